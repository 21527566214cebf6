"""The 8-bit key/value cache, its attention and the log probabilities in
float64 from their definitions, on the CPU, with the error bounds that the
tests of the kernels use."""
from __future__ import annotations

import torch

D = 128
LOG2E = 1.4426950408889634


class Cache:
    """A paged cache on the CPU: codes int8 [pages][kv][page][128], scales
    float32 [pages][kv], for keys (0) and values (1)."""

    def __init__(self, pages, page, kv_heads, table):
        self.page, self.kv = page, kv_heads
        self.codes = [torch.full((pages, kv_heads, page, D), 77, dtype=torch.int8) for _ in range(2)]
        self.scales = [torch.full((pages, kv_heads), float("nan")) for _ in range(2)]
        self.table = table

    def tokens(self, which, seq, begin, end):
        """float64 values of tokens [begin, end) of a sequence, [kv][tokens][128]."""
        pos = torch.arange(begin, end)
        at = self.table[seq].long()[pos // self.page]
        c = self.codes[which][at, :, pos % self.page].double()
        return (c * self.scales[which][at].double()[..., None]).transpose(0, 1)

    def write(self, which, seq, start, x):
        """float32 step by step as the header states it; x: half [n][kv][128]."""
        n, done = x.shape[0], 0
        while done < n:
            t = start + done
            page, slot = int(self.table[seq, t // self.page]), t % self.page
            m = min(self.page - slot, n - done)
            part = x[done:done + m].float()
            codes, scales = self.codes[which][page], self.scales[which][page]
            for h in range(self.kv):
                amax = part[:, h].abs().amax()
                need = amax * torch.tensor(1 / 127, dtype=torch.float32)
                old = scales[h].clone() if slot else torch.tensor(0.0)
                new = torch.maximum(need, old)  # keeps a NaN
                if not torch.isfinite(amax) or not torch.isfinite(old):
                    new = torch.tensor(float("nan"))
                scales[h] = new
                if torch.isnan(new):
                    continue
                if slot and new > old:
                    codes[h, :slot] = (codes[h, :slot].float() * (old / new)).round().to(torch.int8)
                inverse = 1.0 / new if new > 0 else torch.tensor(0.0)
                codes[h, slot:slot + m] = (part[:, h] * inverse).round().clamp(-127, 127).to(torch.int8)
            done += m


def attention(q, k, v, k_scales, v_scales, seen, scale):
    """One head: q [n][128], k / v [length][128] float64 values, *_scales
    [length]; row i sees its first seen[i] tokens.  Returns the output and
    a bound on the error of one that rounds a probability (times the value
    scale, relative to the row's largest) to half, and the output to half.

    Rounding to half is off by 2^-11 of the value, and by 2^-25 of the
    row's largest where it is subnormal.  A score is a float32 sum of 128
    exact products (a code has 7 bits, a half 11): off by at most 128 * 2^-23
    of the sum of their magnitudes.  Its factor is rounded three times, the
    exponent t and its difference to the maximum twice more, each by 2^-24 of
    |t|: 2^-21 |t|.  log2 of a value scale (below 2^5) and the exponential
    (2^-22) add less than 2^-17."""
    n, length = q.shape[0], k.shape[0]
    out = torch.zeros(n, D, dtype=torch.float64)
    bound = torch.full((n, D), 2.0 ** -25, dtype=torch.float64)
    if length == 0:
        return out, bound
    z = q @ k.T * scale
    mass = (q.abs() @ k.abs().T * scale).nan_to_num(0, 0, 0)
    hidden = torch.arange(length) >= seen[:, None]
    z = z.masked_fill(hidden, -torch.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    off = 128 * 2.0 ** -23 * mass.masked_fill(hidden, 0).amax(-1, keepdim=True) + 2.0 ** -17
    off = off + 2.0 ** -21 * LOG2E * z.masked_fill(hidden, 0).abs().amax(-1, keepdim=True)
    spread = p @ v.abs()
    # 2^-25 of the largest p * scale for every token seen, in codes.
    largest = (p * v_scales).amax(-1, keepdim=True)
    codes = torch.where(v_scales > 0, 1 / v_scales.clamp(min=1e-300), 0.0)[:, None] * v.abs()
    tiny = 2.0 ** -25 * largest * ((~hidden).double() @ codes)
    bound = spread * (2.0 ** -11 + 2 * off) + out.abs() * (2.0 ** -11 + off) + tiny + 2.0 ** -25
    return out, bound


def logprobs(x, target, k):
    """One row in float64: (logprob, rank, entropy, top ids, top logprobs)."""
    x = x.double()
    vocab = x.numel()
    nan = float("nan")
    if torch.isnan(x).any() or (x == torch.inf).any() or (x == -torch.inf).all():
        return nan, -1, nan, [-1] * k, [nan] * k
    logp = torch.log_softmax(x, 0)
    p = logp.exp()
    entropy = float(-torch.where(p > 0, p * logp, 0.0).sum())
    order = torch.sort(x, descending=True, stable=True).indices[:k]
    if target < 0 or target >= vocab:
        return 0.0, -1, entropy, order.tolist(), logp[order].tolist()
    rank = int((x > x[target]).sum() + (x[:target] == x[target]).sum())
    return float(logp[target]), rank, entropy, order.tolist(), logp[order].tolist()
