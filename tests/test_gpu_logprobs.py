"""ov_token_logprobs on the B200 against float64 (tests/cache_reference.py)."""
from __future__ import annotations

import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from cache_reference import logprobs  # noqa: E402
from omnivoice_b200 import _native as N  # noqa: E402

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def device_errors():
    flags = ctypes.c_uint32()
    N.check(N.lib().ov_take_device_errors(ctypes.byref(flags), stream()))
    return flags.value


@pytest.fixture(autouse=True)
def _gpu(cuda_device, native):
    yield
    torch.cuda.synchronize()
    assert device_errors() == 0


def run(x, codebooks, vocab, targets, k, entropy=True, rank=True):
    """x: [rows][ld] on the device; targets [codebooks][rows]."""
    rows = x.shape[0]
    t = targets.to(torch.int32).cuda()
    out = {"logprob": torch.full((codebooks, rows), 9.0, device="cuda"),
           "entropy": torch.full((codebooks, rows), 9.0, device="cuda"),
           "rank": torch.full((codebooks, rows), 9, dtype=torch.int32, device="cuda"),
           "ids": torch.full((codebooks, rows, k), 9, dtype=torch.int32, device="cuda"),
           "tops": torch.full((codebooks, rows, k), 9.0, device="cuda")}
    N.check(N.lib().ov_token_logprobs(
        x.data_ptr(), N.OV_LOGITS_F16 if x.dtype == torch.float16 else N.OV_LOGITS_F32,
        x.stride(0), rows, codebooks, vocab, t.data_ptr(), k, out["logprob"].data_ptr(),
        out["entropy"].data_ptr() if entropy else None, out["rank"].data_ptr() if rank else None,
        out["ids"].data_ptr() if k else None, out["tops"].data_ptr() if k else None, stream()))
    torch.cuda.synchronize()
    return {n: v.cpu() for n, v in out.items()}


def check(x, codebooks, vocab, targets, k):
    """x: [rows][>= codebooks * vocab] on the CPU.

    The kernel's float32 error: the exponential's (2^-22, and its argument,
    rounded three times, by up to 1.5 * 2^-23 * |d| for a term e^d whose |d|
    weighs |d| e^d <= 1/e) and a sum of at most 66 terms for a lane or, in
    sums of 4 or 8 values first, vocab / 1024 + 20 for a thread, each off by
    2^-24: a relative error of Z below (vocab / 512 + 200) * 2^-24 + 2^-21.  A log probability adds the
    roundings of x - m, log Z and their difference, 2^-22 of |x - m| + log Z;
    the entropy's sum of e^d d has Z's relative error with |d| up to about
    its own size on top."""
    got = run(x.cuda(), codebooks, vocab, targets, k)
    rel = (vocab / 512 + 200) * 2.0 ** -24 + 2.0 ** -21
    for c in range(codebooks):
        for r in range(x.shape[0]):
            row = x[r, c * vocab:(c + 1) * vocab]
            lp, rank, entropy, ids, tops = logprobs(row, int(targets[c, r]), k)
            at = f"codebook {c}, row {r}"
            assert got["rank"][c, r] == rank, at
            assert got["ids"][c, r].tolist() == ids, at
            span = math.log(vocab) + 1
            for mine, true in [(float(got["logprob"][c, r]), lp),
                               *zip(got["tops"][c, r].tolist(), tops)]:
                if math.isnan(true) or math.isinf(true):
                    assert math.isnan(mine) == math.isnan(true) and (math.isnan(true) or mine == true), at
                else:
                    assert abs(mine - true) <= rel + (abs(true) + span) * 2.0 ** -22, (at, mine, true)
            mine = float(got["entropy"][c, r])
            if math.isnan(entropy):
                assert math.isnan(mine), at
            else:
                assert abs(mine - entropy) <= (2 * rel + 2.0 ** -21) * (2 * span + abs(entropy)), (at, mine, entropy)
    return got


def some_targets(x, codebooks, vocab, g):
    return torch.randint(0, vocab, (codebooks, x.shape[0]), generator=g)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,codebooks,vocab,k", [
    (1, 1, 1, 1), (3, 2, 2, 0), (5, 1, 31, 31), (9, 3, 33, 32), (7, 8, 1025, 5), (20, 1, 1056, 20),
    (4, 8, 1057, 32), (3, 2, 2112, 1), (2, 1, 2113, 32), (6, 3, 4099, 8), (2, 1, 8193, 20),
    (1, 2, 16385, 32), (1, 1, 1 << 20, 32), (2, 1, 30000, 0), (1, 1, 151936, 20), (40, 1, 20011, 5)])
def test_random_rows(rows, codebooks, vocab, k, half):
    """Rows at odd offsets; few rows of a long vocabulary share clusters."""
    g = torch.Generator().manual_seed(rows * vocab)
    x = torch.randn(rows, codebooks * vocab + 3, generator=g) * 3
    x[:, codebooks * vocab:] = float("nan")  # padding columns
    check(x.half() if half else x, codebooks, vocab, some_targets(x, codebooks, vocab, g), k)


@pytest.mark.parametrize("vocab", [1025, 2000, 5000, 40000])
@pytest.mark.parametrize("kind", ["constant", "rising", "falling", "two values", "few open",
                                  "one open", "spike", "crowded thread", "wide", "signed zeros"])
def test_rows_that_crowd_the_alternatives(vocab, kind):
    """Ties, sorted rows and closed tokens, where a threshold keeps
    too much or too little."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.zeros(2, vocab)
    j = torch.arange(vocab).float()
    if kind == "constant":
        x += 1.5
    elif kind == "rising":
        x += j * 0.001
    elif kind == "falling":
        x -= j * 0.001
    elif kind == "two values":
        x += (torch.rand(2, vocab, generator=g) < 0.3).float()
    elif kind == "few open":
        x.fill_(-math.inf)
        x[0, [5, vocab - 2, vocab // 2]] = torch.tensor([1.0, 3.0, 1.0])
        x[1, vocab - 1] = -2.0
    elif kind == "one open":
        x.fill_(-math.inf)
        x[:, vocab // 3] = 1e30
    elif kind == "spike":
        x = torch.randn(2, vocab, generator=g)
        x[0, vocab - 1] = 200.0
    elif kind == "crowded thread":  # one thread's vectors hold all the large values
        x = torch.randn(2, vocab, generator=g)
        x[:, 100:140] += 50
    elif kind == "wide":
        x = torch.randn(2, vocab, generator=g) * 1e4
    else:
        x = torch.where(torch.rand(2, vocab, generator=g) < 0.5, -0.0, 0.0)
    targets = torch.tensor([[vocab // 3, vocab - 1]])
    for k in (1, 20, 32):
        check(x, 1, vocab, targets, k)
        if kind != "one open" and kind != "wide":
            check(x.half(), 1, vocab, targets, k)


@pytest.mark.parametrize("vocab", [1025, 5000, 30000])
@pytest.mark.parametrize("half", [False, True])
def test_masks_of_the_types_lowest_value(vocab, half):
    """Closed with the lowest finite value instead of -inf: no probability
    (beside an open token), but a value of its own; and rows of it alone."""
    g = torch.Generator().manual_seed(vocab)
    t = torch.float16 if half else torch.float32
    lowest = torch.finfo(t).min
    x = torch.randn(5, vocab, generator=g).to(t)
    x[0, ::2] = lowest
    x[1] = lowest
    x[2] = lowest
    x[2, vocab // 2] = 3.0
    x[3] = -math.inf
    x[3, 5::7] = lowest
    x[4, 3::5] = lowest
    x[4, 1::5] = -math.inf
    targets = torch.tensor([[2, 5, vocab // 2, 12, 1]])
    got = run(x.cuda(), 1, vocab, targets, 9)
    for r in range(5):
        lp, rank, entropy, ids, tops = logprobs(x[r], int(targets[0, r]), 9)
        assert got["rank"][0, r] == rank and got["ids"][0, r].tolist() == ids
        for mine, true in [(float(got["logprob"][0, r]), lp), *zip(got["tops"][0, r].tolist(), tops)]:
            # A sum of equal terms as large as their logarithm's rounding.
            assert mine == true or abs(mine - true) <= 2e-5 + abs(true) * 2.0 ** -21
        assert abs(float(got["entropy"][0, r]) - entropy) <= 1e-4


@pytest.mark.parametrize("vocab", [100, 1025, 5000, 30000])
def test_rows_without_a_distribution(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(6, vocab, generator=g)
    x[0, vocab - 1] = float("nan")
    x[1, 3] = math.inf
    x[2] = -math.inf
    x[3, 0] = float("nan")
    x[3, 1] = math.inf
    x[4] = float("nan")
    got = check(x, 1, vocab, torch.zeros(1, 6, dtype=torch.long), 7)
    assert got["logprob"][0, :5].isnan().all() and not got["logprob"][0, 5].isnan()


@pytest.mark.parametrize("vocab", [1025, 5000])
def test_targets_that_ask_for_nothing_and_closed_ones(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(5, vocab, generator=g)
    x[:, ::3] = -math.inf
    targets = torch.tensor([[-1, -2 ** 31, 9, 10, 0]])
    got = check(x, 1, vocab, targets, 4)
    assert got["logprob"][0, :2].tolist() == [0, 0] and got["logprob"][0, 2] == -math.inf
    got = run(x.cuda(), 1, vocab, torch.tensor([[vocab, 2 ** 31 - 1, 10, 10, 10]]), 4)
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
    assert got["logprob"][0, :2].tolist() == [0, 0] and got["rank"][0, :2].tolist() == [-1, -1]


@pytest.mark.parametrize("vocab", [1025, 5000])
def test_outputs_that_are_not_asked_for_stay(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(4, vocab, generator=g).cuda()
    targets = torch.full((1, 4), 7)
    full = run(x, 1, vocab, targets, 5)
    bare = run(x, 1, vocab, targets, 0, entropy=False, rank=False)
    assert torch.equal(full["logprob"], bare["logprob"])
    assert (bare["entropy"] == 9).all() and (bare["rank"] == 9).all()


def test_large_rows_offset():
    """A row stride that puts the last rows past 2^32 bytes."""
    ld = 1 << 28
    x = torch.empty(5, ld, device="cuda")
    g = torch.Generator().manual_seed(1)
    for vocab in (1025, 9000):
        part = torch.randn(5, vocab, generator=g)
        x[:, :vocab] = part.cuda()
        t = torch.full((1, 5), 11)
        got = run(x, 1, vocab, t, 6)
        want = run(part.cuda(), 1, vocab, t, 6)
        assert all(torch.equal(got[n], want[n]) for n in got)


def test_log_probabilities_of_a_generation_step():
    """The audio head's product through the GEMM, its row padding, and the
    codes' log probabilities, as a caller scores generated codes."""
    g = torch.Generator().manual_seed(2)
    frames, codebooks, vocab, width = 24, 8, 1025, 256
    hidden = torch.randn(frames, width, generator=g).half()
    head = (torch.randn(codebooks * vocab, width, generator=g) * 0.05).half()
    ld = 8224
    h, w = hidden.cuda(), head.cuda()
    logits = torch.empty(frames, ld, device="cuda")
    N.check(N.lib().ov_gemm_f16(h.data_ptr(), width, w.data_ptr(), logits.data_ptr(), ld, frames,
                                width, codebooks * vocab, N.OV_EPI_STORE_F32, None, None, 0, stream()))
    torch.cuda.synchronize()
    check(logits[:, :codebooks * vocab].cpu(), codebooks, vocab,
          torch.randint(0, 1024, (codebooks, frames), generator=g), 5)
