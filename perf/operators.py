"""The 8-bit key/value cache, the attention that reads it and the log
probabilities of chosen tokens, in their plain form and through the library.

Three paths:

  cache     rows of keys and values are quantised into the pages of a cache
            (int8, one float32 scale for each page and head) and the pages
            they touched are read back as float16; with nothing to write,
            whole sequences are read back;
  attend    grouped-query attention of each sequence's rows over its cache;
  logprobs  log probability and rank of a given token, entropy of its row and
            the most likely alternatives, for rows of logits.

`run` computes them with elementary torch operations in float32, or, where
`own` is true, with the library's entry points.  `exact` states them again in
float64 from their definitions.
"""
import ctypes
import math

import torch

own = False

HEAD_DIM = 128


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One token of one utterance appended inside a page: the latency of a step.
        cache_case("append 1 token", seqs=1, start=619, new=1, page=64),
        # The prompts (text and reference voice) of a batch of 64 utterances.
        cache_case("write 64 prompts", seqs=64, start=0, new=1500, page=64, ragged=True),
        # Blocks of a long recording, behind what is there already, odd starts.
        cache_case("write 16 x 8191 tokens", seqs=16, start=1001, new=8191, page=128),
        # A batch's sequences handed back in float16, small pages.
        cache_case("read 64 sequences", seqs=64, start=2175, new=0, page=16, ragged=True),
        # One token of one utterance over its prompt.
        attend_case("1 token over 705", seqs=1, new=1, length=705, page=64, causal=True),
        # One token for each utterance of a batch, ragged lengths.
        attend_case("64 x 1 token, ragged", seqs=64, new=1, length=4096, page=64, causal=True,
                    ragged=True),
        # One token of few sequences with long histories, eight query heads for each key head.
        attend_case("4 x 1 token over 65537", seqs=4, new=1, length=65537, page=128, heads=16,
                    kv_heads=2, causal=True),
        # The target frames of one utterance over its prompt and themselves, both directions.
        attend_case("375 frames over 705", seqs=1, new=375, length=705, page=64, causal=False),
        # A batch of long prompts in one pass.
        attend_case("16 x 2175 rows", seqs=16, new=2175, length=2175, page=64, causal=True,
                    ragged=True),
        # The audio head: eight codebooks for each frame of a 10 s utterance, both branches.
        logprobs_case("audio head, 500 rows", rows=500, codebooks=8, vocab=1025, top_k=5),
        # One row over the text vocabulary.
        logprobs_case("text head, 1 row", rows=1, codebooks=1, vocab=151936, top_k=20),
        # A batch of rows over the text vocabulary, half-precision logits.
        logprobs_case("text head, 512 rows, f16", rows=512, codebooks=1, vocab=151936, top_k=20,
                      half=True),
    ]


def cache_case(name, seqs, start, new, page, kv_heads=8, ragged=False):
    return dict(name=name, op="cache", seqs=seqs, start=start, new=new, page=page,
                kv_heads=kv_heads, ragged=ragged)


def attend_case(name, seqs, new, length, page, heads=16, kv_heads=8, causal=True, ragged=False):
    return dict(name=name, op="attend", seqs=seqs, new=new, length=length, page=page, heads=heads,
                kv_heads=kv_heads, causal=causal, ragged=ragged)


def logprobs_case(name, rows, codebooks, vocab, top_k, half=False):
    return dict(name=name, op="logprobs", rows=rows, codebooks=codebooks, vocab=vocab,
                top_k=top_k, half=half)


def log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ranges, no dearer than the dearest listed one."""
    op = rng.choice(["cache", "cache", "attend", "attend", "attend", "logprobs", "logprobs"])
    page = rng.choice([16, 32, 64, 128])
    if op == "cache":
        seqs, kv_heads = log_uniform(rng, 1, 64), rng.choice([1, 2, 4, 8])
        most = min(8191, 120_000 // seqs)
        new = rng.choice([0, 1, log_uniform(rng, 2, most), log_uniform(rng, 2, most)])
        case = cache_case("", seqs, log_uniform(rng, 1, min(2500, most)), new, page, kv_heads,
                          rng.random() < 0.5)
    elif op == "attend":
        heads, kv_heads = rng.choice([(16, 8), (16, 16), (16, 2), (8, 1), (12, 4), (10, 2)])
        seqs = log_uniform(rng, 1, 64)
        length = log_uniform(rng, 1, min(65537, 200_000 // seqs))
        # Scores of the plain form stay under 1.2e9 values.
        most = max(1, min(length, 2175, int(1.2e9 / (seqs * heads * length))))
        new = rng.choice([1, 1, log_uniform(rng, 1, most), log_uniform(rng, 1, most)])
        case = attend_case("", seqs, new, length, page, heads, kv_heads, rng.random() < 0.7,
                           rng.random() < 0.5)
    elif rng.random() < 0.5:
        case = logprobs_case("", log_uniform(rng, 1, 4000), 8, rng.randint(500, 2100),
                             rng.randint(0, 32), rng.random() < 0.5)
    else:
        vocab = log_uniform(rng, 3000, 200_000)
        case = logprobs_case("", log_uniform(rng, 1, min(4000, 60_000_000 // vocab)), 1, vocab,
                             rng.randint(0, 32), rng.random() < 0.5)
    del case["name"]
    return case


def spread(count, most, least, ragged, step):
    """`count` whole numbers of [least, most], the first the largest; even steps of an irrational
    fraction stand for a ragged batch."""
    if not ragged:
        return [most] * count
    return [max(least, most - int((most - least) * ((i * step) % 1.0))) for i in range(count)]


def extents(case):
    """(tokens in the cache before, rows given) of each sequence."""
    n = case["seqs"]
    if case["op"] == "cache":
        starts = spread(n, case["start"], case["start"] // 4, case["ragged"], 0.6180339887)
        return starts, spread(n, case["new"], case["new"] // 8, case["ragged"], 0.4142135623)
    lengths = spread(n, case["length"], max(1, case["length"] // 8), case["ragged"], 0.6180339887)
    rows = spread(n, case["new"], max(1, case["new"] // 4), case["ragged"], 0.4142135623)
    rows = [min(a, b) for a, b in zip(rows, lengths)]
    return [a - b for a, b in zip(lengths, rows)], rows


def work(case):
    if case["op"] == "cache":
        starts, rows = extents(case)
        token = 2 * case["kv_heads"] * HEAD_DIM  # key and value elements of a token
        new = sum(rows)
        back = new + sum(s % case["page"] if n else 0 for s, n in zip(starts, rows))
        if case["new"] == 0:
            return {"bytes": sum(starts) * token * 3, "flops": sum(starts) * token}
        return {"bytes": new * token * 3 + back * token * 3, "flops": new * token * 3 + back * token}
    if case["op"] == "attend":
        starts, rows = extents(case)
        tokens = sum(starts) + sum(rows)
        pairs = sum(n * s + (n * (n + 1) // 2 if case["causal"] else n * n)
                    for s, n in zip(starts, rows))
        return {"bytes": 2 * tokens * case["kv_heads"] * HEAD_DIM
                + 4 * sum(rows) * case["heads"] * HEAD_DIM,
                "flops": 4 * pairs * case["heads"] * HEAD_DIM}
    items = case["rows"] * case["codebooks"]
    return {"bytes": items * (case["vocab"] * (2 if case["half"] else 4) + 16 + 8 * case["top_k"]),
            "flops": items * case["vocab"] * 6}


# ---------------------------------------------------------------- the inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return prepare_logprobs(case, g) if case["op"] == "logprobs" else prepare_cache(case, g)


def prepare_cache(case, g):
    """A cache whose pages lie in no order, with what was written before, and
    the rows of this call as columns of one projection (queries, keys,
    values), as the generator lays them out."""
    starts, rows = extents(case)
    page, kv_heads, seqs = case["page"], case["kv_heads"], case["seqs"]
    heads = case.get("heads", kv_heads)
    totals = [a + b for a, b in zip(starts, rows)]
    max_pages = max(-(-t // page) for t in totals)
    pages = seqs * max_pages
    dev = dict(device="cuda")
    table = torch.randperm(pages, generator=g, **dev).to(torch.int32).view(seqs, max_pages)
    shape = (pages, kv_heads, page, HEAD_DIM)
    s = dict(case)

    def codes():  # normal values on a grid of a page's largest (about four deviations)
        out = torch.empty(shape, dtype=torch.int8, **dev)
        flat = out.view(-1)
        for part in flat.split(1 << 28):
            part.copy_((torch.randn(part.numel(), generator=g, **dev) * 31).round_().clamp_(-127, 127))
        return out

    s["keys"], s["values"] = codes(), codes()
    s["key_scales"] = (0.7 + 0.6 * torch.rand(pages, kv_heads, generator=g, **dev)) / 31
    s["value_scales"] = (0.7 + 0.6 * torch.rand(pages, kv_heads, generator=g, **dev)) / 31
    s["table"] = table
    total = sum(rows)
    width = (heads + 2 * kv_heads) * HEAD_DIM
    qkv = torch.randn(max(total, 1), width, generator=g, **dev, dtype=torch.float32).half()
    s["q"] = qkv[:, :heads * HEAD_DIM]
    s["k"] = qkv[:, heads * HEAD_DIM:(heads + kv_heads) * HEAD_DIM]
    s["v"] = qkv[:, (heads + kv_heads) * HEAD_DIM:]
    s["rows"], s["max_rows"] = total, max(rows)
    s["cu"] = cumulative(rows)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, **dev)
    s["lengths"] = torch.tensor(totals, dtype=torch.int32, **dev)
    s["max_length"] = max(totals)
    s["scale"] = HEAD_DIM ** -0.5
    # What is read back: the pages that the new rows touch, or everything.
    if case["op"] == "cache":
        first = [a // page * page if n else a for a, n in zip(starts, rows)]
        back = [t - f for t, f in zip(totals, first)]
        if case["new"] == 0:
            first, back = [0] * seqs, totals
        s["back_cu"], s["back_rows"], s["back_max"] = cumulative(back), sum(back), max(back)
        s["back_starts"] = torch.tensor(first, dtype=torch.int32, **dev)
        s["out_k"] = torch.empty(sum(back), kv_heads * HEAD_DIM, dtype=torch.float16, **dev)
        s["out_v"] = torch.empty_like(s["out_k"])
    else:
        s["out"] = torch.empty(total, heads * HEAD_DIM, dtype=torch.float16, **dev)
    if own:  # the description of the cache and the scratch that a program keeps
        own_handles(s)
    return s


def cumulative(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def prepare_logprobs(case, g):
    """Logits of a head whose mask class and a few others are closed (-inf),
    and the tokens that were taken."""
    rows, codebooks, vocab = case["rows"], case["codebooks"], case["vocab"]
    ld = -(-codebooks * vocab // 32) * 32
    logits = torch.randn(rows, ld, generator=g, device="cuda") * 2.5
    view = logits[:, :codebooks * vocab].view(rows, codebooks, vocab)
    view[..., vocab - 1] = -math.inf
    view[..., 7 % (vocab - 1)::97] = -math.inf
    s = dict(case, ld=ld, logits=logits.half() if case["half"] else logits)
    targets = torch.randint(0, vocab - 1, (codebooks, rows), generator=g, device="cuda")
    # A target is a token that a sampler could take: not a closed one.
    closed = view.transpose(0, 1).gather(2, targets[..., None])[..., 0] == -math.inf
    targets = torch.where(closed, (targets + 1) % (vocab - 1), targets)
    s["targets"] = targets.to(torch.int32)
    k = case["top_k"]
    s["logprob"] = torch.empty(codebooks, rows, device="cuda")
    s["entropy"] = torch.empty(codebooks, rows, device="cuda")
    s["rank"] = torch.empty(codebooks, rows, dtype=torch.int32, device="cuda")
    s["top_ids"] = torch.empty(codebooks, rows, k, dtype=torch.int32, device="cuda")
    s["top_logprobs"] = torch.empty(codebooks, rows, k, device="cuda")
    return s


# ------------------------------------------------------------------ the runs

def run(s):
    if own:
        return own_run(s)
    if s["op"] == "cache":
        return plain_cache(s)
    return plain_attend(s) if s["op"] == "attend" else plain_logprobs(s)


def own_handles(s):
    from omnivoice_b200 import _native as N
    c = N.KvCache(keys=s["keys"].data_ptr(), values=s["values"].data_ptr(),
                  key_scales=s["key_scales"].data_ptr(), value_scales=s["value_scales"].data_ptr(),
                  page_table=s["table"].data_ptr(), pages=s["keys"].shape[0],
                  page_tokens=s["page"], kv_heads=s["kv_heads"], head_dim=HEAD_DIM,
                  num_seqs=s["seqs"], max_pages=s["table"].shape[1])
    s["cache"] = ctypes.byref(c)
    if s["op"] == "attend":
        need = N.lib().ov_attention_kv_cache_workspace_bytes(
            s["cache"], s["rows"], s["max_rows"], s["max_length"], s["heads"])
        s["workspace"] = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")


def own_run(s):
    from omnivoice_b200 import _native as N
    lib, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    if s["op"] == "cache":
        if s["rows"]:
            N.check(lib.ov_kv_cache_write(
                s["cache"], s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(),
                s["v"].stride(0), s["rows"], s["cu"].data_ptr(), s["starts"].data_ptr(),
                s["max_rows"], stream))
        k, v = s["out_k"], s["out_v"]
        N.check(lib.ov_kv_cache_read(
            s["cache"], s["back_cu"].data_ptr(), s["back_starts"].data_ptr(), s["back_rows"],
            s["back_max"], k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), stream))
        return {"k": k, "v": v}
    if s["op"] == "attend":
        q, out, work_ = s["q"], s["out"], s["workspace"]
        N.check(lib.ov_attention_kv_cache(
            s["cache"], q.data_ptr(), q.stride(0), s["rows"], s["cu"].data_ptr(), s["max_rows"],
            s["lengths"].data_ptr(), s["max_length"], s["heads"], int(s["causal"]), s["scale"],
            out.data_ptr(), out.stride(0), work_.data_ptr(), work_.numel(), stream))
        return {"out": out}
    x = s["logits"]
    N.check(lib.ov_token_logprobs(
        x.data_ptr(), N.OV_LOGITS_F16 if s["half"] else N.OV_LOGITS_F32, s["ld"], s["rows"],
        s["codebooks"], s["vocab"], s["targets"].data_ptr(), s["top_k"], s["logprob"].data_ptr(),
        s["entropy"].data_ptr(), s["rank"].data_ptr(), s["top_ids"].data_ptr(),
        s["top_logprobs"].data_ptr(), stream))
    return {n: s[n] for n in ("logprob", "entropy", "rank", "top_ids", "top_logprobs")}


# ----------------------------------------------------------- the plain forms

def row_places(cu, starts, rows):
    """Sequence and position of every packed row."""
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), r.to(torch.int32), right=True)
    return seq, starts.long()[seq] + r - cu.long()[seq]


def plain_cache(s):
    if s["rows"]:
        for x, codes, scales in ((s["k"], s["keys"], s["key_scales"]),
                                 (s["v"], s["values"], s["value_scales"])):
            plain_write(s, x[:s["rows"]], codes, scales)
    seq, pos = row_places(s["back_cu"], s["back_starts"], s["back_rows"])
    page = s["table"].long()[seq, pos // s["page"]]
    slot = pos % s["page"]
    out = {}
    for name, codes, scales in (("k", s["keys"], s["key_scales"]),
                                ("v", s["values"], s["value_scales"])):
        x = codes[page, :, slot].float() * scales[page][..., None]
        out[name] = x.half().flatten(1)
    return out


def plain_write(s, x, codes, scales):
    """One of keys and values: the scale of a page grows to what its largest
    value needs, what a page keeps is put on the new grid, new rows follow."""
    page, kv_heads, table = s["page"], s["kv_heads"], s["table"].long()
    seq, pos = row_places(s["cu"], s["starts"], s["rows"])
    at, slot = table[seq, pos // page], pos % page
    x = x.float().unflatten(1, (kv_heads, HEAD_DIM))
    need = torch.zeros_like(scales).scatter_reduce_(
        0, at[:, None].expand(-1, kv_heads), x.abs().amax(-1) * (1 / 127), "amax")
    starts = s["starts"].long()
    keeps = (starts % page > 0) & (s["cu"][1:] > s["cu"][:-1])
    first = table[torch.arange(s["seqs"], device="cuda"),
                  torch.clamp(starts // page, max=table.shape[1] - 1)]
    old = scales[first]
    new = torch.maximum(need[first], torch.where(keeps[:, None], old, 0.0))
    ratio = torch.where(new > 0, old / new, 0.0)
    held = codes[first].float()
    kept = (torch.arange(page, device="cuda") < (starts % page)[:, None]) & keeps[:, None]
    moved = torch.where(kept[:, None, :, None], (held * ratio[..., None, None]).round(), held)
    codes[first] = moved.to(torch.int8)
    touched = torch.zeros(scales.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, at, True)
    scales.copy_(torch.where(touched[:, None], need, scales))
    scales[first] = torch.where(keeps[:, None], new, scales[first])
    scale = scales[at]
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    codes[at, :, slot] = (x * inverse[..., None]).round().clamp_(-127, 127).to(torch.int8)


def plain_attend(s):
    seqs, heads, kv_heads, page = s["seqs"], s["heads"], s["kv_heads"], s["page"]
    group, n, length = heads // kv_heads, s["max_rows"], s["max_length"]
    j = torch.arange(length, device="cuda")
    at = s["table"].long()[:, j // page]                                # [seqs, length]
    slot = (j % page).expand_as(at)

    def values(codes, scales):                                          # [seqs, kv, length, d]
        return (codes[at, :, slot].float() * scales[at][..., None]).transpose(1, 2)

    count = (s["cu"][1:] - s["cu"][:-1]).long()
    i = torch.arange(n, device="cuda")
    row = torch.clamp(s["cu"][:-1].long()[:, None] + i, max=s["rows"] - 1)
    q = s["q"][row].float().view(seqs, n, kv_heads, group, HEAD_DIM)
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * n, HEAD_DIM)
    scores = torch.matmul(q, values(s["keys"], s["key_scales"]).transpose(2, 3)) * s["scale"]
    lengths = s["lengths"].long()
    last = lengths[:, None] if not s["causal"] else lengths[:, None] - count[:, None] + i + 1
    seen = j < torch.minimum(last, lengths[:, None]).expand(seqs, n)[..., None]
    seen = seen[:, None, None].expand(seqs, 1, group, n, length).reshape(seqs, 1, group * n, length)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, values(s["values"], s["value_scales"]))
    out = out / torch.where(total == 0, 1.0, total)
    out = out.view(seqs, kv_heads, group, n, HEAD_DIM).permute(0, 3, 1, 2, 4)
    seq, pos = row_places(s["cu"], torch.zeros_like(s["starts"]), s["rows"])
    return {"out": out[seq, pos].reshape(s["rows"], heads * HEAD_DIM).half()}


def plain_logprobs(s):
    rows, codebooks, vocab, k = s["rows"], s["codebooks"], s["vocab"], s["top_k"]
    x = s["logits"][:, :codebooks * vocab].unflatten(1, (codebooks, vocab)).transpose(0, 1).float()
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    shifted = torch.where(e > 0, x - top, 0.0)
    entropy = total.log() - (e * shifted).sum(-1, keepdim=True) / total
    lse = top + total.log()
    t = s["targets"].long()[..., None]
    taken = x.gather(2, t)
    index = torch.arange(vocab, device="cuda")
    rank = ((x > taken) | ((x == taken) & (index < t))).sum(-1)
    # One key orders by value and, where values are equal, by the lower index.
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + ((1 << 20) - 1 - index)
    ids = (1 << 20) - 1 - (key.topk(k, dim=-1).values & ((1 << 20) - 1))
    return {"logprob": (taken - lse)[..., 0], "entropy": entropy[..., 0],
            "rank": rank.to(torch.int32), "top_ids": ids.to(torch.int32),
            "top_logprobs": x.gather(2, ids) - lse}


# ------------------------------------------------- the definitions in float64

def exact(case, seed):
    s = prepare(case, seed)
    return {"cache": exact_cache, "attend": exact_attend, "logprobs": exact_logprobs}[s["op"]](s)


def history(s, codes, scales, i, length):
    """The first `length` tokens that sequence i's pages stand for, [kv][length][d]."""
    pages = s["table"][i, :-(-length // s["page"])].long()
    x = codes[pages].double() * scales[pages].double()[..., None, None]
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


def exact_cache(s):
    cu, starts = s["cu"].tolist(), s["starts"].tolist()
    back_cu, back_starts = s["back_cu"].tolist(), s["back_starts"].tolist()
    page, kv_heads = s["page"], s["kv_heads"]
    out = {}
    for name, codes, scales in (("k", s["keys"], s["key_scales"]),
                                ("v", s["values"], s["value_scales"])):
        parts = []
        for i in range(s["seqs"]):
            n, start = cu[i + 1] - cu[i], starts[i]
            begin, end = back_starts[i], back_starts[i] + back_cu[i + 1] - back_cu[i]
            if n == 0:
                parts.append(history(s, codes, scales, i, end)[:, begin:].transpose(0, 1).flatten(1))
                continue
            x = s[name][cu[i]:cu[i + 1]].double().unflatten(1, (kv_heads, HEAD_DIM)).transpose(0, 1)
            kept = start - begin
            first = s["table"][i, start // page].long()
            held = codes[first].double()[:, :kept]
            blank = torch.zeros(kv_heads, -(end - begin) % page, HEAD_DIM, device="cuda",
                                dtype=torch.float64)
            rows = torch.cat([torch.zeros_like(held), x, blank], 1)
            rows = rows.unflatten(1, (-1, page))                        # [kv, pages, page, d]
            step = rows.abs().amax((2, 3)) / 127
            if kept:
                step[:, 0] = torch.maximum(step[:, 0], scales[first].double())
            grid = step[..., None, None]
            rows = torch.where(grid > 0, torch.round(rows / grid.clamp(min=1e-300)), 0.0) * grid
            rows = rows.flatten(1, 2)[:, :end - begin]
            if kept:
                old = scales[first].double()[:, None, None]
                rows[:, :kept] = torch.round(held * old / grid[:, 0]) * grid[:, 0]
            parts.append(rows.transpose(0, 1).flatten(1))
        out[name] = torch.cat(parts)
    return out


def exact_attend(s):
    cu, lengths, kv_heads = s["cu"].tolist(), s["lengths"].tolist(), s["kv_heads"]
    group = s["heads"] // kv_heads
    out = torch.zeros(s["rows"], s["heads"], HEAD_DIM, dtype=torch.float64, device="cuda")
    for i in range(s["seqs"]):
        n, length = cu[i + 1] - cu[i], lengths[i]
        k = history(s, s["keys"], s["key_scales"], i, length)
        v = history(s, s["values"], s["value_scales"], i, length)
        q = s["q"][cu[i]:cu[i + 1]].double().view(n, s["heads"], HEAD_DIM)
        hidden = None
        if s["causal"]:
            position = torch.arange(length - n, length, device="cuda")
            hidden = torch.arange(length, device="cuda") > position[:, None]
        for h in range(s["heads"]):
            z = q[:, h] @ k[h // group].T * s["scale"]
            if hidden is not None:
                z = z.masked_fill(hidden, -math.inf)
            out[cu[i]:cu[i + 1], h] = torch.softmax(z, -1) @ v[h // group]
    return {"out": out.flatten(1)}


def exact_logprobs(s):
    codebooks, vocab, k = s["codebooks"], s["vocab"], s["top_k"]
    names = ("logprob", "entropy", "top_logprobs")
    parts = {n: [] for n in names}
    for c in range(codebooks):
        by_rows = {n: [] for n in names}
        for at in torch.arange(s["rows"], device="cuda").split(max(1, 40_000_000 // vocab)):
            x = s["logits"][at][:, c * vocab:(c + 1) * vocab].double()
            logp = torch.log_softmax(x, -1)
            p = logp.exp()
            by_rows["logprob"].append(logp.gather(1, s["targets"][c, at].long()[:, None])[:, 0])
            by_rows["entropy"].append(-torch.where(p > 0, p * logp, 0.0).sum(-1))
            by_rows["top_logprobs"].append(logp.topk(k, -1).values)
        for n in names:
            parts[n].append(torch.cat(by_rows[n]))
    # Ranks and indices are whole numbers: the plain form's are exact.
    return {**{n: torch.stack(parts[n]) for n in names}, "rank": None, "top_ids": None}
