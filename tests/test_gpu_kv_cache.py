"""The paged 8-bit key/value cache and the attention over it on the B200,
through the C-ABI, against tests/cache_reference.py."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

from cache_reference import Cache, D, attention  # noqa: E402
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


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cumulative(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


class GpuCache:
    """The device copy of a reference cache."""

    def __init__(self, ref):
        self.codes = [c.cuda() for c in ref.codes]
        self.scales = [s.cuda() for s in ref.scales]
        self.table = ref.table.to(torch.int32).cuda()
        pages, kv, page, _ = ref.codes[0].shape
        self.desc = N.KvCache(
            keys=self.codes[0].data_ptr(), values=self.codes[1].data_ptr(),
            key_scales=self.scales[0].data_ptr(), value_scales=self.scales[1].data_ptr(),
            page_table=self.table.data_ptr(), pages=pages, page_tokens=page, kv_heads=kv,
            head_dim=D, num_seqs=self.table.shape[0], max_pages=self.table.shape[1])
        self.keep = []

    def write(self, k, v, counts, starts, max_rows=None):
        """k, v: half [rows][>= kv * 128], on the device."""
        cu, st = i32(cumulative(counts)), i32(starts)
        self.keep = [k, v, cu, st]
        N.check(N.lib().ov_kv_cache_write(
            ctypes.byref(self.desc), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
            k.shape[0], cu.data_ptr(), st.data_ptr(),
            max(counts) if max_rows is None else max_rows, stream()))

    def read(self, counts, starts, rows=None, max_rows=None, ld=None, fill=0.0):
        rows = sum(counts) if rows is None else rows
        width = self.desc.kv_heads * D
        k = torch.full((rows, ld or width), fill, dtype=torch.float16, device="cuda")
        v = torch.full_like(k, fill)
        cu, st = i32(cumulative(counts)), i32(starts)
        N.check(N.lib().ov_kv_cache_read(
            ctypes.byref(self.desc), cu.data_ptr(), st.data_ptr(), rows,
            max(counts) if max_rows is None else max_rows, k.data_ptr(), k.stride(0), v.data_ptr(),
            v.stride(0), stream()))
        torch.cuda.synchronize()
        return k, v

    def workspace(self, rows, max_rows, max_length, heads):
        need = N.lib().ov_attention_kv_cache_workspace_bytes(
            ctypes.byref(self.desc), rows, max_rows, max_length, heads)
        return torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")

    def attend(self, q, counts, lengths, heads, causal, scale, out, workspace=None, max_rows=None,
               max_length=None, on=None):
        cu, ln = i32(cumulative(counts)), i32(lengths)
        self.keep = [q, cu, ln]
        N.check(N.lib().ov_attention_kv_cache(
            ctypes.byref(self.desc), q.data_ptr(), q.stride(0), q.shape[0], cu.data_ptr(),
            max(counts) if max_rows is None else max_rows, ln.data_ptr(),
            max(lengths) if max_length is None else max_length, heads, int(causal), scale,
            out.data_ptr(), out.stride(0), workspace.data_ptr() if workspace is not None else None,
            workspace.numel() if workspace is not None else 0, stream() if on is None else on))
        return out


def shuffled_table(seqs, max_pages, extra, g):
    return torch.randperm(seqs * max_pages + extra, generator=g)[:seqs * max_pages].view(seqs, max_pages)


def same_cache(ref, gpu):
    torch.cuda.synchronize()
    for which in range(2):
        assert torch.equal(ref.codes[which], gpu.codes[which].cpu())
        a, b = ref.scales[which], gpu.scales[which].cpu()
        assert torch.equal(a.nan_to_num(-7.0), b.nan_to_num(-7.0))


# ------------------------------------------------------- writing and reading

@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv", [1, 3, 8])
def test_writes_in_pieces_match_the_definition(page, kv):
    """Ragged writes behind one another (a prompt, single tokens, blocks that
    end inside pages, nothing) give the same codes and scales as the float32
    definition, bit for bit, and leave every other slot as it was; what is
    read back is the half of code * scale, and near what was written."""
    g = torch.Generator().manual_seed(page + kv)
    seqs, max_pages = 4, 6
    ref = Cache(seqs * max_pages + 3, page, kv, shuffled_table(seqs, max_pages, 3, g))
    gpu = GpuCache(ref)
    lengths = [0] * seqs
    written = [[torch.zeros(0, kv, D) for _ in range(seqs)] for _ in range(2)]
    for step, counts in enumerate([[page + 3, 1, 0, 2 * page], [1, 1, 1, 1], [0, page - 2, 5, 1],
                                   [7, 0, page, 3], [1, 2, 3, page // 2]]):
        rows = sum(counts) + 2  # two rows behind the last sequence
        x = torch.randn(rows, 2 * kv * D + 8, generator=g) * 2.0 ** (step - 2)
        x[sum(counts):] = float("nan")
        x = x.half()
        d = x.cuda()
        gpu.write(d[:, :kv * D], d[:, kv * D:2 * kv * D], counts, lengths)
        at = 0
        for s, n in enumerate(counts):
            for which in range(2):
                part = x[at:at + n, which * kv * D:(which + 1) * kv * D].view(n, kv, D)
                ref.write(which, s, lengths[s], part)
                written[which][s] = torch.cat([written[which][s], part.float()])
            at += n
            lengths[s] += n
        same_cache(ref, gpu)
    got = gpu.read(lengths, [0] * seqs)
    at = 0
    for s, n in enumerate(lengths):
        for which in range(2):
            value = got[which][at:at + n].cpu().view(n, kv, D)
            pos = torch.arange(n)
            pages = ref.table[s][pos // page]
            want = (ref.codes[which][pages, :, pos % page].float() * ref.scales[which][pages][..., None]).half()
            assert torch.equal(value, want)
            # Half a scale for each of at most five roundings (the first and
            # one for each later write), none on a coarser grid than the last.
            scale = ref.scales[which][pages][..., None].double()
            off = (value.double() - written[which][s].double()).abs()
            assert (off <= 2.5 * scale * (1 + 2.0 ** -20) + value.double().abs() * 2.0 ** -11 + 2.0 ** -25).all()
        at += n


def test_rewriting_a_tail_and_a_page_from_its_start():
    """A start below the current end drops what was behind it; a page that is
    rewritten from its first slot gets a new scale, a smaller one too."""
    g = torch.Generator().manual_seed(3)
    ref = Cache(5, 16, 2, torch.tensor([[4, 1, 0]]))
    gpu = GpuCache(ref)
    for start, n, size in [(0, 40, 4.0), (20, 6, 1.0), (16, 16, 0.01), (10, 7, 0.5)]:
        x = (torch.randn(n, 4 * D, generator=g) * size).half()
        d = x.cuda()
        gpu.write(d[:, :2 * D], d[:, 2 * D:], [n], [start])
        for which in range(2):
            ref.write(which, 0, start, x[:, which * 2 * D:(which + 1) * 2 * D].view(n, 2, D))
        same_cache(ref, gpu)


def test_extreme_values():
    """Zeros, the least and greatest halves, and pages with NaN or infinity:
    those read back as NaN, also after more was written behind, until the
    page is rewritten from its start."""
    ref = Cache(6, 16, 1, torch.arange(6).view(1, 6))
    gpu = GpuCache(ref)
    x = torch.zeros(96, D, dtype=torch.float16)
    x[16:32] = 5.960464477539063e-08
    x[32:48, ::2] = 65504.0
    x[32:48, 1::2] = -65504.0
    x[50, 5] = float("nan")
    x[70, 9] = float("-inf")
    d = x.cuda()
    gpu.write(d, d, [88], [0])
    for which in range(2):
        ref.write(which, 0, 0, x[:88].view(88, 1, D))
    same_scale = [s.isnan().flatten().tolist() for s in ref.scales]
    assert same_scale[0] == [False, False, False, True, True, False]
    k, v = gpu.read([88], [0])
    for got in (k.cpu(), v.cpu()):
        assert torch.equal(got[:48], x[:48])
        assert got[48:80].isnan().all()
        assert torch.equal(got[80:88], x[80:88])
    gpu.write(d[:3], d[:3], [3], [60])  # behind the NaN, in its page
    assert gpu.read([16], [48])[0][:15].isnan().all()
    gpu.write(d[32:48], d[32:48], [16], [48])
    assert torch.equal(gpu.read([16], [48])[0].cpu(), x[32:48])


def test_reading_leaves_other_rows_and_columns():
    g = torch.Generator().manual_seed(5)
    ref = Cache(8, 32, 2, shuffled_table(2, 4, 0, g))
    gpu = GpuCache(ref)
    x = torch.randn(70, 2 * D, generator=g).half()
    gpu.write(x.cuda(), x.cuda(), [33, 37], [0, 0])
    k, v = gpu.read([3, 20], [30, 9], rows=29, max_rows=25, ld=2 * D + 16, fill=-3.0)
    full = gpu.read([33, 37], [0, 0])
    for got, want in ((k, full[0]), (v, full[1])):
        assert torch.equal(got[:3, :2 * D], want[30:33]) and torch.equal(got[3:23, :2 * D], want[42:62])
        assert (got[23:] == -3).all() and (got[:, 2 * D:] == -3).all()


def test_what_only_the_device_sees_is_skipped_and_reported():
    """Pages outside the cache, tokens past the table, negative starts and
    row bounds that decrease or exceed what was announced."""
    g = torch.Generator().manual_seed(6)
    table = torch.tensor([[0, 9, 1], [2, 3, -4], [4, 5, 5], [7, 8, 6]])
    ref = Cache(9, 16, 1, table)
    ref.scales = [torch.full_like(s, 0.01) for s in ref.scales]
    gpu = GpuCache(ref)
    x = torch.randn(160, D, generator=g).half()
    d = x.cuda()
    before = [c.clone() for c in gpu.codes]
    # Sequence 0: its middle page does not exist; 1: nor does its last one;
    # 2: starts below 0; 3: past its table.
    gpu.write(d, d, [40, 40, 3, 20], [0, 0, -1, 40])
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
    ref.write(0, 0, 0, x[:16].view(16, 1, D))
    ref.write(0, 0, 32, x[32:40].view(8, 1, D))
    ref.write(0, 1, 0, x[40:72].view(32, 1, D))
    ref.write(0, 3, 40, x[83:91].view(8, 1, D))  # tokens 40 .. 47 of 48
    torch.cuda.synchronize()
    assert torch.equal(gpu.codes[0].cpu(), ref.codes[0])
    k, _ = gpu.read([48], [0], fill=-3.0)
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
    assert (k[16:32] == -3).all() and not (k[:16] == -3).all()
    for counts, max_rows in (([5, -2, 9, 1], 9), ([200, 0, 0, 0], 200), ([12, 0, 0, 0], 11)):
        held = [c.clone() for c in gpu.codes]
        gpu.write(d, d, counts, [0, 0, 0, 0], max_rows=max_rows)
        assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
        if counts[1] == 0:
            assert all(torch.equal(a, b) for a, b in zip(held, gpu.codes))
    assert not torch.equal(before[0], gpu.codes[0])


def test_what_is_skipped_leaves_keys_values_and_scales():
    """As above, for all that a write touches: codes and scales of keys and of
    values, beside sequences that are written."""
    g = torch.Generator().manual_seed(16)
    table = torch.tensor([[0, 9, 1], [2, 3, -4], [4, 5, 10], [7, 8, 6]])
    ref = Cache(10, 16, 2, table.clamp(0, 9))
    ref.scales = [torch.rand(10, 2, generator=g) for _ in range(2)]
    ref.table = table
    gpu = GpuCache(ref)
    gpu.desc.pages = 9  # page 9 lies behind the cache
    x = torch.randn(120, 4 * D, generator=g).half()
    d = x.cuda()
    k, v = d[:, :2 * D], d[:, 2 * D:]

    def wrote(seq, start, first, end):
        for which in range(2):
            ref.write(which, seq, start, x[first:end, which * 2 * D:(which + 1) * 2 * D].view(end - first, 2, D))

    gpu.write(k, v, [40, 40, 3, 20], [0, 0, -1, 40])
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
    for call in ((0, 0, 0, 16), (0, 32, 32, 40), (1, 0, 40, 72), (3, 40, 83, 91)):
        wrote(*call)
    same_cache(ref, gpu)
    # Bounds that decrease: the other sequences are written.
    gpu.write(k, v, [5, -2, 9, 1], [0, 0, 0, 0], max_rows=9)
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
    for call in ((0, 0, 0, 5), (2, 0, 3, 12), (3, 0, 12, 13)):
        wrote(*call)
    same_cache(ref, gpu)
    # More rows than there are, or than were announced, and a negative first row.
    for counts, max_rows in (([200, 0, 0, 0], 200), ([12, 0, 0, 0], 11), ([-3, 3, 0, 0], 9)):
        gpu.write(k, v, counts, [0, 0, 0, 0], max_rows=max_rows)
        assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
        same_cache(ref, gpu)
    # What is read back of skipped tokens stays, keys and values.
    for got in gpu.read([48], [0], fill=-3.0):
        assert (got[16:32] == -3).all() and not (got[:16] == -3).any()
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT


def test_host_memory_is_refused():
    g = torch.Generator().manual_seed(7)
    gpu = GpuCache(Cache(4, 16, 1, shuffled_table(1, 4, 0, g)))
    host = torch.zeros(4, D, dtype=torch.float16)
    with pytest.raises(N.OmniVoiceError, match="k is not memory of the current device"):
        gpu.write(host, host, [4], [0])


@pytest.mark.parametrize("change", [
    dict(rows=2 ** 63, max_rows=2 ** 63), dict(rows=2 ** 40, max_rows=2 ** 40), dict(heads=2 ** 20),
    dict(num_seqs=2 ** 63), dict(max_length=2 ** 60), dict(kv_heads=0), dict(heads=3)])
def test_no_workspace_size_for_calls_that_are_refused(change):
    args = dict(rows=40, max_rows=40, max_length=64, heads=4, num_seqs=1, kv_heads=2) | change
    d = N.KvCache(kv_heads=args["kv_heads"], num_seqs=args["num_seqs"], head_dim=D, page_tokens=16,
                  pages=4, max_pages=4)
    assert N.lib().ov_attention_kv_cache_workspace_bytes(
        ctypes.byref(d), args["rows"], args["max_rows"], args["max_length"], args["heads"]) == 0


# ---------------------------------------------------------------- attention

def filled(seqs, page, kv, lengths, g, page_sizes=False, extra=2):
    """A cache with random codes up to `lengths`; the slots behind them hold
    codes of the type's ends, pages that no sequence owns NaN scales."""
    max_pages = max(1, max(-(-n // page) for n in lengths) + 1)
    ref = Cache(seqs * max_pages + extra, page, kv, shuffled_table(seqs, max_pages, extra, g))
    for s, n in enumerate(lengths):
        for j in range(-(-n // page)):
            at = int(ref.table[s, j])
            for which in range(2):
                ref.codes[which][at] = torch.randint(-127, 128, (kv, page, D), generator=g).to(torch.int8)
                scale = torch.rand(kv, generator=g) * 0.02 + 0.005
                if page_sizes:  # pages of very different size, some of them zero
                    scale *= 10.0 ** float(torch.randint(-4, 2, (1,), generator=g))
                    if j % 3 == 1:
                        scale[0] = 0.0
                        ref.codes[which][at, 0] = 0
                ref.scales[which][at] = scale
                left = n - j * page
                if left < page:
                    ref.codes[which][at, :, left:] = -128 if which else 127
    return ref


def reference(ref, q, counts, lengths, heads, causal, scale):
    """float64 output and bound for every packed row."""
    out = torch.zeros(q.shape[0], heads, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    group, at = heads // ref.kv, 0
    for s, (n, length) in enumerate(zip(counts, lengths)):
        k, v = ref.tokens(0, s, 0, length), ref.tokens(1, s, 0, length)
        pages = ref.table[s][torch.arange(length) // ref.page]
        i = torch.arange(n)
        seen = (length - n + i + 1).clamp(min=0) if causal else torch.full((n,), length)
        for h in range(heads):
            kvh = h // group
            out[at:at + n, h], bound[at:at + n, h] = attention(
                q[at:at + n, h * D:(h + 1) * D].double(), k[kvh], v[kvh],
                ref.scales[0][pages, kvh].double(), ref.scales[1][pages, kvh].double(), seen, scale)
        at += n
    return out.flatten(1), bound.flatten(1)


def check_attention(ref, counts, lengths, heads, causal, g, workspace=True, scale=D ** -0.5, q_size=1.0):
    rows = sum(counts) + 3  # rows behind the last sequence stay
    q = (torch.randn(rows, heads * D + 24, generator=g) * q_size).half()
    q[sum(counts):] = float("nan")
    want, bound = reference(ref, q[:sum(counts), :heads * D], counts, lengths, heads, causal, scale)
    gpu = GpuCache(ref)
    out = torch.full((rows, heads * D + 8), -3.0, dtype=torch.float16, device="cuda")
    ws = gpu.workspace(rows, max(counts), max(lengths), heads) if workspace else None
    gpu.attend(q.cuda()[:, :heads * D], counts, lengths, heads, causal, scale, out, ws)
    torch.cuda.synchronize()
    got = out.cpu()
    assert (got[sum(counts):] == -3).all() and (got[:, heads * D:] == -3).all()
    off = (got[:sum(counts), :heads * D].double() - want).abs()
    assert torch.isfinite(off).all()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert (off <= bound).all(), f"{worst:.3g} of the bound"
    again = torch.full_like(out, -3.0)
    gpu.attend(q.cuda()[:, :heads * D], counts, lengths, heads, causal, scale, again, ws)
    torch.cuda.synchronize()
    assert torch.equal(out, again)  # also: the workspace was left ready
    return out


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 1), (4, 4), (16, 2), (12, 4), (5, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_single_tokens(page, heads, kv, causal):
    """One row for each sequence, lengths from none to several pages."""
    g = torch.Generator().manual_seed(page + heads)
    lengths = [1, 0, page - 1, page, page + 1, 3 * page + 7, 2, 31, 33, 300]
    check_attention(filled(len(lengths), page, kv, lengths, g), [1] * len(lengths), lengths, heads,
                    causal, g)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("page,heads,kv,lengths", [
    (64, 4, 2, [5000]), (16, 2, 1, [3333, 17]), (128, 8, 1, [4097, 128, 2000]),
    (32, 16, 16, [999, 1, 0, 1000])])
def test_single_tokens_over_long_histories(page, heads, kv, lengths, workspace):
    g = torch.Generator().manual_seed(page)
    check_attention(filled(len(lengths), page, kv, lengths, g), [1] * len(lengths), lengths, heads,
                    True, g, workspace)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("page,heads,kv,counts,lengths", [
    (64, 4, 2, [2, 3, 0, 8], [2, 100, 50, 8]),          # few rows each
    (16, 2, 1, [9, 1, 4], [400, 1, 0]),
    (128, 2, 2, [16], [1000]),
    (32, 8, 1, [2, 1], [77, 500]),
    (64, 4, 2, [17, 40, 1], [17, 300, 64]),             # tens of rows
    (64, 2, 1, [64], [64]), (64, 2, 1, [65], [129]),    # a tile of rows, and one row more
    (16, 16, 2, [33, 5], [33, 257]),
    (128, 4, 4, [130, 0, 127], [400, 3, 127]),
    (32, 3, 1, [50, 100], [333, 100]),                  # three heads of a key head: odd tiles
    (64, 2, 2, [257], [600]), (64, 4, 1, [300], [2100]),
    (16, 2, 1, [513, 2], [1025, 1])])
def test_blocks_of_rows(page, heads, kv, counts, lengths, causal):
    g = torch.Generator().manual_seed(sum(counts))
    check_attention(filled(len(lengths), page, kv, lengths, g), counts, lengths, heads, causal, g)


@pytest.mark.parametrize("n", [1, 3, 30, 200])
def test_more_rows_than_tokens(n):
    """Causal rows before a sequence's first token see nothing: zeros."""
    g = torch.Generator().manual_seed(n)
    lengths = [0, 1, n - 1, n // 2]
    out = check_attention(filled(4, 16, 2, lengths, g), [n] * 4, lengths, 4, True, g)
    assert (out[:n, :4 * D] == 0).all()


@pytest.mark.parametrize("n", [1, 4, 100])
def test_pages_of_very_different_scales(n):
    """Page scales over six decades and pages of zeros, keys and values."""
    g = torch.Generator().manual_seed(n)
    lengths = [700, 95, 1201]
    check_attention(filled(3, 32, 2, lengths, g, page_sizes=True), [n] * 3, lengths, 4, True, g)


@pytest.mark.parametrize("n", [1, 40])
def test_large_scores(n):
    """Scores in the hundreds, as good as one token for each row."""
    g = torch.Generator().manual_seed(n)
    lengths = [500, 64]
    check_attention(filled(2, 64, 1, lengths, g), [n] * 2, lengths, 2, True, g, q_size=30.0)


@pytest.mark.parametrize("n", [1, 40])
def test_a_nan_page_reaches_its_own_sequence_and_head_only(n):
    g = torch.Generator().manual_seed(n)
    lengths = [200, 200]
    for which in range(2):
        ref = filled(2, 64, 2, lengths, g)
        ref.scales[which][int(ref.table[1, 1]), 1] = float("nan")
        q = torch.randn(2 * n, 4 * D, generator=g).half()
        want, bound = reference(ref, q, [n] * 2, lengths, 4, True, 0.1)
        gpu = GpuCache(ref)
        out = torch.zeros(2 * n, 4 * D, dtype=torch.float16, device="cuda")
        gpu.attend(q.cuda(), [n] * 2, lengths, 4, True, 0.1, out,
                   gpu.workspace(2 * n, n, 200, 4))
        got = out.cpu().double()
        clean = torch.ones_like(got, dtype=torch.bool)
        clean[n:, 2 * D:] = False
        assert ((got - want).abs() <= bound)[clean].all()
        assert got[n:, 2 * D:].isnan().all()


@pytest.mark.parametrize("heads", [17, 48, 200])
def test_many_query_heads_of_one_key_head(heads):
    """A single token's heads fill, or pass, a tile of rows."""
    g = torch.Generator().manual_seed(heads)
    lengths = [0, 1, 130, 300]
    check_attention(filled(4, 32, 1, lengths, g), [1, 1, 2, 1], lengths, heads, True, g)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(8, 8), (16, 8), (24, 8)])
def test_lengths_around_the_kernels_key_steps_in_pairs_of_row_tiles(heads, kv, causal):
    """So many sequences that a CTA takes 256 rows, of which the first 128 may
    see up to 128 tokens less than the last."""
    g = torch.Generator().manual_seed(heads + causal)
    lengths = [n + d for n in (64, 128, 192, 256, 320, 640, 1152) for d in (-1, 0, 1)]
    counts = [min(n, 129 + 17 * i) for i, n in enumerate(lengths)]
    counts[:3] = [129, 256, 257]  # more rows than tokens: the first see none
    check_attention(filled(len(lengths), 64, kv, lengths, g), counts, lengths, heads, causal, g)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("length", [1, 63, 64, 65, 127, 128, 129, 193, 256, 257, 384, 449, 511, 640, 1025, 1151])
def test_lengths_around_the_kernels_key_steps_in_single_tiles(length, workspace):
    g = torch.Generator().manual_seed(length)
    check_attention(filled(1, 16, 2, [length], g), [40], [length], 4, True, g, workspace)
    check_attention(filled(1, 128, 2, [length], g), [100], [length], 2, False, g, workspace)


@pytest.mark.parametrize("n", [1, 12, 40])
def test_no_tokens_at_all(n):
    g = torch.Generator().manual_seed(n)
    gpu = GpuCache(filled(3, 16, 2, [0, 0, 0], g))
    q = torch.randn(3 * n, 4 * D, generator=g).half().cuda()
    out = torch.full_like(q, 5.0)
    gpu.attend(q, [n] * 3, [0] * 3, 4, False, 0.1, out, gpu.workspace(3 * n, n, 0, 4))
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("n", [129, 200, 256, 300, 513])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_that_see_nothing_in_pairs_of_row_tiles(n, causal):
    """Both row tiles of a CTA, or the first of them, without a token: zeros,
    whatever the queries hold, in every launch."""
    g = torch.Generator().manual_seed(n + causal)
    lengths = ([0, 1, n - 129, n - 128, n - 127, n] * 4)[:20]
    kv, heads = 4, 4  # 80 items of at least two tiles: more than single tiles fill a GPU with
    check_attention(filled(20, 64, kv, lengths, g), [n] * 20, lengths, heads, causal, g)
    gpu = GpuCache(filled(20, 64, kv, [0] * 20, g))
    rows = 20 * n
    q = torch.full((rows, heads * D), 7.0, dtype=torch.float16, device="cuda")
    ws = gpu.workspace(rows, n, 0, heads)
    for _ in range(8):
        out = torch.full_like(q, 5.0)
        gpu.attend(q, [n] * 20, [0] * 20, heads, causal, 0.1, out, ws)
        torch.cuda.synchronize()
        assert (out == 0).all()


@pytest.mark.parametrize("n,heads,length,page", [(1, 2, 1_300_001, 16), (40, 1, 200_003, 64)])
def test_a_very_long_history(n, heads, length, page):
    """Against float64 on the GPU, in pieces."""
    pages = -(-length // page)
    g = torch.Generator(device="cuda").manual_seed(n)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    codes = [torch.randint(-127, 128, (pages, 1, page, D), generator=g, device="cuda",
                           dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(pages, 1, generator=g, device="cuda") * 0.02 + 0.005 for _ in range(2)]
    gpu = GpuCache(Cache(1, page, 1, torch.zeros(1, 1)))
    gpu.codes, gpu.scales, gpu.table = codes, scales, table
    d = gpu.desc
    d.keys, d.values = codes[0].data_ptr(), codes[1].data_ptr()
    d.key_scales, d.value_scales = scales[0].data_ptr(), scales[1].data_ptr()
    d.page_table, d.pages, d.max_pages = table.data_ptr(), pages, pages
    q = torch.randn(n, heads * D, generator=g, device="cuda").half()
    out = torch.zeros_like(q)
    gpu.attend(q, [n], [length], heads, True, D ** -0.5, out, gpu.workspace(n, n, length, heads))
    torch.cuda.synchronize()
    qd = q.double().view(n * heads, D)
    row = torch.arange(n * heads, device="cuda") // heads
    top = torch.full((n * heads, 1), -torch.inf, dtype=torch.float64, device="cuda")
    total, acc, square = (torch.zeros(n * heads, w, dtype=torch.float64, device="cuda") for w in (1, D, D))
    for p0 in range(0, pages, 20_000 * 16 // page):
        at = table[p0:p0 + 20_000 * 16 // page].long()
        k, v = ((codes[w][at, 0].double() * scales[w][at].double()[..., None]).flatten(0, 1)
                for w in range(2))
        pos = p0 * page + torch.arange(k.shape[0], device="cuda")
        z = (qd @ k.T * D ** -0.5).masked_fill(pos > length - n + row[:, None], -torch.inf)
        z = z.masked_fill(pos >= length, -torch.inf)
        grown = torch.maximum(top, z.amax(-1, keepdim=True))
        old, p = torch.exp(top - grown), torch.exp(z - grown)
        total, acc = total * old + p.sum(-1, keepdim=True), acc * old + p @ v
        square = square * old.square() + p.square() @ v.square()
        top = grown
    want = (acc / total).view(n, heads * D)
    # The roundings of the probabilities to half, each within 2^-11 of its
    # value, hence of a deviation of at most 2^-11 / sqrt(3) of it, are
    # independent: their sum with the values deviates by that times the root of
    # sum (p v)^2.  Seven deviations (2.6e-12 for a value, of 5,120), the
    # output's own rounding, and as much again for float32 sums.
    bound = (7 * 2.0 ** -11 / 3 ** 0.5 * square.sqrt() / total).view(n, heads * D)
    bound = bound + want.abs() * 2.0 ** -10 + 2.0 ** -24
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("seqs,heads,kv", [(33, 4, 2), (64, 8, 8), (300, 2, 1), (1000, 1, 1)])
@pytest.mark.parametrize("n", [1, 9])
def test_many_sequences(seqs, heads, kv, n):
    """More sequences than lanes, some without rows or tokens."""
    g = torch.Generator().manual_seed(seqs)
    lengths = [int(x) for x in torch.randint(0, 90, (seqs,), generator=g)]
    counts = [int(x) for x in torch.randint(0, n + 1, (seqs,), generator=g)]
    lengths[7], counts[7] = 1500, n
    check_attention(filled(seqs, 32, kv, lengths, g), counts, lengths, heads, True, g)


@pytest.mark.parametrize("n", [4, 60])
@pytest.mark.parametrize("which", [0, 1])
def test_a_nan_page_that_only_later_rows_see(n, which):
    g = torch.Generator().manual_seed(n)
    length = 64 + n // 2  # half of the rows end before the second page
    ref = filled(1, 64, 1, [length], g)
    ref.scales[which][int(ref.table[0, 1]), 0] = float("nan")
    q = torch.randn(n, 2 * D, generator=g).half()
    gpu = GpuCache(ref)
    out = torch.zeros(n, 2 * D, dtype=torch.float16, device="cuda")
    gpu.attend(q.cuda(), [n], [length], 2, True, 0.1, out, gpu.workspace(n, n, length, 2))
    got = out.cpu()
    clean = 64 - (length - n)  # rows that see the first page only
    assert got[clean:].isnan().all()
    ref.scales[which][int(ref.table[0, 1]), 0] = 0.01  # not seen by these
    want, bound = reference(ref, q, [n], [length], 2, True, 0.1)
    assert ((got[:clean].double() - want[:clean]).abs() <= bound[:clean]).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_a_nan_page_in_pairs_of_row_tiles(page, which):
    """Each sequence has its NaN page elsewhere: before every row, inside what
    only the later rows of the first tile see, or only the second tile."""
    g = torch.Generator().manual_seed(page + which)
    seqs, n, length = 50, 300, 400
    ref = filled(seqs, page, 1, [length] * seqs, g)
    used = -(-length // page)
    at = [(s, s % used) for s in range(seqs)]
    for s, j in at:
        ref.scales[which][ref.table[s, j], 0] = float("nan")
    q = torch.randn(seqs * n, D, generator=g).half()
    gpu = GpuCache(ref)
    out = torch.zeros(seqs * n, D, dtype=torch.float16, device="cuda")
    gpu.attend(q.cuda(), [n] * seqs, [length] * seqs, 1, True, 0.1, out,
               gpu.workspace(seqs * n, n, length, 1))
    got = out.cpu().view(seqs, n, D)
    for s, j in at:
        ref.scales[which][ref.table[s, j], 0] = 0.01  # not seen by the rows that are compared
    want, bound = reference(ref, q, [n] * seqs, [length] * seqs, 1, True, 0.1)
    want, bound = want.view(seqs, n, D), bound.view(seqs, n, D)
    for s, j in at:
        clean = min(n, max(0, page * j - (length - n)))  # rows that end before the page
        assert got[s, clean:].isnan().all()
        assert ((got[s, :clean].double() - want[s, :clean]).abs() <= bound[s, :clean]).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_bad_pages_in_pairs_of_row_tiles(page, causal):
    """A page outside the cache, elsewhere in each sequence, counts as tokens
    that nothing sees, for both row tiles."""
    g = torch.Generator().manual_seed(page + causal)
    seqs, n, length = 50, 300, 400
    ref = filled(seqs, page, 1, [length] * seqs, g)
    table, used = ref.table.clone(), -(-length // page)
    for s in range(seqs):
        ref.table[s, s % used] = (-1, ref.codes[0].shape[0], 2 ** 31 - 1)[s % 3]
    q = torch.randn(seqs * n, D, generator=g).half()
    gpu = GpuCache(ref)
    out = torch.zeros(seqs * n, D, dtype=torch.float16, device="cuda")
    gpu.attend(q.cuda(), [n] * seqs, [length] * seqs, 1, causal, 0.1, out,
               gpu.workspace(seqs * n, n, length, 1))
    torch.cuda.synchronize()
    assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
    got = out.cpu().double().view(seqs, n, D)
    ref.table = table
    token = torch.arange(length)
    for s in range(seqs):
        keep = token[token // page != s % used]
        k, v = (ref.tokens(w, s, 0, length)[0][keep] for w in range(2))
        pages = table[s][keep // page]
        ends = length - n + 1 + torch.arange(n) if causal else torch.full((n,), length)
        seen = (keep < ends[:, None]).sum(-1)
        want, bound = attention(q[s * n:(s + 1) * n].double(), k, v, ref.scales[0][pages, 0].double(),
                                ref.scales[1][pages, 0].double(), seen, 0.1)
        assert ((got[s] - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [1, 50])
def test_sequences_that_share_pages(n):
    g = torch.Generator().manual_seed(n)
    lengths = [200, 230, 130]
    ref = filled(3, 64, 2, lengths, g)
    ref.table[1, :2] = ref.table[0, :2]
    ref.table[2, :2] = ref.table[0, :2]
    check_attention(ref, [n] * 3, lengths, 4, False, g)


@pytest.mark.parametrize("n", [2, 30])
def test_the_least_scales(n):
    """Factors that underflow: every score is 0, hidden tokens stay hidden."""
    g = torch.Generator().manual_seed(n)
    ref = filled(1, 32, 1, [100], g)
    for s in ref.scales:
        s.copy_(torch.where(s.isnan(), s, 1e-6))
    check_attention(ref, [n], [100], 2, True, g, scale=1e-36)
    ref.scales[0].copy_(torch.where(ref.scales[0].isnan(), ref.scales[0], 1e-38))
    check_attention(ref, [n], [100], 2, True, g, scale=1e-30)


@pytest.mark.parametrize("n", [1, 12, 40, 300])
@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-12, 2.0 ** -33, 2.0 ** -32])
def test_value_scales_below_every_half(n, scale):
    """Codes that are not zero under value scales so small that code * scale
    rounds to 0 (128 * 2^-32 is half of the least half): zeros, as reading the
    cache gives; and nothing beside a page of ordinary values."""
    g = torch.Generator().manual_seed(n)
    seqs = 50 if n == 300 else 2  # pairs of row tiles
    lengths = [320, 90] * (seqs // 2)
    ref = filled(seqs, 32, 1, lengths, g)
    ref.codes[1][..., 5] = -127 if scale == 2.0 ** -32 else -128
    ref.codes[1][..., 9] = 127
    for s in range(seqs):
        ref.scales[1][ref.table[s, :(lengths[s] + 31) // 32]] = scale
    gpu = GpuCache(ref)
    assert (gpu.read(lengths, [0] * seqs)[1] == 0).all()
    q = torch.randn(seqs * n, D, generator=g).half().cuda()
    out = torch.full_like(q, 5.0)
    ws = gpu.workspace(seqs * n, n, 320, 1)
    gpu.attend(q, [n] * seqs, lengths, 1, False, 0.1, out, ws)
    torch.cuda.synchronize()
    assert (out == 0).all()
    # The page in the middle has ordinary values: the others only take their
    # share of the probability.
    ref.scales[1][ref.table[0, 4], 0] = 0.01
    check_attention(ref, [n] * seqs, lengths, 1, False, g)


def test_one_workspace_for_calls_of_any_shape_and_two_graphs():
    """A workspace goes from single tokens of few sequences to many, to
    blocks of rows and back, eagerly and in two graphs that share it."""
    g = torch.Generator().manual_seed(4)
    shapes = [([3000], [1], 4, 2), ([700] * 40, [1] * 40, 4, 4), ([2500], [30], 8, 1),
              ([900, 900], [100, 3], 2, 2), ([3000], [2], 4, 1)]
    calls, need = [], 0
    for lengths, counts, heads, kv in shapes:
        gpu = GpuCache(filled(len(lengths), 32, kv, lengths, g))
        q = torch.randn(sum(counts), heads * D, generator=g).half().cuda()
        own = gpu.workspace(sum(counts), max(counts), max(lengths), heads)
        need = max(need, own.numel())
        want = gpu.attend(q, counts, lengths, heads, True, 0.1, torch.zeros_like(q), own)
        calls.append((gpu, q, counts, lengths, heads, want))
    torch.cuda.synchronize()
    shared = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        for gpu, q, counts, lengths, heads, want in calls:
            got = gpu.attend(q, counts, lengths, heads, True, 0.1, torch.zeros_like(q), shared)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
    lib, s = N.lib(), torch.cuda.Stream()
    graphs, outs, held = [], [], []
    for part in (calls[:3], calls[2:]):
        prepared = [(gpu, q, i32(cumulative(counts)), i32(lengths), counts, lengths, heads,
                     torch.zeros_like(q)) for gpu, q, counts, lengths, heads, _ in part]
        torch.cuda.synchronize()
        graph = ctypes.c_void_p()
        N.check(lib.ov_graph_capture_begin(s.cuda_stream))
        for gpu, q, cu, ln, counts, lengths, heads, out in prepared:
            N.check(lib.ov_attention_kv_cache(
                ctypes.byref(gpu.desc), q.data_ptr(), q.stride(0), q.shape[0], cu.data_ptr(),
                max(counts), ln.data_ptr(), max(lengths), heads, 1, 0.1, out.data_ptr(),
                out.stride(0), shared.data_ptr(), shared.numel(), s.cuda_stream))
        N.check(lib.ov_graph_capture_end(s.cuda_stream, ctypes.byref(graph)))
        graphs.append(graph)
        outs.append([p[-1] for p in prepared])
        held.append(prepared)
    for turn in (0, 1, 1, 0):
        for out in outs[turn]:
            out.zero_()
        torch.cuda.synchronize()
        N.check(lib.ov_graph_launch(graphs[turn], s.cuda_stream))
        torch.cuda.synchronize()
        for out, call in zip(outs[turn], (calls[:3], calls[2:])[turn]):
            assert torch.equal(out, call[5])
    for graph in graphs:
        N.check(lib.ov_graph_destroy(graph))


@pytest.mark.parametrize("n", [1, 40])
def test_bad_pages_and_lengths_are_skipped_and_reported(n):
    """A page outside the cache counts as tokens that nothing sees."""
    g = torch.Generator().manual_seed(n)
    ref = filled(1, 32, 1, [150], g)
    table = ref.table.clone()
    q = torch.randn(n, 2 * D, generator=g).half()
    for bad in (-1, ref.codes[0].shape[0], 2 ** 31 - 1):
        ref.table = table.clone()
        ref.table[0, 2] = bad
        gpu = GpuCache(ref)
        out = torch.zeros(n, 2 * D, dtype=torch.float16, device="cuda")
        gpu.attend(q.cuda(), [n], [150], 2, False, 0.1, out, gpu.workspace(n, n, 150, 2))
        torch.cuda.synchronize()
        assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
        keep = torch.cat([torch.arange(64), torch.arange(96, 150)])
        ref.table = table
        k, v = (ref.tokens(w, 0, 0, 150)[0][keep] for w in range(2))
        pages = table[0][keep // 32]
        for h in range(2):
            want, bound = attention(q[:, h * D:(h + 1) * D].double(), k, v,
                                    ref.scales[0][pages, 0].double(), ref.scales[1][pages, 0].double(),
                                    torch.full((n,), keep.numel()), 0.1)
            off = (out[:, h * D:(h + 1) * D].cpu().double() - want).abs()
            assert (off <= bound).all()
    # A negative length is none; one above max_length is cut there.
    gpu = GpuCache(ref)
    for length, cut in ((-5, 0), (150, 100)):
        got = torch.full((n, 2 * D), 9.0, dtype=torch.float16, device="cuda")
        want = torch.full_like(got, 9.0)
        ws = gpu.workspace(n, n, 100, 2)
        gpu.attend(q.cuda(), [n], [length], 2, False, 0.1, got, ws, max_length=100)
        torch.cuda.synchronize()
        assert device_errors() == N.OV_DEVICE_BAD_ARGUMENT
        gpu.attend(q.cuda(), [n], [cut], 2, False, 0.1, want, ws, max_length=100)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """Pages whose first byte lies past 2^32, written, read and attended."""
    page, kv = 128, 8
    tile = kv * page * D
    pages = 2 ** 32 // tile + 40
    codes = [torch.empty(pages, kv, page, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, kv, device="cuda") for _ in range(2)]
    g = torch.Generator().manual_seed(8)
    small = Cache(3, page, kv, torch.tensor([[2, 0, 1]]))
    gpu = GpuCache(small)
    far = GpuCache(small)
    far.codes, far.scales = codes, scales
    far.table = i32([[pages - 1, pages - 3, pages - 2]])
    far.desc.keys, far.desc.values = codes[0].data_ptr(), codes[1].data_ptr()
    far.desc.key_scales, far.desc.value_scales = scales[0].data_ptr(), scales[1].data_ptr()
    far.desc.page_table, far.desc.pages = far.table.data_ptr(), pages
    x = torch.randn(300, 2 * kv * D, generator=g).half().cuda()
    outs = []
    for c in (gpu, far):
        c.write(x[:, :kv * D], x[:, kv * D:], [300], [0])
        k, v = c.read([300], [0])
        out = []
        for n in (1, 100):
            o = torch.zeros(n, 2 * kv * D, dtype=torch.float16, device="cuda")
            c.attend(x[:n], [n], [300], 2 * kv, True, 0.09, o, c.workspace(n, n, 300, 2 * kv))
            out.append(o)
        torch.cuda.synchronize()
        outs.append([k, v, *out])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert not torch.equal(outs[0][0], torch.zeros_like(outs[0][0]))


def test_another_stream_and_graph_replay():
    """The run of a decoding step (append, attend) captured once and replayed
    with new rows and lengths in the same buffers equals eager calls; an
    eager call works on a stream of its own."""
    g = torch.Generator().manual_seed(9)
    page, kv, heads, seqs = 32, 2, 4, 3
    lengths = [40, 0, 95]
    ref = filled(seqs, page, kv, [n + 8 for n in lengths], g)
    gpu, other = GpuCache(ref), GpuCache(ref)
    width = (heads + 2 * kv) * D
    rows = [torch.randn(seqs, width, generator=g).half().cuda() for _ in range(4)]
    max_length = 128
    lib = N.lib()
    qkv = rows[0].clone()
    cu, starts, ends = i32([0, 1, 2, 3]), i32(lengths), i32([n + 1 for n in lengths])
    out = torch.zeros(seqs, heads * D, dtype=torch.float16, device="cuda")
    ws = gpu.workspace(seqs, 1, max_length, heads)
    s = torch.cuda.Stream()

    def step(c, q, o, w, on):
        k, v = q.data_ptr() + heads * D * 2, q.data_ptr() + (heads + kv) * D * 2
        N.check(lib.ov_kv_cache_write(ctypes.byref(c.desc), k, width, v, width, seqs, cu.data_ptr(),
                                      starts.data_ptr(), 1, on))
        N.check(lib.ov_attention_kv_cache(ctypes.byref(c.desc), q.data_ptr(), width, seqs,
                                          cu.data_ptr(), 1, ends.data_ptr(), max_length, heads, 1,
                                          0.1, o.data_ptr(), heads * D, w.data_ptr(), w.numel(), on))

    torch.cuda.synchronize()
    graph = ctypes.c_void_p()
    N.check(lib.ov_graph_capture_begin(s.cuda_stream))
    step(gpu, qkv, out, ws, s.cuda_stream)
    N.check(lib.ov_graph_capture_end(s.cuda_stream, ctypes.byref(graph)))
    eager = torch.zeros_like(out)
    ws2 = other.workspace(seqs, 1, max_length, heads)
    for r in rows:
        with torch.cuda.stream(s):
            qkv.copy_(r)
            N.check(lib.ov_graph_launch(graph, s.cuda_stream))
        torch.cuda.synchronize()
        step(other, r, eager, ws2, s.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert all(torch.equal(a, b) for a, b in zip(gpu.codes, other.codes))
        assert all(torch.equal(a.nan_to_num(-7.0), b.nan_to_num(-7.0))
                   for a, b in zip(gpu.scales, other.scales))  # unused pages hold NaN
        starts += 1
        ends += 1
        torch.cuda.synchronize()
    N.check(lib.ov_graph_destroy(graph))


def test_a_decoding_step_next_to_the_varlen_attention():
    """Projection with QK norm and RoPE, cache, attention, head and log
    probabilities as a caller chains them; the attention is within what
    rounding keys and values to a page's grid can change of the one that
    ov_attention_varlen computes from the same rows."""
    g = torch.Generator().manual_seed(11)
    heads, kv, width, n, page = 4, 2, 256, 150, 32
    cols = (heads + 2 * kv) * D
    lib = N.lib()
    x = torch.randn(n, width, generator=g).half().cuda()
    w = (torch.randn(cols, width, generator=g) / 16).half().cuda()
    norm = torch.ones(D, device="cuda")
    cos = torch.ones(n, D // 2, device="cuda")
    sin = torch.zeros(n, D // 2, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    args = N.EpilogueArgs(q_norm=norm.data_ptr(), k_norm=norm.data_ptr(), positions=pos.data_ptr(),
                          rope_cos=cos.data_ptr(), rope_sin=sin.data_ptr(), max_positions=n,
                          heads=heads, kv_heads=kv, head_dim=D, epsilon=1e-6)
    qkv = torch.empty(n, cols, dtype=torch.float16, device="cuda")
    N.check(lib.ov_gemm_f16(x.data_ptr(), width, w.data_ptr(), qkv.data_ptr(), cols, n, width, cols,
                            N.OV_EPI_QKNORM_ROPE_F16, ctypes.byref(args), None, 0, stream()))
    plain = torch.empty(n, heads * D, dtype=torch.float16, device="cuda")
    cu = i32([0, n])
    N.check(lib.ov_attention_varlen(qkv.data_ptr(), cols, n, cu.data_ptr(), 1, n, heads, kv, D,
                                    D ** -0.5, plain.data_ptr(), heads * D, stream()))
    gpu = GpuCache(Cache(5, page, kv, torch.tensor([[3, 0, 2, 4, 1]])))
    k, v = qkv[:, heads * D:(heads + kv) * D], qkv[:, (heads + kv) * D:]
    gpu.write(k, v, [n], [0])
    out = torch.empty_like(plain)
    gpu.attend(qkv[:, :heads * D], [n], [n], heads, False, D ** -0.5, out, gpu.workspace(n, n, n, heads))
    last = torch.empty(1, heads * D, dtype=torch.float16, device="cuda")
    gpu.attend(qkv[n - 1:, :heads * D], [1], [n], heads, True, D ** -0.5, last, gpu.workspace(1, 1, n, heads))
    torch.cuda.synchronize()
    # Half a step of at most amax / 127 for a value, and for a key through
    # |q|_1 * step / 2 * scale in each score (a relative change of twice its
    # exponential); halves elsewhere.
    step_k = float(k.abs().max()) / 127
    step_v = float(v.abs().max()) / 127
    shift = float(qkv[:, :heads * D].float().view(n, heads, D).abs().sum(-1).max()) * step_k / 2 * D ** -0.5
    bound = step_v / 2 + float(v.abs().max()) * (torch.tensor(2 * shift).expm1().item() + 2.0 ** -9)
    assert float((out - plain).abs().max()) <= bound
    assert float((last - plain[n - 1:]).abs().max()) <= bound
    # The audio head over the attention's output, four codebooks.
    books, vocab = 4, 1025
    head = (torch.randn(books * vocab, heads * D, generator=g) / 8).half().cuda()
    logits = torch.empty(n, books * vocab + 12, device="cuda")
    N.check(lib.ov_gemm_f16(out.data_ptr(), heads * D, head.data_ptr(), logits.data_ptr(),
                            logits.stride(0), n, heads * D, books * vocab, N.OV_EPI_STORE_F32, None,
                            None, 0, stream()))
    targets = torch.randint(0, vocab, (books, n), generator=g).to(torch.int32).cuda()
    lp = torch.empty(books, n, device="cuda")
    rank = torch.empty(books, n, dtype=torch.int32, device="cuda")
    N.check(lib.ov_token_logprobs(logits.data_ptr(), N.OV_LOGITS_F32, logits.stride(0), n, books,
                                  vocab, targets.data_ptr(), 0, lp.data_ptr(), None,
                                  rank.data_ptr(), None, None, stream()))
    torch.cuda.synchronize()
    z = logits[:, :books * vocab].unflatten(1, (books, vocab)).transpose(0, 1)
    t = targets.long()[..., None]
    want = torch.log_softmax(z.double(), -1).gather(2, t)[..., 0]
    assert float((lp.double() - want).abs().max()) <= 1e-5 * (1 + float(want.abs().max()))
    assert torch.equal(rank.long(), (z > z.gather(2, t)).sum(-1))
