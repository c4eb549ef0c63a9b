"""A paged cache of keys and values against plain torch in 64 bits: rows into pages and back, attention over the pages.

Tolerances.  Writes and reads are exact: codes, powers of two and copies have one right value; only fp32 values read as bf16 are rounded, once.
Attention: let A = sum_j p_j |v_j| and B = the largest sum_d |q_d k_jd| * scale of the row.  A score is off by at most (dim + 8) * 2^-24 * B * 2 (fp32 sums in any
order, the tensor core's truncating adds count twice) plus 2^-20 of its size in exponentials and caps (approximate exp2, tanh), so that a weight is off by that
share; with weights rounded to bf16 (2^-8 each) an output is off by
    A * (2^-8 [bf16 operands] + 2 * (dim + 8) * 2^-23 * B + 2^-17) + |out| * 2^-8 [bf16 output].
"""
import ctypes

import pytest
import torch

from paged_cache import Cache, codes_of

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def backend():
    import gpt_b200
    be = gpt_b200.Backend(0, torch.cuda.current_stream().cuda_stream)
    yield be
    be.close()


def rows_in(rows, width, dtype, extra, seed, scale=1.0):
    """[rows x width] as a slice of wider rows."""
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn(rows, width, generator=g)).to(TYPES[dtype])
    wide = torch.full((rows, width + extra), 7.0, dtype=TYPES[dtype], device="cuda")
    wide[:, :width] = x.cuda()
    return wide[:, :width], x


def places(c):
    """(row, page, token) of every new row that has a place."""
    got = []
    for s, n in enumerate(c.counts):
        for i in range(n):
            p = max(c.lengths[s], 0) - n + i
            if p >= 0:
                got.append((int(c.starts_cpu[s]) + i, int(c.table_cpu[s, p // c.page]), p % c.page))
    return got


SHAPES = [  # lengths, counts, kv heads, dim, page
    ([1], [1], 1, 8, 8), ([5, 0, 17], [5, 0, 3], 3, 40, 8), ([64, 64], [64, 1], 2, 64, 16), ([100, 33, 7, 250], [1, 1, 1, 1], 4, 128, 32), ([300], [257], 8, 96, 64), ([40] * 70, [1] * 70, 4, 64, 16),
    ([2, 3], [5, 3], 2, 72, 16),   # more new rows than tokens: the first ones have no place
    ([5000], [5000], 2, 128, 4096),
]


@pytest.mark.parametrize("kind", ["bf16", "f32", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,counts,kv_heads,dim,page", SHAPES)
def test_write_and_read(backend, lengths, counts, kv_heads, dim, page, dtype, kind):
    c = Cache(kind, lengths, counts, kv_heads, dim, page, seed=len(lengths) + dim, extra_rows=3).cuda()
    width = kv_heads * dim
    k, k_cpu = rows_in(c.rows, width, dtype, 8, 1)
    v, v_cpu = rows_in(c.rows, width, dtype, 16, 2, scale=100.0)
    want, scales = c.data_cpu.float().clone(), c.scales_cpu.clone() if c.scales_cpu is not None else None
    for r, page_id, token in places(c):
        for which, x in ((0, k_cpu), (1, v_cpu)):
            y = x[r].double().reshape(kv_heads, dim)
            if kind == "e4m3":
                codes, e = codes_of(y)
                want[page_id, which, :, token] = codes.float()
                scales[page_id, which, :, token] = e
            else:
                want[page_id, which, :, token] = y.to(c.TYPES[kind]).float()
    dt = {"bf16": 0, "f32": 1}[dtype]
    backend.kv_pages_write(c.pages, c.batch, k, k.stride(0), v, v.stride(0), dt)
    backend.synchronize()
    assert torch.equal(c.data.float().cpu(), want)
    if scales is not None:
        assert torch.equal(c.scales.cpu(), scales)
    ko, _ = rows_in(c.rows, width, dtype, 8, 3)
    vo, _ = rows_in(c.rows, width, dtype, 16, 4)
    before = [ko.clone(), vo.clone()]
    backend.kv_pages_read(ko, ko.stride(0), vo, vo.stride(0), dt, c.pages, c.batch)
    backend.synchronize()
    held = want.double() if scales is None else torch.ldexp(want.double(), scales[..., None].int() - 127)
    for which, x in ((0, before[0].cpu()), (1, before[1].cpu())):
        for r, page_id, token in places(c):
            x[r] = held[page_id, which, :, token].reshape(-1).to(TYPES[dtype])
        assert torch.equal((ko, vo)[which].cpu(), x)       # rows without a place, and those behind the last sequence, as they were
    for wide, width_ in ((k, width), (ko, width), (vo, width)):
        assert (wide._base[:, width_:] == 7.0).all()


def test_write_edges_of_the_format(backend):
    """Zeros, the smallest and largest numbers, halfway cases, infinities and NaN: fp32 rows of 8 into e4m3."""
    tiny, big = 2.0 ** -149, 3.4e38
    x = torch.tensor([[0.0] * 8, [tiny, -tiny, 0, 0, 0, 0, 0, 0], [big, -big, 1, 0, 0, 0, 0, 0], [448, 449, -464, 465, 1, 2, 3, 4], [1.75, 1.76, 0.001, -0.002, 0, 0, 0, 0],
                      [float("inf"), 1, 2, 3, 4, 5, 6, 7], [float("nan"), -float("inf"), 0.1, 0.2, 0.3, 0.4, 0.5, 0.6], [17, 19, 21, 23, 25, 27, 29, 448], [2.0 ** -120, 2.0 ** -126, 2.0 ** -130, 0, 0, 0, 0, 0],
                      [1.0625, 1.1875, 1.3125, -1.4375, 448, 0, 0, 0]], dtype=torch.float32)
    n = x.shape[0]
    c = Cache("e4m3", [n], [n], 1, 8, 16).cuda()
    d = x.cuda()
    backend.kv_pages_write(c.pages, c.batch, d, 8, d, 8, 1)
    out_k, out_v = torch.empty(n, 8, device="cuda"), torch.empty(n, 8, device="cuda")
    backend.kv_pages_read(out_k, 8, out_v, 8, 1, c.pages, c.batch)
    backend.synchronize()
    codes, e = codes_of(x.double())
    want = torch.ldexp(codes, e[:, None].int() - 127)
    for got in (out_k, out_v):
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=1e300), torch.nan_to_num(want, nan=1e300))
    held = (want - x.double()).abs()
    fine = torch.isfinite(x.double()) & (x.abs() >= 2.0 ** -110) & (x.abs() < 3.3e38) & (x.double().abs() >= 2.0 ** -6 * torch.ldexp(torch.ones(n, 1, dtype=torch.float64), e[:, None].int() - 127))
    assert (held[fine] <= 2.0 ** -4 * x.double().abs()[fine]).all()


def attend(be, c, q, heads, dtype, scale, cap=0.0, window=0, sinks=0, extra=0, lse=True):
    width = heads * c.dim
    out, _ = rows_in(c.rows, width, dtype, extra, 99)
    out._base.fill_(77.0)
    sums = torch.full((c.rows + 1, heads), 77.0, device="cuda") if lse else None
    be.attention_paged(out, out.stride(0), sums, q, q.stride(0), {"bf16": 0, "f32": 1}[dtype], heads, c.pages, c.batch, scale, cap, window, sinks)
    return out, sums


def check(c, q, out, sums, heads, dtype, scale, cap=0.0, window=0, sinks=0, kind=None):
    want, lse, spread, slack = c.attention(q, heads, scale, cap, window, sinks)
    end = int(c.starts_cpu[-1])
    got = out.double().cpu()
    assert (got[end:] == 77.0).all() and (out._base[:, heads * c.dim:] == 77.0).all()
    weight = 2.0 ** -8 if dtype == "bf16" else 0.0
    bound = spread * (weight + 2 * (c.dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * HALF[dtype]
    off = (got - want).abs()[:end]
    assert torch.equal(torch.isnan(got[:end]), torch.isnan(want[:end]))
    fine = torch.isfinite(want[:end])
    assert (off[fine] <= bound[:end][fine] + 1e-30).all(), float((off[fine] / (bound[:end][fine] + 1e-30)).max())
    if sums is not None:
        s = sums.double().cpu()
        assert (s[c.rows] == 77.0).all() and (s[end:c.rows] == 77.0).all()
        empty = torch.isinf(lse[:end])
        assert torch.equal(torch.isinf(s[:end]), empty)
        close = (s[:end] - lse[:end]).abs() <= (2 * (c.dim + 8) * 2.0 ** -23 * slack.reshape(c.rows, heads, -1)[:end, :, 0] + 2.0 ** -17 * (1 + lse[:end].abs()))
        assert (close | empty | torch.isnan(lse[:end])).all()


ATTEND = [  # lengths, counts, kv heads, share, dim, page, cap, window, sinks
    ([1], [1], 1, 1, 8, 8, 0.0, 0, 0),
    ([256], [1], 12, 1, 64, 16, 0.0, 0, 0),
    ([1, 2, 15, 16, 17, 64, 65, 300], [1] * 8, 2, 4, 128, 16, 0.0, 0, 0),
    ([7, 1000, 130], [1, 1, 1], 1, 8, 96, 32, 40.0, 0, 0),
    ([700, 40, 9], [1, 1, 1], 2, 3, 128, 64, 0.0, 100, 4),
    ([700, 513], [1, 1], 2, 16, 64, 8, 0.0, 64, 70),
    ([33, 260, 5], [5, 3, 5], 2, 4, 64, 16, 0.0, 0, 0),
    ([90], [40], 1, 20, 40, 8, 5.0, 17, 3),
    ([128], [128], 2, 2, 64, 32, 0.0, 0, 0),
    ([129, 400, 1], [129, 200, 1], 2, 2, 128, 128, 0.0, 0, 0),
    ([513], [513], 1, 4, 80, 64, 40.0, 0, 0),
    ([600, 90], [333, 90], 1, 3, 128, 16, 0.0, 50, 5),
    ([1025], [300], 1, 1, 32, 256, 0.0, 1, 0),
    ([20, 0, 300, 3], [20, 0, 300, 7], 1, 2, 128, 64, 0.0, 0, 0),          # a sequence with more rows than tokens
    ([0, 64], [2, 64], 2, 1, 64, 32, 0.0, 0, 0),                          # one without any token
    ([2000], [260], 1, 8, 128, 32, 0.0, 300, 200),
    ([3000, 10, 1500], [2, 1, 130], 1, 4, 64, 16, 30.0, 0, 0),
]


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32"), ("f32", "e4m3"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("lengths,counts,kv_heads,share,dim,page,cap,window,sinks", ATTEND)
def test_attention(backend, lengths, counts, kv_heads, share, dim, page, cap, window, sinks, dtype, kind):
    c = Cache(kind, lengths, counts, kv_heads, dim, page, seed=dim + len(lengths), extra_rows=2, poison=True).cuda()
    heads, scale = kv_heads * share, dim ** -0.5
    q, _ = rows_in(c.rows, heads * dim, dtype, 8, 5, scale=2.0)
    out, sums = attend(backend, c, q, heads, dtype, scale, cap, window, sinks, extra=8)
    backend.synchronize()
    check(c, q, out, sums, heads, dtype, scale, cap, window, sinks)
    # whatever max_new says, and without the sums
    for most in (0, 1, 100000):
        c.cuda(max_new=most)
        out, sums = attend(backend, c, q, heads, dtype, scale, cap, window, sinks, extra=8, lse=False)
        backend.synchronize()
        check(c, q, out, sums, heads, dtype, scale, cap, window, sinks)


BOTH = [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32")]


@pytest.mark.parametrize("dtype,kind", BOTH + [("f32", "e4m3")])
@pytest.mark.parametrize("lengths,counts,kv_heads,share,dim,window,sinks", [
    ([9000, 3], [1, 1], 1, 8, 32, 0, 0),            # one tile shared by every block of the grid
    ([9000], [1], 1, 1, 128, 0, 0),
    ([7000, 20], [2, 1], 1, 16, 64, 0, 0),
    ([6000], [300], 1, 1, 64, 0, 0),
    ([50000], [1], 1, 16, 16, 0, 0),
    ([20000], [3], 1, 8, 128, 12000, 100),
])
def test_long_sequences(backend, lengths, counts, kv_heads, share, dim, window, sinks, dtype, kind):
    c = Cache(kind, lengths, counts, kv_heads, dim, 64, seed=11, poison=True).cuda()
    heads, scale = kv_heads * share, dim ** -0.5
    q, _ = rows_in(c.rows, heads * dim, dtype, 0, 6)
    out, sums = attend(backend, c, q, heads, dtype, scale, 0.0, window, sinks)
    again, sums_again = attend(backend, c, q, heads, dtype, scale, 0.0, window, sinks)
    backend.synchronize()
    check(c, q, out, sums, heads, dtype, scale, 0.0, window, sinks)
    assert torch.equal(out, again) and torch.equal(sums, sums_again)      # the parts' order does not depend on who arrives last
    backend.set_option("max_sms", 7)                                       # another grid, another cut of the line
    try:
        out, sums = attend(backend, c, q, heads, dtype, scale, 0.0, window, sinks)
        backend.synchronize()
        check(c, q, out, sums, heads, dtype, scale, 0.0, window, sinks)
    finally:
        backend.set_option("max_sms", 0)


@pytest.mark.parametrize("dtype,kind", BOTH + [("f32", "e4m3"), ("bf16", "f32")])
@pytest.mark.parametrize("count", [1, 3, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_does_not_matter(backend, dtype, kind, count, bad):
    """Not finite keys and values that only later rows of the same tile see, or that lie in front of the window: they make those rows, and only those, not finite."""
    dim, heads, window, sinks = 64, 4, 90, 2
    c = Cache(kind, [200, 130], [count, count], 2, dim, 16, seed=3)
    for s, length in enumerate(c.lengths):
        for position in ([length - 1, length - count // 2 - 1] if count > 1 else []) + [20]:
            for which in (0, 1):
                if which == 0 and position != 20:
                    continue      # of keys only one that nobody sees: a not finite score is a not finite row
                page, token = int(c.table_cpu[s, position // c.page]), position % c.page
                data = c.data_cpu.float()
                data[page, which, :, token, 5] = bad
                c.data_cpu = data.to(c.TYPES[kind])
                c.values[page, which, :, token, 5] = float("nan") if kind == "e4m3" else bad
    c.cuda()
    q, _ = rows_in(c.rows, heads * dim, dtype, 0, 8)
    out, sums = attend(backend, c, q, heads, dtype, 0.125, 0.0, window, sinks)
    backend.synchronize()
    want, lse, spread, slack = c.attention(q, heads, 0.125, 0.0, window, sinks)
    got = out.double().cpu()
    fine = torch.isfinite(want)
    assert fine.any() and torch.equal(torch.isfinite(got), fine)
    bound = torch.nan_to_num(spread, nan=0.0, posinf=0.0) * (2.0 ** -8 + 2 * (dim + 8) * 2.0 ** -23 * torch.nan_to_num(slack, nan=0.0, posinf=0.0) + 2.0 ** -17) + want.abs() * HALF[dtype]
    assert ((got - want).abs()[fine] <= bound[fine] + 1e-30).all()


@pytest.mark.parametrize("dtype,kind,share,count", [("bf16", "bf16", 4, 1), ("bf16", "e4m3", 2, 40), ("f32", "f32", 1, 1), ("f32", "f32", 2, 20)])
def test_numbers_that_do_not_fit_are_reported(backend, dtype, kind, share, count):
    import gpt_b200
    lengths, counts = [300, 200, 150], [count] * 3
    c = Cache(kind, lengths, counts, 2, 64, 16, seed=4).cuda()
    q, _ = rows_in(c.rows, 2 * share * 64, dtype, 0, 8)
    k, _ = rows_in(c.rows, 128, dtype, 0, 9)
    dt = {"bf16": 0, "f32": 1}[dtype]
    whole, _ = attend(backend, c, q, 2 * share, dtype, 0.125)
    backend.synchronize()
    want, _, spread, slack = c.attention(q, 2 * share, 0.125)
    bound = spread * ((2.0 ** -8 if dtype == "bf16" else 0.0) + 2 * (c.dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * HALF[dtype]
    before = c.data.view(torch.uint8).clone()
    for array, at, value in [("table", (1, 3), c.num_pages), ("table", (1, 0), -7), ("table", (1, 12), 2**31 - 1), ("len_dev", 1, 10**6), ("len_dev", 1, -5), ("starts", 3, c.rows + 1)]:
        t = getattr(c, array)
        kept = t[at].clone()
        t[at] = value
        out, _ = attend(backend, c, q, 2 * share, dtype, 0.125)
        with pytest.raises(gpt_b200.GptB200Error) as e:
            backend.synchronize()
        assert e.value.status == 1
        if array != "starts":      # the other sequences are served; with other lengths the line of work is cut elsewhere, so that sums are added in another order
            got = out.double().cpu()
            for s in (0, 2):
                r = slice(s * count, s * count + count)
                assert ((got - want).abs() <= bound)[r].all()
                assert array != "table" or torch.equal(out[r], whole[r])
        ko, vo = torch.empty_like(k), torch.empty_like(k)
        backend.kv_pages_read(ko, ko.stride(0), vo, vo.stride(0), dt, c.pages, c.batch)
        if array != "table" or at[1] * 16 >= lengths[1] - count:
            with pytest.raises(gpt_b200.GptB200Error):
                backend.synchronize()
        t[at] = kept
    backend.synchronize()
    assert torch.equal(c.data.view(torch.uint8), before)
    out, _ = attend(backend, c, q, 2 * share, dtype, 0.125)
    backend.synchronize()
    assert torch.equal(out, whole)


def test_refusals_of_the_calls(backend):
    import gpt_b200
    c = Cache("bf16", [20], [2], 2, 64, 16).cuda()
    q = torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(q)
    kv = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda")

    def refused(call):
        n = backend.launch_count()
        with pytest.raises(gpt_b200.GptB200Error) as e:
            call()
        assert e.value.status == 1 and backend.launch_count() == n

    refused(lambda: backend.attention_paged(out, 255, None, q, 256, 0, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.attention_paged(out, 260, None, q, 256, 0, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.attention_paged(out, 256, None, q, 248, 0, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.attention_paged(out.data_ptr() + 2, 256, None, q, 256, 0, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.attention_paged(out, 256, None, None, 256, 0, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.attention_paged(q, 256, None, q, 256, 0, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.attention_paged(out, 256, None, q, 256, 5, 4, c.pages, c.batch, 0.1))
    refused(lambda: backend.kv_pages_write(c.pages, c.batch, kv, 120, kv, 128, 0))
    refused(lambda: backend.kv_pages_write(c.pages, c.batch, kv, 128, kv.data_ptr() + 8, 128, 0))
    refused(lambda: backend.kv_pages_read(kv, 128, None, 128, 0, c.pages, c.batch))
    refused(lambda: backend.kv_pages_read(kv, 128, kv, 130, 1, c.pages, c.batch))
    for sequences, rows in ((0, 3), (1, 0)):                       # nothing to do: nothing is launched
        empty = gpt_b200.KvRows(c.starts, c.len_dev, c.table, sequences, c.pitch, rows, 1)
        n = backend.launch_count()
        backend.attention_paged(out, 256, None, q, 256, 0, 4, c.pages, empty, 0.1)
        backend.kv_pages_write(c.pages, empty, kv, 128, kv, 128, 0)
        assert backend.launch_count() == n


@pytest.mark.parametrize("dtype,kind", BOTH)
@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 40, 1]])
def test_captured_calls_follow_their_arrays(backend, dtype, kind, counts):
    """A step (write, attend) captured twice, on tables and lengths that change between replays; both graphs share the context's scratch."""
    import gpt_b200
    lengths, heads, dim = [700, 300, 90], 8, 64
    c = Cache(kind, lengths, counts, 2, dim, 16, seed=21, spare=40).cuda()
    dt = {"bf16": 0, "f32": 1}[dtype]
    q, _ = rows_in(c.rows, heads * dim, dtype, 0, 8)
    k, k_cpu = rows_in(c.rows, 2 * dim, dtype, 0, 9)
    v, v_cpu = rows_in(c.rows, 2 * dim, dtype, 0, 10)
    side = torch.cuda.Stream()
    be = gpt_b200.Backend(0, side.cuda_stream)
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    torch.cuda.synchronize()
    for out, cap in zip(outs, (0.0, 30.0)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            be.kv_pages_write(c.pages, c.batch, k, k.stride(0), v, v.stride(0), dt)
            be.attention_paged(out, out.stride(0), None, q, q.stride(0), dt, heads, c.pages, c.batch, 0.2, cap)
        graphs.append(g)
    free = [p for p in range(c.num_pages) if p not in c.used]
    for turn in range(3):
        if turn:   # every sequence one token longer, a page more where it needs one; the first one's pages change places
            for s in range(3):
                at = c.lengths[s] // 16
                if c.lengths[s] % 16 == 0:
                    c.table_cpu[s, at] = free.pop()
                c.lengths[s] += 1
            a, b = int(c.table_cpu[0, 1]), int(c.table_cpu[0, 2])
            c.table_cpu[0, 1], c.table_cpu[0, 2] = b, a
            torch.cuda.synchronize()
            c.len_dev.copy_(torch.tensor(c.lengths, dtype=torch.int32))
            c.table.copy_(c.table_cpu)
        for g in graphs:
            with torch.cuda.stream(side):
                g.replay()
        be.synchronize()
        c.data_cpu = c.data.cpu()
        c.values = c.data_cpu.double() if kind != "e4m3" else torch.ldexp(c.data_cpu.float().double(), c.scales.cpu()[..., None].int() - 127)
        for s, page, token in [(r, p, t) for r, p, t in places(c)]:
            x = k_cpu[s].double().reshape(2, dim)
            want = x.to(c.TYPES[kind]).double() if kind != "e4m3" else torch.ldexp(codes_of(x)[0], codes_of(x)[1][:, None].int() - 127)
            assert torch.equal(c.values[page, 0, :, token], want)
        for out, cap in zip(outs, (0.0, 30.0)):
            want, _, spread, slack = c.attention(q, heads, 0.2, cap)
            bound = spread * ((2.0 ** -8 if dtype == "bf16" else 0.0) + 2 * (dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * HALF[dtype]
            assert ((out.double().cpu() - want).abs() <= bound + 1e-30).all()
    del graphs
    be.close()


def test_pools_beyond_two_to_the_31_elements(backend):
    """Pages at the far end of a pool of more than 2^32 bytes, in bf16 and e4m3, for single tokens and a prompt."""
    for kind, dtype, pages in (("bf16", torch.bfloat16, 2100), ("e4m3", torch.float8_e4m3fn, 4200)):
        for count in (1, 70):
            small = Cache(kind, [500, 90], [count, count], 4, 128, 1024, seed=5)
            data = torch.zeros(pages, 2, 4, 1024, 128, dtype=torch.uint8 if kind == "e4m3" else dtype, device="cuda")
            assert data.numel() > 2 ** 31
            n = small.num_pages
            data[-n:] = (small.data_cpu.view(torch.uint8) if kind == "e4m3" else small.data_cpu).cuda()
            scales = torch.zeros(pages, 2, 4, 1024, dtype=torch.uint8, device="cuda") if kind == "e4m3" else None
            if scales is not None:
                scales[-n:] = small.scales_cpu.cuda()
            big = Cache(kind, [500, 90], [count, count], 4, 128, 1024, seed=5)
            big.cuda()
            import gpt_b200
            big.data, big.scales = data.view(torch.float8_e4m3fn) if kind == "e4m3" else data, scales
            big.table = (big.table_cpu + (big.table_cpu >= 0) * (pages - n)).int().cuda()
            big.pages = gpt_b200.KvPages(big.data, scales, Cache.KINDS[kind], pages, 1024, 4, 128)
            big.batch = gpt_b200.KvRows(big.starts, big.len_dev, big.table, 2, big.pitch, big.rows, count)
            q, _ = rows_in(big.rows, 8 * 128, "bf16", 0, 5)
            out, sums = attend(backend, big, q, 8, "bf16", 0.1)
            backend.synchronize()
            check(big, q, out, sums, 8, "bf16", 0.1)
            del data, scales, big
            torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,kind,heads,dim,window,sinks", [("f32", "f32", 12, 64, 0, 0), ("bf16", "e4m3", 8, 128, 60, 4), ("bf16", "bf16", 4, 40, 0, 0)])
def test_a_served_batch(backend, dtype, kind, heads, dim, window, sinks):
    """Prompts in portions, then single tokens, sequences joining and leaving: every step writes its rows and attends over the pages; at the end the cache is read back."""
    import gpt_b200
    g = torch.Generator().manual_seed(13)
    kv_heads, page, num = 4, 16, 60
    dt = {"bf16": 0, "f32": 1}[dtype]
    data = torch.zeros(num, 2, kv_heads, page, dim, dtype=Cache.TYPES[kind] if kind != "e4m3" else torch.uint8, device="cuda")
    scales = torch.zeros(num, 2, kv_heads, page, dtype=torch.uint8, device="cuda") if kind == "e4m3" else None
    pool = gpt_b200.KvPages(data, scales, Cache.KINDS[kind], num, page, kv_heads, dim)
    free, tables, history = list(range(num)), {}, {}
    plan = [{0: 50, 1: 7}, {0: 50, 1: 1}, {0: 1, 1: 1, 2: 33}, {1: 1, 2: 1}, {1: 40, 3: 5}, {1: 1, 3: 1, 2: 1}]
    for turn, step in enumerate(plan):
        if turn == 3:
            free += tables.pop(0)
            history.pop(0)
        order = sorted(step)
        for s in order:
            tables.setdefault(s, [])
            history.setdefault(s, [torch.empty(0, kv_heads, dim, dtype=torch.float64) for _ in (0, 1)])
            while len(tables[s]) * page < history[s][0].shape[0] + step[s]:
                tables[s].append(free.pop(0))
        rows = sum(step.values())
        x = [torch.randn(rows, n * dim, generator=g).to(TYPES[dtype]) for n in (kv_heads, kv_heads, heads)]
        at = 0
        for s in order:
            for which in (0, 1):
                new = x[which][at:at + step[s]].double().reshape(-1, kv_heads, dim)
                if kind == "e4m3":
                    codes, e = codes_of(new)
                    new = torch.ldexp(codes, e[..., None].int() - 127)
                history[s][which] = torch.cat([history[s][which], new])
            at += step[s]
        width = max(len(tables[s]) for s in order)
        table = torch.tensor([tables[s] + [-1] * (width - len(tables[s])) for s in order], dtype=torch.int32).cuda()
        lengths = torch.tensor([history[s][0].shape[0] for s in order], dtype=torch.int32).cuda()
        starts = torch.tensor([0] + [step[s] for s in order]).cumsum(0).int().cuda()
        batch = gpt_b200.KvRows(starts, lengths, table, len(order), width, rows, max(step.values()))
        k, v, q = (t.cuda() for t in x)
        out = torch.empty_like(q)
        backend.kv_pages_write(pool, batch, k, k.stride(0), v, v.stride(0), dt)
        backend.attention_paged(out, out.stride(0), None, q, q.stride(0), dt, heads, pool, batch, dim ** -0.5, 0.0, window, sinks)
        backend.synchronize()
        at = 0
        for s in order:
            dense = Cache.__new__(Cache)
            n, length = step[s], history[s][0].shape[0]
            dense.kv_heads, dense.dim, dense.page, dense.lengths, dense.counts = kv_heads, dim, length, [length], [n]
            dense.starts_cpu, dense.table_cpu, dense.rows = torch.tensor([0, n]), torch.zeros(1, 1, dtype=torch.int32), n
            dense.values = torch.stack([h.permute(1, 0, 2) for h in history[s]])[None]
            want, _, spread, slack = dense.attention(x[2][at:at + n], heads, dim ** -0.5, 0.0, window, sinks)
            bound = spread * ((2.0 ** -8 if dtype == "bf16" else 0.0) + 2 * (dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * HALF[dtype]
            assert ((out[at:at + n].double().cpu() - want).abs() <= bound + 1e-30).all()
            at += n
    order = sorted(history)
    width = max(len(tables[s]) for s in order)
    table = torch.tensor([tables[s] + [-1] * (width - len(tables[s])) for s in order], dtype=torch.int32).cuda()
    counts = [history[s][0].shape[0] for s in order]
    starts, lengths = torch.tensor([0] + counts).cumsum(0).int().cuda(), torch.tensor(counts, dtype=torch.int32).cuda()
    batch = gpt_b200.KvRows(starts, lengths, table, len(order), width, sum(counts), max(counts))
    k, v = (torch.empty(sum(counts), kv_heads * dim, device="cuda") for _ in (0, 1))
    backend.kv_pages_read(k, k.stride(0), v, v.stride(0), 1, pool, batch)
    backend.synchronize()
    for which, got in ((0, k), (1, v)):
        assert torch.equal(got.double().cpu(), torch.cat([history[s][which] for s in order]).reshape(sum(counts), -1).to(torch.float32).double())


@pytest.mark.parametrize("dtype,kind", [("f32", "f32"), ("f32", "e4m3"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("lengths,counts,kv_heads,share,dim,page,cap,window,sinks", [
    ([700, 90, 3], [333, 90, 1], 2, 4, 128, 16, 0.0, 50, 5),
    ([513, 60], [513, 1], 1, 8, 80, 64, 40.0, 0, 0),
    ([6000], [20], 1, 8, 64, 32, 0.0, 0, 0),           # a tile's parts lie all over the grid
    ([40, 41, 31], [33, 9, 31], 1, 8, 8, 8, 0.0, 0, 0),
])
def test_wide_tiles_on_fmas(backend, lengths, counts, kv_heads, share, dim, page, cap, window, sinks, dtype, kind):
    """Calls of many rows of all heads, though most of them may lie behind the last sequence."""
    import gpt_b200
    c = Cache(kind, lengths, counts, kv_heads, dim, page, seed=dim, extra_rows=520, poison=True)
    c.cuda(max_new=max(counts))
    heads, scale = kv_heads * share, dim ** -0.5
    assert gpt_b200.plan_attention_paged(148, {"bf16": 0, "f32": 1}[dtype], heads, c.pages, c.batch, scale, cap, window, sinks)["tile_rows"] == 32
    q, _ = rows_in(c.rows, heads * dim, dtype, 8, 5, scale=2.0)
    out, sums = attend(backend, c, q, heads, dtype, scale, cap, window, sinks, extra=8)
    backend.synchronize()
    check(c, q, out, sums, heads, dtype, scale, cap, window, sinks)
    # a value that is not finite, seen by the last row of a sequence alone
    last, c.values = int(c.table_cpu[0, (lengths[0] - 1) // page]), c.values.clone()
    data = c.data.float()
    data[last, 1, :, (lengths[0] - 1) % page, 5] = float("nan")
    c.data.copy_(data.to(c.data.dtype))
    c.values[last, 1, :, (lengths[0] - 1) % page, 5] = float("nan")
    out, sums = attend(backend, c, q, heads, dtype, scale, cap, window, sinks, extra=8)
    backend.synchronize()
    want, got = c.attention(q, heads, scale, cap, window, sinks)[0], out.double().cpu()
    end = sum(counts)
    assert torch.equal(torch.isnan(got[:end]), torch.isnan(want[:end])) and torch.isnan(want[counts[0] - 1]).any() and not torch.isnan(want[:counts[0] - 1]).any()
