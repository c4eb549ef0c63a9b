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
