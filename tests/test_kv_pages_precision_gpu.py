"""How many bits attention over a paged cache keeps, kernel by kernel, against plain torch in 64 bits.

Tolerances.  With A = sum_j p_j |v_j| and B = the largest sum_d |q_d k_jd| * scale of the row, an output is off by at most
    A * (w + 2 * (dim + 8) * 2^-23 * B + 2^-17) + |out| * h [+ a]
where the second summand is that of fp32 scores in any order (the tensor core's truncating sums count twice), 2^-17 that of approximate exponentials, caps and sums of
some thousand terms, h the output's own rounding (2^-8 bf16, 2^-24 fp32) and w that of the weights, by the kernel that runs:
    few rows over bf16 pages   two bf16 terms, each off by half a step of what it holds: 2^-8 * 2^-8 = 2^-16
    few rows over codes        two fp16 terms: 2^-11 * 2^-11 = 2^-22; besides a = 2^-36 * 448 for every key, times the row's largest p_j 2^(e_j): the second term's
                               smallest step is 2^-24 where the largest weight is 2^11 at least
                               Queries are fp16, the row's largest in [2^15, 2^16) of it (a bf16 number below 2^16 is exact): an element is off by half of fp16's smallest
                               step at most, 2^-25 = 2^-40 * 2^15, a score by 2^-40 * max_d |q_d| * sum_d |k_jd| * scale = C, and an output, whose weights and sum are
                               off by that share, by A * 2 * C
    prompts                    one bf16 term: 2^-8, and as much for their sum
    fp32 FMAs                  0
"""
import pytest
import torch

from paged_cache import Cache, codes_of
from test_kv_pages_gpu import ATTEND, TYPES, attend, backend, rows_in   # noqa: F401 (backend is a fixture)

pytestmark = pytest.mark.gpu

DT = {"bf16": 0, "f32": 1}


def kernel_of(c, heads, dtype, scale, cap=0.0, window=0, sinks=0):
    import gpt_b200
    return gpt_b200.plan_attention_paged(148, DT[dtype], heads, c.pages, c.batch, scale, cap, window, sinks)["kernel"]


def bound_of(c, q, heads, dtype, scale, cap=0.0, window=0, sinks=0):
    want, lse, spread, slack = c.attention(q, heads, scale, cap, window, sinks)
    kernel = kernel_of(c, heads, dtype, scale, cap, window, sinks)
    weight = {"tokens": 2.0 ** -22 if c.kind == "e4m3" else 2.0 ** -16, "prompt": 2.0 ** -7, "few": 0.0, "rows": 0.0}[kernel]
    bound = spread * (weight + 2 * (c.dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24)
    if kernel == "tokens" and c.kind == "e4m3":
        bound = bound + 2.0 ** -36 * 448 * vanishing(c, q, heads, scale, cap, window, sinks).repeat_interleave(c.dim, 1) + 2 * spread * lost(c, q, heads, scale).repeat_interleave(c.dim, 1)
    return want, lse, bound, slack


def lost(c, q, heads, scale):
    """[rows, heads]: 2^-40 * max_d |q_d| * sum_d |k_jd| * scale, for the largest key of the row's sequence and head."""
    most = q.double().cpu().reshape(-1, heads, c.dim).abs().amax(2)
    keys = torch.zeros_like(most)
    for s, n in enumerate(c.counts):
        k = c.sequence(s)[0]
        if n and k.shape[1]:
            r0 = int(c.starts_cpu[s])
            keys[r0:r0 + n] = torch.nan_to_num(k).abs().sum(2).amax(1).repeat_interleave(heads // c.kv_heads)
    return 2.0 ** -40 * most * keys * scale


def vanishing(c, q, heads, scale, cap, window, sinks):
    """[rows, heads]: visible keys times the largest p_j 2^(e_j) among them."""
    q = q.double().cpu().reshape(-1, heads, c.dim)
    got, share = torch.zeros(q.shape[0], heads, dtype=torch.float64), heads // c.kv_heads
    for s, n in enumerate(c.counts):
        length, r0 = max(c.lengths[s], 0), int(c.starts_cpu[s])
        keys = c.sequence(s)[0]
        ids = c.table_cpu[s, :-(-length // c.page)].long()
        powers = torch.exp2(c.scales_cpu[ids, 1].double() - 127.0).permute(1, 0, 2).reshape(c.kv_heads, -1)[:, :length]
        for i in range(n):
            at = length - n + i
            if at < 0:
                continue
            key = torch.arange(length)
            seen = (key <= at) & ((at - key < window) | (key < sinks) if window else key >= 0)
            for h in range(heads):
                x = keys[h // share][seen] @ q[r0 + i, h] * scale
                if cap:
                    x = cap * torch.tanh(x / cap)
                got[r0 + i, h] = seen.sum() * (torch.softmax(x, 0) * powers[h // share][seen]).max()
    return got


def check(c, q, out, sums, heads, dtype, scale, cap=0.0, window=0, sinks=0):
    want, lse, bound, slack = bound_of(c, q, heads, dtype, scale, cap, window, sinks)
    end, got = int(c.starts_cpu[-1]), out.double().cpu()
    off = (got - want).abs()[:end]
    assert torch.isfinite(want[:end]).all() and torch.isfinite(got[:end]).all()
    assert (off <= bound[:end] + 1e-30).all(), float((off / (bound[:end] + 1e-30)).max())
    if sums is not None:
        s, per_row = sums.double().cpu()[:end], slack.reshape(c.rows, heads, -1)[:end, :, 0]
        empty = torch.isinf(lse[:end])
        assert (((s - lse[:end]).abs() <= 2 * (c.dim + 8) * 2.0 ** -23 * per_row + 2.0 ** -17 * (1 + lse[:end].abs())) | empty).all()


def held(kind, k, v, page=16, counts=(1,), extra=0):
    """A cache of one sequence whose keys and values [length, kv heads, dim] are given (float64)."""
    length, kv_heads, dim = k.shape
    c = Cache(kind, [length], list(counts), kv_heads, dim, page, seed=1, extra_rows=extra)
    for which, x in ((0, k), (1, v)):
        where, token = c.table_cpu[0, torch.arange(length) // page].long(), torch.arange(length) % page
        if kind == "e4m3":
            codes, e = codes_of(x)
            data = c.data_cpu.float()
            data[where, which, :, token] = codes.float()
            c.data_cpu, c.scales_cpu[where, which, :, token] = data.to(torch.float8_e4m3fn), e
            c.values[where, which, :, token] = torch.ldexp(codes, e[..., None].int() - 127)
        else:
            c.data_cpu[where, which, :, token] = x.to(c.TYPES[kind])
            c.values[where, which, :, token] = x.to(c.TYPES[kind]).double()
    return c.cuda()


KINDS = [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32"), ("f32", "e4m3"), ("bf16", "f32")]


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("lengths,counts,kv_heads,share,dim,page,cap,window,sinks", ATTEND)
def test_every_shape_within_the_bits_of_its_kernel(backend, lengths, counts, kv_heads, share, dim, page, cap, window, sinks, dtype, kind):
    c = Cache(kind, lengths, counts, kv_heads, dim, page, seed=dim + len(lengths)).cuda()
    heads, scale = kv_heads * share, dim ** -0.5
    q, _ = rows_in(c.rows, heads * dim, dtype, 0, 5, scale=2.0)
    out, sums = attend(backend, c, q, heads, dtype, scale, cap, window, sinks)
    backend.synchronize()
    check(c, q, out, sums, heads, dtype, scale, cap, window, sinks)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("share", [1, 8, 16])
@pytest.mark.parametrize("gap", [12.0, 18.0, 21.0])
def test_many_small_weights_beside_a_large_one(backend, dtype, kind, share, gap):
    """The first key has nearly all of the weight and one dimension to itself; three thousand others, 2^-17 to 2^-30 of it each, are all that the other dimensions have."""
    length, dim = 3001, 64
    k, v = torch.zeros(length, 1, dim, dtype=torch.float64), torch.zeros(length, 1, dim, dtype=torch.float64)
    k[0, 0, 0] = 8.0
    v[0, 0, 0] = 448.0
    v[1:, 0, 1:] = 448.0 * torch.rand(length - 1, dim - 1, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    v[1:, 0, 1] = 448.0
    c = held(kind, k, v)
    q = torch.zeros(1, share * dim, dtype=TYPES[dtype], device="cuda")
    q[:, ::dim] = 1.0
    out, sums = attend(backend, c, q, share, dtype, gap / 8.0)
    backend.synchronize()
    check(c, q, out, sums, share, dtype, gap / 8.0)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("count,share", [(1, 1), (1, 8), (2, 8)])
@pytest.mark.parametrize("apart", [2.0 ** -18, 2.0 ** -24, 2.0 ** -30])
def test_small_queries_beside_a_large_one(backend, dtype, kind, count, share, apart):
    """Dimension 0 of every query is large and meets only zeros; the scores are the others', far smaller ones times large keys."""
    length, dim, g = 200, 64, torch.Generator().manual_seed(3)
    k = torch.randn(length, 1, dim, generator=g, dtype=torch.float64) / apart
    k[:, :, 0] = 0.0
    c = held(kind, k, torch.randn(length, 1, dim, generator=g, dtype=torch.float64), counts=(count,))
    x = 2.0 * apart * torch.randn(count, share, dim, generator=g, dtype=torch.float64)
    x[:, :, 0] = 1.5
    q = x.reshape(count, -1).to(TYPES[dtype]).cuda()
    out, sums = attend(backend, c, q, share, dtype, dim ** -0.5)
    backend.synchronize()
    check(c, q, out, sums, share, dtype, dim ** -0.5)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("count,share", [(1, 1), (1, 8), (2, 8)])
def test_values_that_cancel(backend, dtype, kind, count, share):
    """Two keys with nearly the same weight and opposite values: what is left is the difference of the weights."""
    dim = 64
    k, v = torch.zeros(2, 1, dim, dtype=torch.float64), torch.ones(2, 1, dim, dtype=torch.float64)
    k[1, 0, :share] = torch.arange(8, 8 + share, dtype=torch.float64) / 8.0    # 1 to 2.875: exact in every kind
    v[1] = -1.0
    c = held(kind, torch.cat([k, k[1:]]) if count == 2 else k, torch.cat([v, v[1:]]) if count == 2 else v, counts=(count,))
    x = torch.zeros(count, share, dim)
    x[:, range(share), range(share)] = 1.0
    q = x.reshape(count, -1).to(TYPES[dtype]).cuda()
    out, sums = attend(backend, c, q, share, dtype, 0.003)
    backend.synchronize()
    check(c, q, out, sums, share, dtype, 0.003)


@pytest.mark.parametrize("power", [-120, -60, 60, 110])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_queries_and_keys_of_any_size(backend, kind, power):
    """Queries of 2^power against keys of 2^-power: the scores are ordinary ones."""
    length, dim, share, g = 100, 64, 8, torch.Generator().manual_seed(4)
    c = held(kind, torch.randn(length, 1, dim, generator=g, dtype=torch.float64) * 2.0 ** -power, torch.randn(length, 1, dim, generator=g, dtype=torch.float64))
    q = (torch.randn(1, share * dim, generator=g) * 2.0 ** power).to(torch.bfloat16).cuda()
    out, sums = attend(backend, c, q, share, "bf16", dim ** -0.5)
    backend.synchronize()
    check(c, q, out, sums, share, "bf16", dim ** -0.5)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("count,share", [(4, 2), (64, 1), (300, 4)])
@pytest.mark.parametrize("cap", [20.0, 2.0 ** 10, 2.0 ** 17])
def test_scores_far_below_the_cap_beside_those_beyond_it(backend, dtype, kind, count, share, cap):
    """Every third row's scores are many times the cap; the others' are ordinary ones, and as exact as without those."""
    length, dim, g = count + 200, 64, torch.Generator().manual_seed(5)
    c = held(kind, torch.randn(length, 1, dim, generator=g, dtype=torch.float64), torch.randn(length, 1, dim, generator=g, dtype=torch.float64), counts=(count,))
    x = torch.randn(count, share * dim, generator=g)
    x[::3] *= 8.0 * cap
    q = x.to(TYPES[dtype]).cuda()
    out, sums = attend(backend, c, q, share, dtype, dim ** -0.5, cap)
    backend.synchronize()
    check(c, q, out, sums, share, dtype, dim ** -0.5, cap)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("query,key", [(2.0 ** 125, 2.0 ** -115), (2.0 ** 120, 2.0 ** -118), (2.0 ** -118, 2.0 ** 115), (2.0 ** -110, 2.0 ** 119)])
def test_queries_and_keys_at_the_ends_of_the_range(backend, kind, query, key):
    """Scores of ordinary size: the scale takes what the two leave."""
    length, dim, share, g = 100, 64, 8, torch.Generator().manual_seed(4)
    scale = 2.0 ** -3 / (query * key)
    c = held(kind, torch.randn(length, 1, dim, generator=g, dtype=torch.float64) * key, torch.randn(length, 1, dim, generator=g, dtype=torch.float64))
    q = (torch.randn(1, share * dim, generator=g).clamp(-1.9, 1.9) * query).to(torch.bfloat16).cuda()
    out, sums = attend(backend, c, q, share, "bf16", scale)
    backend.synchronize()
    check(c, q, out, sums, share, "bf16", scale)
