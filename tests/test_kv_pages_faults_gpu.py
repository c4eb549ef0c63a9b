"""Batches on which attention over a paged cache could lose results: tiles that one half of a block works on alone, values that are not finite, arrays that do not fit."""
import pytest
import torch

from paged_cache import Cache
from test_kv_pages_gpu import attend, backend, rows_in   # noqa: F401 (backend is a fixture)
from test_kv_pages_gpu import check as check_wide
from test_kv_pages_precision_gpu import check

pytestmark = pytest.mark.gpu


def put(c, kind, s, position, value, which=1, heads=slice(None), element=5):
    """A key's (0) or value's (1) element of a sequence's token, in the cache and in its 64-bit form."""
    page, token = int(c.table_cpu[s, position // c.page]), position % c.page
    data = c.data_cpu.float()
    data[page, which, heads, token, element] = value
    c.data_cpu = data.to(c.TYPES[kind])
    c.values[page, which, heads, token, element] = float("nan") if kind == "e4m3" else value


NARROW = [  # lengths, counts, share: tiles of 256 rows; those of up to 128 have no rows for the second half of a block
    ([300, 40, 50, 60, 30, 20], [64, 32, 32, 32, 16, 8], 4),
    ([300, 40, 50, 300, 30, 300], [64, 20, 32, 64, 16, 60], 4),
    ([2000, 9, 9, 9, 9, 2000, 9, 9, 9], [200, 9, 9, 9, 9, 100, 9, 9, 9], 2),
    ([10, 40, 3, 300, 100, 90], [64, 64, 64, 64, 32, 32], 4),          # more new rows than tokens: first halves that see nothing
    ([0, 0, 0, 200, 0, 0], [64, 64, 30, 64, 64, 20], 4),
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("blocks", [1, 2, 0])
@pytest.mark.parametrize("lengths,counts,share", NARROW)
def test_tiles_of_one_half(backend, lengths, counts, share, blocks, kind):
    c = Cache(kind, lengths, counts, 2, 64, 16, seed=len(lengths)).cuda()
    heads = 2 * share
    q, _ = rows_in(c.rows, heads * 64, "bf16", 0, 5)
    backend.set_option("max_sms", blocks)
    try:
        for _ in range(3):
            out, sums = attend(backend, c, q, heads, "bf16", 0.125)
            backend.synchronize()
            check(c, q, out, sums, heads, "bf16", 0.125)
    finally:
        backend.set_option("max_sms", 0)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("bad_rows", [1, 40])
def test_rows_formed_again_beside_tiles_of_one_half(backend, kind, bad_rows):
    """The last rows of a tile see a value that is not finite, so that the second half's other rows are formed again while the first half goes on to narrow tiles."""
    lengths, counts, share = [3000, 40, 50, 30, 20, 40, 10], [64, 32, 32, 16, 20, 20, 10], 4
    c = Cache(kind, lengths, counts, 1, 64, 16, seed=3)
    put(c, kind, 0, lengths[0] - bad_rows, float("nan"))
    c.cuda()
    q, _ = rows_in(c.rows, share * 64, "bf16", 0, 5)
    backend.set_option("max_sms", 1)
    try:
        out, sums = attend(backend, c, q, share, "bf16", 0.125)
        backend.synchronize()
    finally:
        backend.set_option("max_sms", 0)
    check_wide(c, q, out, sums, share, "bf16", 0.125)
    got = out.double().cpu()
    assert torch.isnan(got[64 - bad_rows:64, 5::64]).all() and torch.isfinite(got[:64 - bad_rows]).all() and torch.isfinite(got[64:]).all()


def kinds(x):
    """0 finite, 1 NaN, 2 infinite, 3 minus infinite."""
    return torch.where(torch.isnan(x), 1, torch.where(torch.isposinf(x), 2, torch.where(torch.isneginf(x), 3, 0)))


def kinds_by_definition(c, heads, window, sinks):
    """[rows, heads, dim] of the outputs, from the values that each row sees (all scores finite): every weight is positive."""
    want = torch.zeros(c.rows, heads, c.dim, dtype=torch.int64)
    for s, n in enumerate(c.counts):
        length, r0 = c.lengths[s], int(c.starts_cpu[s])
        v = c.sequence(s)[1]
        key = torch.arange(length)
        for i in range(n):
            at = length - n + i
            seen = (key <= at) & ((at - key < window) | (key < sinks) if window else key >= 0)
            x = v[:, seen]
            nan, high, low = torch.isnan(x).any(1), torch.isposinf(x).any(1), torch.isneginf(x).any(1)
            kind = torch.where(nan | (high & low), 1, torch.where(high, 2, torch.where(low, 3, 0)))
            want[r0 + i] = kind.repeat_interleave(heads // c.kv_heads, 0)
    return want.reshape(c.rows, -1)


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32"), ("f32", "e4m3"), ("bf16", "f32")])
@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 2, 1], [40, 1, 33], [200, 100, 7]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
def test_kinds_of_what_is_not_finite(backend, dtype, kind, counts, window, sinks):
    """NaN and infinities at first, old, new and last tokens of a batch: an output is of the kind that the values its row sees make it, and all others are right."""
    inf, nan = float("inf"), float("nan")
    lengths, dim, heads = [400, 300, 40], 64, 4
    c = Cache(kind, lengths, counts, 2, dim, 16, seed=3)
    spots = [(0, 0, 0, inf), (0, 3, 1, -inf), (0, 200, 2, nan), (0, 399, 3, nan), (0, 390, 4, inf), (0, 392, 4, -inf), (0, 398, 6, inf), (1, 1, 7, nan), (1, 4, 63, -inf), (1, 299, 62, inf), (1, 270, 9, inf),
             (1, 230, 9, -inf), (1, 231, 10, inf), (0, 321, 11, nan), (0, 320, 11, inf)]
    for s, position, element, value in spots:
        put(c, kind, s, position, value, heads=position % 2, element=element)
    c.cuda()
    q, _ = rows_in(c.rows, heads * dim, dtype, 0, 8)
    out, sums = attend(backend, c, q, heads, dtype, 0.125, 0.0, window, sinks)
    backend.synchronize()
    got = out.double().cpu()
    assert torch.equal(kinds(got), kinds_by_definition(c, heads, window, sinks))
    # without them, where rows are finite: the same
    for s, position, element, value in spots:
        put(c, kind, s, position, 0.0, heads=position % 2, element=element)
    c.values[torch.isnan(c.values)] = 0.0
    want, lse, spread, slack = c.attention(q, heads, 0.125, 0.0, window, sinks)
    bound = spread * (2.0 ** -7 + 2 * (dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24)
    fine = torch.isfinite(got)
    assert ((got - want).abs() <= bound + 1e-30)[fine].all()
    assert ((sums[:c.rows].double().cpu() - lse).abs() <= 2 * (dim + 8) * 2.0 ** -23 * slack.reshape(c.rows, heads, -1)[:, :, 0] + 2.0 ** -17 * (1 + lse.abs())).all()


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("count,share", [(1, 1), (1, 8), (2, 8), (40, 2), (300, 1)])
def test_sums_that_would_leave_the_range(backend, dtype, kind, count, share):
    """Weights stand against a first score that later ones exceed by a factor of e^19, and values near the type's largest are multiplied by them: the outputs are in range."""
    length, dim = 300 + count, 64
    c = Cache(kind, [length], [count], 1, dim, 16, seed=3)
    for position in range(length):
        page, token = int(c.table_cpu[0, position // 16]), position % 16
        row = torch.zeros(2, dim)
        row[0, 0] = 0.0 if position == 0 else 19.0 if position in (20, 170) else -40.0
        row[1] = 2.0 ** 125 if position in (20, 170) else 1.0
        c.data_cpu[page, :, 0, token] = row.to(c.TYPES[kind])
        c.values[page, :, 0, token] = row.double()
    c.cuda()
    q = torch.zeros(count, share * dim, dtype=torch.bfloat16 if dtype == "bf16" else torch.float32, device="cuda")
    q[:, ::dim] = 1.0
    out, sums = attend(backend, c, q, share, dtype, 1.0)
    backend.synchronize()
    check(c, q, out, sums, share, dtype, 1.0)


def least_ms(call, turns=8):
    """The shortest of some calls' times."""
    begin, end, got = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True), []
    for _ in range(turns):
        begin.record()
        call()
        end.record()
        end.synchronize()
        got.append(begin.elapsed_time(end))
    return min(got)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("which,position,value", [(1, 0, float("nan")), (0, 0, float("nan")), (1, 0, float("inf")), (1, 8191, float("nan"))])
def test_a_poisoned_prompt_beside_a_healthy_one(backend, kind, which, position, value):
    """What a row sees makes it NaN or infinite: it is not formed again for that, the other sequence is as it was, and the call takes no more than twice the time."""
    heads, dim, lengths = 32, 128, [8192, 2000]
    c = Cache(kind, lengths, lengths, 8, dim, 64, seed=3).cuda()
    q, _ = rows_in(c.rows, heads * dim, "bf16", 0, 8)
    out = torch.empty_like(q)
    call = lambda: backend.attention_paged(out, out.stride(0), None, q, q.stride(0), 0, heads, c.pages, c.batch, dim ** -0.5)   # noqa: E731
    healthy = least_ms(call)
    clean = out.clone()
    page, token = int(c.table_cpu[0, position // 64]), position % 64
    value = float("nan") if kind == "e4m3" else value
    if kind == "e4m3":
        c.data.view(torch.uint8)[page, which, :, token, 5] = 0x7f
    else:
        c.data[page, which, :, token, 5] = value
    poisoned = least_ms(call)
    backend.synchronize()
    assert torch.equal(out[8192:], clean[8192:])
    mine, before = out[:8192].reshape(8192, heads, dim), clean[:8192].reshape(8192, heads, dim)
    if which == 0:
        assert torch.isnan(mine[position:]).all() and torch.equal(mine[:position], before[:position])
    else:
        sees = mine[position:, :, 5]
        assert torch.isnan(sees).all() if value != value else (sees == value).all()
        if position == 0:
            keep = [d for d in range(dim) if d != 5]
            assert torch.equal(mine[:, :, keep], before[:, :, keep])
        else:       # rows of the last tiles that do not see it were formed again, in fp32: off by the weights' rounding
            keep = torch.ones_like(mine, dtype=torch.bool)
            keep[position:, :, 5] = False
            assert torch.isfinite(mine[keep]).all() and ((mine - before).abs()[keep] <= 2.0 ** -7 * before.abs()[keep] + 2.0 ** -6).all()
    print(f"{kind} {which} {position} {value}: healthy {healthy * 1e3:.0f} us, poisoned {poisoned * 1e3:.0f} us")
    if position == 0:
        assert poisoned <= 2.0 * healthy, (poisoned, healthy)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("position,value", [(0, float("nan")), (30000, float("nan")), (30000, float("inf"))])
def test_poisoned_tokens_beside_healthy_ones(backend, kind, position, value):
    heads, dim, lengths = 16, 128, [40000, 50000, 7, 20000]
    c = Cache(kind, lengths, [1] * 4, 4, dim, 64, seed=3).cuda()
    q, _ = rows_in(c.rows, heads * dim, "bf16", 0, 8)
    out = torch.empty_like(q)
    call = lambda: backend.attention_paged(out, out.stride(0), None, q, q.stride(0), 0, heads, c.pages, c.batch, dim ** -0.5)   # noqa: E731
    healthy = least_ms(call)
    clean = out.clone()
    page, token = int(c.table_cpu[0, position // 64]), position % 64
    value = float("nan") if kind == "e4m3" else value
    if kind == "e4m3":
        c.data.view(torch.uint8)[page, 1, :, token, 5] = 0x7f
    else:
        c.data[page, 1, :, token, 5] = value
    poisoned = least_ms(call)
    backend.synchronize()
    assert torch.equal(out[1:], clean[1:])
    sees = out[0].reshape(heads, dim)[:, 5]
    assert torch.isnan(sees).all() if value != value else (sees == value).all()
    keep = [d for d in range(dim) if d != 5]
    off = (out[0].reshape(heads, dim)[:, keep].float() - clean[0].reshape(heads, dim)[:, keep].float()).abs()
    assert (off <= 2.0 ** -7 * clean[0].reshape(heads, dim)[:, keep].float().abs() + 2.0 ** -12).all()
    print(f"{kind} {position} {value}: healthy {healthy * 1e3:.0f} us, poisoned {poisoned * 1e3:.0f} us")


def test_rows_formed_again_for_longer_than_a_wait_may_take(backend):
    """The last of 64 new tokens behind 400 000 others holds a NaN that the 63 before it do not see: all of theirs are formed again, which takes a second or so, while the other warps wait."""
    length, count, share, dim = 400000, 64, 4, 64
    c = Cache("bf16", [length, 50], [count, 20], 1, dim, 64, seed=3)
    want, _, spread, slack = c.attention(rows_in(count + 20, share * dim, "bf16", 0, 8)[0], share, 0.125)
    page, token = int(c.table_cpu[0, (length - 1) // 64]), (length - 1) % 64
    c.data_cpu[page, 1, :, token, 5] = float("nan")
    c.cuda()
    q, _ = rows_in(c.rows, share * dim, "bf16", 0, 8)
    out = torch.empty_like(q)
    took = least_ms(lambda: backend.attention_paged(out, out.stride(0), None, q, q.stride(0), 0, share, c.pages, c.batch, 0.125), 1)
    backend.synchronize()
    print(f"{took:.0f} ms")
    got = out.double().cpu()
    assert torch.isnan(got[count - 1, 5::64]).all()
    bound = spread * (2.0 ** -7 + 2 * (dim + 8) * 2.0 ** -23 * slack + 2.0 ** -17) + want.abs() * 2.0 ** -8
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[count - 1, 5::64] = False
    assert ((got - want).abs() <= bound)[keep].all()


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("count", [1, 40, 300])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("entry", [-1, -2**31, 2**31 - 1, "past"])
def test_a_page_that_is_none_brings_in_no_other(backend, dtype, kind, count, page, entry):
    """An entry of the table that names no page of the pool: nothing of the pool's pages that the sequence does not own takes part, whatever they hold."""
    import gpt_b200
    lengths, dim = [1200, 700], 64
    seed = next(s for s in range(100) if not {0} & set(Cache(kind, lengths, [count] * 2, 2, 8, page, seed=s).used))
    c = Cache(kind, lengths, [count] * 2, 2, dim, page, seed=seed)
    foreign = [p for p in range(c.num_pages) if p not in c.used]
    assert 0 in foreign
    c.cuda()
    c.table[0, 1] = c.num_pages if entry == "past" else entry
    q, _ = rows_in(c.rows, 4 * dim, dtype, 0, 8)
    got = []
    for fill in (0.0, float("nan")):
        data = c.data.float()
        data[foreign] = fill
        c.data.copy_(data.to(c.data.dtype))
        out, sums = attend(backend, c, q, 4, dtype, 0.125)
        with pytest.raises(gpt_b200.GptB200Error) as e:
            backend.synchronize()
        assert e.value.status == 1
        got.append((out.clone(), sums.clone()))
    for a, b in zip(*got):
        assert torch.isfinite(b[:c.rows].float()).all() and torch.equal(a, b)


STARTS = [[0, 10, 5, 8], [0, 5, 3, 3], [-3, 2, 4, 8], [0, 4, 8, 13], [8, 8, 4, 2], [0, 2**31 - 1, 5, 8], [12, 0, 0, 0], [0, 0, -1, 0]]


@pytest.mark.parametrize("starts", STARTS)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_starts_out_of_order_are_reported(backend, starts, kind):
    """By every call, whichever rows they leave to no sequence."""
    import gpt_b200
    c = Cache(kind, [20, 30, 40], [4, 4, 4], 2, 64, 16, seed=2).cuda()
    c.starts.copy_(torch.tensor(starts, dtype=torch.int32))
    x, _ = rows_in(c.rows, 128, "bf16", 0, 8)
    q, _ = rows_in(c.rows, 256, "bf16", 0, 8)
    out = torch.empty_like(q)
    k, v = torch.empty_like(x), torch.empty_like(x)
    for call in (lambda: backend.kv_pages_write(c.pages, c.batch, x, 128, x, 128, 0), lambda: backend.kv_pages_read(k, 128, v, 128, 0, c.pages, c.batch),
                 lambda: backend.attention_paged(out, 256, None, q, 256, 0, 4, c.pages, c.batch, 0.125)):
        call()
        with pytest.raises(gpt_b200.GptB200Error) as e:
            backend.synchronize()
        assert e.value.status == 1
        backend.synchronize()      # once
    c.starts.copy_(c.starts_cpu)
    backend.kv_pages_write(c.pages, c.batch, x, 128, x, 128, 0)
    backend.synchronize()


def test_sums_at_an_odd_address_are_refused(backend):
    import gpt_b200
    c = Cache("bf16", [20], [2], 2, 64, 16).cuda()
    q, out = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda")
    sums = torch.zeros(16, device="cuda")
    n = backend.launch_count()
    for off in (1, 2, 3):
        with pytest.raises(gpt_b200.GptB200Error) as e:
            backend.attention_paged(out, 256, sums.data_ptr() + off, q, 256, 0, 4, c.pages, c.batch, 0.1)
        assert e.value.status == 1 and backend.launch_count() == n
    backend.attention_paged(out, 256, sums.data_ptr() + 4, q, 256, 0, 4, c.pages, c.batch, 0.1)
    backend.synchronize()


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("count,share", [(1, 1), (1, 16), (3, 8), (40, 2), (300, 1)])
@pytest.mark.parametrize("below,cap", [(20.0, 0.0), (95.0, 0.0), (300.0, 0.0), (20.0, 30.0), (300.0, 400.0)])
def test_infinite_values_with_next_to_no_weight(backend, dtype, kind, count, share, below, cap):
    """A weight of e^-300 is positive, whatever fp32 makes of it: an infinite value makes the output infinite.  Behind a key that is minus infinite the weight is none, and the product NaN,
    but where a cap bounds the score."""
    inf, length, dim = float("inf"), 500 + count, 64
    c = Cache(kind, [length, 30], [count, 3], 1, dim, 16, seed=3)
    for s in (0, 1):
        for position in range(c.lengths[s]):
            put(c, kind, s, position, 0.0, which=0, element=slice(0, 1))
    put(c, kind, 0, length - count // 2 - 1, float("nan"), element=12)       # some rows do not see it
    for position, key, values in ((7, -below, {3: inf, 4: -inf, 5: inf}), (9, -below, {5: -inf, 6: inf}), (11, -inf, {8: inf, 9: -inf}), (300, -below, {10: inf}), (length - 1, 0.0, {11: inf})):
        put(c, kind, 0, position, key, which=0, element=0)
        for element, value in values.items():
            put(c, kind, 0, position, value, element=element)
    c.cuda()
    q = 0.1 * torch.randn(count + 3, share, dim, generator=torch.Generator().manual_seed(2))
    q[:, :, 0] = 1.0
    q = q.reshape(count + 3, -1).to(torch.bfloat16 if dtype == "bf16" else torch.float32).cuda()
    out, sums = attend(backend, c, q, share, dtype, 1.0, cap)
    backend.synchronize()
    got = kinds(out.double().cpu().reshape(count + 3, share, dim))
    want = torch.zeros_like(got)
    want[:count, :, [3, 6, 10]] = 2
    want[:count, :, 4] = 3
    want[:count, :, 5] = 1
    want[:count, :, 8] = 2 if cap else 1
    want[:count, :, 9] = 3 if cap else 1
    want[count - 1, :, 11] = 2
    want[count - count // 2 - 1:count, :, 12] = 1
    assert torch.equal(got, want)
