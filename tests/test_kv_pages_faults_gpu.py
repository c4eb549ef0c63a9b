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
