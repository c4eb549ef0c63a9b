"""What calls on a paged cache refuse before anything is launched, and what their plan says, without a GPU."""
import pytest
import torch

from test_kv_pages_cpu import BF16, E4M3, F32, pages, plan, rows


@pytest.mark.parametrize("what", [
    dict(scale=3e38), dict(scale=2.4e38), dict(scale=1.0, cap=1e-39), dict(scale=1.0, cap=3e38), dict(scale=1.0, cap=2.3e38), dict(scale=1e-30, cap=1e30), dict(scale=1e10, cap=1e-30), dict(scale=1e-20, cap=1e20),
])
def test_scales_and_caps_beyond_the_range(built_library, what):
    """Kernels multiply by scale, cap and scale / cap, the first two in base 2: none of them may be infinite, nor the quotient nothing."""
    import gpt_b200
    for dtype, kind in ((BF16, BF16), (BF16, E4M3), (F32, F32)):
        with pytest.raises(gpt_b200.GptB200Error) as e:
            plan(dtype=dtype, p=pages(kind=kind), **what)
        assert e.value.status == 1


@pytest.mark.parametrize("what", [dict(scale=2.3e38), dict(scale=1e-30), dict(scale=1.0, cap=1e-37), dict(scale=1.0, cap=8e37), dict(scale=1e-20, cap=1e17), dict(scale=2.0**-10, cap=2.0**100)])
def test_scales_and_caps_within_the_range(built_library, what):
    assert plan(**what)["kernel"] == "tokens"


class OnDevice:
    """A tensor as if it were in device memory."""

    def __init__(self, t):
        self._t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self._t, name)


def device(*shape, dtype=torch.int32):
    return OnDevice(torch.zeros(*shape, dtype=dtype))


def described(starts=None, lengths=None, table=None, sequences=3, pitch=4):
    import gpt_b200
    return gpt_b200.KvRows(device(4) if starts is None else starts, device(3) if lengths is None else lengths, device(3, 4) if table is None else table, sequences, pitch, 9, 4)


def pool(data=None, scales=None, kind=E4M3, num=5):
    import gpt_b200
    return gpt_b200.KvPages(device(5, 2, 3, 16, 64, dtype=torch.uint8) if data is None else data, device(5, 2, 3, 16, dtype=torch.uint8) if scales is None else scales, kind, num, 16, 3, 64)


def test_descriptions_of_tensors_that_fit():
    described()
    described(starts=device(9), lengths=device(7), table=device(20))
    described(table=OnDevice(torch.zeros(3, 8, dtype=torch.int32)[:, :4]), pitch=8)      # a few columns of wider rows
    described(sequences=0)
    pool()
    pool(data=device(7, 2, 3, 16, 64, dtype=torch.float8_e4m3fn))
    pool(data=OnDevice(torch.zeros(2, 5, 2, 3, 16, 64, dtype=torch.uint8)[1]))
    pool(data=device(5, 2, 3, 16, 64, dtype=torch.bfloat16), kind=BF16)
    pool(data=device(5 * 2 * 3 * 16 * 64 * 4, dtype=torch.uint8), kind=F32)            # bytes
    pool(num=0)


@pytest.mark.parametrize("what", [
    dict(lengths=(3, torch.int64)), dict(starts=(4, torch.int64)), dict(table=(12, torch.int64)), dict(lengths=(3, torch.float32)), dict(starts=(4, torch.int16)), dict(lengths=(2, torch.int32)),
    dict(starts=(3, torch.int32)), dict(table=(8, torch.int32)),
])
def test_arrays_that_are_not_what_the_description_says(what):
    """An int64 array, torch's default, would be read as pairs of numbers."""
    (name, (size, dtype)), = what.items()
    with pytest.raises(ValueError, match=name.replace("starts", "row_starts").replace("table", "page_table")):
        described(**{name: device(size, dtype=dtype)})


def test_arrays_with_gaps_or_on_the_host():
    for name in ("starts", "lengths"):
        with pytest.raises(ValueError, match="contiguous"):
            described(**{name: OnDevice(torch.zeros(8, dtype=torch.int32)[::2])})
    with pytest.raises(ValueError, match="contiguous"):
        described(table=OnDevice(torch.zeros(4, 3, dtype=torch.int32).T))
    for name in ("starts", "lengths", "table"):
        with pytest.raises(ValueError, match="device memory"):
            described(**{name: torch.zeros(12, dtype=torch.int32)})


@pytest.mark.parametrize("kind,shape,dtype", [
    (BF16, (5, 2, 3, 16, 64), torch.float32), (BF16, (5, 2, 3, 16, 64), torch.float16), (F32, (5, 2, 3, 16, 64), torch.bfloat16), (E4M3, (5, 2, 3, 16, 64), torch.float8_e5m2), (BF16, (4, 2, 3, 16, 64), torch.bfloat16),
    (E4M3, (5, 2, 3, 16, 63), torch.uint8), (F32, (5, 2, 3, 16, 64), torch.uint8),
])
def test_pools_that_are_not_what_the_description_says(kind, shape, dtype):
    with pytest.raises(ValueError, match="data"):
        pool(data=device(*shape, dtype=dtype), kind=kind)


def test_pools_with_gaps_short_scales_or_on_the_host():
    with pytest.raises(ValueError, match="contiguous"):
        pool(data=OnDevice(torch.zeros(5, 2, 3, 16, 128, dtype=torch.uint8)[..., :64]))
    with pytest.raises(ValueError, match="scales"):
        pool(scales=device(5, 2, 3, 15, dtype=torch.uint8))
    with pytest.raises(ValueError, match="scales"):
        pool(scales=device(5, 2, 3, 16, dtype=torch.float32))
    with pytest.raises(ValueError, match="device memory"):
        pool(data=torch.zeros(5, 2, 3, 16, 64, dtype=torch.uint8))


@pytest.mark.parametrize("name", ["starts", "lengths", "table"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_at_odd_addresses(built_library, name, off):
    """A load of four bytes from there would fault."""
    import gpt_b200
    with pytest.raises(gpt_b200.GptB200Error) as e:
        plan(r=rows(**{name: 0x3000 + off}))
    assert e.value.status == 1
    assert plan(r=rows(**{name: 0x3004}))["kernel"] == "tokens"


@pytest.mark.parametrize("dtype,kind,max_new,kernel,per_sm,most,part", [
    (BF16, BF16, 1, "tokens", 2, 320, 16 * 130), (BF16, E4M3, 1, "tokens", 3, 480, 16 * 130), (BF16, BF16, 100, "prompt", 1, 512, 256 * 132), (F32, F32, 1, "few", 3, 480, 16 * 130),
    (F32, F32, 100, "rows", 3, 480, 16 * 130),
])
@pytest.mark.parametrize("sms", [1, 7, 148, 160, 200, 2000, 2**31 - 1])
def test_plan_on_any_number_of_sms(built_library, dtype, kind, max_new, kernel, per_sm, most, part, sms):
    """The grid that a call launches, and the scratch for two parts per block: no more blocks than parts of a tile have room for."""
    import gpt_b200
    got = gpt_b200.plan_attention_paged(sms, dtype, 4, pages(kind=kind), rows(max_new=max_new), 0.125)
    blocks = min(sms * per_sm, most)
    assert got["kernel"] == kernel and got["blocks"] == blocks and got["scratch_kib"] == 2 * blocks * part * 4 >> 10
