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
