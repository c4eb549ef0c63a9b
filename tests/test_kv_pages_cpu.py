"""Host logic of the paged cache of keys and values, without a GPU: the line of work behind its attention, the choice of kernel, refusals."""
import os
import subprocess

import pytest

from conftest import ROOT

BF16, F32, E4M3 = 0, 1, 2


def test_line_of_work_and_arrays_that_do_not_fit(built_library, tmp_path):
    """tests/kv_line.cu: divisions, blocks of keys, ranges of the line, arrays with any numbers in them, on the host."""
    from gpt_b200 import build
    exe = str(tmp_path / "kv_line")
    res = subprocess.run([build._nvcc(), "-std=c++17", "-O1", *build.ARCH_FLAGS, "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, os.path.join(ROOT, "tests", "kv_line.cu"), "-o", exe],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout


def pages(data=0x1000, scales=0x2000, kind=BF16, num=10, page=16, kv_heads=2, dim=64):
    import gpt_b200
    return gpt_b200.KvPages(data, scales, kind, num, page, kv_heads, dim)


def rows(starts=0x3000, lengths=0x4000, table=0x5000, sequences=2, pitch=4, count=3, max_new=2):
    import gpt_b200
    return gpt_b200.KvRows(starts, lengths, table, sequences, pitch, count, max_new)


def plan(dtype=BF16, heads=4, p=None, r=None, scale=0.125, cap=0.0, window=0, sinks=0):
    import gpt_b200
    return gpt_b200.plan_attention_paged(148, dtype, heads, p or pages(), r or rows(), scale, cap, window, sinks)


@pytest.mark.parametrize("dtype,kind,heads,max_new,want", [
    (BF16, BF16, 2, 1, ("tokens", 8, 296)), (BF16, BF16, 8, 3, ("tokens", 8, 296)), (BF16, BF16, 8, 4, ("tokens", 16, 296)), (BF16, E4M3, 8, 4, ("tokens", 8, 444)),
    (BF16, E4M3, 16, 4, ("tokens", 16, 444)), (BF16, BF16, 16, 5, ("tokens", 16, 296)), (BF16, BF16, 16, 6, ("prompt", 256, 148)), (BF16, E4M3, 2, 96, ("tokens", 16, 444)),
    (BF16, E4M3, 2, 97, ("prompt", 256, 148)), (BF16, BF16, 2, 2**31 - 1, ("prompt", 256, 148)), (BF16, BF16, 2, 0, ("tokens", 8, 296)),
    (F32, F32, 2, 1, ("few", 1, 444)), (F32, E4M3, 4, 2, ("few", 1, 444)), (F32, BF16, 6, 2, ("few", 1, 444)), (F32, F32, 6, 3, ("rows", 16, 444)), (BF16, F32, 2, 100, ("rows", 16, 444)),
])
def test_choice_of_kernel(built_library, dtype, kind, heads, max_new, want):
    got = plan(dtype, heads, pages(kind=kind), rows(max_new=max_new))
    assert (got["kernel"], got["tile_rows"], got["blocks"]) == want
    assert got["blocks"] <= 1024 and got["scratch_kib"] < 1 << 20


def test_nothing_to_do(built_library):
    assert plan(r=rows(sequences=0))["kernel"] == "none" and plan(r=rows(count=0))["kernel"] == "none"
    assert plan(p=pages(data=0), r=rows(count=0, starts=0, lengths=0, table=0))["kernel"] == "none"


@pytest.mark.parametrize("what", [
    dict(dtype=2), dict(dtype=-1), dict(heads=0), dict(heads=3), dict(heads=-2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0),
    dict(cap=float("inf")), dict(cap=float("nan")), dict(window=-1), dict(sinks=-1),
    dict(p=dict(kind=3)), dict(p=dict(kind=-1)), dict(p=dict(data=0)), dict(p=dict(data=0x1008)), dict(p=dict(kind=E4M3, scales=0)), dict(p=dict(kind=E4M3, scales=0x2004)), dict(p=dict(num=-1)),
    dict(p=dict(page=4)), dict(p=dict(page=24)), dict(p=dict(page=8192)), dict(p=dict(page=0)), dict(p=dict(kv_heads=0)), dict(p=dict(dim=0)), dict(p=dict(dim=12)), dict(p=dict(dim=136)), dict(p=dict(dim=-8)),
    dict(r=dict(sequences=-1)), dict(r=dict(count=-1)), dict(r=dict(max_new=-1)), dict(r=dict(pitch=-1)), dict(r=dict(starts=0)), dict(r=dict(lengths=0)), dict(r=dict(table=0)),
])
def test_refusals(built_library, what):
    import gpt_b200
    what = dict(what)
    if "p" in what:
        what["p"] = pages(**what["p"])
    if "r" in what:
        what["r"] = rows(**what["r"])
    with pytest.raises(gpt_b200.GptB200Error) as e:
        plan(**what)
    assert e.value.status == 1   # GPTB200_ERR_INVALID_ARG


def test_sizes_beyond_the_maximum(built_library):
    import gpt_b200
    for what in (dict(heads=2**20), dict(r=rows(count=2**31 - 1)), dict(heads=2, r=rows(sequences=2**31 - 1))):
        with pytest.raises(gpt_b200.GptB200Error) as e:
            plan(**what)
        assert e.value.status == 6   # GPTB200_ERR_TOO_LARGE


def test_null_arguments(built_library):
    import ctypes
    import gpt_b200
    lib, p, r, out = gpt_b200.load_library(), pages().struct, rows().struct, (ctypes.c_int * 4)()
    assert lib.gptb200_plan_attention_paged(148, 0, 4, None, r, 1.0, 0.0, 0, 0, out) == 1 and lib.gptb200_plan_attention_paged(148, 0, 4, p, None, 1.0, 0.0, 0, 0, out) == 1
    assert lib.gptb200_plan_attention_paged(0, 0, 4, p, r, 1.0, 0.0, 0, 0, out) == 1
    assert lib.gptb200_attention_paged(None, 0x1000, 256, None, 0x2000, 256, 0, 4, p, r, 1.0, 0.0, 0, 0) == 1
    assert lib.gptb200_kv_pages_write(None, p, r, 0x1000, 128, 0x2000, 128, 0) == 1 and lib.gptb200_kv_pages_read(None, 0x1000, 128, 0x2000, 128, 0, p, r) == 1


@pytest.mark.parametrize("heads,max_new,count,want", [(32, 2, 4096, 16), (32, 3, 79, 16), (32, 3, 80, 32), (8, 40, 319, 16), (8, 40, 320, 32)])
def test_rows_of_a_tile_on_fmas(built_library, heads, max_new, count, want):
    got = plan(F32, heads, pages(kind=F32), rows(max_new=max_new, count=count))
    assert (got["kernel"], got["tile_rows"]) == ("rows", want)
