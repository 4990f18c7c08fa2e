"""The choice among the dense FP8 product's kernels, without a GPU (a device of 148 SMs is assumed then)."""
import ctypes
import random

import pytest
import torch

F32, F16, BF16, E4M3 = 0, 1, 30, 100


def plan(m, n, k, ty=BF16):
    import darask_inference_engine_b200 as D
    p = (ctypes.c_int * 3)()
    assert D._lib.lib().darask_fp8_linear_plan(m, n, k, ty, p) == 0
    return tuple(p)


def drawn(count=20000):
    rng = random.Random(5)
    for _ in range(count):
        yield int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 15))


def test_every_kernel_is_chosen_by_some_call_and_no_other():
    """The library holds stream kernels of 16, 32 and 128 rows, the one of 16 that quantizes its rows, and the pair kernel."""
    import re
    from pathlib import Path

    import darask_inference_engine_b200 as D
    seen, parts = set(), set()
    for m, n, k in drawn():
        rows, split, fused = plan(m, n, k)
        seen.add((rows, fused))
        parts.add(split)
    assert seen == {(16, 0), (16, 1), (32, 0), (128, 0), (256, 0)} and parts == {1, 2, 4, 8}
    source = (Path(D._lib.__file__).parent / "csrc" / "fp8_linear.cu").read_text()
    compiled = set(re.findall(r"launch_stream<(\d+), (true|false)>\(", source))
    assert {(int(r), int(f == "true")) for r, f in compiled} == seen - {(256, 0)}


def test_codes_are_divided_as_the_rows_they_came_from():
    """So that both give the same bits."""
    for m, n, k in drawn(3000):
        for ty in (F32, F16, BF16):
            assert plan(m, n, k, ty)[:2] == plan(m, n, k, E4M3)[:2] and plan(m, n, k, E4M3)[2] == 0


@pytest.mark.parametrize("bad", [(0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 1, 1, 12), ((1 << 24) + 1, 1, 1, 0)])
def test_refusals(bad):
    import darask_inference_engine_b200 as D
    assert D._lib.lib().darask_fp8_linear_plan(*bad, (ctypes.c_int * 3)()) == 1
    assert D._lib.lib().darask_fp8_linear_plan(1, 1, 1, 0, None) == 1


@pytest.mark.skipif(torch.cuda.is_available(), reason="the sizes below are for the 148 SMs assumed without a device")
def test_some_choices():
    assert plan(1, 4096, 4096) == (16, 8, 1) and plan(256, 4096, 2048) == (32, 1, 0) and plan(4096, 4096, 4096) == (256, 1, 0)
