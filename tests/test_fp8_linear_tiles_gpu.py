"""The dense block-scaled FP8 product where a block goes on: rings, accumulators and factor slots used more than once, several tiles per
pair of blocks, every width and division of k; against the definition in 64 bits, with the tolerance of the tests of the product."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import formats as F
from tests.test_fp8_linear_gpu import TYPES, quantized, weights

pytestmark = pytest.mark.gpu

GGML = {"f32": 0, "f16": 1, "bf16": 30, "codes": 100}


def plan(m, n, k, ty):
    import darask_inference_engine_b200 as D
    p = (ctypes.c_int * 3)()
    assert D._lib.lib().darask_fp8_linear_plan(m, n, k, GGML[ty], p) == 0
    return tuple(p)


def decoded(codes):
    table = torch.from_numpy(F.e4m3_decode(np.arange(256, dtype=np.uint8))).double().cuda()
    return table[codes.long()]


def check(y, xv, xs, w, ws, base=None):
    """y against x . w^T (added to `base`): sums on the GPU in 64 bits."""
    n, k = w.shape
    kb = math.ceil(k / 128)
    x = xv.double().cuda() * xs.double().cuda().repeat_interleave(128, 1)[:, :k]
    wd = decoded(w) * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    ref, size = x @ wd.T, x.abs() @ wd.abs().T
    bound = (kb + 16) * 2.0 ** -23 * size
    if base is not None:
        ref = ref + base.double()
        bound = bound + 2.0 ** -24 * (ref.abs() + bound)
    if y.dtype != torch.float32:
        fi = torch.finfo(y.dtype)
        bound = bound + fi.eps / 2 * (ref.abs() + bound) + fi.tiny * fi.eps
    d = (y.double() - ref).abs()
    assert bool((d <= bound).all()), f"off by {float((d / bound.clamp_min(1e-300)).max()):.3g} of the bound, {int((d > bound).sum())} elements"


def inputs(m, n, k, x_ty):
    w, ws = weights(m + n + k, n, k, pitch=(k + 15) // 16 * 16)
    g = torch.Generator(device="cuda").manual_seed(m * 7 + k)
    if x_ty == "codes":
        x, _ = weights(m * 3 + k, m, k, pitch=(k + 15) // 16 * 16)
        xs = torch.rand(m, math.ceil(k / 128), generator=g, device="cuda") + 0.1
        return x, xs, decoded(x), xs, w, ws
    x = (torch.randn(m, k, generator=g, device="cuda") * 0.05).to(TYPES[x_ty])
    return (x, None, *quantized(x), w, ws)


# rows, columns, 128-column blocks of k (the last one short by 48), rows per tile, parts of k: 17 blocks and more per part, so that
# every ring goes round three times and the third group of factors waits for the first
STREAM = [(9, 130, 17, 16, 4), (100, 5000, 17, 16, 1), (9, 18000, 34, 16, 2), (150, 130, 70, 16, 4), (9, 130, 136, 16, 8), (520, 1100, 17, 32, 1),
          (50, 5000, 34, 32, 2), (600, 130, 70, 32, 4), (300, 130, 136, 32, 8), (70, 18000, 17, 128, 1), (520, 1100, 34, 128, 2), (257, 1100, 75, 128, 4),
          (200, 3400, 136, 128, 8)]


@pytest.mark.parametrize("m,n,kb,rows,parts", STREAM)
@pytest.mark.parametrize("x_ty,out_ty", [("bf16", "bf16"), ("codes", "f32"), ("f32", "f16")])
def test_stream_kernels_over_long_k(m, n, kb, rows, parts, x_ty, out_ty):
    import darask_inference_engine_b200 as D
    k = kb * 128 - 48
    assert plan(m, n, k, x_ty) == (rows, parts, 0)
    x, xs, xv, xsv, w, ws = inputs(m, n, k, x_ty)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = D.fp8.linear(x, w, ws, x_scales=xs, out_dtype=TYPES[out_ty], status=word)
    check(y, xv, xsv, w, ws)
    if out_ty == "f32":
        base = torch.randn(m, n, device="cuda")
        check(D.fp8.linear(x, w, ws, x_scales=xs, out=base.clone(), add=True, status=word), xv, xsv, w, ws, base)
    assert D._lib.take_status(word) == 0


@pytest.mark.parametrize("m", [1, 3, 8])
@pytest.mark.parametrize("n,k,parts", [(130, 32768, 8), (1000, 5100, 8), (18000, 2048, 2), (20000, 3900, 1), (140, 300 * 128, None)])
@pytest.mark.parametrize("x_ty", ["bf16", "f32", "codes"])
def test_a_few_rows(m, n, k, parts, x_ty):
    """Rows quantized in the launch, up to the 32 blocks of k that a block holds; codes, and rows too long for it."""
    import darask_inference_engine_b200 as D
    p = plan(m, n, k, x_ty)
    assert p[0] == 16 and (p[1:] == (parts, int(x_ty != "codes")) if parts else p[2] == 0)
    x, xs, xv, xsv, w, ws = inputs(m, n, k, x_ty)
    check(D.fp8.linear(x, w, ws, x_scales=xs, out_dtype=torch.float32), xv, xsv, w, ws)


@pytest.mark.parametrize("m,n,k", [(520, 18000, 17 * 128 - 48), (2900, 3500, 19 * 128)])
@pytest.mark.parametrize("x_ty,out_ty", [("bf16", "bf16"), ("codes", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("shift", [0, 1])
def test_pairs_that_take_several_tiles(m, n, k, x_ty, out_ty, shift):
    """168 and 213 tiles for 74 pairs, three groups of factors per tile, results by TMA and (one column further) by ordinary stores; what lies
    around the results stays."""
    import darask_inference_engine_b200 as D
    assert plan(m, n, k, x_ty) == (256, 1, 0) and math.ceil(m / 256) * math.ceil(n / 256) > 2 * 74
    x, xs, xv, xsv, w, ws = inputs(m, n, k, x_ty)
    pitch = (n + 31) // 16 * 16
    out = torch.full((m + 1, pitch), -1.5, dtype=TYPES[out_ty], device="cuda")
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = D.fp8.linear(x, w, ws, x_scales=xs, out=out[:m, shift:shift + n], status=word)
    check(y, xv, xsv, w, ws)
    assert bool((out[m] == -1.5).all()) and bool((out[:, :shift] == -1.5).all()) and bool((out[:, shift + n:] == -1.5).all())
    if out_ty == "f32":
        base = torch.randn(m, n, device="cuda")
        check(D.fp8.linear(x, w, ws, x_scales=xs, out=base.clone(), add=True, status=word), xv, xsv, w, ws, base)
    assert D._lib.take_status(word) == 0


def swiglu_reference(x, k, w, ws):
    g, u = x.double().cpu()[:, :k], x.double().cpu()[:, k:]
    return quantized((g / (1 + torch.exp(-g)) * u).float())


@pytest.mark.parametrize("m", [1, 6, 50, 400])
@pytest.mark.parametrize("n,k", [(200, 77), (130, 130), (300, 2050), (150, 384)])
@pytest.mark.parametrize("x_ty", ["f32", "bf16"])
def test_swiglu_rows_whose_products_are_exact(m, n, k, x_ty):
    """Gates of 32, 64, 0 and -200: silu is the gate or zero to the last bit and a power of two, so gate * up is exact and so are the codes; for any
    k, with halves that start on any element."""
    import darask_inference_engine_b200 as D
    w, ws = weights(m + k, n, k, pitch=(k + 15) // 16 * 16)
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    gate = torch.tensor([32.0, 64.0, 0.0, -200.0], device="cuda")[torch.randint(0, 4, (m, k), generator=g, device="cuda")]
    x = torch.cat([gate, torch.randn(m, k, generator=g, device="cuda")], 1).to(TYPES[x_ty])
    y = D.fp8.linear(x, w, ws, swiglu=True, out_dtype=torch.float32)
    v = torch.where(x[:, :k] > 0, x[:, :k].float() * x[:, k:].float(), torch.zeros_like(gate))
    check(y, *quantized(v), w, ws)


def test_swiglu_of_single_rows():
    """Forty rows, each in a call of its own: a SwiGLU product a few float32 steps off moves a code with the chance 2^-17, one row in 300."""
    import darask_inference_engine_b200 as D
    k, n = 384, 200
    w, ws = weights(8, n, k)
    x = torch.randn(40, 2 * k, generator=torch.Generator(device="cuda").manual_seed(40), device="cuda") * 2
    v, s = swiglu_reference(x, k, w, ws)
    xq = v.cuda() * s.double().cuda().repeat_interleave(128, 1)
    wd = decoded(w) * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    ref, size = xq @ wd.T, xq.abs() @ wd.abs().T
    y = torch.cat([D.fp8.linear(x[i:i + 1], w, ws, swiglu=True) for i in range(40)]).double()
    differ = ((y - ref).abs() > 2.0 ** -19 * size).any(1)
    assert int(differ.sum()) <= 2
