"""The dense block-scaled FP8 product against its definition in 64 bits.

Tolerance, per element: with A = sum |x_q| |w_q| (scales included) the kernel's float32 sums are off by at most
2^-23 A per addition of partial sums: one per 128-column block, a few inside a block (the tensor core adds the products of
an instruction and the running sum) and a few where parts of k are joined.  (kb + 16) 2^-23 A covers these.  Storing rounds
once more by at most eps / 2 of the value."""
import math

import numpy as np
import pytest
import torch

from oracle import formats as F
from tests import workloads as W

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def e4m3(codes):
    return torch.from_numpy(F.e4m3_decode(codes.cpu().numpy())).double()


def weights(seed, n, k, pitch=None):
    """codes [n, k] with rows `pitch` bytes apart and one scale per block; values of every exponent, negative zero included."""
    rng = W.rng_for(seed)
    codes = rng.integers(0, 256, (n, pitch or k)).astype(np.uint8)
    codes[(codes & 127) == 127] = 0x80                                  # no NaN
    scales = np.exp(rng.uniform(-4, 1, (math.ceil(n / 128), math.ceil(k / 128)))).astype(np.float32)
    return torch.from_numpy(codes).cuda()[:, :k], torch.from_numpy(scales).cuda()


def quantized(x):
    """Codes (as float64 values) and scales of float rows, block by block, from the rounding steps the quantizer is defined with."""
    x = x.float().cpu().numpy()
    m, k = x.shape
    kb = math.ceil(k / 128)
    val, scale = np.zeros((m, k)), np.ones((m, kb), np.float32)
    for b in range(kb):
        p = x[:, b * 128:(b + 1) * 128]
        top = np.abs(p).max(1)
        scale[:, b] = np.where(top == 0, np.float32(1), top / np.float32(448))
        inv = (np.float32(1) / scale[:, b]).astype(np.float32)
        val[:, b * 128:(b + 1) * 128] = F.e4m3_decode(F.e4m3_encode((p * inv[:, None]).astype(np.float32)))
    return torch.from_numpy(val), torch.from_numpy(scale)


def check(y, xv, xs, w, ws):
    n, k = w.shape
    kb = math.ceil(k / 128)
    x = xv * xs.double().cpu().repeat_interleave(128, 1)[:, :k]
    wd = e4m3(w) * ws.double().cpu().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    ref, size = x @ wd.T, x.abs() @ wd.abs().T
    bound = (kb + 16) * 2.0 ** -23 * size
    if y.dtype != torch.float32:
        bound = bound + torch.finfo(y.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(y.dtype).tiny * torch.finfo(y.dtype).eps
    d = (y.double().cpu() - ref).abs()
    assert bool((d <= bound).all()), f"off by {float((d / bound.clamp_min(1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (2, 129, 144), (7, 1000, 272), (16, 256, 4096), (17, 130, 1040),
                                   (33, 384, 640), (64, 96, 2048), (77, 1000, 1552), (128, 128, 128), (129, 257, 384), (300, 512, 256),
                                   (513, 1100, 912), (1025, 2304, 528), (2048, 2048, 256),
                                   (40, 130, 77), (600, 4100, 205)])
@pytest.mark.parametrize("x_ty,out_ty", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f16"), ("codes", "f32")])
def test_product(m, n, k, x_ty, out_ty):
    import darask_inference_engine_b200 as D
    w, ws = weights(m + n + k, n, k, pitch=(k + 15) // 16 * 16)
    g = torch.Generator(device="cuda").manual_seed(m * 7 + k)
    if x_ty == "codes":
        codes, xs = weights(m * 3 + k, m, k, pitch=(k + 15) // 16 * 16)
        xs = torch.rand(m, math.ceil(k / 128), generator=g, device="cuda") + 0.1
        y = D.fp8.linear(codes, w, ws, x_scales=xs, out_dtype=TYPES[out_ty])
        check(y, e4m3(codes), xs, w, ws)
    else:
        x = (torch.randn(m, k, generator=g, device="cuda") * 0.05).to(TYPES[x_ty])
        y = D.fp8.linear(x, w, ws, out_dtype=TYPES[out_ty])
        check(y, *quantized(x), w, ws)
    assert D.fp8.linear_status() == 0


def test_codes_equal_the_activation_quantizer():
    """Rows quantized inside the call and rows quantized by the stand-alone quantizer give the same bits."""
    import darask_inference_engine_b200 as D
    for m in (1, 5, 40, 700):
        x = torch.randn(m, 640, device="cuda")
        x[0] = 0
        w, ws = weights(3, 300, 640)
        codes, xs = D.quantize.fp8_act(x)
        assert torch.equal(D.fp8.linear(x, w, ws), D.fp8.linear(codes, w, ws, x_scales=xs, out_dtype=torch.float32))


@pytest.mark.parametrize("m", [1, 6, 50, 400])
def test_swiglu_rows(m):
    """gate | up rows: off by the float32 products' rounding (a few ulp), which can move a code by one step: each code is
    within a step 2^-3 of its value (half of it the rounding that the reference makes too), so the outputs agree to the size
    of one such step in one code per block with every other code equal."""
    import darask_inference_engine_b200 as D
    k, n = 384, 200
    x = torch.randn(m, 2 * k, device="cuda") * 2
    w, ws = weights(8, n, k)
    y = D.fp8.linear(x, w, ws, swiglu=True).double().cpu()
    g, u = x.double().cpu()[:, :k], x.double().cpu()[:, k:]
    v, s = quantized((g / (1 + torch.exp(-g)) * u).float())
    xq = v * s.double().repeat_interleave(128, 1)
    wd = e4m3(w) * ws.double().cpu().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    ref, size = xq @ wd.T, xq.abs() @ wd.abs().T
    step = 2.0 ** -3 * (xq.abs().amax(1, keepdim=True) * wd.abs().amax(1)[None]) * 3
    assert bool(((y - ref).abs() <= 2.0 ** -19 * size + step).all())
    # and nearly all rows have every code equal
    same = ((y - ref).abs() <= 2.0 ** -19 * size).all(1)
    assert int((~same).sum()) <= max(1, m // 20)


def test_strides_views_and_an_output_of_the_caller():
    import darask_inference_engine_b200 as D
    m, n, k = 37, 150, 300
    big = torch.randn(m, 2 * k + 9, device="cuda")
    x = big[:, 5:5 + k]                                                   # odd stride, odd start
    w, ws = weights(1, n, k, pitch=320)
    wide = torch.nn.functional.pad(ws, (0, 3), value=float("nan"))[:, :3]
    out = torch.full((m, n + 7), 3.25, dtype=torch.bfloat16, device="cuda")
    y = D.fp8.linear(x, w, wide, out=out[:, 1:1 + n])
    check(y, *quantized(x), w, ws)
    assert y.data_ptr() == out[:, 1:].data_ptr()
    assert bool((out[:, :1] == 3.25).all()) and bool((out[:, 1 + n:] == 3.25).all())
    codes, xs = D.quantize.fp8_act(torch.randn(m, 384, device="cuda"))
    w2, ws2 = weights(2, n, 384, pitch=400)
    padded = torch.zeros(m, 400, dtype=torch.uint8, device="cuda")
    padded[:, :384] = codes
    y = D.fp8.linear(padded[:, :384], w2, ws2, x_scales=xs, out_dtype=torch.float16)
    check(y, e4m3(codes), xs, w2, ws2)


@pytest.mark.parametrize("m", [3, 40, 600])
def test_values_that_are_not_finite_stay_in_their_row(m):
    import darask_inference_engine_b200 as D
    x = torch.randn(m, 256, device="cuda")
    clean = D.fp8.linear(x, *weights(4, 140, 256))
    x[0, 130] = float("inf")
    x[2, 7] = float("nan")
    y = D.fp8.linear(x, *weights(4, 140, 256))
    assert bool(y[0].isnan().all()) and bool(y[2].isnan().all())
    keep = [i for i in range(m) if i not in (0, 2)]
    assert torch.equal(y[keep], clean[keep])


def test_extreme_magnitudes():
    """Rows of 1e-30, of 1e30 and of zeros in one batch: the block scales carry the range."""
    import darask_inference_engine_b200 as D
    for m in (4, 200):
        x = torch.randn(m, 256, device="cuda")
        x[0] *= 1e-30
        x[1] *= 1e30
        x[2] = 0
        w, ws = weights(6, 128, 256)
        y = D.fp8.linear(x, w, ws)
        check(y, *quantized(x), w, ws)
        assert not bool(y[2].any())


def test_same_bits_in_every_call_on_other_streams_and_in_a_graph():
    """Split sums are joined in a fixed order; captured calls with their own scratch replay on new inputs."""
    import darask_inference_engine_b200 as D
    w, ws = weights(9, 520, 2048)
    for m in (1, 20, 130, 900):
        x = torch.randn(m, 2048, device="cuda", dtype=torch.bfloat16)
        first = D.fp8.linear(x, w, ws)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [D.fp8.linear(x, w, ws) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(first, a) for a in again)
        fixed, graphs, outs = x.clone(), [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(D.fp8.linear(fixed, w, ws))
            graphs.append(g)
        fixed.copy_(torch.randn_like(fixed))
        want = D.fp8.linear(fixed, w, ws)
        for g, o in zip(graphs, outs):
            g.replay()
            assert torch.equal(o, want)


def test_empty_batch():
    import darask_inference_engine_b200 as D
    w, ws = weights(9, 64, 128)
    assert tuple(D.fp8.linear(torch.empty(0, 128, device="cuda"), w, ws).shape) == (0, 64)


@pytest.mark.parametrize("out_ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,shift", [(2201, 0), (2201, 1), (2208, 0), (2208, 1)])
def test_many_rows_into_a_view(out_ty, n, shift):
    """256 x 256 tiles cut at both edges, into rows that start and end on a 16-byte boundary and into rows that do not."""
    import darask_inference_engine_b200 as D
    m, k = 1111, 528
    w, ws = weights(12, n, k)
    x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16)
    pitch = (n + 31) // 16 * 16
    out = torch.full((m + 1, pitch + shift), -1.5, dtype=TYPES[out_ty], device="cuda")
    D.fp8.linear(x, w, ws, out=out[:m, shift:shift + n])
    check(out[:m, shift:shift + n], *quantized(x), w, ws)
    assert bool((out[m] == -1.5).all()) and bool((out[:, :shift] == -1.5).all()) and bool((out[:, shift + n:] == -1.5).all())
    assert D.fp8.linear_status() == 0
