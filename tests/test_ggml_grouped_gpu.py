"""The product grouped by expert over Q4_K / Q6_K weights against its definition in 64 bits.

Tolerance, per element, with A = sum |x| (|d sc q| + |dmin m|), the two parts of a Q4_K weight apart:
  float32 sums             2^-23 A per addition of partial sums: (k/256 + 32) 2^-23 A
  rows in two f16 parts    2^-22 A, and 2^-34 of the row's largest value for what the parts cannot hold: 2^-34 max|x| sum|w|
  bf16 / f16 outputs       one f16 part of float32 rows in front of bf16 (2^-12 A); Q6_K integers over 2048 rounded to f16 (2^-12 A)
  SwiGLU                   float32 silu(g) u, 2^-20 A
  storing                  eps / 2 of the value"""
import numpy as np
import pytest
import torch

from oracle import formats as F
from tests import workloads as W

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
Q4, Q6 = F.GGML_Q4_K, F.GGML_Q6_K


def blocks(rng, ty, count):
    """Random GGUF blocks: every code and scale byte, block scales of both signs and of several magnitudes, zero among them."""
    raw = rng.integers(0, 256, (count, 144 if ty == Q4 else 210)).astype(np.uint8)
    d = (rng.choice([-1, 1], count) * np.exp(rng.uniform(-9, -5, count))).astype(np.float16)
    d[rng.random(count) < 0.02] = 0
    dmin = (rng.choice([-1, 1], count) * np.exp(rng.uniform(-9, -5, count))).astype(np.float16)
    if ty == Q4:
        raw[:, 0:2] = d.view(np.uint8).reshape(-1, 2)
        raw[:, 2:4] = dmin.view(np.uint8).reshape(-1, 2)
    else:
        raw[:, 208:210] = d.view(np.uint8).reshape(-1, 2)
    return raw


def weight(seed, ty, groups, n, k):
    """(Weight as a layer holds it, float64 values [groups, n, k], float64 sizes of the two parts)"""
    import darask_inference_engine_b200 as D
    raw = blocks(W.rng_for(seed), ty, groups * n * (k // 256))
    value = F.ggml_decode(raw.reshape(groups * n, -1), ty, k).astype(np.float64).reshape(groups, n, k)
    size = np.abs(value)
    if ty == Q4:
        b = raw.copy()
        b[:, 2:4] = 0                                                   # without the mins
        main = F.ggml_decode(b.reshape(groups * n, -1), ty, k).astype(np.float64).reshape(groups, n, k)
        size = np.abs(main) + np.abs(value - main)
    layer = D.KogarashiMoeLayer(256, 256, 1, 1)
    layer.load("ffn_gate_exps.weight", torch.from_numpy(raw.reshape(-1)), ty, (k, n, groups))
    return layer.weights["ffn_gate_exps.weight"], torch.from_numpy(value), torch.from_numpy(size)


def ranges_of(counts, first=0):
    offs = np.concatenate([[0], np.cumsum(counts)[:-1]]) + first
    return torch.from_numpy(np.stack([np.array(counts), offs], 1).astype(np.int32)).cuda()


def check(y, xs, value, size, counts, first=0, x_f32=False, q6=False, swiglu=False):
    """y [rows, n] against rows xs float64 in dispatch order."""
    k = value.shape[2]
    at = first
    for g, c in enumerate(counts):
        x = xs[at:at + c]
        ref, a = x @ value[g].T, x.abs() @ size[g].T
        rel = (k // 256 + 32) * 2.0 ** -23 + 2.0 ** -22
        if y.dtype == torch.bfloat16 and x_f32:
            rel += 2.0 ** -12
        if y.dtype != torch.float32 and q6:
            rel += 2.0 ** -12
        if swiglu:
            rel += 2.0 ** -20
        bound = rel * a + 2.0 ** -34 * x.abs().amax(1, keepdim=True) * size[g].sum(1)[None] if c else a
        if y.dtype != torch.float32:
            fi = torch.finfo(y.dtype)
            bound = bound + fi.eps / 2 * (ref.abs() + bound) + fi.tiny * fi.eps
        d = (y[at:at + c].double().cpu() - ref).abs()
        assert bool((d <= bound).all()), f"group {g}: off by {float((d / bound.clamp_min(1e-300)).max()):.3g} of the bound"
        at += c


COUNTS = [[1], [0, 1, 0], [3, 0, 17, 1, 64, 0], [130, 5, 128, 0, 257], [16, 15, 33]]


@pytest.mark.parametrize("counts", COUNTS, ids=[str(c) for c in COUNTS])
@pytest.mark.parametrize("n,k", [(128, 256), (1, 512), (200, 768), (300, 2048), (129, 1280)])
@pytest.mark.parametrize("ty", [Q4, Q6])
@pytest.mark.parametrize("x_ty,out_ty", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "bf16")])
def test_product(counts, n, k, ty, x_ty, out_ty):
    import darask_inference_engine_b200 as D
    w, value, size = weight(n + k, ty, len(counts), n, k)
    rows = sum(counts)
    x = torch.randn(rows, k, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(TYPES[x_ty])
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, out_dtype=TYPES[out_ty])
    check(y, x.double().cpu(), value, size, counts, x_f32=x_ty == "f32", q6=ty == Q6)
    assert D.kogarashi.grouped_status() == 0


@pytest.mark.parametrize("ty", [Q4, Q6])
@pytest.mark.parametrize("x_ty,out_ty", [("f32", "f32"), ("bf16", "bf16")])
def test_routes_two_matrices_and_rows_outside_the_ranges(ty, x_ty, out_ty):
    """Dispatch rows fetched through assignments, gate | up side by side, rows that no range covers left alone."""
    import darask_inference_engine_b200 as D
    tokens, topk, groups, n, k = 50, 3, 9, 136, 512
    rng = W.rng_for(5)
    w0, v0, s0 = weight(1, ty, groups, n, k)
    w1, v1, s1 = weight(2, ty, groups, n, k)
    ids = np.argsort(rng.random((tokens, groups)), 1)[:, :topk].reshape(-1)
    order = np.argsort(ids, kind="stable")
    counts = np.bincount(ids, minlength=groups)
    first, rows = 4, tokens * topk + 4 + 3
    asg = np.zeros(rows, np.int32)
    asg[first:first + tokens * topk] = order
    x = torch.randn(tokens, k, device="cuda").to(TYPES[x_ty])
    out = torch.full((rows, 2 * n + 1), 7.0, dtype=TYPES[out_ty], device="cuda")
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts, first), w0, up=w1, assignments=torch.from_numpy(asg).cuda(), topk=topk, out=out[:, :2 * n])
    xs = torch.zeros(rows, k, dtype=torch.float64)
    xs[first:first + tokens * topk] = x.double().cpu()[torch.from_numpy(order // topk)]
    check(y[:, :n], xs, v0, s0, counts, first, x_ty == "f32", ty == Q6)
    check(y[:, n:], xs, v1, s1, counts, first, x_ty == "f32", ty == Q6)
    assert bool((out[:first] == 7).all()) and bool((out[first + tokens * topk:] == 7).all()) and bool((out[:, 2 * n] == 7).all())
    assert D.kogarashi.grouped_status() == 0


@pytest.mark.parametrize("ty", [Q4, Q6])
@pytest.mark.parametrize("x_ty,out_ty", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_swiglu_rows(ty, x_ty, out_ty):
    import darask_inference_engine_b200 as D
    counts, n, k = [5, 0, 140, 31], 150, 512
    w, value, size = weight(3, ty, len(counts), n, k)
    wide = (torch.randn(sum(counts), 2 * k + 3, device="cuda") * 2).to(TYPES[x_ty])
    x = wide[:, 1:1 + 2 * k]
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, swiglu=True, out_dtype=TYPES[out_ty])
    g, u = x.double().cpu()[:, :k], x.double().cpu()[:, k:]
    # silu(g) u is a float32 number here, whatever the type of the rows
    check(y, g / (1 + torch.exp(-g)) * u, value, size, counts, x_f32=True, q6=ty == Q6, swiglu=True)


@pytest.mark.parametrize("ty", [Q4, Q6])
def test_magnitudes_and_values_that_are_not_finite(ty):
    """Rows from 1e-30 to 1e30 (beyond f16), zeros; an infinity or a NaN makes its row NaN and no other."""
    import darask_inference_engine_b200 as D
    counts, n, k = [6, 2], 130, 512
    w, value, size = weight(4, ty, 2, n, k)
    x = torch.randn(8, k, device="cuda")
    x[0] *= 1e-30
    x[1] *= 1e30
    x[2] = 0
    x[3, 5:] = 0
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w)
    check(y, x.double().cpu(), value, size, counts)
    assert not bool(y[2].any())
    z = x.clone()
    z[4, 300], z[7, 0] = float("inf"), float("nan")
    b = D.kogarashi.grouped_gemm(z, ranges_of(counts), w)
    assert bool(b[4].isnan().all()) and bool(b[7].isnan().all())
    keep = [0, 1, 2, 3, 5, 6]
    assert torch.equal(b[keep], y[keep])
    h = (torch.randn(8, k, device="cuda") * 3e4).clamp(-6e4, 6e4).half()   # f16 near its end: the sums must not overflow
    h[1] *= 2.0 ** -24
    y = D.kogarashi.grouped_gemm(h, ranges_of(counts), w, out_dtype=torch.float32)
    check(y, h.double().cpu(), value, size, counts)


def test_bad_ranges_and_routes_are_cut_and_reported():
    import darask_inference_engine_b200 as D
    w, value, size = weight(6, Q4, 3, 128, 256)
    x = torch.randn(10, 256, device="cuda")
    out = torch.full((10, 128), 5.0, device="cuda")
    bad = torch.tensor([[4, 0], [9, 6], [3, 40]], dtype=torch.int32, device="cuda")
    D.kogarashi.grouped_gemm(x, bad, w, out=out)
    assert D.kogarashi.grouped_status() == 2 and D.kogarashi.grouped_status() == 0
    check(out[:4], x.double().cpu(), value, size, [4])
    check(out[6:], x.double().cpu()[6:], value[1:], size[1:], [4])
    assert bool((out[4:6] == 5).all())
    asg = torch.tensor([0, 1, 99, 3], dtype=torch.int32, device="cuda")
    y = D.kogarashi.grouped_gemm(x, ranges_of([4, 0, 0]), w, assignments=asg)
    assert D.kogarashi.grouped_status() == 2
    assert not bool(y[2].any())
    check(y[:2], x.double().cpu(), value, size, [2])


def test_same_bits_on_other_streams_and_in_graphs():
    import darask_inference_engine_b200 as D
    counts = [40, 0, 3, 200]
    w, _, _ = weight(7, Q6, 4, 260, 768)
    x = torch.randn(sum(counts), 768, device="cuda")
    r = ranges_of(counts)
    first = D.kogarashi.grouped_gemm(x, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [D.kogarashi.grouped_gemm(x, r, w) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, a) for a in again)
    fixed, graphs, outs = x.clone(), [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(D.kogarashi.grouped_gemm(fixed, r, w))
        graphs.append(g)
    fixed.copy_(torch.randn_like(fixed))
    want = D.kogarashi.grouped_gemm(fixed, r, w)
    for g, o in zip(graphs, outs):
        g.replay()
        assert torch.equal(o, want)


def test_no_rows():
    import darask_inference_engine_b200 as D
    w, _, _ = weight(7, Q4, 4, 128, 256)
    assert tuple(D.kogarashi.grouped_gemm(torch.empty(0, 256, device="cuda"), ranges_of([0] * 4), w).shape) == (0, 128)
    x = torch.ones(5, 256, device="cuda")
    out = torch.full((5, 128), 2.0, device="cuda")
    D.kogarashi.grouped_gemm(x, ranges_of([0] * 4), w, out=out)            # rows, but none in a range
    assert bool((out == 2).all())


def test_ranges_that_all_hold_every_row():
    """Far more tiles than the rows have: some are left out and reported, the call ends, rows past the ranges stay."""
    import darask_inference_engine_b200 as D
    g, rows, n, k = 64, 600, 130, 256
    w, _, _ = weight(11, Q4, g, n, k)
    x = torch.randn(rows, k, device="cuda")
    D.kogarashi.grouped_status()
    r = torch.tensor([[rows - 1, 0]] * g, dtype=torch.int32, device="cuda")
    out = torch.full((rows, n), 7.0, device="cuda")
    D.kogarashi.grouped_gemm(x, r, w, out=out)
    assert D.kogarashi.grouped_status() == 2
    assert bool((out[-1] == 7.0).all())
