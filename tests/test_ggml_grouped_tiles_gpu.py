"""The grouped GGUF product where a block goes on to further tiles, over long rows and over ranges that overlap; against the definition in
64 bits, with the tolerance of the tests of the product."""
import numpy as np
import pytest
import torch

from oracle import formats as F
from tests import workloads as W
from tests.test_ggml_grouped_gpu import Q4, Q6, TYPES, blocks, check, ranges_of, weight

pytestmark = pytest.mark.gpu


def sampled_weight(seed, ty, groups, n, k, sample):
    """(Weight as a layer holds it, {group: (float64 values [n, k], sizes of the two parts)}), decoded for the sampled groups only."""
    import darask_inference_engine_b200 as D
    raw = blocks(W.rng_for(seed), ty, groups * n * (k // 256)).reshape(groups, n, -1)
    parts = {}
    for g in sample:
        value = F.ggml_decode(raw[g], ty, k).astype(np.float64)
        size = np.abs(value)
        if ty == Q4:
            b = raw[g].reshape(-1, 144).copy()
            b[:, 2:4] = 0                                # without the mins
            main = F.ggml_decode(b.reshape(n, -1), ty, k).astype(np.float64)
            size = np.abs(main) + np.abs(value - main)
        parts[g] = torch.from_numpy(value), torch.from_numpy(size)
    layer = D.KogarashiMoeLayer(256, 256, 1, 1)
    layer.load("ffn_gate_exps.weight", torch.from_numpy(raw.reshape(-1)), ty, (k, n, groups))
    return layer.weights["ffn_gate_exps.weight"], parts


def tiles(counts, n, mats):
    rows = sum(counts)
    height = 32 if rows <= 32 * len(counts) else 128
    return sum(-(-c // height) for c in counts) * -(-n // 128) * mats


# groups, busiest group, columns: 32-row and 128-row tiles, each more than three times the 148 blocks
MANY = [("narrow", 60, 40, 1000), ("wide", 20, 420, 2400)]


@pytest.mark.parametrize("shape", MANY, ids=[m[0] for m in MANY])
@pytest.mark.parametrize("k", [512, 768])
@pytest.mark.parametrize("ty", [Q4, Q6])
@pytest.mark.parametrize("x_ty,out_ty,up", [("f32", "f32", False), ("bf16", "f32", True), ("f16", "f16", False), ("f32", "f16", True), ("bf16", "bf16", True),
                                            ("f32", "bf16", False)])
def test_blocks_that_take_several_tiles(shape, k, ty, x_ty, out_ty, up):
    """Expander sets, rings, accumulators and the search for the group go on from tile to tile, over groups without rows, tiles of every height
    and an even and an odd number of 256-column blocks."""
    import darask_inference_engine_b200 as D
    kind, groups, most, n = shape
    n = n // 2 if up else n
    rng = W.rng_for(k + groups)
    counts = rng.integers(0, most + 1, groups)
    counts[rng.choice(groups, groups // 6, replace=False)] = 0
    counts = [int(c) for c in counts]
    rows = sum(counts)
    assert (rows <= 32 * groups) == (kind == "narrow") and tiles(counts, n, 1 + up) > 3 * 148
    sample = sorted({int(g) for g in rng.choice(groups, 6, replace=False)} | {0, groups - 1, max(g for g in range(groups) if counts[g])})
    w, parts = sampled_weight(k + n, ty, groups, n, k, sample)
    mats = [(w, parts)] + ([sampled_weight(k + n + 1, ty, groups, n, k, sample)] if up else [])
    x = torch.randn(rows, k, generator=torch.Generator(device="cuda").manual_seed(k + rows), device="cuda").to(TYPES[x_ty])
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, up=mats[1][0] if up else None, out_dtype=TYPES[out_ty], status=word)
    xs, first = x.double().cpu(), np.concatenate([[0], np.cumsum(counts)])
    for i, (_, p) in enumerate(mats):
        for g in sample:
            value, size = p[g]
            check(y[:, i * n:(i + 1) * n], xs, value[None], size[None], [counts[g]], int(first[g]))
    # the groups that are not compared: their results exist, and the same rows give the same numbers wherever they are computed
    assert bool(y.isfinite().all())
    g = sample[len(sample) // 2]
    one = D.kogarashi.Weight(w.data.view(groups, -1)[g].clone(), w.ty, k, n, (k, n, 1))
    alone = D.kogarashi.grouped_gemm(x[first[g]:first[g + 1]], ranges_of([counts[g]]), one, out_dtype=TYPES[out_ty])
    if counts[g]:
        check(alone, xs[first[g]:first[g + 1]], parts[g][0][None], parts[g][1][None], [counts[g]])
    assert D._lib.take_status(word) == 0


@pytest.mark.parametrize("counts", [[3, 0, 40], [260]], ids=str)
@pytest.mark.parametrize("k", [4096, 4352, 8448])
@pytest.mark.parametrize("ty", [Q4, Q6])
@pytest.mark.parametrize("x_ty,swiglu,shift", [("f32", False, 0), ("bf16", False, 0), ("f16", False, 0), ("f32", False, 1), ("bf16", False, 1), ("f32", True, 0),
                                               ("bf16", True, 0), ("f16", True, 3)])
def test_long_rows(counts, k, ty, x_ty, swiglu, shift):
    """Rows longer than what a block keeps of them between its passes; aligned and not, each with its largest value behind that."""
    import darask_inference_engine_b200 as D
    n = 130
    w, value, size = weight(k + n, ty, len(counts), n, k)
    rows, cols = sum(counts), 2 * k if swiglu else k
    g = torch.Generator(device="cuda").manual_seed(k + rows)
    wide = torch.randn(rows, cols + 8, generator=g, device="cuda")
    wide[:, shift + k - 3] = 9
    wide = wide.to(TYPES[x_ty])
    x = wide[:, shift:shift + cols]
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, swiglu=swiglu, out_dtype=torch.float32, status=word)
    xs = x.double().cpu()
    if swiglu:
        xs = xs[:, :k] / (1 + torch.exp(-xs[:, :k])) * xs[:, k:]
    check(y, xs, value, size, counts, swiglu=swiglu)
    if not swiglu:                                       # a value that is not finite, behind what is kept, takes its row and no other
        wide[1, shift + k - 1] = float("nan")
        z = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, out_dtype=torch.float32, status=word)
        assert bool(z[1].isnan().all())
        keep = [i for i in range(rows) if i != 1]
        assert torch.equal(z[keep], y[keep])
    assert D._lib.take_status(word) == 0


@pytest.mark.parametrize("ty", [Q4, Q6])
def test_overlapping_ranges_leave_one_of_the_products(ty):
    """Every 16 bytes of a row that several ranges hold are those of one of its groups."""
    import darask_inference_engine_b200 as D
    groups, rows, n, k = 24, 300, 256, 256
    w, value, size = weight(12, ty, groups, n, k)
    x = torch.randn(rows, k, generator=torch.Generator(device="cuda").manual_seed(12), device="cuda")
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = torch.tensor([[rows - 20, 10]] * groups, dtype=torch.int32, device="cuda")
    out = torch.full((rows, n), 7.0, device="cuda")
    D.kogarashi.grouped_gemm(x, r, w, out=out, status=word)
    assert D._lib.take_status(word) == 2                  # ranges that hold many times the rows
    assert bool((out[:10] == 7).all()) and bool((out[-10:] == 7).all())
    xs = x.double()[10:-10]
    some = torch.zeros(rows - 20, n // 4, dtype=torch.bool, device="cuda")
    for g in range(groups):
        v, s = value[g].cuda(), size[g].cuda()
        bound = ((k // 256 + 32) * 2.0 ** -23 + 2.0 ** -22) * (xs.abs() @ s.T) + 2.0 ** -34 * xs.abs().amax(1, keepdim=True) * s.sum(1)[None]
        some |= ((out[10:-10].double() - xs @ v.T).abs() <= bound).view(rows - 20, n // 4, 4).all(2)
    assert bool(some.all())
