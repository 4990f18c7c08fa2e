"""16-bit results of the grouped GGUF product are rounded once.

Tolerance, per element, with A = sum |x| (|d sc q| + |dmin m|) as in the tests of the product: (k/256 + 32) 2^-23 A for the float32 sums,
2^-22 A for rows in two f16 parts (2^-34 of the row's largest value for what these cannot hold), 2^-20 A for float32 SwiGLU, and one
rounding of the result, eps / 2 of the value. Nothing is added for the operands: every integer sc (q - 32) of Q6_K up to 4096 and both parts
of a row have to enter whole."""
import pytest
import torch

from tests.test_ggml_grouped_gpu import Q4, Q6, TYPES, check, ranges_of, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[5, 0, 33, 1, 17], [300, 5, 140]], ids=["narrow", "wide"])
@pytest.mark.parametrize("n,k", [(200, 768), (1000, 768), (129, 1280)])
@pytest.mark.parametrize("ty", [Q6, Q4])
@pytest.mark.parametrize("x_ty,swiglu", [("f16", False), ("f32", False), ("bf16", False), ("f32", True), ("f16", True)])
def test_f16_results_are_rounded_once(counts, n, k, ty, x_ty, swiglu):
    import darask_inference_engine_b200 as D
    w, value, size = weight(n + k + 1, ty, len(counts), n, k)
    rows = sum(counts)
    x = torch.randn(rows, 2 * k if swiglu else k, generator=torch.Generator(device="cuda").manual_seed(k + n), device="cuda").to(TYPES[x_ty])
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, swiglu=swiglu, out_dtype=torch.float16)
    xs = x.double().cpu()
    if swiglu:
        xs = xs[:, :k] / (1 + torch.exp(-xs[:, :k])) * xs[:, k:]
    check(y, xs, value, size, counts, swiglu=swiglu)
    # and the error over all is that of one rounding: half a step at most, 2^-11 of the value
    at, num, den = 0, 0.0, 0.0
    for g, c in enumerate(counts):
        ref = xs[at:at + c] @ value[g].T
        num += float((y[at:at + c].double().cpu() - ref).square().sum())
        den += float(ref.square().sum())
        at += c
    assert (num / den) ** 0.5 < 2.0 ** -11 / 3 ** 0.5 * 0.9
    assert D.kogarashi.grouped_status() == 0


@pytest.mark.parametrize("counts", [[5, 0, 33, 1, 17], [300, 5, 140]], ids=["narrow", "wide"])
@pytest.mark.parametrize("n,k", [(200, 768), (1000, 768), (129, 1280)])
@pytest.mark.parametrize("ty", [Q6, Q4])
@pytest.mark.parametrize("x_ty,swiglu", [("f16", False), ("f32", False), ("bf16", False), ("f32", True), ("bf16", True)])
def test_bf16_results_are_rounded_once(counts, n, k, ty, x_ty, swiglu):
    """Half a step from the exact value, and nearly every result the bf16 number closest to it. An error e in front of the rounding moves a
    result to a neighbour with the chance e / step, a step being 2^-8 to 2^-7 of the value: float32 results are off by 6e-7 of their
    root mean square, which moves 1.5e-4 of them and a few times that where values are small (0.005 allowed). One operand rounded to 11 bits
    (2^-12 / sqrt 3 on average) would move 0.02 to 0.04."""
    import darask_inference_engine_b200 as D
    w, value, size = weight(n + k + 2, ty, len(counts), n, k)
    rows = sum(counts)
    x = torch.randn(rows, 2 * k if swiglu else k, generator=torch.Generator(device="cuda").manual_seed(k + n + 1), device="cuda").to(TYPES[x_ty])
    y = D.kogarashi.grouped_gemm(x, ranges_of(counts), w, swiglu=swiglu, out_dtype=torch.bfloat16)
    xs = x.double().cpu()
    if swiglu:
        xs = xs[:, :k] / (1 + torch.exp(-xs[:, :k])) * xs[:, k:]
    check(y, xs, value, size, counts, swiglu=swiglu)
    ref = torch.cat([r @ value[g].T for g, r in enumerate(xs.split(counts))])
    assert float((y.cpu() != ref.float().bfloat16()).double().mean()) < 0.005
    assert D.kogarashi.grouped_status() == 0
