"""The layers that use the dense FP8 product and the grouped GGUF product: the Kogarashi layer for prompts against the oracle and
against the layer's own decode call, the FP8 layer with a shared expert against its pieces, and the two operators in one run."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import formats as F
from oracle import layers as L
from tests import workloads as W
from tests.test_kogarashi_gpu import run_layer as run_kogarashi

pytestmark = pytest.mark.gpu


def prefill(layer, acts, **kw):
    m, _ = run_kogarashi(layer, acts)                    # loads the weights; its own result is the decode call's
    x, n = torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"]).cuda()
    out, ids, prob = m.prefill(x, n, **kw)
    assert out is x
    return m, x.cpu().numpy(), ids.cpu().numpy(), prob.cpu().numpy()


@pytest.mark.parametrize("tokens,experts,topk,shared,zipf", [(1, 16, 4, True, None), (40, 32, 4, True, 1.1), (300, 16, 2, False, None), (130, 8, 8, True, None)])
def test_prefill_against_the_oracle(tokens, experts, topk, shared, zipf):
    """Routes bit for bit on the same logits, outputs within the layer's bars (relative L2 1e-3, max 2e-3 max|ref|)."""
    layer, acts = W.kogarashi_layer(31 + tokens, hidden=512, inter=256, experts=experts, topk=topk, tokens=tokens, shared=shared, zipf=zipf, pool=8)
    logits = L.kogarashi_logits(layer, acts["n"]) + (acts["bias"] if acts["bias"] is not None else 0)
    logits = np.ascontiguousarray(logits, np.float32)
    ref = L.kogarashi_forward(layer, acts["x"], acts["n"], logits=logits)
    m, out, ids, prob = prefill(layer, acts, logits=torch.from_numpy(logits).cuda())
    assert np.array_equal(ids, ref["ids"])
    assert np.allclose(prob, ref["prob"], rtol=1e-5, atol=1e-7)
    W.check_output(out.astype(np.float64) - acts["x"], ref["out"].astype(np.float64) - acts["x"])


def test_prefill_projects_the_router_itself():
    """Without given logits the routes follow the projection: float32 sums of 512 products, off by 512 2^-24 sum|w x| at most, so that
    tokens whose selection hangs on less are left out of the comparison."""
    layer, acts = W.kogarashi_layer(5, hidden=512, inter=256, experts=24, topk=3, tokens=90, shared=True, pool=8)
    exact = acts["n"].astype(np.float64) @ layer.router.astype(np.float64).T + (acts["bias"] if acts["bias"] is not None else 0)
    doubt = 512 * 2.0 ** -24 * (np.abs(acts["n"]).astype(np.float64) @ np.abs(layer.router).astype(np.float64).T).max(1)
    top = np.sort(exact, 1)[:, ::-1]
    clear = (top[:, :3] - top[:, 1:4]).min(1) > 2 * doubt
    assert clear.sum() > 60
    m, out, ids, prob = prefill(layer, acts)
    want = np.argsort(-exact, 1, kind="stable")[:, :3]
    assert np.array_equal(ids[clear], want[clear])
    ref = L.kogarashi_forward(layer, acts["x"], acts["n"], logits=np.ascontiguousarray(exact, np.float32))
    W.check_output((out.astype(np.float64) - acts["x"])[clear], (ref["out"].astype(np.float64) - acts["x"])[clear])


@pytest.mark.parametrize("down", [F.GGML_Q4_K, F.GGML_Q6_K])
def test_prefill_agrees_with_the_decode_call(down):
    layer, acts = W.kogarashi_layer(8, hidden=768, inter=512, experts=16, topk=4, tokens=24, shared=True, pool=8, down_ty=down)
    m, decode = run_kogarashi(layer, acts)
    x, n = torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"]).cuda()
    m.prefill(x, n, logits=m.logits[:24].clone())
    W.check_output(x.cpu().numpy().astype(np.float64) - acts["x"], decode.astype(np.float64) - acts["x"], rel=1e-4, max_abs=2e-4)


def test_prefill_with_the_layer_entry():
    """Residual add and RMS norm in front, as the decode call has them: the same kernel writes x and n."""
    layer, acts = W.kogarashi_layer(9, hidden=512, inter=256, experts=16, topk=2, tokens=20, shared=True, pool=8)
    m, _ = run_kogarashi(layer, acts)
    attn, w = torch.randn(20, 512, device="cuda"), torch.rand(512, device="cuda") + 0.5
    xa, na = torch.from_numpy(acts["x"].copy()).cuda(), torch.empty(20, 512, device="cuda")
    xb, nb = xa.clone(), na.clone()
    m.forward(xa, na, attn_out=attn, norm_w=w)
    before = torch.from_numpy(acts["x"]).cuda() + attn
    m.prefill(xb, nb, logits=m.logits[:20].clone(), attn_out=attn, norm_w=w)
    assert torch.equal(na, nb)
    W.check_output((xb - before).cpu().numpy(), (xa - before).cpu().numpy(), rel=1e-4, max_abs=2e-4)


def test_prefill_refusals():
    import darask_inference_engine_b200 as D
    m = D.KogarashiMoeLayer(256, 256, 4, 2)
    x = torch.zeros(3, 256, device="cuda")
    for bad in (dict(x=x, n=x[:2]), dict(x=x.half(), n=x.half()), dict(x=x, n=x.clone(), logits=torch.zeros(3, 5, device="cuda")),
                dict(x=x, n=x.clone(), attn_out=x)):
        with pytest.raises(ValueError):
            m.prefill(**bad)
    with pytest.raises(D._lib.CudaError):
        m.prefill(x, x.clone())                          # no weights loaded


def fp8_layer(tokens, hidden=512, inter=256, width=384):
    import darask_inference_engine_b200 as D
    layer, acts = W.fp8_layer(3 + tokens, hidden, inter, 8, 2, tokens)
    m = D.Fp8MoeLayer(hidden, inter, 8, 2, tokens)
    for name in ("gate", "up", "down"):
        mats = getattr(layer, name)
        m.load(name, torch.from_numpy(np.stack([p for p, _ in mats])), torch.from_numpy(np.stack([s for _, s in mats])))
    rng = W.rng_for(17)
    sh = [tuple(torch.from_numpy(a) for a in F.fp8_block_quantize(W.normal(rng, shp, shp[1] ** -0.5))) for shp in ((width, hidden), (width, hidden), (hidden, width))]
    return m, sh, torch.from_numpy(acts["x"]).bfloat16().cuda(), torch.from_numpy(acts["logits"]).cuda()


@pytest.mark.parametrize("tokens", [1, 7, 200])
def test_fp8_layer_with_a_shared_expert(tokens):
    """The sum of the routed experts and of the shared one: the parts on their own give the same bits; the shared part against the
    definition in 64 bits from its float32 gate and up rows."""
    import darask_inference_engine_b200 as D
    m, sh, x, logits = fp8_layer(tokens)
    routed = m.forward(x, logits).clone()
    m.load_shared(*sh)
    out = m.forward(x, logits)
    assert m.status() == 0
    gate, up, down = [(p.cuda(), s.cuda()) for p, s in sh]
    g, u = D.fp8.linear(x, *gate, out_dtype=torch.float32), D.fp8.linear(x, *up, out_dtype=torch.float32)
    both = D.fp8.linear(x, torch.cat([gate[0], up[0]]), torch.cat([gate[1], up[1]]), out_dtype=torch.float32)
    # (the stacked product may divide k otherwise than the single ones: 2^-20 of sum |x| |w| is far above its float32 sums)
    assert torch.allclose(both, torch.cat([g, u], 1), rtol=1e-5, atol=1e-4)
    y = D.fp8.linear(both, *down, swiglu=True, out_dtype=torch.float32)
    assert torch.equal(out, routed + y)
    h = (both[:, :384].double() / (1 + torch.exp(-both[:, :384].double())) * both[:, 384:].double()).float().cpu().numpy()
    codes, scales = F.fp8_act_quantize(h)
    ref = L.fp8_dequant_gemm(codes, scales, down[0].cpu().numpy(), down[1].cpu().numpy())
    W.check_output(y.cpu().numpy(), ref, rel=5e-3, max_abs=2e-2)       # a SwiGLU ulp moves a code by one step now and then


def test_add_to_an_output():
    import darask_inference_engine_b200 as D
    for m, n, k in ((1, 130, 256), (40, 257, 640), (300, 4100, 256), (700, 2048, 512)):
        w, ws = D.quantize.fp8_block(torch.randn(n, k, device="cuda"))
        x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16) if k % 16 == 0 else None
        base = torch.randn(m, n, device="cuda")
        got = base.clone()
        assert D.fp8.linear(x, w, ws, out=got, add=True) is got
        assert torch.equal(got, base + D.fp8.linear(x, w, ws, out_dtype=torch.float32))
    with pytest.raises(ValueError, match="add"):
        D.fp8.linear(x, w, ws, add=True)
    with pytest.raises(ValueError, match="add"):
        D.fp8.linear(x, w, ws, out=torch.zeros(m, n, dtype=torch.bfloat16, device="cuda"), add=True)


def test_the_operators_together_in_a_graph():
    """A block as a prompt meets it: a dense FP8 projection gives the rows that the GGUF experts read, captured once and replayed on other
    tokens; the replay equals the calls."""
    import darask_inference_engine_b200 as D
    t, hidden = 70, 512
    layer, acts = W.kogarashi_layer(21, hidden=hidden, inter=256, experts=16, topk=2, tokens=t, shared=True, pool=8)
    m, _ = run_kogarashi(layer, acts)
    w, ws = D.quantize.fp8_block(torch.randn(hidden, 384, device="cuda") * 384 ** -0.5)
    tokens = torch.randn(t, 384, device="cuda", dtype=torch.bfloat16)
    x0 = torch.randn(t, hidden, device="cuda")
    x, n = x0.clone(), torch.empty(t, hidden, device="cuda")

    def block():
        D.fp8.linear(tokens, w, ws, out=n)
        return m.prefill(x, n)

    block()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
    tokens.copy_(torch.randn_like(tokens))
    x.copy_(x0)
    block()
    want = x.clone()
    x.copy_(x0)
    graph.replay()
    assert torch.equal(x, want)
    # and on another stream
    side = torch.cuda.Stream()
    x.copy_(x0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(x, want)


def test_prefill_refuses_tensors_that_are_elsewhere():
    layer, acts = W.kogarashi_layer(9, hidden=256, inter=256, experts=4, topk=2, tokens=3, shared=False, pool=4)
    m, _ = run_kogarashi(layer, acts)
    x = torch.zeros(3, 256, device="cuda")
    for bad in (dict(x=x.cpu(), n=x), dict(x=x, n=x.cpu()), dict(x=x, n=x.clone(), logits=torch.zeros(3, 4)),
                dict(x=x, n=x.clone(), norm_w=torch.ones(256)), dict(x=x, n=x.clone(), norm_w=x[0].clone(), attn_out=torch.zeros(3, 256))):
        with pytest.raises(ValueError):
            m.prefill(**bad)


@pytest.mark.parametrize("tokens", [1, 33, 70])
def test_prefill_of_rows_on_any_word(tokens):
    """x, n and the router four bytes off: the same bits as on 16-byte boundaries."""
    layer, acts = W.kogarashi_layer(21, hidden=512, inter=256, experts=40, topk=3, tokens=tokens, shared=True, pool=8)
    m, _ = run_kogarashi(layer, acts)
    off = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    x, n = torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"].copy()).cuda()
    y, ids, prob = m.prefill(x.clone(), n)
    y2, ids2, prob2 = m.prefill(off(x), off(n))
    assert torch.equal(y, y2) and torch.equal(ids, ids2) and torch.equal(prob, prob2)


@pytest.mark.parametrize("dtype,ty", [(torch.bfloat16, 30), (torch.float16, 1)])
def test_prefill_with_a_router_of_16_bits(dtype, ty):
    """A 16-bit router and the same numbers in float32: the same bits."""
    import darask_inference_engine_b200 as D
    layer, acts = W.kogarashi_layer(23, hidden=512, inter=256, experts=40, topk=3, tokens=45, shared=True, pool=8)
    m, _ = run_kogarashi(layer, acts)
    runs = []
    router = torch.from_numpy(layer.router).cuda().to(dtype)
    gate = m.weights["ffn_gate_inp_shexp.weight"].data.view(torch.float32).to(dtype)
    for cast, kind in ((torch.float32, 0), (dtype, ty)):
        m.weights["ffn_gate_inp.weight"] = D.kogarashi.Weight(router.to(cast).contiguous().view(torch.uint8).view(-1), kind, 512, 40, (512, 40))
        m.weights["ffn_gate_inp_shexp.weight"] = D.kogarashi.Weight(gate.to(cast).contiguous().view(torch.uint8).view(-1), kind, 512, 1, (512, 1))
        runs.append(m.prefill(torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"]).cuda()))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_two_prompts_at_once_through_one_layer():
    """Scratch and routes belong to the call: prompts of different lengths on two streams, again and again, give the bits of one alone."""
    layer, acts = W.kogarashi_layer(24, hidden=512, inter=256, experts=16, topk=4, tokens=150, shared=True, pool=8)
    m, _ = run_kogarashi(layer, acts)
    x, n = torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"].copy()).cuda()
    parts = [(x[:150], n[:150]), (x[:37], n[:37].flip(0).contiguous())]
    alone = [m.prefill(a.clone(), b)[0] for a, b in parts]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(6):
        for s, (a, b), want in zip(streams, parts, alone):
            with torch.cuda.stream(s):
                outs.append((m.prefill(a.clone(), b)[0], want))
    torch.cuda.synchronize()
    assert all(torch.equal(got, want) for got, want in outs)
