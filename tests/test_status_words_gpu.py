"""Status words of the dense FP8 product, of the grouped GGUF product and of the layers on them: no bit is lost, none is another caller's,
and a layer's own `status` tells what its products met."""
import ctypes
import threading
import time

import numpy as np
import pytest
import torch

from oracle import formats as F
from tests import workloads as W
from tests.test_ggml_grouped_gpu import Q4, ranges_of, weight

pytestmark = pytest.mark.gpu

BAD_ROUTE = 2


def bad_call(groups=1, **kw):
    """A call whose range leaves the rows: it is cut and reported."""
    import darask_inference_engine_b200 as D
    w, _, _ = weight(3, Q4, 1, 128, 256)
    x = torch.ones(4, 256, device="cuda")
    bad = torch.tensor([[9, 0]], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return lambda: D.kogarashi.grouped_gemm(x, bad, w, **kw)


def test_no_bit_is_lost_while_another_thread_reads():
    """One thread reads and clears the device's word all the time, another makes calls that set it: each call is reported. (A copy and a
    clear of their own lost the bits that were set between the two.)"""
    import darask_inference_engine_b200 as D
    call, reads, stop, failed = bad_call(), [], threading.Event(), []

    def reader():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not stop.is_set():
                    reads.append(D.kogarashi.grouped_status())
        except Exception as e:      # noqa: BLE001
            failed.append(e)

    def wait_for(count):
        end = time.monotonic() + 20
        while len(reads) < count and not failed and time.monotonic() < end:
            time.sleep(0)
        assert len(reads) >= count and not failed

    call()
    torch.cuda.synchronize()
    D.kogarashi.grouped_status()
    t = threading.Thread(target=reader, daemon=True)
    t.start()
    lost = 0
    try:
        for _ in range(400):
            wait_for(len(reads) + 1)
            before = len(reads)
            call()
            torch.cuda.current_stream().synchronize()
            wait_for(len(reads) + 2)                     # a whole reading after the call has ended
            lost += not any(v & BAD_ROUTE for v in reads[before:])
    finally:
        stop.set()
        t.join(20)
    assert lost == 0


def test_a_word_of_the_callers():
    """Bits go to the word that a call is given, and to no other; words of two calls on two streams are apart."""
    import darask_inference_engine_b200 as D
    D.kogarashi.grouped_status()
    own, other = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    bad_call(status=own)()
    w, _, _ = weight(3, Q4, 1, 128, 256)
    x = torch.ones(4, 256, device="cuda")
    D.kogarashi.grouped_gemm(x, ranges_of([4]), w, status=other)
    assert D.kogarashi.grouped_status() == 0
    assert D._lib.take_status(own) == BAD_ROUTE and D._lib.take_status(own) == 0 and D._lib.take_status(other) == 0
    cw, cs = D.quantize.fp8_block(torch.randn(64, 128, device="cuda"))
    D.fp8.linear(x[:, :128], cw, cs, status=own)
    assert D._lib.take_status(own) == 0 and D.fp8.linear_status() == 0
    for bad in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="status"):
            D.fp8.linear(x[:, :128], cw, cs, status=bad)
        with pytest.raises(ValueError, match="status"):
            D.kogarashi.grouped_gemm(x, ranges_of([4]), w, status=bad)


def test_two_readers_at_once():
    """Of a bit that is set once, one of the readers hears and the others do not."""
    import darask_inference_engine_b200 as D
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(20):
        word.fill_(5)
        torch.cuda.synchronize()
        got = []

        def read():
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append(D._lib.take_status(word))
        threads = [threading.Thread(target=read) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(20)
        assert sorted(got) == [0, 0, 0, 5]


def test_the_status_of_a_prompt_outlives_its_scratch():
    """Bits in a call's workspace reach the caller's word. The bits come from the test, written to the workspace's status word from another
    stream while the call runs (its own launches have no way to set one for a valid call)."""
    import darask_inference_engine_b200 as D
    from tests.test_kogarashi_gpu import run_layer
    lib = D._lib.lib()
    tokens = 900
    layer, acts = W.kogarashi_layer(26, hidden=512, inter=256, experts=16, topk=4, tokens=tokens, shared=True, pool=8)
    m, _ = run_layer(layer, {**acts, "x": acts["x"][:1], "n": acts["n"][:1]})
    x, n = torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"].copy()).cuda()
    d = m._descriptor(x, n, None, None, 1e-6)
    logits, ids, prob = torch.empty(tokens, 16, device="cuda"), torch.empty(tokens, 4, dtype=torch.int32, device="cuda"), torch.empty(tokens, 4, device="cuda")
    d.logits, d.ids, d.prob = logits.data_ptr(), ids.data_ptr(), prob.data_ptr()
    nbytes = lib.kogarashi_moe_prefill_workspace_bytes(512, 256, 16, 4, tokens)
    ws = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = ws.data_ptr(), nbytes
    total = torch.zeros(1, dtype=torch.int32, device="cuda")
    host = ctypes.c_uint(0)
    # where the workspace keeps its status word: the one that kogarashi_moe_status reads
    for at in range(0, 4096, 256):
        ws.zero_()
        ws[at:at + 4].view(torch.int32).fill_(1 << 20)
        D._lib.check(lib.kogarashi_moe_status(ws.data_ptr(), ctypes.byref(host), D._lib.current_stream(0)), "status")
        if host.value == 1 << 20:
            break
    else:
        raise AssertionError("no status word found")
    word = ws[at:at + 4].view(torch.int32)

    def call():
        D._lib.check(lib.kogarashi_moe_prefill_checked(ctypes.byref(d), 0, total.data_ptr(), D._lib.current_stream(0)), "prefill")
    call()                                               # alone: the bit of before is cleared, none is set
    assert D._lib.take_status(total) == 0
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(400):
            word.fill_(1 << 21)
    seen = 0
    for _ in range(50):                                  # until a call has met one of the writes between its start and its end
        with torch.cuda.stream(side):
            graph.replay()
        for _ in range(4):
            call()
        torch.cuda.synchronize()
        seen |= D._lib.take_status(total)
        if seen:
            break
    assert seen == 1 << 21
    # and the layer's own calls report to the layer
    m.prefill(x, n)
    assert m.status() == 0
    m._prefill_status.fill_(1)
    assert m.status() == 1 and m.status() == 0


def test_prompts_hand_the_layers_word_to_the_library(monkeypatch):
    import darask_inference_engine_b200 as D
    from tests.test_kogarashi_gpu import run_layer
    layer, acts = W.kogarashi_layer(27, hidden=256, inter=256, experts=4, topk=2, tokens=3, shared=False, pool=4)
    m, _ = run_layer(layer, acts)
    real, words = D._lib.lib(), []

    class Recorder:
        def __getattr__(self, name):
            return getattr(real, name)

        def kogarashi_moe_prefill_checked(self, d, given, word, stream):
            words.append(word)
            return real.kogarashi_moe_prefill_checked(d, given, word, stream)
    monkeypatch.setattr(D._lib, "lib", Recorder)
    x, n = torch.from_numpy(acts["x"].copy()).cuda(), torch.from_numpy(acts["n"].copy()).cuda()
    m.prefill(x, n)
    assert words == [m._prefill_status.data_ptr()]
    assert m.status() == 0


def test_the_fp8_layer_reports_its_shared_expert(monkeypatch):
    import darask_inference_engine_b200 as D
    hidden, inter, tokens = 256, 128, 5
    layer, acts = W.fp8_layer(3, hidden, inter, 8, 2, tokens)
    m = D.Fp8MoeLayer(hidden, inter, 8, 2, tokens)
    for name in ("gate", "up", "down"):
        mats = getattr(layer, name)
        m.load(name, torch.from_numpy(np.stack([p for p, _ in mats])), torch.from_numpy(np.stack([s for _, s in mats])))
    rng = W.rng_for(17)
    m.load_shared(*[tuple(torch.from_numpy(a) for a in F.fp8_block_quantize(W.normal(rng, s, s[1] ** -0.5))) for s in ((128, hidden), (128, hidden), (hidden, 128))])
    x, logits = torch.from_numpy(acts["x"]).bfloat16().cuda(), torch.from_numpy(acts["logits"]).cuda()
    want = m.forward(x, logits).clone()
    assert m.status() == 0
    real, words = D.fp8.linear, []

    def linear(*args, status=None, **kw):
        words.append(status)
        out = real(*args, status=status, **kw)
        status.bitwise_or_(len(words))                   # as a wait that runs out in the first or the second product would
        return out
    monkeypatch.setattr(D.fp8, "linear", linear)
    assert torch.equal(m.forward(x, logits), want)
    assert len(words) == 2 and m.status() == 3 and m.status() == 0
    assert D.fp8.linear_status() == 0
