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
