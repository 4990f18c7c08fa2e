"""Refusals of the dense FP8 product and of the grouped GGUF product, without a GPU: descriptors that break a rule return
cudaErrorInvalidValue before anything is enqueued, the Python calls raise ValueError."""
import ctypes

import pytest
import torch

INVALID = 1
FAKE = 0x10000

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up device addresses must never reach a GPU")


def linear(**kw):
    import darask_inference_engine_b200 as D
    d = D._lib.DaraskFp8Linear()
    d.m, d.n, d.k = 40, 200, 300
    d.x, d.x_ty, d.ldx, d.w, d.ldw, d.w_scales, d.ld_ws, d.out, d.out_ty, d.ldo = FAKE, 0, 300, FAKE, 304, FAKE, 3, FAKE, 30, 200
    d.workspace, d.workspace_bytes = FAKE, D._lib.lib().darask_fp8_linear_workspace_bytes(40, 200, 300, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def grouped(**kw):
    import darask_inference_engine_b200 as D
    d = D._lib.DaraskGgmlGrouped()
    d.groups, d.n, d.k, d.rows, d.ranges = 4, 200, 512, 30, FAKE
    d.x, d.x_ty, d.ldx, d.x_rows, d.topk = FAKE, 0, 512, 30, 1
    d.w, d.w_ty, d.out, d.out_ty, d.ldo = FAKE, 12, FAKE, 0, 200
    d.workspace, d.workspace_bytes = FAKE, D._lib.lib().darask_ggml_grouped_workspace_bytes(30, 512, 0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


LINEAR = [dict(m=-1), dict(n=0), dict(k=0), dict(m=1 << 25), dict(x=0), dict(w=0), dict(w_scales=0), dict(out=0), dict(workspace=0), dict(workspace_bytes=64),
          dict(workspace=FAKE + 16), dict(w=FAKE + 8), dict(ldw=300), dict(ldw=288), dict(ldx=299), dict(ldo=199), dict(ld_ws=2), dict(x_ty=12),
          dict(out_ty=100), dict(out_ty=14), dict(x_scales=FAKE, ld_xs=3), dict(swiglu=1), dict(x=FAKE + 2), dict(out=FAKE + 1),
          dict(x_ty=100, ldx=304), dict(x_ty=100, ldx=304, x_scales=FAKE, ld_xs=2), dict(x_ty=100, ldx=300, x_scales=FAKE, ld_xs=3),
          dict(x_ty=100, ldx=304, x_scales=FAKE, ld_xs=3, x=FAKE + 4), dict(x_ty=100, ldx=608, x_scales=FAKE, ld_xs=3, swiglu=1)]
GROUPED = [dict(groups=0), dict(groups=1025), dict(n=0), dict(k=0), dict(k=300), dict(k=65536 + 256), dict(rows=-1), dict(ranges=0), dict(x=0), dict(w=0), dict(out=0),
           dict(w=FAKE + 8), dict(w_up=FAKE + 4), dict(w_ty=0), dict(w_ty=30), dict(x_ty=12), dict(x_ty=100), dict(out_ty=100), dict(ldx=511), dict(swiglu=1, ldx=1023),
           dict(ldo=199), dict(w_up=FAKE, ldo=399), dict(assignments=FAKE, topk=0), dict(workspace=0), dict(workspace_bytes=64), dict(workspace=FAKE + 64),
           dict(x=FAKE + 2), dict(out=FAKE + 2), dict(x_rows=-1)]


@no_gpu
@pytest.mark.parametrize("entry,make,bad", [("darask_fp8_linear", linear, LINEAR), ("darask_ggml_grouped_gemm", grouped, GROUPED)],
                         ids=["linear", "grouped"])
def test_descriptors_that_break_a_rule_are_refused(entry, make, bad):
    import darask_inference_engine_b200 as D
    call = getattr(D._lib.lib(), entry)
    assert call(None, None) == INVALID
    assert call(ctypes.byref(make()), None) != INVALID                    # the base descriptor passes, and ends in the missing driver
    for change in bad:
        assert call(ctypes.byref(make(**change)), None) == INVALID, change


@no_gpu
def test_empty_batches_enqueue_nothing():
    import darask_inference_engine_b200 as D
    lib = D._lib.lib()
    assert lib.darask_fp8_linear(ctypes.byref(linear(m=0, x=0, out=0, workspace=0)), None) == 0
    assert lib.darask_ggml_grouped_gemm(ctypes.byref(grouped(rows=0, x_rows=0, x=0, out=0, ranges=0, workspace=0)), None) == 0


def test_the_structs_of_the_header_match_their_mirrors(tmp_path):
    import os
    import subprocess

    import darask_inference_engine_b200 as D
    structs = [D._lib.DaraskFp8Linear, D._lib.DaraskGgmlGrouped]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "darask_moe_b200.h"', 'int main(void) {']
    for s in structs:
        lines.append(f'  printf("{s.__name__} %zu\\n", sizeof({s.__name__}));')
        lines += [f'  printf("{s.__name__}.{f} %zu\\n", offsetof({s.__name__}, {f}));' for f, _ in s._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ['  printf("e4m3 %d\\n", DARASK_E4M3);', "  return 0;", "}"]) + "\n")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", inc, str(src), "-o", str(exe)], check=True, capture_output=True)
    out = dict(l.split() for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for s in structs:
        assert int(out[s.__name__]) == ctypes.sizeof(s)
        assert all(int(out[f"{s.__name__}.{f}"]) == getattr(s, f).offset for f, _ in s._fields_)
    assert int(out["e4m3"]) == D.fp8.E4M3


def test_python_refusals_of_the_dense_product():
    import darask_inference_engine_b200 as D
    x, w, ws = torch.zeros(4, 256), torch.zeros(130, 256, dtype=torch.uint8), torch.ones(2, 2)
    for bad, match in ((dict(w=w.float()), "uint8"), (dict(w_scales=ws[:1]), "needs scales"), (dict(w_scales=ws.double()), "float32"),
                       (dict(x=x.double()), "columns"), (dict(x=x[:, :255]), "columns"), (dict(swiglu=True), "columns"),
                       (dict(x=w[:4]), "x_scales"), (dict(x_scales=torch.ones(4, 2)), "x_scales"), (dict(x=w[:4], x_scales=torch.ones(4, 1)), "x_scales"),
                       (dict(out=torch.zeros(4, 129)), "out must"), (dict(out=torch.zeros(4, 130), out_dtype=torch.float16), "out must"), (dict(), "CUDA device")):
        with pytest.raises(ValueError, match=match):
            D.fp8.linear(**{**dict(x=x, w=w, w_scales=ws), **bad})


def test_python_refusals_of_the_grouped_product():
    import darask_inference_engine_b200 as D
    W = D.kogarashi.Weight
    good = W(torch.zeros(3 * 64 * 288, dtype=torch.uint8), 12, 512, 64, (512, 64, 3))
    x, r = torch.zeros(5, 512), torch.zeros(3, 2, dtype=torch.int32)
    for bad, match in ((dict(weight=W(good.data, 0, 512, 64, (512, 64, 3))), "Q4_K or Q6_K"), (dict(weight=W(good.data, 14, 512, 64, (512, 64, 3))), "bytes"),
                       (dict(weight=W(good.data[1:], 12, 512, 64, (512, 64, 3))), "bytes"), (dict(up=W(good.data, 14, 512, 64, (512, 64, 3))), "up must"),
                       (dict(x=x[:, :256]), "columns"), (dict(x=x.double()), "columns"), (dict(swiglu=True), "columns"), (dict(ranges=r[:2]), "ranges"),
                       (dict(ranges=r.long()), "ranges"), (dict(assignments=torch.zeros(5)), "assignments"),
                       (dict(assignments=torch.zeros(5, dtype=torch.int32), topk=0), "assignments"), (dict(out=torch.zeros(5, 63)), "out must"), (dict(), "CUDA device")):
        with pytest.raises(ValueError, match=match):
            D.kogarashi.grouped_gemm(**{**dict(x=x, ranges=r, weight=good), **bad})


@no_gpu
@pytest.mark.parametrize("entry,make,bad", [("darask_fp8_linear", linear, [dict(w_scales=FAKE + 2), dict(x_ty=100, ldx=304, x_scales=FAKE + 1, ld_xs=3)]),
                                            ("darask_ggml_grouped_gemm", grouped, [dict(ranges=FAKE + 2), dict(assignments=FAKE + 1)])], ids=["linear", "grouped"])
def test_scales_and_index_lists_off_their_words_are_refused(entry, make, bad):
    import darask_inference_engine_b200 as D
    for change in bad:
        assert getattr(D._lib.lib(), entry)(ctypes.byref(make(**change)), None) == INVALID, change


@no_gpu
def test_more_tiles_than_the_kernel_counts_are_refused():
    import darask_inference_engine_b200 as D
    d = grouped(groups=1024, n=1 << 20, rows=1 << 25, x_rows=1 << 25, w_up=FAKE, ldo=2 << 20, workspace_bytes=1 << 50)
    assert D._lib.lib().darask_ggml_grouped_gemm(ctypes.byref(d), None) == INVALID


def prefill(**kw):
    import darask_inference_engine_b200 as D
    d = D._lib.KogarashiMoe()
    d.hidden, d.inter, d.experts, d.topk, d.tokens = 512, 256, 8, 2, 5
    for name in ("router_w", "gate_w", "up_w", "down_w", "n", "x", "logits", "ids", "prob", "workspace"):
        setattr(d, name, FAKE)
    d.router_ty, d.gate_ty, d.up_ty, d.down_ty = 0, 12, 12, 14
    for k, v in kw.items():
        setattr(d, k, v)
    d.workspace_bytes = kw.get("workspace_bytes", D._lib.lib().kogarashi_moe_prefill_workspace_bytes(d.hidden, d.inter, d.experts, d.topk, d.tokens))
    return d


@no_gpu
def test_the_prompt_layer_refuses_before_anything_is_enqueued():
    import darask_inference_engine_b200 as D
    call = D._lib.lib().kogarashi_moe_prefill
    assert call(None, 0, None) == INVALID
    assert call(ctypes.byref(prefill()), 0, None) != INVALID              # passes, and ends in the missing driver
    shared = dict(sh_gate_w=FAKE, sh_up_w=FAKE, sh_down_w=FAKE, sh_inp_w=FAKE)
    for change in (dict(gate_w=FAKE + 8), dict(up_w=FAKE + 4), dict(down_w=FAKE + 8), dict(shared, sh_down_w=FAKE + 8), dict(n=FAKE + 2), dict(logits=FAKE + 1),
                   dict(ids=FAKE + 2), dict(hidden=65536 + 256), dict(inter=65536 + 256), dict(workspace=FAKE + 16), dict(workspace_bytes=64), dict(tokens=0),
                   dict(tokens=1 << 27), dict(topk=9), dict(gate_ty=0, up_ty=0), dict(down_ty=30), dict(shared, sh_up_w=0)):
        assert call(ctypes.byref(prefill(**change)), 0, None) == INVALID, change
