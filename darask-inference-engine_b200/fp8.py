"""Host-side mirror of the FP8 prefill MoE path: block-scaled e4m3 expert weights, e4m3 activations, grouped
products on the tcgen05 tensor cores.

Reference: `prefill_experts`, engines/hayate/crates/models/src/glm53/gpu.rs:2068-2566 (route, group the routes by
expert, gather rows, grouped gate/up product, SwiGLU, grouped down product, scatter with the routing weights); weight
format `Fp8Block`, engines/hayate/crates/kernels/src/cpu/glm53.rs:23-24.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

E4M3 = 100      # DARASK_E4M3: rows of e4m3 codes where a float type is named otherwise


def grouped_gemm(a_codes, a_scales, ranges, w0, sw0, w1=None, sw1=None, quantize=False, row_map=None):
    """Ragged grouped product. a_codes uint8 [rows(+pad), k], a_scales float32 [rows(+pad), k/128], ranges uint32
    [E, 2] = {rows, offset}, w uint8 [E, n, k], sw float32 [E, n/128, k/128].  Without w1: float32 a w0^T (dispatch
    row i written to row row_map[i] when a map is given).  With w1: bf16 silu(a w0^T) * (a w1^T), or with `quantize`
    its e4m3 codes and float32 scales per row and 128 columns.  Rows outside every range are left untouched."""
    experts, n, k = w0.shape
    rows = a_codes.shape[0]
    dev = a_codes.device
    mode = 0 if w1 is None else (2 if quantize else 1)
    out = torch.zeros(rows, n, dtype=(torch.float32, torch.bfloat16, torch.uint8)[mode], device=dev)
    scales = torch.zeros(rows, n // 128, dtype=torch.float32, device=dev) if mode == 2 else None
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    st = torch.cuda.current_stream(dev).cuda_stream
    _lib.check(_lib.lib().darask_fp8_grouped_gemm(
        a_codes.data_ptr(), a_scales.data_ptr(), rows, w0.data_ptr(), w1.data_ptr() if mode else None, sw0.data_ptr(),
        sw1.data_ptr() if mode else None, experts, n, k, mode, ranges.data_ptr(), out.data_ptr(),
        scales.data_ptr() if mode == 2 else None, row_map.data_ptr() if row_map is not None else None, status.data_ptr(), st),
        "darask_fp8_grouped_gemm")
    if int(status.item()):
        raise RuntimeError(f"darask_fp8_grouped_gemm: device status {int(status.item()):#x}")
    return (out, scales) if mode == 2 else out


def linear(x, w, w_scales, x_scales=None, swiglu=False, out_dtype=None, out=None, add=False, status=None):
    """Dense product in block-scaled FP8, x [m, k] -> [m, n].  w uint8 (e4m3 codes) [n, k], w_scales float32 [ceil(n/128), >= ceil(k/128)]
    (``quantize.fp8_block``).  x float32, float16 or bfloat16 is quantized by the call with one scale per row and 128 columns; with
    `swiglu` its rows hold gate | up ([m, 2k]) and silu(gate) * up is quantized.  x uint8 holds e4m3 codes, with x_scales float32
    [m, >= ceil(k/128)] (``quantize.fp8_act``).  Sums are float32; `out_dtype` (float32, float16, bfloat16) defaults to x's type, or
    bfloat16 for codes.  With `add` the product is added to what a float32 `out` holds.  `out` must not overlap an input.  Rows
    may be strided; rows of w and of codes start on 16-byte boundaries.  Any m, including 0; k as w has it.
    `status`: one int32 on the device to which the call's status bits are added (OR); without it they go to the device's shared word,
    which `linear_status` reads.  Runs on the current stream of x's device and does not synchronize; the scratch belongs to the call."""
    if w.dim() != 2 or w.dtype is not torch.uint8 or w_scales.dim() != 2 or w_scales.dtype is not torch.float32:
        raise ValueError("w must be uint8 [n, k] and w_scales float32 [n blocks, k blocks]")
    n, k = w.shape
    kb = (k + 127) // 128
    ws_rows, ws_cols = w_scales.shape
    if n < 1 or k < 1 or ws_rows < (n + 127) // 128 or ws_cols < kb:
        raise ValueError(f"w [{n}, {k}] needs scales [{(n + 127) // 128}, {kb}], got {list(w_scales.shape)}")
    codes = x.dtype is torch.uint8
    ty = E4M3 if codes else _lib.float_type(x.dtype)
    if ty is None or x.dim() != 2 or x.shape[1] != (2 * k if swiglu else k) or (codes and swiglu):
        raise ValueError(f"x must be uint8 codes or float32 / float16 / bfloat16 rows of {2 * k if swiglu else k} columns")
    m = x.shape[0]
    if codes is (x_scales is None) or (codes and (x_scales.dim() != 2 or x_scales.dtype is not torch.float32 or x_scales.shape[0] != m or
                                                  x_scales.shape[1] < kb)):
        raise ValueError(f"codes come with x_scales float32 [{m}, {kb}], float rows without")
    if add and (out is None or out.dtype is not torch.float32):
        raise ValueError("add needs a float32 out to add to")
    if out is None:
        out = x.new_empty((m, n), dtype=out_dtype or (torch.bfloat16 if codes else x.dtype))
    elif tuple(out.shape) != (m, n) or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out must be [{m}, {n}]")
    out_ty = _lib.float_type(out.dtype)
    dev = x.get_device()
    ldx, ldw, ldws, ldo, ldxs = _lib.row_stride(x), _lib.row_stride(w), _lib.row_stride(w_scales), _lib.row_stride(out), 0
    if codes:
        ldxs = _lib.row_stride(x_scales) if x_scales.get_device() == dev else -1
    if out_ty is None or dev < 0 or w.get_device() != dev or w_scales.get_device() != dev or out.get_device() != dev or \
            min(ldx, ldw, ldws, ldo, ldxs) < 0:
        raise ValueError("tensors must share one CUDA device, with unit column stride and rows that do not overlap; "
                         "out must be float32, float16 or bfloat16")
    xp, wp = x.data_ptr(), w.data_ptr()
    if wp % 16 or ldw % 16 or (codes and m and (xp % 16 or ldx % 16)):
        raise ValueError("rows of w and of codes must start on 16-byte boundaries")
    word = None if status is None else _lib.status_pointer(status, dev)
    if m == 0:
        return out
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return linear(x, w, w_scales, x_scales, swiglu, None, out, add, status)
    lib = _lib.lib()
    nbytes = lib.darask_fp8_linear_workspace_bytes(m, n, k, ty)
    scratch = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    d = _lib.DaraskFp8Linear(m, n, k, xp, ty, ldx, x_scales.data_ptr() if codes else None, ldxs, 1 if swiglu else 0, wp, ldw,
                             w_scales.data_ptr(), ldws, out.data_ptr(), out_ty, ldo, 1 if add else 0, scratch.data_ptr() if nbytes else None, nbytes,
                             word)
    _lib.check(lib.darask_fp8_linear(ctypes.byref(d), _lib.current_stream(dev)), "darask_fp8_linear")
    return out


def linear_status(device="cuda") -> int:
    """Status bits that `linear` calls without a `status` of their own have set on this device since the last look; clears them and
    synchronizes the current stream."""
    s = ctypes.c_uint(0)
    device = torch.device(device)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().darask_fp8_linear_status(ctypes.byref(s), torch.cuda.current_stream(device).cuda_stream), "darask_fp8_linear_status")
    return s.value


class Fp8MoeLayer:
    def __init__(self, hidden: int, inter: int, experts: int, topk: int, max_tokens: int, device="cuda"):
        self.hidden, self.inter, self.experts, self.topk, self.max_tokens = hidden, inter, experts, topk, max_tokens
        self.device = torch.device(device)
        nbytes = _lib.lib().darask_fp8_moe_workspace_bytes(hidden, inter, experts, topk, max_tokens)
        self.workspace = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        self.ids = torch.empty(max_tokens, topk, dtype=torch.int32, device=self.device)
        self.prob = torch.empty(max_tokens, topk, dtype=torch.float32, device=self.device)
        self.w = {}
        self.shared = None
        self._shared_status = torch.zeros(1, dtype=torch.int32, device=self.device)

    def _stream(self):
        return torch.cuda.current_stream(self.device).cuda_stream

    def load_shared(self, gate, up, down) -> None:
        """An always-on shared expert in the same format, added to the routed sum (hayate cu/glm53/decode.cu:55-59): gate and up
        (payload uint8 [F, H], scales float32 [F/128, H/128]), down (payload [H, F], scales [H/128, F/128]); F a multiple of 128 of
        its own.  Its products are the dense ones of `linear`: gate | up in one, SwiGLU and the quantizer in front of down."""
        f = gate[0].shape[0]
        if f < 128 or f % 128:
            raise ValueError("the shared expert's intermediate width must be a multiple of 128")
        for name, (p, s), (n, k) in (("gate", gate, (f, self.hidden)), ("up", up, (f, self.hidden)), ("down", down, (self.hidden, f))):
            if tuple(p.shape) != (n, k) or tuple(s.shape) != (n // 128, k // 128):
                raise ValueError(f"shared {name}: expected payload [{n},{k}] and scales [{n // 128},{k // 128}]")
        put = lambda t, ty: t.to(self.device, ty).contiguous()
        self.shared = (put(torch.cat([gate[0], up[0]]), torch.uint8), put(torch.cat([gate[1], up[1]]), torch.float32),
                       put(down[0], torch.uint8), put(down[1], torch.float32))

    def load(self, name: str, payload: torch.Tensor, scales: torch.Tensor) -> None:
        """name in gate|up|down; payload uint8 [E, n, k]; scales float32 [E, n/128, k/128]."""
        n, k = (self.hidden, self.inter) if name == "down" else (self.inter, self.hidden)
        if tuple(payload.shape) != (self.experts, n, k) or tuple(scales.shape) != (self.experts, n // 128, k // 128):
            raise ValueError(f"{name}: expected payload [E,{n},{k}] and scales [E,{n // 128},{k // 128}]")
        self.w[name] = (payload.to(self.device, torch.uint8).contiguous(), scales.to(self.device, torch.float32).contiguous())

    def forward(self, x: torch.Tensor, logits: torch.Tensor) -> torch.Tensor:
        """x bf16 [T,H], logits float32 [T,E] -> float32 [T,H] (the routed experts' weighted sum, and the shared expert if loaded)."""
        t = x.shape[0]
        if t > self.max_tokens or x.dtype != torch.bfloat16 or logits.dtype != torch.float32 or not x.is_contiguous() or not logits.is_contiguous():
            raise ValueError("x must be contiguous bf16 [T<=max_tokens,H], logits contiguous float32 [T,E]")
        out = torch.empty(t, self.hidden, dtype=torch.float32, device=self.device)
        d = _lib.DaraskFp8Moe()
        d.hidden, d.inter, d.experts, d.topk, d.tokens = self.hidden, self.inter, self.experts, self.topk, t
        d.x, d.logits = x.data_ptr(), logits.data_ptr()
        (gw, gs), (uw, us), (dw, ds) = self.w["gate"], self.w["up"], self.w["down"]
        d.gate_w, d.up_w, d.down_w = gw.data_ptr(), uw.data_ptr(), dw.data_ptr()
        d.gate_s, d.up_s, d.down_s = gs.data_ptr(), us.data_ptr(), ds.data_ptr()
        d.out, d.ids, d.prob = out.data_ptr(), self.ids.data_ptr(), self.prob.data_ptr()
        d.workspace, d.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
        _lib.check(_lib.lib().darask_fp8_moe_layer(ctypes.byref(d), self._stream()), "darask_fp8_moe_layer")
        if self.shared is not None:
            gu_w, gu_s, down_w, down_s = self.shared
            rows = linear(x, gu_w, gu_s, out_dtype=torch.float32, status=self._shared_status)
            linear(rows, down_w, down_s, swiglu=True, out=out, add=True, status=self._shared_status)
        return out

    def status(self) -> int:
        """Status bits of the last call's routed experts and of the shared expert's products since the last look; synchronizes."""
        s = ctypes.c_uint(0)
        _lib.check(_lib.lib().darask_fp8_moe_status(self.workspace.data_ptr(), ctypes.byref(s), self._stream()), "darask_fp8_moe_status")
        return s.value | _lib.take_status(self._shared_status)
