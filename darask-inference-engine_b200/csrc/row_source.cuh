// Rows of activations as the dense FP8 product and the grouped GGUF product read them: float32, bf16 or f16 with a row
// stride, either as they are or as gate | up halves of which silu(gate) * up is taken (float32, both halves exact).
#pragma once
#include "../../include/darask_moe_b200.h"
#include "common.cuh"

namespace dmoe {

struct RowSource {
  const void* x;
  long long ld;          // elements from row to row
  int ty;                // DARASK_GGML_F32 / F16 / BF16
  int k;                 // columns of the operand; swiglu: column c of the gate half, k + c of the up half
  int swiglu;
  int vec;               // 1: four elements from a multiple of four columns can be loaded as one word; 2: eight 16-bit ones too
};

// The four-wide loads need the base and the row stride (and, for the up half, k) on a boundary of four elements.
inline int row_source_vec(const void* x, int ty, long long ld, int k, int swiglu) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  if (at % (ty == DARASK_GGML_F32 ? 16 : 8) || ld % 4 || (swiglu && k % 4)) return 0;
  return ty != DARASK_GGML_F32 && at % 16 == 0 && ld % 8 == 0 ? 2 : 1;
}
inline size_t row_type_bytes(int ty) { return ty == DARASK_GGML_F32 ? 4 : ty == DARASK_GGML_F16 || ty == DARASK_GGML_BF16 ? 2 : 0; }

// Loads pass L1 by here and in the kernels behind: nothing says that a launch which starts while its predecessor drains finds L1
// cleared of lines that have been rewritten since.
DEVI float load_elem(const void* p, int ty, size_t i) {
  if (ty == DARASK_GGML_F32) return __ldcg(static_cast<const float*>(p) + i);
  const unsigned short u = __ldcg(static_cast<const unsigned short*>(p) + i);
  return ty == DARASK_GGML_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float(uint32_t(u) << 16);
}
// elements i .. i + 3, i a multiple of four on an aligned base
DEVI void load_elem4(const void* p, int ty, size_t i, float (&v)[4]) {
  if (ty == DARASK_GGML_F32) {
    const float4 f = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    return;
  }
  const uint2 u = __ldcg(reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i));
  if (ty == DARASK_GGML_F16) {
    v[0] = half_lo(u.x); v[1] = half_hi(u.x); v[2] = half_lo(u.y); v[3] = half_hi(u.y);
  } else {
    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}
// columns c .. c + 3 of a row (c a multiple of four); columns past k read as zero
DEVI void row_source_load4(const RowSource& s, long long row, int c, float (&v)[4]) {
  const size_t at = size_t(row) * size_t(s.ld) + size_t(c);
  if (s.vec && c + 4 <= s.k) {
    load_elem4(s.x, s.ty, at, v);
    if (s.swiglu) {
      float u[4];
      load_elem4(s.x, s.ty, at + size_t(s.k), u);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = silu_mul(v[i], u[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = 0.f;
    if (c + i < s.k) {
      v[i] = load_elem(s.x, s.ty, at + i);
      if (s.swiglu) v[i] = silu_mul(v[i], load_elem(s.x, s.ty, at + size_t(s.k) + i));
    }
  }
}

// one result in the output's type, rounded once from float32; `add`: on top of what is there
DEVI void store_elem(void* out, int ty, size_t i, float v, int add = 0) {
  if (add) v += load_elem(out, ty, i);
  if (ty == DARASK_GGML_F32) static_cast<float*>(out)[i] = v;
  else if (ty == DARASK_GGML_F16) static_cast<__half*>(out)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

}  // namespace dmoe
