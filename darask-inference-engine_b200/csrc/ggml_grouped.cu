// Product grouped by expert over GGUF Q4_K / Q6_K weights:
//   out[i][j] = x[row(i)] . W_g[j]      for the dispatch rows i of every group g
// Q4_K: w = d sc_b q - dmin m_b (sub-blocks of 32 columns), Q6_K: w = d sc_b (q - 32) (sub-blocks of 16 columns), per block
// of 256 columns (kogarashi kernels/native.cu:21-41).
#include "../../include/darask_moe_b200.h"
#include "ggml_grouped.cuh"
#include "status.cuh"

namespace dmoe {

static __device__ unsigned g_ggml_grouped_status;
static cudaError_t status_word(unsigned** p) {
  static unsigned* known[64] = {};
  return device_word(g_ggml_grouped_status, known, p);
}

static int ggml_row_bytes(int ty, int k) {
  return ty == DARASK_GGML_Q4_K ? k / 256 * 144 : ty == DARASK_GGML_Q6_K ? k / 256 * 208 + (2 * (k / 256) + 15) / 16 * 16 : 0;
}

// f16 parts of a row: float32 numbers (the rows themselves, or SwiGLU products of any rows) take two
static int row_parts(int x_ty, int swiglu) { return x_ty == DARASK_GGML_F32 || swiglu ? 2 : 1; }

struct GroupedWs { __half* planes; __half* sum; float* scale; size_t bytes; };
static GroupedWs carve(void* base, long long rows, int k, int parts) {
  GroupedWs w;
  uint8_t* p = static_cast<uint8_t*>(base);
  size_t off = 0;
  auto take = [&](size_t bytes) { uint8_t* q = p ? p + off : nullptr; off = (off + bytes + 255) / 256 * 256; return q; };
  w.planes = reinterpret_cast<__half*>(take(size_t(parts) * size_t(rows) * k * 2));
  w.sum = reinterpret_cast<__half*>(take(size_t(rows) * (k / 256) * 32));
  w.scale = reinterpret_cast<float*>(take(size_t(rows) * 4));
  w.bytes = off;
  return w;
}

template <bool Q6, int NT, int NX, typename OUT>
static cudaError_t launch_products(const CUtensorMap (&m)[6], const GgArgs& a, cudaStream_t st) {
  using S = GgShape<Q6, NT, NX>;
  static_assert(S::kSmem + 3 * 1024 <= kSmemBudget, "rings and 3 KB of barriers and scales must fit one block");
  static bool configured[64] = {};      // the opt-in is per device and per kernel
  const int dev = current_device_slot();
  if (dev < 0) return cudaErrorInvalidDevice;
  auto kernel = ggml_grouped_kernel<Q6, NT, NX, OUT>;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_pdl(kernel, dim3(sm_count()), dim3(S::kThreads), size_t(S::kSmem), st, m[0], m[1], m[2], m[3], m[4], m[5], a);
}

template <int KIND>
static cudaError_t launch_rows(const GgRowsArgs& r, int parts, bool sums, cudaStream_t st) {
  constexpr bool kOne = KIND == 2 || KIND == 3;          // plain 16-bit rows have one part, float32 and SwiGLU rows two
  auto kernel = sums ? ggml_rows_kernel<KIND, !kOne, true> : ggml_rows_kernel<KIND, !kOne, false>;
  if constexpr (KIND == 0)
    if (parts == 1) kernel = sums ? ggml_rows_kernel<KIND, false, true> : ggml_rows_kernel<KIND, false, false>;
  const size_t smem = size_t(r.src.k < kGgRowHeld ? r.src.k : kGgRowHeld) * sizeof(float);
  return launch_pdl(kernel, dim3(unsigned(r.rows)), dim3(kGgRowThreads), smem, st, r);
}

// Every output type takes all that the operands hold. With one part of two-part rows (11 bits of 22) and one term of Q6_K's integers in front
// of bf16 and f16, bf16 results were off by up to 1.73e-3 and f16 ones by 2.6e-4, where their own roundings are 1.66e-3 and 2.07e-4; the
// second part and the second term cost bf16 results 12 to 30 % of the time (32768 rows, 128 groups of 2048 x 768 Q6_K: 286 -> 314 us for bf16
// rows, 288 -> 347 us for float32 rows).
template <bool Q6, int NT, typename OUT>
static cudaError_t launch_by_parts(int parts, const CUtensorMap (&m)[6], const GgArgs& a, cudaStream_t st) {
  return parts == 2 ? launch_products<Q6, NT, 2, OUT>(m, a, st) : launch_products<Q6, NT, 1, OUT>(m, a, st);
}
template <bool Q6, int NT>
static cudaError_t launch_by_type(int out_ty, int parts, const CUtensorMap (&m)[6], const GgArgs& a, cudaStream_t st) {
  if (out_ty == DARASK_GGML_F32) return launch_by_parts<Q6, NT, float>(parts, m, a, st);
  if (out_ty == DARASK_GGML_F16) return launch_by_parts<Q6, NT, __half>(parts, m, a, st);
  return launch_by_parts<Q6, NT, __nv_bfloat16>(parts, m, a, st);
}

}  // namespace dmoe

using namespace dmoe;

extern "C" size_t darask_ggml_grouped_workspace_bytes(long long rows, int k, int x_ty, int swiglu) {
  if (rows < 1 || k < 256 || k % 256 || !row_type_bytes(x_ty)) return 0;
  return carve(nullptr, rows, k, row_parts(x_ty, swiglu)).bytes;
}

// Few rows per group, narrow tiles: the weights' bytes pace the product then (16 rows in 256 groups: 85 us). The host knows the rows and the
// groups, not which groups have rows: where a few of many groups take nearly all rows, these go through narrow tiles too and expand
// their codes four times as often as wide ones would.
static bool grouped_narrow(const DaraskGgmlGrouped* d) { return d->rows <= 32ll * d->groups; }
// one more than the tiles of ranges that do not overlap
static long long grouped_tile_cap(const DaraskGgmlGrouped* d) {
  return (d->rows / (grouped_narrow(d) ? 32 : 128) + d->groups) * ((d->n + 127) / 128) * (d->w_up ? 2 : 1) + 1;
}
static bool grouped_ok(const DaraskGgmlGrouped* d) {
  if (!d || d->groups < 1 || d->groups > 1024 || d->n < 1 || d->n > (1 << 20) || d->k < 256 || d->k > (1 << 16) || d->k % 256) return false;
  if (d->rows < 0 || d->rows > (1ll << 27) || d->x_rows < 0 || d->x_rows > (1ll << 31) - 1) return false;
  if (!d->w || reinterpret_cast<uintptr_t>(d->w) % 16 || reinterpret_cast<uintptr_t>(d->w_up) % 16 || !ggml_row_bytes(d->w_ty, d->k)) return false;
  const size_t eb = row_type_bytes(d->x_ty), ob = row_type_bytes(d->out_ty);
  if (!eb || !ob || d->ldx < (d->swiglu ? 2ll : 1ll) * d->k || d->ldo < (d->w_up ? 2ll : 1ll) * d->n) return false;
  if (reinterpret_cast<uintptr_t>(d->status) % 4) return false;
  if (d->assignments && (d->topk < 1 || reinterpret_cast<uintptr_t>(d->assignments) % 4)) return false;
  if (grouped_tile_cap(d) >= 1ll << 30) return false;      // tiles are counted in 32 bits, two counts added
  if (d->rows == 0) return true;
  if (!d->ranges || reinterpret_cast<uintptr_t>(d->ranges) % 4 || !d->out || reinterpret_cast<uintptr_t>(d->out) % ob) return false;
  if (d->x_rows > 0 && (!d->x || reinterpret_cast<uintptr_t>(d->x) % eb)) return false;
  return d->workspace && reinterpret_cast<uintptr_t>(d->workspace) % 256 == 0 &&
         d->workspace_bytes >= darask_ggml_grouped_workspace_bytes(d->rows, d->k, d->x_ty, d->swiglu);
}

extern "C" int darask_ggml_grouped_gemm(const DaraskGgmlGrouped* d, cudaStream_t st) {
  if (!grouped_ok(d)) return cudaErrorInvalidValue;
  if (d->rows == 0) return cudaSuccess;
  unsigned* status = d->status;
  cudaError_t e = cudaSuccess;
  if (!status && (e = status_word(&status))) return e;
  const bool q6 = d->w_ty == DARASK_GGML_Q6_K;
  const int parts = row_parts(d->x_ty, d->swiglu), row_bytes = ggml_row_bytes(d->w_ty, d->k), nblk = d->k / 256;
  const GroupedWs ws = carve(d->workspace, d->rows, d->k, parts);
  GgRowsArgs r = {};
  r.src = RowSource{d->x, d->ldx, d->x_ty, d->k, d->swiglu, row_source_vec(d->x, d->x_ty, d->ldx, d->k, d->swiglu)};
  r.rows = d->rows; r.x_rows = d->x_rows; r.assignments = d->assignments; r.topk = d->topk;
  r.planes = ws.planes; r.sum = ws.sum; r.scale = ws.scale;
  const unsigned long long wrows = (unsigned long long)d->groups * d->n, wcols = (unsigned long long)nblk * (q6 ? 208 : 144);
  const unsigned box = q6 ? 208 : 144;
  CUtensorMap m[6];                     // weights (two matrices), rows of x by 32 and by 128, their sums by 32 and by 128
  if (!byte_map(m + 0, d->w, wrows, wcols, row_bytes, 128, box, CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !byte_map(m + 1, d->w_up ? d->w_up : d->w, wrows, wcols, row_bytes, 128, box, CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !byte_map(m + 2, ws.planes, (unsigned long long)parts * d->rows, d->k * 2ull, d->k * 2ull, 32, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !byte_map(m + 3, ws.planes, (unsigned long long)parts * d->rows, d->k * 2ull, d->k * 2ull, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !byte_map(m + 4, ws.sum, d->rows, nblk * 32ull, nblk * 32ull, 32, 32, CU_TENSOR_MAP_SWIZZLE_32B) ||
      !byte_map(m + 5, ws.sum, d->rows, nblk * 32ull, nblk * 32ull, 128, 32, CU_TENSOR_MAP_SWIZZLE_32B))
    return cudaErrorInvalidValue;
  // eight columns at a time where the rows allow it
  const bool whole = r.src.vec >= (d->x_ty == DARASK_GGML_F32 ? 1 : 2) && d->ldx % (d->x_ty == DARASK_GGML_F32 ? 4 : 8) == 0;
  const int kind = !whole ? 0 : (d->x_ty == DARASK_GGML_F32 ? 1 : d->x_ty == DARASK_GGML_F16 ? 2 : 3) + (d->swiglu ? 3 : 0);
  switch (kind) {
    case 0: e = launch_rows<0>(r, parts, !q6, st); break;
    case 1: e = launch_rows<1>(r, parts, !q6, st); break;
    case 2: e = launch_rows<2>(r, parts, !q6, st); break;
    case 3: e = launch_rows<3>(r, parts, !q6, st); break;
    case 4: e = launch_rows<4>(r, parts, !q6, st); break;
    case 5: e = launch_rows<5>(r, parts, !q6, st); break;
    default: e = launch_rows<6>(r, parts, !q6, st);
  }
  if (e) return e;
  GgArgs a = {};
  a.ranges = d->ranges; a.groups = d->groups; a.n = d->n; a.nblk = nblk; a.mats = d->w_up ? 2 : 1; a.row_bytes = row_bytes; a.rows = d->rows;
  a.w[0] = static_cast<const uint8_t*>(d->w); a.w[1] = static_cast<const uint8_t*>(d->w_up);
  a.xscale = ws.scale; a.out = d->out; a.ldo = d->ldo; a.tile_cap = int(grouped_tile_cap(d));
  const size_t ob = row_type_bytes(d->out_ty);
  a.aligned = reinterpret_cast<uintptr_t>(d->out) % 16 == 0 && d->ldo * ob % 16 == 0 && (!d->w_up || d->n * ob % 16 == 0);
  a.status = status;
  const bool narrow = grouped_narrow(d);
  if (q6) return narrow ? launch_by_type<true, 32>(d->out_ty, parts, m, a, st) : launch_by_type<true, 128>(d->out_ty, parts, m, a, st);
  return narrow ? launch_by_type<false, 32>(d->out_ty, parts, m, a, st) : launch_by_type<false, 128>(d->out_ty, parts, m, a, st);
}

extern "C" int darask_ggml_grouped_status(unsigned* host_status, cudaStream_t st) {
  if (!host_status) return cudaErrorInvalidValue;
  unsigned* p = nullptr;
  const cudaError_t e = status_word(&p);
  return e ? e : darask_status_take(p, host_status, st);
}
