// Product grouped by expert over GGUF Q4_K / Q6_K weights:
//   out[i][j] = x[row(i)] . W_g[j]      for the dispatch rows i of every group g
// Q4_K: w = d sc_b q - dmin m_b (sub-blocks of 32 columns), Q6_K: w = d sc_b (q - 32) (sub-blocks of 16 columns), per block
// of 256 columns (kogarashi kernels/native.cu:21-41).
#include "../../include/darask_moe_b200.h"
#include "row_source.cuh"
#include "stream_launch.cuh"

namespace dmoe {

static __device__ unsigned g_ggml_grouped_status;

struct GgmlArgs {
  int groups, n, k;
  long long rows;
  const unsigned* ranges;
  RowSource x;
  long long x_rows;
  const unsigned* assignments;
  int topk;
  const uint8_t* w[2];
  int w_ty, row_bytes;
  void* out;
  int out_ty;
  long long ldo;
  unsigned* status;
};

// column c of a 256-column block at `b` (Q4_K: 144 bytes; Q6_K: the 208 bytes of the device layout, block scale d apart)
DEVI float q4k_value(const uint8_t* b, int c) {
  const float d = __half2float(*reinterpret_cast<const __half*>(b)), dm = __half2float(*reinterpret_cast<const __half*>(b + 2));
  const int s = c >> 5, q = (b[16 + (c >> 6) * 32 + (c & 31)] >> (4 * (s & 1))) & 15;
  const int sc = s < 4 ? b[4 + s] & 63 : (b[8 + s] & 15) | ((b[s] >> 6) << 4);
  const int mi = s < 4 ? b[8 + s] & 63 : (b[8 + s] >> 4) | ((b[4 + s] >> 6) << 4);
  return fmaf(d * sc, float(q), -dm * mi);
}
DEVI float q6k_value(const uint8_t* b, float d, int c) {
  const int h = c >> 7, p = (c >> 5) & 3, l = c & 31;
  const int q = ((b[h * 64 + (p & 1) * 32 + l] >> (p >> 1) * 4) & 15) | (((b[128 + h * 32 + l] >> (2 * p)) & 3) << 4);
  return d * float(int(static_cast<int8_t>(b[192 + (c >> 4)])) * (q - 32));
}

// Block (32 weight rows, matrix and group): 32 rows at a time, one 256-column block of both operands in shared memory.
__global__ void __launch_bounds__(256) ggml_grouped_kernel(const GgmlArgs a) {
  extern __shared__ float sm[];
  float(*wt)[257] = reinterpret_cast<float(*)[257]>(sm);
  float(*xt)[257] = reinterpret_cast<float(*)[257]>(sm + 32 * 257);
  pdl_wait();
  pdl_launch();
  const int j0 = blockIdx.x * 32, g = blockIdx.y, mat = blockIdx.z, nblk = a.k / 256;
  long long rows = a.ranges[2 * g];
  const long long first = a.ranges[2 * g + 1];
  if (first + rows > a.rows) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadRoute);
    rows = first < a.rows ? a.rows - first : 0;
  }
  const uint8_t* w = a.w[mat] + size_t(g) * a.n * a.row_bytes;
  const int tj = threadIdx.x & 31, ti = threadIdx.x >> 5;
  for (long long i0 = 0; i0 < rows; i0 += 32) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < nblk; ++b) {
      __syncthreads();
      for (int e = threadIdx.x; e < 32 * 256; e += 256) {
        const int r = e >> 8, c = e & 255;
        float v = 0.f;
        if (j0 + r < a.n) {
          const uint8_t* row = w + size_t(j0 + r) * a.row_bytes;
          v = a.w_ty == DARASK_GGML_Q4_K
                  ? q4k_value(row + b * 144, c)
                  : q6k_value(row + b * 208, __half2float(*reinterpret_cast<const __half*>(row + nblk * 208 + 2 * b)), c);
        }
        wt[r][c] = v;
      }
      for (int e = threadIdx.x; e < 32 * 64; e += 256) {
        const int r = e >> 6, c = (e & 63) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (i0 + r < rows) {
          const long long row = a.assignments ? a.assignments[first + i0 + r] / a.topk : first + i0 + r;
          if (row < a.x_rows) row_source_load4(a.x, row, b * 256 + c, v);
          else atomicOr(a.status, kStatusBadRoute);
        }
        for (int q = 0; q < 4; ++q) xt[r][c + q] = v[q] - v[q] == 0.f ? v[q] : __uint_as_float(0x7fffffffu);   // infinities as NaN
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float p = 0.f;
        for (int c = 0; c < 256; ++c) p = fmaf(xt[ti + 8 * q][c], wt[tj][c], p);
        acc[q] += p;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i0 + ti + 8 * q < rows && j0 + tj < a.n)
        store_elem(a.out, a.out_ty, size_t(first + i0 + ti + 8 * q) * size_t(a.ldo) + size_t(mat) * a.n + j0 + tj, acc[q]);
  }
}

}  // namespace dmoe

using namespace dmoe;

static int ggml_row_bytes(int ty, int k) {
  return ty == DARASK_GGML_Q4_K ? k / 256 * 144 : ty == DARASK_GGML_Q6_K ? k / 256 * 208 + (2 * (k / 256) + 15) / 16 * 16 : 0;
}

extern "C" size_t darask_ggml_grouped_workspace_bytes(long long rows, int k, int x_ty) {
  return rows < 1 || k < 1 || !row_type_bytes(x_ty) ? 0 : 256;
}

static bool grouped_ok(const DaraskGgmlGrouped* d) {
  if (!d || d->groups < 1 || d->groups > 1024 || d->n < 1 || d->n > (1 << 20) || d->k < 256 || d->k > (1 << 16) || d->k % 256) return false;
  if (d->rows < 0 || d->rows > (1ll << 27) || d->x_rows < 0 || d->x_rows > (1ll << 31) - 1) return false;
  if (!d->w || reinterpret_cast<uintptr_t>(d->w) % 16 || reinterpret_cast<uintptr_t>(d->w_up) % 16 || !ggml_row_bytes(d->w_ty, d->k)) return false;
  const size_t eb = row_type_bytes(d->x_ty), ob = row_type_bytes(d->out_ty);
  if (!eb || !ob || d->ldx < (d->swiglu ? 2ll : 1ll) * d->k || d->ldo < (d->w_up ? 2ll : 1ll) * d->n) return false;
  if (d->assignments && d->topk < 1) return false;
  if (d->rows == 0) return true;
  if (!d->ranges || !d->out || reinterpret_cast<uintptr_t>(d->out) % ob) return false;
  if (d->x_rows > 0 && (!d->x || reinterpret_cast<uintptr_t>(d->x) % eb)) return false;
  return d->workspace && reinterpret_cast<uintptr_t>(d->workspace) % 256 == 0 &&
         d->workspace_bytes >= darask_ggml_grouped_workspace_bytes(d->rows, d->k, d->x_ty);
}

extern "C" int darask_ggml_grouped_gemm(const DaraskGgmlGrouped* d, cudaStream_t st) {
  if (!grouped_ok(d)) return cudaErrorInvalidValue;
  if (d->rows == 0) return cudaSuccess;
  void* status = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&status, g_ggml_grouped_status);
  if (e) return e;
  GgmlArgs a = {};
  a.groups = d->groups; a.n = d->n; a.k = d->k; a.rows = d->rows; a.ranges = d->ranges;
  a.x = RowSource{d->x, d->ldx, d->x_ty, d->k, d->swiglu, row_source_vec(d->x, d->x_ty, d->ldx, d->k, d->swiglu)};
  a.x_rows = d->x_rows; a.assignments = d->assignments; a.topk = d->topk;
  a.w[0] = static_cast<const uint8_t*>(d->w); a.w[1] = static_cast<const uint8_t*>(d->w_up);
  a.w_ty = d->w_ty; a.row_bytes = ggml_row_bytes(d->w_ty, d->k);
  a.out = d->out; a.out_ty = d->out_ty; a.ldo = d->ldo; a.status = static_cast<unsigned*>(status);
  const size_t smem = 2 * 32 * 257 * 4;
  if ((e = cudaFuncSetAttribute(ggml_grouped_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)))) return e;
  return launch_pdl(ggml_grouped_kernel, dim3((d->n + 31) / 32, d->groups, d->w_up ? 2 : 1), dim3(256), smem, st, a);
}

extern "C" int darask_ggml_grouped_status(unsigned* host_status, cudaStream_t st) {
  if (!host_status) return cudaErrorInvalidValue;
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_ggml_grouped_status);
  if (!e) e = cudaMemcpyAsync(host_status, p, 4, cudaMemcpyDeviceToHost, st);
  if (!e) e = cudaMemsetAsync(p, 0, 4, st);
  return e ? e : cudaStreamSynchronize(st);
}
