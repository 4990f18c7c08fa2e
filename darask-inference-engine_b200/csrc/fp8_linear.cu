// Dense product in block-scaled FP8:
//   out[i][j] = sum over 128-column blocks b of (code(x)[i][b] . W[j][b]) * sx[i][b] * sw[j / 128][b]
// W: e4m3, one float32 scale per 128 x 128 block (hayate `Fp8Block`, cpu/glm53.rs:23-24). x: float rows, quantized here to
// e4m3 with one float32 scale per row and 128 columns (as darask_quantize_fp8_act), or codes and scales as they are.
#include "../../include/darask_moe_b200.h"
#include <cuda_fp8.h>
#include "row_source.cuh"
#include "stream_launch.cuh"

namespace dmoe {

static __device__ unsigned g_fp8_linear_status;

struct Fp8LinearArgs {
  int m, n, k;
  const uint8_t* codes;  // e4m3 rows
  long long ldx;
  const float* xs;
  long long ld_xs;
  const uint8_t* w;
  long long ldw;
  const float* ws;
  long long ld_ws;
  void* out;
  int out_ty;
  long long ldo;
};

// One warp per row and 128 columns, four columns per lane: scale = absmax / 448 (1 for zeros), code = e4m3(x * (1 / scale)),
// every step rounded to float32. A group with an infinity or a NaN gets the scale NaN, so that the row's products say so.
__global__ void __launch_bounds__(256) fp8_linear_quant_kernel(const RowSource src, long long groups, int kb, uint8_t* codes, float* scales) {
  pdl_wait();
  pdl_launch();
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (w >= groups) return;
  const int lane = threadIdx.x & 31, b = int(w % kb);
  float v[4];
  row_source_load4(src, w / kb, b * 128 + lane * 4, v);
  // the bits of |v| grow with |v|, infinity and NaN on top
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  const float scale = top == 0u ? 1.f : top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __uint_as_float(top) / 448.f;
  const float inv = 1.f / scale;
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = v[i] * inv;            // 0 times the infinite reciprocal of a subnormal scale stays 0
    out |= uint32_t(__nv_cvt_float_to_fp8(y == y ? fminf(fmaxf(y, -448.f), 448.f) : 0.f, __NV_SATFINITE, __NV_E4M3)) << (8 * i);
  }
  if (lane == 0) scales[w] = scale;
  reinterpret_cast<uint32_t*>(codes)[w * 32 + lane] = out;
}

// 32 x 32 outputs per block, operands of one 128-column block in shared memory as float32.
__global__ void __launch_bounds__(256) fp8_linear_kernel(const Fp8LinearArgs a) {
  __shared__ float xt[32][129], wt[32][129];
  pdl_wait();
  pdl_launch();
  const int j0 = blockIdx.x * 32;
  for (int i0 = blockIdx.y * 32; i0 < a.m; i0 += gridDim.y * 32) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int tj = threadIdx.x & 31, ti = threadIdx.x >> 5;
    for (int b = 0; b * 128 < a.k; ++b) {
      __syncthreads();
      for (int e = threadIdx.x; e < 32 * 128; e += 256) {
        const int r = e >> 7, c = b * 128 + (e & 127);
        const bool xin = i0 + r < a.m && c < a.k, win = j0 + r < a.n && c < a.k;
        const uint8_t xc = xin ? a.codes[size_t(i0 + r) * size_t(a.ldx) + c] : 0, wc = win ? a.w[size_t(j0 + r) * size_t(a.ldw) + c] : 0;
        xt[r][e & 127] = __half2float(__half(__nv_cvt_fp8_to_halfraw(xc, __NV_E4M3)));
        wt[r][e & 127] = __half2float(__half(__nv_cvt_fp8_to_halfraw(wc, __NV_E4M3)));
      }
      __syncthreads();
      if (j0 + tj < a.n) {
        const float sw = a.ws[size_t((j0 + tj) / 128) * size_t(a.ld_ws) + b];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = ti + 8 * q;
          if (i0 + i >= a.m) continue;
          float p = 0.f;
          for (int c = 0; c < 128; ++c) p = fmaf(xt[i][c], wt[tj][c], p);
          acc[q] = fmaf(p, a.xs[size_t(i0 + i) * size_t(a.ld_xs) + b] * sw, acc[q]);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i0 + ti + 8 * q < a.m && j0 + tj < a.n) store_elem(a.out, a.out_ty, size_t(i0 + ti + 8 * q) * size_t(a.ldo) + j0 + tj, acc[q]);
  }
}

static size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace dmoe

using namespace dmoe;

extern "C" size_t darask_fp8_linear_workspace_bytes(int m, int n, int k, int x_ty) {
  if (m < 1 || n < 1 || k < 1 || x_ty == DARASK_E4M3) return 0;
  const size_t kb = (size_t(k) + 127) / 128;
  return round_up(size_t(m) * kb * 128, 256) + round_up(size_t(m) * kb * 4, 256);
}

static bool linear_ok(const DaraskFp8Linear* d) {
  if (!d || d->m < 0 || d->n < 1 || d->k < 1 || d->m > (1 << 24) || d->n > (1 << 24) || d->k > (1 << 20)) return false;
  if (!d->w || !d->w_scales || reinterpret_cast<uintptr_t>(d->w) % 16 || d->ldw % 16 || d->ldw < d->k) return false;
  const long long kb = (d->k + 127) / 128;
  if (d->ld_ws < kb || !row_type_bytes(d->out_ty) || d->ldo < d->n) return false;
  if (d->m == 0) return true;
  if (!d->x || !d->out || reinterpret_cast<uintptr_t>(d->out) % row_type_bytes(d->out_ty)) return false;
  if (d->x_ty == DARASK_E4M3)
    return d->x_scales && d->ld_xs >= kb && !d->swiglu && reinterpret_cast<uintptr_t>(d->x) % 16 == 0 && d->ldx % 16 == 0 && d->ldx >= d->k;
  const size_t eb = row_type_bytes(d->x_ty);
  if (!eb || d->x_scales || reinterpret_cast<uintptr_t>(d->x) % eb || d->ldx < (d->swiglu ? 2ll : 1ll) * d->k) return false;
  return d->workspace && reinterpret_cast<uintptr_t>(d->workspace) % 256 == 0 &&
         d->workspace_bytes >= darask_fp8_linear_workspace_bytes(d->m, d->n, d->k, d->x_ty);
}

extern "C" int darask_fp8_linear(const DaraskFp8Linear* d, cudaStream_t st) {
  if (!linear_ok(d)) return cudaErrorInvalidValue;
  if (d->m == 0) return cudaSuccess;
  const int kb = (d->k + 127) / 128;
  Fp8LinearArgs a = {};
  a.m = d->m; a.n = d->n; a.k = d->k;
  a.w = static_cast<const uint8_t*>(d->w); a.ldw = d->ldw; a.ws = d->w_scales; a.ld_ws = d->ld_ws;
  a.out = d->out; a.out_ty = d->out_ty; a.ldo = d->ldo;
  if (d->x_ty == DARASK_E4M3) {
    a.codes = static_cast<const uint8_t*>(d->x); a.ldx = d->ldx; a.xs = d->x_scales; a.ld_xs = d->ld_xs;
  } else {
    uint8_t* codes = static_cast<uint8_t*>(d->workspace);
    float* scales = reinterpret_cast<float*>(codes + round_up(size_t(d->m) * kb * 128, 256));
    const RowSource src{d->x, d->ldx, d->x_ty, d->k, d->swiglu, row_source_vec(d->x, d->x_ty, d->ldx, d->k, d->swiglu)};
    const long long groups = (long long)d->m * kb;
    const cudaError_t e = launch_pdl(fp8_linear_quant_kernel, dim3(unsigned((groups + 7) / 8)), dim3(256), 0, st, src, groups, kb, codes, scales);
    if (e) return e;
    a.codes = codes; a.ldx = (long long)kb * 128; a.xs = scales; a.ld_xs = kb;
  }
  return launch_pdl(fp8_linear_kernel, dim3((d->n + 31) / 32, unsigned((d->m + 31) / 32 < 65535 ? (d->m + 31) / 32 : 65535)), dim3(256), 0, st, a);
}

extern "C" int darask_fp8_linear_status(unsigned* host_status, cudaStream_t st) {
  if (!host_status) return cudaErrorInvalidValue;
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_fp8_linear_status);
  if (!e) e = cudaMemcpyAsync(host_status, p, 4, cudaMemcpyDeviceToHost, st);
  if (!e) e = cudaMemsetAsync(p, 0, 4, st);
  return e ? e : cudaStreamSynchronize(st);
}
