// Dense product in block-scaled FP8:
//   out[i][j] = sum over 128-column blocks b of (code(x)[i][b] . W[j][b]) * sx[i][b] * sw[j / 128][b]
// W: e4m3, one float32 scale per 128 x 128 block (hayate `Fp8Block`, cpu/glm53.rs:23-24). x: float rows, quantized here to
// e4m3 with one float32 scale per row and 128 columns (as darask_quantize_fp8_act), or codes and scales as they are.
#include "../../include/darask_moe_b200.h"
#include <cuda_fp8.h>
#include "fp8_linear_stream.cuh"
#include "fp8_linear_tile.cuh"
#include "status.cuh"

namespace dmoe {

static __device__ unsigned g_fp8_linear_status;
static cudaError_t status_word(unsigned** p) {
  static unsigned* known[64] = {};
  return device_word(g_fp8_linear_status, known, p);
}

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
  uint32_t out;
  const float scale = fp8_group(v, &out);
  if (lane == 0) scales[w] = scale;
  reinterpret_cast<uint32_t*>(codes)[w * 32 + lane] = out;
}

// What a call runs. `fused` (rows quantized in the product's launch) depends on m and k alone, as the workspace does. It saves a launch, 4 us
// on the host, which is what bounds such calls when they are made one by one (9.8 us a call for 8 rows of 4096 x 4096 bf16); in a
// captured graph it gains nothing for small matrices (4.9 against 5.0 us for 6 rows of 2048 x 2048) and loses for large ones, where
// every block quantizes its part of k again (9.2 against 7.8 us for 8 rows of 4096 x 4096).
struct LinearPlan { int nt, splits; bool fused, tile; };
static bool linear_small(int m, int kb) { return m <= 8 && kb <= 8 * kFsResident; }
// Rows of x per tile, blocks per cluster and kind of kernel by the time they are expected to take, in ns. The weights are fitted to a
// sweep over 17 to 1024 rows of matrices from 1024 x 1536 to 8192 x 4096: a 128-column block of k takes 310, 390 or 780 ns with
// 16, 32 or 128 rows (64 rows took 510, which 32 or 128 always beat, so there are no such tiles; 1.3 times as long where two blocks share an SM), joining S parts 450 S (1 + NT / 64), a 256 x 256 tile of the
// pair kernel 550 ns per block of k and 900 more to start. (4096 x 4096, 256 rows: 128 rows in two parts 18.7 us, 32 rows undivided
// 19.6, pairs 22.0; 512 rows: pairs 23.2, 128 rows 30.5.)
static LinearPlan linear_plan(int m, int n, int kb, bool codes) {
  LinearPlan p = {};
  const long long sms = sm_count() > 1 ? sm_count() : 148;
  const long long tiles_n = (n + 127) / 128;
  if (linear_small(m, kb)) {             // codes are divided the same way: they give the same bits as the rows they came from
    p.fused = !codes;
    p.nt = 16;
    p.splits = 1;
    while (p.splits < 8 && p.splits * 2 <= kb && (tiles_n * p.splits * 2 <= 2 * sms || (kb + p.splits - 1) / p.splits > kFsResident)) p.splits *= 2;
    return p;
  }
  long long best = -1;
  for (int unit = 0; unit < 3; ++unit) {
    static const int kRows[3] = {16, 32, 128}, kUnit[3] = {310, 390, 780};
    const int nt = kRows[unit];
    if (nt > 16 && nt / 2 >= m) break;                 // no wider than the rows need
    const long long tiles = tiles_n * ((m + nt - 1) / nt);
    for (int splits = 1; splits <= 8 && splits <= kb; splits *= 2) {
      const long long blocks = tiles * splits, slots = nt <= 32 ? 2 * sms : sms, kbs = (kb + splits - 1) / splits;
      long long cost = (blocks + slots - 1) / slots * kbs * kUnit[unit];
      if (blocks > sms && nt <= 32) cost = cost * 13 / 10;
      if (splits > 1) cost += 450ll * splits * (64 + nt) / 64;
      if (best < 0 || cost < best) { best = cost; p.nt = nt; p.splits = splits; }
    }
  }
  if (m > 128) {
    const long long tiles = (long long)((n + 255) / 256) * ((m + 255) / 256), pairs = sms / 2;
    p.tile = 900 + (tiles + pairs - 1) / pairs * kb * 550 < best;
  }
  return p;
}

template <int NT, bool FUSED>
static cudaError_t launch_stream(const CUtensorMap& mw, const CUtensorMap& mx, const FsArgs& a, int tiles, int splits, cudaStream_t st) {
  static bool configured[64] = {};      // the opt-in is per device and per kernel
  const int dev = current_device_slot();
  if (dev < 0) return cudaErrorInvalidDevice;
  auto kernel = fp8_linear_stream_kernel<NT, FUSED>;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               FUSED ? kFsFusedSmem + kFsResident * (2048 + 64) : FsShape<NT>::kSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const size_t smem = FUSED ? size_t(kFsFusedSmem) + size_t((a.kb + splits - 1) / splits) * (2048 + 64) : size_t(FsShape<NT>::kSmem);
  return launch_cluster(kernel, dim3(unsigned(tiles) * unsigned(splits)), dim3(kFsThreads), smem, unsigned(splits), st, mw, mx, a);
}

static cudaError_t launch_tile(const DaraskFp8Linear* d, const FsArgs& s, const uint8_t* xc, unsigned long long cols, unsigned long long pitch,
                               cudaStream_t st) {
  CUtensorMap mx, mw, mo;
  if (!byte_map(&mx, xc, d->m, cols, pitch, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
  if (!byte_map(&mw, d->w, d->n, d->k, d->ldw, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
  const unsigned long long es = row_type_bytes(d->out_ty);
  // a TMA store writes whole 16-byte pieces: rows that end inside one would lose what lies behind them
  const bool aligned = reinterpret_cast<uintptr_t>(d->out) % 16 == 0 && d->ldo * es % 16 == 0 && d->n * es % 16 == 0;
  FtArgs a = {};
  a.m = d->m; a.n = d->n; a.kb = s.kb; a.xs = s.xs; a.ld_xs = s.ld_xs; a.ws = s.ws; a.ld_ws = s.ld_ws;
  a.out = d->out; a.out_ty = d->out_ty; a.ldo = d->ldo; a.add = d->add; a.status = s.status;
  a.tma_store = aligned && !d->add && byte_map(&mo, d->out, d->m, d->n * es, d->ldo * es, 32, 128, CU_TENSOR_MAP_SWIZZLE_128B, unsigned(es));
  if (!a.tma_store) mo = mx;            // not used
  a.tiles_m = (d->m + 255) / 256; a.tiles_n = (d->n + 255) / 256;
  if ((long long)a.tiles_m * a.tiles_n > 0x3fffffffll) return cudaErrorInvalidValue;
  static bool configured[64] = {};      // the opt-in is per device
  const int dev = current_device_slot();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fp8_linear_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFtSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_pdl(fp8_linear_tile_kernel, dim3(unsigned(sm_count() / 2 * 2)), dim3(kFtThreads), size_t(kFtSmem), st, mx, mw, mo, a);
}

static size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace dmoe

using namespace dmoe;

extern "C" size_t darask_fp8_linear_workspace_bytes(int m, int n, int k, int x_ty) {
  if (m < 1 || n < 1 || k < 1 || x_ty == DARASK_E4M3) return 0;
  const size_t kb = (size_t(k) + 127) / 128;
  if (linear_small(m, int(kb))) return 0;
  return round_up(size_t(m) * kb * 128, 256) + round_up(size_t(m) * kb * 4, 256);
}

static bool linear_ok(const DaraskFp8Linear* d) {
  if (!d || d->m < 0 || d->n < 1 || d->k < 1 || d->m > (1 << 24) || d->n > (1 << 24) || d->k > (1 << 20)) return false;
  if (!d->w || !d->w_scales || reinterpret_cast<uintptr_t>(d->w_scales) % 4 || reinterpret_cast<uintptr_t>(d->w) % 16 || d->ldw % 16 || d->ldw < d->k) return false;
  const long long kb = (d->k + 127) / 128;
  if (reinterpret_cast<uintptr_t>(d->status) % 4) return false;
  if (d->ld_ws < kb || !row_type_bytes(d->out_ty) || d->ldo < d->n || (d->add && d->out_ty != DARASK_GGML_F32)) return false;
  if (d->m == 0) return true;
  if (!d->x || !d->out || reinterpret_cast<uintptr_t>(d->out) % row_type_bytes(d->out_ty)) return false;
  if (d->x_ty == DARASK_E4M3)
    return d->x_scales && reinterpret_cast<uintptr_t>(d->x_scales) % 4 == 0 && d->ld_xs >= kb && !d->swiglu && reinterpret_cast<uintptr_t>(d->x) % 16 == 0 && d->ldx % 16 == 0 && d->ldx >= d->k;
  const size_t eb = row_type_bytes(d->x_ty);
  if (!eb || d->x_scales || reinterpret_cast<uintptr_t>(d->x) % eb || d->ldx < (d->swiglu ? 2ll : 1ll) * d->k) return false;
  const size_t need = darask_fp8_linear_workspace_bytes(d->m, d->n, d->k, d->x_ty);
  return need == 0 || (d->workspace && reinterpret_cast<uintptr_t>(d->workspace) % 256 == 0 &&
         d->workspace_bytes >= need);
}

extern "C" int darask_fp8_linear(const DaraskFp8Linear* d, cudaStream_t st) {
  if (!linear_ok(d)) return cudaErrorInvalidValue;
  if (d->m == 0) return cudaSuccess;
  const int kb = (d->k + 127) / 128;
  unsigned* status = d->status;
  cudaError_t e = cudaSuccess;
  if (!status && (e = status_word(&status))) return e;
  const bool codes = d->x_ty == DARASK_E4M3;
  const LinearPlan p = linear_plan(d->m, d->n, kb, codes);
  FsArgs a = {};
  a.m = d->m; a.n = d->n; a.kb = kb;
  a.ws = d->w_scales; a.ld_ws = d->ld_ws;
  a.out = d->out; a.out_ty = d->out_ty; a.ldo = d->ldo;
  a.add = d->add;
  a.tiles_n = (d->n + 127) / 128;
  a.status = status;
  a.src = RowSource{d->x, d->ldx, d->x_ty, d->k, d->swiglu, codes ? 0 : row_source_vec(d->x, d->x_ty, d->ldx, d->k, d->swiglu)};
  const uint8_t* xc = static_cast<const uint8_t*>(d->x);
  unsigned long long pitch = d->ldx, cols = d->k;
  a.xs = d->x_scales; a.ld_xs = d->ld_xs;
  if (!codes && !p.fused) {
    uint8_t* q = static_cast<uint8_t*>(d->workspace);
    float* scales = reinterpret_cast<float*>(q + round_up(size_t(d->m) * kb * 128, 256));
    const long long groups = (long long)d->m * kb;
    if ((e = launch_pdl(fp8_linear_quant_kernel, dim3(unsigned((groups + 7) / 8)), dim3(256), 0, st, a.src, groups, kb, q, scales))) return e;
    xc = q; pitch = cols = (unsigned long long)kb * 128; a.xs = scales; a.ld_xs = kb;
  }
  CUtensorMap mw, mx;
  if (p.tile) return launch_tile(d, a, xc, cols, pitch, st);
  if (!byte_map(&mw, d->w, d->n, d->k, d->ldw, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
  if (p.fused) mx = mw;                 // not read
  else if (!byte_map(&mx, xc, d->m, cols, pitch, p.nt, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
  const long long tiles = (long long)a.tiles_n * ((d->m + p.nt - 1) / p.nt);
  if (tiles * p.splits > 0x7fffffffll) return cudaErrorInvalidValue;
  if (p.fused) return launch_stream<16, true>(mw, mx, a, int(tiles), p.splits, st);
  switch (p.nt) {
    case 16: return launch_stream<16, false>(mw, mx, a, int(tiles), p.splits, st);
    case 32: return launch_stream<32, false>(mw, mx, a, int(tiles), p.splits, st);
    default: return launch_stream<128, false>(mw, mx, a, int(tiles), p.splits, st);
  }
}

extern "C" int darask_fp8_linear_plan(int m, int n, int k, int x_ty, int* plan) {
  if (!plan || m < 1 || n < 1 || k < 1 || m > (1 << 24) || n > (1 << 24) || k > (1 << 20) || (x_ty != DARASK_E4M3 && !row_type_bytes(x_ty))) return cudaErrorInvalidValue;
  const LinearPlan p = linear_plan(m, n, (k + 127) / 128, x_ty == DARASK_E4M3);
  plan[0] = p.tile ? 256 : p.nt;
  plan[1] = p.tile ? 1 : p.splits;
  plan[2] = p.fused;
  return cudaSuccess;
}

extern "C" int darask_fp8_linear_status(unsigned* host_status, cudaStream_t st) {
  if (!host_status) return cudaErrorInvalidValue;
  unsigned* p = nullptr;
  const cudaError_t e = status_word(&p);
  return e ? e : darask_status_take(p, host_status, st);
}
