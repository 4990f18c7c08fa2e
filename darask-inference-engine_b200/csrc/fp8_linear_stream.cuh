// Few rows of x: the dense block-scaled FP8 product as a stream of the weights.
// A block computes 128 weight rows x NT rows of x over its part of k: the weight tile is the M = 128 operand and the rows of x
// are the N operand of tcgen05.mma kind::f8f6f4, so a single token costs a 16-wide tile and not a 128-wide one. The `cluster`
// blocks of a cluster split k (128-column blocks) among them and add their float32 tiles through distributed shared memory in
// rank order: no scratch in HBM, no atomics, the same bits in every call.
//   warp 0      TMA: weight tile (and the tile of x unless it is quantized here) of one 128-column block per ring stage
//   warp 1      tcgen05.mma, four per block of k, into one of four TMEM buffers of NT columns
//   warps 2-3   the factors sx * sw of the blocks, eight blocks of k at a time, two groups ahead of their use
//   warps 4-7   tcgen05.ld of the block's partial tile (thread = one weight row), times the factors, added in registers
// FUSED: x comes as float rows; before the loop all warps but 0 quantize this block's part of x straight into the
// swizzled operand tiles, which stay in shared memory (one tile of 16 for up to 8 rows, at most kFsResident blocks of k): one launch.
// Bound: a single row by the latency of one pass (4096 x 4096 in a graph of calls: 6.3 us with other weights in every call, 2.65 TB/s, 5.9 with
// the same ones, which L2 holds; 2.6 us at the rate of a copy; start, quantizer, four dependent ring rounds and the join are the rest),
// more rows by the promotion, which costs a block of k 310 ns with 16 rows and 780 with 128 (256 rows of 4096 x 2048: 14.6 us with the
// quantizer in front, in tiles of 32 rows). Rows as the N operand: as M they would cost a 128-row tile for one token.
#pragma once
#include <cuda_fp8.h>
#include "row_source.cuh"
#include "tcgen05.cuh"

namespace dmoe {

constexpr int kFsThreads = 256;
constexpr int kFsResident = 32;              // blocks of k a FUSED block holds of x
constexpr int kFsGroup = 8;                  // blocks of k whose factors travel together
constexpr int kFsFlight = 6;                 // groups of x a warp has in flight while it quantizes
constexpr int kFsBufs = 4;                   // TMEM buffers

struct FsArgs {
  int m, n, kb;                              // kb: blocks of k in all
  RowSource src;                             // FUSED
  const float* xs;                           // otherwise [m][ld_xs]
  long long ld_xs;
  const float* ws;                           // [ceil(n/128)][ld_ws]
  long long ld_ws;
  void* out;
  int out_ty;
  long long ldo;
  int add;                                   // on top of what out holds
  int tiles_n;                               // ceil(n/128)
  unsigned* status;
};

template <int NT>
struct FsShape {
  static constexpr int kStages = NT <= 32 ? 5 : 6;
  static constexpr int kStageBytes = 128 * 128 + NT * 128;
  static constexpr int kFactorFloats = 2 * kFsGroup * NT;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kTmemCols = kFsBufs * NT < 32 ? 32 : kFsBufs * NT;
  static constexpr int kSmem = 1024 + kRingBytes + kFactorFloats * 4;
  static_assert(kRingBytes >= NT * 128 * 4, "the joined tile reuses the ring");
};
// FUSED: ring of weight tiles only, resident x tiles and their factors
constexpr int kFsFusedStages = 5;
constexpr int kFsFusedSmem = 1024 + kFsFusedStages * 128 * 128;       // + blocks of k of this block * (16 * 128 + 16 * 4)

// scale and e4m3 codes of one 128-column group, four columns per lane (see fp8_linear_quant_kernel)
DEVI float fp8_group(const float (&v)[4], uint32_t* codes) {
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
  *codes = out;
  return scale;
}

// Block `rank` adds and stores every SPLITS-th row of x of the cluster's tile: a warp per row, four weight rows per lane, eight pieces
// from other blocks in flight; added in rank order.
template <int SPLITS, int NT>
DEVI void fs_join(const FsArgs& a, float* part, uint32_t rank, int n0, int t0) {
  constexpr int U = 8 / SPLITS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = n0 + lane * 4;
  uint32_t from[SPLITS];
#pragma unroll
  for (int s = 0; s < SPLITS; ++s) from[s] = cluster_map(smem_u32(part) + lane * 16, s);
  for (int c0 = int(rank) + warp * SPLITS; c0 < NT && t0 + c0 < a.m; c0 += 8 * SPLITS * U) {
    float4 v[U][SPLITS];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < SPLITS; ++s) {
        const int c = c0 + u * 8 * SPLITS;
        if (c < NT) v[u][s] = ld_cluster_f32x4(from[s] + c * 512);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 8 * SPLITS;
      if (c >= NT || t0 + c >= a.m) break;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < SPLITS; ++s) { y[0] += v[u][s].x; y[1] += v[u][s].y; y[2] += v[u][s].z; y[3] += v[u][s].w; }
      const size_t at = size_t(t0 + c) * size_t(a.ldo) + col;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (col + q < a.n) store_elem(a.out, a.out_ty, at + q, y[q], a.add);
    }
  }
}

template <int NT, bool FUSED>
__global__ void __launch_bounds__(kFsThreads, NT <= 32 ? 2 : 1) fp8_linear_stream_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                       const __grid_constant__ CUtensorMap map_x, const FsArgs a) {
  static_assert(!FUSED || NT == 16, "rows quantized in the kernel: one tile of 16");
  using S = FsShape<NT>;
  constexpr int kStages = FUSED ? kFsFusedStages : S::kStages;
  constexpr int kStageBytes = FUSED ? 128 * 128 : S::kStageBytes;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kStages], empty[kStages], tfull[kFsBufs], tempty[kFsBufs], ffull[2], fempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t rank = cluster_rank();
  const int tile = int(blockIdx.x / splits), n0 = (tile % a.tiles_n) * 128, t0 = (tile / a.tiles_n) * NT;
  const int kb0 = int((long long)a.kb * rank / splits), kbs = int((long long)a.kb * (rank + 1) / splits) - kb0;
  uint8_t* xres = ring + kFsFusedStages * 128 * 128;                               // FUSED: kbs tiles of 16 x 128 bytes
  float* factors = reinterpret_cast<float*>(FUSED ? xres + size_t(kbs) * 16 * 128 : ring + S::kRingBytes);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int b = 0; b < kFsBufs; ++b) { mbar_init(tfull + b, 1); mbar_init(tempty + b, 4); }
    for (int b = 0; b < 2; ++b) { mbar_init(ffull + b, 2); mbar_init(fempty + b, 4); }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<S::kTmemCols>(&tmem_slot);
  pdl_wait();
  pdl_launch();
  auto load_stage = [&](int i) {
    const int s = i % kStages;
    const uint32_t dst = smem_u32(ring + s * kStageBytes);
    mbar_arrive_expect_tx(full + s, kStageBytes);
    tma_load_2d(dst, &map_w, (kb0 + i) * 128, n0, full + s);
    if (!FUSED) tma_load_2d(dst + 128 * 128, &map_x, (kb0 + i) * 128, t0, full + s);
  };
  if (FUSED) {
    // the first weight tiles travel while x is quantized (thread 0 has initialised the barriers that it uses here)
    if (threadIdx.x == 0)
      for (int i = 0; i < kStages && i < kbs; ++i) load_stage(i);
    if (warp >= 1) {
      // group = (block of k, row), a handful per warp in flight; rows past m stay as they are: what they give is never stored
      const int groups = kbs * a.m;
      const float* ws = a.ws + size_t(n0 / 128) * size_t(a.ld_ws) + kb0;
      for (int g0 = warp - 1; g0 < groups; g0 += 7 * kFsFlight) {
        float v[kFsFlight][4], w[kFsFlight];
#pragma unroll
        for (int u = 0; u < kFsFlight; ++u) {
          const int g = g0 + 7 * u, b = g / a.m;
          if (g < groups) {
            row_source_load4(a.src, g - b * a.m, (kb0 + b) * 128 + lane * 4, v[u]);
            w[u] = __ldcg(ws + b);
          }
        }
#pragma unroll
        for (int u = 0; u < kFsFlight; ++u) {
          const int g = g0 + 7 * u, b = g / a.m, row = g - b * a.m;
          if (g >= groups) break;
          uint32_t codes;
          const float scale = fp8_group(v[u], &codes);
          // 128-byte rows, 16-byte pieces swizzled by the row in its group of eight
          *reinterpret_cast<uint32_t*>(xres + size_t(b) * 2048 + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) = codes;
          if (lane == 0) factors[b * 16 + row] = scale * w[u];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;
  constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(NT >> 3) << 17) | (uint32_t(128 >> 4) << 24);
  float acc[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) acc[c] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      int issued = FUSED ? (kbs < kStages ? kbs : kStages) : 0;
      for (int i = issued; i < kbs && !abort_flag; ++i, ++issued) {
        if (i >= kStages && !pipe_wait(empty + i % kStages, ((i / kStages) & 1) ^ 1, a.status)) { abort_flag = 1; break; }
        load_stage(i);
      }
      // after a timeout the copies in flight land before the block ends
      if (abort_flag)
        for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i) pipe_wait(full + i % kStages, (i / kStages) & 1, a.status);
    }
  } else if (warp == 1) {
    // (the lanes stay together: operands of tcgen05.mma live in uniform registers)
    const uint32_t go = elect_lane();
    const uint64_t d0 = umma_desc_k128(smem_u32(ring)), dres = umma_desc_k128(smem_u32(xres));
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < kbs; ++i) {
      const int s = i % kStages, buf = i % kFsBufs;
      if (i >= kFsBufs) ok = warp_wait(tempty + buf, ((i / kFsBufs) & 1) ^ 1, a.status);
      ok = warp_wait(full + s, (i / kStages) & 1, a.status) && ok;
      if (!ok) { abort_flag = 1; break; }
      tmem_fence_after();
      const uint64_t dw = d0 + uint32_t(s * (kStageBytes >> 4)), dx = FUSED ? dres + uint32_t(i * (2048 >> 4)) : dw + (128 * 128 >> 4);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        asm volatile(
            "{\n\t.reg .pred p, g;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 g, %5, 0;\n\t"
            "@g tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(tmem + buf * NT), "l"(dw + 2 * q), "l"(dx + 2 * q), "r"(kIdesc), "r"(q ? 1u : 0u), "r"(go) : "memory");
      umma_commit_if(empty + s, go);
      umma_commit_if(tfull + buf, go);
    }
  } else if (warp < 4) {
    if (!FUSED) {
      const int ft = threadIdx.x - 64;                            // 0 .. 63
      const float* ws = a.ws + size_t(n0 / 128) * size_t(a.ld_ws) + kb0;
      for (int g = 0; g * kFsGroup < kbs; ++g) {
        const int slot = g & 1, b0 = g * kFsGroup;
        float v[NT * kFsGroup / 64];
#pragma unroll
        for (int j = 0; j < NT * kFsGroup / 64; ++j) {             // element = (row, block of k): eight neighbours share a row
          const int e = j * 64 + ft, row = e / kFsGroup, b = b0 + e % kFsGroup;
          v[j] = t0 + row < a.m && b < kbs ? __ldcg(a.xs + size_t(t0 + row) * size_t(a.ld_xs) + kb0 + b) * __ldcg(ws + b) : 0.f;
        }
        int ok = 1;
        if (g >= 2 && lane == 0) ok = pipe_wait(fempty + slot, ((g >> 1) & 1) ^ 1, a.status) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok || abort_flag) { abort_flag = 1; break; }
#pragma unroll
        for (int j = 0; j < NT * kFsGroup / 64; ++j) {
          const int e = j * 64 + ft;
          factors[slot * kFsGroup * NT + (e % kFsGroup) * NT + e / kFsGroup] = v[j];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(ffull + slot);
      }
    }
  } else {
    const uint32_t tl = tmem + (uint32_t((warp - 4) * 32) << 16);
    for (int i = 0; i < kbs; ++i) {
      const int buf = i % kFsBufs, g = i / kFsGroup;
      bool ok = warp_wait(tfull + buf, (i / kFsBufs) & 1, a.status);
      if (!FUSED && i % kFsGroup == 0) ok = warp_wait(ffull + (g & 1), (g >> 1) & 1, a.status) && ok;
      if (!ok) { abort_flag = 1; break; }
      tmem_fence_after();
      const float4* f = reinterpret_cast<const float4*>(factors + (FUSED ? i : (g & 1) * kFsGroup + i % kFsGroup) * NT);
      if (NT == 16) {
        uint32_t v[16];
        tmem_ld16(tl + buf * NT, v);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 fq = f[q];
          acc[4 * q] = fmaf(__uint_as_float(v[4 * q]), fq.x, acc[4 * q]);
          acc[4 * q + 1] = fmaf(__uint_as_float(v[4 * q + 1]), fq.y, acc[4 * q + 1]);
          acc[4 * q + 2] = fmaf(__uint_as_float(v[4 * q + 2]), fq.z, acc[4 * q + 2]);
          acc[4 * q + 3] = fmaf(__uint_as_float(v[4 * q + 3]), fq.w, acc[4 * q + 3]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < NT; c += 32) {
          uint32_t v[32];
          tmem_ld32(tl + buf * NT + c, v);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 fq = f[c / 4 + q];
            acc[(c + 4 * q) % NT] = fmaf(__uint_as_float(v[4 * q]), fq.x, acc[(c + 4 * q) % NT]);
            acc[(c + 4 * q + 1) % NT] = fmaf(__uint_as_float(v[4 * q + 1]), fq.y, acc[(c + 4 * q + 1) % NT]);
            acc[(c + 4 * q + 2) % NT] = fmaf(__uint_as_float(v[4 * q + 2]), fq.z, acc[(c + 4 * q + 2) % NT]);
            acc[(c + 4 * q + 3) % NT] = fmaf(__uint_as_float(v[4 * q + 3]), fq.w, acc[(c + 4 * q + 3) % NT]);
          }
        }
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(tempty + buf);
        if (!FUSED && (i % kFsGroup == kFsGroup - 1)) mbar_arrive(fempty + (g & 1));
      }
    }
  }
  __syncwarp();
  // ---- join and store: thread = one weight row, one element per row of x -----------------------------------------------
  const int row = threadIdx.x - 128, col = n0 + row;              // epilogue threads
  if (splits == 1) {
    if (warp >= 4 && col < a.n) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (t0 + c < a.m) store_elem(a.out, a.out_ty, size_t(t0 + c) * size_t(a.ldo) + col, acc[c], a.add);
    }
  } else {
    float* part = reinterpret_cast<float*>(ring);                  // [NT][128]: every copy into the ring has been read
    if (warp >= 4) {
#pragma unroll
      for (int c = 0; c < NT; ++c) part[c * 128 + row] = acc[c];
    }
    cluster_sync();
    if (splits == 2) fs_join<2, NT>(a, part, rank, n0, t0);
    else if (splits == 4) fs_join<4, NT>(a, part, rank, n0, t0);
    else fs_join<8, NT>(a, part, rank, n0, t0);
    cluster_sync();                                                // nobody leaves while its tile is being read
  }
  tmem_fence_before();
  __syncthreads();
  if (warp == 1) tmem_free<S::kTmemCols>(tmem);
}

}  // namespace dmoe
