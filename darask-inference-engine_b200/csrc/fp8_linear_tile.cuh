// Many rows of x: the dense block-scaled FP8 product as 256 x 256 output tiles of pairs of blocks (tcgen05 cta_group::2).
// A block of a pair holds 128 rows of x and 128 rows of w of the tile in shared memory and the float32 partial products of its
// 128 rows of x and all 256 rows of w in TMEM: per 128-column block of k each SM fetches and reads 32 KB for 512 cycles of the
// tensor pipe, where a tile of its own (128 x 256) would take 48 KB; shared memory, not the pipe, bounds that one.
// The block scales are arbitrary float32 numbers, so a block of k is promoted outside the tensor core: partial * (sx * sw)
// is added to float32 registers while the next block multiplies into the other TMEM buffer.
//   warp 0     TMA loads of this block's halves into a ring; the copies of both blocks count on the first block's barrier
//   warp 1     (first block) tcgen05.mma M256 N256 K32, four per block of k; commits arrive in both blocks
//   warps 2-3  scales of the rows and of the two 128-row groups of w, eight blocks of k at a time
//   warps 4-11 promotion (thread = one row of x, 128 of the 256 columns) and, per tile, the store: rounded once, staged per
//              warp as 32 rows of 128 bytes and written by TMA (unaligned outputs: element by element)
// Bound: the tensor pipe with the promotion beside it (8192 x 8192 x 4096: 291 us, 1.89 PFLOP/s, the pipe active 56 % of the
// cycles, half of all issue slots taken).
// Persistent: one pair per two SMs takes tiles in steps of the number of pairs, rows of x fastest.
#pragma once
#include "row_source.cuh"
#include "tcgen05.cuh"

namespace dmoe {

constexpr int kFtThreads = 384;
constexpr int kFtStages = 5;
constexpr int kFtStageBytes = 2 * 128 * 128;
constexpr int kFtGroup = 8;                                      // blocks of k whose scales travel together
constexpr int kFtStoreBytes = 8 * 32 * 128;                      // 8 warps x 32 rows x 128 bytes
constexpr int kFtFactorFloats = 2 * kFtGroup * (128 + 2);
constexpr int kFtSmem = 1024 + kFtStages * kFtStageBytes + kFtStoreBytes + kFtFactorFloats * 4;

struct FtArgs {
  int m, n, kb;
  const float* xs;
  long long ld_xs;
  const float* ws;
  long long ld_ws;
  void* out;
  int out_ty;
  long long ldo;
  int add;                    // on top of what out holds (not with tma_store)
  int tma_store;              // the output's rows can be written by TMA
  int tiles_m, tiles_n;       // of 256
  unsigned* status;
};

DEVI void tma_load_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {      // barrier of either block of the pair
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
DEVI void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
DEVI void umma_commit_pair(uint64_t* bar, uint32_t go) {          // arrives on the barrier at this offset in both blocks
  asm volatile(
      "{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %2, 0;\n\t"
      "@g tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
      ::"r"(smem_u32(bar)), "h"(uint16_t(3)), "r"(go) : "memory");
}
DEVI void umma_f8_pair(uint32_t d, uint64_t da, uint64_t db, uint32_t accumulate, uint32_t go) {      // M256 N256 K32
  constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(256 >> 3) << 17) | (uint32_t(256 >> 4) << 24);
  asm volatile(
      "{\n\t.reg .pred p, g;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 g, %5, 0;\n\t"
      "@g tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(kIdesc), "r"(accumulate), "r"(go) : "memory");
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFtThreads, 1)
fp8_linear_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_out, const FtArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* store_stage = ring + kFtStages * kFtStageBytes;
  float* fx = reinterpret_cast<float*>(store_stage + kFtStoreBytes);      // [2][kFtGroup][128] scales of this block's rows
  float* fw = fx + 2 * kFtGroup * 128;                                    // [2][kFtGroup][2] scales of the two halves of the columns
  __shared__ uint64_t full[kFtStages], empty[kFtStages], tfull[2], tempty[2], ffull[2], fempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kFtStages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(tfull + b, 1); mbar_init(tempty + b, 16); mbar_init(ffull + b, 2); mbar_init(fempty + b, 8); }
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch();
  tmem_fence_before();
  __syncthreads();
  cluster_sync();                        // the peer's barriers are initialised
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;
  const int total = a.tiles_m * a.tiles_n, step = int(gridDim.x >> 1), first = int(blockIdx.x >> 1);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // (the lanes of warps 0 and 1 stay together: operands of the copies and of tcgen05.mma live in uniform registers)
    if (warp == 0) {
      const uint32_t go = elect_lane();
      const uint32_t full0 = cluster_map(smem_u32(full), 0), ring0 = smem_u32(ring);
      int s = 0, used = 0;               // stage; stages filled so far (up to the first round)
      uint32_t ph = 1;                   // parity of the "empty" phase
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += step) {
        const int r0 = (tile % a.tiles_m) * 256 + int(rank) * 128, w0 = (tile / a.tiles_m) * 256 + int(rank) * 128;
#pragma unroll 1
        for (int kb = 0; kb < a.kb; ++kb) {
          if (used == kFtStages) ok = warp_wait(empty + s, ph, a.status);
          else ++used;
          if (!ok) break;
          if (go) {
            const uint32_t dst = ring0 + s * kFtStageBytes, bar = full0 + s * 8;
            if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * kFtStageBytes);
            tma_load_pair(dst, &map_x, kb * 128, r0, bar);
            tma_load_pair(dst + 128 * 128, &map_w, kb * 128, w0, bar);
          }
          if (++s == kFtStages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok) {                         // after a timeout the copies in flight land before the pair ends
        abort_flag = 1;
        if (rank == 0)
          for (int i = 0; i < used; ++i) pipe_wait(full + i, i < s ? ph ^ 1 : ph, a.status);
      }
    } else if (warp == 1) {
      if (rank == 0) {
        const uint32_t go = elect_lane();
        const uint64_t d0 = umma_desc_k128(smem_u32(ring));
        int s = 0;
        uint32_t ph = 0, it = 0;
        bool ok = true;
        for (int tile = first; tile < total && ok; tile += step) {
#pragma unroll 1
          for (int kb = 0; kb < a.kb; ++kb, ++it) {
            const uint32_t buf = it & 1;
            if (it >= 2) ok = warp_wait(tempty + buf, ((it >> 1) & 1) ^ 1, a.status);
            ok = warp_wait(full + s, ph, a.status) && ok;
            if (!ok) break;
            tmem_fence_after();
            const uint64_t dx = d0 + uint32_t(s * (kFtStageBytes >> 4)), dw = dx + (128 * 128 >> 4);
#pragma unroll
            for (int q = 0; q < 4; ++q) umma_f8_pair(tmem + buf * 256, dx + 2 * q, dw + 2 * q, q ? 1u : 0u, go);
            umma_commit_pair(empty + s, go);
            umma_commit_pair(tfull + buf, go);
            if (++s == kFtStages) { s = 0; ph ^= 1; }
          }
        }
        if (!ok) abort_flag = 1;
      }
    } else if (warp >= 2) {
      const int ft = threadIdx.x - 64;
      int fg = 0;
      for (int tile = first; tile < total && !abort_flag; tile += step) {
        const int r0 = (tile % a.tiles_m) * 256 + int(rank) * 128, nb = (tile / a.tiles_m) * 2;
        for (int b0 = 0; b0 < a.kb; b0 += kFtGroup, ++fg) {
          const int slot = fg & 1;
          float v[128 * kFtGroup / 64];
#pragma unroll
          for (int j = 0; j < 128 * kFtGroup / 64; ++j) {          // eight neighbouring threads share a row
            const int row = r0 + j * 8 + ft / 8, b = b0 + ft % 8;
            v[j] = row < a.m && b < a.kb ? __ldcg(a.xs + size_t(row) * size_t(a.ld_xs) + b) : 0.f;
          }
          float w = 0.f;
          if (ft < 2 * kFtGroup && (nb + (ft & 1)) * 128 < a.n && b0 + ft / 2 < a.kb)
            w = __ldcg(a.ws + size_t(nb + (ft & 1)) * size_t(a.ld_ws) + b0 + ft / 2);
          int ok = 1;
          if (fg >= 2 && lane == 0) ok = pipe_wait(fempty + slot, ((fg >> 1) & 1) ^ 1, a.status) ? 1 : 0;
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) abort_flag = 1;
          if (abort_flag) break;
#pragma unroll
          for (int j = 0; j < 128 * kFtGroup / 64; ++j) fx[(slot * kFtGroup + ft % 8) * 128 + j * 8 + ft / 8] = v[j];
          if (ft < 2 * kFtGroup) fw[slot * 2 * kFtGroup + ft] = w;
          __syncwarp();
          if (lane == 0) mbar_arrive(ffull + slot);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
    const uint32_t tl = tmem + (uint32_t(quarter * 32) << 16) + 128 * half;
    const uint32_t tempty_addr = cluster_map(smem_u32(tempty), 0);
    uint8_t* mine = store_stage + (warp - 4) * 32 * 128;
    int it = 0, fg = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += step) {
      float acc[128];
#pragma unroll
      for (int c = 0; c < 128; ++c) acc[c] = 0.f;
      for (int kb = 0; kb < a.kb; ++kb, ++it) {
        const int buf = it & 1, slot = fg & 1;
        if (kb % kFtGroup == 0) ok = warp_wait(ffull + slot, (fg >> 1) & 1, a.status);
        ok = warp_wait(tfull + buf, (it >> 1) & 1, a.status) && ok;
        if (!ok) { abort_flag = 1; break; }
        tmem_fence_after();
        const float f = fx[(slot * kFtGroup + kb % kFtGroup) * 128 + row] * fw[(slot * kFtGroup + kb % kFtGroup) * 2 + half];
        uint32_t v[64];
        tmem_ld64(tl + buf * 256, v);
#pragma unroll
        for (int c = 0; c < 64; ++c) acc[c] = fmaf(__uint_as_float(v[c]), f, acc[c]);
        tmem_ld64(tl + buf * 256 + 64, v);
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_addr + buf * 8);
#pragma unroll
        for (int c = 0; c < 64; ++c) acc[64 + c] = fmaf(__uint_as_float(v[c]), f, acc[64 + c]);
        if (kb % kFtGroup == kFtGroup - 1 || kb == a.kb - 1) {
          if (lane == 0) mbar_arrive(fempty + slot);
          ++fg;
        }
      }
      if (!ok) break;
      // ---- store: pieces of 128 bytes per row -----------------------------------------------------------------------
      const int r0 = (tile % a.tiles_m) * 256 + int(rank) * 128 + quarter * 32, c0 = (tile / a.tiles_m) * 256 + 128 * half;
      auto put = [&](const uint4 (&piece)[8], int col, int per) {         // `per` columns from col of this warp's rows
        if (lane == 0 && a.tma_store) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(mine + lane * 128 + ((j ^ (lane & 7)) << 4)) = piece[j];
        if (a.tma_store) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && r0 < a.m && col < a.n) {
            tma_store_2d(&map_out, smem_u32(mine), col, r0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          __syncwarp();
          const int es = 128 / per;
          for (int r = 0; r < 32 && r0 + r < a.m; ++r)
            for (int c = lane; c < per && col + c < a.n; c += 32) {
              const uint8_t* src = mine + r * 128 + (((c * es >> 4) ^ (r & 7)) << 4) + ((c * es) & 15);
              const size_t at = size_t(r0 + r) * size_t(a.ldo) + size_t(col + c);
              if (es == 4) store_elem(a.out, a.out_ty, at, *reinterpret_cast<const float*>(src), a.add);
              else static_cast<unsigned short*>(a.out)[at] = *reinterpret_cast<const unsigned short*>(src);
            }
          __syncwarp();
        }
      };
      uint4 piece[8];
      if (a.out_ty == DARASK_GGML_F32) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            piece[j] = make_uint4(__float_as_uint(acc[p * 32 + 4 * j]), __float_as_uint(acc[p * 32 + 4 * j + 1]),
                                  __float_as_uint(acc[p * 32 + 4 * j + 2]), __float_as_uint(acc[p * 32 + 4 * j + 3]));
          put(piece, c0 + p * 32, 32);
        }
      } else {
        const bool f16 = a.out_ty == DARASK_GGML_F16;
        auto pack = [&](float lo, float hi) {
          if (f16) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&h); }
          const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
          return *reinterpret_cast<const uint32_t*>(&b);
        };
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int c = p * 64 + 8 * j;
            piece[j] = make_uint4(pack(acc[c], acc[c + 1]), pack(acc[c + 2], acc[c + 3]), pack(acc[c + 4], acc[c + 5]), pack(acc[c + 6], acc[c + 7]));
          }
          put(piece, c0 + p * 64, 64);
        }
      }
    }
    if (lane == 0 && a.tma_store) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  cluster_sync();                        // neither block leaves while the other's operands or barriers are in use
  tmem_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace dmoe
