// Product grouped by expert over GGUF Q4_K / Q6_K weights on the 5th-generation tensor cores:
//   out[i][j] = x[row(i)] . W_g[j]      for the dispatch rows i of every group g
// A block of 256 weights is d times integers, sc_b q (Q4_K, at most 945) or sc_b (q - 32) (Q6_K, at most 4096), less dmin
// times integers m_b that multiply the sums of x over 32 columns (Q4_K). The tensor cores multiply these integers: f16 holds
// Q4_K's exactly (11 significant bits) and Q6_K's to 2^-12 (a second f16 term holds the rest), so a weight is never rounded and
// has no range to lose, whatever the type of the output. d and dmin are applied in float32 once per 256 columns, when the partial
// product leaves TMEM. A row of x is divided by a power of two (largest value into [2^9, 2^10)) and split into one or two f16
// parts (float32: 22 bits); the power of two comes back in the store.
//
// One block computes 128 weight rows x up to 128 dispatch rows of one group; the weight rows are the M operand, so that few
// rows cost a narrow tile (N a multiple of 16). The weight operand is written straight into TMEM (tcgen05.st), where
// tcgen05.mma reads it: it costs shared memory neither space nor bandwidth.
//   warps 0, 2    TMA: rows of x and their sums per 128 columns; packed weight rows (128 x 144 or 208 bytes) per 256 columns
//   warp 1        tcgen05.mma kind::f16 into one of two accumulators
//   then          two to four sets of four expander warps: thread = one weight row; codes -> integers in f16 -> TMEM, a step of 128
//                 columns of k in the set's slot
//   the last 4-8  promotion (thread = one weight row): acc += d * main - dmin * min, and the store at the end of a tile
// TMEM: two accumulators of NT columns, Q4_K's min products, the slots, Q6_K's second terms.
// Persistent: tiles are dealt out in steps of the grid, the row tiles of a group's weight tile next to each other.
// Bound: instructions and their latencies. A tile's 256 columns cost about 5000 warp instructions (2.1 per cycle), most of them the
// expanders', whatever its rows: 32768 rows over 128 groups of 2 x 768 x 2048 Q4_K (bf16) take 430 us, 352 when the groups are even and
// fill their tiles (585 TFLOP/s), 2048 rows over 256 groups of 2 x 1024 x 2048 232 us (2.6 TB/s).
#pragma once
#include "row_source.cuh"
#include "tcgen05.cuh"

namespace dmoe {

constexpr int kGgMaxGroups = 1024;

struct GgArgs {
  const unsigned* ranges;                                // [groups][2]
  int groups, n, nblk, mats, row_bytes;
  long long rows;
  const uint8_t* w[2];                                   // Q6_K: the block scales d are read from here
  const float* xscale;                                   // [rows] powers of two; negative: row(i) does not exist
  void* out;
  long long ldo;
  int tile_cap;                                          // more tiles than ranges that do not overlap can have, below 2^30
  int aligned;                                           // 16-byte pieces of the output's rows start on 16-byte boundaries
  unsigned* status;
};

// NT: rows of x per tile, NX: f16 parts of a row of x. A step is 128 columns of k.
template <bool Q6, int NT, int NX>
struct GgShape {
  // TMEM holds the weights of kSets steps, and a set of four expander warps belongs to each slot. Few rows leave room for four slots,
  // whose sets hide their latencies from each other; 128 rows leave two (there, sets that fill each step together took 439 us where
  // these take 423, and four promotion warps instead of eight 466: 32768 rows, 128 groups of 2 x 768 x 2048).
  static constexpr bool kWide = NT > 32;
  static constexpr int kSets = kWide ? 2 : Q6 ? 3 : 4;
  static constexpr int kPromote = kWide ? 8 : 4;         // warps that promote and store: two per quarter of the weight rows, half of x each
  static constexpr int kThreads = 128 * (1 + kSets) + 32 * kPromote;
  // wide: registers of the roles, the expanders and the promotion; their sum is what the block is launched with (640 x 96)
  static constexpr int kRegRoles = 48, kRegExpand = 88, kRegPromote = 128;
  static_assert(kRegRoles + 2 * kRegExpand + 2 * kRegPromote <= 5 * 96, "setmaxnreg draws on the launch's registers");
  static constexpr int kRawBytes = Q6 ? 208 : 144;
  static constexpr int kRawStage = 128 * kRawBytes;
  static constexpr int kBox = NT * 128;                  // NT rows x 64 columns of f16
  static constexpr int kPart = 2 * kBox;                 // one part of a step
  static constexpr int kSums = Q6 ? 0 : NT * 32;         // NT rows x 16 f16: the sums of eight groups of 32 columns, high and low parts
  static constexpr int kXStage = NX * kPart + kSums;     // Q4_K: the sums travel with the second step of a block
  static constexpr int kXStages = kWide && NX == 2 ? 2 : 4;
  // Partial products per block of 256 columns. The tensor core cuts the sum of every 16 columns to the accumulator's 24 bits, toward
  // zero, so that the error grows with the number of sums and does not average out; products of two parts have bits to lose. In turn in
  // one accumulator they lost 1.5e-6 of the result (Q4_K, whose codes have no sign and largely cancel against the mins) and 8e-7 (Q6_K).
  // The small products go first (Q6_K: 6e-7; an accumulator per step would bring 2e-7, but took 513 us where this took 449: 32768 rows, 128
  // groups of 2048 x 768), and Q4_K has an accumulator of its own for every step as well (4e-7 for 4 % of the time).
  static constexpr int kSteps = Q6 ? 1 : NX;
  static_assert(kSteps == 2 || kXStages == 4 || Q6, "the promotion takes the stage of a block's second step from its buffer");
  static constexpr int kMins = Q6 ? 0 : kSets / 2;       // 128 rows x 32 bytes each
  static constexpr int kOffMin = kXStages * kXStage;
  static constexpr int kOffRaw = kOffMin + kMins * 4096;
  static constexpr int kStore = kPromote * 1024;         // per warp 16 output rows x 32 columns (8 rows of float32)
  static constexpr int kTail = kStore + 4 * 128 * 8 + (kGgMaxGroups + 4) * 4;
  static constexpr int kFit = (kSmemBudget - 4 * 1024 - kOffRaw - kTail) / kRawStage;
  static constexpr int kRawStages = kFit < 8 ? kFit : 8;
  static constexpr int kOffStore = kOffRaw + kRawStages * kRawStage;
  static constexpr int kOffD = kOffStore + kStore;
  static constexpr int kOffEnds = kOffD + 4 * 128 * 8;
  static constexpr int kSmem = 1024 + kOffStore + kTail;
  // TMEM columns: two main buffers, one or two of min products, the weights, their second terms
  static constexpr int kMinBufs = Q6 ? 0 : kWide ? 1 : 2;
  static constexpr uint32_t kColMin = 2 * NT, kColA = kColMin + kMinBufs * NT, kColA2 = kColA + 64 * kSets;
  static_assert(kRawStages >= 3 && kColA2 + (Q6 ? 64 * kSets : 0) <= 512, "rings must fit");
};

// ---- rows of x -> f16 parts --------------------------------------------------------------------------------------------
// One block per dispatch row: largest magnitude, then x * 2^-e as one or two f16 parts, four columns at a time in the order
// 0 2 1 3 in which the expanders leave the weights, and (Q4_K) the sums of 32 columns as f16 high and low parts.
struct GgRowsArgs {
  RowSource src;
  long long rows, x_rows;
  const unsigned* assignments;
  int topk;
  __half* planes;                                        // [parts][rows][k]
  __half* sum;                                           // [rows][k / 256][16]: 8 high, 8 low
  float* scale;                                          // [rows]
};
constexpr int kGgRowThreads = 128;
constexpr int kGgRowHeld = 4096;                         // columns that stay in shared memory between the passes; what is behind them is read twice
// KIND: 0 any rows (four elements at a time, strides and SwiGLU as they come); rows on 16-byte boundaries: 1 float32, 2 f16, 3 bf16;
// 4, 5, 6 the same three as gate | up halves. One loop of few registers for all: held in registers, rows of 2048 bf16 left room for
// eight blocks per SM, and the code of unrolled SwiGLU products came through the instruction cache anew for every block (32768 rows:
// 2048 bf16 53 us instead of 65, 2 x 768 float32 50 instead of 83).
template <int KIND>
DEVI void rows_load8(const RowSource& s, const void* at, long long row, int c, float (&v)[8]) {
  if constexpr (KIND == 0) {
    float a[4], b[4];
    row_source_load4(s, row, c, a);
    row_source_load4(s, row, c + 4, b);
#pragma unroll
    for (int q = 0; q < 4; ++q) { v[q] = a[q]; v[4 + q] = b[q]; }
  } else if constexpr (KIND >= 4) {
    float u[8];
    rows_load8<KIND - 3>(s, at, row, c, v);
    rows_load8<KIND - 3>(s, at, row, c + s.k, u);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = silu_mul(v[q], u[q]);
  } else if constexpr (KIND == 1) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(at) + c);
    const float4 a = __ldcg(p), b = __ldcg(p + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = __ldcg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(at) + c));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[2 * q] = KIND == 2 ? half_lo(w[q]) : __uint_as_float(w[q] << 16);
      v[2 * q + 1] = KIND == 2 ? half_hi(w[q]) : __uint_as_float(w[q] & 0xffff0000u);
    }
  }
}
template <int KIND, bool PARTS, bool SUMS>
__global__ void __launch_bounds__(kGgRowThreads) ggml_rows_kernel(const GgRowsArgs a) {
  constexpr int kUnroll = KIND == 0 || KIND >= 4 ? 1 : 2;
  extern __shared__ __align__(16) float row_smem[];      // [min(k, kGgRowHeld)]
  __shared__ uint32_t red[kGgRowThreads / 32];
  pdl_wait();
  pdl_launch();
  const long long i = blockIdx.x;
  const int k = a.src.k;
  long long row = i;
  if (a.assignments) row = __ldcg(a.assignments + i) / unsigned(a.topk);
  const bool exists = row < a.x_rows;
  const void* at = static_cast<const uint8_t*>(a.src.x) + row * a.src.ld * (KIND == 1 || KIND == 4 ? 4 : 2);       // KIND 0: unused
  uint32_t top = 0;
  auto scan = [&](const float (&v)[8]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) top = max(top, __float_as_uint(v[q]) & 0x7fffffffu);
  };
  if (exists) {
#pragma unroll kUnroll
    for (int c = threadIdx.x * 8; c < k; c += kGgRowThreads * 8) {
      float v[8];
      rows_load8<KIND>(a.src, at, row, c, v);
      scan(v);
      if (c < kGgRowHeld) {
        *reinterpret_cast<float4*>(row_smem + c) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row_smem + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kGgRowThreads / 32; ++q) top = max(top, red[q]);
  // exponent of the largest magnitude (not below 2^-117: the factor stays finite), moved to 2^9
  const bool finite = top < 0x7f800000u;
  const int e = max(int(top >> 23) - 127, -117) - 9;
  const bool live = exists && finite;
  const float down = live ? __uint_as_float(uint32_t(127 - e) << 23) : 0.f;
  if (threadIdx.x == 0)
    a.scale[i] = !exists ? -1.f : top == 0u ? 1.f : finite ? __uint_as_float(uint32_t(127 + e) << 23) : __uint_as_float(0x7fffffffu);
  auto put = [&](int c, float (&v)[8]) {
    uint32_t hi[4], lo[4];
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      v[q] = live ? v[q] * down : 0.f;         // (a row that does not exist was never loaded)
      s += v[q];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {                        // columns 0 2 | 1 3 of each four
      const float p0 = v[(q >> 1) * 4 + (q & 1)], p1 = v[(q >> 1) * 4 + (q & 1) + 2];
      const __half2 h = __floats2half2_rn(p0, p1);
      hi[q] = *reinterpret_cast<const uint32_t*>(&h);
      if (PARTS) {
        const float2 back = __half22float2(h);
        const __half2 l = __floats2half2_rn(p0 - back.x, p1 - back.y);
        lo[q] = *reinterpret_cast<const uint32_t*>(&l);
      }
    }
    *reinterpret_cast<uint4*>(a.planes + size_t(i) * k + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (PARTS) *reinterpret_cast<uint4*>(a.planes + (size_t(a.rows) + size_t(i)) * k + c) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    if (SUMS) {                                          // k is a multiple of 256: groups of four lanes are here or not as one
      const unsigned mask = 0xfu << (threadIdx.x & 28);
      s += __shfl_xor_sync(mask, s, 1);
      s += __shfl_xor_sync(mask, s, 2);
      if ((threadIdx.x & 3) == 0) {
        const __half h = __float2half_rn(s);
        __half* p = a.sum + (size_t(i) * (k / 256) + c / 256) * 16 + (c % 256) / 32;
        p[0] = h;
        p[8] = __float2half_rn(s - __half2float(h));
      }
    }
  };
#pragma unroll 1
  for (int c = threadIdx.x * 8; c < k; c += kGgRowThreads * 8) {         // what this thread has left there itself
    float v[8] = {};
    if (live && c < kGgRowHeld) {
      const float4 p = *reinterpret_cast<const float4*>(row_smem + c), q = *reinterpret_cast<const float4*>(row_smem + c + 4);
      v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
    } else if (live) {
      rows_load8<KIND>(a.src, at, row, c, v);
    }
    put(c, v);
  }
}

// ---- expanders ---------------------------------------------------------------------------------------------------------
DEVI __half2 as_half2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
DEVI uint32_t as_word(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// (a & b) | c as one instruction: with both constants written out the compiler takes two, and the integer pipe paces the expanders
DEVI uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
DEVI uint32_t opaque(uint32_t v) {       // a constant that stays in a register
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// byte `i` of w as an integer in both halves (1024 + byte is exact in f16, so is the difference)
template <int I>
DEVI __half2 byte_half2(uint32_t w, float offset) {
  return __hsub2(as_half2(__byte_perm(w, 0x64006400u, 0x5050 + 0x0101 * I)), __float2half2_rn(offset));
}
DEVI void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
DEVI uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// d = a (TMEM) x b (shared memory) in f16, float32 accumulation; issued by the lane with `go` set. The eight products of a step, 64
// columns of k per box of b, in one piece with one predicate: fewer instructions for the one warp that issues (Q6_K down 447 -> 435 us).
DEVI void umma_f16_ts_step(uint32_t d, uint32_t a_tmem, uint64_t box0, uint64_t box1, uint32_t idesc, uint32_t accumulate, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, g, one;\n\t.reg .b32 t;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 g, %6, 0;\n\tsetp.eq.b32 one, 0, 0;\n\t"
      "@g tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %4, p;\n\t"
      "add.u32 t, %1, 8;\n\tadd.s64 b, %2, 2;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], b, %4, one;\n\t"
      "add.u32 t, %1, 16;\n\tadd.s64 b, %2, 4;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], b, %4, one;\n\t"
      "add.u32 t, %1, 24;\n\tadd.s64 b, %2, 6;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], b, %4, one;\n\t"
      "add.u32 t, %1, 32;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], %3, %4, one;\n\t"
      "add.u32 t, %1, 40;\n\tadd.s64 b, %3, 2;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], b, %4, one;\n\t"
      "add.u32 t, %1, 48;\n\tadd.s64 b, %3, 4;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], b, %4, one;\n\t"
      "add.u32 t, %1, 56;\n\tadd.s64 b, %3, 6;\n\t@g tcgen05.mma.cta_group::1.kind::f16 [%0], [t], b, %4, one;\n\t"
      "}"
      ::"r"(d), "r"(a_tmem), "l"(box0), "l"(box1), "r"(idesc), "r"(accumulate), "r"(go) : "memory");
}
DEVI void umma_f16_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, g;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 g, %5, 0;\n\t"
      "@g tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(go) : "memory");
}
// K-major operand tile, rows of 32 bytes, 32-byte swizzle, 8-row groups 256 bytes apart
DEVI uint64_t umma_desc_k32(uint32_t smem_addr) {
  return uint64_t((smem_addr & 0x3FFFFu) >> 4) | (uint64_t(256 >> 4) << 32) | (1ull << 46) | (6ull << 61);
}

struct GgTile { int group = 0, n0, mat, rows; long long first; };  // rows of the tile, its first dispatch row

template <typename T> DEVI T from_float(float v);
template <> DEVI float from_float<float>(float v) { return v; }
template <> DEVI __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> DEVI __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <bool Q6, int NT, int NX, typename OUT>
__global__ void __launch_bounds__((GgShape<Q6, NT, NX>::kThreads), 1)
ggml_grouped_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                    const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_x4, const __grid_constant__ CUtensorMap map_sum,
                    const __grid_constant__ CUtensorMap map_sum4, const GgArgs a) {
  using S = GgShape<Q6, NT, NX>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float2* dring = reinterpret_cast<float2*>(smem + S::kOffD);               // [4][128] {d, dmin} of the rows
  int* ends = reinterpret_cast<int*>(smem + S::kOffEnds);                   // [groups + 1] cumulative tile counts
  // A step (128 columns of k) has one "full" barrier, on which its tile of x and its expander warps count, and one "empty"
  // barrier, on which the tensor core reports it read: the loader, the expanders (kSets steps on) and, at the end of a block of
  // 256 columns, the promotion all wait for that one. Waits and commits are what the MMA warp spends its time on.
  // With two stages and nothing but the buffers between them (Q6_K) the tensor core could report the next block before a late warp
  // has looked for this one, so the promotion has barriers of its own there.
  constexpr bool kOwnDone = Q6 && S::kXStages == 2;
  __shared__ uint64_t wfull[S::kRawStages], wempty[S::kRawStages], full[S::kXStages], empty[S::kXStages], tempty[2], done[2], mfree;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float xsc[S::kPromote][NT / (S::kPromote / 4)];
  __shared__ volatile int abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < S::kRawStages; ++s) { mbar_init(wfull + s, 1); mbar_init(wempty + s, 8); }
    for (int s = 0; s < S::kXStages; ++s) { mbar_init(full + s, 5); mbar_init(empty + s, 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(tempty + s, S::kPromote); mbar_init(done + s, 1); }
    mbar_init(&mfree, S::kPromote);
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<512>(&tmem_slot);
  pdl_wait();
  pdl_launch();
  // rows of a group that lie inside [0, a.rows)
  auto group_rows = [&](int g, long long* first) {
    const unsigned r = __ldcg(a.ranges + 2 * g), o = __ldcg(a.ranges + 2 * g + 1);
    *first = o;
    return (long long)o + r <= a.rows ? int(r) : o < a.rows ? int(a.rows - o) : 0;
  };
  const int tiles_n = (a.n + 127) / 128 * a.mats;
  for (int g = threadIdx.x; g < a.groups; g += S::kThreads) {
    long long first;
    const int r = group_rows(g, &first);
    if (unsigned(r) != __ldcg(a.ranges + 2 * g) && blockIdx.x == 0) atomicOr(a.status, kStatusBadRoute);
    ends[g] = (r + NT - 1) / NT * tiles_n;
  }
  __syncthreads();
  if (warp == 0) {                       // inclusive scan, consecutive groups per lane
    // ranges that overlap can count more tiles than the rows hold: the sum stops at tile_cap, groups behind it get none
    const int per = (a.groups + 31) / 32;
    int sum = 0;
    for (int i = 0; i < per; ++i) { const int g = lane * per + i; if (g < a.groups) sum = min(sum + ends[g], a.tile_cap); }
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run = min(run + t, a.tile_cap); }
    int off = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) off = 0;
    for (int i = 0; i < per; ++i) { const int g = lane * per + i; if (g < a.groups) { off = min(off + ends[g], a.tile_cap); ends[g] = off; } }
    if (lane == 31) {
      ends[a.groups] = run;
      if (run == a.tile_cap && blockIdx.x == 0) atomicOr(a.status, kStatusBadRoute);
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot, tmem_min = tmem + S::kColMin, tmem_a = tmem + S::kColA, tmem_a2 = tmem + S::kColA2;
  const int total = ends[a.groups];
  // a warp's tiles come in ascending order: the search for the group goes on from the last one
  auto locate = [&](int tile, GgTile& t) {
    int g = t.group;                     // (ends[groups] is above every tile, what lies behind it is not looked at)
    for (;;) {                           // 32 groups at a time
      const uint32_t found = __ballot_sync(0xffffffffu, g + lane <= a.groups && tile < ends[min(g + lane, a.groups)]);
      if (found) { g += __ffs(found) - 1; break; }
      g += 32;
    }
    const int local = tile - (g ? ends[g - 1] : 0);
    t.group = g;
    const int r = group_rows(g, &t.first);
    // row tiles of equal height, a multiple of 16
    const int tiles_m = (r + NT - 1) / NT;
    int m = 0, nt = local;
    if (tiles_m > 1) {
      const int h = ((r + tiles_m - 1) / tiles_m + 15) / 16 * 16;
      nt = local / tiles_m;
      m = local - nt * tiles_m;
      t.first += m * h;
      t.rows = r - m * h < h ? r - m * h : h;
    } else {
      t.rows = r;
    }
    t.n0 = (a.mats == 2 ? nt >> 1 : nt) * 128;
    t.mat = a.mats == 2 ? nt & 1 : 0;
  };

  if (warp < 4) {
    if (S::kWide) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRegRoles));
    if (warp == 0) {
      // ---- TMA, rows of x ----------------------------------------------------------------------------------------------
      const uint32_t go = elect_lane();
      int xs = 0, used = 0;              // stage; stages filled so far (up to the first round)
      uint32_t ph = 1;                   // parity of the "empty" phase
      bool ok = true;
      GgTile t;
      for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
        locate(tile, t);
        // rows of x in boxes of 32, or one box of 128
        const bool wide = S::kWide && t.rows > 96;
        const CUtensorMap *mx = wide ? &map_x4 : &map_x, *ms = wide ? &map_sum4 : &map_sum;
        const int boxes = wide ? 1 : (t.rows + 31) / 32, height = wide ? 128 : 32, first = int(t.first);
#pragma unroll 1
        for (int c = 0; c < 2 * a.nblk; ++c) {
          if (used == S::kXStages) ok = warp_wait(empty + xs, ph, a.status);
          else ++used;
          if (!ok) break;
          if (go) {
            const uint32_t dst = smem_u32(smem + xs * S::kXStage);
            const bool with_sums = !Q6 && (c & 1);
            mbar_arrive_expect_tx(full + xs, boxes * height * (NX * 256 + (with_sums ? 32 : 0)));
#pragma unroll 1
            for (int q = 0; q < boxes; ++q) {
              const int r = first + 32 * q;
              tma_load_2d(dst + q * 32 * 128, mx, c * 256, r, full + xs);
              tma_load_2d(dst + q * 32 * 128 + S::kBox, mx, c * 256 + 128, r, full + xs);
              if (NX == 2) {
                tma_load_2d(dst + q * 32 * 128 + S::kPart, mx, c * 256, int(a.rows) + r, full + xs);
                tma_load_2d(dst + q * 32 * 128 + S::kPart + S::kBox, mx, c * 256 + 128, int(a.rows) + r, full + xs);
              }
              if (with_sums) tma_load_2d(dst + NX * S::kPart + q * 32 * 32, ms, (c >> 1) * 32, r, full + xs);
            }
          }
          if (++xs == S::kXStages) { xs = 0; ph ^= 1; }
        }
      }
      if (!ok) {                         // after a timeout the copies in flight land before the block ends
        abort_flag = 1;
        for (int i = 0; i < used; ++i) pipe_wait(full + i, i < xs ? ph ^ 1 : ph, a.status);
      }
    } else if (warp == 2) {
      // ---- TMA, packed weights: on their own, as far ahead as the ring allows ------------------------------------------------
      const uint32_t go = elect_lane();
      int ws = 0, used = 0;
      uint32_t ph = 1;
      bool ok = true;
      GgTile t;
      for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
        locate(tile, t);
        const CUtensorMap* mw = t.mat ? &map_w1 : &map_w0;
        const int wrow = t.group * a.n + t.n0;
#pragma unroll 1
        for (int b = 0; b < a.nblk; ++b) {
          if (used == S::kRawStages) ok = warp_wait(wempty + ws, ph, a.status);
          else ++used;
          if (!ok) break;
          if (go) {
            mbar_arrive_expect_tx(wfull + ws, S::kRawStage);
            tma_load_2d(smem_u32(smem + S::kOffRaw + ws * S::kRawStage), mw, b * S::kRawBytes, wrow, wfull + ws);
          }
          if (++ws == S::kRawStages) { ws = 0; ph ^= 1; }
        }
      }
      if (!ok) {
        abort_flag = 1;
        for (int i = 0; i < used; ++i) pipe_wait(wfull + i, i < ws ? ph ^ 1 : ph, a.status);
      }
    } else if (warp == 1) {
      // ---- MMA ---------------------------------------------------------------------------------------------------------
      const uint32_t go = elect_lane();
      const uint64_t dx0 = umma_desc_k128(smem_u32(smem)), dmin = umma_desc_k32(smem_u32(smem + S::kOffMin));
      const uint64_t dsum0 = umma_desc_k32(smem_u32(smem + NX * S::kPart));
      uint32_t wi = 0, slot = 0;
      bool ok = true;
      GgTile t;
      for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
        locate(tile, t);
        const uint32_t idesc = __shfl_sync(0xffffffffu, (1u << 4) | (uint32_t((t.rows + 15) / 16 * 2) << 17) | (uint32_t(128 >> 4) << 24), 0);
#pragma unroll 1
        for (int b = 0; b < a.nblk && ok; ++b, ++wi) {
          const uint32_t buf = wi & 1;
          // stage of the first step and its parity: two or four stages
          const uint32_t x0 = S::kXStages == 4 ? buf * 2 : 0u, ph = S::kXStages == 4 ? (wi >> 1) & 1 : wi & 1;
          // TMEM slots of the two steps
          const uint32_t a0 = slot, a1 = slot + 1 == S::kSets ? 0u : slot + 1;
          slot = a1 + 1 == S::kSets ? 0u : a1 + 1;
          // the buffers are free: the block before the last has been promoted
          if (S::kSteps == 1 && wi >= 2) ok = warp_wait(tempty + buf, ((wi >> 1) & 1) ^ 1, a.status);
          if (S::kSteps == 2 && wi >= 1) ok = warp_wait(tempty, (wi & 1) ^ 1, a.status);
          ok = warp_wait(full + x0, ph, a.status) && ok;
          if (!ok) break;
          tmem_fence_after();
#pragma unroll
          for (int step = 0; step < 2; ++step) {
            if (step == 1) {
              // one buffer of mins: the promotion of the last block has read it
              if (S::kMinBufs == 1 && wi >= 1) ok = warp_wait(&mfree, (wi - 1) & 1, a.status);
              if (S::kSteps == 2 && wi >= 1) ok = warp_wait(tempty + 1, (wi & 1) ^ 1, a.status) && ok;
              ok = warp_wait(full + x0 + 1, ph, a.status) && ok;
              if (!ok) break;
              tmem_fence_after();
            }
            const uint64_t dx = dx0 + (x0 + step) * uint32_t(S::kXStage >> 4);
            const uint32_t at = tmem_a + (step ? a1 : a0) * 64, a2 = tmem_a2 + (step ? a1 : a0) * 64;
            const uint32_t d = tmem + (S::kSteps == 2 ? uint32_t(step) : buf) * NT;
            const uint32_t first = S::kSteps == 2 || step == 0 ? 0u : 1u;
            const uint64_t dx1 = dx + (S::kBox >> 4), dl = dx + (S::kPart >> 4), dl1 = dl + (S::kBox >> 4);
            if (NX == 2) umma_f16_ts_step(d, at, dl, dl1, idesc, first, go);
            if (Q6) umma_f16_ts_step(d, a2, dx, dx1, idesc, NX == 2 ? 1u : first, go);
            umma_f16_ts_step(d, at, dx, dx1, idesc, NX == 2 || Q6 ? 1u : first, go);
            if (!Q6 && step == 1)                            // sums times mins
              umma_f16_ss(tmem_min + (S::kMinBufs == 2 ? buf * NT : 0u), dmin + (S::kMins == 2 ? buf * (4096u >> 4) : 0u), dsum0 + (x0 + step) * uint32_t(S::kXStage >> 4), idesc, 0u, go);
            umma_commit_if(empty + x0 + step, go);
          }
          if (kOwnDone && ok) umma_commit_if(done + buf, go);
        }
      }
      if (!ok) abort_flag = 1;
    }
  } else if (warp < 4 + 4 * S::kSets) {
    if (S::kWide) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRegExpand));
    // ---- expanders: four warps, one for each quarter of the TMEM lanes, take every kSets-th step --------------------------------
    const int set = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t tl = (uint32_t((warp & 3) * 32) << 16) + set * 64;       // the set's TMEM slot
    const uint32_t magic = opaque(0x64006400u);      // 1024 in both halves
    uint32_t wi0 = 0;                    // blocks of 256 columns before the tile
    bool ok = true;
    GgTile t;
    for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x, wi0 += a.nblk) {
      locate(tile, t);
      const __half* dq = nullptr;        // Q6_K: the row's block scales
      if (Q6) {
        const int r = t.n0 + row < a.n ? t.n0 + row : a.n - 1;
        dq = reinterpret_cast<const __half*>(a.w[t.mat] + (size_t(t.group) * a.n + r) * a.row_bytes + size_t(a.nblk) * 208);
      }
      // steps of the tile whose number, counted from the first tile on, is `set` modulo kSets
#pragma unroll 1
      for (uint32_t own = (set + 2u * S::kSets - (2u * wi0) % S::kSets) % S::kSets; own < 2u * a.nblk; own += S::kSets) {
          const uint32_t b = own >> 1, h = own & 1, wi = wi0 + b, ws = wi % S::kRawStages;
          __half d_now = {};
          if (Q6 && h == 0) d_now = __ldcg(dq + b);
          ok = warp_wait(wfull + ws, (wi / S::kRawStages) & 1, a.status);
          const uint32_t raw = smem_u32(smem + S::kOffRaw + ws * S::kRawStage) + row * S::kRawBytes;
          // Q4_K: d, dmin, 6-bit scales and mins; Q6_K: the sixteen int8 scales
          const uint4 head = lds128(raw + (Q6 ? 192 : 0));
          // the TMEM slot is free when the step kSets before has been read
          const uint32_t ps = 2 * wi + h - S::kSets;
          if (2 * wi + h >= uint32_t(S::kSets)) ok = warp_wait(empty + ps % S::kXStages, (ps / S::kXStages) & 1, a.status) && ok;
          if (!ok) break;
          tmem_fence_after();
          if (h == 0) {
            const __half2 dd = as_half2(head.x);
            dring[(wi & 3) * 128 + row] = Q6 ? make_float2(__half2float(d_now), 0.f) : make_float2(__low2float(dd), -__high2float(dd));
          } else if (!Q6) {
            // m_0 .. m_7 twice (for the high and the low parts of the sums): 32 bytes, the same whatever the swizzle
            const uint32_t m0 = head.z & 0x3f3f3f3fu, m1 = ((head.w >> 4) & 0x0f0f0f0fu) | ((head.z >> 2) & 0x30303030u);
            auto pair = [](uint32_t w, int sel) { return as_word(__hsub2(as_half2(__byte_perm(w, 0x64646464u, sel)), __float2half2_rn(1024.f))); };
            const uint4 m = make_uint4(pair(m0, 0x4140), pair(m0, 0x4342), pair(m1, 0x4140), pair(m1, 0x4342));
            uint4* p = reinterpret_cast<uint4*>(smem + S::kOffMin + (S::kMins == 2 ? (wi & 1) * 4096 : 0) + row * 32);
            p[0] = m;
            p[1] = m;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          // Q4_K: the four scales of the step; Q6_K: the step is one half of the block
          const uint32_t scales = h == 0 ? head.y & 0x3f3f3f3fu : (head.w & 0x0f0f0f0fu) | ((head.y >> 2) & 0x30303030u);
#pragma unroll 1
          for (int cc = 0; cc < 2; ++cc) {                // 64 columns
            const uint32_t dst = tl + cc * 32;
            const uint32_t at = raw + (Q6 ? 128 + h * 32 : 16 + (h * 2 + cc) * 32);
            const uint4 w0 = lds128(at), w1 = lds128(at + 16);        // Q4_K: codes; Q6_K: upper bits
            const uint32_t scw = scales >> (16 * cc);
          if (!Q6) {
            // low nibbles: columns 0-31 of the step, high nibbles: 32-63; (1024 + q) sc - 1024 sc, every term exact
            const __half2 s0 = byte_half2<0>(scw, 1024.f), s1 = byte_half2<1>(scw, 1024.f);
            const __half2 k0 = __hmul2(s0, __float2half2_rn(-1024.f)), s1d = __hmul2(s1, __float2half2_rn(0.0625f)), k1 = __hmul2(s1, __float2half2_rn(-64.f));
            uint32_t lo[16], hi[16];
            const uint32_t wd[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const uint32_t w = wd[q], u = w >> 8;
              lo[2 * q] = as_word(__hfma2(as_half2(and_or(w, 0x000f000fu, magic)), s0, k0));
              lo[2 * q + 1] = as_word(__hfma2(as_half2(and_or(u, 0x000f000fu, magic)), s0, k0));
              hi[2 * q] = as_word(__hfma2(as_half2(and_or(w, 0x00f000f0u, magic)), s1d, k1));
              hi[2 * q + 1] = as_word(__hfma2(as_half2(and_or(u, 0x00f000f0u, magic)), s1d, k1));
            }
            tmem_st16(tmem_a + dst, lo);
            tmem_st16(tmem_a + dst + 16, hi);
          } else {
            uint32_t sc4 = (h == 0 ? (cc == 0 ? head.x : head.y) : (cc == 0 ? head.z : head.w)) ^ 0x80808080u;
            const int down = 4 * cc;                    // the second 64 columns of a half block have the high nibbles and the upper bit pairs
            const uint32_t hq[8] = {w0.x >> down, w0.y >> down, w0.z >> down, w0.w >> down, w1.x >> down, w1.y >> down, w1.z >> down, w1.w >> down};
#pragma unroll 1
            for (int part = 0; part < 2; ++part, sc4 >>= 16) {       // 32 columns: the first or the second 32 bytes of ql
              const uint4 l0 = lds128(raw + h * 64 + part * 32), l1 = lds128(raw + h * 64 + part * 32 + 16);
              const uint32_t wd[8] = {l0.x, l0.y, l0.z, l0.w, l1.x, l1.y, l1.z, l1.w};
              const __half2 sa = byte_half2<0>(sc4, 1152.f), sb = byte_half2<1>(sc4, 1152.f);
              const int up = 4 - 2 * part;
              uint32_t v[16], r[16];
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const __half2 sc = q < 4 ? sa : sb;
                const uint32_t w = wd[q] >> down, h = hq[q] << up;
#pragma unroll
                for (int o = 0; o < 2; ++o) {            // even and odd bytes
                  const __half2 z = __hsub2(as_half2(and_or(o ? h >> 8 : h, 0x00300030u, and_or(o ? w >> 8 : w, 0x000f000fu, magic))),
                                            __float2half2_rn(1056.f));                    // q - 32
                  const __half2 p = __hmul2(z, sc);
                  v[2 * q + o] = as_word(p);
                  r[2 * q + o] = as_word(__hfma2(z, sc, __hneg2(p)));
                }
              }
              tmem_st16(tmem_a + dst + part * 16, v);
              tmem_st16(tmem_a2 + dst + part * 16, r);
            }
          }
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(full + (2 * wi + h) % S::kXStages);
            mbar_arrive(wempty + ws);
          }
      }
    }
    if (!ok) abort_flag = 1;
  } else {
    if (S::kWide) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kRegPromote));
    // ---- promotion and store ---------------------------------------------------------------------------------------------
    constexpr int kFirst = 4 + 4 * S::kSets, kHalf = NT / (S::kPromote / 4);       // rows of x per warp
    const int quarter = warp & 3, row = quarter * 32 + lane, c0 = ((warp - kFirst) >> 2) * kHalf;
    const uint32_t tl = (uint32_t(quarter * 32) << 16) + c0;
    float* scale = xsc[warp - kFirst];
    uint32_t wi = 0, pi = 0;             // blocks of 256 columns and partial products so far
    bool ok = true;
    GgTile t;
    for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
      locate(tile, t);
      const int rows = min(t.rows - c0, kHalf);            // of this warp's; may be none
      __syncwarp();
#pragma unroll
      for (int q = 0; q < kHalf / 32; ++q) {
        const int r = q * 32 + lane;
        const float v = r < rows ? __ldcg(a.xscale + t.first + c0 + r) : 0.f;
        if (v < 0.f && quarter == 0) atomicOr(a.status, kStatusBadRoute);
        scale[r] = fabsf(v);
      }
      __syncwarp();
      float acc[kHalf];
#pragma unroll
      for (int c = 0; c < kHalf; ++c) acc[c] = 0.f;
#pragma unroll 1
      for (int b = 0; b < a.nblk; ++b, ++wi) {
#pragma unroll 1
        for (int u = 0; u < S::kSteps; ++u, ++pi) {
          const uint32_t buf = pi & 1;
          uint64_t* bar = kOwnDone ? done + buf : empty + (S::kSteps == 2 ? pi % S::kXStages : buf * 2 + 1);
          const uint32_t ph = S::kSteps == 2 ? pi / S::kXStages : pi >> 1;
          if (!warp_wait(bar, ph & 1, a.status)) { ok = false; break; }
          tmem_fence_after();
          const float2 d = dring[(wi & 3) * 128 + row];   // {d, -dmin}
          auto add = [&](uint32_t from, float f) {        // acc += f * columns
#pragma unroll
            for (int c = 0; c < kHalf; c += 32) {
              if (c < rows) {
                uint32_t v[32];
                tmem_ld32(from + c, v);
#pragma unroll
                for (int q = 0; q < 32; ++q) acc[c + q] = fmaf(f, __uint_as_float(v[q]), acc[c + q]);
              }
            }
          };
          if (!Q6 && u == S::kSteps - 1) {
            add(tmem_min + tl + (S::kMinBufs == 2 ? (wi & 1) * NT : 0u), d.y);
            if (S::kMinBufs == 1) {
              tmem_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&mfree);
            }
          }
          add(tmem + tl + buf * NT, d.x);
          if (b + 1 < a.nblk || u + 1 < S::kSteps) {
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty + buf);
          }
        }
        if (!ok) break;
      }
      if (!ok) break;
      // The sums go through the buffer just read, which is not handed back yet: a loop of few instructions stores them (128 stores
      // in a row would come through the instruction cache anew for every tile).
      const uint32_t last = (pi - 1) & 1, stage = tmem + tl + last * NT;
#pragma unroll
      for (int c = 0; c < kHalf; c += 16) {
        if (c < rows) {
          uint32_t v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(acc[c + j]);
          tmem_st16(stage + c, v);
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      // a few output rows at a time: this warp's 32 columns of them through shared memory, out in pieces of 16 bytes
      constexpr int kAtOnce = 32 / int(sizeof(OUT)), kPieces = int(sizeof(OUT)) * 2;     // rows; pieces per row
      OUT* mine = reinterpret_cast<OUT*>(smem + S::kOffStore + (warp - kFirst) * 1024);
      const int col = t.n0 + quarter * 32;
      OUT* base = static_cast<OUT*>(a.out) + size_t(t.first + c0) * size_t(a.ldo) + size_t(t.mat) * a.n + col;
      const bool whole = a.aligned && col + 32 <= a.n;
#pragma unroll 1
      for (int c = 0; c < rows; c += 16) {
        uint32_t v[16];
        tmem_ld16(stage + c, v);
#pragma unroll
        for (int g = 0; g < 16; g += kAtOnce) {
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) mine[q * 32 + lane] = from_float<OUT>(__uint_as_float(v[g + q]) * scale[c + g + q]);
          __syncwarp();
          if (whole) {
#pragma unroll
            for (int i = lane; i < 64; i += 32) {
              const int r = i / kPieces, part = i % kPieces;
              if (c + g + r < rows)
                reinterpret_cast<uint4*>(base + size_t(c + g + r) * size_t(a.ldo))[part] = reinterpret_cast<const uint4*>(mine + r * 32)[part];
            }
          } else if (col + lane < a.n) {
            for (int r = 0; r < kAtOnce && c + g + r < rows; ++r) base[size_t(c + g + r) * size_t(a.ldo) + lane] = mine[r * 32 + lane];
          }
          __syncwarp();
        }
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty + last);
    }
    if (!ok) abort_flag = 1;
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 1) tmem_free<512>(tmem);
}

}  // namespace dmoe
