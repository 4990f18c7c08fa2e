// Tensor-core, TMEM, cluster and tensor-map helpers that the operators next to the MoE layers share.
#pragma once
#include "grouped_fp8.cuh"
#include "stream_launch.cuh"

namespace dmoe {

// ---- host: tensor maps -----------------------------------------------------------------------------------------------
typedef CUresult (*TensorMapEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                    const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                    CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorMapEncode tensor_map_encode() {
  static TensorMapEncode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<TensorMapEncode>(p)
               : nullptr;
  }();
  return fn;
}
// Tensor [rows][cols] of `es`-byte elements (box and columns given in bytes), rows `pitch` bytes apart (16-byte aligned base and pitch), box [box_rows][box_cols]; reads past
// the last row or column give zeros.
inline bool byte_map(CUtensorMap* m, const void* base, unsigned long long rows, unsigned long long cols, unsigned long long pitch,
                     unsigned box_rows, unsigned box_cols, CUtensorMapSwizzle swizzle, unsigned es = 1) {
  const TensorMapEncode enc = tensor_map_encode();
  if (!enc) return false;
  const cuuint64_t dims[2] = {cols / es, rows}, strides[1] = {pitch};
  const cuuint32_t box[2] = {box_cols / es, box_rows}, estr[2] = {1, 1};
  return enc(m, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : es == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Launch with programmatic dependent launch and a cluster of `cluster` blocks along x.
template <typename Kernel, typename... Args>
inline cudaError_t launch_cluster(Kernel kernel, dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- TMEM ------------------------------------------------------------------------------------------------------------
template <int COLS>
DEVI void tmem_alloc(uint32_t* slot) {      // one whole warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(uint32_t(COLS)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
DEVI void tmem_free(uint32_t base) {            // the warp that allocated
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(uint32_t(COLS)) : "memory");
}
// 32 columns of this warp's 32 TMEM lanes -> registers, complete on return
DEVI void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}

// 64 columns, complete on return
#define DMOE_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define DMOE_R16(r, i) DMOE_R4(r, i), DMOE_R4(r, i + 4), DMOE_R4(r, i + 8), DMOE_R4(r, i + 12)
DEVI void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : DMOE_R16(r, 0), DMOE_R16(r, 16), DMOE_R16(r, 32), DMOE_R16(r, 48)
      : "r"(taddr) : "memory");
}
#undef DMOE_R16
#undef DMOE_R4

// Bounded waits for a phase. What a wait costs when the phase is over already is most of what these kernels' single warps spend:
// one probe without a branch around it (70 cycles beside twenty busy warps; a probe inside a loop of its own 160, a broadcast from
// one lane 250). After that each probe suspends the thread for up to 2 us, and a million of them set the status bit.
DEVI uint32_t phase_over(uint32_t addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(addr), "r"(parity)
      : "memory");
  return ok;
}
DEVI uint32_t phase_probe(uint32_t addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 2000;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(addr), "r"(parity)
      : "memory");
  return ok;
}
DEVI bool pipe_wait(uint64_t* bar, uint32_t parity, unsigned* status) {      // one thread
  const uint32_t addr = smem_u32(bar);
  if (__builtin_expect(phase_over(addr, parity), 1)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < 1000000u; ++i)
    if (phase_probe(addr, parity)) return true;
  atomicOr(status, kStatusWaitTimeout);
  return false;
}
// A whole warp; the vote keeps the lanes together, so that loops around the wait stay on the uniform datapath, where the operands of
// tcgen05.mma and of the tensor copies live.
DEVI bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* status) {
  const uint32_t addr = smem_u32(bar);
  if (__builtin_expect(__all_sync(0xffffffffu, phase_over(addr, parity)), 1)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < 1000000u; ++i)
    if (__all_sync(0xffffffffu, phase_probe(addr, parity))) return true;
  if ((threadIdx.x & 31) == 0) atomicOr(status, kStatusWaitTimeout);
  return false;
}
DEVI uint32_t elect_lane() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}
// commits by the lane with `go` set
DEVI void umma_commit_if(uint64_t* bar, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %1, 0;\n\t"
      "@g tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(go) : "memory");
}

// ---- clusters --------------------------------------------------------------------------------------------------------
DEVI uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
DEVI void cluster_sync() {       // all threads of all blocks of the cluster
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same shared-memory location in block `rank` of the cluster
DEVI uint32_t cluster_map(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Barrier anywhere in the cluster, address from cluster_map. It hands over TMEM, which tcgen05.fence orders: a release at the scope of
// the cluster would wait here for everything this thread has in flight (400 to 2000 cycles).
DEVI void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
DEVI float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

}  // namespace dmoe
