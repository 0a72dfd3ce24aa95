// What the attention kernels on tcgen05 share: barriers with bounded waits, 128-byte swizzled tiles and their descriptors, the
// products (operands in shared memory, or the first in tensor memory), reads and writes of tensor memory, packed arithmetic and
// the tensor maps.
//
// A file that includes this has HEAD_DIM (64 or 128) and, in front of the include, the constants below; all of a kernel's shared
// memory is `fa_raw`, its last word is set by a wait that ran out.
//   FA_WAIT_LIMIT   polls of a wait
//   kSubTile        bytes of a [128 x 64] bfloat16 swizzled tile
//   kFaSmem         bytes of a block's shared memory
#pragma once
#include <cuda.h>

#include "common.cuh"

extern __shared__ __align__(1024) unsigned char fa_raw[];      // swizzle atoms: 1024-byte aligned

__device__ __forceinline__ unsigned fa_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
// the word that a wait that ran out sets
__device__ __forceinline__ unsigned fa_gave_up_at() { return fa_smem(fa_raw) + (unsigned)(kFaSmem - 4); }
__device__ __forceinline__ void fa_mbar_init(unsigned long long* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(fa_smem(bar)), "r"(count));
}
__device__ __forceinline__ void fa_mbar_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(fa_smem(bar)) : "memory");
}
__device__ __forceinline__ bool fa_mbar_wait(unsigned long long* bar, unsigned parity) {
  const unsigned addr = fa_smem(bar);
  // the thread sleeps in hardware until the phase completes or the hint runs out, so
  // waiting warps do not take issue slots from working ones
  const unsigned suspend_ns = 20000u;
  // Unrolled, and with the report of a wait that ran out at each of its two dozen places, this loop made half of the
  // kernel's 115 KB of code.  Behind a layer's other kernels that code starts cold, and its misses stand in a row: one
  // portion of 128 tokens behind 256 MB of other traffic took 16.1 us (14 heads of 64) and 17.3 (12 of 128), and 9.3 and
  // 11.8 with this, loops of the loaders kept as loops and the block's start in the order it has now; 2,048 tokens 36.4 ->
  // 28.1 and 36.7 -> 32.3.
#pragma unroll 1
  for (unsigned spin = 0; spin < FA_WAIT_LIMIT; ++spin) {
    unsigned done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(addr), "r"(parity), "r"(suspend_ns) : "memory");
    if (done) return true;
  }
  asm volatile("st.shared.u32 [%0], 1;" ::"r"(fa_gave_up_at()) : "memory");      // reported at the block's end
  return false;
}
// byte offset of element (row, 16-byte piece c) in a [rows x 64] bfloat16 tile with 128-byte swizzle
__device__ __forceinline__ int swz(int row, int c) {
  return (row >> 3) * 1024 + (row & 7) * 128 + ((c ^ (row & 7)) << 4);
}
__device__ __forceinline__ bool fa_elect() {
  unsigned one;
  asm volatile("{\n.reg .pred p;\n.reg .b32 r;\nelect.sync r|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}
// Matrix descriptors of tiles of 128-byte swizzled rows, 8-row groups 1024 bytes apart (stride offset); the low word is
// the tile's address in 16 bytes and the leading offset, which steps inside a tile only add to.
//   K-major (q, k): no leading offset;  MN-major (v: a key per 128-byte row of 64 lanes): 64-lane pieces of the head
//   one sub-tile apart
constexpr unsigned kDescHigh = 64u | (1u << 14) | (2u << 29);
constexpr unsigned kDescK = 1u << 16, kDescV = (unsigned)(kSubTile >> 4) << 16;
// the product of a K-major a and b
__device__ __forceinline__ void fa_mma(unsigned tmem_d, unsigned a_at, unsigned b_at, unsigned idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n"
      ::"r"(tmem_d), "r"(a_at | kDescK), "r"(b_at | kDescK), "r"(idesc), "r"((unsigned)accumulate), "r"(kDescHigh)
      : "memory");
}
// the first operand from tensor memory (16 bits, two to a column: a product's 16 lanes of k are 8 columns)
__device__ __forceinline__ void fa_mma_ts(unsigned tmem_d, unsigned tmem_a, unsigned b_at, unsigned idesc,
                                          bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 b, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n"
      ::"r"(tmem_d), "r"(tmem_a), "r"(b_at | kDescV), "r"(idesc), "r"((unsigned)accumulate), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void fa_commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
               ::"r"(fa_smem(bar)) : "memory");
}
// columns of this thread's row, waited for in the same statement (nothing may use a register before the wait)
__device__ __forceinline__ void fa_tmem_load64(unsigned taddr, float (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
      ",%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      ",%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47"
      ",%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void fa_tmem_load16(unsigned taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
      "}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void fa_tmem_store16(unsigned taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16"
      "};\n"
      :: "r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
        "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void fa_tmem_store32(unsigned taddr, const unsigned (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16"
      ",%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32"
      "};\n"
      :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// two 32-bit values in one 64-bit register, for the packed arithmetic of sm_100
__device__ __forceinline__ unsigned long long fa_pack2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void fa_unpack2(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long fa_fma2(unsigned long long a, unsigned long long b,
                                                      unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long fa_add2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float fa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void fa_copy16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(fa_smem(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void fa_expect(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(fa_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fa_tma(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(fa_smem(dst)), "l"(map), "r"(fa_smem(bar)), "r"(x), "r"(y) : "memory");
}

// ---- host side ----------------------------------------------------------------
typedef CUresult (*FaEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static FaEncodeFn fa_encode() {
  static const FaEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<FaEncodeFn>(p);
  }();
  return fn;
}

// A map over row-major [rows, lanes] bfloat16, boxes of box_rows x 64 lanes, 128-byte swizzle, zeros outside.
static int fa_map(CUtensorMap* map, const void* base, long long rows, long long lanes, int box_rows) {
  const FaEncodeFn fn = fa_encode();
  if (!fn) return TOKB200_BAD_SIZE;
  const cuuint64_t dims[2] = {(cuuint64_t)lanes, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)lanes * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TOKB200_OK : TOKB200_BAD_ALIGNMENT;
}
