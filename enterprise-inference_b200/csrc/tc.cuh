// tcgen05 / TMA / mbarrier primitives shared by the attention kernels whose query side fills the MMA's M dimension.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace b200 {

int get_tensor_map_2d(const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, CUtensorMap* out);
int get_tensor_map_3d(const void* ptr, uint32_t slabs, uint64_t rows, uint64_t cols, uint32_t box_rows, CUtensorMap* out);

namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits are bounded.  One that a defect keeps from completing runs out after kWaitTries (4 us each: two seconds): it marks the CTA, whose other
// waits then return as soon as they would have to wait, and sets a word in host memory that the next call reports as an error (waits.cu).  The
// TMA warp stops at the mark, the other roles run through their finite loops; what is in flight then finishes (bounded again) before shared
// and tensor memory are given up.  Tries are counted because a clock costs, even one that is only read after 64 of them: 2 048 prefill rows
// 108 us with either count or no limit at all, 118 with it.
constexpr int kWaitTries = 1 << 19;
struct Waits {
  uint32_t* mark;     // shared: a wait of this CTA ran out
  uint32_t* status;   // host memory
  int limit;
  __device__ __forceinline__ Waits(uint32_t* m, uint32_t* st, int tries = kWaitTries) : mark(m), status(st), limit(tries) {}
  __device__ __forceinline__ bool marked() const { return *reinterpret_cast<volatile uint32_t*>(mark) != 0; }
  __device__ __forceinline__ bool stop() const { return __any_sync(0xffffffffu, marked()); }   // the whole warp's answer
  __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) const {
    for (int i = 0; !mbar_try(bar, parity); ++i)
      if ((i & 63) == 63 && (marked() || i > limit)) {
        *reinterpret_cast<volatile uint32_t*>(mark) = 1;
        if (status) *reinterpret_cast<volatile uint32_t*>(status) = 1;
        return;
      }
  }
  // after the mark: for what is still in flight
  __device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) const {
    for (int i = 0; !mbar_try(bar, parity) && i < limit; ++i) {}
  }
};
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
// The columns at the end of cached rows that are no whole box of 64, of 64 rows, by a warp: where a box would have put them (128-byte swizzle, `dst` at a multiple of 1024).  Boxes that
// reach past a row's end are not used where a map declares more rows than the memory behind it has: steps with such rows (64 bytes under a box of 128) ended in illegal addresses
// three times, each behind hundreds of other calls, and nothing else of them was out of range.  `row`: the first one, below 0 where a block is none: zeros, as boxes have them; ld and cols
// multiples of 16, `from` the first row's columns
__device__ __forceinline__ void copy_tail_start(unsigned char* dst, const __nv_bfloat16* from, int row, int ld, int cols) {
  const int bytes = row < 0 ? 0 : 16, each = cols & 16 ? 1 : 2;   // 2 or 4 lanes a row: its 16-byte pieces are neighbours (a row to a lane touches 32 lines with every copy)
  const int lane = threadIdx.x & 31, r0 = lane >> each;
  const __nv_bfloat16* const src = from + (int64_t)max(row, 0) * ld;
  for (int x = lane & ((1 << each) - 1); x < cols >> 3; x += 1 << each)
#pragma unroll 4
    for (int r = r0; r < 64; r += 32 >> each)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * 128 + ((x ^ (r & 7)) << 4))), "l"(src + (int64_t)r * ld + x * 8), "r"(bytes) : "memory");
}
// behind copy_tail_start: the columns arrive at the barrier by themselves (a lane's arrival counts itself in, so before the phase's own one).  They are ordinary writes to the tensor
// cores: who waits for the barrier fences (fence_async_smem) before the products.  16 heads over 256 + 32, with a wait for the columns here instead, before the next tile is asked for, and so:
// 64 rows at 1 000 tokens 18.7 us, 16.7 (18.7 too with a row to a lane), 100 at 3 000 63.0, 57.5, one at 3 000 16.5, 15.1 (over 256 + 64, boxes alone: 16.6, 59.6, 14.6)
__device__ __forceinline__ void copy_tail_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
  __syncwarp();
}
// bytes that copies will bring, without the arrival of mbar_expect_tx
__device__ __forceinline__ void mbar_expect_more(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar)), "r"(one)
      : "memory");
}
// D += A B with A in shared memory, by the lane whose `one` is set.  The predicate is the instruction's, not a branch's: in convergent code
// the operands of a warp-uniform loop stay in uniform registers (inside `if (one)` each is moved there for every instruction).
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
// D += A B with A in tensor memory: lane = row, one 32-bit column = two neighbouring k
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
// SWIZZLE_128B operand in shared memory.  K-major: rows of 128 bytes, groups of 8 rows sbo bytes apart (lbo unused).
// MN-major: atoms of 64 MN elements x 8 k rows; k groups sbo apart, the next 64 MN elements lbo bytes away.
__device__ __forceinline__ uint64_t make_desc(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3fff);
  d |= (uint64_t)((lbo_bytes >> 4) & 0x3fff) << 16;
  d |= (uint64_t)((sbo_bytes >> 4) & 0x3fff) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// bf16 x bf16 -> fp32, M = 128
__host__ __device__ constexpr uint32_t idesc_bf16(int n, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      :
      "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
      "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      :
      "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
      "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
      "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
      "=r"(r[31])
      : "r"(taddr));
}
// waits for the thread's loads; the registers pass through so that no use moves ahead of the wait
template <int N>
__device__ __forceinline__ void ld_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :
      : "r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      :
      : "r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// 16 lanes x 32 columns: registers 4 i + {0, 1} of lane x hold columns 8 i + 2 (x % 4) + {0, 1} of row x / 4, {2, 3} those of row x / 4 + 8
__device__ __forceinline__ void st_16x256b_x4(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :
      : "r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// one whole 32-byte sector per thread (p 32-byte aligned)
__device__ __forceinline__ void store_sector(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}
// the largest of 64 scores, in eight chains (one would be 64 dependent steps)
__device__ __forceinline__ float max64(const uint32_t* s) {
  float m[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) m[j] = __uint_as_float(s[j]);
#pragma unroll
  for (int j = 8; j < 64; ++j) m[j & 7] = fmaxf(m[j & 7], __uint_as_float(s[j]));
  return fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
}
// 2^x on the hardware's exponential
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace tc
}  // namespace b200
