// Attention over the 8-bit cache: what its kernels (attn_kv8_cols.cu, attn_kv8_rows.cu) and their host side (attn_kv8.cu) share.
#pragma once
#include "kv8.cuh"
#include "tc.cuh"

namespace b200 {

constexpr int kKv8Tile = 128;          // tokens of a tile
constexpr int kKv8Cols = 32;           // (row, head) pairs of a group at most
constexpr int kKv8PartFloats = 132;    // of a pair in a part: 128 sums, their maximum (log2 domain), the denominator

// rows [row0, row0 + nrows) of one sequence that share its keys and values; nrows 0: none
struct Kv8Group {
  int row0, nrows, seq, ctx;   // ctx: the longest context, within the block table
};

// CTA a's last item continues in `parts` - 1 further CTAs
struct Kv8Cut {
  int row0, nrows, kvh, parts;
};

struct Kv8Params {
  const __nv_bfloat16* q;
  int64_t ldq;
  const int32_t *block_table, *row_to_seq, *ctx_lens;
  const uint8_t *ke, *ve;
  __nv_bfloat16* out;
  int64_t ldo;
  const Kv8Group* groups;      // a plan's groups (groups[-1].row0 of them), or null: found among the rows themselves
  float* part;                 // [CTA][2][pairs][kKv8PartFloats]: of an item that began in an earlier CTA, of one that goes on in the next
  Kv8Cut* cuts;                // [CTA]
  uint32_t* status;
  int64_t n_blocks;
  int bt_stride, T, hq, hkv, block_size, group_rows;   // group_rows: rows of a group at most
  float scale2;                // scale * log2 e
};

// maps of the codes: [cells][128] bytes, boxes of so many rows, 128-byte swizzle
struct Kv8Maps {
  CUtensorMap k, v;
};
int kv8_maps(const Kv8Attn& a, int box_rows, Kv8Maps* m);

int kv8_cols_launch(const Kv8Maps& m, const Kv8Params& p, int cols, int grid, cudaStream_t s);

__device__ __forceinline__ int kv8_ctx(const Kv8Params& p, int row) {
  return (int)min((int64_t)__ldg(p.ctx_lens + row), (int64_t)p.bt_stride * p.block_size);
}

// the warp's largest value; NaN if one is
__device__ __forceinline__ float warp_max_f32(float v) {
  float m;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

namespace tc {

// has the phase completed?  (mbar_try may wait for a while)
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __shfl_sync(0xffffffffu, ok, 0) != 0;   // one answer for the warp
}
// D += A B, e4m3 operands in shared memory
__device__ __forceinline__ void mma_f8_ss(uint32_t one, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
// e4m3 x e4m3 -> fp32, M = 128
__host__ __device__ constexpr uint32_t idesc_e4m3(int n, int a_mn_major) {
  return (1u << 4) | ((uint32_t)a_mn_major << 15) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// N 32-bit columns of the warp's lanes, not waited for
template <int N>
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t* r) {
  if constexpr (N == 1) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r[0]) : "r"(taddr));
  } else if constexpr (N == 2) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(taddr));
  } else if constexpr (N == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr));
  } else {
    static_assert(N == 8, "width");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  }
}

}  // namespace tc
}  // namespace b200
