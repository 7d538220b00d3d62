// Attention over the 8-bit cache: what its kernels (attn_kv8_cols.cu, attn_kv8_rows.cu) and their host side (attn_kv8.cu) share.
#pragma once
#include "f32x2.cuh"
#include "kv8.cuh"
#include "tc.cuh"

namespace b200 {

constexpr int kKv8Tile = 128;          // tokens of a tile
constexpr int kKv8Cols = 16;           // (row, head) pairs of a group at most
constexpr int kKv8Span = 100;          // bits between value exponents that are told apart: 2^that times a long context's weights is an fp32 number
constexpr int kKv8PartFloats = 132;    // of a pair in a part: 128 sums, their maximum (log2 domain), the denominator

// rows [row0, row0 + nrows) of one sequence that share its keys and values; nrows 0: none
struct Kv8Group {
  int row0, nrows, seq, ctx;   // ctx: the longest context, within the block table
};

// work of the rows kernel: rows of one sequence and a kv head over the cache tiles [tile0, tile1); parts > 1: further CTAs have the rest, each leaves its sums in
// a slot.  A CTA's items follow one another; cta -1: none
struct alignas(16) Kv8Rows {
  int row0, nrows, seq, ctx, tile0, tile1, kvh, cta, parts, slot, pad[2];
};
// what a plan found; its groups come right behind
struct Kv8Head {
  int groups, two, pad[2];   // two: items have up to two tiles of pairs
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
  const Kv8Head* groups_head;  // of a plan
  Kv8Rows* items;
  int* starts;                 // [CTA] its first item (-1: none)
  Kv8Cut* cuts_rows;           // [CTA]
  const float* q_scale;        // [row][head]: what the rows kernel's scores are multiplied by
  float* part_rows;            // [CTA][2][128 pairs][kKv8PartFloats], as part
  uint32_t* status;
  int64_t n_blocks;
  int bt_stride, T, hq, hkv, block_size, group_rows;   // group_rows: rows of a group at most
  float scale2;                // scale * log2 e
};

// maps of the codes: [cells][128] bytes, boxes of so many rows, 128-byte swizzle; of the rows kernel's queries in two terms: [rows][heads][128] bytes, boxes of the
// rows that fill a tile of 128 pairs (or 32: few) by the heads of a kv head
struct Kv8Maps {
  CUtensorMap k, v;
};
struct Kv8QueryMaps {
  CUtensorMap hi, lo;
};
int kv8_maps(const Kv8Attn& a, int box_rows, Kv8Maps* m);

int kv8_cols_launch(const Kv8Maps& m, const Kv8Params& p, int cols, int grid, cudaStream_t s);
// few: items of at most 32 pairs
int kv8_rows_launch(const Kv8Maps& m, const Kv8QueryMaps& q, const Kv8Params& p, bool few, int grid, cudaStream_t s);

__device__ __forceinline__ int kv8_ctx(const Kv8Params& p, int row) {
  return (int)min((int64_t)__ldg(p.ctx_lens + row), (int64_t)p.bt_stride * p.block_size);
}

// byte (row r, byte b) of an operand in rows of 128 bytes, 128-byte swizzle
__device__ __forceinline__ int operand_off(int r, int b) { return (r >> 3) * 1024 + (r & 7) * 128 + ((((b >> 4) ^ r) & 7) << 4) + (b & 15); }

// e4m3 by integer operations.  A value times 2^-120 has e4m3's exponent in its low bits, subnormals included: the code of x >= 0 is its bits from 20 on, rounded to
// nearest (halves up).
constexpr float kE4m3Unit = 7.52316384526264e-37f;   // 2^-120
__device__ __forceinline__ uint32_t e4m3_bits(float scaled) { return (__float_as_uint(scaled) + 0x80000u) & 0xfff00000u; }   // of a rounded value, times 2^-120
// the codes of hi and of LO times what its rounding left, for x >= 0 times 2^-120: bits 0..7 and 8..15
template <int LO>
__device__ __forceinline__ uint32_t e4m3_two(float scaled) {
  const uint32_t h = e4m3_bits(scaled);
  const float rest = (scaled - __uint_as_float(h)) * (float)LO;
  const uint32_t l = (__float_as_uint(rest) & 0x7fffffffu) + 0x80000u;   // (sign apart)
  return h >> 20 | (l >> 12 & 0x7f00u) | (__float_as_uint(rest) >> 16 & 0x8000u);
}

// A query scaled by a power of two to [128, 256), as e4m3 and LO times what that rounding left.  With LO = 16 both terms are exact down to 2^-14 of the largest
// entry, with 1 to 2^-10, and off by at most 2^-23 (2^-19) of it below.
// the largest magnitude of eight entries, as bf16 bits
__device__ __forceinline__ uint32_t query_max(const uint4 v) {
  const uint32_t x[4] = {v.x, v.y, v.z, v.w};
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) m = max(m, max(x[j] & 0x7fffu, (x[j] >> 16) & 0x7fffu));
  return m;
}
__device__ __forceinline__ uint32_t query_exponent(uint32_t max_bits) { return max(max_bits >> 7, 8u); }   // biased; 255: not a number
__device__ __forceinline__ float query_back(uint32_t e) { return __uint_as_float((min(e, 254u) - 7u) << 23); }   // undoes the scaling
template <int LO>
__device__ __forceinline__ void split_query(const uint4 v, uint32_t e, uint2& hi, uint2& lo) {
  const uint32_t x[4] = {v.x, v.y, v.z, v.w};
  const float f = __uint_as_float((261u - min(e, 254u)) << 23);   // (and the unit, as a product of its own: their exponents may not fit in one)
  uint32_t h4[4], l4[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a = e4m3_two<LO>(fabsf(bf16lo(x[j])) * f * kE4m3Unit), b = e4m3_two<LO>(fabsf(bf16hi(x[j])) * f * kE4m3Unit);
    const uint32_t s = (x[j] >> 8 & 0x80u) | (x[j] >> 16 & 0x8000u);
    h4[j] = (__byte_perm(a, b, 0x7740) & 0xffffu) ^ s;
    l4[j] = (__byte_perm(a, b, 0x7751) & 0xffffu) ^ s;
    if (e == 255u) h4[j] = 0x7f7fu;
  }
  hi = make_uint2(h4[0] | h4[1] << 16, h4[2] | h4[3] << 16);
  lo = make_uint2(l4[0] | l4[1] << 16, l4[2] | l4[3] << 16);
}

// the warp's largest value; NaN if one is
__device__ __forceinline__ float warp_max_f32(float v) {
  float m;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

namespace tc {

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)), "l"(map),
               "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
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
__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :
               : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
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
