// The 8-bit paged cache: per token and kv head 128 e4m3 codes and one exponent byte, value = code * 2^(byte - 127).
//
// A power of two as scale costs a float format nothing but the bottom of its range (e4m3 keeps its four significant bits at any exponent), makes
// the value an exact bf16, and is one byte beside 128.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {

constexpr int kKv8MinExp = -100;   // exponent of rows of zeros, and of rows that need a smaller one

// cache blocks: whole boxes of rows of a 128-token tile, or whole tiles
inline bool kv8_block_ok(int block_size) { return block_size == 16 || block_size == 32 || block_size == 64 || (block_size > 0 && block_size % 128 == 0); }
// rows (token, kv head) of a cache stay below 2^31: TMA coordinates are 32-bit
inline bool kv8_rows_ok(int64_t n_blocks, int hkv, int block_size) {
  return n_blocks > 0 && n_blocks <= 0x7fffffffll / ((int64_t)hkv * block_size);
}

// the byte of a row whose largest magnitude has these fp32 bits: the smallest e >= kKv8MinExp with amax <= 448 * 2^e = 1.75 * 2^(e + 8); 255 for inf and NaN
__device__ __forceinline__ uint32_t kv8_exp_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(max(e, kKv8MinExp) + 127);
}
// two codes, the first in the low byte; magnitudes above 448 do not occur (kv8_exp_byte)
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

int rope_kv_append_fp8(const __nv_bfloat16* qkv, int64_t ld, const int32_t* positions, const int32_t* slots, const __nv_bfloat16* cos_sin,
                       __nv_bfloat16* q_out, int64_t ldq, uint8_t* kc, uint8_t* vc, uint8_t* ke, uint8_t* ve, int64_t n_blocks, int T, int hq, int hkv,
                       int block_size, cudaStream_t s);

struct Kv8Attn {
  const __nv_bfloat16* q;
  int64_t ldq;
  const uint8_t *kc, *vc, *ke, *ve;
  int64_t n_blocks;
  const int32_t* block_table;
  int bt_stride;
  const int32_t *row_to_seq, *ctx_lens;
  __nv_bfloat16* out;
  int64_t ldo;
  int T, hq, hkv, block_size;
  float scale;
};
int64_t paged_attn_fp8_workspace_bytes(int T, int hq, int hkv);
// most: rows of a sequence are at most so many (1: decode rows), 0: not known
int paged_attn_fp8(const Kv8Attn& a, int most, void* ws, int64_t ws_bytes, cudaStream_t s);

int64_t verify_drafts_workspace_bytes(int n_rows, int vocab);
int verify_drafts(const __nv_bfloat16* target, int64_t ldt, const __nv_bfloat16* draft, int64_t ldd, const int32_t* tokens, const int32_t* starts,
                  const float* temperature, const float* uniforms, int n_seqs, int n_rows, int vocab, int32_t* out, int32_t* accepted, void* ws,
                  int64_t ws_bytes, cudaStream_t s);

}  // namespace b200
