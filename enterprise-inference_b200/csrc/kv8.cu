// (a4 + a5 over an 8-bit cache) RoPE of the q and k heads, k and v rows quantised as they are appended.  The cache's form: kv8.cuh.
//
// RoPE in fp32: (x1 c - x2 s, x2 c + x1 s) for the pairs (i, i + 64).  Products of bf16 values are exact in fp32, so every output is rounded once in
// fp32 and once to what it is stored as (bf16 for q, e4m3 for k): closer to the formula than rope_kv_kernel's bf16 arithmetic, which follows the
// reference's image.
// Eight lanes take a head of a row: lane j the entries 8 j .. 8 j + 7 and their partners, 16 bytes each, so that the pairs are rotated and the head's largest
// magnitude found (three shuffles) without shared memory.  A group of lanes for every head: with two or four heads each the loads of a group overlap, but rows of few
// heads take longer (1024 rows, 48 heads: 5.1, 6.0, 8.9 us; 2047 rows, 80 heads: 16.4, 16.8, 23.9).  Bound by the rows' bytes, 4.9 TB/s at 2047.
#include "kv8.cuh"

namespace b200 {
namespace {

constexpr int kAppendThreads = 256;

__device__ __forceinline__ void unpack8(const uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) x[2 * j] = bf16lo(w[j]), x[2 * j + 1] = bf16hi(w[j]);
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

__global__ void __launch_bounds__(kAppendThreads)
rope_kv_append_fp8_kernel(const __nv_bfloat16* qkv, int64_t ld, const int32_t* __restrict__ positions, const int32_t* __restrict__ slots,
                          const __nv_bfloat16* __restrict__ cos_sin, __nv_bfloat16* q_out, int64_t ldq, uint8_t* __restrict__ kc, uint8_t* __restrict__ vc,
                          uint8_t* __restrict__ ke, uint8_t* __restrict__ ve, int64_t n_slots, int T, int hq, int hkv, int block_size) {
  pdl_wait();
  pdl_launch_dependents();
  const int heads = hq + 2 * hkv, j = threadIdx.x & 7;
  const int64_t unit = (int64_t)blockIdx.x * (kAppendThreads / 8) + (threadIdx.x >> 3);
  const int t = (int)(unit / heads), head = (int)(unit % heads);
  const unsigned group = 0xffu << (threadIdx.x & 24);   // the head's lanes
  if (t >= T) return;
  const __nv_bfloat16* x = qkv + (int64_t)t * ld + head * kHeadDim + 8 * j;
  // all that is read, asked for at once
  const uint4 x0 = *reinterpret_cast<const uint4*>(x), x1 = *reinterpret_cast<const uint4*>(x + 64);
  const int slot = slots[t];
  uint4 cs0 = {}, cs1 = {};
  if (head < hq + hkv) {
    const __nv_bfloat16* cs = cos_sin + (int64_t)positions[t] * kHeadDim + 8 * j;
    cs0 = ld_ro(cs), cs1 = ld_ro(cs + 64);
  }
  float a[8], b[8];
  unpack8(x0, a);
  unpack8(x1, b);
  if (head < hq + hkv) {
    float c[8], s[8];
    unpack8(cs0, c);
    unpack8(cs1, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = a[i] * c[i] - b[i] * s[i], w = b[i] * c[i] + a[i] * s[i];
      a[i] = u, b[i] = w;
    }
  }
  if (head < hq) {
    __nv_bfloat16* y = q_out + (int64_t)t * ldq + head * kHeadDim + 8 * j;
    *reinterpret_cast<uint4*>(y) = pack8(a);
    *reinterpret_cast<uint4*>(y + 64) = pack8(b);
    return;
  }
  if (slot < 0 || slot >= n_slots) return;
  // magnitudes as integers: inf and NaN are the largest
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(group, m, o));
  const uint32_t byte = kv8_exp_byte(m);
  uint32_t lo[2], hi[2];
  if (byte == 255u) {
    lo[0] = lo[1] = hi[0] = hi[1] = 0x7f7f7f7fu;
  } else {
    const float f = __uint_as_float((254u - byte) << 23);   // 2^-e
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lo[i] = e4m3x2(a[4 * i] * f, a[4 * i + 1] * f) | e4m3x2(a[4 * i + 2] * f, a[4 * i + 3] * f) << 16;
      hi[i] = e4m3x2(b[4 * i] * f, b[4 * i + 1] * f) | e4m3x2(b[4 * i + 2] * f, b[4 * i + 3] * f) << 16;
    }
  }
  const bool key = head < hq + hkv;
  const int kvh = head - hq - (key ? 0 : hkv);
  const int64_t cell = ((int64_t)(slot / block_size) * hkv + kvh) * block_size + slot % block_size;
  uint8_t* dst = (key ? kc : vc) + cell * kHeadDim + 8 * j;
  *reinterpret_cast<uint2*>(dst) = make_uint2(lo[0], lo[1]);
  *reinterpret_cast<uint2*>(dst + 64) = make_uint2(hi[0], hi[1]);
  if (j == 0) (key ? ke : ve)[cell] = (uint8_t)byte;
}

}  // namespace

int rope_kv_append_fp8(const __nv_bfloat16* qkv, int64_t ld, const int32_t* positions, const int32_t* slots, const __nv_bfloat16* cos_sin,
                       __nv_bfloat16* q_out, int64_t ldq, uint8_t* kc, uint8_t* vc, uint8_t* ke, uint8_t* ve, int64_t n_blocks, int T, int hq, int hkv,
                       int block_size, cudaStream_t s) {
  if (T == 0) return B200_OK;
  const int64_t units = (int64_t)T * (hq + 2 * hkv), per = kAppendThreads / 8;
  B200_CUDA(launch(rope_kv_append_fp8_kernel, dim3((unsigned)((units + per - 1) / per)), dim3(kAppendThreads), 0, s, qkv, ld, positions, slots, cos_sin, q_out,
                   ldq, kc, vc, ke, ve, n_blocks * block_size, T, hq, hkv, block_size));
  return B200_OK;
}

}  // namespace b200

using namespace b200;

static bool kv8_heads_ok(int hq, int hkv) { return hkv > 0 && hq > 0 && hq % hkv == 0; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

extern "C" int b200_rope_kv_append_fp8(const void* qkv, int64_t ld, const int32_t* positions, const int32_t* slot_mapping, const void* cos_sin, void* q_out,
                                       int64_t ldq, void* k_codes, void* v_codes, void* k_exps, void* v_exps, int64_t n_blocks, int32_t T, int32_t hq,
                                       int32_t hkv, int32_t block_size, void* stream) {
  B200_REQUIRE(qkv && positions && slot_mapping && cos_sin && q_out && k_codes && v_codes && k_exps && v_exps, B200_ERR_INVALID, "rope_kv_append_fp8: null");
  B200_REQUIRE(T >= 0 && kv8_heads_ok(hq, hkv), B200_ERR_INVALID, "rope_kv_append_fp8: %d rows, %d heads over %d", T, hq, hkv);
  B200_REQUIRE(kv8_block_ok(block_size), B200_ERR_UNSUPPORTED, "rope_kv_append_fp8: block_size=%d (16, 32, 64 or a multiple of 128)", block_size);
  B200_REQUIRE(kv8_rows_ok(n_blocks, hkv, block_size), B200_ERR_INVALID, "rope_kv_append_fp8: %lld blocks", (long long)n_blocks);
  B200_REQUIRE(ld >= (int64_t)(hq + 2 * hkv) * kHeadDim && ld % 8 == 0 && ldq >= (int64_t)hq * kHeadDim && ldq % 8 == 0, B200_ERR_INVALID,
               "rope_kv_append_fp8: ld and ldq are multiples of 8 that hold a row");
  B200_REQUIRE(aligned16(qkv) && aligned16(cos_sin) && aligned16(q_out) && aligned16(k_codes) && aligned16(v_codes), B200_ERR_INVALID,
               "rope_kv_append_fp8: tensors must be 16-byte aligned");
  return rope_kv_append_fp8(static_cast<const __nv_bfloat16*>(qkv), ld, positions, slot_mapping, static_cast<const __nv_bfloat16*>(cos_sin),
                            static_cast<__nv_bfloat16*>(q_out), ldq, static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(v_codes),
                            static_cast<uint8_t*>(k_exps), static_cast<uint8_t*>(v_exps), n_blocks, T, hq, hkv, block_size, (cudaStream_t)stream);
}

static int attn_fp8(const char* who, const void* q, int64_t ldq, const void* kc, const void* vc, const void* ke, const void* ve, int64_t n_blocks,
                    const int32_t* block_table, int32_t bt_stride, const int32_t* row_to_seq, const int32_t* ctx_lens, void* out, int64_t ldo, int32_t T,
                    int32_t hq, int32_t hkv, int32_t block_size, int32_t most, float scale, void* ws, int64_t ws_bytes, void* stream) {
  B200_REQUIRE(q && kc && vc && ke && ve && block_table && ctx_lens && out, B200_ERR_INVALID, "%s: null", who);
  B200_REQUIRE(T >= 0 && kv8_heads_ok(hq, hkv) && bt_stride > 0 && most >= 0, B200_ERR_INVALID, "%s: %d rows, %d heads over %d, %d block-table columns", who, T,
               hq, hkv, bt_stride);
  B200_REQUIRE(hq / hkv <= 16, B200_ERR_UNSUPPORTED, "%s: %d heads over %d (at most 16 to a kv head)", who, hq, hkv);
  B200_REQUIRE(kv8_block_ok(block_size), B200_ERR_UNSUPPORTED, "%s: block_size=%d (16, 32, 64 or a multiple of 128)", who, block_size);
  B200_REQUIRE(kv8_rows_ok(n_blocks, hkv, block_size), B200_ERR_INVALID, "%s: %lld blocks", who, (long long)n_blocks);
  B200_REQUIRE(ldq >= (int64_t)hq * kHeadDim && ldq % 8 == 0 && ldo >= (int64_t)hq * kHeadDim && ldo % 8 == 0, B200_ERR_INVALID,
               "%s: ldq and ldo are multiples of 8 that hold a row", who);
  B200_REQUIRE(aligned16(q) && aligned16(out) && aligned16(kc) && aligned16(vc) && aligned16(ke) && aligned16(ve), B200_ERR_INVALID,
               "%s: tensors must be 16-byte aligned", who);
  B200_REQUIRE(scale - scale == 0.f, B200_ERR_INVALID, "%s: scale must be finite", who);
  if (T == 0) return B200_OK;
  B200_REQUIRE(ws && aligned16(ws) && ws_bytes >= paged_attn_fp8_workspace_bytes(T, hq, hkv), B200_ERR_INVALID,
               "%s: the workspace is 16-byte aligned and has at least %lld bytes (%lld)", who, (long long)paged_attn_fp8_workspace_bytes(T, hq, hkv),
               (long long)ws_bytes);
  const Kv8Attn a = {static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const uint8_t*>(kc), static_cast<const uint8_t*>(vc),
                     static_cast<const uint8_t*>(ke), static_cast<const uint8_t*>(ve), n_blocks, block_table, bt_stride, row_to_seq, ctx_lens,
                     static_cast<__nv_bfloat16*>(out), ldo, T, hq, hkv, block_size, scale};
  return paged_attn_fp8(a, most, ws, ws_bytes, (cudaStream_t)stream);
}

extern "C" int64_t b200_paged_attn_fp8_workspace_bytes(int32_t T, int32_t hq, int32_t hkv) {
  return T > 0 && kv8_heads_ok(hq, hkv) ? paged_attn_fp8_workspace_bytes(T, hq, hkv) : 0;
}
extern "C" int b200_paged_attn_decode_fp8(const void* q, int64_t ldq, const void* k_codes, const void* v_codes, const void* k_exps, const void* v_exps,
                                          int64_t n_blocks, const int32_t* block_table, int32_t bt_stride, const int32_t* row_to_seq,
                                          const int32_t* ctx_lens, void* out, int64_t ldo, int32_t T, int32_t hq, int32_t hkv, int32_t block_size, float scale,
                                          void* ws, int64_t ws_bytes, void* stream) {
  return attn_fp8("paged_attn_decode_fp8", q, ldq, k_codes, v_codes, k_exps, v_exps, n_blocks, block_table, bt_stride, row_to_seq, ctx_lens, out, ldo, T, hq,
                  hkv, block_size, 1, scale, ws, ws_bytes, stream);
}
extern "C" int b200_paged_attn_prefill_fp8(const void* q, int64_t ldq, const void* k_codes, const void* v_codes, const void* k_exps, const void* v_exps,
                                           int64_t n_blocks, const int32_t* block_table, int32_t bt_stride, const int32_t* row_to_seq,
                                           const int32_t* ctx_lens, void* out, int64_t ldo, int32_t T, int32_t hq, int32_t hkv, int32_t block_size,
                                           int32_t max_rows, float scale, void* ws, int64_t ws_bytes, void* stream) {
  return attn_fp8("paged_attn_prefill_fp8", q, ldq, k_codes, v_codes, k_exps, v_exps, n_blocks, block_table, bt_stride, row_to_seq, ctx_lens, out, ldo, T, hq,
                  hkv, block_size, max_rows, scale, ws, ws_bytes, stream);
}

extern "C" int64_t b200_verify_drafts_workspace_bytes(int32_t n_rows, int32_t vocab) {
  return n_rows > 0 && vocab > 0 ? verify_drafts_workspace_bytes(n_rows, vocab) : 0;
}
extern "C" int b200_verify_drafts(const void* target_logits, int64_t ldt, const void* draft_logits, int64_t ldd, const int32_t* draft_tokens,
                                  const int32_t* row_starts, const float* temperature, const float* uniforms, int32_t n_seqs, int32_t n_rows, int32_t vocab,
                                  int32_t* out_tokens, int32_t* out_accepted, void* ws, int64_t ws_bytes, void* stream) {
  B200_REQUIRE(target_logits && draft_tokens && row_starts && out_tokens && out_accepted && (uniforms || !temperature), B200_ERR_INVALID, "verify_drafts: null");
  B200_REQUIRE(n_seqs >= 0 && n_rows >= 0 && vocab > 0 && ldt >= vocab && (!draft_logits || ldd >= vocab), B200_ERR_INVALID,
               "verify_drafts: %d sequences, %d rows of %d entries, ldt=%lld ldd=%lld", n_seqs, n_rows, vocab, (long long)ldt, (long long)ldd);
  if (n_seqs == 0) return B200_OK;
  const int64_t need = verify_drafts_workspace_bytes(n_rows, vocab);
  B200_REQUIRE((ws && aligned16(ws) && ws_bytes >= need) || need == 0, B200_ERR_INVALID,
               "verify_drafts: the workspace is 16-byte aligned and has at least %lld bytes (%lld)", (long long)need, (long long)ws_bytes);
  return verify_drafts(static_cast<const __nv_bfloat16*>(target_logits), ldt, static_cast<const __nv_bfloat16*>(draft_logits), ldd, draft_tokens, row_starts,
                       temperature, uniforms, n_seqs, n_rows, vocab, out_tokens, out_accepted, ws, ws_bytes, (cudaStream_t)stream);
}
