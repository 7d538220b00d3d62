// Attention over the paged cache with a mask per row (b200_paged_attn_tree): trees of drafted tokens, beams that share a prompt.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),  over the tokens j that the row sees: those in front of ctx_lens[t], and ctx_lens[t] + i for each
//   bit i of its mask.
//
// Rows of one sequence that follow one another share its keys and values: a CTA takes up to 32 (row, head) pairs of a kv head and walks the sequence in tiles of 64
// tokens, all in fp32 (one pass, running maximum and sum).
#include <algorithm>

#include "kv8.cuh"
#include "tc.cuh"

namespace b200 {
namespace {

constexpr int kTreeThreads = 256, kTreePairs = 32, kTreeKeys = 64, kMostWords = 32;

struct TreeParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t ldq, n_blocks;
  const int32_t *block_table, *row_to_seq, *ctx_lens;
  const uint32_t* masks;
  __nv_bfloat16* out;
  int64_t ldo;
  int bt_stride, words, T, hq, hkv, block_size;
  float scale;
};

__device__ __forceinline__ int64_t tree_tokens(const TreeParams& p) { return (int64_t)p.bt_stride * p.block_size; }
// tokens up to the last one that a row sees
__device__ __forceinline__ int tree_end(const TreeParams& p, int row) {
  const int64_t most = tree_tokens(p);
  int64_t end = min((int64_t)max(__ldg(p.ctx_lens + row), 0), most);
  for (int w = p.words - 1; w >= 0; --w) {
    const uint32_t m = __ldg(p.masks + (int64_t)row * p.words + w);
    if (m) return (int)min(most, (int64_t)max(__ldg(p.ctx_lens + row), 0) + 32 * w + 32 - __clz(m));
  }
  return (int)end;
}
__device__ __forceinline__ bool tree_sees(const TreeParams& p, int row, int ctx, int j) {
  if (j < ctx) return true;
  const int i = j - ctx;
  return i < 32 * p.words && (__ldg(p.masks + (int64_t)row * p.words + (i >> 5)) >> (i & 31) & 1);
}

__global__ void __launch_bounds__(kTreeThreads) attn_tree_kernel(const TreeParams p, int R) {
  __shared__ float qs[kTreePairs][kHeadDim], sc[kTreePairs][kTreeKeys + 1];
  __shared__ __nv_bfloat16 ks[kTreeKeys][kHeadDim + 8];
  __shared__ int sh_end;
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x, G = p.hq / p.hkv;
  auto seq_of = [&](int r) { return p.row_to_seq ? __ldg(p.row_to_seq + r) : r; };
  const int seq = seq_of(row0);
  int back = 0;   // rows of the sequence in front
  while (back < row0 && seq_of(row0 - back - 1) == seq) ++back;
  if (back % R) return;
  int rows = 1;
  while (rows < R && row0 + rows < p.T && seq_of(row0 + rows) == seq) ++rows;
  if (tid == 0) sh_end = 0;
  for (int e = tid; e < kTreePairs * kHeadDim; e += kTreeThreads) {
    const int pr = e / kHeadDim, d = e % kHeadDim, r = pr / G;
    qs[pr][d] = r < rows ? __bfloat162float(p.q[(int64_t)(row0 + r) * p.ldq + (kvh * G + pr % G) * kHeadDim + d]) : 0.f;
  }
  __syncthreads();
  if (tid < rows) atomicMax(&sh_end, tree_end(p, row0 + tid));
  __syncthreads();
  const int end = sh_end, pr = tid >> 3, sub = tid & 7, r = pr / G;
  const bool alive = r < rows;
  const int row = row0 + min(r, rows - 1), ctx = (int)min((int64_t)max(__ldg(p.ctx_lens + row), 0), tree_tokens(p));
  float m = -INFINITY, l = 0.f, o[16] = {};
  auto stage = [&](const __nv_bfloat16* cache, int k0) {
    for (int e = tid; e < kTreeKeys * 16; e += kTreeThreads) {
      const int j = k0 + (e >> 4), c = (e & 15) * 8;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (j < end) {
        const int64_t blk = __ldg(p.block_table + (int64_t)seq * p.bt_stride + j / p.block_size);
        if (blk >= 0 && blk < p.n_blocks) x = ld_ro(cache + ((blk * p.hkv + kvh) * p.block_size + j % p.block_size) * kHeadDim + c);
      }
      *reinterpret_cast<uint4*>(&ks[e >> 4][c]) = x;
    }
  };
  for (int k0 = 0; k0 < end; k0 += kTreeKeys) {
    __syncthreads();
    stage(p.k, k0);
    __syncthreads();
    float s[8], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = sub + 8 * i;
      float a = 0.f;
      for (int d = 0; d < kHeadDim; ++d) a = fmaf(qs[pr][d], __bfloat162float(ks[j][d]), a);
      s[i] = alive && k0 + j < end && tree_sees(p, row, ctx, k0 + j) ? a * p.scale : -INFINITY;
      top = fmaxf(top, s[i]);
    }
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float mn = fmaxf(m, top), f = m > -INFINITY ? expf(m - mn) : 0.f;
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = s[i] > -INFINITY || s[i] != s[i] ? expf(s[i] - mn) : 0.f;
      sc[pr][sub + 8 * i] = s[i] == -INFINITY ? -1.f : e;   // -1: not seen
      part += e;
    }
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) part += __shfl_xor_sync(0xffffffffu, part, x);
    l = l * f + part;
    m = mn;
    __syncthreads();
    stage(p.v, k0);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < 16; ++d) o[d] *= f;
    for (int j = 0; j < kTreeKeys; ++j) {
      const float w = sc[pr][j];
      if (w == -1.f) continue;   // (whatever stands in a token that the row does not see)
#pragma unroll
      for (int d = 0; d < 16; ++d) o[d] = fmaf(w, __bfloat162float(ks[j][sub * 16 + d]), o[d]);
    }
  }
  if (!alive) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* to = p.out + (int64_t)row * p.ldo + (kvh * G + pr % G) * kHeadDim + sub * 16;
#pragma unroll
  for (int d = 0; d < 16; ++d) to[d] = __float2bfloat16_rn(o[d] * inv);
}

}  // namespace
}  // namespace b200

using namespace b200;

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool tree_heads_ok(int hq, int hkv) { return hkv > 0 && hq > 0 && hq % hkv == 0; }

extern "C" int64_t b200_paged_attn_tree_workspace_bytes(int32_t T, int32_t hq, int32_t hkv) { return T > 0 && tree_heads_ok(hq, hkv) ? 16 : 0; }

extern "C" int b200_paged_attn_tree(const void* q, int64_t ldq, const void* k_cache_layer, const void* v_cache_layer, int64_t n_blocks, const int32_t* block_table,
                                    int32_t bt_stride, const int32_t* row_to_seq, const int32_t* ctx_lens, const uint32_t* tree_masks, int32_t mask_words, void* out,
                                    int64_t ldo, int32_t T, int32_t hq, int32_t hkv, int32_t block_size, float scale, void* ws, int64_t ws_bytes, void* stream) {
  B200_REQUIRE(q && k_cache_layer && v_cache_layer && block_table && ctx_lens && out && (tree_masks || mask_words == 0), B200_ERR_INVALID, "paged_attn_tree: null");
  B200_REQUIRE(T >= 0 && tree_heads_ok(hq, hkv) && bt_stride > 0 && mask_words >= 0, B200_ERR_INVALID,
               "paged_attn_tree: %d rows, %d heads over %d, %d block-table columns, %d mask words", T, hq, hkv, bt_stride, mask_words);
  B200_REQUIRE(hq / hkv <= 16, B200_ERR_UNSUPPORTED, "paged_attn_tree: %d heads over %d (at most 16 to a kv head)", hq, hkv);
  B200_REQUIRE(mask_words <= kMostWords, B200_ERR_UNSUPPORTED, "paged_attn_tree: %d mask words (at most %d)", mask_words, kMostWords);
  B200_REQUIRE(kv8_block_ok(block_size), B200_ERR_UNSUPPORTED, "paged_attn_tree: block_size=%d (16, 32, 64 or a multiple of 128)", block_size);
  B200_REQUIRE(kv8_rows_ok(n_blocks, hkv, block_size), B200_ERR_INVALID, "paged_attn_tree: %lld blocks", (long long)n_blocks);
  B200_REQUIRE((int64_t)bt_stride * block_size <= 0x7fffffff - 256, B200_ERR_UNSUPPORTED, "paged_attn_tree: block tables of %lld tokens", (long long)bt_stride * block_size);
  B200_REQUIRE(ldq >= (int64_t)hq * kHeadDim && ldq % 8 == 0 && ldo >= (int64_t)hq * kHeadDim && ldo % 8 == 0, B200_ERR_INVALID,
               "paged_attn_tree: ldq and ldo are multiples of 8 that hold a row");
  B200_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_cache_layer) && aligned16(v_cache_layer), B200_ERR_INVALID, "paged_attn_tree: tensors must be 16-byte aligned");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(tree_masks) & 3) == 0, B200_ERR_INVALID, "paged_attn_tree: masks must be 4-byte aligned");
  B200_REQUIRE(scale > 0.f && scale - scale == 0.f, B200_ERR_INVALID, "paged_attn_tree: scale must be positive and finite");
  if (T == 0) return B200_OK;
  const int64_t need = b200_paged_attn_tree_workspace_bytes(T, hq, hkv);
  B200_REQUIRE(ws && aligned16(ws) && ws_bytes >= need, B200_ERR_INVALID, "paged_attn_tree: the workspace is 16-byte aligned and has at least %lld bytes (%lld)",
               (long long)need, (long long)ws_bytes);
  const TreeParams p = {static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k_cache_layer), static_cast<const __nv_bfloat16*>(v_cache_layer), ldq,
                        n_blocks, block_table, row_to_seq, ctx_lens, tree_masks, static_cast<__nv_bfloat16*>(out), ldo, bt_stride, mask_words, T, hq, hkv, block_size, scale};
  B200_CUDA(launch(attn_tree_kernel, dim3((unsigned)T, (unsigned)hkv), dim3(kTreeThreads), (size_t)0, (cudaStream_t)stream, p, kTreePairs / (hq / hkv)));
  return B200_OK;
}
