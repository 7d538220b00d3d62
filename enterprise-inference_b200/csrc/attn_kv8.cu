// Host side of the attention over the 8-bit cache: maps, workspace, routes, and the joining of parts.
#include <algorithm>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

// an item that several CTAs share, column by column: out = sum of a_i 2^(m_i - m) / sum of l_i 2^(m_i - m)
// (a warp a column, four entries a lane)
__global__ void __launch_bounds__(256) kv8_join_kernel(const Kv8Params p) {
  pdl_wait();
  pdl_launch_dependents();
  const Kv8Cut cut = p.cuts[blockIdx.x];
  const int G = p.hq / p.hkv, lane = threadIdx.x & 31;
  if (cut.parts < 2) return;
  for (int c = blockIdx.y * 8 + (threadIdx.x >> 5); c < cut.nrows * G; c += 8 * gridDim.y) {
    auto part = [&](int i) { return p.part + ((int64_t)(2 * (blockIdx.x + i) + (i == 0)) * kKv8Cols + c) * kKv8PartFloats; };
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < cut.parts; i += 32) m = fmaxf(m, part(i)[128]);
    m = warp_max(m);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < cut.parts; ++i) {
      const float* x = part(i);
      const float f = m == -INFINITY ? 1.f : tc::exp2_fast(x[128] - m);
      const float4 v = reinterpret_cast<const float4*>(x)[lane];
      l += x[129] * f;
      a.x += v.x * f, a.y += v.y * f, a.z += v.z * f, a.w += v.w * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + (int64_t)(cut.row0 + c / G) * p.ldo + (cut.kvh * G + c % G) * kHeadDim + 4 * lane) =
        make_uint2(pack_bf16(a.x * inv, a.y * inv), pack_bf16(a.z * inv, a.w * inv));
  }
}

constexpr int64_t kCutBytes = (kNumSMs * sizeof(Kv8Cut) + 255) / 256 * 256;
constexpr int64_t kPartBytes = (int64_t)kNumSMs * 2 * kKv8Cols * kKv8PartFloats * 4;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    cudaGetLastError();
    return EncodeTiledFn(nullptr);
  }();
  return fn;
}

}  // namespace

// encoded anew by every call (1 us): a map that is kept would go by the cache's address
int kv8_maps(const Kv8Attn& a, int box_rows, Kv8Maps* m) {
  const EncodeTiledFn fn = encode_fn();
  B200_REQUIRE(fn != nullptr, B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t cells = (cuuint64_t)a.n_blocks * a.hkv * a.block_size, dims[2] = {kHeadDim, cells}, stride[1] = {kHeadDim};
  const cuuint32_t box[2] = {kHeadDim, (cuuint32_t)box_rows}, one[2] = {1, 1};
  CUresult r = CUDA_SUCCESS;
  const std::pair<CUtensorMap*, const uint8_t*> codes[2] = {{&m->k, a.kc}, {&m->v, a.vc}};
  for (int i = 0; i < 2 && r == CUDA_SUCCESS; ++i)
    r = fn(codes[i].first, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes[i].second), dims, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B200_REQUIRE(r == CUDA_SUCCESS, B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %lld rows", (int)r, (long long)cells);
  return B200_OK;
}

int64_t paged_attn_fp8_workspace_bytes(int T, int hq, int hkv) { return kCutBytes + kPartBytes; }

int paged_attn_fp8(const Kv8Attn& a, int most, void* ws, int64_t ws_bytes, cudaStream_t s) {
  B200_REQUIRE((int64_t)a.T * a.hkv * (((int64_t)a.bt_stride * a.block_size + kKv8Tile - 1) / kKv8Tile) < 0x7fffffffll, B200_ERR_UNSUPPORTED,
               "paged_attn_fp8: %d rows of up to %lld tokens", a.T, (long long)a.bt_stride * a.block_size);
  Kv8Maps maps;
  if (const int rc = kv8_maps(a, std::min(a.block_size, kKv8Tile), &maps)) return rc;
  const int G = a.hq / a.hkv;
  Kv8Params p = {};
  p.q = a.q;
  p.ldq = a.ldq;
  p.block_table = a.block_table;
  p.row_to_seq = a.row_to_seq;
  p.ctx_lens = a.ctx_lens;
  p.ke = a.ke;
  p.ve = a.ve;
  p.out = a.out;
  p.ldo = a.ldo;
  p.cuts = static_cast<Kv8Cut*>(ws);
  p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + kCutBytes);
  p.status = wait_status_word();
  p.n_blocks = a.n_blocks;
  p.bt_stride = a.bt_stride;
  p.T = a.T;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.block_size = a.block_size;
  p.scale2 = a.scale * 1.4426950408889634f;
  p.group_rows = most == 1 ? 1 : most > 0 && most * G <= kKv8Cols ? most : kKv8Cols / G;
  if (const int rc = kv8_cols_launch(maps, p, p.group_rows * G, kNumSMs, s)) return rc;
  const PdlScope join;
  B200_CUDA(launch(kv8_join_kernel, dim3(kNumSMs, (p.group_rows * G + 7) / 8), dim3(256), 0, s, p));
  return B200_OK;
}

}  // namespace b200
