// Paged attention over the 8-bit cache (kv8.cuh): a warp per (row, kv head) walks the context token by token, all G query heads at once.
#include "kv8.cuh"

namespace b200 {
namespace {

constexpr int kMostHeads = 16;

__device__ __forceinline__ void codes4(uint32_t c, float (&x)[4]) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xffffu), __NV_E4M3),
                    hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3);
  const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

__global__ void __launch_bounds__(32) paged_attn_fp8_kernel(const Kv8Attn a) {
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, kvh = blockIdx.y, lane = threadIdx.x, G = a.hq / a.hkv;
  const int seq = a.row_to_seq ? a.row_to_seq[t] : t;
  const int ctx = (int)min((int64_t)a.ctx_lens[t], (int64_t)a.bt_stride * a.block_size);
  float q[kMostHeads][4], o[kMostHeads][4] = {}, m[kMostHeads], l[kMostHeads] = {};
#pragma unroll
  for (int g = 0; g < kMostHeads; ++g) {
    m[g] = -INFINITY;
    if (g >= G) continue;
    const uint2 v = *reinterpret_cast<const uint2*>(a.q + (int64_t)t * a.ldq + (kvh * G + g) * kHeadDim + 4 * lane);
    q[g][0] = bf16lo(v.x), q[g][1] = bf16hi(v.x), q[g][2] = bf16lo(v.y), q[g][3] = bf16hi(v.y);
  }
  for (int j = 0; j < ctx; ++j) {
    const int blk = a.block_table[(int64_t)seq * a.bt_stride + j / a.block_size];
    float k[4] = {}, v[4] = {}, ks = 0.f, vs = 0.f;
    if (blk >= 0 && blk < a.n_blocks) {
      const int64_t cell = ((int64_t)blk * a.hkv + kvh) * a.block_size + j % a.block_size;
      codes4(*reinterpret_cast<const uint32_t*>(a.kc + cell * kHeadDim + 4 * lane), k);
      codes4(*reinterpret_cast<const uint32_t*>(a.vc + cell * kHeadDim + 4 * lane), v);
      ks = kv8_scale(a.ke[cell]);
      vs = kv8_scale(a.ve[cell]);
    }
#pragma unroll
    for (int g = 0; g < kMostHeads; ++g) {
      if (g >= G) continue;
      const float s = warp_sum(q[g][0] * k[0] + q[g][1] * k[1] + q[g][2] * k[2] + q[g][3] * k[3]) * ks * a.scale;
      const float mn = fmaxf(m[g], s), f = mn == -INFINITY ? 1.f : expf(m[g] - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
      m[g] = mn;
      l[g] = l[g] * f + p;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[g][i] = o[g][i] * f + p * (v[i] * vs);
    }
  }
#pragma unroll
  for (int g = 0; g < kMostHeads; ++g) {
    if (g >= G) continue;
    const float inv = l[g] == 0.f ? 0.f : 1.f / l[g];
    *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.ldo + (kvh * G + g) * kHeadDim + 4 * lane) =
        make_uint2(pack_bf16(o[g][0] * inv, o[g][1] * inv), pack_bf16(o[g][2] * inv, o[g][3] * inv));
  }
}

}  // namespace

int64_t paged_attn_fp8_workspace_bytes(int T, int hq, int hkv) { return 16; }

int paged_attn_fp8(const Kv8Attn& a, int most, void* ws, int64_t ws_bytes, cudaStream_t s) {
  B200_CUDA(launch(paged_attn_fp8_kernel, dim3(a.T, a.hkv), dim3(32), 0, s, a));
  return B200_OK;
}

}  // namespace b200
