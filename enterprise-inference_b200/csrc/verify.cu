// Check of drafted tokens against the target's probabilities (b200_verify_drafts): a CTA takes a sequence, its rows in order, in 64 bits.
#include "kv8.cuh"

namespace b200 {
namespace {

constexpr int kVerifyThreads = 1024;

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
  for (int i = 0; i < kVerifyThreads / 32; ++i) t += sh[i];
  __syncthreads();
  return t;
}
// largest value of a row and its first place
__device__ __forceinline__ float row_max(const __nv_bfloat16* l, int vocab, int* at, float* shv, int* shi) {
  float m = -INFINITY;
  int i0 = 0x7fffffff;
  for (int i = threadIdx.x; i < vocab; i += kVerifyThreads) {
    const float v = __bfloat162float(l[i]);
    if (v > m || i0 == 0x7fffffff) m = v, i0 = i;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, m, o);
    const int i = __shfl_xor_sync(0xffffffffu, i0, o);
    if (v > m || (v == m && i < i0)) m = v, i0 = i;
  }
  if ((threadIdx.x & 31) == 0) shv[threadIdx.x >> 5] = m, shi[threadIdx.x >> 5] = i0;
  __syncthreads();
  for (int w = 0; w < kVerifyThreads / 32; ++w)
    if (shv[w] > m || (shv[w] == m && shi[w] < i0)) m = shv[w], i0 = shi[w];
  __syncthreads();
  *at = i0;
  return m;
}

__global__ void __launch_bounds__(kVerifyThreads)
verify_kernel(const __nv_bfloat16* target, int64_t ldt, const __nv_bfloat16* draft, int64_t ldd, const int32_t* tokens, const int32_t* starts,
              const float* temperature, const float* uniforms, int n_rows, int vocab, int32_t* out, int32_t* accepted) {
  __shared__ double sh[kVerifyThreads / 32], part[kVerifyThreads];
  __shared__ float shv[32];
  __shared__ int shi[32], found;
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x, r0 = max(starts[s], 0), r1 = min(starts[s + 1], n_rows);
  const double temp = temperature ? (double)temperature[s] : 0.0;
  int taken = 0, token = -1;
  for (int r = r0; r < r1; ++r) {
    const bool last = r == r1 - 1;
    const __nv_bfloat16* l = target + (int64_t)r * ldt;
    const __nv_bfloat16* d = draft ? draft + (int64_t)r * ldd : nullptr;
    const int x = last ? -1 : tokens[r];
    int best;
    const float m = row_max(l, vocab, &best, shv, shi);
    if (!(temp > 0.0) || m == -INFINITY) {
      token = best;
      if (best == x && m > -INFINITY) {
        if (threadIdx.x == 0) out[r0 + taken] = x;
        ++taken;
        continue;
      }
      break;
    }
    double z = 0, zd = 0;
    float md = 0;
    for (int i = threadIdx.x; i < vocab; i += kVerifyThreads) z += exp((double)(__bfloat162float(l[i]) - m) / temp);
    z = block_sum(z, sh);
    if (d && !last) {
      int at;
      md = row_max(d, vocab, &at, shv, shi);
      for (int i = threadIdx.x; i < vocab && md > -INFINITY; i += kVerifyThreads) zd += exp((double)(__bfloat162float(d[i]) - md) / temp);
      zd = block_sum(zd, sh);
    }
    auto p = [&](int i) { return exp((double)(__bfloat162float(l[i]) - m) / temp) / z; };
    auto q = [&](int i) {
      if (last) return 0.0;
      if (!d) return i == x ? 1.0 : 0.0;
      return zd > 0 ? exp((double)(__bfloat162float(d[i]) - md) / temp) / zd : 0.0;
    };
    if (!last && x >= 0 && x < vocab && (double)uniforms[2 * r] * q(x) < p(x)) {
      if (threadIdx.x == 0) out[r0 + taken] = x;
      ++taken;
      continue;
    }
    const int per = (vocab + kVerifyThreads - 1) / kVerifyThreads, i0 = min((int)threadIdx.x * per, vocab), i1 = min(i0 + per, vocab);
    for (int pass = 0; pass < 2; ++pass) {   // what is left of p; p itself where nothing is
      auto w = [&](int i) { return pass ? p(i) : fmax(p(i) - q(i), 0.0); };
      double own = 0;
      for (int i = i0; i < i1; ++i) own += w(i);
      part[threadIdx.x] = own;
      if (threadIdx.x == 0) found = 0x7fffffff;
      __syncthreads();
      double before = 0, all = 0;
      for (int i = 0; i < kVerifyThreads; ++i) {
        if (i == (int)threadIdx.x) before = all;
        all += part[i];
      }
      const double limit = (double)uniforms[2 * r + 1] * all;
      double c = before;
      for (int i = i0; i < i1; ++i) {
        c += w(i);
        if (c > limit) {
          atomicMin(&found, i);
          break;
        }
      }
      __syncthreads();
      token = found;
      __syncthreads();
      if (all > 0) break;
    }
    break;
  }
  if (threadIdx.x == 0) {
    accepted[s] = taken;
    for (int r = r0 + taken; r < r1; ++r) out[r] = r == r0 + taken ? token : -1;
  }
}

}  // namespace

int64_t verify_drafts_workspace_bytes(int n_rows, int vocab) { return 0; }

int verify_drafts(const __nv_bfloat16* target, int64_t ldt, const __nv_bfloat16* draft, int64_t ldd, const int32_t* tokens, const int32_t* starts,
                  const float* temperature, const float* uniforms, int n_seqs, int n_rows, int vocab, int32_t* out, int32_t* accepted, void* ws,
                  int64_t ws_bytes, cudaStream_t s) {
  B200_CUDA(launch(verify_kernel, dim3(n_seqs), dim3(kVerifyThreads), 0, s, target, ldt, draft, ldd, tokens, starts, temperature, uniforms, n_rows, vocab, out,
                   accepted));
  return B200_OK;
}

}  // namespace b200
