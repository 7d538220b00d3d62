// Check of drafted tokens against the target's probabilities (b200_verify_drafts), two launches.
//
// stats: a CTA takes a slice of a logit row (target rows, and the rows that drafts were drawn from) and leaves its largest logit m, the first place of it and the sum
// of 2^((l - m) c), c = log2e / T, in fp32 on the hardware's exponential: enough for a draft's limit u q(x) < p(x).  The difference of two logits is exact, or
// rounded once, and never above zero, whatever the temperature: l c by itself has no bits left for its fraction where T is small.  A thread compares 32 entries with its maximum at once; the place is looked for at the end, by the threads that met the CTA's
// largest (with a place kept by every thread the same took 23.5 million instructions for 64 x 5 drafts over 128256 entries, this 15.2; differences and products in place of one
// fused operation made them 16.1, in the same time).  35 us there, 4.2 TB/s;
// bound by the exponentials (four a cycle and quarter of an SM: 16 us) and the latency of short loops.
// draw: a cluster of eight CTAs takes a sequence: the kept drafts from the slices' sums, then the token from the one row that draws it.  A draw next to a border of
// the cumulated weights has to come out as in exact arithmetic (128 k borders: sums that are off by 1e-9 pick another token once in 4000 draws), so weights and
// sums are fp64 there: 2^t by a table of 32 powers and a cubic, relative error below 2e-13, ten fp64 operations a weight (16 powers and a degree of 5, with selects for
// masked entries: 45 instructions a weight in all and 49 us, this 30 and 40).  Each CTA owns an eighth of the row in chunks of 256 entries, the target's fetched once
// into shared memory; sums are taken in a fixed order, chunk by chunk.  Bound by the instructions of the weights: 27 thousand a quarter of an SM.
#include <cooperative_groups.h>

#include <algorithm>

#include "kv8.cuh"
#include "f32x2.cuh"
#include "tc.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kStatGroups = 4, kLeastSlice = 2048, kWholeSlice = kStatThreads * 8 * kStatGroups;
constexpr float kLeastScale = 1.4426950408889634e-30f, kMostScale = 1.4426950408889634e30f;   // log2e / T of temperatures between 1e30 (masked entries weigh nothing) and 1e-30
constexpr int kDrawThreads = 256, kDrawCtas = 8, kChunk = 256, kMostChunks = 192;
constexpr int kMostVocab = kDrawCtas * kMostChunks * kChunk, kMostPart = kMostChunks * kChunk * 2;

struct alignas(16) Stat {
  float m, s;
  int at;
};
constexpr int kKnownRows = 64;   // rows of a sequence whose largest logits are kept

// eight entries from index i on (-inf behind the end), 16 bytes at a time where the address allows it
__device__ __forceinline__ bool whole8(const __nv_bfloat16* row, int i, int n) { return i + 8 <= n && (reinterpret_cast<uintptr_t>(row + i) & 15) == 0; }
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int i, int n) {
  if (whole8(row, i, n)) return ld_ro(row + i);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = i + 2 * j;
    const uint32_t a = k < n ? __bfloat16_as_ushort(row[k]) : 0xff80u, b = k + 1 < n ? __bfloat16_as_ushort(row[k + 1]) : 0xff80u;
    w[j] = a | b << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void fetch8(uint4* dst, const __nv_bfloat16* row, int i, int n) {   // -> shared memory
  if (whole8(row, i, n)) f2::cp16(dst, row + i);
  else *dst = load8(row, i, n);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__global__ void __launch_bounds__(kStatThreads)
verify_stats_kernel(const __nv_bfloat16* __restrict__ target, int64_t ldt, const __nv_bfloat16* __restrict__ draft, int64_t ldd, const int32_t* __restrict__ starts,
                    const float* __restrict__ temperature, int n_seqs, int vocab, int slice_len, Stat* __restrict__ stats) {
  __shared__ int found, first;
  __shared__ float sh_m[kStatThreads / 32], sh_s[kStatThreads / 32];
  pdl_wait();
  const int slice = blockIdx.x, row = blockIdx.y, which = blockIdx.z;
  if (threadIdx.x == 0) found = -1, first = 0x7fffffff;
  __syncthreads();
  for (int s = threadIdx.x; s < n_seqs; s += kStatThreads)
    if (starts[s] <= row && row < starts[s + 1]) found = s;
  __syncthreads();
  const int seq = found;
  if (seq < 0) return;
  const float temp = temperature ? temperature[seq] : 0.f;
  if (which && (!(temp > 0.f) || row == starts[seq + 1] - 1)) return;   // no probabilities asked for
  const __nv_bfloat16* l = which ? draft + (int64_t)row * ldd : target + (int64_t)row * ldt;
  // entries from i0 on in groups of eight that start at 16-byte addresses (the slice's ends may lie inside a group)
  const int shift = (int)((reinterpret_cast<uintptr_t>(l) >> 1) & 7);
  const int i0 = slice * slice_len, i1 = min(vocab, i0 + slice_len), a0 = i0 - shift;
  float m = -INFINITY, s = 0.f;
  int at = 0x7fffffff;
  const float c = temp > 0.f ? fmaxf(fminf(1.4426950408889634f / temp, kMostScale), kLeastScale) : 0.f;
  constexpr int U = kStatGroups, S = kStatThreads * 8;
  for (int g0 = a0 + threadIdx.x * 8; g0 < i1; g0 += U * S) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = g0 + u * S;
      v[u] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
      if (i >= i0 && i + 8 <= i1) {
        v[u] = ld_stream(l + i);
      } else if (i + 8 > i0 && i < i1) {   // a group that crosses the slice's ends: its entries one by one
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = i + 2 * j;
          const uint32_t x = k >= i0 && k < i1 ? __bfloat16_as_ushort(l[k]) : 0xff80u, y = k + 1 >= i0 && k + 1 < i1 ? __bfloat16_as_ushort(l[k + 1]) : 0xff80u;
          w[j] = x | y << 16;
        }
        v[u] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    uint32_t h = 0xff80ff80u;
#pragma unroll
    for (int u = 0; u < U; ++u) h = max2(h, max2(max2(v[u].x, v[u].y), max2(v[u].z, v[u].w)));
    const float top = fmaxf(bf16lo(h), bf16hi(h));
    if (top > m) {
      s *= tc::exp2_fast((m - top) * c);   // (nothing yet: 2^-inf)
      m = top;
      at = g0;
    }
    if (!(temp > 0.f)) continue;
    const float from = m > -INFINITY ? -m : 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g0 + u * S >= i1) break;
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      uint64_t e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t t = f2::mul(f2::add(f2::pack(bf16lo(w[j]), bf16hi(w[j])), f2::both(from)), f2::both(c));
        e[j] = f2::pack(tc::exp2_fast(f2::lo(t)), tc::exp2_fast(f2::hi(t)));
      }
      s += f2::sum(f2::add(f2::add(e[0], e[1]), f2::add(e[2], e[3])));
    }
  }
  pdl_launch_dependents();   // (before the rows are read the next launch's CTAs would only take their places: 112 -> 141 us)
  const float most = warp_max(m);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh_m[warp] = most;
  __syncthreads();
  float all = sh_m[0];
#pragma unroll
  for (int w = 1; w < kStatThreads / 32; ++w) all = fmaxf(all, sh_m[w]);
  // the first place of the largest entry: those look for it who met it
  if (m == all && m > -INFINITY) {
    bool there = false;
    for (int u = 0; u < U && !there; ++u)
      for (int k = max(at + u * S, i0), end = min(at + u * S + 8, i1); k < end && !there; ++k)
        if (__bfloat162float(l[k]) == m) atomicMin(&first, k), there = true;
  }
  s = warp_sum(m > -INFINITY ? s * tc::exp2_fast((m - all) * c) : 0.f);
  if (lane == 0) sh_s[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kStatThreads / 32; ++w) s += sh_s[w];
    stats[((int64_t)row * 2 + which) * gridDim.x + slice] = {all, s, first};
  }
}

// a bf16 in its fp32 bits -> the double of 2^-896 times its value (the exponent's bits moved as they are; denormals stay what they are, -inf comes out as
// -2^128 times that: nothing beside any logit that counts)
__device__ __forceinline__ double scaled_double(uint32_t f) { return __hiloint2double((int)f >> 3 & (int)0x8fffffffu, 0); }
__device__ __forceinline__ double scaled_double(float x) { return scaled_double(__float_as_uint(x)); }
constexpr double kScaledBack = 0x1p896;
// 2^t for t <= 0, 2^-1017 below that: t = n / 32 + r, 2^(n / 32) = 2^(n >> 5) table[n & 31], 2^r = 1 + r q(r), |r| <= 1 / 64: the series of (2^r - 1) / r
// with its terms above the third taken down to a cubic by Chebyshev polynomials, 1.6e-13 of 2^r
__device__ __forceinline__ double exp2_table(double t, const double* table) {
  t = __hiloint2double((int)min((uint32_t)__double2hiint(t), 0xc08fc800u), __double2loint(t));
  const double u = t + 211106232532992.0;   // 1.5 * 2^47: n in the low bits
  const double r = t - (u - 211106232532992.0);
  const int n = __double2loint(u);
  double q = fma(r, 0.00961817611557608, 0.05550443419199583);
  q = fma(q, r, 0.24022650695623157);
  q = fma(q, r, 0.693147180550011);
  const double b = table[n & 31], e = fma(b * r, q, b);
  return __hiloint2double(__double2hiint(e) + ((n & ~31) << 15), __double2loint(e));
}
// what 2^t gives for a masked entry, 7.2e-307, is no weight, nor is a chunk's sum of them: a chunk whose sum is one has an entry that is, a row whose sum is one a chunk
constexpr double kLeastWeight = 1e-306, kLeastChunk = kChunk * kLeastWeight, kNothing = 1e-300;
static_assert(kDrawCtas * kMostChunks * kLeastChunk < kNothing, "weights");
__device__ __forceinline__ double warp_sum_double(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kDrawThreads, 4) __cluster_dims__(kDrawCtas, 1, 1)
verify_draw_kernel(const __nv_bfloat16* __restrict__ target, int64_t ldt, const __nv_bfloat16* __restrict__ draft, int64_t ldd,
                   const int32_t* __restrict__ tokens, const int32_t* __restrict__ starts, const float* __restrict__ temperature,
                   const float* __restrict__ uniforms, int n_rows, int vocab, int n_slices, const Stat* __restrict__ stats, int32_t* __restrict__ out,
                   int32_t* __restrict__ accepted) {
  extern __shared__ __align__(16) unsigned char row_smem[];   // the CTA's part of the target row
  __shared__ double table[32], chunk_sum[kMostChunks], chunk_q[kMostChunks], warp_part[2][kDrawThreads / 32], mine[2], shared_w, known_ratio[kKnownRows], sh_ratio;
  __shared__ int sh_refused, sh_best, sh_chunk, known_at[kKnownRows];
  __shared__ float sh_m[2], known_m[kKnownRows][2];
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), s = blockIdx.x / kDrawCtas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  pdl_wait();
  pdl_launch_dependents();
  const int r0 = min(max(starts[s], 0), n_rows), r1 = min(max(starts[s + 1], r0), n_rows);
  const float temp = temperature ? temperature[s] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double c = greedy ? 0.0 : fmax(fmin(1.4426950408889634 / (double)temp, (double)kMostScale), (double)kLeastScale);
  const double cf = greedy ? 0.0 : (double)fmaxf(fminf(1.4426950408889634f / temp, kMostScale), kLeastScale);   // what the sums have
  if (tid == 0) sh_refused = max(r1 - r0 - 1, 0);
  __syncthreads();
  // a row's largest logits, their first place and (relative to them) the sums, from the slices (by a warp)
  auto row_stats = [&](int r, float (&m)[2], double (&z)[2], int& at, bool sums) {
    at = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[k] = -INFINITY, z[k] = 0.0;
      if (k && (greedy || r == r1 - 1 || !draft)) continue;
      const Stat* st = stats + ((int64_t)r * 2 + k) * n_slices;
      for (int i = lane; i < n_slices; i += 32) {
        const Stat x = st[i];
        if (!k && (x.m > m[0] || (x.m == m[0] && x.at < at))) at = x.at;
        m[k] = fmaxf(m[k], x.m);
      }
      const float own = m[k];
      m[k] = warp_max(own);
      if (!k) at = __reduce_min_sync(0xffffffffu, own == m[0] ? at : 0x7fffffff);
      if (!sums || !(m[k] > -INFINITY)) continue;
      for (int i = lane; i < n_slices; i += 32)
        if (st[i].m > -INFINITY) z[k] += (double)st[i].s * exp2_table(((double)st[i].m - (double)m[k]) * cf, table);
      z[k] = warp_sum_double(z[k]);
    }
    if (m[0] == -INFINITY) at = 0;
  };
  // the sums of a row's target over its draft, each relative to its largest logit, as near as fp32 has them
  auto ratio = [&](const double (&z)[2]) { return z[1] > 0.0 ? z[0] / z[1] : 0.0; };
  // the probability of an entry (its bits) of a row, down to the least number there is (the table's powers end before)
  auto probability = [&](uint32_t bits, float m, double z) { return exp2(((double)__uint_as_float(bits << 16) - (double)m) * cf) / z; };
  // a warp a row: is the draft refused?
  for (int r = r0 + warp; r < r1; r += kDrawThreads / 32) {
    double z[2];
    float m[2];
    int at;
    const bool last = r == r1 - 1;
    const int x = last ? -1 : tokens[r];
    bool ok = !last && x >= 0 && x < vocab;
    // (asked for before the sums are there)
    const uint32_t lx = ok ? __bfloat16_as_ushort(target[(int64_t)r * ldt + x]) : 0u, dx = ok && draft ? __bfloat16_as_ushort(draft[(int64_t)r * ldd + x]) : 0u;
    const double u = ok && !greedy ? (double)uniforms[2 * r] : 0.0;
    row_stats(r, m, z, at, !greedy);
    if (lane == 0 && r - r0 < kKnownRows) {
      known_m[r - r0][0] = m[0], known_m[r - r0][1] = m[1], known_at[r - r0] = at;
      known_ratio[r - r0] = ratio(z);
    }
    ok = ok && m[0] > -INFINITY;
    if (ok && greedy) {
      ok = x == at;
    } else if (ok) {
      const double p = probability(lx, m[0], z[0]), q = !draft ? 1.0 : m[1] > -INFINITY ? probability(dx, m[1], z[1]) : 0.0;
      ok = u * q < p;
    }
    if (!ok && lane == 0) atomicMin(&sh_refused, r - r0);
  }
  __syncthreads();
  const int taken = sh_refused, row = r0 + taken;
  const bool any = r1 > r0, last = row == r1 - 1;
  // the row that draws: its largest logits
  if (any && taken < kKnownRows) {
    if (tid == 0) sh_m[0] = known_m[taken][0], sh_m[1] = known_m[taken][1], sh_best = known_at[taken], sh_ratio = known_ratio[taken];
  } else if (any && warp == 0) {
    double z[2];
    float m[2];
    int at;
    row_stats(row, m, z, at, !greedy);
    if (lane == 0) sh_m[0] = m[0], sh_m[1] = m[1], sh_best = at, sh_ratio = ratio(z);
  }
  __syncthreads();
  if (rank == 0) {
    if (tid == 0) accepted[s] = taken;
    for (int r = r0 + tid; r < r1; r += kDrawThreads)
      if (r != row) out[r] = r < row ? tokens[r] : -1;
    if (any && tid == 0) out[row] = sh_best;   // greedy, or nothing to draw from (or, with NaN among the logits, no border found); else a draw's CTA writes again
  }
  if (!any || greedy || sh_m[0] == -INFINITY) return;   // (the cluster's CTAs all leave here)

  const __nv_bfloat16* l = target + (int64_t)row * ldt;
  const bool residual = !last, probs = residual && draft && sh_m[1] > -INFINITY;
  const __nv_bfloat16* d = probs ? draft + (int64_t)row * ldd : nullptr;
  const int x = residual && !draft ? tokens[row] : -1;   // a certain draft: what is left has nothing of it
  const double mp = scaled_double(sh_m[0]), mq = probs ? scaled_double(sh_m[1]) : 0.0, scale = c * kScaledBack;
  const int n_chunks = (vocab + kChunk - 1) / kChunk, per = (n_chunks + kDrawCtas - 1) / kDrawCtas;
  const int ch0 = min(n_chunks, rank * per), ch1 = min(n_chunks, ch0 + per);
  // the CTA's entries, -inf behind the end (a thread reads back what it wrote: its eight of every 16th chunk)
  uint4* part_p = reinterpret_cast<uint4*>(row_smem);
  for (int ch = ch0 + warp; ch < ch1; ch += kDrawThreads / 32) {
    const int i = ch * kChunk + 8 * lane, at = (ch - ch0) * (kChunk / 8) + lane;
    fetch8(part_p + at, l, i, vocab);
  }
  f2::cp_wait_all();
  // entry j of eight, relative to the row's largest logit (m: scaled as they are)
  auto weight = [&](const uint32_t* w, int j, double m) { return exp2_table((scaled_double(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16) - m) * scale, table); };
  // running sums of the chunks, by a warp: kMostChunks / 32 neighbours a lane, then over the lanes; returns their sum
  auto running = [&](double* v) {
    constexpr int N = kMostChunks / 32;
    double t[N], sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = lane * N + i;
      sum += at < ch1 - ch0 ? v[at] : 0.0;
      t[i] = sum;
    }
    double front = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double w = __shfl_up_sync(0xffffffffu, front, o);
      if (lane >= o) front += w;
    }
    const double prev = __shfl_up_sync(0xffffffffu, front, 1), base = lane ? prev : 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane * N + i < ch1 - ch0) v[lane * N + i] = base + t[i];
    return __shfl_sync(0xffffffffu, front, 31);
  };
  double to_p = 1.0, to_q = 1.0;   // one over the rows' sums
  if (probs) {
    // One pass over both rows: their sums, and for each chunk the sums A of e^p and B of e^q over the entries of which p is the larger, going by the ratio of the rows' sums
    // in fp32: max(p - q, 0) then sums to A / Zp - B / Zq.  A chunk with an entry of equal p and q to within 2^-17 (the ratio is good to 2^-19) is marked, and
    // taken entry by entry below, as is one whose difference loses four digits.
    const double rho = sh_ratio;
    double zp = 0.0, zq = 0.0;
    uint4 next = ch0 + warp < ch1 ? load8(d, (ch0 + warp) * kChunk + 8 * lane, vocab) : uint4{};
    for (int ch = ch0 + warp; ch < ch1; ch += kDrawThreads / 32) {
      const uint4 v = part_p[(ch - ch0) * (kChunk / 8) + lane], w = next;
      if (ch + kDrawThreads / 32 < ch1) next = load8(d, (ch + kDrawThreads / 32) * kChunk + 8 * lane, vocab);
      const uint32_t p4[4] = {v.x, v.y, v.z, v.w}, q4[4] = {w.x, w.y, w.z, w.w};
      double a = 0.0, b = 0.0;
      bool near = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double ep = weight(p4, j, mp), eq = weight(q4, j, mq), more = fma(-rho, eq, ep);
        zp += ep, zq += eq;
        near |= (__double2hiint(more) & 0x7fffffff) + (17 << 20) < __double2hiint(ep);
        if (more > 0.0) a += ep, b += eq;
      }
      a = warp_sum_double(a), b = warp_sum_double(b);
      near = __any_sync(0xffffffffu, near);
      if (lane == 0) chunk_sum[ch - ch0] = near ? -1.0 : a, chunk_q[ch - ch0] = b;
    }
    zp = warp_sum_double(zp), zq = warp_sum_double(zq);
    if (lane == 0) warp_part[0][warp] = zp, warp_part[1][warp] = zq;
    __syncthreads();
    if (tid < 2) {
      double z = 0.0;
      for (int w = 0; w < kDrawThreads / 32; ++w) z += warp_part[tid][w];
      mine[tid] = z;
    }
    cluster.sync();
    zp = zq = 0.0;
#pragma unroll
    for (int k = 0; k < kDrawCtas; ++k) {
      const double* other = cluster.map_shared_rank(mine, k);
      zp += other[0], zq += other[1];
    }
    cluster.sync();   // (nobody writes again while another reads)
    to_p = 1.0 / zp, to_q = 1.0 / zq;
  }
  for (int pass = residual ? 0 : 1; pass < 2; ++pass) {   // what the draft leaves of p; p itself behind the last draft, and where nothing is left
    auto weights8 = [&](int ch, double (&w)[8]) {
      const int at = (ch - ch0) * (kChunk / 8) + lane, i = ch * kChunk + 8 * lane;
      const uint4 v = part_p[at];
      const uint32_t p4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = weight(p4, j, mp);
      if (pass) return;
      if (probs) {
        const uint4 q = load8(d, i, vocab);
        const uint32_t q4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double left = __dsub_rn(__dmul_rn(w[j], to_p), __dmul_rn(weight(q4, j, mq), to_q));   // (equal rows leave zeros)
          w[j] = left > 0.0 ? left : 0.0;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j == x) w[j] = 0.0;
    };
    for (int ch = ch0 + warp; ch < ch1; ch += kDrawThreads / 32) {
      double t = -1.0;
      if (probs && !pass) {
        const double a = chunk_sum[ch - ch0] * to_p;
        t = a - chunk_q[ch - ch0] * to_q;
        if (!(t > 1e-4 * a) && a != 0.0) t = -1.0;
      }
      if (t < 0.0) {
        double w[8];
        weights8(ch, w);
        t = warp_sum_double(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
      }
      __syncwarp();
      if (lane == 0) chunk_sum[ch - ch0] = t > kLeastChunk ? t : 0.0;   // (a draw of 0 takes the first chunk that is not 0)
    }
    __syncthreads();
    if (warp == 0) {
      const double t = running(chunk_sum);
      if (lane == 0) mine[0] = shared_w = t;
    }
    cluster.sync();
    double all = 0.0, before = 0.0;   // of all CTAs' weights, of those in front of this one's
#pragma unroll
    for (int k = 0; k < kDrawCtas; ++k) {
      const double w = *cluster.map_shared_rank(mine, k);
      if (k == rank) before = all;
      all += w;
    }
    cluster.sync();   // (nobody writes again, or leaves, while another reads)
    if (!pass && !(all > kNothing)) continue;   // nothing left: the cluster agrees
    const double limit = (double)uniforms[2 * row + 1] * all;
    if (tid == 0) sh_chunk = 0x7fffffff;
    __syncthreads();
    if (before + shared_w > limit && !(before > limit)) {   // the CTA that holds the border (each adds up the same numbers: there is one)
      for (int i = tid; i < ch1 - ch0; i += kDrawThreads)
        if (before + chunk_sum[i] > limit) atomicMin(&sh_chunk, i);   // (rounding may leave none: the last)
      __syncthreads();
      if (warp == 0) {
        const int at = min(sh_chunk, ch1 - ch0 - 1), i = (ch0 + at) * kChunk + 8 * lane;
        double w[8], t = 0.0;
        weights8(ch0 + at, w);   // (another warp's entries: the barriers in between)
#pragma unroll
        for (int j = 0; j < 8; ++j) t += w[j];
        double front = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, front, o);
          if (lane >= o) front += v;
        }
        front += before + (at > 0 ? chunk_sum[at - 1] : 0.0) - t;
        int token = 0x7fffffff, some = -1;   // the first entry above the limit; the last of any weight
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          front += w[j];
          if (w[j] > kLeastWeight) {
            some = i + j;
            if (front > limit && token == 0x7fffffff) token = i + j;
          }
        }
        token = __reduce_min_sync(0xffffffffu, token);
        some = __reduce_max_sync(0xffffffffu, some);
        if (lane == 0 && some >= 0) out[row] = token == 0x7fffffff ? some : token;   // (a chunk that only rounding let through: the largest entry stays)
      }
    }
    break;
  }
}

// slices of a row: about 24 CTAs an SM (12 and 48: 64 x 5 drafts 67.5 and 68.9 us, with 24 67.0), each of whole turns of its loop (lengths between leave the last
// turn's groups empty) or, where rows are few, of at least kLeastSlice entries (with 1024: 5 rows 20.2 us instead of
// 18.0, 20 rows 40.3 instead of 28.4)
int slice_length(int n_rows, int vocab) {
  const int64_t want = std::max<int64_t>(1, kNumSMs * 24 / std::max(1, 2 * n_rows)), len = (vocab + want - 1) / want;
  return (int)(len > kWholeSlice / 2 ? (len + kWholeSlice - 1) / kWholeSlice * kWholeSlice : std::max<int64_t>(kLeastSlice, (len + 7) / 8 * 8));
}
int slices(int n_rows, int vocab) {
  const int len = slice_length(n_rows, vocab);
  return (vocab + len - 1) / len;
}

}  // namespace

// enough for this many rows and for any smaller number (rows times slices falls where slices get longer): a row has at most want slices, and so many of kLeastSlice
int64_t verify_drafts_workspace_bytes(int n_rows, int vocab) {
  const int64_t most = ((int64_t)vocab + kLeastSlice - 1) / kLeastSlice;
  return std::min(n_rows * most, std::max<int64_t>(n_rows, kNumSMs * 24 / 2)) * 2 * (int64_t)sizeof(Stat);
}

int verify_drafts(const __nv_bfloat16* target, int64_t ldt, const __nv_bfloat16* draft, int64_t ldd, const int32_t* tokens, const int32_t* starts,
                  const float* temperature, const float* uniforms, int n_seqs, int n_rows, int vocab, int32_t* out, int32_t* accepted, void* ws,
                  int64_t ws_bytes, cudaStream_t s) {
  B200_REQUIRE(vocab <= kMostVocab, B200_ERR_UNSUPPORTED, "verify_drafts: vocab=%d (at most %d)", vocab, kMostVocab);
  B200_REQUIRE(n_rows <= 65535, B200_ERR_UNSUPPORTED, "verify_drafts: %d rows (at most 65535)", n_rows);
  B200_REQUIRE(n_seqs <= 0x7fffffff / kDrawCtas, B200_ERR_UNSUPPORTED, "verify_drafts: %d sequences (at most %d)", n_seqs, 0x7fffffff / kDrawCtas);
  Stat* stats = static_cast<Stat*>(ws);
  const int n = slices(n_rows, vocab), per = ((vocab + kChunk - 1) / kChunk + kDrawCtas - 1) / kDrawCtas, smem = per * kChunk * 2;
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(verify_draw_kernel, kMostPart, done));
  if (n_rows > 0)
    B200_CUDA(launch(verify_stats_kernel, dim3(n, n_rows, draft && temperature ? 2 : 1), dim3(kStatThreads), 0, s, target, ldt, draft, ldd, starts,
                     temperature, n_seqs, vocab, slice_length(n_rows, vocab), stats));
  const PdlScope draw(n_rows > 0);
  B200_CUDA(launch(verify_draw_kernel, dim3(n_seqs * kDrawCtas), dim3(kDrawThreads), (size_t)smem, s, target, ldt, draft, ldd, tokens, starts, temperature, uniforms, n_rows,
                   vocab, n, stats, out, accepted));
  return B200_OK;
}

}  // namespace b200
