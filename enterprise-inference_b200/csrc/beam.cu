// A beam search's selection over beams and vocabulary (b200_beam_select), two launches.
//
// score(r, i) = scores[r] + x_ri - log sum_j exp x_rj; a sequence takes the K largest of its rows and all their entries, ties by row, then by entry.
// blocks: a warp takes 2 048 neighbouring logits, all in registers at once, and leaves their largest, m, and the sum of exp(x - m).  No barriers, nothing is selected.
// merge: a cluster takes a sequence.  One of its CTAs joins the blocks' sums; a number that more than K blocks' largest scores reach bounds the K-th score from below, and only
// the blocks that reach it, little more than K, are read again.  Where a sequence has less than kBlocksEach blocks for each of the K, their largest entries may lie far behind the K-th: groups of
// eight entries give the limit then; and a list that is longer than K + kSpare is cut by a limit of its own entries (ranks take as long as the square of their number), one that has no room for
// all by a limit of all: 40 000 entries near the limit in 4 rows of 32 768, 16 to take, 120 us, 88 with a limit of the 1 024 that found room, in 16 rows of 16 384 186 and 815.  50 x 3 rows of 26 316
// entries, 20 to take, 17 us, 37 to 296 without the two; 8 rows of 1 024, 64 to take, 18 and 134; they cost the others 0.3.  (With a selection of its own in every slice of 16 384 logits the first kernel had twice the instructions.)  Order
// is decided in 64 bits: sums of fp32 exponentials are good to kNear, so where two rows' candidates are nearer to each other than that, the cluster adds up those rows in 64 bits (half of the entries
// to a CTA) and the CTA picks again.  Entries of one row never need it.
// Bound by the bytes of the logits, and where these are few by latency: 4 rows of 128 256 entries 10.2 us, 32 sequences of up to 5 rows of 32 000 12.9, 512 rows of 128 256 (131 MB) 33.8,
// of which the merge takes some 6; 66 where one sequence has two rows that are near.  Logits through shared memory by asynchronous copies, two or three blocks a warp ahead, are no
// faster (39 to 41 us against 38 then): what is left beside the copy rate's 20 us is the first kernel's start and end.
#include <cooperative_groups.h>

#include <algorithm>

#include "f32x2.cuh"
#include "tc.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kBlockThreads = 256, kBlockGroups = 8, kBlock = 32 * 8 * kBlockGroups, kBlockCtas = 4 * kNumSMs;
constexpr int kMostTake = 128, kMostVocab = 393216;
constexpr int kMergeThreads = 1024, kMergeCtas = 2, kMergeList = kMergeThreads, kKnownRows = 64;
constexpr int kBlocksEach = 3, kSpare = 128;
constexpr float kLog2e = 1.4426950408889634f;
// What a row's log-sum may be off by: exponents of base 2 are rounded once (2^-24 of up to 17 in the mean over the weights, times ln 2: 7e-7) and have log2 e to 2^-26 (2e-7), the
// hardware's exponential has 2^-22 (2.4e-7), for a term and for its block's largest, and nine sums and products follow one another in a lane (5e-7); behind them everything is fp64
constexpr double kNear = 2e-6;

struct RowStat {
  double base, near;   // scores[r] - the log-sum (-inf: no candidates), and how far it may be off (below 0: as far, and asked for in 64 bits)
};

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float max8(const uint4& v) {
  const uint32_t h = max2(max2(v.x, v.y), max2(v.z, v.w));
  return fmaxf(bf16lo(h), bf16hi(h));
}
// numbers in an order that unsigned ones have (zeros alike), and back
__device__ __forceinline__ uint32_t ordered_f32(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float f32_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

// eight logits from entry i0 on, of which some lie outside the row (-inf), entry by entry, all asked for at once (one after another: 57 x 2 rows of 571 entries 19.8 us, 15.1 so)
__device__ __forceinline__ uint4 load_edge(const __nv_bfloat16* l, int i0, int vocab) {
  uint32_t e[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) e[q] = i0 + q >= 0 && i0 + q < vocab ? __bfloat16_as_ushort(l[i0 + q]) : 0xff80u;
  return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}
// a lane's eight groups of eight logits of a row's block (-inf outside the row); groups start at 16-byte addresses: entry i of a row is at place i + shift.  Returns the first one's index
__device__ __forceinline__ int load_block(const __nv_bfloat16* l, int block, int vocab, uint4 (&v)[kBlockGroups]) {
  const int shift = (int)((reinterpret_cast<uintptr_t>(l) >> 1) & 7), p0 = block * kBlock + (threadIdx.x & 31) * 8 - shift;
  if (block * kBlock >= shift && (block + 1) * kBlock - shift <= vocab) {
    const __nv_bfloat16* at = l + p0;
#pragma unroll
    for (int j = 0; j < kBlockGroups; ++j) v[j] = ld_stream(at + j * 256);
    return p0;
  }
  // groups that cross the row's start (the first lane's first) or its end
  const int lane = threadIdx.x & 31, place = vocab + shift, at = (place >> 3) - block * (kBlock / 8), end = (place & 7) && at >= 0 && at < kBlock / 8 && (at & 31) == lane ? at >> 5 : -1;
  const bool start = block == 0 && lane == 0 && shift;
  const int g = start ? 0 : end;
  uint4 w = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  if (g >= 0) w = load_edge(l, p0 + g * 256, vocab);
#pragma unroll
  for (int j = 0; j < kBlockGroups; ++j) {
    const int i = p0 + j * 256;
    v[j] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    if (i >= 0 && i + 8 <= vocab) v[j] = ld_stream(l + i);
    else if (j == g) v[j] = w;
  }
  if (start && end > 0) {
    w = load_edge(l, p0 + end * 256, vocab);
#pragma unroll
    for (int j = 0; j < kBlockGroups; ++j)
      if (j == end) v[j] = w;
  }
  return p0;
}

// stats [row][block]: the largest logit, the sum of exp(x - it)
__global__ void __launch_bounds__(kBlockThreads, 4)
beam_blocks_kernel(const __nv_bfloat16* __restrict__ logits, int64_t ld, int n_rows, int per_row, int vocab, float2* __restrict__ stats) {
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
  for (int b = warp * gridDim.x + blockIdx.x; b < n_rows * per_row; b += kBlockThreads / 32 * gridDim.x) {
    const int row = b / per_row;
    uint4 v[kBlockGroups];
    load_block(logits + (int64_t)row * ld, b - row * per_row, vocab, v);
    uint32_t h = 0xff80ff80u;
#pragma unroll
    for (int j = 0; j < kBlockGroups; ++j) h = max2(h, max2(max2(v[j].x, v[j].y), max2(v[j].z, v[j].w)));
    const float m = warp_max_redux(fmaxf(bf16lo(h), bf16hi(h)));
    // exp(x - m) as 2^(a x - c) with c = a m rounded: the exponents' own rounding apart, all terms are off by one factor, 2^(c - a m), by which the sum is multiplied.  Far from zero,
    // where it might be large, neighbouring bf16 values are so far apart that any a tells them from the largest: a = 1
    const bool far = fabsf(m) >= 65536.f;
    const float a = far ? 1.f : kLog2e, c = m > -INFINITY ? a * m : 0.f;
    const uint64_t a2 = f2::both(a), c2 = f2::both(-c);
    uint64_t part[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kBlockGroups; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint64_t t = f2::fma(f2::pack(bf16lo(w[q]), bf16hi(w[q])), a2, c2);
        part[q] = f2::add(part[q], f2::pack(tc::exp2_fast(f2::lo(t)), tc::exp2_fast(f2::hi(t))));
      }
    }
    double s = (double)f2::sum(f2::add(f2::add(part[0], part[1]), f2::add(part[2], part[3])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) stats[b] = make_float2(m, (float)(far || !(m > -INFINITY) ? s : s * (double)tc::exp2_fast(fmaf(-a, m, c))));
  }
}

// scores as unsigned numbers in their order (compares of 64-bit integers; fp64's have several times the latency), zeros alike, and back
__device__ __forceinline__ uint64_t ordered_f64(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x == 0.0 ? 0.0 : x);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double f64_of_ordered(uint64_t o) { return __longlong_as_double((long long)(o & 0x8000000000000000ull ? o ^ 0x8000000000000000ull : ~o)); }
struct Best {
  uint64_t score, id;
};
// what decides between scores that are alike: the lower row; within a row (where a log-sum may be large beside the logits) the larger logit, the lower entry
__device__ __forceinline__ uint64_t id_of(int row, float x, int entry) { return (uint64_t)row << 48 | (uint64_t)(0xffffu - (ordered_f32(x) >> 16)) << 32 | (uint32_t)entry; }
__device__ __forceinline__ int row_of(uint64_t id) { return (int)(id >> 48); }
__device__ __forceinline__ bool better(const Best& a, const Best& b) { return a.score > b.score || (a.score == b.score && a.id < b.id); }

// Sums of exp(x - m) in units of 2^-62, high and low 32 bits of the terms apart: exact whatever the order, so that rows of the same entries in other places stay alike (fp64 sums differ in
// their last bit).  Units of 393 216 terms make 9e-14
struct alignas(16) UnitSum {
  unsigned long long high, low;
};
__device__ __forceinline__ void operator+=(UnitSum& a, const UnitSum& b) { a.high += b.high, a.low += b.low; }
__device__ __forceinline__ double value_of(const UnitSum& a) { return (double)a.high * 0x1p-30 + (double)a.low * 0x1p-62; }
// exp(d), d <= 0, in these units (0 below 2^-64): d = n ln 2 / 16 + r ln 2 / 16, |r| <= 1 / 2, 2^(n / 16) by its whole part and a table, 2^(r / 16) by its series up to the sixth power (5e-16
// of it).  Conversions, which the hardware has at a quarter of its fp64 rate or less, are left out: n stands in the low word of a sum, the units are the shifted bits
__constant__ double kSixteenths[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
                                       1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
                                       1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
                                       1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};
__device__ __forceinline__ unsigned long long units_of(double d, const double* table) {
  if (!(d >= -45.0)) return 0;
  constexpr double kScale = 23.083120654223414, kShift = 0x1.8p52;   // 16 / ln 2
  const double k = fma(d, kScale, kShift), r = fma(d, kScale, kShift - k);
  const int n = __double2loint(k);
  double e = 9.181219573844438e-12;   // (ln 2 / 16)^6 / 6!, and so on
  e = fma(e, r, 1.2715871950558131e-09), e = fma(e, r, 1.467610032291943e-07), e = fma(e, r, 1.3550807779497457e-05), e = fma(e, r, 0.0009383847928089872), e = fma(e, r, 0.04332169878499658);
  e = fma(e, r, 1.0) * table[n & 15];
  const int shift = (__double2hiint(e) >> 20) - 1023 + (n >> 4) + 10;   // 2^62 = 2^52 x 2^10
  const unsigned long long bits = ((unsigned long long)__double_as_longlong(e) & 0xfffffffffffffull) | 0x10000000000000ull;
  return shift >= 0 ? bits << shift : bits >> -shift;
}
// bf16 bits as fp64 (below the normal numbers: 0, next to which they are nothing in an exponent)
__device__ __forceinline__ double f64_of(uint32_t b) {
  return (b & 0x7fffu) < 0x80u ? 0.0 : __hiloint2double((int)((b & 0x8000u) << 16 | (((b & 0x7fffu) << 13) + (896u << 20))), 0);
}
// What a CTA's share of a row's entries has (of eight at a 16-byte address, four such loads at once); of a row with numbers that are none: anything.  bf16 has 4096 values from 2^-8 up to
// 2^8: those are counted, and what each has goes into the sum as often (an exponential for every entry takes 80 issue slots of a warp); the few that are nearer to zero, or
// further from it, by themselves
constexpr uint32_t kCountFrom = (127 - 8) << 7, kCounted = 16 << 7;   // of either sign
__device__ __noinline__ UnitSum row_part(const __nv_bfloat16* l, int vocab, int cta, double m, const double* table, uint32_t* counts) {
  const int shift = (int)((reinterpret_cast<uintptr_t>(l) >> 1) & 7), groups = (vocab + shift + 7) / 8;
  const int from = (int)((int64_t)groups * cta / kMergeCtas), to = (int)((int64_t)groups * (cta + 1) / kMergeCtas);
  UnitSum sum = {0, 0};
  for (int i = threadIdx.x; i < 2 * (int)kCounted; i += kMergeThreads) counts[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int g0 = from + threadIdx.x; g0 < to; g0 += 4 * kMergeThreads) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int g = g0 + j * kMergeThreads, i = g * 8 - shift;
      v[j] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
      if (g < to) {
        if (i >= 0 && i + 8 <= vocab) v[j] = ld_stream(l + i);
        else v[j] = load_edge(l, i, vocab);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll 1
      for (int q = 0; q < 8; ++q) {
        const uint32_t x = v[j].x & 0xffffu, at = (x & 0x7fffu) - kCountFrom;
        v[j].x = __funnelshift_r(v[j].x, v[j].y, 16), v[j].y = __funnelshift_r(v[j].y, v[j].z, 16), v[j].z = __funnelshift_r(v[j].z, v[j].w, 16), v[j].w >>= 16;
        if (at < kCounted) {
          atomicAdd(counts + (x >> 15) * kCounted + at, 1u);
        } else if (x != 0xff80u) {
          const unsigned long long t = units_of(f64_of(x) - m, table);
          sum += {t >> 32, t & 0xffffffffu};
        }
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < 2 * kCounted; i += kMergeThreads) {
    const unsigned long long n = counts[i];
    if (n == 0) continue;
    const unsigned long long t = units_of(f64_of(i < kCounted ? i + kCountFrom : 0x8000u | (i - kCounted + kCountFrom)) - m, table);
    sum += {n * (t >> 32), n * (t & 0xffffffffu)};
  }
  __syncthreads();   // (before they are counted again)
  return sum;
}
__device__ __noinline__ double row_base(const float* scores, int r, double m, double sum) {
  const double base = (scores ? (double)scores[r] : 0.0) - (m + log(sum));
  return base - base == 0.0 ? base : -INFINITY;
}
// Limits: a number that more than `take` scores reach, and not many more, as fp32 (rounded down); -inf: there are no more than `take`.  Scores are counted by their distance from the
// largest, in steps of a sixteenth of a power of two; the number is the far end of the step in which the count passes `take` (by halves, with a barrier for each, this took 3 000
// cycles)
constexpr int kSteps = 512;
constexpr uint32_t kFirstStep = __builtin_bit_cast(uint32_t, 0x1p-23f) >> 19;
__device__ __forceinline__ int at_step(int k) { return k + k / (kSteps / 32); }   // (no bank conflicts)
__device__ __forceinline__ void count_step(int* steps, float most, float top, int n = 1) {
  const uint32_t far = __float_as_uint(most - top) >> 19;   // (by a sixteenth of a power of two each)
  atomicAdd(&steps[at_step(far < kFirstStep ? 0 : min(far - kFirstStep + 1, kSteps - 1u))], n);
}
__device__ __forceinline__ float far_end(const int* steps, float most, int take) {
  const int lane = threadIdx.x & 31;
  auto scan = [&](int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    return x;
  };
  int count = 0;   // a lane's kSteps / 32, then of one lane's
#pragma unroll
  for (int k = 0; k < kSteps / 32; ++k) count += steps[at_step(lane * (kSteps / 32) + k)];
  const int until = scan(count);
  const uint32_t past = __ballot_sync(0xffffffffu, until > take);
  if (!past) return -INFINITY;
  const int owner = __ffs(past) - 1, before = __shfl_sync(0xffffffffu, until - count, owner);
  const int within = scan(lane < kSteps / 32 ? steps[at_step(owner * (kSteps / 32) + lane)] : 0);
  const int step = owner * (kSteps / 32) + __ffs(__ballot_sync(0xffffffffu, before + within > take)) - 1;
  if (step == kSteps - 1) return f32_of(ordered_f32(-INFINITY) + 1);   // (the last one has no end)
  const float end = most - __uint_as_float((kFirstStep + step) << 19);
  return end - (fabsf(most) + fabsf(end)) * 0x1p-22f;   // (distances are rounded)
}
// Limits from the blocks' entries: where there are few blocks for those to take, of the largest entries of groups of eight; where more entries reach the limit than the list holds, of all of
// them (those that found room differ from call to call, and with a limit by them what has to be added up in 64 bits)
struct Listed {   // blocks whose scores reach `least`
  const __nv_bfloat16* logits;
  const float2* stats;   // of the sequence
  const RowStat* rows;   // of the sequence
  const int* blocks;     // NULL: all n
  int64_t ld;
  int n, per_row, vocab;
  double least;
};
template <bool kAll>
__device__ __noinline__ float limit_of_entries(const Listed& b, const double* known, int* steps, float* warp_tops, int take) {
  constexpr int kWarps = kMergeThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kSteps) steps[at_step(tid)] = 0;
  float most = -INFINITY;
  auto base_of = [&](int r) { return r < kKnownRows ? known[r] : b.rows[r].base; };
  for (int e = tid; e < b.n; e += kMergeThreads) {
    const int k = b.blocks ? b.blocks[e] : e;
    most = fmaxf(most, __double2float_rd(base_of(k / b.per_row) + (double)b.stats[k].x));   // (no number: left out)
  }
  most = warp_max_redux(most);
  if (lane == 0) warp_tops[warp] = most;
  __syncthreads();
  most = warp_max_redux(warp_tops[lane & (kWarps - 1)]);
#pragma unroll 1
  for (int e = warp; e < b.n; e += kWarps) {
    const int k = b.blocks ? b.blocks[e] : e, r = k / b.per_row;
    const double base = base_of(r);
    if (!(base > -INFINITY)) continue;
    uint4 v[kBlockGroups];
    load_block(b.logits + (int64_t)r * b.ld, k - r * b.per_row, b.vocab, v);
    if constexpr (kAll) {
      // neighbours alike, of which there may be thousands, are counted together
      float last = -INFINITY;
      int n = 0;
      auto count = [&] {
        const double score = base + (double)last;
        const float top = __double2float_rd(score);
        if (n > 0 && score >= b.least && top > -INFINITY) count_step(steps, most, top, n);
      };
#pragma unroll 1
      for (int j = 0; j < kBlockGroups; ++j) {
        uint4 w = v[0];
#pragma unroll
        for (int i = 1; i < kBlockGroups; ++i)
          if (i == j) w = v[i];
        if (!(base + (double)max8(w) >= b.least)) continue;
        if (w.x == w.y && w.z == w.w && w.x == w.z && w.x == __funnelshift_l(w.x, w.x, 16)) {
          if (bf16lo(w.x) != last) count(), last = bf16lo(w.x), n = 0;
          n += 8;
          continue;
        }
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
          const float x = bf16lo(w.x);
          w.x = __funnelshift_r(w.x, w.y, 16), w.y = __funnelshift_r(w.y, w.z, 16), w.z = __funnelshift_r(w.z, w.w, 16), w.w >>= 16;
          if (x != last) count(), last = x, n = 0;
          ++n;
        }
      }
      count();
      continue;
    }
#pragma unroll
    for (int j = 0; j < kBlockGroups; ++j) {
      const double score = base + (double)max8(v[j]);
      const float top = __double2float_rd(score);
      if (score >= b.least && top > -INFINITY) count_step(steps, most, top);
    }
  }
  __syncthreads();
  return far_end(steps, most, take);
}
// The same of the first n of the list
__device__ __noinline__ float limit_of_list(const Best* cand, int n, int* steps, float* warp_tops, int take) {
  constexpr int kWarps = kMergeThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kSteps) steps[at_step(tid)] = 0;
  const float top = tid < n ? __double2float_rd(f64_of_ordered(cand[tid].score)) : -INFINITY, wm = warp_max_redux(top);
  if (lane == 0) warp_tops[warp] = wm;
  __syncthreads();
  const float most = warp_max_redux(warp_tops[lane & (kWarps - 1)]);
  if (top > -INFINITY) count_step(steps, most, top);
  __syncthreads();
  return far_end(steps, most, take);
}
__global__ void __launch_bounds__(kMergeThreads, 1) __cluster_dims__(kMergeCtas, 1, 1)
beam_merge_kernel(const __nv_bfloat16* __restrict__ logits, int64_t ld, const float* __restrict__ scores, const int32_t* __restrict__ starts, int n_rows, int per_row, int vocab, int take,
                  const float2* __restrict__ stats, RowStat* rows, UnitSum* parts, int32_t* out_rows, int32_t* out_tokens, float* out_scores) {
  constexpr int kWarps = kMergeThreads / 32;
  __shared__ Best cand[kMergeList];
  __shared__ Best sorted[kMostTake + 1];
  __shared__ float warp_tops[kWarps], block_tops[kMergeList];
  __shared__ int steps[kSteps + 32];
  __shared__ UnitSum sh_part[kWarps];
  __shared__ double sixteenths[16], known[kKnownRows];   // known: bases of the first rows
  __shared__ int need[2 * kMergeList], blocks[kMergeList], n_need, n_list, n_blocks, seen_all, asked;
  __shared__ uint32_t asked_for[kMergeList / 32], exact_rows[kMergeList / 32];   // rows of the sequence that are in need, and that have been added up in 64 bits (of the first kMergeList)
  __shared__ Best limit;
  __shared__ Listed reaching;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (before shared memory of the other CTA is written, it runs)
  pdl_wait();
  const cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), seq = blockIdx.x / kMergeCtas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = min(max(starts[seq], 0), n_rows), r1 = min(max(starts[seq + 1], r0), n_rows), all_blocks = (r1 - r0) * per_row;
  const float2* const mine = stats + (int64_t)r0 * per_row;   // block b of the sequence: of row r0 + b / per_row
  auto top_of = [&](int r) {   // a row's largest logit
    float m = -INFINITY;
#pragma unroll 1
    for (int i = lane; i < per_row; i += 32) m = fmaxf(m, stats[(int64_t)r * per_row + i].x);
    return warp_max(m);
  };
  auto base_of = [&](int r) { return r - r0 < kKnownRows ? known[r - r0] : rows[r].base; };
  auto near_of = [&](int r) { return r - r0 >= kMergeList ? fabs(rows[r].near) : exact_rows[(r - r0) >> 5] >> ((r - r0) & 31) & 1 ? 0.0 : kNear; };
  if (cta == 0) {
    if (tid < kMergeList / 32) exact_rows[tid] = 0;
    // log-sums of the rows; the first kHeld x 32 blocks of a row stay in registers between the maximum and the sum
    constexpr int kHeld = 4;
#pragma unroll 1
    for (int r = r0 + warp; r < r1; r += kWarps) {
      const float2* st = stats + (int64_t)r * per_row;
      float2 held[kHeld];
#pragma unroll
      for (int j = 0; j < kHeld; ++j) held[j] = 32 * j + lane < per_row ? st[32 * j + lane] : make_float2(-INFINITY, 0.f);
      float m = fmaxf(fmaxf(held[0].x, held[1].x), fmaxf(held[2].x, held[3].x));
#pragma unroll 1
      for (int i = 32 * kHeld + lane; i < per_row; i += 32) m = fmaxf(m, st[i].x);
      m = warp_max_redux(m);
      double s = 0.0;
      auto add = [&](const float2& t) { s += (double)t.y * (double)tc::exp2_fast((t.x - m) * kLog2e); };   // (both -inf: no number, as the sum of a row that has none)
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (32 * j + lane < per_row) add(held[j]);
#pragma unroll 1
      for (int i = 32 * kHeld + lane; i < per_row; i += 32) add(st[i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) {
        const double base = row_base(scores, r, (double)m, s);
        rows[r] = {base, kNear};
        if (r - r0 < kKnownRows) known[r - r0] = base;
      }
    }
    __syncthreads();
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  bool exact = false;   // every row added up in 64 bits
#pragma unroll 1
  for (;;) {
    if (cta == 0) {
      double margin = exact ? 0.0 : 2 * kNear;
      auto limit_of = [&](double best) {
        const float top = __double2float_rd(best), wm = warp_max_redux(top);
        __syncthreads();
        if (lane == 0) warp_tops[warp] = wm;
        if (tid < kSteps) steps[at_step(tid)] = 0;
        __syncthreads();
        const float most = warp_max_redux(warp_tops[lane & (kWarps - 1)]);
        if (top > -INFINITY) count_step(steps, most, top);
        __syncthreads();
        return far_end(steps, most, take);
      };
      // blocks by their largest entry
      if (tid == 0) n_list = 0, n_need = 0, n_blocks = 0, seen_all = 1;
      if (tid < kMergeList / 32) asked_for[tid] = 0;
      auto block_score = [&](int b, float& x) {
        x = mine[b].x;
        return base_of(r0 + b / per_row) + (double)x;
      };
      double best = -INFINITY, last_score = -INFINITY;
      float last_top = -INFINITY;
#pragma unroll 1
      for (int b = tid; b < all_blocks; b += kMergeThreads) {
        last_score = block_score(b, last_top);
        if (last_score > best) best = last_score;
      }
      Best at = {ordered_f64((double)limit_of(best)), ~0ull};
      const double lowest = f64_of_ordered(at.score) - margin;
#pragma unroll 1
      for (int b = tid; b < all_blocks; b += kMergeThreads) {
        float x = last_top;
        const double t = all_blocks <= kMergeThreads ? last_score : block_score(b, x);
        if (t > -INFINITY && t >= lowest) {
          const int k = atomicAdd(&n_blocks, 1);
          if (k < kMergeList) blocks[k] = b, block_tops[k] = x;
        }
      }
      __syncthreads();
      const int listed = n_blocks;
      // a warp looks through a block: f(score, id) for its entries whose score is `least` or more
      auto each = [&](double least, auto f) {
#pragma unroll 1
        for (int e = warp; e < (listed <= kMergeList ? listed : all_blocks); e += kWarps) {
          const int b = listed <= kMergeList ? blocks[e] : e, r = r0 + b / per_row;
          const double base = base_of(r);
          const float x0 = __double2float_rd(least - base - fabs(base) * 0x1p-50);   // (in the logits' own terms; where the sum is rounded to fp64, a little less)
          if (!(base > -INFINITY) || !((listed <= kMergeList ? block_tops[e] : mine[b].x) >= x0)) continue;
          uint4 v[kBlockGroups];
          const int p0 = load_block(logits + (int64_t)r * ld, b - (r - r0) * per_row, vocab, v);
          uint32_t hot = 0;
#pragma unroll
          for (int j = 0; j < kBlockGroups; ++j) hot |= (max8(v[j]) >= x0 ? 1u : 0u) << j;
#pragma unroll 1
          for (; hot; hot &= hot - 1) {   // (few lanes have one)
            const int g = __ffs(hot) - 1;
            uint4 w = v[0];
#pragma unroll
            for (int j = 1; j < kBlockGroups; ++j)
              if (j == g) w = v[j];
#pragma unroll 1
            for (int i = p0 + g * 256, end = i + 8; i < end; ++i) {   // (outside the row: -inf)
              const float x = bf16lo(w.x);
              w.x = __funnelshift_r(w.x, w.y, 16), w.y = __funnelshift_r(w.y, w.z, 16), w.z = __funnelshift_r(w.z, w.w, 16), w.w >>= 16;
              if (!(x >= x0 && x > -INFINITY)) continue;
              const double t = base + (double)x;
              if (t >= least) f(Best{ordered_f64(t), id_of(r, x, i)});
            }
          }
        }
      };
      // f(entry, its place) for the first n of the list: a warp an entry
      auto each_place = [&](int n, auto f) {
#pragma unroll 1
        for (int e = warp; e < n; e += kWarps) {
          const Best x = cand[e];
          int before = 0;
#pragma unroll 1
          for (int k = lane; k < n; k += 32) before += better(cand[k], x);
          before = __reduce_add_sync(0xffffffffu, before);
          if (lane == 0) f(x, before);
        }
      };
      // a limit by the entries of the blocks that reach this one
      auto look = [&](auto limit_of_those) {
        if (tid == 0)
          reaching = {logits + (int64_t)r0 * ld, mine, rows + r0, listed <= kMergeList ? blocks : nullptr, ld, listed <= kMergeList ? listed : all_blocks, per_row, vocab,
                      f64_of_ordered(at.score) - margin};
        __syncthreads();
        const uint64_t reached = ordered_f64((double)limit_of_those(reaching, known, steps, warp_tops, take));
        __syncthreads();
        return reached;
      };
      if (all_blocks < kBlocksEach * take || !(f64_of_ordered(at.score) > -INFINITY)) at.score = max(at.score, look(limit_of_entries<false>));
      bool too_many = false, closer = false;
#pragma unroll 1
      for (;;) {
        if (too_many) {
          Best own = {0, ~0ull - tid};   // (with none: behind all others, and no two alike)
          each(f64_of_ordered(at.score) - margin, [&](const Best& x) {
            if (better(x, own) && !better(at, x)) own = x;
          });
          // the entry behind the best `take` threads' own is a limit nearer to the end (of 64 rows of 128 256 entries alike, the best rows last, the list would leave out a thousand at a
          // time).  It leaves take + 1 threads with any: then it is the one behind the best `take` of those that found room, which leaves out all but `take` of them.  Either way
          // fewer are left
          if (__syncthreads_count(own.score > 0) > take + 1) cand[tid] = own;
          __syncthreads();
          each_place(kMergeList, [&](const Best& x, int place) {
            if (place == take) limit = x;
          });
          __syncthreads();
          at = limit;
        }
        each(f64_of_ordered(at.score) - margin, [&](const Best& x) {
          if (margin > 0.0 || !better(at, x)) {
            const int k = atomicAdd(&n_list, 1);
            if (k < kMergeList) cand[k] = x;
          }
        });
        __syncthreads();
        const int found = n_list;
        if (found <= take + kSpare) break;
        if (!closer) {   // a limit by these: ranks take as long as the square of their number
          closer = true;
          const uint64_t reached = found > kMergeList ? look(limit_of_entries<true>) : ordered_f64((double)limit_of_list(cand, found, steps, warp_tops, take));
          if (reached > at.score) {
            at.score = reached;
            const Best x = cand[tid];
            __syncthreads();
            if (tid == 0) n_list = 0;
            __syncthreads();
            if (found > kMergeList) continue;   // from the blocks again
            if (tid < found && f64_of_ordered(x.score) >= f64_of_ordered(reached) - margin) cand[atomicAdd(&n_list, 1)] = x;
            __syncthreads();
            break;
          }
        }
        if (found <= kMergeList) break;
        __syncthreads();
        if (tid == 0) n_list = 0, seen_all = margin == 0.0 && seen_all;   // (those next to the limit will not all be seen)
        margin = 0.0;
        too_many = true;
        __syncthreads();
      }
      const int n = n_list;
      each_place(n, [&](const Best& x, int place) {
        if (place <= take) sorted[place] = x;
      });
      __syncthreads();
      if (!exact) {
        // candidates of two rows that are nearer to each other than their sums are good for: neighbours among those taken, and the last of them and whatever comes behind
#pragma unroll 1
        for (int e = tid; e < take + n; e += kMergeThreads) {
          const int k = e < take ? e : take - 1;
          if (k >= n || (e < take && e + 1 >= n)) continue;
          const Best x = sorted[k], y = e < take ? sorted[e + 1] : cand[e - take];
          const int ra = row_of(x.id), rb = row_of(y.id);
          if (ra == rb || !better(x, y)) continue;
          const double na = near_of(ra), nb = near_of(rb);
          if (na + nb > 0.0 && f64_of_ordered(x.score) - f64_of_ordered(y.score) <= na + nb) {
#pragma unroll 1
            for (int side = 0; side < 2; ++side) {
              const int r = side ? rb : ra;
              if (!((side ? nb : na) > 0.0)) continue;
              const uint32_t bit = 1u << ((r - r0) & 31);
              if (r - r0 < kMergeList) {
                if (atomicOr(&asked_for[(r - r0) >> 5], bit) & bit) continue;
              } else if (__longlong_as_double((long long)atomicExch(reinterpret_cast<unsigned long long*>(&rows[r].near), (unsigned long long)__double_as_longlong(-kNear))) < 0.0) {
                continue;
              }
              need[atomicAdd(&n_need, 1)] = r;   // (two for each of n entries at most)
            }
          }
        }
        __syncthreads();
      }
      const bool all_rows = !exact && !seen_all;
      const int wanted = exact ? 0 : all_rows ? -1 : n_need;
      if (wanted == 0) {
#pragma unroll 1
        for (int k = tid; k < take; k += kMergeThreads) {
          const int64_t to = (int64_t)seq * take + k;
          const Best x = k < n ? sorted[k] : Best{0, 0};
          out_rows[to] = k < n ? row_of(x.id) : -1;
          out_tokens[to] = k < n ? (int)(uint32_t)x.id : -1;
          out_scores[to] = k < n ? (float)f64_of_ordered(x.score) : -INFINITY;
        }
      }
      if (tid < kMergeCtas) *cluster.map_shared_rank(&asked, tid) = wanted;
      exact = exact || all_rows;
    }
    cluster.sync();   // the other CTAs have waited here: their help is asked for where `asked` is not 0 (-1: all rows)
    if (asked == 0) return;
    const int wanted = asked < 0 ? r1 - r0 : asked;
    const int* list = cluster.map_shared_rank(need, 0);
    static_assert(sizeof(cand) == 8 * kCounted, "counts of a row's values lie where the list was");
    uint32_t* const counts = reinterpret_cast<uint32_t*>(cand);
    auto wanted_row = [&](int i) { return asked < 0 ? r0 + i : list[i]; };
    if (tid < 16) sixteenths[tid] = kSixteenths[tid];
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < wanted; ++i) {
      const int r = wanted_row(i);
      UnitSum sum = row_part(logits + (int64_t)r * ld, vocab, cta, (double)top_of(r), sixteenths, counts);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += {__shfl_xor_sync(0xffffffffu, sum.high, o), __shfl_xor_sync(0xffffffffu, sum.low, o)};
      __syncthreads();
      if (lane == 0) sh_part[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) sum += sh_part[w];
        parts[(int64_t)r * kMergeCtas + cta] = sum;
      }
    }
    __threadfence();
    cluster.sync();   // (and nobody goes on while another one reads its list)
    if (cta == 0) {
#pragma unroll 1
      for (int i = warp; i < wanted; i += kWarps) {
        const int r = wanted_row(i);
        const float m = top_of(r);
        if (lane == 0) {
          UnitSum sum = {0, 0};
          for (int k = 0; k < kMergeCtas; ++k) {
            const ulonglong2 t = __ldcg(reinterpret_cast<const ulonglong2*>(parts) + (int64_t)r * kMergeCtas + k);
            sum += {t.x, t.y};
          }
          const double base = rows[r].base > -INFINITY ? row_base(scores, r, (double)m, value_of(sum)) : -INFINITY;   // (a row that is none stays none)
          rows[r] = {base, 0.0};
          if (r - r0 < kKnownRows) known[r - r0] = base;
          if (r - r0 < kMergeList) atomicOr(&exact_rows[(r - r0) >> 5], 1u << ((r - r0) & 31));
        }
      }
      __syncthreads();
    }
  }
}

int per_row_of(int vocab) { return (vocab + 7 + kBlock - 1) / kBlock; }   // blocks, of places from a 16-byte address on: up to seven more than entries

}  // namespace

int64_t beam_select_workspace_bytes(int n_rows, int vocab) {
  return (int64_t)n_rows * (per_row_of(vocab) * (int64_t)sizeof(float2) + (int64_t)sizeof(RowStat) + kMergeCtas * (int64_t)sizeof(UnitSum)) + 64;
}

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_beam_select_workspace_bytes(int32_t n_rows, int32_t vocab, int32_t n_select) {
  return n_rows > 0 && vocab > 0 && n_select > 0 ? beam_select_workspace_bytes(n_rows, vocab) : 0;
}
extern "C" int b200_beam_select(const void* logits, int64_t ld, const float* scores, const int32_t* row_starts, int32_t n_seqs, int32_t n_rows, int32_t vocab,
                                int32_t n_select, int32_t* out_rows, int32_t* out_tokens, float* out_scores, void* ws, int64_t ws_bytes, void* stream) {
  B200_REQUIRE(logits && row_starts && out_rows && out_tokens && out_scores, B200_ERR_INVALID, "beam_select: null");
  B200_REQUIRE(n_seqs >= 0 && n_rows >= 0 && vocab > 0 && ld >= vocab && n_select > 0, B200_ERR_INVALID, "beam_select: %d sequences, %d rows of %d entries, ld=%lld, %d to select",
               n_seqs, n_rows, vocab, (long long)ld, n_select);
  B200_REQUIRE(vocab <= kMostVocab, B200_ERR_UNSUPPORTED, "beam_select: vocab=%d (at most %d)", vocab, kMostVocab);
  B200_REQUIRE(n_select <= kMostTake, B200_ERR_UNSUPPORTED, "beam_select: %d to select (at most %d)", n_select, kMostTake);
  B200_REQUIRE(n_rows <= 65535, B200_ERR_UNSUPPORTED, "beam_select: %d rows (at most 65535)", n_rows);
  B200_REQUIRE(n_seqs < 1 << 28, B200_ERR_UNSUPPORTED, "beam_select: %d sequences (at most 2^28 - 1)", n_seqs);
  if (n_seqs == 0) return B200_OK;
  const int64_t need = n_rows > 0 ? beam_select_workspace_bytes(n_rows, vocab) : 0;
  B200_REQUIRE(need == 0 || (ws && (reinterpret_cast<uintptr_t>(ws) & 15) == 0 && ws_bytes >= need), B200_ERR_INVALID,
               "beam_select: the workspace is 16-byte aligned and has at least %lld bytes (%lld)", (long long)need, (long long)ws_bytes);
  B200_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 1) == 0, B200_ERR_INVALID, "beam_select: logits must be 2-byte aligned");
  const cudaStream_t s = (cudaStream_t)stream;
  const __nv_bfloat16* l = static_cast<const __nv_bfloat16*>(logits);
  const int per_row = per_row_of(vocab);
  RowStat* rows = static_cast<RowStat*>(ws);
  UnitSum* parts = reinterpret_cast<UnitSum*>(rows + n_rows);
  float2* stats = reinterpret_cast<float2*>(parts + (int64_t)n_rows * kMergeCtas);
  if (n_rows > 0)
    B200_CUDA(launch(beam_blocks_kernel, dim3((unsigned)std::min(kBlockCtas, n_rows * per_row)), dim3(kBlockThreads), (size_t)0, s, l, ld, n_rows, per_row, vocab, stats));
  const PdlScope merge(n_rows > 0);
  B200_CUDA(launch(beam_merge_kernel, dim3((unsigned)(n_seqs * kMergeCtas)), dim3(kMergeThreads), (size_t)0, s, l, ld, scores, row_starts, n_rows, per_row, vocab, n_select, stats, rows,
                   parts, out_rows, out_tokens, out_scores));
  return B200_OK;
}
