// A beam search's selection over beams and vocabulary (b200_beam_select), two launches.
//
// score(r, i) = scores[r] + x_ri - log sum_j exp x_rj; a sequence takes the K largest of its rows and all their entries, ties by row, then by entry.
// slices: a CTA takes a slice of a row, all of it in registers at once: its largest logit m, the sum of exp(x - m) and its own K largest entries.  A thread's largest
// entry is compared first: any number that K threads' largest reach is a limit that the slice's K largest reach too, and it leaves little more than K entries, which
// are then counted against each other.
// merge: a cluster takes a sequence; every CTA of it joins the slices' sums and picks the K best of the slices' candidates in the same way.  Order is decided in 64 bits:
// sums of fp32 exponentials are good to kNear, so where two rows' candidates are nearer to each other than that, the cluster adds up those rows in fp64 (an eighth of the
// entries to a CTA) and picks again.  Entries of one row never need it.
// Bound by the bytes of the logits.
#include <cooperative_groups.h>

#include <algorithm>

#include "f32x2.cuh"
#include "tc.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kSliceThreads = 256, kMostGroups = 8, kLeastSlice = kSliceThreads * 8, kMostSlice = kLeastSlice * kMostGroups;
constexpr int kMostTake = 128, kMostVocab = 393216, kFewCtas = 8 * kNumSMs, kSliceList = 512;
constexpr int kMergeThreads = 256, kMergeCtas = 8, kMergeList = 1024;
// What a row's log-sum may be off by: exponents are rounded once (2^-24 of up to 20 in the mean over the weights, in units of log2e), the hardware's exponential has
// 2^-22, sixteen sums of 2^-24 follow one another in a thread; behind it everything is fp64
constexpr double kNear = 2e-6;

struct alignas(16) SliceStat {
  double sum;
  float m;
  int pad;
};
struct RowStat {
  double base, near;   // scores[r] - the log-sum (-inf: no candidates), and how far it may be off
};

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// fp32 bits of a bf16 in an order that unsigned numbers have (zeros alike), and back; -inf is kNoEntry
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) >> 16;
}
__device__ __forceinline__ float entry_of(uint32_t o) {
  const uint32_t b = o & 0x8000u ? o ^ 0x8000u : ~o & 0xffffu;
  return __uint_as_float(b << 16);
}
constexpr uint32_t kNoEntry = 0x007fu;   // ordered(-inf)

// 0xffff in the halves of x that reach (are above) y's
__device__ __forceinline__ uint32_t reach(uint32_t x, uint32_t y) {
  return __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
}

// candidates [row][slice][take]: an entry's index (-1: none) and its logit
template <int J>
__global__ void __launch_bounds__(kSliceThreads, J == 8 ? 4 : 6)
beam_slices_kernel(const __nv_bfloat16* __restrict__ logits, int64_t ld, const int32_t* __restrict__ starts, int n_seqs, int n_slices, int vocab, int take,
                   SliceStat* __restrict__ stats, int2* __restrict__ cands) {
  constexpr int kWarps = kSliceThreads / 32, kWords = 4 * J, kSets = (kWords + 15) / 16;
  __shared__ float sh_m[kWarps];
  __shared__ double sh_s[kWarps];
  __shared__ int count, sum_of[2];
  __shared__ uint2 list[kSliceList];   // ordered entry, index
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slice = blockIdx.x % n_slices, row = blockIdx.x / n_slices;
  const __nv_bfloat16* l = logits + (int64_t)row * ld;
  const int shift = (int)((reinterpret_cast<uintptr_t>(l) >> 1) & 7);   // groups of eight start at 16-byte addresses: entry i is at place i + shift
  uint4 v[J];
  const int p0 = slice * (kLeastSlice * J) + tid * 8 - shift;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = p0 + j * kLeastSlice;
    v[j] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    if (i >= 0 && i + 8 <= vocab) v[j] = ld_stream(l + i);
  }
  const bool none = row < __ldg(starts) || row >= __ldg(starts + n_seqs);
  // a group that crosses the row's ends: the first one's, or the last one's (a thread has one of them at most, or the one that is both)
  const int last = (vocab - 1 - p0) / kLeastSlice;
  const bool head = p0 < 0 && p0 + 8 > 0, tail = vocab - 1 >= p0 && last < J && p0 + last * kLeastSlice + 8 > vocab;
  if (head || tail) {
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      const int g = side ? last : 0;
      if (side ? !tail || (head && last == 0) : !head) continue;
      uint32_t w[4] = {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = p0 + g * kLeastSlice + k;
        if (i >= 0 && i < vocab) w[k >> 1] = k & 1 ? (w[k >> 1] & 0xffffu) | (uint32_t)__bfloat16_as_ushort(l[i]) << 16 : (w[k >> 1] & 0xffff0000u) | __bfloat16_as_ushort(l[i]);
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j == g) v[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (none) return;
  uint32_t h = 0xff80ff80u;
#pragma unroll
  for (int j = 0; j < J; ++j) h = max2(h, max2(max2(v[j].x, v[j].y), max2(v[j].z, v[j].w)));
  const float mine = fmaxf(bf16lo(h), bf16hi(h));
  const float wm = warp_max_redux(mine);
  if (lane == 0) sh_m[warp] = wm;
  if (tid == 0) count = 0;
  __syncthreads();
  float m = sh_m[lane & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  // exp(x - m) = 2^((x - m) log2 e): the difference is exact, or rounded once
  const uint64_t minus = f2::both(m > -INFINITY ? -m : 0.f), log2e = f2::both(1.4426950408889634f);
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t t = f2::mul(f2::add(f2::pack(bf16lo(w[k]), bf16hi(w[k])), minus), log2e);
      sum[k & 1] = f2::add(sum[k & 1], f2::pack(tc::exp2_fast(f2::lo(t)), tc::exp2_fast(f2::hi(t))));
    }
  }
  double s = ((double)f2::lo(sum[0]) + (double)f2::hi(sum[0])) + ((double)f2::lo(sum[1]) + (double)f2::hi(sum[1]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh_s[warp] = s;
  // a limit that at least `take` threads' largest entries reach, and few more (all entries: too few threads have any)
  const uint32_t key = ordered(mine);
  uint32_t limit = kNoEntry + 1, top = ordered(m);   // top: too few reach a number above it
  const int enough = __syncthreads_count(key >= limit);
  if (tid == 0) {
    double all = sh_s[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) all += sh_s[w];
    stats[blockIdx.x] = {all, m, 0};
  }
  if (enough > take) {
    uint32_t low = limit;
    int got = enough;
    while (low < top && got > take + (take >> 2) + 4) {
      const uint32_t mid = (low + top + 1) >> 1;
      const int n = __syncthreads_count(key >= mid);
      if (n >= take) low = mid, got = n;
      else top = mid - 1;
    }
    limit = low;
  }
  // the entries that reach a number, as bits: 16 words to a set, the word's lower half in bit k, its upper half in bit 16 + k
  auto reaching = [&](uint32_t least, uint32_t (&bits)[kSets]) {
    const uint32_t y = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(entry_of(least))) * 0x10001u;
#pragma unroll
    for (int q = 0; q < kSets; ++q) bits[q] = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) bits[(4 * j + k) / 16] |= reach(w[k], y) & (0x10001u << ((4 * j + k) & 15));
    }
  };
  auto index_of = [&](int q, int b) {   // of bit b of set q
    const int word = 16 * q + (b & 15);
    return p0 + (word >> 2) * kLeastSlice + 2 * (word & 3) + (b >> 4);
  };
  // entries that reach `least`, those at it up to an index -> the list
  auto collect = [&](uint32_t least, int most_index) {
    if (key >= least) {
      uint32_t bits[kSets];
      reaching(least, bits);
#pragma unroll
      for (int q = 0; q < kSets; ++q)
#pragma unroll 1
        for (uint32_t rest = bits[q]; rest; rest &= rest - 1) {
          const int i = index_of(q, __ffs(rest) - 1);
          const uint32_t x = ordered(__bfloat162float(l[i]));
          if (x > least || i <= most_index) {
            const int at = atomicAdd(&count, 1);
            if (at < kSliceList) list[at] = make_uint2(x, (uint32_t)i);
          }
        }
    }
    __syncthreads();
  };
  int from = 0x7fffffff;
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    collect(limit, from);
    if (pass || count <= kSliceList) break;
    // many entries to a thread, or alike: the exact limit, and the index up to which entries at it count, bit by bit
    auto total = [&](uint32_t least, int most_index) {
      uint32_t bits[kSets], above[kSets];
      reaching(least, bits);
      reaching(least + 1, above);
      int c = 0;
#pragma unroll
      for (int q = 0; q < kSets; ++q) {
        c += __popc(above[q]);
#pragma unroll 1
        for (uint32_t rest = bits[q] & ~above[q]; rest; rest &= rest - 1) c += index_of(q, __ffs(rest) - 1) <= most_index;
      }
      c = __reduce_add_sync(0xffffffffu, c);
      __syncthreads();
      if (tid == 0) sum_of[0] = 0;
      __syncthreads();
      if (lane == 0) atomicAdd(&sum_of[0], c);
      __syncthreads();
      return sum_of[0];
    };
    uint32_t low = limit, high = ordered(m);
    int to = vocab;
    from = 0;   // the smallest index that is enough
#pragma unroll 1
    while (low < high || from < to) {
      const bool keys = low < high;
      const uint32_t mid = (low + high + 1) >> 1;
      const int at = (from + to) >> 1;
      const bool is = total(keys ? mid : low, keys ? 0x7fffffff : at) >= take;
      if (keys && is) low = mid;
      else if (keys) high = mid - 1;
      else if (is) to = at;
      else from = at + 1;
    }
    limit = low;
    if (tid == 0) count = 0;
    __syncthreads();
  }
  const int n = count;
  int2* out = cands + (int64_t)blockIdx.x * take;
  for (int e = tid; e < max(n, take); e += kSliceThreads) {
    if (e < n) {
      const uint2 x = list[e];
      int rank = 0;
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const uint2 y = list[k];
        rank += y.x > x.x || (y.x == x.x && y.y < x.y);
      }
      if (rank < take) out[rank] = make_int2((int)x.y, __float_as_int(entry_of(x.x)));
    } else {
      out[e] = make_int2(-1, 0);
    }
  }
}

struct Best {
  double s;
  uint64_t id;
};
// what decides between scores that are alike: the lower row; within a row (where a log-sum may be large beside the logits) the larger logit, the lower entry
__device__ __forceinline__ uint64_t id_of(int row, float x, int entry) { return (uint64_t)row << 48 | (uint64_t)(0xffffu - ordered(x)) << 32 | (uint32_t)entry; }
__device__ __forceinline__ int row_of(uint64_t id) { return (int)(id >> 48); }
__device__ __forceinline__ bool better(double s, uint64_t id, double t, uint64_t od) { return s > t || (s == t && id < od); }

// the log-sum of a row, its largest logit at m: an eighth of the entries
__device__ __noinline__ double row_part(const __nv_bfloat16* row, int from, int to, double m) {
  double sum = 0.0;
  for (int k = from + threadIdx.x; k < to; k += kMergeThreads) sum += exp((double)__bfloat162float(row[k]) - m);
  return sum;
}
__device__ __noinline__ double row_base(const float* scores, int r, double m, double sum) {
  const double base = (scores ? (double)scores[r] : 0.0) - (m + log(sum));
  return base - base == 0.0 ? base : -INFINITY;
}
__device__ __forceinline__ uint32_t ordered_f32(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float f32_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

__global__ void __launch_bounds__(kMergeThreads) __cluster_dims__(kMergeCtas, 1, 1)
beam_merge_kernel(const __nv_bfloat16* __restrict__ logits, int64_t ld, const float* __restrict__ scores, const int32_t* __restrict__ starts, int n_rows, int n_slices,
                  int vocab, int take, const SliceStat* __restrict__ stats, const int2* __restrict__ cands, RowStat* rows, double* parts, int32_t* out_rows,
                  int32_t* out_tokens, float* out_scores) {
  constexpr int kWarps = kMergeThreads / 32;
  __shared__ double sh_s[kMergeList], sh_sum[kWarps];
  __shared__ uint64_t sh_id[kMergeList];
  __shared__ Best sorted[kMostTake + 1];
  __shared__ int need[2 * kMergeList], n_need, n_list, seen_all;
  __shared__ uint32_t asked_for[kMergeList / 32];   // rows of the sequence that are in need (of the first kMergeList)
  __shared__ Best limit;
  pdl_wait();
  const cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), seq = blockIdx.x / kMergeCtas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = min(max(starts[seq], 0), n_rows), r1 = min(max(starts[seq + 1], r0), n_rows);
  const int per_row = n_slices * take;
  auto top_of = [&](int r) {   // a row's largest logit
    float m = -INFINITY;
#pragma unroll 1
    for (int i = lane; i < n_slices; i += 32) m = fmaxf(m, stats[(int64_t)r * n_slices + i].m);
    return warp_max(m);
  };
  if (cta == 0) {
    // log-sums of the rows
#pragma unroll 1
    for (int r = r0 + warp; r < r1; r += kWarps) {
      const SliceStat* st = stats + (int64_t)r * n_slices;
      const float m = top_of(r);
      double s = 0.0;
#pragma unroll 1
      for (int i = lane; i < n_slices; i += 32) {
        const float d = st[i].m - m;   // (exact, or rounded once; both -inf: no number, as the sum of a row that has none)
        s += st[i].sum * (double)tc::exp2_fast(d * 1.4426950408889634f);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) rows[r] = {row_base(scores, r, (double)m, s), kNear};
    }
    __syncthreads();
  }
  bool exact = false;   // every row added up in fp64
#pragma unroll 1
  for (;;) {
    if (cta == 0) {
      auto each = [&](auto f) {   // the thread's share of the candidates
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
          const double base = rows[r].base;
          if (base == -INFINITY) continue;
          const int2* mine = cands + (int64_t)r * per_row;
#pragma unroll 2
          for (int i = tid; i < per_row; i += kMergeThreads) {
            const int2 c = mine[i];
            if (c.x >= 0) f(base + (double)__int_as_float(c.y), id_of(r, __int_as_float(c.y), c.x));
          }
        }
      };
      // the largest of each thread; a number that more than `take` of them reach, and few more, as fp32 (rounded down)
      double best = -INFINITY;
      each([&](double t, uint64_t) { best = fmax(best, t); });
      const uint32_t key = ordered_f32(__double2float_rd(best));
      if (tid == 0) n_list = 0, n_need = 0, seen_all = 1;
      if (tid < kMergeList / 32) asked_for[tid] = 0;
      uint32_t low = ordered_f32(-INFINITY) + 1, high = ordered_f32(INFINITY);
      int got = __syncthreads_count(key >= low);
      const bool limited = got > take;
#pragma unroll 1
      while (limited && low < high && got > take + 1 + (take >> 2) + 4) {
        const uint32_t mid = low + ((high - low + 1) >> 1);
        const int n = __syncthreads_count(key >= mid);
        if (n > take) low = mid, got = n;
        else high = mid - 1;
      }
      if (tid == 0) limit = {limited ? (double)f32_of(low) : -INFINITY, ~0ull};
      __syncthreads();
      double margin = exact ? 0.0 : 2 * kNear;
#pragma unroll 1
      for (;;) {
        const Best b = limit;
        each([&](double t, uint64_t od) {
          if (t > b.s - margin || !better(b.s, b.id, t, od)) {
            const int at = atomicAdd(&n_list, 1);
            if (at < kMergeList) sh_s[at] = t, sh_id[at] = od;
          }
        });
        __syncthreads();
        if (n_list <= kMergeList) break;
        // too many: the entry behind the best `take` of those that found room is a limit nearer to the end.  Those next to it are not all seen
#pragma unroll 1
        for (int e = tid; e < kMergeList; e += kMergeThreads) {
          int before = 0;
#pragma unroll 1
          for (int k = 0; k < kMergeList; ++k) before += better(sh_s[k], sh_id[k], sh_s[e], sh_id[e]);
          if (before == take) limit = {sh_s[e], sh_id[e]};
        }
        __syncthreads();
        if (tid == 0) n_list = 0, seen_all = margin == 0.0 && seen_all;
        margin = 0.0;
        __syncthreads();
      }
      const int n = n_list;
#pragma unroll 1
      for (int e = tid; e < n; e += kMergeThreads) {
        int before = 0;
#pragma unroll 2
        for (int k = 0; k < n; ++k) before += better(sh_s[k], sh_id[k], sh_s[e], sh_id[e]);
        if (before <= take) sorted[before] = {sh_s[e], sh_id[e]};
      }
      __syncthreads();
      if (!exact) {
        // candidates of two rows that are nearer to each other than their sums are good for: neighbours among those taken, and the last of them and whatever comes behind
#pragma unroll 1
        for (int e = tid; e < take + n; e += kMergeThreads) {
          const int k = e < take ? e : take - 1;
          if (k >= n || (e < take && e + 1 >= n)) continue;
          const Best a = sorted[k], c = e < take ? sorted[e + 1] : Best{sh_s[e - take], sh_id[e - take]};
          if (!better(a.s, a.id, c.s, c.id)) continue;
          const int ra = row_of(a.id), rb = row_of(c.id);
          const double na = rows[ra].near, nb = rows[rb].near;
          if (ra != rb && na + nb > 0.0 && a.s - c.s <= na + nb) {
#pragma unroll 1
            for (int side = 0; side < 2; ++side) {
              const int r = side ? rb : ra;
              if (!((side ? nb : na) > 0.0)) continue;
              const uint32_t bit = 1u << ((r - r0) & 31);
              if (r - r0 < kMergeList && (atomicOr(&asked_for[(r - r0) >> 5], bit) & bit)) continue;
              need[atomicAdd(&n_need, 1)] = r;   // (two for each of n entries at most)
            }
          }
        }
        __syncthreads();
      }
      const bool all_rows = !exact && !seen_all;
      if (tid == 0 && all_rows) n_need = -1;
      if (exact || (n_need == 0 && !all_rows)) {
#pragma unroll 1
        for (int k = tid; k < take; k += kMergeThreads) {
          const int64_t at = (int64_t)seq * take + k;
          out_rows[at] = k < n ? row_of(sorted[k].id) : -1;
          out_tokens[at] = k < n ? (int)(uint32_t)sorted[k].id : -1;
          out_scores[at] = k < n ? (float)sorted[k].s : -INFINITY;
        }
      }
      exact = exact || all_rows;
    }
    cluster.sync();   // the other CTAs have waited here: their help is asked for where n_need is not 0 (-1: all rows)
    const int* asked = cluster.map_shared_rank(&n_need, 0);
    const int* list = cluster.map_shared_rank(need, 0);
    const int wanted = *asked < 0 ? r1 - r0 : *asked;
    const bool by_list = *asked >= 0;
    const int from = (int)((int64_t)vocab * cta / kMergeCtas), to = (int)((int64_t)vocab * (cta + 1) / kMergeCtas);
    auto wanted_row = [&](int i) { return by_list ? list[i] : r0 + i; };
#pragma unroll 1
    for (int i = 0; i < wanted; ++i) {
      const int r = wanted_row(i);
      double sum = row_part(logits + (int64_t)r * ld, from, to, (double)top_of(r));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncthreads();
      if (lane == 0) sh_sum[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) sum += sh_sum[w];
        parts[(int64_t)r * kMergeCtas + cta] = sum;
      }
    }
    __threadfence();
    cluster.sync();   // (and nobody has left while another one reads its list)
    if (wanted == 0) return;
    if (cta == 0) {
#pragma unroll 1
      for (int i = warp; i < wanted; i += kWarps) {
        const int r = wanted_row(i);
        const float m = top_of(r);
        if (lane == 0) {
          double sum = 0.0;
          for (int k = 0; k < kMergeCtas; ++k) sum += __ldcg(parts + (int64_t)r * kMergeCtas + k);
          rows[r] = {row_base(scores, r, (double)m, sum), 0.0};
        }
      }
      __syncthreads();
    }
  }
}

// groups of eight entries a thread: the shortest slices that make no more than kFewCtas CTAs, else the longest
int slice_groups(int n_rows, int vocab) {
  int j = 1;
  while (j < kMostGroups && (int64_t)n_rows * ((vocab + 7 + kLeastSlice * j - 1) / (kLeastSlice * j)) > kFewCtas) j *= 2;
  return j;
}
int slices(int vocab, int groups) { return (vocab + 7 + kLeastSlice * groups - 1) / (kLeastSlice * groups); }

// slices of all rows at most, for this many rows and for any smaller number
int64_t most_slices(int n_rows, int vocab) {
  return std::min((int64_t)n_rows * slices(vocab, 1), std::max<int64_t>(kFewCtas, (int64_t)n_rows * slices(vocab, kMostGroups)));
}

}  // namespace

int64_t beam_select_workspace_bytes(int n_rows, int vocab, int take) {
  return most_slices(n_rows, vocab) * (int64_t)(sizeof(SliceStat) + take * sizeof(int2)) + (int64_t)n_rows * (sizeof(RowStat) + kMergeCtas * sizeof(double)) + 64;
}

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_beam_select_workspace_bytes(int32_t n_rows, int32_t vocab, int32_t n_select) {
  return n_rows > 0 && vocab > 0 && n_select > 0 ? beam_select_workspace_bytes(n_rows, vocab, n_select) : 0;
}
extern "C" int b200_beam_select(const void* logits, int64_t ld, const float* scores, const int32_t* row_starts, int32_t n_seqs, int32_t n_rows, int32_t vocab,
                                int32_t n_select, int32_t* out_rows, int32_t* out_tokens, float* out_scores, void* ws, int64_t ws_bytes, void* stream) {
  B200_REQUIRE(logits && row_starts && out_rows && out_tokens && out_scores, B200_ERR_INVALID, "beam_select: null");
  B200_REQUIRE(n_seqs >= 0 && n_rows >= 0 && vocab > 0 && ld >= vocab && n_select > 0, B200_ERR_INVALID, "beam_select: %d sequences, %d rows of %d entries, ld=%lld, %d to select",
               n_seqs, n_rows, vocab, (long long)ld, n_select);
  B200_REQUIRE(vocab <= kMostVocab, B200_ERR_UNSUPPORTED, "beam_select: vocab=%d (at most %d)", vocab, kMostVocab);
  B200_REQUIRE(n_select <= kMostTake, B200_ERR_UNSUPPORTED, "beam_select: %d to select (at most %d)", n_select, kMostTake);
  B200_REQUIRE(n_rows <= 65535, B200_ERR_UNSUPPORTED, "beam_select: %d rows (at most 65535)", n_rows);
  B200_REQUIRE(n_seqs <= 0x7fffffff / kMergeCtas, B200_ERR_UNSUPPORTED, "beam_select: %d sequences (at most %d)", n_seqs, 0x7fffffff / kMergeCtas);
  if (n_seqs == 0) return B200_OK;
  const int64_t need = n_rows > 0 ? beam_select_workspace_bytes(n_rows, vocab, n_select) : 0;
  B200_REQUIRE(need == 0 || (ws && (reinterpret_cast<uintptr_t>(ws) & 15) == 0 && ws_bytes >= need), B200_ERR_INVALID,
               "beam_select: the workspace is 16-byte aligned and has at least %lld bytes (%lld)", (long long)need, (long long)ws_bytes);
  B200_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 1) == 0, B200_ERR_INVALID, "beam_select: logits must be 2-byte aligned");
  const cudaStream_t s = (cudaStream_t)stream;
  const __nv_bfloat16* l = static_cast<const __nv_bfloat16*>(logits);
  const int groups = slice_groups(n_rows, vocab), n = slices(vocab, groups);
  SliceStat* stats = static_cast<SliceStat*>(ws);
  RowStat* rows = reinterpret_cast<RowStat*>(stats + (int64_t)n_rows * n);
  double* parts = reinterpret_cast<double*>(rows + n_rows);
  int2* cands = reinterpret_cast<int2*>(parts + (int64_t)n_rows * kMergeCtas);
  if (n_rows > 0) {
    const auto kernel = groups == 1 ? beam_slices_kernel<1> : groups == 2 ? beam_slices_kernel<2> : groups == 4 ? beam_slices_kernel<4> : beam_slices_kernel<8>;
    B200_CUDA(launch(kernel, dim3((unsigned)(n_rows * n)), dim3(kSliceThreads), (size_t)0, s, l, ld, row_starts, n_seqs, n, vocab, n_select, stats, cands));
  }
  const PdlScope merge(n_rows > 0);
  B200_CUDA(launch(beam_merge_kernel, dim3((unsigned)(n_seqs * kMergeCtas)), dim3(kMergeThreads), (size_t)0, s, l, ld, scores, row_starts, n_rows, n, vocab, n_select, stats,
                   cands, rows, parts, out_rows, out_tokens, out_scores));
  return B200_OK;
}
