// Paged attention of runs of rows over the 8-bit cache, on tcgen05: the (row, head) pairs of one kv head fill the MMA's M dimension.
//
// A work item is up to two tiles of 128 pairs (consecutive rows of one sequence times the G heads of a kv head) that share every key and value tile:
//   S_x[128][64 keys] = Q_x . K^T      (e4m3; a query in two terms that are exact together, the keys' codes as the cache has them)
//   O_x[128][128] += P_x . V           (f16; weights from TMEM, values widened by four warps: code * 2^(exponent - reference), exact)
// Here one column of scores belongs to one thread's pair, so nothing is reduced across lanes, and a weight is one f16: 11 bits, and 2^-31 of the largest before
// it is lost (e4m3 in two terms would lose it at 2^-22, and cost twice the conversions).  Widening the values is shared by 256 pairs.  The reference
// exponent of the values follows the largest one seen (two bits ahead of it); where it rises O is rescaled, as it is where a row's maximum rises by more than 2^8.
// The reference is shared by rows that see different tokens, and values far below it would lose bits to ones that a row does not see or hardly weighs: from the tile
// on where they are more than 2^kSpan apart, an item's weights carry the value exponents themselves, relative to the row's own largest share (always: 2048 rows 120 us
// instead of 104; where they do from the start 203).  Items of few pairs always do: their softmax is short, and the widening, which bounds them, has nothing to scale (200 x 5 rows over
// 300 tokens 108 -> 102.5 us).
//
// Bound by the warp that issues the MMAs (1000 to 1250 cycles for a half of 64 keys and 128 pairs: 12 MMAs, whose operands take 640 cycles of shared memory's reads, commits and
// three waits) and, beside it, by the softmax of the half (900) and the widening (1900 for both halves of a tile).  2048 rows behind 1000 tokens, 32 heads over 8, 104 us, 650
// TFLOP/s; 300 rows of three sequences behind 6000 tokens 68 us.  An item's end costs 7000 cycles: its last product, results by way of shared memory, the next one's first scores.
#include <algorithm>
#include <type_traits>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr int kThreads = 512, kHalf = 64;            // keys of a score tile: half of a tile of the cache
constexpr int kOperand = 128 * 128;                  // a term of 128 queries; a tile of keys or values in codes: 16 KiB
constexpr int kKSlots = 3, kVSlots = 2, kWide = 3;   // tiles of codes, halves of widened values
constexpr int kFacBytes = 3 * kHalf * 4 + 16;        // the keys' factors; the values' reference exponent (-1: in the weights); their own exponents; (few) 2^-those
constexpr int kSpan = 14;   // bits between an item's value exponents up to which they have one reference (a weight is good to 2^-32 of the largest, a share then to
                            // 2^-17 of the row's largest share)
constexpr int kStage = 8 * 2048;
constexpr int kBars = 2 * kKSlots + 2 * kVSlots + 2 * kWide + 12 + 3 + 1;   // (and the two words behind them)
constexpr int kSmem = 1024 + 4 * kOperand + kWide * kOperand + (kKSlots + kVSlots) * kOperand + kStage + kWide * kFacBytes + kBars * 8 + 16;
static_assert(kSmem <= 232448, "shared memory");

__device__ __forceinline__ uint32_t idesc_f16(int n) { return (1u << 4) | (1u << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

// FEW: items of at most 32 pairs, which are there in each quarter of the MMA's rows: a quarter's warp takes a quarter of the keys.  Softmax is half the work then, and
// the second group of softmax warps widens every other half instead (48 x 5 rows of 4 heads over 2500 tokens 79 us; as items of 128 pairs 90).
template <bool FEW>
__global__ void __launch_bounds__(kThreads, 1)
kv8_rows_kernel(const __grid_constant__ Kv8Maps maps, const __grid_constant__ Kv8QueryMaps qmaps, const Kv8Params p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* qs = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);   // [tile][term]
  unsigned char* wide = qs + 4 * kOperand;               // [kWide][2 x 64 dims][64 keys] f16
  unsigned char* kring = wide + kWide * kOperand;
  unsigned char* vring = kring + kKSlots * kOperand;
  unsigned char* ostage = vring + kVSlots * kOperand;
  unsigned char* facs = ostage + kStage;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(facs + kWide * kFacBytes);
  uint64_t* k_free = k_full + kKSlots;
  uint64_t* v_full = k_free + kKSlots;
  uint64_t* v_free = v_full + kVSlots;
  uint64_t* w_full = v_free + kVSlots;                   // a half's values are widened, its keys' factors there
  uint64_t* w_free = w_full + kWide;
  uint64_t* s_full = w_free + kWide;                     // [tile of pairs][2]
  uint64_t* p_ready = s_full + 4;
  uint64_t* o_full = p_ready + 4;
  uint64_t* q_ready = o_full + 4;
  uint64_t* q_free = q_ready + 1;
  uint64_t* last = q_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Waits wait(tmem_slot + 1, p.status);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kKSlots; ++s) mbar_init(k_full + s, 1), mbar_init(k_free + s, 1);
    for (int s = 0; s < kVSlots; ++s) mbar_init(v_full + s, 1), mbar_init(v_free + s, FEW ? 8 : 4);
    for (int s = 0; s < kWide; ++s) mbar_init(w_full + s, 4), mbar_init(w_free + s, 1);
    for (int s = 0; s < 4; ++s) mbar_init(s_full + s, 1), mbar_init(p_ready + s, 4), mbar_init(o_full + s, 1);
    mbar_init(q_ready, 1);
    mbar_init(q_free, 1);
    mbar_init(last, 1);
    tmem_slot[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  if (p.starts[blockIdx.x] < 0) return;   // nothing for this CTA
  const bool two = !FEW && p.groups_head->two != 0;   // items of two tiles of pairs; else of one, whose halves the two groups of softmax warps take in turn
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;   // per tile of pairs 256 columns: scores of even, odd halves, O; few: scores of even, odd tiles, O
  constexpr int kO = FEW ? 256 : 128;
  const int G = p.hq / p.hkv, R = (FEW ? 32 : 128) / G;
  // the CTA's items, in the plan's order; the one behind the next is asked for
  int at = p.starts[blockIdx.x];
  Kv8Rows ahead = p.items[at];
  auto next_unit = [&](Kv8Rows& u) {
    u = ahead;
    if (u.cta != (int)blockIdx.x) return false;
    ahead = p.items[++at];
    return true;
  };
  // does the item that was asked for come next? (its block numbers, contexts and factors may be asked for)
  auto comes_next = [&]() { return ahead.cta == (int)blockIdx.x; };

  // ===== values of a half -> f16, factors of its keys: every half (group -1), or one of each tile's =====
  auto widen = [&](int group) {
    Kv8Rows w;
    const int w4 = warp & 3, stride = p.hkv * p.block_size;
    const int r_own = 16 * w4 + 2 * (lane >> 3) + (lane >> 2 & 1), c_own = (lane & 3) + (lane & 4);
    const float sign = p.scale2 < 0.f ? -1.f : 1.f;
    int half = 0, slot = 0;
    uint32_t ph = 0;
    while (next_unit(w)) {
        // a lane's four tokens of a tile: their exponents are fetched a tile ahead, their block two
      const int32_t* bt = p.block_table + (int64_t)w.seq * p.bt_stride;
      const int h1 = min(2 * w.tile1, (w.ctx + kHalf - 1) / kHalf);
      int tok = w.tile0 * kKv8Tile + 4 * lane, at = tok / p.block_size, off = tok - at * p.block_size, blk = 0, cell = -1;
      auto place = [&]() {
        cell = tok < w.ctx ? w.kvh * p.block_size + off : -1;
        blk = __ldg(tok < w.ctx ? bt + at : p.block_table);
        tok += kKv8Tile, off += kKv8Tile;
        while (off >= p.block_size) off -= p.block_size, ++at;
      };
      uint32_t k_next = 0u, v_next = 0u;
      auto fetch = [&]() {
        k_next = v_next = 0u;
        if (cell >= 0 && blk >= 0 && blk < p.n_blocks) {   // (outside the cache: zeros)
          const int64_t c = (int64_t)blk * stride + cell;
          k_next = __ldg(reinterpret_cast<const uint32_t*>(p.ke + c)), v_next = __ldg(reinterpret_cast<const uint32_t*>(p.ve + c));
        }
      };
      place();
      fetch();
      place();
      int ref = 0;
      bool apart = false;
#pragma unroll 1
      for (int t = w.tile0; t < w.tile1; ++t) {
        const uint32_t k4 = k_next, v4 = v_next;
        fetch();
        place();
        // the reference: two bits above the largest exponent so far
        const int left = w.ctx - t * kKv8Tile;
        uint32_t mx = 1u, mn = 255u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t v = (v4 >> (8 * j)) & 255u;
          if (4 * lane + j < left && v != 255u) mx = max(mx, v), mn = min(mn, v - 1u);   // (0 stands for nothing)
        }
        mx = __reduce_max_sync(0xffffffffu, mx);
        mn = __reduce_min_sync(0xffffffffu, mn);
        if (t == w.tile0 || (int)mx > ref) ref = (int)mx + 2;
        apart |= (int)mn + 1 < ref - 2 - kSpan;
        const int least = max(ref - 2 - kKv8Span, kKv8MinExp + 127);   // (few) values below are nothing beside the largest so far
        wait(v_full + slot, ph);
        const int halves = min(2, h1 - 2 * t);
#pragma unroll 1
        for (int hh = 0; hh < halves; ++hh, ++half) {
          const int b = half % kWide;
          if (FEW && hh != group) continue;   // the other warps'
          if (half >= kWide) wait(w_free + b, (half / kWide - 1) & 1);
          const unsigned char* raw = vring + slot * kOperand + hh * kHalf * 128;
          unsigned char* dst = wide + b * kOperand;
          // pieces of 16 dims: eight lanes take four of a row and the other four of the next, so that neither the reads nor the writes (two pieces of f16 each)
          // meet a bank twice; all are asked for before anything is stored
          uint4 c[4];
          uint32_t f[2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = r_own + 8 * (i >> 1);
            c[i] = *reinterpret_cast<const uint4*>(raw + r * 128 + (((c_own ^ 4 * (i & 1)) ^ (r & 7)) << 4));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int rt = hh * kHalf + r_own + 8 * i;   // row of the tile
            const uint32_t ve = (__shfl_sync(0xffffffffu, v4, rt >> 2) >> (8 * (rt & 3))) & 255u;
            if constexpr (FEW) {   // codes as they are
              f[i] = rt >= left || ve == 255u || (int)ve < least ? 0x80008000u : 0u;
            } else {
              const int d = apart ? 5 : (int)ve - ref + 7;   // code * 2^d: exact, 5 - kSpan or more, but for bytes of 0
              const uint32_t f1 = rt >= left || ve == 255u ? 0x8000u : (uint32_t)max(d + 15, 0) << 10;
              f[i] = f1 | f1 << 16;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = r_own + 8 * (i >> 1), cc = c_own ^ 4 * (i & 1);
            if (f[i >> 1] == 0x80008000u) c[i] = make_uint4(0u, 0u, 0u, 0u);   // behind the context, not a number, or (few) nothing: zeros, whatever the codes
            const uint32_t c4[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c4[j >> 1] >> (16 * (j & 1))), __NV_E4M3));
              const __half2 v = FEW ? a : __hmul2(a, *reinterpret_cast<const __half2*>(&f[i >> 1]));
              o[j] = *reinterpret_cast<const uint32_t*>(&v);
            }
            unsigned char* row = dst + (cc >> 2) * (kOperand / 2) + r * 128;
            *reinterpret_cast<uint4*>(row + ((((cc & 3) * 2) ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(row + ((((cc & 3) * 2 + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
          {
            // a value row that is not a number: the rows that see it are none either (its key's factor)
            const int r = 16 * w4 + (lane & 15), rt = hh * kHalf + r;
            const uint32_t ke = (__shfl_sync(0xffffffffu, k4, rt >> 2) >> (8 * (rt & 3))) & 255u, ve = (__shfl_sync(0xffffffffu, v4, rt >> 2) >> (8 * (rt & 3))) & 255u;
            float* fk = reinterpret_cast<float*>(facs + b * kFacBytes);
            if (lane < 16) fk[r] = ve == 255u && rt < left ? __uint_as_float(0x7fffffffu) : sign * __uint_as_float(ke << 23);
            if constexpr (FEW) {
              const int e = rt >= left || ve == 255u ? 0 : max((int)ve, least) - 127;
              if (lane < 16) fk[kHalf + 4 + r] = (float)e, fk[2 * kHalf + 4 + r] = __uint_as_float((uint32_t)(127 - e) << 23);
            } else {
              if (lane < 16 && apart) fk[kHalf + 4 + r] = ve == 255u ? 0.f : (float)(int)ve;
              if (w4 == 0 && lane == 16) reinterpret_cast<int*>(fk)[kHalf] = apart ? -1 : ref;
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(w_full + b);
        }
        if (lane == 0) mbar_arrive(v_free + slot);
        if (++slot == kVSlots) slot = 0, ph ^= 1;
      }
    }
  };

  if (FEW && warp >= 4 && warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    widen(1);
  } else if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // ===== softmax and output: a thread owns a pair of tile x =====
    const int x = warp >> 2, quad = warp & 3, m = quad * 32 + lane;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + x * 256;
    const int r = m / G, row = (two ? x : 0) * R + r, step = two ? 1 : 2, first = two ? 0 : x;
    unsigned char* const exchange = qs + 2 * kOperand;   // (items of one tile: the second one's queries are not there)
    int n = 0, half = 0, tiles = 0;   // halves of this group of warps', of the CTA; (few) tiles of the items before this one
    auto rescale = [&](int n, float fo) {   // O of the halves before n
      if (FEW) wait(o_full + ((n - 1) & 3), ((n - 1) >> 2) & 1);
      else wait(o_full + 2 * x + ((n - 1) & 1), ((n - 1) >> 1) & 1);
      fence_after();
#pragma unroll 1
      for (int c = 0; c < kHeadDim; c += 16) {
        uint32_t o[16];
        ld16(base + kO + c, o);
        ld_wait<16>(o);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * fo);
        st16(base + kO + c, o);
      }
    };
    // The weights of a half whose values' exponents they carry: 2^(score + exponent) relative to the largest one that the row has met, `share` (followed to within 2^8, as
    // mu is), which O is relative to then; the denominators stay relative to mu.  Scores are read twice: registers are for the halves that have a reference
    auto carry = [&](uint32_t s_addr, const float* f, int live, float qf, int n, bool rescales, float& mu, float& l, float& share) {
      uint32_t s[16];
      auto read = [&](int c) {
        ld16(s_addr + 16 * c, s);
        ld_wait<16>(s);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = 16 * c + j < live ? __float_as_uint(__uint_as_float(s[j]) * f[16 * c + j] * qf) : 0xff800000u;
      };
      float ms = -INFINITY, mt = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        read(c);
#pragma unroll
        for (int j = 0; j < 16; ++j) ms = fmaxf(ms, __uint_as_float(s[j])), mt = fmaxf(mt, __uint_as_float(s[j]) + f[kHalf + 4 + 16 * c + j]);
      }
      if (ms > mu + 8.f) l *= exp2_fast(mu - ms), mu = ms;   // (nothing yet: l is 0)
      float fo = 1.f;
      if (mt > share + 8.f) {
        if (share > -INFINITY) fo = exp2_fast(share - mt);
        share = mt;
      }
      if (rescales && __any_sync(0xffffffffu, fo != 1.f)) rescale(n, fo);
      const float less = 7.f - (share > -INFINITY ? share : 0.f), shift = 7.f - (mu > -INFINITY ? mu : 0.f);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        read(c);
        uint32_t pk[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float s0 = __uint_as_float(s[2 * j]), s1 = __uint_as_float(s[2 * j + 1]);
          const float* g = f + kHalf + 4 + 16 * c + 2 * j;
          l += exp2_fast(s0 + shift) + exp2_fast(s1 + shift);
          const __half2 h2 = __floats2half2_rn(exp2_fast(s0 + g[0] + less), exp2_fast(s1 + g[1] + less));
          pk[j] = *reinterpret_cast<const uint32_t*>(&h2);
        }
        st8(s_addr + 8 * c, pk);   // (below what is still to be read)
      }
    };
    // what a row's O is times its result's denominator: values and weights as they are, but for the 2^7 that l has too
    auto undone = [&](int ref, float mu, float share, bool carried) {
      return carried && mu > -INFINITY ? exp2_fast(share - mu - 132.f) : __uint_as_float((uint32_t)max(ref - 7, 1) << 23);
    };
    // 32 columns of the warp's pairs from shared memory to their rows: a row's 64 bytes leave from four neighbouring lanes
    auto store_staged = [&](const unsigned char* st, const Kv8Rows& w, int c) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int rr = k * 8 + (lane >> 2), mm = quad * 32 + rr, row2 = (two ? x : 0) * R + mm / G, col = c + (lane & 3) * 8;
        const uint4 v = *reinterpret_cast<const uint4*>(st + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
        if (mm / G < R && row2 < w.nrows)
          *reinterpret_cast<uint4*>(p.out + (int64_t)(w.row0 + row2) * p.ldo + (int64_t)(w.kvh * G + mm % G) * kHeadDim + col) = v;
      }
    };
    // (few) what a lane's pair sees, and its scores' factor: the next item's are asked for before this one's results are written
    int ctx_next = 0;
    float qf_next = 1.f;
    bool led = false;
    auto ask = [&](const Kv8Rows& w) {
      const int t = w.row0 + lane / G;
      const bool alive = lane < w.nrows * G;
      ctx_next = alive ? kv8_ctx(p, t) : 0;
      qf_next = alive ? __ldg(p.q_scale + (int64_t)t * p.hq + w.kvh * G + lane % G) : 1.f;
    };
    // an item of at most 32 pairs: lane = pair, this warp's 16 keys of each half; the four quarters' sums are joined at the end
    auto few = [&](const Kv8Rows& w, int h0, int h1, int& n, int half) {
      const bool alive = lane < w.nrows * G;
      const int t = w.row0 + lane / G;
      if (!led) ask(w);
      const int ctx = ctx_next;
      const float qf = qf_next;
      float share = -INFINITY, l = 0.f;   // the largest 2^(score + exponent) so far (followed to within 2^8), which O and the denominator are relative to
#pragma unroll 1
      for (int h = h0; h < h1; ++h, ++n) {
        const int at = half + h - h0, b = at % kWide;
        const float* f = reinterpret_cast<const float*>(facs + b * kFacBytes);
        const int tile = tiles + (h >> 1) - w.tile0;
        if ((h & 1) == 0) wait(s_full + (tile & 1), (tile >> 1) & 1);
        wait(w_full + b, (at / kWide) & 1);
        fence_after();
        const uint32_t s_addr = base + (tile & 1) * 128 + (h & 1) * kHalf;
        uint32_t s[16];
        ld16(s_addr + 16 * quad, s);
        const int live = ctx - h * kHalf - 16 * quad;
        float k[16], e[16], back[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          *reinterpret_cast<float4*>(k + 4 * j) = reinterpret_cast<const float4*>(f)[4 * quad + j];
          *reinterpret_cast<float4*>(e + 4 * j) = reinterpret_cast<const float4*>(f + kHalf + 4)[4 * quad + j];
          *reinterpret_cast<float4*>(back + 4 * j) = reinterpret_cast<const float4*>(f + 2 * kHalf + 4)[4 * quad + j];
        }
        ld_wait<16>(s);
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float v = j < live ? fmaf(__uint_as_float(s[j]) * k[j], qf, e[j]) : -INFINITY;
          s[j] = __float_as_uint(v);
          mx = fmaxf(mx, v);
        }
        const bool jump = mx > share + 8.f;
        if (__any_sync(0xffffffffu, jump)) {
          const float mn = jump ? mx : share, fo = jump && share != -INFINITY ? exp2_fast(share - mn) : 1.f;
          l *= fo;
          share = mn;
          if (h > h0 && __any_sync(0xffffffffu, fo != 1.f)) rescale(n, fo);
        }
        const float shift = 7.f - (share > -INFINITY ? share : 0.f);
        uint32_t pk[8], none[8];
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float p0 = exp2_fast(__uint_as_float(s[2 * j]) + shift), p1 = exp2_fast(__uint_as_float(s[2 * j + 1]) + shift);
          sum = fmaf(p0, back[2 * j], fmaf(p1, back[2 * j + 1], sum));
          const __half2 h2 = __floats2half2_rn(p0, p1);
          pk[j] = *reinterpret_cast<const uint32_t*>(&h2);
          none[j] = 0u;
        }
        l += sum;
#pragma unroll
        for (int c = 0; c < 4; ++c) st8(s_addr + 8 * c, c == quad ? pk : none);   // (other quarters' keys: nothing)
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + (n & 3));
      }
      if ((led = comes_next())) ask(ahead);
      wait(o_full + ((n - 1) & 3), ((n - 1) >> 2) & 1);
      fence_after();
      // the quarters' maxima and denominators, then their sums, 32 columns at a time
      float2* ml = reinterpret_cast<float2*>(exchange);
      ml[m] = make_float2(share, l > 3e38f ? 3e38f : l);   // (not infinite: times nothing it would not be a number)
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float top = -INFINITY, all = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[32 * k + lane].x);
#pragma unroll
      for (int k = 0; k < 4; ++k) all += ml[32 * k + lane].y * (top == -INFINITY ? 0.f : exp2_fast(ml[32 * k + lane].x - top));
      const float own = share == -INFINITY ? 0.f : exp2_fast(share - top), mult = w.parts > 1 ? own : all == 0.f ? 0.f : own / all;
      float* part = p.part_rows + ((int64_t)w.slot * 128 + lane) * kKv8PartFloats;
      if (w.parts > 1 && alive && quad == 0) part[128] = top, part[129] = all;
#pragma unroll 1
      for (int c = 0; c < kHeadDim; c += 32) {
        uint32_t o[32];
        ld32(base + kO + c, o);
        ld_wait<32>(o);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float4*>(ostage + quad * 4096 + j * 512 + lane * 16) =
              make_float4(__uint_as_float(o[4 * j]) * mult, __uint_as_float(o[4 * j + 1]) * mult, __uint_as_float(o[4 * j + 2]) * mult, __uint_as_float(o[4 * j + 3]) * mult);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float y[8] = {};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(ostage + k * 4096 + (2 * quad + j) * 512 + lane * 16);
            y[4 * j] += v.x, y[4 * j + 1] += v.y, y[4 * j + 2] += v.z, y[4 * j + 3] += v.w;
          }
        if (alive && w.parts > 1) {
          *reinterpret_cast<float4*>(part + c + 8 * quad) = make_float4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<float4*>(part + c + 8 * quad + 4) = make_float4(y[4], y[5], y[6], y[7]);
        } else if (alive) {
          *reinterpret_cast<uint4*>(p.out + (int64_t)t * p.ldo + (w.kvh * G + lane % G) * kHeadDim + c + 8 * quad) =
              make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      fence_before();
    };
    Kv8Rows w;
    while (next_unit(w)) {
      const int h0 = 2 * w.tile0, h1 = min(2 * w.tile1, (w.ctx + kHalf - 1) / kHalf);
      const int at0 = half;
      half += h1 - h0;
      if (two && x == 1 && w.nrows <= R) continue;   // the item has one tile of pairs
      if constexpr (FEW) {
        few(w, h0, h1, n, at0);
        tiles += w.tile1 - w.tile0;
        continue;
      }
      const bool alive = r < R && row < w.nrows, any = __any_sync(0xffffffffu, alive);
      const int t = w.row0 + row, ctx = alive ? kv8_ctx(p, t) : 0;
      const float qf = alive ? __ldg(p.q_scale + (int64_t)t * p.hq + w.kvh * G + m % G) : 1.f;
      float mu = -INFINITY, l = 0.f, share = -INFINITY;
      int ref = 0, h = h0 + first;
      auto handed = [&]() {
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 2 * x + (n & 1));
      };
      for (; h < h1; h += step, ++n) {
        const int at = at0 + h - h0, b = at % kWide;
        const float* f = reinterpret_cast<const float*>(facs + b * kFacBytes);
        wait(s_full + 2 * x + (n & 1), (n >> 1) & 1);
        wait(w_full + b, (at / kWide) & 1);   // (after the scores: this tile's warps may have passed items over, and the phase three halves ago is complete now)
        if (!any) {   // no pair of this warp's: its weights may be anything
          if (lane == 0) mbar_arrive(p_ready + 2 * x + (n & 1));
          continue;
        }
        fence_after();
        const uint32_t s_addr = base + (n & 1) * kHalf;
        uint32_t s[64];
        ld32(s_addr, s);
        ld32(s_addr + 32, s + 32);
        const int ref_new = reinterpret_cast<const int*>(f)[kHalf], live = ctx - h * kHalf;
        ld_wait<64>(s);
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          const float4 k = reinterpret_cast<const float4*>(f)[j >> 2];
          const uint64_t a = f2::mul(f2::pack(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), f2::pack(k.x, k.y)),
                         c = f2::mul(f2::pack(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), f2::pack(k.z, k.w));
          s[j] = (uint32_t)a, s[j + 1] = (uint32_t)(a >> 32), s[j + 2] = (uint32_t)c, s[j + 3] = (uint32_t)(c >> 32);
        }
        if (__any_sync(0xffffffffu, live < kHalf)) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j >= live) s[j] = 0xff800000u;   // -inf
        }
        const float mx = max64(s) * qf;
        const bool jump = mx > mu + 8.f;   // also the first live key (mu = -inf)
        if (__any_sync(0xffffffffu, jump) || ref_new != ref) {
          if (ref_new < 0) break;   // from here on the weights carry the exponents
          const float mn = jump ? mx : mu;
          float fo = jump && mu != -INFINITY ? exp2_fast(mu - mn) : 1.f;
          l *= fo;
          mu = mn;
          if (h > h0 + first) {
            fo *= __uint_as_float((uint32_t)max(127 - (ref_new - ref), 0) << 23);
            if (__any_sync(0xffffffffu, fo != 1.f)) rescale(n, fo);
          }
          ref = ref_new;
        }
        // weights times 2^7: up to 2^15 where the maximum has risen by 2^8 since it was followed
        const uint64_t shift = f2::both(7.f - (mu > -INFINITY ? mu : 0.f)), qf2 = f2::both(qf);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int i = c * 32 + 2 * j;
            const uint64_t e = f2::fma(f2::pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), qf2, shift);
            const float p0 = exp2_fast(f2::lo(e)), p1 = exp2_fast(f2::hi(e));
            sum[j & 1] = f2::add(sum[j & 1], f2::pack(p0, p1));
            const __half2 h2 = __floats2half2_rn(p0, p1);
            pk[j] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          st16(s_addr + c * 16, pk);
        }
        l += f2::sum(sum[0]) + f2::sum(sum[1]);
        handed();
      }
      const bool carried = h < h1;
      if (carried) share = mu + (float)(ref - 2);
#pragma unroll 1
      for (; h < h1; h += step, ++n) {
        const int at = at0 + h - h0, b = at % kWide;
        wait(s_full + 2 * x + (n & 1), (n >> 1) & 1);
        wait(w_full + b, (at / kWide) & 1);
        fence_after();
        carry(base + (n & 1) * kHalf, reinterpret_cast<const float*>(facs + b * kFacBytes), ctx - h * kHalf, qf, n, h > h0 + first, mu, l, share);
        handed();
      }
      const bool some = h0 + first < h1;
      if (some) {
        wait(o_full + 2 * x + ((n - 1) & 1), ((n - 1) >> 1) & 1);
        fence_after();
      }
      const float back = undone(ref, mu, share, carried);
      if (!two) {   // the other group's halves: its sums come over through shared memory, 32 columns at a time in two buffers
        float2* ml = reinterpret_cast<float2*>(ostage + 8192);
        ml[threadIdx.x] = make_float2(mu, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float2 other = ml[threadIdx.x ^ 128];
        const float top = fmaxf(mu, other.x), own = mu == -INFINITY ? 0.f : exp2_fast(mu - top);
        const float all = l * own + other.y * (other.x == -INFINITY ? 0.f : exp2_fast(other.x - top));
        const float mult = own * (w.parts > 1 ? back : all == 0.f ? 0.f : back / all);
        float* dst = p.part_rows + ((int64_t)w.slot * 128 + m) * kKv8PartFloats;
        if (w.parts > 1 && alive && x == 0) dst[128] = top, dst[129] = all;
        unsigned char* st = ostage + warp * 2048;
#pragma unroll 1
        for (int c = 0; c < kHeadDim; c += 32) {
          uint32_t o[32];
          if (any && some) {
            ld32(base + kO + c, o);
            ld_wait<32>(o);
          }
          unsigned char* xb = exchange + (c & 32) * (kOperand / 32) + m * 16;
          if (x == 1 && any) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(xb + j * 2048) = some ? make_float4(__uint_as_float(o[4 * j]) * mult, __uint_as_float(o[4 * j + 1]) * mult,
                                                                            __uint_as_float(o[4 * j + 2]) * mult, __uint_as_float(o[4 * j + 3]) * mult)
                                                               : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (x == 0 && any) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 v = *reinterpret_cast<const float4*>(xb + j * 2048);
              const float y0 = fmaf(__uint_as_float(o[4 * j]), mult, v.x), y1 = fmaf(__uint_as_float(o[4 * j + 1]), mult, v.y),
                          y2 = fmaf(__uint_as_float(o[4 * j + 2]), mult, v.z), y3 = fmaf(__uint_as_float(o[4 * j + 3]), mult, v.w);
              if (w.parts > 1) {
                if (alive) *reinterpret_cast<float4*>(dst + c + 4 * j) = make_float4(y0, y1, y2, y3);
              } else {
                *reinterpret_cast<uint2*>(st + lane * 64 + (((j >> 1) ^ ((lane >> 1) & 3)) << 4) + (j & 1) * 8) = make_uint2(pack_bf16(y0, y1), pack_bf16(y2, y3));
              }
            }
            if (w.parts == 1) {
              __syncwarp();
              store_staged(st, w, c);
              __syncwarp();
            }
          }
        }
        fence_before();
        continue;
      }
      if (!any) continue;
      const float mult = l == 0.f ? 0.f : back / l;
      unsigned char* st = ostage + warp * 2048;
#pragma unroll 1
      for (int c = 0; c < kHeadDim; c += 32) {
        uint32_t o[32];
        ld32(base + kO + c, o);
        ld_wait<32>(o);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = pack_bf16(__uint_as_float(o[8 * k + 2 * j]) * mult, __uint_as_float(o[8 * k + 2 * j + 1]) * mult);
          *reinterpret_cast<uint4*>(st + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        __syncwarp();
        store_staged(st, w, c);
        __syncwarp();
      }
      fence_before();
      // all four warps of a tile have read its O before any of them hands over the next item's first weights (whose product restarts O)
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int box = min(p.block_size, kKv8Tile), per_tile = kKv8Tile / box;   // boxes of a tile
    Kv8Rows w;
    if (warp == 8 || warp == 10) {
      // ===== TMA: warp 8 keys, warp 10 values, a tile of 128 tokens at a time =====
      const bool issuer = elect_one(), values = warp == 10;
      const CUtensorMap* map = values ? &maps.v : &maps.k;
      unsigned char* ring = values ? vring : kring;
      uint64_t *full = values ? v_full : k_full, *freed = values ? v_free : k_free;
      const int slots = values ? kVSlots : kKSlots, cells = (int)(p.n_blocks * p.hkv * p.block_size);
      int slot = 0;
      uint32_t ph = 1;
      bool stop = false;
      // the first cell of an item's box number `at` (of those that hold something), a box to a lane
      auto cell_of = [&](const Kv8Rows& w, int at) {
        const int tok = w.tile0 * kKv8Tile + at * box;
        if (tok >= min(w.ctx, w.tile1 * kKv8Tile)) return 0;
        const int blk = __ldg(p.block_table + (int64_t)w.seq * p.bt_stride + tok / p.block_size);
        return blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + w.kvh) * p.block_size + tok % p.block_size : cells;   // behind the cache: zeros
      };
      int lead = 0;   // (few) the next item's first 32 boxes, asked for behind this one's first tile (longer items gain nothing)
      bool led = false;
      while (!stop && next_unit(w)) {
        const int boxes = (min(w.ctx, w.tile1 * kKv8Tile) - w.tile0 * kKv8Tile + box - 1) / box;
        int have = led ? lead : cell_of(w, lane), next = 32 < boxes ? cell_of(w, 32 + lane) : 0;
        for (int b = 0; b < boxes && !(stop = wait.stop()); b += per_tile) {
          if (b && (b & 31) == 0) have = next, next = cell_of(w, b + 32 + lane);
          const int k = min(per_tile, boxes - b);
          wait(freed + slot, ph);
          if (issuer) mbar_expect_tx(full + slot, k * box * 128);
          __syncwarp();
          for (int i = 0; i < k; ++i) {
            const int cell = __shfl_sync(0xffffffffu, have, (b & 31) + i);
            if (issuer) tma_load_2d(ring + slot * kOperand + i * box * 128, map, 0, cell, full + slot);
          }
          if (FEW && b == 0 && (led = comes_next())) lead = cell_of(ahead, lane);
          if (++slot == slots) slot = 0, ph ^= 1;
        }
      }
      if (wait.stop())   // the loads in flight: a slot's last one filled it in this round of the ring or in the one before
        for (int s = 0; s < slots; ++s) wait.drain(full + s, s < slot ? ph ^ 1 : ph);
    } else if (warp == 11) {
      // ===== TMA: an item's queries, in the two terms that the plan's launch left =====
      const bool issuer = elect_one();
      int done = 0;
      while (!wait.stop() && next_unit(w)) {
        const int copies = FEW ? 4 : w.nrows > R ? 2 : 1, bytes = R * G * 128;
        if (done > 0) wait(q_free, (done - 1) & 1);
        ++done;
        if (issuer) {
          mbar_expect_tx(q_ready, 2 * copies * bytes);
          for (int i = 0; i < copies; ++i) {
            unsigned char* dst = qs + i * (FEW ? 32 * 128 : 2 * kOperand);
            const int row = w.row0 + (FEW ? 0 : i * R);
            tma_load_3d(dst, &qmaps.hi, 0, w.kvh * G, row, q_ready);
            tma_load_3d(dst + kOperand, &qmaps.lo, 0, w.kvh * G, row, q_ready);
          }
        }
        __syncwarp();
      }
      if (wait.stop() && done > 0) wait.drain(q_ready, (done - 1) & 1);
    } else if (warp == 9) {
      // ===== MMA: per half, for either tile of pairs: the next half's scores, then this one's second product =====
      const uint32_t one = elect_one() ? 1u : 0u, tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t desc_q = make_desc(smem_u32(qs), 16, 1024), desc_k = make_desc(smem_u32(kring), 16, 1024), desc_v = make_desc(smem_u32(wide), kOperand / 2, 1024);
      constexpr uint32_t id_s = idesc_e4m3(kHalf, 0);
      const uint32_t id_o = idesc_f16(kHeadDim);
      int n[2] = {0, 0}, half = 0, tile = 0, slot = 0, done = 0;   // half, tile: of the CTA; slot: of the keys
      uint32_t ph = 0;
      // an item of nh halves: straight code for either count of tiles (branches between the MMAs cost the issuing warp more than the MMAs take)
      auto walk = [&](auto tiles_c, int nh) {
        constexpr int TILES = decltype(tiles_c)::value;
        auto scores = [&](int x, int nx, int i) {
          const uint64_t da = desc_q + (uint64_t)((x * 2 * kOperand) >> 4), db = desc_k + (uint64_t)((slot * kOperand + (i & 1) * kHalf * 128) >> 4);
          const uint32_t d = tm + x * 256 + (nx & 1) * kHalf;
#pragma unroll
          for (int j = 0; j < 8; ++j) mma_f8_ss(one, d, da + ((j >> 2) * kOperand + (j & 3) * 32) / 16, db + ((j & 3) * 32) / 16, id_s, j ? 1u : 0u);
          commit(one, s_full + 2 * x + (nx & 1));
        };
        auto scored = [&](int i) {   // half i's scores are on their way: the last of a tile, of the item
          const bool end = i + 1 == nh;
          commit((i & 1) || end ? one : 0u, k_free + slot);
          commit(end ? one : 0u, q_free);
          if (((i & 1) || end) && ++slot == kKSlots) slot = 0, ph ^= 1;
        };
        wait(k_full + slot, ph);
        fence_after();
#pragma unroll
        for (int x = 0; x < TILES; ++x) scores(x, n[x], 0);
        scored(0);
        int b = half % kWide;
        uint32_t bph = (half / kWide) & 1;
        auto step = [&](auto more_c, int i) {   // half i's product, behind the scores of half i + 1
          constexpr bool MORE = decltype(more_c)::value;
          if (MORE && (i & 1)) {
            wait(k_full + slot, ph);
            fence_after();
          }
          const uint64_t dv = desc_v + (uint64_t)((b * kOperand) >> 4);
#pragma unroll
          for (int x = 0; x < TILES; ++x) {
            if constexpr (MORE) scores(x, n[x] + 1, i + 1);
            if (MORE && x == TILES - 1) scored(i + 1);
            if (x == 0) wait(w_full + b, bph);
            wait(p_ready + 2 * x + (n[x] & 1), (n[x] >> 1) & 1);
            fence_after();
            const uint32_t pa = tm + x * 256 + (n[x] & 1) * kHalf, d = tm + x * 256 + 128;
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_ts(one, d, pa + j * 8, dv + (uint64_t)((j * 2048) >> 4), id_o, (i | j) ? 1u : 0u);
            if (x == TILES - 1) commit(one, w_free + b);
            commit(one, o_full + 2 * x + (n[x] & 1));
            ++n[x];
          }
          if (++b == kWide) b = 0, bph ^= 1;
        };
        for (int i = 0; i + 1 < nh; ++i) step(std::true_type(), i);
        step(std::false_type(), nh - 1);
        half += nh;
      };
      // few pairs: the scores of whole tiles (the queries' operands are read once for 128 keys: 200 x 5 rows over 300 tokens 120 -> 109 us, 48 x 5 over 2500 81 -> 79.5), a tile ahead.  Four barriers for the halves in turn: at half n all products of
      // the tile before the last are known to be complete, n - 4 among them, and a wait for the one before n - 1 in its place must not be one for n - 1
      auto walk_few = [&](int nh) {
        const int nt = (nh + 1) >> 1;
        auto scores = [&](int t) {
          wait(k_full + slot, ph);
          fence_after();
          const uint64_t db = desc_k + (uint64_t)((slot * kOperand) >> 4);
          const uint32_t d = tm + ((tile + t) & 1) * 128;
#pragma unroll
          for (int j = 0; j < 8; ++j) mma_f8_ss(one, d, desc_q + ((j >> 2) * kOperand + (j & 3) * 32) / 16, db + ((j & 3) * 32) / 16, idesc_e4m3(128, 0), j ? 1u : 0u);
          commit(one, s_full + ((tile + t) & 1));
          commit(one, k_free + slot);
          commit(t + 1 == nt ? one : 0u, q_free);
          if (++slot == kKSlots) slot = 0, ph ^= 1;
        };
        scores(0);
        int b = half % kWide;
        uint32_t bph = (half / kWide) & 1;
#pragma unroll 1
        for (int i = 0; i < nh; ++i) {
          if ((i & 1) == 0 && (i >> 1) + 1 < nt) scores((i >> 1) + 1);
          wait(w_full + b, bph);
          wait(p_ready + (n[0] & 3), (n[0] >> 2) & 1);
          fence_after();
          const uint32_t pa = tm + ((tile + (i >> 1)) & 1) * 128 + (i & 1) * kHalf, d = tm + kO;
          const uint64_t dv = desc_v + (uint64_t)((b * kOperand) >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_ts(one, d, pa + j * 8, dv + (uint64_t)((j * 2048) >> 4), id_o, (i | j) ? 1u : 0u);
          commit(one, w_free + b);
          commit(one, o_full + (n[0] & 3));
          ++n[0];
          if (++b == kWide) b = 0, bph ^= 1;
        }
        half += nh, tile += nt;
      };
      // one tile of pairs, its even halves to the first group of softmax warps, its odd ones to the second: scores two halves ahead
      auto walk_in_turn = [&](int nh) {
        int s_slot = slot;
        uint32_t s_ph = ph;
        auto scores = [&](int i) {
          if ((i & 1) == 0) {
            wait(k_full + s_slot, s_ph);
            fence_after();
          }
          const int x = i & 1, nx = (x ? n[1] : n[0]) + (i >> 1);
          const uint64_t db = desc_k + (uint64_t)((s_slot * kOperand + (i & 1) * kHalf * 128) >> 4);
          const uint32_t d = tm + x * 256 + (nx & 1) * kHalf;
#pragma unroll
          for (int j = 0; j < 8; ++j) mma_f8_ss(one, d, desc_q + ((j >> 2) * kOperand + (j & 3) * 32) / 16, db + ((j & 3) * 32) / 16, id_s, j ? 1u : 0u);
          commit(one, s_full + 2 * x + (nx & 1));
          const bool end = i + 1 == nh;
          commit(x || end ? one : 0u, k_free + s_slot);
          commit(end ? one : 0u, q_free);
          if ((x || end) && ++s_slot == kKSlots) s_slot = 0, s_ph ^= 1;
        };
        int b = half % kWide;
        uint32_t bph = (half / kWide) & 1;
#pragma unroll 1
        for (int i = -2; i < nh; ++i) {
          if (i + 2 < nh) scores(i + 2);
          if (i < 0) continue;
          const int x = i & 1, nx = (x ? n[1] : n[0]) + (i >> 1);
          wait(w_full + b, bph);
          wait(p_ready + 2 * x + (nx & 1), (nx >> 1) & 1);
          fence_after();
          const uint32_t pa = tm + x * 256 + (nx & 1) * kHalf, d = tm + x * 256 + 128;
          const uint64_t dv = desc_v + (uint64_t)((b * kOperand) >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_ts(one, d, pa + j * 8, dv + (uint64_t)((j * 2048) >> 4), id_o, (i > 1 || j) ? 1u : 0u);
          commit(one, w_free + b);
          commit(one, o_full + 2 * x + (nx & 1));
          if (++b == kWide) b = 0, bph ^= 1;
        }
        n[0] += (nh + 1) >> 1, n[1] += nh >> 1;
        half += nh;
        slot = s_slot, ph = s_ph;
      };
      for (;;) {
        const bool more = next_unit(w);
        if (!__shfl_sync(0xffffffffu, more, 0)) break;
        const int nh = __shfl_sync(0xffffffffu, min(2 * w.tile1, (w.ctx + kHalf - 1) / kHalf) - 2 * w.tile0, 0);
        const int tiles = __shfl_sync(0xffffffffu, w.nrows > R ? 2 : 1, 0);
        wait(q_ready, done++ & 1);
        if constexpr (FEW) {
          walk_few(nh);
          continue;
        }
        if (!two) walk_in_turn(nh);
        else if (tiles == 2) walk(std::integral_constant<int, 2>(), nh);
        else walk(std::integral_constant<int, 1>(), nh);
      }
      if (wait.stop()) {
        commit(one, last);
        wait.drain(last, 0);
      }
    } else {
      widen(FEW ? 0 : -1);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace

int kv8_rows_launch(const Kv8Maps& m, const Kv8QueryMaps& q, const Kv8Params& p, bool few, int grid, cudaStream_t s) {
  if (const int e = wait_status()) return e;
  static bool done[2][64] = {};
  B200_CUDA(few ? ensure_dynamic_smem(kv8_rows_kernel<true>, kSmem, done[1]) : ensure_dynamic_smem(kv8_rows_kernel<false>, kSmem, done[0]));
  B200_CUDA(launch(few ? kv8_rows_kernel<true> : kv8_rows_kernel<false>, dim3(grid), dim3(kThreads), (size_t)kSmem, s, m, q, p));
  return B200_OK;
}

}  // namespace b200
