// Paged attention of runs of rows over the 8-bit cache, on tcgen05: the (row, head) pairs of one kv head fill the MMA's M dimension.
//
// A work item is up to two tiles of 128 pairs (consecutive rows of one sequence times the G heads of a kv head) that share every key and value tile:
//   S_x[128][64 keys] = Q_x . K^T      (e4m3; a query in two terms that are exact together, the keys' codes as the cache has them)
//   O_x[128][128] += P_x . V           (f16; weights from TMEM, values widened by four warps: code * 2^(exponent - reference), exact)
// Here one column of scores belongs to one thread's pair, so nothing is reduced across lanes, and a weight is one f16: 11 bits, and 2^-31 of the largest before
// it is lost (e4m3 in two terms would lose it at 2^-22, and cost twice the conversions).  Widening the values is shared by 256 pairs.  The reference
// exponent of the values follows the largest one seen (two bits ahead of it); where it rises O is rescaled, as it is where a row's maximum rises by more than 2^8.
//
// Bound by the exponentials (16 a cycle and SM) and by the shared-memory reads of the MMAs' operands.
#include <algorithm>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr int kThreads = 512, kHalf = 64;            // keys of a score tile: half of a tile of the cache
constexpr int kOperand = 128 * 128;                  // a term of 128 queries; a tile of keys or values in codes: 16 KiB
constexpr int kKSlots = 3, kVSlots = 2, kWide = 3;   // tiles of codes, halves of widened values
constexpr int kFacBytes = kHalf * 4 + 16;            // the keys' factors; the values' reference exponent
constexpr int kStage = 8 * 2048;
constexpr int kBars = 2 * kKSlots + 2 * kVSlots + 2 * kWide + 12 + 3 + 1;
constexpr int kSmem = 1024 + 4 * kOperand + kWide * kOperand + (kKSlots + kVSlots) * kOperand + kStage + kWide * kFacBytes + 2 * 256 * 4 + kBars * 8 + 16;
static_assert(kSmem <= 232448, "shared memory");

__device__ __forceinline__ uint32_t idesc_f16(int n) { return (1u << 4) | (1u << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

struct Unit {
  Kv8Rows w;
  int kvh, slot;
};

// an item's queries -> the two terms of its one or two tiles, and their factors, by 128 threads: 16 lanes a pair
__device__ __forceinline__ void stage_queries(const Kv8Params& p, unsigned char* qs, float* scale, const Unit& u, int R, int G, int thread) {
  const int pieces = (u.w.nrows > R ? 2 : 1) * 128 * 16, chunk = thread & 15;
  const __nv_bfloat16* q0 = p.q + (int64_t)u.w.row0 * p.ldq + (int64_t)u.kvh * G * kHeadDim + chunk * 8;
  constexpr int U = 4;
#pragma unroll 1
  for (int e0 = thread; e0 < pieces; e0 += U * 128) {
    uint4 v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int m = (e0 + i * 128) >> 4, r = (m & 127) / G, row = (m >> 7) * R + r;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < R && row < u.w.nrows) v[i] = __ldg(reinterpret_cast<const uint4*>(q0 + (int64_t)row * p.ldq + ((m & 127) % G) * kHeadDim));
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int m = (e0 + i * 128) >> 4;
      uint2 hi, lo;
      const float back = split_query<1>(v[i], hi, lo);
      unsigned char* dst = qs + (m >> 7) * 2 * kOperand + operand_off(m & 127, chunk * 8);
      *reinterpret_cast<uint2*>(dst) = hi;
      *reinterpret_cast<uint2*>(dst + kOperand) = lo;
      if (chunk == 0) scale[m] = fmaxf(back * fabsf(p.scale2), 1e-37f);   // (a scale of zero: keys behind the context are still -inf)
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
kv8_rows_kernel(const __grid_constant__ Kv8Maps maps, const Kv8Params p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* qs = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);   // [tile][term]
  unsigned char* wide = qs + 4 * kOperand;               // [kWide][2 x 64 dims][64 keys] f16
  unsigned char* kring = wide + kWide * kOperand;
  unsigned char* vring = kring + kKSlots * kOperand;
  unsigned char* ostage = vring + kVSlots * kOperand;
  unsigned char* facs = ostage + kStage;
  float* q_scale = reinterpret_cast<float*>(facs + kWide * kFacBytes);   // [2 items][256]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(q_scale + 2 * 256);
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
    for (int s = 0; s < kVSlots; ++s) mbar_init(v_full + s, 1), mbar_init(v_free + s, 4);
    for (int s = 0; s < kWide; ++s) mbar_init(w_full + s, 4), mbar_init(w_free + s, 1);
    for (int s = 0; s < 4; ++s) mbar_init(s_full + s, 1), mbar_init(p_ready + s, 4), mbar_init(o_full + s, 1);
    mbar_init(q_ready, 4);
    mbar_init(q_free, 1);
    mbar_init(last, 1);
    tmem_slot[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  const Kv8Head head = *p.head;
  const int n_units = head.items * p.hkv, grid = gridDim.x;
  if ((int)blockIdx.x >= n_units) return;
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;   // per tile of pairs 256 columns: scores of even, odd halves, O
  const int G = p.hq / p.hkv, R = 128 / G;
  // units in turn, the longest first, every other round backwards
  auto unit = [&](int round, Unit& u) {
    const int i = round * grid + ((round & 1) ? grid - 1 - (int)blockIdx.x : (int)blockIdx.x);
    if (i >= n_units) return false;
    u.slot = n_units - 1 - i;
    u.kvh = u.slot % p.hkv;
    u.w = p.items[u.slot / p.hkv];
    return u.w.tile1 > u.w.tile0;   // (rows that see nothing: the plan wrote their zeros)
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // ===== softmax and output: a thread owns a pair of tile x =====
    const int x = warp >> 2, quad = warp & 3, m = quad * 32 + lane;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + x * 256;
    const int r = m / G, row = x * R + r;
    int n = 0, half = 0, item = 0;   // halves of this tile of pairs, of the CTA; items
    Unit u;
    for (int round = 0; round * grid < n_units; ++round) {
      if (!unit(round, u)) continue;
      const Kv8Rows& w = u.w;
      const int h0 = 2 * w.tile0, h1 = min(2 * w.tile1, (w.ctx + kHalf - 1) / kHalf);
      ++item;
      if (x == 1 && w.nrows <= R) {   // the item has one tile of pairs
        half += h1 - h0;
        continue;
      }
      const bool alive = r < R && row < w.nrows, any = __any_sync(0xffffffffu, alive);
      const int t = w.row0 + row, ctx = alive ? kv8_ctx(p, t) : 0;
      float qf = 0.f, mu = -INFINITY, l = 0.f;
      int ref = 0;
      for (int h = h0; h < h1; ++h, ++n, ++half) {
        const int b = half % kWide;
        const float* f = reinterpret_cast<const float*>(facs + b * kFacBytes);
        wait(s_full + 2 * x + (n & 1), (n >> 1) & 1);
        wait(w_full + b, (half / kWide) & 1);   // (after the scores: this tile's warps may have passed items over, and the phase three halves ago is complete now)
        if (!any) {   // no pair of this warp's: its weights may be anything
          if (lane == 0) mbar_arrive(p_ready + 2 * x + (n & 1));
          continue;
        }
        if (h == h0) qf = q_scale[(item & 1) * 256 + x * 128 + m];
        fence_after();
        const uint32_t s_addr = base + (n & 1) * kHalf;
        uint32_t s[64];
        ld32(s_addr, s);
        ld32(s_addr + 32, s + 32);
        const int ref_new = reinterpret_cast<const int*>(f)[kHalf];
        ld_wait<64>(s);
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          const float4 k = reinterpret_cast<const float4*>(f)[j >> 2];
          const uint64_t a = f2::mul(f2::pack(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), f2::pack(k.x, k.y)),
                         c = f2::mul(f2::pack(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), f2::pack(k.z, k.w));
          s[j] = (uint32_t)a, s[j + 1] = (uint32_t)(a >> 32), s[j + 2] = (uint32_t)c, s[j + 3] = (uint32_t)(c >> 32);
        }
        const int live = ctx - h * kHalf;
        if (__any_sync(0xffffffffu, live < kHalf)) {
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j >= live) s[j] = 0xff800000u;   // -inf
        }
        const float mx = max64(s) * qf;
        const bool jump = mx > mu + 8.f;   // also the first live key (mu = -inf)
        if (__any_sync(0xffffffffu, jump) || ref_new != ref) {
          const float mn = jump ? mx : mu;
          float fo = jump && mu != -INFINITY ? exp2_fast(mu - mn) : 1.f;
          l *= fo;
          mu = mn;
          if (h > h0) {
            fo *= __uint_as_float((uint32_t)max(127 - (ref_new - ref), 0) << 23);
            if (__any_sync(0xffffffffu, fo != 1.f)) {
              wait(o_full + 2 * x + ((n - 1) & 1), ((n - 1) >> 1) & 1);
              fence_after();
#pragma unroll 1
              for (int c = 0; c < kHeadDim; c += 16) {
                uint32_t o[16];
                ld16(base + 128 + c, o);
                ld_wait<16>(o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * fo);
                st16(base + 128 + c, o);
              }
            }
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
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 2 * x + (n & 1));
      }
      wait(o_full + 2 * x + ((n - 1) & 1), ((n - 1) >> 1) & 1);
      fence_after();
      if (!any) continue;
      const float back = __uint_as_float((uint32_t)max(ref - 7, 1) << 23);   // 2^(ref - 134): values and weights as they are, but for the 2^7 that l has too
      const float mult = w.parts > 1 ? back : l == 0.f ? 0.f : back / l;
      if (w.parts > 1) {
        float* dst = p.part_rows + ((int64_t)u.slot * 128 + m) * kKv8PartFloats;
        if (alive) dst[128] = mu, dst[129] = l;
#pragma unroll 1
        for (int c = 0; c < kHeadDim; c += 16) {
          uint32_t o[16];
          ld16(base + 128 + c, o);
          ld_wait<16>(o);
          if (alive) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(dst + c + j) = make_float4(__uint_as_float(o[j]) * mult, __uint_as_float(o[j + 1]) * mult, __uint_as_float(o[j + 2]) * mult,
                                                                    __uint_as_float(o[j + 3]) * mult);
          }
        }
      } else {
        // 32 columns at a time through shared memory: a row's 64 bytes leave from four neighbouring lanes
        unsigned char* st = ostage + warp * 2048;
#pragma unroll 1
        for (int c = 0; c < kHeadDim; c += 32) {
          uint32_t o[32];
          ld32(base + 128 + c, o);
          ld_wait<32>(o);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = pack_bf16(__uint_as_float(o[8 * k + 2 * j]) * mult, __uint_as_float(o[8 * k + 2 * j + 1]) * mult);
            *reinterpret_cast<uint4*>(st + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int rr = k * 8 + (lane >> 2), mm = quad * 32 + rr, row2 = x * R + mm / G, col = c + (lane & 3) * 8;
            const uint4 v = *reinterpret_cast<const uint4*>(st + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
            if (mm / G < R && row2 < w.nrows)
              *reinterpret_cast<uint4*>(p.out + (int64_t)(w.row0 + row2) * p.ldo + (int64_t)(u.kvh * G + mm % G) * kHeadDim + col) = v;
          }
          __syncwarp();
        }
      }
      fence_before();
      // all four warps of a tile have read its O before any of them hands over the next item's first weights (whose product restarts O)
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int box = min(p.block_size, kKv8Tile), per_tile = kKv8Tile / box;   // boxes of a tile
    Unit u;
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
      for (int round = 0; round * grid < n_units && !stop; ++round) {
        if (!unit(round, u)) continue;
        const int32_t* bt = p.block_table + (int64_t)u.w.seq * p.bt_stride;
        const int b0 = u.w.tile0 * per_tile, b1 = (min(u.w.ctx, u.w.tile1 * kKv8Tile) + box - 1) / box;
        auto cell_of = [&](int b) {
          if (b >= b1) return 0;
          const int tok = b * box, blk = __ldg(bt + tok / p.block_size);
          return blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + u.kvh) * p.block_size + tok % p.block_size : cells;   // behind the cache: zeros
        };
        int have = cell_of(b0 + lane), next = b0 + 32 < b1 ? cell_of(b0 + 32 + lane) : 0;
        for (int b = b0; b < b1 && !(stop = wait.stop()); b += per_tile) {
          if (b - b0 && ((b - b0) & 31) == 0) have = next, next = cell_of(b + 32 + lane);
          const int k = min(per_tile, b1 - b);
          wait(freed + slot, ph);
          if (issuer) mbar_expect_tx(full + slot, k * box * 128);
          __syncwarp();
          for (int i = 0; i < k; ++i) {
            const int cell = __shfl_sync(0xffffffffu, have, ((b - b0) & 31) + i);
            if (issuer) tma_load_2d(ring + slot * kOperand + i * box * 128, map, 0, cell, full + slot);
          }
          if (++slot == slots) slot = 0, ph ^= 1;
        }
      }
      if (wait.stop())   // the loads in flight: a slot's last one filled it in this round of the ring or in the one before
        for (int s = 0; s < slots; ++s) wait.drain(full + s, s < slot ? ph ^ 1 : ph);
    } else if (warp == 9) {
      // ===== MMA: per half, for either tile of pairs: the next half's scores, then this one's second product =====
      const uint32_t one = elect_one() ? 1u : 0u, tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t desc_q = make_desc(smem_u32(qs), 16, 1024), desc_k = make_desc(smem_u32(kring), 16, 1024), desc_v = make_desc(smem_u32(wide), kOperand / 2, 1024);
      constexpr uint32_t id_s = idesc_e4m3(kHalf, 0);
      const uint32_t id_o = idesc_f16(kHeadDim);
      int n[2] = {0, 0}, half = 0, slot = 0, done = 0;   // half: of the CTA; slot: of the keys
      uint32_t ph = 0;
      for (int round = 0; round * grid < n_units; ++round) {
        const bool have = unit(round, u);
        if (!__shfl_sync(0xffffffffu, have, 0)) continue;
        const int nh = __shfl_sync(0xffffffffu, min(2 * u.w.tile1, (u.w.ctx + kHalf - 1) / kHalf) - 2 * u.w.tile0, 0);
        const int tiles = __shfl_sync(0xffffffffu, u.w.nrows > R ? 2 : 1, 0);
        wait(q_ready, done++ & 1);
        // step i: scores of half i (i < nh), the product of half i - 1 (i > 0)
        for (int i = 0; i <= nh; ++i) {
          if (i < nh && (i & 1) == 0) wait(k_full + slot, ph);
          fence_after();
#pragma unroll 1
          for (int x = 0; x < tiles; ++x) {
            if (i < nh) {
              const uint64_t da = desc_q + (uint64_t)((x * 2 * kOperand) >> 4), db = desc_k + (uint64_t)((slot * kOperand + (i & 1) * kHalf * 128) >> 4);
              const int nx = n[x] + (i > 0 ? 1 : 0);
              const uint32_t d = tm + x * 256 + (nx & 1) * kHalf;
#pragma unroll
              for (int j = 0; j < 8; ++j) mma_f8_ss(one, d, da + ((j >> 2) * kOperand + (j & 3) * 32) / 16, db + ((j & 3) * 32) / 16, id_s, j ? 1u : 0u);
              commit(one, s_full + 2 * x + (nx & 1));
              if (x + 1 == tiles) {
                commit(((i & 1) || i + 1 == nh) ? one : 0u, k_free + slot);
                commit(i + 1 == nh ? one : 0u, q_free);   // the item's last scores are on their way
              }
            }
            if (i > 0) {
              const int b = half % kWide;
              if (x == 0) wait(w_full + b, (half / kWide) & 1);
              wait(p_ready + 2 * x + (n[x] & 1), (n[x] >> 1) & 1);
              fence_after();
              const uint32_t pa = tm + x * 256 + (n[x] & 1) * kHalf, d = tm + x * 256 + 128;
              const uint64_t dv = desc_v + (uint64_t)((b * kOperand) >> 4);
#pragma unroll
              for (int j = 0; j < 4; ++j) mma_ts(one, d, pa + j * 8, dv + (uint64_t)((j * 2048) >> 4), id_o, (i > 1 || j) ? 1u : 0u);
              if (x + 1 == tiles) commit(one, w_free + b);
              commit(one, o_full + 2 * x + (n[x] & 1));
              ++n[x];
            }
          }
          if (i > 0) ++half;
          if (i < nh && ((i & 1) || i + 1 == nh) && ++slot == kKSlots) slot = 0, ph ^= 1;
        }
      }
      if (wait.stop()) {
        commit(one, last);
        wait.drain(last, 0);
      }
    } else if (warp >= 12) {
      // ===== queries of an item -> two terms; values of a half -> f16, factors of its keys =====
      const int w4 = warp - 12, cl = lane & 7, stride = p.hkv * p.block_size;
      const float sign = p.scale2 < 0.f ? -1.f : 1.f;
      int half = 0, slot = 0, done = 0;
      uint32_t ph = 0;
      for (int round = 0; round * grid < n_units; ++round) {
        if (!unit(round, u)) continue;
        const Kv8Rows& w = u.w;
        // exponents: lanes 0..15 four keys each, 16..31 four values; fetched a half ahead, their block two
        const int32_t* bt = p.block_table + (int64_t)w.seq * p.bt_stride;
        const uint8_t* src = lane < 16 ? p.ke : p.ve;
        const int h0 = 2 * w.tile0, h1 = min(2 * w.tile1, (w.ctx + kHalf - 1) / kHalf);
        int tok = h0 * kHalf + 4 * (lane & 15), at = tok / p.block_size, off = tok - at * p.block_size;
        int blk = 0, cell = -1;
        auto place = [&]() {
          cell = tok < w.ctx ? u.kvh * p.block_size + off : -1;
          blk = __ldg(tok < w.ctx ? bt + at : p.block_table);
          tok += kHalf, off += kHalf;
          while (off >= p.block_size) off -= p.block_size, ++at;
        };
        auto fetch = [&]() {
          uint32_t v = 0u;
          if (cell >= 0 && blk >= 0 && blk < p.n_blocks) v = __ldg(reinterpret_cast<const uint32_t*>(src + blk * stride + cell));   // (outside the cache: zeros)
          return v;
        };
        place();
        uint32_t e_next = fetch();
        place();
        if (done > 0) wait(q_free, (done - 1) & 1);
        ++done;
        stage_queries(p, qs, q_scale + (done & 1) * 256, u, R, G, threadIdx.x - 384);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
        int ref = 0;
#pragma unroll 1
        for (int h = h0; h < h1; ++h, ++half) {
          const uint32_t e4 = e_next;
          e_next = fetch();
          place();
          const int b = half % kWide, live = w.ctx - h * kHalf;   // tokens of the half
          // the reference: two bits above the largest exponent so far
          uint32_t mx = 1u;
          if (lane >= 16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t v = (e4 >> (8 * j)) & 255u;
              if (4 * (lane & 15) + j < live && v != 255u) mx = max(mx, v);
            }
          }
          mx = __reduce_max_sync(0xffffffffu, mx);
          if (h == h0 || (int)mx > ref) ref = (int)mx + 2;
          if ((h & 1) == 0) wait(v_full + slot, ph);
          if (half >= kWide) wait(w_free + b, (half / kWide - 1) & 1);
          const unsigned char* raw = vring + slot * kOperand + (h & 1) * kHalf * 128;
          unsigned char* dst = wide + b * kOperand;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 16 * w4 + 4 * i + (lane >> 3);
            const uint32_t ve = (__shfl_sync(0xffffffffu, e4, 16 + (r >> 2)) >> (8 * (r & 3))) & 255u;
            const bool dead = r >= live || ve == 255u;
            const int d = (int)ve - ref + 7;   // code * 2^d, exact while d >= -15
            const uint32_t f1 = d >= -14 ? (uint32_t)(d + 15) << 10 : d >= -24 ? 1u << (d + 24) : 0u, f = f1 | f1 << 16;
            const uint4 c = *reinterpret_cast<const uint4*>(raw + r * 128 + ((cl ^ (r & 7)) << 4));
            const uint32_t c4[4] = {c.x, c.y, c.z, c.w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c4[j >> 1] >> (16 * (j & 1))), __NV_E4M3));
              const __half2 v = __hmul2(a, *reinterpret_cast<const __half2*>(&f));
              o[j] = dead ? 0u : *reinterpret_cast<const uint32_t*>(&v);
            }
            // 16 dims: two pieces of the first or the second 64; odd lanes' halves in another order, so that eight lanes meet no bank twice
            unsigned char* row = dst + (cl >> 2) * (kOperand / 2) + r * 128;
            const int i0 = (cl & 3) * 2, swap = cl >> 2;
            *reinterpret_cast<uint4*>(row + (((i0 + swap) ^ (r & 7)) << 4)) = swap ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(row + (((i0 + 1 - swap) ^ (r & 7)) << 4)) = swap ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(o[4], o[5], o[6], o[7]);
          }
          {
            // a value row that is not a number: the rows that see it are none either (its key's factor)
            const int r = 16 * w4 + (lane & 15);
            const uint32_t ke = (__shfl_sync(0xffffffffu, e4, r >> 2) >> (8 * (r & 3))) & 255u, ve = (__shfl_sync(0xffffffffu, e4, 16 + (r >> 2)) >> (8 * (r & 3))) & 255u;
            float* fk = reinterpret_cast<float*>(facs + b * kFacBytes);
            if (lane < 16) fk[r] = ve == 255u && r < live ? __uint_as_float(0x7fffffffu) : sign * __uint_as_float(ke << 23);
            if (warp == 12 && lane == 16) reinterpret_cast<int*>(fk)[kHalf] = ref;
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(w_full + b);
            if ((h & 1) || h + 1 == h1) mbar_arrive(v_free + slot);
          }
          if (((h & 1) || h + 1 == h1) && ++slot == kVSlots) slot = 0, ph ^= 1;
        }
      }
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

int kv8_rows_launch(const Kv8Maps& m, const Kv8Params& p, int grid, cudaStream_t s) {
  if (const int e = wait_status()) return e;
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(kv8_rows_kernel, kSmem, done));
  B200_CUDA(launch(kv8_rows_kernel, dim3(grid), dim3(kThreads), (size_t)kSmem, s, m, p));
  return B200_OK;
}

}  // namespace b200
