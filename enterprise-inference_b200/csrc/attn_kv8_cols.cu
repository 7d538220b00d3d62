// Paged attention of few (row, head) pairs over the 8-bit cache, on tcgen05 in e4m3: the 128 tokens of a tile fill the MMA's M, the pairs of a
// kv head are its columns (decode rows: the G heads; drafts: rows x G, up to 32).
//
//   S^T[128 tokens][2 NP] = K_tile . Q^T        (A = K as the cache has it, K-major)
//   O^T[128 dims][2 NP] = V_tile^T . W^T        (A = V as the cache has it, MN-major)
//
// The codes go to the tensor core as they are: nothing is widened.  Each column is there twice, as e4m3 and as 16 times what that rounding left: for a
// bf16 query scaled by a power of two both terms together are exact (4 + 4 significant bits), for a weight they have eight.  A token's exponents are
// applied in fp32: the key's to its scores, the value's to its weights, relative to the largest one of the tile.  The weights of a tile are taken
// relative to the tile's own maximum and its product is added to the running sums in registers, so that the 22 bits between the largest and the
// smallest code pair only have to span one tile (weights relative to a running maximum would lose a long context's small ones).
//
// The flattened list of (group, kv head, tile) is cut into equal shares, one per SM: contexts may differ as they like.  An item that a cut goes through
// leaves its sums as parts, joined by the next launch.
//
// Bound by the cache's bytes: 258 a token and kv head.
#include <algorithm>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr int kSlotBytes = kKv8Tile * 128;   // a tile of keys or of values: 16 KiB
constexpr int kTable = 96;                   // items of a CTA that are described at a time
constexpr int kExpBytes = 2 * kKv8Tile;      // a tile's exponents: keys', values'
constexpr int kStageWarps = 4;               // TMA, MMA, queries, table

struct Kv8Item {
  int row0, nrows, seq, kvh, tile0, tile1, ctx, ends;   // ends: 1 begins in an earlier CTA, 2 goes on in the next
};

template <int NC>
struct Cols {
  static constexpr int NP = NC < 8 ? 8 : NC;               // columns of either term: N = 2 NP is a multiple of 16
  static constexpr int CG = NC >= 4 ? 4 : NC;              // groups of four softmax warps that share the columns
  static constexpr int NCG = NC / CG;
  static constexpr int kThreads = (kStageWarps + 4 * CG) * 32;
  static constexpr int kOperand = 2 * NP * 128;            // queries, or weights, of an item or tile
  static constexpr int kSlots = NP <= 16 ? 12 : 10;          // even: keys and values in turn
  static constexpr int kExps = kSlots / 2 + 3;             // tiles whose exponents are kept: a ring ahead of the scores, and two behind them
  static constexpr uint32_t kTmem = 8 * NP;                // S, S, O, O
  static constexpr int kSmem = 1024 + kSlots * kSlotBytes + 4 * kOperand + kExps * kExpBytes + kTable * (int)sizeof(Kv8Item) + (2 * kSlots + 16 + kExps) * 8 +
                               (4 * 32 + CG * 4 * NCG + CG * 2 * 4 * (NCG + 1)) * 4 + 256;
  static_assert(kSmem <= 232448, "shared memory");
};

// byte (row r, byte b) of an operand in rows of 128 bytes
__device__ __forceinline__ int operand_off(int r, int b) { return (r >> 3) * 1024 + (r & 7) * 128 + ((((b >> 4) ^ r) & 7) << 4) + (b & 15); }

// group i: of the plan, or the one that starts at row i
__device__ __forceinline__ Kv8Group find_group(const Kv8Params& p, int i) {
  if (p.groups) return p.groups[i];
  Kv8Group g = {i, 1, p.row_to_seq ? __ldg(p.row_to_seq + i) : i, kv8_ctx(p, i)};
  if (p.group_rows == 1 || !p.row_to_seq) return g;
  int before = 0;   // rows of the sequence in front of this one
  while (i - before > 0 && __ldg(p.row_to_seq + i - before - 1) == g.seq) ++before;
  if (before % p.group_rows) {
    g.nrows = g.ctx = 0;
    return g;
  }
  while (g.nrows < p.group_rows && i + g.nrows < p.T && __ldg(p.row_to_seq + i + g.nrows) == g.seq) g.ctx = max(g.ctx, kv8_ctx(p, i + g.nrows++));
  return g;
}
__device__ __forceinline__ int group_tiles(const Kv8Group& g) { return g.nrows > 0 && g.ctx > 0 ? (g.ctx + kKv8Tile - 1) / kKv8Tile : 0; }

template <int NC>
__global__ void __launch_bounds__(Cols<NC>::kThreads, 1)
kv8_cols_kernel(const __grid_constant__ Kv8Maps maps, const Kv8Params p) {
  using C = Cols<NC>;
  constexpr int NP = C::NP, CG = C::CG, NCG = C::NCG, kSlots = C::kSlots, kThreads = C::kThreads;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* qs = ring + kSlots * kSlotBytes;          // [2] queries of an item
  unsigned char* ws = qs + 2 * C::kOperand;                // [2] weights of a tile
  unsigned char* exps = ws + 2 * C::kOperand;              // [kExps][keys', values']
  Kv8Item* table = reinterpret_cast<Kv8Item*>(exps + C::kExps * kExpBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(table + kTable);   // [kSlots]: K, V, K, V, ...
  uint64_t* freed = full + kSlots;
  uint64_t* s_full = freed + kSlots;                       // [2]
  uint64_t* w_ready = s_full + 2;
  uint64_t* o_full = w_ready + 2;
  uint64_t* q_ready = o_full + 2;
  uint64_t* q_free = q_ready + 2;
  uint64_t* q_info = q_free + 2;                           // [4]: an item's scales, for the softmax warps (who may be three items behind)
  uint64_t* e_full = q_info + 4;                           // [kExps]
  uint64_t* last = e_full + C::kExps;
  float* q_scale = reinterpret_cast<float*>(last + 1);     // [4 items][32]
  float* x_sum = q_scale + 4 * 32;                         // [CG][4][NCG]
  int* x_max = reinterpret_cast<int*>(x_sum + CG * 4 * NCG);   // [CG][2][4][NCG + 1]
  int* shared_int = x_max + CG * 2 * 4 * (NCG + 1);        // 0: tensor memory, 1: a wait ran out, 2: items in the table, 3: next group, 4..: where the share starts
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Waits wait(reinterpret_cast<uint32_t*>(shared_int + 1), p.status);
  __shared__ int64_t scan_warp[kThreads / 32];

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(full + s, 1), mbar_init(freed + s, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(w_ready + s, 4 * CG);
      mbar_init(o_full + s, 1);
      mbar_init(q_ready + s, 1);
      mbar_init(q_free + s, 1);
    }
    for (int s = 0; s < 4; ++s) mbar_init(q_info + s, 1);
    for (int s = 0; s < C::kExps; ++s) mbar_init(e_full + s, 1);
    mbar_init(last, 1);
    shared_int[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(shared_int)), "r"(C::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  for (int i = threadIdx.x; i < 4 * C::kOperand / 16; i += kThreads) reinterpret_cast<uint4*>(qs)[i] = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  pdl_wait();
  pdl_launch_dependents();

  // ---- the CTA's share of the tiles ----
  const int n_groups = p.groups ? p.groups[-1].row0 : p.T, each = (n_groups + kThreads - 1) / kThreads;
  int64_t sum = 0;   // tiles of this thread's groups
  for (int i = threadIdx.x * each; i < min((int)(threadIdx.x + 1) * each, n_groups); ++i) sum += group_tiles(find_group(p, i));
  int64_t before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) scan_warp[warp] = before;
  before -= sum;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scan_warp[w];
    total += scan_warp[w];
  }
  const int64_t tiles = total * p.hkv, share = (tiles + gridDim.x - 1) / gridDim.x;
  const int64_t begin = min(tiles, share * blockIdx.x), end = min(tiles, begin + share);
  const int n_tiles = (int)(end - begin);
  if (begin < end && begin >= before * p.hkv && begin < (before + sum) * p.hkv) {   // one thread's groups hold the first tile
    int i = threadIdx.x * each;
    for (;; ++i) {
      const int nt = group_tiles(find_group(p, i));
      if (begin < (before + nt) * p.hkv) break;
      before += nt;
    }
    shared_int[3] = i;
    *reinterpret_cast<int64_t*>(shared_int + 4) = before * p.hkv;
  }
  if (threadIdx.x == 0) p.cuts[blockIdx.x].parts = 0;
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = (uint32_t)shared_int[0];

  // table of the next items, by warp 3 (all threads come here); false: there are none
  int64_t table_base = n_tiles > 0 ? *reinterpret_cast<int64_t*>(shared_int + 4) : 0;   // flat index of the next group's first tile (warp 3's is kept up to date)
  int table_group = shared_int[3], table_skip = 0;   // items of that group that are in earlier tables
  bool table_done = n_tiles == 0;
  auto next_table = [&]() {
    __syncthreads();
    if (warp == 3) {
      int count = 0;
      while (!table_done && count < kTable) {
        const int i = table_group + lane;
        Kv8Group g = {0, 0, 0, 0};
        if (i < n_groups) g = find_group(p, i);
        const int nt = group_tiles(g);
        int at = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += v;
        }
        const int64_t base = table_base + (int64_t)(at - nt) * p.hkv;   // this group's first tile
        // kv heads [h0, h1) whose tiles are in the share
        int h0 = 0, h1 = 0;
        if (nt > 0) {
          h0 = (int)min((int64_t)p.hkv, max((int64_t)0, (begin - base) / nt));
          h1 = (int)min((int64_t)p.hkv, max((int64_t)0, (end - base + nt - 1) / nt));
          if (lane == 0) h0 = max(h0, table_skip);
          h1 = max(h1, h0);
        }
        const int mine = h1 - h0;
        int pos = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, pos, o);
          if (lane >= o) pos += v;
        }
        const int all = __shfl_sync(0xffffffffu, pos, 31);
        pos += count - mine;
        for (int h = h0; h < h1 && pos + h - h0 < kTable; ++h) {
          Kv8Item w = {g.row0, g.nrows, g.seq, h, 0, nt, g.ctx, 0};
          const int64_t b = base + (int64_t)h * nt;
          if (b < begin) w.tile0 = (int)(begin - b), w.ends |= 1;
          if (b + nt > end) {
            w.tile1 = (int)(end - b), w.ends |= 2;
            if (!(w.ends & 1)) p.cuts[blockIdx.x] = {g.row0, g.nrows, h, (int)((b + nt - 1) / share) - (int)blockIdx.x + 1};
          }
          table[pos + h - h0] = w;
        }
        if (count + all > kTable) {   // full inside this lane's group: the next table goes on there
          const unsigned over = __ballot_sync(0xffffffffu, pos + mine > kTable);
          const int who = __ffs(over) - 1;
          table_skip = __shfl_sync(0xffffffffu, h0 + kTable - pos, who);
          table_base = __shfl_sync(0xffffffffu, base, who);
          table_group += who;
          count = kTable;
        } else {
          count += all;
          table_base += (int64_t)__shfl_sync(0xffffffffu, at, 31) * p.hkv;
          table_group += 32;
          table_skip = 0;
          table_done = table_base >= end || table_group >= n_groups;
        }
      }
      if (lane == 0) shared_int[2] = count;
    }
    __syncthreads();
    return shared_int[2];
  };

  if (warp == 0) {
    // ===== TMA: a tile's keys with all its exponents, its values =====
    const bool issuer = elect_one();
    if (issuer) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    const int box = min(p.block_size, kKv8Tile), per_tile = kKv8Tile / box;   // boxes of a tile
    const int cells = (int)(p.n_blocks * p.hkv * p.block_size);
    int slot = 0, exp_slot = 0;
    uint32_t ph = 1, eph = 1;
    bool stop = false;
    for (int count; (count = next_table()) > 0;) {
      for (int it = 0; it < count && !stop; ++it) {
        const Kv8Item w = table[it];
        const int32_t* bt = p.block_table + (int64_t)w.seq * p.bt_stride;
        const int b0 = w.tile0 * per_tile, b1 = (min(w.ctx, w.tile1 * kKv8Tile) + box - 1) / box;   // boxes that hold something
        // the first cells of the boxes, a box to a lane
        auto cell_of = [&](int b) {
          if (b >= b1) return 0;
          const int tok = b * box, blk = __ldg(bt + tok / p.block_size);
          return blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + w.kvh) * p.block_size + tok % p.block_size : cells;   // behind the cache: zeros
        };
        int have = cell_of(b0 + lane), next = cell_of(b0 + 32 + lane);
        for (int b = b0; b < b1 && !(stop = wait.stop()); b += per_tile) {
          if (b - b0 && ((b - b0) & 31) == 0) have = next, next = cell_of(b + 32 + lane);
          const int n = min(per_tile, b1 - b);
          wait(freed + slot, ph);
          unsigned char* eb = exps + exp_slot * kExpBytes;   // (its tile of a ring ago is long done: the keys' ring is shorter)
          const unsigned lanes = (n == 32 ? 0xffffffffu : (1u << n) - 1u) << ((b - b0) & 31);
          const unsigned outside = __ballot_sync(0xffffffffu, have == cells) & lanes;   // boxes outside the cache: no exponents to fetch
          if (issuer) {
            for (unsigned o = outside; o; o &= o - 1) {
              const int i = __ffs(o) - 1 - ((b - b0) & 31);
              for (int j = 0; j < box; j += 4) *reinterpret_cast<uint32_t*>(eb + i * box + j) = *reinterpret_cast<uint32_t*>(eb + kKv8Tile + i * box + j) = 0u;
            }
            mbar_expect_tx(full + slot, n * box * 128);
            mbar_expect_tx(e_full + exp_slot, (n - __popc(outside)) * box * 2);
          }
          __syncwarp();
          for (int i = 0; i < n; ++i) {
            const int cell = __shfl_sync(0xffffffffu, have, (b - b0 + i) & 31);
            if (issuer) {
              tma_load_2d(ring + slot * kSlotBytes + i * box * 128, &maps.k, 0, cell, full + slot);
              if (cell != cells) {
                bulk_load(eb + i * box, p.ke + cell, box, e_full + exp_slot);
                bulk_load(eb + kKv8Tile + i * box, p.ve + cell, box, e_full + exp_slot);
              }
            }
          }
          if (++slot == kSlots) slot = 0, ph ^= 1;
          if (++exp_slot == C::kExps) exp_slot = 0, eph ^= 1;
          wait(freed + slot, ph);
          if (issuer) mbar_expect_tx(full + slot, n * box * 128);
          __syncwarp();
          for (int i = 0; i < n; ++i) {
            const int cell = __shfl_sync(0xffffffffu, have, (b - b0 + i) & 31);
            if (issuer) tma_load_2d(ring + slot * kSlotBytes + i * box * 128, &maps.v, 0, cell, full + slot);
          }
          if (++slot == kSlots) slot = 0, ph ^= 1;
        }
      }
    }
    if (wait.stop()) {   // the loads in flight: a slot's last one filled it in this round of the ring or in the one before
      for (int s = 0; s < kSlots; ++s) wait.drain(full + s, s < slot ? ph ^ 1 : ph);
      for (int s = 0; s < C::kExps; ++s) wait.drain(e_full + s, s < exp_slot ? eph ^ 1 : eph);
    }
  } else if (warp == 1) {
    // ===== MMA: the scores of tile n + 1, of the next item if need be, then tile n's second product =====
    const uint32_t one = elect_one() ? 1u : 0u, tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t desc_ring = make_desc(smem_u32(ring), 16, 1024), desc_q = make_desc(smem_u32(qs), 16, 1024), desc_w = make_desc(smem_u32(ws), 16, 1024);
    constexpr uint32_t id_s = idesc_e4m3(2 * NP, 0), id_o = idesc_e4m3(2 * NP, 1);
    int slot = 0, n = 0, item = 0;   // slot: of the next tile's keys
    uint32_t ph = 0;
    int prev_v = 0;                  // slot and phase of tile n's values
    uint32_t prev_ph = 0;
    bool pending = false;
    auto product = [&](int m) {      // tile m's weights and values
      wait(full + prev_v, prev_ph);
      wait(w_ready + (m & 1), (m >> 1) & 1);
      fence_after();
      const uint64_t dv = desc_ring + (uint64_t)((prev_v * kSlotBytes) >> 4), dw = desc_w + (uint64_t)(((m & 1) * C::kOperand) >> 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_f8_ss(one, tm + 4 * NP + (m & 1) * 2 * NP, dv + (j * 4096) / 16, dw + (j * 32) / 16, id_o, j ? 1u : 0u);
      commit(one, freed + prev_v);
      commit(one, o_full + (m & 1));
    };
    for (int count; (count = __shfl_sync(0xffffffffu, next_table(), 0)) > 0;) {
      for (int it = 0; it < count; ++it, ++item) {
        const int nt = __shfl_sync(0xffffffffu, table[it].tile1 - table[it].tile0, 0);
        wait(q_ready + (item & 1), (item >> 1) & 1);
        const uint64_t dq = desc_q + (uint64_t)(((item & 1) * C::kOperand) >> 4);
        for (int i = 0; i < nt; ++i, ++n) {
          wait(full + slot, ph);
          fence_after();
          const uint64_t dk = desc_ring + (uint64_t)((slot * kSlotBytes) >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_f8_ss(one, tm + (n & 1) * 2 * NP, dk + (j * 32) / 16, dq + (j * 32) / 16, id_s, j ? 1u : 0u);
          commit(one, freed + slot);
          commit(one, s_full + (n & 1));
          commit(i + 1 == nt ? one : 0u, q_free + (item & 1));
          if (++slot == kSlots) slot = 0, ph ^= 1;
          if (pending) product(n - 1);
          pending = true;
          prev_v = slot, prev_ph = ph;
          if (++slot == kSlots) slot = 0, ph ^= 1;
        }
      }
      if (pending) product(n - 1);   // (the softmax warps finish a table's last item before they come to the next table)
      pending = false;
    }
    if (wait.stop()) {
      commit(one, last);
      wait.drain(last, 0);
    }
  } else if (warp == 2) {
    // ===== queries: 16 lanes a pair, scaled to [128, 256), in two terms =====
    const int G = p.hq / p.hkv;
    int item = 0;
    for (int count; (count = next_table()) > 0;) {
      for (int it = 0; it < count; ++it, ++item) {
        const Kv8Item w = table[it];
        if (item >= 2) wait(q_free + (item & 1), ((item >> 1) - 1) & 1);
        unsigned char* qb = qs + (item & 1) * C::kOperand;
        const int ncol = w.nrows * G, d = (lane & 15) * 8;
        for (int c = lane >> 4; c < ((ncol + 1) & ~1); c += 2) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (c < ncol) v = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)(w.row0 + c / G) * p.ldq + (w.kvh * G + c % G) * kHeadDim + d));
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
          uint32_t m = 0;   // the largest magnitude, as bf16 bits
#pragma unroll
          for (int j = 0; j < 4; ++j) m = max(m, max(x[j] & 0x7fffu, (x[j] >> 16) & 0x7fffu));
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          const uint32_t e = max(m >> 7, 8u);   // biased exponent
          const float f = __uint_as_float((261u - min(e, 254u)) << 23);
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            hi[j] = lo[j] = 0u;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float a = bf16lo(x[2 * j + k]) * f, b = bf16hi(x[2 * j + k]) * f;
              const uint32_t h = e == 255u ? 0x7f7fu : e4m3x2(a, b);
              const float2 r = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h, __NV_E4M3)));
              hi[j] |= h << (16 * k);
              lo[j] |= e4m3x2((a - r.x) * 16.f, (b - r.y) * 16.f) << (16 * k);
            }
          }
          if (c < ncol) {
            *reinterpret_cast<uint2*>(qb + operand_off(c, d)) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(qb + operand_off(NP + c, d)) = make_uint2(lo[0], lo[1]);
            if ((lane & 15) == 0) q_scale[(item & 3) * 32 + c] = __uint_as_float((min(e, 254u) - 7u) << 23) * p.scale2;
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready + (item & 1)), mbar_arrive(q_info + (item & 3));
      }
    }
  } else if (warp == 3) {
    // ===== rows that see nothing: zeros, by the CTAs in turn =====
    if (!p.groups)
      for (int r = blockIdx.x; r < p.T; r += gridDim.x)
        if (__ldg(p.ctx_lens + r) <= 0)
          for (int i = lane; i < p.hq * kHeadDim / 8; i += 32) *reinterpret_cast<uint4*>(p.out + (int64_t)r * p.ldo + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
    while (next_table() > 0) {
    }
  } else {
    // ===== softmax: a thread owns a token of the scores and an entry of the result; the columns are dealt to CG groups of four warps =====
    const int grp = (warp - kStageWarps) >> 2, quad = warp & 3, tau = quad * 32 + lane, G = p.hq / p.hkv, c0 = grp * NCG;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + c0;
    int* xm = x_max + grp * 2 * 4 * (NCG + 1);
    float* xs = x_sum + grp * 4 * NCG;
    int n = 0, item = 0, v_slot = 1, exp_slot = 0;
    uint32_t ph = 0, eph = 0;
    for (int count; (count = next_table()) > 0;) {
      for (int it = 0; it < count; ++it, ++item) {
        const Kv8Item w = table[it];
        const int ncol = w.nrows * G;
        int ctx[NCG];
        float qf[NCG], mu[NCG], l[NCG], acc[NCG], keep[NCG], take[NCG];   // keep, take: what becomes of the sums, and of the previous tile's product
        wait(q_info + (item & 3), (item >> 2) & 1);
#pragma unroll
        for (int j = 0; j < NCG; ++j) {
          const bool live = c0 + j < ncol;
          ctx[j] = !live ? 0 : w.nrows == 1 ? w.ctx : kv8_ctx(p, w.row0 + (c0 + j) / G);
          qf[j] = live ? q_scale[(item & 3) * 32 + c0 + j] : 0.f;
          mu[j] = -INFINITY;
          l[j] = acc[j] = 0.f;
        }
        auto fold = [&](int m) {   // tile m's product
          wait(o_full + (m & 1), (m >> 1) & 1);
          fence_after();
          uint32_t hi[NCG], lo[NCG];
          ld_cols<NCG>(base + 4 * NP + (m & 1) * 2 * NP, hi);
          ld_cols<NCG>(base + 4 * NP + (m & 1) * 2 * NP + NP, lo);
          ld_wait<NCG>(hi);
#pragma unroll
          for (int j = 0; j < NCG; ++j) {
            asm volatile("" : "+r"(lo[j]));
            acc[j] = acc[j] * keep[j] + fmaf(__uint_as_float(lo[j]), 0.0625f, __uint_as_float(hi[j])) * take[j];
          }
        };
        for (int i = w.tile0; i < w.tile1; ++i, ++n) {
          const int tok = i * kKv8Tile + tau, n_valid = w.ctx - i * kKv8Tile;
          wait(e_full + exp_slot, eph);
          uint32_t ve = exps[exp_slot * kExpBytes + kKv8Tile + tau];
          // a value row that is not a number: the columns that see it are none either, the others must not meet it
          const float ks = ve == 255u ? __uint_as_float(0x7fffffffu) : kv8_scale(exps[exp_slot * kExpBytes + tau]);
          const bool dead = tau >= n_valid || ve == 255u;
          if (dead) ve = 0u;
          int* xt = xm + (n & 1) * 4 * (NCG + 1);
          const uint32_t vw = __reduce_max_sync(0xffffffffu, ve);
          wait(s_full + (n & 1), (n >> 1) & 1);
          fence_after();
          uint32_t hi[NCG], lo[NCG];
          ld_cols<NCG>(base + (n & 1) * 2 * NP, hi);
          ld_cols<NCG>(base + (n & 1) * 2 * NP + NP, lo);
          ld_wait<NCG>(hi);
          float s[NCG];
#pragma unroll
          for (int j = 0; j < NCG; ++j) {
            asm volatile("" : "+r"(lo[j]));
            s[j] = tok < ctx[j] ? fmaf(__uint_as_float(lo[j]), 0.0625f, __uint_as_float(hi[j])) * (ks * qf[j]) : -INFINITY;
            const float m = warp_max_redux(s[j]);
            if (lane == 0) xt[quad * (NCG + 1) + j] = __float_as_int(m);
          }
          if (lane == 0) xt[quad * (NCG + 1) + NCG] = (int)vw;
          asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
          const int vmax = max(max(xt[NCG], xt[2 * NCG + 1]), max(xt[3 * NCG + 2], xt[4 * NCG + 3]));
          // 256 * 2^(ve - vmax), and what it is relative to
          const float vf = dead ? 0.f : __uint_as_float((uint32_t)max((int)ve - vmax + 127 + 8, 0) << 23);
          const float vr = __uint_as_float((uint32_t)max(vmax - 8, 1) << 23);
          float wt[NCG], keep1[NCG], take1[NCG];
#pragma unroll
          for (int j = 0; j < NCG; ++j) {
            const float mt = fmaxf(fmaxf(__int_as_float(xt[j]), __int_as_float(xt[NCG + 1 + j])),
                                   fmaxf(__int_as_float(xt[2 * (NCG + 1) + j]), __int_as_float(xt[3 * (NCG + 1) + j])));
            const bool none = mt == -INFINITY;   // a column whose row does not see this tile
            const float mn = fmaxf(mu[j], mt), e = none ? 0.f : exp2_fast(s[j] - mt), b = none ? 0.f : exp2_fast(mt - mn);
            keep1[j] = mn == -INFINITY ? 1.f : exp2_fast(mu[j] - mn);
            take1[j] = b * vr;
            l[j] = l[j] * keep1[j] + e * b;
            mu[j] = mn;
            wt[j] = none ? 0.f : e * vf;
          }
          unsigned char* wb = ws + (n & 1) * C::kOperand;
#pragma unroll
          for (int j = 0; j < NCG; j += 2) {
            const float a = wt[j], b = j + 1 < NCG ? wt[(j + 1) % NCG] : 0.f;
            const uint32_t h = e4m3x2(a, b);
            const float2 r = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h, __NV_E4M3)));
            const uint32_t g = e4m3x2((a - r.x) * 16.f, (b - r.y) * 16.f);
            wb[operand_off(c0 + j, tau)] = (unsigned char)h;
            wb[operand_off(NP + c0 + j, tau)] = (unsigned char)g;
            if (j + 1 < NCG) {
              wb[operand_off(c0 + j + 1, tau)] = (unsigned char)(h >> 8);
              wb[operand_off(NP + c0 + j + 1, tau)] = (unsigned char)(g >> 8);
            }
          }
          if (grp == 0 && __any_sync(0xffffffffu, dead)) {
            // value rows behind the context may hold anything, and 0 * NaN = NaN: zero them under their zero weights
            wait(full + v_slot, ph);
            if (dead) {
              unsigned char* vb = ring + v_slot * kSlotBytes + tau * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vb + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_async_smem();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(w_ready + (n & 1));
          if (i > w.tile0) fold(n - 1);
#pragma unroll
          for (int j = 0; j < NCG; ++j) keep[j] = keep1[j], take[j] = take1[j];
          v_slot += 2;
          if (v_slot >= kSlots) v_slot -= kSlots, ph ^= 1;
          if (++exp_slot == C::kExps) exp_slot = 0, eph ^= 1;
        }
        fold(n - 1);
        // the denominators: every token's share
#pragma unroll
        for (int j = 0; j < NCG; ++j) {
          const float v = warp_sum(l[j]);
          if (lane == 0) xs[quad * NCG + j] = v;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
#pragma unroll
        for (int j = 0; j < NCG; ++j) {
          const int c = c0 + j;
          if (c >= ncol) continue;
          const float sum_l = (xs[j] + xs[NCG + j]) + (xs[2 * NCG + j] + xs[3 * NCG + j]);
          if (w.ends == 0) {
            p.out[(int64_t)(w.row0 + c / G) * p.ldo + (w.kvh * G + c % G) * kHeadDim + tau] = __float2bfloat16_rn(sum_l == 0.f ? 0.f : acc[j] / sum_l);
          } else {
            float* dst = p.part + ((int64_t)(2 * blockIdx.x + ((w.ends & 1) ? 0 : 1)) * kKv8Cols + c) * kKv8PartFloats;
            dst[tau] = acc[j];
            if (tau == 0) dst[128] = mu[j], dst[129] = sum_l;
          }
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");   // xs is written again
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem));
  }
}

template <int NC>
int launch_cols(const Kv8Maps& m, const Kv8Params& p, int grid, cudaStream_t s) {
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(kv8_cols_kernel<NC>, Cols<NC>::kSmem, done));
  B200_CUDA(launch(kv8_cols_kernel<NC>, dim3(grid), dim3(Cols<NC>::kThreads), (size_t)Cols<NC>::kSmem, s, m, p));
  return B200_OK;
}

}  // namespace

int kv8_cols_launch(const Kv8Maps& m, const Kv8Params& p, int cols, int grid, cudaStream_t s) {
  if (const int e = wait_status()) return e;
  if (cols <= 2) return launch_cols<2>(m, p, grid, s);
  if (cols <= 4) return launch_cols<4>(m, p, grid, s);
  if (cols <= 8) return launch_cols<8>(m, p, grid, s);
  if (cols <= 16) return launch_cols<16>(m, p, grid, s);
  return launch_cols<32>(m, p, grid, s);
}

}  // namespace b200
