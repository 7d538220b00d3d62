// Host side of the attention over the 8-bit cache: maps, workspace, routes, and the joining of parts.
#include <algorithm>
#include <type_traits>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

// sums `a`, their maximum (log2 domain) and denominator of `parts` parts, one after another `step` floats apart -> out = sum of a_i 2^(m_i - m) / sum of l_i 2^(m_i - m),
// by LANES neighbouring lanes.  Eight where an item of 128 pairs has few parts (a warp would wait for its parts four times: 2.5 us more behind 300 rows), a warp where
// it has many (eight lanes: 1 row over 8000 tokens 21 us instead of 17, 5 rows over 3000 28 instead of 24)
constexpr int kManyParts = 4;
template <int LANES>
__device__ __forceinline__ void join_parts(const float* first, const float* rest, int64_t step, int parts, __nv_bfloat16* out) {
  constexpr int K = 32 / LANES;   // four entries at a time
  const int lane = threadIdx.x & (LANES - 1);
  const unsigned group = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
  auto part = [&](int i) { return i ? rest + (i - 1) * step : first; };
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < parts; i += LANES) m = fmaxf(m, part(i)[128]);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(group, m, o));
  float4 a[K];
#pragma unroll
  for (int k = 0; k < K; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll (LANES == 32 ? 4 : 2)
  for (int i = 0; i < parts; ++i) {
    const float* x = part(i);
    const float f = m == -INFINITY ? 1.f : tc::exp2_fast(x[128] - m);
    l += x[129] * f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float4 v = reinterpret_cast<const float4*>(x)[lane + LANES * k];
      a[k].x += v.x * f, a[k].y += v.y * f, a[k].z += v.z * f, a[k].w += v.w * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < K; ++k)
    *reinterpret_cast<uint2*>(out + 4 * (lane + LANES * k)) = make_uint2(pack_bf16(a[k].x * inv, a[k].y * inv), pack_bf16(a[k].z * inv, a[k].w * inv));
}

// blocks [0, kNumSMs): items of the columns kernel that several CTAs share; [kNumSMs, 2 kNumSMs): items of the rows kernel in parts
__global__ void __launch_bounds__(256, 4) kv8_join_kernel(const Kv8Params p, int base) {
  pdl_wait();
  pdl_launch_dependents();
  const int G = p.hq / p.hkv, block = blockIdx.x + base;
  if (block < kNumSMs) {
    const Kv8Cut cut = p.cuts[block];
    if (cut.parts < 2) return;
    const int64_t step = 2ll * kKv8Cols * kKv8PartFloats;
    for (int c = blockIdx.y * 8 + (threadIdx.x >> 5); c < cut.nrows * G; c += 8 * gridDim.y) {
      const float* x = p.part + (2 * (int64_t)block * kKv8Cols + c) * kKv8PartFloats;
      join_parts<32>(x + kKv8Cols * kKv8PartFloats, x + step, step, cut.parts, p.out + (int64_t)(cut.row0 + c / G) * p.ldo + (cut.kvh * G + c % G) * kHeadDim);
    }
    return;
  }
  const Kv8Cut cut = p.cuts_rows[block - kNumSMs];
  if (cut.parts < 2) return;
  const int64_t step = 2ll * 128 * kKv8PartFloats;
  auto join = [&](auto lanes_c) {
    constexpr int LANES = decltype(lanes_c)::value, EACH = 256 / LANES;
    for (int c = blockIdx.y * EACH + threadIdx.x / LANES; c < cut.nrows * G; c += EACH * gridDim.y) {
      const float* x = p.part_rows + (2 * (int64_t)(block - kNumSMs) * 128 + c) * kKv8PartFloats;
      join_parts<LANES>(x + 128 * kKv8PartFloats, x + step, step, cut.parts, p.out + (int64_t)(cut.row0 + c / G) * p.ldo + (cut.kvh * G + c % G) * kHeadDim);
    }
  };
  if (cut.parts > kManyParts) join(std::integral_constant<int, 32>());
  else join(std::integral_constant<int, 8>());
}

// ---- plan: rows -> runs of one sequence -> groups of few pairs (columns kernel) and items of a tile of pairs or two (rows kernel).  One CTA. ----
constexpr int kPlanThreads = 1024, kPlanNear = 2048;   // (steps of at most so many rows: the lists in shared memory, 1 us of 300 rows' 69)

// exclusive scan over the CTA of two counts; returns the totals
__device__ __forceinline__ int2 plan_scan(int& a, int& b, int2* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) x += u, y += v;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = make_int2(x, y);
  __syncthreads();
  int2 w = sh[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w.x, o), v = __shfl_up_sync(0xffffffffu, w.y, o);
    if (lane >= o) w.x += u, w.y += v;
  }
  const int fx = __shfl_sync(0xffffffffu, w.x, max(warp - 1, 0)), fy = __shfl_sync(0xffffffffu, w.y, max(warp - 1, 0));
  a = x - a + (warp ? fx : 0), b = y - b + (warp ? fy : 0);
  return make_int2(__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31));
}

// block 0: the plan; the others: the rows kernel's queries, as two e4m3 terms and a factor each (16 lanes a query), and zeros for rows that see nothing (by the plan's block, 236 idle
// sequences of five rows beside 20 others took 188 us)
__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(const Kv8Params p, int short_rows, int R, Kv8Head* head, Kv8Group* groups, Kv8Group* rows, int* runs,
                                                                uint8_t* q_hi, uint8_t* q_lo, float* q_scale) {
  __shared__ int2 sh[32];
  __shared__ int near_runs[kPlanNear];
  __shared__ Kv8Group near_rows[kPlanNear];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.T <= kPlanNear) runs = near_runs, rows = near_rows;   // every pass over the lists waits for the one before
  if (blockIdx.x > 0) {
    const int64_t pairs = (int64_t)p.T * p.hq, step = (int64_t)(gridDim.x - 1) * (kPlanThreads / 16);
    for (int64_t i0 = (int64_t)(blockIdx.x - 1) * (kPlanThreads / 16); i0 < pairs; i0 += step) {
      const int64_t i = i0 + (tid >> 4);
      const bool in = i < pairs;
      const int row = in ? (int)(i / p.hq) : 0, h = in ? (int)(i % p.hq) : 0, d = (tid & 15) * 8;
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)row * p.ldq + h * kHeadDim + d));
      uint32_t m = query_max(v);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint32_t e = query_exponent(m);
      uint2 hi, lo;
      split_query<1>(v, e, hi, lo);
      if (in) {
        *reinterpret_cast<uint2*>(q_hi + i * kHeadDim + d) = hi;
        *reinterpret_cast<uint2*>(q_lo + i * kHeadDim + d) = lo;
        if (kv8_ctx(p, row) <= 0) *reinterpret_cast<uint4*>(p.out + (int64_t)row * p.ldo + h * kHeadDim + d) = make_uint4(0u, 0u, 0u, 0u);
        if (d == 0) q_scale[i] = fmaxf(query_back(e) * fabsf(p.scale2), 1e-37f);   // (a scale of zero: keys behind the context are still -inf)
      }
    }
    return;
  }
  auto seq_of = [&](int r) { return p.row_to_seq ? __ldg(p.row_to_seq + r) : r; };
  // the runs' first rows
  int n_runs = 0;
  for (int r0 = 0; r0 < p.T; r0 += kPlanThreads) {
    const int r = r0 + tid;
    const int flag = r < p.T && (r == 0 || seq_of(r) != seq_of(r - 1));
    int at = flag, none = 0;
    const int n = plan_scan(at, none, sh).x;
    if (flag) runs[n_runs + at] = r;
    n_runs += n;
  }
  __syncthreads();
  auto run_rows = [&](int i) { return i < n_runs ? (i + 1 < n_runs ? runs[i + 1] : p.T) - runs[i] : 0; };
  // Items of two tiles of pairs, which share what is widened (2048 rows over 1000 tokens: 103 us, of one tile 159), where most of them are full and whole items keep
  // four of seven SMs busy in every round (of 8 kv heads, 1024 rows, 128 items: 55 and 72 us; 700 rows, 88: 50 and 54; of 16, 640 rows, 160: 182 and 163)
  int n1 = 0, n2 = 0;
  for (int i = tid; i < n_runs; i += kPlanThreads) {
    const int n = run_rows(i);
    if (n > short_rows) n1 += (n + R - 1) / R, n2 += (n + 2 * R - 1) / (2 * R);
  }
  const int2 both = plan_scan(n1, n2, sh);
  const int pairs2 = both.y * p.hkv, rounds2 = (pairs2 + kNumSMs - 1) / kNumSMs;
  const bool two = R * (p.hq / p.hkv) > 32 && 7 * (int64_t)pairs2 >= 4ll * kNumSMs * rounds2 && 2 * both.x >= 3 * both.y && both.y > 0;
  const int per = two ? 2 * R : R;
  int n_groups = 0, n_items = 0;
  for (int i0 = 0; i0 < n_runs; i0 += kPlanThreads) {
    const int i = i0 + tid, n = run_rows(i);
    const int mine = n > short_rows ? (n + per - 1) / per : 0;
    int ga = n > 0 && n <= short_rows, it = mine;
    const bool group = ga;
    const int2 all = plan_scan(ga, it, sh);
    if (group) groups[n_groups + ga] = {runs[i], n, seq_of(runs[i]), 0};
    if (mine <= 2) {
      for (int k = 0; k < mine; ++k) rows[n_items + it + k] = {runs[i] + k * per, min(per, n - k * per), seq_of(runs[i]), 0};
    }
    for (unsigned many = __ballot_sync(0xffffffffu, mine > 2); many; many &= many - 1) {   // a run of many items: by its warp
      const int from = __ffs(many) - 1, row0 = __shfl_sync(0xffffffffu, i < n_runs ? runs[i] : 0, from), rn = __shfl_sync(0xffffffffu, n, from),
                to = n_items + __shfl_sync(0xffffffffu, it, from), count = __shfl_sync(0xffffffffu, mine, from), seq = seq_of(row0);
      for (int k = lane; k < count; k += 32) rows[to + k] = {row0 + k * per, min(per, rn - k * per), seq, 0};
    }
    n_groups += all.x, n_items += all.y;
  }
  __syncthreads();
  // the longest context of each
  for (int i = warp; i < n_groups + n_items; i += kPlanThreads / 32) {
    Kv8Group* const g = i < n_groups ? groups + i : rows + i - n_groups;
    const int row0 = g->row0, n = g->nrows;
    int ctx = 0;
    for (int r = lane; r < n; r += 32) ctx = max(ctx, kv8_ctx(p, row0 + r));
    ctx = __reduce_max_sync(0xffffffffu, ctx);
    if (lane == 0) g->ctx = ctx;
  }
  __syncthreads();
  // Items that see nothing leave the list: a CTA takes the first place that is not its own for the end of its items, and the shares are of tiles.  `runs` holds the
  // tiles in front of an item (of one kv head) from here on; nobody needs the runs' first rows any more
  int kept = 0, tiles = 0;
  for (int i0 = 0; i0 < n_items; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const Kv8Group g = i < n_items ? rows[i] : Kv8Group{0, 0, 0, 0};
    int front = (max(g.ctx, 0) + kKv8Tile - 1) / kKv8Tile, at = front > 0;
    const bool sees = front > 0;
    const int2 all = plan_scan(front, at, sh);   // (all have read theirs: places in front are written)
    if (sees) rows[kept + at] = g, runs[kept + at] = tiles + front;
    tiles += all.x, kept += all.y;
  }
  n_items = kept;
  const int n_list = n_items * p.hkv + 2 * kNumSMs + 1;   // places that the list may use, and the one behind them
  for (int i = tid; i < n_list; i += kPlanThreads) p.items[i].cta = -1;
  if (tid < kNumSMs) p.starts[tid] = -1, p.cuts_rows[tid].parts = 0;
  __syncthreads();
  if (two) {
    // whole items, the longest contexts (the last rows) first, every other round backwards
    const int n = n_items * p.hkv, rounds = (n + kNumSMs - 1) / kNumSMs;
    for (int i = tid; i < n; i += kPlanThreads) {
      const int round = i / kNumSMs, k = i % kNumSMs, cta = round & 1 ? kNumSMs - 1 - k : k, u = n - 1 - i;
      const Kv8Group g = rows[u / p.hkv];
      // a CTA's items have places of their own: one a round, and one behind them (the last round may have nothing for it)
      p.items[cta * (rounds + 1) + round] = {g.row0, g.nrows, g.seq, g.ctx, 0, (g.ctx + kKv8Tile - 1) / kKv8Tile, u % p.hkv, cta, 1, 0, {0, 0}};
      if (round == 0) p.starts[cta] = cta * (rounds + 1);
    }
  } else {
    // one tile of pairs: the flattened list of (item, kv head, tile) in equal shares
    const int share = max(1, (tiles * p.hkv + kNumSMs - 1) / kNumSMs);
    for (int u = tid; u < n_items * p.hkv; u += kPlanThreads) {
      const int i = u / p.hkv, h = u % p.hkv;
      const Kv8Group g = rows[i];
      const int nt = (g.ctx + kKv8Tile - 1) / kKv8Tile, base = runs[i] * p.hkv + h * nt;
      const int k0 = base / share, k1 = (base + nt - 1) / share;
      for (int k = k0; k <= k1; ++k) {
        const int from = max(base, k * share), to = min(base + nt, (k + 1) * share), place = u + k;
        p.items[place] = {g.row0, g.nrows, g.seq, g.ctx, from - base, to - base, h, k, k1 - k0 + 1, 2 * k + (k == k0 ? 1 : 0), {0, 0}};
        if (from == k * share) p.starts[k] = place;
        if (k == k0 && k1 > k0) p.cuts_rows[k] = {g.row0, g.nrows, h, k1 - k0 + 1};
      }
    }
  }
  if (tid == 0) *head = {n_groups, two, {0, 0}};
}

constexpr int64_t kMostTokens = 0x7fffffff - 2 * kKv8Tile;   // of a block table: the kernels count tokens, up to two tiles past a context's end, in 32 bits
// rows beside the longest run, times the tokens that a block table has room for: up to here their groups are not worth the columns kernel's launch (64 rows of a chunk and 16
// others over 500 or 2000 tokens: 34 and 53 us without it, 45 and 60 with; over 8000 140 and 99)
constexpr int64_t kFewTokens = 32768;
// (row, head) pairs of a run, or group, for the columns kernel (48 runs of 8 pairs over 2000 tokens: 47 us, by the rows kernel 77; of 12: 83 and 77, of 16: 88 and 77)
constexpr int kShortPairs = 8;
constexpr int64_t kCutBytes = (kNumSMs * sizeof(Kv8Cut) + 255) / 256 * 256;
constexpr int64_t kPartBytes = (int64_t)kNumSMs * 2 * kKv8Cols * kKv8PartFloats * 4, kPartRowsBytes = (int64_t)kNumSMs * 2 * 128 * kKv8PartFloats * 4;
// places of the list of items: one for each and one for each CTA, or (whole items) a round's for every CTA and one behind them
int64_t list_places(int T, int hkv) { return (int64_t)T * hkv + 3 * kNumSMs; }
int64_t plan_bytes(int T, int hkv) {
  return (2 * kCutBytes + (int64_t)sizeof(Kv8Head) + 2ll * T * sizeof(Kv8Group) + list_places(T, hkv) * sizeof(Kv8Rows) + (int64_t)T * 4 + 255) / 256 * 256;
}
int64_t query_bytes(int T, int hq) { return (int64_t)T * hq * kHeadDim; }   // of a term; a 32nd of it the factors

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

// [rows][heads][128] bytes of a query's term, boxes of n rows by the heads of a kv head
int kv8_query_map(const uint8_t* q, int T, int hq, int G, int n, CUtensorMap* m) {
  const EncodeTiledFn fn = encode_fn();
  B200_REQUIRE(fn != nullptr, B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[3] = {kHeadDim, (cuuint64_t)hq, (cuuint64_t)T}, stride[2] = {kHeadDim, (cuuint64_t)hq * kHeadDim};
  const cuuint32_t box[3] = {kHeadDim, (cuuint32_t)G, (cuuint32_t)n}, one[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(q), dims, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B200_REQUIRE(r == CUDA_SUCCESS, B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %d rows of %d queries", (int)r, T, hq);
  return B200_OK;
}

int64_t paged_attn_fp8_workspace_bytes(int T, int hq, int hkv) { return kCutBytes + kPartBytes + kPartRowsBytes + plan_bytes(T, hkv) + 2 * query_bytes(T, hq) + query_bytes(T, hq) / 32; }

int paged_attn_fp8(const Kv8Attn& a, int most, void* ws, int64_t ws_bytes, cudaStream_t s) {
  B200_REQUIRE((int64_t)a.T * a.hkv * (((int64_t)a.bt_stride * a.block_size + kKv8Tile - 1) / kKv8Tile) < 0x7fffffffll, B200_ERR_UNSUPPORTED,
               "paged_attn_fp8: %d rows of up to %lld tokens", a.T, (long long)a.bt_stride * a.block_size);
  B200_REQUIRE((int64_t)a.bt_stride * a.block_size <= kMostTokens, B200_ERR_UNSUPPORTED, "paged_attn_fp8: block tables of %lld tokens (at most %lld)",
               (long long)a.bt_stride * a.block_size, (long long)kMostTokens);
  Kv8Maps maps;
  if (const int rc = kv8_maps(a, std::min(a.block_size, kKv8Tile), &maps)) return rc;
  const int G = a.hq / a.hkv;
  const int64_t pairs = (int64_t)most * G;   // of a run of rows, where that is known
  char* const w = static_cast<char*>(ws);
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
  p.cuts = reinterpret_cast<Kv8Cut*>(w);
  p.part = reinterpret_cast<float*>(w + kCutBytes);
  p.part_rows = reinterpret_cast<float*>(w + kCutBytes + kPartBytes);
  p.status = wait_status_word();
  p.n_blocks = a.n_blocks;
  p.bt_stride = a.bt_stride;
  p.T = a.T;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.block_size = a.block_size;
  p.scale2 = a.scale * 1.4426950408889634f;
  if (most == 1 || (most > 0 && pairs <= kShortPairs)) {   // few pairs in every run: found by the kernel itself
    p.group_rows = most;
    if (const int rc = kv8_cols_launch(maps, p, most * G, kNumSMs, s)) return rc;
    const PdlScope join;
    B200_CUDA(launch(kv8_join_kernel, dim3(kNumSMs, (most * G + 7) / 8), dim3(256), 0, s, p, 0));
    return B200_OK;
  }
  char* at = w + kCutBytes + kPartBytes + kPartRowsBytes;
  p.cuts_rows = reinterpret_cast<Kv8Cut*>(at);
  p.starts = reinterpret_cast<int*>(at + kCutBytes);
  Kv8Head* const head = reinterpret_cast<Kv8Head*>(at + 2 * kCutBytes);
  Kv8Group *const groups = reinterpret_cast<Kv8Group*>(head + 1), *const rows = groups + a.T;
  p.items = reinterpret_cast<Kv8Rows*>(rows + a.T);
  // runs of a tile of pairs at most, or little beside the longest run: all of them to the rows kernel
  const bool drafts = most > 0 && (pairs <= 128 || std::max<int64_t>(a.T - most, 0) * a.bt_stride * a.block_size <= kFewTokens);
  const int short_rows = drafts ? 0 : std::max(1, kShortPairs / G);
  uint8_t* const q_hi = reinterpret_cast<uint8_t*>(w + kCutBytes + kPartBytes + kPartRowsBytes + plan_bytes(a.T, a.hkv));
  uint8_t* const q_lo = q_hi + query_bytes(a.T, a.hq);
  float* const q_scale = reinterpret_cast<float*>(q_lo + query_bytes(a.T, a.hq));
  const bool few = most > 0 && pairs <= 32;
  const int tile_rows = (few ? 32 : 128) / G;
  Kv8QueryMaps qm;
  if (const int rc = kv8_query_map(q_hi, a.T, a.hq, G, tile_rows, &qm.hi)) return rc;
  if (const int rc = kv8_query_map(q_lo, a.T, a.hq, G, tile_rows, &qm.lo)) return rc;
  const int64_t blocks = ((int64_t)a.T * a.hq + kPlanThreads / 16 - 1) / (kPlanThreads / 16);
  B200_CUDA(launch(kv8_plan_kernel, dim3(1 + (int)std::min<int64_t>(blocks, 2 * kNumSMs)), dim3(kPlanThreads), 0, s, p, short_rows, tile_rows, head, groups, rows,
                   reinterpret_cast<int*>(p.items + list_places(a.T, a.hkv)), q_hi, q_lo, q_scale));
  const PdlScope after;
  p.q_scale = q_scale;
  p.groups_head = head;
  if (!drafts) {
    p.groups = groups;
    if (const int rc = kv8_cols_launch(maps, p, short_rows * G, kNumSMs, s)) return rc;
  }
  if (const int rc = kv8_rows_launch(maps, qm, p, few, kNumSMs, s)) return rc;
  B200_CUDA(launch(kv8_join_kernel, dim3(drafts ? kNumSMs : 2 * kNumSMs, 4), dim3(256), 0, s, p, drafts ? kNumSMs : 0));
  return B200_OK;
}

}  // namespace b200
