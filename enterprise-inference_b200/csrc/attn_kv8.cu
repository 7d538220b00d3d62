// Host side of the attention over the 8-bit cache: maps, workspace, routes, and the joining of parts.
#include <algorithm>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

// sums `a`, their maximum (log2 domain) and denominator of `parts` parts, one after another `step` floats apart -> out = sum of a_i 2^(m_i - m) / sum of l_i 2^(m_i - m),
// by a warp, four entries a lane
__device__ __forceinline__ void join_parts(const float* first, const float* rest, int64_t step, int parts, __nv_bfloat16* out) {
  const int lane = threadIdx.x & 31;
  auto part = [&](int i) { return i ? rest + (i - 1) * step : first; };
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, part(i)[128]);
  m = warp_max(m);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* x = part(i);
    const float f = m == -INFINITY ? 1.f : tc::exp2_fast(x[128] - m);
    const float4 v = reinterpret_cast<const float4*>(x)[lane];
    l += x[129] * f;
    a.x += v.x * f, a.y += v.y * f, a.z += v.z * f, a.w += v.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(out + 4 * lane) = make_uint2(pack_bf16(a.x * inv, a.y * inv), pack_bf16(a.z * inv, a.w * inv));
}

// blocks [0, kNumSMs): items of the columns kernel that several CTAs share; [kNumSMs, 2 kNumSMs): items of the rows kernel in parts
__global__ void __launch_bounds__(256) kv8_join_kernel(const Kv8Params p, int base) {
  pdl_wait();
  pdl_launch_dependents();
  const int G = p.hq / p.hkv, warp = threadIdx.x >> 5, block = blockIdx.x + base;
  if (block < kNumSMs) {
    const Kv8Cut cut = p.cuts[block];
    if (cut.parts < 2) return;
    const int64_t step = 2ll * kKv8Cols * kKv8PartFloats;
    for (int c = blockIdx.y * 8 + warp; c < cut.nrows * G; c += 8 * gridDim.y) {
      const float* x = p.part + (2 * (int64_t)block * kKv8Cols + c) * kKv8PartFloats;
      join_parts(x + kKv8Cols * kKv8PartFloats, x + step, step, cut.parts, p.out + (int64_t)(cut.row0 + c / G) * p.ldo + (cut.kvh * G + c % G) * kHeadDim);
    }
    return;
  }
  const int slot = block - kNumSMs;
  if (slot >= p.head->items * p.hkv) return;
  const Kv8Rows w = p.items[slot / p.hkv];
  if (w.parts < 2 || w.first != slot / p.hkv) return;
  const int64_t step = (int64_t)p.hkv * 128 * kKv8PartFloats;
  for (int c = blockIdx.y * 8 + warp; c < w.nrows * G; c += 8 * gridDim.y) {
    const float* x = p.part_rows + ((int64_t)slot * 128 + c) * kKv8PartFloats;
    join_parts(x, x + step, step, w.parts, p.out + (int64_t)(w.row0 + c / G) * p.ldo + (slot % p.hkv * G + c % G) * kHeadDim);
  }
}

// ---- plan: rows -> runs of one sequence -> groups of few pairs (columns kernel) and items of a tile of pairs or two (rows kernel).  One CTA. ----
constexpr int kPlanThreads = 1024, kLeastPart = 4;   // tiles of a part at least

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

__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(const Kv8Params p, int short_rows, Kv8Head* head, Kv8Group* groups, Kv8Rows* items, int* starts) {
  __shared__ int2 sh[32];
  __shared__ Kv8Rows whole[kNumSMs];
  __shared__ int sh_length;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = 128 / (p.hq / p.hkv);
  auto seq_of = [&](int r) { return p.row_to_seq ? __ldg(p.row_to_seq + r) : r; };
  // the runs' first rows
  int n_runs = 0;
  for (int r0 = 0; r0 < p.T; r0 += kPlanThreads) {
    const int r = r0 + tid;
    const int flag = r < p.T && (r == 0 || seq_of(r) != seq_of(r - 1));
    int at = flag, none = 0;
    const int n = plan_scan(at, none, sh).x;
    if (flag) starts[n_runs + at] = r;
    n_runs += n;
  }
  __syncthreads();
  auto run_rows = [&](int i) { return i < n_runs ? (i + 1 < n_runs ? starts[i + 1] : p.T) - starts[i] : 0; };
  // items of two tiles of pairs where that leaves every SM one
  int n1 = 0, n2 = 0;
  for (int i = tid; i < n_runs; i += kPlanThreads) {
    const int n = run_rows(i);
    if (n > short_rows) n1 += (n + R - 1) / R, n2 += (n + 2 * R - 1) / (2 * R);
  }
  const int2 both = plan_scan(n1, n2, sh);
  const int per = both.y * p.hkv >= kNumSMs ? 2 * R : R;
  int n_groups = 0, n_items = 0;
  for (int i0 = 0; i0 < n_runs; i0 += kPlanThreads) {
    const int i = i0 + tid, n = run_rows(i);
    const int mine = n > short_rows ? (n + per - 1) / per : 0;
    int ga = n > 0 && n <= short_rows, it = mine;
    const bool group = ga;
    const int2 all = plan_scan(ga, it, sh);
    if (group) groups[n_groups + ga] = {starts[i], n, seq_of(starts[i]), 0};
    for (int k = 0; k < mine; ++k) items[n_items + it + k] = {starts[i] + k * per, min(per, n - k * per), seq_of(starts[i]), 0, 0, 0, n_items + it + k, 1};
    n_groups += all.x, n_items += all.y;
  }
  __syncthreads();
  // the longest context of each; zeros for rows of which none sees anything
  for (int i = warp; i < n_groups + n_items; i += kPlanThreads / 32) {
    const bool group = i < n_groups;
    const int row0 = group ? groups[i].row0 : items[i - n_groups].row0, n = group ? groups[i].nrows : items[i - n_groups].nrows;
    int ctx = 0;
    for (int r = lane; r < n; r += 32) ctx = max(ctx, kv8_ctx(p, row0 + r));
    ctx = __reduce_max_sync(0xffffffffu, ctx);
    if (lane == 0) {
      if (group) groups[i].ctx = ctx;
      else items[i - n_groups].ctx = ctx, items[i - n_groups].tile1 = (ctx + kKv8Tile - 1) / kKv8Tile;
    }
    if (ctx <= 0)
      for (int r = 0; r < n; ++r)
        for (int c = lane; c < p.hq * kHeadDim / 8; c += 32) *reinterpret_cast<uint4*>(p.out + (int64_t)(row0 + r) * p.ldo + 8 * c) = make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();
  // fewer items than SMs: their contexts in parts, as short as lets every SM have one part at most
  const int room = kNumSMs / p.hkv;
  if (n_items > 0 && n_items < room) {
    if (tid < n_items) whole[tid] = items[tid];
    __syncthreads();
    if (warp == 0) {
      int lo = kLeastPart, hi = 1;
      for (int i = lane; i < n_items; i += 32) hi = max(hi, whole[i].tile1);
      hi = max(lo, __reduce_max_sync(0xffffffffu, hi));
      while (lo < hi) {   // the smallest length whose parts fit
        const int mid = (lo + hi) / 2;
        int n = 0;
        for (int i = lane; i < n_items; i += 32) n += max(1, (whole[i].tile1 + mid - 1) / mid);
        n = __reduce_add_sync(0xffffffffu, n);
        if (n <= room) hi = mid;
        else lo = mid + 1;
      }
      if (lane == 0) sh_length = lo;
    }
    __syncthreads();
    const int length = sh_length, parts = tid < n_items ? max(1, (whole[tid].tile1 + length - 1) / length) : 0;
    int at = parts, none = 0;
    const int n = plan_scan(at, none, sh).x;
    for (int k = 0; k < parts; ++k) {
      Kv8Rows w = whole[tid];
      w.tile0 = k * length, w.tile1 = min(w.tile1, (k + 1) * length), w.first = at, w.parts = parts;
      items[at + k] = w;
    }
    n_items = n;
  }
  if (tid == 0) *head = {n_groups, n_items, {0, 0}};
}

constexpr int kShortPairs = 8;    // (row, head) pairs of a group of the columns kernel in steps of longer runs
constexpr int64_t kCutBytes = (kNumSMs * sizeof(Kv8Cut) + 255) / 256 * 256;
constexpr int64_t kPartBytes = (int64_t)kNumSMs * 2 * kKv8Cols * kKv8PartFloats * 4, kPartRowsBytes = (int64_t)kNumSMs * 128 * kKv8PartFloats * 4;
int64_t plan_bytes(int T) { return (int64_t)sizeof(Kv8Head) + (int64_t)T * sizeof(Kv8Group) + ((int64_t)T + kNumSMs) * sizeof(Kv8Rows) + (int64_t)T * 4; }

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

int64_t paged_attn_fp8_workspace_bytes(int T, int hq, int hkv) { return kCutBytes + kPartBytes + kPartRowsBytes + plan_bytes(T); }

int paged_attn_fp8(const Kv8Attn& a, int most, void* ws, int64_t ws_bytes, cudaStream_t s) {
  B200_REQUIRE((int64_t)a.T * a.hkv * (((int64_t)a.bt_stride * a.block_size + kKv8Tile - 1) / kKv8Tile) < 0x7fffffffll, B200_ERR_UNSUPPORTED,
               "paged_attn_fp8: %d rows of up to %lld tokens", a.T, (long long)a.bt_stride * a.block_size);
  Kv8Maps maps;
  if (const int rc = kv8_maps(a, std::min(a.block_size, kKv8Tile), &maps)) return rc;
  const int G = a.hq / a.hkv;
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
  if (most == 1 || (most > 0 && most * G <= kShortPairs)) {   // few pairs in every run: found by the kernel itself
    p.group_rows = most;
    if (const int rc = kv8_cols_launch(maps, p, most * G, kNumSMs, s)) return rc;
    const PdlScope join;
    B200_CUDA(launch(kv8_join_kernel, dim3(kNumSMs, (most * G + 7) / 8), dim3(256), 0, s, p, 0));
    return B200_OK;
  }
  Kv8Head* const head = reinterpret_cast<Kv8Head*>(w + kCutBytes + kPartBytes + kPartRowsBytes);
  Kv8Group* const groups = reinterpret_cast<Kv8Group*>(head + 1);
  Kv8Rows* const items = reinterpret_cast<Kv8Rows*>(groups + a.T);
  const bool drafts = most > 0 && most * G <= 128;   // runs of a tile of pairs at most: all of them to the rows kernel
  const int short_rows = drafts ? 0 : std::max(1, kShortPairs / G);
  B200_CUDA(launch(kv8_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, short_rows, head, groups, items, reinterpret_cast<int*>(items + a.T + kNumSMs)));
  const PdlScope after;
  p.head = head;
  p.items = items;
  if (!drafts) {
    p.groups = groups;
    if (const int rc = kv8_cols_launch(maps, p, short_rows * G, kNumSMs, s)) return rc;
  }
  if (const int rc = kv8_rows_launch(maps, p, kNumSMs, s)) return rc;
  B200_CUDA(launch(kv8_join_kernel, dim3(drafts ? kNumSMs : 2 * kNumSMs, 4), dim3(256), 0, s, p, drafts ? kNumSMs : 0));
  return B200_OK;
}

}  // namespace b200
