// The walk through a checked tree of drafts (b200_accept_tree), and cached rows or states that move to new places (b200_cache_move).
#include <algorithm>

#include "f32x2.cuh"
#include "tc.cuh"

namespace b200 {
namespace {

// A warp walks a sequence's tree.  A node's parent stands before it, so one pass over the rows in order is enough: of each 32 rows a vote finds the first child of
// the present node that has the token which the target chose there, again and again until there is none.  Rows are read kAhead x 32 at a time: the walk itself then
// waits for no memory.  Bound by latency: a tree of 8 nodes 2.6 us, 64 of 50 3.0.
constexpr int kAhead = 4;

__global__ void __launch_bounds__(32)
accept_tree_kernel(const int32_t* __restrict__ target, const int32_t* __restrict__ drafts, const int32_t* __restrict__ parents, const int32_t* __restrict__ starts,
                   const int32_t* __restrict__ slots, int n_rows, int32_t* __restrict__ out_tokens, int32_t* out_rows, int32_t* __restrict__ accepted,
                   int32_t* __restrict__ move_src, int32_t* __restrict__ move_dst) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.x, lane = threadIdx.x;
  const int r0 = min(max(__ldg(starts + s), 0), n_rows), n = min(max(__ldg(starts + s + 1), r0), n_rows) - r0;
  int node = 0, taken = 0;   // the present node, and how many lie behind the root
  int token = n > 0 ? __ldg(target + r0) : 0;
  if (lane == 0 && n > 0) out_rows[r0] = r0, out_tokens[r0] = token;
  for (int base = 0; base < n; base += 32 * kAhead) {
    int parent[kAhead], draft[kAhead], chosen[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = base + 32 * k + lane;
      const bool in = r > 0 && r < n;
      parent[k] = in ? __ldg(parents + r0 + r) : -1;
      draft[k] = in ? __ldg(drafts + r0 + r) : 0;
      chosen[k] = in ? __ldg(target + r0 + r) : 0;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int first = base + 32 * k;
      for (;;) {
        const unsigned found = __ballot_sync(0xffffffffu, first + lane > node && parent[k] == node && draft[k] == token);
        if (!found) break;
        const int at = __ffs(found) - 1;
        node = first + at;
        token = __shfl_sync(0xffffffffu, chosen[k], at);
        ++taken;
        if (lane == 0) out_rows[r0 + taken] = r0 + node, out_tokens[r0 + taken] = token;
      }
    }
  }
  if (lane == 0) accepted[s] = taken;
  __syncwarp();
  for (int i = lane; i < n; i += 32) {
    const bool on = i <= taken;
    if (!on) out_rows[r0 + i] = -1, out_tokens[r0 + i] = -1;
    if (slots) {
      const int row = on ? out_rows[r0 + i] : r0 + i;   // (written by this warp)
      const bool moves = row != r0 + i;
      move_src[r0 + i] = moves ? __ldg(slots + row) : -1;
      move_dst[r0 + i] = moves ? __ldg(slots + r0 + i) : -1;
    }
  }
}

// Moves of a group happen at once: whatever is read is what was there before.  A CTA takes pieces of rows ("units": a column range of a plane) of one group; all the
// group's moves of a unit go through its shared memory, loads first, then, behind a barrier, stores.  Two halves of it: one batch of units is stored while the next is on its
// way.  A thread keeps its column and steps through (unit, move) by additions, or, where a unit's row has a piece for each thread, through the moves alone (16 x 8 states of 2 MB
// 72.7 us, 5.3 TB/s, against 74.2; 48 x up to 32 rows of 32 layers 6.8 against 7.4); where a unit lies is worked out once a batch (with divisions for every 16 bytes the states
// took 254 us).  Bound by bytes, read and written in turn, or by the launch where they are few.
constexpr int kMoveThreads = 256, kMoveStage = 32768, kMostGroup = 1024, kMoveUnits = 128, kMoveCtas = 3 * kNumSMs, kMoveColumns = 4096;

struct MoveUnit {
  unsigned char* base;
  int64_t left;   // bytes of the row from here on
};
struct MoveParams {
  unsigned char *a, *b;
  int64_t layer_stride, row_bytes, slots;
  const int32_t *src, *dst, *starts;
  int layers, heads, block_size, max_group, splits, columns, piece_bits;   // splits: CTAs of a group; columns: bytes of a unit's row, 2^piece_bits pieces
};

template <int VEC>
__device__ __forceinline__ void move_in(unsigned char* to, const unsigned char* from) {
  if constexpr (VEC == 16) f2::cp16(to, from);
  else if constexpr (VEC == 4) f2::cp4(to, from);
  else *to = *from;
}
template <int VEC>
__device__ __forceinline__ void move_out(unsigned char* to, const unsigned char* from) {
  if constexpr (VEC == 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
  else *to = *from;
}

template <int VEC>
__global__ void __launch_bounds__(kMoveThreads) cache_move_kernel(const __grid_constant__ MoveParams p) {
  extern __shared__ __align__(16) unsigned char stage[];   // two halves, then where moves come from and go to
  __shared__ MoveUnit where[3][kMoveUnits];   // (of the batch that is stored, the next one, and of the one before, which a slow warp may still store)
  __shared__ int n_valid;
  int64_t *const from = reinterpret_cast<int64_t*>(stage + 2 * kMoveStage), *const to = from + p.max_group;
  pdl_wait();
  pdl_launch_dependents();
  const int g = blockIdx.x / p.splits, part = blockIdx.x % p.splits, tid = threadIdx.x;
  const int s0 = __ldg(p.starts + g), len = min(__ldg(p.starts + g + 1) - s0, p.max_group);
  if (tid == 0) n_valid = 0;
  __syncthreads();
  auto place = [&](int slot) { return ((int64_t)(slot / p.block_size) * p.heads * p.block_size + slot % p.block_size) * p.row_bytes; };
  for (int i = tid; i < len; i += kMoveThreads) {
    const int src = __ldg(p.src + s0 + i), dst = __ldg(p.dst + s0 + i);
    if (src >= 0 && src < p.slots && dst >= 0 && dst < p.slots && src != dst) {
      const int at = atomicAdd(&n_valid, 1);
      from[at] = place(src), to[at] = place(dst);
    }
  }
  __syncthreads();
  const int m = n_valid;
  if (m == 0) return;
  const int per_plane = (int)((p.row_bytes + p.columns - 1) / p.columns), units = (p.b ? 2 : 1) * p.layers * p.heads * per_plane;
  const int u0 = (int)((int64_t)units * part / p.splits), u1 = (int)((int64_t)units * (part + 1) / p.splits);
  const int batch = min(kMoveUnits, max(1, kMoveStage / (m * p.columns)));
  // a thread's column (or columns, kMoveThreads pieces apart) and its steps through the pairs of unit and move
  const int piece0 = tid & ((1 << p.piece_bits) - 1), lanes = max(1, kMoveThreads >> p.piece_bits), first = p.piece_bits < 31 ? tid >> p.piece_bits : 0;
  const int unit_step = lanes / m, move_step = lanes % m, unit0 = first / m, move0 = first % m;
  auto find = [&](int u, int count, MoveUnit* w) {
    if (tid < count) {
      const int plane = (u + tid) / per_plane, head = plane % p.heads, layer = plane / p.heads;
      const int64_t col = (int64_t)(u + tid - plane * per_plane) * p.columns;
      unsigned char* const base = layer < p.layers ? p.a + layer * p.layer_stride : p.b + (layer - p.layers) * p.layer_stride;
      w[tid] = {base + (int64_t)head * p.block_size * p.row_bytes + col, p.row_bytes - col};
    }
  };
  auto walk = [&](int count, const MoveUnit* w, const int64_t* moves, auto f) {   // f(place in the half, address) for all of the thread's
    if (lanes == 1) {
      for (int piece = piece0; piece < 1 << p.piece_bits; piece += kMoveThreads)
        for (int unit = 0; unit < count; ++unit) {
          const MoveUnit t = w[unit];
          if (piece * VEC >= t.left) continue;
          unsigned char* const at = t.base + piece * VEC;
          int e = unit * m * p.columns + piece * VEC;
#pragma unroll 4
          for (int mv = 0; mv < m; ++mv, e += p.columns) f(e, at + moves[mv]);
        }
      return;
    }
    for (int unit = unit0, mv = move0; unit < count;) {
      const MoveUnit t = w[unit];
      if (piece0 * VEC < t.left) f((((unit * m + mv) << p.piece_bits) + piece0) * VEC, t.base + moves[mv] + piece0 * VEC);
      unit += unit_step, mv += move_step;
      if (mv >= m) mv -= m, ++unit;
    }
  };
  auto load = [&](int count, const MoveUnit* w, int half) {
    walk(count, w, from, [&](int e, const unsigned char* src) { move_in<VEC>(stage + half * kMoveStage + e, src); });
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto count_at = [&](int u) { return max(0, min(batch, u1 - u)); };
  find(u0, count_at(u0), where[0]);
  __syncthreads();
  load(count_at(u0), where[0], 0);
  int half = 0, w = 0;
  for (int u = u0; u < u1; u += batch, half ^= 1) {
    const int more = count_at(u + batch), next = w == 2 ? 0 : w + 1;
    find(u + batch, more, where[next]);
    __syncthreads();   // (the other half has been stored, and its units are there)
    if (more) {
      load(more, where[next], half ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    walk(count_at(u), where[w], to, [&](int e, unsigned char* dst) { move_out<VEC>(dst, stage + half * kMoveStage + e); });
    w = next;
  }
}

template <int VEC>
int move_launch(const MoveParams& p, int n_groups, cudaStream_t s) {
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(cache_move_kernel<VEC>, 2 * kMoveStage + kMostGroup * 16, done));
  B200_CUDA(launch(cache_move_kernel<VEC>, dim3((unsigned)(n_groups * p.splits)), dim3(kMoveThreads), (size_t)(2 * kMoveStage + p.max_group * 16), s, p));
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_accept_tree(const int32_t* target_tokens, const int32_t* draft_tokens, const int32_t* parents, const int32_t* row_starts,
                                const int32_t* slot_mapping, int32_t n_seqs, int32_t n_rows, int32_t* out_tokens, int32_t* out_rows, int32_t* out_accepted,
                                int32_t* move_src, int32_t* move_dst, void* stream) {
  B200_REQUIRE(target_tokens && draft_tokens && parents && row_starts && out_tokens && out_rows && out_accepted, B200_ERR_INVALID, "accept_tree: null");
  B200_REQUIRE((slot_mapping != nullptr) == (move_src != nullptr) && (slot_mapping != nullptr) == (move_dst != nullptr), B200_ERR_INVALID,
               "accept_tree: slot_mapping, move_src and move_dst go together");
  B200_REQUIRE(n_seqs >= 0 && n_rows >= 0, B200_ERR_INVALID, "accept_tree: %d sequences, %d rows", n_seqs, n_rows);
  if (n_seqs == 0) return B200_OK;
  B200_CUDA(launch(accept_tree_kernel, dim3((unsigned)n_seqs), dim3(32), (size_t)0, (cudaStream_t)stream, target_tokens, draft_tokens, parents, row_starts, slot_mapping,
                   n_rows, out_tokens, out_rows, out_accepted, move_src, move_dst));
  return B200_OK;
}

extern "C" int b200_cache_move(void* cache_a, void* cache_b, int32_t n_layers, int64_t layer_stride, int64_t n_blocks, int32_t heads, int32_t block_size,
                               int64_t row_bytes, const int32_t* src_slots, const int32_t* dst_slots, const int32_t* group_starts, int32_t n_groups,
                               int32_t max_group, void* stream) {
  B200_REQUIRE(cache_a && src_slots && dst_slots && group_starts, B200_ERR_INVALID, "cache_move: null");
  B200_REQUIRE(n_layers > 0 && n_blocks > 0 && heads > 0 && block_size > 0 && row_bytes > 0 && n_groups >= 0 && max_group >= 0, B200_ERR_INVALID,
               "cache_move: %d layers of %lld blocks of %d heads x %d rows of %lld bytes, %d groups of up to %d moves", n_layers, (long long)n_blocks, heads, block_size,
               (long long)row_bytes, n_groups, max_group);
  B200_REQUIRE(max_group <= kMostGroup, B200_ERR_UNSUPPORTED, "cache_move: groups of %d moves (at most %d)", max_group, kMostGroup);
  B200_REQUIRE(n_blocks <= 0x7fffffff / block_size, B200_ERR_UNSUPPORTED, "cache_move: %lld blocks of %d rows (at most 2^31 - 1 rows)", (long long)n_blocks, block_size);
  const __int128 plane = (__int128)n_blocks * heads * block_size * row_bytes;
  B200_REQUIRE(plane < ((__int128)1 << 62), B200_ERR_INVALID, "cache_move: a layer of more bytes than there are");
  B200_REQUIRE(n_layers == 1 || layer_stride >= (int64_t)plane, B200_ERR_INVALID, "cache_move: layers of %lld bytes, %lld apart", (long long)plane, (long long)layer_stride);
  if (n_groups == 0 || max_group == 0) return B200_OK;
  if (cache_b == cache_a) cache_b = nullptr;   // (values that are the keys: moved once, by one CTA a piece, or what is read might have been written already)
  const uint64_t all = reinterpret_cast<uintptr_t>(cache_a) | reinterpret_cast<uintptr_t>(cache_b) | (uint64_t)row_bytes | (n_layers > 1 ? (uint64_t)layer_stride : 0);
  const int vec = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
  MoveParams p = {static_cast<unsigned char*>(cache_a), static_cast<unsigned char*>(cache_b), layer_stride, row_bytes, n_blocks * block_size, src_slots, dst_slots, group_starts,
                  n_layers, heads, block_size, max_group, 1, vec, 0};
  // a unit's row: as much of a row as leaves room for all moves of a group
  const int64_t room = std::min<int64_t>(kMoveStage / max_group, kMoveColumns);
  while (2 * p.columns <= room && p.columns < row_bytes) p.columns *= 2, ++p.piece_bits;
  const __int128 units = (__int128)(cache_b ? 2 : 1) * n_layers * heads * ((row_bytes + p.columns - 1) / p.columns);
  B200_REQUIRE(units < 0x7fffffff, B200_ERR_UNSUPPORTED, "cache_move: rows of %lld bytes in %d planes", (long long)row_bytes, n_layers * heads);
  p.splits = (int)std::min<int64_t>((int64_t)units, std::max(1, kMoveCtas / n_groups));
  B200_REQUIRE((int64_t)n_groups * p.splits < 0x7fffffff, B200_ERR_UNSUPPORTED, "cache_move: %d groups", n_groups);
  const cudaStream_t s = (cudaStream_t)stream;
  return vec == 16 ? move_launch<16>(p, n_groups, s) : vec == 4 ? move_launch<4>(p, n_groups, s) : move_launch<1>(p, n_groups, s);
}
