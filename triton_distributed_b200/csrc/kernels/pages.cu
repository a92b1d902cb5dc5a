// Pages of a cache that several sequences may hold: forking, room for more tokens (copy on write), trimming, compaction, copies.
//
// State on the device: block_table int32 [R, W], where entry w of row r is the page of tokens w * page ... and -1 marks what a row does not
// hold (held entries come first); kv_lens int32 [R]; refs int32 [N], by how many table entries each page is held. A page whose count is zero
// is free: there is no list of free pages to keep. Nothing here waits for the host, so all of it can be captured in a graph.
//
// Whatever could be done in several orders is defined: free pages are given out in ascending order to the rows in ascending order, and
// counts change by integer atomics, so results do not depend on the schedule. Page numbers and rows out of range are skipped.
//
// What bounds them: the moves are copies at the memory's rate; the tables are small and their kernels take launch and latency.
#include "b200/host.h"
#include "b200/primitives.cuh"

#include <cstring>

namespace b200 {

constexpr int kPlanThreads = 1024;
constexpr int kLongRows = 64;

// Inclusive sum over the threads of a CTA of kPlanThreads; `total` is the CTA's. All threads call it.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += x;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int front = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return v + (warp > 0 ? front : 0);
}

// The counts of pages i ... i + 3, one beyond the last page as `none`.
__device__ __forceinline__ int4 four_counts(const int* refs, int i, int N, int none) {
  if (i + 4 <= N && (reinterpret_cast<uintptr_t>(refs) & 15u) == 0) return *reinterpret_cast<const int4*>(refs + i);
  return make_int4(i < N ? refs[i] : none, i + 1 < N ? refs[i + 1] : none, i + 2 < N ? refs[i + 2] : none, i + 3 < N ? refs[i + 3] : none);
}

// ---- fork ------------------------------------------------------------------------------------
__device__ __forceinline__ int pages_of(int len, int page) { return len / page + (len % page != 0); }   // (any length, also one that no table holds)

// A CTA per pair: the new row i in `staged` [n, W] and its length (-1: the pair is skipped), the counts of what is taken and let go. The table is only
// read here, so that a row may be both a source and a destination (every pair sees the table as it was).
__global__ void fork_stage_kernel(const int* __restrict__ table, const int* __restrict__ lens, int* refs, const int* __restrict__ src,
                                  const int* __restrict__ dst, int n, int R, int W, int N, int page, int* __restrict__ staged, int* __restrict__ staged_len) {
  __shared__ int again;
  griddep_wait();
  griddep_launch_dependents();
  const int i = blockIdx.x, s = src[i], d = dst[i];
  if (threadIdx.x == 0) again = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < i; j += blockDim.x)
    if (dst[j] == d && src[j] >= 0 && src[j] < R) again = 1;   // of several pairs with one destination the first one inside the table counts
  __syncthreads();
  if (again || s < 0 || s >= R || d < 0 || d >= R) {
    if (threadIdx.x == 0) staged_len[i] = -1;
    return;
  }
  const int len = max(0, lens[s]), held = pages_of(len, page);
  for (int w = threadIdx.x; w < W; w += blockDim.x) {
    const int old = table[static_cast<size_t>(d) * W + w];
    if (old >= 0 && old < N) atomicAdd(refs + old, -1);
    const int take = w < held ? table[static_cast<size_t>(s) * W + w] : -1;
    if (take >= 0 && take < N) atomicAdd(refs + take, 1);
    staged[static_cast<size_t>(i) * W + w] = take;
  }
  if (threadIdx.x == 0) staged_len[i] = len;
}
__global__ void fork_store_kernel(int* __restrict__ table, int* __restrict__ lens, const int* __restrict__ dst, int W, const int* __restrict__ staged,
                                  const int* __restrict__ staged_len) {
  griddep_wait();
  griddep_launch_dependents();
  const int i = blockIdx.x, len = staged_len[i];
  if (len < 0) return;
  const int d = dst[i];
  for (int w = threadIdx.x; w < W; w += blockDim.x) table[static_cast<size_t>(d) * W + w] = staged[static_cast<size_t>(i) * W + w];
  if (threadIdx.x == 0) lens[d] = len;
}

// Both at once, by one CTA, for as many rows as its shared memory holds (four rows of a few pages: 2.2 us for 3.6, and a launch less).
constexpr int kForkFew = 256, kForkEntries = 8192;   // pairs, entries
__global__ void __launch_bounds__(kPlanThreads) fork_few_kernel(int* table, int* lens, int* refs, const int* __restrict__ src, const int* __restrict__ dst, int n,
                                                                int R, int W, int N, int page) {
  __shared__ int staged[kForkEntries], s_len[kForkFew];
  griddep_wait();
  griddep_launch_dependents();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = src[i], d = dst[i];
    bool ok = s >= 0 && s < R && d >= 0 && d < R;
    for (int j = 0; j < i && ok; ++j) ok = dst[j] != d || src[j] < 0 || src[j] >= R;   // of several pairs with one destination the first one inside the table counts
    s_len[i] = ok ? max(0, lens[s]) : -1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * W; e += kPlanThreads) {
    const int i = e / W, w = e - i * W, len = s_len[i];
    if (len < 0) continue;
    const int old = table[static_cast<size_t>(dst[i]) * W + w], take = w < pages_of(len, page) ? table[static_cast<size_t>(src[i]) * W + w] : -1;
    if (old != take) {
      if (old >= 0 && old < N) atomicAdd(refs + old, -1);
      if (take >= 0 && take < N) atomicAdd(refs + take, 1);
    }
    staged[e] = take;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * W; e += kPlanThreads) {
    const int i = e / W;
    if (s_len[i] >= 0) table[static_cast<size_t>(dst[i]) * W + e - i * W] = staged[e];
  }
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (s_len[i] >= 0) lens[dst[i]] = s_len[i];
}

// ---- trim ------------------------------------------------------------------------------------
__global__ void trim_kernel(int* __restrict__ table, int* __restrict__ lens, int* refs, const int* __restrict__ rows, const int* __restrict__ to, int R, int W,
                            int N, int page) {
  griddep_wait();
  griddep_launch_dependents();
  const int r = rows ? rows[blockIdx.x] : blockIdx.x;
  if (r < 0 || r >= R) return;
  const int want = to ? to[blockIdx.x] : 0;
  if (want < 0) return;   // this row stays as it is
  const int len = min(max(0, lens[r]), want), keep = min(W, pages_of(len, page));
  for (int w = keep + threadIdx.x; w < W; w += blockDim.x) {
    // (exchanged, so that a row named twice lets go of its pages once)
    const int old = atomicExch(table + static_cast<size_t>(r) * W + w, -1);
    if (old >= 0 && old < N) atomicAdd(refs + old, -1);
  }
  __syncthreads();
  if (threadIdx.x == 0) atomicMin(lens + r, want);
}

// ---- room for more tokens --------------------------------------------------------------------
// One CTA plans: which rows write into a page that others hold (they get a copy; if all its holders write, the first row keeps the page), how
// many fresh pages each row needs, and which free pages they are. moves[k] = {from, to, tokens, 0} for the copies, *n_moves their number.
// If there are too few pages (1), a row becomes too long for the table (2) or has no page for its last token (3: its length went on after a call that
// found no room, and pages behind the gap would be attended as if the gap held keys), nothing is changed: *status says so and *n_moves is zero.
struct RowPlan {
  int copy;         // the page that is copied, or -1
  int held, need;   // entries [held, need) are given fresh pages
  int first;        // the row's first request among all
};
struct ReserveParams {
  int* table;
  const int* lens;
  int* refs;
  const int* counts;   // nullable [R]; else `count` for every row
  int count, R, W, N, page;
  int* asks;           // [N] scratch: how many rows write into a shared page
  int* lowest;         // [N] scratch: the first of them
  int* fresh;          // [N] scratch: free pages in ascending order (as many as are asked for)
  RowPlan* rows;       // [R] scratch
  int4* moves;         // [R]
  int* n_moves;
  int* status;
  int keep;            // whether *status is raised to this outcome, but never lowered
};
__global__ void __launch_bounds__(kPlanThreads) reserve_plan_kernel(const ReserveParams p) {
  __shared__ int warp_sums[32];
  __shared__ int s_too_long, s_gap, s_moves, s_n_long, s_long[kLongRows];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x;
  if (tid == 0) { s_too_long = 0; s_gap = 0; s_moves = 0; s_n_long = 0; }
  const int each = (p.R + kPlanThreads - 1) / kPlanThreads;   // thread t plans rows [t * each, (t + 1) * each)
  const int r0 = min(p.R, tid * each), r1 = min(p.R, r0 + each);
  auto entry = [&](int r, int w) -> int& { return p.table[static_cast<size_t>(r) * p.W + w]; };
  auto count_of = [&](int r) { return p.counts ? max(0, p.counts[r]) : p.count; };
  // ---- shared pages that are written into ----
  bool gap = false;
  for (int r = r0; r < r1; ++r) {
    const int c = count_of(r), len = max(0, p.lens[r]);
    int copy = -1;
    if (c > 0 && len > 0 && (len - 1) / p.page < p.W) {
      const int pg = entry(r, (len - 1) / p.page);   // of the last token
      gap |= pg < 0;
      if (len % p.page != 0 && pg >= 0 && pg < p.N && p.refs[pg] > 1) copy = pg;
    }
    p.rows[r].copy = copy;
    if (copy >= 0) { p.asks[copy] = 0; p.lowest[copy] = 0x7fffffff; }
  }
  __syncthreads();
  for (int r = r0; r < r1; ++r) {
    const int copy = p.rows[r].copy;
    if (copy >= 0) { atomicAdd(p.asks + copy, 1); atomicMin(p.lowest + copy, r); }
  }
  __syncthreads();
  // ---- requests, in the order of the rows ----
  int sum = 0, total;
  for (int r = r0; r < r1; ++r) {
    RowPlan plan = p.rows[r];
    const int c = count_of(r), len = max(0, p.lens[r]);
    if (plan.copy >= 0 && __ldcg(p.asks + plan.copy) == p.refs[plan.copy] && __ldcg(p.lowest + plan.copy) == r) plan.copy = -1;
    const long long need = c > 0 ? (static_cast<long long>(len) + c + p.page - 1) / p.page : 0;
    if (need > p.W) atomicExch(&s_too_long, 1);
    plan.need = static_cast<int>(min(need, static_cast<long long>(p.W)));
    plan.held = min(plan.need, pages_of(len, p.page));
    while (plan.held < plan.need && entry(r, plan.held) >= 0) ++plan.held;   // room from an earlier call
    plan.first = sum;
    sum += (plan.copy >= 0) + plan.need - plan.held;
    p.rows[r] = plan;
  }
  if (gap) atomicExch(&s_gap, 1);
  const int before = block_scan(sum, warp_sums, total) - sum;
  // ---- the lowest free pages, as many as are asked for ----
  int found = 0;
  for (int i0 = 0; i0 < p.N && found < total; i0 += 4 * kPlanThreads) {
    const int i = i0 + 4 * tid;
    const int4 c = four_counts(p.refs, i, p.N, 1);
    const int here = (c.x <= 0) + (c.y <= 0) + (c.z <= 0) + (c.w <= 0);
    int in_tile, k = found + block_scan(here, warp_sums, in_tile) - here;
    if (c.x <= 0 && k < total) p.fresh[k] = i;
    k += c.x <= 0;
    if (c.y <= 0 && k < total) p.fresh[k] = i + 1;
    k += c.y <= 0;
    if (c.z <= 0 && k < total) p.fresh[k] = i + 2;
    k += c.z <= 0;
    if (c.w <= 0 && k < total) p.fresh[k] = i + 3;
    found += in_tile;
  }
  const bool fits = s_too_long == 0 && s_gap == 0 && total <= found;
  __syncthreads();
  if (fits) {
    for (int r = r0; r < r1; ++r) {
      const RowPlan plan = p.rows[r];
      const int first = before + plan.first;
      p.rows[r].first = first;
      if (plan.copy >= 0) {
        const int to = p.fresh[first], len = p.lens[r];
        p.moves[atomicAdd(&s_moves, 1)] = make_int4(plan.copy, to, len % p.page, 0);
        entry(r, len / p.page) = to;
        atomicAdd(p.refs + plan.copy, -1);
        p.refs[to] = 1;
      }
    }
    __syncthreads();
    auto give = [&](int r, const RowPlan& plan, int thread, int threads) {
      const int first = plan.first + (plan.copy >= 0) - plan.held;
      for (int w = plan.held + thread; w < plan.need; w += threads) {
        const int to = p.fresh[first + w];
        entry(r, w) = to;
        p.refs[to] = 1;
      }
    };
    for (int r = tid >> 5; r < p.R; r += kPlanThreads / 32) {   // a row by a warp; a prompt (as many as are remembered) by the CTA
      const RowPlan plan = p.rows[r];
      int place = kLongRows;
      if (plan.need - plan.held > 256) {
        if ((tid & 31) == 0) place = atomicAdd(&s_n_long, 1);
        place = __shfl_sync(0xffffffffu, place, 0);
      }
      if (place < kLongRows) s_long[place] = r;
      else give(r, plan, tid & 31, 32);
    }
    __syncthreads();
    for (int i = 0; i < min(s_n_long, kLongRows); ++i) give(s_long[i], p.rows[s_long[i]], tid, kPlanThreads);
  }
  __syncthreads();
  if (tid == 0) {
    *p.n_moves = s_moves;
    const int outcome = s_too_long ? 2 : s_gap ? 3 : total > found ? 1 : 0;
    *p.status = p.keep ? max(*p.status, outcome) : outcome;
  }
}

// ---- compaction ------------------------------------------------------------------------------
// One CTA plans: the k-th page in use behind the first `live` ones moves to the k-th free page among them; the least that can move. remap[page] is
// where a page is afterwards.
struct CompactParams {
  const int* refs;
  int* refs_out;    // may be refs
  int N, page;
  int* from;        // [N] scratch
  int* to;          // [N] scratch
  int* remap;       // [N]
  int4* moves;      // [N]
  int* n_moves;
};
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactParams p) {
  __shared__ int warp_sums[32];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x;
  int n = 0, live;
#pragma unroll 4
  for (int i = 4 * tid; i < p.N; i += 4 * kPlanThreads) {
    const int4 c = four_counts(p.refs, i, p.N, 0);
    n += (c.x > 0) + (c.y > 0) + (c.z > 0) + (c.w > 0);
  }
  block_scan(n, warp_sums, live);
  int movers = 0, holes = 0;
  for (int base = 0; base < p.N; base += 4 * kPlanThreads) {
    const int i = base + 4 * tid;
    const int4 c = four_counts(p.refs, i, p.N, i >= live ? 0 : 1);   // (pages that are not there neither move nor are holes)
    const int count[4] = {c.x, c.y, c.z, c.w};
    int here = 0, in_tile;   // pages that move, holes << 16
#pragma unroll
    for (int e = 0; e < 4; ++e) here += count[e] > 0 && i + e >= live && i + e < p.N ? 1 : count[e] <= 0 && i + e < live ? 1 << 16 : 0;
    const int front = block_scan(here, warp_sums, in_tile) - here;
    int km = movers + (front & 0xffff), kh = holes + (front >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e >= p.N) break;
      if (count[e] > 0 && i + e >= live) p.from[km++] = i + e;
      if (count[e] <= 0 && i + e < live) p.to[kh++] = i + e;
      p.remap[i + e] = i + e;
      if (p.refs_out != p.refs) p.refs_out[i + e] = count[e];
    }
    movers += in_tile & 0xffff;
    holes += in_tile >> 16;
  }
  __syncthreads();
  for (int k = tid; k < movers; k += kPlanThreads) {   // as many holes as movers
    const int from = p.from[k], to = p.to[k];
    p.moves[k] = make_int4(from, to, p.page, 0);
    p.remap[from] = to;
    p.refs_out[to] = p.refs[from];
    p.refs_out[from] = 0;
  }
  if (tid == 0) *p.n_moves = movers;
}

// ---- moves -----------------------------------------------------------------------------------
constexpr int kMoveTensors = 16;      // per launch
constexpr int kMoveThreads = 256;
constexpr int kMoveChunk = 16384;     // bytes that a CTA copies at a time

struct MoveTensor {
  uint8_t* base;
  long long layer_stride, page_bytes;   // bytes
  int layers, row_bytes;                // row: a token's
  int chunks;                           // per page
  int units;                            // layers * chunks, those of the tensors in front added
};
struct MoveParams {
  const int4* moves;    // {from, to, tokens, -}
  const int* n_moves;   // nullable: n
  int n, N, tensors;
  const int* table;     // nullable: [entries] -> table_out by remap
  int* table_out;
  const int* remap;
  int entries;
  MoveTensor t[kMoveTensors];
};

// Units of work: a chunk of a page of a layer of a tensor of a move. Vec: the widest type that all addresses and rows are multiples of.
template <typename Vec>
__global__ void __launch_bounds__(kMoveThreads) move_pages_kernel(const __grid_constant__ MoveParams p) {
  griddep_wait();
  griddep_launch_dependents();
  for (int i = blockIdx.x * kMoveThreads + threadIdx.x; i < p.entries; i += gridDim.x * kMoveThreads) {
    const int pg = p.table[i];
    p.table_out[i] = pg >= 0 && pg < p.N ? p.remap[pg] : pg;
  }
  const int n = p.n_moves ? *p.n_moves : p.n;
  const int per_move = p.t[p.tensors - 1].units;
  const long long units = static_cast<long long>(n) * per_move;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int m = static_cast<int>(u / per_move);
    int rest = static_cast<int>(u - static_cast<long long>(m) * per_move), i = 0;
    while (rest >= p.t[i].units) ++i;
    if (i > 0) rest -= p.t[i - 1].units;
    const MoveTensor& t = p.t[i];
    const int layer = rest / t.chunks, chunk = rest - layer * t.chunks;
    const int4 move = p.moves[m];
    if (move.x < 0 || move.x >= p.N || move.y < 0 || move.y >= p.N) continue;
    const long long bytes = min(t.page_bytes, static_cast<long long>(move.z) * t.row_bytes);
    const long long begin = static_cast<long long>(chunk) * kMoveChunk, size = min(static_cast<long long>(kMoveChunk), bytes - begin);
    if (size <= 0) continue;
    const uint8_t* layer_base = t.base + layer * t.layer_stride;
    const Vec* src = reinterpret_cast<const Vec*>(layer_base + move.x * t.page_bytes + begin);
    Vec* dst = reinterpret_cast<Vec*>(const_cast<uint8_t*>(layer_base) + move.y * t.page_bytes + begin);
    const int vecs = static_cast<int>(size / static_cast<int>(sizeof(Vec)));
    constexpr int kFlight = sizeof(Vec) == 16 ? kMoveChunk / 16 / kMoveThreads : 8;
    for (int v0 = threadIdx.x; v0 < vecs; v0 += kMoveThreads * kFlight) {
      Vec x[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        if (v0 + j * kMoveThreads < vecs) x[j] = src[v0 + j * kMoveThreads];
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        if (v0 + j * kMoveThreads < vecs) dst[v0 + j * kMoveThreads] = x[j];
    }
  }
}

// Mirrored by ops.py: a tensor whose pages move.
struct PageTensor {
  void* base;
  long long layers, layer_stride, page_bytes, row_bytes;
};

static int move_pages(MoveParams p, const PageTensor* tensors, int n_tensors, long long most_moves, cudaStream_t s) {
  long long align = 16;
  for (int i = 0; i < n_tensors; ++i) {
    const PageTensor& t = tensors[i];
    B200_REQUIRE(t.base != nullptr && t.layers >= 1 && t.layers < 1 << 20 && t.page_bytes >= 1 && t.row_bytes >= 1 && t.row_bytes <= t.page_bytes &&
                 t.page_bytes < 1LL << 40, "pages: bad tensor %d", i);
    for (long long x : {static_cast<long long>(reinterpret_cast<uintptr_t>(t.base)), t.layer_stride, t.page_bytes, t.row_bytes})
      while (x % align) align /= 2;
  }
  for (int first = 0; first == 0 || first < n_tensors; first += kMoveTensors) {
    p.tensors = n_tensors - first < kMoveTensors ? n_tensors - first : kMoveTensors;
    long long units = 0;
    for (int i = 0; i < p.tensors; ++i) {
      const PageTensor& t = tensors[first + i];
      const long long chunks = (t.page_bytes + kMoveChunk - 1) / kMoveChunk;
      units += t.layers * chunks;
      B200_REQUIRE(units <= 0x7fffffff, "pages: too many layers and bytes");
      p.t[i] = {static_cast<uint8_t*>(t.base), t.layer_stride, t.page_bytes, static_cast<int>(t.layers), static_cast<int>(t.row_bytes), static_cast<int>(chunks),
                static_cast<int>(units)};
    }
    if (p.tensors == 0) { p.tensors = 1; memset(p.t, 0, sizeof(p.t[0])); }   // the table alone
    long long want = units * most_moves, ctas = 8LL * sm_count();
    if (p.entries > 0 && want < (p.entries + kMoveThreads - 1) / kMoveThreads) want = (p.entries + kMoveThreads - 1) / kMoveThreads;
    if (want < 1) want = 1;
    if (ctas > want) ctas = want;
    switch (align) {
      case 16: B200_CHECK_CUDA(launch_pdl(move_pages_kernel<uint4>, static_cast<unsigned>(ctas), kMoveThreads, 0, s, p)); break;
      case 8: B200_CHECK_CUDA(launch_pdl(move_pages_kernel<uint2>, static_cast<unsigned>(ctas), kMoveThreads, 0, s, p)); break;
      case 4: B200_CHECK_CUDA(launch_pdl(move_pages_kernel<uint32_t>, static_cast<unsigned>(ctas), kMoveThreads, 0, s, p)); break;
      case 2: B200_CHECK_CUDA(launch_pdl(move_pages_kernel<uint16_t>, static_cast<unsigned>(ctas), kMoveThreads, 0, s, p)); break;
      default: B200_CHECK_CUDA(launch_pdl(move_pages_kernel<uint8_t>, static_cast<unsigned>(ctas), kMoveThreads, 0, s, p)); break;
    }
    p.entries = 0;
  }
  return kOk;
}

}  // namespace b200

using namespace b200;

// Rows dst[i] become copies of rows src[i] (int32 [n] on the device; all sources are read as they were before the call): they let go of
// their pages and hold the ceil(len / page) first ones of the source. Pairs out of range are skipped, and of the others all but the first of a
// destination. scratch: int32 [n * (W + 1)]; unused, and may be null, for at most 256 pairs and 8192 entries (n * W).
B200_API int b200_fork_pages(int* table, int* lens, int* refs, const int* src, const int* dst, int n, int R, int W, int N, int page, int* scratch,
                             void* stream) {
  B200_REQUIRE(n >= 0 && R >= 1 && W >= 1 && N >= 1 && page >= 1, "fork_pages: bad sizes");
  if (n == 0) return kOk;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n <= kForkFew && static_cast<long long>(n) * W <= kForkEntries) {
    B200_CHECK_CUDA(launch_pdl(fork_few_kernel, 1, kPlanThreads, 0, s, table, lens, refs, src, dst, n, R, W, N, page));
    return kOk;
  }
  const int threads = W > 256 ? 256 : 128;
  int* staged_len = scratch + static_cast<size_t>(n) * W;
  B200_CHECK_CUDA(launch_pdl(fork_stage_kernel, n, threads, 0, s, table, lens, refs, src, dst, n, R, W, N, page, scratch, staged_len));
  B200_CHECK_CUDA(launch_pdl(fork_store_kernel, n, threads, 0, s, table, lens, dst, W, scratch, staged_len));
  return kOk;
}

// Row rows[i] (null: row i) keeps the pages of its first min(len, to[i]) tokens (null: none) and that length; to[i] < 0 leaves it alone.
B200_API int b200_trim_pages(int* table, int* lens, int* refs, const int* rows, const int* to, int n, int R, int W, int N, int page, void* stream) {
  B200_REQUIRE(n >= 0 && R >= 1 && W >= 1 && N >= 1 && page >= 1, "trim_pages: bad sizes");
  if (n == 0) return kOk;
  B200_CHECK_CUDA(launch_pdl(trim_kernel, n, 128, 0, static_cast<cudaStream_t>(stream), table, lens, refs, rows, to, R, W, N, page));
  return kOk;
}

// int32 words of scratch that b200_reserve_pages (8 R + 3 N + 1) and b200_compact_pages (7 N + 1) need (16-byte aligned).
B200_API long long b200_pages_scratch(int R, int N) { return 8LL * R + 8LL * N + 16; }

// Room for counts[r] (null: count) more tokens in every row, see ReserveParams; the copies are made in `tensors`. keep: *status becomes the larger of
// what it was and this call's outcome.
B200_API int b200_reserve_pages(int* table, const int* lens, int* refs, const int* counts, int count, int R, int W, int N, int page, const void* tensors,
                                int n_tensors, int* scratch, int* status, int keep, void* stream) {
  B200_REQUIRE(R >= 1 && W >= 1 && N >= 1 && page >= 1 && count >= 0 && n_tensors >= 0, "reserve_pages: bad sizes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ReserveParams p;
  p.table = table; p.lens = lens; p.refs = refs; p.counts = counts; p.count = count; p.R = R; p.W = W; p.N = N; p.page = page;
  p.moves = reinterpret_cast<int4*>(scratch);
  p.rows = reinterpret_cast<RowPlan*>(scratch + 4 * static_cast<size_t>(R));
  p.asks = scratch + 8 * static_cast<size_t>(R);
  p.lowest = p.asks + N;
  p.fresh = p.lowest + N;
  p.n_moves = p.fresh + N;
  p.status = status; p.keep = keep;
  B200_CHECK_CUDA(launch_pdl(reserve_plan_kernel, 1, kPlanThreads, 0, s, p));
  if (n_tensors == 0) return kOk;
  MoveParams m;
  memset(&m, 0, sizeof(m));
  m.moves = p.moves; m.n_moves = p.n_moves; m.N = N;
  return move_pages(m, static_cast<const PageTensor*>(tensors), n_tensors, R, s);
}

// The pages in use move to the front, see CompactParams; table_out and refs_out may be the tables that are read.
B200_API int b200_compact_pages(const int* table, int* table_out, const int* refs, int* refs_out, int R, int W, int N, int page, const void* tensors, int n_tensors,
                                int* scratch, void* stream) {
  B200_REQUIRE(R >= 1 && W >= 1 && N >= 1 && page >= 1 && n_tensors >= 0 && static_cast<long long>(R) * W < 1LL << 30, "compact_pages: bad sizes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CompactParams p;
  p.refs = refs; p.refs_out = refs_out; p.N = N; p.page = page;
  p.moves = reinterpret_cast<int4*>(scratch);
  p.from = scratch + 4 * static_cast<size_t>(N);
  p.to = p.from + N;
  p.remap = p.to + N;
  p.n_moves = p.remap + N;
  B200_CHECK_CUDA(launch_pdl(compact_plan_kernel, 1, kPlanThreads, 0, s, p));
  MoveParams m;
  memset(&m, 0, sizeof(m));
  m.moves = p.moves; m.n_moves = p.n_moves; m.N = N; m.table = table; m.table_out = table_out; m.remap = p.remap; m.entries = R * W;
  return move_pages(m, static_cast<const PageTensor*>(tensors), n_tensors, N / 2 + 1, s);
}

// Pages moves[k].x -> moves[k].y (int32 [n, 4]: from, to, tokens, unused) of all tensors.
B200_API int b200_copy_pages(const void* tensors, int n_tensors, const void* moves, int n, int N, void* stream) {
  B200_REQUIRE(n >= 0 && N >= 1 && n_tensors >= 0, "copy_pages: bad sizes");
  if (n == 0 || n_tensors == 0) return kOk;
  MoveParams m;
  memset(&m, 0, sizeof(m));
  m.moves = static_cast<const int4*>(moves); m.n = n; m.N = N;
  return move_pages(m, static_cast<const PageTensor*>(tensors), n_tensors, n, static_cast<cudaStream_t>(stream));
}
