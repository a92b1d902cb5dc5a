// Attention over a paged cache for a batch whose sequences begin with the same keys: the shared keys are read once for the rows of all
// sequences, everybody's own keys once for the rows of that sequence, and the partial results are merged.
//
//   n = kv_len[b] - tokens + t + 1 keys are visible to query token t of sequence b (the new tokens are in the cache)
//   o = sum_{j < n} p_j v_j / sum_{j < n} p_j,  p_j = exp(scale q . k_j - m)      (zeros and a log-sum-exp of -inf for n <= 0)
//
// A row (token and query head) is split over disjoint ranges of keys. Every range leaves its normalised output o_i and its
// log-sum-exp l_i; the whole is sum_i exp(l_i - l) o_i with l = log sum_i exp(l_i).
//
// This file holds the kernel on warp-level products (m16n8k16) with the keys on the wide side: S^T [16 keys, 8 rows] = K Q^T and O^T [D, 8 rows]
// += V^T P^T, for 8, 16 or 32 rows that share a KV head per CTA. Each of the four warps streams its own slices of 16 keys through a
// private ring of three (cp.async, no barrier of the CTA in the loop), its reference, sum and output in registers; the reference is the
// maximum when it was last raised, and a slice in which no row's score lies more than 8 above it rescales nothing (one vote; 64 / 8 heads, 32768 + 1024
// keys: 93.7 -> 92.7 us). It takes the own keys of every sequence and, while the rows per KV head are few,
// the shared keys; both in one launch, the shared ones first because their CTAs run longest. What bounds it is the read of the keys, and in short
// sequences the latency of starting and merging. The first form, with the rows on the 16 rows of the product, took 1136 instructions a
// slice and fetched them from beyond the instruction cache (86 us for the own keys of 64 sequences of 544 keys, 8 KV heads).
// Many rows go to the tensor-core kernel in shared_prefix_sm100.cu.
//
// A sequence that does not reach beyond the shared keys (a row of the batch that holds none, or a shorter one) is attended by
// itself, over its own page table from key 0 on, so that no key of the shared range is ever masked for a row.
// Page numbers outside the cache and table columns outside the table are not read; their keys count as zeros.
#include "b200/host.h"
#include "b200/elem.cuh"
#include "b200/mma_sync.cuh"
#include "b200/primitives.cuh"
#include "b200/shared_prefix.cuh"

#include <cstring>

namespace b200 {

constexpr int kSpanThreads = 128;
constexpr int kSpanSlice = 16;   // keys per slice of a warp
constexpr int kSpanRing = 3;     // slices in flight per warp
constexpr float kSpanRaise = 8.f;   // a score (as a power of two) so far above its row's reference raises it; weights are up to 2^8

constexpr int kSpanMostRows = 32;   // per CTA
template <int D>
constexpr int span_smem() {         // the rings; in the end the four warps' maxima, sums and outputs (rows D + 4 floats apart)
  constexpr int rings = 4 * kSpanRing * 2 * kSpanSlice * D * 2, merge = 4 * kSpanMostRows * (2 + D + 4) * 4;
  return (rings > merge ? rings : merge) + kSpanMostRows * D * 2 /*queries*/;
}

__device__ __forceinline__ float span_exp2(float x) {   // one instruction; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Whether a slice of values holds one that is not finite.
template <bool BF16, int D>
__device__ __forceinline__ bool slice_has_nonfinite(uint32_t vs, int lane) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < kSpanSlice * D * 2 / 512; ++i) {
    uint32_t x[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(vs + (i * 32 + lane) * 16));
    constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;   // the exponent's bits
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= ((x[j] & e) == e || (x[j] >> 16 & e) == e) ? 1u : 0u;
  }
  return __any_sync(0xffffffffu, bad != 0u);
}

// The queries of a CTA's rows (row r: query token first_token + (row0 + r) / G) to shared memory: 16-byte chunk c of row r lies at chunk c ^ (r & 7).
// Rows that do not exist are zero. Commits a group.
template <int D, int NB>
__device__ __forceinline__ void span_fetch_queries(const SharedPrefixParams& p, uint8_t* smem, int kvh, int first_token, int row0, int nrows) {
  constexpr int kChunks = D / 8, kLaneRows = 32 / kChunks;
  const uint32_t qs = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + span_smem<D>() - kSpanMostRows * D * 2;
  const int G = p.Hq / p.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = row0 + min(lane, nrows - 1);   // lane r knows where row r lies
  const long long at = (static_cast<long long>(first_token + g / G) * p.ldq + static_cast<long long>(kvh * G + g % G) * D) * 2;
#pragma unroll
  for (int r0 = 0; r0 < NB * 8; r0 += 4 * kLaneRows) {
    const int r = r0 + warp * kLaneRows + lane / kChunks, chunk = lane % kChunks;
    const long long row_at = __shfl_sync(0xffffffffu, at, r & 31);
    if (r < NB * 8) cp_async_16(qs + r * D * 2 + ((chunk ^ (r & 7)) * 16), static_cast<const uint8_t*>(p.q) + row_at + chunk * 16, r < nrows ? 16 : 0);
  }
  cp_async_commit();
}

// Where the slice of keys from token `tok` on (a multiple of 16) begins in the cache, in slices; -1: nowhere. (Pages of a multiple of 16 keys.)
__device__ __forceinline__ int span_slice_at(const SharedPrefixParams& p, const int* table, int width, unsigned tok) {
  const unsigned w = tok / p.page;
  const int blk = w < static_cast<unsigned>(width) ? table[w] : -1;
  return blk >= 0 && blk < p.num_blocks ? blk * (p.page / kSpanSlice) + static_cast<int>(tok % p.page) / kSpanSlice : -1;
}

// One CTA: 8 NB rows of KV head `kvh` from row `row0` of a group of `rows`, over keys [t0, t1) of the pages in `table`. A row r of
// the group is query token first_token + r / G, head kvh * G + r % G. `own`: the rows are one sequence's and see keys below `limit0` + r / G.
// The rows' queries are on their way (span_fetch_queries). `ahead`: this lane's span_slice_at of slice warp + 4 * lane counted from key `ahead_base` on, where that has been read already.
template <bool BF16, int D, int NB>
__device__ __forceinline__ void span_body(const SharedPrefixParams& p, uint8_t* smem, int kvh, int first_token, int row0, int rows, const int* table,
                                          int width, int t0, int t1, bool own, int limit0, int split, int ahead_base, int ahead) {
  constexpr int kKK = D / 16, kRowBytes = D * 2, kChunks = D / 8, kSliceBytes = kSpanSlice * kRowBytes;
  constexpr int kLaneRows = 32 / kChunks;                  // keys that a warp copies with one instruction
  constexpr int kCopies = kSpanSlice / kLaneRows;
  const int G = p.Hq / p.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = lane >> 2, col = (lane & 3) * 2;         // of an accumulator tile: key (or output column), row of the group and the next
  const int nrows = min(NB * 8, rows - row0);
  auto row_id = [&](int r) {   // of row r of this CTA, among all rows of the call
    const int g = row0 + r;
    return static_cast<size_t>(first_token + g / G) * p.Hq + kvh * G + g % G;
  };
  if (t0 >= t1) {
    cp_async_wait<0>();
    for (int r = threadIdx.x; r < nrows; r += kSpanThreads) p.lse_part[row_id(r) * p.S + split] = -INFINITY;
    return;
  }

  // ---- this warp's ring: slot s holds K at +0 and V behind it; slices begin at multiples of 16 keys ----
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (kSpanRing * 2 * kSliceBytes);
  const uint8_t *kc = static_cast<const uint8_t*>(p.k_cache), *vc = static_cast<const uint8_t*>(p.v_cache);
  const int base = t0 & ~(kSpanSlice - 1);
  const int n_slices = (t1 - base + kSpanSlice - 1) / kSpanSlice;
  const int mine = n_slices > warp ? (n_slices - warp + 3) / 4 : 0;   // slices warp, warp + 4, ...
  const bool page_fast = p.page % kSpanSlice == 0;                    // a slice lies in one page
  auto page_of = [&](int tok) -> int {   // -1: there is none
    const int w = tok / p.page;
    const int blk = w < width ? table[w] : -1;
    return blk < p.num_blocks ? blk : -1;
  };
  const int hi = lane / kChunks, chunk = lane % kChunks;
  const size_t token_bytes = static_cast<size_t>(p.Hkv) * kRowBytes, step = token_bytes * kLaneRows;
  const size_t lane_off = hi * token_bytes + static_cast<size_t>(kvh) * kRowBytes + chunk * 16;
  // lane i knows where slices i and i + 32 of a window of this warp's slices begin
  auto slice_at = [&](int j) { return span_slice_at(p, table, width, static_cast<unsigned>(base) + (warp + 4 * (j + lane)) * kSpanSlice); };
  int window = !page_fast ? 0 : base == ahead_base ? ahead : slice_at(0);
  int next = page_fast && mine > 32 ? slice_at(32) : 0;
  auto load_slice = [&](int j) {   // always commits a group, so that the counting stays uniform
    if (j < mine) {
      const int st0 = base + (warp + 4 * j) * kSpanSlice;
      const uint32_t slot = ring + (j % kSpanRing) * (2 * kSliceBytes);
      if (page_fast) {
        if (j > 0 && j % 32 == 0) {
          window = next;
          if (j + 32 < mine) next = slice_at(j + 32);
        }
        const int at_slice = __shfl_sync(0xffffffffu, window, j % 32);
        const bool all = at_slice >= 0 && st0 >= t0 && st0 + kSpanSlice <= t1;
        const size_t off = static_cast<size_t>(max(at_slice, 0)) * (kSpanSlice * token_bytes) + lane_off;
        const uint8_t *ks = kc + off, *vs = vc + off;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int tok_in = i * kLaneRows + hi, tok = st0 + tok_in;
          const uint32_t at = slot + tok_in * kRowBytes + ((chunk ^ (tok_in & 7)) * 16);
          const int bytes = all || (at_slice >= 0 && tok >= t0 && tok < t1) ? 16 : 0;   // (the address is inside the page either way)
          cp_async_16(at, ks + i * step, bytes);
          cp_async_16(at + kSliceBytes, vs + i * step, bytes);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kCopies; ++i) {
          const int tok_in = i * kLaneRows + hi, tok = st0 + tok_in;
          const int page = tok >= t0 && tok < t1 ? page_of(tok) : -1;
          const size_t off = page >= 0 ? (static_cast<size_t>(page) * p.page + tok % p.page) * token_bytes + lane_off - hi * token_bytes : 0;
          const uint32_t at = slot + tok_in * kRowBytes + ((chunk ^ (tok_in & 7)) * 16);
          cp_async_16(at, kc + off, page >= 0 ? 16 : 0);
          cp_async_16(at + kSliceBytes, vc + off, page >= 0 ? 16 : 0);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kSpanRing - 1; ++j) load_slice(j);

  // ---- Q^T fragments: row nb * 8 + lane / 4, elements 16 kk + col, + 1 and eight further ----
  uint32_t qb[NB][kKK][2];
  cp_async_wait<kSpanRing - 1>();   // (all groups but the slices')
  __syncthreads();
  const uint32_t qs = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + span_smem<D>() - kSpanMostRows * kRowBytes;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int kk = 0; kk < kKK; kk += 2)
      ldmatrix_x4(qs + (nb * 8 + (lane & 7)) * kRowBytes + (((2 * kk + (lane >> 3)) ^ (lane & 7)) * 16), qb[nb][kk][0], qb[nb][kk][1], qb[nb][kk + 1][0],
                  qb[nb][kk + 1][1]);
  int limit[NB][2];   // of rows nb * 8 + col, + 1
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) limit[nb][h] = own ? min(t1, limit0 + (row0 + nb * 8 + col + h) / G) : t1;
  const int safe = own ? min(t1, limit0 + row0 / G) : t1;   // keys below are visible to every row of this CTA

  float m_run[NB][2], l_run[NB][2], oacc[NB][kKK][4];   // of rows col, col + 1; l_run: this lane's keys; oacc: columns 16 dn + row (and + 8)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) { m_run[nb][h] = -INFINITY; l_run[nb][h] = 0.f; }
#pragma unroll
    for (int i = 0; i < kKK; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) oacc[nb][i][e] = 0.f;
  }
  const int mi = lane >> 3, mr = lane & 7;
  const uint32_t k_row = ((mi & 1) * 8 + mr) * kRowBytes, v_row = ((mi >> 1) * 8 + mr) * kRowBytes;
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    load_slice(j + kSpanRing - 1);       // into the slot of the iteration before
    cp_async_wait<kSpanRing - 1>();      // this lane's part of slice j has landed; the barrier covers the other lanes
    __syncwarp();
    const uint32_t ks = ring + (j % kSpanRing) * (2 * kSliceBytes), vs = ks + kSliceBytes;
    const int st0 = base + (warp + 4 * j) * kSpanSlice;
    // ---- S^T of 16 keys; for one block of rows two sums, so that no product waits for the one before it ----
    constexpr int kSums = NB == 1 ? 2 : 1;
    float s[NB][kSums][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int x = 0; x < kSums; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nb][x][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      uint32_t a[4];
      ldmatrix_x4(ks + k_row + (((2 * kk + (mi >> 1)) ^ mr) * 16), a[0], a[1], a[2], a[3]);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) mma16816<BF16>(s[nb][kk % kSums], a, qb[nb][kk][0], qb[nb][kk][1]);
    }
    const bool whole = st0 >= t0 && st0 + kSpanSlice <= safe;
    float v[NB][4];   // keys row, row, row + 8, row + 8 of rows col, col + 1, col, col + 1
    bool raise = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[nb][e] = (kSums == 2 ? s[nb][0][e] + s[nb][kSums - 1][e] : s[nb][0][e]) * p.scale_log2e;
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = st0 + row + 8 * (e >> 1);
          if (tok < t0 || tok >= limit[nb][e & 1]) v[nb][e] = -INFINITY;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) raise |= fmaxf(v[nb][h], v[nb][h + 2]) > m_run[nb][h] + kSpanRaise;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(v[nb][h], v[nb][h + 2]);
#pragma unroll
          for (int m = 4; m < 32; m <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
          const float m_new = fmaxf(m_run[nb][h], mx);
          const float corr = m_new == -INFINITY ? 0.f : span_exp2(m_run[nb][h] - m_new);   // m_run = -inf -> 0
          m_run[nb][h] = m_new;
          l_run[nb][h] *= corr;
#pragma unroll
          for (int i = 0; i < kKK; ++i) {
            oacc[nb][i][h] *= corr;
            oacc[nb][i][2 + h] *= corr;
          }
        }
    }
    // the weights are rounded to the type of the values: the product's operand has it (each relative to itself, also those above one)
    uint32_t pb[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = span_exp2(v[nb][e] - (m_run[nb][e & 1] == -INFINITY ? 0.f : m_run[nb][e & 1]));
      l_run[nb][0] += w[0] + w[2];
      l_run[nb][1] += w[1] + w[3];
#pragma unroll
      for (int x = 0; x < 2; ++x) pb[nb][x] = movmatrix_trans(BF16 ? pack_bf16x2(w[2 * x], w[2 * x + 1]) : pack_f16x2(w[2 * x], w[2 * x + 1]));
    }
    if (!whole && own && slice_has_nonfinite<BF16, D>(vs, lane)) {
      // ---- rare: between drafted tokens a key is masked for some rows, and zero times an infinity or NaN must not reach them. Token by
      // token from the last one on: the keys that it does not see are zeroed, and the product is kept for its rows alone. ----
      const int t_first = row0 / G, t_last = (row0 + nrows - 1) / G;
#pragma unroll 1
      for (int t = t_last; t >= t_first; --t) {
        const int seen = max(0, min(kSpanSlice, min(t1, limit0 + t) - st0));
        __syncwarp();
        for (int i = seen * kChunks + lane; i < kSpanSlice * kChunks; i += 32)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs + i * 16), "r"(0u) : "memory");
        __syncwarp();
#pragma unroll
        for (int dn = 0; dn < kKK; ++dn) {
          uint32_t a[4];
          ldmatrix_x4_trans(vs + v_row + (((2 * dn + (mi & 1)) ^ mr) * 16), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float d[4] = {oacc[nb][dn][0], oacc[nb][dn][1], oacc[nb][dn][2], oacc[nb][dn][3]};
            mma16816<BF16>(d, a, pb[nb][0], pb[nb][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((row0 + nb * 8 + col + (e & 1)) / G == t) oacc[nb][dn][e] = d[e];
          }
        }
      }
    } else {
#pragma unroll
      for (int dn = 0; dn < kKK; ++dn) {
        uint32_t a[4];
        ldmatrix_x4_trans(vs + v_row + (((2 * dn + (mi & 1)) ^ mr) * 16), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16816<BF16>(oacc[nb][dn], a, pb[nb][0], pb[nb][1]);
      }
    }
    __syncwarp();   // the slot is free for the copies of the next iteration
  }
  cp_async_wait<0>();
  __syncthreads();  // all rings are idle: their memory becomes the merge area

  // ---- merge of the four warps ----
  static_assert(NB * 8 <= kSpanMostRows, "the merge area holds the rows of a CTA");
  constexpr int kRows = NB * 8, kPitch = D + 4;      // (lanes of one store are columns of four rows: 4 words apart in the banks)
  float* red_m = reinterpret_cast<float*>(smem);     // [4][rows]
  float* red_l = red_m + 4 * kRows;                  // [4][rows]
  float* red_o = red_l + 4 * kRows;                  // [4][rows][pitch]
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int m = 4; m < 32; m <<= 1) l_run[nb][h] += __shfl_xor_sync(0xffffffffu, l_run[nb][h], m);
      const int r = warp * kRows + nb * 8 + col + h;
      if (row == 0) { red_m[r] = m_run[nb][h]; red_l[r] = l_run[nb][h]; }
      float* o = red_o + r * kPitch + row;
#pragma unroll
      for (int i = 0; i < kKK; ++i) {
        o[16 * i] = oacc[nb][i][h];
        o[16 * i + 8] = oacc[nb][i][2 + h];
      }
    }
  __syncthreads();
  constexpr int kVecs = D / 4, kWarpRows = 32 / kVecs;
  const long long my_id = static_cast<long long>(row_id(min(lane, nrows - 1)));   // lane r knows where row r goes
#pragma unroll 2
  for (int r0 = warp * kWarpRows; r0 < nrows; r0 += 4 * kWarpRows) {
    const int r = r0 + lane / kVecs, c = lane % kVecs;
    const size_t id = static_cast<size_t>(__shfl_sync(0xffffffffu, my_id, r & 31)) * p.S + split;
    if (r >= nrows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, red_m[w * kRows + r]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = red_m[w * kRows + r], f = mw == -INFINITY ? 0.f : span_exp2(mw - top);   // (a sum that is NaN stays one)
      const float4 x = *reinterpret_cast<const float4*>(red_o + (w * kRows + r) * kPitch + c * 4);
      l += red_l[w * kRows + r] * f;
      o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    *reinterpret_cast<float4*>(p.o_part + id * D + c * 4) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (c == 0) p.lse_part[id] = l > 0.f ? top * 0.6931471805599453f + logf(l) : (l == l ? -INFINITY : l);
  }
}

// blockIdx.x: first the CTAs of the shared keys (split fastest, then row group, then KV head), then those of the own keys (split
// fastest, then row group, KV head, sequence).
template <bool BF16, int D, int NBP, int NBO>
__global__ void __launch_bounds__(kSpanThreads) shared_prefix_span_kernel(const SharedPrefixParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  if (!p.late_wait) griddep_wait();
  griddep_launch_dependents();
  const int G = p.Hq / p.Hkv;
  int at = blockIdx.x;
  if constexpr (NBP > 0) {
    if (at < p.prefix_ctas) {
      const int split = at % p.prefix_splits;
      at /= p.prefix_splits;
      const int groups = p.prefix_ctas / p.prefix_splits / p.Hkv;
      const int kvh = at / groups, group = at % groups;
      const int t0 = split * p.prefix_chunk, t1 = min(p.shared, t0 + p.prefix_chunk);
      span_fetch_queries<D, NBP>(p, smem, kvh, 0, group * NBP * 8, min(NBP * 8, p.B * p.T * G - group * NBP * 8));
      span_body<BF16, D, NBP>(p, smem, kvh, 0, group * NBP * 8, p.B * p.T * G, p.prefix_table, (p.shared + p.page - 1) / p.page, t0, t1, false, 0, split, -1, 0);
      // rows of sequences that do not reach beyond the shared keys are attended by themselves
      __syncthreads();
      for (int r = threadIdx.x; r < NBP * 8; r += kSpanThreads) {
        const int g = group * NBP * 8 + r;
        if (g >= p.B * p.T * G) break;
        const int token = g / G;
        if (prefix_len(p, token / p.T) - p.T + 1 < p.shared) p.lse_part[(static_cast<size_t>(token) * p.Hq + kvh * G + g % G) * p.S + split] = -INFINITY;
      }
      return;
    }
  }
  at -= p.prefix_ctas;
  const int split = at % p.own_splits;
  at /= p.own_splits;
  const int rows = p.T * G, groups = (rows + NBO * 8 - 1) / (NBO * 8);
  const int group = at % groups;
  at /= groups;
  const int kvh = at % p.Hkv, b = at / p.Hkv;
  span_fetch_queries<D, NBO>(p, smem, kvh, b * p.T, group * NBO * 8, min(NBO * 8, rows - group * NBO * 8));
  const int* table = p.block_table + static_cast<size_t>(b) * p.bt_stride;
  const int len = prefix_len(p, b);
  // The first pages as they are for a sequence that reaches beyond the shared keys: read together with its length, not after it. (With a window of 32
  // page numbers a warp instead of one ahead, and the merge's outputs fetched before its weights: 2 sequences of 32 / 8 heads, 1000 + 64 keys 8.8 ->
  // 6.9 us; 16 of 64 / 8 heads, 2048 + 512 17.0 -> 14.6; 48 x 3 tokens of 14 / 2 heads of 64, 16384 + 700 33.7 -> 29.0.)
  const bool known = p.own_splits == 1 && p.page % kSpanSlice == 0;
  const int ahead_base = known ? p.shared & ~(kSpanSlice - 1) : -1;
  const int ahead = known ? span_slice_at(p, table, p.width, static_cast<unsigned>(ahead_base) + ((threadIdx.x >> 5) + 4 * (threadIdx.x & 31)) * kSpanSlice) : 0;
  const int start = len - p.T + 1 >= p.shared ? p.shared : 0;
  int chunk = (len - start + p.own_splits - 1) / p.own_splits;
  chunk = (chunk + 4 * kSpanSlice - 1) / (4 * kSpanSlice) * (4 * kSpanSlice);
  const int t0 = start + split * chunk, t1 = min(len, t0 + chunk);
  span_body<BF16, D, NBO>(p, smem, kvh, b * p.T, group * NBO * 8, rows, table, p.width, t0, t1, true, len - p.T + 1, p.prefix_splits + split,
                          ahead_base, ahead);
  // The kernel in front (the shared keys') has to be complete before this one is. One CTA sees to that: if all of them waited, they would keep the
  // SMs that the kernel in front leaves free (64 / 8 heads, batch 64, with 64 CTAs in front: 155 us for 130).
  if (p.late_wait && blockIdx.x == gridDim.x - 1) griddep_wait();
}

// The merge: a warp per row, the weights of up to 32 ranges at a time in its lanes.
template <typename T, int D>
__global__ void __launch_bounds__(128) shared_prefix_merge_kernel(const float* __restrict__ o_part, const float* __restrict__ lse_part, int rows, int S,
                                                                  T* __restrict__ out, float* __restrict__ out_lse) {
  griddep_wait();
  griddep_launch_dependents();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  const float* l_row = lse_part + static_cast<size_t>(row) * S;
  constexpr int kV = D / 32, kAhead = 8;   // columns per lane; ranges in flight while those before are added
  const float* o_row = o_part + static_cast<size_t>(row) * S * D + lane * kV;
  float v[2][kAhead][kV];
  auto fetch = [&](int s0, float (&x)[kAhead][kV]) {   // (an empty range has left nothing there: read, but not used)
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (s0 + i < S) {
        const float* src = o_row + static_cast<size_t>(s0 + i) * D;
        if (kV == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(src);
      }
  };
  fetch(0, v[0]);
  float l = lane < S ? l_row[lane] : -INFINITY;
  float top = l;
  for (int s = lane + 32; s < S; s += 32) top = fmaxf(top, l_row[s]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[kV] = {0.f}, den = 0.f, mine = 0.f;
  for (int s0 = 0; s0 < S; s0 += 2 * kAhead) {
    if (s0 % 32 == 0) {
      if (s0 > 0) l = s0 + lane < S ? l_row[s0 + lane] : -INFINITY;
      mine = l == -INFINITY ? 0.f : expf(l - ref);   // the weight of range s0 + lane
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int s1 = s0 + half * kAhead;
      if (s1 + kAhead < S) fetch(s1 + kAhead, v[half ^ 1]);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float w = __shfl_sync(0xffffffffu, mine, (s1 + i) % 32);
        if (s1 + i < S && w != 0.f) {
          den += w;
#pragma unroll
          for (int e = 0; e < kV; ++e) acc[e] += w * v[half][i][e];
        }
      }
    }
  }
  T* dst = out + static_cast<size_t>(row) * D + lane * kV;
#pragma unroll
  for (int e = 0; e < kV; ++e) dst[e] = from_float<T>(den > 0.f || den != den ? acc[e] / den : 0.f);
  if (lane == 0 && out_lse != nullptr) out_lse[row] = den > 0.f || den != den ? ref + logf(den) : -INFINITY;
}

template <bool BF16, int D, int NBP, int NBO>
static int launch_span(const SharedPrefixParams& p, int ctas, cudaStream_t s) {
  static bool configured[64] = {false};
  int dev = 0;
  B200_CHECK_CUDA(cudaGetDevice(&dev));
  auto kernel = shared_prefix_span_kernel<BF16, D, NBP, NBO>;
  if (!configured[dev & 63]) {
    B200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, span_smem<D>()));
    configured[dev & 63] = true;
  }
  B200_CHECK_CUDA(launch_pdl(kernel, ctas, kSpanThreads, span_smem<D>(), s, p));
  return kOk;
}

// Blocks of eight rows per CTA for a number of rows: 1, 2 or 4.
static int span_blocks(long long rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

template <int D>
static int launch_span_form(const SharedPrefixParams& p, bool bf16, int nbp, int nbo, int ctas, cudaStream_t s) {
#define B200_SPAN(A, C) (bf16 ? launch_span<true, D, A, C>(p, ctas, s) : launch_span<false, D, A, C>(p, ctas, s))
  if (nbp == 0) return nbo == 1 ? B200_SPAN(0, 1) : nbo == 2 ? B200_SPAN(0, 2) : B200_SPAN(0, 4);
  if (nbp == 1) return B200_SPAN(1, 1);
  if (nbp == 2) return nbo == 1 ? B200_SPAN(2, 1) : B200_SPAN(2, 2);
  return nbo == 1 ? B200_SPAN(4, 1) : nbo == 2 ? B200_SPAN(4, 2) : B200_SPAN(4, 4);
#undef B200_SPAN
}

}  // namespace b200

using namespace b200;

// q [B * T, Hq, D] with ldq elements between tokens; caches [num_blocks, page, Hkv, D] contiguous; kv_lens int32 [B]; block_table int32
// [B, width] with bt_stride between rows; prefix_table int32 [>= ceil(shared / page)]; o_part fp32 [B * T * Hq, prefix_splits +
// own_splits, D] and lse_part fp32 [B * T * Hq, prefix_splits + own_splits] are scratch; out [B * T, Hq, D] contiguous, out_lse nullable
// fp32 [B * T, Hq]. 16-byte aligned q, caches, out. tc: the shared keys go to the tensor-core kernel. With shared = 0:
// tc = 0, prefix_splits = 0.
B200_API int b200_shared_prefix_attention(const void* q, long long ldq, const void* k_cache, const void* v_cache, const int* kv_lens, const int* block_table,
                                          int bt_stride, int width, const int* prefix_table, int B, int T, int Hq, int Hkv, int D, int num_blocks,
                                          int page, int shared, float scale, int tc, int prefix_splits, int own_splits, float* o_part, float* lse_part, void* out,
                                          float* out_lse, int dtype, uint32_t* status, void* stream) {
  B200_REQUIRE(dtype == kBF16 || dtype == kF16, "shared-prefix attention supports bf16/f16");
  B200_REQUIRE(D == 64 || D == 128, "shared-prefix attention supports head sizes 64 and 128, got %d", D);
  B200_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "Hq (%d) must be a multiple of Hkv (%d)", Hq, Hkv);
  B200_REQUIRE(B >= 0 && T >= 1 && page >= 1 && num_blocks >= 1 && width >= 0 && shared >= 0 && shared <= kPrefixMostKeys && ldq % 8 == 0, "shared-prefix attention: bad sizes");
  B200_REQUIRE(scale > 0.f, "the score scale must be positive");
  B200_REQUIRE(own_splits >= 1 && (shared == 0 ? prefix_splits == 0 : prefix_splits >= 1), "shared-prefix attention: bad split counts");
  if (B == 0) return kOk;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  SharedPrefixParams p;
  memset(&p, 0, sizeof(p));
  p.q = q; p.ldq = ldq; p.k_cache = k_cache; p.v_cache = v_cache; p.kv_lens = kv_lens; p.block_table = block_table; p.prefix_table = prefix_table;
  p.bt_stride = bt_stride; p.width = width; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.num_blocks = num_blocks; p.page = page; p.shared = shared;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.prefix_splits = prefix_splits; p.own_splits = own_splits; p.S = prefix_splits + own_splits;
  p.o_part = o_part; p.lse_part = lse_part; p.status = status;
  const int G = Hq / Hkv;
  const long long prefix_rows = static_cast<long long>(B) * T * G, own_rows = static_cast<long long>(T) * G;
  B200_REQUIRE(prefix_rows * Hkv <= 1 << 30, "shared-prefix attention: too many rows");
  const int nbp = tc || shared == 0 ? 0 : span_blocks(prefix_rows), nbo = span_blocks(own_rows);
  long long ctas = 0;
  if (tc) {
    B200_REQUIRE(shared_prefix_tc_takes(p, D), "shared-prefix attention: these heads or pages are not for the tensor-core kernel");
    p.prefix_chunk = ((shared + prefix_splits - 1) / prefix_splits + 127) / 128 * 128;
    const int rc = shared_prefix_tc_launch(p, D, dtype, s);
    if (rc != kOk) return rc;
    p.late_wait = pdl_enabled();
  } else if (shared > 0) {
    p.prefix_chunk = ((shared + prefix_splits - 1) / prefix_splits + 63) / 64 * 64;
    ctas = (prefix_rows + nbp * 8 - 1) / (nbp * 8) * Hkv * prefix_splits;
    p.prefix_ctas = static_cast<int>(ctas);
  }
  ctas += (own_rows + nbo * 8 - 1) / (nbo * 8) * Hkv * B * own_splits;
  B200_REQUIRE(ctas <= 0x7fffffffLL, "shared-prefix attention: grid is too large");
  const int rc = D == 128 ? launch_span_form<128>(p, dtype == kBF16, nbp, nbo, static_cast<int>(ctas), s)
                          : launch_span_form<64>(p, dtype == kBF16, nbp, nbo, static_cast<int>(ctas), s);
  if (rc != kOk) return rc;
  const int rows = B * T * Hq;
#define B200_MERGE(TT, DD)                                                                                                     \
  B200_CHECK_CUDA(launch_pdl(shared_prefix_merge_kernel<TT, DD>, (rows + 3) / 4, 128, 0, s, o_part, lse_part, rows, p.S, static_cast<TT*>(out), out_lse))
  if (dtype == kBF16) {
    if (D == 128) B200_MERGE(__nv_bfloat16, 128); else B200_MERGE(__nv_bfloat16, 64);
  } else {
    if (D == 128) B200_MERGE(__half, 128); else B200_MERGE(__half, 64);
  }
#undef B200_MERGE
  return kOk;
}
