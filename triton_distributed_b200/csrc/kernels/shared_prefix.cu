// Attention over a paged cache for a batch whose sequences begin with the same keys: the shared keys are read once for the rows of all
// sequences, everybody's own keys once for the rows of that sequence, and the partial results are merged.
//
//   n = kv_len[b] - tokens + t + 1 keys are visible to query token t of sequence b (the new tokens are in the cache)
//   o = sum_{j < n} p_j v_j / sum_{j < n} p_j,  p_j = exp(scale q . k_j - m)      (zeros and a log-sum-exp of -inf for n <= 0)
//
// A row (token and query head) is split over disjoint ranges of keys. Every range leaves its normalised output o_i and its
// log-sum-exp l_i; the whole is sum_i exp(l_i - l) o_i with l = log sum_i exp(l_i).
//
// This file holds the kernel on warp-level products (m16n8k16): 16 or 32 rows that share a KV head per CTA, each of the four warps
// streaming its own slices of 16 keys through a private ring of three (cp.async, no barrier of the CTA in the loop), its running
// maximum, sum and output in registers. It takes the own keys of every sequence and, while the rows per KV head are few, the
// shared keys; both in one launch, the shared ones first because their CTAs run longest. What bounds it is the read of the keys.
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

template <int D>
constexpr int span_smem() { return 4 * kSpanRing * 2 * kSpanSlice * D * 2; }

// The value rows of a slice in which some keys are masked for some rows (between drafted tokens): a masked key has weight zero, and
// zero times an infinity or NaN must not reach the row. Tells whether the slice holds such a value.
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

// One CTA: NM x 16 rows of KV head `kvh` from row `row0` of a group of `rows`, over keys [t0, t1) of the pages in `table`. A row r of
// the group is query token first_token + r / G, head kvh * G + r % G. `own`: the rows are one sequence's and see keys below `limit0` + r / G.
template <bool BF16, int D, int NM>
__device__ void span_body(const SharedPrefixParams& p, uint8_t* smem, int kvh, int first_token, int row0, int rows, const int* table, int width,
                          int t0, int t1, bool own, int limit0, int split) {
  constexpr int kKK = D / 16, kRowBytes = D * 2, kChunks = D / 8, kSliceBytes = kSpanSlice * kRowBytes;
  const int G = p.Hq / p.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r_lo = lane >> 2;
  const int nrows = min(NM * 16, rows - row0);
  auto row_id = [&](int r) {   // of row r of this CTA, among all rows of the call
    const int g = row0 + r;
    return static_cast<size_t>(first_token + g / G) * p.Hq + kvh * G + g % G;
  };
  if (t0 >= t1) {
    for (int r = threadIdx.x; r < nrows; r += kSpanThreads) p.lse_part[row_id(r) * p.S + split] = -INFINITY;
    return;
  }

  // ---- query fragments; rows that do not exist are zero ----
  uint32_t qa[NM][kKK][4];
  int limit[NM][2];
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = m * 16 + r_lo + 8 * h, g = row0 + r;
      const bool in = r < nrows;
      limit[m][h] = own ? min(t1, limit0 + g / G) : t1;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.q) + (static_cast<size_t>(first_token + g / G) * p.ldq +
                                                              static_cast<size_t>(kvh * G + g % G) * D) * 2) + (lane & 3);
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {
        qa[m][kk][h] = in ? src[kk * 8] : 0u;
        qa[m][kk][h + 2] = in ? src[kk * 8 + 4] : 0u;
      }
    }

  // ---- this warp's ring: slot s holds K at +0 and V behind it; slices begin at multiples of 16 keys ----
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (kSpanRing * 2 * kSliceBytes);
  const uint8_t *kc = static_cast<const uint8_t*>(p.k_cache), *vc = static_cast<const uint8_t*>(p.v_cache);
  const int base = t0 & ~(kSpanSlice - 1);
  const int n_slices = (t1 - base + kSpanSlice - 1) / kSpanSlice;
  const int mine = n_slices > warp ? (n_slices - warp + 3) / 4 : 0;   // slices warp, warp + 4, ...
  const bool page_fast = p.page % kSpanSlice == 0;
  auto page_of = [&](int tok) -> long long {   // first slot of the page that holds a token, or -1
    const int w = tok / p.page;
    const int blk = w < width ? table[w] : -1;
    return blk >= 0 && blk < p.num_blocks ? static_cast<long long>(blk) * p.page : -1;
  };
  auto load_slice = [&](int j) {   // always commits a group, so that the counting stays uniform
    if (j < mine) {
      const int st0 = base + (warp + 4 * j) * kSpanSlice;
      const uint32_t slot = ring + (j % kSpanRing) * (2 * kSliceBytes);
      const long long first = page_fast ? page_of(st0) : 0;
#pragma unroll
      for (int i = 0; i < kSpanSlice * kChunks / 32; ++i) {
        const int tok_in = (i * 32 + lane) / kChunks, c = lane % kChunks;
        const int tok = st0 + tok_in;
        bool valid = tok >= t0 && tok < t1;
        long long page0 = first;
        if (!page_fast && valid) page0 = page_of(tok);
        valid = valid && page0 >= 0;
        const size_t off = valid ? ((static_cast<size_t>(page0 + tok % p.page) * p.Hkv + kvh) * D + c * 8) * 2 : 0;
        const uint32_t so = tok_in * kRowBytes + ((c ^ (tok_in & 7)) * 16);
        cp_async_16(slot + so, kc + off, valid ? 16 : 0);
        cp_async_16(slot + kSliceBytes + so, vc + off, valid ? 16 : 0);
      }
    }
    cp_async_commit();
  };

  float m_run[NM][2], l_run[NM][2], oacc[NM][2 * kKK][4];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
#pragma unroll
    for (int h = 0; h < 2; ++h) { m_run[m][h] = -INFINITY; l_run[m][h] = 0.f; }
#pragma unroll
    for (int i = 0; i < 2 * kKK; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) oacc[m][i][e] = 0.f;
  }
  const int safe = own ? min(t1, limit0 + row0 / G) : t1;   // keys below are visible to every row of this CTA
#pragma unroll
  for (int j = 0; j < kSpanRing - 1; ++j) load_slice(j);
  for (int j = 0; j < mine; ++j) {
    load_slice(j + kSpanRing - 1);       // into the slot of the iteration before
    cp_async_wait<kSpanRing - 1>();      // this lane's part of slice j has landed; the barrier covers the other lanes
    __syncwarp();
    const uint32_t ks = ring + (j % kSpanRing) * (2 * kSliceBytes), vs = ks + kSliceBytes;
    const int st0 = base + (warp + 4 * j) * kSpanSlice;
    // ---- scores of 16 keys ----
    float s[NM][2][4];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[m][0][e] = s[m][1][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      const int mat = lane >> 3, tok_in = (mat >> 1) * 8 + (lane & 7), c = 2 * kk + (mat & 1);
      uint32_t b0, b1, b2, b3;
      ldmatrix_x4(ks + tok_in * kRowBytes + ((c ^ (tok_in & 7)) * 16), b0, b1, b2, b3);
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        mma16816<BF16>(s[m][0], qa[m][kk], b0, b1);
        mma16816<BF16>(s[m][1], qa[m][kk], b2, b3);
      }
    }
    const bool whole = st0 >= t0 && st0 + kSpanSlice <= safe;
    uint32_t pa[NM][4];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = s[m][nb][2 * h + e] * p.scale_log2e;
            const int tok = st0 + nb * 8 + (lane & 3) * 2 + e;
            if (!whole && (tok < t0 || tok >= limit[m][h])) v = -INFINITY;
            s[m][nb][2 * h + e] = v;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run[m][h], mx);
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float corr = exp2f(m_run[m][h] - ref);   // -inf -> 0
        m_run[m][h] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float w = exp2f(s[m][nb][2 * h + e] - ref);
            s[m][nb][2 * h + e] = w;
            sum += w;
          }
        l_run[m][h] = l_run[m][h] * corr + sum;
#pragma unroll
        for (int i = 0; i < 2 * kKK; ++i) {
          oacc[m][i][2 * h] *= corr;
          oacc[m][i][2 * h + 1] *= corr;
        }
      }
      // the weights are rounded to the type of the values: the product's A operand has it (the row's largest is one, exactly)
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pa[m][nb * 2 + h] = BF16 ? pack_bf16x2(s[m][nb][2 * h], s[m][nb][2 * h + 1]) : pack_f16x2(s[m][nb][2 * h], s[m][nb][2 * h + 1]);
    }
    if (!whole && own && slice_has_nonfinite<BF16, D>(vs, lane)) {
      // ---- rare: what is not finite is added for the rows that see its key, and is zero in the product. The weights go through the
      // slice's K slot, which has been used. ----
      __syncwarp();
      const uint32_t smem0 = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
      float* w_sh = reinterpret_cast<float*>(smem + (ks - smem0));   // [16 rows][16 keys]
      uint8_t* v_sh = smem + (vs - smem0);
      constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
      for (int m = 0; m < NM; ++m) {
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) w_sh[(r_lo + 8 * (e >> 1)) * 16 + nb * 8 + (lane & 3) * 2 + (e & 1)] = s[m][nb][e];
        __syncwarp();
#pragma unroll 1
        for (int key = 0; key < kSpanSlice; ++key) {
          const float w0 = w_sh[r_lo * 16 + key], w1 = w_sh[(r_lo + 8) * 16 + key];
#pragma unroll
          for (int i = 0; i < 2 * kKK; ++i) {
            const uint32_t raw = *reinterpret_cast<const uint32_t*>(v_sh + key * kRowBytes + ((i ^ (key & 7)) * 16) + (lane & 3) * 4);
            const float2 v = BF16 ? unpack_bf16x2(raw) : unpack_f16x2(raw);
            const bool x = (raw & kExp) == kExp, y = (raw >> 16 & kExp) == kExp;
            if (x && w0 > 0.f) oacc[m][i][0] += w0 * v.x;
            if (y && w0 > 0.f) oacc[m][i][1] += w0 * v.y;
            if (x && w1 > 0.f) oacc[m][i][2] += w1 * v.x;
            if (y && w1 > 0.f) oacc[m][i][3] += w1 * v.y;
          }
        }
        __syncwarp();
      }
      for (int i = lane; i < kSliceBytes / 4; i += 32) {
        uint32_t* at = reinterpret_cast<uint32_t*>(v_sh) + i;
        const uint32_t raw = *at;
        *at = ((raw & kExp) == kExp ? 0u : raw & 0xffffu) | ((raw >> 16 & kExp) == kExp ? 0u : raw & 0xffff0000u);
      }
      __syncwarp();
    }
#pragma unroll
    for (int dn = 0; dn < kKK; ++dn) {
      const int mat = lane >> 3, tok_in = (mat & 1) * 8 + (lane & 7), c = 2 * dn + (mat >> 1);
      uint32_t b0, b1, b2, b3;
      ldmatrix_x4_trans(vs + tok_in * kRowBytes + ((c ^ (tok_in & 7)) * 16), b0, b1, b2, b3);
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        mma16816<BF16>(oacc[m][2 * dn], pa[m], b0, b1);
        mma16816<BF16>(oacc[m][2 * dn + 1], pa[m], b2, b3);
      }
    }
    __syncwarp();   // the slot is free for the copies of the next iteration
  }
  cp_async_wait<0>();
  __syncthreads();  // all rings are idle: their memory becomes the merge area

  // ---- merge of the four warps ----
  float* red_m = reinterpret_cast<float*>(smem);     // [4][NM * 16]
  float* red_l = red_m + 4 * NM * 16;                // [4][NM * 16]
  float* red_o = red_l + 4 * NM * 16;                // [4][NM * 16][D]
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l_run[m][h] += __shfl_xor_sync(0xffffffffu, l_run[m][h], 1);
      l_run[m][h] += __shfl_xor_sync(0xffffffffu, l_run[m][h], 2);
      if ((lane & 3) == 0) {
        red_m[(warp * NM + m) * 16 + r_lo + 8 * h] = m_run[m][h];
        red_l[(warp * NM + m) * 16 + r_lo + 8 * h] = l_run[m][h];
      }
    }
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int i = 0; i < 2 * kKK; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(red_o + (static_cast<size_t>(warp * NM + m) * 16 + r_lo + 8 * h) * D + i * 8 + (lane & 3) * 2) =
            make_float2(oacc[m][i][2 * h], oacc[m][i][2 * h + 1]);
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * D; i += kSpanThreads) {
    const int r = i / D, c = i - r * D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, red_m[w * NM * 16 + r]);
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = red_m[w * NM * 16 + r], f = mw == -INFINITY ? 0.f : exp2f(mw - top);   // (a sum that is NaN stays one)
      l += red_l[w * NM * 16 + r] * f;
      o += red_o[static_cast<size_t>(w * NM * 16 + r) * D + c] * f;
    }
    const size_t id = row_id(r) * p.S + split;
    p.o_part[id * D + c] = l > 0.f ? o / l : (l == l ? 0.f : l);
    if (c == 0) p.lse_part[id] = l > 0.f ? top * 0.6931471805599453f + logf(l) : (l == l ? -INFINITY : l);
  }
}

// blockIdx.x: first the CTAs of the shared keys (split fastest, then row group, then KV head), then those of the own keys (split
// fastest, then row group, KV head, sequence).
template <bool BF16, int D, int NMP, int NMO>
__global__ void __launch_bounds__(kSpanThreads) shared_prefix_span_kernel(const SharedPrefixParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  if (!p.late_wait) griddep_wait();
  griddep_launch_dependents();
  const int G = p.Hq / p.Hkv;
  int at = blockIdx.x;
  if (at < p.prefix_ctas) {
    const int split = at % p.prefix_splits;
    at /= p.prefix_splits;
    const int groups = p.prefix_ctas / p.prefix_splits / p.Hkv;
    const int kvh = at / groups, group = at % groups;
    const int t0 = split * p.prefix_chunk, t1 = min(p.shared, t0 + p.prefix_chunk);
    span_body<BF16, D, NMP>(p, smem, kvh, 0, group * NMP * 16, p.B * p.T * G, p.prefix_table, (p.shared + p.page - 1) / p.page, t0,
                            t1, false, 0, split);
    // rows of sequences that do not reach beyond the shared keys are attended by themselves
    __syncthreads();
    for (int r = threadIdx.x; r < NMP * 16; r += kSpanThreads) {
      const int g = group * NMP * 16 + r;
      if (g >= p.B * p.T * G) break;
      const int token = g / G;
      if (p.kv_lens[token / p.T] - p.T + 1 < p.shared) p.lse_part[(static_cast<size_t>(token) * p.Hq + kvh * G + g % G) * p.S + split] = -INFINITY;
    }
  } else {
    at -= p.prefix_ctas;
    const int split = at % p.own_splits;
    at /= p.own_splits;
    const int rows = p.T * G, groups = (rows + NMO * 16 - 1) / (NMO * 16);
    const int group = at % groups;
    at /= groups;
    const int kvh = at % p.Hkv, b = at / p.Hkv;
    const int len = max(0, p.kv_lens[b]), start = len - p.T + 1 >= p.shared ? p.shared : 0;
    int chunk = (len - start + p.own_splits - 1) / p.own_splits;
    chunk = (chunk + 4 * kSpanSlice - 1) / (4 * kSpanSlice) * (4 * kSpanSlice);
    const int t0 = start + split * chunk, t1 = min(len, t0 + chunk);
    span_body<BF16, D, NMO>(p, smem, kvh, b * p.T, group * NMO * 16, rows, p.block_table + static_cast<size_t>(b) * p.bt_stride, p.width, t0, t1,
                            true, len - p.T + 1, p.prefix_splits + split);
  }
  if (p.late_wait) griddep_wait();   // the kernel in front (the shared keys') is complete before this one is
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
  const float* o_row = o_part + static_cast<size_t>(row) * S * D;
  constexpr int kV = D / 32;   // columns per lane
  float top = -INFINITY;
  for (int s = lane; s < S; s += 32) top = fmaxf(top, l_row[s]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[kV] = {0.f}, den = 0.f;
  for (int s0 = 0; s0 < S; s0 += 32) {
    const float l = s0 + lane < S ? l_row[s0 + lane] : -INFINITY;
    const float mine = l == -INFINITY ? 0.f : expf(l - ref);
    const int n = min(32, S - s0);
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float w = __shfl_sync(0xffffffffu, mine, s);
      float v[kV];
      const float* src = o_row + static_cast<size_t>(s0 + s) * D + lane * kV;
      if (kV == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
      den += w;
      if (w != 0.f)   // an empty range has left nothing there
#pragma unroll
        for (int e = 0; e < kV; ++e) acc[e] += w * v[e];
    }
  }
  T* dst = out + static_cast<size_t>(row) * D + lane * kV;
#pragma unroll
  for (int e = 0; e < kV; ++e) dst[e] = from_float<T>(den > 0.f || den != den ? acc[e] / den : 0.f);
  if (lane == 0 && out_lse != nullptr) out_lse[row] = den > 0.f || den != den ? ref + logf(den) : -INFINITY;
}

template <bool BF16, int D, int NMP, int NMO>
static int launch_span(const SharedPrefixParams& p, int ctas, cudaStream_t s) {
  static bool configured[64] = {false};
  int dev = 0;
  B200_CHECK_CUDA(cudaGetDevice(&dev));
  auto kernel = shared_prefix_span_kernel<BF16, D, NMP, NMO>;
  if (!configured[dev & 63]) {
    B200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, span_smem<D>()));
    configured[dev & 63] = true;
  }
  B200_CHECK_CUDA(launch_pdl(kernel, ctas, kSpanThreads, span_smem<D>(), s, p));
  return kOk;
}

template <int D>
static int launch_span_form(const SharedPrefixParams& p, bool bf16, int nmp, int nmo, int ctas, cudaStream_t s) {
#define B200_SPAN(A, C) (bf16 ? launch_span<true, D, A, C>(p, ctas, s) : launch_span<false, D, A, C>(p, ctas, s))
  return nmo == 2 ? B200_SPAN(2, 2) : nmp == 2 ? B200_SPAN(2, 1) : B200_SPAN(1, 1);
#undef B200_SPAN
}

}  // namespace b200

using namespace b200;

// q [B * T, Hq, D] with ldq elements between tokens; caches [num_blocks, page, Hkv, D] contiguous; kv_lens int32 [B]; block_table int32
// [B, width] with bt_stride between rows; prefix_table int32 [>= ceil(shared / page)]; o_part fp32 [B * T * Hq, prefix_splits +
// own_splits, D] and lse_part fp32 [B * T * Hq, prefix_splits + own_splits] are scratch; out [B * T, Hq, D] contiguous, out_lse nullable
// fp32 [B * T, Hq]. 16-byte aligned q, caches, out. tc: the shared keys go to the tensor-core kernel (an even number of ranges where all rows
// of a KV head fit one tile of floor(128 / (Hq / Hkv)) tokens). With shared = 0: tc = 0, prefix_splits = 0.
B200_API int b200_shared_prefix_attention(const void* q, long long ldq, const void* k_cache, const void* v_cache, const int* kv_lens, const int* block_table,
                                          int bt_stride, int width, const int* prefix_table, int B, int T, int Hq, int Hkv, int D, int num_blocks,
                                          int page, int shared, float scale, int tc, int prefix_splits, int own_splits, float* o_part, float* lse_part, void* out,
                                          float* out_lse, int dtype, uint32_t* status, void* stream) {
  B200_REQUIRE(dtype == kBF16 || dtype == kF16, "shared-prefix attention supports bf16/f16");
  B200_REQUIRE(D == 64 || D == 128, "shared-prefix attention supports head sizes 64 and 128, got %d", D);
  B200_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "Hq (%d) must be a multiple of Hkv (%d)", Hq, Hkv);
  B200_REQUIRE(B >= 0 && T >= 1 && page >= 1 && num_blocks >= 1 && width >= 0 && shared >= 0 && ldq % 8 == 0, "shared-prefix attention: bad sizes");
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
  const int nmp = prefix_rows > 16 ? 2 : 1, nmo = own_rows > 16 ? 2 : 1;
  long long ctas = 0;
  if (tc) {
    B200_REQUIRE(shared_prefix_tc_takes(p, D), "shared-prefix attention: these heads or pages are not for the tensor-core kernel");
    const bool two_ranges = static_cast<long long>(B) * T <= 128 / G;
    B200_REQUIRE(!two_ranges || prefix_splits % 2 == 0, "shared-prefix attention: rows of one tile take pairs of ranges");
    const int per_row = two_ranges ? prefix_splits / 2 : prefix_splits;
    p.prefix_chunk = ((shared + per_row - 1) / per_row + 127) / 128 * 128;
    const int rc = shared_prefix_tc_launch(p, D, dtype, s);
    if (rc != kOk) return rc;
    p.late_wait = pdl_enabled();
  } else if (shared > 0) {
    p.prefix_chunk = ((shared + prefix_splits - 1) / prefix_splits + 63) / 64 * 64;
    ctas = (prefix_rows + nmp * 16 - 1) / (nmp * 16) * Hkv * prefix_splits;
    p.prefix_ctas = static_cast<int>(ctas);
  }
  ctas += (own_rows + nmo * 16 - 1) / (nmo * 16) * Hkv * B * own_splits;
  B200_REQUIRE(ctas <= 0x7fffffffLL, "shared-prefix attention: grid is too large");
  const int rc = D == 128 ? launch_span_form<128>(p, dtype == kBF16, nmp, nmo, static_cast<int>(ctas), s)
                          : launch_span_form<64>(p, dtype == kBF16, nmp, nmo, static_cast<int>(ctas), s);
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
