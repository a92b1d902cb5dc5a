// Which of a sequence's drafted tokens stand, and the token behind them (speculative sampling with the random numbers given).
//
//   drafts d_0 ... d_{len-1} with draft probabilities q_i and target probabilities p_0 ... p_len, uniform numbers u_0 ... u_K in [0, 1):
//   d_i is accepted if all before it are and u_i q_i(d_i) < p_i(d_i); n = number of accepted drafts
//   w = p_len if n = len, else max(p_n - q_n, 0), or p_n where that is zero everywhere
//   the next token is the first j with w_0 + ... + w_j > u_K * sum(w)
// so that the tokens are distributed as if drawn from the target alone. Without draft probabilities a draft was picked without
// chance: q_i is one at d_i, and w is p_n without d_n.
//
// The comparison is exact: products of two 32-bit (or 16-bit) values are exact in 64 bits, and so are the differences but for one
// rounding. The sums are kept in 64 bits: with 32, which of two neighbours among 152 K tokens is drawn would depend on the order of the
// additions. Values that are not positive and finite count as zero, drafts outside the vocabulary are never accepted.
//
// A cluster of CTAs takes a sequence: all find n for themselves (a few loads), then every warp adds up its own contiguous run
// of the one row (two with draft probabilities) that is needed, keeping the sums of its parts, and the CTAs write their sums into each other's shared
// memory. The warp whose interval holds the target reads the part with the target once more, which the caches still have. One pass over memory.
#include "b200/host.h"
#include "b200/elem.cuh"
#include "b200/primitives.cuh"

#include <cooperative_groups.h>
#include <cstring>

namespace b200 {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCtas = 16;   // per sequence
constexpr int kVerifySlots = 16;     // sums that every lane keeps of its part of the warp's run

struct VerifyParams {
  const long long* drafts;   // [B, K]
  const void* target;        // [B, K + 1, V], strides in elements
  const void* draft;         // nullable [B, K, V]
  const float* uniform;      // [B, K + 1]
  const int* lens;           // nullable [B]
  long long t_b, t_k, d_b, d_k;
  int K, V;
  int* accepted;             // [B]
  long long* tokens;         // [B, K + 1]
};

__device__ __forceinline__ float probability(float x) { return __float_as_uint(x) < 0x7f800000u ? x : 0.f; }   // (a sign makes the bits larger)

// The weights of a row, in blocks of N = 16 bytes' worth of tokens that begin where the target's row is 16-byte aligned: block k holds
// tokens [k N - off, ...) of [0, V). max(p - q, 0) with draft probabilities, else p without the refused token.
template <typename T>
struct Weights {
  static constexpr int N = 16 / sizeof(T);
  const T* p;
  const T* q;       // nullable
  int hole;         // a token without a weight, or -1
  int V, off;
  bool q_wide;      // q's row is aligned like p's

  __device__ __forceinline__ void set(const T* p_, const T* q_, long long hole_, int V_) {
    p = p_; q = q_; hole = hole_ >= 0 && hole_ < V_ ? static_cast<int>(hole_) : -1; V = V_;
    off = static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(T) % N);
    q_wide = static_cast<int>(reinterpret_cast<uintptr_t>(q) / sizeof(T) % N) == off;
  }
  __device__ __forceinline__ int blocks() const { return (V + off + N - 1) / N; }
  // Blocks of [k0, k1) that the row's ends do not cut: [first_whole, last_whole)
  __device__ __forceinline__ int first_whole(int k0) const { return max(k0, off > 0 ? 1 : 0); }
  __device__ __forceinline__ int last_whole(int k1) const { return min(k1, (V + off) / N); }
  // Both rows' values of block k, zeros where it is not before `end` or there is no such token.
  __device__ __forceinline__ void fetch(int k, int end, uint4& a, uint4& b) const {
    const int j = k * N - off;
    a = b = make_uint4(0u, 0u, 0u, 0u);
    const bool whole = k < end && j >= 0 && j + N <= V;
    if (whole) a = *reinterpret_cast<const uint4*>(p + j);
    if (whole && q != nullptr && q_wide) b = *reinterpret_cast<const uint4*>(q + j);
    if (k < end && (!whole || (q != nullptr && !q_wide))) {
      T *x = reinterpret_cast<T*>(&a), *y = reinterpret_cast<T*>(&b);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < V) {
          if (!whole) x[e] = p[j + e];
          if (q != nullptr) y[e] = q[j + e];
        }
    }
  }
  // Weight of token j from its two values. (The difference has its one rounding in 64 bits.)
  __device__ __forceinline__ double weight(int j, T at_p, T at_q) const {
    const float x = probability(to_float(at_p)), y = q ? probability(to_float(at_q)) : j == hole ? x : 0.f;
    return static_cast<double>(x) - static_cast<double>(fminf(x, y));
  }
  __device__ __forceinline__ double one(int j) const { return weight(j, p[j], q ? q[j] : p[j]); }
};

// Whether none of the values that went into `most` (a maximum of their bits as unsigned numbers) is negative, infinite or NaN.
template <typename T> __device__ __forceinline__ unsigned max_bits(unsigned a, unsigned b, unsigned c) { return __vimax3_u16x2(a, b, c); }
template <> __device__ __forceinline__ unsigned max_bits<float>(unsigned a, unsigned b, unsigned c) { return max(a, max(b, c)); }
template <typename T> __device__ __forceinline__ bool all_plain(unsigned most);
template <> __device__ __forceinline__ bool all_plain<float>(unsigned most) { return most < 0x7f800000u; }
template <> __device__ __forceinline__ bool all_plain<__nv_bfloat16>(unsigned most) { return (most & 0xffffu) < 0x7f80u && (most >> 16) < 0x7f80u; }
template <> __device__ __forceinline__ bool all_plain<__half>(unsigned most) { return (most & 0xffffu) < 0x7c00u && (most >> 16) < 0x7c00u; }

template <typename T, int kQ> constexpr int kGroupRows = sizeof(T) == 2 && kQ ? 2 : 4;   // rows of 32 blocks
template <typename T> constexpr int kGroupBlocks = 32 * kGroupRows<T, 1>;                             // of which sums are kept

// The sum of the weights of blocks [k0, k1), by a warp; `sums` [kVerifySlots][32] receives each lane's sums of `per_slot` groups of kGroupBlocks. (Adding
// them up over the lanes, ten shuffles and five dependent additions in 64 bits a group, took 3 us of 64 sequences' 24.) kQ: 0 without draft
// probabilities, 1 with them aligned like the target's, 2 otherwise: the draft's values are then loaded one by one (64 sequences with draft probabilities,
// 50257 tokens for 50256: 12.6 us for 10.8 in 32 bits, 9.7 for 7.6 in 16).
// Whole blocks in groups of loads, each issued before the values of the group in front are used; loads behind the end are of the last block, without a
// weight, so that no branch stands between loads. A block that the row's ends cut is read token by token.
// The first form looked at every value for what is no probability and kept the last token with a weight: about thirty instructions a
// token bound it (64 sequences of 151936: 31 us). Now a group's values are looked at by one maximum of their bits, and the last token
// is looked for where it is needed; two conversions to 64 bits a token, a minimum and two additions are left.
template <typename T, int kQ>
__device__ __noinline__ double warp_mass_of(const Weights<T> w, int k0, int k1, double* sums, int per_slot) {
  constexpr int N = Weights<T>::N, kRows = kGroupRows<T, kQ>, kParts = kRows / kGroupRows<T, 1>;
  const int lane = threadIdx.x & 31;
  const int i0 = w.first_whole(k0), i1 = w.last_whole(k1);
  const int hole_block = w.hole >= 0 ? (w.hole + w.off) / N : -1;
  uint4 a[2][kRows], b[2][kRows];
  auto fetch = [&](int k, uint4& x, uint4& y) {
    const int j = min(k, i1 - 1) * N - w.off;
    x = *reinterpret_cast<const uint4*>(w.p + j);
    if (kQ == 1) y = *reinterpret_cast<const uint4*>(w.q + j);
    if (kQ == 2) {
      T* e = reinterpret_cast<T*>(&y);
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = w.q[j + i];
    }
  };
  // the tokens of a first block that the row's begin cuts belong to the first sum, those of the last to the last
  double total = 0.0, slot_sum = 0.0;
  if (k0 == 0 && lane >= w.off && lane < N && w.off > 0 && lane - w.off < w.V) slot_sum = w.one(lane - w.off);
  int left = per_slot;   // groups until the sum is complete
  sums += lane;
  auto use = [&](int at, const uint4 (&x)[kRows], const uint4 (&y)[kRows]) {   // blocks at, at + 32, ... of this lane
    unsigned most = 0u;
#pragma unroll
    for (int g = 0; g < kRows; ++g) {
      most = max_bits<T>(most, x[g].x, x[g].y);
      most = max_bits<T>(most, x[g].z, x[g].w);
      if (kQ) {
        most = max_bits<T>(most, y[g].x, y[g].y);
        most = max_bits<T>(most, y[g].z, y[g].w);
      }
    }
    const bool plain = all_plain<T>(most);
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      double sum[2] = {0.0, 0.0};
#pragma unroll
      for (int g = part * kRows / kParts; g < (part + 1) * kRows / kParts; ++g) {
        const int k = at + g * 32;
        if (k >= i1) break;
        if (!plain || (kQ == 0 && k == hole_block)) {   // rare: token by token
#pragma unroll 1
          for (int e = 0; e < N; ++e) sum[0] += w.one(k * N - w.off + e);
          continue;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {   // max(u - v, 0) = u - min(u, v)
          const float u = to_float(reinterpret_cast<const T*>(&x[g])[e]);
          double d = u;
          if (kQ) d -= static_cast<double>(fminf(u, to_float(reinterpret_cast<const T*>(&y[g])[e])));
          sum[e & 1] += d;
        }
      }
      slot_sum += sum[0] + sum[1];
      // (a last group that is not full stays open: what follows it belongs to its sum)
      if (--left == 0 && at - lane + (part + 1) * kGroupBlocks<T> <= i1) {
        *sums = slot_sum;
        sums += 32;
        total += slot_sum;
        slot_sum = 0.0;
        left = per_slot;
      }
    }
  };
  constexpr int kStep = kRows * 32;
  if (i0 < i1) {
#pragma unroll
    for (int g = 0; g < kRows; ++g) fetch(i0 + g * 32 + lane, a[0][g], b[0][g]);
#pragma unroll 1
    for (int k = i0; k < i1; k += 2 * kStep) {
#pragma unroll
      for (int turn = 0; turn < 2; ++turn) {
        const int at = k + turn * kStep;
        if (turn == 1 && at >= i1) break;
        if (at + kStep < i1)
#pragma unroll
          for (int g = 0; g < kRows; ++g) fetch(at + kStep + g * 32 + lane, a[turn ^ 1][g], b[turn ^ 1][g]);
        use(at + lane, a[turn], b[turn]);
      }
    }
  }
  if (k0 < k1 && i1 < k1 && i1 * N - w.off + lane >= 0 && i1 * N - w.off + lane < w.V && (i1 > 0 || w.off == 0)) slot_sum += w.one(i1 * N - w.off + lane);   // (fewer than N are left)
  *sums = slot_sum;
  total += slot_sum;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  return total;
}
template <typename T>
__device__ __forceinline__ double warp_mass(const Weights<T>& w, int k0, int k1, double* sums, int per_slot) {
  return w.q == nullptr ? warp_mass_of<T, 0>(w, k0, k1, sums, per_slot)
                        : w.q_wide ? warp_mass_of<T, 1>(w, k0, k1, sums, per_slot) : warp_mass_of<T, 2>(w, k0, k1, sums, per_slot);
}
// The last token of [j0, j1) that has a weight, or -1; by a whole CTA.
template <typename T>
__device__ __noinline__ int last_weight(const Weights<T> w, int j0, int j1, int* shared) {
  __syncthreads();
  if (threadIdx.x == 0) *shared = -1;
  __syncthreads();
  int last = -1;
  for (int j = j0 + threadIdx.x; j < j1; j += kVerifyThreads)
    if (w.one(j) > 0.0) last = j;
  if (last >= 0) atomicMax(shared, last);
  __syncthreads();
  return *shared;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_drafts_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double warp_sums[kVerifyWarps];
  __shared__ double all_total[2][kVerifyMaxCtas];   // written by all CTAs of the cluster, for each attempt
  __shared__ double slots[kVerifyWarps][kVerifySlots * 32];   // sums of each lane's groups
  __shared__ int s_accepted, s_last;
  const int crank = static_cast<int>(cluster.block_rank()), csize = static_cast<int>(cluster.num_blocks());
  const int b = blockIdx.x / csize;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // the others' shared memory may be written once all have started
  griddep_wait();
  griddep_launch_dependents();

  // ---- how many drafts stand ----
  const int len = p.lens ? max(0, min(p.K, p.lens[b])) : p.K;
  const long long* d_row = p.drafts + static_cast<size_t>(b) * p.K;
  const float* u_row = p.uniform + static_cast<size_t>(b) * (p.K + 1);
  const T* target = static_cast<const T*>(p.target) + b * p.t_b;
  const T* draft = p.draft ? static_cast<const T*>(p.draft) + b * p.d_b : nullptr;
  const double u_last = u_row[p.K];
  if (warp == 0) {
    int n = 0;
    for (int k0 = 0; k0 < len; k0 += 32) {
      bool stands = false;
      if (k0 + lane < len) {
        const long long d = d_row[k0 + lane];
        const double u = u_row[k0 + lane];
        if (d >= 0 && d < p.V) {
          const double pd = probability(to_float(target[(k0 + lane) * p.t_k + d]));
          const double qd = draft ? static_cast<double>(probability(to_float(draft[(k0 + lane) * p.d_k + d]))) : 1.0;
          stands = u * qd < pd;
        }
      }
      const uint32_t yes = __ballot_sync(0xffffffffu, stands);
      const int run = yes == 0xffffffffu ? 32 : __ffs(~yes) - 1;
      n += run;
      if (run < 32) break;
    }
    if (lane == 0) { s_accepted = n; }
  }
  __syncthreads();
  const int n = s_accepted;
  const bool rest = n < len;                                   // a draft was refused
  Weights<T> weights;
  weights.set(target + n * p.t_k, rest && draft ? draft + n * p.d_k : nullptr, rest && !draft ? d_row[n] : -1, p.V);

  // the row's blocks in equal runs of 32 k, one for each warp of the cluster
  const int blocks = weights.blocks(), runs = csize * kVerifyWarps, per_warp = (blocks + runs * 32 - 1) / (runs * 32) * 32;
  const int lo = min(blocks, (crank * kVerifyWarps + warp) * per_warp), hi = min(blocks, lo + per_warp);
  const int groups = (per_warp + kGroupBlocks<T> - 1) / kGroupBlocks<T>, per_slot = (groups + kVerifySlots - 2) / (kVerifySlots - 1);   // (and one for the rest)
  // The edges of this warp's interval. Neighbours compute a common edge by the same additions, so the intervals have neither gaps nor
  // overlaps whatever the rounding.
  double before = 0.0, behind = 0.0, total = 0.0;
  for (int attempt = 0; attempt < 2; ++attempt) {
    const double sum = warp_mass(weights, lo, hi, slots[warp], per_slot);
    if (lane == 0) warp_sums[warp] = sum;
    __syncthreads();
    double in_cta = 0.0;
#pragma unroll
    for (int w = 0; w < kVerifyWarps; ++w) {
      if (w == warp) before = in_cta;
      in_cta += warp_sums[w];
      if (w == warp) behind = in_cta;
    }
    if (attempt == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (threadIdx.x < csize) *cluster.map_shared_rank(&all_total[attempt][crank], threadIdx.x) = in_cta;
    cluster.sync();
    total = 0.0;
    double front = 0.0;
    for (int c = 0; c < csize; ++c) {
      if (c == crank) front = total;
      total += all_total[attempt][c];
    }
    before += front;
    behind += front;
    if (total > 0.0 || !rest || (weights.q == nullptr && weights.hole < 0)) break;
    weights.q = nullptr;   // the target has nothing beyond the draft: its own probabilities
    weights.hole = -1;
  }

  // ---- the drawn token: the warp whose interval holds the target finds the sum that holds it, reads these groups again, and in a group the row, the
  // lane and the token. Where the rounding of other orders of addition leaves nothing beyond the target: the last token with a weight. ----
  const double aim = fmax(u_last * total, 0.0);
  long long* out = p.tokens + static_cast<size_t>(b) * (p.K + 1);
  if (before <= aim && aim < behind) {
    constexpr int N = Weights<T>::N, kTokens = kGroupBlocks<T> / 32;   // blocks of a group per lane
    const int i0 = weights.first_whole(lo), n_slots = max(0, weights.last_whole(hi) - i0) / kGroupBlocks<T> / per_slot + 1;
    __syncwarp();
    // the sums over the lanes: in each step a lane keeps half of the sums and takes the other lane's part of them, so that lane l ends with sum l / 2
    double of[kVerifySlots];
#pragma unroll
    for (int i = 0; i < kVerifySlots; ++i) of[i] = i < n_slots ? slots[warp][i * 32 + lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 1; o >>= 1)
#pragma unroll
      for (int i = 0; i < o / 2; ++i) {
        const bool up = (lane & o) != 0;
        const double keep = up ? of[i + o / 2] : of[i], give = up ? of[i] : of[i + o / 2];
        of[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    const double own = of[0] + __shfl_xor_sync(0xffffffffu, of[0], 1);
    double upto = own;
#pragma unroll
    for (int o = 2; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t with = __ballot_sync(0xffffffffu, own > 0.0), beyond = __ballot_sync(0xffffffffu, own > 0.0 && before + upto > aim);
    const int at = beyond ? __ffs(beyond) - 1 : with ? 31 - __clz(with) : 0, slot = at >> 1;   // that with the target, or the last one with a weight
    double run = before + __shfl_sync(0xffffffffu, upto - own, at);
    int pick = -1, kept = -1;   // the token; the last one with a weight so far
    const int span = per_slot * kGroupBlocks<T>, end = min(hi, i0 + (slot + 1) * span);
    for (int k = slot == 0 ? lo : i0 + slot * span; k < end && pick < 0; k += kGroupBlocks<T>) {   // kTokens neighbouring blocks a lane
      uint4 a[kTokens], b[kTokens];
#pragma unroll
      for (int r = 0; r < kTokens; ++r) weights.fetch(k + lane * kTokens + r, end, a[r], b[r]);
      double d[kTokens][N], part[kTokens], mine = 0.0;
      const int j0 = (k + lane * kTokens) * N - weights.off;   // the lane's first token
#pragma unroll
      for (int r = 0; r < kTokens; ++r) {
        part[r] = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) part[r] += d[r][e] = weights.weight(j0 + r * N + e, reinterpret_cast<const T*>(&a[r])[e], reinterpret_cast<const T*>(&b[r])[e]);
        mine += part[r];
      }
      double incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t some = __ballot_sync(0xffffffffu, mine > 0.0), hit = __ballot_sync(0xffffffffu, mine > 0.0 && run + incl > aim);
      if (some) {
        const int holder = hit ? __ffs(hit) - 1 : 31 - __clz(some);
        int found = -1, last = -1;
        if (lane == holder) {
          double here = run + (incl - mine);
#pragma unroll
          for (int r = 0; r < kTokens; ++r) {
            if (found < 0 && part[r] > 0.0) {
              double t = here;
#pragma unroll
              for (int e = 0; e < N; ++e) {
                t += d[r][e];
                if (d[r][e] > 0.0) {
                  last = j0 + r * N + e;
                  if (found < 0 && t > aim) found = last;
                }
              }
            }
            here += part[r];
          }
        }
        kept = __shfl_sync(0xffffffffu, hit && found >= 0 ? found : last, holder);
        if (hit) pick = kept;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) out[n] = pick >= 0 ? pick : kept;
  }
  if (crank == 0) {
    if (!(aim < total)) {   // nothing has a weight (-1), or a number that is not below one
      const int last = total > 0.0 ? last_weight(weights, 0, p.V, &s_last) : -1;
      if (threadIdx.x == 0) out[n] = last;
    }
    if (threadIdx.x == 0) p.accepted[b] = n;
    for (int k = threadIdx.x; k <= p.K; k += kVerifyThreads)
      if (k != n) out[k] = k < n ? d_row[k] : -1;
  }
}

template <typename T>
static int launch_verify(const VerifyParams& p, int B, cudaStream_t s) {
  // CTAs per sequence: a wave of two per SM, but at least 32 KB of the rows to each
  const long long row = static_cast<long long>(p.V) * sizeof(T) * (p.draft ? 2 : 1);
  int ctas = 1;
  while (ctas < kVerifyMaxCtas && 2LL * ctas * B <= 2 * sm_count() && row / (2 * ctas) >= 32 << 10) ctas *= 2;
  auto kernel = verify_drafts_kernel<T>;
  static bool configured[64] = {false};
  int dev = 0;
  B200_CHECK_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    B200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(B) * ctas);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  B200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return kOk;
}

}  // namespace b200

using namespace b200;

// drafts int64 [B, K]; target [B, K + 1, V] and draft (nullable) [B, K, V] of one type (bf16, f16, f32) with unit stride along V and the given
// strides; uniform fp32 [B, K + 1]; lens nullable int32 [B]; accepted int32 [B]; tokens int64 [B, K + 1].
B200_API int b200_verify_drafts(const long long* drafts, const void* target, long long t_b, long long t_k, const void* draft, long long d_b, long long d_k,
                                const float* uniform, const int* lens, int B, int K, int V, int* accepted, long long* tokens, int dtype, void* stream) {
  B200_REQUIRE(B >= 0 && K >= 0 && V >= 1, "verify_drafts: bad sizes");
  B200_REQUIRE(B <= 1 << 24 && V <= 1 << 30, "verify_drafts: too many sequences or tokens");
  if (B == 0) return kOk;
  VerifyParams p;
  p.drafts = drafts; p.target = target; p.draft = draft; p.uniform = uniform; p.lens = lens; p.t_b = t_b; p.t_k = t_k; p.d_b = d_b; p.d_k = d_k;
  p.K = K; p.V = V; p.accepted = accepted; p.tokens = tokens;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  B200_DISPATCH_FLOAT(dtype, return launch_verify<T>(p, B, s););
}
