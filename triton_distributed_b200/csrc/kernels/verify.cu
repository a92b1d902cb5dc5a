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
// of the one row (two with draft probabilities) that is needed and the CTAs write their sums into each other's shared memory. The CTA with
// the warp whose interval holds the target cuts that run (which the caches still have) into a part for each warp, and the warp with the target walks its part. One
// pass over memory.
#include "b200/host.h"
#include "b200/elem.cuh"
#include "b200/primitives.cuh"

#include <cooperative_groups.h>
#include <cstring>

namespace b200 {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCtas = 16;   // per sequence

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

__device__ __forceinline__ float probability(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

// Elements that a lane reads at a time: 16 bytes where both rows start on 16 bytes, else one.
template <typename T, int N>
struct Lanes {
  float v[N];
  __device__ __forceinline__ void load(const T* p) {
    if (N == 1) { v[0] = to_float(p[0]); return; }
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = to_float(x[e]);
  }
};

// The weights of a row: max(p - q, 0) with q, p without the refused token otherwise.
template <typename T>
struct Weights {
  const T* p;
  const T* q;       // nullable
  long long hole;   // a token without a weight, or -1
  template <int N>
  __device__ __forceinline__ void operator()(int j, double (&w)[N]) const {   // of tokens j ... j + N - 1
    Lanes<T, N> a, b;
    a.load(p + j);
    if (q) b.load(q + j);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      w[e] = probability(a.v[e]);
      if (q) w[e] = fmax(w[e] - static_cast<double>(probability(b.v[e])), 0.0);
      else if (j + e == hole) w[e] = 0.0;
    }
  }
};

// The sum of the weights of [lo, hi) and the last token among them that has one (-1), by a warp; lo and hi are multiples of N but for the
// row's end. Groups of loads before any of their values is used.
template <typename T, int N>
__device__ __forceinline__ double warp_mass(const Weights<T>& weights, int lo, int hi, int& last) {
  constexpr int kStep = 32 * N, kGroup = N == 1 ? 8 : N == 8 ? 2 : 4;
  const int lane = threadIdx.x & 31;
  double sum[2] = {0.0, 0.0};
  int j = lo + lane * N;
  last = -1;
  for (; j + (kGroup - 1) * kStep + N <= hi; j += kGroup * kStep) {
    Lanes<T, N> a[kGroup], b[kGroup];
#pragma unroll
    for (int g = 0; g < kGroup; ++g) a[g].load(weights.p + j + g * kStep);
    if (weights.q)
#pragma unroll
      for (int g = 0; g < kGroup; ++g) b[g].load(weights.q + j + g * kStep);
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int at = j + g * kStep + e;
        const float x = probability(a[g].v[e]), y = weights.q ? probability(b[g].v[e]) : at == weights.hole ? x : 0.f;
        // (of the difference's double rounding nothing is lost where the sign is decided in 32 bits: it is exact there)
        if (x > y) {
          sum[e & 1] += static_cast<double>(x) - static_cast<double>(y);
          last = at;
        }
      }
  }
  for (; j < hi; j += kStep) {
    if (j + N <= hi) {
      double w[N];
      weights(j, w);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (w[e] > 0.0) { sum[e & 1] += w[e]; last = j + e; }
    } else {
      for (int e = 0; j + e < hi; ++e) {
        double w[1];
        weights(j + e, w);
        if (w[0] > 0.0) { sum[0] += w[0]; last = j + e; }
      }
    }
  }
  double total = sum[0] + sum[1];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  }
  return total;
}

template <typename T, int N>
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double warp_sums[kVerifyWarps];
  __shared__ int warp_last[kVerifyWarps];
  __shared__ double all_total[2][kVerifyMaxCtas];   // written by all CTAs of the cluster, for each attempt
  __shared__ int all_last[2][kVerifyMaxCtas];
  __shared__ int s_accepted, s_run;
  __shared__ double s_before;
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
    if (lane == 0) { s_accepted = n; s_run = -1; }
  }
  __syncthreads();
  const int n = s_accepted;
  const bool rest = n < len;                                   // a draft was refused
  Weights<T> weights = {target + n * p.t_k, rest && draft ? draft + n * p.d_k : nullptr, rest && !draft ? d_row[n] : -1};

  // CTA c takes [c * per_cta, ...), its warp w [w * per_warp, ...) of that; all but the row's end are multiples of 32 N
  constexpr int kUnit = 32 * N;
  const int per_warp = (p.V + csize * kVerifyWarps * kUnit - 1) / (csize * kVerifyWarps * kUnit) * kUnit;
  const int lo = static_cast<int>(min(static_cast<long long>(p.V), (static_cast<long long>(crank) * kVerifyWarps + warp) * per_warp));
  const int hi = min(p.V, lo + per_warp);
  // The edges of this warp's interval. Neighbours compute a common edge by the same additions, so the intervals have neither gaps nor
  // overlaps whatever the rounding.
  double before = 0.0, behind = 0.0, total = 0.0;
  int last = -1;
  for (int attempt = 0; attempt < 2; ++attempt) {
    int my_last;
    const double sum = warp_mass<T, N>(weights, lo, hi, my_last);
    if (lane == 0) { warp_sums[warp] = sum; warp_last[warp] = my_last; }
    __syncthreads();
    double in_cta = 0.0;
    int cta_last = -1;
#pragma unroll
    for (int w = 0; w < kVerifyWarps; ++w) {
      if (w == warp) before = in_cta;
      in_cta += warp_sums[w];
      if (w == warp) behind = in_cta;
      cta_last = max(cta_last, warp_last[w]);
    }
    if (attempt == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (threadIdx.x < csize) {
      *cluster.map_shared_rank(&all_total[attempt][crank], threadIdx.x) = in_cta;
      *cluster.map_shared_rank(&all_last[attempt][crank], threadIdx.x) = cta_last;
    }
    cluster.sync();
    total = 0.0;
    last = -1;
    double front = 0.0;
    for (int c = 0; c < csize; ++c) {
      if (c == crank) front = total;
      total += all_total[attempt][c];
      last = max(last, all_last[attempt][c]);
    }
    before += front;
    behind += front;
    if (total > 0.0 || !rest || (weights.q == nullptr && weights.hole < 0)) break;
    weights.q = nullptr;   // the target has nothing beyond the draft: its own probabilities
    weights.hole = -1;
  }

  // ---- the drawn token: the CTA that has the warp whose interval holds the target cuts that interval anew, a part to each warp ----
  const double aim = fmax(u_last * total, 0.0);
  long long* out = p.tokens + static_cast<size_t>(b) * (p.K + 1);
  if (lane == 0 && before <= aim && aim < behind) { s_run = lo; s_before = before; }
  __syncthreads();
  if (s_run >= 0) {
    const int run_lo = s_run, run_hi = min(p.V, run_lo + per_warp);
    const int part = (per_warp / kVerifyWarps + N - 1) / N * N;   // (per_warp is at least 32 N, twice the warps)
    const int a0 = min(run_hi, run_lo + warp * part), a1 = warp == kVerifyWarps - 1 ? run_hi : min(run_hi, a0 + part);
    int my_last;
    const double sum = warp_mass<T, N>(weights, a0, a1, my_last);
    __syncthreads();
    if (lane == 0) { warp_sums[warp] = sum; warp_last[warp] = my_last; }
    __syncthreads();
    double edge = s_before;
    int chosen = -1, fallback = -1;
    double from = 0.0;
#pragma unroll
    for (int w = 0; w < kVerifyWarps; ++w) {
      const double next = edge + warp_sums[w];
      if (chosen < 0 && aim < next) { chosen = w; from = edge; }
      if (warp_last[w] >= 0) fallback = w;
      edge = next;
    }
    if (chosen < 0) {   // the new sums are a rounding shorter: the last token with a weight
      if (threadIdx.x == 0) out[n] = warp_last[fallback < 0 ? 0 : fallback];
    } else if (warp == chosen) {
      double run = from;
      int pick = -1, kept = -1;
      for (int j0 = a0; j0 < a1 && pick < 0; j0 += 32) {
        double w[1] = {0.0};
        if (j0 + lane < a1) weights(j0 + lane, w);
        double incl = w[0];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, w[0] > 0.0 && run + incl > aim), some = __ballot_sync(0xffffffffu, w[0] > 0.0);
        if (hit) pick = j0 + __ffs(hit) - 1;
        if (some) kept = j0 + 31 - __clz(some);
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) out[n] = pick >= 0 ? pick : kept;   // (the walk's own rounding at the end: the last with a weight)
    }
  }
  if (crank == 0) {
    if (threadIdx.x == 0) {
      p.accepted[b] = n;
      if (!(aim < total)) out[n] = last;   // nothing has a weight (-1), or a number that is not below one
    }
    for (int k = threadIdx.x; k <= p.K; k += kVerifyThreads)
      if (k != n) out[k] = k < n ? d_row[k] : -1;
  }
}

template <typename T, int N>
static int launch_verify(const VerifyParams& p, int B, cudaStream_t s) {
  // CTAs per sequence: enough of them to keep the memory busy
  const int ctas = B <= 18 ? 16 : B <= 37 ? 8 : B <= 148 ? 4 : 2;
  auto kernel = verify_drafts_kernel<T, N>;
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
  B200_REQUIRE(B <= 1 << 24, "verify_drafts: too many sequences");
  if (B == 0) return kOk;
  VerifyParams p;
  p.drafts = drafts; p.target = target; p.draft = draft; p.uniform = uniform; p.lens = lens; p.t_b = t_b; p.t_k = t_k; p.d_b = d_b; p.d_k = d_k;
  p.K = K; p.V = V; p.accepted = accepted; p.tokens = tokens;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // rows that all start on 16 bytes are read 16 bytes at a time
  const long long size = dtype_size(dtype);
  const bool wide = (reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft) | static_cast<uintptr_t>(t_b * size) |
                     static_cast<uintptr_t>(t_k * size) | (draft ? static_cast<uintptr_t>(d_b * size) | static_cast<uintptr_t>(d_k * size) : 0)) % 16 == 0;
  B200_DISPATCH_FLOAT(dtype, if (wide) return launch_verify<T, 16 / sizeof(T)>(p, B, s); return launch_verify<T, 1>(p, B, s););
}
