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
// of the one row (two with draft probabilities) that is needed, the CTAs exchange their sums through distributed shared memory,
// and the warp whose interval holds the target walks its run once more, which the caches still have. One pass over memory.
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

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double warp_sum_of[kVerifyWarps];
  __shared__ double x_total, all_total[kVerifyMaxCtas];
  __shared__ int x_last, all_last[kVerifyMaxCtas];
  __shared__ int s_accepted, s_last;
  const int crank = static_cast<int>(cluster.block_rank()), csize = static_cast<int>(cluster.num_blocks());
  const int b = blockIdx.x / csize;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch_dependents();

  // ---- how many drafts stand ----
  const int len = p.lens ? max(0, min(p.K, p.lens[b])) : p.K;
  const long long* d_row = p.drafts + static_cast<size_t>(b) * p.K;
  const float* u_row = p.uniform + static_cast<size_t>(b) * (p.K + 1);
  const T* target = static_cast<const T*>(p.target) + b * p.t_b;
  const T* draft = p.draft ? static_cast<const T*>(p.draft) + b * p.d_b : nullptr;
  if (warp == 0) {
    int n = 0;
    for (int k0 = 0; k0 < len; k0 += 32) {
      bool stands = false;
      if (k0 + lane < len) {
        const long long d = d_row[k0 + lane];
        if (d >= 0 && d < p.V) {
          const double pd = probability(to_float(target[(k0 + lane) * p.t_k + d]));
          const double qd = draft ? static_cast<double>(probability(to_float(draft[(k0 + lane) * p.d_k + d]))) : 1.0;
          stands = static_cast<double>(u_row[k0 + lane]) * qd < pd;
        }
      }
      const uint32_t yes = __ballot_sync(0xffffffffu, stands);
      const int run = yes == 0xffffffffu ? 32 : __ffs(~yes) - 1;
      n += run;
      if (run < 32) break;
    }
    if (lane == 0) s_accepted = n;
  }
  __syncthreads();
  const int n = s_accepted;
  const T* pr = target + n * p.t_k;
  const bool rest = n < len;                                   // a draft was refused
  const T* qr = rest && draft ? draft + n * p.d_k : nullptr;
  const long long refused = rest && !draft ? d_row[n] : -1;    // has no weight

  const int per_cta = (p.V + csize - 1) / csize;
  const int per_warp = ((per_cta + kVerifyWarps - 1) / kVerifyWarps + 31) / 32 * 32;
  const int c0 = min(p.V, crank * per_cta), c1 = min(p.V, c0 + per_cta);
  const int lo = min(c1, c0 + warp * per_warp), hi = min(c1, lo + per_warp);
  bool minus = true;   // subtract the draft's probabilities
  auto weight = [&](int j) -> double {
    double w = probability(to_float(pr[j]));
    if (minus) {
      if (qr) w = fmax(w - static_cast<double>(probability(to_float(qr[j]))), 0.0);
      else if (j == refused) w = 0.0;
    }
    return w;
  };
  // The edges of this warp's interval. Neighbours compute a common edge by the same additions, so the intervals have neither gaps nor
  // overlaps whatever the rounding.
  double before = 0.0, behind = 0.0, total = 0.0;
  int last = -1;
  for (int attempt = 0; attempt < 2; ++attempt) {
    double sum = 0.0;
    last = -1;   // the last token with a weight
    for (int j = lo + lane; j < hi; j += 32) {
      const double w = weight(j);
      sum += w;
      if (w > 0.0) last = j;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    }
    if (threadIdx.x == 0) s_last = -1;
    __syncthreads();
    if (lane == 0) {
      warp_sum_of[warp] = sum;
      atomicMax(&s_last, last);
    }
    __syncthreads();
    double in_cta = 0.0;
    for (int w = 0; w < kVerifyWarps; ++w) {
      if (w == warp) before = in_cta;
      in_cta += warp_sum_of[w];
      if (w == warp) behind = in_cta;
    }
    if (threadIdx.x == 0) {
      x_total = in_cta;
      x_last = s_last;
    }
    cluster.sync();
    if (threadIdx.x < csize) {
      all_total[threadIdx.x] = *cluster.map_shared_rank(&x_total, threadIdx.x);
      all_last[threadIdx.x] = *cluster.map_shared_rank(&x_last, threadIdx.x);
    }
    cluster.sync();
    total = 0.0;
    last = -1;
    double front = 0.0;
    for (int c = 0; c < csize; ++c) {
      if (c == crank) front = total;
      total += all_total[c];
      last = max(last, all_last[c]);
    }
    before += front;
    behind += front;
    if (total > 0.0 || !rest || !minus) break;
    minus = false;   // the target has nothing beyond the draft: its own probabilities
  }

  // ---- the drawn token: the warp whose interval holds the target walks its run ----
  const double aim = fmax(static_cast<double>(u_row[p.K]) * total, 0.0);
  long long* out = p.tokens + static_cast<size_t>(b) * (p.K + 1);
  if (before <= aim && aim < behind) {
    double run = before;
    int pick = -1, kept = -1;
    for (int j0 = lo; j0 < hi && pick < 0; j0 += 32) {
      const double w = j0 + lane < hi ? weight(j0 + lane) : 0.0;
      double incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, w > 0.0 && run + incl > aim), some = __ballot_sync(0xffffffffu, w > 0.0);
      if (hit) pick = j0 + __ffs(hit) - 1;
      if (some) kept = j0 + 31 - __clz(some);
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) out[n] = pick >= 0 ? pick : kept;   // (the walk's own rounding at the interval's end: the last with a weight)
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

template <typename T>
static int launch_verify(const VerifyParams& p, int B, cudaStream_t s) {
  // CTAs per sequence: enough of them to keep the memory busy
  const int ctas = B <= 18 ? 16 : B <= 37 ? 8 : B <= 148 ? 4 : 2;
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
  B200_REQUIRE(B <= 1 << 24, "verify_drafts: too many sequences");
  if (B == 0) return kOk;
  VerifyParams p;
  p.drafts = drafts; p.target = target; p.draft = draft; p.uniform = uniform; p.lens = lens; p.t_b = t_b; p.t_k = t_k; p.d_b = d_b; p.d_k = d_k;
  p.K = K; p.V = V; p.accepted = accepted; p.tokens = tokens;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  B200_DISPATCH_FLOAT(dtype, return launch_verify<T>(p, B, s););
}
