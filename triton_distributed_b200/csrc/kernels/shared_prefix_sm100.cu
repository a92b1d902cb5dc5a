// The shared keys of a batch on the tensor cores: partial attention of all rows that share a KV head over a range of the shared keys
// (what is merged and when this kernel is taken: shared_prefix.cu).
//
// A row is a query token and one of the G query heads of a KV head; a tile holds floor(128 / G) tokens, 128 rows at most. Every row sees
// every shared key (sequences that do not are attended by themselves), so nothing is masked but what lies behind the last key.
// A CTA takes two tiles over one range of keys in steps of 128; the tiles are two blocks of rows that use the same K and V tiles in
// shared memory, or, where all rows fit one tile (kTwoRanges), the same rows over the even and the odd steps, each with K and V tiles of
// its own. While the softmax of one tile runs, the tensor core computes the other tile's products (two tiles in turn: published as
// ping-pong scheduling, FlashAttention-3, Shah et al. 2024):
//   warps 0-3    softmax of tile 0, one thread per row
//   warps 4-7    softmax of tile 1
//   warp 8       TMA producer: the query tiles, then K and V tiles page by page through their rings (128-byte swizzle)
//   warp 9       one elected thread issues tcgen05.mma, for each step and tile O += P V of this step, then S = Q K^T of the next
// Tensor memory: S of tile t at columns 128 t, O of tile t at 256 + 128 t. P is written over S as 16-bit pairs and is the A operand of
// the second product; V is read in place as an MN-major B operand.
// The softmax of a step does not wait for its maximum: the weights are taken against the reference of the steps before (at the first step: the maximum
// of its first 32 keys), and only if one of a warp's scores lies above it by more than 8 (a factor of 256; published as conditional rescaling,
// FlashAttention-4, Zadouri et al. 2026) the warp raises its rows' references to their maxima, rescales their output and takes the step's weights
// anew from the scores, which are still there because the weights stay in registers until then. The maximum
// of the first keys mostly stands, so this is rare, and the chain of a step is one pass over the scores instead of two (two passes at the first step
// only, for the maximum of all its keys: 18.0 instead of 17.1 us for 16 rows of 64 / 8 heads over 2048 keys). Weights above one are rounded like those
// below (relative to themselves); what is lost is that a row's largest weight was held exactly: error against 64 bits 2.3e-3 of the norm both ways.
// Pages: a step's 128 keys are one copy, or 128 / p of p keys, p the largest power of two that divides a page; page numbers are read a window of 32 ahead by
// the producer's lanes. Pages outside the cache are copies from behind its end, which give zeros.
// Rows leave their normalised output in fp32 and their log-sum-exp, one range per CTA.
#include "b200/host.h"
#include "b200/packed_f32.cuh"
#include "b200/primitives.cuh"
#include "b200/shared_prefix.cuh"
#include "b200/tcgen05.cuh"

namespace b200 {

constexpr int kXM = 128, kXN = 128;            // rows per tile, keys per step
constexpr int kXAtom = 128 * 64 * 2;           // 128 rows x 64 columns of 16 bits: 16 KB
constexpr int kXThreads = 384;
constexpr int kXSoftmaxRegs = 208, kXOtherRegs = 88;   // 256 x 208 + 128 x 88 = 384 x 168, what the block starts with
constexpr float kXRaise = 8.f;                 // a score so far above the reference raises it (weights up to 2^8; f16 holds 2^8 times as much)
template <int kAtoms, bool kTwoRanges>
struct PrefixShape {
  static constexpr int kTile = kAtoms * kXAtom;
  static constexpr int kQTiles = kTwoRanges ? 1 : 2;
  static constexpr int kStages = kTwoRanges ? (kAtoms == 2 ? 3 : 4) : (kAtoms == 2 ? 2 : 4);   // of K, and as many of V
  static constexpr int kSmem = kQTiles * kTile + 2 * kStages * kTile + 1024 /*alignment*/ + 256 /*barriers*/;
};

// Keys per copy: the largest power of two that divides a page, so that a copy lies in one page, and steps consist of whole copies.
__host__ __device__ __forceinline__ int prefix_copy_rows(int page) {
  const int rows = page & -page;
  return rows < kXN ? rows : kXN;
}
__device__ __forceinline__ float prefix_exp2(float x) {   // one instruction; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {   // NaN if one of them is
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ void store_32_bytes(float* dst, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
               "f"(v[6]), "f"(v[7]) : "memory");
}

// blockIdx: x = range of keys, y = pair of tiles (kTwoRanges: tile), z = KV head
template <int kAtoms, bool BF16, bool kTwoRanges>
__global__ void __launch_bounds__(kXThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const SharedPrefixParams p) {
  using Shape = PrefixShape<kAtoms, kTwoRanges>;
  constexpr int kTile = Shape::kTile, kSt = Shape::kStages, D = kAtoms * 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                              // [query tiles][atoms]
  uint8_t* sK = sQ + Shape::kQTiles * kTile;       // [stages][atoms]
  uint8_t* sV = sK + kSt * kTile;                  // [stages][atoms]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kSt * kTile);
  uint64_t* q_full = bars;           // [1]
  uint64_t* k_full = bars + 1;       // [4]
  uint64_t* k_empty = bars + 5;      // [4]
  uint64_t* v_full = bars + 9;       // [4]
  uint64_t* v_empty = bars + 13;     // [4]
  uint64_t* s_full = bars + 17;      // [2 tiles] scores are in tensor memory (and the tile's earlier products are done)
  uint64_t* p_full = bars + 19;      // [2 tiles] probabilities are in tensor memory, and the output has been rescaled
  uint64_t* o_full = bars + 21;      // [2 tiles] the last product is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t timeout_ns = 4000000000ull;
  const int G = p.Hq / p.Hkv, tile_tokens = kXM / G, tile_rows = tile_tokens * G, all_tokens = p.B * p.T;
  const int kvh = blockIdx.z, split = blockIdx.x;
  // tile t: rows of tokens [token0[t], ...), steps[t] steps of 128 keys
  const int key0 = split * p.prefix_chunk, key1 = min(p.shared, key0 + p.prefix_chunk);
  const int n_steps = max(0, (key1 - key0 + kXN - 1) / kXN);   // (none in a range behind the last key)
  auto token0_of = [&](int t) { return (kTwoRanges ? static_cast<int>(blockIdx.y) : 2 * static_cast<int>(blockIdx.y) + t) * tile_tokens; };
  auto steps_of = [&](int t) { return kTwoRanges ? (n_steps + 1 - t) / 2 : token0_of(t) < all_tokens ? n_steps : 0; };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_full + t, 4);
      mbar_init(o_full + t, 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // rows of a tile that hold no head: zeros, so that nothing (not even NaN) keeps the rescaling busy
  for (int i = threadIdx.x; i < Shape::kQTiles * kAtoms * (kXM - tile_rows) * 8; i += kXThreads) {
    const int chunk = i & 7, r = (i >> 3) % (kXM - tile_rows) + tile_rows, a = (i >> 3) / (kXM - tile_rows);
    *reinterpret_cast<uint4*>(sQ + a * kXAtom + r * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_view_async_shared();
  if (warp == 10) tmem_alloc(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kXOtherRegs));
    if (warp == 8) {
      // ---------------------------------------------------------------- TMA producer: the warp reads page numbers, every lane copies a part of a step
      const int rows = prefix_copy_rows(p.page), pieces = kXN / rows;   // keys per copy, copies per step
      const int piece0 = key0 / rows, piece_end = (p.shared + rows - 1) / rows;   // copies are numbered from the first key on
      auto page_at = [&](int piece) -> int {   // first slot of a copy (behind the cache's end where there is no such page)
        if (piece >= piece_end) return 0;
        const int per_page = p.page / rows, blk = p.prefix_table[piece / per_page];
        return blk >= 0 && blk < p.num_blocks ? blk * p.page + piece % per_page * rows : p.num_blocks * p.page;
      };
      bool ok = true;
      if (lane == 0 && n_steps > 0) {
        int tiles = 0;
        for (int t = 0; t < Shape::kQTiles; ++t) tiles += token0_of(t) < all_tokens;
        mbar_expect_tx(q_full, tiles * kAtoms * tile_rows * 128);
        for (int t = 0; t < Shape::kQTiles; ++t)
          if (token0_of(t) < all_tokens)
#pragma unroll
            for (int a = 0; a < kAtoms; ++a) tma_load_3d(sQ + t * kTile + a * kXAtom, &tmQ, q_full, 64 * a, kvh * G, token0_of(t));
      }
      int window = piece0, now = page_at(piece0 + lane), next = page_at(piece0 + 32 + lane);
      const int piece = lane / kAtoms, atom = lane % kAtoms;   // each lane makes one copy of a step (24 x 5 drafts, pages of 16: 33.5 us, 40 with one lane for all)
      int done = 0;
      for (int j = 0; j < n_steps; ++j) {
        const int st = j % kSt;
        const int first = piece0 + j * pieces, n = min(pieces, (key1 - key0 - j * kXN + rows - 1) / rows);
        if (first - window >= 32) {   // (pieces divide 32: a step never straddles two windows)
          window += 32;
          now = next;
          next = page_at(window + 32 + lane);
        }
        const int slot = __shfl_sync(0xffffffffu, now, first - window + piece);   // (of the lanes' copies; behind the step's last one unused)
        ok = mbar_wait(k_empty + st, ((j / kSt) & 1) ^ 1, abort_flag, timeout_ns);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(k_full + st, n * rows * 128 * kAtoms);
        __syncwarp();
        if (piece < n) tma_load_3d(sK + st * kTile + atom * kXAtom + piece * rows * 128, &tmK, k_full + st, 64 * atom, kvh, slot);
        ok = mbar_wait(v_empty + st, ((j / kSt) & 1) ^ 1, abort_flag, timeout_ns);
        if (!__all_sync(0xffffffffu, ok)) { done = -(j + 1); break; }   // (K of this step is on its way)
        if (lane == 0) mbar_expect_tx(v_full + st, n * rows * 128 * kAtoms);
        __syncwarp();
        if (piece < n) tma_load_3d(sV + st * kTile + atom * kXAtom + piece * rows * 128, &tmV, v_full + st, 64 * atom, kvh, slot);
        done = j + 1;
      }
      // after an abort nothing waits for the last copies any more: they have to land before shared memory is given back
      if (lane == 0 && n_steps > 0 && *abort_flag != 0u) {
        volatile uint32_t never = 0;
        const int kc = done < 0 ? -done : done, vc = done < 0 ? -done - 1 : done;
        mbar_wait(q_full, 0, &never, timeout_ns);
        for (int c = max(0, kc - kSt); c < kc; ++c) mbar_wait(k_full + c % kSt, (c / kSt) & 1, &never, timeout_ns);
        for (int c = max(0, vc - kSt); c < vc; ++c) mbar_wait(v_full + c % kSt, (c / kSt) & 1, &never, timeout_ns);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---------------------------------------------------------------- MMA issuer
      if (elect_one()) {
        const uint32_t idesc_s = umma_idesc_f16(kXM, kXN, BF16);
        const uint32_t idesc_o = umma_idesc_f16(kXM, D, BF16) | 1u << 16;   // V as it stands is an MN-major B operand
        // Descriptors differ in their low word. The compiler must not see that the words below come from loop invariants: it would keep
        // dozens of finished descriptors and spill.
        const uint64_t dk = umma_desc_sw128_kmajor(0), dv = umma_desc_sw128_mnmajor(0, kXAtom);
        const uint32_t hi = static_cast<uint32_t>(dk >> 32), lo_k = static_cast<uint32_t>(dk), lo_v = static_cast<uint32_t>(dv);
        auto hide = [](uint32_t x) { asm volatile("" : "+r"(x)); return x; };
        auto desc = [&](uint32_t lo) { return static_cast<uint64_t>(hi) << 32 | lo; };
        auto scores = [&](int t, int st) {   // S_t = Q_t K^T
          const uint32_t a = hide(lo_k + (smem_u32(sQ + (kTwoRanges ? 0 : t) * kTile) >> 4)), b = hide(lo_k + (smem_u32(sK + st * kTile) >> 4));
#pragma unroll
          for (int kk = 0; kk < kAtoms * 4; ++kk) {
            const uint32_t step = ((kk >> 2) * kXAtom >> 4) + 2 * (kk & 3);
            umma_f16(tmem_base + t * kXN, desc(a + step), desc(b + step), idesc_s, kk != 0);
          }
          umma_commit(s_full + t);
        };
        auto output = [&](int t, int st, bool more) {   // O_t (+)= P_t V
          const uint32_t b = hide(lo_v + (smem_u32(sV + st * kTile) >> 4));
#pragma unroll
          for (int kk = 0; kk < kXN / 16; ++kk)
            umma_f16_ta(tmem_base + 2 * kXN + t * 128, tmem_base + t * kXN + kk * 8, desc(b + (kk * 16 * 128 >> 4)), idesc_o, more || kk != 0);
        };
        bool ok = n_steps > 0 && mbar_wait(q_full, 0, abort_flag, timeout_ns);
        if (kTwoRanges) {
          auto begin = [&](int c) {   // scores of step c
            ok = ok && mbar_wait(k_full + c % kSt, (c / kSt) & 1, abort_flag, timeout_ns);
            if (!ok) return;
            tc_fence_after_sync();
            scores(c & 1, c % kSt);
            umma_commit(k_empty + c % kSt);
          };
          if (ok) begin(0);
          if (n_steps > 1) begin(1);
          for (int c = 0; c < n_steps && ok; ++c) {
            const int t = c & 1;
            ok = mbar_wait(v_full + c % kSt, (c / kSt) & 1, abort_flag, timeout_ns) && mbar_wait(p_full + t, (c >> 1) & 1, abort_flag, timeout_ns);
            if (!ok) break;
            tc_fence_after_sync();
            output(t, c % kSt, c > 1);
            umma_commit(v_empty + c % kSt);
            if (c + 2 >= n_steps) umma_commit(o_full + t);
            else begin(c + 2);
          }
        } else {
          const bool two = steps_of(1) > 0;
          ok = ok && mbar_wait(k_full, 0, abort_flag, timeout_ns);
          if (ok) {
            tc_fence_after_sync();
            scores(0, 0);
            if (two) scores(1, 0);
            umma_commit(k_empty);
          }
          for (int j = 0; j < n_steps && ok; ++j) {
            const int st = j % kSt, st1 = (j + 1) % kSt;
            ok = mbar_wait(v_full + st, (j / kSt) & 1, abort_flag, timeout_ns);
            for (int t = 0; t < (two ? 2 : 1) && ok; ++t) {
              ok = mbar_wait(p_full + t, j & 1, abort_flag, timeout_ns);
              if (!ok) break;
              tc_fence_after_sync();
              output(t, st, j != 0);
              if (j == n_steps - 1) umma_commit(o_full + t);
              else {
                ok = mbar_wait(k_full + st1, ((j + 1) / kSt) & 1, abort_flag, timeout_ns);
                if (!ok) break;
                tc_fence_after_sync();
                scores(t, st1);
              }
            }
            if (!ok) break;
            umma_commit(v_empty + st);
            if (j + 1 < n_steps) umma_commit(k_empty + st1);
          }
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ softmax, one thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kXSoftmaxRegs));
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_addr = lanes + t * kXN, o_addr = lanes + 2 * kXN + t * 128;
    const int steps = steps_of(t);
    const int token = token0_of(t) + row / G;
    const bool mine = row < tile_rows && token < all_tokens;
    const bool valid = mine && n_steps > 0 && prefix_len(p, token / p.T) - p.T + 1 >= p.shared;   // (else the sequence ends inside the shared keys)
    float ref = -INFINITY, sum = 0.f;   // the row's reference (of scaled scores) and the sum of 2^(score - reference)
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int c_step = kTwoRanges ? 2 * j + t : j;
      ok = __all_sync(0xffffffffu, mbar_wait(s_full + t, j & 1, abort_flag, timeout_ns));
      if (!ok) break;
      tc_fence_after_sync();
      const int visible = key1 - key0 - c_step * kXN;
      uint32_t packed[4][16];
      f32x2 sums[2];
      auto fetch = [&](int c, uint32_t (&r)[32]) { tmem_ld_32x32(s_addr + c * 32, r); };
      auto hide_tail = [&](int c, uint32_t (&r)[32]) {   // scores behind the last key
        if (visible < (c + 1) * 32) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e >= visible) r[e] = __float_as_uint(-INFINITY);
        }
      };
      const f32x2 scale2 = pack2(p.scale_log2e, p.scale_log2e);
      auto weigh = [&](int c, const uint32_t (&r)[32], f32x2 base2) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          // 2^(s * scale - reference): one fused multiply-add for two scores, one special-function instruction each
          const float2 x = unpack2(fma2(pack2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), scale2, base2));
          const float p0 = prefix_exp2(x.x), p1 = prefix_exp2(x.y);
          sums[e & 1] = add2(sums[e & 1], pack2(p0, p1));
          packed[c][e] = BF16 ? pack_bf16x2(p0, p1) : pack_f16x2(p0, p1);
        }
      };
      float mx = -INFINITY;   // of the scores; NaN if one of them is
      auto look = [&](const uint32_t (&r)[32]) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) mx = max3_nan(mx, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
      };
      sums[0] = sums[1] = pack2(0.f, 0.f);
      {
        uint32_t r[2][32];
        fetch(0, r[0]);
        tmem_ld_wait();
        fetch(1, r[1]);
        hide_tail(0, r[0]);
        look(r[0]);
        if (j == 0) ref = mx * p.scale_log2e;   // the first reference: the maximum of the first keys (none if that is NaN)
        const f32x2 base2 = pack2(-ref, -ref);
        weigh(0, r[0], base2);
#pragma unroll
        for (int c = 1; c < 4; ++c) {
          tmem_ld_wait();
          if (c < 3) fetch(c + 1, r[(c + 1) & 1]);
          hide_tail(c, r[c & 1]);
          weigh(c, r[c & 1], base2);
          look(r[c & 1]);
        }
      }
      const bool raise = __any_sync(0xffffffffu, !(mx * p.scale_log2e - ref <= kXRaise));   // (also without a reference, and with NaN)
      if (raise) {
        const float top = fmaxf(ref, mx * p.scale_log2e), base = top == -INFINITY ? 0.f : top;
        const float corr = ref == -INFINITY || ref != ref ? 0.f : prefix_exp2(ref - base);
        ref = top;
        sum *= corr;
        if (j > 0) {
          // the scores of this step were issued after the tile's last product, so O is complete and nothing writes it now
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x16(o_addr + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st_32x16(o_addr + c * 16, o);
          }
        }
        sums[0] = sums[1] = pack2(0.f, 0.f);
        const f32x2 base2 = pack2(-base, -base);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          fetch(c, r);
          tmem_ld_wait();
          hide_tail(c, r);
          weigh(c, r, base2);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_st_32x16(s_addr + c * 16, packed[c]);
      sum += sum2(add2(sums[0], sums[1]));
      if (visible < kXN && (kTwoRanges || t == 0)) {
        // value rows behind the last key are zero for the product, whatever the stage held before. (Both tiles' products of this
        // step are issued after tile 0's probabilities have been announced.)
        const int st = c_step % kSt;
        ok = __all_sync(0xffffffffu, mbar_wait(v_full + st, (c_step / kSt) & 1, abort_flag, timeout_ns));
        if (!ok) break;
        for (int i = threadIdx.x & 127; i < (kXN - visible) * kAtoms * 8; i += 128) {
          const int key = visible + i / (kAtoms * 8), chunk = i % (kAtoms * 8);
          *reinterpret_cast<uint4*>(sV + st * kTile + (chunk >> 3) * kXAtom + key * 128 + (chunk & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_view_async_shared();
      }
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + t);
    }
    // ---- the row's range ----
    if (ok && steps > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(o_full + t, 0, abort_flag, timeout_ns));
      tc_fence_after_sync();
    }
    const size_t range = (static_cast<size_t>(token) * p.Hq + kvh * G + row % G) * p.S + split;
    float weight = 1.f, weight_other = 0.f;   // of this tile's output and of the other steps'
    // With two ranges the tiles exchange halves of their columns and each stores one. The K ring holds the halves, row by row, the 16-byte
    // chunks exchanged so that rows lie in all banks. (A tile's last product is issued after all products of scores, so nothing reads K now.)
    constexpr int kCols = kTwoRanges ? D / 2 : D, kChunks = D / 8;   // columns that a thread stores; 16-byte chunks of a half row
    static_assert(!kTwoRanges || 2 * kXM * (kChunks * 16 + 8) <= kSt * kTile, "the K ring holds both tiles' halves, references and sums");
    const int col0 = kTwoRanges ? t * kCols : 0;
    float4* other = reinterpret_cast<float4*>(sK) + (t * kXM + row) * kChunks;   // what the other tile left of this tile's columns
    float2* s_stat = reinterpret_cast<float2*>(sK + 2 * kXM * kChunks * 16);   // [2 tiles][128 rows] references and sums
    const bool both = kTwoRanges && n_steps > 1;
    if constexpr (kTwoRanges) {
      if (both && ok) {
        float4* left = reinterpret_cast<float4*>(sK) + ((t ^ 1) * kXM + row) * kChunks;
        s_stat[t * kXM + row] = make_float2(ref, sum);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[16];
          tmem_ld_32x16(o_addr + (D / 2 - col0) + c * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            left[(c * 4 + q) ^ (row & (kChunks - 1))] = make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]), __uint_as_float(o[4 * q + 2]),
                                                                    __uint_as_float(o[4 * q + 3]));
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");   // (both tiles' warps get here, after an abort too)
      if (both && *abort_flag == 0u) {
        const float2 x = s_stat[(t ^ 1) * kXM + row];
        const float top = fmaxf(ref, x.x), base = top == -INFINITY ? 0.f : top;
        weight = prefix_exp2(ref - base);
        weight_other = prefix_exp2(x.x - base);
        sum = sum * weight + x.y * weight_other;
        ref = top;
      }
    }
    const bool stores = ok && (kTwoRanges ? both || t == 0 : true);   // (with one step the first tile has all columns)
    if (stores && mine && (!kTwoRanges || t == 0)) p.lse_part[range] = valid && steps > 0 ? (ref + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    if (stores && steps > 0) {
      const float inv = 1.f / sum;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        if (kTwoRanges && c >= kCols / 16 && both) break;
        const int col = (kTwoRanges && !both ? 0 : col0) + c * 16;
        uint32_t o[16];
        tmem_ld_32x16(o_addr + col, o);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[q * 8 + e]) * weight;
          if (both) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float4 x = other[(c * 4 + q * 2 + h) ^ (row & (kChunks - 1))];
              v[4 * h] += x.x * weight_other; v[4 * h + 1] += x.y * weight_other; v[4 * h + 2] += x.z * weight_other; v[4 * h + 3] += x.w * weight_other;
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= inv;
          if (valid) store_32_bytes(p.o_part + range * D + col + q * 8, v);
        }
      }
    }
  }

  // ---------------------------------------------------------------------- teardown
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 10) tmem_dealloc(tmem_base, 512);
  if (threadIdx.x == 0 && *abort_flag != 0u && p.status != nullptr) atomicMax(p.status, static_cast<uint32_t>(kStatusPipeTimeout));
}

template <int kAtoms, bool BF16, bool kTwoRanges>
static int launch_prefix(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const SharedPrefixParams& p, dim3 grid, cudaStream_t s) {
  constexpr int kSmem = PrefixShape<kAtoms, kTwoRanges>::kSmem;
  static bool configured[64] = {false};
  int dev = 0;
  B200_CHECK_CUDA(cudaGetDevice(&dev));
  auto kernel = shared_prefix_kernel<kAtoms, BF16, kTwoRanges>;
  if (!configured[dev & 63]) {
    cudaFuncAttributes attr;
    B200_CHECK_CUDA(cudaFuncGetAttributes(&attr, kernel));   // the warps' register shares must not exceed what the block starts with
    if (attr.numRegs * kXThreads < 256 * kXSoftmaxRegs + 128 * kXOtherRegs)
      return set_error(kErrUnsupported, "shared-prefix kernel was compiled for %d registers", attr.numRegs);
    B200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    configured[dev & 63] = true;
  }
  B200_CHECK_CUDA(launch_pdl(kernel, grid, kXThreads, kSmem, s, tq, tk, tv, p));
  return kOk;
}

static int row_tiles(const SharedPrefixParams& p) {
  const int tokens = kXM / (p.Hq / p.Hkv);   // of a tile
  return (p.B * p.T + tokens - 1) / tokens;
}

// Whether the kernel handles a call at all: whole groups of query heads in a tile, pages of whole swizzle atoms (8 keys), slots that a 32-bit
// coordinate reaches, pairs of tiles and KV heads that a grid holds.
bool shared_prefix_tc_takes(const SharedPrefixParams& p, int D) {
  return p.shared > 0 && p.Hq / p.Hkv <= kXM && (D == 64 || D == 128) && p.page % 8 == 0 &&
         static_cast<long long>(p.num_blocks) * p.page < 0x7fffff00LL && p.Hkv <= 65535 && row_tiles(p) <= 2 * 65535;
}

// p.prefix_splits ranges of p.prefix_chunk keys (a multiple of 128).
int shared_prefix_tc_launch(const SharedPrefixParams& p, int D, int dtype, cudaStream_t s) {
  const int G = p.Hq / p.Hkv, tile_tokens = kXM / G, tiles = row_tiles(p);
  const bool two_ranges = tiles == 1;
  const int rows = prefix_copy_rows(p.page);
  const uint64_t slots = static_cast<uint64_t>(p.num_blocks) * p.page;
  CUtensorMap tq, tk, tv;
  int rc = make_tma_3d(&tq, p.q, dtype, D, p.Hq, static_cast<uint64_t>(p.B) * p.T, D, static_cast<uint64_t>(p.ldq), 64, G, tile_tokens, true);
  if (rc == kOk) rc = make_tma_3d(&tk, p.k_cache, dtype, D, p.Hkv, slots, D, static_cast<uint64_t>(p.Hkv) * D, 64, 1, rows, true);
  if (rc == kOk) rc = make_tma_3d(&tv, p.v_cache, dtype, D, p.Hkv, slots, D, static_cast<uint64_t>(p.Hkv) * D, 64, 1, rows, true);
  if (rc != kOk) return rc;
  const dim3 grid(p.prefix_splits, two_ranges ? 1 : (tiles + 1) / 2, p.Hkv);
#define B200_PREFIX(A, TWO) (dtype == kBF16 ? launch_prefix<A, true, TWO>(tq, tk, tv, p, grid, s) : launch_prefix<A, false, TWO>(tq, tk, tv, p, grid, s))
  if (D == 128) return two_ranges ? B200_PREFIX(2, true) : B200_PREFIX(2, false);
  return two_ranges ? B200_PREFIX(1, true) : B200_PREFIX(1, false);
#undef B200_PREFIX
}

}  // namespace b200
