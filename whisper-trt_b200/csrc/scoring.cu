// Log-probabilities of given tokens, with entropy and best alternatives, from logits in hand: per row the log-softmax at
// one token, -sum p ln p, and the `top` largest logits with their tokens.
//
// Bound by the one read of the logits. A row is a CTA of 128 threads, 8 of them to an SM, or a cluster of up to 8 CTAs where
// there are few rows, exchanging through distributed shared memory. A thread takes every 128th 16-byte piece, four a
// round, the next round's loads out before this one's sums. In a round the maximum comes first (packed pairs for 16-bit logits),
// then the two sums of scoring.cuh, in paired fp32 instructions.
// The alternatives cost the pass nothing but that maximum: the `top` best tokens of a row lie with the `top` threads whose
// own best are best, so those threads are found (sorted by warp, then counted into place), and their pieces alone, about
// top / 128 of the row, are read again, from L2.
// Measured: 7136 rows x 51865, bf16 (740 MB) 131 us without alternatives (5.7 TB/s), 146 / 155 / 236 with 1 / 3 / 16, fp32 225
// (6.6 TB/s); in 16 bits the exponentials (16 a cycle) take 82 of it by themselves. A mask that leaves no piece alone:
// 236. 5 rows of fp32 with a mask and 5 alternatives, 8 CTAs each: 9.8.
#include <cooperative_groups.h>

#include "scoring.cuh"

namespace wt {
namespace {

constexpr int kLpThreads = 128;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpPieces = 4;        // 16-byte pieces per thread and round
constexpr int kLpRound = kLpThreads * kLpPieces;
constexpr int kLpCtas = 8;          // per SM
constexpr int kLpMaxCluster = 8;
constexpr int kLpMaxVocab = 1 << 20;  // (the suppressed tokens' bits in shared memory: 128 KB)
constexpr int kLpLists = kLpWarps > kLpMaxCluster ? kLpWarps : kLpMaxCluster;

template <typename T> struct Piece {  // a 16-byte piece of logits
  static constexpr int n = 8;
  static constexpr uint32_t kLow = Elem<T>::code == WT_BF16 ? 0xff80u : 0xfc00u;  // -inf
  static __device__ __forceinline__ void get(const uint4 &u, float *f) {
    unpack8<T>(u, *reinterpret_cast<float(*)[8]>(f));
  }
  static __device__ __forceinline__ float one(const T *p) { return Elem<T>::to_float(*p); }
  static __device__ __forceinline__ uint32_t raw(const T *p) { return *reinterpret_cast<const uint16_t *>(p); }
  // element i of a piece put into it
  static __device__ __forceinline__ void put(uint32_t (&w)[4], int i, uint32_t v) {
    w[i >> 1] = (i & 1) ? (w[i >> 1] & 0xffffu) | (v << 16) : (w[i >> 1] & 0xffff0000u) | v;
  }
  using P2 = typename Elem<T>::pair;
  static __device__ __forceinline__ P2 pair(uint32_t w) { return *reinterpret_cast<const P2 *>(&w); }
  static __device__ __forceinline__ P2 max2(const uint4 &u) {
    return __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w)));
  }
  static __device__ __forceinline__ float larger(P2 m) {
    const float2 f = Elem<T>::to_float2(*reinterpret_cast<const uint32_t *>(&m));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ float max(const uint4 &u) { return larger(max2(u)); }  // (NaN aside)
  static __device__ __forceinline__ float max4(const uint4 (&u)[4]) {
    return larger(__hmax2(__hmax2(max2(u[0]), max2(u[1])), __hmax2(max2(u[2]), max2(u[3]))));
  }
};
template <> struct Piece<float> {
  static constexpr int n = 4;
  static constexpr uint32_t kLow = 0xff800000u;
  static __device__ __forceinline__ void get(const uint4 &u, float *f) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float one(const float *p) { return *p; }
  static __device__ __forceinline__ uint32_t raw(const float *p) { return __float_as_uint(*p); }
  static __device__ __forceinline__ void put(uint32_t (&w)[4], int i, uint32_t v) { w[i] = v; }
  static __device__ __forceinline__ float max(const uint4 &u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ float max4(const uint4 (&u)[4]) {
    return fmaxf(fmaxf(max(u[0]), max(u[1])), fmaxf(max(u[2]), max(u[3])));
  }
};

struct LpShared {
  SoftStat stat[kLpWarps];
  Key list[kLpLists * kMaxTop];         // warps' (or CTAs') lists side by side
  Key best[kMaxTop];                    // what merge_lists leaves
  SoftStat cta;                         // this CTA's statistics, for the cluster
};

// The lists' `top` best -> sh.best.
__device__ __forceinline__ void merge_lists(LpShared &sh, int n, int top) {
  count_into_place(sh.list, n, top, sh.best);
}

struct LpArgs {
  const void *logits;
  const int64_t *tokens;
  const uint8_t *suppress;
  ScoreOut out;
  long long stride;
  int rows, vocab, top, cl;
};

template <typename T, bool MASKED>
__global__ void __launch_bounds__(kLpThreads, kLpCtas) logprobs_kernel(const LpArgs a) {
  namespace cg = cooperative_groups;
  using P = Piece<T>;
  extern __shared__ uint32_t bits[];  // the suppressed tokens of this CTA's pieces
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % a.cl;
  const uint32_t cid = blockIdx.x / a.cl, ncl = gridDim.x / a.cl;

  pdl_wait();
  pdl_launch_dependents();

  // Pieces of a row: 16-byte aligned ones; the first and the last may be cut short by the row's ends. With this CTA's
  // share [p0, p1) of them, its tokens lie within [p0 * n - (n - 1), p1 * n) whatever the row's alignment.
  const int npieces = (a.vocab + P::n - 1) / P::n + 1;
  const int p0 = static_cast<int>(static_cast<long long>(npieces) * rank / a.cl);
  const int p1 = static_cast<int>(static_cast<long long>(npieces) * (rank + 1) / a.cl);
  const int bit0 = (max(0, p0 * P::n - P::n) & ~31) - 32;  // the token of the first bit (a word before any there is)
  if (MASKED) {
    const int words = (min(a.vocab, p1 * P::n) - bit0 + 31) / 32 + 1;  // (one more: bits are read across words)
    const bool vec = (reinterpret_cast<uintptr_t>(a.suppress) & 15u) == 0;
    for (int w = tid; w < words; w += kLpThreads) {
      const int v = bit0 + w * 32;
      uint32_t b = 0;
      if (vec && v >= 0 && v + 32 <= a.vocab) {
        const uint4 lo = ldg16(a.suppress + v), hi = ldg16(a.suppress + v + 16);
        const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int k = 0; k < 8; ++k)  // four 0/1 bytes -> four bits
          b |= ((((u[k] & 0x01010101u) * 0x01020408u) >> 24) & 0xfu) << (4 * k);
      } else {
        for (int k = 0; k < 32; ++k) b |= v + k >= 0 && v + k < a.vocab && a.suppress[v + k] != 0 ? 1u << k : 0u;
      }
      bits[w] = b;
    }
    __syncthreads();
  }
  auto suppressed = [&](int v) { return (bits[(v - bit0) >> 5] >> ((v - bit0) & 31)) & 1u; };

  for (uint32_t row = cid; row < static_cast<uint32_t>(a.rows); row += ncl) {  // (rows < 2^31, ncl <= 2^30: no wrap)
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));  // piece 0 starts here
    // piece p: tokens p * n - shift .. + n - 1; `count` pieces from p0 on, the first and last may be cut short
    const int count = max(min(p1, (a.vocab + shift + P::n - 1) / P::n) - p0, 0);
    const int64_t tok = a.tokens[row];  // (for the end: on its way early)
    const bool has = tok >= 0 && tok < a.vocab;
    float xt = kNegInf;
    if (tid == 0 && rank == 0 && has && !(MASKED && a.suppress[tok] != 0)) xt = P::one(x + tok);
    auto load = [&](int i) {  // the i-th piece, -inf where there is no token
      const int v0 = (p0 + i) * P::n - shift;
      if (i < count && v0 >= 0 && v0 + P::n <= a.vocab) return ldg_stream(x + v0);
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < P::n; ++e)
        P::put(w, e, i < count && v0 + e >= 0 && v0 + e < a.vocab ? P::raw(x + v0 + e) : P::kLow);
      return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto mask = [&](int i, uint4 &u) {  // the suppressed ones out
      const int at = (p0 + i) * P::n - shift - bit0;
      const uint32_t gone = __funnelshift_r(bits[at >> 5], bits[(at >> 5) + 1], at & 31) & ((1u << P::n) - 1);
      if (gone != 0) {
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < P::n; ++e)
          if ((gone >> e) & 1u) P::put(w, e, P::kLow);
        u = make_uint4(w[0], w[1], w[2], w[3]);
      }
    };
    SoftStat st = soft_empty();
    int best_p = 0;  // the piece of this thread's (first) largest logit
    const T *at = x + (static_cast<long long>(p0 + tid) * P::n - shift);
    uint4 next[kLpPieces];
#pragma unroll
    for (int j = 0; j < kLpPieces; ++j) next[j] = load(j * kLpThreads + tid);
    for (int i0 = 0; i0 < count; i0 += kLpRound) {
      uint4 u[kLpPieces];
#pragma unroll
      for (int j = 0; j < kLpPieces; ++j) u[j] = next[j];
      at += kLpRound * P::n;
      if (i0 + 2 * kLpRound < count) {  // (the next round is whole, and the row goes on behind it)
#pragma unroll
        for (int j = 0; j < kLpPieces; ++j) next[j] = ldg_stream(at + j * kLpThreads * P::n);
      } else if (i0 + kLpRound < count) {
#pragma unroll
        for (int j = 0; j < kLpPieces; ++j) next[j] = load(i0 + kLpRound + j * kLpThreads + tid);
      }
      if (MASKED) {
#pragma unroll
        for (int j = 0; j < kLpPieces; ++j)
          if (i0 + j * kLpThreads + tid < count) mask(i0 + j * kLpThreads + tid, u[j]);
      }
      const float cm = P::max4(u);
      if (cm > st.m) {
        soft_raise(st, cm);
#pragma unroll
        for (int j = kLpPieces - 1; j >= 0; --j)
          if (P::max(u[j]) == cm) best_p = p0 + i0 + j * kLpThreads + tid;
      }
      const float base = soft_base(st.m);
      SoftSum sum;
      bool again = MASKED || i0 + kLpRound > count;  // (logits of -inf are expected)
      if (!again) {
#pragma unroll
        for (int j = 0; j < kLpPieces; ++j) {
          float f[P::n];
          P::get(u[j], f);
          sum.template add<P::n, false>(f, base);
        }
        again = sum.broken();  // (there was one, or a NaN)
      }
      if (again) {
        sum.restart();
#pragma unroll
        for (int j = 0; j < kLpPieces; ++j) {
          float f[P::n];
          P::get(u[j], f);
          sum.template add<P::n, true>(f, base);
        }
      }
      sum.into(st);
    }

    // the statistics of the CTA's threads; and, with alternatives, every warp's best threads, by their best token (the
    // piece it lies in gives the same order: a piece is one thread's)
    Key best_key = key_of(st.m, best_p);
    st = soft_merge_lanes(st);
    if (lane == 0) sh.stat[warp] = st;
    if (a.top > 0) {
      warp_sort(best_key);
      if (lane < a.top) sh.list[warp * a.top + lane] = best_key;
      merge_lists(sh, kLpWarps * a.top, a.top);
      // those threads' tokens again, as far as they reach the last of those maxima
      const float last_v = key_value(sh.best[a.top - 1]);
      Key found = 0;
      for (int k = warp; k < a.top; k += kLpWarps) {
        const int best = key_token(sh.best[k]);
        if (best < 0) break;
        const int th = (best - p0) % kLpThreads;
        const int tokens = (count - th + kLpThreads - 1) / kLpThreads * P::n;  // (cut short or not)
        constexpr int kBatch = 8;  // 32 tokens each, a token a lane, their loads together
        for (int e0 = lane; e0 - lane < tokens; e0 += 32 * kBatch) {
          float f[kBatch];
          int id[kBatch];
#pragma unroll
          for (int q = 0; q < kBatch; ++q) {
            const int e = e0 + q * 32, v = (p0 + th + e / P::n * kLpThreads) * P::n - shift + e % P::n;
            id[q] = v;
            f[q] = e < tokens && v >= 0 && v < a.vocab && !(MASKED && suppressed(v)) ? P::one(x + v) : kNegInf;
          }
#pragma unroll
          for (int q = 0; q < kBatch; ++q)
            if (__any_sync(0xffffffffu, f[q] >= last_v && f[q] > kNegInf))
              warp_insert(found, a.top, f[q] >= last_v ? key_of(f[q], id[q]) : 0);
        }
      }
      __syncthreads();  // (every warp has read the lists)
      if (lane < a.top) sh.list[warp * a.top + lane] = found;
      merge_lists(sh, kLpWarps * a.top, a.top);
    } else {
      __syncthreads();
    }
    if (warp == 0) {
      st = soft_merge_lanes(lane < kLpWarps ? sh.stat[lane] : soft_empty());
      if (lane == 0) sh.cta = st;
    }
    if (a.cl > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      if (rank == 0) {
        const int e = tid / kMaxTop, k = tid % kMaxTop;
        if (e < a.cl && k < a.top) {
          const LpShared *peer = cluster.map_shared_rank(&sh, e);
          sh.list[e * a.top + k] = peer->best[k];
        }
        if (warp == 0)
          st = soft_merge_lanes(lane < a.cl ? cluster.map_shared_rank(&sh, lane)->cta : soft_empty());
      }
      cluster.sync();  // (the peers' results may be overwritten, and the peers may leave)
      if (rank == 0 && a.top > 0) merge_lists(sh, a.cl * a.top, a.top);
    }
    if (rank == 0 && warp == 0) {
      write_scores(a.out, row, a.top, st, lane < a.top ? sh.best[lane] : 0, has, xt);
    }
    __syncthreads();  // (the shared arrays are free for the next row)
  }
}

template <typename T, bool MASKED>
int launch_logprobs(LpArgs a, int sms, void *stream) {
  // CTAs per row: as many as keep about 2 CTAs on every SM, and at least a round of pieces for each
  a.cl = 1;
  while (a.cl < kLpMaxCluster && a.rows <= sms / a.cl && a.vocab >= a.cl * 2 * kLpThreads * Piece<T>::n) a.cl *= 2;
  // with suppressed tokens a CTA's rows share the bits it makes of them; without, a CTA is a row
  constexpr int kMaxGrid = 1 << 30;
  int ncl = a.rows < kMaxGrid ? a.rows : kMaxGrid;
  if (MASKED && ncl > kLpCtas * sms / a.cl) ncl = kLpCtas * sms / a.cl;
  const int smem = MASKED ? ((a.vocab + 31) / 32 + 5) * 4 : 0;
  const int st = opt_in_smem<logprobs_kernel<T, MASKED>>(smem, "token_logprobs");
  if (st != WT_OK) return st;
  const dim3 grid(ncl * a.cl), block(kLpThreads);
  if (a.cl > 1) return launch_clustered("token_logprobs", logprobs_kernel<T, MASKED>, grid, block, smem, stream, a.cl, a);
  return launch("token_logprobs", logprobs_kernel<T, MASKED>, grid, block, smem, stream, a);
}

}  // namespace
}  // namespace wt

extern "C" int wt_token_logprobs(int dtype, const void *logits, long long row_stride, const int64_t *tokens,
                                 const uint8_t *suppress, float *logprob, float *entropy, float *top_logprob,
                                 int64_t *top_token, int rows, int vocab, int top, void *stream) {
  using namespace wt;
  WT_REQUIRE(rows > 0 && vocab > 0 && row_stride >= vocab, WT_ERR_ARG,
             "token_logprobs: sizes must be positive, the row stride at least the vocabulary (rows %d, vocab %d, stride "
             "%lld)",
             rows, vocab, row_stride);
  WT_REQUIRE(logits && tokens && logprob && entropy && (top == 0 || (top_logprob && top_token)), WT_ERR_ARG,
             "token_logprobs: null pointer");
  WT_REQUIRE(top >= 0 && top <= kMaxTop, WT_ERR_ARG, "token_logprobs: top %d (0 to %d)", top, kMaxTop);
  WT_REQUIRE(vocab <= kLpMaxVocab, WT_ERR_UNSUPPORTED, "token_logprobs: vocab %d (at most %d)", vocab, kLpMaxVocab);
  WT_REQUIRE(dtype == WT_F16 || dtype == WT_BF16 || dtype == WT_F32, WT_ERR_DTYPE, "token_logprobs: unknown dtype %d",
             dtype);
  WT_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == WT_F32 ? 4 : 2) == 0, WT_ERR_ALIGN,
             "token_logprobs: logits are not aligned to their type");
  const int sms = device_sm_count();
  if (sms <= 0) return WT_ERR_CUDA;
  const LpArgs a{logits, tokens, suppress, {logprob, entropy, top_logprob, top_token}, row_stride, rows, vocab, top, 1};
  const bool m = suppress != nullptr;
  if (dtype == WT_F32) return m ? launch_logprobs<float, true>(a, sms, stream) : launch_logprobs<float, false>(a, sms, stream);
  if (dtype == WT_BF16)
    return m ? launch_logprobs<__nv_bfloat16, true>(a, sms, stream) : launch_logprobs<__nv_bfloat16, false>(a, sms, stream);
  return m ? launch_logprobs<__half, true>(a, sms, stream) : launch_logprobs<__half, false>(a, sms, stream);
}
