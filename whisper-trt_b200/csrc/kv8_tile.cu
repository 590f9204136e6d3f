// Cross-attention of many queries per window over an 8-bit cache (kv8.cuh): more than a decode step has, a transcript
// forced through the decoder.
//
// With many queries a key serves many of them, and the work is products: these run on the 5th-generation tensor cores. A
// CTA takes 128 queries of a (window, head) over blocks of 64 frames, S = Q K^T (M 128, N 64, K 64) and O += P V (the same
// shape), both accumulators in tensor memory:
//   * warps 0-7 are the softmax, 16 queries each, 4 lanes a query, in the layout of an MMA's accumulator: maxima and sums
//     cross lanes in two shuffles, and the weights go, as 16-bit pairs, over the scores they come from, from where the
//     second product takes them (no trip through shared memory: with it and a thread a query the 16 windows below took 51
//     us instead of 43, weights then in one part). They are relative to a maximum that lags: only when a score exceeds it
//     by 2^kLag does the warp take the output out of tensor memory and rescale it, which is rare after the first block.
//   * warps 8-11 bring a block in: e4m3 bytes by asynchronous copies three ahead, converted once for all queries -- exactly,
//     to fp16 -- and stored as they lie, 64 rows of 128 swizzled bytes: K's is the product's K-major operand, V's its
//     MN-major one (transposing V on the way took 47 us instead of 43, likewise).
//   * warp 12 issues the MMAs: the next two blocks' S before it waits for a block's weights.
// Windows of different lengths go longest first, so that no long one is left to the end on its own: every CTA reads the
// lengths and counts its window's place (57 -> 51 us). Where there are too few tiles of queries for the SMs, a cluster of 2 or
// 4 CTAs shares a tile's frames; their sums meet through distributed shared memory.
// 16 windows x 223 queries x 16 heads, lengths 375 to 1500, bf16: 51 us, of which the weights' second part takes 7; memory
// alone 8, exponentials (16 a cycle) 14.
// Bound by hand-offs: a block's way from MMA to softmax to MMA takes some 1000 cycles with nothing to compute, 1300 with it;
// two CTAs on an SM and three S in flight hide part of it. Fewer copies, one exponential for all, a stage more: 2 to 5%.
//
// Scales: a score is multiplied by the block's key scale and the query's power (query_exp), a weight by the block's
// value scale over the row's reference, which follows, like its maximum and as lazily, the largest product of a weight and a
// value scale so far: a block of large values that no weight falls on costs the others no bits. Weights enter as fp16, 2^kUp
// times themselves (at most 2^15), normal down to 2^-(14 + kUp) of the reference and never off by more than 2^-(25 + kUp) of
// it, in two parts, hi + lo, so that their rounding does not add to the output's. Waits are bounded as in the other tcgen05
// kernels: a wait that runs out sets the error word and a stop flag.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "kv8_tile.cuh"
#include "tc05.cuh"
#include "tma.cuh"

namespace wt {
namespace {

constexpr int kTQ = kTileQueries, kTK = 64;
constexpr int kTSoftmax = 8, kTLoaders = 4, kTThreads = (kTSoftmax + kTLoaders + 1) * 32;  // warps; threads
constexpr int kTQTile = kTQ * 128, kTKTile = kTK * 128;  // bytes: 128 or 64 rows of 64 16-bit values
constexpr float kLag = 8.f, kUp = 7.f;                   // (kLag + kUp = 15: fp16's largest power of two)
constexpr float kLow = -3e38f, kNoRef = -150.f;          // a row's maximum and value reference before any score: below all
constexpr int kTErrTimeout = 1;
constexpr int kTCluster = 4;
constexpr int kTRec = 68;                                // floats of a row of a CTA's share (64, apart in the banks)
constexpr uint32_t kTTmem = 256;                         // S, then P, kTScores of them; O

struct TileArgs {
  const void *q;  // [W, S, H 64]
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  const int64_t *lengths;  // [W] or null
  void *y;
  int W, S, H, T, tiles, cl;  // tiles: of 128 queries; cl: CTAs that share a tile's frames
  float scale;
  int *err;
  uint32_t polls;
  int withhold;
};

constexpr int kTSlots = 3;   // loads in flight: 64 bytes of a loading thread each
constexpr int kTSlotBytes = 128 * 64;
constexpr int kTStages = 4;  // K and V tiles
constexpr int kTScores = 3;  // S, then P, in tensor memory
constexpr int kTKv = kTQTile, kTSlotsAt = kTKv + kTStages * 2 * kTKTile, kTBars = kTSlotsAt + kTSlots * kTSlotBytes,
              kTBytes = kTBars + (2 * kTStages + 3 * kTScores + 2) * 8 + 16 + 1024;
static_assert(kTQ * kTRec * 4 <= kTStages * 2 * kTKTile, "a CTA's share lies over the tiles");
static_assert(2 * (kTBytes + 5 * 1024) <= 228 * 1024, "two CTAs on an SM (static arrays and the reserved 1 KB with them)");

// Tensor memory of 16 rows by 64 or 16 columns, as an MMA's accumulator lies in registers: of each 8 columns a lane holds
// columns 2 (lane % 4) and + 1 of rows lane / 4 (r[4 i], r[4 i + 1]) and + 8 (r[4 i + 2], r[4 i + 3]).
__device__ __forceinline__ void tmem_ld_rows64(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_rows16(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_rows16(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 rows by 32 columns of two 16-bit values each: of each 4 columns a lane holds column lane % 4 of rows lane / 4 and + 8.
__device__ __forceinline__ void tmem_st_pairs(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D[tmem] (+)= A[tmem, two fp16 a column] . B[smem desc]^T
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// SHARED: a cluster's CTAs share a tile's frames.
template <typename T, bool SHARED>
__global__ void __launch_bounds__(kTThreads, 2) tile8_kernel(const TileArgs a) {
  namespace cg = cooperative_groups;
  const int cl = SHARED ? a.cl : 1;
  constexpr int kStages = kTStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *qt = smem, *kv = smem + kTKv;
  uint64_t *kv_full = reinterpret_cast<uint64_t *>(smem + kTBars), *kv_empty = kv_full + kStages;
  uint64_t *s_full = kv_empty + kStages, *p_full = s_full + kTScores, *pv_done = p_full + kTScores;
  uint64_t *drained = pv_done + kTScores, *q_full = drained + 1;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(q_full + 1);
  volatile int *stop = reinterpret_cast<volatile int *>(tmem_holder + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int lens[kTThreads], chosen;
  __shared__ float q_fac[kTQ];
  __shared__ float state[3][SHARED ? kTQ : 1];  // this CTA's rows' maxima, sums, value references

  if (warp == 0) {
    tmem_alloc(tmem_holder, kTTmem);
    tmem_relinquish();
  }
  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&kv_full[s], kTLoaders);
      mbar_init(&kv_empty[s], 1);  // a commit
    }
    for (int s = 0; s < kTScores; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], kTSoftmax);
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(drained, 1);
    mbar_init(q_full, kTSoftmax);
    *stop = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder, tmem_o = tmem + kTScores * kTK;
  pdl_wait();
  pdl_launch_dependents();

  const int unit = blockIdx.x / cl, rank = blockIdx.x - unit * cl;
  int b = unit / (a.H * a.tiles);  // window
  const int rest = unit - b * a.H * a.tiles, h = rest / a.tiles, q0 = (rest - h * a.tiles) * kTQ;
  int len = a.T;
  if (a.lengths != nullptr) {
    auto length = [&](int w) {
      const int64_t l = a.lengths[w];
      return static_cast<int>(l < 0 ? 0 : (l > a.T ? a.T : l));
    };
    if (a.W <= kTThreads) {  // the b-th longest window (more windows are many rounds of CTAs, in any order)
      if (tid < a.W) lens[tid] = length(tid);
      __syncthreads();
      if (tid < a.W) {
        const int mine = lens[tid];
        int before = 0;
        for (int w = 0; w < a.W; ++w) before += lens[w] > mine || (lens[w] == mine && w < tid);
        if (before == b) chosen = tid;
      }
      __syncthreads();
      b = chosen;
      len = lens[b];
    } else {
      len = length(b);
    }
  }
  const size_t wh = static_cast<size_t>(b) * a.H + h, HD = static_cast<size_t>(a.H) * 64;
  const T *qb = static_cast<const T *>(a.q) + static_cast<size_t>(b) * a.S * HD + static_cast<size_t>(h) * 64;
  // this CTA's share of the blocks; everything below sees a window of its frames alone
  const int all = (len + kTK - 1) / kTK, first = all * rank / cl, nb = all * (rank + 1) / cl - first;
  len = min(len - first * kTK, nb * kTK);

  // a warp's wait, decided together (its tensor-memory loads are warp-wide): one look first, since most are over already
  auto wait = [&](uint64_t *bar, uint32_t phase) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, phase)) ||
           __all_sync(0xffffffffu, mbar_wait_role(bar, phase, a.err, kTErrTimeout, a.polls, stop));
  };
  if (warp < kTSoftmax) {
    // ---- the softmax: 16 queries a warp, 4 lanes a query -------------------------------------------------------
    {  // the query tile (rows past S are zeros), 2 threads a row
      const int row = tid >> 1, s = q0 + row, half = (tid & 1) * 4;
      uint4 u[4];
      uint32_t mag = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = s < a.S ? ldg16(qb + static_cast<size_t>(s) * HD + (half + i) * 8) : make_uint4(0, 0, 0, 0);
        mag = Mag<T>::max8(u[i], mag);
      }
      mag = max(mag & 0xffffu, mag >> 16);
      mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
      const int e = query_exp<T>(mag);
      const float inv = exp2_int(-e);
      if ((tid & 1) == 0) q_fac[row] = exp2_int(e) * a.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4 *>(qt + swz128(row, half + i)) =
            make_uint4(query_f16<T>(u[i].x, inv), query_f16<T>(u[i].y, inv), query_f16<T>(u[i].z, inv),
                       query_f16<T>(u[i].w, inv));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const int row0 = (warp & 3) * 32 + (warp >> 2) * 16;  // a warp reaches the 32 rows of its quarter: 16 of them its own
    const uint32_t rows = static_cast<uint32_t>(row0) << 16;
    const size_t sbase = wh * ((a.T + kFrameBlock - 1) / kFrameBlock) + first;
    // a row's maximum, sum and value reference (whole numbers in log2 units: moving them is exact)
    float m[2] = {kLow, kLow}, l[2] = {0.f, 0.f}, ref[2] = {kNoRef, kNoRef};
    float next_k = nb > 0 ? a.ks[sbase] : 0.f, next_v = nb > 0 ? a.vs[sbase] : 0.f;  // the next block's scales
    bool ok = wait(q_full, 0), far = false;  // far: one of the warp's maxima is
    const float factor[2] = {ok ? q_fac[row0 + (lane >> 2)] : 0.f, ok ? q_fac[row0 + (lane >> 2) + 8] : 0.f};
    for (int i = 0; i < nb && ok; ++i) {
      const uint32_t at = tmem + rows + static_cast<uint32_t>(i % kTScores * kTK);
      // (held above 0, where zero or tiny queries meet zero or tiny keys: frames that are not there are -inf before it)
      constexpr float kLeast = 1.17549435e-38f;
      float f[2] = {fmaxf(next_k * factor[0], kLeast), fmaxf(next_k * factor[1], kLeast)};
      const float ve = static_cast<float>(static_cast<int>(__float_as_uint(next_v) >> 23) - 127);
      if (i + 1 < nb) {
        next_k = a.ks[sbase + i + 1];
        next_v = a.vs[sbase + i + 1];
      }
      ok = wait(&s_full[i % kTScores], (i / kTScores) & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t raw[32];
      tmem_ld_rows64(at, raw);
      tmem_wait_ld();
      float x[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(raw[j]);
      const int lim = len - 1 - i * kTK - 2 * (lane & 3);  // of this lane's columns, the last frame that is there
      if (len - i * kTK < kTK) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (8 * (j >> 2) + (j & 1) > lim) x[j] = kNegInf;
      }
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m2[2] = {x[2 * e], x[2 * e + 1]};
#pragma unroll
        for (int j = 1; j < 8; ++j) {
          m2[0] = fmaxf(m2[0], x[4 * j + 2 * e]);
          m2[1] = fmaxf(m2[1], x[4 * j + 2 * e + 1]);
        }
        mx[e] = fmaxf(m2[0], m2[1]);
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2)) * f[e];  // (f > 0)
      }
      const bool late = mx[0] > m[0] + kLag || mx[1] > m[1] + kLag || mx[0] - m[0] + ve > ref[0] + kLag ||
                        mx[1] - m[1] + ve > ref[1] + kLag;
      if (__any_sync(0xffffffffu, late)) {
        float by[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float up = ceilf(mx[e]), mn = fmaxf(m[e], up), go = m[e] - mn, rn = fmaxf(ref[e] + go, up - mn + ve);
          l[e] *= ex2f(go);
          by[e] = ex2f(ref[e] + go - rn);
          m[e] = mn;
          ref[e] = rn;
        }
        far = __any_sync(0xffffffffu, fmaxf(fabsf(m[0]), fabsf(m[1])) >= kFarMax);
        if (i > 0) {  // the output so far, once block i - 1 is in it
          ok = wait(&pv_done[(i - 1) % kTScores], ((i - 1) / kTScores) & 1);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[8];
            tmem_ld_rows16(tmem_o + rows + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by[(j >> 1) & 1]);
            tmem_st_rows16(tmem_o + rows + 16 * c, o);
          }
        }
      }
      // Weights, over the scores that they come from. (The value scale over the row's reference, a power of two, goes into
      // the exponent, and out of the sum again. Below 2^-90 the weights themselves would leave fp32; what such values give
      // is below 2^-81 of the largest.)
      const float shift[2] = {fmaxf(ve - ref[0], -90.f), fmaxf(ve - ref[1], -90.f)};
      float up[2] = {kUp - m[0] + shift[0], kUp - m[1] + shift[1]};
      if (far) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (fabsf(m[e]) >= kFarMax) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (((j >> 1) & 1) == e) x[j] = __fsub_rn(__fmul_rn(x[j], f[e]), m[e]);  // (rounded like the maxima)
            f[e] = 1.f;
            up[e] = kUp + shift[e];
          }
      }
      const Pair f2[2] = {pair_of(f[0], f[0]), pair_of(f[1], f[1])}, up2[2] = {pair_of(up[0], up[0]), pair_of(up[1], up[1])};
      uint32_t hi[16], lo[16];
      Pair sum[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int e = j & 1;
        float p0, p1;
        halves(fma2(pair_of(x[2 * j], x[2 * j + 1]), f2[e], up2[e]), p0, p1);
        p0 = ex2f(p0);
        p1 = ex2f(p1);
        const Pair p = pair_of(p0, p1);
        sum[e] = add2(sum[e], p);
        hi[j] = Elem<__half>::from_float2(p0, p1);
        const float2 r = Elem<__half>::to_float2(hi[j]);
        halves(add2(p, pair_of(-r.x, -r.y)), p0, p1);
        lo[j] = Elem<__half>::from_float2(p0, p1);
      }
      tmem_st_pairs(at, hi);
      tmem_st_pairs(at + 32, lo);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float s0, s1;
        halves(sum[e], s0, s1);
        l[e] = fmaf(s0 + s1, ex2f(-shift[e]), l[e]);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i % kTScores]);
    }
    if (ok && nb > 0) ok = wait(&pv_done[(nb - 1) % kTScores], ((nb - 1) / kTScores) & 1);
    if (ok) {
      tc_fence_after();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      }
      uint32_t o[32];
      if (nb > 0) {
        tmem_ld_rows64(tmem_o + rows, o);
        tmem_wait_ld();
      } else {  // (no frame: zeros)
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = 0;
      }
      if constexpr (SHARED) {  // this CTA's share of the sums, over the tiles of keys that every MMA is done with
        float *to = reinterpret_cast<float *>(kv) + (row0 + (lane >> 2)) * kTRec + 2 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          *reinterpret_cast<float2 *>(to + (j & 1) * 8 * kTRec + (j >> 1) * 8) =
              make_float2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
        if ((lane & 3) == 0) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            state[0][row0 + (lane >> 2) + 8 * e] = m[e];
            state[1][row0 + (lane >> 2) + 8 * e] = l[e];
            state[2][row0 + (lane >> 2) + 8 * e] = ref[e];
          }
        }
      } else {  // by way of the query tile, which every MMA is done with, as whole pieces of rows
        unsigned char *to = qt + row0 * 128;
        // (no frame: zeros; nothing but scores of -inf: NaN)
        const float f[2] = {nb > 0 ? 1.f / l[0] : 0.f, nb > 0 ? 1.f / l[1] : 0.f}, r[2] = {ex2f(ref[0]), ex2f(ref[1])};
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int e = j & 1;
          *reinterpret_cast<uint32_t *>(to + swz128((lane >> 2) + 8 * e, j >> 1) + 4 * (lane & 3)) =
              Elem<T>::from_float2(__uint_as_float(o[2 * j]) * f[e] * r[e], __uint_as_float(o[2 * j + 1]) * f[e] * r[e]);
        }
        __syncwarp();
        T *yr = static_cast<T *>(a.y) + (static_cast<size_t>(b) * a.S + q0 + row0) * HD + static_cast<size_t>(h) * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = i * 4 + (lane >> 3), c = lane & 7;
          if (q0 + row0 + row < a.S)
            *reinterpret_cast<uint4 *>(yr + static_cast<size_t>(row) * HD + c * 8) =
                *reinterpret_cast<const uint4 *>(to + swz128(row, c));
        }
      }
    }
  } else if (warp < kTSoftmax + kTLoaders) {
    // ---- the loaders ---------------------------------------------------------------------------------------------
    const int t = tid - kTSoftmax * 32;
    const size_t base = wh * a.T + static_cast<size_t>(first) * kTK;
    // A load is 64 bytes a thread, into its own places of a slot, which it reads back itself: rows t / 4 and + 32, piece
    // t % 4.
    unsigned char *slots = smem + kTSlotsAt;
    auto issue = [&](int n) {
      if (n < nb) {
        unsigned char *slot = slots + n % kTSlots * kTSlotBytes, *mine = slot + t * 16;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = n * kTK + (t >> 2) + 32 * e;
          const size_t from = j < len ? (base + j) * 64 + (t & 3) * 16 : 0;
          cp16(mine + e * 2048, a.k8 + from, j < len);
          cp16(mine + (2 + e) * 2048, a.v8 + from, j < len);
        }
      }
      cp_commit_group();
    };
#pragma unroll
    for (int n = 0; n < kTSlots; ++n) issue(n);
    for (int i = 0; i < nb; ++i) {
      const int st = i % kStages, use = i / kStages;
      if (use >= 1 && !wait(&kv_empty[st], (use - 1) & 1)) break;
      cp_wait_group<kTSlots - 1>();
      const unsigned char *slot = slots + i % kTSlots * kTSlotBytes;
      uint4 u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = *reinterpret_cast<const uint4 *>(slot + e * 2048 + t * 16);
      unsigned char *tile = kv + st * 2 * kTKTile;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // K's two rows, V's two
        unsigned char *to = tile + (e >> 1) * kTKTile;
        const int r = (t >> 2) + 32 * (e & 1), c = 2 * (t & 3);
        *reinterpret_cast<uint4 *>(to + swz128(r, c)) = widen_f16(u[e].x, u[e].y);
        *reinterpret_cast<uint4 *>(to + swz128(r, c + 1)) = widen_f16(u[e].z, u[e].w);
      }
      issue(i + kTSlots);
      fence_proxy_async_smem();
      __syncwarp();
      // (test hook: the first CTA's first block is never said to be there)
      if (lane == 0 && !(a.withhold && i == 0 && blockIdx.x == 0)) mbar_arrive(&kv_full[st]);
    }
    cp_wait_group<0>();
  } else if (lane == 0) {
    // ---- the MMAs ------------------------------------------------------------------------------------------------------
    constexpr uint32_t idesc = idesc_f16(kTQ, kTK, false), idesc_v = idesc | 1u << 16;  // (V: rows along K)
    const uint64_t qd = sw128_desc(smem_addr(qt)), kvd = sw128_desc(smem_addr(kv));
    auto wait1 = [&](uint64_t *bar, uint32_t phase) {
      return mbar_try_wait(bar, phase) || mbar_wait_role(bar, phase, a.err, kTErrTimeout, a.polls, stop);
    };
    auto pv = [&](int i) {  // O (+)= P V of block i
      if (!wait1(&p_full[i % kTScores], (i / kTScores) & 1)) return false;
      tc_fence_after();
      const uint64_t vd = kvd + ((i % kStages) * 2 + 1) * (kTKTile >> 4);
      const uint32_t pa = tmem + static_cast<uint32_t>(i % kTScores * kTK);
#pragma unroll
      for (int s = 0; s < 8; ++s)  // (the second parts stand behind the first)
        umma_f16_ta(tmem_o, pa + 8 * s, vd + (2048 >> 4) * (s & 3), idesc_v, i > 0 || s > 0);
      umma_commit(&kv_empty[i % kStages]);
      umma_commit(&pv_done[i % kTScores]);
      return true;
    };
    // S of the next blocks first, kTScores - 1 of them; a block's S goes over the weights of kTScores blocks before it,
    // which the MMAs issued before it read
    bool ok = nb > 0 && wait1(q_full, 0);
    for (int i = 0; i < nb + kTScores - 1 && ok; ++i) {
      if (i < nb) {
        ok = wait1(&kv_full[i % kStages], (i / kStages) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t kd = kvd + (i % kStages) * 2 * (kTKTile >> 4);
#pragma unroll
        for (int s = 0; s < 4; ++s)
          umma_f16(tmem + static_cast<uint32_t>(i % kTScores * kTK), qd + 2 * s, kd + 2 * s, idesc, s > 0);
        umma_commit(&s_full[i % kTScores]);
      }
      if (i >= kTScores - 1) ok = pv(i - kTScores + 1);
    }
    umma_commit(drained);  // every MMA issued has completed before the tensor memory is freed (bounded)
    mbar_wait_bounded(drained, 0, nullptr, 0, a.polls);
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (SHARED) {
    // the shares of the cluster's CTAs -> the output: 8 threads a query, 8 head dims each
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int t = rank * kTThreads + tid; t < kTQ * 8; t += cl * kTThreads) {
      const int row = t >> 3, d8 = (t & 7) * 8;
      if (q0 + row >= a.S) continue;
      float4 o[kTCluster][2];
      float m[kTCluster], l[kTCluster], r[kTCluster], top = kLow, v = kNoRef, den = 0.f;
#pragma unroll
      for (int c = 0; c < kTCluster; ++c) {  // (all loads together)
        const int from = c < cl ? c : rank;
        const float *st = cluster.map_shared_rank(&state[0][row], from);
        const float4 *at = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(
                                                                cluster.map_shared_rank(kv, from)) + row * kTRec + d8);
        m[c] = st[0];
        l[c] = c < cl ? st[kTQ] : 0.f;
        r[c] = st[2 * kTQ];
        o[c][0] = at[0];
        o[c][1] = at[1];
      }
      float num[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kTCluster; ++c)
        if (l[c] != 0.f) top = fmaxf(top, m[c]);  // (it has seen a frame)
#pragma unroll
      for (int c = 0; c < kTCluster; ++c)
        if (l[c] != 0.f) v = fmaxf(v, m[c] - top + r[c]);
#pragma unroll
      for (int c = 0; c < kTCluster; ++c)
        if (l[c] != 0.f) {
          const float w = ex2f(m[c] - top), wv = ex2f(m[c] - top + r[c] - v);
          den = fmaf(w, l[c], den);
          num[0] = fmaf(wv, o[c][0].x, num[0]);
          num[1] = fmaf(wv, o[c][0].y, num[1]);
          num[2] = fmaf(wv, o[c][0].z, num[2]);
          num[3] = fmaf(wv, o[c][0].w, num[3]);
          num[4] = fmaf(wv, o[c][1].x, num[4]);
          num[5] = fmaf(wv, o[c][1].y, num[5]);
          num[6] = fmaf(wv, o[c][1].z, num[6]);
          num[7] = fmaf(wv, o[c][1].w, num[7]);
        }
      const float f = all == 0 ? 0.f : 1.f / den, by = ex2f(v);  // (no frame: zeros; none but of score -inf: NaN)
#pragma unroll
      for (int i = 0; i < 8; ++i) num[i] = num[i] * f * by;
      *reinterpret_cast<uint4 *>(static_cast<T *>(a.y) + (static_cast<size_t>(b) * a.S + q0 + row) * HD +
                                 static_cast<size_t>(h) * 64 + d8) = pack8<T>(num);
    }
    cluster.sync();  // (no CTA leaves while another reads its share)
  } else {
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc(tmem, kTTmem);
}

template <typename T>
int launch_tile(TileArgs a, int sms, void *stream) {
  a.tiles = static_cast<int>(kv8_cross_tiles(a.S));
  const long long units = static_cast<long long>(a.W) * a.H * a.tiles;  // (fewer than 2^30)
  // CTAs per tile of queries, a cluster that shares its frames: as many as two on each SM hold, of 3 blocks at least. Measured
  // (us, 20 heads x 1500 frames, fp16, with / without): 1 window x 33 queries 12.2 / 25.0, x 128 14.0 / 25.5, x 223 19.3 / 25.7;
  // 2 windows x 128 19.3 / 25.6; 4 windows x 64, which take every second place of the SMs' already, 24.6 / 25.9.
  a.cl = 1;
  while (a.cl < kTCluster && units * a.cl * 2 <= 2LL * sms && a.T > a.cl * 2 * 3 * kTK) a.cl *= 2;
  constexpr int smem = kTBytes;
  const dim3 grid(static_cast<unsigned>(units * a.cl)), block(kTThreads);
  if (a.cl > 1) {
    const int st = opt_in_smem<tile8_kernel<T, true>>(smem, "kv8_cross_attn");
    if (st != WT_OK) return st;
    return launch_clustered("kv8_cross_attn", tile8_kernel<T, true>, grid, block, smem, stream, a.cl, a);
  }
  const int st = opt_in_smem<tile8_kernel<T, false>>(smem, "kv8_cross_attn");
  if (st != WT_OK) return st;
  return launch("kv8_cross_attn", tile8_kernel<T, false>, grid, block, smem, stream, a);
}

}  // namespace

int kv8_cross_tile(int dtype, const void *q, const void *k8, const void *v8, const float *ks, const float *vs,
                   const int64_t *lengths, void *y, int windows, int queries, int heads, int frames, int sms,
                   int *err, void *stream) {
  const TileArgs a{q, static_cast<const uint8_t *>(k8), static_cast<const uint8_t *>(v8), ks, vs, lengths, y, windows,
                   queries, heads, frames, 0, 1, static_cast<float>(0.125 * 1.4426950408889634), err, wait_limit(),
                   test_withhold_stage()};
  if (dtype == WT_BF16) return launch_tile<__nv_bfloat16>(a, sms, stream);
  return launch_tile<__half>(a, sms, stream);
}

}  // namespace wt
