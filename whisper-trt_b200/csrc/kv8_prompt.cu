// Self-attention of S new tokens per row (a prompt) over the row's cached slots of an 8-bit cache (kv8.cuh), read through
// the slot table, and causally over each other.
//
// One CTA of 4 warps per 64 queries of a (row, head): queries are the M of mma.sync.m16n8k16 (16 a warp), keys the N, in
// blocks of 64; the longest CTAs come first. A row's keys are few (a prompt and what stands before it), so a CTA lives
// for a handful of blocks, and its start and the exchange between its warps count for as much as its products: on tcgen05
// (a form of kv8_tile.cu's kernel with a softmax thread a query and the weights through shared memory, M 128, the new tokens
// as further blocks; the present form was not tried) 32 rows x 223 tokens x 20 heads took 79 us, here 58 (memory alone: 9). Bound by latency: 4 CTAs on an SM in 128 registers, a few of them spilled; 3 CTAs in 168
// took 64, 32 keys at a time 63 (4 CTAs) and 73 (5).
// With many queries a key serves the whole CTA, so a block is converted once, on its way into shared memory: the next
// block's e4m3 bytes (and slot-table entries, a block earlier still) are loaded into registers while the current one is
// worked on, then stored as 16-bit, 128-byte-swizzled tiles that ldmatrix reads. The conversions are exact; the scales
// act in fp32: scores times the key's scale and the query's power (query_exp), and the weights times their slots'
// scales, as bf16 hi + lo parts (16 significant bits over fp32's range of exponents) beside the values in bf16. The new
// tokens' keys and values enter at their own 16 bits, copied asynchronously, weights as hi + lo in that type. Weights in
// two parts err by less than 2^-16, so that the output's own rounding is what is left.
#include <type_traits>

#include "cross_math.cuh"
#include "kv8.cuh"
#include "kv8_tile.cuh"

namespace wt {
namespace {

constexpr int kTQ = 64, kTK = 64, kTThreads = 128;
constexpr int kTTile = 64 * 128;  // 64 rows of 128 bytes

__device__ __forceinline__ uint32_t f16x2_to_bf16x2(uint32_t h) {
  const float2 f = Elem<__half>::to_float2(h);
  return Elem<__nv_bfloat16>::from_float2(f.x, f.y);
}
__device__ __forceinline__ uint4 widen_bf16(uint32_t a, uint32_t b) {
  const uint4 u = widen_f16(a, b);
  return make_uint4(f16x2_to_bf16x2(u.x), f16x2_to_bf16x2(u.y), f16x2_to_bf16x2(u.z), f16x2_to_bf16x2(u.w));
}

struct PromptArgs {
  const void *qkv;  // [N, S, 3 H 64]
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  const int64_t *offset;
  const int32_t *src;
  void *y;
  int N, S, H, C;
  float scale;
};

// One block of 64 keys into the running softmax of a warp's 16 queries. TK, TV: the 16-bit types of the K and V tiles (and
// of the weights, which enter as hi + lo). CACHED: per-key factors kscale and vscale in shared memory. Keys from jb; lim0 /
// lim1: the last visible key of query rows g and g + 8; qw0: the warp's first query; nact: 8-key tiles that can hold a visible key; up: the weights (and
// sums) are 2^up times themselves (15 where fp16 weights occur: normal down to 2^-29 of the largest, never off by more
// than 2^-40 of it).
template <typename TK, typename TV, bool CACHED>
__device__ __forceinline__ void prompt_block(float (&o)[8][4], float (&m)[2], float (&l)[2], const unsigned char *qt,
                                             const unsigned char *kt, const unsigned char *vt, const float *kscale,
                                             const float *vscale, float qs0, float qs1, int jb, int lim0, int lim1,
                                             int nact, float up, int qw0, int warp, int lane) {
  const int t = lane & 3;
  uint32_t qa[4][4];
#pragma unroll
  for (int s = 0; s < 4; ++s) ldmatrix_x4(qa[s], qt + swizzle128(warp * 16 + (lane & 15), 2 * s + (lane >> 4)));
  float sc[8][4];
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) {
    sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
    if (CACHED || nt < nact) {
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        uint32_t kf[4];
        ldmatrix_x4(kf, kt + swizzle128(nt * 8 + (lane & 7), 4 * kp + (lane >> 3)));
        Mma<TK>::run(sc[nt], qa[2 * kp][0], qa[2 * kp][1], qa[2 * kp][2], qa[2 * kp][3], kf[0], kf[1]);
        Mma<TK>::run(sc[nt], qa[2 * kp + 1][0], qa[2 * kp + 1][1], qa[2 * kp + 1][2], qa[2 * kp + 1][3], kf[2], kf[3]);
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) {
    Pair f0 = pair_of(qs0, qs0), f1 = pair_of(qs1, qs1);
    if (CACHED) {
      const Pair f = *reinterpret_cast<const Pair *>(kscale + nt * 8 + 2 * t);
      f0 = mul2(f0, f);
      f1 = mul2(f1, f);
    }
    halves(mul2(pair_of(sc[nt][0], sc[nt][1]), f0), sc[nt][0], sc[nt][1]);
    halves(mul2(pair_of(sc[nt][2], sc[nt][3]), f1), sc[nt][2], sc[nt][3]);
  }
  if (__any_sync(0xffffffffu, lim0 - jb < kTK - 1 || lim1 - jb < kTK - 1)) {
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = jb + nt * 8 + 2 * t + e;
        if (j > lim0) sc[nt][e] = kNegInf;
        if (j > lim1) sc[nt][2 + e] = kNegInf;
      }
  }
  float mx0 = kNegInf, mx1 = kNegInf;
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) {
    mx0 = fmaxf(mx0, fmaxf(sc[nt][0], sc[nt][1]));
    mx1 = fmaxf(mx1, fmaxf(sc[nt][2], sc[nt][3]));
  }
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
  }
  if (__any_sync(0xffffffffu, mx0 > m[0] || mx1 > m[1])) {
    const float mn0 = fmaxf(m[0], mx0), mn1 = fmaxf(m[1], mx1);
    const float a0 = ex2f(m[0] - (mn0 == kNegInf ? 0.f : mn0)), a1 = ex2f(m[1] - (mn1 == kNegInf ? 0.f : mn1));
    m[0] = mn0;
    m[1] = mn1;
    l[0] *= a0;
    l[1] *= a1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i][0] *= a0;
      o[i][1] *= a0;
      o[i][2] *= a1;
      o[i][3] *= a1;
    }
  }
  float b0 = m[0] == kNegInf ? 0.f : m[0], b1 = m[1] == kNegInf ? 0.f : m[1];
  if (up != 0.f && __any_sync(0xffffffffu, fmaxf(fabsf(b0), fabsf(b1)) >= kFarMax)) {
    const float f0 = far_part(b0), f1 = far_part(b1);
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      sc[nt][0] -= f0;
      sc[nt][1] -= f0;
      sc[nt][2] -= f1;
      sc[nt][3] -= f1;
    }
    b0 = fabsf(b0) >= kFarMax ? 0.f : b0;
    b1 = fabsf(b1) >= kFarMax ? 0.f : b1;
  }
  const float up0 = up - b0, up1 = up - b1;
  // The keys that stand beside these queries: what a later token's value holds stays away from the earlier queries (a zero
  // weight alone would make NaN of it), so values that are not finite go around the product.
  const int beside = CACHED ? -1 : (qw0 - jb) >> 4;
  bool around = false;
  if (!CACHED && beside < 4) {
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = *reinterpret_cast<const uint4 *>(vt + swizzle128(16 * beside + 4 * i + (lane >> 3), lane & 7));
      odd |= Mag<TV>::not_finite(u.x) | Mag<TV>::not_finite(u.y) | Mag<TV>::not_finite(u.z) | Mag<TV>::not_finite(u.w);
    }
    around = __any_sync(0xffffffffu, odd != 0);
  }
  Pair ps[2] = {0, 0};
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (!CACHED && 2 * kk >= nact) break;
    uint32_t ph[4], pl[4];  // the weights of 16 keys: (row g, g + 8) x (keys 2t, 2t + 1 of each 8-key tile)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int nt = 2 * kk + e;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float up_q = q == 0 ? up0 : up1;
        float p0, p1;
        halves(add2(pair_of(sc[nt][2 * q], sc[nt][2 * q + 1]), pair_of(up_q, up_q)), p0, p1);
        Pair p = pair_of(ex2f(p0), ex2f(p1));
        ps[q] = add2(ps[q], p);
        if (CACHED) p = mul2(p, *reinterpret_cast<const Pair *>(vscale + nt * 8 + 2 * t));
        halves(p, p0, p1);
        const uint32_t hi = Elem<TV>::from_float2(p0, p1);
        const float2 x = Elem<TV>::to_float2(hi);
        halves(add2(p, pair_of(-x.x, -x.y)), p0, p1);
        ph[2 * e + q] = hi;
        pl[2 * e + q] = Elem<TV>::from_float2(p0, p1);
      }
    }
    auto product = [&](auto clean) {
#pragma unroll
      for (int dp = 0; dp < 4; ++dp) {
        uint32_t vf[4];
        ldmatrix_x4_trans(vf, vt + swizzle128(16 * kk + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * dp + (lane >> 4)));
        if constexpr (decltype(clean)::value) {
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[i] &= ~__vcmpeq2(vf[i] & Mag<TV>::kInf2, Mag<TV>::kInf2);
        }
        Mma<TV>::run(o[2 * dp], ph[0], ph[1], ph[2], ph[3], vf[0], vf[1]);
        Mma<TV>::run(o[2 * dp + 1], ph[0], ph[1], ph[2], ph[3], vf[2], vf[3]);
        Mma<TV>::run(o[2 * dp], pl[0], pl[1], pl[2], pl[3], vf[0], vf[1]);
        Mma<TV>::run(o[2 * dp + 1], pl[0], pl[1], pl[2], pl[3], vf[2], vf[3]);
      }
    };
    if (around && kk == beside)
      product(std::true_type());
    else
      product(std::false_type());
  }
  if (around) {  // (whatever its weight, such a value decides the sum)
    for (int j = 0; j < 16; ++j) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const uint32_t u = *reinterpret_cast<const uint32_t *>(vt + swizzle128(16 * beside + j, dt) + 4 * t);
        const float2 f = Elem<TV>::to_float2(u & __vcmpeq2(u & Mag<TV>::kInf2, Mag<TV>::kInf2));
        if (qw0 + j <= lim0) o[dt][0] += f.x, o[dt][1] += f.y;
        if (qw0 + j <= lim1) o[dt][2] += f.x, o[dt][3] += f.y;
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float s0, s1;
    halves(ps[q], s0, s1);
    l[q] += s0 + s1;
  }
}

template <typename T>
__global__ void __launch_bounds__(kTThreads, 4) prompt8_kernel(const PromptArgs p) {
  constexpr bool kBf = Elem<T>::code == WT_BF16;
  constexpr float kShift = kBf ? 0.f : 15.f;
  extern __shared__ unsigned char smem_raw[];  // Q (bf16: as it is, and as fp16), two buffers of K, V and their scales
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *q_raw = smem, *q_f16 = smem + kTTile, *kv = smem + (kBf ? 2 : 1) * kTTile;
  float *facs = reinterpret_cast<float *>(kv + 4 * kTTile);  // [buffer][K, V][key]
  __shared__ float q_fac[kTQ];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.H, h = blockIdx.x - b * p.H;
  const int q0 = static_cast<int>(gridDim.y - 1 - blockIdx.y) * kTQ;  // (the longest first)
  const size_t HD = static_cast<size_t>(p.H) * 64;
  const size_t qstride = 3 * HD;
  const T *qb = static_cast<const T *>(p.qkv) + static_cast<size_t>(b) * p.S * qstride + static_cast<size_t>(h) * 64;

  pdl_wait();
  pdl_launch_dependents();

  const int64_t o64 = p.offset[b];
  const int off = static_cast<int>(o64 < 0 ? 0 : (o64 > p.C ? p.C : o64));
  // the query tile (rows past S are zeros); 2 threads a row find its power and, for bf16, write the fp16 form
  {
    const int r = tid >> 1, s = q0 + r, half = (tid & 1) * 4;
    uint4 u[4];
    uint32_t mag = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = s < p.S ? ldg16(qb + static_cast<size_t>(s) * qstride + (half + i) * 8) : make_uint4(0, 0, 0, 0);
      mag = Mag<T>::max8(u[i], mag);
      *reinterpret_cast<uint4 *>(q_raw + swizzle128(r, half + i)) = u[i];
    }
    mag = max(mag & 0xffffu, mag >> 16);
    mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
    const int e = query_exp<T>(mag);
    if (kBf) {
      const float inv = exp2_int(-e);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4 *>(q_f16 + swizzle128(r, half + i)) =
            make_uint4(query_f16<T>(u[i].x, inv), query_f16<T>(u[i].y, inv), query_f16<T>(u[i].z, inv),
                       query_f16<T>(u[i].w, inv));
    }
    if ((tid & 1) == 0) q_fac[r] = exp2_int(e) * p.scale;
  }
  const int nbc = (off + kTK - 1) / kTK;                                      // blocks of cached places
  const int nbn = (min(p.S, q0 + kTQ) + kTK - 1) / kTK;                       // blocks of new tokens, up to these queries
  const int nb = nbc + nbn;

  // loads of block kb: cached, thread (row tid / 4 and + 32, piece tid % 4); new, (row tid / 8 and + 16 .., piece tid % 8)
  const size_t head = static_cast<size_t>(h) * p.C;
  uint4 pre[4];
  float fac = 0.f;
  int idx[3] = {0, 0, 0};  // slot-table entries of the next cached block: of this thread's two rows, and of key tid % 64
  auto load_idx = [&](int kb) {
    if (kb >= nbc) return;
    const int32_t *srow = p.src + static_cast<size_t>(b) * p.C;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int j = kb * kTK + (i < 2 ? (tid >> 2) + 32 * i : (tid & 63));
      const int v = j < off ? srow[j] : 0;
      idx[i] = v < 0 ? 0 : (v > p.N - 1 ? p.N - 1 : v);
    }
  };
  auto load = [&](int kb) {
    if (kb < nbc) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = kb * kTK + (tid >> 2) + 32 * i;
        const bool in = j < off;
        const size_t place = static_cast<size_t>(idx[i]) * p.H * p.C + head + j;
        pre[i] = in ? ldg16(p.k8 + place * 64 + (tid & 3) * 16) : make_uint4(0, 0, 0, 0);
        pre[2 + i] = in ? ldg16(p.v8 + place * 64 + (tid & 3) * 16) : make_uint4(0, 0, 0, 0);
      }
      const int j = kb * kTK + (tid & 63);
      const size_t place = static_cast<size_t>(idx[2]) * p.H * p.C + head + j;
      fac = j < off ? (tid < 64 ? p.ks : p.vs)[place] : 0.f;
      load_idx(kb + 1);
    } else {  // (the buffer's last block, kb - 2, is done with: every warp has met the others since)
      unsigned char *kt = kv + (kb & 1) * 2 * kTTile, *vt = kt + kTTile;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (tid >> 3) + 16 * i, j = (kb - nbc) * kTK + r;
        const T *kp = qb + static_cast<size_t>(j < p.S ? j : 0) * qstride + HD + (tid & 7) * 8;
        cp16(kt + swizzle128(r, tid & 7), kp, j < p.S);
        cp16(vt + swizzle128(r, tid & 7), kp + HD, j < p.S);
      }
      cp_commit_group();
    }
  };
  auto store = [&](int kb) {
    unsigned char *kt = kv + (kb & 1) * 2 * kTTile, *vt = kt + kTTile;
    if (kb < nbc) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (tid >> 2) + 32 * i, c = 2 * (tid & 3);
        *reinterpret_cast<uint4 *>(kt + swizzle128(r, c)) = widen_f16(pre[i].x, pre[i].y);
        *reinterpret_cast<uint4 *>(kt + swizzle128(r, c + 1)) = widen_f16(pre[i].z, pre[i].w);
        const uint4 v = pre[2 + i];
        *reinterpret_cast<uint4 *>(vt + swizzle128(r, c)) = widen_bf16(v.x, v.y);
        *reinterpret_cast<uint4 *>(vt + swizzle128(r, c + 1)) = widen_bf16(v.z, v.w);
      }
      facs[(kb & 1) * 2 * kTK + tid] = fac;
    } else {
      cp_wait_group<0>();
    }
  };
  load_idx(0);
  if (nb > 0) load(0);

  const int g = lane >> 2, t = lane & 3;
  const int qw0 = q0 + warp * 16, sq0 = qw0 + g, sq1 = sq0 + 8;
  const bool active = qw0 < p.S;
  float o[8][4], m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  for (int kb = 0; kb < nb; ++kb) {
    store(kb);  // (every warp is past block kb - 2 here: it has met the others since)
    __syncthreads();
    if (kb + 1 < nb) load(kb + 1);
    if (!active) continue;
    const unsigned char *kt = kv + (kb & 1) * 2 * kTTile, *vt = kt + kTTile;
    const float *ks = facs + (kb & 1) * 2 * kTK, *vs = ks + kTK;
    if (kb < nbc) {
      prompt_block<__half, __nv_bfloat16, true>(o, m, l, kBf ? q_f16 : q_raw, kt, vt, ks, vs, q_fac[warp * 16 + g],
                                                q_fac[warp * 16 + g + 8], kb * kTK, off - 1, off - 1, 8, kShift, qw0, warp, lane);
    } else {
      const int jb = (kb - nbc) * kTK;
      if (qw0 + 15 >= jb)
        prompt_block<T, T, false>(o, m, l, q_raw, kt, vt, nullptr, nullptr, p.scale, p.scale, jb, min(sq0, p.S - 1),
                                  min(sq1, p.S - 1), min(8, (qw0 + 15 - jb) / 8 + 1), kShift, qw0, warp,
                                  lane);
    }
  }
  __syncthreads();  // (the query tile is read no more)
  if (!active) return;
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    l[0] += __shfl_xor_sync(0xffffffffu, l[0], x);
    l[1] += __shfl_xor_sync(0xffffffffu, l[1], x);
  }
  const float r0 = 1.f / l[0], r1 = 1.f / l[1];  // (a query sees itself at least; nothing but scores of -inf: NaN)
  unsigned char *os = q_raw + warp * 16 * 128;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) {
    *reinterpret_cast<uint32_t *>(os + swizzle128(g, dt) + 4 * t) = Elem<T>::from_float2(o[dt][0] * r0, o[dt][1] * r0);
    *reinterpret_cast<uint32_t *>(os + swizzle128(g + 8, dt) + 4 * t) =
        Elem<T>::from_float2(o[dt][2] * r1, o[dt][3] * r1);
  }
  __syncwarp();
  T *yb = static_cast<T *>(p.y) + static_cast<size_t>(b) * p.S * HD + static_cast<size_t>(h) * 64;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = i * 32 + lane, r = x >> 3, c = x & 7, s = qw0 + r;
    if (s < p.S)
      *reinterpret_cast<uint4 *>(yb + static_cast<size_t>(s) * HD + c * 8) =
          *reinterpret_cast<const uint4 *>(os + swizzle128(r, c));
  }
}

template <typename T>
int launch_prompt(const PromptArgs &a, void *stream) {
  constexpr int smem = (Elem<T>::code == WT_BF16 ? 6 : 5) * kTTile + 4 * kTK * 4 + 1024;
  const int st = opt_in_smem<prompt8_kernel<T>>(smem, "kv8_self_attn");
  if (st != WT_OK) return st;
  const dim3 grid(static_cast<unsigned>(a.N) * a.H, (a.S + kTQ - 1) / kTQ), block(kTThreads);
  return launch("kv8_self_attn", prompt8_kernel<T>, grid, block, smem, stream, a);
}

}  // namespace

int kv8_self_prompt(int dtype, const void *qkv, const void *k8, const void *v8, const float *ks, const float *vs,
                    const int64_t *offset, const int32_t *src, void *y, int rows, int new_tokens, int heads,
                    int capacity, void *stream) {
  const PromptArgs a{qkv, static_cast<const uint8_t *>(k8), static_cast<const uint8_t *>(v8), ks, vs, offset, src, y, rows,
                     new_tokens, heads, capacity, static_cast<float>(0.125 * 1.4426950408889634)};
  if (dtype == WT_BF16) return launch_prompt<__nv_bfloat16>(a, stream);
  return launch_prompt<__half>(a, stream);
}

}  // namespace wt
