// Cross-attention of few queries per window over an 8-bit cache (kv8.cuh), a decode step's: softmax(q k^T / 8) v per window and head
// over the window's first lengths[w] frames, k = k8 * k_scale and v = v8 * v_scale with a scale for each 64 frames.
//
// The decode step's queries (a window's beams) share one stream of 2 bytes per frame and head dim, about 5 queries x 4
// flops for each: bound by HBM. So the shape follows the stream: a window and head is one CTA of 4 warps, or a
// cluster of 2 or 4 such CTAs where there are too few of them to fill the SMs, and its 32-frame units go round the
// warps. Each warp keeps a ring of units in flight with 16-byte asynchronous copies, whose completion it can wait for
// without a barrier, and brings a running maximum, sum and output along (log2 units, fp32); the warps' states meet in
// shared memory, the CTAs' through distributed shared memory. No scratch in HBM, no counters, nothing kept between
// calls.
//
// The products run on mma.sync with keys as rows: S^T = K Q^T, O^T += V^T P^T, 16 keys by 8 queries. e4m3 converts to
// fp16 exactly, so the operands are the stored values and the fp16 queries (query_exp: bf16 ones scaled), and the scales
// are applied to the fp32 results: the scores times k_scale and the query's power, a unit's output times v_scale as
// it is added. The weights enter as fp16 in two parts, hi + lo (22 significant bits): one part alone errs by 2^-12 of the
// sum of p |v|, which shows in any output that is small beside it, bf16 ones too.
// How the operands come to lie in registers: unit_scores and unit_values in kv8.cuh.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "kv8_tile.cuh"

namespace wt {
namespace {

constexpr int few_ctas(int nt) { return nt == 1 ? 5 : (nt < 4 ? 3 : 2); }  // CTAs per SM, by tiles of 8 queries

template <typename T, int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, few_ctas(NT))
    cross8_kernel(const T *__restrict__ q, const uint8_t *__restrict__ k8, const uint8_t *__restrict__ v8,
                  const float *__restrict__ ks, const float *__restrict__ vs, const int64_t *__restrict__ lengths,
                  T *__restrict__ y, int S, int H, int Tn, int nblk, int cl, float scale) {
  namespace cg = cooperative_groups;
  constexpr int kRing = STAGES * kUnitBytes;
  static_assert(NT * 8 * kRec * 4 <= kRing, "a warp's records lie over its ring");
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int wh = blockIdx.x / cl, rank = blockIdx.x - wh * cl;
  const int w = wh / H, h = wh - w * H;
  unsigned char *ring = smem + warp * kRing;

  pdl_wait();
  pdl_launch_dependents();

  int len = Tn;
  if (lengths != nullptr) {
    const int64_t l = lengths[w];
    len = static_cast<int>(l < 0 ? 0 : (l > Tn ? Tn : l));
  }
  const int units = (len + kUnit - 1) / kUnit;
  const int step = cl * WARPS, first = warp * cl + rank;  // (the CTAs of a cluster share the last, partial round)
  const size_t base = static_cast<size_t>(wh) * Tn * 64;
  const int krow = unit_key(g);
  const uint8_t *kl = k8 + base + krow * 64 + 16 * c, *vl = v8 + base + g * 64 + 16 * c;  // this lane's pieces
  unsigned char *kd = ring + lane * 16, *vd = ring + kUnit * 64 + g * 64 + ((c ^ (g & 2)) << 4);
  auto issue = [&](int u, int stage) {
    const size_t from = static_cast<size_t>(u) * (kUnit * 64);
    const int to = stage * kUnitBytes, rows = len - u * kUnit;
    if (rows >= kUnit) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        cp16_all(kd + to + a * 512, kl + from + a * 512);
        cp16_all(vd + to + a * 512, vl + from + a * 512);
      }
    } else {  // (the last unit: frames past the window's read as zeros, and are not read)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const bool in_k = 8 * a + krow < rows, in_v = 8 * a + g < rows;
        cp16(kd + to + a * 512, in_k ? kl + from + a * 512 : k8, in_k);
        cp16(vd + to + a * 512, in_v ? vl + from + a * 512 : v8, in_v);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (first + s * step < units) issue(first + s * step, s);
    cp_commit_group();
  }

  // this window's queries: lane (g, c) holds head dims 16 c .. + 15 of query g of each tile
  const size_t HD = static_cast<size_t>(H) * 64;
  const T *qw = q + static_cast<size_t>(w) * S * HD + static_cast<size_t>(h) * 64 + 16 * c;
  uint32_t qf[NT][8];
  float qs[NT][2];  // the factors of the scores of queries 2c and 2c + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int qi = nt * 8 + g;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (qi < S) {
      a = ldg16(qw + static_cast<size_t>(qi) * HD);
      b = ldg16(qw + static_cast<size_t>(qi) * HD + 8);
    }
    uint32_t m = Mag<T>::max8(b, Mag<T>::max8(a, 0));
    m = max(m & 0xffffu, m >> 16);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const int e = query_exp<T>(m);
    const float inv = exp2_int(-e);
    qf[nt][0] = query_f16<T>(a.x, inv);
    qf[nt][1] = query_f16<T>(a.y, inv);
    qf[nt][2] = query_f16<T>(a.z, inv);
    qf[nt][3] = query_f16<T>(a.w, inv);
    qf[nt][4] = query_f16<T>(b.x, inv);
    qf[nt][5] = query_f16<T>(b.y, inv);
    qf[nt][6] = query_f16<T>(b.z, inv);
    qf[nt][7] = query_f16<T>(b.w, inv);
    const float f = exp2_int(e) * scale;
    qs[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c);
    qs[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
  }

  float m[NT][2], l[NT][2], o[NT][4][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = kLowest;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
  }
  const size_t sbase = static_cast<size_t>(wh) * nblk;
  float ksc = 0.f, vsc = 0.f;
  if (first < units) {
    ksc = ks[sbase + (first * kUnit) / kFrameBlock];
    vsc = vs[sbase + (first * kUnit) / kFrameBlock];
  }
  int stage = 0;
  for (int u = first; u < units; u += step) {
    const int ahead = u + (STAGES - 1) * step;
    if (ahead < units) issue(ahead, stage == 0 ? STAGES - 1 : stage - 1);
    cp_commit_group();
    const float k_now = ksc, v_now = vsc;
    if (u + step < units) {  // (the next unit's scales, while this one is worked on)
      ksc = ks[sbase + ((u + step) * kUnit) / kFrameBlock];
      vsc = vs[sbase + ((u + step) * kUnit) / kFrameBlock];
    }
    cp_wait_group<STAGES - 1>();
    __syncwarp();  // (V is read by other lanes than copied it)
    const unsigned char *kt = ring + stage * kUnitBytes, *vt = kt + kUnit * 64;
    const int rows = len - u * kUnit;

    float sc[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < 2; ++t) sc[nt][t][0] = sc[nt][t][1] = sc[nt][t][2] = sc[nt][t][3] = 0.f;
    unit_scores<NT>(sc, kt, qf, lane);
    uint32_t va[2][4][4];
    unit_values(va, vt, lane);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // sc[t]: (key g, query 2c), (key g, query 2c + 1), (key g + 8, query 2c), (key g + 8, query 2c + 1) of tile t
      const float f0 = k_now * qs[nt][0], f1 = k_now * qs[nt][1];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[nt][t][j] *= (j & 1) ? f1 : f0;
      if (rows < kUnit) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (16 * t + krow + (j & 2) * 4 >= rows) sc[nt][t][j] = kNegInf;
      }
      float mx0 = fmaxf(fmaxf(sc[nt][0][0], sc[nt][0][2]), fmaxf(sc[nt][1][0], sc[nt][1][2]));
      float mx1 = fmaxf(fmaxf(sc[nt][0][1], sc[nt][0][3]), fmaxf(sc[nt][1][1], sc[nt][1][3]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
      }
      const float mn0 = fmaxf(m[nt][0], mx0), mn1 = fmaxf(m[nt][1], mx1);
      if (__any_sync(0xffffffffu, mn0 != m[nt][0] || mn1 != m[nt][1])) {  // (rarer and rarer)
        const float al0 = ex2f(m[nt][0] - mn0), al1 = ex2f(m[nt][1] - mn1);
        m[nt][0] = mn0;
        m[nt][1] = mn1;
        l[nt][0] *= al0;
        l[nt][1] *= al1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[nt][i][0] *= al0;
          o[nt][i][1] *= al1;
          o[nt][i][2] *= al0;
          o[nt][i][3] *= al1;
        }
      }
      // (past kFarMax weights of at most 1, exact: what fp16 makes of them errs by 2^-25 of the largest)
      const bool near0 = fabsf(mn0) < kFarMax, near1 = fabsf(mn1) < kFarMax;
      const float up0 = (near0 ? kWeightExp : 0.f) - mn0, up1 = (near1 ? kWeightExp : 0.f) - mn1;
      const float inv0 = near0 ? kWeightInv : 1.f, inv1 = near1 ? kWeightInv : 1.f;
      float tmp[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmp[i][0] = tmp[i][1] = tmp[i][2] = tmp[i][3] = 0.f;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float p0 = ex2f(sc[nt][t][0] + up0), p1 = ex2f(sc[nt][t][1] + up1);
        const float p2 = ex2f(sc[nt][t][2] + up0), p3 = ex2f(sc[nt][t][3] + up1);
        s0 += p0 + p2;
        s1 += p1 + p3;
        unit_output(tmp, va[t], p0, p1, p2, p3);
      }
      l[nt][0] = fmaf(s0, inv0, l[nt][0]);
      l[nt][1] = fmaf(s1, inv1, l[nt][1]);
      const float v0 = v_now * inv0, v1 = v_now * inv1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[nt][i][0] = fmaf(tmp[i][0], v0, o[nt][i][0]);
        o[nt][i][1] = fmaf(tmp[i][1], v1, o[nt][i][1]);
        o[nt][i][2] = fmaf(tmp[i][2], v0, o[nt][i][2]);
        o[nt][i][3] = fmaf(tmp[i][3], v1, o[nt][i][3]);
      }
    }
    __syncwarp();  // (every lane has read the stage before it is filled again)
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  cp_wait_group<0>();
  __syncwarp();

  // this warp's state over the start of its ring: per query 64 outputs, maximum, sum
  float *rec = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], x);
      l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], x);
    }
    float *r0 = rec + (nt * 8 + 2 * c) * kRec, *r1 = r0 + kRec;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<float2 *>(r0 + 8 * g + 2 * i) = make_float2(o[nt][i][0], o[nt][i][2]);
      *reinterpret_cast<float2 *>(r1 + 8 * g + 2 * i) = make_float2(o[nt][i][1], o[nt][i][3]);
    }
    if (g == 0) {
      r0[64] = m[nt][0];
      r0[65] = l[nt][0];
      r1[64] = m[nt][1];
      r1[65] = l[nt][1];
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (cl > 1)
    cluster.sync();
  else
    __syncthreads();
  // all states -> the output: 8 threads a query, 8 head dims each; a cluster's CTAs share the (query, dims) items
  for (int t = rank * WARPS * 32 + threadIdx.x; t < S * 8; t += cl * WARPS * 32) {
    const int qq = t >> 3, d8 = (t & 7) * 8;
    float top = kLowest, den = 0.f, num[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int cr = 0; cr < cl; ++cr) {
      const unsigned char *peer = cl > 1 ? cluster.map_shared_rank(smem, cr) : smem;
#pragma unroll
      for (int wi = 0; wi < WARPS; ++wi) {
        const float *r = reinterpret_cast<const float *>(peer + wi * kRing) + qq * kRec;
        const float mr = r[64], lr = r[65];
        const float4 a = *reinterpret_cast<const float4 *>(r + d8), b = *reinterpret_cast<const float4 *>(r + d8 + 4);
        const float mn = fmaxf(top, mr), wa = ex2f(top - mn), wb = ex2f(mr - mn);
        top = mn;
        den = den * wa + lr * wb;
        num[0] = num[0] * wa + a.x * wb;
        num[1] = num[1] * wa + a.y * wb;
        num[2] = num[2] * wa + a.z * wb;
        num[3] = num[3] * wa + a.w * wb;
        num[4] = num[4] * wa + b.x * wb;
        num[5] = num[5] * wa + b.y * wb;
        num[6] = num[6] * wa + b.z * wb;
        num[7] = num[7] * wa + b.w * wb;
      }
    }
    const float inv = len == 0 ? 0.f : 1.f / den;  // (no frame: zeros; none but of score -inf: NaN)
#pragma unroll
    for (int i = 0; i < 8; ++i) num[i] *= inv;
    *reinterpret_cast<uint4 *>(y + (static_cast<size_t>(w) * S + qq) * HD + static_cast<size_t>(h) * 64 + d8) =
        pack8<T>(num);
  }
  if (cl > 1) cluster.sync();  // (no CTA leaves while another reads its records)
}

template <typename T, int NT, int WARPS, int STAGES>
int launch_cross8(const void *q, const void *k8, const void *v8, const float *ks, const float *vs,
                  const int64_t *lengths, void *y, int W, int S, int H, int Tn, int cl, void *stream) {
  constexpr int smem = WARPS * STAGES * kUnitBytes;
  auto kernel = cross8_kernel<T, NT, WARPS, STAGES>;
  const int st = opt_in_smem<cross8_kernel<T, NT, WARPS, STAGES>>(smem, "kv8_cross_attn");
  if (st != WT_OK) return st;
  const float scale = static_cast<float>(0.125 * 1.4426950408889634);
  const dim3 grid(W * H * cl), block(WARPS * 32);
  const int nblk = (Tn + kFrameBlock - 1) / kFrameBlock;
  if (cl > 1)
    return launch_clustered("kv8_cross_attn", kernel, grid, block, smem, stream, cl, static_cast<const T *>(q),
                            static_cast<const uint8_t *>(k8), static_cast<const uint8_t *>(v8), ks, vs, lengths,
                            static_cast<T *>(y), S, H, Tn, nblk, cl, scale);
  return launch("kv8_cross_attn", kernel, grid, block, smem, stream, static_cast<const T *>(q),
                static_cast<const uint8_t *>(k8), static_cast<const uint8_t *>(v8), ks, vs, lengths, static_cast<T *>(y),
                S, H, Tn, nblk, cl, scale);
}

template <typename T>
int cross8(const void *q, const void *k8, const void *v8, const float *ks, const float *vs, const int64_t *lengths,
           void *y, int W, int S, int H, int Tn, int sms, void *stream) {
  const int nt = (S + 7) / 8;  // tiles of 8 queries: 1 to 4
  const long long units = static_cast<long long>(W) * H;
  // CTAs per (window, head): 2 or 4 where the SMs then still hold them all, and a warp has a few units left. Measured at 20
  // heads x 1500 frames x 5 queries, fp16 (us per launch), by 1 / 2 / 4 / 8 CTAs: 1 window - / 7.3 / 6.3 / 8.0; 8
  // windows - / 11.3 / 11.8 / -; 32 windows 24.8 / 33 (of 3 warps' rings) / - / -.
  int cl = 1;
  while (cl < 4 && units * cl * 2 <= 3LL * sms && Tn > cl * 4 * kUnit) cl *= 2;
  // 4 warps with rings of 2 units, 5 CTAs on an SM: 32 windows of 20 heads then run as one wave. Measured (us at 1 / 8 / 16
  // / 32 / 64 windows): 4 warps x 2 units 6.3 / 11.3 / 17.0 / 24.8 / 41.7; 4 x 3 (4 CTAs) 7.8 / 10.7 / 16.4 / 26.9 / 44.3;
  // 4 x 4 (3 CTAs) 7.9 / 11.0 / 17.2 / 26.8 / 44.9; 2 x 4 6.5 / 12.8 / 21.5 / 29.1 / 47.2; 8 x 2 11.0 / 12.9 / 16.7 /
  // 26.3 / 44.8.
  if (nt == 1) return launch_cross8<T, 1, 4, 2>(q, k8, v8, ks, vs, lengths, y, W, S, H, Tn, cl, stream);
  // More queries take more registers: 9 to 24 run with 3 CTAs on an SM. Measured (us at 32 windows, fp16): 16 queries 34.7, in as
  // many registers as they like (2 CTAs, rings of 4 units) 42.6, 4 CTAs 37.5; 24 queries 48.7, with 2 CTAs 53.2, as 4 tiles
  // 66.6; 32 queries 67.4, with 3 CTAs 68.4. In bf16, whose queries are scaled first, 35.5, 51.0 and 70.3.
  if (nt == 2) return launch_cross8<T, 2, 4, 2>(q, k8, v8, ks, vs, lengths, y, W, S, H, Tn, cl, stream);
  if (nt == 3) return launch_cross8<T, 3, 4, 2>(q, k8, v8, ks, vs, lengths, y, W, S, H, Tn, cl, stream);
  return launch_cross8<T, 4, 4, 3>(q, k8, v8, ks, vs, lengths, y, W, S, H, Tn, cl, stream);
}

}  // namespace
}  // namespace wt

extern "C" int wt_kv8_cross_attn(int dtype, const void *q, const void *k8, const void *v8, const float *k_scale,
                                 const float *v_scale, const int64_t *lengths, void *y, int windows, int queries,
                                 int heads, int frames, int head_dim, int *err, void *stream) {
  using namespace wt;
  WT_REQUIRE(windows > 0 && queries > 0 && heads > 0 && frames > 0, WT_ERR_ARG,
             "kv8_cross_attn: sizes must be positive (windows %d, queries %d, heads %d, frames %d)", windows, queries,
             heads, frames);
  WT_REQUIRE(q && k8 && v8 && k_scale && v_scale && y && err, WT_ERR_ARG, "kv8_cross_attn: null pointer");
  WT_ALIGNED(q);
  WT_ALIGNED(k8);
  WT_ALIGNED(v8);
  WT_ALIGNED(y);
  WT_REQUIRE(dtype == WT_F16 || dtype == WT_BF16, WT_ERR_DTYPE, "kv8_cross_attn: unknown dtype %d", dtype);
  WT_REQUIRE(head_dim == 64, WT_ERR_UNSUPPORTED, "kv8_cross_attn: head_dim %d (supported: 64)", head_dim);
  WT_REQUIRE(static_cast<long long>(windows) * heads < (1LL << 27), WT_ERR_ARG,
             "kv8_cross_attn: grid too large (windows %d x heads %d)", windows, heads);
  WT_REQUIRE(queries < (1 << 30) && static_cast<long long>(windows) * heads * kv8_cross_tiles(queries) < (1LL << 30),
             WT_ERR_ARG, "kv8_cross_attn: too many queries (%d windows x %d heads x %d)", windows, heads, queries);
  const int sms = device_sm_count();
  if (sms <= 0) return WT_ERR_CUDA;
  // Up to 32 queries share one read of the keys here, and the tile kernel's 128 rows would be mostly empty. Measured (us, here
  // / tile kernel, 20 heads x 1500 frames, fp16): 1 window x 32 queries 11.2 / 11.9; 16 windows x 32 43.7 / 56.8, of which it
  // takes 64 in 57.4. (A second round of 32 queries here took 13.1 at 1 window x 33, the tile kernel 12.2; 26.6 / 23.3 at 4
  // windows.)
  if (queries > 32)
    return kv8_cross_tile(dtype, q, k8, v8, k_scale, v_scale, lengths, y, windows, queries, heads, frames, sms, err,
                          stream);
  if (dtype == WT_BF16)
    return cross8<__nv_bfloat16>(q, k8, v8, k_scale, v_scale, lengths, y, windows, queries, heads, frames, sms, stream);
  return cross8<__half>(q, k8, v8, k_scale, v_scale, lengths, y, windows, queries, heads, frames, sms, stream);
}
