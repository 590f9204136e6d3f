// Self-attention of one new token per row over an 8-bit cache (kv8.cuh) read through the slot table: cached slot j <
// offset[r] comes, e4m3 values and scales, from the row src[r, j] names; the new token itself at 16 bits from qkv.
//
// Each (row, head) gathers offset slots of 64 + 64 bytes and two scales, about 2 flops a byte: bound by memory, and
// behind that by the instructions a gathered row costs. A (row, head) is a CTA of one warp where there are enough of them
// to fill the SMs (no warp waits for another, and 24 of them hide the chain of dependent loads, slot table to keys, that
// stands before the first unit), of 4 warps where not, or a cluster of such CTAs for few rows over long caches. 32-key
// units go round the warps, through a ring of asynchronous copies per warp, the slot-table entries of a unit loaded one
// unit earlier. The unit runs on mma.sync although there is a single query (all 8 columns hold it): converting 16 keys for the tensor cores and reading one column back takes 9 instructions a key, where
// dot products and weighted sums on FMAs took 28 and bound the kernel (160 rows x 20 heads x 335 slots: 41 us).
// Scales differ from slot to slot: a score is multiplied by its key's, a weight by its value's, and the unit's products by
// the power of two that brings the largest of them near fp16's largest value, whose inverse the unit's output takes as it is
// added: a slot of large values that no weight falls on costs the others no bits. The new token is attended in fp32. The warps' states
// meet in shared memory, a cluster's through distributed shared memory.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "kv8_tile.cuh"

namespace wt {
namespace {

constexpr int kSStages = 2;
constexpr int kSStageBytes = kUnitBytes + kUnit * 8;  // K, V, (k, v) scales
constexpr int kSRing = kSStages * kSStageBytes;
constexpr int kSResident = 24;  // warps per SM: 209 KB of rings

template <typename T, int kSWarps>
__global__ void __launch_bounds__(kSWarps * 32, kSResident / kSWarps)
    self8_step_kernel(const T *__restrict__ qkv, const uint8_t *__restrict__ k8, const uint8_t *__restrict__ v8,
                      const float *__restrict__ ks, const float *__restrict__ vs, const int64_t *__restrict__ offset,
                      const int32_t *__restrict__ src, T *__restrict__ y, int N, int H, int C, int cl, float scale) {
  namespace cg = cooperative_groups;
  __shared__ __align__(128) unsigned char smem[kSWarps * kSRing];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int rh = blockIdx.x / cl, rank = blockIdx.x - rh * cl;
  const int r = rh / H, h = rh - r * H;
  const size_t HD = static_cast<size_t>(H) * 64;
  unsigned char *ring = smem + warp * kSRing;

  pdl_wait();
  pdl_launch_dependents();

  const int step = cl * kSWarps, first = warp * cl + rank;
  const int32_t *srow = src + static_cast<size_t>(r) * C;
  const uint32_t row_stride = static_cast<uint32_t>(H) * C, head = static_cast<uint32_t>(h) * C;  // in slots
  const int krow = unit_key(g);
  // the place (a cache's slots fit 32 bits: checked at the entry) of the unit's key `lane`, by the slot table (clamped)
  // -- not of the keys below the offset alone: the first load then does not wait for it
  auto load_place = [&](int u) {
    const int j = u * kUnit + lane;
    const int v = j < C ? srow[j] : 0;
    return static_cast<uint32_t>(v < 0 ? 0 : (v > N - 1 ? N - 1 : v)) * row_stride + head + (j < C ? j : 0);
  };
  uint32_t place = load_place(first);
  const int64_t o64 = offset[r];
  const int off = static_cast<int>(o64 < 0 ? 0 : (o64 > C ? C : o64));
  const int units = (off + kUnit - 1) / kUnit;
  unsigned char *kd = ring + lane * 16, *vd = ring + kUnit * 64 + unit_v_at(g, c), *sd = ring + kUnitBytes + lane * 8;
  const uint8_t *kl = k8 + 16 * c, *vl = v8 + 16 * c;
  auto issue = [&](int u, int stage, uint32_t place) {
    const int to = stage * kSStageBytes, rows = off - u * kUnit;
    if (rows >= kUnit) {
      cp4_all(sd + to, ks + place);
      cp4_all(sd + to + 4, vs + place);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const uint32_t pk = __shfl_sync(0xffffffffu, place, 8 * a + krow);
        const uint32_t pv = __shfl_sync(0xffffffffu, place, 8 * a + g);
        cp16_all(kd + to + a * 512, kl + static_cast<size_t>(pk) * 64);
        cp16_all(vd + to + a * 512, vl + static_cast<size_t>(pv) * 64);
      }
    } else {  // (the last unit: keys past the offset read as zeros, and are not read)
      cp4(sd + to, ks + place, lane < rows);
      cp4(sd + to + 4, vs + place, lane < rows);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const uint32_t pk = __shfl_sync(0xffffffffu, place, 8 * a + krow);
        const uint32_t pv = __shfl_sync(0xffffffffu, place, 8 * a + g);
        cp16(kd + to + a * 512, kl + static_cast<size_t>(pk) * 64, 8 * a + krow < rows);
        cp16(vd + to + a * 512, vl + static_cast<size_t>(pv) * 64, 8 * a + g < rows);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < kSStages - 1; ++s) {
    const int u = first + s * step;
    if (u < units) issue(u, s, place);
    place = load_place(u + step);
    cp_commit_group();
  }

  const T *qrow = qkv + static_cast<size_t>(r) * 3 * HD + static_cast<size_t>(h) * 64;
  const uint4 qa = ldg16(qrow + 16 * c), qb = ldg16(qrow + 16 * c + 8);
  uint32_t mag = Mag<T>::max8(qb, Mag<T>::max8(qa, 0));
  mag = max(mag & 0xffffu, mag >> 16);
  mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
  mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
  const int qe = query_exp<T>(mag);
  const float qinv = exp2_int(-qe), qscale = exp2_int(qe) * scale;
  const uint32_t qf[1][8] = {{query_f16<T>(qa.x, qinv), query_f16<T>(qa.y, qinv), query_f16<T>(qa.z, qinv),
                              query_f16<T>(qa.w, qinv), query_f16<T>(qb.x, qinv), query_f16<T>(qb.y, qinv),
                              query_f16<T>(qb.z, qinv), query_f16<T>(qb.w, qinv)}};

  float m = kNegInf, l = 0.f, o[4][4];  // (all columns alike; l: of this lane's keys)
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  if (rank == 0 && warp == 0) {  // the new token, at 16 bits: every row attends to it
    float q[16], k[16], v[8];
    unpack8<T>(qa, *reinterpret_cast<float(*)[8]>(q));
    unpack8<T>(qb, *reinterpret_cast<float(*)[8]>(q + 8));
    unpack8<T>(ldg16(qrow + HD + 16 * c), *reinterpret_cast<float(*)[8]>(k));
    unpack8<T>(ldg16(qrow + HD + 16 * c + 8), *reinterpret_cast<float(*)[8]>(k + 8));
    unpack8<T>(ldg16(qrow + 2 * HD + 8 * g), v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s = fmaf(q[i], k[i], s);
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    s *= scale;
    if (s != kNegInf) {  // (a score that is not finite: as the softmax of it)
      const bool fine = fabsf(s) < __uint_as_float(0x7f800000u);
      m = fine ? s : kNegInf;
      l = g != 0 ? 0.f : (fine ? 1.f : __uint_as_float(0x7fffffffu));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i][0] = o[i][1] = v[2 * i];
        o[i][2] = o[i][3] = v[2 * i + 1];
      }
    }
  }

  int stage = 0;
  for (int u = first; u < units; u += step) {
    const int ahead = u + (kSStages - 1) * step;
    if (ahead < units) issue(ahead, stage == 0 ? kSStages - 1 : stage - 1, place);
    place = load_place(ahead + step);
    cp_commit_group();
    cp_wait_group<kSStages - 1>();
    __syncwarp();  // (values and scales are read by other lanes than copied them)
    const unsigned char *kt = ring + stage * kSStageBytes, *vt = kt + kUnit * 64;
    const float2 *sc_s = reinterpret_cast<const float2 *>(kt + kUnitBytes);  // (k, v) scale of a key
    const int rows = off - u * kUnit;
    float sc[1][2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) sc[0][t][0] = sc[0][t][1] = sc[0][t][2] = sc[0][t][3] = 0.f;
    unit_scores<1>(sc, kt, qf, lane);
    uint32_t va[2][4][4];
    unit_values(va, vt, lane);
    // this lane's keys: 16 t + krow (+ 8)
    float x[2][2], w[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = sc_s[16 * t + krow + 8 * e];
        x[t][e] = sc[0][t][2 * e] * f.x * qscale;
        w[t][e] = f.y;
      }
    if (rows < kUnit) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (16 * t + krow + 8 * e >= rows) x[t][e] = kNegInf;
    }
    float mx = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
#pragma unroll
    for (int s = 4; s < 32; s <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    if (mx > m) {  // (the same in all lanes; rarer and rarer)
      const float al = ex2f(m - mx);
      m = mx;
      l *= al;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i][0] *= al;
        o[i][1] *= al;
        o[i][2] *= al;
        o[i][3] *= al;
      }
    }
    const float base = m == kNegInf ? 0.f : m;
    float sum = 0.f;
    uint32_t top = 0;  // (not negative: their bits are in their order)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float p = ex2f(x[t][e] - base);
        sum += p;
        w[t][e] *= p;
        top = max(top, __float_as_uint(w[t][e]));
      }
    l += sum;
    // the power of two that brings the largest into 2^14 .. 2^15 (of 2^-112 at least), and its inverse
    const uint32_t big = max(__reduce_max_sync(0xffffffffu, top) >> 23 & 0xffu, 15u);
    const float inv = __uint_as_float((127u + 14u + 127u - big) << 23), by = __uint_as_float((big - 14u) << 23);
    float tmp[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) tmp[i][0] = tmp[i][1] = tmp[i][2] = tmp[i][3] = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float p0 = w[t][0] * inv, p1 = w[t][1] * inv;
      unit_output(tmp, va[t], p0, p0, p1, p1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = fmaf(tmp[i][e], by, o[i][e]);
    __syncwarp();  // (every lane has read the stage before it is filled again)
    stage = stage + 1 == kSStages ? 0 : stage + 1;
  }
  cp_wait_group<0>();
  __syncwarp();

  // the warp's state over its ring; then the states -> the output
#pragma unroll
  for (int s = 4; s < 32; s <<= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
  float *rec = reinterpret_cast<float *>(ring);
  if (c == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float2 *>(rec + 8 * g + 2 * i) = make_float2(o[i][0], o[i][2]);
    if (g == 0) {
      rec[64] = m;
      rec[65] = l;
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (cl > 1)
    cluster.sync();
  else
    __syncthreads();
  if (rank == 0 && threadIdx.x < 8) {
    const int d8 = threadIdx.x * 8;
    float top = kNegInf, den = 0.f, num[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int cr = 0; cr < cl; ++cr) {
      const unsigned char *peer = cl > 1 ? cluster.map_shared_rank(smem, cr) : smem;
#pragma unroll
      for (int wi = 0; wi < kSWarps; ++wi) {
        const float *x = reinterpret_cast<const float *>(peer + wi * kSRing);
        const float mn = fmaxf(top, x[64]), mu = mn == kNegInf ? 0.f : mn;
        const float wa = ex2f(top - mu), wb = ex2f(x[64] - mu);
        top = mn;
        den = den * wa + x[65] * wb;
#pragma unroll
        for (int i = 0; i < 8; ++i) num[i] = num[i] * wa + x[d8 + i] * wb;
      }
    }
    const float inv = 1.f / den;
#pragma unroll
    for (int i = 0; i < 8; ++i) num[i] *= inv;
    *reinterpret_cast<uint4 *>(y + static_cast<size_t>(r) * HD + static_cast<size_t>(h) * 64 + d8) = pack8<T>(num);
  }
  if (cl > 1) cluster.sync();
}

template <typename T, int kSWarps>
int launch_self8(const void *qkv, const void *k8, const void *v8, const float *ks, const float *vs,
                 const int64_t *offset, const int32_t *src, void *y, int N, int H, int C, int cl, void *stream) {
  const float scale = static_cast<float>(0.125 * 1.4426950408889634);
  const dim3 grid(static_cast<unsigned>(static_cast<long long>(N) * H * cl)), block(kSWarps * 32);
  auto kernel = self8_step_kernel<T, kSWarps>;
  if (cl > 1)
    return launch_clustered("kv8_self_attn", kernel, grid, block, 0, stream, cl, static_cast<const T *>(qkv),
                            static_cast<const uint8_t *>(k8), static_cast<const uint8_t *>(v8), ks, vs, offset, src,
                            static_cast<T *>(y), N, H, C, cl, scale);
  return launch("kv8_self_attn", kernel, grid, block, 0, stream, static_cast<const T *>(qkv),
                static_cast<const uint8_t *>(k8), static_cast<const uint8_t *>(v8), ks, vs, offset, src,
                static_cast<T *>(y), N, H, C, cl, scale);
}

// One warp per (row, head) from 16 of them per SM on, else 4. Measured (us at 5 / 40 / 160 / 320 rows x 20 heads, some 335
// slots, and at 160 rows x 75 slots): 1 warp 5.3 / 17.9 / 31.4 / 56.3 / 12.2; 2 warps 5.2 / 14.1 / 34.9 / 60.5 / 15.7; 4 warps
// 4.5 / 11.9 / 36.2 / 65.1 / 18.4; 8 warps 5.2 / 15.8 / 54.0 / 103 / 39.3. Rings of 3 or 4 units, which leave room for
// fewer warps: 39.1 and 38.4 at 160 rows (1 warp); persistent CTAs whose copies run on into the next (row, head), 4 warps
// of 3 units: 45. Clusters of 2 and 4 of the 4-warp CTAs at 5 rows: 4.7 and 6.2, so only where a warp has 8 units or more.
template <typename T>
int self8_step(const void *qkv, const void *k8, const void *v8, const float *ks, const float *vs,
               const int64_t *offset, const int32_t *src, void *y, int N, int H, int C, int sms, void *stream) {
  const long long units = static_cast<long long>(N) * H;
  if (units >= 16LL * sms) return launch_self8<T, 1>(qkv, k8, v8, ks, vs, offset, src, y, N, H, C, 1, stream);
  int cl = 1;
  while (cl < 8 && units * cl * 2 <= (kSResident / 4) * sms && C > cl * 4 * kUnit * 8) cl *= 2;
  return launch_self8<T, 4>(qkv, k8, v8, ks, vs, offset, src, y, N, H, C, cl, stream);
}

}  // namespace
}  // namespace wt

extern "C" int wt_kv8_self_attn(int dtype, const void *qkv, void *k8, void *v8, float *k_scale, float *v_scale,
                                const int64_t *offset, const int32_t *src, void *y, int rows, int new_tokens,
                                int heads, int capacity, int head_dim, int write_cache, void *stream) {
  using namespace wt;
  WT_REQUIRE(rows > 0 && new_tokens > 0 && heads > 0 && capacity > 0, WT_ERR_ARG,
             "kv8_self_attn: sizes must be positive (rows %d, new_tokens %d, heads %d, capacity %d)", rows, new_tokens,
             heads, capacity);
  WT_REQUIRE(qkv && k8 && v8 && k_scale && v_scale && offset && src && y, WT_ERR_ARG, "kv8_self_attn: null pointer");
  WT_ALIGNED(qkv);
  WT_ALIGNED(k8);
  WT_ALIGNED(v8);
  WT_ALIGNED(y);
  WT_REQUIRE(dtype == WT_F16 || dtype == WT_BF16, WT_ERR_DTYPE, "kv8_self_attn: unknown dtype %d", dtype);
  WT_REQUIRE(head_dim == 64, WT_ERR_UNSUPPORTED, "kv8_self_attn: head_dim %d (supported: 64)", head_dim);
  WT_REQUIRE(static_cast<long long>(rows) * heads < (1LL << 27) && capacity <= (1 << 30) && new_tokens <= (1 << 20),
             WT_ERR_ARG, "kv8_self_attn: too large (rows %d x heads %d, %d slots, %d new tokens)", rows, heads, capacity,
             new_tokens);
  WT_REQUIRE(static_cast<unsigned long long>(rows) * heads * capacity < (1ULL << 32), WT_ERR_ARG,
             "kv8_self_attn: the cache has 2^32 slots or more (rows %d x heads %d x %d)", rows, heads, capacity);
  WT_REQUIRE(!write_cache || static_cast<long long>(rows) * heads * new_tokens * 2 < (1LL << 31), WT_ERR_ARG,
             "kv8_self_attn: too many new tokens to append (%d rows x heads %d x %d)", rows, heads, new_tokens);
  const int sms = device_sm_count();
  if (sms <= 0) return WT_ERR_CUDA;
  int st;
  if (new_tokens == 1)
    st = dtype == WT_BF16 ? self8_step<__nv_bfloat16>(qkv, k8, v8, k_scale, v_scale, offset, src, y, rows, heads,
                                                      capacity, sms, stream)
                          : self8_step<__half>(qkv, k8, v8, k_scale, v_scale, offset, src, y, rows, heads, capacity,
                                               sms, stream);
  else
    st = kv8_self_prompt(dtype, qkv, k8, v8, k_scale, v_scale, offset, src, y, rows, new_tokens, heads, capacity, stream);
  if (st != WT_OK || !write_cache) return st;
  return kv8_append(dtype, qkv, offset, k8, v8, k_scale, v_scale, rows, new_tokens, heads, capacity, stream);
}
