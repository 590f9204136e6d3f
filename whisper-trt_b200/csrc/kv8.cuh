// Shared pieces of the 8-bit cache kernels: e4m3 values with power-of-two scales, and what reads them as fp16.
//
// A cache value is stored * scale, stored in e4m3 (4 significant bits, largest 448), scale a float32 power of two shared
// by a block of one head's places: the smallest one, not below 2^-120, under which the block's largest finite magnitude
// is at most 448. A power of two because e4m3 is a floating-point format: it loses nothing against an exact
// amax / 448 except at the subnormal end, x / scale is then exact, so that the one rounding is the one to e4m3 (half to
// even), and multiplying by a scale is exact wherever a kernel does it. Infinities and NaN are stored as NaN and do
// not enter the scale.
#pragma once

#include "common.cuh"

namespace wt {

constexpr int kFrameBlock = 64;  // frames of a cross-attention cache that share a scale
constexpr int kMinScaleExp = -120;  // (its inverse, 2^120, is a float too)

// The exponent of the scale of a block whose largest finite magnitude is `amax`: 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kMinScaleExp ? kMinScaleExp : e;
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Two floats (already divided by the scale: at most 448, or not finite) as e4m3, `a` in the low byte. Infinities become
// NaN: the conversion itself would saturate them to 448.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  a = fabsf(a) <= 448.f ? a : __uint_as_float(0x7fffffffu);
  b = fabsf(b) <= 448.f ? b : __uint_as_float(0x7fffffffu);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
// 8 values of type T (16 bytes) times `inv` as 8 e4m3 bytes.
template <typename T>
__device__ __forceinline__ uint2 quantize8(const uint4 &u, float inv) {
  float f[8];
  unpack8<T>(u, f);
  uint2 r;
  r.x = to_e4m3x2(f[0] * inv, f[1] * inv) | (to_e4m3x2(f[2] * inv, f[3] * inv) << 16);
  r.y = to_e4m3x2(f[4] * inv, f[5] * inv) | (to_e4m3x2(f[6] * inv, f[7] * inv) << 16);
  return r;
}

// The largest of 8 packed 16-bit magnitudes, as bits (for both types the order of the bits is that of the values, and
// infinities and NaN come last); `kInf` is where they begin.
template <typename T>
struct Mag {
  static constexpr uint32_t kInf = Elem<T>::code == WT_BF16 ? 0x7f80u : 0x7c00u;
  static constexpr uint32_t kInf2 = kInf | kInf << 16;
  static __device__ __forceinline__ uint32_t max8(const uint4 &u, uint32_t m) {
    m = __vmaxu2(m, __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu));
    return __vmaxu2(m, __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
  }
  // not zero if one of two is not finite: its exponent, all ones, carries over
  static __device__ __forceinline__ uint32_t not_finite(uint32_t u) {
    constexpr uint32_t kLast = Elem<T>::code == WT_BF16 ? 0x00800080u : 0x04000400u;
    return ((u & kInf2) + kLast) & 0x80008000u;
  }
  // the same over the finite ones alone (a block that holds something else: rare)
  static __device__ __forceinline__ uint32_t finite(uint32_t u) {
    const uint32_t lo = u & 0x7fffu, hi = (u >> 16) & 0x7fffu;
    return (lo < kInf ? lo : 0u) | ((hi < kInf ? hi : 0u) << 16);
  }
  static __device__ __forceinline__ uint32_t max8_finite(const uint4 &u, uint32_t m) {
    m = __vmaxu2(m, __vmaxu2(finite(u.x), finite(u.y)));
    return __vmaxu2(m, __vmaxu2(finite(u.z), finite(u.w)));
  }
  static __device__ __forceinline__ float value(uint32_t bits) {
    return Elem<T>::to_float2(bits & 0xffffu).x;
  }
};

// Two e4m3 values (in the low 16 bits) as fp16 (exact).
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(x)));
  return r;
}

// 8 e4m3 values as fp16.
__device__ __forceinline__ uint4 widen_f16(uint32_t a, uint32_t b) {
  return make_uint4(e4m3_to_f16x2(a), e4m3_to_f16x2(a >> 16), e4m3_to_f16x2(b), e4m3_to_f16x2(b >> 16));
}

__device__ __forceinline__ float ex2f(float x) {  // 2^x on the special-function unit (2^-inf = 0)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Asynchronous copies into shared memory; `valid` false writes zeros and reads nothing.
__device__ __forceinline__ void cp16(void *dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp16_all(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp4_all(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp4(void *dst, const void *src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(valid ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait_group() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// d += a . b, fp16 operands (exact stored values and weights), fp32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// fp16 weights enter the products times 2^15 (the largest is then 2^15, and a unit's sums are divided by it again as
// they are added): normal down to 2^-29 of the largest, and never off by more than 2^-40 of it.
constexpr float kWeightExp = 15.f, kWeightInv = 1.f / 32768.f;
// An exponent is score + (15 - maximum): one addition a weight. From maxima of 2^22 on the bracket rounds by more than 1/4,
// and a weight could pass fp16's largest value: there the maximum is subtracted from the scores first, or the 15 left out.
// (A row's own matter: the others' results do not change by it.)
constexpr float kFarMax = 4194304.f;
constexpr float kLowest = -3.402823466e38f;  // a maximum before any score: no score but -inf is below it
__device__ __forceinline__ float far_part(float b) { return fabsf(b) >= kFarMax ? b : 0.f; }

// Queries enter the products as fp16 beside the fp16 form of the stored keys. fp16 queries do so as they are; a bf16
// query is first divided by a power of two that brings its largest magnitude near 2^12, where fp16 holds all of its 8
// significant bits down to 2^-27 of that magnitude, and below that errs by less than fp32 sums do. This is that power's
// exponent, from the packed magnitudes of the query's values (0 for fp16); the score is multiplied by it afterwards.
template <typename T>
__device__ __forceinline__ int query_exp(uint32_t mag_bits) {
  if (Elem<T>::code != WT_BF16) return 0;
  const int e = static_cast<int>((mag_bits & 0x7fffu) >> 7) - 127 - 12;
  return e < -100 ? -100 : e;
}
// Two query values as fp16, times 2^-e.
template <typename T>
__device__ __forceinline__ uint32_t query_f16(uint32_t u, float inv) {
  if (Elem<T>::code != WT_BF16) return u;
  const float2 f = Elem<T>::to_float2(u);
  return Elem<__half>::from_float2(f.x * inv, f.y * inv);
}

// ---- the decode kernels' unit: 32 keys of one head against tiles of 8 queries, by one warp ----------------------
// S^T = K Q^T and O^T += V^T P^T on m16n8k16, keys (then head dims) as rows, queries as columns. Register layouts are met
// by naming the keys and head dims of an mma's rows as the loads give them, for lane (g, c) = (lane / 4, lane % 4):
//   K: row g of a 16-key tile is key unit_key(g), row g + 8 the key 8 further, and the lane holds of both the head dims 16 c
//      .. 16 c + 15, one 16-byte piece: four k-steps. In shared memory a lane's pieces lie at lane * 16 + 512 a for the keys
//      unit_key(g) + 8 a: each lane reads back what it copied itself. The queries' fragments are head dims 16 c ..
//      16 c + 15 of query g, in order.
//   V: k index 2c, 2c + 1, 2c + 8, 2c + 9 is then key c, c + 4, c + 8, c + 12 of the tile, of which the lane reads head dims
//      8 g .. 8 g + 7 (conflict-free with chunk j of row r stored at j ^ (r & 2)), interleaved bytewise into pairs of
//      keys before they are converted. Output row g (g + 8) of tile i is head dim 8 g + 2 i (+ 1).
constexpr int kUnit = 32;
constexpr int kUnitBytes = kUnit * 64 * 2;  // K, then V
constexpr int kRec = 68;  // floats of a query's record between warps: output 64, maximum, sum (in 16-byte rows)

__device__ __forceinline__ int unit_key(int g) { return (g >> 1) + 4 * (g & 1); }
__device__ __forceinline__ int unit_v_at(int row, int chunk) { return row * 64 + ((chunk ^ (row & 2)) << 4); }
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// sc[nt][t] += (key g, query 2c), (key g, query 2c + 1), (key g + 8, query 2c), (key g + 8, query 2c + 1) of 16-key tile t
template <int NT>
__device__ __forceinline__ void unit_scores(float (&sc)[NT][2][4], const unsigned char *kt, const uint32_t (&qf)[NT][8],
                                            int lane) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint4 lo = *reinterpret_cast<const uint4 *>(kt + (2 * t) * 512 + lane * 16);
    const uint4 hi = *reinterpret_cast<const uint4 *>(kt + (2 * t + 1) * 512 + lane * 16);
    const uint32_t lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t a0 = e4m3_to_f16x2(lw[s]), a1 = e4m3_to_f16x2(hw[s]);
      const uint32_t a2 = e4m3_to_f16x2(lw[s] >> 16), a3 = e4m3_to_f16x2(hw[s] >> 16);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(sc[nt][t], a0, a1, a2, a3, qf[nt][2 * s], qf[nt][2 * s + 1]);
    }
  }
}
__device__ __forceinline__ void unit_values(uint32_t (&va)[2][4][4], const unsigned char *vt, int lane) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    uint2 r[4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
      r[a] = *reinterpret_cast<const uint2 *>(vt + unit_v_at(16 * t + c + 4 * a, g >> 1) + (g & 1) * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w0 = i < 2 ? r[0].x : r[0].y, w1 = i < 2 ? r[1].x : r[1].y;
      const uint32_t w2 = i < 2 ? r[2].x : r[2].y, w3 = i < 2 ? r[3].x : r[3].y;
      const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
      const uint32_t p01 = __byte_perm(w0, w1, sel), p23 = __byte_perm(w2, w3, sel);
      va[t][i][0] = e4m3_to_f16x2(p01);
      va[t][i][1] = e4m3_to_f16x2(p01 >> 16);
      va[t][i][2] = e4m3_to_f16x2(p23);
      va[t][i][3] = e4m3_to_f16x2(p23 >> 16);
    }
  }
}
// One tile's weights (in unit_scores' order) as hi + lo parts in fp16 into the output.
__device__ __forceinline__ void unit_output(float (&o)[4][4], const uint32_t (&va)[4][4], float p0, float p1, float p2,
                                            float p3) {
  const uint32_t h01 = Elem<__half>::from_float2(p0, p1), h23 = Elem<__half>::from_float2(p2, p3);
  const uint32_t pb0 = movmatrix(h01), pb1 = movmatrix(h23);
#pragma unroll
  for (int i = 0; i < 4; ++i) mma_f16(o[i], va[i][0], va[i][1], va[i][2], va[i][3], pb0, pb1);
  const float2 f01 = Elem<__half>::to_float2(h01), f23 = Elem<__half>::to_float2(h23);
  const uint32_t lb0 = movmatrix(Elem<__half>::from_float2(p0 - f01.x, p1 - f01.y));
  const uint32_t lb1 = movmatrix(Elem<__half>::from_float2(p2 - f23.x, p3 - f23.y));
#pragma unroll
  for (int i = 0; i < 4; ++i) mma_f16(o[i], va[i][0], va[i][1], va[i][2], va[i][3], lb0, lb1);
}

}  // namespace wt
