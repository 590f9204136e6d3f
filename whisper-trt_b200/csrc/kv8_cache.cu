// Filling the 8-bit caches: a window's encoder keys and values (a scale for each block of 64 frames and head), and the
// new tokens of the self-attention (a scale for each slot and head). The format and its scales: kv8.cuh.
//
// Both are bound by memory: 2 bytes in, 1 byte and a little out per value. A block of the cross cache, 64 frames x 64
// head dims x 16 bits = 8 KB, is one warp's work: it stays in the warp's registers (256 bytes a lane, all loads in flight at
// once) between the pass for the largest magnitude and the pass that rounds, so each value is read once: 32 windows of
// 375 to 1500 frames x 20 heads in 41 us, 5.6 TB/s.
#include "kv8.cuh"

namespace wt {
namespace {

constexpr int kQWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kQWarps * 32)
    quantize_cross_kernel(const T *__restrict__ k, const T *__restrict__ v, const int64_t *__restrict__ lengths,
                          uint8_t *__restrict__ k8, uint8_t *__restrict__ v8, float *__restrict__ ks,
                          float *__restrict__ vs, int H, int Tn, int nblk, int units) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x * kQWarps + (threadIdx.x >> 5);  // (window, head, block)
  if (unit >= units) return;
  const int wh = unit / nblk, b = unit - wh * nblk;
  const int t0 = b * kFrameBlock;
  int len = Tn;
  if (lengths != nullptr) {
    const int64_t l = lengths[wh / H];
    len = static_cast<int>(l < 0 ? 0 : (l > Tn ? Tn : l));
  }
  if (t0 >= len) return;  // (nothing of this block is valid: it and its scale stay as they are)
  const bool is_v = blockIdx.y != 0;
  const size_t base = (static_cast<size_t>(wh) * Tn + t0) * 64;
  const T *x = (is_v ? v : k) + base;
  uint8_t *out = (is_v ? v8 : k8) + base;
  // pass i: 8 frames; this lane 16 values of frame 8 i + lane / 4
  const int rows = len - t0, row = lane >> 2, col = (lane & 3) * 16;
  uint4 a[8][2];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = 8 * i + row < rows;
    const T *p = x + (8 * i + row) * 64 + col;
    a[i][0] = in ? ldg_stream(p) : make_uint4(0, 0, 0, 0);
    a[i][1] = in ? ldg_stream(p + 8) : make_uint4(0, 0, 0, 0);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = Mag<T>::max8(a[i][1], Mag<T>::max8(a[i][0], m));
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
  if (m >= Mag<T>::kInf) {  // something here is not finite (the whole warp agrees)
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = Mag<T>::max8_finite(a[i][1], Mag<T>::max8_finite(a[i][0], m));
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
  }
  const int e = scale_exp(Mag<T>::value(m));
  const float inv = exp2_int(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (8 * i + row >= rows) break;
    const uint2 lo = quantize8<T>(a[i][0], inv), hi = quantize8<T>(a[i][1], inv);
    *reinterpret_cast<uint4 *>(out + (8 * i + row) * 64 + col) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  if (lane == 0) (is_v ? vs : ks)[unit] = exp2_int(e);
}

// New tokens into the self-attention cache. The largest magnitude of 8 or 16 values a lane over LANES lanes, those that are
// not finite left out: the token's exponent.
template <typename T, int LANES, int N>
__device__ __forceinline__ int token_exp(const uint4 (&x)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = Mag<T>::max8(x[i], m);
  m = max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int o = LANES / 2; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (__any_sync(0xffffffffu, m >= Mag<T>::kInf)) {
    m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = Mag<T>::max8_finite(x[i], m);
    m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int o = LANES / 2; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  return scale_exp(Mag<T>::value(m));
}

// The kernels below are launched behind a call's attention kernel, which may still be at work when they start: the new
// tokens and offsets, complete since before that kernel let this one start, are read (from L2) and rounded meanwhile, and
// only the stores wait (160 rows 32.9 -> 32.0 us, 5 rows 5.5 -> 4.9, attention and append). They let nothing behind them
// start before they end: a trigger in front of the wait would let it run beside the attention, and one behind the wait costs
// more than it gives (32 rows x 223 tokens in fp16 51.9 -> 52.4 us).
template <typename T>
__device__ __forceinline__ uint4 ld_l2(const T *p) {
  return __ldcg(reinterpret_cast<const uint4 *>(p));
}
__device__ __forceinline__ int clamp_offset(int64_t o, int C) { return static_cast<int>(o < 0 ? 0 : (o > C ? C : o)); }

// A decode step's few tokens: 8 lanes per (row, key or value, head, token), 8 values a lane.
constexpr int kAThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kAThreads)
    append8_step_kernel(const T *__restrict__ qkv, const int64_t *__restrict__ offset, uint8_t *__restrict__ k8,
                        uint8_t *__restrict__ v8, float *__restrict__ ks, float *__restrict__ vs, int S, int H, int C,
                        uint32_t total) {
  const uint32_t item = blockIdx.x * (kAThreads / 8) + (threadIdx.x >> 3), it = item < total ? item : 0;  // (all shuffle)
  const uint32_t rk = it / S, h2 = 2 * H, r = rk / h2, s = it - rk * S;
  const int sub = threadIdx.x & 7;
  const uint4 x[1] = {
      ld_l2(qkv + (static_cast<size_t>(r * S + s) * 3 * H + H + (rk - r * h2)) * 64 + sub * 8)};
  const int off = clamp_offset(__ldcg(reinterpret_cast<const long long *>(offset) + r), C);
  const int e = token_exp<T, 8>(x);
  const uint2 stored = quantize8<T>(x[0], exp2_int(-e));
  pdl_wait();  // (the attention has read the cache)
  const int kvh = static_cast<int>(rk - r * h2), h = kvh < H ? kvh : kvh - H;
  if (item >= total || static_cast<int>(s) >= C - off) return;  // (past the cache: dropped)
  const size_t slot = (static_cast<size_t>(r) * H + h) * C + off + s;
  *reinterpret_cast<uint2 *>((kvh < H ? k8 : v8) + slot * 64 + sub * 8) = stored;
  if (sub == 0) (kvh < H ? ks : vs)[slot] = exp2_int(e);
}

// A prompt: a CTA per 128 tokens of one (row, key or value, head), whose slots follow one another; 4 lanes a token, 16
// values a lane, two tokens a lane. Bound by the instructions issued once the tokens lie in L2: with a step's mapping 32
// rows x 223 tokens x 20 heads took 16.2 us behind the attention, here 8.3.
constexpr int kATokens = kAThreads / 4;
template <typename T>
__global__ void __launch_bounds__(kAThreads)
    append8_prompt_kernel(const T *__restrict__ qkv, const int64_t *__restrict__ offset, uint8_t *__restrict__ k8,
                          uint8_t *__restrict__ v8, float *__restrict__ ks, float *__restrict__ vs, int S, int H, int C) {
  const int r = blockIdx.x / (2 * H), kvh = blockIdx.x - r * 2 * H, h = kvh < H ? kvh : kvh - H;
  const int sub = threadIdx.x & 3, s0 = blockIdx.y * 2 * kATokens + (threadIdx.x >> 2);
  const T *src = qkv + (static_cast<size_t>(r) * S * 3 * H + H + kvh) * 64 + sub * 16;
  uint4 x[2][2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int s = min(s0 + u * kATokens, S - 1);  // (every lane shuffles)
    const T *at = src + static_cast<size_t>(s) * 3 * H * 64;
    x[u][0] = ld_l2(at);
    x[u][1] = ld_l2(at + 8);
  }
  const int off = clamp_offset(__ldcg(reinterpret_cast<const long long *>(offset) + r), C);
  const size_t slot0 = (static_cast<size_t>(r) * H + h) * C + off;
  uint8_t *out = (kvh < H ? k8 : v8) + slot0 * 64 + sub * 16;
  float *scale = (kvh < H ? ks : vs) + slot0;
  int e[2];
  uint4 stored[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    e[u] = token_exp<T, 4>(x[u]);
    const float inv = exp2_int(-e[u]);
    const uint2 lo = quantize8<T>(x[u][0], inv), hi = quantize8<T>(x[u][1], inv);
    stored[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  pdl_wait();  // (the attention has read the cache)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int s = s0 + u * kATokens;
    if (s >= S || s >= C - off) continue;  // (past the cache: dropped)
    *reinterpret_cast<uint4 *>(out + static_cast<size_t>(s) * 64) = stored[u];
    if (sub == 0) scale[s] = exp2_int(e[u]);
  }
}

template <typename T>
int launch_append(const void *qkv, const int64_t *offset, void *k8, void *v8, float *ks, float *vs, int R, int S, int H,
                  int C, void *stream) {
  const T *x = static_cast<const T *>(qkv);
  uint8_t *k = static_cast<uint8_t *>(k8), *v = static_cast<uint8_t *>(v8);
  const dim3 block(kAThreads);
  if (S >= kATokens / 2)  // (below, half of a prompt CTA's lanes would idle)
    return launch_behind("kv8_self_attn", append8_prompt_kernel<T>,
                         dim3(static_cast<unsigned>(R) * 2 * H, (S + 2 * kATokens - 1) / (2 * kATokens)), block, 0,
                         stream, x, offset, k, v, ks, vs, S, H, C);
  const uint32_t total = static_cast<uint32_t>(R) * S * 2 * H;
  return launch_behind("kv8_self_attn", append8_step_kernel<T>, dim3((total + kAThreads / 8 - 1) / (kAThreads / 8)),
                       block, 0, stream, x, offset, k, v, ks, vs, S, H, C, total);
}

}  // namespace

int kv8_append(int dtype, const void *qkv, const int64_t *offset, void *k8, void *v8, float *ks, float *vs, int rows,
               int new_tokens, int heads, int capacity, void *stream) {
  if (dtype == WT_BF16)
    return launch_append<__nv_bfloat16>(qkv, offset, k8, v8, ks, vs, rows, new_tokens, heads, capacity, stream);
  return launch_append<__half>(qkv, offset, k8, v8, ks, vs, rows, new_tokens, heads, capacity, stream);
}

}  // namespace wt

extern "C" int wt_kv8_quantize_cross(int dtype, const void *k, const void *v, const int64_t *lengths, void *k8,
                                     void *v8, float *k_scale, float *v_scale, int windows, int heads, int frames,
                                     int head_dim, void *stream) {
  using namespace wt;
  WT_REQUIRE(windows > 0 && heads > 0 && frames > 0, WT_ERR_ARG,
             "kv8_quantize_cross: sizes must be positive (windows %d, heads %d, frames %d)", windows, heads, frames);
  WT_REQUIRE(k && v && k8 && v8 && k_scale && v_scale, WT_ERR_ARG, "kv8_quantize_cross: null pointer");
  WT_ALIGNED(k);
  WT_ALIGNED(v);
  WT_ALIGNED(k8);
  WT_ALIGNED(v8);
  WT_REQUIRE(dtype == WT_F16 || dtype == WT_BF16, WT_ERR_DTYPE, "kv8_quantize_cross: unknown dtype %d", dtype);
  WT_REQUIRE(head_dim == 64, WT_ERR_UNSUPPORTED, "kv8_quantize_cross: head_dim %d (supported: 64)", head_dim);
  const int nblk = (frames + kFrameBlock - 1) / kFrameBlock;
  const long long units = static_cast<long long>(windows) * heads * nblk;
  WT_REQUIRE(units < (1LL << 31) - kQWarps, WT_ERR_ARG, "kv8_quantize_cross: too large");
  const dim3 grid(static_cast<unsigned>((units + kQWarps - 1) / kQWarps), 2), block(kQWarps * 32);
  uint8_t *ko = static_cast<uint8_t *>(k8), *vo = static_cast<uint8_t *>(v8);
  if (dtype == WT_BF16)
    return launch("kv8_quantize_cross", quantize_cross_kernel<__nv_bfloat16>, grid, block, 0, stream,
                  static_cast<const __nv_bfloat16 *>(k), static_cast<const __nv_bfloat16 *>(v), lengths, ko, vo, k_scale,
                  v_scale, heads, frames, nblk, static_cast<int>(units));
  return launch("kv8_quantize_cross", quantize_cross_kernel<__half>, grid, block, 0, stream,
                static_cast<const __half *>(k), static_cast<const __half *>(v), lengths, ko, vo, k_scale, v_scale, heads,
                frames, nblk, static_cast<int>(units));
}
