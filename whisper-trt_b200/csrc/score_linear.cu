// Log-probabilities of given tokens, entropy and best alternatives straight from hidden states: the vocabulary
// projection x [N, d] . w [V, d]^T with scoring.cuh's statistics taken from its accumulators, so that the N x V
// logits never reach memory (a batch of forced transcripts would write and read back gigabytes of them).
//
// Few rows (a decode step): bound by the one read of w. Many rows: bound by the tensor cores. Both on pairs of CTAs
// (tcgen05, cta_group::2): an MMA covers 256 rows of x by up to 256 tokens, each CTA of the pair holding its own 128
// rows of x and half of the tokens' rows of w, so w crosses into shared memory once for 256 rows.
//   * Work: the vocabulary is cut into slices of a few such tiles, and items are (slice, 256 rows), slices outermost:
//     the pairs at work share a few slices of w and all of x in L2. A pair walks an item's tiles with its statistics
//     in registers and leaves them, with the best groups of tokens, in a scratch record per row; a second kernel merges a
//     row's records. The cut is the one that leaves the least of the last round idle (plan below).
//   * Per CTA: warp 0 issues the TMA loads (64-element blocks of d, 128-byte swizzle, completing on the first CTA's
//     barrier), warp 1 of the first CTA the MMAs, into two accumulators of 256 columns in turn; warps 2-9 of both take
//     an accumulator's statistics -- a row is a thread, half of a tile's tokens each -- while the other is filled.
//   * The statistics are a maximum per 32 tokens, then per token an exponent, two sums: some 7 instructions, a fifth of
//     the time a tile's MMAs take at d = 1280. The alternatives are not sought token by token (a list per row that takes
//     in a token at a time, 32 rows to a warp, each diverging at its own, took twice the MMAs' time in a short walk):
//     the `top` best tokens of a walk lie in the `top` groups of 32 tokens with the largest maxima. A thread keeps
//     those groups' maxima, and copies the 32 logits of a group that enters to the place of the one that leaves; the merge
//     kernel looks into the few groups whose maxima can matter.
// Measured, 51865 tokens, d 1280: 7136 states 605 to 662 us (1565 to 1430 TFLOP/s, by the power cap), 0.40 us for a block of
// 64 of d where a library product takes 0.37; 160 states with 5 alternatives 44.5 us (w alone 20), 11 of them the merge.
// Waits are bounded as in the other tcgen05 kernels: a wait that runs out sets the error word and a stop flag, and the
// CTA drains what it has issued, meets its pair and returns.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "scoring.cuh"
#include "tc05.cuh"
#include "tma.cuh"

namespace wt {
namespace {

constexpr int kSlEpiWarps = 8;
constexpr int kSlThreads = 32 * (2 + kSlEpiWarps);
constexpr int kSlRows = 128;        // rows of x per CTA (256 per pair)
constexpr int kSlTile = 256;        // tokens per tile, at most
constexpr int kSlStages = 6;
constexpr int kSlABytes = kSlRows * 128;
constexpr int kSlStageBytes = 2 * kSlABytes;  // x block, then the CTA's half of the w block (at most 128 rows)
constexpr int kSlSmem = 1024 + kSlStages * kSlStageBytes + (2 * kSlStages + 5) * 8 + 16;
constexpr int kSlTmem = 512;
constexpr int kSlErrTimeout = 1;
constexpr int kSlMaxVocab = 1 << 20, kSlMaxRows = 1 << 24;

// ---- pairs of CTAs -----------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t in_first_cta(const void *p) {  // the same place in the pair's first CTA
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_addr(p)));
  return r;
}
__device__ __forceinline__ void pair_tma_load(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// the barrier at this place in both CTAs gets one arrival when the MMAs issued so far have completed
__device__ __forceinline__ void pair_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

constexpr int kSlGroup = 32;                // tokens per group: what a thread takes at a time
static_assert(kMaxTop <= kSlGroup, "a group's place fits below its first token");

struct SlPlan {
  int mblk, nmma, tiles, slices, items, pairs, kblocks, rec, parts;
};

// The cut of the vocabulary: `tiles` tiles of `nmma` tokens a slice. An item costs its tiles, each nmma tokens plus about
// 16 for the hand-over, and the records' writes, about 32 more; the cheapest number of rounds over the pairs wins.
SlPlan sl_plan(int rows, int vocab, int d, int top, int sms) {
  SlPlan p{};
  p.mblk = (rows + 2 * kSlRows - 1) / (2 * kSlRows);
  p.kblocks = (d + 63) / 64;
  const int pairs = sms / 2 > 0 ? sms / 2 : 1;
  long long best = -1;
  for (int nmma = kSlTile; nmma >= 128; nmma -= 32)
    for (int tiles = 1; tiles <= 16; ++tiles) {
      const long long slices = (vocab + nmma * tiles - 1) / (nmma * tiles);
      const long long rounds = (slices * p.mblk + pairs - 1) / pairs;
      const long long cost = rounds * (tiles * (nmma + 16) + 32);
      if (best < 0 || cost < best) {
        best = cost;
        p.nmma = nmma;
        p.tiles = tiles;
        p.slices = static_cast<int>(slices);
      }
    }
  p.items = p.slices * p.mblk;
  p.pairs = p.items < pairs ? p.items : pairs;
  // floats of a record: m, s, t, (padding), the best groups' maxima, tokens + places, logits
  p.rec = 4 + (2 * top + 3) / 4 * 4 + top * kSlGroup;
  p.parts = 2 * p.slices;             // records of a row (two halves of each slice's tiles)
  return p;
}

struct SlArgs {
  const int64_t *tokens;
  const uint8_t *suppress;
  float *part;   // [rows / 32, parts][rec words of 32 rows each]: a warp's rows side by side (logits: 16 bytes a row)
  float *token;  // [rows]: the given tokens' logits
  int N, V, top;
  SlPlan p;
  int *err;
  uint32_t polls;
  int withhold;
};

// Where the record of part `part` of the 32 rows from row0 on begins.
__device__ __forceinline__ size_t record_at(const SlArgs &a, int row0, int part) {
  return (static_cast<size_t>(row0 / 32) * a.p.parts + part) * (32 * a.p.rec);
}

// KK: the length of a row's list in registers, 0 without alternatives.
template <bool BF16, int KK>
__global__ void __launch_bounds__(kSlThreads, 1)
    score_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const SlArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kSlStages * kSlStageBytes);
  uint64_t *empty = full + kSlStages;
  uint64_t *acc_full = empty + kSlStages;
  uint64_t *acc_empty = acc_full + 2;
  uint64_t *drained = acc_empty + 2;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drained + 1);
  volatile int *stop = reinterpret_cast<volatile int *>(tmem_holder + 1);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), pair = blockIdx.x >> 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nmma = a.p.nmma, half_n = nmma / 2, kblocks = a.p.kblocks;

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_holder)),
                 "r"(static_cast<uint32_t>(kSlTmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&xmap);
    for (int s = 0; s < kSlStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kSlEpiWarps);  // (both CTAs' epilogue warps, at the first CTA's)
    }
    mbar_init(drained, 1);
    *stop = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  cluster.sync();  // (the pair's barriers stand before anything of either arrives on them)
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {  // producer: this CTA's x block and half of the w block of every stage
      const bool hold = a.withhold && blockIdx.x == 0;  // (test hook: the first stage's x block is left out)
      const uint32_t first_full = in_first_cta(full);  // (the first CTA's barriers count both CTAs' copies)
      int it = 0, s = 0;
      uint32_t phase = 1;  // (of the empty barriers: the first round finds them free)
      bool halt = false;
      for (int item = pair; item < a.p.items && !halt; item += a.p.pairs) {
        const int slice = item / a.p.mblk, mfirst = (item - slice * a.p.mblk) * 2 * kSlRows, m0 = mfirst + rank * kSlRows;
        // (a second CTA none of whose rows exist loads no x, and what its half of the accumulator holds is not read)
        const uint32_t bytes =
            static_cast<uint32_t>((mfirst + kSlRows < a.N ? 2 : 1) * kSlABytes + 2 * half_n * 128);
        for (int tile = 0; tile < a.p.tiles && !halt; ++tile) {
          const int v0 = (slice * a.p.tiles + tile) * nmma;
          if (v0 >= a.V) break;
          for (int kb = 0; kb < kblocks; ++kb, ++it) {
            if (it >= kSlStages && !mbar_try_wait(&empty[s], phase) &&
                !mbar_wait_role(&empty[s], phase, a.err, kSlErrTimeout, a.polls, stop)) {
              halt = true;
              break;
            }
            unsigned char *st = smem + s * kSlStageBytes;
            if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
            if (m0 < a.N && !(hold && it == 0)) pair_tma_load(st, &xmap, kb * 64, m0, first_full + 8 * s);
            pair_tma_load(st + kSlABytes, &wmap, kb * 64, v0 + rank * half_n, first_full + 8 * s);
            if (++s == kSlStages) {
              s = 0;
              phase ^= 1;
            }
          }
        }
      }
      // every copy of the pair has landed, and every arrival that the MMAs owe this CTA's barriers has come, before
      // the shared memory goes away (bounded)
      for (int i = it > kSlStages ? it - kSlStages : 0; i < it; ++i) {
        if (rank == 0) mbar_wait_bounded(&full[i % kSlStages], (i / kSlStages) & 1, nullptr, 0, a.polls);
        if (!halt && !*stop) mbar_wait_bounded(&empty[i % kSlStages], (i / kSlStages) & 1, nullptr, 0, a.polls);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {  // MMA issuer for the pair: tile j into accumulator j % 2
      // (one thread feeds the tensor cores of both SMs, 512 cycles of them with each k block: what it computes between
      // the blocks is kept to a few instructions)
      const uint32_t idesc = idesc_f16(2 * kSlRows, nmma, BF16);
      const uint64_t adesc0 = sw128_desc(smem_addr(smem)), bdesc0 = sw128_desc(smem_addr(smem) + kSlABytes);
      constexpr uint64_t kDescStage = kSlStageBytes >> 4;  // (a descriptor's address is in units of 16 bytes)
      uint64_t adesc = adesc0, bdesc = bdesc0;
      int s = 0, j = 0;
      uint32_t phase = 0;
      bool halt = false;
      for (int item = pair; item < a.p.items && !halt; item += a.p.pairs) {
        const int slice = item / a.p.mblk;
        for (int tile = 0; tile < a.p.tiles && !halt; ++tile) {
          if ((slice * a.p.tiles + tile) * nmma >= a.V) break;
          const int b = j & 1, use = j >> 1;
          if (use >= 1 && !mbar_wait_role(&acc_empty[b], (use - 1) & 1, a.err, kSlErrTimeout, a.polls, stop)) {
            halt = true;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + static_cast<uint32_t>(b * kSlTile);
          for (int kb = 0; kb < kblocks; ++kb) {
            if (!mbar_try_wait(&full[s], phase) &&
                !mbar_wait_role(&full[s], phase, a.err, kSlErrTimeout, a.polls, stop)) {
              halt = true;
              break;
            }
            tc_fence_after();
            pair_umma(d, adesc, bdesc, idesc, kb != 0);
            pair_umma(d, adesc + 2, bdesc + 2, idesc, 1);
            pair_umma(d, adesc + 4, bdesc + 4, idesc, 1);
            pair_umma(d, adesc + 6, bdesc + 6, idesc, 1);
            pair_commit(&empty[s]);
            adesc += kDescStage;
            bdesc += kDescStage;
            if (++s == kSlStages) {
              s = 0;
              phase ^= 1;
              adesc = adesc0;
              bdesc = bdesc0;
            }
          }
          if (!halt) pair_commit(&acc_full[b]);
          ++j;
        }
      }
      pair_commit(drained);  // every MMA issued has completed before the tensor memory is freed (bounded)
    }
    if (lane == 0) mbar_wait_bounded(drained, 0, nullptr, 0, a.polls);
  } else {
    // epilogue: thread = row (lane quarter warp % 4), half of the tile's tokens
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    int j = 0;
    bool halt = false;
    for (int item = pair; item < a.p.items && !halt; item += a.p.pairs) {
      const int slice = item / a.p.mblk;
      const int row = (item - slice * a.p.mblk) * 2 * kSlRows + rank * kSlRows + quarter * 32 + lane;
      const int64_t tok64 = row < a.N ? a.tokens[row] : -1;
      const int tok = tok64 >= 0 && tok64 < a.V ? static_cast<int>(tok64) : -1;
      SoftStat st = soft_empty();
      // the best groups: maxima in order, and their first tokens (multiples of 32) + places; of KK, the first KK - top
      // stay at infinity
      float lv[KK > 0 ? KK : 1];
      int ls[KK > 0 ? KK : 1];
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        lv[i] = i < KK - a.top ? -kNegInf : kNegInf;
        ls[i] = i - (KK - a.top);
      }
      float *rec = a.part + record_at(a, row - lane, slice * 2 + half) + lane;
      const bool idle = row - lane >= a.N;  // (none of this warp's rows exist)
      for (int tile = 0; tile < a.p.tiles; ++tile) {
        const int v0 = (slice * a.p.tiles + tile) * nmma;
        if (v0 >= a.V) break;
        const int b = j & 1, use = j >> 1;
        if (!__all_sync(0xffffffffu,
                        mbar_wait_role(&acc_full[b], use & 1, a.err, kSlErrTimeout, a.polls, stop))) {
          halt = true;
          break;
        }
        tc_fence_after();
        const uint32_t base_t = tmem + static_cast<uint32_t>(b * kSlTile) + (static_cast<uint32_t>(quarter * 32) << 16);
        for (int c = half * 32; c < nmma && !idle; c += 64) {
          const int v = v0 + c;
          uint32_t raw[32];
          tmem_ld32(base_t + static_cast<uint32_t>(c), raw);
          const bool out = v + lane >= a.V || (a.suppress != nullptr && a.suppress[v + lane] != 0);
          const unsigned gone = __ballot_sync(0xffffffffu, out);  // tokens that are suppressed or past the vocabulary
          tmem_wait_ld();
          float x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(raw[i]);
          const int at = tok - v;
          if (__any_sync(0xffffffffu, at >= 0 && at < 32 && row < a.N)) {
            float xt = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) xt = at == i ? x[i] : xt;
            if (at >= 0 && at < 32 && row < a.N) a.token[row] = (gone >> at) & 1u ? kNegInf : xt;
          }
          if (gone != 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = (gone >> i) & 1u ? kNegInf : x[i];
          }
          float cm = x[0];
#pragma unroll
          for (int i = 1; i < 32; ++i) cm = fmaxf(cm, x[i]);
          if (cm > st.m) soft_raise(st, cm);
          const float base = soft_base(st.m);
          float cs = 0.f, ct = 0.f;  // (the chunk's sums apart: a row's thousands of terms in one chain would round more)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float y = soft_floor((x[i] - base) * kLog2e), e = sc_ex2(y);
            cs += e;
            ct = fmaf(e, y, ct);
          }
          st.s += cs;
          st.t += ct;
          if (KK > 0 && cm > lv[KK > 0 ? KK - 1 : 0] && row < a.N) {
            const int place = ls[KK > 0 ? KK - 1 : 0] & (kSlGroup - 1);
            lv[KK > 0 ? KK - 1 : 0] = cm;
            ls[KK > 0 ? KK - 1 : 0] = v | place;
#pragma unroll
            for (int i = KK - 1; i > 0; --i)
              if (lv[i] > lv[i - 1]) {
                const float tv = lv[i];
                lv[i] = lv[i - 1];
                lv[i - 1] = tv;
                const int ti = ls[i];
                ls[i] = ls[i - 1];
                ls[i - 1] = ti;
              }
            float *to = rec - lane + 32 * (3 + 2 * a.top + place * kSlGroup) + 4 * lane;
#pragma unroll
            for (int i = 0; i < kSlGroup; i += 4)
              *reinterpret_cast<float4 *>(to + 32 * i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(in_first_cta(&acc_empty[b]));
        ++j;
      }
      if (!halt && row < a.N) {
        rec[0] = st.m;
        rec[32] = st.s;
        rec[64] = st.t;
#pragma unroll
        for (int i = 0; i < KK; ++i) {
          const int k = i - (KK - a.top);
          if (k >= 0) {
            rec[32 * (3 + k)] = lv[i];
            rec[32 * (3 + a.top + k)] = __int_as_float(ls[i]);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster.sync();  // (neither CTA of the pair leaves, or frees tensor memory, while the other is at work)
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(static_cast<uint32_t>(kSlTmem))
                 : "memory");
}

// A group's first token + place names its record: the slice and the half (of a tile's 32-token chunks every other one).
__device__ __forceinline__ int part_of(const SlArgs &a, int token_place) {
  const int per_slice = a.p.tiles * a.p.nmma, slice = token_place / per_slice;
  return 2 * slice + ((token_place - slice * per_slice) % a.p.nmma / 32 & 1);
}
// A logit of a row's stored group.
__device__ __forceinline__ float group_logit(const SlArgs &a, int row, int token_place, int i) {
  return a.part[record_at(a, row, part_of(a, token_place)) +
                32 * (3 + 2 * a.top + (token_place & (kSlGroup - 1)) * kSlGroup + (i & ~3)) + 4 * (row & 31) + (i & 3)];
}
__device__ __forceinline__ SoftStat record_stat(const SlArgs &a, int row, int part) {
  const float *rec = a.part + record_at(a, row, part) + (row & 31);
  return SoftStat{rec[0], rec[32], rec[64]};
}
// The k-th best group of a row's record (maximum, first token + place). What a call that gave up a wait left behind may be
// anything: a group that cannot be is not one.
__device__ __forceinline__ Key record_group(const SlArgs &a, int row, int part, int k) {
  const float *rec = a.part + record_at(a, row, part) + (row & 31);
  const float v = rec[32 * (3 + k)];
  const int id = __float_as_int(rec[32 * (3 + a.top + k)]);
  return id >= 0 && (id & ~(kSlGroup - 1)) < a.V && (id & (kSlGroup - 1)) < a.top ? key_of(v, id) : 0;
}

// A row's records -> its outputs. The `top` best groups lie in the `top` records whose own best are best, and the `top` best
// tokens in those groups: so first the records' best in order, then the groups of the first of them, then their tokens that
// reach the last group's maximum. Few records: a warp a row, two records a lane.
__global__ void __launch_bounds__(128) score_merge_kernel(const SlArgs a, const ScoreOut out) {
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, top = a.top;
  if (row >= a.N) return;
  const int64_t tok = a.tokens[row];
  const bool has = tok >= 0 && tok < a.V;
  const float xt = has ? a.token[row] : 0.f;
  SoftStat st = soft_empty();
  Key best = 0;
  for (int p = lane; p - lane < a.p.parts; p += 32) {
    Key more = 0;
    if (p < a.p.parts) {
      st = soft_merge(st, record_stat(a, row, p));
      if (top > 0) more = record_group(a, row, p, 0);
    }
    if (top > 0) warp_sorted_add(best, more, p == lane);
  }
  st = soft_merge_lanes(st);
  if (top > 1) {
    const Key records = best;
    for (int c = lane; c - lane < top * top; c += 32) {
      const Key of = __shfl_sync(0xffffffffu, records, c < top * top ? c / top : 0);
      warp_sorted_add(best, c < top * top && of != 0 ? record_group(a, row, part_of(a, key_token(of)), c % top) : 0,
                      c == lane);
    }
  }
  Key found = 0;
  if (top > 0) {
    const int group = key_token(best);
    const float last = __shfl_sync(0xffffffffu, key_value(best), top - 1);  // (-inf: there are fewer)
    float v[kMaxTop];
#pragma unroll
    for (int k = 0; k < kMaxTop; ++k) {  // (all loads together)
      const int token = __shfl_sync(0xffffffffu, group, k < top ? k : 0);
      v[k] = k < top && token >= 0 ? group_logit(a, row, token, lane) : kNegInf;
    }
#pragma unroll
    for (int k = 0; k < kMaxTop; ++k)
      if (k < top) {
        const int first = __shfl_sync(0xffffffffu, group, k) & ~(kSlGroup - 1);
        warp_insert(found, top, v[k] >= last ? key_of(v[k], first + lane) : 0);
      }
  }
  write_scores(out, row, top, st, found, has, xt);
}

// Many records: a CTA of 8 warps a row. A warp keeps the best groups of its records, which it loads at once: few of those
// behind the records' best enter the list. The warps' lists, then the groups' tokens, are counted into place.
__global__ void __launch_bounds__(256) score_merge_wide_kernel(const SlArgs a, const ScoreOut out) {
  constexpr int kWarps = 8;
  static_assert(kMaxTop * (kWarps + 1) <= kWarps * 32 && kMaxTop <= 2 * kWarps, "an entry a thread; two groups a warp");
  __shared__ SoftStat stat_s[kWarps];
  __shared__ Key list[kMaxTop * (kWarps + 1)], best[kMaxTop];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x, top = a.top;
  const int64_t tok = a.tokens[row];
  const bool has = tok >= 0 && tok < a.V;
  const float xt = has ? a.token[row] : 0.f;
  // of the k-th best group only the first top - k tokens can be among the best: these, one after another
  const int few = top * (top + 1) / 2;
  auto at = [&](int k, int j) { return k * top - k * (k - 1) / 2 + j; };
  SoftStat st = soft_empty();
  Key mine = 0;  // this warp's best groups
  for (int p0 = 0; p0 < a.p.parts; p0 += kWarps * 32) {
    const int p = p0 + warp + kWarps * lane;  // (what there is, spread over the warps)
    const bool in = p < a.p.parts;
    Key key[kMaxTop];
#pragma unroll
    for (int k = 0; k < kMaxTop; ++k) key[k] = in && k < top ? record_group(a, row, p, k) : 0;  // (all loads together)
    if (in) st = soft_merge(st, record_stat(a, row, p));
    if (top > 0) warp_sorted_add(mine, key[0], p0 == 0);
#pragma unroll
    for (int k = 1; k < kMaxTop; ++k) {
      if (k >= top || !__any_sync(0xffffffffu, key[k] > __shfl_sync(0xffffffffu, mine, top - 1))) break;  // (in order)
      warp_insert(mine, top, key[k]);
    }
  }
  if (top > 0) {
    if (lane < top) list[warp * top + lane] = mine;
    __syncthreads();
    count_into_place(list, kWarps * top, top, best);
  }
  if (top > 0) {
    const float last = key_value(best[top - 1]);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = warp + q * kWarps;
      if (k >= top) break;
      const int id = key_token(best[k]);
      const float v = id >= 0 ? group_logit(a, row, id, lane) : kNegInf;
      Key key = v >= last ? key_of(v, (id & ~(kSlGroup - 1)) + lane) : 0;
      warp_sort(key);
      if (k + lane < top) list[at(k, lane)] = key;
    }
    __syncthreads();
    count_into_place(list, few, top, best);
  }
  st = soft_merge_lanes(st);
  if (lane == 0) stat_s[warp] = st;
  __syncthreads();
  if (warp != 0) return;
  st = soft_merge_lanes(lane < kWarps ? stat_s[lane] : soft_empty());
  write_scores(out, row, top, st, lane < top ? best[lane] : 0, has, xt);
}

size_t sl_token_bytes(int rows) { return (static_cast<size_t>(rows) * 4 + 255) / 256 * 256; }
size_t sl_bytes(const SlPlan &p, int rows) {
  return sl_token_bytes(rows) + static_cast<size_t>((rows + 31) / 32 * 32) * p.parts * p.rec * sizeof(float);
}

// Rows a pass of the two kernels takes: all of them, or as many equal shares (of whole 256-row blocks) as keep the scratch
// within kSlScratch, which a pass of 7136 rows with 5 alternatives fits; the passes use it in turn.
constexpr size_t kSlScratch = 320u << 20;
int sl_pass_rows(int rows, int vocab, int d, int top, int sms, SlPlan *plan) {
  int take = rows;
  *plan = sl_plan(take, vocab, d, top, sms);
  for (long long n = 2; sl_bytes(*plan, take) > kSlScratch && take > 2 * kSlRows; ++n) {
    const long long least = static_cast<long long>((sl_bytes(*plan, take) + kSlScratch - 1) / kSlScratch) * rows / take;
    n = n > least ? n : least;
    take = static_cast<int>((rows + n - 1) / n + 2 * kSlRows - 1) / (2 * kSlRows) * (2 * kSlRows);
    *plan = sl_plan(take, vocab, d, top, sms);
  }
  return take;
}

template <bool BF16, int KK>
int launch_score(const CUtensorMap &wm, const CUtensorMap &xm, const SlArgs &a, void *stream) {
  const int st = opt_in_smem<score_kernel<BF16, KK>>(kSlSmem, "score_tokens");
  if (st != WT_OK) return st;
  return launch_clustered("score_tokens", score_kernel<BF16, KK>, dim3(2 * a.p.pairs), dim3(kSlThreads), kSlSmem, stream,
                          2, wm, xm, a);
}

// The same cut of the vocabulary for fewer rows (a call's last pass: the others' scratch holds it).
SlPlan sl_with_rows(SlPlan p, int rows) {
  p.mblk = (rows + 2 * kSlRows - 1) / (2 * kSlRows);
  p.items = p.slices * p.mblk;
  p.pairs = p.items < p.pairs ? p.items : p.pairs;
  return p;
}

// One pass: x [a.N, d] (16-bit values of either type).
int score_rows(int dtype, const uint16_t *x, const void *w, int d, const SlArgs &a, const ScoreOut &out, void *stream) {
  CUtensorMap wm, xm;
  int st = encode_tile_map(&wm, w, static_cast<unsigned long long>(a.V), static_cast<unsigned long long>(d), a.p.nmma / 2,
                           dtype);
  if (st != WT_OK) return st;
  st = encode_tile_map(&xm, x, static_cast<unsigned long long>(a.N), static_cast<unsigned long long>(d), kSlRows, dtype);
  if (st != WT_OK) return st;
  const bool bf = dtype == WT_BF16;
#define WT_SCORE_CASE(kk) st = bf ? launch_score<true, kk>(wm, xm, a, stream) : launch_score<false, kk>(wm, xm, a, stream)
  if (a.top == 0)
    WT_SCORE_CASE(0);
  else if (a.top == 1)
    WT_SCORE_CASE(1);
  else if (a.top <= 4)
    WT_SCORE_CASE(4);
  else if (a.top <= 8)
    WT_SCORE_CASE(8);
  else
    WT_SCORE_CASE(16);
#undef WT_SCORE_CASE
  if (st != WT_OK) return st;
  // (with 5 alternatives of 51866 tokens, us of the whole call by a warp / a CTA a row: 160 rows x 136 records 48.9 / 44.5,
  // 512 x 74 82.2 / 82.1, 1024 x 36 124 / 134, 7136 x 58 770 to 829 by the power cap / 864)
  if (a.p.parts <= 64)
    return launch("score_tokens", score_merge_kernel, dim3((a.N + 3) / 4), dim3(128), 0, stream, a, out);
  return launch("score_tokens", score_merge_wide_kernel, dim3(a.N), dim3(256), 0, stream, a, out);
}

}  // namespace
}  // namespace wt

extern "C" size_t wt_score_tokens_workspace(int rows, int vocab, int d_model, int top) {
  using namespace wt;
  if (rows <= 0 || vocab <= 0 || d_model <= 0 || top < 0 || top > kMaxTop || vocab > kSlMaxVocab || rows > kSlMaxRows)
    return 0;
  const int sms = device_sm_count();
  SlPlan p;
  const int take = sl_pass_rows(rows, vocab, d_model, top, sms > 0 ? sms : 148, &p);
  return sl_bytes(p, take);
}

extern "C" int wt_score_tokens(int dtype, const void *x, const void *w, const int64_t *tokens, const uint8_t *suppress,
                               float *logprob, float *entropy, float *top_logprob, int64_t *top_token, int rows,
                               int vocab, int d_model, int top, int *err, void *workspace, size_t workspace_bytes,
                               void *stream) {
  using namespace wt;
  WT_REQUIRE(rows > 0 && vocab > 0 && d_model > 0, WT_ERR_ARG,
             "score_tokens: sizes must be positive (rows %d, vocab %d, d_model %d)", rows, vocab, d_model);
  WT_REQUIRE(x && w && tokens && logprob && entropy && err && (top == 0 || (top_logprob && top_token)), WT_ERR_ARG,
             "score_tokens: null pointer");
  WT_REQUIRE(top >= 0 && top <= kMaxTop, WT_ERR_ARG, "score_tokens: top %d (0 to %d)", top, kMaxTop);
  WT_ALIGNED(x);
  WT_ALIGNED(w);
  WT_ALIGNED(workspace);
  WT_REQUIRE(d_model % 8 == 0, WT_ERR_UNSUPPORTED, "score_tokens: d_model %d is not a multiple of 8", d_model);
  WT_REQUIRE(vocab <= kSlMaxVocab && rows <= kSlMaxRows, WT_ERR_UNSUPPORTED,
             "score_tokens: too large (rows %d, vocab %d)", rows, vocab);
  WT_REQUIRE(dtype == WT_F16 || dtype == WT_BF16, WT_ERR_DTYPE, "score_tokens: unknown dtype %d", dtype);
  const int sms = device_sm_count();
  if (sms <= 0) return WT_ERR_CUDA;
  SlPlan p;
  const int take = sl_pass_rows(rows, vocab, d_model, top, sms, &p);
  WT_REQUIRE(workspace && workspace_bytes >= sl_bytes(p, take), WT_ERR_WORKSPACE,
             "score_tokens: needs a workspace of %zu bytes (given %zu)", sl_bytes(p, take),
             workspace ? workspace_bytes : 0);
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  int st = WT_OK;
  for (int row = 0; row < rows && st == WT_OK; row += take) {
    const int n = rows - row < take ? rows - row : take;
    const SlArgs a{tokens + row, suppress, reinterpret_cast<float *>(ws + sl_token_bytes(take)),
                   reinterpret_cast<float *>(ws), n, vocab, top, n == take ? p : sl_with_rows(p, n), err, wait_limit(),
                   test_withhold_stage()};
    const size_t at = static_cast<size_t>(row);
    st = score_rows(dtype, static_cast<const uint16_t *>(x) + at * d_model, w, d_model, a,
                    ScoreOut{logprob + at, entropy + at, top ? top_logprob + at * top : nullptr,
                             top ? top_token + at * top : nullptr},
                    stream);
  }
  return st;
}
