// Attention over the 8-bit K/V cache, and attention in which every query has its own span of keys.
//
// Both run the loop of the bf16 cache kernel: one CTA per (pair of 128-row query tiles, head, row), one thread issues
// S = Q K^T and O += P V (tcgen05, fp32 in TMEM), a softmax warpgroup per query tile, K/V through a ring of five
// 32 KB tiles handed over as pairs (V_j, K_j+1), lazy rescaling of O.  What differs:
//
// kQ8.  K/V tiles are not copied by TMA: four warps load the cache's bytes into registers one tile ahead, expand them
//   to bf16 and store them in the layout the tensor cores read.  A tile of K carries the largest exponent E of its
//   tokens: it holds m * 2^(e-E-6), and 2^(E+6) joins the softmax scale of that tile, one multiplication per tile.  V
//   tiles use R, the largest exponent of V so far, the same way; when R grows O is rescaled, as for a grown maximum.
//   So a byte costs 1.5 instructions (permute, mask, multiply), the products see exactly the values the cache holds,
//   and exponents may differ by 2^120 inside a head.
//
// Spans.  Row i attends keys [begin_i, end_i).  A CTA walks the key tiles between the smallest begin and the largest
//   end of its rows; a thread masks its own row, and only in tiles that its span does not cover.  V rows that no row
//   of the CTA attends are cleared on chip (0 x NaN would reach the output otherwise); one that some row of it attends stays,
//   so an infinity or NaN in it reaches the CTA's other rows too.  Rows with an empty span give 0.
//
// Split tiles write unnormalised O, the running maximum, sum and V exponent to scratch; combine_kernel merges them.
//
// Bound by the chain S -> softmax -> P V of a query tile, two of which share the tensor pipe and the exp unit (both some
// 60 % busy): 3800 cycles a step of 128 keys for 256 queries.  14040 queries in three blocks over 14040 keys x 12 heads:
// 664-676 us, 1.2 PFLOP/s, where the clock stays up (756-786 us elsewhere and in long runs under the power cap); 2 x 3120
// queries over 32760 keys x 12 heads expanded first 1.15 ms of 1.24 in such a run, 2 % more than the bf16 cache kernel takes
// over the same scratch (it refuses empty rows and keeps its partial results in the one workspace of a device, where a call
// here has its own); expanded here, 256 queries over 32760 keys x 12 heads 73 us.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "attn_items.cuh"
#include "attn_tiles.cuh"
#include "ptx.cuh"
#include "q8.cuh"
#include "sdv2_internal.h"

namespace sdv2 {
namespace attnx {

using namespace attn;

enum Mode {
  kModeSpans,   // K/V tensors by TMA, a span of keys per query
  kModeExpand,  // 8-bit cache, expanded in the kernel
  kModeLens,    // K/V tensors by TMA, one length per row: the 8-bit cache after kv_read_q8_kernel
};

constexpr int kExpandWarps = 4;
// Warpgroups: 0 = the issuing warp (and the TMA warp), then with kModeExpand one that expands the cache's bytes, then one
// softmax warpgroup per query tile.  Registers move from the former to the latter: 2 x 176 + 48 + 112 of 4 x 128 a thread
// at launch, 2 x 200 + 104 of 3 x 168 without the expand warpgroup, 200 + 56 of 2 x 128 with one query tile.
//
// One query tile (kTiles 1) is for short key ranges: 256 TMEM columns and 98 KB let two CTAs share an SM, so that one's
// set-up, first loads and epilogue pass behind the other's products.  K and V have one slot each there: K_j+1 is loaded
// while the softmax of tile j runs, V_j+1 while that of tile j+1 does.  Two query tiles share every K/V tile, which long
// key ranges need: the L2 could not feed two CTAs' own tiles.
template <int kMode, int kTiles>
struct Shape {
  static constexpr bool kExpand = kMode == kModeExpand;
  static constexpr int kSoftmaxWarp0 = kExpand ? 8 : 4;
  static constexpr int kThreads = (kSoftmaxWarp0 + 4 * kTiles) * 32;
  static constexpr int kCtasPerSm = kTiles == 1 ? 2 : 1;
  static constexpr int kRegsIssue = kExpand ? 48 : kTiles == 1 ? 56 : 104, kRegsExpand = 112;
  static constexpr int kRegsSoftmax = kExpand ? 176 : 200;
  static constexpr int kRegsLaunch = kExpand || kTiles == 1 ? 128 : 168;
  static_assert((kExpand ? kRegsIssue + kRegsExpand : kRegsIssue) + kTiles * kRegsSoftmax <= kRegsLaunch * kThreads / 128,
                "the warpgroups' shares add up to more than the launch provides");
  // shared memory: Q tiles | K/V slots | barriers and words | alignment slack
  static constexpr int kRing = kTiles == 1 ? 2 : 5;
  static constexpr uint32_t kSmemKV = kTiles * kTileBytes;
  static constexpr uint32_t kSmemBar = kSmemKV + kRing * kTileBytes;
  static constexpr uint32_t kSmemBytes = kSmemBar + 256 + 1024;
  static constexpr uint32_t kTmemCols = 256 * kTiles;
  static constexpr uint32_t kColS = 0, kColO = 128 * kTiles;
};
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

constexpr int kPairBars = 3;
constexpr int kBarQFull = 0;                       // [2]
constexpr int kBarK0Full = 2;                      // K_0 in place
constexpr int kBarPairFull = 3;                    // [kPairBars] V_g and K_{g+1} in place
constexpr int kBarPairDone = 3 + kPairBars;        // [kPairBars] every MMA reading V_g or K_{g+1} (or older) completed
constexpr int kBarSFull = 3 + 2 * kPairBars;       // [2]
constexpr int kBarPFull = kBarSFull + 2;           // [2]
constexpr int kBarOFull = kBarPFull + 2;           // [2]
constexpr int kBarPHalf = kBarOFull + 2;           // [2] first 64 key columns of P written
constexpr int kBarMask = kBarPHalf + 2;            // the four warps of query tile 0 have noted which keys are attended
constexpr int kNumBars = kBarMask + 1;
// with one query tile, by key tile: K in place, V in place, K read, V read
constexpr int kBarKFull = kBarK0Full, kBarVFull = kBarPairFull, kBarKFree = kBarPairDone, kBarVFree = kBarPairDone + 1;
// words behind the barriers: abort flag, TMEM base, hull of the spans, exponents of the last four key tiles, keys of a
// tile that some row attends (three sets of 128 bits in turn)
constexpr int kWordAbort = 0, kWordTmem = 1, kWordLo = 2, kWordHi = 3, kWordFullLo = 4, kWordFullHi = 5, kWordExpK = 6,
              kWordExpV = 10, kWordMask = 14, kNumWords = 26;
static_assert(kNumBars * 8 + kNumWords * 4 <= 256, "barrier block too small");

constexpr float kRescaleThreshold = 8.0f;  // log2 units

// ------------------------------------------------------------------ expanding the 8-bit cache (kQ8)
// A tile is 8 steps x 4 warps of four tokens.  A lane has 16 bytes of one token: in every eight lanes, 64 bytes of an
// even token and of the odd one after it, whose swizzled chunks never share a bank.
constexpr int kSteps = 8;

struct TileBytes {
  uint4 raw[kSteps];
};
__device__ __forceinline__ int lane_token(int lane) { return ((lane >> 4) << 1) | ((lane >> 2) & 1); }  // 0..3
__device__ __forceinline__ int lane_byte(int lane) { return ((lane >> 3) & 1) * 64 + (lane & 3) * 16; }

// Four of the 128 exponents of a tile: tokens lane, lane + 32, ...  Tokens past the end get the smallest exponent.
struct TileExps {
  int e[4];
  __device__ __forceinline__ void load(const int8_t* base, int64_t stride_tok, int tok0, int seq_len, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = tok0 + i * 32 + lane;
      e[i] = t < seq_len ? base[t * stride_tok] : q8::kMinExp;
    }
  }
  // largest of the tile's exponents; vectors that are not finite carry -128 and leave it to the others
  __device__ __forceinline__ int top() const {
    return __reduce_max_sync(0xffffffffu, max(max(max(e[0], e[1]), max(e[2], e[3])), q8::kMinExp));
  }
  __device__ __forceinline__ uint32_t packed() const {
    return __byte_perm(__byte_perm(e[0], e[1], 0x0040), __byte_perm(e[2], e[3], 0x0040), 0x5410);
  }
};

// 16 bytes that no one reads again on this SM: not kept in L1, which shared memory leaves little of
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// `base`: this lane's bytes of token 0; `tok`: this lane's token of step 0.
__device__ __forceinline__ void load_bytes(TileBytes& t, const uint8_t* base, int64_t stride_tok, int tok, int seq_len) {
  const uint8_t* src = base + tok * stride_tok;
  const int64_t step = 16 * stride_tok;
  if (__all_sync(0xffffffffu, tok + 16 * (kSteps - 1) < seq_len)) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) t.raw[i] = ld_stream(src + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      t.raw[i] = tok + 16 * i < seq_len ? ld_stream(src + i * step) : make_uint4(0u, 0u, 0u, 0u);
  }
}

// Store the tile as bf16 m * 2^(e - ref - 6) in the 128-byte-swizzled layout of two 64-column halves.
__device__ __forceinline__ void expand_tile(const TileBytes& t, uint32_t exps, int ref, uint32_t tile, int w, int lane) {
  const int sub = w * 4 + lane_token(lane);  // token of step i: 16 i + sub
  // the four exponents of the tokens sub + 32 k and of sub + 16 + 32 k
  const uint32_t even = __shfl_sync(0xffffffffu, exps, sub), odd = __shfl_sync(0xffffffffu, exps, sub + 16);
  const uint32_t row = tile + ((lane >> 3) & 1) * kHalfTile + sub * 128;
  const uint32_t first = row + ((((lane & 3) * 2) ^ (sub & 7)) << 4), second = row + ((((lane & 3) * 2 + 1) ^ (sub & 7)) << 4);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int e = static_cast<int8_t>(((i & 1) ? odd : even) >> (8 * (i >> 1)));
    // 2^(127 + e - ref) times the subnormal m * 2^-133; e <= ref, so the multiplier is a normal bf16 number
    const uint32_t s2 = e == q8::kNotFinite ? 0x7FC07FC0u : static_cast<uint32_t>(254 + e - ref) * 0x00800080u;
    const uint32_t in[4] = {t.raw[i].x, t.raw[i].y, t.raw[i].z, t.raw[i].w};
    uint32_t o[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      q8::spread4(in[k], o[2 * k], o[2 * k + 1]);
      o[2 * k] = q8::mul_bf16x2(o[2 * k], s2);
      o[2 * k + 1] = q8::mul_bf16x2(o[2 * k + 1], s2);
    }
    st_shared_v4(first + i * 2048, o[0], o[1], o[2], o[3]);
    st_shared_v4(second + i * 2048, o[4], o[5], o[6], o[7]);
  }
}

// ------------------------------------------------------------------ the kernel
template <bool kSpans>
__device__ __forceinline__ Item find_item(const AttnXParams& p, int i) {
  if (!kSpans) return find_item_lens(p, i);
  // late query tiles first: with masks that grow along the sequence they are the long ones
  Item it;
  int tile = i;
  it.part = -1;
  it.parts = 1;
  it.slot = 0;
  if (i >= p.n_full) {
    it.slot = i - p.n_full;
    tile = p.n_full + it.slot / p.split;
    it.parts = p.split;
    if (p.split > 1) it.part = it.slot % p.split;
  }
  const int per = p.heads * p.rows;
  it.tile = p.pair_tiles - 1 - tile / per;
  it.h = tile % per % p.heads;
  it.b = tile % per / p.heads;
  it.len = 0;
  return it;
}

// Bits lo .. hi - 1 of word w of a tile's 128 key bits.
__device__ __forceinline__ uint32_t span_bits(int lo, int hi, int w) {
  const int a = max(lo - 32 * w, 0), e = min(hi - 32 * w, 32);
  if (a >= e) return 0u;
  return (e == 32 ? 0xFFFFFFFFu : (1u << e) - 1u) & (0xFFFFFFFFu << a);
}

template <int kMode, int kTiles>
__global__ void __launch_bounds__(Shape<kMode, kTiles>::kThreads, Shape<kMode, kTiles>::kCtasPerSm)
attn_x_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnXParams p) {
  constexpr bool kQ8 = kMode == kModeExpand, kSpans = kMode == kModeSpans;
  using Sh = Shape<kMode, kTiles>;
  constexpr int kRing = Sh::kRing;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + Sh::kSmemBar;
  auto bar = [&](int i) { return bar0 + 8u * i; };
  volatile int* words = reinterpret_cast<volatile int*>(gbase + Sh::kSmemBar + kNumBars * 8);
  volatile int* abort_flag = words + kWordAbort;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const Item item = find_item<kSpans>(p, blockIdx.x);
  const int b = item.b, h = item.h, q0 = item.tile * (kTiles * kBM);
  const bool two_tiles = kTiles == 2 && q0 + kBM < p.q_tokens;
  const int n_stage = two_tiles ? 2 : 1;
  const int bk = p.kv_row_broadcast ? 0 : b;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    words[kWordLo] = words[kWordFullHi] = 0x7FFFFFFF;
    words[kWordHi] = words[kWordFullLo] = 0;
    for (int i = 0; i < 12; ++i) words[kWordMask + i] = 0;
    mbar_init(bar(kBarMask), 4);
    for (int i = 0; i < 2; ++i) mbar_init(bar(kBarQFull + i), 1);
    mbar_init(bar(kBarK0Full), kQ8 ? kExpandWarps : 1);
    for (int i = 0; i < kPairBars; ++i) {
      mbar_init(bar(kBarPairFull + i), kQ8 ? kExpandWarps : 1);
      mbar_init(bar(kBarPairDone + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kBarSFull + i), 1);
      mbar_init(bar(kBarPFull + i), kBM);
      mbar_init(bar(kBarPHalf + i), kBM);
      mbar_init(bar(kBarOFull + i), 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    if (!kQ8) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(const_cast<int*>(words + kWordTmem)), Sh::kTmemCols);
    tmem_relinquish();
  }
  wait_for_previous_kernel();
  if (threadIdx.x == 0) {
    for (int s = 0; s < n_stage; ++s) {  // the queries are wanted whatever the keys; the issuing thread waits for them
      mbar_expect_tx(bar(kBarQFull + s), kTileBytes);
      tma_load_4d(base + s * kTileBytes, &tm_q, bar(kBarQFull + s), 0, h, q0 + s * kBM, b);
      tma_load_4d(base + s * kTileBytes + kHalfTile, &tm_q, bar(kBarQFull + s), 64, h, q0 + s * kBM, b);
    }
  }
  // this thread's query row (softmax warps) and its span, clipped to the keys there are; for the threads of query tile 0
  // that of the row 128 further on too
  constexpr int kSoftmaxWarp0 = Sh::kSoftmaxWarp0;
  const int my_row = q0 + (warp - kSoftmaxWarp0) * 32 + lane;  // four warps for the 128 rows of a query tile
  int span_lo = 0, span_hi = 0, span2_lo = 0, span2_hi = 0;
  auto load_span = [&](int row, int& lo, int& hi) {
    if (row >= p.q_tokens) return;
    hi = min(p.end[b * p.end_stride_row + static_cast<int64_t>(row) * p.end_stride_tok], p.kv_tokens);
    lo = p.begin == nullptr ? 0 : max(p.begin[b * p.begin_stride_row + static_cast<int64_t>(row) * p.begin_stride_tok], 0);
    if (lo >= hi) lo = hi = 0;
  };
  if (kSpans && warp >= kSoftmaxWarp0) {
    load_span(my_row, span_lo, span_hi);
    if (kTiles == 2 && warp < kSoftmaxWarp0 + 4) load_span(my_row + kBM, span2_lo, span2_hi);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_kernel_in();
  if (kSpans) {
    const bool some = span_hi > span_lo;
    const int lo = __reduce_min_sync(0xffffffffu, some ? span_lo : 0x7FFFFFFF);
    const int hi = __reduce_max_sync(0xffffffffu, some ? span_hi : 0);
    const int flo = __reduce_max_sync(0xffffffffu, some ? span_lo : 0);
    const int fhi = __reduce_min_sync(0xffffffffu, some ? span_hi : 0x7FFFFFFF);
    if (warp >= kSoftmaxWarp0 && lane == 0) {
      atomicMin(const_cast<int*>(words + kWordLo), lo);
      atomicMax(const_cast<int*>(words + kWordHi), hi);
      atomicMax(const_cast<int*>(words + kWordFullLo), flo);
      atomicMin(const_cast<int*>(words + kWordFullHi), fhi);
    }
    __syncthreads();
  }
  const uint32_t tmem = static_cast<uint32_t>(words[kWordTmem]);
  // the keys that some row attends, the key tiles they lie in, and this item's share of those
  const int key_lo = kSpans ? words[kWordLo] : 0, key_hi = kSpans ? words[kWordHi] : item.len;
  const int tile_lo = kSpans && key_lo < key_hi ? key_lo / kBN : 0;
  const int n_kv_all = key_lo < key_hi ? (key_hi + kBN - 1) / kBN - tile_lo : 0;
  const int j0 = tile_lo + (item.part < 0 ? 0 : static_cast<int>(static_cast<int64_t>(item.part) * n_kv_all / item.parts));
  const int j1 = tile_lo + (item.part < 0 ? n_kv_all
                                          : static_cast<int>(static_cast<int64_t>(item.part + 1) * n_kv_all / item.parts));
  const int n_kv = j1 - j0;  // may be 0: nothing to attend

  auto slot_off = [&](int it) { return Sh::kSmemKV + (it % kRing) * kTileBytes; };

  if (warp < 4) regs_dec<Sh::kRegsIssue>();
  if (warp == 0) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t sq[2] = {base, base + kTileBytes};
      const uint32_t tS[2] = {tmem + Sh::kColS, tmem + Sh::kColS + 128};
      const uint32_t tO[2] = {tmem + Sh::kColO, tmem + Sh::kColO + 128};
      // without condition: this thread must not leave while its copies are in flight
      bool ok = true;
      for (int s = 0; s < n_stage; ++s) ok = mbar_wait(bar(kBarQFull + s), 0, abort_flag, p.status, WAIT_Q_FULL) && ok;
      ok = ok && n_kv > 0 && mbar_wait(bar(kBarK0Full), 0, abort_flag, p.status, WAIT_KV_FULL);
      for (int s = 0; s < n_stage && ok; ++s) {
        tc_fence_after();
        issue_qk(tS[s], sq[s], base + slot_off(0));
        umma_commit(bar(kBarSFull + s));
      }
      if (kTiles == 1) {
        if (ok) umma_commit(bar(kBarKFree));
        for (int j = 0; j < n_kv && ok; ++j) {
          const uint32_t sk = base + slot_off(0), sv = base + slot_off(1);
          ok = mbar_wait(bar(kBarPHalf), j & 1, abort_flag, p.status, WAIT_P_FULL) &&
               mbar_wait(bar(kBarVFull), j & 1, abort_flag, p.status, WAIT_KV_FULL);
          if (!ok) break;
          tc_fence_after();
          issue_pv(tO[0], tS[0], sv, j > 0, 0, 4);
          ok = mbar_wait(bar(kBarPFull), j & 1, abort_flag, p.status, WAIT_P_FULL);
          if (!ok) break;
          tc_fence_after();
          issue_pv(tO[0], tS[0], sv, true, 4, 8);
          umma_commit(bar(kBarVFree));
          if (j + 1 < n_kv) {
            ok = mbar_wait(bar(kBarKFull), (j + 1) & 1, abort_flag, p.status, WAIT_KV_FULL);
            if (!ok) break;
            tc_fence_after();
            issue_qk(tS[0], sq[0], sk);
            umma_commit(bar(kBarSFull));
            umma_commit(bar(kBarKFree));
          } else {
            umma_commit(bar(kBarOFull));
          }
        }
        ok = false;  // done; the loop below is that of two query tiles
      }
      // step j: O += P_j V_j and S = Q K_{j+1}^T for each query tile; V_j and K_{j+1} are pair j of the ring
      int slot_v = 1 % kRing, slot_k = 2 % kRing, pair_bar = 0, pair_par = 0;
      for (int j = 0; kTiles == 2 && j < n_kv && ok; ++j) {
        const bool more = j + 1 < n_kv;
        const uint32_t sv = base + Sh::kSmemKV + slot_v * kTileBytes, sk = base + Sh::kSmemKV + slot_k * kTileBytes;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (s >= n_stage || !ok) break;
          // opaque to the compiler: descriptors are rebuilt from one address per tile instead of being kept, hoisted out
          // of the loop, in registers that this warp does not have (spilled, they cost 300 cycles an MMA)
          uint32_t q_tile = sq[s], s_col = tS[s], o_col = tO[s];
          asm volatile("" : "+r"(q_tile), "+r"(s_col), "+r"(o_col));
          ok = mbar_wait(bar(kBarPHalf + s), j & 1, abort_flag, p.status, WAIT_P_FULL);
          if (ok && s == 0) ok = mbar_wait(bar(kBarPairFull + pair_bar), pair_par, abort_flag, p.status, WAIT_KV_FULL);
          if (!ok) break;
          tc_fence_after();
          issue_pv(o_col, s_col, sv, j > 0, 0, 4);
          ok = mbar_wait(bar(kBarPFull + s), j & 1, abort_flag, p.status, WAIT_P_FULL);
          if (!ok) break;
          tc_fence_after();
          issue_pv(o_col, s_col, sv, true, 4, 8);
          if (more) {
            issue_qk(s_col, q_tile, sk);
            umma_commit(bar(kBarSFull + s));
          } else {
            umma_commit(bar(kBarOFull + s));
          }
        }
        if (ok) umma_commit(bar(kBarPairDone + pair_bar));
        slot_v = slot_v + 2 >= kRing ? slot_v + 2 - kRing : slot_v + 2;
        slot_k = slot_k + 2 >= kRing ? slot_k + 2 - kRing : slot_k + 2;
        if (++pair_bar == kPairBars) {
          pair_bar = 0;
          pair_par ^= 1;
        }
      }
    }
  } else if (warp < kSoftmaxWarp0) {
    if (kQ8 && warp >= 4) {
      // ---------------------------------------------------------------- expand warps
      regs_dec<Sh::kRegsExpand>();
      const int w = warp - 4;
      const int tok = j0 * kBN + w * 4 + lane_token(lane);
      const uint8_t* kb = static_cast<const uint8_t*>(p.k.ptr) + bk * p.k.stride_row + h * p.k.stride_head + lane_byte(lane);
      const uint8_t* vb = static_cast<const uint8_t*>(p.v.ptr) + bk * p.v.stride_row + h * p.v.stride_head + lane_byte(lane);
      const int8_t* keb = static_cast<const int8_t*>(p.k_exp.ptr) + bk * p.k_exp.stride_row + h * p.k_exp.stride_head;
      const int8_t* veb = static_cast<const int8_t*>(p.v_exp.ptr) + bk * p.v_exp.stride_row + h * p.v_exp.stride_head;
      TileBytes rk, rv;
      TileExps ek, ev;
      uint32_t ev_now = 0;
      int ref_v = q8::kMinExp, ref_next = q8::kMinExp;
      // K of a tile together with the exponents of its V, whose running maximum is published with K
      auto load_k = [&](int g) {
        ek.load(keb, p.k_exp.stride_tok, (j0 + g) * kBN, key_hi, lane);
        ev.load(veb, p.v_exp.stride_tok, (j0 + g) * kBN, key_hi, lane);
        load_bytes(rk, kb, p.k.stride_tok, tok + g * kBN, key_hi);
      };
      auto expand_k = [&](int g, int it) {
        const int ref = ek.top();
        ref_next = max(ref_next, ev.top());
        if (w == 0 && lane == 0) {
          words[kWordExpK + (g & 3)] = ref;
          words[kWordExpV + (g & 3)] = ref_next;
        }
        expand_tile(rk, ek.packed(), ref, base + slot_off(it), w, lane);
      };
      auto arrive = [&](int i) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(i));
      };
      if (n_kv > 0) {
        load_k(0);
        load_bytes(rv, vb, p.v.stride_tok, tok, key_hi);
        expand_k(0, 0);
        arrive(kBarK0Full);
      }
      for (int g = 0; g < n_kv; ++g) {  // pair g = items 2g+1 (V_g) and 2g+2 (K_{g+1})
        const bool more = g + 1 < n_kv;
        ev_now = ev.packed();
        ref_v = ref_next;
        if (more) load_k(g + 1);
        // the slots of pair g held K_{g-2} and V_{g-2}: free once step g-2 of the issuer has completed
        if (g >= 2) {
          bool ok = mbar_wait(bar(kBarPairDone + (g - 2) % kPairBars), ((g - 2) / kPairBars) & 1, abort_flag, p.status,
                              WAIT_KV_EMPTY);
          if (!__all_sync(0xffffffffu, ok)) break;
        }
        expand_tile(rv, ev_now, ref_v, base + slot_off(2 * g + 1), w, lane);
        if (more) {
          load_bytes(rv, vb, p.v.stride_tok, tok + (g + 1) * kBN, key_hi);
          expand_k(g + 1, 2 * g + 2);
        }
        arrive(kBarPairFull + g % kPairBars);
      }
    } else if (!kQ8 && warp == 1 && lane == 0 && n_kv > 0) {
      // ---------------------------------------------------------------- TMA producer
      auto load_tile = [&](const CUtensorMap* tm, int it, int kv_tile, uint32_t full_bar) {
        tma_load_4d(base + slot_off(it), tm, full_bar, 0, h, (j0 + kv_tile) * kBN, bk);
        tma_load_4d(base + slot_off(it) + kHalfTile, tm, full_bar, 64, h, (j0 + kv_tile) * kBN, bk);
      };
      mbar_expect_tx(bar(kBarK0Full), kTileBytes);
      load_tile(&tm_k, 0, 0, bar(kBarK0Full));
      bool ok = true;
      if (kTiles == 1) {
        int g = 0;
        bool k_ahead = false;  // the K load of tile g was made
        for (; g < n_kv; ++g) {
          k_ahead = g == 0;
          if (g > 0) {
            ok = mbar_wait(bar(kBarKFree), (g - 1) & 1, abort_flag, p.status, WAIT_KV_EMPTY);
            if (!ok) break;
            mbar_expect_tx(bar(kBarKFull), kTileBytes);
            load_tile(&tm_k, 0, g, bar(kBarKFull));
            k_ahead = true;
            ok = mbar_wait(bar(kBarVFree), (g - 1) & 1, abort_flag, p.status, WAIT_KV_EMPTY);
            if (!ok) break;
          }
          mbar_expect_tx(bar(kBarVFull), kTileBytes);
          load_tile(&tm_v, 1, g, bar(kBarVFull));
        }
        if (!ok) {  // leave no copy in flight: the last of either kind (an earlier one has been consumed)
          const long long t0 = clock64();
          const int last_k = k_ahead ? g : g - 1;
          while (!mbar_try_wait(bar(kBarKFull), last_k & 1) && clock64() - t0 < kWaitBudgetCycles) {
          }
          const long long t1 = clock64();
          while (g > 0 && !mbar_try_wait(bar(kBarVFull), (g - 1) & 1) && clock64() - t1 < kWaitBudgetCycles) {
          }
        }
        ok = true;  // done; the rest is for two query tiles
      }
      int issued = 0;  // pairs requested
      for (int g = 0; kTiles == 2 && g < n_kv; ++g) {
        if (g >= 2)
          ok = mbar_wait(bar(kBarPairDone + (g - 2) % kPairBars), ((g - 2) / kPairBars) & 1, abort_flag, p.status,
                         WAIT_KV_EMPTY);
        if (!ok) break;
        const bool more = g + 1 < n_kv;
        const uint32_t full = bar(kBarPairFull + g % kPairBars);
        mbar_expect_tx(full, more ? 2 * kTileBytes : kTileBytes);
        load_tile(&tm_v, 2 * g + 1, g, full);
        if (more) load_tile(&tm_k, 2 * g + 2, g + 1, full);
        issued = g + 1;
      }
      if (!ok) {
        // leave no copy in flight: wait (bounded) for the tiles already requested
        const long long t0 = clock64();
        while (!mbar_try_wait(bar(kBarK0Full), 0) && clock64() - t0 < kWaitBudgetCycles) {
        }
        for (int g = (issued > kPairBars ? issued - kPairBars : 0); g < issued; ++g) {
          const long long t1 = clock64();
          while (!mbar_try_wait(bar(kBarPairFull + g % kPairBars), (g / kPairBars) & 1) &&
                 clock64() - t1 < kWaitBudgetCycles) {
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    regs_inc<Sh::kRegsSoftmax>();
    const int stage = (warp - kSoftmaxWarp0) >> 2;
    if (stage == 0 || two_tiles) {
      const int quad = warp & 3;
      const int row = quad * 32 + lane;
      const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
      const uint32_t tS = tmem + lane_base + Sh::kColS + stage * 128;
      const uint32_t tO = tmem + lane_base + Sh::kColO + stage * 128;
      const int full_lo = kSpans ? words[kWordFullLo] : 0, full_hi = kSpans ? words[kWordFullHi] : key_hi;
      float m_used = -INFINITY;  // running maximum (lags by up to the threshold); -inf: no key so far
      float l = 0.f;
      int ref_v = 0;  // V exponent the accumulator is in (kQ8)
      bool ok = true;
      int n_mixed = 0;
      for (int j = 0; j < n_kv; ++j) {
        const int key0 = (j0 + j) * kBN;
        // V rows that no query row of this CTA attends lie inside the tensor, so the TMA did not zero-fill them and they
        // may hold anything, NaN included; P is 0 there, but 0 x NaN would poison output rows.  Query tile 0 clears
        // them in shared memory before it reports P (tile 1's P V is issued later), and before it holds a tile of S in
        // registers.  (kQ8: expanded as zeros.)
        if (!kQ8 && stage == 0 && (key0 < full_lo || key0 + kBN > full_hi)) {
          // which keys some row attends: each warp adds its rows' (and those 128 further on) to the tile's 128 bits
          bool attended = key0 + row < key_hi;  // kModeLens: one length for all
          if (kSpans) {
            volatile int* bits = words + kWordMask + (n_mixed % 3) * 4;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t mine = span_bits(span_lo - key0, span_hi - key0, w);
              if (kTiles == 2) mine |= span_bits(span2_lo - key0, span2_hi - key0, w);
              mine = __reduce_or_sync(0xffffffffu, mine);
              if (lane == w) {
                atomicOr(const_cast<int*>(bits + w), static_cast<int>(mine));
                // the set of the next mixed tile: everyone has read what it held two tiles ago
                if (quad == 0) words[kWordMask + ((n_mixed + 1) % 3) * 4 + w] = 0;
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kBarMask));
            ok = mbar_wait(bar(kBarMask), n_mixed & 1, abort_flag, p.status, WAIT_MASK);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            attended = (static_cast<uint32_t>(bits[row >> 5]) >> (row & 31)) & 1u;
            ++n_mixed;
          }
          // With one V slot the barrier's phase says only whether tile j or j - 1 is the last to have arrived, and tile j - 1
          // may still be on its way if it was not a mixed one.  S_j is issued behind P V of tile j - 1, so it settles that;
          // with three pair barriers pair j - 3 has long arrived.
          if (kTiles == 1) ok = mbar_wait(bar(kBarSFull), j & 1, abort_flag, p.status, WAIT_S_FULL);
          ok = ok && (kTiles == 1 ? mbar_wait(bar(kBarVFull), j & 1, abort_flag, p.status, WAIT_KV_FULL)
                                  : mbar_wait(bar(kBarPairFull + j % kPairBars), (j / kPairBars) & 1, abort_flag, p.status,
                                              WAIT_KV_FULL));
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (!attended) {
            uint8_t* vrow = gbase + slot_off(2 * j + 1) + row * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              *reinterpret_cast<uint4*>(vrow + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
              *reinterpret_cast<uint4*>(vrow + kHalfTile + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_smem();
        }
        ok = mbar_wait(bar(kBarSFull + stage), j & 1, abort_flag, p.status, WAIT_S_FULL);
        if (kQ8 && ok)  // K_j's and V_j's exponents were published with K_j: already complete, read for its ordering
          ok = j == 0 ? mbar_wait(bar(kBarK0Full), 0, abort_flag, p.status, WAIT_KV_FULL)
                      : mbar_wait(bar(kBarPairFull + (j - 1) % kPairBars), ((j - 1) / kPairBars) & 1, abort_flag, p.status,
                                  WAIT_KV_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, s[c]);
        tmem_wait_ld();
        const int lo = kSpans ? span_lo - key0 : 0, hi = (kSpans ? span_hi : key_hi) - key0;
        if (__any_sync(0xffffffffu, lo > 0 || hi < kBN)) {
          const uint32_t width = static_cast<uint32_t>(max(hi - lo, 0));
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (static_cast<uint32_t>(c * 32 + i - lo) >= width) s[c][i] = 0xFF800000u;  // -inf
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            mx0 = fmaxf(mx0, __uint_as_float(s[c][i]));
            mx1 = fmaxf(mx1, __uint_as_float(s[c][i + 1]));
            mx2 = fmaxf(mx2, __uint_as_float(s[c][i + 2]));
            mx3 = fmaxf(mx3, __uint_as_float(s[c][i + 3]));
          }
        float scale = p.scale_log2;
        int ref_new = 0;
        if (kQ8) {
          scale = fmaxf(scale * exp2_int(words[kWordExpK + (j & 3)] + 6), 1.17549435e-38f);
          ref_new = words[kWordExpV + (j & 3)];
        }
        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * scale;
        if (j == 0) {
          m_used = mx;
          ref_v = ref_new;
        } else {
          const bool grow = mx > m_used + kRescaleThreshold;
          const bool shift = kQ8 && ref_new != ref_v;  // the same for every row
          if (__any_sync(0xffffffffu, grow || shift)) {
            const float m_new = grow ? mx : m_used;
            float alpha = grow ? ex2_approx(m_used - m_new) : 1.f;
            m_used = m_new;
            l *= alpha;
            if (kQ8) alpha *= exp2_int(ref_v - ref_new);
            ref_v = ref_new;
            // O of this stage is idle here: P V of the previous kv tile completed before S arrived
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(tO + c * 32, o);
            }
          }
        }
        const float m_sub = m_used == -INFINITY ? 0.f : m_used;  // no key yet: exponentials of -inf, not of -inf + inf
        // P goes to bf16 because the product takes nothing wider beside V's bf16; the sum keeps fp32.  It puts the output off
        // by 2^-9 of itself (root mean square, values of random signs), as much as rounding the output to bf16 does.
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p0 = ex2_approx(fmaf(__uint_as_float(s[c][2 * i]), scale, -m_sub));
            const float p1 = ex2_approx(fmaf(__uint_as_float(s[c][2 * i + 1]), scale, -m_sub));
            sum0 += p0;
            sum1 += p1;
            pk[i] = pack_bf16x2(p0, p1);
          }
          tmem_st16(tS + c * 16, pk);
          if (c == 1) {  // the first 64 keys of P are complete: their share of P V can start
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(kBarPHalf + stage));
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(kBarPFull + stage));
        l += sum0 + sum1;
      }
      if (ok && n_kv > 0) {
        ok = mbar_wait(bar(kBarOFull + stage), 0, abort_flag, p.status, WAIT_O_FULL);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (ok && item.part < 0) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float unit = kQ8 ? exp2_int(ref_v + 6) : 1.f;
        const int q_row = q0 + stage * kBM + row;
        __nv_bfloat16* op = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(b) * p.out_stride_row +
                            static_cast<int64_t>(q_row) * p.out_stride_tok +
                            static_cast<int64_t>(h) * p.out_stride_head;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          if (n_kv > 0) {
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
          }
          if (q_row < p.q_tokens) {
            float y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              y[i] = l == 0.f ? 0.f : __uint_as_float(o[i]) * inv;
              if (kQ8) y[i] *= unit;
            }
            // a thread has a row of its own, so a store of 32 bytes touches half as many sectors as two of 16
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t w[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) w[k] = pack_bf16x2(y[16 * i + 2 * k], y[16 * i + 2 * k + 1]);
              if (p.out_wide) {
                st_global_v8(op + c * 32 + i * 16, w);
              } else {
                reinterpret_cast<uint4*>(op + c * 32 + i * 16)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                reinterpret_cast<uint4*>(op + c * 32 + i * 16)[1] = make_uint4(w[4], w[5], w[6], w[7]);
              }
            }
          }
        }
      } else if (ok) {
        // partial result of one key range: unnormalised accumulator, running maximum and sum, V exponent
        float* po = p.part_o + (static_cast<size_t>(item.slot) * kTiles + stage) * (kBM * kHD) + row * kHD;
        float* pm = p.part_meta + (static_cast<size_t>(item.slot) * kTiles + stage) * (3 * kBM);
        pm[row] = m_used;
        pm[kBM + row] = l;
        pm[2 * kBM + row] = static_cast<float>(ref_v);
        if (n_kv > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t w[8] = {o[8 * i],     o[8 * i + 1], o[8 * i + 2], o[8 * i + 3],
                                     o[8 * i + 4], o[8 * i + 5], o[8 * i + 6], o[8 * i + 7]};
              st_global_v8(po + c * 32 + i * 8, w);
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmemCols);
  }
}

// Merge the parts of the split tiles.  Block = (split tile, query tile, group of 8 rows), a warp a row, a lane four dims.
// out = sum_k w_k O_k / sum_k 2^(m_k - m) l_k with w_k = 2^(m_k - m + R_k - R) and the result in units of 2^(R+6); a part
// without a key has l_k = 0 and no accumulator (what lies in its place is not used).  Bound by the latency of its loads: the
// first kAhead parts' are made before the weights are known, and a lane has the weights of every 32nd part.
constexpr int kMergeRows = 8;
template <int kMode, int kTiles>
__global__ void __launch_bounds__(kMergeRows * 32) combine_kernel(const __grid_constant__ AttnXParams p) {
  constexpr bool kQ8 = kMode == kModeExpand, kSpans = kMode == kModeSpans;
  constexpr int kAhead = 8;
  const int stage = blockIdx.y, lane = threadIdx.x & 31;
  const int row = blockIdx.z * kMergeRows + (threadIdx.x >> 5);
  const Item item =
      find_item<kSpans>(p, kSpans ? p.n_full + static_cast<int>(blockIdx.x) * p.split : first_item_lens(p, blockIdx.x));
  const int q_row = item.tile * (kTiles * kBM) + stage * kBM + row;
  begin_after_previous_kernel();  // the parts are complete
  if (item.part < 0 || q_row >= p.q_tokens) return;
  const float* pm = p.part_meta + (static_cast<size_t>(item.slot) * kTiles + stage) * (3 * kBM) + row;
  const float* po = p.part_o + (static_cast<size_t>(item.slot) * kTiles + stage) * (kBM * kHD) + row * kHD + lane * 4;
  constexpr size_t pm_step = kTiles * 3 * kBM, po_step = static_cast<size_t>(kTiles) * kBM * kHD;
  float4 a[kAhead];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (k0 + i < item.parts) a[i] = *reinterpret_cast<const float4*>(po + (k0 + i) * po_step);
  };
  load(0);
  float mk[2], lk[2], rk[2];  // of parts lane, lane + 32; later ones (few queries' worth of tiles) are read again
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int k = lane + 32 * i;
    mk[i] = k < item.parts ? pm[k * pm_step] : -INFINITY;
    lk[i] = k < item.parts ? pm[k * pm_step + kBM] : 0.f;
    rk[i] = kQ8 && lk[i] != 0.f ? pm[k * pm_step + 2 * kBM] : q8::kMinExp;
  }
  float m = fmaxf(mk[0], mk[1]), ref = fmaxf(rk[0], rk[1]);
  for (int k = 64 + lane; k < item.parts; k += 32) {
    m = fmaxf(m, pm[k * pm_step]);
    if (kQ8 && pm[k * pm_step + kBM] != 0.f) ref = fmaxf(ref, pm[k * pm_step + 2 * kBM]);
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
    if (kQ8) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, i));
  }
  const float m_sub = m == -INFINITY ? 0.f : m;
  auto shift = [&](float r) { return kQ8 ? exp2_int(static_cast<int>(r - ref)) : 1.f; };
  float wk[2], l = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float up = lk[i] == 0.f ? 0.f : exp2f(mk[i] - m_sub);
    l += up * lk[i];
    wk[i] = up * shift(rk[i]);
  }
  for (int k = 64 + lane; k < item.parts; k += 32)
    if (pm[k * pm_step + kBM] != 0.f) l += exp2f(pm[k * pm_step] - m_sub) * pm[k * pm_step + kBM];
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < item.parts; k0 += kAhead) {
    if (k0 > 0) load(k0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int k = k0 + i;
      if (k >= item.parts) break;
      float w, lp;
      if (k < 64) {
        w = __shfl_sync(0xffffffffu, k < 32 ? wk[0] : wk[1], k & 31);
        lp = __shfl_sync(0xffffffffu, k < 32 ? lk[0] : lk[1], k & 31);
      } else {
        w = exp2f(pm[k * pm_step] - m_sub) * shift(pm[k * pm_step + 2 * kBM]);
        lp = pm[k * pm_step + kBM];
      }
      if (lp == 0.f) continue;
      acc.x += w * a[i].x; acc.y += w * a[i].y; acc.z += w * a[i].z; acc.w += w * a[i].w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float unit = kQ8 ? exp2_int(static_cast<int>(ref) + 6) : 1.f;
  __nv_bfloat16* op = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(item.b) * p.out_stride_row +
                      static_cast<int64_t>(q_row) * p.out_stride_tok +
                      static_cast<int64_t>(item.h) * p.out_stride_head + lane * 4;
  *reinterpret_cast<uint2*>(op) =
      make_uint2(pack_bf16x2(acc.x * inv * unit, acc.y * inv * unit), pack_bf16x2(acc.z * inv * unit, acc.w * inv * unit));
}

template <int kMode, int kTiles>
cudaError_t launch(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttnXParams& p,
                   cudaStream_t stream) {
  constexpr bool kSpans = kMode == kModeSpans;
  static DynamicSmemGrant smem_grant;  // one per instantiation
  DeviceInfo di;
  cudaError_t e = device_info(&di);
  if (e == cudaSuccess) e = smem_grant.ensure(attn_x_kernel<kMode, kTiles>, static_cast<int>(Shape<kMode, kTiles>::kSmemBytes), di.device);
  if (e != cudaSuccess) return e;
  const int items = p.n_full + p.n_parts;
  e = launch_chained(attn_x_kernel<kMode, kTiles>, dim3(items), dim3(Shape<kMode, kTiles>::kThreads),
                     Shape<kMode, kTiles>::kSmemBytes, stream, tm_q, tm_k, tm_v, p);
  if (e != cudaSuccess || p.split == 1) return e;
  const int merged = p.n_tiles - p.n_full;
  return launch_chained(combine_kernel<kMode, kTiles>, dim3(merged, kTiles == 2 && p.q_tokens > kBM ? 2 : 1, kBM / kMergeRows),
                        dim3(kMergeRows * 32), 0, stream, p);
}

}  // namespace attnx

cudaError_t launch_attn_q8_expand(const CUtensorMap& tm_q, const AttnXParams& p, cudaStream_t stream) {
  return attnx::launch<attnx::kModeExpand, 2>(tm_q, tm_q, tm_q, p, stream);
}

cudaError_t launch_attn_lens(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                             const AttnXParams& p, cudaStream_t stream) {
  return attnx::launch<attnx::kModeLens, 2>(tm_q, tm_k, tm_v, p, stream);
}

cudaError_t launch_attn_spans(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                              const AttnXParams& p, cudaStream_t stream) {
  return p.tiles == 1 ? attnx::launch<attnx::kModeSpans, 1>(tm_q, tm_k, tm_v, p, stream)
                      : attnx::launch<attnx::kModeSpans, 2>(tm_q, tm_k, tm_v, p, stream);
}

// Spans live on the device, so the host cuts the tail's tiles by their number and the number of keys alone; a part whose
// share is empty costs little.  Tiles before the tail run late queries first.
//
// One query tile to a CTA up to kShortKeys keys, two beyond (3120 queries, microseconds with one and with two): 300 keys
// x 12 heads 21.2 and 22.1, 512 x 48 heads 58.5 and 60.7, 1024 x 24 heads 53.7 and 54.9; 2048 x 24 heads 94.0 and 89.2, 4680 x
// 12 heads 107 and 99.5.  That holds for 128 queries too, whose second tile is empty: its ring is deeper (12 heads x
// 16384 keys 34.4 and 30.0).
//
// A part has at least two key tiles where everything fits one wave, else four.  One wave, with two and with four: 1001 tokens
// in five clips x 3 heads 10.9 and 12.3 us, 2 x 200 queries over 700 keys x 6 heads 12.4 and 15.5, 256 over 1536 x 12 heads 16.1
// and 16.9 (against it 600 over 800 x 12 heads, 21.0 and 18.0).  Beyond, the tail overlaps the waves before it, and merging
// parts of two tiles each mostly costs more than it saves: 4 x 3120 queries over text of 512, 77, 226 and 0 keys x 12 heads
// 42.7 and 40.0, 3120 over 512 x 48 heads 60.7 and 59.0, over 2048 x 24 heads 88.6 and 87.9 (against it 1024 x 13 heads, 34.0
// and 36.3).
int plan_spans(AttnXParams& p, int sms) {
  constexpr int kShortKeys = 1024;
  p.tiles = p.kv_tokens <= kShortKeys ? 1 : 2;
  p.pair_tiles = (p.q_tokens + 128 * p.tiles - 1) / (128 * p.tiles);
  const int wave = p.tiles == 1 ? 2 * sms : sms;
  const int64_t n_tiles = static_cast<int64_t>(p.pair_tiles) * p.heads * p.rows;
  if (n_tiles > 0x7FFFFFFFLL / 64) return -1;
  p.n_tiles = static_cast<int>(n_tiles);
  const int tail = p.n_tiles % wave;
  p.n_full = p.n_tiles - tail;
  const int min_tiles = p.n_full == 0 ? 2 : 4;
  p.split = tail == 0 ? 1 : max(1, min(min(wave / tail, 64), (p.kv_tokens + 127) / 128 / min_tiles));
  p.n_parts = tail * p.split;
  return p.split > 1 ? p.n_parts : 0;
}

}  // namespace sdv2
