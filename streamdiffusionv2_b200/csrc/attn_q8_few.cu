// Attention of a few queries over the 8-bit cache: up to 16 query rows to a block, bound by reading the cache once.
//
// A block's four warps take 32 keys each in turn.  A warp has the bytes of its keys' K and V copied into its own ring of
// shared-memory stages (TMA, the next stage in flight) and works on them with m16n8k16 bf16 products, keys (for S^T = K Q^T)
// and dims (for O^T = V^T P^T) as M and eight queries as N: the tcgen05 kernel's 128 query rows would be empty, and its
// tiles would have to pass through shared memory as bf16, four times these bytes; with the queries as M (16 of them) a
// step has twice the products and twice the exponentials.  A fragment's order of dims and keys is free as long as both
// operands agree on it, so a lane loads 16 consecutive bytes of a key and expands them in registers: for K the four dims
// of a word become one k-step's pair of registers, for V the same byte of two keys becomes one register (one permute
// takes both, one mask follows).
//
// The products take the values as they come out of that, bf16 subnormals +-m * 2^-133, without a multiplication: the
// queries are scaled up by a power of two beforehand (2^qs, as far as their largest element allows), the weights by
// 2^(120 - R) with R the largest V exponent so far; a key's own powers of two join its score and its weight.  All of it
// is exact.  The running maximum is exact too (weights stay at most 1 and weight * 2^(e - R + 120) below 2^121); the
// accumulator is rescaled when it or R moves.  The warps' results merge in shared memory, the parts of a split row in
// combine_few_kernel.
//
// One query over 4 rows x 12 heads x 32760 keys (405 MB): 70-71 us, 5.7 TB/s; over one such row 25 us, of which about 10 are
// launch, first tiles and merging.  With the queries as the products' 16 rows: 77 and 33 us.  9 to 16 queries: 85-91 and 33 us.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "attn_items.cuh"
#include "ptx.cuh"
#include "q8.cuh"
#include "sdv2_internal.h"

namespace sdv2 {
namespace few {

using attnx::Item;

constexpr int kWarps = 4;
constexpr int kKeys = kFewStageKeys;  // keys of a stage
constexpr int kBlocks = kKeys / 16;   // ... in products of 16
constexpr int kStages = 2;
constexpr int kStageBytes = kKeys * 128 * 2;
constexpr int kSmemBar = kWarps * kStages * kStageBytes;
constexpr int kSmemBytes = kSmemBar + kWarps * kStages * 8 + 16 + 1024;  // barriers, abort flag, alignment
static_assert(kSmemBar >= kWarps * kFewRows * (128 + 2) * 4, "the warps' results reuse the ring");

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// D += A (16 x 16, row) * B (16 x 8, col), bf16 with fp32 accumulation
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit values spread over the warp (lane: row lane / 4, columns 2 (lane % 4), + 1).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 16-byte chunk `c` of row `r` of a stage, as the TMA's 128-byte swizzle places it.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Place of four dims in a block's row of results: the lanes of a quarter warp store to different banks.
__device__ __forceinline__ int result_chunk(int query, int c4) { return c4 ^ ((query >> 1) & 3); }

constexpr int kQueryExp = 110;   // queries enter the product as q * 2^kQueryExp
constexpr int kScoreExp = 20;    // scores are kept in units of 2^kScoreExp, so that fp32 holds the factor of every K exponent
constexpr float kScoreUnit = 1 << kScoreExp;
constexpr int kWeightExp = 120;  // weights enter the product as p * 2^(e - R + kWeightExp)

// kN: eights of query rows
template <int kN>
__global__ void __launch_bounds__(kWarps * 32, kFewBlocksPerSm)
attn_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ AttnXParams p) {
  constexpr int kRows = 8 * kN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base_addr = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_addr - raw);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemBar + kWarps * kStages * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = base_addr + warp * kStages * kStageBytes;
  const uint32_t bars = base_addr + kSmemBar + warp * kStages * 8;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (lane == 0) {  // a warp's barriers are its own
    for (int i = 0; i < kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  const Item item = attnx::find_item_lens(p, blockIdx.x);
  const int b = item.b, h = item.h, q0 = item.tile * kRows;
  const int n_all = (item.len + 127) / 128;
  const int key0 = (item.part < 0 ? 0 : static_cast<int>(static_cast<int64_t>(item.part) * n_all / item.parts)) * 128;
  const int key1 = min(item.len, (item.part < 0 ? n_all
                                                : static_cast<int>(static_cast<int64_t>(item.part + 1) * n_all / item.parts)) * 128);
  constexpr int kStride = kWarps * kKeys;
  const int first0 = key0 + warp * kKeys;
  static_assert(kKeys == 32, "a lane has the exponents of one key");
  const int8_t* keb = static_cast<const int8_t*>(p.k_exp.ptr) + b * p.k_exp.stride_row + h * p.k_exp.stride_head;
  const int8_t* veb = static_cast<const int8_t*>(p.v_exp.ptr) + b * p.v_exp.stride_row + h * p.v_exp.stride_head;
  int exp_k = 0, exp_v = 0, next_k = 0, next_v = 0;  // of this lane's key in this stage and in the next
  auto load = [&](int stage, int first) {
    if (first >= key1) return;
    if (lane == 0) {
      const uint32_t dst = ring + stage * kStageBytes, bar = bars + 8 * stage;
      mbar_expect_tx(bar, kStageBytes);
      tma_load_4d(dst, &tm_k, bar, 0, h, first, b & p.k_row_mask);
      tma_load_4d(dst + kKeys * 128, &tm_v, bar, 0, h, first, b & p.v_row_mask);
    }
    const int64_t key = min(first + lane, key1 - 1);
    next_k = keb[key * p.k_exp.stride_tok];
    next_v = veb[key * p.v_exp.stride_tok];
  };
  begin_after_previous_kernel();
  load(0, first0);

  // query fragments: k-step hf * 4 + w holds dims hf * 64 + t4 * 16 + w * 4 + {0, 1} and {2, 3} of query g
  uint32_t qb[kN][8][2];
#pragma unroll
  for (int nb = 0; nb < kN; ++nb) {
    const int row = q0 + nb * 8 + g;
    const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(p.q.ptr) + b * p.q.stride_row +
                              static_cast<int64_t>(row) * p.q.stride_tok + h * p.q.stride_head + t4 * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row < p.q_tokens) v = *reinterpret_cast<const uint4*>(qp + (i >> 1) * 64 + (i & 1) * 8);
      qb[nb][2 * i][0] = v.x;
      qb[nb][2 * i][1] = v.y;
      qb[nb][2 * i + 1][0] = v.z;
      qb[nb][2 * i + 1][1] = v.w;
    }
  }
  __syncthreads();  // the abort flag belongs to all warps

  // scale the queries by 2^110; a row whose largest element would pass 2^120 by less (none, with an infinity or NaN: its
  // scores are not finite either way), one whose elements all lie below 2^-17 by 2^127: only keys near the largest that
  // the format holds give it scores that matter, and at 2^110 such products would be subnormal numbers
  float row_fix[kN][2];  // of queries 2 t4, 2 t4 + 1, as all that follows
  bool plain = true;
#pragma unroll
  for (int nb = 0; nb < kN; ++nb) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __vmaxu2(top, __vmaxu2(qb[nb][i][0] & 0x7FFF7FFFu, qb[nb][i][1] & 0x7FFF7FFFu));
    top = max(top & 0xFFFFu, top >> 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int field = static_cast<int>(top >> 7);  // the exponent's
    const int qs = top != 0 && field < 127 - 17 ? 127 : min(max(246 - field, 0), kQueryExp);
    const uint32_t q2 = q8::scale_bits(qs, false);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qb[nb][i][0] = q8::mul_bf16x2(qb[nb][i][0], q2);
      qb[nb][i][1] = q8::mul_bf16x2(qb[nb][i][1], q2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) row_fix[nb][i] = attnx::exp2_int(kQueryExp - __shfl_sync(0xffffffffu, qs, 4 * (2 * t4 + i)));
    plain = plain && qs == kQueryExp;
  }
  plain = __all_sync(0xffffffffu, plain);

  float m[kN][2], l[kN][2];
  int ref_v = q8::kMinExp;  // R
  float o[kN][8][4];        // dims g * 16 + 2 j + {0, 0, 1, 1}, queries 2 t4 + {0, 1, 0, 1}
#pragma unroll
  for (int nb = 0; nb < kN; ++nb) {
    m[nb][0] = m[nb][1] = -INFINITY;
    l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
  }

  bool ok = true;
  static_assert(kStages == 2, "one stage in use, one on its way");
  int stage = 0;
  uint32_t parity = 0;
#pragma unroll 1
  for (int first = first0; first < key1; first += kStride, stage ^= 1, parity ^= stage == 0) {
    __syncwarp();  // every lane is done with the stage that the next copy overwrites
    exp_k = next_k;
    exp_v = next_v;
    load(stage ^ 1, first + kStride);
    ok = mbar_wait(bars + 8 * stage, parity, abort_flag, p.status, WAIT_KV_FULL);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {  // a wait ran out (reported): leave no copy of this warp in flight
      for (int i = 0; i < kStages && first + i * kStride < key1; ++i) {
        const long long t0 = clock64();
        while (!mbar_try_wait(bars + 8 * (stage ^ i), parity ^ (stage & i)) && clock64() - t0 < kWaitBudgetCycles) {
        }
      }
      break;
    }
    const uint32_t ks = ring + stage * kStageBytes, vs = ks + kKeys * 128;

    // S^T = K Q^T, 16 keys a block; a lane holds keys g, g + 8 of each and queries 2 t4, 2 t4 + 1 (c: with
    // one eight of queries two chains of products, their latencies side by side)
    float s[kBlocks][kN][4];
    {
      constexpr int kChains = kN == 1 ? 2 : 1;
      float c[kChains][kBlocks][kN][4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) {
#pragma unroll
          for (int nb = 0; nb < kN && hf < kChains; ++nb)
            c[hf][kb][nb][0] = c[hf][kb][nb][1] = c[hf][kb][nb][2] = c[hf][kb][nb][3] = 0.f;
          const uint4 lo = ld_shared_v4(ks + chunk_at(kb * 16 + g, hf * 4 + t4));
          const uint4 hi = ld_shared_v4(ks + chunk_at(kb * 16 + g + 8, hf * 4 + t4));
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a[4];
            q8::spread4(word(lo, w), a[0], a[2]);
            q8::spread4(word(hi, w), a[1], a[3]);
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) mma(c[hf % kChains][kb][nb], a, qb[nb][hf * 4 + w][0], qb[nb][hf * 4 + w][1]);
          }
        }
#pragma unroll
      for (int i = 0; i < kBlocks * kN * 4; ++i)
        s[i / (4 * kN)][i / 4 % kN][i % 4] =
            c[0][i / (4 * kN)][i / 4 % kN][i % 4] + (kChains == 2 ? c[kChains - 1][i / (4 * kN)][i / 4 % kN][i % 4] : 0.f);
    }
    // this lane's key: its exponents as factors of a score and of a weight, and R
    const int left = key1 - first;
    const int ref_new = max(ref_v, __reduce_max_sync(0xffffffffu, exp_v));
    float fk = fmaxf(attnx::exp2_int(exp_k + 133 - kQueryExp - kScoreExp) * p.scale_log2, 1.17549435e-38f);
    float fv = attnx::exp2_int(exp_v - ref_new + kWeightExp);
    if (exp_k == q8::kNotFinite) fk = NAN;
    if (exp_v == q8::kNotFinite) fv = NAN;
    if (lane >= left) fv = 0.f;
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = __shfl_sync(0xffffffffu, fk, kb * 16 + i * 8 + g);
#pragma unroll
        for (int nb = 0; nb < kN; ++nb) {
          s[kb][nb][2 * i] *= f;
          s[kb][nb][2 * i + 1] *= f;
        }
      }
    if (!plain) {
#pragma unroll
      for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
        for (int nb = 0; nb < kN; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kb][nb][i] *= row_fix[nb][i & 1];
    }
    if (left < kKeys) {
#pragma unroll
      for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kb * 16 + (i >> 1) * 8 + g >= left) {
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) s[kb][nb][i] = -INFINITY;
          }
    }
    float mx[kN][2];
    bool grow = ref_new != ref_v;
#pragma unroll
    for (int nb = 0; nb < kN; ++nb)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(s[0][nb][i], s[0][nb][2 + i]);
#pragma unroll
        for (int kb = 1; kb < kBlocks; ++kb) x = fmaxf(x, fmaxf(s[kb][nb][i], s[kb][nb][2 + i]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
        x *= kScoreUnit;
        mx[nb][i] = x;
        grow = grow || x > m[nb][i];
      }
    if (__any_sync(0xffffffffu, grow)) {
      const float shift = attnx::exp2_int(ref_v - ref_new);
      ref_v = ref_new;
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float m_new = fmaxf(m[nb][i], mx[nb][i]);
          const float alpha = m_new == m[nb][i] ? 1.f : ex2_approx(m[nb][i] - m_new);
          m[nb][i] = m_new;
          l[nb][i] *= alpha;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[nb][j][i] *= alpha * shift;
            o[nb][j][2 + i] *= alpha * shift;
          }
        }
    }
    uint32_t pb[kBlocks][kN][2];
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = __shfl_sync(0xffffffffu, fv, kb * 16 + i * 8 + g);
#pragma unroll
        for (int nb = 0; nb < kN; ++nb) {
          float w[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            w[q] = ex2_approx(fmaf(s[kb][nb][2 * i + q], kScoreUnit, m[nb][q] == -INFINITY ? 0.f : -m[nb][q]));
            l[nb][q] += w[q];
          }
          // bf16 as in the tensor-core kernels: 2^-9 of the output, as much as its own rounding
          pb[kb][nb][i] = transpose8(pack_bf16x2(w[0] * f, w[1] * f));  // now of query g, keys 2 t4, 2 t4 + 1
        }
      }
    // O^T += V^T P^T, 16 keys a step: row g of the dims' block j is dim g * 16 + 2 j, row g + 8 the dim after it
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = ld_shared_v4(vs + chunk_at(kb * 16 + 2 * t4 + (i & 1) + (i >> 1) * 8, g));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t a[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t sel = 0x4400u + 0x1111u * (2 * (j & 1) + i);  // that byte of the first key doubled, of the second
          a[i] = __byte_perm(word(v[0], j >> 1), word(v[1], j >> 1), sel) & 0x807F807Fu;
          a[2 + i] = __byte_perm(word(v[2], j >> 1), word(v[3], j >> 1), sel) & 0x807F807Fu;
        }
#pragma unroll
        for (int nb = 0; nb < kN; ++nb) mma(o[nb][j], a, pb[kb][nb][0], pb[kb][nb][1]);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) return;

  // merge the warps: results to shared memory (the ring is free now), then a thread per dim
  float* so = reinterpret_cast<float*>(smem);    // [warp][row][128]
  float* sm = so + kWarps * kRows * 128;         // [warp][2][row]
  // every result is divided by its own sum before it leaves its unit 2^(R + 13): so it is a mean of V and stays finite
  const float unit = attnx::exp2_int(ref_v + 6);
#pragma unroll
  for (int nb = 0; nb < kN; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int query = nb * 8 + 2 * t4 + i;
      float sum = l[nb][i];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float inv = sum == 0.f ? 0.f : exp2f(133 - 6 - kWeightExp) / sum;
      float* dst = so + (warp * kRows + query) * 128;
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        *reinterpret_cast<float4*>(dst + 4 * result_chunk(query, g * 4 + (j >> 1))) =
            make_float4(o[nb][j][i] * inv * unit, o[nb][j][2 + i] * inv * unit, o[nb][j + 1][i] * inv * unit,
                        o[nb][j + 1][2 + i] * inv * unit);
      if (g == 0) {
        sm[(warp * 2) * kRows + query] = m[nb][i];
        sm[(warp * 2 + 1) * kRows + query] = sum;
      }
    }
  __syncthreads();
  const int dim = threadIdx.x;
  const int rows = min(kRows, p.q_tokens - q0);
#pragma unroll 2
  for (int row = 0; row < rows; ++row) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w * 2 * kRows + row]);
    const float m_sub = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, weight[kWarps];  // shares of the sum, so that the merged mean stays finite as well
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float lw = sm[(w * 2 + 1) * kRows + row];
      weight[w] = lw == 0.f ? 0.f : ex2_approx(sm[w * 2 * kRows + row] - m_sub) * lw;
      ll += weight[w];
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    const int at = 4 * result_chunk(row, dim >> 2) + (dim & 3);
    float acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) acc += weight[w] * inv * so[(w * kRows + row) * 128 + at];
    if (item.part < 0) {
      static_cast<__nv_bfloat16*>(p.out)[b * p.out_stride_row + static_cast<int64_t>(q0 + row) * p.out_stride_tok +
                                         h * p.out_stride_head + dim] = __float2bfloat16_rn(acc);
    } else {
      p.part_o[(static_cast<size_t>(item.slot) * kFewRows + row) * 128 + dim] = acc;
      if (dim == 0) {
        p.part_meta[(static_cast<size_t>(item.slot) * 2) * kFewRows + row] = mm;
        p.part_meta[(static_cast<size_t>(item.slot) * 2 + 1) * kFewRows + row] = ll;
      }
    }
  }
}

// Merge the parts of a split tile: block = (tile, query row), 256 threads = 8 groups of parts x 32 groups of 4 dims.  What
// it waits for is the latency of its loads, so those of the first 64 parts are all made before any is used.
__global__ void __launch_bounds__(256) combine_few_kernel(const __grid_constant__ AttnXParams p) {
  constexpr int kAhead = 8, kFirst = 8 * kAhead;
  __shared__ float4 part_acc[8][32];
  const int row = blockIdx.y, lane = threadIdx.x & 31, c0 = lane * 4, grp = threadIdx.x >> 5;
  const Item item = attnx::find_item_lens(p, attnx::first_item_lens(p, blockIdx.x));
  const int q_row = item.tile * p.few_rows + row;
  begin_after_previous_kernel();  // the parts are complete
  if (item.part < 0 || q_row >= p.q_tokens) return;
  const float* pm = p.part_meta + static_cast<size_t>(item.slot) * 2 * kFewRows + row;
  const float* po = p.part_o + (static_cast<size_t>(item.slot) * kFewRows + row) * 128 + c0;
  constexpr int kStepM = 2 * kFewRows, kStepO = kFewRows * 128;
  float mk[2], lk[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int k = lane + 32 * i;
    mk[i] = k < item.parts ? pm[k * kStepM] : -INFINITY;
    lk[i] = k < item.parts ? pm[k * kStepM + kFewRows] : 0.f;
  }
  float4 a[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int k = grp + 8 * i;
    a[i] = k < item.parts ? *reinterpret_cast<const float4*>(po + static_cast<size_t>(k) * kStepO) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float m = fmaxf(mk[0], mk[1]);
  for (int k = kFirst + lane; k < item.parts; k += 32) m = fmaxf(m, pm[k * kStepM]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  const float m_sub = m == -INFINITY ? 0.f : m;
  float wk[2], l = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    wk[i] = lk[i] == 0.f ? 0.f : ex2_approx(mk[i] - m_sub) * lk[i];
    l += wk[i];
  }
  for (int k = kFirst + lane; k < item.parts; k += 32) l += ex2_approx(pm[k * kStepM] - m_sub) * pm[k * kStepM + kFewRows];
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const float f = __shfl_sync(0xffffffffu, wk[i / 4], grp + 8 * (i % 4)) * inv;
    acc.x += f * a[i].x; acc.y += f * a[i].y; acc.z += f * a[i].z; acc.w += f * a[i].w;
  }
#pragma unroll 4
  for (int k = kFirst + grp; k < item.parts; k += 8) {
    const float4 x = *reinterpret_cast<const float4*>(po + static_cast<size_t>(k) * kStepO);
    const float f = ex2_approx(pm[k * kStepM] - m_sub) * pm[k * kStepM + kFewRows] * inv;
    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
  }
  part_acc[grp][lane] = acc;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    const float4 x = part_acc[k][lane];
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  }
  __nv_bfloat16* op = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(item.b) * p.out_stride_row +
                      static_cast<int64_t>(q_row) * p.out_stride_tok + static_cast<int64_t>(item.h) * p.out_stride_head + c0;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
}

template <int kN>
cudaError_t launch(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttnXParams& p, cudaStream_t stream) {
  static DynamicSmemGrant smem_grant;  // one per instantiation
  DeviceInfo di;
  cudaError_t e = device_info(&di);
  if (e == cudaSuccess) e = smem_grant.ensure(attn_few_kernel<kN>, kSmemBytes, di.device);
  if (e != cudaSuccess) return e;
  e = launch_chained(attn_few_kernel<kN>, dim3(p.n_full + p.n_parts), dim3(kWarps * 32), kSmemBytes, stream, tm_k, tm_v, p);
  if (e != cudaSuccess || p.split == 1) return e;
  return launch_chained(combine_few_kernel, dim3(p.n_tiles - p.n_full, min(p.q_tokens, p.few_rows)), dim3(256), 0, stream, p);
}

}  // namespace few

cudaError_t launch_attn_few(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttnXParams& p, cudaStream_t stream) {
  return p.few_rows == 8 ? few::launch<1>(tm_k, tm_v, p, stream) : few::launch<2>(tm_k, tm_v, p, stream);
}

// Splitting along the keys.  With `wave` CTAs on the GPU at a time, n_tiles = waves * wave + tail leaves only `tail` of
// those places busy at the end (all of them, when there are few tiles).  Rows are taken longest first, and the tail's tiles
// are cut into parts of about c tiles of 128 keys, c the smallest for which the parts fit the places: short items
// share one as far as they end with the others (an item costs `setup` key tiles beside its own).  A part costs its set-up
// and a pass over its accumulator, so c stays at min_tiles or more.  Rows so long that a tile of theirs would outlast all
// else (twice a place's share) belong to the tail whole: one row of 32760 keys among fifteen of 100 x 40 heads would
// keep 40 places busy and leave 400 idle (one token: 234 us, cut up 67).
int plan_lens(AttnXParams& p, int wave, int min_tiles, int setup) {
  const int per_row = p.pair_tiles * p.heads;
  int n_kv[SDV2_MAX_ROWS], first[SDV2_MAX_ROWS];
  for (int r = 1; r < p.rows; ++r) {  // insertion sort, longest row first
    const AttnXParams::Row x = p.by_length[r];
    int at = r;
    for (; at > 0 && p.by_length[at - 1].len < x.len; --at) p.by_length[at] = p.by_length[at - 1];
    p.by_length[at] = x;
  }
  const int64_t n_tiles = static_cast<int64_t>(per_row) * p.rows;
  if (n_tiles > 0x7FFFFFFFLL / 64) return -1;
  p.n_tiles = static_cast<int>(n_tiles);
  int n_long = 0;
  if (p.n_tiles >= wave) {
    int64_t work = 0;
    for (int r = 0; r < p.rows; ++r) work += static_cast<int64_t>(per_row) * ((p.by_length[r].len + 127) / 128);
    while (n_long < p.rows && (p.by_length[n_long].len + 127) / 128 > max(2 * work / wave, static_cast<int64_t>(min_tiles))) ++n_long;
    std::rotate(p.by_length, p.by_length + n_long, p.by_length + p.rows);
  }
  const int n_other = p.n_tiles - n_long * per_row;
  p.n_full = n_other - n_other % wave;
  int longest = 0;
  for (int r = 0; r < p.rows; ++r) {
    n_kv[r] = (p.by_length[r].len + 127) / 128;
    first[r] = max(r * per_row, p.n_full);
    if ((r + 1) * per_row > p.n_full) longest = max(longest, n_kv[r]);
  }
  auto parts_at = [&](int c, int r) { return n_kv[r] <= c ? 1 : (n_kv[r] + c - 1) / c; };
  auto places_at = [&](int c) {
    double n = 0.;
    for (int r = 0; r < p.rows; ++r) {
      const int parts = parts_at(c, r);
      n += static_cast<double>(max((r + 1) * per_row - first[r], 0)) * parts / ((c + setup) / ((n_kv[r] + parts - 1) / parts + setup));
    }
    return n;
  };
  int lo = min_tiles, hi = max(longest, min_tiles);  // the smallest c in [lo, hi] whose parts fit, else hi
  while (lo < hi) {
    const int c = (lo + hi) / 2;
    if (places_at(c) <= wave) hi = c;
    else lo = c + 1;
  }
  p.split = 1;
  int item = 0;
  for (int r = 0; r < p.rows; ++r) {
    const int parts = parts_at(lo, r);
    p.by_length[r].tail_tile0 = first[r];
    p.by_length[r].item0 = item;
    p.by_length[r].parts = parts;
    const int tiles = max((r + 1) * per_row - first[r], 0);
    if (tiles > 0) p.split = max(p.split, parts);
    item += tiles * parts;
  }
  p.n_parts = item;
  return p.split > 1 ? p.n_parts : 0;
}

}  // namespace sdv2
