// Attention of a few queries over the 8-bit cache: up to 16 query rows to a block, bound by reading the cache once.
//
// A block's four warps take 32 keys each in turn.  A warp has the bytes of its keys' K and V copied into its own ring of
// shared-memory stages (TMA, the next stage in flight) and works on them with m16n8k16 bf16 products, the 16 query rows as M:
// the tcgen05 kernel's 128 rows would be empty, and its tiles would have to pass through shared memory as bf16, four
// times these bytes.  A fragment's order of dims and keys is free as long as both operands agree on it, so a lane loads
// 16 consecutive bytes of a key and expands them in registers: for K the four dims of a word become one k-step's pair
// of registers, for V the same byte of two keys becomes one register (one permute takes both, one mask follows).
//
// The products take the values as they come out of that, bf16 subnormals +-m * 2^-133, without a multiplication: the
// queries are scaled up by a power of two beforehand (2^qs, as far as their largest element allows), the weights by
// 2^(120 - R) with R the largest V exponent so far; a key's own powers of two join its score and its weight.  All of it
// is exact.  The running maximum is exact too (weights stay at most 1 and weight * 2^(e - R + 120) below 2^121); the
// accumulator is rescaled when it or R moves.  The warps' results merge in shared memory, the parts of a split row in
// combine_few_kernel.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "attn_items.cuh"
#include "ptx.cuh"
#include "q8.cuh"
#include "sdv2_internal.h"

namespace sdv2 {
namespace few {

using attnx::Item;

constexpr int kRows = kFewRows;       // query rows of a block
constexpr int kWarps = 4;
constexpr int kKeys = kFewStageKeys;  // keys of a stage
constexpr int kBlocks = kKeys / 8;    // ... in products of eight
constexpr int kStages = 2;
constexpr int kStageBytes = kKeys * 128 * 2;
constexpr int kSmemBar = kWarps * kStages * kStageBytes;
constexpr int kSmemBytes = kSmemBar + kWarps * kStages * 8 + 16 + 1024;  // barriers, abort flag, alignment
static_assert(kSmemBar >= kWarps * kRows * (128 + 2) * 4, "the warps' results reuse the ring");

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

// 16-byte chunk `c` of row `r` of a stage, as the TMA's 128-byte swizzle places it.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

constexpr int kQueryExp = 110;   // queries enter the product as q * 2^kQueryExp
constexpr int kWeightExp = 120;  // weights enter the product as p * 2^(e - R + kWeightExp)

__global__ void __launch_bounds__(kWarps * 32, kFewBlocksPerSm)
attn_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ AttnXParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base_addr = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_addr - raw);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemBar + kWarps * kStages * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = base_addr + warp * kStages * kStageBytes;
  const uint32_t bars = base_addr + kSmemBar + warp * kStages * 8;
  if (lane == 0) {
    *abort_flag = 0;
    for (int i = 0; i < kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncthreads();  // the abort flag belongs to all warps
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merging kernel may be set up meanwhile
  const Item item = attnx::find_item_lens(p, blockIdx.x);
  const int b = item.b, h = item.h, q0 = item.tile * kRows;
  const int len = p.seq_lens[b];
  const int n_all = (len + 127) / 128;
  const int key0 = (item.part < 0 ? 0 : static_cast<int>(static_cast<int64_t>(item.part) * n_all / item.parts)) * 128;
  const int key1 = min(len, (item.part < 0 ? n_all
                                           : static_cast<int>(static_cast<int64_t>(item.part + 1) * n_all / item.parts)) * 128);
  constexpr int kStride = kWarps * kKeys;
  const int first0 = key0 + warp * kKeys;
  static_assert(kKeys == 32, "a lane has the exponents of one key");
  const int8_t* keb = static_cast<const int8_t*>(p.k_exp.ptr) + b * p.k_exp.stride_row + h * p.k_exp.stride_head;
  const int8_t* veb = static_cast<const int8_t*>(p.v_exp.ptr) + b * p.v_exp.stride_row + h * p.v_exp.stride_head;
  int exp_k[kStages], exp_v[kStages];
  auto load = [&](int stage, int first) {
    if (first >= key1) return;
    if (lane == 0) {
      const uint32_t dst = ring + stage * kStageBytes, bar = bars + 8 * stage;
      mbar_expect_tx(bar, kStageBytes);
      tma_load_4d(dst, &tm_k, bar, 0, h, first, b & p.k_row_mask);
      tma_load_4d(dst + kKeys * 128, &tm_v, bar, 0, h, first, b & p.v_row_mask);
    }
    const int64_t key = min(first + lane, key1 - 1);
    exp_k[stage] = keb[key * p.k_exp.stride_tok];
    exp_v[stage] = veb[key * p.v_exp.stride_tok];
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i, first0 + i * kStride);

  // query fragments: k-step s of half hf holds dims hf * 64 + t4 * 16 + s * 4 + {0, 1} and {2, 3}
  uint32_t qa[8][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = q0 + g + 8 * i;
    const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(p.q.ptr) + b * p.q.stride_row +
                              static_cast<int64_t>(row) * p.q.stride_tok + h * p.q.stride_head + t4 * 16;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int half16 = 0; half16 < 2; ++half16) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < p.q_tokens) v = __ldg(reinterpret_cast<const uint4*>(qp + hf * 64 + half16 * 8));
        qa[hf * 4 + half16 * 2][i] = v.x;
        qa[hf * 4 + half16 * 2][i + 2] = v.y;
        qa[hf * 4 + half16 * 2 + 1][i] = v.z;
        qa[hf * 4 + half16 * 2 + 1][i + 2] = v.w;
      }
  }

  // scale the queries by 2^110, a row whose largest finite element would pass 2^120 by less
  float row_fix[2];
  bool plain = true;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    uint32_t top = 0;  // exponent field
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = r; j < 4; j += 2)
#pragma unroll
        for (int k = 7; k < 32; k += 16) {
          const uint32_t e = (qa[i][j] >> k) & 0xFFu;
          if (e != 255u) top = max(top, e);
        }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int qs = min(max(246 - static_cast<int>(top), 0), kQueryExp);
    const uint32_t q2 = q8::scale_bits(qs, false);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = r; j < 4; j += 2) qa[i][j] = q8::mul_bf16x2(qa[i][j], q2);
    row_fix[r] = attnx::exp2_int(kQueryExp - qs);
    plain = plain && qs == kQueryExp;
  }
  plain = __all_sync(0xffffffffu, plain);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int ref_v = q8::kMinExp;  // R
  float o[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;

  bool ok = true;
  uint32_t parity = 0;
  for (int base = first0; base < key1 && ok; base += kStages * kStride, parity ^= 1) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      const int first = base + st * kStride;
      if (first >= key1) break;  // warp-uniform
      __syncwarp();              // every lane is done with the stage that the next copy overwrites
      load((st + kStages - 1) % kStages, first + (kStages - 1) * kStride);
      ok = mbar_wait(bars + 8 * st, parity, abort_flag, p.status, WAIT_KV_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {  // a wait ran out (reported): leave no copy of this warp in flight
        for (int i = 0; i < kStages && first + i * kStride < key1; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(bars + 8 * ((st + i) % kStages), st + i < kStages ? parity : parity ^ 1) &&
                 clock64() - t0 < kWaitBudgetCycles) {
          }
        }
        break;
      }
      const uint32_t ks = ring + st * kStageBytes, vs = ks + kKeys * 128;

      // S = Q K^T, eight keys a block; a lane holds keys 2 t4, 2 t4 + 1 of each
      float s[kBlocks][4];
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint4 kv[kBlocks];
#pragma unroll
        for (int nb = 0; nb < kBlocks; ++nb) kv[nb] = ld_shared_v4(ks + chunk_at(nb * 8 + g, hf * 4 + t4));
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int nb = 0; nb < kBlocks; ++nb) {
            uint32_t lo, hi;
            q8::spread4(word(kv[nb], w), lo, hi);
            mma(s[nb], qa[hf * 4 + w], lo, hi);
          }
      }
      // this lane's key: its exponents as factors of a score and of a weight, and R
      const int left = key1 - first;
      const int ref_new = max(ref_v, __reduce_max_sync(0xffffffffu, exp_v[st]));
      float fk = fmaxf(attnx::exp2_int(exp_k[st] + 133 - kQueryExp) * p.scale_log2, 1.17549435e-38f);
      float fv = attnx::exp2_int(exp_v[st] - ref_new + kWeightExp);
      if (exp_k[st] == q8::kNotFinite) fk = NAN;
      if (exp_v[st] == q8::kNotFinite) fv = NAN;
      if (lane >= left) fv = 0.f;
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float f = __shfl_sync(0xffffffffu, fk, nb * 8 + 2 * t4 + i);
          s[nb][i] *= f;
          s[nb][2 + i] *= f;
        }
      if (!plain) {
#pragma unroll
        for (int i = 0; i < 4 * kBlocks; ++i) s[i >> 2][i & 3] *= row_fix[(i >> 1) & 1];
      }
      if (left < kKeys) {
#pragma unroll
        for (int i = 0; i < 2 * kBlocks; ++i)
          if ((i >> 1) * 8 + 2 * t4 + (i & 1) >= left) s[i >> 1][i & 1] = s[i >> 1][2 + (i & 1)] = -INFINITY;
      }
      float mx[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
        for (int nb = 1; nb < kBlocks; ++nb) mx[r] = fmaxf(mx[r], fmaxf(s[nb][2 * r], s[nb][2 * r + 1]));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1] || ref_new != ref_v)) {
        const float shift = attnx::exp2_int(ref_v - ref_new);
        ref_v = ref_new;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float m_new = fmaxf(m[r], mx[r]);
          const float alpha = m_new == m[r] ? 1.f : ex2_approx(m[r] - m_new);
          m[r] = m_new;
          l[r] *= alpha;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            o[j][2 * r] *= alpha * shift;
            o[j][2 * r + 1] *= alpha * shift;
          }
        }
      }
      uint32_t pa[kBlocks / 2][4];
      const float m_sub[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
        const float f0 = __shfl_sync(0xffffffffu, fv, nb * 8 + 2 * t4), f1 = __shfl_sync(0xffffffffu, fv, nb * 8 + 2 * t4 + 1);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p0 = ex2_approx(s[nb][2 * r] - m_sub[r]), p1 = ex2_approx(s[nb][2 * r + 1] - m_sub[r]);
          l[r] += p0 + p1;
          pa[nb >> 1][(nb & 1) * 2 + r] = pack_bf16x2(p0 * f0, p1 * f1);
        }
      }
      // O += P V, 16 keys a step: this lane's column of every block of eight dims is dim g * 16 + block, its keys are the
      // four above
#pragma unroll
      for (int kk = 0; kk < kBlocks / 2; ++kk) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = ld_shared_v4(vs + chunk_at(kk * 16 + 2 * t4 + (i & 1) + (i >> 1) * 8, g));
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const uint32_t sel = 0x4400u + 0x1111u * d;  // byte d of the first key doubled, of the second doubled
            mma(o[w * 4 + d], pa[kk], __byte_perm(word(v[0], w), word(v[1], w), sel) & 0x807F807Fu,
                __byte_perm(word(v[2], w), word(v[3], w), sel) & 0x807F807Fu);
          }
      }
    }
  }
  __syncthreads();
  if (*abort_flag) return;

  // merge the warps: results to shared memory (the ring is free now), then 128 threads = 16 rows x 8 groups of 16 dims
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  float* so = reinterpret_cast<float*>(smem);                    // [warp][row][128]
  float* sm = so + kWarps * kRows * 128;                         // [warp][2][row]
  // every result is divided by its own sum before it leaves its unit 2^(R + 13): so it is a mean of V and stays finite
  const float unit = attnx::exp2_int(ref_v + 6);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = g + 8 * r;
    const float inv = l[r] == 0.f ? 0.f : exp2f(133 - 6 - kWeightExp) / l[r];
    // column j of a lane's block is dim n * 16 + j for the accumulator's columns n = 2 t4, 2 t4 + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float* dst = so + (warp * kRows + row) * 128 + (2 * t4 + c) * 16;
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<float4*>(dst + j) =
            make_float4(o[j][2 * r + c] * inv * unit, o[j + 1][2 * r + c] * inv * unit, o[j + 2][2 * r + c] * inv * unit,
                        o[j + 3][2 * r + c] * inv * unit);
    }
    if (t4 == 0) {
      sm[(warp * 2) * kRows + row] = m[r];
      sm[(warp * 2 + 1) * kRows + row] = l[r];
    }
  }
  __syncthreads();
  const int row = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 16;
  if (q0 + row >= p.q_tokens) return;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w * 2 * kRows + row]);
  const float m_sub = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, weight[kWarps], acc[16];  // shares of the sum, so that the merged mean stays finite as well
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float lw = sm[(w * 2 + 1) * kRows + row];
    weight[w] = lw == 0.f ? 0.f : exp2f(sm[w * 2 * kRows + row] - m_sub) * lw;
    ll += weight[w];
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] += weight[w] * inv * so[(w * kRows + row) * 128 + c0 + j];
  if (item.part < 0) {
    __nv_bfloat16* op = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(b) * p.out_stride_row +
                        static_cast<int64_t>(q0 + row) * p.out_stride_tok + static_cast<int64_t>(h) * p.out_stride_head + c0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<uint4*>(op + 8 * i) =
          make_uint4(pack_bf16x2(acc[8 * i], acc[8 * i + 1]), pack_bf16x2(acc[8 * i + 2], acc[8 * i + 3]),
                     pack_bf16x2(acc[8 * i + 4], acc[8 * i + 5]), pack_bf16x2(acc[8 * i + 6], acc[8 * i + 7]));
  } else {
    float* po = p.part_o + (static_cast<size_t>(item.slot) * kRows + row) * 128 + c0;
#pragma unroll
    for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(po + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    if (c0 == 0) {
      p.part_meta[(static_cast<size_t>(item.slot) * 2) * kRows + row] = mm;
      p.part_meta[(static_cast<size_t>(item.slot) * 2 + 1) * kRows + row] = ll;
    }
  }
}

// Merge the parts of a split tile: block = (tile, query row), 256 threads = 8 groups of parts x 32 groups of 4 dims.
__global__ void __launch_bounds__(256) combine_few_kernel(const __grid_constant__ AttnXParams p) {
  __shared__ float4 part_acc[8][32];
  const int row = blockIdx.y, c0 = (threadIdx.x & 31) * 4, grp = threadIdx.x >> 5;
  const Item item = attnx::find_item_lens(p, attnx::first_item_lens(p, blockIdx.x));
  const int q_row = item.tile * kRows + row;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are complete
  if (item.part < 0 || q_row >= p.q_tokens) return;
  const float* pm = p.part_meta + static_cast<size_t>(item.slot) * 2 * kRows + row;
  const float* po = p.part_o + (static_cast<size_t>(item.slot) * kRows + row) * 128 + c0;
  float m = -INFINITY;
  for (int k = threadIdx.x & 31; k < item.parts; k += 32) m = fmaxf(m, pm[k * 2 * kRows]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  const float m_sub = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int k = threadIdx.x & 31; k < item.parts; k += 32) l += exp2f(pm[k * 2 * kRows] - m_sub) * pm[k * 2 * kRows + kRows];
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = grp; k < item.parts; k += 8) {
    const float4 a = *reinterpret_cast<const float4*>(po + static_cast<size_t>(k) * kRows * 128);
    const float f = exp2f(pm[k * 2 * kRows] - m_sub) * pm[k * 2 * kRows + kRows] * inv;
    acc.x += f * a.x; acc.y += f * a.y; acc.z += f * a.z; acc.w += f * a.w;
  }
  part_acc[grp][threadIdx.x & 31] = acc;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    const float4 a = part_acc[k][threadIdx.x];
    acc.x += a.x; acc.y += a.y; acc.z += a.z; acc.w += a.w;
  }
  __nv_bfloat16* op = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(item.b) * p.out_stride_row +
                      static_cast<int64_t>(q_row) * p.out_stride_tok + static_cast<int64_t>(item.h) * p.out_stride_head + c0;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
}

}  // namespace few

cudaError_t launch_attn_few(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttnXParams& p, cudaStream_t stream) {
  static DynamicSmemGrant smem_grant;
  DeviceInfo di;
  cudaError_t e = device_info(&di);
  if (e == cudaSuccess) e = smem_grant.ensure(few::attn_few_kernel, few::kSmemBytes, di.device);
  if (e != cudaSuccess) return e;
  few::attn_few_kernel<<<p.n_full + p.n_parts, few::kWarps * 32, few::kSmemBytes, stream>>>(tm_k, tm_v, p);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.split == 1) return e;
  return launch_dependent(few::combine_few_kernel, dim3(p.n_tiles - p.n_full, min(p.q_tokens, kFewRows)), dim3(256), stream, p);
}

// Splitting along the keys.  With `wave` CTAs on the GPU at a time, n_tiles = waves * wave + tail leaves only `tail` of
// those places busy at the end (all of them, when there are few tiles).  The tail's tiles - those of the shortest rows,
// rows are taken longest first - are cut into parts of about c tiles of 128 keys, c the smallest for which the parts
// still fit one wave.  A part costs its set-up and a pass over its accumulator, so c stays at min_tiles or more.
int plan_lens(AttnXParams& p, int wave, int min_tiles) {
  const int per_row = p.pair_tiles * p.heads;
  int n_kv[SDV2_MAX_ROWS], first[SDV2_MAX_ROWS];
  for (int r = 0; r < p.rows; ++r) {  // insertion sort, longest row first
    int at = r;
    while (at > 0 && p.seq_lens[p.order[at - 1]] < p.seq_lens[r]) {
      p.order[at] = p.order[at - 1];
      --at;
    }
    p.order[at] = r;
  }
  const int64_t n_tiles = static_cast<int64_t>(per_row) * p.rows;
  if (n_tiles > 0x7FFFFFFFLL / 64) return -1;
  p.n_tiles = static_cast<int>(n_tiles);
  p.n_full = p.n_tiles - p.n_tiles % wave;
  int longest = 0;
  for (int r = 0; r < p.rows; ++r) {
    n_kv[r] = (p.seq_lens[p.order[r]] + 127) / 128;
    first[r] = max(r * per_row, p.n_full);
    if ((r + 1) * per_row > p.n_full) longest = max(longest, n_kv[r]);
  }
  auto parts_at = [&](int c, int r) { return n_kv[r] <= c ? 1 : (n_kv[r] + c - 1) / c; };
  auto items_at = [&](int c) {
    int64_t n = 0;
    for (int r = 0; r < p.rows; ++r) n += static_cast<int64_t>(max((r + 1) * per_row - first[r], 0)) * parts_at(c, r);
    return n;
  };
  int lo = min_tiles, hi = max(longest, min_tiles);  // the smallest c in [lo, hi] whose parts fit; hi always does
  while (lo < hi) {
    const int c = (lo + hi) / 2;
    if (items_at(c) <= wave) hi = c;
    else lo = c + 1;
  }
  p.split = 1;
  int item = 0;
  for (int r = 0; r < p.rows; ++r) {
    p.tail_tile0[r] = first[r];
    p.item0[r] = item;
    p.parts[r] = parts_at(lo, r);
    const int tiles = max((r + 1) * per_row - first[r], 0);
    if (tiles > 0) p.split = max(p.split, p.parts[r]);
    item += tiles * p.parts[r];
  }
  p.n_parts = item;
  return p.split > 1 ? p.n_parts : 0;
}

}  // namespace sdv2
