// Tile shapes and the two tensor-core contractions that the attention kernels share.
#pragma once
#include <stdint.h>

#include "ptx.cuh"

namespace sdv2 {
namespace attn {

constexpr int kBM = 128;   // query rows per tile
constexpr int kBN = 128;   // kv rows per tile
constexpr int kHD = 128;   // head dim
constexpr uint32_t kTileBytes = kBN * kHD * 2;
constexpr uint32_t kHalfTile = kTileBytes / 2;  // one 64-column box

constexpr uint32_t kIdescQK = umma_idesc_bf16(kBM, kBN, false, false);
constexpr uint32_t kIdescPV = umma_idesc_bf16(kBM, kHD, false, true);

// S[stage] = Q[stage] (128 x 128, K-major) * K_tile^T (128 x 128, K-major); 8 steps of K = 16.
__device__ __forceinline__ void issue_qk(uint32_t tmem_s, uint32_t sq, uint32_t sk) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t off = (k >> 2) * kHalfTile + (k & 3) * 32;
    umma_ss(tmem_s, umma_smem_desc(sq + off, 16, 1024), umma_smem_desc(sk + off, 16, 1024), kIdescQK,
            k > 0 ? 1u : 0u);
  }
}
// O[stage] (+)= P[stage] (128 x 128 bf16 in TMEM, 8 columns per K step) * V_tile (kv x d, MN-major).
// k_begin..k_end select 16-key steps, so that the first half of a tile can be issued while the
// softmax warps are still producing the second half of P.
// a_from_smem (the rate measurement only): A is the K-major shared-memory tile at sa instead of P.
__device__ __forceinline__ void issue_pv(uint32_t tmem_o, uint32_t tmem_p, uint32_t sv, bool accumulate,
                                         int k_begin = 0, int k_end = 8, bool a_from_smem = false, uint32_t sa = 0) {
#pragma unroll
  for (int k = k_begin; k < k_end; ++k) {
    const uint32_t acc = (accumulate || k > k_begin) ? 1u : 0u;
    const uint64_t b_desc = umma_smem_desc(sv + k * 2048, kHalfTile, 1024);
    if (a_from_smem)
      umma_ss(tmem_o, umma_smem_desc(sa + (k >> 2) * kHalfTile + (k & 3) * 32, 16, 1024), b_desc, kIdescPV, acc);
    else
      umma_ts(tmem_o, tmem_p + k * 8, b_desc, kIdescPV, acc);
  }
}

}  // namespace attn
}  // namespace sdv2
