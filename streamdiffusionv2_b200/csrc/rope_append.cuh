// What the append kernels share: rope arithmetic, table and slot lookups, the index writes.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"
#include "sdv2_internal.h"

namespace sdv2 {

// (a + ib) * (c + id) with every product and sum rounded separately, as the reference's CPU
// complex128 multiply does; then fp64 -> fp32 (RN).  bf16 storage adds a second RNE step.
__device__ __forceinline__ void rope_pair(double a, double b, double2 cs, float& re, float& im) {
  re = __double2float_rn(__dsub_rn(__dmul_rn(a, cs.x), __dmul_rn(b, cs.y)));
  im = __double2float_rn(__dadd_rn(__dmul_rn(a, cs.y), __dmul_rn(b, cs.x)));
}

// n / d for n * d < 2^32 with m = ceil(2^32 / d), which is 0 in 32 bits for d = 1
__device__ __forceinline__ int fast_div(uint32_t n, uint32_t m) { return static_cast<int>(m == 0 ? n : __umulhi(n, m)); }

// table entry for complex column `col` of a token at (time row, grid row y, grid column x)
__device__ __forceinline__ const double2* table_place(const AppendParams& p, int col, int64_t trow, int y, int x) {
  const int64_t row = col < p.cols_t ? trow : (col < p.cols_t + p.cols_h ? y : x);
  return p.table + row * p.half + col;
}
// ... for kernels that start when everything before them has ended
__device__ __forceinline__ double2 table_entry(const AppendParams& p, int col, int64_t trow, int y, int x) {
  return __ldg(table_place(p, col, trow, y, x));
}

// Per-row slot parameters come from the launch parameters or, for launches that must not carry
// per-step values (a captured graph), from a device array the host refreshes between steps.
__device__ __forceinline__ int64_t row_start_frame(const AppendParams& p, int b) {
  return p.step_dev != nullptr ? p.step_dev[b] : p.start_frame[b];
}
__device__ __forceinline__ int64_t row_dst_begin(const AppendParams& p, int b) {
  return p.step_dev != nullptr ? p.step_dev[p.rows + b] : p.dst_begin[b];
}

// Device-resident parameters cannot be validated by the host: every thread checks them (the same
// few cached loads) and the whole launch writes nothing when a slot would leave the cache or a
// frame the rope table.  Block 0 records that in the status word.
__device__ __forceinline__ bool step_params_ok(const AppendParams& p) {
  if (p.step_dev == nullptr) return true;
  bool ok = true;
  for (int b = 0; b < p.rows; ++b) {
    const int64_t f = p.step_dev[b], d = p.step_dev[p.rows + b];
    ok = ok && f >= 0 && f + p.grid_f <= p.table_rows && d >= 0 && d + p.tokens <= p.cache_tokens;
  }
  return ok;
}

__device__ __forceinline__ void write_index(const AppendParams& p) {
  if (p.global_end_dev != nullptr) {
    for (int b = 0; b < p.rows; ++b) {
      p.global_end_dev[b] = p.step_dev != nullptr ? p.step_dev[2 * p.rows + b] : p.global_end_val[b];
      p.local_end_dev[b] = p.step_dev != nullptr ? p.step_dev[3 * p.rows + b] : p.local_end_val[b];
    }
  }
}

__device__ __forceinline__ void report_bad_step_params(const AppendParams& p) {
  if (p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(BAD_STEP_PARAMS));
}

inline uint32_t magic_of(uint32_t d) { return static_cast<uint32_t>(((1ull << 32) + d - 1) / d); }

}  // namespace sdv2
