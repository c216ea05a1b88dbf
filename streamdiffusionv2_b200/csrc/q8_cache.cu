// The K/V cache in 8 bits: written with the rotary embedding fused in, and read back.
//
// Format, per (row, token, head) vector x of 128 values: e = max(floor(log2(max|x|)) - 6, -126) and, per value, a
// sign bit above a 7-bit magnitude m = min(rint(|x| / 2^e), 127); the vector holds sign * m * 2^e.  The exponent is
// kept as one int8 beside the 128 bytes.  A power of two as the scale makes every held value a bf16 value, so
// reading back and the attention kernel's tiles lose nothing; it follows from the exponent bits of the maximum
// alone, so no rounding enters the choice.  |x - held| <= 2^(e-1), except that magnitudes above 127.5 go to 127
// (at most one step).  A vector with a value that fp32 cannot hold as a finite number gets e = -128 and reads back
// as NaN.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "q8.cuh"
#include "rope_append.cuh"
#include "sdv2_internal.h"

namespace sdv2 {
namespace q8 {

constexpr int kLanesPerHead = 16;  // 8 values a lane

// Eight values of a lane as loaded.
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Raw8<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const uint4*>(p));
    b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  }
};

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&y)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                                            pack_bf16x2(y[6], y[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&y)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(y[0], y[1], y[2], y[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(y[4], y[5], y[6], y[7]);
}

// max over the 16 lanes of a head vector
__device__ __forceinline__ uint32_t head_max(uint32_t v) {
#pragma unroll
  for (int o = kLanesPerHead / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ uint2 pack_bytes(const uint32_t (&m)[8]) {
  return make_uint2(m[0] | (m[1] << 8) | (m[2] << 16) | (m[3] << 24), m[4] | (m[5] << 8) | (m[6] << 16) | (m[7] << 24));
}

// Quantise the lane's eight doubles; the exponent comes back in `e`.  |y| * 2^-e < 128 is exact, and adding 2^52
// in one fused step rounds it to the nearest integer, ties to even, into the low word: no conversion instruction.
__device__ __forceinline__ uint2 quantise(const double (&y)[8], int& e) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, static_cast<uint32_t>(__double2hiint(y[i])) & 0x7FFFFFFFu);
  const int log2_top = static_cast<int>(head_max(top) >> 20) - 1023;
  if (log2_top > 127) {
    e = kNotFinite;
    return make_uint2(0u, 0u);
  }
  e = max(log2_top - 6, kMinExp);
  const double inv = __hiloint2double((1023 - e) << 20, 0);
  uint32_t m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t v = static_cast<uint32_t>(__double2loint(__fma_rn(fabs(y[i]), inv, 4503599627370496.0)));
    m[i] = min(v, 127u) | ((static_cast<uint32_t>(__double2hiint(y[i])) >> 24) & 0x80u);
  }
  return pack_bytes(m);
}

// The same for floats (values that are not rotated).
__device__ __forceinline__ uint2 quantise(const float (&y)[8], int& e) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
  const int log2_top = static_cast<int>(head_max(top) >> 23) - 127;
  if (log2_top > 127) {
    e = kNotFinite;
    return make_uint2(0u, 0u);
  }
  e = max(log2_top - 6, kMinExp);
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  uint32_t m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t v = __float_as_uint(__fmaf_rn(fabsf(y[i]), inv, 8388608.0f)) & 0x7FFFFFu;
    m[i] = min(v, 127u) | ((__float_as_uint(y[i]) >> 24) & 0x80u);
  }
  return pack_bytes(m);
}

// One warp per (row, token, group of heads): half a warp holds one head vector, eight values (four complex pairs) a
// lane, and the two halves walk the heads side by side.  A lane's four multipliers belong to its columns and serve
// every head of the token, so the rope table is read once per token and not once per head.
template <typename T>
__global__ void __launch_bounds__(256) rope_kv_append_q8_kernel(const __grid_constant__ Q8AppendParams qp) {
  const AppendParams& p = qp.a;
  if (!step_params_ok(p)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) report_bad_step_params(p);
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) write_index(p);
  const int lane = threadIdx.x & 31;
  const int c = lane & (kLanesPerHead - 1);
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t token = warp / qp.head_groups;
  const int hg = static_cast<int>(warp - token * qp.head_groups);
  if (token >= static_cast<int64_t>(p.rows) * p.tokens) return;  // whole warps leave
  const int b = static_cast<int>(token / p.tokens);
  const int t = static_cast<int>(token - static_cast<int64_t>(b) * p.tokens);
  const int f = fast_div(t, p.magic_plane);
  const int rem = t - f * p.plane;
  const int y = fast_div(rem, p.magic_w);
  const int x = rem - y * p.grid_w;
  double2 cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = table_entry(p, c * 4 + i, row_start_frame(p, b) + f, y, x);
  const int64_t slot = row_dst_begin(p, b) + t;
  const T* q_src = static_cast<const T*>(p.q.ptr) + b * p.q.stride_row + t * p.q.stride_tok + c * 8;
  const T* k_src = static_cast<const T*>(p.k.ptr) + b * p.k.stride_row + t * p.k.stride_tok + c * 8;
  const T* v_src = static_cast<const T*>(p.v.ptr) + b * p.v.stride_row + t * p.v.stride_tok + c * 8;
  T* q_dst = static_cast<T*>(p.q_out.ptr) + b * p.q_out.stride_row + t * p.q_out.stride_tok + c * 8;
  uint8_t* k_dst = static_cast<uint8_t*>(p.k_cache.ptr) + b * p.k_cache.stride_row + slot * p.k_cache.stride_tok + c * 8;
  uint8_t* v_dst = static_cast<uint8_t*>(p.v_cache.ptr) + b * p.v_cache.stride_row + slot * p.v_cache.stride_tok + c * 8;
  int8_t* ke_dst = static_cast<int8_t*>(qp.k_exp.ptr) + b * qp.k_exp.stride_row + slot * qp.k_exp.stride_tok;
  int8_t* ve_dst = static_cast<int8_t*>(qp.v_exp.ptr) + b * qp.v_exp.stride_row + slot * qp.v_exp.stride_tok;
  const int h_end = min(p.heads, (hg + 1) * qp.heads_per_group);
  for (int h0 = hg * qp.heads_per_group; h0 < h_end; h0 += 2) {
    const int h = h0 + (lane >> 4);
    const bool on = h < h_end;
    const int hc = on ? h : h0;  // the idle half of an odd count repeats its neighbour's loads and stores nothing
    Raw8<T> rq, rk, rv;
    rq.load(q_src + hc * p.q.stride_head);
    rk.load(k_src + hc * p.k.stride_head);
    rv.load(v_src + hc * p.v.stride_head);
    float xs[8], ys[8];
    rq.get(xs);
#pragma unroll
    for (int i = 0; i < 4; ++i) rope_pair(xs[2 * i], xs[2 * i + 1], cs[i], ys[2 * i], ys[2 * i + 1]);
    if (on) store8(q_dst + hc * p.q_out.stride_head, ys);
    rk.get(xs);
    double yd[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double re = xs[2 * i], im = xs[2 * i + 1];
      yd[2 * i] = __dsub_rn(__dmul_rn(re, cs[i].x), __dmul_rn(im, cs[i].y));
      yd[2 * i + 1] = __dadd_rn(__dmul_rn(re, cs[i].y), __dmul_rn(im, cs[i].x));
    }
    int ke, ve;
    const uint2 kb = quantise(yd, ke);
    rv.get(xs);
    const uint2 vb = quantise(xs, ve);
    if (on) {
      *reinterpret_cast<uint2*>(k_dst + hc * p.k_cache.stride_head) = kb;
      *reinterpret_cast<uint2*>(v_dst + hc * p.v_cache.stride_head) = vb;
      if (c == 0) {
        ke_dst[hc * qp.k_exp.stride_head] = static_cast<int8_t>(ke);
        ve_dst[hc * qp.v_exp.stride_head] = static_cast<int8_t>(ve);
      }
    }
  }
}

// A block reads `block_tokens` tokens of one row; a thread takes 8 bytes of a head vector, for K and V.
__global__ void __launch_bounds__(256) kv_read_q8_kernel(const __grid_constant__ Q8ReadParams p) {
  const int b = blockIdx.y;
  const int t0 = blockIdx.x * p.block_tokens;
  const int n = min(p.block_tokens, p.count[b] - t0) * p.row_vecs;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int j = fast_div(i, p.magic_row_vecs);
    const int r = i - j * p.row_vecs;
    const int h = r >> 4, c = r & 15;
    const int64_t src = p.begin[b] + t0 + j;
    const int64_t dst = t0 + j;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const sdv2_view& cv = which ? p.v : p.k;
      const sdv2_view& ev = which ? p.v_exp : p.k_exp;
      const sdv2_view& ov = which ? p.v_out : p.k_out;
      const uint2 raw = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(cv.ptr) + b * cv.stride_row +
                                                             src * cv.stride_tok + h * cv.stride_head + c * 8));
      const int e = static_cast<const int8_t*>(ev.ptr)[b * ev.stride_row + src * ev.stride_tok + h * ev.stride_head];
      uint32_t w[4];
      const uint32_t s2 = scale_bits(e + 6, e == kNotFinite);
      decode4(raw.x, s2, w[0], w[1]);
      decode4(raw.y, s2, w[2], w[3]);
      const int64_t o = b * ov.stride_row + dst * ov.stride_tok + h * ov.stride_head + c * 8;
      if (p.dtype == SDV2_DTYPE_BF16) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(ov.ptr) + o) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float4* op = reinterpret_cast<float4*>(static_cast<float*>(ov.ptr) + o);
        op[0] = make_float4(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u),
                            __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xFFFF0000u));
        op[1] = make_float4(__uint_as_float(w[2] << 16), __uint_as_float(w[2] & 0xFFFF0000u),
                            __uint_as_float(w[3] << 16), __uint_as_float(w[3] & 0xFFFF0000u));
      }
    }
  }
}

}  // namespace q8

cudaError_t launch_rope_kv_append_q8(const Q8AppendParams& p_in, int dtype, cudaStream_t stream) {
  Q8AppendParams p = p_in;
  AppendParams& a = p.a;
  a.plane = a.grid_h * a.grid_w;
  a.magic_plane = magic_of(a.plane);
  a.magic_w = magic_of(a.grid_w);
  // fast_div is exact while numerator * divisor < 2^32
  if (static_cast<uint64_t>(a.tokens) * a.plane >= (1ull << 32)) return cudaErrorInvalidValue;
  p.heads_per_group = a.heads;
  p.head_groups = 1;
  const int64_t warps = static_cast<int64_t>(a.rows) * a.tokens * p.head_groups;
  const int64_t blocks = (warps + 7) / 8;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  if (dtype == SDV2_DTYPE_BF16)
    q8::rope_kv_append_q8_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  else
    q8::rope_kv_append_q8_kernel<float><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv_read_q8(const Q8ReadParams& p_in, cudaStream_t stream) {
  Q8ReadParams p = p_in;
  p.row_vecs = p.heads * q8::kLanesPerHead;
  p.magic_row_vecs = magic_of(p.row_vecs);
  p.block_tokens = p.row_vecs >= 1024 ? 1 : (1024 + p.row_vecs - 1) / p.row_vecs;
  if (static_cast<uint64_t>(p.block_tokens) * p.row_vecs * p.row_vecs >= (1ull << 32)) return cudaErrorInvalidValue;
  const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens, p.rows);
  q8::kv_read_q8_kernel<<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace sdv2
