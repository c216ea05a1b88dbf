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
constexpr int kWarpsPerBlock = 4;
constexpr int kHeadsPerWarp = 24;  // at most
constexpr int kReadLanesPerHead = 8, kReadUnroll = 2;

// Eight values of a lane as loaded.
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
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
    a = reinterpret_cast<const uint4*>(p)[0];
    b = reinterpret_cast<const uint4*>(p)[1];
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

// Bytes i of four words, one above the other.
template <int kByte>
__device__ __forceinline__ uint32_t gather4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  constexpr uint32_t kPair = kByte | ((4 + kByte) << 4);
  return __byte_perm(__byte_perm(a, b, kPair), __byte_perm(c, d, kPair), 0x5410);
}
// Magnitudes 0..128 (low bytes of m) with 128 lowered to 127, under the signs (top bits of s).
__device__ __forceinline__ uint2 pack_bytes(const uint32_t (&m)[8], const uint32_t (&s)[8]) {
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = gather4<0>(m[4 * i], m[4 * i + 1], m[4 * i + 2], m[4 * i + 3]);
    const uint32_t sign = gather4<3>(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]) & 0x80808080u;
    o[i] = (v - ((v >> 7) & 0x01010101u)) | sign;
  }
  return make_uint2(o[0], o[1]);
}

__device__ __forceinline__ int clamp_exp(int log2_top) { return log2_top > 127 ? kNotFinite : max(log2_top - 6, kMinExp); }

// floor(log2) + 1023 of the largest of eight doubles, + 127 of the largest of eight floats (denormals: 0)
__device__ __forceinline__ uint32_t top_exponent(const double (&y)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    top = __vimax3_u32(top, __double2hiint(y[i]) & 0x7FFFFFFFu, __double2hiint(y[i + 1]) & 0x7FFFFFFFu);
  return top >> 20;
}
__device__ __forceinline__ uint32_t top_exponent(const float (&y)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    top = __vimax3_u32(top, __float_as_uint(y[i]) & 0x7FFFFFFFu, __float_as_uint(y[i + 1]) & 0x7FFFFFFFu);
  return top >> 23;
}

// The eight values of a lane in units of 2^e.  |y| * 2^-e < 128 is exact, and adding 2^52 (2^23 for floats) in one
// fused step rounds it to the nearest integer, ties to even, into the low bits: no conversion instruction.
__device__ __forceinline__ uint2 quantise(const double (&y)[8], int e) {
  if (e == kNotFinite) return make_uint2(0u, 0u);
  const double inv = __hiloint2double((1023 - e) << 20, 0);
  uint32_t m[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = static_cast<uint32_t>(__double2loint(__fma_rn(fabs(y[i]), inv, 4503599627370496.0)));
    s[i] = static_cast<uint32_t>(__double2hiint(y[i]));
  }
  return pack_bytes(m, s);
}
__device__ __forceinline__ uint2 quantise(const float (&y)[8], int e) {
  if (e == kNotFinite) return make_uint2(0u, 0u);
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  uint32_t m[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = __float_as_uint(__fmaf_rn(fabsf(y[i]), inv, 8388608.0f));
    s[i] = __float_as_uint(y[i]);
  }
  return pack_bytes(m, s);
}

// One warp per (row, token, group of heads): half a warp holds one head vector, eight values (four complex pairs) a
// lane, and the two halves walk the heads side by side, the next pair's loads in flight.  A lane's four multipliers
// belong to its columns and serve every head of the token, so the rope table is read once per token and not once per head.
// Bound by HBM at large sizes, 1282 bytes a head vector in bf16: 4 rows x 3120 tokens x 40 heads 114.5 us (5.6 TB/s), 2 x
// 3120 x 12 20.8 us (4.6 TB/s; some 3 us are start and drain).
template <typename T>
__global__ void __launch_bounds__(kWarpsPerBlock * 32, sizeof(T) == 2 ? 6 : 5)
rope_kv_append_q8_kernel(const __grid_constant__ Q8AppendParams qp) {
  const AppendParams& p = qp.a;
  begin_after_previous_kernel();
  if (!step_params_ok(p)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) report_bad_step_params(p);
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) write_index(p);
  const int lane = threadIdx.x & 31;
  const int c = lane & (kLanesPerHead - 1);
  const uint32_t warp = blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);  // the launcher keeps the count below 2^31
  const uint32_t token = warp / static_cast<uint32_t>(qp.head_groups);
  const int hg = static_cast<int>(warp - token * qp.head_groups);
  if (token >= static_cast<uint32_t>(p.rows) * p.tokens) return;  // whole warps leave
  const int b = static_cast<int>(token / static_cast<uint32_t>(p.tokens));
  const int t = static_cast<int>(token - static_cast<uint32_t>(b) * p.tokens);
  const int f = fast_div(t, p.magic_plane);
  const int rem = t - f * p.plane;
  const int y = fast_div(rem, p.magic_w);
  const int x = rem - y * p.grid_w;
  const int64_t slot = row_dst_begin(p, b) + t;
  const int h_end = min(p.heads, (hg + 1) * qp.heads_per_group);
  // the half without a head, at the end of an odd count, works on its neighbour's and stores nothing
  int h = hg * qp.heads_per_group + (lane >> 4);
  const int h_first = min(h, h_end - 1);
  const T* q_src = static_cast<const T*>(p.q.ptr) + b * p.q.stride_row + t * p.q.stride_tok + h_first * p.q.stride_head + c * 8;
  const T* k_src = static_cast<const T*>(p.k.ptr) + b * p.k.stride_row + t * p.k.stride_tok + h_first * p.k.stride_head + c * 8;
  const T* v_src = static_cast<const T*>(p.v.ptr) + b * p.v.stride_row + t * p.v.stride_tok + h_first * p.v.stride_head + c * 8;
  Raw8<T> rq, rk, rv;
  rq.load(q_src);
  rk.load(k_src);
  rv.load(v_src);
  double2 cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = *table_place(p, c * 4 + i, row_start_frame(p, b) + f, y, x);
  T* q_dst = static_cast<T*>(p.q_out.ptr) + b * p.q_out.stride_row + t * p.q_out.stride_tok + h_first * p.q_out.stride_head + c * 8;
  uint8_t* k_dst = static_cast<uint8_t*>(p.k_cache.ptr) + b * p.k_cache.stride_row + slot * p.k_cache.stride_tok +
                   h_first * p.k_cache.stride_head + c * 8;
  uint8_t* v_dst = static_cast<uint8_t*>(p.v_cache.ptr) + b * p.v_cache.stride_row + slot * p.v_cache.stride_tok +
                   h_first * p.v_cache.stride_head + c * 8;
  int8_t* ke_dst = static_cast<int8_t*>(qp.k_exp.ptr) + b * qp.k_exp.stride_row + slot * qp.k_exp.stride_tok +
                   h_first * qp.k_exp.stride_head;
  int8_t* ve_dst = static_cast<int8_t*>(qp.v_exp.ptr) + b * qp.v_exp.stride_row + slot * qp.v_exp.stride_tok +
                   h_first * qp.v_exp.stride_head;
#pragma unroll 1
  while (true) {
    const bool on = h < h_end;
    const bool more = __any_sync(0xffffffffu, h + 2 < h_end);
    float xs[8];
    rk.get(xs);
    double yd[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double re = xs[2 * i], im = xs[2 * i + 1];
      yd[2 * i] = __dsub_rn(__dmul_rn(re, cs[i].x), __dmul_rn(im, cs[i].y));
      yd[2 * i + 1] = __dadd_rn(__dmul_rn(re, cs[i].y), __dmul_rn(im, cs[i].x));
    }
    float xv[8], xq[8];
    rv.get(xv);
    rq.get(xq);
    if (more) {  // the next pair of heads is on its way while this one is worked on
      const int64_t step = h + 2 < h_end ? 2 : 0;
      q_src += step * p.q.stride_head;
      k_src += step * p.k.stride_head;
      v_src += step * p.v.stride_head;
      rq.load(q_src);
      rk.load(k_src);
      rv.load(v_src);
    }
    // both exponents through one reduction over the 16 lanes of the head
    uint32_t top = (top_exponent(yd) << 16) | top_exponent(xv);
#pragma unroll
    for (int o = kLanesPerHead / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int ke = clamp_exp(static_cast<int>(top >> 16) - 1023), ve = clamp_exp(static_cast<int>(top & 0xFFFFu) - 127);
    const uint2 kb = quantise(yd, ke), vb = quantise(xv, ve);
    if (on) {
      *reinterpret_cast<uint2*>(k_dst) = kb;
      *reinterpret_cast<uint2*>(v_dst) = vb;
      if (c == 0) {
        *ke_dst = static_cast<int8_t>(ke);
        *ve_dst = static_cast<int8_t>(ve);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) rope_pair(xq[2 * i], xq[2 * i + 1], cs[i], xs[2 * i], xs[2 * i + 1]);
    if (on) store8(q_dst, xs);
    if (!more) break;
    h += 2;
    q_dst += 2 * p.q_out.stride_head;
    k_dst += 2 * p.k_cache.stride_head;
    v_dst += 2 * p.v_cache.stride_head;
    ke_dst += 2 * qp.k_exp.stride_head;
    ve_dst += 2 * qp.v_exp.stride_head;
  }
}

// 32 bytes: one store where the tensor's layout keeps 32-byte alignment, else two
template <bool kWide>
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  if (!kWide) {
    static_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    return;
  }
  st_global_v8(p, w);
}

// A block reads `block_tokens` tokens of one row.  A thread takes 16 bytes of a head vector, of K and of V and of
// kReadUnroll vectors at a time, and writes them as whole 32-byte sectors (2 rows x 32760 tokens x 12 heads to bf16: 100 us,
// 6.05 TB/s, bound by HBM; 110 us with two 16-byte stores in their place).
template <bool kBf16, bool kWide>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(const __grid_constant__ Q8ReadParams p) {
  begin_after_previous_kernel();
  const int b = blockIdx.y;
  const int t0 = blockIdx.x * p.block_tokens;
  const int n = min(p.block_tokens, p.count[b] - t0) * p.row_vecs;
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * kReadUnroll) {
    uint4 raw[kReadUnroll][2];
    int e[kReadUnroll][2];
    int64_t out[kReadUnroll][2];
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
      const int i = min(i0 + u * 256, n - 1);
      const int j = fast_div(i, p.magic_row_vecs);
      const int r = i - j * p.row_vecs;
      const int h = r >> 3, c = (r & 7) * 16;
      const int64_t src = p.begin[b] + t0 + j, dst = t0 + j;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const sdv2_view& cv = which ? p.v : p.k;
        const sdv2_view& ev = which ? p.v_exp : p.k_exp;
        const sdv2_view& ov = which ? p.v_out : p.k_out;
        raw[u][which] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(cv.ptr) + b * cv.stride_row +
                                                        src * cv.stride_tok + h * cv.stride_head + c);
        e[u][which] = static_cast<const signed char*>(ev.ptr)[b * ev.stride_row + src * ev.stride_tok + h * ev.stride_head];
        out[u][which] = b * ov.stride_row + dst * ov.stride_tok + h * ov.stride_head + c;
      }
    }
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
      if (i0 + u * 256 >= n) break;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t s2 = scale_bits(min(e[u][which], 121) + 6, e[u][which] == kNotFinite);
        uint32_t w[8];
        decode4(raw[u][which].x, s2, w[0], w[1]);
        decode4(raw[u][which].y, s2, w[2], w[3]);
        decode4(raw[u][which].z, s2, w[4], w[5]);
        decode4(raw[u][which].w, s2, w[6], w[7]);
        const sdv2_view& ov = which ? p.v_out : p.k_out;
        if (kBf16) {
          store32<kWide>(static_cast<__nv_bfloat16*>(ov.ptr) + out[u][which], w);
        } else {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t x[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              x[2 * k] = w[hf * 4 + k] << 16;
              x[2 * k + 1] = w[hf * 4 + k] & 0xFFFF0000u;
            }
            store32<kWide>(static_cast<float*>(ov.ptr) + out[u][which] + hf * 8, x);
          }
        }
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
  // few tokens: fewer heads to a warp, so that every scheduler has warps to switch between (390 tokens x 12 heads: 4.1 us
  // with four heads, 5.8 with all twelve); enough of them: more, for one look at the table serves them all (2 rows x 3120
  // tokens x 12 heads: 20.8 us with twelve, 24.0 with four)
  DeviceInfo di;
  const cudaError_t e = device_info(&di);
  if (e != cudaSuccess) return e;
  int per_warp = q8::kHeadsPerWarp;
  while (per_warp > 4 && static_cast<int64_t>(a.rows) * a.tokens * ((a.heads + per_warp - 1) / per_warp) < 12 * di.sms) per_warp /= 2;
  p.head_groups = (a.heads + per_warp - 1) / per_warp;
  p.heads_per_group = (((a.heads + p.head_groups - 1) / p.head_groups) + 1) & ~1;  // groups of equal, even size
  p.head_groups = (a.heads + p.heads_per_group - 1) / p.heads_per_group;
  const int64_t warps = static_cast<int64_t>(a.rows) * a.tokens * p.head_groups;
  if (warps > 0x7FFFFF00LL) return cudaErrorInvalidValue;
  const int64_t blocks = (warps + q8::kWarpsPerBlock - 1) / q8::kWarpsPerBlock;
  constexpr int kThreads = q8::kWarpsPerBlock * 32;
  auto* kernel = dtype == SDV2_DTYPE_BF16 ? q8::rope_kv_append_q8_kernel<__nv_bfloat16> : q8::rope_kv_append_q8_kernel<float>;
  return launch_chained(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, p);
}

cudaError_t launch_kv_read_q8(const Q8ReadParams& p_in, cudaStream_t stream) {
  Q8ReadParams p = p_in;
  p.row_vecs = p.heads * q8::kReadLanesPerHead;
  p.magic_row_vecs = magic_of(p.row_vecs);
  constexpr int kPass = 256 * q8::kReadUnroll;
  p.block_tokens = p.row_vecs >= kPass ? 1 : (kPass + p.row_vecs - 1) / p.row_vecs;
  if (static_cast<uint64_t>(p.block_tokens) * p.row_vecs * p.row_vecs >= (1ull << 32)) return cudaErrorInvalidValue;
  const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens, p.rows);
  const int esize = p.dtype == SDV2_DTYPE_BF16 ? 2 : 4;
  auto wide = [&](const sdv2_view& v) {
    const int64_t any = (v.stride_row | v.stride_tok | v.stride_head) * esize | static_cast<int64_t>(reinterpret_cast<uintptr_t>(v.ptr));
    return (any & 31) == 0;
  };
  const bool w = wide(p.k_out) && wide(p.v_out);
  auto* kernel = p.dtype == SDV2_DTYPE_BF16 ? (w ? q8::kv_read_q8_kernel<true, true> : q8::kv_read_q8_kernel<true, false>)
                                            : (w ? q8::kv_read_q8_kernel<false, true> : q8::kv_read_q8_kernel<false, false>);
  return launch_chained(kernel, grid, dim3(256), 0, stream, p);
}

}  // namespace sdv2
