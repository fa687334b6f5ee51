// Pieces shared by the kernels over the 8-bit KV cache (k_kv8.cu, k_kv8_step.cu,
// k_kv8_flash.cu).
//
// A cached row (one position of one kv head, D values) is stored as D codes of
// one byte and one fp32 scale:
//   s = fl32(max|x| / M),  code = round-half-even(x / s),  value = code * s,
// M = 127 for int8 codes and 448 for e4m3 codes. x is the real-number result
// of the head norm and rotary on the fp32 inputs: it is formed in double, so
// the code is the right one also next to a rounding border. A row with a
// value that is not finite gets a NaN scale and zero codes (it reads back as
// NaN and poisons only the queries that see it).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "b2m_internal.cuh"
#include "ptx.cuh"

namespace kv8 {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_max_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Nearest e4m3 code (ties to even) of t, |t| <= 448. The hardware conversion
// takes fp32, and rounding a double to fp32 first could land on a border that
// the double is not on: t goes to fp32 toward zero with the lost bits ORed
// into the last place, which the second rounding then sees as "above".
__device__ __forceinline__ uint8_t e4m3_code(double t) {
  float f = __double2float_rz(t);
  if ((double)f != t) f = __uint_as_float(__float_as_uint(f) | 1u);
  return (uint8_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
}

// The value a code stands for, before its row's scale.
template <bool E4M3>
__device__ __forceinline__ float code_value(uint8_t c) {
  if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
  return (float)(int8_t)c;
}

// One new row: quantised into codes[0..D) and *scale by one warp. `xs` is the
// row's fp32 input staged in shared memory. norm: multiply by gain[d] /
// sqrt(mean + eps) first; cos != null: rotary at `pos` on the first rot values.
__device__ __forceinline__ void quantise_row(const float *xs, int D, const float *gain, double eps, const float *cos,
                                             const float *sin, int64_t pos, int half, int rot, int interleaved,
                                             bool e4m3, uint8_t *codes, float *scale, int lane) {
  double inv = 1.0;
  if (gain) {
    double ss = 0.0;
    for (int d = lane; d < D; d += 32) ss += (double)xs[d] * xs[d];
    inv = 1.0 / sqrt(warp_sum_d(ss) / D + eps);
  }
  auto normed = [&](int d) { return gain ? (double)xs[d] * inv * gain[d] : (double)xs[d]; };
  double x[8];  // D <= 256: four consecutive values of up to two 128-value blocks
  double amax = 0.0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int d = (i >> 2) * 128 + 4 * lane + (i & 3);
    x[i] = 0.0;
    if (d >= D) continue;
    double v = normed(d);
    if (cos && d < rot) {
      const int hr = rot >> 1;
      const bool first = interleaved ? (d & 1) == 0 : d < hr;
      const int pi = interleaved ? d >> 1 : (first ? d : d - hr);
      const int e = interleaved ? (d ^ 1) : (first ? d + hr : d - hr);
      const double c = cos[pos * half + pi], sn = sin[pos * half + pi], w = normed(e);
      v = first ? v * c - w * sn : v * c + w * sn;
    }
    x[i] = v;
    bad |= !isfinite(v);
    amax = fmax(amax, fabs(v));
  }
  bad = __any_sync(0xffffffffu, bad);
  amax = warp_max_d(amax);
  const double top = e4m3 ? 448.0 : 127.0;
  const float s = bad ? __int_as_float(0x7fc00000) : (float)(amax / top);
  if (lane == 0) *scale = s;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int d0 = h * 128 + 4 * lane;
    if (d0 >= D) continue;
    uint32_t w = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      uint32_t c = 0;
      if (s > 0.f) {  // false for NaN
        const double t = fmin(fmax(x[4 * h + u] / (double)s, -top), top);
        c = e4m3 ? e4m3_code(t) : (uint8_t)(int8_t)(int)rint(t);
      }
      w |= c << (8 * u);
    }
    if (d0 + 4 <= D && (reinterpret_cast<uintptr_t>(codes + d0) & 3) == 0) {
      *reinterpret_cast<uint32_t *>(codes + d0) = w;
    } else {
      for (int u = 0; u < 4 && d0 + u < D; u++) codes[d0 + u] = (uint8_t)(w >> (8 * u));
    }
  }
}

// Rotary position of new token i of sequence b; -1 when its depth is outside
// [0, S) (the caller raises the device error).
__device__ __forceinline__ int64_t token_pos(const Kv8Args &a, int b, int i, int past) {
  if (!a.depth) return past + i;
  const int dp = a.depth[(int64_t)b * a.S + i];
  return dp < 0 || dp >= a.S ? -1 : past + dp;
}

// Quantises one side (0: key, 1: value) of new token i of (sequence b, kv head)
// into the cache, by one warp; xs: 256 floats of shared memory of its own.
__device__ __forceinline__ void append_row(const Kv8Args &a, int b, int i, int kvh, int side, int past, float *xs,
                                           int lane) {
  const int64_t pos = token_pos(a, b, i, past);
  if (past < 0 || (a.cos && pos < 0)) {
    if (lane == 0 && a.err) b2m::set_dev_error(a.err, B2M_DEVERR_INDEX);
    return;
  }
  if ((int64_t)past + i >= a.CAP) {
    if (lane == 0 && a.err) b2m::set_dev_error(a.err, B2M_DEVERR_CACHE_FULL);
    return;
  }
  const float *src = (side ? a.v : a.k) + ((int64_t)b * a.S + i) * a.kv_rs + (int64_t)kvh * a.D;
  __syncwarp();
  for (int d = lane; d < a.D; d += 32) xs[d] = src[d];
  __syncwarp();
  const int64_t row = ((int64_t)b * a.KVH + kvh) * a.CAP + past + i;
  // rotary only reads the table where the position is in it: past + depth < CAP
  const float *gain = side || !a.k_gain ? nullptr : a.k_gain + (int64_t)kvh * a.D;
  const float *cos = side || pos >= a.CAP ? nullptr : a.cos;
  quantise_row(xs, a.D, gain, a.eps, cos, a.sin, pos, a.half, a.rot, a.interleaved, a.e4m3,
               (side ? a.vc : a.kc) + row * a.D, (side ? a.vs : a.ks) + row, lane);
}

// Two e-th codes of words a and b interleaved: prmt selectors for codes 0, 1
// and codes 2, 3 of both.
constexpr uint32_t PAIR01 = 0x5140, PAIR23 = 0x7362;

// Word of four codes c0 .. c3 -> (c0, c1) and (c2, c3) as f16 pairs. int8:
// exact values, by the bits of 1024 + (c + 128) minus 1152. e4m3: exactly 2^-8
// of the value, by moving the exponent and mantissa fields into place (every
// bit pattern gives a finite number; the factor is folded into the scales).
template <bool E4M3>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t &p01, uint32_t &p23) {
  if (E4M3) {
    const uint32_t a = b2m::prmt(w, 0u, 0x1404), b = b2m::prmt(w, 0u, 0x3424);
    p01 = ((a >> 1) & 0x3f803f80u) | (a & 0x80008000u);
    p23 = ((b >> 1) & 0x3f803f80u) | (b & 0x80008000u);
  } else {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 k = __half2half2(__ushort_as_half(0x6480));  // 1152
    p01 = b2m::h2_as_u32(__hsub2(b2m::u32_as_h2(b2m::prmt(x, 0x64646464u, 0x4140)), k));
    p23 = b2m::h2_as_u32(__hsub2(b2m::u32_as_h2(b2m::prmt(x, 0x64646464u, 0x4342)), k));
  }
}
template <bool E4M3>
__host__ __device__ constexpr float code_factor() {
  return E4M3 ? 256.f : 1.f;
}

}  // namespace kv8

// The warp-level tensor-core kernel for few query rows per kv head
// (k_kv8_step.cu).
bool kv8_step_shape(const Kv8Args &a);
void launch_kv8_step(const Kv8Args &a, cudaStream_t s);
// The tcgen05 kernel for many rows (k_kv8_flash.cu), after launch_kv8_append.
bool kv8_flash_shape(const Kv8Args &a);
void launch_kv8_flash(const Kv8Args &a, cudaStream_t s);
