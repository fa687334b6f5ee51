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
__device__ __forceinline__ float lg2(float x) {  // -inf for 0
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---- the reference of a row's weights ------------------------------------------
// What goes to the tensor cores is w_j = 2^(x_j - ref) v_j as one or two f16 terms
// (x_j the score in log2 units, v_j the V row's scale over the largest that the
// kernel has met, 0 <= v_j <= 1), and l = sum 2^(x_j - ref) in fp32 beside it. f16
// reaches from 2^-24 to 2^16, so ref has to follow the largest w_j of the row's own
// keys, c = max (x_j + log2 v_j): taken from the scores alone, a loud V row that this
// row does not see, or hardly weighs, would push the others' w_j out of f16 (32 keys
// beside a hidden one 2^20 times as large: 1.7e-4 of error, 2^36: zeros). The largest
// w_j stands at 2^REF_BIAS and may grow by 2^REF_SLACK before ref moves. The plain
// weights are then larger than w_j by up to 1 / v_j; REF_SPAN bounds that, so that sums
// over 2^30 keys stay below 2^120. V rows of one sequence may so differ by 2^85 before
// the small ones of a row that sees no others lose digits. A scale not below V_LOW costs
// none: the largest w_j is then at 2^2 or more, and what two terms cannot hold is below
// 2^-27 of it.
constexpr float REF_BIAS = 10.f, REF_SLACK = 5.f, REF_SPAN = 85.f, V_LOW = 0x1p-8f;
__device__ __forceinline__ float weight_ref(float m, float c) { return fmaxf(c - REF_BIAS, m - REF_SPAN); }

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
  if (!a.depth) return (int64_t)past + i;
  const int dp = a.depth[(int64_t)b * a.S + i];
  return dp < 0 || dp >= a.S ? -1 : (int64_t)past + dp;
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

// ---- the same row with little double arithmetic ----------------------------
// Rows of whole float4s (D % 4 == 0, aligned, rotary pairs in whole float4s): x is
// formed in fp32, and only what that cannot decide goes through double: the
// row's norm factor, the elements that may be the maximum, and an element whose
// fp32 quotient lies within its error of a rounding border. Same codes and
// scales as quantise_row.
struct RowChunk {
  float x[4], w[4];    // values and their rotary partners
  float g[4], gw[4];   // head norm gains of both
  float c[4], sn[4];   // x_rot = x c - w sn (the sign of the second half is in sn)
};

// max(|a|, |b|, |c|), NaN if one is.
__device__ __forceinline__ float max3_nan_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

template <bool NORM, bool ROT>
__device__ __forceinline__ double chunk_exact(const RowChunk &r, int k, double inv, bool turn) {
  const double x = NORM ? (double)r.x[k] * inv * r.g[k] : (double)r.x[k];
  if (!ROT || !turn) return x;
  const double w = NORM ? (double)r.w[k] * inv * r.gw[k] : (double)r.w[k];
  return x * (double)r.c[k] - w * (double)r.sn[k];
}

__device__ __forceinline__ uint32_t exact_code(double x, float s, bool e4m3) {
  const double top = e4m3 ? 448.0 : 127.0, t = fmin(fmax(x / (double)s, -top), top);
  return e4m3 ? e4m3_code(t) : (uint32_t)(uint8_t)(int8_t)(int)rint(t);
}

// Reductions over the LPR lanes (32, or either half of a warp) of a row; the whole
// warp takes part.
template <int LPR>
__device__ __forceinline__ double row_sum_d(double v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LPR>
__device__ __forceinline__ double row_max_d(double v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int LPR>
__device__ __forceinline__ uint32_t row_max_u(uint32_t v) {
  if constexpr (LPR == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}

// NCH chunks of four values per lane, LPR lanes per row: lane l of the row holds
// values 4 (l + LPR i) .. + 3. Writes nothing where !ok.
// NORM: the head norm comes first; ROT: the chunks that `turn` marks are rotated.
template <bool E4M3, int LPR, int NCH, bool NORM, bool ROT>
__device__ __forceinline__ void quantise_chunks(RowChunk (&r)[NCH], int D, double eps, const bool (&turn)[NCH],
                                                uint8_t *codes, float *scale, int l, bool ok) {
  constexpr bool real = NORM || ROT;  // x is more than its fp32 value
  constexpr float top = E4M3 ? 448.f : 127.f;
  double inv = 1.0;
  float invf = 1.f;
  if (NORM) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NCH; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) ss = fma((double)r[i].x[k], (double)r[i].x[k], ss);
    const double v = row_sum_d<LPR>(ss) / D + eps;
    // 1 / sqrt(v): two Newton steps from the fp32 value (relative error 2^-50);
    // outside fp32's comfortable range by the library
    if (v > 1e-30 && v < 1e30) {
      double y = rsqrtf((float)v);
      y = y * fma(-0.5 * v * y, y, 1.5);
      inv = y * fma(-0.5 * v * y, y, 1.5);
    } else {
      inv = 1.0 / sqrt(v);
    }
    invf = (float)inv;
  }
  float x[NCH][4];
  float top_x = 0.f, mag = 0.f;  // largest value; largest sum of the magnitudes that make up one
#pragma unroll
  for (int i = 0; i < NCH; i++) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float v = NORM ? r[i].x[k] * invf * r[i].g[k] : r[i].x[k];
      if (ROT && turn[i]) {
        const float w = NORM ? r[i].w[k] * invf * r[i].gw[k] : r[i].w[k];
        const float p = v * r[i].c[k], q = w * r[i].sn[k];
        v = p - q;
        mag = fmaxf(mag, fabsf(p) + fabsf(q));
      } else if (real) {
        mag = fmaxf(mag, fabsf(v));
      }
      x[i][k] = v;
    }
    top_x = max3_nan_abs(top_x, x[i][0], x[i][1]);
    top_x = max3_nan_abs(top_x, x[i][2], x[i][3]);
  }
  const uint32_t mx = row_max_u<LPR>(__float_as_uint(top_x));  // infinities and NaN order above
  const float amaxf = __uint_as_float(mx);
  // |fp32 x - x|: at most seven roundings of 2^-24 of mag
  const float xerr = real ? __uint_as_float(row_max_u<LPR>(__float_as_uint(mag))) * 0x1p-20f : 0.f;
  float s;
  if (!real) {
    // amaxf / top, rounded once: Markstein's quotient by the rounded reciprocal
    const float t = amaxf * (1.f / top);
    s = fmaf(fmaf(-t, top, amaxf), 1.f / top, t);
  } else {
    double am = 0.0;
    const float near = amaxf - 2.f * xerr;
    if (fabsf(top_x) >= near) {  // few lanes hold a candidate
#pragma unroll
      for (int i = 0; i < NCH; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (fabsf(x[i][k]) >= near) am = fmax(am, fabs(chunk_exact<NORM, ROT>(r[i], k, inv, turn[i])));
    }
    // one lane of the row as a rule
    const unsigned half = LPR == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    const unsigned cand = __ballot_sync(0xffffffffu, am > 0.0) & half;
    if (__any_sync(0xffffffffu, (cand & (cand - 1)) != 0))
      am = row_max_d<LPR>(am);
    else
      am = __shfl_sync(0xffffffffu, am, cand ? __ffs(cand) - 1 : 0);
    s = (float)(am * (1.0 / (double)top));
  }
  // Values near the ends of fp32's range: everything in double.
  const bool slow_row = real ? !(amaxf > 1e-25f && amaxf < 1e30f) : !(amaxf > 1e-30f && mx < 0x7f800000u);
  uint32_t word[NCH];
  if (__any_sync(0xffffffffu, slow_row)) {  // (both rows of a warp: the exact way is right for either)
    double am = 0.0;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < NCH; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const double v = chunk_exact<NORM, ROT>(r[i], k, inv, turn[i]);
        bad |= isfinite(v) ? 0u : 1u;
        am = fmax(am, fabs(v));
      }
    bad = row_max_u<LPR>(bad);
    am = row_max_d<LPR>(am);
    s = bad ? __int_as_float(0x7fc00000) : (float)(am / (double)top);
#pragma unroll
    for (int i = 0; i < NCH; i++) {
      word[i] = 0;
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (s > 0.f) word[i] |= exact_code(chunk_exact<NORM, ROT>(r[i], k, inv, turn[i]), s, E4M3) << (8 * k);
    }
  } else {
    const float is = __fdividef(1.f, s);  // (its error of some 2^-23 is within the 2^-20 below)
    const float wabs = xerr * is;  // |t - x / s| is at most this and 2^-20 of t
    uint32_t doubt[NCH], any = 0;  // bytes whose code depends on the error
#pragma unroll
    for (int i = 0; i < NCH; i++) {
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float t = x[i][k] * is, w = fmaf(fabsf(t), 0x1p-20f, wabs);
        if (E4M3) {
          lo[k] = __nv_cvt_float2_to_fp8x2(make_float2(t - w, t + w), __NV_SATFINITE, __NV_E4M3);
        } else {
          lo[k] = __float_as_uint((t - w) + 12582912.f);
          hi[k] = __float_as_uint((t + w) + 12582912.f);
        }
      }
      if (E4M3) {
        const uint32_t u = b2m::prmt(lo[0], lo[1], 0x5410), v = b2m::prmt(lo[2], lo[3], 0x5410);  // pairs (lo, hi)
        word[i] = b2m::prmt(u, v, 0x6420);
        doubt[i] = word[i] ^ b2m::prmt(u, v, 0x7531);
      } else {
        word[i] = b2m::prmt(b2m::prmt(lo[0], lo[1], 0x0040), b2m::prmt(lo[2], lo[3], 0x0040), 0x5410);
        doubt[i] = word[i] ^ b2m::prmt(b2m::prmt(hi[0], hi[1], 0x0040), b2m::prmt(hi[2], hi[3], 0x0040), 0x5410);
      }
      any |= doubt[i];
    }
    if (any) {
#pragma unroll
      for (int i = 0; i < NCH; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (doubt[i] >> (8 * k) & 0xffu) {
            const uint32_t code = exact_code(chunk_exact<NORM, ROT>(r[i], k, inv, turn[i]), s, E4M3);
            word[i] = (word[i] & ~(0xffu << (8 * k))) | (code << (8 * k));
          }
    }
  }
  if (!ok) return;
  if (l == 0) *scale = s;
#pragma unroll
  for (int i = 0; i < NCH; i++)
    if (4 * (l + LPR * i) < D) *reinterpret_cast<uint32_t *>(codes + 4 * (l + LPR * i)) = word[i];
}

// The rows quantise_chunks takes.
inline bool append_rows_vec(const Kv8Args &a) {
  auto al = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  return a.D % 4 == 0 && a.kv_rs % 4 == 0 && al(a.k) && al(a.v) && al(a.k_gain) &&
         (!a.cos || (a.rot % 8 == 0 && a.half % 4 == 0 && al(a.cos) && al(a.sin)));
}

// Loads one side's row of a new token (position pos for the rotary).
template <int LPR, int NCH>
__device__ __forceinline__ void load_chunks(const Kv8Args &a, const float *src, const float *gain, const float *cos,
                                            int64_t pos, RowChunk (&r)[NCH], bool (&turn)[NCH], int l) {
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int d = 4 * (l + LPR * i);
    turn[i] = false;
    auto put = [](float *dst, const float *p) {
      const float4 v = *reinterpret_cast<const float4 *>(p);
      dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
    };
#pragma unroll
    for (int k = 0; k < 4; k++) r[i].x[k] = r[i].w[k] = r[i].g[k] = r[i].gw[k] = r[i].c[k] = r[i].sn[k] = 0.f;
    if (d >= a.D) continue;
    put(r[i].x, src + d);
    if (gain) put(r[i].g, gain + d);
    if (cos && d < a.rot) {
      turn[i] = true;
      if (a.interleaved) {
        const float2 c2 = *reinterpret_cast<const float2 *>(cos + pos * a.half + (d >> 1));
        const float2 s2 = *reinterpret_cast<const float2 *>(a.sin + pos * a.half + (d >> 1));
        r[i].c[0] = r[i].c[1] = c2.x, r[i].c[2] = r[i].c[3] = c2.y;
        r[i].sn[0] = s2.x, r[i].sn[1] = -s2.x, r[i].sn[2] = s2.y, r[i].sn[3] = -s2.y;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          r[i].w[k] = r[i].x[k ^ 1];
          r[i].gw[k] = r[i].g[k ^ 1];
        }
      } else {
        const int hr = a.rot >> 1;
        const bool first = d < hr;
        const int pi = first ? d : d - hr, e = first ? d + hr : d - hr;
        put(r[i].c, cos + pos * a.half + pi);
        put(r[i].sn, a.sin + pos * a.half + pi);
        put(r[i].w, src + e);
        if (gain) put(r[i].gw, gain + e);
        if (!first)
#pragma unroll
          for (int k = 0; k < 4; k++) r[i].sn[k] = -r[i].sn[k];
      }
    }
  }
}

// Where a new token's row goes; false (and the device error) where it is refused.
struct NewRow {
  int64_t pos, off, row;
  const float *gain, *cos;
};
__device__ __forceinline__ bool place_row(const Kv8Args &a, int b, int i, int kvh, int past, NewRow &w) {
  w.pos = token_pos(a, b, i, past);
  const bool index = past < 0 || (a.cos && w.pos < 0), full = (int64_t)past + i >= a.CAP;
  if ((index || full) && a.err) b2m::set_dev_error(a.err, index ? B2M_DEVERR_INDEX : B2M_DEVERR_CACHE_FULL);
  w.off = ((int64_t)b * a.S + i) * a.kv_rs + (int64_t)kvh * a.D;
  w.row = ((int64_t)b * a.KVH + kvh) * a.CAP + past + i;
  w.gain = a.k_gain ? a.k_gain + (int64_t)kvh * a.D : nullptr;
  w.cos = w.pos < 0 || w.pos >= a.CAP ? nullptr : a.cos;  // the table's positions
  return !index && !full;
}

// append_row for rows that append_rows_vec accepts: the sides of `sides` (bit 0:
// the key, bit 1: the value) of one new token's kv head per LPR lanes, all loads
// ahead of the arithmetic. All 32 lanes call it, `ok` false where there is none.
template <bool E4M3, int LPR, int NCH>
__device__ __forceinline__ void append_vec(const Kv8Args &a, int b, int i, int kvh, int sides, int past, bool ok) {
  const int l = threadIdx.x & (LPR - 1);
  NewRow w;
  ok = ok && place_row(a, b, i, kvh, past, w);
  if (!ok) w.off = 0, w.row = 0, w.pos = 0, w.gain = nullptr, w.cos = nullptr;  // (reads the first row, writes nothing)
  RowChunk rk[NCH], rv[NCH];
  bool tk[NCH], tv[NCH];
  if (sides & 2) load_chunks<LPR, NCH>(a, a.v + w.off, nullptr, nullptr, 0, rv, tv, l);
  if (sides & 1) load_chunks<LPR, NCH>(a, a.k + w.off, w.gain, w.cos, w.pos, rk, tk, l);
  if (sides & 2)
    quantise_chunks<E4M3, LPR, NCH, false, false>(rv, a.D, 0.0, tv, a.vc + w.row * a.D, a.vs + w.row, l, ok);
  if (sides & 1) {
    uint8_t *codes = a.kc + w.row * a.D;
    float *scale = a.ks + w.row;
    if (a.k_gain)  // (ROT without a table: no chunk is marked)
      quantise_chunks<E4M3, LPR, NCH, true, true>(rk, a.D, a.eps, tk, codes, scale, l, ok);
    else if (a.cos)
      quantise_chunks<E4M3, LPR, NCH, false, true>(rk, a.D, 0.0, tk, codes, scale, l, ok);
    else
      quantise_chunks<E4M3, LPR, NCH, false, false>(rk, a.D, 0.0, tk, codes, scale, l, ok);
  }
}

// ---- query rows -------------------------------------------------------------
// Row r of a kv head's query rows is head r % G of token r / G. Eight lanes hold a
// row (lane l8 the float4 chunks l8 + 8 i), four rows a warp: head norm, rotary,
// and a power of two that brings its largest magnitude into [2^9, 2^10), where two
// f16 terms hold 22 bits of it. All 32 lanes call it; rows past the last are zero.
template <int D>
struct QRow {
  float4 v[D / 32];
  float factor;   // what a score of these values is multiplied by (log2 units, K's scale apart)
  int lim;        // last key seen whatever the tree says, -1: none
  uint64_t bits;  // tree bits
};

// What the float4 loads below need.
inline bool q_rows_vec(const Kv8Args &a) {
  auto al = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  return a.D % 32 == 0 && a.q_rs % 4 == 0 && al(a.q) && al(a.q_gain) &&
         (!a.cos || (a.rot % 8 == 0 && a.half % 4 == 0 && al(a.cos) && al(a.sin)));
}

template <int D>
__device__ __forceinline__ void load_q_row(const Kv8Args &a, int b, int kvh, int G, int r, int past, QRow<D> &o) {
  constexpr int NC = D / 32;
  const int l8 = threadIdx.x & 7;
  const bool valid = r < a.S * G;
  const int i = valid ? r / G : 0, h = kvh * G + (valid ? r % G : 0);
  const float *src = a.q + ((int64_t)b * a.S + i) * a.q_rs + (int64_t)h * D;
  const float *gain = a.q_gain ? a.q_gain + (int64_t)h * D : nullptr;
  const int64_t pos = token_pos(a, b, i, past);
  const bool turn = a.cos && pos >= 0 && pos < a.CAP;
  const int hr = a.rot >> 1;
  // The whole head in halves: a chunk's partner is NC / 2 chunks on, in this lane.
  const bool halves = turn && a.rot == D && !a.interleaved && NC % 2 == 0;
  constexpr int NH = NC / 2 > 0 ? NC / 2 : 1;
  float4 g4[NC], c4[NH], n4[NH];  // all loads ahead of the first use
#pragma unroll
  for (int u = 0; u < NC; u++) {
    o.v[u] = *reinterpret_cast<const float4 *>(src + 4 * (l8 + 8 * u));
    if (gain) g4[u] = *reinterpret_cast<const float4 *>(gain + 4 * (l8 + 8 * u));
  }
  if (halves) {
#pragma unroll
    for (int u = 0; u < NC / 2; u++) {
      const int64_t at = pos * a.half + 4 * (l8 + 8 * u);
      c4[u] = *reinterpret_cast<const float4 *>(a.cos + at);
      n4[u] = *reinterpret_cast<const float4 *>(a.sin + at);
    }
  }
  float inv = 1.f, pre = 1.f;
  if (gain) {
    auto squares = [&]() {
      float ss = 0.f;
#pragma unroll
      for (int u = 0; u < NC; u++)
        ss = fmaf(o.v[u].x, o.v[u].x, fmaf(o.v[u].y, o.v[u].y, fmaf(o.v[u].z, o.v[u].z, fmaf(o.v[u].w, o.v[u].w, ss))));
#pragma unroll
      for (int f = 1; f < 8; f <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, f);
      return ss;
    };
    float ss = squares();
    inv = 1.f / sqrtf(ss / D + (float)a.eps);
    // Rows whose squares leave fp32's comfortable range are first brought near 1.
    const bool wide = !(ss > 1e-30f && ss < 1e36f);
    if (__any_sync(0xffffffffu, wide)) {
      if (wide) pre = ss > 1.f ? 0x1p-100f : 0x1p100f;
#pragma unroll
      for (int u = 0; u < NC; u++) o.v[u].x *= pre, o.v[u].y *= pre, o.v[u].z *= pre, o.v[u].w *= pre;
      ss = squares();
      if (wide) inv = (float)(1.0 / sqrt((double)ss / D + a.eps * pre * pre));
    }
  }
  if (gain) {
#pragma unroll
    for (int u = 0; u < NC; u++) {
      o.v[u].x *= inv * g4[u].x, o.v[u].y *= inv * g4[u].y, o.v[u].z *= inv * g4[u].z, o.v[u].w *= inv * g4[u].w;
    }
  }
  if (halves) {
#pragma unroll
    for (int u = 0; u < NC / 2; u++) {
      const float4 c = c4[u], n = n4[u];
      const float4 x = o.v[u], y = o.v[u + NC / 2];
      o.v[u] = make_float4(x.x * c.x - y.x * n.x, x.y * c.y - y.y * n.y, x.z * c.z - y.z * n.z, x.w * c.w - y.w * n.w);
      o.v[u + NC / 2] =
          make_float4(y.x * c.x + x.x * n.x, y.y * c.y + x.y * n.y, y.z * c.z + x.z * n.z, y.w * c.w + x.w * n.w);
    }
  } else if (turn) {
#pragma unroll
    for (int u = 0; u < NC; u++) {
      const int d = 4 * (l8 + 8 * u);
      if (d >= a.rot) continue;
      const float x[4] = {o.v[u].x, o.v[u].y, o.v[u].z, o.v[u].w};
      const bool first = a.interleaved || d < hr;
      float c[4], sn[4], w[4], y[4];
      if (a.interleaved) {
        const float2 c2 = *reinterpret_cast<const float2 *>(a.cos + pos * a.half + (d >> 1));
        const float2 s2 = *reinterpret_cast<const float2 *>(a.sin + pos * a.half + (d >> 1));
        c[0] = c[1] = c2.x, c[2] = c[3] = c2.y;
        sn[0] = s2.x, sn[1] = -s2.x, sn[2] = s2.y, sn[3] = -s2.y;
        w[0] = x[1], w[1] = x[0], w[2] = x[3], w[3] = x[2];
      } else {  // the partner from memory again
        const int pi = first ? d : d - hr, e = first ? d + hr : d - hr;
        const float4 c4 = *reinterpret_cast<const float4 *>(a.cos + pos * a.half + pi);
        const float4 s4 = *reinterpret_cast<const float4 *>(a.sin + pos * a.half + pi);
        float4 w4 = *reinterpret_cast<const float4 *>(src + e);
        if (gain) {
          const float4 g4 = *reinterpret_cast<const float4 *>(gain + e);
          w4.x = w4.x * pre * (inv * g4.x), w4.y = w4.y * pre * (inv * g4.y);
          w4.z = w4.z * pre * (inv * g4.z), w4.w = w4.w * pre * (inv * g4.w);
        }
        c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w;
        const float sg = first ? 1.f : -1.f;
        sn[0] = sg * s4.x, sn[1] = sg * s4.y, sn[2] = sg * s4.z, sn[3] = sg * s4.w;
        w[0] = w4.x, w[1] = w4.y, w[2] = w4.z, w[3] = w4.w;
      }
#pragma unroll
      for (int k = 0; k < 4; k++) y[k] = x[k] * c[k] - w[k] * sn[k];
      o.v[u] = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
  float mx = 0.f;
#pragma unroll
  for (int u = 0; u < NC; u++) {
    if (!valid) o.v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(o.v[u].x), fabsf(o.v[u].y)), fmaxf(fabsf(o.v[u].z), fabsf(o.v[u].w))));
  }
#pragma unroll
  for (int f = 1; f < 8; f <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, f));
  // 2^(e-1) <= mx < 2^e (subnormals count as 2^-126, infinite rows as any), times
  // 2^(10 - e) in two steps, as either may leave the normal range alone.
  const int e = min(max((int)(__float_as_uint(mx) >> 23), 1), 254) - 126;
  const int e1 = (10 - e) / 2, e2 = 10 - e - e1;
  const float f1 = __uint_as_float((uint32_t)(127 + e1) << 23), f2 = __uint_as_float((uint32_t)(127 + e2) << 23);
#pragma unroll
  for (int u = 0; u < NC; u++)
    o.v[u] = make_float4(o.v[u].x * f1 * f2, o.v[u].y * f1 * f2, o.v[u].z * f1 * f2, o.v[u].w * f1 * f2);
  // Never 0 (a row of zeros under a scale below 2^-12 would come to less than the
  // smallest number): hidden scores are -inf before they are multiplied.
  o.factor = fmaxf(a.scale * LOG2E / f1 / f2, __uint_as_float(1u));
  o.lim = !valid ? -1 : (a.tree ? past - 1 : past + i);
  o.bits = valid && a.tree ? a.tree[(int64_t)b * a.S + i] : 0;
}

// Codes as f16 pairs, exactly. int8: the bits of 1024 + (c + 128) minus 1152 (the
// mask, the exponent and the sign flip are one three-input operation); e4m3: the
// hardware's conversion (cached rows never hold a NaN code).
__device__ __forceinline__ uint32_t pair_int8(uint32_t codes02) {  // codes in bytes 0 and 2
  const uint32_t u = (codes02 & 0x00ff00ffu) ^ 0x64806480u;
  return b2m::h2_as_u32(__hsub2(b2m::u32_as_h2(u), __half2half2(__ushort_as_half(0x6480))));
}
__device__ __forceinline__ uint32_t pair_e4m3(uint32_t codes01) {  // codes in bytes 0 and 1
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(codes01));
  return r;
}
__device__ __forceinline__ uint32_t pair_e4m3_hi(uint32_t codes23) {  // codes in bytes 2 and 3
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(codes23));
  return r;
}

// Word of four codes c0 .. c3 as two pairs: (c0, c1) and (c2, c3) for e4m3, (c0,
// c2) and (c1, c3) for int8 (what each takes the fewest operations for).
template <bool E4M3>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t &p, uint32_t &q) {
  if (E4M3) {
    p = pair_e4m3(w);
    q = pair_e4m3_hi(w);
  } else {
    p = pair_int8(w);
    q = pair_int8(w >> 8);
  }
}
// The order of a word's four values in expand4's pairs: position k holds value
// expand_order<E4M3>(k).
template <bool E4M3>
__host__ __device__ constexpr int expand_order(int k) {
  return E4M3 ? k : (k == 1 ? 2 : (k == 2 ? 1 : k));
}

// Words a, b of four codes each -> pairs (a_k, b_k), k = 0 .. 3.
template <bool E4M3>
__device__ __forceinline__ void expand_zip(uint32_t a, uint32_t b, uint32_t (&p)[4]) {
  if (E4M3) {
    const uint32_t x = b2m::prmt(a, b, 0x5140), y = b2m::prmt(a, b, 0x7362);  // a0 b0 a1 b1, a2 b2 a3 b3
    p[0] = pair_e4m3(x), p[1] = pair_e4m3_hi(x);
    p[2] = pair_e4m3(y), p[3] = pair_e4m3_hi(y);
  } else {
    const uint32_t x = b2m::prmt(a, b, 0x5410), y = b2m::prmt(a, b, 0x7632);  // a0 a1 b0 b1, a2 a3 b2 b3
    p[0] = pair_int8(x), p[1] = pair_int8(x >> 8);
    p[2] = pair_int8(y), p[3] = pair_int8(y >> 8);
  }
}

}  // namespace kv8

// The warp-level tensor-core kernel for few query rows per kv head
// (k_kv8_step.cu).
bool kv8_step_shape(const Kv8Args &a);
void launch_kv8_step(const Kv8Args &a, cudaStream_t s);
// The tcgen05 kernel for many rows (k_kv8_flash.cu), after launch_kv8_append.
bool kv8_flash_shape(const Kv8Args &a);
void launch_kv8_flash(const Kv8Args &a, cudaStream_t s);
