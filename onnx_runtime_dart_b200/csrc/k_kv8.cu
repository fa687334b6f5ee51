// 8-bit KV cache: quantised append, read-back, the move of accepted rows, the
// fp32 attention kernel, and the choice between the attention kernels. The
// format is described in kv8_common.cuh.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"

namespace {

using namespace kv8;
using b2m::pdl_launch_dependents;
using b2m::set_dev_error;

// Appends the call's keys and values, one warp per (token, kv head) and side.
__global__ void __launch_bounds__(256) kv8_append_kernel(const Kv8Args a) {
  pdl_launch_dependents();
  __shared__ float stage[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + warp;
  if (item >= (int64_t)a.B * a.S * a.KVH * 2) return;
  const int side = (int)(item & 1);
  const int kvh = (int)((item >> 1) % a.KVH);
  const int64_t bs = (item >> 1) / a.KVH;
  const int i = (int)(bs % a.S), b = (int)(bs / a.S);
  append_row(a, b, i, kvh, side, a.past[b], stage[warp], lane);
}

// The same for rows of whole float4s: half a warp per (token, kv head), both
// sides. Bound by issue slots, not by memory (8 D bytes in, 2 D + 8 out): what a
// row costs beside its elements (the norm factor, the maximum in double) is paid
// once for two rows. 16376 tokens of 8 kv heads of 128, normed and rotated, 73 us
// (2.3 TB/s, issue slots 65% used; 103 us with a warp per row; floor 26).
template <bool E4M3, int NCH>
__global__ void __launch_bounds__(256, NCH == 4 ? 1 : 3) kv8_append_vec_kernel(const Kv8Args a) {
  pdl_launch_dependents();
  const unsigned item = blockIdx.x * 16 + (threadIdx.x >> 4);  // (token, kv head): the launcher keeps it below 2^31
  if ((item & ~1u) >= (unsigned)a.S * (unsigned)a.KVH) return;  // the whole warp
  const unsigned i = item / (unsigned)a.KVH;
  const int b = blockIdx.y;
  append_vec<E4M3, 16, NCH>(a, b, (int)i, (int)(item - i * a.KVH), 3, a.past[b], i < (unsigned)a.S);
}

// The values of n cached positions from start[b] (or 0) on, [B][KVH][n][D]
// fp32: one warp per row. Bound by the stores (8 D bytes for 2 D + 8 read): 34 us
// for 16376 tokens of 8 heads of 128, 5.0 TB/s; 52 us with one code a lane.
template <bool E4M3>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Args a, const int32_t *start, int n, float *k_out,
                                                       float *v_out) {
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + warp;
  if (item >= (int64_t)a.B * a.KVH * n) return;
  const int j = (int)(item % n);
  const int64_t bk = item / n;
  const int64_t pos = (int64_t)(start ? start[bk / a.KVH] : 0) + j;
  if (pos < 0 || pos >= a.CAP) {
    if (lane == 0 && a.err) set_dev_error(a.err, B2M_DEVERR_INDEX);
    return;
  }
  const int64_t row = bk * a.CAP + pos;
  // Four codes a lane where both ends allow it, all loads ahead of the stores.
  auto al16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  if ((a.D & 3) == 0 && al16(k_out) && al16(v_out)) {
    uint32_t w[2][2];
    float s[2];
#pragma unroll
    for (int side = 0; side < 2; side++) {
      if (!(side ? v_out : k_out)) continue;
      s[side] = (side ? a.vs : a.ks)[row];
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (4 * (lane + 32 * u) < a.D)
          w[side][u] = reinterpret_cast<const uint32_t *>((side ? a.vc : a.kc) + row * a.D)[lane + 32 * u];
    }
#pragma unroll
    for (int side = 0; side < 2; side++) {
      float *out = side ? v_out : k_out;
      if (!out) continue;
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (4 * (lane + 32 * u) < a.D) {
          const uint32_t c = w[side][u];
          float4 v;
          v.x = code_value<E4M3>((uint8_t)c) * s[side], v.y = code_value<E4M3>((uint8_t)(c >> 8)) * s[side];
          v.z = code_value<E4M3>((uint8_t)(c >> 16)) * s[side], v.w = code_value<E4M3>((uint8_t)(c >> 24)) * s[side];
          reinterpret_cast<float4 *>(out + item * a.D)[lane + 32 * u] = v;
        }
    }
    return;
  }
#pragma unroll
  for (int side = 0; side < 2; side++) {
    float *out = side ? v_out : k_out;
    if (!out) continue;
    const uint8_t *codes = (side ? a.vc : a.kc) + row * a.D;
    const float s = (side ? a.vs : a.ks)[row];
    for (int d = lane; d < a.D; d += 32) out[item * a.D + d] = code_value<E4M3>(codes[d]) * s;
  }
}

// Moves rows past + path[j] to past + j for j < count, one warp per (layer,
// sequence, kv head) and side. The path is strictly increasing with path[j] >=
// j, so a run of rows can be read whole and then written: no later row is read
// from where an earlier one went. A path that is not (or a count outside [0, n])
// moves nothing and raises the device error. A row's latency is what it costs
// (one row at a time took 20 us for 30 rows of two sequences; runs of 16: 4 us).
__global__ void __launch_bounds__(256) kv8_keep_kernel(const Kv8Args a, int layers, const int32_t *path,
                                                       const int32_t *count, int n) {
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + warp;
  if (item >= (int64_t)layers * a.B * a.KVH * 2) return;
  const int side = (int)(item & 1);
  const int64_t lbk = item >> 1;  // (layer * B + b) * KVH + kvh
  const int b = (int)((lbk / a.KVH) % a.B);
  const int past = a.past[b], c = count[b];
  const int32_t *p = path + (int64_t)b * n;
  bool bad = past < 0 || c < 0 || c > n || (c > 0 && (int64_t)past + p[c - 1] >= a.CAP);
  if (!bad)
    for (int j = lane; j < c; j += 32) bad |= p[j] < j || p[j] >= n || (j > 0 && p[j] <= p[j - 1]);
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0 && a.err) set_dev_error(a.err, B2M_DEVERR_INDEX);
    return;
  }
  uint8_t *codes = side ? a.vc : a.kc;
  float *scale = side ? a.vs : a.ks;
  const int64_t base = lbk * a.CAP + past;
  constexpr int RUN = 16;
  const bool vec = (a.D & 15) == 0 && (reinterpret_cast<uintptr_t>(codes) & 15) == 0;
  for (int j0 = 0; j0 < c; j0 += RUN) {
    const int m = min(RUN, c - j0);
    const float sc = lane < m ? scale[base + p[j0 + lane]] : 0.f;
    if (vec) {
      const int nv = a.D >> 4, items = m * nv;  // 16-byte pieces: at most RUN * 16
      uint4 r[RUN * 16 / 32];
#pragma unroll
      for (int u = 0; u < RUN * 16 / 32; u++) {
        const int it = lane + 32 * u;
        if (it < items)
          r[u] = reinterpret_cast<const uint4 *>(codes + (base + p[j0 + it / nv]) * a.D)[it % nv];
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < RUN * 16 / 32; u++) {
        const int it = lane + 32 * u;
        if (it < items) reinterpret_cast<uint4 *>(codes + (base + j0 + it / nv) * a.D)[it % nv] = r[u];
      }
    } else {
      for (int j = j0; j < j0 + m; j++) {
        const int64_t from = base + p[j], to = base + j;
        if (from != to)
          for (int d = lane; d < a.D; d += 32) codes[to * a.D + d] = codes[from * a.D + d];
        __syncwarp();
      }
    }
    __syncwarp();
    if (lane < m) scale[base + j0 + lane] = sc;
    __syncwarp();
  }
}

// Whether new token i of sequence b sees key j (past = cached positions).
__device__ __forceinline__ bool sees(const Kv8Args &a, int j, int past, int i, uint64_t bits) {
  if (!a.tree) return j <= past + i;
  return j < past || (j - past < 64 && (bits >> (j - past) & 1));
}

// Attention in fp32 on the CUDA cores, any head_dim <= 256: CTA per (token,
// query head, sequence), its eight warps taking keys in turn with an online
// softmax each, merged in shared memory in warp order.
template <bool E4M3>
__global__ void __launch_bounds__(256) kv8_attend_kernel(const Kv8Args a) {
  pdl_launch_dependents();
  __shared__ float qs[256], wo[8][256], wm[8], wl[8];
  __shared__ double sums[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int kvh = h / (a.H / a.KVH), D = a.D;
  const int past = min(max(0, a.past[b]), a.CAP);  // (an append past either has raised its error)
  const int64_t pos = token_pos(a, b, i, past);
  float x = tid < D ? a.q[((int64_t)b * a.S + i) * a.q_rs + (int64_t)h * D + tid] : 0.f;
  if (a.q_gain) {
    const double ss = warp_sum_d((double)x * x);
    if (lane == 0) sums[warp] = ss;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < 8; w++) t += sums[w];
    if (tid < D) x = (float)((double)x * (1.0 / sqrt(t / D + a.eps)) * a.q_gain[(int64_t)h * D + tid]);
  }
  qs[tid] = x;
  __syncthreads();
  if (a.cos && pos >= 0 && pos < a.CAP && tid < a.rot) {
    const int hr = a.rot >> 1;
    const bool first = a.interleaved ? (tid & 1) == 0 : tid < hr;
    const int pi = a.interleaved ? tid >> 1 : (first ? tid : tid - hr);
    const int e = a.interleaved ? (tid ^ 1) : (first ? tid + hr : tid - hr);
    const float c = a.cos[pos * a.half + pi], sn = a.sin[pos * a.half + pi], w = qs[e];
    x = first ? x * c - w * sn : x * c + w * sn;
  }
  __syncthreads();
  qs[tid] = x * a.scale;
  __syncthreads();
  float q[8], o[8];
#pragma unroll
  for (int u = 0; u < 8; u++) {
    q[u] = lane + 32 * u < D ? qs[lane + 32 * u] : 0.f;
    o[u] = 0.f;
  }
  const uint64_t bits = a.tree ? a.tree[(int64_t)b * a.S + i] : 0;
  const int kend = (int)min((int64_t)a.CAP, (int64_t)past + (a.tree ? a.S : i + 1));
  const int64_t base = ((int64_t)b * a.KVH + kvh) * a.CAP;
  float m = -INFINITY, l = 0.f;
  for (int j = warp; j < kend; j += 8) {
    if (!sees(a, j, past, i, bits)) continue;
    const uint8_t *kr = a.kc + (base + j) * D, *vr = a.vc + (base + j) * D;
    float t = 0.f;
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (lane + 32 * u < D) t = fmaf(q[u], code_value<E4M3>(kr[lane + 32 * u]), t);
#pragma unroll
    for (int of = 16; of > 0; of >>= 1) t += __shfl_xor_sync(0xffffffffu, t, of);
    t *= a.ks[base + j];
    const float mn = fmaxf(m, t);
    const float corr = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(t - mn);
    const float pv = p * a.vs[base + j];
    l = l * corr + p;
    m = mn;
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (lane + 32 * u < D) o[u] = fmaf(pv, code_value<E4M3>(vr[lane + 32 * u]), o[u] * corr);
  }
  if (lane == 0) {
    wm[warp] = m;
    wl[warp] = l;
  }
#pragma unroll
  for (int u = 0; u < 8; u++) wo[warp][lane + 32 * u] = o[u];
  __syncthreads();
  if (tid >= D) return;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int w = 0; w < 8; w++) M = fmaxf(M, wm[w]);
  for (int w = 0; w < 8; w++) {
    // l == 0: this warp saw no key (its l is NaN, not 0, when a score was NaN)
    const float f = wl[w] == 0.f ? 0.f : (wm[w] == -INFINITY ? 1.f : __expf(wm[w] - M));
    L += wl[w] * f;
    O += wo[w][tid] * f;
  }
  const float r = L == 0.f ? 0.f : O / L;  // a token that sees nothing: zeros
  const int64_t at = ((int64_t)b * a.S + i) * a.H * D + (int64_t)h * D + tid;
  if (a.out) a.out[at] = r;
  if (a.out16) a.out16[at] = __float2half_rn(r);
}

unsigned blocks_for(int64_t items, int per) {
  const int64_t g = (items + per - 1) / per;
  B2M_REQUIRE(g <= 0x7fffffff, B2M_ERR_INVALID_ARGUMENT, "8-bit KV cache: too many rows in one call");
  return (unsigned)g;
}

}  // namespace

void launch_kv8_append(const Kv8Args &a, cudaStream_t s) {
  const int64_t items = (int64_t)a.B * a.S * a.KVH * 2;
  if (items == 0) return;
  if (append_rows_vec(a) && (int64_t)a.S * a.KVH < ((int64_t)1 << 31) && a.B <= 65535) {
    const dim3 grid((unsigned)(((int64_t)a.S * a.KVH + 15) / 16), (unsigned)a.B);
    auto kern = a.D <= 64 ? (a.e4m3 ? kv8_append_vec_kernel<true, 1> : kv8_append_vec_kernel<false, 1>)
                : a.D <= 128 ? (a.e4m3 ? kv8_append_vec_kernel<true, 2> : kv8_append_vec_kernel<false, 2>)
                             : (a.e4m3 ? kv8_append_vec_kernel<true, 4> : kv8_append_vec_kernel<false, 4>);
    kern<<<grid, 256, 0, s>>>(a);
    B2M_CUDA(cudaGetLastError());
    return;
  }
  kv8_append_kernel<<<blocks_for(items, 8), 256, 0, s>>>(a);
  B2M_CUDA(cudaGetLastError());
}

void launch_kv8_read(const Kv8Args &a, const int32_t *start, int n, float *k_out, float *v_out, cudaStream_t s) {
  const int64_t items = (int64_t)a.B * a.KVH * n;
  if (items == 0) return;
  if (a.e4m3)
    kv8_read_kernel<true><<<blocks_for(items, 8), 256, 0, s>>>(a, start, n, k_out, v_out);
  else
    kv8_read_kernel<false><<<blocks_for(items, 8), 256, 0, s>>>(a, start, n, k_out, v_out);
  B2M_CUDA(cudaGetLastError());
}

void launch_kv8_keep(const Kv8Args &a, int layers, const int32_t *path, const int32_t *count, int n, cudaStream_t s) {
  const int64_t items = (int64_t)layers * a.B * a.KVH * 2;
  if (items == 0 || n == 0) return;
  kv8_keep_kernel<<<blocks_for(items, 8), 256, 0, s>>>(a, layers, path, count, n);
  B2M_CUDA(cudaGetLastError());
}

void launch_kv8_attend(const Kv8Args &a, bool exact, cudaStream_t s) {
  if (!exact && kv8_flash_shape(a)) {
    launch_kv8_append(a, s);
    launch_kv8_flash(a, s);
    return;
  }
  if (!exact && kv8_step_shape(a)) {
    launch_kv8_step(a, s);
    return;
  }
  launch_kv8_append(a, s);
  const dim3 grid((unsigned)a.S, (unsigned)a.H, (unsigned)a.B);
  if (a.e4m3)
    kv8_attend_kernel<true><<<grid, 256, 0, s>>>(a);
  else
    kv8_attend_kernel<false><<<grid, 256, 0, s>>>(a);
  B2M_CUDA(cudaGetLastError());
}
