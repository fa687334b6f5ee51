// Log probabilities of given tokens, entropy and the k likeliest tokens of
// rows of logits, in one pass over each row.
//
// A state (m, c, z, w) stands for a set of logits: m the maximum, c how many
// entries equal it, z = sum of e^(x-m) over the others and w = sum of
// (x-m) e^(x-m). Then
//   ln sum e^x = m + log1p(c - 1 + z),   entropy = log1p(c - 1 + z) - w / (c + z),
// and keeping the maximum's own 1s out of z keeps the log probability of a
// confident row, which 1 + z would lose below 2^-24. Two states join by moving
// the lower one to the higher maximum.
//
// The k best are kept per warp as 32 keys, one per lane in descending order;
// a key is the logit's order-preserving bits over the complement of its index,
// so equal logits fall to the lowest index. An entry is looked at only when
// it beats a threshold that k entries seen by the CTA already reach.
//
// Bound by HBM: 4 V bytes per row are read once, about ten ALU and one MUFU
// instruction per entry.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "b2m_internal.cuh"
#include "ptx.cuh"
#include "tc_common.cuh"

namespace {

namespace cg = cooperative_groups;
using b2m::set_dev_error;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_VEC = 4;  // float4 loads of a thread per batch
typedef unsigned long long u64;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Bits whose unsigned order is the order of the values; -0 as +0, NaN lowest.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t r = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x != x ? 0u : r;
}
__device__ __forceinline__ u64 make_key(float x, uint32_t idx) {
  return ((u64)order_bits(x) << 32) | (u64)(0xffffffffu - idx);
}
__device__ __forceinline__ uint32_t key_index(u64 k) { return 0xffffffffu - (uint32_t)k; }

struct LpState {
  float m, c, z, w;
};

__device__ __forceinline__ LpState lp_join(LpState a, LpState b) {
  if (!(a.m >= b.m)) {  // also when a is NaN: then the result's maximum is b's, marked below
    const LpState t = a;
    a = b;
    b = t;
  }
  if (b.m == a.m) {
    a.c += b.c;
    a.z += b.z;
    a.w += b.w;
  } else if (b.c > 0.f) {
    const float d = b.m - a.m, f = d < -200.f ? 0.f : expf(d);
    const float s = b.c + b.z;
    a.w += (b.w + fmaxf(d, -200.f) * s) * f;
    a.z += s * f;
  }
  return a;
}

// Sorts one key per lane into descending order (bitonic network).
__device__ __forceinline__ u64 warp_sort_desc(u64 v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const u64 o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool up = (lane & k) != 0;  // this run ascends (never at k == 32)
      const bool low = (lane & j) == 0;
      v = (low != up) ? max(v, o) : min(v, o);
    }
  return v;
}

// The 32 best of two descending lists, descending.
__device__ __forceinline__ u64 warp_merge_desc(u64 a, u64 b, int lane) {
  u64 v = max(a, __shfl_xor_sync(0xffffffffu, b, 31));  // a[i] against b[31 - i]: a bitonic sequence
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const u64 o = __shfl_xor_sync(0xffffffffu, v, j);
    v = (lane & j) == 0 ? max(v, o) : min(v, o);
  }
  return v;
}

struct LpArgs {
  const float *x;
  int64_t ld;
  const int64_t *ids;
  int64_t rows, V;
  float *logprob, *entropy;
  int k;
  int64_t *top_ids;
  float *top_lp;
  int32_t *err;
  int cl;  // CTAs (one cluster) per row
};

template <bool TOPK>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const LpArgs a) {
  b2m::pdl_launch_dependents();
  __shared__ LpState st[LP_WARPS];
  __shared__ u64 lists[LP_WARPS][32];
  __shared__ u64 thr_sh;
  __shared__ LpState cta_state;
  __shared__ int bad_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int rank = (int)(blockIdx.x % a.cl);
  const int64_t r = blockIdx.x / a.cl;
  const float *x = a.x + r * a.ld;
  if (tid == 0) {
    thr_sh = 0;
    bad_sh = 0;
  }
  __syncthreads();
  // This CTA's entries [j0, j1): chunks in multiples of four.
  const int64_t per = ((a.V + a.cl - 1) / a.cl + 3) / 4 * 4;
  const int64_t j0 = min(a.V, per * rank), j1 = min(a.V, j0 + per);
  // Aligned float4 body; the entries before and behind it go one by one.
  const int64_t mis = ((16 - (reinterpret_cast<uintptr_t>(x + j0) & 15)) & 15) >> 2;
  const int64_t b0 = min(j1, j0 + mis), nvec = (j1 - b0) >> 2, tail0 = b0 + 4 * nvec;
  const float4 *xv = reinterpret_cast<const float4 *>(x + b0);

  LpState s{-INFINITY, 0.f, 0.f, 0.f};
  bool bad = false;
  u64 list = 0, thr = 0;  // keys must beat thr

  // N values of this lane (index base + 4 * (i / 4) * stride + i % 4), those
  // at or past `valid` being -inf fillers that are never chosen.
  auto take = [&](const float *v, auto nv, auto index, auto valid, bool first) {
    constexpr int NV = decltype(nv)::value;
    float bm = v[0];
#pragma unroll
    for (int i = 1; i < NV; i++) bm = max_nan(bm, v[i]);
    bad |= !(bm < INFINITY);
    const float mn = fmaxf(s.m, bm);
    if (mn > -INFINITY && mn < INFINITY) {
      if (mn > s.m) {  // rare after the first batches
        const float d = s.m - mn, f = d < -200.f ? 0.f : ex2f(d * LOG2E), t = s.c + s.z;
        s.w = t > 0.f ? (s.w + fmaxf(d, -200.f) * t) * f : 0.f;
        s.z = t * f;
        s.c = 0.f;
        s.m = mn;
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const float d = fmaxf(v[i] - s.m, -200.f), e = ex2f(d * LOG2E);
        const bool top = v[i] == s.m;
        s.c += top ? 1.f : 0.f;
        s.z += top ? 0.f : e;
        s.w = fmaf(d, e, s.w);
      }
    }
    if (TOPK) {
      if (first) {
        // The k-th best of the lanes' best: k entries reach it.
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < NV; i++)
          if (valid(i)) best = max(best, make_key(v[i], index(i)));
        const u64 kth = __shfl_sync(0xffffffffu, warp_sort_desc(best, lane), a.k - 1);
        thr = kth ? kth - 1 : 0;
      }
      const u64 shared_thr = *reinterpret_cast<volatile u64 *>(&thr_sh);
      thr = max(thr, shared_thr);
      const bool want = bm != bm || order_bits(bm) >= (uint32_t)(thr >> 32);
      if (__any_sync(0xffffffffu, want)) {
        bool grew = false;
#pragma unroll 1
        for (int i = 0; i < NV; i++) {
          float vi = v[0];
#pragma unroll
          for (int u = 1; u < NV; u++) vi = u == i ? v[u] : vi;
          u64 key = valid(i) ? make_key(vi, index(i)) : 0;
          unsigned todo = __ballot_sync(0xffffffffu, key > thr);
          while (todo) {
            const int src = __ffs(todo) - 1;
            const u64 nk = __shfl_sync(0xffffffffu, key, src);
            const int at = __popc(__ballot_sync(0xffffffffu, list > nk));
            const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
            list = lane < at ? list : (lane == at ? nk : up);
            const u64 kth = __shfl_sync(0xffffffffu, list, a.k - 1);
            if (kth > thr) {
              // the list's k-th entry is in the list: later keys must beat it
              thr = kth;
              grew = true;
            }
            if (lane == src) key = 0;
            todo = __ballot_sync(0xffffffffu, key > thr);
          }
        }
        if (grew && lane == 0) atomicMax(&thr_sh, thr - 1);
      }
    }
  };

  // Body: batches of LP_VEC float4 per thread, the next batch in flight while
  // this one is worked on.
  constexpr int NV = 4 * LP_VEC;
  const int64_t step = (int64_t)LP_THREADS * LP_VEC;
  float nxt[NV];
  auto load = [&](int64_t v0) {
#pragma unroll
    for (int i = 0; i < LP_VEC; i++) {
      const int64_t at = v0 + (int64_t)i * LP_THREADS + tid;
      float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (at < nvec) q = __ldcs(xv + at);
      nxt[4 * i] = q.x, nxt[4 * i + 1] = q.y, nxt[4 * i + 2] = q.z, nxt[4 * i + 3] = q.w;
    }
  };
  if (nvec > 0) load(0);
  for (int64_t v0 = 0; v0 < nvec; v0 += step) {
    float cur[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) cur[i] = nxt[i];
    if (v0 + step < nvec) load(v0 + step);
    take(
        cur, std::integral_constant<int, NV>{},
        [&](int i) { return (uint32_t)(b0 + 4 * (v0 + (int64_t)(i >> 2) * LP_THREADS + tid) + (i & 3)); },
        [&](int i) { return v0 + (int64_t)(i >> 2) * LP_THREADS + tid < nvec; }, v0 == 0);
  }
  if (warp == 0) {  // at most three entries before the body and three behind it
    const int64_t nhead = b0 - j0, nrest = nhead + (j1 - tail0);
    const int64_t j = lane < nhead ? j0 + lane : tail0 + (lane - nhead);
    if (nrest > 0) {
      const float v[1] = {lane < nrest ? x[j] : -INFINITY};
      take(v, std::integral_constant<int, 1>{}, [&](int) { return (uint32_t)j; }, [&](int) { return lane < nrest; }, false);
    }
  }
  // Lanes, then warps, then the cluster's CTAs, each in a fixed order.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpState t;
    t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
    t.c = __shfl_xor_sync(0xffffffffu, s.c, o);
    t.z = __shfl_xor_sync(0xffffffffu, s.z, o);
    t.w = __shfl_xor_sync(0xffffffffu, s.w, o);
    s = lane & o ? lp_join(t, s) : lp_join(s, t);  // the same order of operands in both lanes
  }
  if (lane == 0) st[warp] = s;
  if (TOPK) lists[warp][lane] = list;
  if (bad) bad_sh = 1;
  __syncthreads();
  if (TOPK) {
#pragma unroll
    for (int h = LP_WARPS / 2; h > 0; h >>= 1) {
      if (warp < h) lists[warp][lane] = warp_merge_desc(lists[warp][lane], lists[warp + h][lane], lane);
      __syncthreads();
    }
  }
  if (tid == 0) {
    LpState t = st[0];
    for (int w = 1; w < LP_WARPS; w++) t = lp_join(t, st[w]);
    cta_state = t;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  if (rank == 0 && warp == 0) {
    LpState t = cta_state;
    int bd = bad_sh;
    u64 best = TOPK ? lists[0][lane] : 0;
    for (int q = 1; q < a.cl; q++) {
      t = lp_join(t, *cl.map_shared_rank(&cta_state, q));
      bd |= *cl.map_shared_rank(&bad_sh, q);
      if (TOPK) best = warp_merge_desc(best, cl.map_shared_rank(&lists[0][0], q)[lane], lane);
    }
    // A row with a NaN or +inf entry, or with nothing above -inf, has no
    // distribution: NaN, as the formula gives.
    const double rest = (double)t.c - 1.0 + (double)t.z;
    const bool none = bd || !(t.c > 0.f);
    const float lz = none ? __int_as_float(0x7fc00000) : (float)log1p(rest);
    if (lane == 0) {
      if (a.ids) {
        const int64_t id = a.ids[r];
        const bool in = id >= 0 && id < a.V;
        if (!in && a.err) set_dev_error(a.err, B2M_DEVERR_INDEX);
        a.logprob[r] = in ? (x[id] - t.m) - lz : __int_as_float(0x7fc00000);
      }
      if (a.entropy) a.entropy[r] = none ? lz : (float)(log1p(rest) - (double)t.w / (1.0 + rest));
    }
    if (TOPK && lane < a.k) {
      const uint32_t id = key_index(best);
      a.top_ids[r * a.k + lane] = id;
      if (a.top_lp) a.top_lp[r * a.k + lane] = (x[id] - t.m) - lz;
    }
  }
  cl.sync();  // rank 0 has read the others' shared memory
}

// CTAs per row: as many as bring the launch to about four per SM, a cluster of
// at most 16, each with at least 4096 entries.
int lp_cluster(int64_t rows, int64_t V) {
  int c = 1;
  while (c < 8 && rows * c < 2 * b2m::device_sm_count() && V / (2 * c) >= 4096) c *= 2;
  return c;
}

}  // namespace

void launch_logprobs(const float *x, int64_t ld, const int64_t *ids, int64_t rows, int64_t V, float *logprob,
                     float *entropy, int k, int64_t *top_ids, float *top_lp, int32_t *err, cudaStream_t s) {
  if (rows == 0) return;
  LpArgs a{x, ld, ids, rows, V, logprob, entropy, k, top_ids, top_lp, err, lp_cluster(rows, V)};
  B2M_REQUIRE(rows * a.cl <= 0x7fffffff, B2M_ERR_INVALID_ARGUMENT, "LogProbs: too many rows in one call");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * a.cl));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)a.cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (k > 0)
    B2M_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, a));
  else
    B2M_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, a));
}
