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
// The k best are kept per warp as a descending list of 32 keys; a key is the
// logit's order-preserving bits over the complement of its index, so equal
// logits fall to the lowest index. An entry is looked at only when it reaches
// a threshold that k entries of the CTA are known to reach, first from the
// threads' maxima of the first batch, then from the warps' lists. Such entries go
// to a buffer of the warp that is sorted and merged into its list when 32 are in
// it. No barrier stands in the loop.
//
// Bound by HBM: 4 V bytes per row are read once, about eight issue slots and
// one MUFU operation per entry. Measured on one B200, 1024 rows of 151936: 97 us
// without alternatives (6.4 TB/s), 116 us with k = 1, 131 us with k = 20 (issue
// slots 73% used); one row over a cluster of 16 CTAs 10.5 us with k = 20 (launch, cluster and the
// merge of the lists; its bytes would take 0.1 us).
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
constexpr int LP_VEC = 4;     // float4 loads of a thread per batch
constexpr int LP_FLUSH = 32;  // buffered keys of a warp that are worth a merge
constexpr int LP_BUF = LP_FLUSH - 1 + 32 * 4 * LP_VEC;  // what a flush leaves and one batch
constexpr int LP_CTAS = 4;    // resident per SM
constexpr int LP_MAX_CLUSTER = 16;  // above 8: opted in for the kernel
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

// The value of a key (-0 as +0; -inf for the key of a NaN or none).
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return o < 0x007fffffu ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// (maxima are never NaN; c or z is, for a row that has no distribution)
struct LpState {
  float m, c, z, w;
};

__device__ __forceinline__ LpState lp_join(LpState a, LpState b) {
  if (b.m > a.m) {
    const LpState t = a;
    a = b;
    b = t;
  }
  if (b.m == a.m) {
    a.c += b.c;
    a.z += b.z;
    a.w += b.w;
  } else {
    const float d = b.m - a.m, f = d < -200.f ? 0.f : expf(d);
    const float s = b.c + b.z;
    a.w += (b.w + fmaxf(d, -200.f) * s) * f;
    a.z += s * f;
  }
  return a;
}

// Sorts one key per lane into descending order (bitonic network).
template <class T>
__device__ __forceinline__ T warp_sort_desc(T v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const T o = __shfl_xor_sync(0xffffffffu, v, j);
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

// The 32 best of a descending list and one unordered key per lane, descending.
// Kept out of line: its 20 shuffle steps in every place that merges would push
// the loop out of the instruction cache (measured: 165 against 131 us for 1024
// rows of 151936 with k = 20).
__device__ __noinline__ u64 warp_take_in(u64 list, u64 key, int lane) {
  const u64 sorted = warp_sort_desc(key, lane);
  return __shfl_sync(0xffffffffu, list, 0) == 0 ? sorted : warp_merge_desc(list, sorted, lane);
}

// The largest value of the warp's lanes, NaN if one is NaN.
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

template <bool TOPK>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) logprobs_kernel(const LpArgs a) {
  b2m::pdl_launch_dependents();
  __shared__ LpState st[LP_WARPS], cta_state;
  __shared__ u64 lists[LP_WARPS][32], buf[TOPK ? LP_WARPS : 1][TOPK ? LP_BUF : 1];
  __shared__ volatile uint32_t known[2][LP_WARPS];
  cg::cluster_group cl = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int rank = (int)(blockIdx.x % a.cl);
  const int few = (a.k + LP_WARPS - 1) / LP_WARPS;  // k spread over the warps

  // The row a CTA walks: entries [j0, j1) in multiples of four, of which an
  // aligned float4 body [b0, tail0) in batches of LP_VEC float4 per thread; the
  // (at most three each) entries before and behind it go last. The next batch
  // is in flight while one is worked on. Offsets in a row fit 32 bits.
  constexpr int NV = 4 * LP_VEC, STEP = LP_THREADS * LP_VEC;
  const float *x = nullptr;
  int64_t j0 = 0, b0 = 0, tail0 = 0, j1 = 0;
  int nvec = 0;
  float nxt[NV], x_id = 0.f;
  auto load = [&](int v0) {
    const float4 *xv = reinterpret_cast<const float4 *>(x + b0);
#pragma unroll
    for (int i = 0; i < LP_VEC; i++) {
      const int at = v0 + i * LP_THREADS + tid;
      float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (at < nvec) q = __ldcs(xv + at);
      nxt[4 * i] = q.x, nxt[4 * i + 1] = q.y, nxt[4 * i + 2] = q.z, nxt[4 * i + 3] = q.w;
    }
  };
  // Goes to row r and requests its first batch and the given token's logit.
  auto start_row = [&](int64_t r) {
    x = a.x + r * a.ld;
    const int64_t per = ((a.V + a.cl - 1) / a.cl + 3) / 4 * 4;
    j0 = min(a.V, per * rank), j1 = min(a.V, j0 + per);
    b0 = min(j1, j0 + (int64_t)(((16 - (reinterpret_cast<uintptr_t>(x + j0) & 15)) & 15) >> 2));
    tail0 = b0 + ((j1 - b0) & ~(int64_t)3);
    nvec = (int)((tail0 - b0) >> 2);
    load(0);
    x_id = __int_as_float(0x7fc00000);
    if (a.ids && rank == 0 && tid == 0) {
      const int64_t id = a.ids[r];
      if (id >= 0 && id < a.V)
        x_id = x[id];
      else if (a.err)
        set_dev_error(a.err, B2M_DEVERR_INDEX);
    }
  };
  auto merge_lists = [&]() {
#pragma unroll
    for (int h = LP_WARPS / 2; h > 0; h >>= 1) {
      if (warp < h) lists[warp][lane] = warp_merge_desc(lists[warp][lane], lists[warp + h][lane], lane);
      __syncthreads();
    }
  };
  // Joins the states of `width` lanes, in the same order of operands in all.
  auto join_lanes = [&](LpState &q, int width) {
    for (int o = width / 2; o > 0; o >>= 1) {
      LpState t;
      t.m = __shfl_xor_sync(0xffffffffu, q.m, o);
      t.c = __shfl_xor_sync(0xffffffffu, q.c, o);
      t.z = __shfl_xor_sync(0xffffffffu, q.z, o);
      t.w = __shfl_xor_sync(0xffffffffu, q.w, o);
      q = lane & o ? lp_join(t, q) : lp_join(q, t);
    }
  };

  const int64_t r = blockIdx.x / a.cl;
  if (TOPK && tid < 2 * LP_WARPS) known[tid / LP_WARPS][tid % LP_WARPS] = 0;
  start_row(r);
  __syncthreads();
  {
    // The warp's lanes share one maximum s.m.
    LpState s{-INFINITY, 0.f, 0.f, 0.f};
    bool bad = false;
    u64 list = 0, thr = 0;  // 32 best keys of the warp; keys must beat thr
    float thr_val = -INFINITY;
    int count = 0;          // keys in the warp's buffer

    // Adds N values whose largest over the warp is bm; -inf values add nothing.
    auto add = [&](const float *v, auto nv, float bm) {
      constexpr int N = decltype(nv)::value;
      bad |= !(bm < INFINITY);  // NaN or +inf
      if (bm < s.m) {
#pragma unroll
        for (int i = 0; i < N; i++) {
          const float d = fmaxf(v[i] - s.m, -200.f), e = ex2f(d * LOG2E);
          s.z += e;
          s.w = fmaf(d, e, s.w);
        }
      } else if (bm > -INFINITY && bm < INFINITY) {  // a new or an equal maximum: rare after the first batches
        if (bm > s.m) {
          const float d = s.m - bm, f = d < -200.f ? 0.f : ex2f(d * LOG2E), t = s.c + s.z;
          s.w = t > 0.f ? (s.w + fmaxf(d, -200.f) * t) * f : 0.f;
          s.z = t * f;
          s.c = 0.f;
          s.m = bm;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
          const float d = fmaxf(v[i] - s.m, -200.f), e = ex2f(d * LOG2E);
          const bool top = v[i] == s.m;
          s.c += top ? 1.f : 0.f;
          s.z += top ? 0.f : e;
          s.w = fmaf(d, e, s.w);
        }
      }
    };
    auto set_thr = [&](u64 t) {
      thr = t;
      thr_val = key_value(t);
    };
    // Merges the last 32 buffered keys (or all, if fewer) into the list and
    // tells the other warps which values k / LP_WARPS and k of its keys reach.
    auto flush = [&]() {
      __syncwarp();
      const int from = max(0, count - 32);
      const u64 key = from + lane < count ? buf[warp][from + lane] : 0;
      count = from;
      list = warp_take_in(list, key, lane);
      if (lane == few - 1) known[0][warp] = max(known[0][warp], (uint32_t)(list >> 32));
      if (lane == a.k - 1) known[1][warp] = max(known[1][warp], (uint32_t)(list >> 32));
      const u64 kth = __shfl_sync(0xffffffffu, list, a.k - 1);
      if (kth > thr) set_thr(kth);
      __syncwarp();
    };
    // Buffers the lanes' entries that `ok` marks and that beat the threshold.
    auto push = [&](bool ok, float v, uint32_t index) {
      const u64 key = make_key(v, index);
      ok = ok && key > thr;
      const unsigned take = __ballot_sync(0xffffffffu, ok);
      if (ok) buf[warp][count + __popc(take & ((1u << lane) - 1))] = key;
      count += __popc(take);
    };

    for (int v0 = 0; v0 == 0 || v0 < nvec; v0 += STEP) {
      float cur[NV];
#pragma unroll
      for (int i = 0; i < NV; i++) cur[i] = nxt[i];
      if (v0 + STEP < nvec) load(v0 + STEP);
      float lm = cur[0];
#pragma unroll
      for (int i = 1; i < NV; i++) lm = max_nan(lm, cur[i]);
      const float bm = warp_max_nan(lm);
      add(cur, std::integral_constant<int, NV>{}, bm);
      if (TOPK) {
        if (v0 == 0) {
          // What the threads' best entries tell (those without an entry, or
          // with a NaN, count as none).
          const bool any = tid < nvec && lm == lm && lm > -INFINITY;
          const uint32_t best = warp_sort_desc(any ? order_bits(lm) : 0u, lane);
          if (lane == few - 1) known[0][warp] = best;
          if (lane == a.k - 1) known[1][warp] = best;
          __syncwarp();
        }
        // Values that k entries of the CTA are known to reach: what k / LP_WARPS
        // keys of every warp reach, or k keys of one. Keys with such a value,
        // whatever their index, beat the threshold.
        const uint32_t lo = __reduce_min_sync(0xffffffffu, known[0][lane % LP_WARPS]);
        const uint32_t hi = max(lo, __reduce_max_sync(0xffffffffu, known[1][lane % LP_WARPS]));
        if (hi && ((u64)hi << 32) - 1 > thr) set_thr(((u64)hi << 32) - 1);
        if (!(bm < thr_val)) {
          const bool nans = bm != bm && thr <= 0xffffffffu;  // so far fewer than k numbers: NaNs count
#pragma unroll
          for (int i = 0; i < NV; i++) {
            const int at = v0 + (i >> 2) * LP_THREADS + tid;
            const bool ok = (cur[i] >= thr_val || nans) && at < nvec;
            if (__any_sync(0xffffffffu, ok)) push(ok, cur[i], (uint32_t)(b0 + 4 * (int64_t)at + (i & 3)));
          }
          while (count >= LP_FLUSH) flush();
        }
      }
    }
    if (warp == 0) {
      const int nhead = (int)(b0 - j0), nrest = nhead + (int)(j1 - tail0);
      const int64_t j = lane < nhead ? j0 + lane : tail0 + (lane - nhead);
      const float v[1] = {lane < nrest ? x[j] : -INFINITY};
      add(v, std::integral_constant<int, 1>{}, warp_max_nan(v[0]));
      if (TOPK) push(lane < nrest, v[0], (uint32_t)j);
    }
    // Lanes, then warps, then the cluster's CTAs, each in a fixed order.
    if (TOPK)
      while (count > 0) flush();
    if (bad) s.c = __int_as_float(0x7fc00000);
    join_lanes(s, 32);
    if (lane == 0) st[warp] = s;
    if (TOPK) lists[warp][lane] = list;
    __syncthreads();
    if (TOPK) merge_lists();
    if (warp == 0) {
      LpState q{-INFINITY, 0.f, 0.f, 0.f};
      if (lane < LP_WARPS) q = st[lane];
      join_lanes(q, LP_WARPS);
      if (lane == 0) cta_state = q;
    }
    if (a.cl > 1)
      cl.sync();
    else
      __syncthreads();
    if (rank == 0) {
      if (TOPK && a.cl > 1) {
        const u64 *mine = &lists[0][0];  // rank q's list is its lists[0]
        u64 best = warp < a.cl ? cl.map_shared_rank(mine, warp)[lane] : 0;
        if (warp + LP_WARPS < a.cl)
          best = warp_merge_desc(best, cl.map_shared_rank(mine, warp + LP_WARPS)[lane], lane);
        __syncthreads();  // warp 0 has read this CTA's own
        lists[warp][lane] = best;
        __syncthreads();
        merge_lists();
      }
      if (warp == 0) {
        LpState t{-INFINITY, 0.f, 0.f, 0.f};
        if (lane < a.cl) t = *cl.map_shared_rank(&cta_state, lane);
        join_lanes(t, LP_MAX_CLUSTER);
        // A row with a NaN or +inf entry, or with nothing above -inf, has no
        // distribution: NaN, as the formula gives.
        t.m = __shfl_sync(0xffffffffu, t.m, 0);
        t.c = __shfl_sync(0xffffffffu, t.c, 0);
        t.z = __shfl_sync(0xffffffffu, t.z, 0);
        const double rest = (double)t.c - 1.0 + (double)t.z, ln = log1p(rest);
        const bool none = !(t.c > 0.f);
        const float lz = none ? __int_as_float(0x7fc00000) : (float)ln;
        if (lane == 0) {
          if (a.ids) a.logprob[r] = (x_id - t.m) - lz;
          if (a.entropy) a.entropy[r] = none ? lz : (float)(ln - (double)t.w / (1.0 + rest));
        }
        if (TOPK && lane < a.k) {
          const u64 key = lists[0][lane];
          a.top_ids[r * a.k + lane] = key_index(key);
          if (a.top_lp) a.top_lp[r * a.k + lane] = (key_value(key) - t.m) - lz;
        }
      }
    }
    if (a.cl > 1) cl.sync();  // rank 0 has read the others' shared memory
  }
}

// CTAs per row (one cluster): enough for two per SM, each with at least 4096
// entries.
int lp_cluster(int64_t rows, int64_t V) {
  int c = 1;
  while (c < LP_MAX_CLUSTER && rows * c < 2 * b2m::device_sm_count() && V / (2 * c) >= 4096) c *= 2;
  return c;
}

}  // namespace

void launch_logprobs(const float *x, int64_t ld, const int64_t *ids, int64_t rows, int64_t V, float *logprob,
                     float *entropy, int k, int64_t *top_ids, float *top_lp, int32_t *err, cudaStream_t s) {
  if (rows == 0) return;
  B2M_REQUIRE(rows <= 0x7fffffff / LP_MAX_CLUSTER, B2M_ERR_INVALID_ARGUMENT, "LogProbs: too many rows in one call");
  LpArgs a{x, ld, ids, rows, V, logprob, entropy, k, top_ids, top_lp, err, lp_cluster(rows, V)};
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
  if (k > 0) {
    b2m::allow_large_cluster_once<logprobs_kernel<true>>();
    B2M_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, a));
  } else {
    b2m::allow_large_cluster_once<logprobs_kernel<false>>();
    B2M_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, a));
  }
}
