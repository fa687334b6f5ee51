// Attention over the 8-bit KV cache for few query rows per kv head: a decode
// step (the G query heads of a group), a small drafted tree or a short chunk.
//
// A cluster of CL CTAs serves one (kv head, sequence, tile of 8 NT query rows);
// its CTAs take consecutive key ranges, the four warps of a CTA 16-key tiles of
// its range in turn. Per tile a warp forms, with mma.m16n8k16 (f16 operands,
// fp32 sums),
//   S^T[16 keys][8 rows] = K . Q^T,   O^T[D][8 rows] += V^T . P^T.
// The codes are the A operands: int8 and e4m3 codes are f16 numbers exactly, so
// they are expanded in registers and the scales applied in fp32, K's to the
// scores and V's to the weights. Q and the weights are split into two f16 terms (22
// bits), so the products carry fp32 accuracy, for an f16 output too (one term of the
// weights would put 2.9e-4 of error where the output's own rounding is 2.1e-4). Which
// D index or key an MMA lane holds is free as long as both operands agree: lanes are
// given 16 consecutive bytes of a row, so no data is shuffled on its way to the tensor
// cores; only P^T is transposed between the two products (movmatrix).
//
// Should be bound by HBM (2 D + 8 bytes per key of a kv head): 64 sequences over
// 4096 .. 8191 positions of 8 kv heads take 176 us, 4.8 TB/s (floor 129); the warps'
// own chains (expand, product, exp2, product) and the part-empty last wave are the
// rest, issue slots 50% used. Each lane copies the bytes it will use itself into a
// ring of its own in shared memory (cp.async), two tiles ahead, so that enough
// loads are in flight without registers and no barrier is needed in the loop (when
// all took 168 us: one tile ahead 184, three 169; four CTAs per SM instead of three
// 184, six warps per CTA 185, eight 223).
//
// V scales are taken relative to the largest the warp has met (a power of two). A
// row's softmax reference goes by its own largest weight times V scale (weight_ref)
// and moves only when one passes 2^15, or in tiles with a V scale below 2^-8 (a warp
// vote). Warps, then the cluster's CTAs,
// merge in a fixed order through (distributed) shared memory: no workspace and
// no atomics, so captured graphs share nothing and results repeat.
#include <cooperative_groups.h>

#include <algorithm>

#include "kv8_common.cuh"
#include "tc_common.cuh"

namespace {

namespace cg = cooperative_groups;
using namespace kv8;

constexpr int ST_WARPS = 4, ST_THREADS = 32 * ST_WARPS, ST_STAGES = 3, ST_WINDOW = 16;

template <int N>
__device__ __forceinline__ void cp_async(void *dst, const void *src) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(b2m::smem_u32(dst)), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(b2m::smem_u32(dst)), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// D += A . B (m16n8k16, f16 operands, fp32 sums). Not volatile, so that the
// compiler may interleave independent products.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// How a row of D codes is dealt to the lanes: K rows in NKC chunks of KC bytes
// for each of four lanes, V rows in NVC chunks of VC bytes for each of eight.
template <int D>
struct StepShape {
  static_assert(D % 32 == 0 && D <= 256, "head dim");
  static constexpr int KC = D % 64 == 0 ? 16 : 8, NKC = D / (4 * KC), KW = KC / 4;
  static constexpr int VC = D % 128 == 0 ? 16 : (D % 64 == 0 ? 8 : 4), NVC = D / (8 * VC), VW = VC / 4;
  static constexpr int KSTEPS = D / 16, MT = D / 16;
  // One ring slot of a warp: K chunks [row half][chunk][lane], V chunks
  // [key slot][chunk][lane], one scale per lane.
  static constexpr int K_BYTES = 2 * NKC * 32 * KC, V_BYTES = 4 * NVC * 32 * VC, SLOT = K_BYTES + V_BYTES + 128;
};

template <int D, int NT>
struct StepSmem {
  static constexpr int R = 8 * NT;
  static constexpr int RING = 0;
  static constexpr int QF = RING + ST_WARPS * ST_STAGES * StepShape<D>::SLOT;  // Q fragments [NT][KSTEPS][32] uint4
  static constexpr int ROWS = QF + NT * StepShape<D>::KSTEPS * 512;            // per-row words, below
  // bits[R] (u64), factor[R], lim[R], wm[4][R], wl[4][R], cm[R], cl[R] (m: references)
  static constexpr int BYTES = ROWS + R * (8 + 4 + 4 + 16 + 16 + 8);
  // Warp states O [4][R][D] fp32 reuse the ring (drained by then).
  static_assert(ST_WARPS * R * D * 4 <= QF, "O staging fits the ring");
};

// (The CTAs per SM that the registers allow anyway, said to the compiler: 32 trees
// of 8 tokens 42 us, 45 .. 47 without; 48 with the totals of ST_WINDOW.)
template <bool E4M3, int D, int NT>
__global__ void __launch_bounds__(ST_THREADS, D <= 128 ? (NT == 1 ? 3 : 2) : 1)
    kv8_step_kernel(const Kv8Args a, const int fused_append) {
  using L = StepShape<D>;
  using M = StepSmem<D, NT>;
  constexpr int R = M::R;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t *rows_mem = smem + M::ROWS;
  uint64_t *row_bits = reinterpret_cast<uint64_t *>(rows_mem);
  float *row_factor = reinterpret_cast<float *>(rows_mem + 8 * R);
  int *row_lim = reinterpret_cast<int *>(rows_mem + 12 * R);
  float *wm = reinterpret_cast<float *>(rows_mem + 16 * R), *wl = wm + ST_WARPS * R, *cm = wl + ST_WARPS * R,
        *cl_ = cm + R;
  uint4 *qfrag = reinterpret_cast<uint4 *>(smem + M::QF);

  b2m::pdl_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int g = lane >> 2, t = lane & 3;
  const int row0 = (int)(blockIdx.x / CL) * R, kvh = blockIdx.y, b = blockIdx.z;
  const int G = a.H / a.KVH, nrows = a.S * G;
  const int past = min(max(0, a.past[b]), a.CAP);  // (an append past either has raised its error)
  // keys that the tile's last row sees
  const int n = (int)min((int64_t)a.CAP, (int64_t)past + (a.tree ? a.S : min(a.S, (row0 + R - 1) / G + 1)));
  const int chunk = (((n + CL - 1) / CL) + 15) & ~15;
  const int jbeg = min(n, rank * chunk), jend = min(n, jbeg + chunk);
  const int64_t base = ((int64_t)b * a.KVH + kvh) * a.CAP;

  // Ring of this warp.
  uint8_t *ring = smem + warp * (ST_STAGES * L::SLOT);
  const uint8_t *kcodes = a.kc + base * D, *vcodes = a.vc + base * D;
  const float *kscale = a.ks + base, *vscale = a.vs + base;
  const int ntile = (jend - jbeg + 15) >> 4;
  const uint8_t *kp0 = kcodes + (int64_t)(jbeg + g) * D + t * L::KC;
  const uint8_t *vp0 = vcodes + (int64_t)(jbeg + 2 * t) * D + g * L::VC;
  // lane t of a group: K scale of keys g, g + 8, V scale of keys g, g + 8
  const float *sp0 = (t & 2 ? vscale : kscale) + jbeg + g + 8 * (t & 1);
  auto issue = [&](int tile, int slot) {
    if (tile < ntile) {
      uint8_t *s = ring + slot * L::SLOT;
      const uint8_t *kp = kp0 + (int64_t)tile * (16 * D), *vp = vp0 + (int64_t)tile * (16 * D);
      const float *sp = sp0 + 16 * tile;
      // distances to the tile's other rows; in the last tile no further than its last row
      int kd = 8 * D, vd[4] = {0, D, 8 * D, 9 * D};  // keys 2t, 2t+1, 2t+8, 2t+9
      const int over = jbeg + 16 * tile + 16 - jend;
      if (over > 0) {
        const int left = 15 - over;  // index of the last row
        kp += (int64_t)min(0, left - g) * D;
        kd = (min(left, g + 8) - min(left, g)) * D;
        const int k0 = min(left, 2 * t);
        vp += (int64_t)(k0 - 2 * t) * D;
#pragma unroll
        for (int q = 1; q < 4; q++) vd[q] = (min(left, 2 * t + (q & 1) + 8 * (q >> 1)) - k0) * D;
        sp += min(0, left - g - 8 * (t & 1));
      }
#pragma unroll
      for (int hf = 0; hf < 2; hf++)
#pragma unroll
        for (int c = 0; c < L::NKC; c++)
          cp_async<L::KC>(s + ((hf * L::NKC + c) * 32 + lane) * L::KC, kp + hf * kd + c * 4 * L::KC);
#pragma unroll
      for (int q = 0; q < 4; q++)
#pragma unroll
        for (int c = 0; c < L::NVC; c++)
          cp_async<L::VC>(s + L::K_BYTES + ((q * L::NVC + c) * 32 + lane) * L::VC, vp + vd[q] + c * 8 * L::VC);
      cp_async<4>(s + L::K_BYTES + L::V_BYTES + lane * 4, sp);
    }
    cp_commit();
  };

  // The first tiles are on their way while the rows below are prepared (a tile
  // with rows that this call still appends waits for them). Of what came before
  // the append all is visible: the append was launched without an early start.
  int ahead = 0;
#pragma unroll
  for (int k = 0; k < ST_STAGES - 1; k++)
    if (ahead == k && jbeg + 16 * (warp + k * ST_WARPS) + 16 <= past) {
      issue(warp + k * ST_WARPS, k);
      ahead = k + 1;
    }
  // Work items of the prologue, dealt to the warps: the new rows of this CTA's
  // range (every rank appends its own, the last one also reports those past the
  // capacity), then groups of four query rows.
  {
    const int i0 = max(0, jbeg - past), i1 = !fused_append ? i0 : (rank == CL - 1 ? a.S : min(a.S, jend - past));
    const int nnew = 2 * max(0, i1 - i0);
#pragma unroll 1
    for (int it = warp; it < nnew + R / 4; it += ST_WARPS) {
      if (it < nnew) {
        append_vec<E4M3, 32, (D + 127) / 128>(a, b, i0 + (it >> 1), kvh, 1 << (it & 1), a.past[b], true);
      } else {
        const int rr = 4 * (it - nnew) + (lane >> 3);
        QRow<D> q;
        load_q_row<D>(a, b, kvh, G, row0 + rr, past, q);
#pragma unroll
        for (int u = 0; u < D / 32; u++) {
          // Fragment of values d .. d + 3: the k-step, and the lane of the row's
          // four, whose code words hold them.
          const int d = 4 * ((lane & 7) + 8 * u);
          const int ks = d / (4 * L::KC) * L::KW + d % L::KC / 4, t4 = d / L::KC % 4;
          const float v[4] = {q.v[u].x, q.v[u].y, q.v[u].z, q.v[u].w};
          const float4 x = make_float4(v[0], v[expand_order<E4M3>(1)], v[expand_order<E4M3>(2)], v[3]);
          const __half2 h0 = __floats2half2_rn(x.x, x.y), h1 = __floats2half2_rn(x.z, x.w);
          const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
          qfrag[((rr >> 3) * L::KSTEPS + ks) * 32 + (rr & 7) * 4 + t4] =
              make_uint4(b2m::h2_as_u32(h0), b2m::h2_as_u32(h1),
                         b2m::h2_as_u32(__floats2half2_rn(x.x - f0.x, x.y - f0.y)),
                         b2m::h2_as_u32(__floats2half2_rn(x.z - f1.x, x.w - f1.y)));
        }
        if ((lane & 7) == 0) {
          row_factor[rr] = q.factor;
          row_lim[rr] = q.lim;
          row_bits[rr] = q.bits;
        }
      }
    }
    __syncthreads();
    b2m::pdl_wait();  // an append launched before this kernel is through
#pragma unroll
    for (int k = 0; k < ST_STAGES - 1; k++)
      if (k >= ahead) issue(warp + k * ST_WARPS, k);
  }

  // The tensor cores cut off what an addition to a sum leaves below it, always toward
  // zero: over n additions some n 2^-25 of the sum. So they only sum ST_WINDOW tiles,
  // which are then added, rounded to nearest, to the totals.
  float o[NT][L::MT][4], total[NT][L::MT][4];
  // Per row: the largest score seen, log2 of the largest weight times V scale (at
  // reference weight 1), the reference, the weights' sum, the scores' factor.
  float m[NT][2], c_max[NT][2], ref[NT][2], l[NT][2], rf[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
#pragma unroll
    for (int k = 0; k < L::MT; k++)
#pragma unroll
      for (int u = 0; u < 4; u++) o[nt][k][u] = total[nt][k][u] = 0.f;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      m[nt][u] = c_max[nt][u] = -INFINITY;
      ref[nt][u] = 0.f;
      l[nt][u] = 0.f;
      rf[nt][u] = row_factor[nt * 8 + 2 * t + u];
    }
  }
  float vmax = 0.f, vinv = 0.f;  // largest V scale seen (a power of two above it), and its reciprocal
  const int all_see = a.tree ? past : past + row0 / G + 1;  // keys below this are seen by every row

  auto fold = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int k = 0; k < L::MT; k++)
#pragma unroll
        for (int u = 0; u < 4; u++) {
          total[nt][k][u] += o[nt][k][u];
          o[nt][k][u] = 0.f;
        }
  };

  int slot = 0, window = 0;
#pragma unroll 1
  for (int tile = warp; tile < ntile; tile += ST_WARPS) {
    cp_wait<ST_STAGES - 2>();
    __syncwarp();
    issue(tile + (ST_STAGES - 1) * ST_WARPS, slot == 0 ? ST_STAGES - 1 : slot - 1);
    const uint8_t *s = ring + slot * L::SLOT;
    const int j0 = jbeg + 16 * tile;
    // S^T = K . Q^T
    float c[NT][4], ch[2][NT][4], cl[2][NT][4];  // (four chains of products)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int u = 0; u < 4; u++) ch[0][nt][u] = ch[1][nt][u] = cl[0][nt][u] = cl[1][nt][u] = 0.f;
#pragma unroll
    for (int cc = 0; cc < L::NKC; cc++) {
      uint32_t w0[L::KW], w1[L::KW];
      const uint8_t *p0 = s + (cc * 32 + lane) * L::KC, *p1 = p0 + L::NKC * 32 * L::KC;
      if constexpr (L::KC == 16) {
        const uint4 x = *reinterpret_cast<const uint4 *>(p0), y = *reinterpret_cast<const uint4 *>(p1);
        w0[0] = x.x, w0[1] = x.y, w0[2] = x.z, w0[3] = x.w;
        w1[0] = y.x, w1[1] = y.y, w1[2] = y.z, w1[3] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2 *>(p0), y = *reinterpret_cast<const uint2 *>(p1);
        w0[0] = x.x, w0[1] = x.y;
        w1[0] = y.x, w1[1] = y.y;
      }
#pragma unroll
      for (int w = 0; w < L::KW; w++) {
        uint32_t A[4];
        expand4<E4M3>(w0[w], A[0], A[2]);
        expand4<E4M3>(w1[w], A[1], A[3]);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint4 q = qfrag[(nt * L::KSTEPS + cc * L::KW + w) * 32 + lane];
          mma(ch[w & 1][nt], A, q.x, q.y);
          mma(cl[w & 1][nt], A, q.z, q.w);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int u = 0; u < 4; u++) c[nt][u] = (ch[0][nt][u] + ch[1][nt][u]) + (cl[0][nt][u] + cl[1][nt][u]);
    // Scores in log2 units; masked ones -inf.
    const float4 sc = *reinterpret_cast<const float4 *>(s + L::K_BYTES + L::V_BYTES + g * 16);
    float x[NT][2][2];  // [key g, g + 8][row 2t, 2t + 1]
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        x[nt][0][u] = c[nt][u] * sc.x * rf[nt][u];
        x[nt][1][u] = c[nt][2 + u] * sc.y * rf[nt][u];
      }
    const bool whole = j0 + 16 <= min(jend, all_see);
    uint32_t seen = 0xffffffffu;  // bit (nt * 2 + key) * 2 + row
    if (!whole) {
      seen = 0;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const int j = j0 + g + 8 * k, rr = nt * 8 + 2 * t + u, dj = j - past;
            const bool ok = j < jend && (j <= row_lim[rr] || (dj >= 0 && dj < 64 && (row_bits[rr] >> dj & 1)));
            if (ok)
              seen |= 1u << ((nt * 2 + k) * 2 + u);
            else
              x[nt][k][u] = -INFINITY;
          }
    }
    // Keys past the range stand for its last key: their scales are valid ones.
    bool need = fmaxf(sc.z, sc.w) > vmax || !(fminf(sc.z, sc.w) >= vmax * V_LOW);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int u = 0; u < 2; u++) need |= fmaxf(x[nt][0][u], x[nt][1][u]) > c_max[nt][u] + REF_SLACK;
    if (__any_sync(0xffffffffu, need)) {
      float vm = fmaxf(sc.z, sc.w);
#pragma unroll
      for (int of = 4; of < 32; of <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, of));
      float vf = 1.f;  // old reference over new one
      if (vm > vmax) {
        // the power of two above vm, kept where its reciprocal is a normal number
        const float up = __uint_as_float(min(max((__float_as_uint(vm) >> 23) + 1u, 2u), 252u) << 23);
        vf = vmax * (1.f / up);
        vmax = up;
        vinv = 1.f / up;
      }
      const float lf = lg2(vf), lv0 = lg2(sc.z * vinv), lv1 = lg2(sc.w * vinv);
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float mn = fmaxf(x[nt][0][u], x[nt][1][u]);
          float cn = fmaxf(x[nt][0][u] + lv0, x[nt][1][u] + lv1);  // (a hidden key's NaN is passed over)
#pragma unroll
          for (int of = 4; of < 32; of <<= 1) {
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, of));
            cn = fmaxf(cn, __shfl_xor_sync(0xffffffffu, cn, of));
          }
          mn = fmaxf(mn, m[nt][u]);
          float fo = vf;
          if (mn > -INFINITY) {
            c_max[nt][u] = fmaxf(c_max[nt][u] + lf, cn);
            const float rn = weight_ref(mn, c_max[nt][u]), f = m[nt][u] == -INFINITY ? 0.f : ex2(ref[nt][u] - rn);
            l[nt][u] = l[nt][u] == 0.f ? 0.f : l[nt][u] * f;
            m[nt][u] = mn;
            ref[nt][u] = rn;
            fo *= f;
          }
#pragma unroll
          for (int k = 0; k < L::MT; k++) {
            o[nt][k][u] *= fo;
            o[nt][k][2 + u] *= fo;
            total[nt][k][u] *= fo;
            total[nt][k][2 + u] *= fo;
          }
        }
    }
    // Weights (with V's scales) as two f16 terms, transposed into B fragments.
    const float v0 = sc.z * vinv, v1 = sc.w * vinv;
    uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float w[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const bool ok = seen >> ((nt * 2 + k) * 2 + u) & 1;
          const float p = ok ? ex2(x[nt][k][u] - ref[nt][u]) : 0.f;
          l[nt][u] += p;
          w[u] = ok ? p * (k ? v1 : v0) : 0.f;  // a hidden key's scale may be NaN
        }
        const __half2 h = __floats2half2_rn(w[0], w[1]);
        bh[nt][k] = transpose8x8(b2m::h2_as_u32(h));
        const float2 hf = __half22float2(h);
        bl[nt][k] = transpose8x8(b2m::h2_as_u32(__floats2half2_rn(w[0] - hf.x, w[1] - hf.y)));
      }
    // O^T += V^T . P^T
#pragma unroll
    for (int cc = 0; cc < L::NVC; cc++) {
      uint32_t vw[4][L::VW];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint8_t *p = s + L::K_BYTES + ((q * L::NVC + cc) * 32 + lane) * L::VC;
        if constexpr (L::VC == 16) {
          const uint4 y = *reinterpret_cast<const uint4 *>(p);
          vw[q][0] = y.x, vw[q][1] = y.y, vw[q][2] = y.z, vw[q][3] = y.w;
        } else if constexpr (L::VC == 8) {
          const uint2 y = *reinterpret_cast<const uint2 *>(p);
          vw[q][0] = y.x, vw[q][1] = y.y;
        } else {
          vw[q][0] = *reinterpret_cast<const uint32_t *>(p);
        }
      }
#pragma unroll
      for (int w = 0; w < L::VW; w++) {
        uint32_t lo[4], hi[4];  // dims 4w .. 4w+3 of the chunk: keys (2t, 2t+1), (2t+8, 2t+9)
        expand_zip<E4M3>(vw[0][w], vw[1][w], lo);
        expand_zip<E4M3>(vw[2][w], vw[3][w], hi);
        const uint32_t A[2][4] = {{lo[0], lo[1], hi[0], hi[1]}, {lo[2], lo[3], hi[2], hi[3]}};
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++) mma(o[nt][(cc * L::VW + w) * 2 + hf], A[hf], bh[nt][0], bh[nt][1]);
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++) mma(o[nt][(cc * L::VW + w) * 2 + hf], A[hf], bl[nt][0], bl[nt][1]);
      }
    }
    if (++window == ST_WINDOW) {
      window = 0;
      fold();
    }
    slot = slot + 1 == ST_STAGES ? 0 : slot + 1;
    __syncwarp();  // every lane has read the slot's scales before it is refilled
  }
  cp_wait<0>();
  __syncthreads();  // the rings are drained: the states reuse them

  fold();

  // Warp states: reference, l per row and O (in the values' own scale).
  float *so = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float s = l[nt][u];
#pragma unroll
      for (int of = 4; of < 32; of <<= 1) s += __shfl_xor_sync(0xffffffffu, s, of);
      const int rr = nt * 8 + 2 * t + u;
      if (g == 0) {
        wm[warp * R + rr] = m[nt][u] == -INFINITY ? -INFINITY : ref[nt][u];
        wl[warp * R + rr] = s;
      }
      float *dst = so + (warp * R + rr) * D;
#pragma unroll
      for (int k = 0; k < L::MT; k++) {
        const int cc = (k >> 1) / L::VW, w = (k >> 1) % L::VW;
        const int d = (cc * 8 + g) * L::VC + 4 * w + 2 * (k & 1);
        *reinterpret_cast<float2 *>(dst + d) = make_float2(total[nt][k][u] * vmax, total[nt][k][2 + u] * vmax);
      }
    }
  __syncthreads();
  // A state's share of the joint one: none if it saw no key; with a NaN sum and
  // no reference (all its scores NaN) it passes the NaN on.
  auto share = [](float sm, float sl, float top) {
    return sl == 0.f ? 0.f : (sm == -INFINITY ? 1.f : ex2(sm - top));
  };
  constexpr int D4 = D / 4;
#pragma unroll 1
  for (int e = tid; e < R * D4; e += ST_THREADS) {
    const int rr = e / D4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < ST_WARPS; w++) top = fmaxf(top, wm[w * R + rr]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < ST_WARPS; w++) {
      const float sl = wl[w * R + rr], f = share(wm[w * R + rr], sl, top);
      const float4 v = reinterpret_cast<const float4 *>(so + w * R * D)[e];
      sum += sl * f;
      acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
    }
    reinterpret_cast<float4 *>(so)[e] = acc;
    if (e % D4 == 0) {
      cm[rr] = top;
      cl_[rr] = sum;
    }
  }
  if (CL > 1)
    cluster.sync();
  else
    __syncthreads();
#pragma unroll 1
  for (int e = rank * ST_THREADS + tid; e < R * D4; e += CL * ST_THREADS) {
    const int rr = e / D4, r = row0 + rr;
    if (r >= nrows) continue;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // (eight ranks' loads at once: their latency is what this costs)
    for (int q0 = 0; q0 < CL; q0 += 8) {
      float sm[8], sl[8], was = top;
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int q = q0 + k;
        sm[k] = -INFINITY, sl[k] = 0.f, v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (q < CL) {
          const float4 *src = reinterpret_cast<const float4 *>(so) + e;
          sm[k] = CL > 1 ? *cluster.map_shared_rank(cm + rr, q) : cm[rr];
          sl[k] = CL > 1 ? *cluster.map_shared_rank(cl_ + rr, q) : cl_[rr];
          v[k] = CL > 1 ? *cluster.map_shared_rank(src, q) : *src;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k++) top = fmaxf(top, sm[k]);
      const float keep = share(was, sum, top);
      sum *= keep, acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float f = share(sm[k], sl[k], top);
        sum += sl[k] * f;
        acc.x += v[k].x * f, acc.y += v[k].y * f, acc.z += v[k].z * f, acc.w += v[k].w * f;
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that saw nothing: zeros
    acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    const int64_t at = ((int64_t)b * a.S + r / G) * a.H * D + (int64_t)(kvh * G + r % G) * D + 4 * (e % D4);
    if (a.out) *reinterpret_cast<float4 *>(a.out + at) = acc;
    if (a.out16) {
      const __half2 h0 = __floats2half2_rn(acc.x, acc.y), h1 = __floats2half2_rn(acc.z, acc.w);
      *reinterpret_cast<uint2 *>(a.out16 + at) = make_uint2(b2m::h2_as_u32(h0), b2m::h2_as_u32(h1));
    }
  }
  if (CL > 1) cluster.sync();  // the others have read this CTA's state
}

template <bool E4M3, int D, int NT>
void launch(const Kv8Args &a, cudaStream_t s) {
  using M = StepSmem<D, NT>;
  constexpr auto kern = kv8_step_kernel<E4M3, D, NT>;
  b2m::set_smem_limit_once<kern>(M::BYTES);
  const int nrows = a.S * (a.H / a.KVH), tiles = (nrows + M::R - 1) / M::R;
  // One new row per sequence is appended beside the query rows; more would hold up
  // the CTA whose range they fall into (eight: 7 us longer than a launch of its own).
  const bool fused = a.S == 1 && tiles == 1 && append_rows_vec(a);
  if (!fused) launch_kv8_append(a, s);
  // Key splits. A CTA costs some 8 us however few keys it has, and a cluster is
  // only placed where all its CTAs fit, so a split has to pay for itself: up to one
  // wave of CTAs that are resident together (three per SM for 8 query rows, two for
  // 16), at least 128 cache positions each, 16 CTAs at most; and two for calls of
  // between one and two waves of long rows, whose second wave would be mostly
  // empty (64 sequences over 4096 .. 8191 positions: 176 us, 207
  // unsplit, 202 with four; 32 trees over 1500: 48 us unsplit, 51 and 70 with two and
  // four). Three sequences over 40000 (12 x 16 CTAs) are bound by the SMs that hold
  // two CTAs: 41 us; clusters of 8 and 4: 52 and 94.
  const int64_t ctas = (int64_t)a.B * a.KVH * tiles;
  const int64_t wave = (NT == 1 ? 3 : 2) * (int64_t)b2m::device_sm_count();
  int cl = 1;
  while (cl < 16 && ctas * cl * 2 <= wave && a.CAP >= 256 * cl) cl *= 2;
  if (cl == 1 && NT == 1 && ctas > wave && ctas < 2 * wave && a.CAP >= 2048) cl = 2;
  b2m::allow_large_cluster_once<kern>();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * cl), (unsigned)a.KVH, (unsigned)a.B);
  cfg.blockDim = dim3(ST_THREADS);
  cfg.dynamicSmemBytes = M::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // starts beside its own append
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = fused ? 1 : 2;
  B2M_CUDA(cudaLaunchKernelEx(&cfg, kern, a, fused ? 1 : 0));
}

template <bool E4M3, int D>
void launch_rows(const Kv8Args &a, cudaStream_t s) {
  if (a.S * (a.H / a.KVH) <= 8)
    launch<E4M3, D, 1>(a, s);
  else
    launch<E4M3, D, 2>(a, s);
}

template <bool E4M3>
void launch_dim(const Kv8Args &a, cudaStream_t s) {
  switch (a.D) {
    case 32: return launch_rows<E4M3, 32>(a, s);
    case 64: return launch_rows<E4M3, 64>(a, s);
    case 96: return launch_rows<E4M3, 96>(a, s);
    case 128: return launch_rows<E4M3, 128>(a, s);
    default: return launch<E4M3, 256, 1>(a, s);
  }
}

}  // namespace

// Head dims the kernel is compiled for, cache rows it can copy 16 bytes at a
// time, query rows and outputs it can take four values at a time.
bool kv8_step_shape(const Kv8Args &a) {
  auto al = [](const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  return (a.D == 32 || a.D == 64 || a.D == 96 || a.D == 128 || a.D == 256) && q_rows_vec(a) && al(a.kc, 16) &&
         al(a.vc, 16) && al(a.out, 16) && al(a.out16, 8) && a.KVH <= 65535;
}

void launch_kv8_step(const Kv8Args &a, cudaStream_t s) {
  if (a.e4m3)
    launch_dim<true>(a, s);
  else
    launch_dim<false>(a, s);
}
