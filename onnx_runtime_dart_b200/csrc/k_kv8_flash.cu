// Attention over the 8-bit KV cache for many query rows per kv head (prompts,
// chunks, wide drafted trees) on tcgen05; head_dim 64 or 128.
//
// A CTA takes 128 query rows of one (kv head, sequence): row r is query head
// r % G of token r / G, so the heads of a group share the K / V tiles. Keys come
// in tiles of 64. Roles:
//   warps 4-7  expand a tile's codes (exact f16 numbers) into shared memory, K as
//              [64 keys][D], V transposed as [D][64 keys] (128-byte swizzle), the
//              next tile's codes already in flight in registers;
//   warp 8     (of a third warpgroup) one thread issues S_j = Q . K_j^T (S in TMEM,
//              two buffers) and O += P_j . V_j with P in TMEM as the A operand;
//              S_{j+1} is issued before P_j is waited for, so the tensor cores
//              work under the softmax;
//   warps 0-3  a thread per query row (= TMEM lane): scores times K's scale,
//              the causal or tree mask, exp2 against a reference that only moves
//              when a weight would pass 2^15 (O in TMEM is rescaled then), the
//              weights times V's scale as f16 back into S's columns. V's scales
//              are kept over the largest of the CTA's keys, hidden ones included;
//              the reference goes by what the row itself sees (weight_ref), which
//              costs extra operations only in tiles with a scale below 2^-8 of that.
// No cross-thread reduction is left in the softmax. Two CTAs share an SM, so one's
// exponentials run under the other's products.
//
// Q and P are split into two f16 terms (22 bits, two products each), for an f16
// output too: with one term of Q its error against 64 bits was 2.8e-4, the output's own
// rounding is 2.1e-4.
//
// Few row tiles over many keys (a tree on long sequences): the CTAs of a cluster
// split the keys and merge their O, reference and l through distributed shared memory in
// rank order; no workspace, no atomics.
//
// 4 x 2048 causal tokens (16 heads on 8) take 275 us with their append: 250 TFLOP/s
// of wanted products, tensor pipe 29% busy (second terms included), issue slots 46%.
// What bounds it is the instructions of the softmax and of the expansion (some
// 4500 per 64-key tile and CTA), the single K and V tile, and each CTA's start, totals
// and end, which only the SM's other CTA covers. 237 us were without the second term
// of Q, whose room held another tile of each, and without the totals; 257 without the
// totals alone.
//
// Every wait is bounded; one that gives up records the device error and all
// roles leave their loops.
#include <cooperative_groups.h>

#include <algorithm>

#include "kv8_common.cuh"
#include "tc_common.cuh"

namespace {

namespace cg = cooperative_groups;
using namespace kv8;
using namespace b2m;

constexpr int FL_MAX_CLUSTER = 8, FL_THREADS = 384, FL_TILE = 64, FL_ROWS = 128, FL_SLOTS = 4,
              FL_WINDOW = 8;  // tiles whose products the tensor cores add up (see the softmax's totals)
// Registers per thread: at launch (two CTAs per SM), then per role, and the
// launch's number again for the common end. The CTA's three warpgroups share
// what it was launched with: the roles' sum is no more.
constexpr int FL_REGS = 80, FL_REGS_SOFTMAX = 136, FL_REGS_TILES = 64, FL_REGS_MMA = 40;
static_assert(FL_REGS_SOFTMAX + FL_REGS_TILES + FL_REGS_MMA <= 3 * FL_REGS, "register split");

__device__ __forceinline__ uint32_t sw128(int r, int k) {  // byte offset of 16-bit element k < 64 of row r
  return (uint32_t)(r * 128 + ((((k >> 3) ^ (r & 7)) << 4) | ((k & 7) << 1)));
}

// True in one lane of a converged warp. Code behind it may keep its addresses and
// descriptors in uniform registers, where tcgen05.mma takes them from; behind a
// test of the lane number each would be moved there first (100 cycles a product).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Two fp32 operations per instruction on register pairs.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 32 lanes x 32 consecutive 32-bit TMEM columns -> 16 register pairs per thread.
__device__ __forceinline__ void tmem_ld32x2(uint32_t taddr, f32x2 *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}

// Waits for phase `parity` of a barrier, suspended in the hardware for up to a
// millisecond per try: at two CTAs per SM a dozen warps wait at any time, and
// polling took half of the issue slots. Gives up when another thread has, or
// after two seconds (and records the error).
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int32_t *dev_err) {
#pragma unroll 1
  for (int i = 0; i < 2000; i++) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  if (dev_err) set_dev_error(dev_err, B2M_DEVERR_MBAR_TIMEOUT);
  return false;
}
// The same for a whole warp, one verdict for all lanes.
__device__ __forceinline__ bool warp_wait_phase(uint64_t *bar, uint32_t parity, volatile int *abort_flag,
                                                int32_t *dev_err) {
  return __all_sync(0xffffffffu, wait_phase(bar, parity, abort_flag, dev_err));
}

template <int D>
struct FlashLayout {
  static constexpr int ND = D / 64;
  static constexpr uint32_t QH = 0, QL = ND * 16384;
  static constexpr uint32_t K = QL + ND * 16384;  // one K and one V tile (two of each are more than half of an SM's memory)
  static constexpr uint32_t V = K + ND * 8192;
  static constexpr uint32_t TILES = V + D * 128;
  // O staging [128][D + 4] fp32 at the end, over Q, K and V
  static constexpr int OST = D + 4;
  static constexpr uint32_t SCALES0 = 128 * OST * 4 > TILES ? 128 * OST * 4 : TILES;
  // ks[SLOTS][64], vs[SLOTS][64], vf[SLOTS], vflag[SLOTS], vref; then per row: factor, limit,
  // bits, reference, l; barriers
  static constexpr uint32_t SCALES = SCALES0;
  static constexpr uint32_t VF = SCALES + FL_SLOTS * 64 * 8, VFLAG = VF + FL_SLOTS * 4, VREF = VFLAG + FL_SLOTS * 4;
  static constexpr uint32_t ROWS = VREF + 16;
  static constexpr uint32_t BARS = ROWS + 128 * (8 + 4 + 4 + 4 + 4);
  static constexpr uint32_t SLOT = BARS + 10 * 8, FLAG = SLOT + 4;
  static constexpr uint32_t BYTES = FLAG + 4;
  static constexpr uint32_t T_O = 128;  // TMEM: S / P buffers at 0 and 64, O at 128
  static_assert(BYTES <= 113 * 1024, "two CTAs per SM");
};

template <bool E4M3, int D>
__global__ void __launch_bounds__(FL_THREADS, 2) kv8_flash_kernel(const Kv8Args a) {
  using L = FlashLayout<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  float *ks_s = reinterpret_cast<float *>(smem + L::SCALES), *vs_s = ks_s + FL_SLOTS * 64;
  float *vf_s = reinterpret_cast<float *>(smem + L::VF), *vref_s = reinterpret_cast<float *>(smem + L::VREF);
  int *vflag_s = reinterpret_cast<int *>(smem + L::VFLAG);  // bit 0: a NaN scale, bit 1: one far below vref
  uint64_t *row_bits = reinterpret_cast<uint64_t *>(smem + L::ROWS);
  float *row_factor = reinterpret_cast<float *>(row_bits + 128);
  int *row_lim = reinterpret_cast<int *>(row_factor + 128);
  float *row_ref = reinterpret_cast<float *>(row_lim + 128), *row_l = row_ref + 128;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BARS);
  uint64_t *k_full = bars, *k_empty = bars + 1, *v_full = bars + 2, *v_empty = bars + 3, *s_full = bars + 4,
           *p_full = bars + 6, *o_done = bars + 8, *all_done = bars + 9;
  uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::SLOT);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::FLAG);

  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, tid = threadIdx.x;
  const int row0 = (int)(gridDim.z - 1 - blockIdx.z) * FL_ROWS;  // the longest rows of all first
  const int kvh = (int)(blockIdx.x / CL), b = blockIdx.y;
  const int G = a.H / a.KVH, nrows = a.S * G;
  const int past = min(max(0, a.past[b]), a.CAP);  // (an append past either has raised its error)
  const int last_token = min(a.S - 1, (row0 + FL_ROWS - 1) / G);
  const int n = (int)min((int64_t)a.CAP, (int64_t)past + (a.tree ? a.S : last_token + 1));
  const int all_tiles = (n + FL_TILE - 1) / FL_TILE, per = (all_tiles + CL - 1) / CL;
  const int t0 = min(all_tiles, rank * per), ntile = min(all_tiles, t0 + per) - t0;
  const int64_t base = ((int64_t)b * a.KVH + kvh) * a.CAP;

  if (tid == 0) {
    mbar_init(k_full, 128);
    mbar_init(k_empty, 1);
    mbar_init(v_full, 128);
    mbar_init(v_empty, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
    }
    mbar_init(o_done, 1);
    mbar_init(all_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(slot, 256);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *slot, 0);
  // Behind the allocation: a dependent kernel that fits beside this CTA and wants
  // all of TMEM could otherwise take it first and then wait for this grid, which
  // would wait for TMEM.
  pdl_launch_dependents();

  // The query rows, by the warps that will use them; the others start on the tiles.
  if (warp < 4 || warp >= 8) {
#pragma unroll 1
    for (int rr = (warp < 4 ? warp : warp - 4) * 4 + (lane >> 3); rr < FL_ROWS; rr += 32) {
      QRow<D> q;
      load_q_row<D>(a, b, kvh, G, row0 + rr, past, q);
#pragma unroll
      for (int u = 0; u < D / 32; u++) {
        const int d = 4 * ((lane & 7) + 8 * u);
        // (in the order of K's expanded codes)
        const float v[4] = {q.v[u].x, q.v[u].y, q.v[u].z, q.v[u].w};
        const float4 x = make_float4(v[0], v[expand_order<E4M3>(1)], v[expand_order<E4M3>(2)], v[3]);
        const __half2 h0 = __floats2half2_rn(x.x, x.y), h1 = __floats2half2_rn(x.z, x.w);
        const uint32_t at = (uint32_t)(d >> 6) * 16384u + sw128(rr, d & 63);
        *reinterpret_cast<uint2 *>(smem + L::QH + at) = make_uint2(h2_as_u32(h0), h2_as_u32(h1));
        const float2 g0 = __half22float2(h0), g1 = __half22float2(h1);
        *reinterpret_cast<uint2 *>(smem + L::QL + at) = make_uint2(
            h2_as_u32(__floats2half2_rn(x.x - g0.x, x.y - g0.y)), h2_as_u32(__floats2half2_rn(x.z - g1.x, x.w - g1.y)));
      }
      if ((lane & 7) == 0) {
        row_factor[rr] = q.factor;
        row_lim[rr] = q.lim;
        row_bits[rr] = q.bits;
      }
    }
    fence_proxy_async_smem();
    named_barrier_sync(1, FL_THREADS - 128);
  }

  if (warp >= 4 && warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FL_REGS_TILES));
    // ---- K / V tiles -------------------------------------------------------
    const int ct = tid - 128, cw = warp - 4;
    constexpr int KI = 64 * (D / 16) / 128, VI = D / 64;  // 16-byte items per thread: K; V (per key of the pair)
    uint4 kreg[KI], vreg[2][VI];
    float sc[2];
    const uint8_t *kc = a.kc + base * D, *vc = a.vc + base * D;
    // K: eight lanes take eight rows of one 16-byte chunk (conflict-free stores)
    auto k_item = [&](int u, int &row, int &c) {
      const int it = ct + 128 * u;
      row = (it & 7) + 8 * (it / (8 * (D / 16)));
      c = (it >> 3) % (D / 16);
    };
    auto load_k = [&](int t) {
      const int j0 = (t0 + t) * FL_TILE;
#pragma unroll
      for (int u = 0; u < KI; u++) {
        int row, c;
        k_item(u, row, c);
        kreg[u] = *reinterpret_cast<const uint4 *>(kc + (int64_t)min(j0 + row, n - 1) * D + 16 * c);
      }
      // warps 0, 1: K's scales (one per lane); warps 2, 3: V's (two per lane)
      if (cw < 2) {
        sc[0] = a.ks[base + min(j0 + ct, n - 1)];
      } else {
        sc[0] = a.vs[base + min(j0 + lane, n - 1)];
        sc[1] = a.vs[base + min(j0 + 32 + lane, n - 1)];
      }
    };
    // V: lane p takes keys 2p, 2p + 1, warp w the chunks w VI ...
    auto load_v = [&](int t) {
      const int j0 = (t0 + t) * FL_TILE;
#pragma unroll
      for (int q = 0; q < 2; q++)
#pragma unroll
        for (int u = 0; u < VI; u++)
          vreg[q][u] = *reinterpret_cast<const uint4 *>(vc + (int64_t)min(j0 + 2 * lane + q, n - 1) * D +
                                                        16 * (cw * VI + u));
    };
    float vref = 0.f, vinv = 0.f;
    auto put_k = [&](int t) {
      const int sl = t % FL_SLOTS;
      if (t > 0 && !warp_wait_phase(k_empty, (uint32_t)(t - 1) & 1u, abort_flag, a.err)) return false;
      uint8_t *kd = smem + L::K;
#pragma unroll
      for (int u = 0; u < KI; u++) {
        int row, c;
        k_item(u, row, c);
        const uint32_t w[4] = {kreg[u].x, kreg[u].y, kreg[u].z, kreg[u].w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; k++) expand4<E4M3>(w[k], o[2 * k], o[2 * k + 1]);
        uint8_t *blk = kd + (c >> 2) * 8192;
        *reinterpret_cast<uint4 *>(blk + sw128(row, (16 * c) & 63)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4 *>(blk + sw128(row, ((16 * c) & 63) + 8)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
      if (cw < 2) {
        ks_s[sl * 64 + ct] = sc[0];
      } else {
        // V's scales over the power of two above the largest so far (both warps
        // come to the same one); a change tells the softmax to rescale O.
        float vm = fmaxf(sc[0], sc[1]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
        float vf = 1.f;
        if (vm > vref) {
          const float up = __uint_as_float(min(max((__float_as_uint(vm) >> 23) + 1u, 2u), 252u) << 23);
          vinv = 1.f / up;
          vf = vref * vinv;
          vref = up;
        }
        if (cw == 2)
          vs_s[sl * 64 + lane] = sc[0] * vinv;
        else
          vs_s[sl * 64 + 32 + lane] = sc[1] * vinv;
        const bool nan = __any_sync(0xffffffffu, sc[0] != sc[0] || sc[1] != sc[1]);
        const bool low = __any_sync(0xffffffffu, !(sc[0] * vinv >= V_LOW) || !(sc[1] * vinv >= V_LOW));
        if (cw == 2 && lane == 0) {
          vflag_s[sl] = (nan ? 1 : 0) | (low ? 2 : 0);
          vf_s[sl] = vf;
          *vref_s = vref;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(k_full);
      return true;
    };
    // The append of the call's rows may still run: tiles without new rows go ahead
    // (what came before the append is visible: it was launched without an early start).
    bool appended = false;
    auto reach = [&](int t) {
      if (!appended && (t0 + t + 1) * (int64_t)FL_TILE > past) {
        pdl_wait();
        appended = true;
      }
    };
    if (ntile > 0) {
      reach(0);
      load_k(0);
      load_v(0);
      put_k(0);
      if (ntile > 1) {
        reach(1);
        load_k(1);
      }
    }
    // K_{t+1} before V_t: its products are wanted first (under tile t's softmax).
#pragma unroll 1
    for (int t = 0; t < ntile; t++) {
      if (t + 1 < ntile) {
        if (!put_k(t + 1)) break;
        if (t + 2 < ntile) {
          reach(t + 2);
          load_k(t + 2);
        }
      }
      if (t > 0 && !warp_wait_phase(v_empty, (uint32_t)(t - 1) & 1u, abort_flag, a.err)) break;
      uint8_t *vd = smem + L::V;
#pragma unroll
      for (int u = 0; u < VI; u++) {
        const uint32_t w0[4] = {vreg[0][u].x, vreg[0][u].y, vreg[0][u].z, vreg[0][u].w};
        const uint32_t w1[4] = {vreg[1][u].x, vreg[1][u].y, vreg[1][u].z, vreg[1][u].w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          uint32_t o[4];  // dims 4k .. 4k+3: keys (2p, 2p+1)
          expand_zip<E4M3>(w0[k], w1[k], o);
#pragma unroll
          for (int e = 0; e < 4; e++)
            *reinterpret_cast<uint32_t *>(vd + sw128(16 * (cw * VI + u) + 4 * k + e, 2 * lane)) = o[e];
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(v_full);
      if (t + 1 < ntile) load_v(t + 1);
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FL_REGS_MMA));
    // ---- tensor cores ------------------------------------------------------
    if (warp == 8 && ntile > 0 && elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc(128, FL_TILE, 1u, 0u, 0u), idesc_o = umma_idesc(128, D, 1u, 0u, 0u);
      const uint32_t sb = smem_u32(smem);
      const uint64_t d_qh = sw128_kmajor_desc(sb + L::QH), d_ql = sw128_kmajor_desc(sb + L::QL);
      auto issue_s = [&](int t) {
        const uint64_t dk = sw128_kmajor_desc(sb + L::K);
        const uint32_t ts = tmem + (uint32_t)(t & 1) * 64u;
        // the lower terms first: fewer additions to a sum of full size
#pragma unroll
        for (int part = 0; part < 2; part++)
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++) {
            const uint64_t oq = ((kk >> 2) * 16384u + (kk & 3) * 32u) >> 4,
                           ok = ((kk >> 2) * 8192u + (kk & 3) * 32u) >> 4;
            umma_f16(ts, (part ? d_qh : d_ql) + oq, dk + ok, idesc_s, part || kk ? 1u : 0u);
          }
        umma_commit(s_full + (t & 1));
        umma_commit(k_empty);
      };
      bool ok = wait_phase(k_full, 0u, abort_flag, a.err);
      if (ok) {
        tc_fence_after();
        issue_s(0);
      }
#pragma unroll 1
      for (int t = 0; ok && t < ntile; t++) {
        if (t + 1 < ntile) {
          // S_{t+1} takes the columns of P_{t-1}: products of different shapes are
          // not ordered among themselves, so P_{t-1} . V must be through.
          ok = (t == 0 || wait_phase(o_done, (uint32_t)(t - 1) & 1u, abort_flag, a.err)) &&
               wait_phase(k_full, (uint32_t)(t + 1) & 1u, abort_flag, a.err);
          if (!ok) break;
          tc_fence_after();
          issue_s(t + 1);
        }
        ok = wait_phase(v_full, (uint32_t)t & 1u, abort_flag, a.err) &&
             wait_phase(p_full + (t & 1), (uint32_t)(t >> 1) & 1u, abort_flag, a.err);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = sw128_kmajor_desc(sb + L::V);
        const uint32_t tp = tmem + (uint32_t)(t & 1) * 64u;
#pragma unroll
        for (int part = 0; part < 2; part++)
#pragma unroll
          for (int kk = 0; kk < FL_TILE / 16; kk++)
            umma_f16_ts(tmem + L::T_O, tp + (part ? 0u : 32u) + 8u * kk, dv + ((kk * 32u) >> 4), idesc_o,
                        t % FL_WINDOW || part || kk ? 1u : 0u);
        umma_commit(v_empty);
        umma_commit(o_done);
        // A barrier of its own for the last one: a waiter that has not seen the
        // phase before could take o_done's parity for the one it waits for. (In the
        // loop S_t is there, and S_t was issued behind phase t - 2.)
        if (t + 1 == ntile) umma_commit(all_done);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FL_REGS_SOFTMAX));
    // ---- softmax -----------------------------------------------------------
    const int rr = tid;
    const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
    const float rf = row_factor[rr];
    const int lim = row_lim[rr];
    const uint64_t bits = row_bits[rr];
    const int all_see = a.tree ? past : past + row0 / G + 1;  // keys below this are seen by every row
    // Largest score seen, log2 of the largest weight times V scale (at the reference
    // weight 1), the reference the weights are taken against, their sum.
    float m = -INFINITY, c_max = -INFINITY, ref = 0.f, l = 0.f;
    // The tensor cores cut off what an addition to O leaves below it, always toward
    // zero: eight times per tile, 1.6e-7 of a sum of equal signs (1e-5 after 60 tiles,
    // without a bound as sequences grow). So O starts anew every FL_WINDOW tiles, and
    // the row's thread adds what it held, rounded to nearest, to totals of its own:
    // thread-local memory, which is laid out across a warp's threads and stays in L2 (the
    // driver keeps 190 MB of it for the device). `carry` is what the totals are to be multiplied by since the last time.
    alignas(16) float total[D];
    float carry = 1.f;
    // Waits for phase `parity` of `done`, then calls put(d, totals + O of dimensions d ..
    // d + 3) for all of them; 64 totals at a time are requested ahead (as long a way as
    // a tile's products take).
    auto with_totals = [&](bool any, uint64_t *done, uint32_t parity, auto put) {
      float4 held[16];
      int d0 = 0;
      asm volatile("" : "+r"(d0));  // (an index the compiler knows would put the totals into registers that are not there)
      auto fetch = [&](int d) {
#pragma unroll
        for (int k = 0; k < 16; k++)
          held[k] = any ? reinterpret_cast<const float4 *>(total + d)[k] : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      fetch(d0);
      if (!warp_wait_phase(done, parity, abort_flag, a.err)) return false;
      tc_fence_after();
#pragma unroll 1
      for (int d = d0; d < D; d += 64) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint32_t u[16];
          tmem_ld16(trow + L::T_O + d + 16u * q, u);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float4 v = held[4 * q + k];
            put(d + 16 * q + 4 * k, make_float4(fmaf(v.x, carry, __uint_as_float(u[4 * k])),
                                                fmaf(v.y, carry, __uint_as_float(u[4 * k + 1])),
                                                fmaf(v.z, carry, __uint_as_float(u[4 * k + 2])),
                                                fmaf(v.w, carry, __uint_as_float(u[4 * k + 3]))));
          }
        }
        if (d + 64 < D) fetch(d + 64);
      }
      return true;
    };
    bool ok = true;
#pragma unroll 1
    for (int t = 0; t < ntile; t++) {
      const bool anew = t % FL_WINDOW == 0;
      const int sl = t % FL_SLOTS, j0 = (t0 + t) * FL_TILE;
      ok = warp_wait_phase(s_full + (t & 1), (uint32_t)(t >> 1) & 1u, abort_flag, a.err);
      if (!ok) break;
      tc_fence_after();
      if (anew && t > 0) {
        ok = with_totals(t > FL_WINDOW, o_done, (uint32_t)(t - 1) & 1u,
                         [&](int d, const float4 &v) { *reinterpret_cast<float4 *>(total + d) = v; });
        if (!ok) break;
        carry = 1.f;
      }
      const uint32_t ts = trow + (uint32_t)(t & 1) * 64u;
      // Scores of the row's 64 keys as 32 pairs, times K's scales.
      f32x2 x[FL_TILE / 2];
      tmem_ld32x2(ts, x);
      tmem_ld32x2(ts + 32u, x + 16);
      tmem_ld_wait();
      const ulonglong2 *kp = reinterpret_cast<const ulonglong2 *>(ks_s + sl * 64);
#pragma unroll
      for (int c = 0; c < FL_TILE / 4; c++) {
        const ulonglong2 k4 = kp[c];
        x[2 * c] = mul2(x[2 * c], k4.x);
        x[2 * c + 1] = mul2(x[2 * c + 1], k4.y);
      }
      const bool whole = j0 + FL_TILE <= min(n, all_see);
      uint64_t seen = ~0ull;
      if (!whole) {
        // Bit c: key j0 + c. Causal (and cached) keys up to lim; tree bits from past on.
        const int below = min(lim + 1, n) - j0;
        seen = below >= 64 ? ~0ull : (below <= 0 ? 0ull : (1ull << below) - 1);
        if (a.tree) {
          const int sh = past - j0;  // the tree's bit 0 is key j0 + sh
          uint64_t tb = sh >= 64 || sh <= -64 ? 0ull : (sh >= 0 ? bits << sh : bits >> -sh);
          const int end = n - j0;
          if (end < 64) tb &= end <= 0 ? 0ull : (1ull << end) - 1;
          seen |= tb;
        }
        const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
        for (int c = 0; c < FL_TILE / 2; c++) {
          float x0, x1;
          unpack2(x[c], x0, x1);
          const uint32_t w = c < 16 ? s0 : s1;
          x0 = w >> (2 * c & 31) & 1 ? x0 : -INFINITY;
          x1 = w >> (2 * c + 1 & 31) & 1 ? x1 : -INFINITY;
          x[c] = pack2(x0, x1);
        }
      }
      float xm;
      {
        float q[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < FL_TILE / 2; c++) {
          float x0, x1;
          unpack2(x[c], x0, x1);
          q[c & 3] = max3(q[c & 3], x0, x1);
        }
        xm = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3])) * rf;  // rf > 0; -inf stays
      }
      const float vf = vf_s[sl];
      const int vflag = vflag_s[sl];
      const ulonglong2 *vp = reinterpret_cast<const ulonglong2 *>(vs_s + sl * 64);
      float cm = xm;  // the row's largest score + log2(V scale); exact where the tile's scales differ much
      if (vflag & 2) {
        cm = -INFINITY;
#pragma unroll
        for (int c = 0; c < FL_TILE / 4; c++) {
          const ulonglong2 v4 = vp[c];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float x0, x1, v0, v1;
            unpack2(x[2 * c + k], x0, x1);
            unpack2(k ? v4.y : v4.x, v0, v1);
            cm = max3(cm, fmaf(x0, rf, lg2(v0)), fmaf(x1, rf, lg2(v1)));  // (a hidden key's NaN is passed over)
          }
        }
      }
      if (__any_sync(0xffffffffu, cm > c_max + REF_SLACK || xm > m + REF_SLACK || vf != 1.f)) {
        float f = vf;
        const float mn = fmaxf(m, xm);
        if (mn > -INFINITY) {
          c_max = fmaxf(c_max + lg2(vf), cm);
          const float rn = weight_ref(mn, c_max), fr = m == -INFINITY ? 0.f : ex2(ref - rn);
          l = l == 0.f ? 0.f : l * fr;
          f *= fr;
          m = mn;
          ref = rn;
        }
        carry *= f;
        if (!anew) {  // O holds the tiles before: rescale it once their products are done
          ok = warp_wait_phase(o_done, (uint32_t)(t - 1) & 1u, abort_flag, a.err);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            f32x2 u[16];
            uint32_t w[32];
            tmem_ld32x2(trow + L::T_O + 32u * c, u);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; k++) {
              float u0, u1;
              unpack2(u[k], u0, u1);
              w[2 * k] = __float_as_uint(u0 * f);
              w[2 * k + 1] = __float_as_uint(u1 * f);
            }
            tmem_st32(trow + L::T_O + 32u * c, w);
          }
          tmem_st_wait();
        }
      }
      const f32x2 rf2 = pack2(rf, rf), mr2 = pack2(-ref, -ref);
      uint32_t ph[32], pl[32];
      f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < FL_TILE / 4; c++) {
        const ulonglong2 v4 = vp[c];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          float e0, e1;
          unpack2(fma2(x[2 * c + k], rf2, mr2), e0, e1);
          const f32x2 p = pack2(ex2(e0), ex2(e1));
          sum[k] = add2(sum[k], p);
          float w0, w1;
          unpack2(mul2(p, k ? v4.y : v4.x), w0, w1);
          const __half2 h = __floats2half2_rn(w0, w1);
          ph[2 * c + k] = h2_as_u32(h);
          const float2 g = __half22float2(h);
          pl[2 * c + k] = h2_as_u32(__floats2half2_rn(w0 - g.x, w1 - g.y));
        }
      }
      if ((vflag & 1) && !whole) {
        // A key that this row does not see has a NaN scale: its weight is nothing.
        const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
        for (int c = 0; c < FL_TILE / 2; c++) {
          const uint32_t w = c < 16 ? s0 : s1;
          const uint32_t keep = (w >> (2 * c & 31) & 1 ? 0xffffu : 0u) | (w >> (2 * c + 1 & 31) & 1 ? 0xffff0000u : 0u);
          ph[c] &= keep;
          pl[c] &= keep;
        }
      }
      {
        float a0, a1, b0, b1;
        unpack2(sum[0], a0, a1);
        unpack2(sum[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
      }
      tmem_st32(ts, ph);
      tmem_st32(ts + 32u, pl);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full + (t & 1));  // two: a warp may be a tile ahead of another (S_{t+1} is there early)
    }
    // O (in the values' own scale), reference and l to shared memory: Q, K and V are no
    // longer read (the last products have completed).
    float *ost = reinterpret_cast<float *>(smem) + rr * L::OST;
    if (ok && ntile > 0) {
      // (alone, a CTA divides here; a row that saw nothing: zeros)
      float vo = 0.f;
      ok = with_totals(ntile > FL_WINDOW, all_done, 0u, [&](int d, const float4 &v) {
        if (d == 0) vo = CL > 1 ? *vref_s : (l == 0.f ? 0.f : *vref_s / l);
        *reinterpret_cast<float4 *>(ost + d) = make_float4(v.x * vo, v.y * vo, v.z * vo, v.w * vo);
      });
    } else if (ok) {
#pragma unroll 4
      for (int d = 0; d < D; d += 4) *reinterpret_cast<float4 *>(ost + d) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    row_ref[rr] = m == -INFINITY ? -INFINITY : ref;
    row_l[rr] = l;
  }
  // All roles meet before any takes registers back: a warp that gave its up and
  // took them again at once could leave the softmax waiting for its share. Behind
  // the barrier the softmax gives, the others take, and none waits for another.
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (warp < 4)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FL_REGS));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FL_REGS));
  if (CL > 1) cluster.sync();
  pdl_wait();  // no CTA ends before the append it was launched beside
  // Rows to memory, a cluster's ranks sharing them.
  const float *o_s = reinterpret_cast<const float *>(smem);
  constexpr int D4 = D / 4;
  const int rows = *abort_flag ? 0 : min(FL_ROWS, nrows - row0);  // (a wait that gave up: nothing)
  auto put = [&](int rr, int c, const float4 &acc) {
    const int r = row0 + rr;
    const int64_t at = ((int64_t)b * a.S + r / G) * a.H * D + (int64_t)(kvh * G + r % G) * D + 4 * c;
    if (a.out) *reinterpret_cast<float4 *>(a.out + at) = acc;
    if (a.out16) {
      const __half2 h0 = __floats2half2_rn(acc.x, acc.y), h1 = __floats2half2_rn(acc.z, acc.w);
      *reinterpret_cast<uint2 *>(a.out16 + at) = make_uint2(h2_as_u32(h0), h2_as_u32(h1));
    }
  };
  if (CL == 1) {
#pragma unroll 4
    for (int e = tid; e < rows * D4; e += FL_THREADS)
      put(e / D4, e % D4, *reinterpret_cast<const float4 *>(o_s + e / D4 * L::OST + 4 * (e % D4)));
  } else {
#pragma unroll 1
    for (int e = rank * FL_THREADS + tid; e < rows * D4; e += CL * FL_THREADS) {
      const int rr = e / D4, c = e % D4;
      const float *src = o_s + rr * L::OST + 4 * c;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      // four ranks at once, their loads ahead of the first use (one after the other: 56 us for 53)
      float top = -INFINITY, sum = 0.f;
      for (int q0 = 0; q0 < CL; q0 += 4) {
        float sm[4], sl[4];
        const float was = top;
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int q = q0 + k;
          sm[k] = -INFINITY, sl[k] = 0.f, v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (q < CL) {
            sm[k] = *cluster.map_shared_rank(row_ref + rr, q);
            sl[k] = *cluster.map_shared_rank(row_l + rr, q);
            v[k] = *cluster.map_shared_rank(reinterpret_cast<const float4 *>(src), q);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) top = fmaxf(top, sm[k]);
        // none if a rank saw no key; with a NaN sum and no reference the NaN is passed on
        const float keep = sum == 0.f ? 0.f : (was == -INFINITY ? 1.f : ex2(was - top));
        sum *= keep, acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float f = sl[k] == 0.f ? 0.f : (sm[k] == -INFINITY ? 1.f : ex2(sm[k] - top));
          sum += sl[k] * f;
          acc.x += v[k].x * f, acc.y += v[k].y * f, acc.z += v[k].z * f, acc.w += v[k].w * f;
        }
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
      put(rr, c, acc);
    }
  }
  if (CL > 1) cluster.sync();  // the others have read this CTA's rows
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// The register split needs what the kernel was designed to be launched with: a
// build with fewer would wait for registers that are not there.
template <auto Kern>
void require_regs_once() {
  static std::atomic<int> regs{0};
  if (regs.load(std::memory_order_acquire) == 0) {
    cudaFuncAttributes at;
    B2M_CUDA(cudaFuncGetAttributes(&at, Kern));
    regs.store(at.numRegs, std::memory_order_release);
  }
  B2M_REQUIRE(regs.load(std::memory_order_acquire) >= FL_REGS, B2M_ERR_UNSUPPORTED,
              "GroupQueryAttention (8-bit cache): the flash kernel was built with another register count");
}

template <bool E4M3, int D>
void launch(const Kv8Args &a, cudaStream_t s) {
  using L = FlashLayout<D>;
  constexpr auto kern = kv8_flash_kernel<E4M3, D>;
  set_smem_limit_once<kern>((int)L::BYTES);
  require_regs_once<kern>();
  const int nrows = a.S * (a.H / a.KVH), tiles = (nrows + FL_ROWS - 1) / FL_ROWS;
  // Key splits up to one wave (two CTAs per SM), each with two tiles or more; and
  // two for calls of one to two waves over a long cache, whose second wave would
  // be part empty (400 CTAs of 59 tiles: 283 us, 326 unsplit, 321 with four; a causal
  // call from an empty cache, 512 CTAs of 1 to 32 tiles, loses: 179 us, 153 unsplit).
  const int64_t ctas = (int64_t)a.B * a.KVH * tiles, wave = 2 * (int64_t)device_sm_count();
  int cl = 1;
  while (cl < FL_MAX_CLUSTER && ctas * cl * 2 <= wave && a.CAP > 2 * FL_TILE * cl) cl *= 2;
  if (cl == 1 && ctas > wave && ctas < 2 * wave && a.CAP >= 2048) cl = 2;
  allow_large_cluster_once<kern>();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.KVH * cl), (unsigned)a.B, (unsigned)tiles);
  cfg.blockDim = dim3(FL_THREADS);
  cfg.dynamicSmemBytes = L::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // starts beside the call's append
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  B2M_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
}

}  // namespace

// Enough rows, head dims and alignments the kernel takes. The other kernel reads
// the cache once per 16 rows: from 33 rows on this one is faster where the other's
// CTAs are more than one wave (32 x 8 (sequence, kv head)s over 1500 keys: 40 rows
// 98 us, 137 there, 48 rows 99 and 139; 32 rows 98 and 97). With few CTAs it takes over
// from 49 rows (2 x 8 over 6000 keys: 48 rows 53 us, 45 there, 64 rows 54 and 46: the
// border lies higher still).
bool kv8_flash_shape(const Kv8Args &a) {
  auto al = [](const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  const int64_t rows = (int64_t)a.S * (a.H / a.KVH);
  const bool enough = rows > 48 || (rows > 32 && (int64_t)a.B * a.KVH * 3 > 2 * (int64_t)device_sm_count());
  return (a.D == 64 || a.D == 128) && enough && rows <= 65535 * FL_ROWS && a.KVH <= 65535 && q_rows_vec(a) &&
         al(a.kc, 16) && al(a.vc, 16) && al(a.out, 16) && al(a.out16, 8);
}

// The launch before this one must be that of the call's append.
void launch_kv8_flash(const Kv8Args &a, cudaStream_t s) {
  if (a.e4m3) {
    if (a.D == 128)
      launch<true, 128>(a, s);
    else
      launch<true, 64>(a, s);
  } else {
    if (a.D == 128)
      launch<false, 128>(a, s);
    else
      launch<false, 64>(a, s);
  }
}
