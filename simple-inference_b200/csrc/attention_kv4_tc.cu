// attention_kv4_tc.cu -- prompt attention over the paged KV cache in 4 bits, on
// the tcgen05 tensor cores.
//
// The function of attention_kv4.cu for a run of consecutive tokens of one
// sequence: token t of the run, at position prefix + t, attends positions 0 ..
// prefix + t.
//
// Arithmetic.  Both contractions are sums of three fp16 MMAs with fp32
// accumulators, over operands split in two:
//   K and V: scale * (code - 8) has 15 bits, hi = fp16(x) and lo = fp16(x - hi)
//            hold them exactly;
//   Q and P: hi has 8 bits and lo the next 11;
//   a.b = a_hi.b_hi + a_hi.b_lo + a_lo.b_hi (lo.lo is below 2^-20 of it).
// A tensor-core accumulator cuts off, towards zero, what lies below its 24 bits
// at every MMA, so what is added to a large sum, and how often, decides the
// error: the scores' two small products are summed first; the output's go to an
// accumulator of their own; the short hi halves make the large products 19
// bits long; and every kWindow tiles the softmax warps add both accumulators
// into a third with fp32 adds.  Operands are scaled by powers of two (Q per row,
// K and V per KV head) to just below 2^14, so that a cache of small values keeps
// its bits.
//
// Layout.  Pre-passes write the split operands: Q [T][Hq][D], K [Hkv][Lp][D], V
// transposed [Hkv][D][Lp] (Lp = the context rounded up to 64 keys).  A CTA takes
// 128 query rows -- TQ tokens x the G heads of a KV group -- and a split of
// their keys, in tiles of 64:
//   S = Q.K^T   TMEM, 128 x 64 fp32, two buffers
//   P           TMEM, over its own scores: 32 columns of hi pairs, 32 of lo pairs
//   O += P.V    TMEM, P as the MMA's TMEM operand; O, O_lo and the windows' sum
// Warp roles (320 threads): warp 0 TMA producer, warp 1 MMA issue, warps 2-5 and
// 6-9 softmax, the two groups taking turns at the tiles, so that one tile's
// softmax runs beside the next tile's scores and the previous tile's P.V.  The
// running maximum is handed from tile to tile through shared memory; it is only
// raised by a score more than 2^8 above it.  Every wait is bounded (about 2 s;
// SI_ERR_TIMEOUT in the context's error word); on expiry every role stops, the
// CTA's own copies and MMAs in flight are waited for (bounded) and TMEM is freed.
#include <algorithm>

#include "si_common.cuh"
#include "si_kernels.cuh"
#include "si_tc.cuh"
#include "si_tma.cuh"

namespace si {
namespace k4tc {
using namespace si::tc;

constexpr int BK = 64;     // keys per tile
constexpr int ROWS = 128;  // query rows per CTA
constexpr int THREADS = 320;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kWindow = 4;  // tiles per window
constexpr int kMaxSplits = 32;

template <int D>
struct Shape {
  static constexpr int NC = D / 64;               // 128-byte swizzle columns of a Q or K row
  static constexpr int Q_CHUNK = ROWS * 128;
  static constexpr int Q_BYTES = NC * Q_CHUNK;    // one split of Q
  static constexpr int K_CHUNK = BK * 128;
  static constexpr int K_BYTES = NC * K_CHUNK;    // one split of a K tile
  static constexpr int V_BYTES = D * 128;         // one split of a V^T tile
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * Q_BYTES;        // [stage][hi, lo]
  static constexpr int OFF_V = OFF_K + 4 * K_BYTES;        // [stage][hi, lo]
  static constexpr int OFF_BAR = OFF_V + 4 * V_BYTES;
  static constexpr int OFF_M = OFF_BAR + 256;              // running maximum per row
  static constexpr int OFF_L = OFF_M + ROWS * 4;           // row sums of the two groups
  static constexpr int SMEM = OFF_L + 2 * ROWS * 4 + 1024;
  static constexpr uint32_t COL_S = 0, COL_O = 128, COL_OL = 128 + D, COL_OT = 128 + 2 * D;
};
static_assert(Shape<128>::SMEM <= 232448, "shared memory budget");

struct Params {
  int T, Hq, G, TQ, prefix, Lp, ntiles_rows, nsplit;
  float *out;   // rows [T][Hq][D]
  float *part;  // with splits: (m, l) [T][Hq][nsplit], then O [T][Hq][nsplit][D]
  int *err;
  const float *rowf;  // [T][Hq]: takes a row's scores to log2 units
  const int *bits;    // [Hkv][2]: largest |scale| of K and V as fp16 bits
};

// The power of two by which a KV head's K or V operands are scaled: |scale| <
// 2^(e + 1), so values are below 2^(e + 4) and operands below 2^14.
__device__ __forceinline__ int operand_shift(int bits) { return 10 - ((bits >> 10) - 15); }

__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// The left operand from TMEM: lane = row, a column holds two fp16 of the row.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int c0, int c1,
                                            int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ bool mbar_drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_sleep(bar, parity))
    if (globaltimer() - t0 > 2000000000ull) return false;
  return true;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float bf16_part(float x) {  // the nearest number of 8 bits
  return __uint_as_float((__float_as_uint(x) + 0x8000u) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_h2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
    k_attn_kv4_tc(const __grid_constant__ CUtensorMap tmQh, const __grid_constant__ CUtensorMap tmQl,
                  const __grid_constant__ CUtensorMap tmKh, const __grid_constant__ CUtensorMap tmKl,
                  const __grid_constant__ CUtensorMap tmVh, const __grid_constant__ CUtensorMap tmVl,
                  const Params p) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_align<1024>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.y;
  const int rt = p.ntiles_rows - 1 - (int)blockIdx.x;  // longest row tiles first
  const int t0 = rt * p.TQ;
  const int rows = p.G * p.TQ;
  const int last_tok = min(p.T, t0 + p.TQ) - 1;
  // This split's key tiles [kt0, kt0 + nkt) of the row tile's.
  const int all_kt = (p.prefix + last_tok + 1 + BK - 1) / BK;
  const int per = (all_kt + p.nsplit - 1) / p.nsplit;
  const int kt0 = (int)blockIdx.z * per;
  const int nkt = min(all_kt - kt0, per);
  const int nsplits = (all_kt + per - 1) / per;
  if (nkt <= 0) return;

  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::OFF_BAR);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int B_Q = 0, B_KF = 1, B_KE = 3, B_VF = 5, B_VE = 7, B_SF = 9, B_PF = 11, B_MX = 13,
                B_OD = 15, B_FIN = 17, NBAR = 18;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + S::OFF_BAR + NBAR * 8);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::OFF_BAR + NBAR * 8 + 16);
  float *m_s = reinterpret_cast<float *>(smem + S::OFF_M);
  float *l_s = reinterpret_cast<float *>(smem + S::OFF_L);

  if (threadIdx.x == 0) {
    for (int i = 0; i < NBAR; ++i)
      mbar_init(bar(i), (i >= B_PF && i < B_OD) ? 4 : 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&]() {
    if (p.err) atomicCAS(p.err, 0, 6 /* SI_ERR_TIMEOUT */);
    *abort_flag = 1;
  };

  if (warp == 0) {
    // ---------------- producer ----------------
    if (lane == 0) {
      const uint32_t qb = smem_u32(smem + S::OFF_Q);
      mbar_expect_tx(bar(B_Q), 2 * S::NC * 128 * rows);
      for (int c = 0; c < S::NC; ++c) {
        tma_load_3d(qb + c * S::Q_CHUNK, &tmQh, c * 64, g * p.G, t0, bar(B_Q));
        tma_load_3d(qb + S::Q_BYTES + c * S::Q_CHUNK, &tmQl, c * 64, g * p.G, t0, bar(B_Q));
      }
      int nk = 0, nv = 0;
      bool ok = true;
      for (int i = 0; i < nkt; ++i) {
        const int s = i & 1, par = ((i >> 1) & 1) ^ 1;
        if (!mbar_wait(bar(B_KE + s), par, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t kb = smem_u32(smem + S::OFF_K + s * 2 * S::K_BYTES);
        mbar_expect_tx(bar(B_KF + s), 2 * S::K_BYTES);
        const int krow = g * p.Lp + (kt0 + i) * BK;
        for (int c = 0; c < S::NC; ++c) {
          tma_load_2d(kb + c * S::K_CHUNK, &tmKh, c * 64, krow, bar(B_KF + s));
          tma_load_2d(kb + S::K_BYTES + c * S::K_CHUNK, &tmKl, c * 64, krow, bar(B_KF + s));
        }
        ++nk;
        if (!mbar_wait(bar(B_VE + s), par, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t vb = smem_u32(smem + S::OFF_V + s * 2 * S::V_BYTES);
        mbar_expect_tx(bar(B_VF + s), 2 * S::V_BYTES);
        tma_load_2d(vb, &tmVh, (kt0 + i) * BK, g * D, bar(B_VF + s));
        tma_load_2d(vb + S::V_BYTES, &tmVl, (kt0 + i) * BK, g * D, bar(B_VF + s));
        ++nv;
      }
      if (!ok) {
        fail();
        mbar_drain(bar(B_Q), 0);
        for (int k = nk > 2 ? nk - 2 : 0; k < nk; ++k) mbar_drain(bar(B_KF + (k & 1)), (k >> 1) & 1);
        for (int k = nv > 2 ? nv - 2 : 0; k < nv; ++k) mbar_drain(bar(B_VF + (k & 1)), (k >> 1) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t qh = smem_u32(smem + S::OFF_Q), ql = qh + S::Q_BYTES;
      constexpr uint32_t id_s = idesc_f16(ROWS, BK), id_o = idesc_f16(ROWS, D);
      bool ok = mbar_wait(bar(B_Q), 0, abort_flag);
      for (int i = 0; ok && i <= nkt; ++i) {
        if (i < nkt) {
          // S_i goes over P_(i-2), which P.V_(i-2) must have read.
          const int s = i & 1;
          if (!mbar_wait(bar(B_KF + s), (i >> 1) & 1, abort_flag) ||
              (i >= 2 && !mbar_wait(bar(B_OD + s), ((i >> 1) - 1) & 1, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t kh = smem_u32(smem + S::OFF_K + s * 2 * S::K_BYTES), kl = kh + S::K_BYTES;
          const uint32_t d = tmem + S::COL_S + s * BK;
          uint32_t acc = 0;
#pragma unroll
          for (int pass = 0; pass < 3; ++pass) {  // small products first
            const uint32_t a = pass == 1 ? ql : qh, b = pass == 0 ? kl : kh;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t off = (k & 3) * 32;
              mma_ss(d, smem_desc(a + (k >> 2) * S::Q_CHUNK + off),
                     smem_desc(b + (k >> 2) * S::K_CHUNK + off), id_s, acc);
              acc = 1;
            }
          }
          mma_commit(bar(B_SF + s));
          mma_commit(bar(B_KE + s));
        }
        if (i >= 1) {
          const int j = i - 1, s = j & 1;
          if (!mbar_wait(bar(B_VF + s), (j >> 1) & 1, abort_flag) ||
              !mbar_wait(bar(B_PF + s), (j >> 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t vh = smem_u32(smem + S::OFF_V + s * 2 * S::V_BYTES), vl = vh + S::V_BYTES;
          const uint32_t ph = tmem + S::COL_S + s * BK, pl = ph + BK / 2;
          // A window's first tile overwrites (the softmax warps have moved it on).
          const uint32_t first = j % kWindow != 0;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ts(tmem + S::COL_OL, ph + 8 * k, smem_desc(vl + k * 32), id_o, k ? 1u : first);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ts(tmem + S::COL_OL, pl + 8 * k, smem_desc(vh + k * 32), id_o, 1u);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ts(tmem + S::COL_O, ph + 8 * k, smem_desc(vh + k * 32), id_o, k ? 1u : first);
          mma_commit(bar(B_OD + s));
          mma_commit(bar(B_VE + s));
        }
      }
      if (!ok) fail();
      mma_commit(bar(B_FIN));
      mbar_drain(bar(B_FIN), 0);
    }
    __syncwarp();
  } else {
    // ---------------- softmax (two groups of four warps) and epilogue ----------------
    const int grp = (warp - 2) >> 2;
    const int q = warp & 3;  // TMEM lane quarter
    const int r = q * 32 + lane;
    const int tl = r / p.G, hh = r - tl * p.G;
    const int tok = t0 + tl;
    const bool valid = r < rows && tok < p.T;
    const int pos = valid ? p.prefix + tok : -1;  // a padding row attends nothing
    const float rf = valid ? p.rowf[(size_t)tok * p.Hq + (size_t)g * p.G + hh] : 0.0f;
    const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16);
    float mine = -INFINITY, l = 0.0f;  // this group's sum, relative to the maximum `mine`
    bool ok = true;
    for (int i = grp; i < nkt; i += 2) {
      const uint32_t t_s = t_row + S::COL_S + grp * BK;
      if (!mbar_wait_warp(bar(B_SF + grp), (i >> 1) & 1, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float sv[BK];
      {
        uint32_t a[32], b[32];
        tmem_ld32(t_s, a);
        tmem_ld32(t_s + 32, b);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          sv[j] = __uint_as_float(a[j]);
          sv[32 + j] = __uint_as_float(b[j]);
        }
      }
      const int key0 = (kt0 + i) * BK;
      if (__any_sync(0xffffffffu, key0 + BK - 1 > pos)) {
#pragma unroll
        for (int j = 0; j < BK; ++j)
          if (key0 + j > pos) sv[j] = -INFINITY;
      }
      float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
      for (int j = 4; j < BK; ++j) mx[j & 3] = fmaxf(mx[j & 3], sv[j]);
      float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      mt = mt == -INFINITY ? mt : mt * rf;
      // The maximum as the previous tile left it, raised if need be, passed on.
      float m = -INFINITY;
      if (i > 0) {
        if (!mbar_wait_warp(bar(B_MX + ((i - 1) & 1)), ((i - 1) >> 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        m = m_s[r];
      }
      const bool resc = mt > m + kRescaleLog2;
      const float alpha = resc ? ex2(m - mt) : 1.0f;  // 0 from no keys yet
      if (resc) m = mt;
      m_s[r] = m;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_MX + grp));
      if (m != mine) {
        l *= ex2(mine - m);
        mine = m;
      }
      // A window that tile i - 1 closed goes into the sum; a raised maximum
      // rescales what there is.  Both once P.V_(i-1) is done.
      const bool flush = i > 0 && i % kWindow == 0;
      const bool have_total = i > kWindow;  // before this tile's flush
      if (flush || (i > 0 && __any_sync(0xffffffffu, resc))) {
        if (!mbar_wait_warp(bar(B_OD + ((i - 1) & 1)), ((i - 1) >> 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16], ol[16], ot[16];
          tmem_ld16(t_row + S::COL_O + c, o);
          tmem_ld16(t_row + S::COL_OL + c, ol);
          if (have_total) tmem_ld16(t_row + S::COL_OT + c, ot);
          tmem_wait_ld();
          if (flush) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float w = __uint_as_float(o[k]) + __uint_as_float(ol[k]);
              ot[k] = __float_as_uint((have_total ? __uint_as_float(ot[k]) + w : w) * alpha);
            }
            tmem_st16(t_row + S::COL_OT + c, ot);
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              ol[k] = __float_as_uint(__uint_as_float(ol[k]) * alpha);
            }
            tmem_st16(t_row + S::COL_O + c, o);
            tmem_st16(t_row + S::COL_OL + c, ol);
            if (have_total) {
#pragma unroll
              for (int k = 0; k < 16; ++k) ot[k] = __float_as_uint(__uint_as_float(ot[k]) * alpha);
              tmem_st16(t_row + S::COL_OT + c, ot);
            }
          }
        }
        tmem_wait_st();
      }
      const float mu = m == -INFINITY ? 0.0f : m;
      float sum0 = 0.0f, sum1 = 0.0f;
      uint32_t hw[32], lw[32];
#pragma unroll
      for (int j = 0; j < BK; j += 2) {
        // (-inf * 0 of a padding row would be NaN; its results are not used)
        const float p0 = ex2(fmaf(sv[j], rf, -mu)), p1 = ex2(fmaf(sv[j + 1], rf, -mu));
        sum0 += p0;
        sum1 += p1;
        const float h0 = bf16_part(p0), h1 = bf16_part(p1);
        hw[j / 2] = pack_h2(h0, h1);
        lw[j / 2] = pack_h2(p0 - h0, p1 - h1);
      }
      l += sum0 + sum1;
      tmem_st32(t_s, hw);
      tmem_st32(t_s + 32, lw);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_PF + grp));
    }
    // The last maximum, both groups' sums relative to it, and the last P.V.
    float m = -INFINITY;
    if (ok && !mbar_wait_warp(bar(B_MX + ((nkt - 1) & 1)), ((nkt - 1) >> 1) & 1, abort_flag))
      ok = false;
    if (ok) {
      m = m_s[r];
      if (m != mine) l *= ex2(mine - m);
      l_s[grp * ROWS + r] = l;
    }
    if (ok && !mbar_wait_warp(bar(B_OD + ((nkt - 1) & 1)), ((nkt - 1) >> 1) & 1, abort_flag))
      ok = false;
    if (!ok && lane == 0) fail();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (ok) {
      tc_fence_after();
      l = l_s[r] + l_s[ROWS + r];
      const float back = ldexpf(1.0f, -operand_shift(p.bits[2 * g + 1]));
      const size_t head = (size_t)g * p.G + hh;
      float *orow = p.out + ((size_t)tok * p.Hq + head) * D;
      float f = back;
      if (nsplits == 1) {
        f = l == 0.0f ? 0.0f : back / l;
      } else if (valid) {
        const size_t slot = ((size_t)tok * p.Hq + head) * p.nsplit + blockIdx.z;
        orow = p.part + (size_t)p.T * p.Hq * p.nsplit * 2 + slot * D;
        if (grp == 0) reinterpret_cast<float2 *>(p.part)[slot] = make_float2(m, l);
      }
      const bool have_total = nkt > kWindow;
#pragma unroll 1
      for (int c = grp * (D / 2); c < (grp + 1) * (D / 2); c += 16) {
        uint32_t o[16], ol[16], ot[16];
        tmem_ld16(t_row + S::COL_O + c, o);
        tmem_ld16(t_row + S::COL_OL + c, ol);
        if (have_total) tmem_ld16(t_row + S::COL_OT + c, ot);
        tmem_wait_ld();
        if (valid) {
          float w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            w[k] = __uint_as_float(o[k]) + __uint_as_float(ol[k]);
            if (have_total) w[k] += __uint_as_float(ot[k]);
            w[k] *= f;
          }
#pragma unroll
          for (int k = 0; k < 16; k += 4)
            *reinterpret_cast<float4 *>(orow + c + k) =
                make_float4(w[k], w[k + 1], w[k + 2], w[k + 3]);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Splits of a token merged in order: grid (Hq, T), a thread per dim.
template <int D>
__global__ void __launch_bounds__(D) k_kv4_tc_combine(const Params p) {
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.y;
  const int last_tok = min(p.T, (t / p.TQ + 1) * p.TQ) - 1;
  const int all_kt = (p.prefix + last_tok + 1 + BK - 1) / BK;
  const int per = (all_kt + p.nsplit - 1) / p.nsplit;
  const int ns = (all_kt + per - 1) / per;
  if (ns == 1) return;  // already written
  const size_t row = (size_t)t * p.Hq + blockIdx.x, slot = row * p.nsplit;
  const float2 *ml = reinterpret_cast<const float2 *>(p.part) + slot;
  const float *po = p.part + (size_t)p.T * p.Hq * p.nsplit * 2 + slot * D;
  float M = -INFINITY;
  for (int i = 0; i < ns; ++i) M = fmaxf(M, ml[i].x);
  const float Mu = M == -INFINITY ? 0.0f : M;
  float L = 0.0f, o = 0.0f;
  for (int i = 0; i < ns; ++i) {
    const float2 x = ml[i];
    const float f = ex2(x.x - Mu);
    L = fmaf(x.y, f, L);
    o = fmaf(po[(size_t)i * D + threadIdx.x], f, o);
  }
  p.out[row * D + threadIdx.x] = L == 0.0f ? 0.0f : o / L;
}

// ---- operands from the cache (layout in kv4.cu) ----------------------------
// Largest |scale| of K and of V over positions [0, L) of one KV head, as fp16
// bits: grid (pieces of 1024 positions, Hkv); bits [Hkv][2] start at 0.
template <int D>
__global__ void __launch_bounds__(256) k_kv4_absmax(const __grid_constant__ Kv4View kv, int seq,
                                                    int L, int *__restrict__ bits) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32, GB = kv4_group_bytes(D);
  const int head = blockIdx.y, gpp = kv.page_len / kKv4Group;
  const int *table = kv.tables + (size_t)seq * kv.max_pages;
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pos = blockIdx.x * 1024 + i * 256 + threadIdx.x;
    if (pos >= L) break;
    const int gi = pos / kKv4Group, page = table[gi / gpp];
    if (page < 0 || page >= kv.n_pages) continue;
    const uint8_t *g = kv.pool + (((size_t)page * kv.n_kv_heads + head) * gpp + gi % gpp) * GB +
                       kKv4Group * (D / 2) + (pos % kKv4Group) * (2 * NB);
    // (infinite and NaN scales, 0x7c00 and above, do not count)
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) {
      const uint32_t k = reinterpret_cast<const uint32_t *>(g)[b] & 0x7fff7fffu;
      const uint32_t v = reinterpret_cast<const uint32_t *>(g + GB / 2)[b] & 0x7fff7fffu;
      mk = __vmaxu2(mk, k & __vcmpltu2(k, 0x7c007c00u));
      mv = __vmaxu2(mv, v & __vcmpltu2(v, 0x7c007c00u));
    }
  }
  mk = __reduce_max_sync(0xffffffffu, max(mk & 0xffffu, mk >> 16));
  mv = __reduce_max_sync(0xffffffffu, max(mv & 0xffffu, mv >> 16));
  if ((threadIdx.x & 31) == 0) {
    atomicMax(bits + 2 * head, (int)mk);
    atomicMax(bits + 2 * head + 1, (int)mv);
  }
}

// q * scale, times the power of two that puts the row's largest value just
// below 2^14, split; rowf undoes it and the K operand's.  One warp per (token,
// head) row.
template <int D>
__global__ void __launch_bounds__(256) k_split_q4(const float *__restrict__ q, int rows, int Hq,
                                                  int G, float scale, const int *__restrict__ bits,
                                                  __half *__restrict__ qh, __half *__restrict__ ql,
                                                  float *__restrict__ rowf) {
  pdl_trigger();
  pdl_wait();
  constexpr int N = D / 32;  // values per lane
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  float x[N], am = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 v = *reinterpret_cast<const float2 *>(q + (size_t)row * D + lane * N + i);
    x[i] = __fmul_rn(v.x, scale);
    x[i + 1] = __fmul_rn(v.y, scale);
    am = fmaxf(am, fmaxf(fabsf(x[i]), fabsf(x[i + 1])));
  }
  const int ex = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(am)) >> 23);
  const int e = max(-126, min(127, 13 - (ex - 127)));
  const float up = __int_as_float((e + 127) << 23);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float a = x[i] * up, b = x[i + 1] * up;
    const float ha = bf16_part(a), hb = bf16_part(b);
    reinterpret_cast<uint32_t *>(qh)[((size_t)row * D + lane * N + i) / 2] = pack_h2(ha, hb);
    reinterpret_cast<uint32_t *>(ql)[((size_t)row * D + lane * N + i) / 2] = pack_h2(a - ha, b - hb);
  }
  // (kept above zero: a masked score times it stays -inf)
  if (lane == 0)
    rowf[row] = fmaxf(ldexpf(1.0f, -e - operand_shift(bits[2 * (row % Hq / G)])), 1.2e-38f);
}

// K as [Hkv][Lp][D] and V transposed as [Hkv][D][Lp], hi and lo halves, zero
// past L: one CTA per (64 positions, KV head), a thread per half-word of four
// codes; V goes through shared memory for the transpose.
template <int D>
__global__ void __launch_bounds__(256) k_split_kv4(const __grid_constant__ Kv4View kv, int seq,
                                                   int L, int Lp, const int *__restrict__ bits,
                                                   __half *__restrict__ kh, __half *__restrict__ kl,
                                                   __half *__restrict__ vh, __half *__restrict__ vl,
                                                   int *err) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32, GB = kv4_group_bytes(D);
  __shared__ __half sh[BK][D + 8], sl[BK][D + 8];
  const int p0 = blockIdx.x * BK, head = blockIdx.y, gpp = kv.page_len / kKv4Group;
  const int *table = kv.tables + (size_t)seq * kv.max_pages;
  const float ck = ldexpf(1.0f, operand_shift(bits[2 * head]));
  const float cv = ldexpf(1.0f, operand_shift(bits[2 * head + 1]));
  for (int e = threadIdx.x; e < BK * (D / 4); e += blockDim.x) {
    const int pp = e / (D / 4), hw = e % (D / 4), pos = p0 + pp;
    const int b = hw % NB, d = 32 * b + 4 * (hw / NB);
    uint32_t wk = 0x8888u, wv = 0x8888u;
    float sk = 0.0f, sv = 0.0f;
    if (pos < L) {
      const int gi = pos / kKv4Group, page = table[gi / gpp], r = pos % kKv4Group;
      if (page >= 0 && page < kv.n_pages) {
        const uint8_t *g = kv.pool + (((size_t)page * kv.n_kv_heads + head) * gpp + gi % gpp) * GB;
        const uint16_t *c = reinterpret_cast<const uint16_t *>(g + r * (D / 2)) + hw;
        const uint16_t *s = reinterpret_cast<const uint16_t *>(g + kKv4Group * (D / 2)) + r * NB + b;
        wk = c[0];
        wv = c[GB / 4];
        sk = f16_to_f32(s[0]) * ck;
        sv = f16_to_f32(s[GB / 4]) * cv;
        // A V scale that is no number must not reach the queries before it, whose
        // probability 0 would not mask it: its key's scores become NaN instead,
        // and with them the rows that attend it.
        if ((s[GB / 4] & 0x7c00u) == 0x7c00u) {
          sv = 0.0f;
          sk = __int_as_float(0x7fffffff);
        }
      } else {
        raise_error(err, 1);
      }
    }
    __half khi[4], klo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float k = sk * (float)((int)((wk >> (4 * i)) & 15u) - 8);
      const float v = sv * (float)((int)((wv >> (4 * i)) & 15u) - 8);
      khi[i] = __float2half_rn(k);
      klo[i] = __float2half_rn(k - __half2float(khi[i]));
      const __half vhi = __float2half_rn(v);
      sh[pp][d + i] = vhi;
      sl[pp][d + i] = __float2half_rn(v - __half2float(vhi));
    }
    const size_t kd = ((size_t)head * Lp + pos) * D + d;
    *reinterpret_cast<uint2 *>(kh + kd) = *reinterpret_cast<const uint2 *>(khi);
    *reinterpret_cast<uint2 *>(kl + kd) = *reinterpret_cast<const uint2 *>(klo);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < BK * D / 2; e += blockDim.x) {
    const int d = e / (BK / 2), pp = e % (BK / 2) * 2;
    const size_t vd = ((size_t)head * D + d) * Lp + p0 + pp;
    *reinterpret_cast<__half2 *>(vh + vd) = __halves2half2(sh[pp][d], sh[pp + 1][d]);
    *reinterpret_cast<__half2 *>(vl + vd) = __halves2half2(sl[pp][d], sl[pp + 1][d]);
  }
}

// Where the pieces of the scratch lie.
struct Scratch {
  size_t qh, ql, kh, kl, vh, vl, bits, rowf, part, bytes;
  int nsplit;
};
static Scratch carve(const Kv4PromptArgs &a) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const int D = a.kv.head_dim, Hkv = a.kv.n_kv_heads, G = a.n_q_heads / Hkv;
  const size_t L = (size_t)a.prefix + a.T, Lp = (L + BK - 1) / BK * BK;
  const size_t q = up((size_t)a.T * a.n_q_heads * D * 2), kv = up(Hkv * Lp * D * 2);
  Scratch s;
  s.qh = 0;
  s.ql = s.qh + q;
  s.kh = s.ql + q;
  s.kl = s.kh + kv;
  s.vh = s.kl + kv;
  s.vl = s.vh + kv;
  s.bits = s.vl + kv;
  s.rowf = s.bits + up(2 * Hkv * sizeof(int));
  s.part = s.rowf + up((size_t)a.T * a.n_q_heads * sizeof(float));
  // Splits of the keys where the row tiles alone leave SMs idle; a split has
  // eight tiles at least.
  const int TQ = ROWS / G;
  const long long ctas = (long long)((a.T + TQ - 1) / TQ) * Hkv;
  const long long tiles = (long long)(Lp / BK);
  s.nsplit = (int)std::max<long long>(
      1, std::min<long long>({148 / ctas, tiles / 8, (long long)kMaxSplits}));
  s.bytes = s.part + (s.nsplit > 1 ? (size_t)a.T * a.n_q_heads * s.nsplit * (D + 2) * 4 : 0);
  return s;
}

template <int D>
cudaError_t launch(const Kv4PromptArgs &a, char *base, const Scratch &sc, cudaStream_t s) {
  using S = Shape<D>;
  const int Hkv = a.kv.n_kv_heads, Hq = a.n_q_heads, G = Hq / Hkv, TQ = ROWS / G;
  const int L = a.prefix + a.T, Lp = (L + BK - 1) / BK * BK;
  __half *qh = reinterpret_cast<__half *>(base + sc.qh), *ql = reinterpret_cast<__half *>(base + sc.ql);
  __half *kh = reinterpret_cast<__half *>(base + sc.kh), *kl = reinterpret_cast<__half *>(base + sc.kl);
  __half *vh = reinterpret_cast<__half *>(base + sc.vh), *vl = reinterpret_cast<__half *>(base + sc.vl);
  int *bits = reinterpret_cast<int *>(base + sc.bits);
  float *rowf = reinterpret_cast<float *>(base + sc.rowf);
  const float scale = 1.4426950408889634f / sqrtf((float)D);
  const int rows = a.T * Hq;
  cudaError_t e = cudaMemsetAsync(bits, 0, 2 * Hkv * sizeof(int), s);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k_kv4_absmax<D>, dim3((L + 1023) / 1024, Hkv), dim3(256), 0, s, a.kv, a.seq, L,
                 bits);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k_split_q4<D>, dim3((rows + 7) / 8), dim3(256), 0, s, a.q, rows, Hq, G, scale,
                 bits, qh, ql, rowf);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k_split_kv4<D>, dim3(Lp / BK, Hkv), dim3(256), 0, s, a.kv, a.seq, L, Lp, bits, kh,
                 kl, vh, vl, a.err);
  if (e != cudaSuccess) return e;

  CUtensorMap mQh, mQl, mKh, mKl, mVh, mVl;
  cuuint64_t dQ[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)a.T};
  cuuint64_t sQ[2] = {(cuuint64_t)D * 2, (cuuint64_t)Hq * D * 2};
  cuuint32_t bQ[3] = {64, (cuuint32_t)G, (cuuint32_t)TQ};
  cuuint64_t dK[2] = {(cuuint64_t)D, (cuuint64_t)Hkv * Lp};
  cuuint64_t sK[1] = {(cuuint64_t)D * 2};
  cuuint32_t bK[2] = {64, (cuuint32_t)BK};
  cuuint64_t dV[2] = {(cuuint64_t)Lp, (cuuint64_t)Hkv * D};
  cuuint64_t sV[1] = {(cuuint64_t)Lp * 2};
  cuuint32_t bV[2] = {(cuuint32_t)BK, (cuuint32_t)D};
  const auto F16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const auto SW = CU_TENSOR_MAP_SWIZZLE_128B;
  if (!tma_encode(&mQh, F16, 3, qh, dQ, sQ, bQ, SW) || !tma_encode(&mQl, F16, 3, ql, dQ, sQ, bQ, SW) ||
      !tma_encode(&mKh, F16, 2, kh, dK, sK, bK, SW) || !tma_encode(&mKl, F16, 2, kl, dK, sK, bK, SW) ||
      !tma_encode(&mVh, F16, 2, vh, dV, sV, bV, SW) || !tma_encode(&mVl, F16, 2, vl, dV, sV, bV, SW))
    return cudaErrorInvalidValue;
  Params p{};
  p.T = a.T; p.Hq = Hq; p.G = G; p.TQ = TQ; p.prefix = a.prefix; p.Lp = Lp;
  p.ntiles_rows = (a.T + TQ - 1) / TQ; p.nsplit = sc.nsplit; p.out = a.out;
  p.part = reinterpret_cast<float *>(base + sc.part);
  p.err = a.err; p.rowf = rowf; p.bits = bits;
  e = cudaFuncSetAttribute(k_attn_kv4_tc<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e != cudaSuccess) return e;
  count_launch();
  k_attn_kv4_tc<D><<<dim3(p.ntiles_rows, Hkv, p.nsplit), THREADS, S::SMEM, s>>>(mQh, mQl, mKh, mKl,
                                                                               mVh, mVl, p);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.nsplit == 1) return e;
  return launch_pdl(k_kv4_tc_combine<D>, dim3(Hq, a.T), dim3(D), 0, s, p);
}

}  // namespace k4tc

size_t kv4_prompt_scratch_bytes(const Kv4PromptArgs &a) { return k4tc::carve(a).bytes; }

cudaError_t launch_attention_kv4_prompt(const Kv4PromptArgs &a, void *scratch, size_t scratch_bytes,
                                        cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  const k4tc::Scratch sc = k4tc::carve(a);
  if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255) || scratch_bytes < sc.bytes ||
      !tma_encode_fn() || a.n_q_heads / a.kv.n_kv_heads > 8)
    return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a.q) & 15) || (reinterpret_cast<uintptr_t>(a.out) & 15))
    return cudaErrorMisalignedAddress;
  char *base = static_cast<char *>(scratch);
  return a.kv.head_dim == 128 ? k4tc::launch<128>(a, base, sc, s) : k4tc::launch<64>(a, base, sc, s);
}

}  // namespace si
