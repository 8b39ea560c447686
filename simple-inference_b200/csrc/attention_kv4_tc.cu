// attention_kv4_tc.cu -- prompt attention over the paged KV cache in 4 bits, on
// the tcgen05 tensor cores.
//
// The function of attention_kv4.cu for runs of consecutive tokens: token t of a
// run, at position prefix + t of its sequence, attends positions 0 .. prefix + t.
// Up to eight runs go through one launch of each kernel (7B, four of 300 tokens on
// 400: 49 us, one after the other 100; eight of 64 on 836: 38 and 83).
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
// transposed [Hkv][D][Lp], the runs one after the other, each one's keys rounded up
// to 64.  A CTA takes 128 query rows of a run -- TQ tokens x the G heads of a KV
// group -- and a split of their keys, in tiles of 64 (rows and keys of the next run
// that a copy takes in are not used):
//   S = Q.K^T   TMEM, two tiles by one MMA of 128 columns (one of 64 columns takes
//               the tensor pipe as long)
//   P           TMEM, hi and lo, a buffer for each tile of a pair: the MMA takes its
//               left operand from there, which halves its shared-memory reads
//   O += P.V    TMEM: O and O_lo; finished windows in the softmax warps' registers,
//               half of the dims in each group
// Warp roles (384 threads): warp 0 loads K (and Q at the start), warp 2 V (TMA), warp 1 issues
// the MMAs of the scores, warp 3 those of P.V (a thread's wait on a barrier takes
// some 300 cycles even when it is open, during which the other one's MMAs run),
// warps 4-7 and 8-11 are two softmax groups, one for each tile of a pair.  The
// scores of pair n + 1 follow as soon as both groups have read those of pair n, so
// the tensor pipe has work while the softmax of pair n runs.  The running maximum
// is handed from tile to tile through shared memory, by a tagged word per row (a
// barrier's wait took 300 to 800 cycles there); the reference of the probabilities is
// only raised by a score more than 2^6 above the maximum that set it.  Every wait is
// bounded (about 2 s; SI_ERR_TIMEOUT in the context's error word); on expiry every role
// stops, the CTA's own copies and MMAs in flight are waited for (bounded) and TMEM is
// freed.
//
// Bound by the tensor pipe and shared memory together: an MMA of 128 x 128 x 16
// takes 64 cycles and reads 8 KB of shared memory, all that there is in that time,
// 4 KB with P from TMEM; a pair of tiles takes about 3900 cycles, 3100 of them MMAs.
// 72B heads, 509 tokens on 7680 positions: P through shared memory and one issuing
// warp 417 us, P from TMEM 362, windows taken at the next pair 337, keys a third
// ahead 322, operands by packed arithmetic 305, now 302 (three MMAs a product: 430 TFLOP/s are
// 1290); 7B, a prompt of 2048: 101.  These are runs of some milliseconds; in series of half a
// second and more the card's power lowers the clock: 351 and 109.
#include <algorithm>
#include <atomic>

#include "si_common.cuh"
#include "si_kernels.cuh"
#include "si_tc.cuh"
#include "si_tma.cuh"

namespace si {
namespace k4tc {
using namespace si::tc;

constexpr int BK = 64;     // keys per tile
constexpr int ROWS = 128;  // query rows per CTA
constexpr int PK = 2 * BK;   // keys per score MMA
constexpr int THREADS = 384;
// Registers: launched with kRegs a thread; the control warps give up what the
// softmax warps take (the sums match, else the kernel would wait for good).
constexpr int kRegs = 168, kRegsControl = 56, kRegsSoftmax = 224;
static_assert(THREADS * kRegs >= 128 * kRegsControl + 256 * kRegsSoftmax, "register split");
// Probabilities are 2^(score - reference), at most 2^kTopLog2; a score above that sets
// its row's reference kLiftLog2 below itself.  fp16 has no step finer than 2^-24: with
// the maximum itself as the reference, keys of 2^-17 of the largest one's weight, which
// together may make the whole output, kept 8 bits (a first key 10 nats above 40000
// others: 8e-5 of the row, now 2e-6).  A higher lift makes the reference rise more
// often (11: 7B, a prompt of 2048 tokens 100.7 -> 106.0 us; 7 and 9 cost nothing).
constexpr float kTopLog2 = 15.0f, kLiftLog2 = 9.0f;
constexpr int kWindow = 6;  // tiles per window
constexpr int kMaxSplits = 32;

template <int D>
struct Shape {
  static constexpr int NC = D / 64;               // 128-byte swizzle columns of a Q or K row
  static constexpr int Q_CHUNK = ROWS * 128;
  static constexpr int Q_BYTES = NC * Q_CHUNK;    // one split of Q
  static constexpr int K_CHUNK = PK * 128;
  static constexpr int K_BYTES = NC * K_CHUNK;    // one split of a pair of K tiles
  static constexpr int V_BYTES = D * 128;         // one split of a V^T tile
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * Q_BYTES;        // ring of three: lo, hi, lo, ...
  static constexpr int OFF_V = OFF_K + 3 * K_BYTES;        // [stage][hi, lo]
  static constexpr int OFF_BAR = OFF_V + 4 * V_BYTES;
  static constexpr int OFF_M = OFF_BAR + 256;              // (running maximum, tile) per row
  static constexpr int OFF_L = OFF_M;                      // later: row sums of the two groups
  static constexpr int SMEM = OFF_M + ROWS * 8 + 1024;
  static constexpr uint32_t COL_S = 0, COL_P = 128, COL_O = 256, COL_OL = 256 + D;
};
static_assert(Shape<128>::SMEM <= 232448, "shared memory budget");

// The runs of a launch and where their parts of the operands begin; the last one's
// end stands behind it.
struct Run {
  int seq, prefix, T;
  int row;     // first row of q and out
  int nsplit;  // splits of the keys
  int tok0;    // first token of the Q operand
  int tile0;   // first row tile
  int key0;    // first key of the K and V operands
  int piece0;  // first piece of 256 keys
};
struct Runs {
  int n;
  Run r[kKv4MaxPrompts + 1];
};
// The run that item i of those counted by `first` belongs to.
__device__ __forceinline__ const Run &run_of(const Runs &runs, int Run::*first, int i) {
  int k = 0;
  while (k + 1 < runs.n && runs.r[k + 1].*first <= i) ++k;
  return runs.r[k];
}

struct Params {
  Runs run;
  int T, Hq, G, TQ, Lp, nsplit;  // tokens, keys and most splits of all runs
  float *out;   // rows [.][Hq][D]
  float *part;  // with splits: O [T][Hq][nsplit][D], then (m, l) [T][Hq][nsplit]
  int *err;
  const float *rowf;  // [T][Hq]: with K's power of two takes a row's scores to log2 units
  const int *bits;    // [run][Hkv][2]: largest |scale| of K and V as fp16 bits
};

// The power of two by which a KV head's K or V operands are scaled: |scale| <
// 2^(e + 1), so values are below 2^(e + 4) and operands below 2^14.
__device__ __forceinline__ int operand_shift(int bits) { return 10 - ((bits >> 10) - 15); }

__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
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
// Two waits, asked for at once.
__device__ __forceinline__ bool mbar_wait2(uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2,
                                           volatile int *abort) {
  const bool t1 = mbar_try(b1, p1), t2 = mbar_try(b2, p2);
  return (t1 || mbar_wait(b1, p1, abort)) && (t2 || mbar_wait(b2, p2, abort));
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

__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
    k_attn_kv4_tc(const __grid_constant__ CUtensorMap tmQh, const __grid_constant__ CUtensorMap tmQl,
                  const __grid_constant__ CUtensorMap tmKh, const __grid_constant__ CUtensorMap tmKl,
                  const __grid_constant__ CUtensorMap tmVh, const __grid_constant__ CUtensorMap tmVl,
                  const __grid_constant__ Params p) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_align<1024>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.y;
  const Run &run = run_of(p.run, &Run::tile0, blockIdx.x);
  const int rt = (&run)[1].tile0 - 1 - (int)blockIdx.x;  // longest row tiles first
  const int t0 = rt * p.TQ;
  const int rows = p.G * p.TQ;
  const int last_tok = min(run.T, t0 + p.TQ) - 1;
  // This split's key tiles [kt0, kt0 + nkt) of the row tile's.
  const int all_kt = (run.prefix + last_tok + 1 + BK - 1) / BK;
  const int per = (all_kt + run.nsplit - 1) / run.nsplit;
  const int kt0 = (int)blockIdx.z * per;
  const int nkt = min(all_kt - kt0, per);
  const int nsplits = (all_kt + per - 1) / per;
  const int npair = (nkt + 1) / 2;
  if (nkt <= 0) return;

  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::OFF_BAR);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int B_Q = 0, B_KF = 1, B_KE = 4, B_SF = 7, B_SE = 8, B_VF = 9, B_VE = 11, B_PF = 13,
                B_OD = 15, B_FL = 19, B_FIN = 20, NBAR = 22;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + S::OFF_BAR + NBAR * 8);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::OFF_BAR + NBAR * 8 + 16);
  // A row's maximum as a tile left it, with the tile: one 8-byte word, which the
  // next tile's thread of the row polls.
  volatile unsigned long long *m_s =
      reinterpret_cast<volatile unsigned long long *>(smem + S::OFF_M);
  float *l_s = reinterpret_cast<float *>(smem + S::OFF_L);

  // K comes in units of a pair's lo, then its hi, through a ring of three: the next lo
  // is there when a pair's scores begin, its hi follows into the place of the present
  // lo, which the first third of the MMAs has read.
  auto load_k = [&](int u) {
    const uint32_t dst = smem_u32(smem + S::OFF_K) + u % 3 * S::K_BYTES;
    mbar_expect_tx(bar(B_KF + u % 3), S::K_BYTES);
    // (rows past this run's are read with an odd last tile, and not used)
    const int krow = g * p.Lp + run.key0 + (kt0 + (u & ~1)) * BK;
    for (int c = 0; c < S::NC; ++c)
      tma_load_2d(dst + c * S::K_CHUNK, u & 1 ? &tmKh : &tmKl, c * 64, krow, bar(B_KF + u % 3));
  };
  const int k_first = min(2 * npair, 3);  // units that find the ring empty

  if (threadIdx.x < ROWS) m_s[threadIdx.x] = ~0ull;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NBAR; ++i)
      mbar_init(bar(i), i == B_SE || i == B_FL ? 8 : i >= B_PF && i < B_OD ? 4 : 1);  // warps
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
    // Q and the first of K are on their way while TMEM is allocated.
    pdl_wait();
    const uint32_t qb = smem_u32(smem + S::OFF_Q);
    mbar_expect_tx(bar(B_Q), 2 * S::NC * 128 * rows);
    for (int c = 0; c < S::NC; ++c)
      tma_load_3d(qb + c * S::Q_CHUNK, &tmQh, c * 64, g * p.G, run.tok0 + t0, bar(B_Q));
    load_k(0);
    for (int c = 0; c < S::NC; ++c)
      tma_load_3d(qb + S::Q_BYTES + c * S::Q_CHUNK, &tmQl, c * 64, g * p.G, run.tok0 + t0, bar(B_Q));
    for (int u = 1; u < k_first; ++u) load_k(u);
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
  pdl_wait();  // the operands' kernels
  const uint32_t tmem = *tmem_slot;
  auto fail = [&]() {
    if (p.err) atomicCAS(p.err, 0, 6 /* SI_ERR_TIMEOUT */);
    *abort_flag = 1;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == 0) {
      // ---------------- K producer ----------------
      if (lane == 0) {
        int u = k_first;
        for (; u < 2 * npair; ++u) {
          if (!mbar_wait(bar(B_KE + u % 3), ((u / 3) & 1) ^ 1, abort_flag)) break;
          load_k(u);
        }
        if (u < 2 * npair) fail();
        mbar_drain(bar(B_Q), 0);  // no copy outlives the CTA
        for (int k = max(u - 3, 0); k < u; ++k) mbar_drain(bar(B_KF + k % 3), (k / 3) & 1);
      }
      __syncwarp();
    } else if (warp == 2) {
      // ---------------- V producer ----------------
      if (lane == 0) {
        int i = 0;
        for (; i < nkt; ++i) {
          const int s = i & 1;
          if (!mbar_wait(bar(B_VE + s), ((i >> 1) & 1) ^ 1, abort_flag)) break;
          const uint32_t vb = smem_u32(smem + S::OFF_V + s * 2 * S::V_BYTES);
          mbar_expect_tx(bar(B_VF + s), 2 * S::V_BYTES);
          const int key = run.key0 + (kt0 + i) * BK;
          tma_load_2d(vb, &tmVh, key, g * D, bar(B_VF + s));
          tma_load_2d(vb + S::V_BYTES, &tmVl, key, g * D, bar(B_VF + s));
        }
        if (i < nkt) fail();
        for (int k = max(i - 2, 0); k < i; ++k) mbar_drain(bar(B_VF + (k & 1)), (k >> 1) & 1);
      }
      __syncwarp();
    } else if (warp == 1) {
      // ---------------- S issuer ----------------
      if (lane == 0) {
        const uint32_t qh = smem_u32(smem + S::OFF_Q), ql = qh + S::Q_BYTES;
        const uint32_t kb = smem_u32(smem + S::OFF_K);
        constexpr uint32_t id_s = idesc_f16(ROWS, PK);
        bool ok = mbar_wait(bar(B_Q), 0, abort_flag);
        for (int n = 0; ok && n < npair; ++n) {
          // The scores of two tiles, over those that the softmax warps have read;
          // small products first.
          const int ul = 2 * n, uh = 2 * n + 1;
          const uint32_t kl = kb + ul % 3 * S::K_BYTES, kh = kb + uh % 3 * S::K_BYTES;
          const int full = bar(B_KF + ul % 3), par = (ul / 3) & 1;
          if (n >= 1 ? !mbar_wait2(full, par, bar(B_SE), (n - 1) & 1, abort_flag)
                     : !mbar_wait(full, par, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          auto pass = [&](uint32_t a, uint32_t b, uint32_t acc) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t off = (k & 3) * 32;
              mma_f16(tmem + S::COL_S, smem_desc(a + (k >> 2) * S::Q_CHUNK + off),
                      smem_desc(b + (k >> 2) * S::K_CHUNK + off), id_s, k ? 1u : acc);
            }
          };
          pass(qh, kl, 0);
          mma_commit(bar(B_KE + ul % 3));
          if (!mbar_wait(bar(B_KF + uh % 3), (uh / 3) & 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          pass(ql, kh, 1);
          pass(qh, kh, 1);
          mma_commit(bar(B_SF));
          mma_commit(bar(B_KE + uh % 3));
        }
        if (!ok) fail();
        mma_commit(bar(B_FIN));
        mbar_drain(bar(B_FIN), 0);
      }
      __syncwarp();
    } else if (warp == 3) {
      // ---------------- P.V issuer ----------------
      if (lane == 0) {
        constexpr uint32_t id_o = idesc_f16(ROWS, D);
        bool ok = true;
        for (int j = 0; j < nkt; ++j) {
          const int s = j & 1;
          // (a window's first tile also: both groups have taken the last window's sums)
          if (!mbar_wait2(bar(B_VF + s), (j >> 1) & 1, bar(B_PF + s), (j >> 1) & 1, abort_flag) ||
              (j > 0 && j % kWindow == 0 &&
               !mbar_wait(bar(B_FL), (j / kWindow - 1) & 1, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t vh = smem_u32(smem + S::OFF_V + s * 2 * S::V_BYTES), vl = vh + S::V_BYTES;
          const uint32_t ph = tmem + S::COL_P + s * BK, pl = ph + BK / 2;
          const uint32_t first = j % kWindow != 0;  // a window's first tile overwrites
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ts(tmem + S::COL_OL, ph + 8 * k, smem_desc(vl + k * 32), id_o, k ? 1u : first);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ts(tmem + S::COL_OL, pl + 8 * k, smem_desc(vh + k * 32), id_o, 1u);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ts(tmem + S::COL_O, ph + 8 * k, smem_desc(vh + k * 32), id_o, k ? 1u : first);
          mma_commit(bar(B_OD + (j & 3)));
          mma_commit(bar(B_VE + s));
        }
        if (!ok) fail();
        mma_commit(bar(B_FIN + 1));
        mbar_drain(bar(B_FIN + 1), 0);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------- softmax (two groups of four warps) and epilogue ----------------
    const int grp = (warp - 4) >> 2;
    const int q = warp & 3;  // TMEM lane quarter
    const int r = q * 32 + lane;
    const int tl = r / p.G, hh = r - tl * p.G;
    const int tok = t0 + tl;
    const bool valid = r < rows && tok < run.T;
    const int pos = valid ? run.prefix + tok : -1;  // a padding row attends nothing
    const int *bits = p.bits + 2 * ((int)(&run - p.run.r) * (int)gridDim.y + g);
    const int kshift = operand_shift(bits[0]), vshift = operand_shift(bits[1]);
    // (kept above zero: a masked score times it stays -inf)
    const size_t frow = (size_t)(run.tok0 + tok) * p.Hq + (size_t)g * p.G + hh;
    const float rf = valid ? fmaxf(ldexpf(p.rowf[frow], -kshift), 1.2e-38f) : 0.0f;
    const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16);
    constexpr int H = D / 2;   // this group keeps dims [grp * H, grp * H + H) of the sums
    const uint32_t t_o = t_row + S::COL_O + grp * H, t_ol = t_row + S::COL_OL + grp * H;
    const uint32_t t_p = t_row + S::COL_P + grp * BK;
    float tot[H];              // finished windows, relative to the maximum `mine`
#pragma unroll
    for (int k = 0; k < H; ++k) tot[k] = 0.0f;
    float mine = -INFINITY, l = 0.0f;  // l: this group's tiles, relative to `mine`
    bool ok = true;
    // tot * f1 and the window's sums, times f2
    auto take_window = [&](float f1, float f2) {
#pragma unroll
      for (int c = 0; c < H; c += 32) {
        uint32_t o[32], ol[32];
        tmem_ld32(t_o + c, o);
        tmem_ld32(t_ol + c, ol);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k)
          tot[c + k] = fmaf(tot[c + k], f1, __uint_as_float(o[k]) + __uint_as_float(ol[k])) * f2;
      }
    };
    // The row's maximum as tile j left it (bounded as the other waits).
    auto max_of = [&](int j, float &m) {
      unsigned long long w = m_s[r];
      if (__any_sync(0xffffffffu, (uint32_t)(w >> 32) != (uint32_t)j)) {
        const uint64_t begin = globaltimer();
        bool here;
        do {
          w = m_s[r];
          here = (uint32_t)(w >> 32) == (uint32_t)j;
        } while (!__all_sync(0xffffffffu, here) &&
                 !__any_sync(0xffffffffu, *abort_flag || globaltimer() - begin > 2000000000ull));
        if (!__all_sync(0xffffffffu, here)) return false;
      }
      m = __uint_as_float((uint32_t)w);
      return true;
    };
    auto wait_od = [&](int j) {  // P.V of tile j is done
      return mbar_wait_warp(bar(B_OD + (j & 3)), (j >> 2) & 1, abort_flag);
    };
    for (int i = grp; i < nkt; i += 2) {
      const uint32_t t_s = t_row + S::COL_S + grp * BK;
      if (!mbar_wait_warp(bar(B_SF), (i >> 1) & 1, abort_flag)) {
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
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_SE));
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
      if (i > 0 && !max_of(i - 1, m)) {
        ok = false;
        break;
      }
      const bool resc = mt > m + kTopLog2;
      const float raised = mt - kLiftLog2;
      const float alpha = resc ? ex2(m - raised) : 1.0f;  // 0 from no keys yet
      const float sync = m != mine ? ex2(mine - m) : 1.0f;  // 0 from no keys yet
      if (resc) m = raised;
      m_s[r] = ((unsigned long long)(uint32_t)i << 32) | __float_as_uint(m);
      mine = m;
      l *= sync * alpha;
      // A pair whose first tile begins a window: the last one's sums are taken
      // below, before P.V of that tile overwrites them.
      const int i0 = i & ~1;
      const bool take = i0 > 0 && i0 % kWindow == 0;
      if (!take && __any_sync(0xffffffffu, sync * alpha != 1.0f)) {
#pragma unroll
        for (int k = 0; k < H; ++k) tot[k] *= sync * alpha;
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
      // The P buffer is free once P.V two tiles ago is done.
      if (i >= 2 && !wait_od(i - 2)) {
        ok = false;
        break;
      }
      tc_fence_after();
      tmem_st32(t_p, hw);
      tmem_st32(t_p + 32, lw);
      if (take) {
        if (!wait_od(i0 - 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // The window is relative to the maximum as tile i0 - 1 left it: what group
        // 0 has read, and group 1's own last one.
        take_window(grp == 0 ? sync : 1.0f, grp == 0 ? alpha : sync * alpha);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_FL));
      }
      // A raised maximum rescales the open window, once the previous tile's P.V is
      // done.
      if (i > 0 && !(take && grp == 0) && __any_sync(0xffffffffu, resc)) {
        if (!wait_od(i - 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 2 * D; c += 16) {  // O and O_lo are neighbours
          uint32_t o[16];
          tmem_ld16(t_row + S::COL_O + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tmem_st16(t_row + S::COL_O + c, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_PF + grp));
    }
    // A window that begins with an odd last tile: group 1 has no tile to take the
    // last one's sums at.
    if (ok && grp == 1 && (nkt & 1) && nkt > 1 && (nkt - 1) % kWindow == 0) {
      if (wait_od(nkt - 2)) {
        tc_fence_after();
        take_window(1.0f, 1.0f);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_FL));
      } else {
        ok = false;
      }
    }
    // The last maximum, both groups' sums relative to it, and the last P.V.
    float m = -INFINITY;
    if (ok && !max_of(nkt - 1, m)) ok = false;
    if (ok && m != mine) {
      const float f = ex2(mine - m);
      l *= f;
#pragma unroll
      for (int k = 0; k < H; ++k) tot[k] *= f;
    }
    if (ok && !wait_od(nkt - 1)) ok = false;
    if (!ok && lane == 0) fail();
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the maxima are read
    l_s[grp * ROWS + r] = l;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (ok) {
      tc_fence_after();
      l = l_s[r] + l_s[ROWS + r];
      const float back = ldexpf(1.0f, -vshift);
      const size_t head = (size_t)g * p.G + hh;
      float *orow = p.out + ((size_t)(run.row + tok) * p.Hq + head) * D;
      float f = back;
      if (nsplits == 1) {
        f = l == 0.0f ? 0.0f : back / l;
      } else if (valid) {
        const size_t slot = ((size_t)(run.tok0 + tok) * p.Hq + head) * p.nsplit + blockIdx.z;
        orow = p.part + kv4_part_out(slot, D);
        if (grp == 0)
          *reinterpret_cast<float2 *>(
              p.part + kv4_part_ml((size_t)p.T * p.Hq * p.nsplit, slot, D)) = make_float2(m, l);
      }
      take_window(1.0f, f);
      if (valid) {
#pragma unroll
        for (int k = 0; k < H; k += 4)
          *reinterpret_cast<float4 *>(orow + grp * H + k) =
              make_float4(tot[k], tot[k + 1], tot[k + 2], tot[k + 3]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Splits of a row merged: a warp per (token, head), a lane D / 32 dims and one
// split's maximum and sum; the first splits' sums are asked for before the weights
// are known.
static_assert(kMaxSplits <= 32, "a split per lane");
template <int D>
__global__ void __launch_bounds__(256) k_kv4_tc_combine(const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  constexpr int N = D / 32, AHEAD = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + warp, tt = row / p.Hq;
  if (tt >= p.T) return;
  const Run &run = run_of(p.run, &Run::tok0, tt);
  const int last_tok = min(run.T, ((tt - run.tok0) / p.TQ + 1) * p.TQ) - 1;
  const int all_kt = (run.prefix + last_tok + 1 + BK - 1) / BK;
  const int per = (all_kt + run.nsplit - 1) / run.nsplit;
  const int ns = (all_kt + per - 1) / per;
  if (ns == 1) return;  // already written
  const size_t slot = (size_t)row * p.nsplit;
  const float *po = p.part + kv4_part_out(slot, D) + lane * N;
  float v[AHEAD][N], o[N] = {};
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i0 + i < ns) {
        const float *src = po + (size_t)(i0 + i) * D;
        if constexpr (N == 4) {
          const float4 x = *reinterpret_cast<const float4 *>(src);
          v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2 *>(src);
          v[i][0] = x.x; v[i][1] = x.y;
        }
      }
  };
  load(0);
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (lane < ns)
    ml = *reinterpret_cast<const float2 *>(
        p.part + kv4_part_ml((size_t)p.T * p.Hq * p.nsplit, slot + lane, D));
  float M = ml.x;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
  const float f = ex2(ml.x - (M == -INFINITY ? 0.0f : M));
  float L = ml.y * f;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
  for (int i0 = 0; i0 < ns; i0 += AHEAD) {
    if (i0) load(i0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float w = __shfl_sync(0xffffffffu, f, (i0 + i) & 31);
      if (i0 + i < ns)
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] = fmaf(v[i][k], w, o[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) o[k] = L == 0.0f ? 0.0f : o[k] / L;
  float *dst = p.out + ((size_t)(run.row - run.tok0) * p.Hq + row) * D + lane * N;
  if constexpr (N == 4) *reinterpret_cast<float4 *>(dst) = make_float4(o[0], o[1], o[2], o[3]);
  else *reinterpret_cast<float2 *>(dst) = make_float2(o[0], o[1]);
}

// ---- operands from the cache (layout in kv4.cu) ----------------------------
// Largest |scale| of K and of V of each piece of 256 positions of a run and each KV
// head, as fp16 bits: grid (pieces, Hkv), part [Hkv][pieces].
template <int D>
__global__ void __launch_bounds__(256) k_kv4_absmax(const __grid_constant__ Kv4View kv,
                                                    const __grid_constant__ Runs runs,
                                                    uint2 *__restrict__ part) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32, GB = kv4_group_bytes(D);
  const int head = blockIdx.y, gpp = kv.gpp;
  const Run &run = run_of(runs, &Run::piece0, blockIdx.x);
  const int L = run.prefix + run.T;
  const int *table = kv.tables + (size_t)run.seq * kv.max_pages;
  uint32_t mk = 0, mv = 0;
  const int pos = ((int)blockIdx.x - run.piece0) * 256 + threadIdx.x;
  const int gi = pos / kKv4Group, pi = kv.page_of(gi), page = pos < L ? table[pi] : -1;
  if (page >= 0 && page < kv.n_pages) {
    const uint8_t *g = kv.pool + (((size_t)page * kv.n_kv_heads + head) * gpp + gi - pi * gpp) * GB +
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
  __shared__ uint2 w_s[8];
  if ((threadIdx.x & 31) == 0) w_s[threadIdx.x >> 5] = make_uint2(mk, mv);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) {
      mk = max(mk, w_s[i].x);
      mv = max(mv, w_s[i].y);
    }
    part[(size_t)head * gridDim.x + blockIdx.x] = make_uint2(mk, mv);
  }
}

// The split operands of Q, K and V, in one launch: the first Hkv * Lp / 64 CTAs
// take (64 positions, KV head) of the cache, the others kQRows query rows each.
//
// Q: q * scale, times the power of two that puts the row's largest value just
// below 2^14, split; rowf undoes it.  A warp takes rows one by one, the loads of
// four ahead of their arithmetic.
// K as [Hkv][Lp][D] and V transposed as [Hkv][D][Lp], hi and lo halves, zero
// past a run's end: every CTA first finds its run's and head's largest scales among
// the pieces' (the first one writes them down for the attention).  A thread takes 16 bytes of
// codes, four times eight neighbouring dims, by packed fp16 arithmetic: the rounded
// product is hi, its exact remainder lo.  (The scale times the head's power of two
// is an fp16 number again; of scales 2^-25 of the largest and less it loses bits
// that lie below 2^-36 of the largest value.)  V goes through shared memory for the
// transpose, two dims of eight positions per thread; the 16-byte pieces are XORed by
// the position's octet and parity, so that neither side meets a bank twice.
constexpr int kQRows = 32;
struct SplitArgs {
  Kv4View kv;
  Runs run;
  int Hq, Lp, pieces, q_rows;  // keys, pieces and query rows of all runs
  float scale;
  const float *q;
  const uint2 *part;  // [Hkv][pieces] largest |scale| of K and V, as fp16 bits
  int *bits;          // [run][Hkv][2]
  __half *qh, *ql, *kh, *kl, *vh, *vl;
  float *rowf;
  int *err;
};
template <int D>
__global__ void __launch_bounds__(256) k_split(const __grid_constant__ SplitArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32, GB = kv4_group_bytes(D);
  __shared__ __align__(16) __half sh[BK * D], sl[BK * D];
  const int kv_ctas = a.Lp / BK * a.kv.n_kv_heads;
  if ((int)blockIdx.x >= kv_ctas) {
    constexpr int N = D / 32, R = kQRows / 8;  // values per lane, rows per warp
    const int row0 = (blockIdx.x - kv_ctas) * kQRows + (threadIdx.x >> 5) * R, lane = threadIdx.x & 31;
    float x[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= a.q_rows) break;
      const Run &run = run_of(a.run, &Run::tok0, (row0 + r) / a.Hq);
      const int to_q = (run.row - run.tok0) * a.Hq;  // from the operand's rows to those of q
      const float *src = a.q + (size_t)(row0 + r + to_q) * D + lane * N;
      if constexpr (N == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(src);
        x[r][0] = v.x; x[r][1] = v.y; x[r][2] = v.z; x[r][3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2 *>(src);
        x[r][0] = v.x; x[r][1] = v.y;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + r;
      if (row >= a.q_rows) return;
      float am = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[r][i] = __fmul_rn(x[r][i], a.scale);
        am = fmaxf(am, fabsf(x[r][i]));
      }
      const int ex = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(am)) >> 23);
      const int e = max(-126, min(127, 13 - (ex - 127)));
      const float up = __int_as_float((e + 127) << 23);
      uint32_t h[N / 2], l[N / 2];
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float u = x[r][i] * up, v = x[r][i + 1] * up;
        const float hu = bf16_part(u), hv = bf16_part(v);
        h[i / 2] = pack_h2(hu, hv);
        l[i / 2] = pack_h2(u - hu, v - hv);
      }
      const size_t at = (size_t)row * D + lane * N;
      if constexpr (N == 4) {
        *reinterpret_cast<uint2 *>(a.qh + at) = make_uint2(h[0], h[1]);
        *reinterpret_cast<uint2 *>(a.ql + at) = make_uint2(l[0], l[1]);
      } else {
        *reinterpret_cast<uint32_t *>(a.qh + at) = h[0];
        *reinterpret_cast<uint32_t *>(a.ql + at) = l[0];
      }
      if (lane == 0) a.rowf[row] = ldexpf(1.0f, -e);
    }
    return;
  }
  const int head = blockIdx.x / (a.Lp / BK), at0 = blockIdx.x % (a.Lp / BK) * BK;
  const Run &run = run_of(a.run, &Run::key0, at0);
  const int p0 = at0 - run.key0, L = run.prefix + run.T, gpp = a.kv.gpp;
  const int *table = a.kv.tables + (size_t)run.seq * a.kv.max_pages;
  __shared__ uint2 w_s[8];
  uint2 mx = make_uint2(0, 0);
  for (int i = run.piece0 + threadIdx.x; i < (&run)[1].piece0; i += blockDim.x) {
    const uint2 x = a.part[(size_t)head * a.pieces + i];
    mx = make_uint2(max(mx.x, x.x), max(mx.y, x.y));
  }
  mx.x = __reduce_max_sync(0xffffffffu, mx.x);
  mx.y = __reduce_max_sync(0xffffffffu, mx.y);
  if ((threadIdx.x & 31) == 0) w_s[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = make_uint2(max(mx.x, w_s[i].x), max(mx.y, w_s[i].y));
  if (p0 == 0 && threadIdx.x == 0) {
    int *bits = a.bits + 2 * ((int)(&run - a.run.r) * a.kv.n_kv_heads + head);
    bits[0] = (int)mx.x;
    bits[1] = (int)mx.y;
  }
  const float ck = ldexpf(1.0f, operand_shift((int)mx.x));
  const float cv = ldexpf(1.0f, operand_shift((int)mx.y));
  // (K or V, position, 16 bytes of its codes)
  constexpr int PIECES = D / 32;
  for (int e = threadIdx.x; e < 2 * BK * PIECES; e += blockDim.x) {
    const bool is_v = e >= BK * PIECES;
    const int pp = e / PIECES % BK, t = e % PIECES, pos = p0 + pp;
    uint4 w = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
    uint32_t sc[NB / 2] = {};
    bool bad[NB] = {};
    if (pos < L) {
      const int gi = pos / kKv4Group, pi = a.kv.page_of(gi), page = table[pi], r = pos % kKv4Group;
      if (page >= 0 && page < a.kv.n_pages) {
        const uint8_t *g =
            a.kv.pool + (((size_t)page * a.kv.n_kv_heads + head) * gpp + gi - pi * gpp) * GB;
        const uint8_t *scales = g + kKv4Group * (D / 2) + r * (2 * NB);
        w = *reinterpret_cast<const uint4 *>(g + (is_v ? GB / 2 : 0) + r * (D / 2) + 16 * t);
        // A V scale that is no number must not reach the queries before it, whose
        // probability 0 would not mask it: its key's scores become NaN instead,
        // and with them the rows that attend it.
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          const uint32_t sv = reinterpret_cast<const uint32_t *>(scales + GB / 2)[i];
          sc[i] = is_v ? sv : reinterpret_cast<const uint32_t *>(scales)[i];
          bad[2 * i] = (sv & 0x7c00u) == 0x7c00u;
          bad[2 * i + 1] = (sv & 0x7c000000u) == 0x7c000000u;
        }
      } else {
        raise_error(a.err, 1);
      }
    }
    const uint32_t wq[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Eight dims of block b: half-words of the groups 2k and 2k + 1 of this piece.
      const int b = NB == 4 ? i : i >> 1, k = NB == 4 ? 0 : i & 1;
      const int d = 32 * b + 8 * (NB == 4 ? t : 2 * t + k);
      const uint32_t sel = (b & 1) ? 0x7632 : 0x5410;
      const uint32_t c = NB == 4 ? __byte_perm(wq[b >> 1], wq[2 + (b >> 1)], sel)
                                 : __byte_perm(wq[2 * k], wq[2 * k + 1], sel);
      float f = f16_to_f32((uint16_t)(sc[b >> 1] >> (16 * (b & 1)))) * (is_v ? cv : ck);
      if (bad[b]) f = is_v ? 0.0f : __int_as_float(0x7fffffff);
      const __half2 f2 = __float2half2_rn(f);
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // dims j and j + 4: n - 8 by way of 1024 + n
        const uint32_t m = ((c >> (4 * j)) & 0x000f000fu) | 0x64006400u;
        const __half2 n = __hsub2(as_h2(m), __half2half2(__ushort_as_half(0x6408)));
        const __half2 x = __hmul2_rn(f2, n);
        h[j] = h2bits(x);
        l[j] = h2bits(__hfma2(f2, n, __hneg2(x)));
      }
      const uint4 hi = make_uint4(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410),
                                  __byte_perm(h[0], h[1], 0x7632), __byte_perm(h[2], h[3], 0x7632));
      const uint4 lo = make_uint4(__byte_perm(l[0], l[1], 0x5410), __byte_perm(l[2], l[3], 0x5410),
                                  __byte_perm(l[0], l[1], 0x7632), __byte_perm(l[2], l[3], 0x7632));
      if (is_v) {
        const int at = pp * D + (d ^ (8 * ((pp >> 3) ^ ((pp & 1) << 2))));
        *reinterpret_cast<uint4 *>(sh + at) = hi;
        *reinterpret_cast<uint4 *>(sl + at) = lo;
      } else {
        const size_t kd = ((size_t)head * a.Lp + at0 + pp) * D + d;
        *reinterpret_cast<uint4 *>(a.kh + kd) = hi;
        *reinterpret_cast<uint4 *>(a.kl + kd) = lo;
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < D / 2 * (BK / 8); e += blockDim.x) {  // two dims' eight positions
    const int d = e / (BK / 8) * 2, o = e % (BK / 8);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const __half *src = part ? sl : sh;
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = *reinterpret_cast<const uint32_t *>(src + (8 * o + j) * D + (d ^ (8 * (o ^ ((j & 1) << 2)))));
      const size_t vd = ((size_t)head * D + d) * a.Lp + at0 + 8 * o;
      __half *dst = part ? a.vl : a.vh;
      *reinterpret_cast<uint4 *>(dst + vd) =
          make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410),
                     __byte_perm(x[4], x[5], 0x5410), __byte_perm(x[6], x[7], 0x5410));
      *reinterpret_cast<uint4 *>(dst + vd + a.Lp) =
          make_uint4(__byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632),
                     __byte_perm(x[4], x[5], 0x7632), __byte_perm(x[6], x[7], 0x7632));
    }
  }
}

// The runs' places, and those of the pieces of the scratch.
struct Scratch {
  Runs run;
  int T, Lp, pieces, tiles, nsplit;  // of all runs; most splits
  size_t qh, ql, kh, kl, vh, vl, bits, part_max, rowf, part, bytes;
};
static Scratch carve(const Kv4PromptArgs &a) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const int D = a.kv.head_dim, Hkv = a.kv.n_kv_heads, TQ = ROWS / (a.n_q_heads / Hkv);
  Scratch s{};
  Run *r = s.run.r;
  s.run.n = a.n;
  int longest = 0;
  for (int i = 0; i < a.n; ++i) {
    const Kv4Prompt &x = a.run[i];
    const int L = x.prefix + x.T, keys = (L + BK - 1) / BK * BK;
    r[i].seq = x.seq; r[i].prefix = x.prefix; r[i].T = x.T; r[i].row = x.row;
    r[i + 1].tok0 = r[i].tok0 + x.T;
    r[i + 1].tile0 = r[i].tile0 + (x.T + TQ - 1) / TQ;
    r[i + 1].key0 = r[i].key0 + keys;
    r[i + 1].piece0 = r[i].piece0 + (L + 255) / 256;
    longest = std::max(longest, keys / BK);
  }
  s.T = r[a.n].tok0;
  s.tiles = r[a.n].tile0;
  s.Lp = r[a.n].key0;
  s.pieces = r[a.n].piece0;
  const size_t rows = (size_t)s.T * a.n_q_heads, q = up(rows * D * 2), kv = up((size_t)Hkv * s.Lp * D * 2);
  s.qh = 0;
  s.ql = s.qh + q;
  s.kh = s.ql + q;
  s.kl = s.kh + kv;
  s.vh = s.kl + kv;
  s.vl = s.vh + kv;
  s.bits = s.vl + kv;
  s.part_max = s.bits + up((size_t)a.n * 2 * Hkv * sizeof(int));
  s.rowf = s.part_max + up((size_t)Hkv * s.pieces * sizeof(uint2));
  s.part = s.rowf + up(rows * sizeof(float));
  // Splits of the keys, into about as many tiles each, where the row tiles alone
  // leave SMs idle, as many as take the least time by this count: some 1 us a tile,
  // for the merge 3.5 us and its sums written and read at 4 TB/s.  (7B, 64 tokens on
  // 4136: 84, 56, 41, 34 us in 1, 2, 4 and 9; 300 on 400: 26 us, 29 in two; 72B, 64 on
  // 1436: 39, 35, 30 in 1, 2 and 4.)
  auto splits = [&](int i, int n) {  // of run i, where the longest has n
    const int per = (longest + n - 1) / n, tiles = (r[i + 1].key0 - r[i].key0) / BK;
    return (tiles + per - 1) / per;
  };
  double best = longest;
  s.nsplit = 1;
  for (int n = 2; n <= std::min(longest, kMaxSplits); ++n) {
    long long ctas = 0;
    for (int i = 0; i < a.n; ++i)
      ctas += (long long)(r[i + 1].tile0 - r[i].tile0) * Hkv * splits(i, n);
    if (ctas > 148) break;
    const double t = (double)((longest + n - 1) / n) + 3.5 + (double)rows * n * (D + 2) * 8 / 4e6;
    if (t < best) {
      best = t;
      s.nsplit = n;
    }
  }
  for (int i = 0; i < a.n; ++i) r[i].nsplit = s.nsplit > 1 ? splits(i, s.nsplit) : 1;
  s.bytes = s.part + (s.nsplit > 1 ? kv4_part_size(rows * s.nsplit, D) * sizeof(float) : 0);
  return s;
}

template <int D>
cudaError_t launch(const Kv4PromptArgs &a, char *base, const Scratch &sc, cudaStream_t s) {
  using S = Shape<D>;
  const int Hkv = a.kv.n_kv_heads, Hq = a.n_q_heads, G = Hq / Hkv, TQ = ROWS / G;
  const int Lp = sc.Lp;
  __half *qh = reinterpret_cast<__half *>(base + sc.qh), *ql = reinterpret_cast<__half *>(base + sc.ql);
  __half *kh = reinterpret_cast<__half *>(base + sc.kh), *kl = reinterpret_cast<__half *>(base + sc.kl);
  __half *vh = reinterpret_cast<__half *>(base + sc.vh), *vl = reinterpret_cast<__half *>(base + sc.vl);
  int *bits = reinterpret_cast<int *>(base + sc.bits);
  float *rowf = reinterpret_cast<float *>(base + sc.rowf);
  const float scale = 1.4426950408889634f / sqrtf((float)D);
  const int rows = sc.T * Hq;
  uint2 *part = reinterpret_cast<uint2 *>(base + sc.part_max);
  cudaError_t e = launch_pdl(k_kv4_absmax<D>, dim3(sc.pieces, Hkv), dim3(256), 0, s, a.kv, sc.run,
                             part);
  if (e != cudaSuccess) return e;
  SplitArgs sa{a.kv, sc.run, Hq, Lp, sc.pieces, rows, scale, a.q, part, bits, qh, ql, kh, kl, vh, vl,
               rowf, a.err};
  e = launch_pdl(k_split<D>, dim3(Lp / BK * Hkv + (rows + kQRows - 1) / kQRows), dim3(256), 0, s, sa);
  if (e != cudaSuccess) return e;

  CUtensorMap mQh, mQl, mKh, mKl, mVh, mVl;
  cuuint64_t dQ[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)sc.T};
  cuuint64_t sQ[2] = {(cuuint64_t)D * 2, (cuuint64_t)Hq * D * 2};
  cuuint32_t bQ[3] = {64, (cuuint32_t)G, (cuuint32_t)TQ};
  cuuint64_t dK[2] = {(cuuint64_t)D, (cuuint64_t)Hkv * Lp};
  cuuint64_t sK[1] = {(cuuint64_t)D * 2};
  cuuint32_t bK[2] = {64, (cuuint32_t)PK};
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
  p.run = sc.run;
  p.T = sc.T; p.Hq = Hq; p.G = G; p.TQ = TQ; p.Lp = Lp; p.nsplit = sc.nsplit; p.out = a.out;
  p.part = reinterpret_cast<float *>(base + sc.part);
  p.err = a.err; p.rowf = rowf; p.bits = bits;
  e = cudaFuncSetAttribute(k_attn_kv4_tc<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e != cudaSuccess) return e;
  // The register split needs the count that the kernel was to be compiled to.  (A query
  // that fails is asked again by the next call.)
  static std::atomic<int> regs{0};
  if (regs.load() == 0) {
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, k_attn_kv4_tc<D>);
    if (e != cudaSuccess) return e;
    regs.store(fa.numRegs);
  }
  if (regs.load() < kRegs) return cudaErrorInvalidConfiguration;
  e = launch_pdl(k_attn_kv4_tc<D>, dim3(sc.tiles, Hkv, p.nsplit), dim3(THREADS), S::SMEM, s, mQh,
                 mQl, mKh, mKl, mVh, mVl, p);
  if (e != cudaSuccess || p.nsplit == 1) return e;
  return launch_pdl(k_kv4_tc_combine<D>, dim3((rows + 7) / 8), dim3(256), 0, s, p);
}

}  // namespace k4tc

size_t kv4_prompt_scratch_bytes(const Kv4PromptArgs &a) { return k4tc::carve(a).bytes; }

cudaError_t launch_attention_kv4_prompt(const Kv4PromptArgs &a, void *scratch, size_t scratch_bytes,
                                        cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
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
