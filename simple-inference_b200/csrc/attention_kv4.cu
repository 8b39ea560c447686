// attention_kv4.cu -- decode attention over the paged KV cache in 4 bits.
//
// Per query token and head h of KV group g = h / (Hq/Hkv), over the token's
// keys t: s_t = q.k_t / sqrt(D), out = sum_t softmax(s)_t v_t, where
// k_t = d_kt,b (n_kt - 8) per block b of 32 dims (d the fp16 scale, n the code)
// and v_t alike.  A token without keys gives a row of zeros.
//
// Arithmetic.  Both contractions run on fp16 matrix instructions with fp32
// accumulators, and no input is rounded to fewer than 22 bits:
//   * two codes n masked out of their word and ORed into the mantissa of 1024
//     are the fp16 numbers 1024 + n (nibbles 0 and 2) or 1024 + 16 n (nibbles 1
//     and 3); one packed subtraction leaves n - 8 or 16 (n - 8), exactly.  The 16
//     goes into the other operand or the result.  (The masked word by itself,
//     the subnormal n 2^-24, would save both steps, but the instruction aligns
//     its products by the operands' nominal exponents and loses the low bits:
//     2.5e-6 relative error against 2e-7);
//   * a query is scaled by a power of two so that its largest value is just
//     below 2^15 and split into two halves, hi = fp16(q), lo = fp16(q - hi).
//     The instruction has 16 rows and a KV group at most 8 heads: hi is rows
//     0-7 and lo rows 8-15, whose results land in the same lane and are added,
//     so the split costs no further instruction;
//   * a block's sum of q (n - 8) is multiplied by d_k in fp32 and added to the
//     score;
//   * P.V: p d_v per block is the left operand, again as hi and lo rows.  p is
//     split once per key; the product's hi is the rounded fp16 product and its
//     lo the exact remainder of that (a fused multiply-add) plus p_lo d_v.  Powers
//     of two that follow the largest |d_v| seen keep both in range, so a cache of
//     small values keeps its bits;
//   * running maximum, sum and output are fp32 per warp, merged over the warps
//     of the CTA and over splits at the end.  The maximum is raised only by a
//     score more than 2^4 above it, so probabilities stay below 16 and the
//     output is rarely rescaled.
//
// Work split.  A CTA of four warps takes one (token, KV head, split of the
// keys); a warp walks every fourth tile of 32 keys of its split on its own.  A
// tile is two contiguous groups of 16 positions with their scales, which one lane
// brings by two bulk copies into the warp's private ring of two, so there is no
// barrier between the warps until the merge.  The query operand is made once per
// CTA and read from shared memory, which leaves registers for three CTAs per SM
// (four with spills: 58 against 55 us).  Up to eight splits of a token are one
// thread-block cluster and merge through distributed shared memory (72B, 8 x 4096
// keys: 23.2 -> 19.7 us); more go through scratch and a second kernel.
//
// Not bound by the cache's bytes: a tile of 4608 bytes takes 823 instructions, some 350
// of them to bring the codes into the operands, at 2.3 of 4 a cycle and SM.  Three warps
// a scheduler are too few to fill the rest: of the stalls the fixed latencies of
// dependent instructions come first (0.99 of an issue), then full math pipes (0.79; the
// fullest, the ALU, is busy 45 % of the time).  72B heads on B200: 131071 keys 53.0 us
// (2.8 TB/s; the copies alone 35.5 us), 8 x 4096 keys 19.4 us.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "si_common.cuh"
#include "si_kernels.cuh"
#include "si_tma.cuh"

namespace si {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 2 * kKv4Group;       // keys per warp step
constexpr int kMinSplit = kWarps * kTile;  // a split has at least one tile per warp
constexpr int kStages = 2;
constexpr int kHeads = 8;                  // query heads of a KV group, at most
constexpr int kCtasPerSm = 3;
constexpr int kMaxCluster = 8;             // splits that are merged within the kernel
constexpr float kStaleMax = 4.0f;          // log2 units a score may lie above the maximum

template <int D>
struct Shape {
  static constexpr int NB = D / 32;
  static constexpr int GB = kv4_group_bytes(D);
  static constexpr int TILE = 2 * GB;
  static constexpr int S_OFF = kKv4Group * (D / 2);  // K scales in a group
  static constexpr int V_OFF = GB / 2;               // V codes in a group
  static constexpr int OROW = D + 4;                 // merge row, one 16-byte step of padding
  static constexpr int RING = kWarps * kStages * TILE;
  static constexpr int MERGE = kWarps * kHeads * (OROW + 2) * 4;
  static constexpr int Q = NB * 2 * 32 * 16;         // query operand
  static constexpr int AMAX = (NB > 2 ? NB : 2) * kHeads * 4;  // later (m, l) per head
  static constexpr int BARS = kWarps * kStages * 8;
  static constexpr int SMEM = Q + AMAX + BARS + (RING > MERGE ? RING : MERGE);
};

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error below 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1,
                                         const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
}
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
// (hi, lo) fp16 pairs of two floats: 22 significant bits together.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2bits(h);
  lo = h2bits(__floats2half2_rn(x - f.x, y - f.y));
}
// The codes of one nibble position of a word of four: n - 8 (low nibble of each
// byte) or 16 (n - 8) (high nibble), two per register.  `one_k` is 1024 twice,
// taken from the kernel's arguments: as a constant the compiler would mask and
// OR in two steps, since an instruction holds one constant (72B, 131071 keys:
// 66.2 -> 61.3 us).
__device__ __forceinline__ uint32_t codes_lo(uint32_t w, uint32_t one_k) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(x) : "r"(w), "r"(one_k));
  return h2bits(__hsub2(as_h2(x), __half2half2(__ushort_as_half(0x6408))));
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w, uint32_t one_k) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(x) : "r"(w), "r"(one_k));
  return h2bits(__hsub2(as_h2(x), __half2half2(__ushort_as_half(0x6480))));
}
__device__ __forceinline__ float half_at(const uint32_t *w, int i) {
  const __half2 h = as_h2(w[i >> 1]);
  return (i & 1) ? __high2float(h) : __low2float(h);
}
__device__ __forceinline__ float pow2(int e) {  // 2^e, 0 below the normal range
  return e < -126 ? 0.0f : __int_as_float((e + 127) << 23);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// The whole warp waits for a stage's copies, 2 s at most.
__device__ __forceinline__ bool wait_tile(uint32_t bar, uint32_t parity) {
  bool ok = mbar_try(bar, parity);
  if (!ok) {
    const uint64_t t0 = globaltimer();
    while (!(ok = mbar_try(bar, parity)) && globaltimer() - t0 < 2000000000ull) {}
  }
  return __all_sync(0xffffffffu, ok) != 0;
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void *p, int cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(cta));
  return r;
}
__device__ __forceinline__ float2 cluster_ld2(const float2 *p, int cta) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(cluster_addr(p, cta))
               : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_ld4(const float *p, int cta) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr(p, cta))
               : "memory");
  return v;
}

struct Token {
  int seq, len, row;
};
__device__ __forceinline__ Token token_of(const Kv4AttnArgs &a, int t) {
  Token k;
  if (a.tok_ctx) {
    k.seq = k.row = t;
    k.len = a.tok_ctx[t];
  } else {
    int lo = 0, hi = a.runs.n;
    k.row = a.runs.row0[0] + t;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.runs.row0[mid] <= k.row) lo = mid;
      else hi = mid;
    }
    k.seq = a.runs.seq[lo];
    k.len = a.runs.pos[lo] + (k.row - a.runs.row0[lo]) + 1;
  }
  const long long most = (long long)a.kv.max_pages * a.kv.page_len;
  k.len = k.len < 0 ? 0 : ((long long)k.len > most ? (int)most : k.len);
  if (k.seq < 0 || k.seq >= a.kv.n_seqs) k.len = 0;
  return k;
}
// Keys per split of a token of `len` keys: an even share, so that a token's
// splits, which are one cluster, end together.
__host__ __device__ __forceinline__ int split_keys(int len, int nsplit) {
  const int per = (len + nsplit - 1) / nsplit;
  const int up = (per + kTile - 1) / kTile * kTile;
  return up > kMinSplit ? up : kMinSplit;
}
// Two fp32 operations per instruction, each rounded on its own.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mov.b64 rc, {%6, %7};\n\tfma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm)
    k_attn_kv4(const __grid_constant__ Kv4AttnArgs a) {
  using S = Shape<D>;
  constexpr int NB = S::NB;
  extern __shared__ __align__(16) uint8_t smem_all[];
  uint4 *q_s = reinterpret_cast<uint4 *>(smem_all);                  // [NB][2][32 lanes]
  float *amax_s = reinterpret_cast<float *>(smem_all + S::Q);        // [NB][8 heads]
  uint8_t *smem = smem_all + S::Q + S::AMAX + S::BARS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;  // operand row (head) and column group
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.x, kvh = blockIdx.y;
  const Token tk = token_of(a, blockIdx.z);
  const int G = a.n_q_heads / a.kv.n_kv_heads;
  const int per = split_keys(tk.len, a.nsplit);
  const int ns = tk.len > 0 ? (tk.len + per - 1) / per : 1;
  if (split >= ns) return;
  const int k0 = split * per, k1 = min(tk.len, k0 + per);
  const int ntiles = (k1 - k0 + kTile - 1) / kTile;
  const int mine = ntiles > warp ? (ntiles - warp + kWarps - 1) / kWarps : 0;

  // This warp's part of the query (see below), asked for before the tables.
  float x[8] = {};
  if (warp < NB && g < G) {
    const float *q = a.q + ((size_t)tk.row * a.n_q_heads + (size_t)kvh * G + g) * D + 32 * warp + 8 * t;
    const float4 u = *reinterpret_cast<const float4 *>(q);
    const float4 v = *reinterpret_cast<const float4 *>(q + 4);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  }

  // Group addresses of this warp's tiles, 16 tiles at a time: lane j holds the
  // pool index of group j & 1 of tile j / 2 of the batch, -1 past the keys or
  // where the table has no page (which is recorded).
  const int gpp = a.kv.gpp;
  const int *table = a.kv.tables + (size_t)tk.seq * a.kv.max_pages;
  uint8_t *ring = smem + warp * (kStages * S::TILE);
  int gidx = -1;
  const uint32_t bars = smem_u32(smem_all + S::Q + S::AMAX) + warp * (kStages * 8);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  uint32_t okb = 0;  // group validity of the tiles in flight, 2 bits each
  auto issue = [&](int n) {
    if ((n & 15) == 0) {
      const int key = k0 + (warp + kWarps * (n + (lane >> 1))) * kTile + (lane & 1) * kKv4Group;
      gidx = -1;
      if (key < k1) {
        const int gi = key / kKv4Group, pi = a.kv.page_of(gi);
        const int page = table[pi];
        if (page >= 0 && page < a.kv.n_pages)
          gidx = (page * a.kv.n_kv_heads + kvh) * gpp + (gi - pi * gpp);
        else
          raise_error(a.err, 1);
      }
    }
    const int g0 = __shfl_sync(0xffffffffu, gidx, (2 * n) & 31);
    const int g1 = __shfl_sync(0xffffffffu, gidx, (2 * n + 1) & 31);
    const int sh = (n & 15) * 2;
    okb = (okb & ~(3u << sh)) | ((uint32_t)(g0 >= 0) << sh) | ((uint32_t)(g1 >= 0) << (sh + 1));
    if (lane == 0) {
      const uint32_t bar = bars + 8 * (n % kStages), dst = smem_u32(ring + (n % kStages) * S::TILE);
      mbar_expect_tx(bar, (g0 >= 0 ? S::GB : 0) + (g1 >= 0 ? S::GB : 0));
      if (g0 >= 0) bulk_load(dst, a.kv.pool + (size_t)(uint32_t)g0 * S::GB, S::GB, bar);
      if (g1 >= 0) bulk_load(dst + S::GB, a.kv.pool + (size_t)(uint32_t)g1 * S::GB, S::GB, bar);
    }
  };
#pragma unroll
  for (int n = 0; n < kStages - 1; ++n)
    if (n < mine) issue(n);

  // The query operand: head g's values of dims 32b + 8t + 0..7, scaled and
  // split, block b by warp b.
  float sc;  // score in log2 units per unit of the accumulators
  {
    if (warp < NB) {
      float am = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) am = fmaxf(am, fabsf(x[i]));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      if (t == 0) amax_s[warp * kHeads + g] = am;
    }
    __syncthreads();
    float am = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) am = fmaxf(am, amax_s[b * kHeads + g]);
    const int e = min(127, 14 - ((int)(__float_as_uint(am) >> 23) - 127));
    const float up = pow2(e);
    sc = ldexpf(1.4426950408889634f / sqrtf((float)D), -e);
    if (warp < NB) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // k columns 2t, 2t+1: nibble 2i of the two half-words; 2t+8, 2t+9:
        // nibble 2i + 1, whose codes come 16-fold.
        uint4 f;
        split2(x[2 * i] * up, x[2 * i + 4] * up, f.x, f.y);
        split2(x[2 * i + 1] * up * 0.0625f, x[2 * i + 5] * up * 0.0625f, f.z, f.w);
        q_s[(warp * 2 + i) * 32 + lane] = f;
      }
    }
    __syncthreads();
  }

  const uint32_t one_k = a.one_k;
  float acc[NB * 4][4];
#pragma unroll
  for (int i = 0; i < NB * 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  // P.V operands are (p 2^p_shift) (d_v 2^d_shift) for |d_v| < 2^(eR + 1); both factors
  // and the product stay below 2^15 (p below 2^4).  fp16 has no step finer than 2^-24,
  // so that keys far below the maximum keep their bits p and the products both have to
  // lie high: the largest d_v goes to 2^-3 to 2.  (Unscaled from 2^-8 to 2^8, with p
  // making room for it, a first key 12 nats above 2100 others of size 300 or 0.01 cost
  // those 1e-4 of their sum, now 2e-6.)  Only eR is kept: with the shifts in registers
  // of their own 131071 keys took 53.6 us instead of 52.9.
  int eR = -1000;
  auto scaled = [](int e) { return e < -2 || e > 0; };  // values outside 1 to 8
  auto d_shift = [&](int e) { return scaled(e) ? -e : 0; };
  auto p_shift = [&](int e) { return scaled(e) || e == 0 ? 10 : 11; };

  for (int n = 0; n < mine; ++n) {
    if (n + kStages - 1 < mine) issue(n + kStages - 1);
    if (!wait_tile(bars + 8 * (n % kStages), (n / kStages) & 1)) {
      // The copies that are still under way are given as long again, then the
      // warp stops.
      if (lane == 0) raise_error(a.err, 6 /* SI_ERR_TIMEOUT */);
      if (n + 1 < mine) wait_tile(bars + 8 * ((n + 1) % kStages), ((n + 1) / kStages) & 1);
      break;
    }
    uint8_t *st = ring + (n % kStages) * S::TILE;
    const int lim = k1 - (k0 + (warp + kWarps * n) * kTile);  // keys of this tile, >= 1
    const uint32_t ok2 = (okb >> ((n & 15) * 2)) & 3u;
    const bool full = lim >= kTile && ok2 == 3u;
    // Lane = key: the scales of keys that do not take part are cleared (their
    // rows may hold anything), and the largest |d_v| of the tile is found.
    const bool in = lane < lim && ((ok2 >> (lane >> 4)) & 1u);
    uint8_t *srow = st + (lane >> 4) * S::GB + S::S_OFF + (lane & 15) * (2 * NB);
    if (!full) {
      if (!in) {
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          reinterpret_cast<uint32_t *>(srow)[i] = 0;
          reinterpret_cast<uint32_t *>(srow + S::V_OFF)[i] = 0;
        }
        fence_proxy_async();  // before the stage's next copy
      }
      __syncwarp();
    }
    uint32_t vmax = 0;
#pragma unroll
    for (int i = 0; i < NB / 2; ++i)
      vmax = __vmaxu2(vmax, reinterpret_cast<const uint32_t *>(srow + S::V_OFF)[i] & 0x7fff7fffu);
    vmax = max(vmax & 0xffffu, vmax >> 16);

    // Scores: n-tile (grp, nt) column c is key 16 grp + 8 nt + c / 2 + 4 (c & 1).
    float s[8];
    {
      uint32_t w[4][NB], d0[4][NB / 2], d1[4][NB / 2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // n-tile (grp, nt) = (i / 2, i % 2)
        const uint8_t *gp = st + (i >> 1) * S::GB;
        const int nt = i & 1;
        const uint8_t *kr = gp + (8 * nt + (g >> 1) + 4 * (g & 1)) * (D / 2) + t * (4 * NB);
        const uint8_t *dp = gp + S::S_OFF + (8 * nt + t) * (2 * NB);
        if constexpr (NB == 4) {
          const uint4 r = *reinterpret_cast<const uint4 *>(kr);
          w[i][0] = __byte_perm(r.x, r.z, 0x5410);
          w[i][1] = __byte_perm(r.x, r.z, 0x7632);
          w[i][2] = __byte_perm(r.y, r.w, 0x5410);
          w[i][3] = __byte_perm(r.y, r.w, 0x7632);
          const uint2 r0 = *reinterpret_cast<const uint2 *>(dp);
          const uint2 r1 = *reinterpret_cast<const uint2 *>(dp + 4 * (2 * NB));
          d0[i][0] = r0.x; d0[i][1] = r0.y; d1[i][0] = r1.x; d1[i][1] = r1.y;
        } else {
          const uint2 r = *reinterpret_cast<const uint2 *>(kr);
          w[i][0] = __byte_perm(r.x, r.y, 0x5410);
          w[i][1] = __byte_perm(r.x, r.y, 0x7632);
          d0[i][0] = *reinterpret_cast<const uint32_t *>(dp);
          d1[i][0] = *reinterpret_cast<const uint32_t *>(dp + 4 * (2 * NB));
        }
      }
      float2 s2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s2[i] = make_float2(0.f, 0.f);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint4 qa = q_s[(b * 2) * 32 + lane], qb = q_s[(b * 2 + 1) * 32 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          float c[4];
          const uint32_t x = w[i][b], h = x >> 8;
          mma16816(c, qa.x, qa.y, qa.z, qa.w, codes_lo(x, one_k), codes_hi(x, one_k), zero);
          mma16816(c, qb.x, qb.y, qb.z, qb.w, codes_lo(h, one_k), codes_hi(h, one_k), c);
          s2[i] = fma2(make_float2(half_at(d0[i], b), half_at(d1[i], b)),
                       add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])), s2[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[2 * i] = s2[i].x * sc;
        s[2 * i + 1] = s2[i].y * sc;
      }
    }
    if (!full) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = (i >> 2) * 16 + ((i >> 1) & 1) * 8 + t + 4 * (i & 1);
        if (key >= lim || !((ok2 >> (i >> 2)) & 1u)) s[i] = -INFINITY;
      }
    }
    float mt = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mt = fmaxf(mt, s[i]);
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
    // A raised maximum or a larger V scale rescales the sums; rare after the
    // first tile.
    const bool raise = mt > m + kStaleMax;
    const bool grow = (int)(vmax >> 10) - 15 > eR;
    if (__any_sync(0xffffffffu, raise || grow)) {
      float f = 1.0f;
      if (raise) {
        f = ex2(m - mt);  // 0 from no keys yet
        m = mt;
        l *= f;
      }
      const uint32_t vm = __reduce_max_sync(0xffffffffu, vmax);
      if ((int)(vm >> 10) - 15 > eR) {
        const int old = p_shift(eR) + d_shift(eR);
        eR = (int)(vm >> 10) - 15 + 1;  // one binade ahead
        f *= pow2(p_shift(eR) + d_shift(eR) - old);  // (the sums are 0 at the first tile)
      }
#pragma unroll
      for (int i = 0; i < NB * 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= f;
    }
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = ex2(s[i] - mu);
      l += s[i];
    }
#pragma unroll
    for (int grp = 0; grp < 2; ++grp) {
      const uint8_t *vp = st + grp * S::GB + S::V_OFF;
      uint32_t cw[4][NB / 2], dv[4][NB / 2];  // keys t, t + 4, t + 8, t + 12
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint8_t *cp = vp + (t + 4 * e) * (D / 2) + g * (2 * NB);
        const uint8_t *dp = vp + S::S_OFF + (t + 4 * e) * (2 * NB);
        if constexpr (NB == 4) {
          const uint2 x = *reinterpret_cast<const uint2 *>(cp);
          const uint2 y = *reinterpret_cast<const uint2 *>(dp);
          cw[e][0] = x.x; cw[e][1] = x.y; dv[e][0] = y.x; dv[e][1] = y.y;
        } else {
          cw[e][0] = *reinterpret_cast<const uint32_t *>(cp);
          dv[e][0] = *reinterpret_cast<const uint32_t *>(dp);
        }
      }
      const float up = p_shift(eR) == 11 ? 2048.0f : 1024.0f;
      float ps[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) ps[e] = s[grp * 4 + e] * up;
      if (scaled(eR)) {  // (3 to 4 % of the call)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // Scaling d down would cost the small d of a key that dominates: there p, which
          // has bits to spare, takes the factor.
          const float c = pow2(-eR);
          const bool by_p = eR > 0 && s[grp * 4 + e] >= 0.5f;
          if (by_p) ps[e] *= c;
          const __half2 c2 = __float2half2_rn(by_p ? 1.0f : c);
#pragma unroll
          for (int i = 0; i < NB / 2; ++i) dv[e][i] = h2bits(__hmul2(as_h2(dv[e][i]), c2));
        }
      }
      uint32_t ph01, pl01, ph23, pl23;
      split2(ps[0], ps[1], ph01, pl01);
      split2(ps[2], ps[3], ph23, pl23);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t sel = (b & 1) ? 0x7632 : 0x5410;
        const __half2 d01 = as_h2(__byte_perm(dv[0][b >> 1], dv[1][b >> 1], sel));
        const __half2 d23 = as_h2(__byte_perm(dv[2][b >> 1], dv[3][b >> 1], sel));
        const __half2 q01 = __hmul2_rn(as_h2(ph01), d01), q23 = __hmul2_rn(as_h2(ph23), d23);
        const uint32_t h01 = h2bits(q01), h23 = h2bits(q23);
        const uint32_t l01 =
            h2bits(__hfma2(as_h2(pl01), d01, __hfma2(as_h2(ph01), d01, __hneg2(q01))));
        const uint32_t l23 =
            h2bits(__hfma2(as_h2(pl23), d23, __hfma2(as_h2(ph23), d23, __hneg2(q23))));
        uint32_t x = __byte_perm(cw[0][b >> 1], cw[1][b >> 1], sel);
        uint32_t y = __byte_perm(cw[2][b >> 1], cw[3][b >> 1], sel);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          if (j == 2) {
            x >>= 8;
            y >>= 8;
          }
          mma16816(acc[b * 4 + j], h01, l01, h23, l23, codes_lo(x, one_k), codes_lo(y, one_k),
                   acc[b * 4 + j]);
          mma16816(acc[b * 4 + j + 1], h01, l01, h23, l23, codes_hi(x, one_k), codes_hi(y, one_k),
                   acc[b * 4 + j + 1]);
        }
      }
    }
    __syncwarp();  // the stage may be refilled
  }
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();

  // Merge of the warps over the ring's memory.
  float *ow = reinterpret_cast<float *>(smem);
  float2 *ml = reinterpret_cast<float2 *>(smem + kWarps * kHeads * S::OROW * 4);
  float2 *cta_ml = reinterpret_cast<float2 *>(amax_s);  // [8 heads]
  {
    const float f0 = mine ? ldexpf(1.0f, -(p_shift(eR) + d_shift(eR))) : 0.0f, f1 = f0 * 0.0625f;
    float *o = ow + (warp * kHeads + g) * S::OROW + 8 * t;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int u = 0; u < 2; ++u)  // column 2t: dims 8t + j; 2t + 1: dims 8t + 4 + j
        *reinterpret_cast<float4 *>(o + 32 * b + 4 * u) =
            make_float4((acc[b * 4][u] + acc[b * 4][u + 2]) * f0,
                        (acc[b * 4 + 1][u] + acc[b * 4 + 1][u + 2]) * f1,
                        (acc[b * 4 + 2][u] + acc[b * 4 + 2][u + 2]) * f0,
                        (acc[b * 4 + 3][u] + acc[b * 4 + 3][u + 2]) * f1);
    }
    if (t == 0) ml[warp * kHeads + g] = make_float2(m, l);
  }
  __syncthreads();
  // The CTA's sums over its warps go to the output (one split), to warp 0's place
  // for the cluster's merge, or to the scratch.
  for (int i = threadIdx.x; i < G * (D / 4); i += kWarps * 32) {
    const int h = i / (D / 4), c = i % (D / 4);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w * kHeads + h].x);
    const float Mu = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = ml[w * kHeads + h];
      const float f = ex2(x.x - Mu);
      const float4 y = *reinterpret_cast<const float4 *>(ow + (w * kHeads + h) * S::OROW + 4 * c);
      L = fmaf(x.y, f, L);
      o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y);
      o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
    }
    const size_t head = (size_t)kvh * G + h;
    if (ns == 1) {
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      *reinterpret_cast<float4 *>(a.out + ((size_t)tk.row * a.n_q_heads + head) * D + 4 * c) =
          make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else if (a.cluster) {
      *reinterpret_cast<float4 *>(ow + h * S::OROW + 4 * c) = o;  // read by this thread alone
      if (c == 0) cta_ml[h] = make_float2(M, L);
    } else {
      const size_t slot = ((size_t)blockIdx.z * a.n_q_heads + head) * a.nsplit + split;
      const size_t slots = (size_t)gridDim.z * a.n_q_heads * a.nsplit;
      if (c == 0)
        *reinterpret_cast<float2 *>(a.part + kv4_part_ml(slots, slot, D)) = make_float2(M, L);
      *reinterpret_cast<float4 *>(a.part + kv4_part_out(slot, D) + 4 * c) = o;
    }
  }
  if (ns == 1 || !a.cluster) return;
  // The splits of a token are one cluster: each CTA merges its share of the output
  // from the others' shared memory, in the order of the splits.
  cluster_sync_all();
  for (int i = split * (kWarps * 32) + threadIdx.x; i < G * (D / 4); i += ns * (kWarps * 32)) {
    const int h = i / (D / 4), c = i % (D / 4);
    float2 x[kMaxCluster];
    float M = -INFINITY;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      x[r] = r < ns ? cluster_ld2(cta_ml + h, r) : make_float2(-INFINITY, 0.0f);
      M = fmaxf(M, x[r].x);
    }
    const float Mu = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      if (r >= ns) break;
      const float f = ex2(x[r].x - Mu);
      const float4 y = cluster_ld4(ow + h * S::OROW + 4 * c, r);
      L = fmaf(x[r].y, f, L);
      o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y);
      o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<float4 *>(a.out + ((size_t)tk.row * a.n_q_heads + (size_t)kvh * G + h) * D +
                                4 * c) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
  cluster_sync_all();  // no CTA leaves while another may still read its sums
}

// Splits of a token merged: grid (Hq, T).  A warp takes every eighth split, a lane
// four dims (D = 64: half a warp a split), all its loads in flight; the warps'
// sums are then added in order.
constexpr int kCombineWarps = 8;
template <int D>
__global__ void __launch_bounds__(kCombineWarps * 32)
    k_kv4_combine(const __grid_constant__ Kv4AttnArgs a) {
  constexpr int LPR = D / 4, GROUPS = kCombineWarps * 32 / LPR;  // splits read at once
  __shared__ float4 o_s[GROUPS][LPR];
  __shared__ float l_s[GROUPS], m_s[kCombineWarps];
  pdl_trigger();
  pdl_wait();
  const Token tk = token_of(a, blockIdx.y);
  const int per = split_keys(tk.len, a.nsplit);
  const int ns = tk.len > 0 ? (tk.len + per - 1) / per : 1;
  if (ns == 1) return;  // already written
  const size_t slot = ((size_t)blockIdx.y * a.n_q_heads + blockIdx.x) * a.nsplit;
  const size_t slots = (size_t)gridDim.y * a.n_q_heads * a.nsplit;
  const float2 *ml = reinterpret_cast<const float2 *>(a.part + kv4_part_ml(slots, slot, D));
  const float *po = a.part + kv4_part_out(slot, D);
  const int grp = threadIdx.x / LPR, c = threadIdx.x % LPR;
  float M = -INFINITY;
  for (int i = threadIdx.x; i < ns; i += blockDim.x) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((threadIdx.x & 31) == 0) m_s[threadIdx.x >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kCombineWarps; ++w) M = fmaxf(M, m_s[w]);
  const float Mu = M == -INFINITY ? 0.0f : M;
  float L = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = grp; i < ns; i += GROUPS) {
    const float2 x = ml[i];
    const float4 y = *reinterpret_cast<const float4 *>(po + (size_t)i * D + 4 * c);
    const float f = ex2(x.x - Mu);
    L = fmaf(x.y, f, L);
    o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y);
    o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
  }
  o_s[grp][c] = o;
  if (c == 0) l_s[grp] = L;
  __syncthreads();
  if (grp) return;
  for (int i = 1; i < GROUPS; ++i) {
    const float4 y = o_s[i][c];
    o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
    L += l_s[i];
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<float4 *>(a.out + ((size_t)tk.row * a.n_q_heads + blockIdx.x) * D + 4 * c) =
      make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <int D>
cudaError_t launch(Kv4AttnArgs a, cudaStream_t s) {
  // Once per device: more shared memory than a kernel has by default.
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!((ready.load() >> (dev & 63)) & 1)) {
    e = cudaFuncSetAttribute(k_attn_kv4<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Shape<D>::SMEM);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  a.one_k = 0x64006400u;
  a.cluster = a.nsplit > 1 && a.nsplit <= kMaxCluster;
  const dim3 grid(a.nsplit, a.kv.n_kv_heads, a.T);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = Shape<D>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if ((unsigned long long)grid.x * grid.y * grid.z <= kPdlMaxCtas) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  if (a.cluster) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = a.nsplit;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  count_launch();
  e = cudaLaunchKernelEx(&cfg, k_attn_kv4<D>, a);
  if (e != cudaSuccess || a.nsplit == 1 || a.cluster) return e;
  return launch_pdl(k_kv4_combine<D>, dim3(a.n_q_heads, a.T), dim3(kCombineWarps * 32), 0, s, a);
}

}  // namespace

// The number of splits that takes the least time by this count, in keys of one
// slot: with all CTAs at once, the longest split; else what the slots have to do on
// average plus half a split at the end, or whole waves where lengths are equal.  A
// CTA costs some 300 keys by itself, the merge kernel for more than kMaxCluster
// splits 600.  (7B, 64 of 0 to 8191 keys: 130, 82, 81, 78, 84, 82, 93 us for 1 to 6
// and 8 splits; 72B, 8 x 4096: 51, 38, 30, 24, 22, 20, 28 us.)
constexpr int kSlots = 148 * kCtasPerSm;  // CTAs that run at once
constexpr int kCtaKeys = 300, kMergeKeys = 600;

void kv4_pick_splits(Kv4AttnArgs &a) {
  const int Hkv = a.kv.n_kv_heads;
  if (a.tok_ctx) {
    // Lengths up to the cache's are possible: enough splits for one wave.  (The lengths
    // themselves are not known here: long ragged batches get fewer splits than above,
    // short tokens of a long cache a second kernel that they do not need.)
    const int most = a.kv.max_pages * a.kv.page_len;
    a.nsplit = std::max(1, std::min(kSlots / (a.T * Hkv), (most + kMinSplit - 1) / kMinSplit));
    return;
  }
  double keys = 0;
  int longest = 1;
  for (int i = 0; i < a.runs.n; ++i) {
    const int c = a.runs.row0[i + 1] - a.runs.row0[i], len = a.runs.pos[i] + c;
    keys += (double)c * len;
    longest = std::max(longest, len);
  }
  const double even = keys * Hkv / kSlots;
  const int most = (longest + kMinSplit - 1) / kMinSplit;
  const int wave = kSlots / std::max(1, std::min(kSlots, a.T * Hkv));
  double best = 0;
  auto consider = [&](int ns) {
    double n = 0;
    for (int i = 0; i < a.runs.n; ++i) {
      const int c = a.runs.row0[i + 1] - a.runs.row0[i], len = a.runs.pos[i] + c;
      n += (double)c * std::max(1, std::min(ns, (len + kMinSplit - 1) / kMinSplit));
    }
    const double waves = n * Hkv / kSlots, piece = split_keys(longest, ns);
    double cost = waves <= 1 ? piece : std::min(std::ceil(waves) * piece, even + piece / 2);
    cost += kCtaKeys * std::max(1.0, waves) + (ns > kMaxCluster ? kMergeKeys : 0);
    if (best == 0 || cost < 0.97 * best) {
      best = cost;
      a.nsplit = ns;
    }
  };
  for (int ns = 1; ns <= std::min(most, kMaxCluster); ++ns) consider(ns);
  if (most > kMaxCluster && wave > kMaxCluster) consider(std::min(most, wave));
}

size_t kv4_part_floats(const Kv4AttnArgs &a) {
  return a.nsplit > kMaxCluster
             ? kv4_part_size((size_t)a.T * a.n_q_heads * a.nsplit, a.kv.head_dim) : 0;
}

cudaError_t launch_attention_kv4(const Kv4AttnArgs &a, cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  if (reinterpret_cast<uintptr_t>(a.q) & 15 || reinterpret_cast<uintptr_t>(a.out) & 15)
    return cudaErrorMisalignedAddress;
  return a.kv.head_dim == 128 ? launch<128>(a, s) : launch<64>(a, s);
}

}  // namespace si
