// attention_kv4.cu -- decode attention over the paged KV cache in 4 bits.
//
// Per query token and head h of KV group g = h / (Hq/Hkv), over the token's
// keys t: s_t = q.k_t / sqrt(D), out = sum_t softmax(s)_t v_t, where
// k_t = d_kt,b (n_kt - 8) per block b of 32 dims (d the fp16 scale, n the code)
// and v_t alike.  A token without keys gives a row of zeros.
//
// Arithmetic.  Both contractions run on fp16 matrix instructions with fp32
// accumulators, and no input is rounded to fewer than 22 bits:
//   * a code n masked out of its word is the fp16 subnormal n 2^-24 (nibbles 0
//     and 2) or n 2^-20 (nibbles 1 and 3) as it stands, so unpacking is one AND
//     per two codes and a shift per eight; the powers of two go into the other
//     operand or the result;
//   * a query is scaled by a power of two so that its largest value is just
//     below 2^15 and split into two halves, hi = fp16(q), lo = fp16(q - hi).
//     The instruction has 16 rows and a KV group at most 8 heads: hi is rows
//     0-7 and lo rows 8-15, whose results land in the same lane and are added,
//     so the split costs no further instruction;
//   * a block's sum of q (n - 8) is the instruction's sum of q n started at
//     -8 sum q, then times d_k in fp32 and added to the score;
//   * P.V: p d_v per block is the left operand, again as hi and lo rows, scaled
//     by a power of two per warp that follows the largest |d_v| seen (so that a
//     cache of small values keeps its bits); codes become n - 8 by one packed
//     subtraction, exact in fp16;
//   * running maximum, sum and output are fp32 per warp, merged over the warps
//     of the CTA and over splits at the end.
//
// Work split.  A CTA of four warps takes one (token, KV head, split of the
// keys); a warp walks every fourth tile of 32 keys of its split on its own, its
// tiles staged by cp.async into a private ring (a tile is two contiguous
// groups of 16 positions with their scales), so there is no barrier between
// the warps until the merge.
#include "si_common.cuh"
#include "si_kernels.cuh"
#include "si_tma.cuh"

namespace si {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 2 * kKv4Group;       // keys per warp step
constexpr int kSplitUnit = kWarps * kTile; // a split's keys are a multiple of this
constexpr int kStages = 3;
constexpr int kHeads = 8;                  // query heads of a KV group, at most

template <int D>
struct Shape {
  static constexpr int NB = D / 32;
  static constexpr int GB = kv4_group_bytes(D);
  static constexpr int TILE = 2 * GB;
  static constexpr int CHUNKS = TILE / 16;
  static constexpr int S_OFF = kKv4Group * (D / 2);  // K scales in a group
  static constexpr int V_OFF = GB / 2;               // V codes in a group
  static constexpr int OROW = D + 4;                 // merge row, one 16-byte step of padding
  static constexpr int RING = kWarps * kStages * TILE;
  static constexpr int MERGE = kWarps * kHeads * (OROW + 2) * 4;
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
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
__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
// (hi, lo) fp16 pairs of two floats: 22 significant bits together.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2bits(h);
  lo = h2bits(__floats2half2_rn(x - f.x, y - f.y));
}
__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<const __half2 *>(&a),
                            *reinterpret_cast<const __half2 *>(&b));
  return h2bits(r);
}
__device__ __forceinline__ float half_at(const uint32_t *w, int i) {
  return f16_to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
}
__device__ __forceinline__ float pow2(int e) {  // 2^e, 0 below the normal range
  return e < -126 ? 0.0f : __int_as_float((e + 127) << 23);
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
// Keys per split of a token of `len` keys, and the splits it needs.
__device__ __forceinline__ int split_keys(int len, int nsplit) {
  const int per = (len + nsplit - 1) / nsplit;
  return (per + kSplitUnit - 1) / kSplitUnit * kSplitUnit;
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32, 3) k_attn_kv4(const __grid_constant__ Kv4AttnArgs a) {
  using S = Shape<D>;
  constexpr int NB = S::NB;
  extern __shared__ __align__(16) uint8_t smem[];
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

  // Group addresses of this warp's tiles, 16 tiles at a time: lane j holds the
  // pool index of group j & 1 of tile j / 2 of the batch, -1 past the keys or
  // where the table has no page (which is recorded).
  const int gpp = a.kv.page_len / kKv4Group;
  const int *table = a.kv.tables + (size_t)tk.seq * a.kv.max_pages;
  uint8_t *ring = smem + warp * (kStages * S::TILE);
  int gidx = -1;
  uint32_t okb = 0;  // group validity of the tiles in flight, 2 bits each
  auto issue = [&](int n) {
    if ((n & 15) == 0) {
      const int key = k0 + (warp + kWarps * (n + (lane >> 1))) * kTile + (lane & 1) * kKv4Group;
      gidx = -1;
      if (key < k1) {
        const int gi = key / kKv4Group, pi = gi / gpp;
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
    const uint8_t *p0 = a.kv.pool + (size_t)(uint32_t)g0 * S::GB;
    const uint8_t *p1 = a.kv.pool + (size_t)(uint32_t)g1 * S::GB;
    const uint32_t dst = smem_u32(ring + (n % kStages) * S::TILE);
#pragma unroll
    for (int i = 0; i < (S::CHUNKS + 31) / 32; ++i) {
      const int c = lane + 32 * i;
      const bool second = c >= S::CHUNKS / 2;
      const uint8_t *src = second ? p1 + (c - S::CHUNKS / 2) * 16 : p0 + c * 16;
      if (c < S::CHUNKS && (second ? g1 : g0) >= 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + c * 16), "l"(src)
                     : "memory");
    }
  };
#pragma unroll
  for (int n = 0; n < kStages - 1; ++n) {
    if (n < mine) issue(n);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // The query operand: head g's values of dims 32b + 8t + 0..7, scaled and split.
  uint32_t aq[NB][2][4];
  float cinit[NB];
  float sc;  // score in log2 units per unit of the accumulators
  {
    float x[NB][8];
    float amax = 0.0f;
    const float *q = a.q + ((size_t)tk.row * a.n_q_heads + (size_t)kvh * G + g) * D + 8 * t;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
      if (g < G) {
        u = *reinterpret_cast<const float4 *>(q + 32 * b);
        v = *reinterpret_cast<const float4 *>(q + 32 * b + 4);
      }
      x[b][0] = u.x; x[b][1] = u.y; x[b][2] = u.z; x[b][3] = u.w;
      x[b][4] = v.x; x[b][5] = v.y; x[b][6] = v.z; x[b][7] = v.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[b][i]));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = min(127, 14 - ((int)(__float_as_uint(amax) >> 23) - 127));
    const float up = pow2(e);
    sc = ldexpf(1.4426950408889634f / sqrtf((float)D), 24 - e);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float sum = 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        // k columns 2t, 2t+1: nibble 2s of the two half-words; 2t+8, 2t+9:
        // nibble 2s + 1, whose codes carry 2^4 more.
        const float x0 = x[b][2 * s] * up, x1 = x[b][2 * s + 4] * up;
        const float y0 = x[b][2 * s + 1] * up, y1 = x[b][2 * s + 5] * up;
        split2(x0, x1, aq[b][s][0], aq[b][s][1]);
        split2(y0 * 0.0625f, y1 * 0.0625f, aq[b][s][2], aq[b][s][3]);
        sum += (x0 + x1) + (y0 + y1);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      cinit[b] = sum * (-8.0f / 16777216.0f);
    }
  }

  float acc[NB * 4][4];
#pragma unroll
  for (int i = 0; i < NB * 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  int eR = -1000;  // P.V operands are p d_v 2^(13 - eR)
  float up_v = 0.0f;

  for (int n = 0; n < mine; ++n) {
    if (n + kStages - 1 < mine) issue(n + kStages - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
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
      }
      __syncwarp();
    }
    uint32_t vmax = 0;
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t *>(srow + S::V_OFF)[i] & 0x7fff7fffu;
      vmax = max(vmax, max(w & 0xffffu, w >> 16));
    }
    vmax = __reduce_max_sync(0xffffffffu, vmax);

    // Scores: n-tile (grp, nt) column c is key 16 grp + 8 nt + c / 2 + 4 (c & 1).
    float s[8];
#pragma unroll
    for (int grp = 0; grp < 2; ++grp) {
      const uint8_t *gp = st + grp * S::GB;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const uint8_t *kr = gp + (8 * nt + (g >> 1) + 4 * (g & 1)) * (D / 2) + t * (4 * NB);
        uint32_t w[NB];
        if constexpr (NB == 4) {
          const uint4 r = *reinterpret_cast<const uint4 *>(kr);
          w[0] = __byte_perm(r.x, r.z, 0x5410);
          w[1] = __byte_perm(r.x, r.z, 0x7632);
          w[2] = __byte_perm(r.y, r.w, 0x5410);
          w[3] = __byte_perm(r.y, r.w, 0x7632);
        } else {
          const uint2 r = *reinterpret_cast<const uint2 *>(kr);
          w[0] = __byte_perm(r.x, r.y, 0x5410);
          w[1] = __byte_perm(r.x, r.y, 0x7632);
        }
        uint32_t d0[NB / 2], d1[NB / 2];
        const uint8_t *sp = gp + S::S_OFF + (8 * nt + t) * (2 * NB);
        if constexpr (NB == 4) {
          const uint2 r0 = *reinterpret_cast<const uint2 *>(sp);
          const uint2 r1 = *reinterpret_cast<const uint2 *>(sp + 4 * (2 * NB));
          d0[0] = r0.x; d0[1] = r0.y; d1[0] = r1.x; d1[1] = r1.y;
        } else {
          d0[0] = *reinterpret_cast<const uint32_t *>(sp);
          d1[0] = *reinterpret_cast<const uint32_t *>(sp + 4 * (2 * NB));
        }
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float ci[4] = {cinit[b], cinit[b], 0.0f, 0.0f};
          float c[4];
          mma16816(c, aq[b][0][0], aq[b][0][1], aq[b][0][2], aq[b][0][3], w[b] & 0x000f000fu,
                   w[b] & 0x00f000f0u, ci);
          const uint32_t h = w[b] >> 8;
          mma16816(c, aq[b][1][0], aq[b][1][1], aq[b][1][2], aq[b][1][3], h & 0x000f000fu,
                   h & 0x00f000f0u, c);
          s0 = fmaf(half_at(d0, b), c[0] + c[2], s0);
          s1 = fmaf(half_at(d1, b), c[1] + c[3], s1);
        }
        s[grp * 4 + nt * 2] = s0 * sc;
        s[grp * 4 + nt * 2 + 1] = s1 * sc;
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
    // A raised maximum (or a larger V scale) rescales the sums; rare after the
    // first tiles.
    const int ev = (int)(vmax >> 10) - 15;
    const bool grow = ev > eR + 1;  // the same in every lane
    if (__any_sync(0xffffffffu, mt > m) || grow) {
      const float mn = fmaxf(m, mt);
      const float alpha = mn == -INFINITY ? 1.0f : ex2(m - mn);
      float f = alpha;
      if (grow) {
        f *= pow2(eR - ev);
        eR = ev;
        up_v = pow2(13 - ev);
      }
      m = mn;
      l *= alpha;
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
      float p[4];
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
        p[e] = s[grp * 4 + e] * up_v;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t h01, l01, h23, l23;
        split2(p[0] * half_at(dv[0], b), p[1] * half_at(dv[1], b), h01, l01);
        split2(p[2] * half_at(dv[2], b), p[3] * half_at(dv[3], b), h23, l23);
        const uint32_t sel = (b & 1) ? 0x7632 : 0x5410;
        uint32_t x = __byte_perm(cw[0][b >> 1], cw[1][b >> 1], sel);
        uint32_t y = __byte_perm(cw[2][b >> 1], cw[3][b >> 1], sel);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          if (j == 2) {
            x >>= 8;
            y >>= 8;
          }
          // -8 as 2^-24 and 2^-20 multiples: 0x8008 and 0x8080
          mma16816(acc[b * 4 + j], h01, l01, h23, l23, sub_h2(x & 0x000f000fu, 0x80088008u),
                   sub_h2(y & 0x000f000fu, 0x80088008u), acc[b * 4 + j]);
          mma16816(acc[b * 4 + j + 1], h01, l01, h23, l23,
                   sub_h2(x & 0x00f000f0u, 0x80808080u), sub_h2(y & 0x00f000f0u, 0x80808080u),
                   acc[b * 4 + j + 1]);
        }
      }
    }
    __syncwarp();  // the stage may be refilled
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();

  // Merge of the warps over the ring's memory.
  float *ow = reinterpret_cast<float *>(smem);
  float2 *ml = reinterpret_cast<float2 *>(smem + kWarps * kHeads * S::OROW * 4);
  {
    const float f0 = mine ? ldexpf(1.0f, 24 - (13 - eR)) : 0.0f, f1 = f0 * 0.0625f;
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
    } else {
      const size_t slot = ((size_t)blockIdx.z * a.n_q_heads + head) * a.nsplit + split;
      float2 *pml = reinterpret_cast<float2 *>(a.part);
      float *po = a.part + (size_t)gridDim.z * a.n_q_heads * a.nsplit * 2;
      if (c == 0) pml[slot] = make_float2(M, L);
      *reinterpret_cast<float4 *>(po + slot * D + 4 * c) = o;
    }
  }
}

// Splits of a token merged in order: grid (Hq, T), a thread per dim.
template <int D>
__global__ void __launch_bounds__(D) k_kv4_combine(const __grid_constant__ Kv4AttnArgs a) {
  pdl_trigger();
  pdl_wait();
  const Token tk = token_of(a, blockIdx.y);
  const int per = split_keys(tk.len, a.nsplit);
  const int ns = tk.len > 0 ? (tk.len + per - 1) / per : 1;
  if (ns == 1) return;  // already written
  const size_t slot = ((size_t)blockIdx.y * a.n_q_heads + blockIdx.x) * a.nsplit;
  const float2 *ml = reinterpret_cast<const float2 *>(a.part) + slot;
  const float *po = a.part + (size_t)gridDim.y * a.n_q_heads * a.nsplit * 2 + slot * D;
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
  a.out[((size_t)tk.row * a.n_q_heads + blockIdx.x) * D + threadIdx.x] = L == 0.0f ? 0.0f : o / L;
}

template <int D>
cudaError_t launch(const Kv4AttnArgs &a, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(k_attn_kv4<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Shape<D>::SMEM);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k_attn_kv4<D>, dim3(a.nsplit, a.kv.n_kv_heads, a.T), dim3(kWarps * 32),
                 Shape<D>::SMEM, s, a);
  if (e != cudaSuccess || a.nsplit == 1) return e;
  return launch_pdl(k_kv4_combine<D>, dim3(a.n_q_heads, a.T), dim3(D), 0, s, a);
}

}  // namespace

int kv4_pick_splits(int T, int n_kv_heads, long long keys, int longest) {
  // About three CTAs per SM over the whole call, a split no shorter than one
  // tile per warp.
  const long long target = 148 * 3;
  long long per = (keys * n_kv_heads + target - 1) / target;
  per = (per + kSplitUnit - 1) / kSplitUnit * kSplitUnit;
  if (per < kSplitUnit) per = kSplitUnit;
  const long long ns = (longest + per - 1) / per;
  (void)T;
  return ns < 1 ? 1 : (int)ns;
}

size_t kv4_part_floats(int T, int n_q_heads, int head_dim, int nsplit) {
  return nsplit > 1 ? (size_t)T * n_q_heads * nsplit * (head_dim + 2) : 0;
}

cudaError_t launch_attention_kv4(const Kv4AttnArgs &a, cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  if (reinterpret_cast<uintptr_t>(a.q) & 15 || reinterpret_cast<uintptr_t>(a.out) & 15)
    return cudaErrorMisalignedAddress;
  return a.kv.head_dim == 128 ? launch<128>(a, s) : launch<64>(a, s);
}

}  // namespace si
