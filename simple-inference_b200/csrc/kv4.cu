// kv4.cu -- the paged KV cache in 4 bits: writing rows, reading them back, and
// the device side of its page bookkeeping (table entries, reference counts,
// page copies).
//
// Format.  A row of D values (one position, one KV head, K or V) is quantised
// in blocks of 32 dims by the GGUF Q4_0 rule that the weights follow: m = the
// block's value of largest magnitude (the first at a tie), d = m / -8 in fp32,
// code = min(15, trunc(x * (1/d) + 8.5)), scale = fp16(d); a code stands for
// scale * (code - 8).  Each product and sum is one rounded fp32 operation.
//
// Layout.  A page holds page_len positions (a multiple of 16) of every KV head:
//   pool[page][head][page_len / 16] groups of 16 positions, a group being
//   16 rows of K codes (D/2 bytes), 16 rows of K scales (D/32 fp16), the same
//   two for V: 2304 bytes at D = 128, 72 per row.
// The attention reads a group as one contiguous piece.  Within a row the codes
// lie in 16-bit groups of four neighbouring dims, nibble i = dim i: the group of
// dims 32b + 4g .. 32b + 4g + 3 is half-word g * (D/32) + b, so that the 2*D/32
// bytes of one g hold the same four dims of every block -- what one lane of a
// matrix instruction's operand takes, in one load.
#include <type_traits>

#include "si_common.cuh"
#include "si_kernels.cuh"

namespace si {
namespace {

// The group of position pos of sequence seq for KV head 0, or null where the
// table has no page there.
__device__ __forceinline__ uint8_t *kv4_group(const Kv4View &kv, int seq, int pos, int *page_out) {
  if (seq < 0 || seq >= kv.n_seqs || pos < 0 || pos >= kKv4MaxCtx) return nullptr;
  const int group = pos >> 4, i = kv.page_of(group);
  if (i >= kv.max_pages) return nullptr;
  const int page = kv.tables[(size_t)seq * kv.max_pages + i];
  if (page < 0 || page >= kv.n_pages) return nullptr;
  *page_out = page;
  const size_t g = (size_t)page * kv.n_kv_heads * kv.gpp + (group - i * kv.gpp);
  return kv.pool + g * kv4_group_bytes(kv.head_dim);
}
static_assert(kKv4Group == 16, "positions are split by shifts");

__device__ __forceinline__ int kv4_run_of(const Kv4Runs &r, int t) {
  int lo = 0, hi = r.n;  // the last run with row0 <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (r.row0[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The later of two values of a row, in their order, if its magnitude is larger (as
// bits: a NaN is largest of all), else the first.
__device__ __forceinline__ float larger(float first, float later) {
  return __float_as_uint(fabsf(later)) > __float_as_uint(fabsf(first)) ? later : first;
}

// A warp takes whole rows: lane j of the D/4 lanes of a row holds dims 4j ..
// 4j + 3, one 16-byte load, which is one half-word of the row (block b = j / 8,
// group g = j % 8), so no code moves between lanes.  At D = 64 a warp takes two
// rows at once.  The N rows of a lane are quantised together: the eight lanes of a
// block halve the rows they hold at each exchange, so that lane g ends with the
// extreme of row g % N, divides once and stores one scale (one row after the
// other, with everything in every lane: 2.5 us more of 17 for 4099 tokens of 72B).
// Row k is row r16 of the half-group dst(k), null for one that is not stored.
template <int D, int N, typename Dst>
__device__ __forceinline__ void kv4_store_rows(const float4 (&x)[N], int j, int r16, Dst dst) {
  static_assert(N == 2 || N == 4, "rows of a lane");
  constexpr int NB = D / 32;
  const int b = j >> 3, g = j & 7;
  float m[N];
#pragma unroll
  for (int k = 0; k < N; ++k)
    m[k] = larger(larger(larger(x[k].x, x[k].y), x[k].z), x[k].w);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const bool up = g & o;  // the other lane's values come before this one's
#pragma unroll
    for (int k = 0; k < (o < N ? N / (2 * o) : 1); ++k) {
      float own = m[k], send = m[k];
      if (o < N) {  // of rows 2k and 2k + 1 of those still held, keep one
        own = up ? m[2 * k + 1] : m[2 * k];
        send = up ? m[2 * k] : m[2 * k + 1];
      }
      const float other = __shfl_xor_sync(0xffffffffu, send, o);
      m[k] = larger(up ? other : own, up ? own : other);
    }
  }
  const float d = __fmul_rn(m[0], -0.125f);  // m / -8, exact
  const float id = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float r = __shfl_sync(0xffffffffu, id, (threadIdx.x & 24) + k);
    // The code in the last bits of 2^23 + code, rounded towards zero; what is no
    // number gives 0.
    auto code = [r](float v) {
      const float t = fminf(fmaxf(__fadd_rn(__fmul_rn(v, r), 8.5f), 0.0f), 15.5f);
      return __float_as_uint(__fadd_rz(t, 8388608.0f));
    };
    const uint32_t w = code(x[k].x) + (code(x[k].y) << 4) + (code(x[k].z) << 8) +
                       (code(x[k].w) << 12);
    if (uint8_t *half = dst(k))
      reinterpret_cast<uint16_t *>(half + r16 * (D / 2))[g * NB + b] = (uint16_t)w;
  }
  if (g < N)
    if (uint8_t *half = dst(g))
      reinterpret_cast<uint16_t *>(half + kKv4Group * (D / 2))[r16 * NB + b] = f32_to_f16(d);
}

// CTAs of kWarps warps, grid (tokens, ceil(units / kUnits)): a unit is a query head
// (rotated into q_out; none without q_out), then the K rows, then the V rows of
// the token; a warp loads its kRows units before it works on them.  Bound by the
// latency of the loads and the warps that an SM holds: rows written and read back,
// 4099 tokens of 72B, 24 us with four warps of four rows, 27 with two rows each, 31
// in eight warps, 29 with eight rows each, 24 in two warps of eight (their bytes alone
// would take 12).  In a layer step (STEP) the K rows and queries are
// rotated first (rope_kv.cu's arithmetic).  A position without a page, or whose page other
// sequences hold too, is not written and recorded as SI_ERR_INVALID.
constexpr int kWarps = 4, kRows = 4, kUnits = kWarps * kRows;

template <int D, bool VEC, bool STEP>
__global__ void __launch_bounds__(32 * kWarps) k_kv4_append(const __grid_constant__ Kv4AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int HALF = D / 2, LPR = D / 4, RPW = 32 / LPR;  // lanes per row, rows per warp
  constexpr int N = kRows / RPW;
  const int t = blockIdx.x, lane = threadIdx.x & 31, j = lane % LPR;
  const int nq = STEP ? a.n_q_heads : 0, Hkv = a.kv.n_kv_heads, units = nq + 2 * Hkv;
  int seq, pos, row = t;
  if (a.tok_ctx) {
    seq = t;
    pos = a.tok_ctx[t] - 1;
  } else {
    row = a.runs.row0[0] + t;
    const int r = kv4_run_of(a.runs, row);
    seq = a.runs.seq[r];
    pos = a.runs.pos[r] + row - a.runs.row0[r];
  }
  const int u0 = blockIdx.y * kUnits + (threadIdx.x >> 5) * (N * RPW) + lane / LPR;
  const size_t qat = STEP ? (size_t)row * a.ldq + 4 * j : 0, at = (size_t)row * a.ldkv + 4 * j;
  float4 x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = u0 + k * RPW;
    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (u < units) {
      const bool is_q = STEP && u < nq, is_v = u >= nq + Hkv;
      const float *src = (is_q ? a.q : is_v ? a.v : a.k) + (is_q ? qat : at) +
                         (is_q ? u : is_v ? u - nq - Hkv : u - nq) * D;
      if constexpr (VEC) x[k] = *reinterpret_cast<const float4 *>(src);
      else x[k] = make_float4(src[0], src[1], src[2], src[3]);
    }
  }
  int page = 0;
  uint8_t *grp = kv4_group(a.kv, seq, pos, &page);
  if (grp && a.kv.refs[page] != 1) grp = nullptr;
  if (!grp && threadIdx.x == 0 && blockIdx.y == 0) raise_error(a.err, 1);
  if constexpr (STEP) {
    if (pos < 0 || pos >= a.max_positions) return;  // never read outside the tables
    const int i = (4 * j) % HALF;
    const float4 c = *reinterpret_cast<const float4 *>(a.cos_tab + (size_t)pos * HALF + i);
    const float4 s = *reinterpret_cast<const float4 *>(a.sin_tab + (size_t)pos * HALF + i);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int u = u0 + k * RPW;
      float4 y;  // the other half of the pair
      y.x = __shfl_xor_sync(0xffffffffu, x[k].x, LPR / 2);
      y.y = __shfl_xor_sync(0xffffffffu, x[k].y, LPR / 2);
      y.z = __shfl_xor_sync(0xffffffffu, x[k].z, LPR / 2);
      y.w = __shfl_xor_sync(0xffffffffu, x[k].w, LPR / 2);
      if (u < nq + Hkv) {
        auto rot = [&](float own, float other, float c, float s) {
          return j < LPR / 2 ? __fsub_rn(__fmul_rn(own, c), __fmul_rn(other, s))
                             : __fadd_rn(__fmul_rn(own, c), __fmul_rn(other, s));
        };
        x[k] = make_float4(rot(x[k].x, y.x, c.x, s.x), rot(x[k].y, y.y, c.y, s.y),
                           rot(x[k].z, y.z, c.z, s.z), rot(x[k].w, y.w, c.w, s.w));
      }
      if (u < nq)
        *reinterpret_cast<float4 *>(a.q_out + ((size_t)row * a.n_q_heads + u) * D + 4 * j) = x[k];
    }
    if (!__any_sync(0xffffffffu, u0 + (N - 1) * RPW >= nq)) return;  // queries alone
  }
  const uint32_t head_bytes = (uint32_t)a.kv.gpp * kv4_group_bytes(D);  // below 2^20
  kv4_store_rows<D, N>(x, j, pos & 15, [&](int k) -> uint8_t * {
    const int h = u0 + k * RPW - nq;
    if (!grp || h < 0 || h >= 2 * Hkv) return nullptr;
    return grp + (h < Hkv ? h * head_bytes : (h - Hkv) * head_bytes + kv4_group_bytes(D) / 2);
  });
}

// Code i of a half-word less 8, exact: placed behind 2^23.
__device__ __forceinline__ float code_at(uint32_t w, int i) {
  return __uint_as_float(((w >> (4 * i)) & 15u) | 0x4b000000u) - 8388616.0f;
}

// Rows back to fp32, laid out as above: grid (tokens, ceil(2 Hkv / kUnits)).  A
// position without a page reads as zeros and is recorded.  MARK, for an attention whose
// probability 0 would not mask a V that is no number from the queries before it: its key's
// scores become NaN instead, and with them the rows that attend it.
template <int D, bool MARK>
__global__ void __launch_bounds__(32 * kWarps) k_kv4_read(const __grid_constant__ Kv4ReadArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32, LPR = D / 4, RPW = 32 / LPR, N = kRows / RPW;
  const int lane = threadIdx.x & 31, j = lane % LPR, Hkv = a.kv.n_kv_heads;
  const int row = a.runs.row0[0] + blockIdx.x, r = kv4_run_of(a.runs, row);
  const int pos = a.runs.pos[r] + row - a.runs.row0[r];
  int page;
  const uint8_t *grp = kv4_group(a.kv, a.runs.seq[r], pos, &page);
  if (!grp && threadIdx.x == 0 && blockIdx.y == 0) raise_error(a.err, 1);
  const uint32_t head_bytes = (uint32_t)a.kv.gpp * kv4_group_bytes(D);
  const int r16 = pos & 15, b = j >> 3, g = j & 7;
  const int u0 = blockIdx.y * kUnits + (threadIdx.x >> 5) * (N * RPW) + lane / LPR;
  uint32_t w[N];
  float sc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = u0 + k * RPW;
    w[k] = 0x8888u;
    sc[k] = 0.0f;
    if (grp && u < 2 * Hkv) {
      const uint8_t *p =
          grp + (u < Hkv ? u * head_bytes : (u - Hkv) * head_bytes + kv4_group_bytes(D) / 2);
      w[k] = reinterpret_cast<const uint16_t *>(p + r16 * (D / 2))[g * NB + b];
      const uint16_t *scale = reinterpret_cast<const uint16_t *>(p + kKv4Group * (D / 2)) + r16 * NB + b;
      sc[k] = f16_to_f32(*scale);
      if constexpr (MARK) {
        const uint16_t v = u < Hkv ? scale[kv4_group_bytes(D) / 4] : *scale;  // the V half's
        if ((v & 0x7c00u) == 0x7c00u) sc[k] = u < Hkv ? __int_as_float(0x7fffffff) : 0.0f;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = u0 + k * RPW;
    if (u >= 2 * Hkv) continue;
    float *out = u < Hkv ? a.k : a.v;
    if (!out) continue;
    *reinterpret_cast<float4 *>(out + ((size_t)row * Hkv + (u < Hkv ? u : u - Hkv)) * D + 4 * j) =
        make_float4(sc[k] * code_at(w[k], 0), sc[k] * code_at(w[k], 1), sc[k] * code_at(w[k], 2),
                    sc[k] * code_at(w[k], 3));
  }
}

// Bookkeeping: table entries from kernel parameters (the host's tables may change
// again at once), the reference counts that follow them, and page copies in the same launch: the
// last kWriters CTAs write the entries, the others copy kCopyBytes each of a
// page.  The words are read through a generic pointer: as constants, whose lanes
// read different addresses, they would come one at a time.
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16 * 4;
constexpr int kWriters = 4;

template <int WORDS>
__global__ void __launch_bounds__(kCopyThreads)
    k_kv4_update(const __grid_constant__ Kv4Update<WORDS> u) {
  pdl_trigger();
  pdl_wait();
  const int pieces = (int)((u.page_bytes + kCopyBytes - 1) / kCopyBytes);
  const int *word = u.word;
  asm volatile("" : "+l"(word));
  if (blockIdx.x >= gridDim.x - kWriters) {
    const int w0 = blockIdx.x - (gridDim.x - kWriters), t0 = w0 * kCopyThreads + threadIdx.x;
    auto set = [&](int *entry, int page) {
      const int old = *entry;
      *entry = page;
      if (old >= 0) atomicSub(u.refs + old, 1);
      if (page >= 0) atomicAdd(u.refs + page, 1);
    };
    for (int j = t0 >> 5; j < u.n_spans; j += kWriters * kCopyThreads / 32) {
      int *to = u.tables + word[3 * j];
      const int n = word[3 * j + 1], from = word[3 * j + 2];
      for (int i = threadIdx.x & 31; i < n; i += 32)
        set(to + i, from == -1 ? -1 : from >= 0 ? u.tables[from + i] : word[-2 - from + i]);
    }
    const int *w = word + 3 * u.n_spans;
    for (int i = t0; i < u.n_table; i += kWriters * kCopyThreads) set(u.tables + w[2 * i], w[2 * i + 1]);
    return;
  }
  const int *w = word + 3 * u.n_spans + 2 * u.n_table + 2 * (blockIdx.x / pieces);
  const size_t off = (size_t)(blockIdx.x % pieces) * kCopyBytes;
  const uint8_t *src = u.pool + (size_t)w[0] * u.page_bytes + off;
  uint8_t *dst = u.pool + (size_t)w[1] * u.page_bytes + off;
  const int n = (int)(min(u.page_bytes - off, (size_t)kCopyBytes) / 16);
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = threadIdx.x + i * kCopyThreads;
    if (c < n) v[i] = reinterpret_cast<const uint4 *>(src)[c];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = threadIdx.x + i * kCopyThreads;
    if (c < n) reinterpret_cast<uint4 *>(dst)[c] = v[i];
  }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendArgs &a, cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  const int units = (a.q_out ? a.n_q_heads : 0) + 2 * a.kv.n_kv_heads;
  const dim3 grid(a.T, (units + kUnits - 1) / kUnits);
  const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
            reinterpret_cast<uintptr_t>(a.v) | 4 * a.ldq | 4 * a.ldkv) & 15) == 0;
  auto pick = [&](auto d, auto step) {
    return vec ? k_kv4_append<d.value, true, step.value> : k_kv4_append<d.value, false, step.value>;
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  auto *kern = a.kv.head_dim == 128 ? (a.q_out ? pick(d128, std::true_type()) : pick(d128, std::false_type()))
                                    : (a.q_out ? pick(d64, std::true_type()) : pick(d64, std::false_type()));
  return launch_pdl(kern, grid, dim3(32 * kWarps), 0, s, a);
}

cudaError_t launch_kv4_read(const Kv4ReadArgs &a, cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  const dim3 grid(a.T, (2 * a.kv.n_kv_heads + kUnits - 1) / kUnits);
  auto *kern = a.kv.head_dim == 128 ? (a.mark ? k_kv4_read<128, true> : k_kv4_read<128, false>)
                                    : (a.mark ? k_kv4_read<64, true> : k_kv4_read<64, false>);
  return launch_pdl(kern, grid, dim3(32 * kWarps), 0, s, a);
}

template <int WORDS>
static cudaError_t update(const Kv4Update<WORDS> &u, cudaStream_t s) {
  const int pieces = (int)((u.page_bytes + kCopyBytes - 1) / kCopyBytes);
  return launch_pdl(k_kv4_update<WORDS>, dim3(u.n_copies * pieces + kWriters), dim3(kCopyThreads), 0, s,
                    u);
}
cudaError_t launch_kv4_update(const Kv4Update<kKv4SmallWords> &u, cudaStream_t s) {
  return update(u, s);
}
cudaError_t launch_kv4_update(const Kv4Update<kKv4MediumWords> &u, cudaStream_t s) {
  return update(u, s);
}
cudaError_t launch_kv4_update(const Kv4Update<kKv4LargeWords> &u, cudaStream_t s) {
  return update(u, s);
}

}  // namespace si
