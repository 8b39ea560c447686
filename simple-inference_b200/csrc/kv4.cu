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
#include "si_common.cuh"
#include "si_kernels.cuh"

namespace si {
namespace {

// The row (16-position group, row in it) of position pos of sequence seq, or
// null where the table has no page there.
__device__ __forceinline__ uint8_t *kv4_group(const Kv4View &kv, int seq, int pos, int head,
                                              int *page_out) {
  if (seq < 0 || seq >= kv.n_seqs || pos < 0 || pos / kv.page_len >= kv.max_pages) return nullptr;
  const int page = kv.tables[(size_t)seq * kv.max_pages + pos / kv.page_len];
  if (page < 0 || page >= kv.n_pages) return nullptr;
  if (page_out) *page_out = page;
  const int gpp = kv.page_len / kKv4Group;
  const size_t g = ((size_t)page * kv.n_kv_heads + head) * gpp + pos % kv.page_len / kKv4Group;
  return kv.pool + g * kv4_group_bytes(kv.head_dim);
}

__device__ __forceinline__ int kv4_run_of(const Kv4Runs &r, int t) {
  int lo = 0, hi = r.n;  // the last run with row0 <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (r.row0[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One warp writes one row: lane = dim within each block of 32.  The codes of
// four neighbouring lanes make a half-word, which lane 4g stores for its g.
template <int D>
__device__ __forceinline__ void kv4_store_row(const float (&x)[D / 32], uint8_t *codes,
                                              uint16_t *scales, int lane) {
  constexpr int NB = D / 32;
  uint32_t hw[NB];
  uint16_t sc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t a = __float_as_uint(fabsf(x[b]));
    const uint32_t amax = __reduce_max_sync(0xffffffffu, a);
    const int first = __ffs(__ballot_sync(0xffffffffu, a == amax)) - 1;
    const float m = __shfl_sync(0xffffffffu, x[b], first);
    const float d = __fmul_rn(m, -0.125f);  // m / -8, exact
    const float id = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
    int q = __float2int_rz(__fadd_rn(__fmul_rn(x[b], id), 8.5f));
    q = min(max(q, 0), 15);
    uint32_t v = (uint32_t)q;
    v |= __shfl_down_sync(0xffffffffu, v, 1) << 4;
    v |= __shfl_down_sync(0xffffffffu, v, 2) << 8;
    hw[b] = v & 0xffffu;
    sc[b] = f32_to_f16(d);
  }
  if ((lane & 3) == 0) {
    uint32_t *dst = reinterpret_cast<uint32_t *>(codes + (lane >> 2) * 2 * NB);
#pragma unroll
    for (int b = 0; b < NB; b += 2) dst[b / 2] = hw[b] | (hw[b + 1] << 16);
  }
  if (lane == 0) {
    uint32_t *dst = reinterpret_cast<uint32_t *>(scales);
#pragma unroll
    for (int b = 0; b < NB; b += 2) dst[b / 2] = sc[b] | ((uint32_t)sc[b + 1] << 16);
  }
}

// One warp per row: grid (tokens, ceil(units / 8)); units are the query heads
// (rotated into q_out; none without q_out), then the K rows, then the V rows.
// With tables the K rows and queries are rotated first (rope_kv.cu's
// arithmetic).  A position without a page, or whose page other sequences hold
// too, is not written and recorded as SI_ERR_INVALID.
template <int D>
__global__ void __launch_bounds__(256) k_kv4_append(const __grid_constant__ Kv4AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32, HALF = D / 2;
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int nq = a.q_out ? a.n_q_heads : 0, Hkv = a.kv.n_kv_heads;
  const int u = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (u >= nq + 2 * Hkv) return;
  int seq, pos, row = t;
  if (a.tok_ctx) {
    seq = t;
    pos = a.tok_ctx[t] - 1;
  } else {
    const int r = kv4_run_of(a.runs, a.runs.row0[0] + t);
    row = a.runs.row0[0] + t;
    seq = a.runs.seq[r];
    pos = a.runs.pos[r] + row - a.runs.row0[r];
  }
  const bool is_v = u >= nq + Hkv;
  const int head = u < nq ? u : (u - nq) % Hkv;
  const float *src = u < nq ? a.q + (size_t)row * a.ldq + (size_t)u * D
                            : (is_v ? a.v : a.k) + (size_t)row * a.ldkv + (size_t)head * D;
  float x[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) x[b] = src[32 * b + lane];
  if (a.cos_tab && !is_v) {
    if (pos < 0 || pos >= a.max_positions) return;  // never read outside the tables
    const float *ct = a.cos_tab + (size_t)pos * HALF, *st = a.sin_tab + (size_t)pos * HALF;
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) {
      const float c = ct[32 * b + lane], s = st[32 * b + lane];
      const float x0 = x[b], x1 = x[b + NB / 2];
      x[b] = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
      x[b + NB / 2] = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s));
    }
  }
  if (u < nq) {
    float *q = a.q_out + ((size_t)row * a.n_q_heads + u) * D;
#pragma unroll
    for (int b = 0; b < NB; ++b) q[32 * b + lane] = x[b];
    return;
  }
  int page = 0;
  uint8_t *g = kv4_group(a.kv, seq, pos, head, &page);
  if (!g || a.kv.refs[page] != 1) {
    if (lane == 0) raise_error(a.err, 1);
    return;
  }
  const int r16 = pos % kKv4Group;
  g += is_v ? kv4_group_bytes(D) / 2 : 0;
  kv4_store_row<D>(x, g + r16 * (D / 2),
                   reinterpret_cast<uint16_t *>(g + kKv4Group * (D / 2)) + r16 * NB, lane);
}

// Rows back to fp32, one warp per row: grid (tokens, ceil(2 Hkv / 8)).  A
// half-word's four values are one 16-byte store; the warp covers the row.  A
// position without a page reads as zeros and is recorded.
template <int D>
__global__ void __launch_bounds__(256) k_kv4_read(const __grid_constant__ Kv4ReadArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int NB = D / 32;
  const int lane = threadIdx.x & 31, Hkv = a.kv.n_kv_heads;
  const int u = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (u >= 2 * Hkv) return;
  const bool is_v = u >= Hkv;
  float *out = is_v ? a.v : a.k;
  if (!out) return;
  const int row = a.runs.row0[0] + blockIdx.x, head = u % Hkv;
  const int r = kv4_run_of(a.runs, row);
  const int pos = a.runs.pos[r] + row - a.runs.row0[r];
  const uint8_t *g = kv4_group(a.kv, a.runs.seq[r], pos, head, nullptr);
  if (!g && lane == 0) raise_error(a.err, 1);
  out += ((size_t)row * Hkv + head) * D;
  const int r16 = pos % kKv4Group;
  if (g) g += is_v ? kv4_group_bytes(D) / 2 : 0;
#pragma unroll
  for (int i = 0; i < D / 4; i += 32) {
    const int h = i + lane;
    if (h >= D / 4) break;  // D = 64: 16 half-words
    const int b = h % NB, gg = h / NB;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g) {
      const uint32_t w = reinterpret_cast<const uint16_t *>(g + r16 * (D / 2))[h];
      const float s = f16_to_f32(
          reinterpret_cast<const uint16_t *>(g + kKv4Group * (D / 2))[r16 * NB + b]);
      o = make_float4(s * (float)((int)(w & 15) - 8), s * (float)((int)((w >> 4) & 15) - 8),
                      s * (float)((int)((w >> 8) & 15) - 8), s * (float)((int)(w >> 12) - 8));
    }
    *reinterpret_cast<float4 *>(out + 32 * b + 4 * gg) = o;
  }
}

// Bookkeeping: entries and reference counts from kernel parameters (the host's
// tables may change again at once), and page copies in the same launch: the
// last CTA writes the entries, the others copy kCopyBytes each of a page.
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16 * 4;

template <int WORDS>
__global__ void __launch_bounds__(kCopyThreads)
    k_kv4_update(const __grid_constant__ Kv4Update<WORDS> u) {
  pdl_trigger();
  pdl_wait();
  const int pieces = (int)((u.page_bytes + kCopyBytes - 1) / kCopyBytes);
  if (blockIdx.x == gridDim.x - 1) {
    for (int j = threadIdx.x >> 5; j < u.n_spans; j += kCopyThreads / 32) {
      int *to = u.tables + u.word[3 * j];
      const int n = u.word[3 * j + 1], from = u.word[3 * j + 2];
      for (int i = threadIdx.x & 31; i < n; i += 32) to[i] = from < 0 ? -1 : u.tables[from + i];
    }
    const int *w = u.word + 3 * u.n_spans;
    for (int i = threadIdx.x; i < u.n_table; i += kCopyThreads) u.tables[w[2 * i]] = w[2 * i + 1];
    w += 2 * u.n_table;
    for (int i = threadIdx.x; i < u.n_refs; i += kCopyThreads) u.refs[w[2 * i]] = w[2 * i + 1];
    return;
  }
  const int *w = u.word + 3 * u.n_spans + 2 * (u.n_table + u.n_refs) +
                 2 * (blockIdx.x / pieces);
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
  const dim3 grid(a.T, (units + 7) / 8);
  return a.kv.head_dim == 128 ? launch_pdl(k_kv4_append<128>, grid, dim3(256), 0, s, a)
                              : launch_pdl(k_kv4_append<64>, grid, dim3(256), 0, s, a);
}

cudaError_t launch_kv4_read(const Kv4ReadArgs &a, cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  const dim3 grid(a.T, (2 * a.kv.n_kv_heads + 7) / 8);
  return a.kv.head_dim == 128 ? launch_pdl(k_kv4_read<128>, grid, dim3(256), 0, s, a)
                              : launch_pdl(k_kv4_read<64>, grid, dim3(256), 0, s, a);
}

template <int WORDS>
static cudaError_t update(const Kv4Update<WORDS> &u, cudaStream_t s) {
  const int pieces = (int)((u.page_bytes + kCopyBytes - 1) / kCopyBytes);
  return launch_pdl(k_kv4_update<WORDS>, dim3(u.n_copies * pieces + 1), dim3(kCopyThreads), 0, s,
                    u);
}
cudaError_t launch_kv4_update(const Kv4Update<kKv4SmallWords> &u, cudaStream_t s) {
  return update(u, s);
}
cudaError_t launch_kv4_update(const Kv4Update<kKv4LargeWords> &u, cudaStream_t s) {
  return update(u, s);
}

}  // namespace si
