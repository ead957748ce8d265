// Rotary positions and the append to the paged int8 cache: tables of cos and
// sin with scaled positions, rotation of row heads (with the head norm before
// and the int8 codes after it), and the same on the way of new K/V rows into
// their pages.  Tables and rows are bound by HBM when they are many, the append by its
// look-ups; few of any by launch and load latency.
#include <math.h>

#include "q3_paged.cuh"

namespace q3 {

static __device__ unsigned int g_rope_error = 0;

int rope_device_status_take() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_rope_error, sizeof v) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_rope_error, &zero, sizeof zero);
  return static_cast<int>(v);
}

namespace rope {

// ---------------------------------------------------------------------------
// tables: angle of position p and pair i in turns = p * turn[i], turn[i] a 64-bit
// binary fraction of one turn.  p * turn[i] modulo 2^64 is exact, so far
// positions lose nothing: the error is p times that of turn[i] (2^-64).  The
// nearest quarter turn is taken off the leading 32 bits, and sin and cos of the rest,
// at most 1/8 turn = pi/4, are their Taylor series (to x^9 and x^10: remainders below
// 2^-29); conversion, series and scaling stay within 2^-22.  131072 positions of 64 pairs are bound by
// their stores (67 MB in 13.2 us, 5.1 TB/s; with two CTAs an SM 15.7), 4096 by launch
// (2.4 us; 3.1 if not launched as a dependent).
// ---------------------------------------------------------------------------
constexpr int MAX_PAIRS = 128;
struct TableArgs {
  uint64_t turn[MAX_PAIRS];
  char *cos, *sin;
  long cos_rb, sin_rb;
  int rows, half;
  uint32_t pos0;
  float a;
};

// (2 pi 2^-32)^n / n!, exact in binary but for the rounding of the constant
__host__ __device__ constexpr double turn_power(int n) {
  double x = 1.0;
  for (int i = 1; i <= n; ++i) x = x * 6.283185307179586476925286766559 / 4294967296.0 / i;
  return x;
}

__global__ void k_rope_tables(const __grid_constant__ TableArgs p) {
  pdl_trigger();
  __shared__ uint64_t turn[MAX_PAIRS];
  for (int i = threadIdx.x; i < p.half; i += blockDim.x) turn[i] = p.turn[i];
  __syncthreads();
  const int per = blockDim.x / p.half;             // positions a block does at once
  const int i = threadIdx.x % p.half, r0 = threadIdx.x / p.half;
  if (r0 >= per) return;   // (others of the block wait below)
  const long step = static_cast<long>(gridDim.x) * per;
  long r = static_cast<long>(blockIdx.x) * per + r0;
  uint64_t t = turn[i] * (static_cast<uint64_t>(p.pos0) + static_cast<uint64_t>(r));
  const uint64_t dt = turn[i] * static_cast<uint64_t>(step);
  char *cp = p.cos + r * p.cos_rb + i * 4, *sp = p.sin + r * p.sin_rb + i * 4;
  pdl_wait();
#pragma unroll 4
  for (; r < p.rows; r += step) {
    const uint32_t hi = static_cast<uint32_t>(t >> 32);
    const uint32_t q = (hi + 0x20000000u) >> 30;   // nearest quarter turn
    const float x = __int2float_rn(static_cast<int>(hi - (q << 30)));   // 2^-32 turns
    // in units of u = (x 2^-29)^2 <= 1 the coefficients stay in float32's range
    const float y = __fmul_rn(x, 1.862645149230957e-09f), u = __fmul_rn(y, y);
    constexpr double k = 536870912.0, k2 = k * k;  // 2^29
    constexpr float s1 = static_cast<float>(turn_power(1) * k),
                    s3 = static_cast<float>(-turn_power(3) * k * k2),
                    s5 = static_cast<float>(turn_power(5) * k * k2 * k2),
                    s7 = static_cast<float>(-turn_power(7) * k * k2 * k2 * k2),
                    s9 = static_cast<float>(turn_power(9) * k * k2 * k2 * k2 * k2),
                    c2 = static_cast<float>(-turn_power(2) * k2),
                    c4 = static_cast<float>(turn_power(4) * k2 * k2),
                    c6 = static_cast<float>(-turn_power(6) * k2 * k2 * k2),
                    c8 = static_cast<float>(turn_power(8) * k2 * k2 * k2 * k2),
                    c10 = static_cast<float>(-turn_power(10) * k2 * k2 * k2 * k2 * k2);
    float s = __fmaf_rn(u, s9, s7), c = __fmaf_rn(u, c10, c8);
    s = __fmaf_rn(u, s, s5);
    c = __fmaf_rn(u, c, c6);
    s = __fmaf_rn(u, s, s3);
    c = __fmaf_rn(u, c, c4);
    s = __fmul_rn(__fmul_rn(u, s), y);
    c = __fmaf_rn(u, c, c2);
    s = __fmaf_rn(y, s1, s);
    c = __fmaf_rn(u, c, 1.0f);
    // quarter q: (c, s), (-s, c), (-c, -s), (s, -c)
    const float cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;
    const float ca = __uint_as_float(__float_as_uint(p.a) ^ (((q + 1) & 2) << 30));
    const float sa = __uint_as_float(__float_as_uint(p.a) ^ ((q & 2) << 30));
    *reinterpret_cast<float *>(cp) = __fmul_rn(cc, ca);
    *reinterpret_cast<float *>(sp) = __fmul_rn(ss, sa);
    t += dt;
    cp += step * p.cos_rb;
    sp += step * p.sin_rb;
  }
}

// ---------------------------------------------------------------------------
// One head in GL lanes: lane g of them holds columns g*N .. g*N+N-1 (head_dim =
// GL N), a warp 32 / GL heads; N is what 16 bytes hold, or 8.  The float32 steps and
// their order are those of the norm-rope-quant epilogue
// (tools/ref_qwen3.py:161-191), so the codes are the same bits.
// ---------------------------------------------------------------------------
constexpr int U = 4;                               // heads a lane holds at once
template <int N, int GL>
__device__ __forceinline__ float head_mean(const float (&x)[N], float inv_hd) {
  // squares by adjacent pairs within 32-column blocks of 32/N lanes ...
  float s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = __fmul_rn(x[i], x[i]);
#pragma unroll
  for (int k = 1; k < N; k <<= 1)
#pragma unroll
    for (int i = 0; i < N; i += 2 * k) s[i] = __fadd_rn(s[i], s[i + k]);
#pragma unroll
  for (int o = 1; o < 32 / N; o <<= 1) s[0] = __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], o));
  // ... and the blocks in order
  float ss = 0.0f;
#pragma unroll
  for (int b = 0; b < GL * N / 32; ++b)
    ss = __fadd_rn(ss, __shfl_sync(0xffffffffu, s[0], b * (32 / N), GL));
  return __fadd_rn(__fmul_rn(ss, inv_hd), kEps);
}

template <int N, int GL>
__device__ __forceinline__ void head_scale(float (&x)[N], const float (&w)[N], float r) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
}
// the roots of U heads at once: that of head u in the lanes with g % U == u
template <typename T, int N, int GL>
__device__ __forceinline__ float head_rsqrt(const Elems<T, N> (&e)[U], float inv_hd, int g) {
  float m = 1.0f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float x[N];
    to_f32(e[u], x);
    const float y = head_mean<N, GL>(x, inv_hd);
    m = (g % U) == u ? y : m;
  }
  return rsqrt_ref(m);
}

// c, s: cos and sin of this lane's columns (half layout: of column mod half, s negated in the lower
// half, so that x c + y s is both x c - y s and y s + x c, with the same rounding; interleaved: c[i],
// s[i] for pair i of the lane in i < N/2)
template <int N, int GL>
__device__ __forceinline__ void head_rotate(float (&x)[N], const float (&c)[N], const float (&s)[N],
                                            int half, bool inter, int g) {
  if (inter) {
    if (g * N < 2 * half) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float a = x[i], b = x[i + 1];
        x[i] = __fsub_rn(__fmul_rn(a, c[i / 2]), __fmul_rn(b, s[i / 2]));
        x[i + 1] = __fadd_rn(__fmul_rn(a, s[i / 2]), __fmul_rn(b, c[i / 2]));
      }
    }
    return;
  }
  const int hl = half / N;                        // lanes of half a rotation
  const bool in = half * 2 == GL * N || g < 2 * hl;   // (the first for the compiler: often all columns)
  const int other = in ? (g < hl ? g + hl : g - hl) : g;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = __shfl_sync(0xffffffffu, x[i], other, GL);
    const float z = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y, s[i]));
    x[i] = in ? z : x[i];
  }
}

struct Turn {   // one view of the tables
  const char *cos, *sin;
  long cos_rb, sin_rb;
  int rows, half;
  int inter;
};

// this lane's cos and sin at row `pos` (columns beyond the rotated part: unused)
template <int N>
__device__ __forceinline__ void load_turn(const Turn &t, long pos, int g, float (&c)[N],
                                          float (&s)[N]) {
  const float *cp = reinterpret_cast<const float *>(t.cos + pos * t.cos_rb);
  const float *sp = reinterpret_cast<const float *>(t.sin + pos * t.sin_rb);
  if (g * N >= 2 * t.half) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = s[i] = 0.0f;
    return;
  }
  if (t.inter) {
    Elems<float, N / 2> a, b;
    a.load(cp + g * (N / 2));
    b.load(sp + g * (N / 2));
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = a.e[i % (N / 2)], s[i] = b.e[i % (N / 2)];
  } else {
    const int at = g * N < t.half ? g * N : g * N - t.half;
    Elems<float, N> a, b;
    a.load(cp + at);
    b.load(sp + at);
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = a.e[i], s[i] = g * N < t.half ? -b.e[i] : b.e[i];
  }
}

// codes of one head's columns (stored where ok) and its scale = RN(absmax * RN(1/127))
template <int N, int GL>
__device__ __forceinline__ float head_int8(const float (&x)[N], void *codes, bool ok) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
  if constexpr (GL == 32) {
    m = warp_tree_max(m);
  } else {
#pragma unroll
    for (int o = 1; o < GL; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  const float scale = __fmul_rn(m, kInv127);
  uint32_t w[N / 4];
  quant_pack_absmax<N>(x, scale, w);
  Elems<int8_t, N> e;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint32_t *>(e.e)[i] = w[i];
  if (ok) e.store(codes);
  return scale;
}

// ---------------------------------------------------------------------------
// rotation of rows.  A warp takes U times its 32 / GL heads of a row: U 16-byte loads a
// lane in flight, one read of the row's cos and sin for them.  Loads and stores
// stream past the caches (8192 rows of 16 heads: 28.2 us against 29.0; 5003
// bf16 rows of 40 heads 25.8 against 28.5).  Bound by HBM and, with the norm, nearly by issue
// slots: pairs of 16-bit elements converted at once, one multiply-add form for both halves
// and one root for U heads brought 24.3 and 20.7 us (5.7 and 5.0 TB/s), 8192 bf16 rows of 32 heads
// with norm 42.7 -> 33.3.  Registers are held to what 8 CTAs an SM leave (9 for f32; 7 and 5 for
// heads in a whole warp): without the limit 23 us, at 10 CTAs 39 for the bf16 rows with norm.
// (The limit spills in the 16-bit forms, 12 to 24 bytes a thread.)  int8 codes out take 27.3 us for the
// 8192 rows and 27.2 for the 5003, bound by the instructions of the codes; a decode batch 2.8, floats 2.4.
// ---------------------------------------------------------------------------
struct RowArgs {
  const char *x;
  char *out, *scale;
  long x_rb, out_rb, scale_rb;
  const float *nw;
  const int32_t *pos;
  Turn t;
  int rows, heads, out_dt;
  float inv_hd;
};

template <typename T, int N, int GL>
__global__ void __launch_bounds__(128, sizeof(T) == 2 ? (GL == 32 ? 7 : 8) : N == 8 ? 5 : 9)
    k_rope_rows(RowArgs p) {
  constexpr int HD = GL * N, HW = 32 / GL;         // heads a warp holds at once
  pdl_trigger();
  const int lane = threadIdx.x & 31, g = lane % GL, hl = lane / GL;
  const int chunks = (p.heads + U * HW - 1) / (U * HW);
  const long unit = static_cast<long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long r = unit / chunks;
  if (r >= p.rows) return;
  const int h0 = static_cast<int>(unit - r * chunks) * (U * HW);
  pdl_wait();
  Elems<T, N> e[U];
  const char *xp = p.x + r * p.x_rb + (static_cast<long>(h0 + hl) * HD + g * N) * sizeof(T);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + u * HW + hl < p.heads) e[u].load_stream(xp + static_cast<long>(u) * HW * HD * sizeof(T));
    else e[u].zero();
  float w[N], c[N], s[N];
  if (p.nw) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p.nw[g * N + i];
  }
  const int pos = p.pos[r];
  if (pos < 0 || pos >= p.t.rows) {
    if (lane == 0) atomicOr(&g_rope_error, kBadPosition);
    return;
  }
  load_turn<N>(p.t, pos, g, c, s);
  float rs = 0.0f;
  if (p.nw) rs = head_rsqrt<T, N, GL>(e, p.inv_hd, g);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (h0 + u * HW >= p.heads) break;
    const int h = h0 + u * HW + hl;
    const bool ok = h < p.heads;
    float x[N];
    to_f32(e[u], x);
    if (p.nw) head_scale<N, GL>(x, w, __shfl_sync(0xffffffffu, rs, u, GL));
    head_rotate<N, GL>(x, c, s, p.t.half, p.t.inter, g);
    const long col = static_cast<long>(h) * HD + g * N;
    char *o = p.out + r * p.out_rb;
    if (p.out_dt == Q3_DT_I8) {
      const float sc = head_int8<N, GL>(x, o + col, ok);
      if (g == 0 && ok) reinterpret_cast<float *>(p.scale + r * p.scale_rb)[h] = sc;
    } else if (ok) {
      if (p.out_dt == Q3_DT_F32) store_row_stream<float, N>(x, o + col * 4);
      else if (p.out_dt == Q3_DT_F16) store_row_stream<__half, N>(x, o + col * 2);
      else store_row_stream<__nv_bfloat16, N>(x, o + col * 2);
    }
  }
}

// ---------------------------------------------------------------------------
// append.  A warp takes U KV heads of K or of V of one row; the row's data is
// requested before the dependent lookups (row -> sequence -> position -> page -> table row), which are the
// bound: 64 rows of 8 KV heads 3.5 us, 3472 of them, 21.5 MB, 9.8 us at 2.2 TB/s.
// ---------------------------------------------------------------------------
struct AppendArgs {
  const char *k, *v;
  long k_rb, v_rb;
  const float *nw;
  Turn t;                       // t.half == 0: no rotation
  float inv_hd;
  char *pk, *pv, *pks, *pvs;
  uint32_t page_tokens, page_bytes, row_bytes, scale_page_bytes, scale_row_bytes;
  uint32_t num_pages, max_pages;
  const uint16_t *tables;
  const int32_t *row0, *kv_len;
  int n_seqs, rows, kv_heads;
};

template <typename T, int N, int GL>
__global__ void k_kv_append(AppendArgs p) {
  constexpr int HD = GL * N, HW = 32 / GL;
  pdl_trigger();
  const int lane = threadIdx.x & 31, g = lane % GL, hl = lane / GL;
  const int chunks = (p.kv_heads + U * HW - 1) / (U * HW);
  long unit = static_cast<long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long r = unit / (2 * chunks);
  if (r >= p.rows) {
    // one warp more than the rows need: do the sequences' rows exist?
    if (unit != static_cast<long>(p.rows) * (2 * chunks)) return;
    pdl_wait();
    bool bad = false;
    for (int s = lane; s < p.n_seqs; s += 32)
      bad = bad || rows_missing(p.row0[s], p.row0[s + 1], p.rows);
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(&g_rope_error, kBadRagged);
    return;
  }
  unit -= r * (2 * chunks);
  const bool is_v = unit >= chunks;
  const int h0 = static_cast<int>(is_v ? unit - chunks : unit) * (U * HW);
  pdl_wait();
  Elems<T, N> e[U];
  const char *xp = (is_v ? p.v + r * p.v_rb : p.k + r * p.k_rb) +
                   (static_cast<long>(h0 + hl) * HD + g * N) * sizeof(T);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + u * HW + hl < p.kv_heads) e[u].load_stream(xp + static_cast<long>(u) * HW * HD * sizeof(T));
    else e[u].zero();
  const bool norm = !is_v && p.nw, turn = !is_v && p.t.half;
  float w[N], c[N], s[N];
  if (norm) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p.nw[g * N + i];
  }
  int first, count;
  const int q = find_seq(p.row0, p.n_seqs, static_cast<int>(r), lane, first, count);
  // a row that belongs to nobody, or to a sequence that the extra warp reports
  if (q < 0 || rows_missing(first, first + count, p.rows)) return;
  const long pos = static_cast<long>(p.kv_len[q]) - count + (r - first);
  const long lp = pos < 0 ? 0 : static_cast<long>(static_cast<uint64_t>(pos) / p.page_tokens);
  unsigned bad = 0;
  uint32_t page = 0;
  if (pos < 0) bad = kBadRagged;
  else if (lp >= p.max_pages) bad = kBadTable;
  else if (p.t.half && pos >= p.t.rows) bad = kBadPosition;   // (V is not rotated, but goes with its K)
  else {
    page = p.tables[static_cast<long>(q) * p.max_pages + lp];
    if (page >= p.num_pages) bad = kBadPage;
  }
  if (bad) {
    if (lane == 0) atomicOr(&g_rope_error, bad);
    return;
  }
  if (turn) load_turn<N>(p.t, pos, g, c, s);
  float rs = 0.0f;
  if (norm) rs = head_rsqrt<T, N, GL>(e, p.inv_hd, g);
  const uint32_t slot = static_cast<uint32_t>(pos - lp * p.page_tokens);
  char *codes = (is_v ? p.pv : p.pk) + static_cast<size_t>(page) * p.page_bytes +
                static_cast<size_t>(slot) * p.row_bytes;
  float *scale = reinterpret_cast<float *>((is_v ? p.pvs : p.pks) +
                                           static_cast<size_t>(page) * p.scale_page_bytes +
                                           static_cast<size_t>(slot) * p.scale_row_bytes);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (h0 + u * HW >= p.kv_heads) break;
    const int h = h0 + u * HW + hl;
    const bool ok = h < p.kv_heads;
    float x[N];
    to_f32(e[u], x);
    if (norm) head_scale<N, GL>(x, w, __shfl_sync(0xffffffffu, rs, u, GL));
    if (turn) head_rotate<N, GL>(x, c, s, p.t.half, p.t.inter, g);
    const float sc = head_int8<N, GL>(x, codes + static_cast<long>(h) * HD + g * N, ok);
    if (g == 0 && ok) scale[h] = sc;
  }
}

}  // namespace rope
}  // namespace q3

// ===========================================================================
// C ABI
// ===========================================================================
using namespace q3;
using namespace q3h;
using namespace q3::rope;

// a strided row view of one of the float types, vector accesses allowed
static int check_rows(const q3_view *v, uint32_t cols) {
  if (!v || !v->data) return Q3_ERR_NULL;
  if (v->dtype != Q3_DT_F32 && v->dtype != Q3_DT_F16 && v->dtype != Q3_DT_BF16) return Q3_ERR_DTYPE;
  Q3_TRY(check_view(v, v->dtype, 16));
  return v->cols < cols ? Q3_ERR_SHAPE : Q3_OK;
}

// head_dim, norm weights and tables; *t describes the tables
static int check_head(const q3_view *nw, const q3_view *cos, const q3_view *sin, uint32_t head_dim,
                      int interleaved, Turn *t) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return Q3_ERR_SHAPE;
  if (nw) {
    Q3_TRY(check_view(nw, Q3_DT_F32));
    if (nw->rows != 1 && nw->cols != 1) return Q3_ERR_SHAPE;
    if (nw->rows * nw->cols < head_dim) return Q3_ERR_SHAPE;
    if (nw->rows > 1 && nw->row_bytes != 4) return Q3_ERR_SHAPE;
  }
  *t = Turn{};
  if (!cos && !sin) return Q3_OK;
  if (!cos || !sin) return Q3_ERR_NULL;
  Q3_TRY(check_view(cos, Q3_DT_F32, 16));
  Q3_TRY(check_view(sin, Q3_DT_F32, 16));
  if (cos->cols != sin->cols || cos->rows != sin->rows || cos->rows > 0x7fffffffu)
    return Q3_ERR_SHAPE;
  if (cos->cols == 0 || cos->cols % 8 || 2 * cos->cols > head_dim) return Q3_ERR_SHAPE;
  *t = Turn{(const char *)cos->data, (const char *)sin->data, cos->row_bytes, sin->row_bytes,
            (int)cos->rows, (int)cos->cols, interleaved ? 1 : 0};
  return Q3_OK;
}

extern "C" int q3_rope_tables(const q3_rope_spec *spec, uint32_t pos0, const q3_view *cos,
                              const q3_view *sin, void *stream) {
  if (!spec) return Q3_ERR_NULL;
  Q3_TRY(check_view(cos, Q3_DT_F32));
  Q3_TRY(check_view(sin, Q3_DT_F32));
  if (spec->scaling < Q3_ROPE_NONE || spec->scaling > Q3_ROPE_YARN) return Q3_ERR_MODE;
  const uint32_t half = cos->cols;
  if (half == 0 || half > MAX_PAIRS || sin->cols != half || sin->rows != cos->rows ||
      cos->rows > 0x7fffffffu)
    return Q3_ERR_SHAPE;
  const bool scaled = spec->scaling != Q3_ROPE_NONE, yarn = spec->scaling == Q3_ROPE_YARN;
  if (!(spec->theta > 1.0 && spec->theta < INFINITY)) return Q3_ERR_SHAPE;
  if (scaled && !(spec->factor >= 1.0 && spec->factor < INFINITY)) return Q3_ERR_SHAPE;
  if (yarn && !(spec->original_max >= 1.0 && spec->original_max < INFINITY &&
                spec->beta_slow > 0.0 && spec->beta_fast >= spec->beta_slow &&
                spec->beta_fast < INFINITY))
    return Q3_ERR_SHAPE;
  if (!((float)spec->attn_factor < INFINITY)) return Q3_ERR_SHAPE;
  if (cos->rows == 0) return Q3_OK;

  TableArgs p;
  // Pair i turns theta^(-2i/rot) / (2 pi) of a turn a position.  YaRN (the
  // published method): pairs that turn more than beta_fast times within
  // original_max keep their frequency, those below beta_slow turns have it
  // divided by factor, a linear ramp over the pair index between them.
  const long double pi = 3.14159265358979323846264338327950288L;
  const double rot = 2.0 * half;
  double low = 0.0, high = 0.0;
  if (yarn) {
    const double per = rot / (2.0 * log(spec->theta));
    low = floor(per * log(spec->original_max / (spec->beta_fast * 2.0 * (double)pi)));
    high = ceil(per * log(spec->original_max / (spec->beta_slow * 2.0 * (double)pi)));
    low = low < 0.0 ? 0.0 : low;
    high = high > rot - 1.0 ? rot - 1.0 : high;
  }
  const double span = high - low > 1e-3 ? high - low : 1e-3;
  // powers by products: 128 roundings of 2^-64 stay below 2^-56
  const long double ratio = expl(-2.0L / rot * logl((long double)spec->theta));
  long double power = 1.0L;
  for (uint32_t i = 0; i < half; ++i, power *= ratio) {
    long double f = power;
    if (spec->scaling == Q3_ROPE_LINEAR) f /= spec->factor;
    if (yarn) {
      double ramp = (i - low) / span;
      ramp = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
      f = f * (1.0L - ramp) + f / spec->factor * ramp;
    }
    const long double turn = f / (2.0L * pi);      // < 1/6
    p.turn[i] = (uint64_t)(turn * 18446744073709551616.0L);
  }
  p.a = spec->attn_factor > 0.0 ? (float)spec->attn_factor
        : yarn                  ? (float)(0.1 * log(spec->factor) + 1.0)
                                : 1.0f;
  p.cos = (char *)cos->data;
  p.sin = (char *)sin->data;
  p.cos_rb = cos->row_bytes;
  p.sin_rb = sin->row_bytes;
  p.rows = (int)cos->rows;
  p.half = (int)half;
  p.pos0 = pos0;
  const int threads = 256, per = threads / (int)half;
  const long blocks = ((long)p.rows + per - 1) / per, most = 4L * sm_count();
  return launch_ex(true, k_rope_tables, dim3((unsigned)(blocks < most ? blocks : most)), dim3(threads), 0,
                   (cudaStream_t)stream, p);
}

template <typename T>
static int launch_rows(const RowArgs &p, uint32_t hd, cudaStream_t s) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));   // head_dim 256: 8 columns a lane
  const int per = U * (hd >= 32 * N ? 1 : 32 * N / static_cast<int>(hd));   // heads of a warp
  const long warps = static_cast<long>(p.rows) * ((p.heads + per - 1) / per);
  const unsigned blocks = (unsigned)((warps + 3) / 4);
  const dim3 grid(blocks), block(128);
  return hd == 64    ? launch_ex(true, k_rope_rows<T, N, 64 / N>, grid, block, 0, s, p)
         : hd == 128 ? launch_ex(true, k_rope_rows<T, N, 128 / N>, grid, block, 0, s, p)
                     : launch_ex(true, k_rope_rows<T, 8, 32>, grid, block, 0, s, p);
}

extern "C" int q3_rope_rows(const q3_view *x, const q3_view *nw, const int32_t *pos,
                            const q3_view *cos, const q3_view *sin, const q3_view *out,
                            const q3_view *scale, uint32_t heads, uint32_t head_dim,
                            int interleaved, float inv_hd, void *stream) {
  if (!pos || !cos || !sin) return Q3_ERR_NULL;
  RowArgs p{};
  if (heads == 0 || heads > 65535) return Q3_ERR_SHAPE;
  Q3_TRY(check_head(nw, cos, sin, head_dim, interleaved, &p.t));
  Q3_TRY(check_rows(x, heads * head_dim));
  if (!out || !out->data) return Q3_ERR_NULL;
  if (out->dtype == Q3_DT_I8) {
    Q3_TRY(check_view(out, Q3_DT_I8, 16));
    Q3_TRY(check_view(scale, Q3_DT_F32));
    if (scale->cols < heads || scale->rows < x->rows) return Q3_ERR_SHAPE;
    p.scale = (char *)scale->data;
    p.scale_rb = scale->row_bytes;
  } else {
    Q3_TRY(check_rows(out, 0));
  }
  if (out->rows < x->rows || out->cols < heads * head_dim || x->rows > 0x7fffffffu)
    return Q3_ERR_SHAPE;
  // in place: the same elements, of the same size (a warp reads its heads before it writes them)
  if (out->data == x->data && (out->dtype != x->dtype || out->row_bytes != x->row_bytes))
    return Q3_ERR_SHAPE;
  if (x->rows == 0) return Q3_OK;
  p.x = (const char *)x->data;
  p.x_rb = x->row_bytes;
  p.out = (char *)out->data;
  p.out_rb = out->row_bytes;
  p.out_dt = out->dtype;
  p.nw = nw ? (const float *)nw->data : nullptr;
  p.pos = pos;
  p.rows = (int)x->rows;
  p.heads = (int)heads;
  p.inv_hd = inv_hd;
  cudaStream_t s = (cudaStream_t)stream;
  return x->dtype == Q3_DT_F32   ? launch_rows<float>(p, head_dim, s)
         : x->dtype == Q3_DT_F16 ? launch_rows<__half>(p, head_dim, s)
                                 : launch_rows<__nv_bfloat16>(p, head_dim, s);
}

template <typename T>
static int launch_append(const AppendArgs &p, uint32_t hd, cudaStream_t s) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));   // head_dim 256: 8 columns a lane
  const int per = U * (hd >= 32 * N ? 1 : 32 * N / static_cast<int>(hd));   // heads of a warp
  const long warps = static_cast<long>(p.rows) * 2 * ((p.kv_heads + per - 1) / per) + 1;
  const unsigned blocks = (unsigned)((warps + 3) / 4);
  const dim3 grid(blocks), block(128);
  return hd == 64    ? launch_ex(true, k_kv_append<T, N, 64 / N>, grid, block, 0, s, p)
         : hd == 128 ? launch_ex(true, k_kv_append<T, N, 128 / N>, grid, block, 0, s, p)
                     : launch_ex(true, k_kv_append<T, 8, 32>, grid, block, 0, s, p);
}

namespace q3 {
// the pool of a ragged operator: `align` bytes for the code rows
int check_pool(const q3_paged_kv *kv, uint32_t kv_heads, uint32_t head_dim, uint32_t num_pages,
               uint32_t max_pages, uint32_t align) {
  if (!kv || !kv->k || !kv->v || !kv->ks || !kv->vs) return Q3_ERR_NULL;
  if (kv_heads == 0 || kv_heads > 4096 || num_pages == 0 || num_pages > 65536 || max_pages == 0)
    return Q3_ERR_SHAPE;
  // (positions rounded up to a tile of keys stay below 2^31)
  if (kv->page_tokens == 0 || kv->page_tokens > 32768 ||
      (uint64_t)max_pages * kv->page_tokens > 0x7fffff00u)
    return Q3_ERR_SHAPE;
  if (kv->row_bytes < kv_heads * head_dim || kv->scale_row_bytes < kv_heads * 4 ||
      (uint64_t)kv->page_tokens * kv->row_bytes > kv->page_bytes ||
      (uint64_t)kv->page_tokens * kv->scale_row_bytes > kv->scale_page_bytes)
    return Q3_ERR_SHAPE;
  if ((uintptr_t)kv->k % align || (uintptr_t)kv->v % align || kv->row_bytes % align ||
      kv->page_bytes % align)
    return Q3_ERR_ALIGN;
  if ((uintptr_t)kv->ks % 4 || (uintptr_t)kv->vs % 4 || kv->scale_row_bytes % 4 ||
      kv->scale_page_bytes % 4)
    return Q3_ERR_ALIGN;
  return Q3_OK;
}
}  // namespace q3

extern "C" int q3_paged_kv_append_batch(const q3_view *k, const q3_view *v, const q3_view *nw,
                                        float inv_hd, const q3_view *cos, const q3_view *sin,
                                        int interleaved, const q3_paged_kv *kv, uint32_t num_pages,
                                        const uint16_t *tables, uint32_t max_pages,
                                        const int32_t *row0, const int32_t *kv_len,
                                        uint32_t n_seqs, uint32_t kv_heads, uint32_t head_dim,
                                        void *stream) {
  if (!tables || !row0 || !kv_len) return Q3_ERR_NULL;
  AppendArgs p{};
  Q3_TRY(check_head(nw, cos, sin, head_dim, interleaved, &p.t));
  Q3_TRY(check_pool(kv, kv_heads, head_dim, num_pages, max_pages, 16));
  Q3_TRY(check_rows(k, kv_heads * head_dim));
  Q3_TRY(check_rows(v, kv_heads * head_dim));
  if (k->dtype != v->dtype) return Q3_ERR_DTYPE;
  if (k->rows != v->rows || k->rows > 0x7fffffffu || n_seqs > 0x7ffffffeu) return Q3_ERR_SHAPE;
  if (k->rows == 0 || n_seqs == 0) return Q3_OK;
  p.k = (const char *)k->data;
  p.v = (const char *)v->data;
  p.k_rb = k->row_bytes;
  p.v_rb = v->row_bytes;
  p.nw = nw ? (const float *)nw->data : nullptr;
  p.inv_hd = inv_hd;
  p.pk = (char *)kv->k;
  p.pv = (char *)kv->v;
  p.pks = (char *)kv->ks;
  p.pvs = (char *)kv->vs;
  p.page_tokens = kv->page_tokens;
  p.page_bytes = kv->page_bytes;
  p.row_bytes = kv->row_bytes;
  p.scale_page_bytes = kv->scale_page_bytes;
  p.scale_row_bytes = kv->scale_row_bytes;
  p.num_pages = num_pages;
  p.max_pages = max_pages;
  p.tables = tables;
  p.row0 = row0;
  p.kv_len = kv_len;
  p.n_seqs = (int)n_seqs;
  p.rows = (int)k->rows;
  p.kv_heads = (int)kv_heads;
  cudaStream_t s = (cudaStream_t)stream;
  return k->dtype == Q3_DT_F32   ? launch_append<float>(p, head_dim, s)
         : k->dtype == Q3_DT_F16 ? launch_append<__half>(p, head_dim, s)
                                 : launch_append<__nv_bfloat16>(p, head_dim, s);
}
