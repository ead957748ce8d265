// Attention of a ragged batch of new rows over the paged int8 cache: what its
// kernels share (q3_attention_chunk.cu).
#pragma once

#include "q3_paged.cuh"

namespace q3 {
namespace chunk {

struct Args {
  const char *q, *qs;
  char *o, *os;
  long q_rb, qs_rb, o_rb, os_rb;
  int q_dt, o_dt;
  const char *k, *v, *ks, *vs;
  uint32_t page_tokens, page_bytes, row_bytes, scale_page_bytes, scale_row_bytes;
  uint32_t num_pages, max_pages;
  const uint16_t *tables;
  const int32_t *row0, *kv_len;
  int n_seqs, rows, max_rows, heads, kv_heads, group;
  int causal, window;
  float scale_log2;              // qk_scale * log2(e)
  int splits;                    // parts of the key range (1: results go to o)
  int tiles;                     // many rows: tiles of the batch; few rows, whole: tiles of a sequence
  int few_rows;                  // packed rows of a sequence that k_attn_few takes
  int min_units;                 // least units of a slice
  int row_shift;                 // log2 of the packed rows of its row tiles, and of a part
  int whole;                     // it takes a sequence's keys as a whole
  int page_shift;                // log2 of page_tokens, or -1
  int whole_blocks;              // a 32-key block lies in one page
  float *part_o, *part_ml;       // parts: sums [..][hd], and their (maximum, sum of weights); of one part: the
                                 // sums of row r and head h at (r heads + h) hd
};

// Rows of sequence s as the device sees them; ok = false: nothing to do
// (no rows), or arrays that do not fit (err set).
struct Seq {
  int first, n, kv, pos0;        // rows first .. first+n-1 at positions pos0 ..
  bool ok;
};
__device__ __forceinline__ Seq load_seq(const Args &p, int s, unsigned *err) {
  Seq q;
  q.first = p.row0[s];
  const int end = p.row0[s + 1];
  q.n = end - q.first;
  q.kv = p.kv_len[s];
  q.pos0 = q.kv - q.n;
  q.ok = q.n > 0;
  if (q.n == 0) return q;
  if (rows_missing(q.first, end, p.rows) || q.n > p.max_rows || q.kv < q.n) {
    *err |= kBadRagged;
    q.ok = false;
  } else if (static_cast<uint32_t>(q.kv) > p.max_pages * p.page_tokens) {
    *err |= kBadTable;
    q.ok = false;
  }
  return q;
}

// Keys [lo, hi) that some row at positions p0..p1 sees
__device__ __forceinline__ void key_range(const Args &p, const Seq &s, int p0, int p1, int &lo,
                                          int &hi) {
  hi = p.causal ? p1 + 1 : s.kv;
  lo = p.window > 0 && p0 >= p.window ? p0 - p.window + 1 : 0;
}
__device__ __forceinline__ uint32_t page_index(const Args &p, uint32_t j) {
  return p.page_shift >= 0 ? j >> p.page_shift : j / p.page_tokens;
}
__device__ __forceinline__ uint32_t page_slot(const Args &p, uint32_t j) {
  return p.page_shift >= 0 ? j & (p.page_tokens - 1) : j % p.page_tokens;
}
// Part z of `splits` of key blocks [b0, b1): equal runs, the first ones longer
__device__ __forceinline__ void split_range(int b0, int b1, int splits, int z, int &z0, int &z1) {
  const int n = b1 - b0, each = n / splits, more = n % splits;
  z0 = b0 + z * each + min(z, more);
  z1 = z0 + each + (z < more ? 1 : 0);
}

constexpr float kVsMin = 7.888609052210118e-31f;   // 2^-100
// Weights are formed relative to a reference kRefBelow under the maximum so far (in powers of two) and
// it moves when one outgrows it by 2^kRefMove: they stay within f16's range, and those down to
// 2^-32 of the largest are not lost in the sums over the fraction while those under it, in
// float32, have them.  The sums of p / vs carry 2^-kRefBelow (in rv): no term passes 2^108.
constexpr float kRefBelow = 7.0f, kRefMove = 15.0f, kSumScale = 0.0078125f;
// the sums over the fraction by those under it (no key seen: zeros)
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : __fdiv_rn(kSumScale, l); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four int8 codes, bytes xor 0x80 (u = code + 128): f16 0x6400 + u is 1024 + u
__device__ __forceinline__ uint32_t f16_pair(uint32_t u, uint32_t sel) {
  const uint32_t m = __byte_perm(u, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&m), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// bf16 rows: 2^up brings the row's maximum m to [2^10, 2^11) (zero, subnormal or infinite m: the
// nearest exponent in range); `down` is its inverse.
__device__ __forceinline__ void bf16_scale(float m, float &up, float &down) {
  const int ex = static_cast<int>(__float_as_uint(m) >> 23);
  const int e = min(max(137 - ex, -120), 110);
  up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
  down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
}

// One head of a result row (whole warp, lane: columns lane*N ..) to o / os.
template <int N>
__device__ __forceinline__ void store_out(const Args &p, long r, int h, int lane, float (&x)[N]) {
  constexpr int HD = 32 * N;
  char *o = p.o + r * p.o_rb;
  const long col = static_cast<long>(h) * HD + lane * N;
  if (p.o_dt == Q3_DT_F16) store_row<__half, N>(x, o + col * 2);
  else if (p.o_dt == Q3_DT_BF16) store_row<__nv_bfloat16, N>(x, o + col * 2);
  else {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
    const float scale = __fmul_rn(warp_tree_max(m), kInv127);
    int c[N];
    quant_n_absmax<N>(x, scale, c);
    Elems<int8_t, N> e;
#pragma unroll
    for (int i = 0; i < N; ++i) e.e[i] = static_cast<int8_t>(c[i]);
    e.store(o + col);
    if (lane == 0) reinterpret_cast<float *>(p.os + r * p.os_rb)[h] = scale;
  }
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
// Sequence of unit `unit` when sequence s has units(s) of them (whole warp); before: those of the
// sequences before it.  -1: there is no such unit.
template <typename F>
__device__ __forceinline__ int find_unit(int n_seqs, long unit, int lane, long &before, F units) {
  before = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    const long mine = s0 + lane < n_seqs ? units(s0 + lane) : 0;
    long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned m = __ballot_sync(0xffffffffu, before + upto > unit);
    if (m) {
      const int l = __ffs(m) - 1;
      before += __shfl_sync(0xffffffffu, upto - mine, l);
      return s0 + l;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return -1;
}

// Many rows (q3_attention_chunk_tc.cu): sequences with more than few_rows packed rows.  `tiles` is the
// number of 256-row tiles that the batch can have.
constexpr int TC_ROWS = 256, TC_KEYS = 128;
// Its sums of values run over at most FOLD_TILES key tiles in the tensor cores, which cut the bits that a
// running sum cannot hold, always towards zero (3.3e-3 of it over 500000 keys); then they are added to
// float32 sums in the workspace.
constexpr int FOLD_TILES = 64, FOLD_KEYS = FOLD_TILES * TC_KEYS;
__device__ __forceinline__ long tiles_of(const Args &p, int s, unsigned *err) {
  const Seq q = load_seq(p, s, err);
  const int packed = q.n * p.group;
  return q.ok && packed > p.few_rows ? (packed + TC_ROWS - 1) / TC_ROWS : 0;
}
// Sequence of tile `id` of the batch, -1: there is no such tile, and its place in the sequence: the last
// one, which has most keys, first (whole warp)
__device__ __forceinline__ int find_tile(const Args &p, int id, int lane, unsigned *err, int &tile) {
  long before;
  const int s = find_unit(p.n_seqs, id, lane, before, [&](int x) { return tiles_of(p, x, err); });
  tile = s < 0 ? 0 : static_cast<int>(tiles_of(p, s, err) - 1 - (id - before));
  return s;
}
int launch_tc(const Args &p, int head_dim, cudaStream_t s);

}  // namespace chunk
}  // namespace q3
