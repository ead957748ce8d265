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
  int tiles;                     // query tiles a sequence may have
  int few_rows;                  // packed rows of a sequence that k_attn_few takes
  int part_rows;                 // rows of one of its parts
  int page_shift;                // log2 of page_tokens, or -1
  float *part_o, *part_ml;       // parts: sums [..][hd], and their (maximum, sum of weights)
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
  if (q.n < 0 || q.first < 0 || end > p.rows || q.n > p.max_rows || q.kv < q.n) {
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

}  // namespace chunk
}  // namespace q3
