// Attention of a ragged batch of new rows over the paged int8 cache.
//
// With codes K8, V8 and scales ks, vs per key, a_i the row's scale in base-2 units
// (qk_scale * log2 e * the scale of q):
//     t_ij = a_i ks_j (q_i . K8_j) + log2 vs_j,   M_i = max_j t_ij,
//     p_ij = 2^(t_ij - M_i) <= 1,
//     o_i  = sum_j p_ij V8_j  /  sum_j p_ij / vs_j.
// The V scale rides in the exponent, so p spans [0, 1] whatever the scales are
// and the f16 rounding of p (2^-11 relative, the only rounding to fewer than 32
// bits) falls on weights relative to the row's largest contribution.  The codes
// are exact in f16, the products are summed in float32, and one pass keeps the
// running maximum: the accumulators are rescaled only when it grows by more
// than 2^8 over the reference in use (p then stays below 2^8, far inside f16).
//
// bf16 queries are multiplied by a power of two per row, which brings the row's
// maximum to [2^10, 2^11): their 8 bits then fit f16 exactly down to 2^-24 of
// the row's maximum, and one f16 path serves all query types.
#include "q3_attention_chunk.h"

namespace q3 {

static __device__ unsigned int g_chunk_error = 0;

int chunk_device_status_take() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_chunk_error, sizeof v) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_chunk_error, &zero, sizeof zero);
  return static_cast<int>(v);
}

namespace chunk {

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
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// One query row of a tile into shared memory as f16 (whole warp), and its a_i.
template <int HD>
__device__ __forceinline__ float stage_q(const Args &p, long r, int h, int lane, __half *dst) {
  constexpr int N = HD / 32;
  const char *qp = p.q + r * p.q_rb;
  if (p.q_dt == Q3_DT_I8) {
    Elems<int8_t, N> e;
    e.load(qp + static_cast<long>(h) * HD + lane * N);
#pragma unroll
    for (int i = 0; i < N; ++i) dst[lane * N + i] = __int2half_rn(e.e[i]);
    return __fmul_rn(p.scale_log2, reinterpret_cast<const float *>(p.qs + r * p.qs_rb)[h]);
  }
  if (p.q_dt == Q3_DT_F16) {
    Elems<__half, N> e;
    e.load(qp + (static_cast<long>(h) * HD + lane * N) * 2);
    e.store(dst + lane * N);
    return p.scale_log2;
  }
  Elems<__nv_bfloat16, N> e;
  e.load(qp + (static_cast<long>(h) * HD + lane * N) * 2);
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(to_f32(e.e[i])));
  m = warp_tree_max(m);
  // 2^up with m * 2^up in [2^10, 2^11) (m zero, subnormal or infinite: the nearest exponent)
  const int ex = static_cast<int>(__float_as_uint(m) >> 23);
  const int up = min(max(137 - ex, -120), 110);
  const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
#pragma unroll
  for (int i = 0; i < N; ++i) dst[lane * N + i] = __float2half_rn(__fmul_rn(to_f32(e.e[i]), f));
  return __fmul_rn(p.scale_log2, __uint_as_float(static_cast<uint32_t>(127 - up) << 23));
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

// ---------------------------------------------------------------------------
// Few rows.  CTA = (sequence, tile of 8 NT packed rows, KV head, part of the
// keys); packed row m is head m % group of new row m / group.  The warps take
// 32-key blocks in turn, each with its own running maximum and sums, merged in
// shared memory at the end.
//
// Keys are the M side of the products (S^T = K8 q^T, o^T = V8^T p^T), so a decode
// step with a group of 2 wastes 6 of 8 columns instead of 14 of 16 rows, and a
// thread's fragment is built from 16-byte global loads without shared memory:
// the contraction over d and the rows of o^T may be permuted freely, so a thread
// takes the bytes it loaded.  Reading K8, V8 once is the bound.
// ---------------------------------------------------------------------------
constexpr int WARPS = 4;
constexpr int KB = 32;                             // keys of a block

template <int HD, int NT>
struct FewSmem {
  static constexpr int Q = 8 * NT;                 // packed rows
  static constexpr int OS = HD + 4;                // row stride of the merged sums
  static constexpr int bytes =
      Q * HD * 2 + Q * 4 + WARPS * Q * 2 * 4 + WARPS * Q * OS * 4;
};

template <int HD, int NT>
__global__ void __launch_bounds__(WARPS * 32) k_attn_few(const Args p) {
  using S = FewSmem<HD, NT>;
  constexpr int Q = S::Q, KW = HD / 16, VW = HD / 32;   // k16 steps; words of a thread's V bytes
  extern __shared__ __align__(16) char smem[];
  __half *sq = reinterpret_cast<__half *>(smem);                   // [Q][HD]
  float *sa = reinterpret_cast<float *>(smem + Q * HD * 2);        // [Q]
  float *sml = sa + Q;                                             // [WARPS][Q][2]
  float *so = sml + WARPS * Q * 2;                                 // [WARPS][Q][OS]
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int s = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles, kvh = blockIdx.y;
  unsigned err = 0;
  const Seq sq_ = load_seq(p, s, &err);
  if (err && threadIdx.x == 0) atomicOr(&g_chunk_error, err);
  const int packed = sq_.n * p.group;
  const int m0 = tile * Q;
  if (!sq_.ok || m0 >= packed) return;
  const int mq = min(Q, packed - m0);
  // positions of the tile's rows, its key blocks and this part's
  const int p0 = sq_.pos0 + m0 / p.group, p1 = sq_.pos0 + (m0 + mq - 1) / p.group;
  int lo, hi, b0, b1;
  key_range(p, sq_, p0, p1, lo, hi);
  split_range(lo / KB, (hi + KB - 1) / KB, p.splits, blockIdx.z, b0, b1);

  for (int m = wid; m < Q; m += WARPS) {
    if (m < mq) {
      const float a = stage_q<HD>(p, sq_.first + (m0 + m) / p.group,
                                  kvh * p.group + (m0 + m) % p.group, lane, sq + m * HD);
      if (lane == 0) sa[m] = a;
    } else {
      for (int d = lane; d < HD; d += 32) sq[m * HD + d] = __ushort_as_half(0);
      if (lane == 0) sa[m] = 0.0f;
    }
  }
  __syncthreads();
  // q fragments: column n = g of tile nt; k16 step w of thread t4 holds the 4 bytes of
  // word w of its chunks (16 bytes at t4*16, and at HD/2 + t4*16 when HD = 128)
  uint32_t qf[NT][KW][2];
  float a[NT][2], mref[NT][2], lsum[NT][2];
  int pq[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const int d = (w / 4) * 64 + t4 * 16 + (w % 4) * 4;
      const uint2 x = *reinterpret_cast<const uint2 *>(sq + (n * 8 + g) * HD + d);
      qf[n][w][0] = x.x;
      qf[n][w][1] = x.y;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = n * 8 + t4 * 2 + j;
      a[n][j] = sa[m];
      pq[n][j] = sq_.pos0 + min(m0 + m, packed - 1) / p.group;
      mref[n][j] = kNegInf;
      lsum[n][j] = 0.0f;
    }
  }
  float o[HD / 16][NT][4];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][n][c] = 0.0f;

  const uint16_t *table = p.tables + static_cast<long>(s) * p.max_pages;
  const long kcol = static_cast<long>(kvh) * HD;
  // place of key b*32 + lane: page << 16 | slot, or -1 (beyond kv_len or the pool)
  auto place = [&](int b) -> uint32_t {
    const int j = b * KB + lane;
    if (b >= b1 || j >= sq_.kv) return 0xffffffffu;
    const uint32_t page = table[j / p.page_tokens];
    if (page >= p.num_pages) {
      atomicOr(&g_chunk_error, kBadPage);
      return 0xffffffffu;
    }
    return (page << 16) | (j % p.page_tokens);
  };
  uint32_t next = place(b0 + wid);
  for (int b = b0 + wid; b < b1; b += WARPS) {
    const uint32_t here = next;
    next = place(b + WARPS);
    // scales of keys i*8 + g, K rows of the same keys, V rows of this thread's 8 keys
    float ks[4], lv[4], rv[4];
    uint32_t kw[4][KW], vw[2][4][VW];
    bool in[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = __shfl_sync(0xffffffffu, here, i * 8 + g);
      in[i] = at != 0xffffffffu;
      ks[i] = 0.0f;
      lv[i] = 1.0f;
#pragma unroll
      for (int w = 0; w < KW; ++w) kw[i][w] = 0;
      if (in[i]) {
        const size_t page = at >> 16, slot = at & 0xffffu;
        const char *kr = p.k + page * p.page_bytes + slot * p.row_bytes + kcol + t4 * 16;
#pragma unroll
        for (int c = 0; c < KW / 4; ++c) {
          const uint4 x = __ldg(reinterpret_cast<const uint4 *>(kr + c * 64));
          kw[i][c * 4] = x.x, kw[i][c * 4 + 1] = x.y, kw[i][c * 4 + 2] = x.z, kw[i][c * 4 + 3] = x.w;
        }
        const size_t so_ = page * p.scale_page_bytes + slot * p.scale_row_bytes + kvh * 4;
        ks[i] = __ldg(reinterpret_cast<const float *>(p.ks + so_));
        lv[i] = __ldg(reinterpret_cast<const float *>(p.vs + so_));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = i * 16 + (j >> 1) * 8 + t4 * 2 + (j & 1);
        const uint32_t at = __shfl_sync(0xffffffffu, here, key);
#pragma unroll
        for (int w = 0; w < VW; ++w) vw[i][j][w] = 0;
        if (at != 0xffffffffu) {
          const char *vr = p.v + static_cast<size_t>(at >> 16) * p.page_bytes +
                           static_cast<size_t>(at & 0xffffu) * p.row_bytes + kcol + g * (HD / 8);
          if constexpr (HD == 128) {
            const uint4 x = __ldg(reinterpret_cast<const uint4 *>(vr));
            vw[i][j][0] = x.x, vw[i][j][1] = x.y, vw[i][j][2] = x.z, vw[i][j][3] = x.w;
          } else {
            const uint2 x = __ldg(reinterpret_cast<const uint2 *>(vr));
            vw[i][j][0] = x.x, vw[i][j][1] = x.y;
          }
        }
      }
    // S^T
    float st[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) st[i][n][c] = 0.0f;
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t x = kw[2 * i][w] ^ 0x80808080u, y = kw[2 * i + 1][w] ^ 0x80808080u;
        const uint32_t af[4] = {f16_pair(x, 0x4140), f16_pair(y, 0x4140), f16_pair(x, 0x4342),
                                f16_pair(y, 0x4342)};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816(st[i][n], af, qf[n][w][0], qf[n][w][1]);
      }
    // t = a ks S + log2 vs, masked; the block's maximum per row
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = fmaxf(lv[i], kVsMin);        // (a NaN scale: fmaxf drops it ...
      rv[i] = rcp(v);
      lv[i] = lv[i] != lv[i] ? lv[i] : lg2(v);     // ... and the row that sees it gets NaN)
    }
    const bool masked = b * KB + KB - 1 > p0 || p.window > 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = kNegInf;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float &x = st[i >> 1][n][(i & 1) * 2 + j];
          x = __fmaf_rn(__fmul_rn(x, ks[i]), a[n][j], lv[i]);
          bool see = in[i];
          if (masked) {
            const int key = b * KB + i * 8 + g;
            see = see && !(p.causal && key > pq[n][j]) &&
                  !(p.window > 0 && key <= pq[n][j] - p.window);
          }
          x = see ? x : kNegInf;
          mx = fmaxf(mx, x);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        // a new reference when the maximum outgrows the old one by 2^8
        const bool grow = mx > __fadd_rn(mref[n][j], 8.0f);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? ex2(__fsub_rn(mref[n][j], mx)) : 1.0f;
          mref[n][j] = grow ? mx : mref[n][j];
          lsum[n][j] = __fmul_rn(lsum[n][j], f);
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            o[d][n][j] = __fmul_rn(o[d][n][j], f);
            o[d][n][2 + j] = __fmul_rn(o[d][n][2 + j], f);
          }
        }
        const float base = mref[n][j] == kNegInf ? 0.0f : mref[n][j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float &x = st[i >> 1][n][(i & 1) * 2 + j];
          x = ex2(__fsub_rn(x, base));
          lsum[n][j] = __fmaf_rn(x, rv[i], lsum[n][j]);
        }
      }
    // o^T += V8^T p^T
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        pf[n][0] = transpose8(pack_f16(st[i][n][0], st[i][n][1]));
        pf[n][1] = transpose8(pack_f16(st[i][n][2], st[i][n][3]));
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        // bytes of keys (0, 1) and (2, 3) of the thread, by column
        const uint32_t l01 = __byte_perm(vw[i][0][w], vw[i][1][w], 0x5140) ^ 0x80808080u;
        const uint32_t h01 = __byte_perm(vw[i][0][w], vw[i][1][w], 0x7362) ^ 0x80808080u;
        const uint32_t l23 = __byte_perm(vw[i][2][w], vw[i][3][w], 0x5140) ^ 0x80808080u;
        const uint32_t h23 = __byte_perm(vw[i][2][w], vw[i][3][w], 0x7362) ^ 0x80808080u;
        const uint32_t fl[4] = {f16_pair(l01, 0x4140), f16_pair(l01, 0x4342),
                                f16_pair(l23, 0x4140), f16_pair(l23, 0x4342)};
        const uint32_t fh[4] = {f16_pair(h01, 0x4140), f16_pair(h01, 0x4342),
                                f16_pair(h23, 0x4140), f16_pair(h23, 0x4342)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_16816(o[2 * w][n], fl, pf[n][0], pf[n][1]);
          mma_16816(o[2 * w + 1][n], fh, pf[n][0], pf[n][1]);
        }
      }
    }
  }
  // merge: row m of o^T tile i is column g*(HD/8) + 2i (c0, c1) and + 1 (c2, c3)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float l = lsum[n][j];
      l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 4));
      l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 8));
      l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 16));
      const int m = n * 8 + t4 * 2 + j;
      if (g == 0) {
        sml[(wid * Q + m) * 2] = mref[n][j];
        sml[(wid * Q + m) * 2 + 1] = l;
      }
      float *row = so + (wid * Q + m) * S::OS + g * (HD / 8);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        row[2 * i] = o[i][n][j];
        row[2 * i + 1] = o[i][n][2 + j];
      }
    }
  __syncthreads();
  constexpr int N = HD / 32;
  for (int m = wid; m < mq; m += WARPS) {
    float mm = kNegInf, l = 0.0f, x[N];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, sml[(w * Q + m) * 2]);
    const float base = mm == kNegInf ? 0.0f : mm;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2(__fsub_rn(sml[(w * Q + m) * 2], base));
      l = __fmaf_rn(f, sml[(w * Q + m) * 2 + 1], l);
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[i] = __fmaf_rn(f, so[(w * Q + m) * S::OS + lane * N + i], x[i]);
    }
    const long r = sq_.first + (m0 + m) / p.group;
    const int h = kvh * p.group + (m0 + m) % p.group;
    if (p.splits == 1) {
      const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);   // no key seen: zeros
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __fmul_rn(x[i], inv);
      store_out<N>(p, r, h, lane, x);
    } else {
      const long at = (static_cast<long>(blockIdx.z) * p.rows + r) * p.heads + h;
#pragma unroll
      for (int i = 0; i < N; ++i) p.part_o[at * HD + lane * N + i] = x[i];
      if (lane == 0) {
        p.part_ml[at * 2] = mm;
        p.part_ml[at * 2 + 1] = l;
      }
    }
  }
}

// The parts of a row head joined (one warp each).
template <int HD>
__global__ void k_attn_join(const Args p) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const long unit = static_cast<long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long r = unit / p.heads;
  const int h = static_cast<int>(unit % p.heads);
  if (r >= p.rows) return;
  int first, count;
  const int s = find_seq(p.row0, p.n_seqs, static_cast<int>(r), lane, first, count);
  if (s < 0) return;
  unsigned err = 0;
  if (!load_seq(p, s, &err).ok) return;
  float mm = kNegInf, l = 0.0f, x[N];
  for (int z = 0; z < p.splits; ++z)
    mm = fmaxf(mm, p.part_ml[((static_cast<long>(z) * p.rows + r) * p.heads + h) * 2]);
  const float base = mm == kNegInf ? 0.0f : mm;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.0f;
  for (int z = 0; z < p.splits; ++z) {
    const long at = (static_cast<long>(z) * p.rows + r) * p.heads + h;
    const float f = ex2(__fsub_rn(p.part_ml[at * 2], base));
    l = __fmaf_rn(f, p.part_ml[at * 2 + 1], l);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmaf_rn(f, p.part_o[at * HD + lane * N + i], x[i]);
  }
  const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __fmul_rn(x[i], inv);
  store_out<N>(p, r, h, lane, x);
}

// How a call is cut: query tiles of 8*nt packed rows, parts of the key range
struct Plan {
  int nt, tiles, splits;
};
static Plan make_plan(uint32_t rows, uint32_t n_seqs, uint32_t max_rows, uint32_t max_kv,
                      uint32_t heads, uint32_t kv_heads) {
  Plan c;
  const long packed = static_cast<long>(max_rows < rows ? max_rows : rows) * (heads / kv_heads);
  c.nt = packed > 8 ? 2 : 1;
  c.tiles = static_cast<int>((packed + 8 * c.nt - 1) / (8 * c.nt));
  const long ctas = static_cast<long>(n_seqs) * c.tiles * kv_heads;
  long z = (3L * q3h::sm_count() + ctas - 1) / ctas;
  const long most = (max_kv + 511) / 512;          // 4 blocks a warp at least
  z = z < most ? z : most;
  c.splits = static_cast<int>(z < 1 ? 1 : z > 64 ? 64 : z);
  return c;
}

}  // namespace chunk

int check_pool(const q3_paged_kv *kv, uint32_t kv_heads, uint32_t head_dim, uint32_t num_pages,
               uint32_t max_pages, uint32_t align);

}  // namespace q3

// ===========================================================================
// C ABI
// ===========================================================================
using namespace q3;
using namespace q3h;

extern "C" size_t q3_attention_chunk_workspace_bytes(uint32_t rows, uint32_t n_seqs,
                                                     uint32_t max_rows, uint32_t max_kv,
                                                     uint32_t heads, uint32_t kv_heads,
                                                     uint32_t head_dim) {
  if (!rows || !n_seqs || !max_rows || !max_kv || !heads || !kv_heads || heads % kv_heads) return 0;
  const chunk::Plan c = chunk::make_plan(rows, n_seqs, max_rows, max_kv, heads, kv_heads);
  return c.splits == 1 ? 0 : static_cast<size_t>(c.splits) * rows * heads * (head_dim + 2) * 4;
}

template <int HD, int NT>
static int launch_few(const chunk::Args &p, int splits, cudaStream_t s) {
  constexpr int smem = chunk::FewSmem<HD, NT>::bytes;
  static_assert(smem <= 48 * 1024, "no opt-in needed");
  const dim3 grid(static_cast<unsigned>(p.n_seqs) * p.tiles, p.kv_heads, splits);
  chunk::k_attn_few<HD, NT><<<grid, chunk::WARPS * 32, smem, s>>>(p);
  return launch_status();
}

extern "C" int q3_attention_chunk_batch(const q3_view *q, const q3_view *q_scale,
                                        const q3_paged_kv *kv, uint32_t num_pages,
                                        const uint16_t *tables, uint32_t max_pages,
                                        const int32_t *row0, const int32_t *kv_len,
                                        uint32_t n_seqs, uint32_t max_rows, const q3_view *o,
                                        const q3_view *os, uint32_t heads, uint32_t kv_heads,
                                        uint32_t head_dim, int causal, uint32_t window,
                                        float qk_scale, void *workspace, size_t workspace_bytes,
                                        void *stream) {
  if (!tables || !row0 || !kv_len || !q || !q->data || !o || !o->data) return Q3_ERR_NULL;
  if (head_dim != 64 && head_dim != 128) return Q3_ERR_SHAPE;
  Q3_TRY(check_pool(kv, kv_heads, head_dim, num_pages, max_pages, 16));
  if (heads == 0 || heads % kv_heads || heads / kv_heads > 16) return Q3_ERR_SHAPE;
  if (causal != 0 && causal != 1) return Q3_ERR_MODE;
  if (window && (!causal || window > 0x7fffffffu)) return Q3_ERR_SHAPE;
  if (!(qk_scale > 0.0f && qk_scale < INFINITY)) return Q3_ERR_SHAPE;
  for (int i = 0; i < 2; ++i) {
    const q3_view *x = i ? o : q, *xs = i ? os : q_scale;
    if (x->dtype != Q3_DT_I8 && x->dtype != Q3_DT_F16 && x->dtype != Q3_DT_BF16)
      return Q3_ERR_DTYPE;
    Q3_TRY(check_view(x, x->dtype, 16));
    if (x->cols < heads * head_dim) return Q3_ERR_SHAPE;
    if (x->dtype == Q3_DT_I8) {
      Q3_TRY(check_view(xs, Q3_DT_F32));
      if (xs->cols < heads || xs->rows < q->rows) return Q3_ERR_SHAPE;
    }
  }
  const uint32_t rows = q->rows;
  if (o->rows < rows || rows > 0x7fffffffu / 16 || n_seqs > 0x7ffffffeu) return Q3_ERR_SHAPE;
  if (rows == 0 || n_seqs == 0) return Q3_OK;
  if (max_rows == 0) return Q3_ERR_SHAPE;
  const uint32_t max_kv = max_pages * kv->page_tokens;
  const chunk::Plan c = chunk::make_plan(rows, n_seqs, max_rows, max_kv, heads, kv_heads);
  if (static_cast<uint64_t>(n_seqs) * c.tiles > 0x7fffffffu || kv_heads > 65535) return Q3_ERR_SHAPE;
  chunk::Args p{};
  if (c.splits > 1) {
    const size_t n = static_cast<size_t>(c.splits) * rows * heads;
    if (!workspace) return Q3_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return Q3_ERR_ALIGN;
    if (workspace_bytes < n * (head_dim + 2) * 4) return Q3_ERR_CAPACITY;
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = p.part_o + n * head_dim;
  }
  p.q = (const char *)q->data;
  p.q_rb = q->row_bytes;
  p.q_dt = q->dtype;
  if (q->dtype == Q3_DT_I8) p.qs = (const char *)q_scale->data, p.qs_rb = q_scale->row_bytes;
  p.o = (char *)o->data;
  p.o_rb = o->row_bytes;
  p.o_dt = o->dtype;
  if (o->dtype == Q3_DT_I8) p.os = (char *)os->data, p.os_rb = os->row_bytes;
  p.k = (const char *)kv->k;
  p.v = (const char *)kv->v;
  p.ks = (const char *)kv->ks;
  p.vs = (const char *)kv->vs;
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
  p.rows = (int)rows;
  p.max_rows = max_rows > 0x7fffffffu ? 0x7fffffff : (int)max_rows;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads);
  p.causal = causal;
  p.window = (int)window;
  p.scale_log2 = (float)((double)qk_scale * 1.4426950408889634);
  p.splits = c.splits;
  p.tiles = c.tiles;
  cudaStream_t s = (cudaStream_t)stream;
  timer_begin(TIMER_ATTENTION, s);
  int st = head_dim == 128 ? (c.nt == 1 ? launch_few<128, 1>(p, c.splits, s)
                                        : launch_few<128, 2>(p, c.splits, s))
                           : (c.nt == 1 ? launch_few<64, 1>(p, c.splits, s)
                                        : launch_few<64, 2>(p, c.splits, s));
  if (st == Q3_OK && c.splits > 1) {
    const long warps = static_cast<long>(rows) * heads;
    const unsigned blocks = (unsigned)((warps + 3) / 4);
    if (head_dim == 128) chunk::k_attn_join<128><<<blocks, 128, 0, s>>>(p);
    else chunk::k_attn_join<64><<<blocks, 128, 0, s>>>(p);
    st = launch_status();
  }
  timer_end(TIMER_ATTENTION, s);
  return st;
}
