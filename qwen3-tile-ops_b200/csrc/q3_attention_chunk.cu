// Attention of a ragged batch of new rows over the paged int8 cache.
//
// With codes K8, V8 and scales ks, vs per key, a_i the row's scale in base-2 units
// (qk_scale * log2 e * the scale of q):
//     t_ij = a_i ks_j (q_i . K8_j) + log2 vs_j,   M_i = max_j t_ij,
//     p_ij = 2^(t_ij - M_i) <= 1,
//     o_i  = sum_j p_ij V8_j  /  sum_j p_ij / vs_j.
// The V scale rides in the exponent, so p spans [0, 1] whatever the scales are
// and the f16 rounding of p falls on weights relative to the row's largest
// contribution: 2^-11 of a weight, and 2^-32 of the largest one for weights below
// 2^-21 of it.  The codes are exact in f16, the products are summed in float32,
// and one pass keeps the running maximum: M is in fact a reference 2^7 below
// the maximum at the time it was set, and the accumulators are rescaled only when
// a weight outgrows it by 2^15 (p stays inside f16).
//
// bf16 queries are multiplied by a power of two per row, which brings the row's
// maximum to [2^10, 2^11) (many rows: or by 2^10, where that serves as well): their
// 8 bits then fit f16 exactly down to 2^-24 of the row's maximum, and one f16
// path serves all query types.
#include <atomic>

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

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += a b, the product by itself, then added in float32: in a running sum the tensor cores cut the bits that
// it cannot hold, always towards zero (over 500000 keys 3.3e-3 of the sum; the adds cost 0.2 us of 54, 0.4 of 18)
__device__ __forceinline__ void add_product(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  float x[4];
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.0f));
  // two at once
#pragma unroll
  for (int i = 0; i < 4; i += 2)
    asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n"
        " add.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
        : "+f"(c[i]), "+f"(c[i + 1])
        : "f"(x[i]), "f"(x[i + 1]));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// ---------------------------------------------------------------------------
// Few rows: sequences with at most few_rows packed rows (packed row m is head m %
// group of new row m / group of the sequence), in row tiles of 8 NT.  A unit of work is
// one 32-key block for one row tile; the units of the whole batch, in order, are cut into equal slices,
// and a warp takes one KV head of a slice, so ragged lengths and any number of
// sequences fill one resident wave evenly, and the heads of a token, which lie side
// by side in memory, are read at about the same time.  A warp works alone: it keeps
// the running maximum and sums of its run of a row tile and stores the result when
// it has all of its blocks, else a part (at most two a warp: of its first and its last
// row tile) that k_attn_join joins.
//
// Keys are the M side of the products (S^T = K8 q^T, o^T = V8^T p^T), so a decode
// step with a group of 2 wastes 6 of 8 columns instead of 14 of 16 rows.  A warp
// keeps STAGES blocks in shared memory or on their way there (cp.async); a fragment
// is built from 16-byte reads of codes, since the contraction over d and the rows of
// o^T may be permuted freely.
//
// Reading the cache once is the bound: 64 sequences of 2048 tokens (277 MB) 54 us, 5.1 TB/s, and
// 5.9 TB/s between the start and the end; the loads alone take as long.  Units that
// take one KV head each, dealt evenly, took 64 us, and 71 against 56 for 2 x 65011 tokens.
// Two stages of 32 keys: three leave fewer warps an SM (58 us); L2 prefetch of later pages 61 us.
// ---------------------------------------------------------------------------
constexpr int WARPS = 4;
// CTAs an SM: what registers give without spills (head_dim 64: three CTAs with two stages each 17.1 us for 24
// sequences of 5 new rows and 70 for 64 of 20; two CTAs with four stages 17.8 and 78)
__host__ __device__ constexpr int few_ctas_sm(int hd, int nt) { return hd == 64 || nt == 1 ? 3 : 2; }
constexpr int KB = 32;                             // keys of a block
// Least units of a slice.  Alone, short slices spread a small batch (one sequence of 2000 tokens 8.5 us;
// slices of 4 10.2, of 1 8.5 with more parts).  Beside the many-row kernel this one has the SMs that
// are left, and many short slices queue there (16 ragged sequences 64 us; of 2 72, of 32 79).
constexpr int ALONE_UNITS = 2, BESIDE_UNITS = 8;
// Most packed rows of a sequence of this kernel, in tiles that read the keys again.  Alone: 2 sequences of
// 48 packed rows over 1000 tokens 15.1 us, in the many-row kernel 20.4; 64 over 2000 177 and 181; 8 of 64
// rows over 4000 63 and 54.  Beside the many-row kernel: 16 ragged sequences 62.8 us, with 32 rows 64.0.
// That batch has few sequences between the two bounds; with many the step down costs: 63 of 20 packed
// rows over 2000 tokens take 113 us alone, 176 where max_rows allows more than 48 packed ones, and 209
// with a chunk of 1000 rows (itself 55).
constexpr int ALONE_ROWS = 48, BESIDE_ROWS = 16;
constexpr uint32_t WHOLE_KEYS = 256;               // most keys of a sequence that one warp takes (make_plan)

template <int HD>
struct FewStage {
  static constexpr int STAGES = 2;
  uint4 k[KB * HD / 16], v[KB * HD / 16];
  float ks[KB], vs[KB];
};

// Row tiles of sequence s, of 2^row_shift packed rows
__device__ __forceinline__ int row_tiles(const Args &p, const Seq &s) {
  return (s.n * p.group + (1 << p.row_shift) - 1) >> p.row_shift;
}
// Blocks of sequence s (0: not this kernel's) and the first of them; a tile's units are its blocks
__device__ __forceinline__ int seq_blocks(const Args &p, const Seq &s, int &b0) {
  b0 = 0;
  if (!s.ok || s.n * p.group > p.few_rows) return 0;
  int lo, hi;
  key_range(p, s, s.pos0, s.kv - 1, lo, hi);
  b0 = lo / KB;
  return (hi + KB - 1) / KB - b0;
}
__device__ __forceinline__ int units_of(const Args &p, int s, unsigned *err) {
  int b0;
  const Seq q = load_seq(p, s, err);
  const int n = seq_blocks(p, q, b0);
  return n ? n * row_tiles(p, q) : 0;
}
// All units, and those of the sequences before s0 (whole warp; the host bounds them by 3 2^30)
__device__ __forceinline__ uint32_t count_units(const Args &p, int s0, int lane, unsigned *err,
                                                uint32_t &before) {
  uint32_t x = 0, y = 0;
  for (int s = lane; s < p.n_seqs; s += 32) {
    const uint32_t n = units_of(p, s, err);
    x += n;
    y += s < s0 ? n : 0;
  }
  before = __reduce_add_sync(0xffffffffu, y);
  return __reduce_add_sync(0xffffffffu, x);
}
// The slices of `total` units: the first `more` have each + 1 of them
struct Slices {
  uint32_t n, each, more;
  __device__ __forceinline__ Slices(uint32_t total, uint32_t most, uint32_t least) {
    n = (total + least - 1) / least;
    n = n < most ? n : most;
    n = n ? n : 1;
    each = total / n;
    more = total - each * n;
  }
  __device__ __forceinline__ uint32_t first(uint32_t w) const { return w * each + min(w, more); }
  __device__ __forceinline__ uint32_t of(uint32_t unit) const {
    const uint32_t big = more * (each + 1);
    return unit < big ? unit / (each + 1) : more + (unit - big) / each;
  }
};

// 16 (HD 64: 8) columns at g * HD/8 of one row head, a row spread over the 8 lanes of equal t4
template <int N>
__device__ __forceinline__ void store_part8(const Args &p, long r, int h, int g, bool ok,
                                            float (&x)[N]) {
  constexpr int HD = 8 * N;
  const long col = static_cast<long>(h) * HD + g * N;
  char *o = p.o + r * p.o_rb;
  if (p.o_dt == Q3_DT_I8) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    const float scale = __fmul_rn(m, kInv127);
    uint32_t c[N / 4];
    quant_pack_absmax<N>(x, scale, c);
    if (!ok) return;
    Elems<int8_t, N> e;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint32_t *>(e.e)[i] = c[i];
    e.store(o + col);
    if (g == 0) reinterpret_cast<float *>(p.os + r * p.os_rb)[h] = scale;
  } else if (ok) {
    if (p.o_dt == Q3_DT_F16) store_row<__half, N>(x, o + col * 2);
    else store_row<__nv_bfloat16, N>(x, o + col * 2);
  }
}

__device__ __forceinline__ void cp4(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0)
               : "memory");
}

template <int HD, int NT>
__global__ void __launch_bounds__(WARPS * 32, few_ctas_sm(HD, NT)) k_attn_few(const Args p) {
  constexpr int KW = HD / 16, VW = HD / 32;   // k16 steps; words of a thread's V bytes
  constexpr int CH = HD / 16;                 // 16-byte chunks of a row
  using Stage = FewStage<HD>;
  constexpr int STAGES = Stage::STAGES;
  extern __shared__ __align__(128) char smem[];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  Stage *ring = reinterpret_cast<Stage *>(smem) + wid * STAGES;
  const uint32_t w = blockIdx.x * WARPS + wid, slice = w / p.kv_heads;
  const int kvh = w - slice * p.kv_heads;

  pdl_trigger();   // the join may start: it looks up its parts while this kernel works
  unsigned err = 0;
  uint32_t u = 0, u1 = 1;
  long before = 0;
  int s = -1;
  int m0 = 0;                                      // first packed row of this warp's
  if (p.whole) {   // 8 NT packed rows of a sequence a slice: nothing to look up, no parts
    const uint32_t at = slice / p.tiles;
    m0 = static_cast<int>(slice - at * p.tiles) * (8 * NT);
    if (at < static_cast<uint32_t>(p.n_seqs)) s = at;
    if (s >= 0 && kvh == 0 && m0 == 0) {
      load_seq(p, s, &err);
      if (err && lane == 0) atomicOr(&g_chunk_error, err);
    }
  } else {
    // sequences 0 .. 31 in registers; more are looked up in turn
    const uint32_t mine = lane < p.n_seqs ? units_of(p, lane, &err) : 0;
    uint32_t total = __reduce_add_sync(0xffffffffu, mine);
    for (int x = 32 + lane; x - lane < p.n_seqs; x += 32)
      total += __reduce_add_sync(0xffffffffu, x < p.n_seqs ? units_of(p, x, &err) : 0);
    if (w == 0 && err) atomicOr(&g_chunk_error, err);
    const Slices cut(total, gridDim.x * WARPS / p.kv_heads, p.min_units);
    if (total && slice < cut.n) {
      u = cut.first(slice);
      u1 = cut.first(slice + 1);
      s = find_unit(p.n_seqs, u, lane, before,
                    [&](int x) { return x == lane ? mine : units_of(p, x, &err); });
    }
  }
  if (s >= 0) {
    while (u < u1 && s < p.n_seqs) {
      // the sequence of unit u, its blocks [pb0, pb0 + pn), and this warp's run [b, be) of them
      const Seq q = load_seq(p, s, &err);
      int pb0, pn = seq_blocks(p, q, pb0);
      int off = static_cast<int>(u - static_cast<uint32_t>(before));
      m0 = p.whole ? m0 : 0;
      if (!p.whole && off >= pn && pn) {           // a row tile behind the first
        m0 = off / pn;
        off -= m0 * pn;
        m0 *= 8 * NT;
      }
      const int packed = min(8 * NT, q.n * p.group - m0);
      if (pn == 0 || packed <= 0) {
        if (p.whole) break;
        ++s;                                       // (a sequence without units)
        continue;
      }
      const int pmin = q.pos0 + m0 / p.group;      // position of the first of the rows
      if (p.whole) {
        int lo, hi;
        key_range(p, q, pmin, q.pos0 + (m0 + packed - 1) / p.group, lo, hi);
        pb0 = lo / KB;
        pn = (hi + KB - 1) / KB - pb0;
        u1 = pn;
      }
      const int b = pb0 + off;
      const int run = static_cast<int>(u1 - u) < pn - off ? static_cast<int>(u1 - u) : pn - off;
      const int be = b + run;
      const bool whole = off == 0 && run == pn;
      const uint16_t *table = p.tables + static_cast<long>(s) * p.max_pages;
      const long kcol = static_cast<long>(kvh) * HD;
      // table index and slot of key x*32 + lane; its page is requested one step before it is used
      auto page_of = [&](int x) -> int {
        const int j = x * KB + lane;
        return x < be && j < q.kv ? table[page_index(p, j)] : -1;
      };
      // this lane's part of a block: chunk lane % CH of rows lane / CH, + 32 / CH, ...; in places
      // that make the fragment reads conflict-free (see there)
      const int fr = lane / CH, fc = lane % CH;
      const long from = kcol + static_cast<long>(fr) * p.row_bytes + fc * 16;
      const uint32_t step = (32 / CH) * p.row_bytes;
      const int kto = HD == 128 ? fr * 8 + (fc ^ ((fr & 1) << 2)) : (fr >> 1) * 8 + (fr & 1) * 4 + fc;
      const int vto = HD == 128 ? fr * 8 + (fc ^ (fr & 2)) : kto ^ (((fr >> 1) & 3) << 1);
      auto fetch = [&](int x, int pg) -> unsigned {   // block x into its stage; its keys that exist
        Stage &st = ring[x % STAGES];
        const uint32_t kd = static_cast<uint32_t>(__cvta_generic_to_shared(st.k + kto)),
                       vd = static_cast<uint32_t>(__cvta_generic_to_shared(st.v + vto)),
                       sd = static_cast<uint32_t>(__cvta_generic_to_shared(st.ks + lane));
        unsigned have = 0;
        if (x < be) {
          const int j = x * KB + lane;
          const bool ok = pg >= 0 && static_cast<uint32_t>(pg) < p.num_pages;
          if (pg >= 0 && !ok) atomicOr(&g_chunk_error, kBadPage);
          have = __ballot_sync(0xffffffffu, ok);
          const uint32_t slot = page_slot(p, j);
          if (p.whole_blocks && have == 0xffffffffu) {
            // one page, all of its keys: rows at equal steps
            const size_t at = static_cast<size_t>(pg) * p.page_bytes +
                              static_cast<size_t>(slot - lane) * p.row_bytes + from;
            const char *k = p.k + at, *v = p.v + at;
#pragma unroll
            for (int i = 0; i < CH; ++i) {
              cp16(kd + i * 512, k, true);
              cp16((HD == 128 && (i & 1) ? vd ^ 64 : vd) + i * 512, v, true);
              k += step;
              v += step;
            }
          } else {
            const uint32_t mine = ok ? (static_cast<uint32_t>(pg) << 16) | slot : 0xffffffffu;
#pragma unroll 2
            for (int i = 0; i < CH; ++i) {
              const uint32_t ra = __shfl_sync(0xffffffffu, mine, i * (32 / CH) + fr);
              const bool rok = ra != 0xffffffffu;
              const size_t at = rok ? static_cast<size_t>(ra >> 16) * p.page_bytes +
                                          static_cast<size_t>(ra & 0xffffu) * p.row_bytes + kcol +
                                          fc * 16
                                    : 0;
              cp16(kd + i * 512, p.k + at, rok);
              cp16((HD == 128 && (i & 1) ? vd ^ 64 : vd) + i * 512, p.v + at, rok);
            }
          }
          const size_t so = ok ? static_cast<size_t>(pg) * p.scale_page_bytes +
                                     static_cast<size_t>(slot) * p.scale_row_bytes + kvh * 4
                               : 0;
          cp4(sd, p.ks + so, ok);
          cp4(sd + KB * 4, p.vs + so, ok);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return have;
      };
      int pg[STAGES];
      unsigned have[STAGES];
#pragma unroll
      for (int i = 0; i < STAGES; ++i) pg[i] = page_of(b + i);

      // query fragments: column n*8 + g; k16 step x of thread t4 takes the 4 codes of word x of
      // its chunks (16 bytes at t4*16, and at 64 + t4*16 when HD = 128)
      uint32_t qf[NT][KW][2];
      float a[NT][2], mref[NT][2], lsum[NT][2];
      int pq[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int m = n * 8 + g;
        float scale = 0.0f;
#pragma unroll
        for (int x = 0; x < KW; ++x) qf[n][x][0] = qf[n][x][1] = 0;
        const int mm = m0 + min(m, packed - 1);
        const long r = q.first + mm / p.group;
        const int h = kvh * p.group + mm % p.group;
        const char *qp = p.q + r * p.q_rb;
        if (p.q_dt == Q3_DT_I8) {
          if (m < packed) {
            scale = reinterpret_cast<const float *>(p.qs + r * p.qs_rb)[h];
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
              Elems<uint32_t, 4> e;
              e.load(qp + static_cast<long>(h) * HD + c * 64 + t4 * 16);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t x = e.e[i] ^ 0x80808080u;
                qf[n][c * 4 + i][0] = f16_pair(x, 0x4140);
                qf[n][c * 4 + i][1] = f16_pair(x, 0x4342);
              }
            }
          }
        } else {
          scale = 1.0f;
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) {
            Elems<uint32_t, 8> e;
            e.load(qp + (static_cast<long>(h) * HD + c * 64 + t4 * 16) * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              qf[n][c * 4 + i][0] = e.e[2 * i];
              qf[n][c * 4 + i][1] = e.e[2 * i + 1];
            }
          }
          if (p.q_dt == Q3_DT_BF16) {
            float mx = 0.0f;
#pragma unroll
            for (int x = 0; x < KW; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                mx = fmaxf(mx, fabsf(__uint_as_float(qf[n][x][i] << 16)));
                mx = fmaxf(mx, fabsf(__uint_as_float(qf[n][x][i] & 0xffff0000u)));
              }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            float up;
            bf16_scale(mx, up, scale);
#pragma unroll
            for (int x = 0; x < KW; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                qf[n][x][i] = pack_f16(__fmul_rn(__uint_as_float(qf[n][x][i] << 16), up),
                                       __fmul_rn(__uint_as_float(qf[n][x][i] & 0xffff0000u), up));
          }
        }
        scale = __fmul_rn(scale, p.scale_log2);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          a[n][j] = __shfl_sync(0xffffffffu, scale, (t4 * 2 + j) * 4);
          pq[n][j] = q.pos0 + (m0 + min(n * 8 + t4 * 2 + j, packed - 1)) / p.group;
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

#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) have[i] = fetch(b + i, pg[i]);
      int pnext = pg[STAGES - 1];
      for (int x = b; x < be; ++x) {
        const unsigned newest = fetch(x + STAGES - 1, pnext);
        pnext = page_of(x + STAGES);
        unsigned mask = have[0];
#pragma unroll
        for (int i = 0; i + 2 < STAGES; ++i) have[i] = have[i + 1];
        have[STAGES - 2] = newest;
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const Stage &st = ring[x % STAGES];
        // S^T: rows g and g + 8 of the two 16-key tiles
        float sc[2][NT][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t kw[2][KW];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int row = i * 16 + y * 8 + g;
#pragma unroll
            for (int c = 0; c < KW / 4; ++c) {
              // a quarter warp reads 4 chunks of two rows: the odd row's lie in the other half
              const int at = HD == 128 ? row * 8 + ((c * 4 + t4) ^ ((row & 1) << 2)) : row * 4 + t4;
              const uint4 z = st.k[at];
              kw[y][c * 4] = z.x ^ 0x80808080u, kw[y][c * 4 + 1] = z.y ^ 0x80808080u;
              kw[y][c * 4 + 2] = z.z ^ 0x80808080u, kw[y][c * 4 + 3] = z.w ^ 0x80808080u;
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) sc[i][n][c] = 0.0f;
#pragma unroll
          for (int c = 0; c < KW; ++c) {
            const uint32_t af[4] = {f16_pair(kw[0][c], 0x4140), f16_pair(kw[1][c], 0x4140),
                                    f16_pair(kw[0][c], 0x4342), f16_pair(kw[1][c], 0x4342)};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816(sc[i][n], af, qf[n][c][0], qf[n][c][1]);
          }
        }
        // t = a ks S + log2 vs, masked; the block's maximum per row
        float ks[4], lv[4], rv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ks[i] = st.ks[i * 8 + g];
          const float v = st.vs[i * 8 + g];
          rv[i] = __fmul_rn(rcp(fmaxf(v, kVsMin)), kSumScale);   // (NaN: fmaxf drops it ...
          lv[i] = v != v ? v : lg2(fmaxf(v, kVsMin));// ... and the rows that see it get NaN)
        }
        const bool masked = mask != 0xffffffffu || x * KB + KB - 1 > pmin || p.window > 0;
        // relative to the reference of the row's weights, which moves when one outgrows it by 2^kRefMove
        float top[NT][2];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float base = mref[n][j] == kNegInf ? 0.0f : mref[n][j];
            float mx = kNegInf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float &y = sc[i >> 1][n][(i & 1) * 2 + j];
              y = __fsub_rn(__fmaf_rn(__fmul_rn(y, ks[i]), a[n][j], lv[i]), base);
              if (masked) {
                const int key = x * KB + i * 8 + g;
                const bool see = ((mask >> (i * 8 + g)) & 1) && !(p.causal && key > pq[n][j]) &&
                                 !(p.window > 0 && key <= pq[n][j] - p.window);
                y = see ? y : kNegInf;
              }
              mx = fmaxf(mx, y);
            }
            top[n][j] = mx;
            grow = grow || mx > kRefMove || mref[n][j] == kNegInf;
          }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float mx = top[n][j];
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const bool none = mref[n][j] == kNegInf;
              const bool move = mx > (none ? kNegInf : kRefMove);
              const float up = move ? __fsub_rn(mx, kRefBelow) : 0.0f;
              const float f = none ? 1.0f : ex2(-up);    // (without a reference the sums are zero)
              if (move) mref[n][j] = none ? up : __fadd_rn(mref[n][j], up);
              lsum[n][j] = __fmul_rn(lsum[n][j], f);
#pragma unroll
              for (int d = 0; d < HD / 16; ++d) {
                o[d][n][j] = __fmul_rn(o[d][n][j], f);
                o[d][n][2 + j] = __fmul_rn(o[d][n][2 + j], f);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float &y = sc[i >> 1][n][(i & 1) * 2 + j];
                y = __fsub_rn(y, up);
              }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float &y = sc[i >> 1][n][(i & 1) * 2 + j];
              y = ex2(y);
              lsum[n][j] = __fmaf_rn(y, rv[i], lsum[n][j]);
            }
        // o^T += V8^T p^T
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t pf[NT][2], vw[4][VW];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            pf[n][0] = transpose8(pack_f16(sc[i][n][0], sc[i][n][1]));
            pf[n][1] = transpose8(pack_f16(sc[i][n][2], sc[i][n][3]));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // a quarter (HD 64: half) warp reads 2 chunks of rows 0, 2, 4, 6 (+ const)
            const int row = i * 16 + (j >> 1) * 8 + t4 * 2 + (j & 1);
            if constexpr (HD == 128) {
              const uint4 z = st.v[row * 8 + (g ^ (row & 6))];
              vw[j][0] = z.x, vw[j][1] = z.y, vw[j][2] = z.z, vw[j][3] = z.w;
            } else {
              const int line = row >> 1, c = ((row & 1) * 4 + (g >> 1)) ^ ((line & 3) << 1);
              const uint2 z = reinterpret_cast<const uint2 *>(st.v)[(line * 8 + c) * 2 + (g & 1)];
              vw[j][0] = z.x, vw[j][1] = z.y;
            }
          }
#pragma unroll
          for (int c = 0; c < VW; ++c) {
            // codes of keys (0, 1) and (2, 3) of the thread side by side, by column
            const uint32_t l01 = __byte_perm(vw[0][c], vw[1][c], 0x5140) ^ 0x80808080u;
            const uint32_t h01 = __byte_perm(vw[0][c], vw[1][c], 0x7362) ^ 0x80808080u;
            const uint32_t l23 = __byte_perm(vw[2][c], vw[3][c], 0x5140) ^ 0x80808080u;
            const uint32_t h23 = __byte_perm(vw[2][c], vw[3][c], 0x7362) ^ 0x80808080u;
            const uint32_t fl[4] = {f16_pair(l01, 0x4140), f16_pair(l01, 0x4342),
                                    f16_pair(l23, 0x4140), f16_pair(l23, 0x4342)};
            const uint32_t fh[4] = {f16_pair(h01, 0x4140), f16_pair(h01, 0x4342),
                                    f16_pair(h23, 0x4140), f16_pair(h23, 0x4342)};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              add_product(o[2 * c][n], fl, pf[n]);
              add_product(o[2 * c + 1][n], fh, pf[n]);
            }
          }
        }
        __syncwarp();   // the stage is read before the next fetch overwrites it
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      // column g*(HD/8) + 2i of o^T in o[i][n][j], + 1 in o[i][n][2 + j], row n*8 + t4*2 + j
      const long slot = 2 * static_cast<long>(w) + (off == 0 ? 1 : 0);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float l = lsum[n][j];
          l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 4));
          l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 8));
          l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 16));
          const int m = n * 8 + t4 * 2 + j;
          const bool ok = m < packed;
          float y[HD / 8];
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            y[2 * i] = o[i][n][j];
            y[2 * i + 1] = o[i][n][2 + j];
          }
          if (whole) {
            const float inv = inverse_sum(l);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) y[i] = __fmul_rn(y[i], inv);
            const int mm = m0 + min(m, packed - 1);
            store_part8<HD / 8>(p, q.first + mm / p.group, kvh * p.group + mm % p.group, g, ok, y);
          } else if (ok) {
            const long at = slot * (8 * NT) + m;
            Elems<float, HD / 8> e;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) e.e[i] = y[i];
            e.store(p.part_o + at * HD + g * (HD / 8));
            if (g == 0) {
              p.part_ml[at * 2] = mref[n][j];
              p.part_ml[at * 2 + 1] = l;
            }
          }
        }
      u += run;
      if (m0 + 8 * NT >= q.n * p.group || p.whole) {   // on to the next sequence
        before += static_cast<long>(pn) * row_tiles(p, q);
        ++s;
      }
    }
  }
  // as a dependent of the many-row kernel it began when all CTAs of that were running; what comes
  // after waits for both
  pdl_wait();
}

// Parts joined: a CTA takes R packed rows of a (sequence, KV head) pair, 8 / R warps a row, which take its
// parts in turn, JOIN_AT loads at once.  Bound by latency: look-ups, which hide behind the kernel
// before it only where its CTAs leave room on the SMs, then the parts (111 a sequence at 2 x 65011
// tokens).  R is the least of 1, 2, 4, 8 that leaves 6 CTAs an SM or fewer: whole calls with R = 1, 2,
// 4, 8 take 8.4, 9.2, 10.0, 12.4 us (16 rows in all), 57.0, 53.8, 53.7, 54.6 (64 x 2048 tokens, 1024 rows),
// 92, 79, 72, 69 (8192 rows).
constexpr int JOIN_WARPS = 8, JOIN_AT = 4;
template <int HD, int R>
__global__ void __launch_bounds__(JOIN_WARPS * 32) k_attn_join(const Args p, uint32_t most) {
  constexpr int N = HD / 32, WR = JOIN_WARPS / R;  // warps of a row
  __shared__ float so[JOIN_WARPS][HD], sm[JOIN_WARPS], sl[JOIN_WARPS];
  __shared__ uint32_t units[2];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int s = blockIdx.x, kvh = blockIdx.y;
  unsigned err = 0;
  const Seq q = load_seq(p, s, &err);
  int pb0;
  const int pn = seq_blocks(p, q, pb0);
  const int m = blockIdx.z * R + wid / WR, wr = wid % WR;   // packed row
  // (also a CTA with nothing to join waits: when this grid ends, the results are there)
  if (pn == 0 || static_cast<int>(blockIdx.z) * R >= q.n * p.group) {   // refused, or the other kernel's
    pdl_wait();
    return;
  }
  if (wid == 0) {
    uint32_t before;
    const uint32_t total = count_units(p, s, lane, &err, before);
    if (lane == 0) units[0] = total, units[1] = before;
  }
  __syncthreads();
  // the slices that have units of the row's tile
  const Slices cut(units[0], most, p.min_units);
  const uint32_t u0 = units[1] + (m >> p.row_shift) * pn, w0 = cut.of(u0), w1 = cut.of(u0 + pn - 1);
  pdl_wait();
  const bool join = m < q.n * p.group && w0 != w1;   // (one slice: stored whole)
  const long r = q.first + m / p.group;
  const int h = kvh * p.group + m % p.group;
  float mm = kNegInf, l = 0.0f, x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.0f;
  for (uint32_t w = w0 + wr; join && w <= w1; w += WR * JOIN_AT) {
    float pm[JOIN_AT], pl[JOIN_AT];
    Elems<float, N> e[JOIN_AT];
#pragma unroll
    for (int k = 0; k < JOIN_AT; ++k) {
      const uint32_t wk = w + k * WR;
      pm[k] = kNegInf;
      pl[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) e[k].e[i] = 0.0f;
      if (wk <= w1) {   // the warp's part: of its last sequence if this one begins with it
        const long at = ((2 * (static_cast<long>(wk) * p.kv_heads + kvh) + (wk == w0 ? 1 : 0))
                         << p.row_shift) + (m & ((1 << p.row_shift) - 1));
        pm[k] = p.part_ml[at * 2];
        pl[k] = p.part_ml[at * 2 + 1];
        e[k].load(p.part_o + at * HD + lane * N);
      }
    }
#pragma unroll
    for (int k = 0; k < JOIN_AT; ++k) {
      const float top = fmaxf(mm, pm[k]), base = top == kNegInf ? 0.0f : top;
      const float f0 = ex2(__fsub_rn(mm, base)), f1 = ex2(__fsub_rn(pm[k], base));
      mm = top;
      l = __fmaf_rn(f1, pl[k], __fmul_rn(f0, l));
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __fmaf_rn(f1, e[k].e[i], __fmul_rn(f0, x[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) so[wid][lane * N + i] = x[i];
  if (lane == 0) sm[wid] = mm, sl[wid] = l;
  __syncthreads();
  if (wr || !join) return;
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < WR; ++i) top = fmaxf(top, sm[wid + i]);
  const float base = top == kNegInf ? 0.0f : top;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.0f;
#pragma unroll
  for (int k = 0; k < WR; ++k) {
    const float f = ex2(__fsub_rn(sm[wid + k], base));
    l = __fmaf_rn(f, sl[wid + k], l);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmaf_rn(f, so[wid + k][lane * N + i], x[i]);
  }
  const float inv = inverse_sum(l);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __fmul_rn(x[i], inv);
  store_out<N>(p, r, h, lane, x);
}

// The parts of k_attn_tc's key ranges, 256 rows each in the order of its CTAs: a warp a packed row of a
// tile.  Bound by latency; 20 MB written and read at most, since keys are split only while the tiles
// cannot fill the card (148 parts of 256 rows).
constexpr int TILE_WARPS = 4;
template <int HD>
__global__ void __launch_bounds__(TILE_WARPS * 32) k_join_tiles(const Args p) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % p.kv_heads, row = blockIdx.y * TILE_WARPS + (threadIdx.x >> 5);
  unsigned err = 0;
  int tile;
  const int s = find_tile(p, blockIdx.x / p.kv_heads, lane, &err, tile);
  if (s < 0) return;
  const Seq q = load_seq(p, s, &err);
  const int m = tile * TC_ROWS + row;
  if (m >= q.n * p.group) return;
  const long r = q.first + m / p.group;
  const int h = kvh * p.group + m % p.group;
  // lane z has the maximum and sum of part z, and of z + 32 (splits <= 64)
  const long at = static_cast<long>(blockIdx.x) * p.splits * TC_ROWS + row, step = TC_ROWS;
  float pm[2], pl[2], f[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int z = lane + i * 32;
    pm[i] = z < p.splits ? p.part_ml[(z * step + at) * 2] : kNegInf;
    pl[i] = z < p.splits ? p.part_ml[(z * step + at) * 2 + 1] : 0.0f;
  }
  const float mm = warp_tree_max(fmaxf(pm[0], pm[1])), base = mm == kNegInf ? 0.0f : mm;
#pragma unroll
  for (int i = 0; i < 2; ++i) f[i] = ex2(__fsub_rn(pm[i], base));
  const float l = warp_tree_sum(__fmaf_rn(f[1], pl[1], __fmul_rn(f[0], pl[0])));
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.0f;
  for (int z0 = 0; z0 < p.splits; z0 += JOIN_AT) {
    Elems<float, N> e[JOIN_AT];
    float fz[JOIN_AT];
#pragma unroll
    for (int k = 0; k < JOIN_AT; ++k) {
      const int z = z0 + k;
      fz[k] = __shfl_sync(0xffffffffu, z < 32 ? f[0] : f[1], z & 31);
      if (fz[k] != 0.0f) e[k].load(p.part_o + (z * step + at) * HD + lane * N);
      else e[k].zero();                              // (a part without keys has no sums)
    }
#pragma unroll
    for (int k = 0; k < JOIN_AT; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __fmaf_rn(fz[k], e[k].e[i], x[i]);
  }
  const float inv = inverse_sum(l);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __fmul_rn(x[i], inv);
  store_out<N>(p, r, h, lane, x);
}

// How a call is cut.  Sequences with at most few_rows packed rows go to k_attn_few (nt tiles of 8),
// the others to the tensor-core kernel of many rows.  Which of them there are is known on the device
// only, so k_attn_few (and, unless `whole`, its join) is always launched, the other kernel where
// max_rows allows such sequences (tiles > 0).
struct Plan {
  long packed;                                     // most packed rows of a sequence
  int nt, few_rows, min_units;
  long few_ctas, few_tiles;
  bool whole;                                      // their keys are not cut
  long tiles;                                      // 0: no sequence can have more than few_rows
  int splits;
  size_t few_slots, bytes;                         // parts of k_attn_few; the whole workspace
};
static Plan make_plan(uint32_t rows, uint32_t n_seqs, uint32_t max_rows, uint32_t max_kv,
                      uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  Plan c{};
  const long group = heads / kv_heads;
  // (one with more new rows than its table holds tokens is refused)
  const uint32_t most_new = max_rows < rows ? max_rows : rows;
  const long packed = c.packed = static_cast<long>(most_new < max_kv ? most_new : max_kv) * group;
  const int sms = q3h::sm_count();
  const bool mixed = packed > ALONE_ROWS;
  c.few_rows = mixed ? BESIDE_ROWS : ALONE_ROWS;
  c.min_units = mixed ? BESIDE_UNITS : ALONE_UNITS;
  c.nt = packed > 8 ? 2 : 1;
  // Up to 256 keys a warp takes a whole sequence if that gives each SM a warp (64 sequences of 220
  // keys 12.5 us, cut 17.4; 8 of them 11.4 and 10.1), or to spare the many-row kernel (4 x 60 rows 15 us
  // against 17)
  c.whole = max_kv <= WHOLE_KEYS && (packed > 16 || static_cast<long>(n_seqs) * kv_heads > sms);
  const long most_rows = packed < c.few_rows ? packed : c.few_rows;
  const long units = static_cast<long>(n_seqs) * ((max_kv + KB - 1) / KB) *
                     ((most_rows + 8 * c.nt - 1) / (8 * c.nt));
  const long slices = (units + c.min_units - 1) / c.min_units;
  const long most = static_cast<long>(sms) * few_ctas_sm(head_dim, c.nt), least = (kv_heads + WARPS - 1) / WARPS;
  long ctas = (slices * kv_heads + WARPS - 1) / WARPS;
  ctas = ctas < most ? ctas : most;
  ctas = ctas > least ? ctas : least;              // a slice at least
  if (c.whole) {   // then all rows go there, in tiles
    c.few_rows = 0x7fffffff;
    c.few_tiles = (packed + 8 * c.nt - 1) / (8 * c.nt);
    ctas = (static_cast<long>(n_seqs) * c.few_tiles * kv_heads + WARPS - 1) / WARPS;
  }
  c.few_ctas = ctas;
  if (!c.whole) c.few_slots = 2 * static_cast<size_t>(c.few_ctas) * WARPS * 8 * c.nt;
  c.splits = 1;
  if (packed > c.few_rows) {
    const long all = static_cast<long>(rows) * group / TC_ROWS + n_seqs;
    const long each = (packed + TC_ROWS - 1) / TC_ROWS * n_seqs;
    c.tiles = all < each ? all : each;
    const long ctas = c.tiles * kv_heads;
    long z = ctas >= sms ? 1 : sms / ctas;         // one CTA on each SM
    // (parts of at least two key tiles: 200 rows over 1000 tokens 24.8 us; of four 27.2)
    const long most = (max_kv + 2 * TC_KEYS - 1) / (2 * TC_KEYS);
    z = z < most ? z : most;
    c.splits = static_cast<int>(z < 1 ? 1 : z > 64 ? 64 : z);
  }
  const size_t parts = c.splits > 1 ? static_cast<size_t>(c.splits) * c.tiles * kv_heads * TC_ROWS : 0;
  const bool fold = c.tiles && c.splits == 1 && max_kv > FOLD_KEYS;
  c.bytes = (c.few_slots + parts) * (head_dim + 2) * 4 +
            (fold ? static_cast<size_t>(rows) * heads * head_dim * 4 : 0);
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
  if (!rows || !n_seqs || !max_rows || !max_kv || !heads || !kv_heads || heads % kv_heads ||
      heads / kv_heads > 16 || (head_dim != 64 && head_dim != 128))
    return 0;
  return chunk::make_plan(rows, n_seqs, max_rows, max_kv, heads, kv_heads, head_dim).bytes;
}

// Dynamic shared memory above 48 KB is opted into once per kernel and device.
template <auto kernel>
static int opt_in(int bytes) {
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_cuda_error(e);
      return Q3_ERR_CUDA;
    }
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return Q3_OK;
}

template <int HD, int NT>
static int launch_few(const chunk::Args &p, long packed, int ctas, bool beside, cudaStream_t s) {
  constexpr int smem = chunk::WARPS * chunk::FewStage<HD>::STAGES * (int)sizeof(chunk::FewStage<HD>);
  Q3_TRY((opt_in<&chunk::k_attn_few<HD, NT>>(smem)));
  Q3_TRY(launch_ex(beside, chunk::k_attn_few<HD, NT>, dim3(ctas), dim3(chunk::WARPS * 32), smem, s, p));
  const unsigned z = static_cast<unsigned>(packed < p.few_rows ? packed : p.few_rows);
  if (p.whole) return Q3_OK;
  const uint32_t most = static_cast<uint32_t>(ctas) * chunk::WARPS / p.kv_heads;
  const long pairs = static_cast<long>(p.n_seqs) * p.kv_heads, room = 6L * sm_count();
  const unsigned r = pairs * z <= room               ? 1
                     : pairs * ((z + 1) / 2) <= room ? 2
                     : pairs * ((z + 3) / 4) <= room ? 4
                                                     : 8;
  const auto join = r == 1   ? chunk::k_attn_join<HD, 1>
                    : r == 2 ? chunk::k_attn_join<HD, 2>
                    : r == 4 ? chunk::k_attn_join<HD, 4>
                             : chunk::k_attn_join<HD, 8>;
  return launch_ex(true, join, dim3(p.n_seqs, p.kv_heads, (z + r - 1) / r),
                   dim3(chunk::JOIN_WARPS * 32), 0, s, p, most);
}

template <int HD>
static int launch_many(const chunk::Args &p, long packed, cudaStream_t s) {
  Q3_TRY(chunk::launch_tc(p, HD, s));
  if (p.splits == 1) return Q3_OK;
  const unsigned rows = packed < chunk::TC_ROWS ? (unsigned)packed : chunk::TC_ROWS;   // of a tile
  chunk::k_join_tiles<HD><<<dim3(p.tiles * p.kv_heads, (rows + chunk::TILE_WARPS - 1) / chunk::TILE_WARPS),
                            chunk::TILE_WARPS * 32, 0, s>>>(p);
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
  const float scale_log2 = (float)((double)qk_scale * 1.4426950408889634);
  if (!(qk_scale > 0.0f && scale_log2 < INFINITY)) return Q3_ERR_SHAPE;
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
  // (packed rows, rounded up to a tile, stay below 2^31)
  if (o->rows < rows || rows > 0x7fffff00u / 16 || n_seqs > 0x7ffffffeu) return Q3_ERR_SHAPE;
  if (rows == 0 || n_seqs == 0) return Q3_OK;
  if (max_rows == 0) return Q3_ERR_SHAPE;
  const uint32_t max_kv = max_pages * kv->page_tokens;
  const chunk::Plan c =
      chunk::make_plan(rows, n_seqs, max_rows, max_kv, heads, kv_heads, head_dim);
  if (c.few_ctas > 0x7fffffff / chunk::WARPS || c.tiles * kv_heads > 0x7fffffff ||
      static_cast<uint64_t>(n_seqs) * max_kv > 0x7fffffffull * 16)
    return Q3_ERR_SHAPE;
  if (c.bytes) {
    if (!workspace) return Q3_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return Q3_ERR_ALIGN;
    if (workspace_bytes < c.bytes) return Q3_ERR_CAPACITY;
  }
  chunk::Args p{};
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
  p.scale_log2 = scale_log2;
  p.page_shift = (p.page_tokens & (p.page_tokens - 1)) ? -1 : __builtin_ctz(p.page_tokens);
  p.whole_blocks = p.page_tokens % chunk::KB == 0;
  p.few_rows = c.few_rows;
  cudaStream_t s = (cudaStream_t)stream;
  timer_begin(TIMER_ATTENTION, s);
  int st = Q3_OK;
  float *ws = static_cast<float *>(workspace);
  if (c.tiles) {
    chunk::Args t = p;
    t.splits = c.splits;
    t.tiles = static_cast<int>(c.tiles);
    t.part_o = ws + c.few_slots * (head_dim + 2);
    t.part_ml = t.part_o + static_cast<size_t>(c.splits) * c.tiles * kv_heads * chunk::TC_ROWS * head_dim;
    st = head_dim == 128 ? launch_many<128>(t, c.packed, s) : launch_many<64>(t, c.packed, s);
  }
  if (st == Q3_OK) {
    p.row_shift = c.nt == 1 ? 3 : 4;
    p.whole = c.whole;
    p.min_units = c.min_units;
    p.tiles = static_cast<int>(c.few_tiles);
    p.part_o = ws;
    p.part_ml = ws + c.few_slots * head_dim;
    const bool beside = c.tiles && c.splits == 1;   // the kernel before is the many-row one
    const int ctas = static_cast<int>(c.few_ctas);
    st = head_dim == 128 ? (c.nt == 1 ? launch_few<128, 1>(p, c.packed, ctas, beside, s)
                                      : launch_few<128, 2>(p, c.packed, ctas, beside, s))
                         : (c.nt == 1 ? launch_few<64, 1>(p, c.packed, ctas, beside, s)
                                      : launch_few<64, 2>(p, c.packed, ctas, beside, s));
  }
  timer_end(TIMER_ATTENTION, s);
  return st;
}
