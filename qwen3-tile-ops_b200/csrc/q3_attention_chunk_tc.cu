// Attention of a ragged batch over the paged int8 cache, sequences with many new
// rows, on the 5th-generation tensor cores (the formulas: q3_attention_chunk.cu).
//
// CTA = (sequence, 256 packed rows, KV head, part of the keys); packed row m is
// head m % group of new row m / group, so a KV head is read once for its whole
// group.  Two 128-row tiles of scores by halves of a key tile (128 rows x 64 keys), two
// halves each in TMEM: while the rows turn one into weights, the tensor cores use
// the weights of another and form the scores after it.
//   warps 0-15   rows: eight warps a tile, two a TMEM lane quadrant, 16 rows each
//   warps 16-23  codes of K and V from global memory, widened to f16 (exact), into a
//                ring of three operand tiles in the 128-byte-swizzled layout
//   warp 24      page lookups, the keys' scales: ks qk_scale log2 e (2^-10), log2 vs, 2^-7 / vs
//   warp 25      issues the products: S = Q K8^T (both operands in shared
//                memory), O += P V8 (P in TMEM, over its scores)
// The loads are plain ones because each code passes through registers on its
// way (the tensor cores take no f16 x int8); rows of pages of any length then need
// no tile shape of their own.
//
// 2 x 4096 rows behind 4096 tokens, 16 heads over 8: 503 us, 820 TFLOP/s, four sets of inputs (over L2) in turn
// in a graph (mma.sync for the same rows: 5.4 ms); with int8 output 514, not causal 691.
// A key tile takes 2.8 us for the 256 rows, of which the tensor cores need 1.5: the row warps' issue
// slots and the widening are the bound (385 us with rows that do nothing), and a CTA takes about
// 10 us to start and end.  Sixteen row warps hold 64 keys of 16 rows each in registers (4 bytes a thread
// spill since the sums are folded); 256 rows share one widening of K and V.
#include <atomic>

#include "q3_attention_chunk.h"
#include "q3_tc.cuh"

namespace q3 {

static __device__ unsigned int g_chunk_tc_error = 0;

int chunk_tc_device_status_take() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_chunk_tc_error, sizeof v) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_chunk_tc_error, &zero, sizeof zero);
  return static_cast<int>(v);
}

namespace chunk {

using namespace tcx;

constexpr unsigned kErrWait = 1u << 18;
constexpr int ROW_WARPS = 16, LOADERS = 8;
constexpr int INFO_WARP = ROW_WARPS + LOADERS, MMA_WARP = INFO_WARP + 1;
constexpr int TC_THREADS = 896;                    // whole warpgroups: two warps idle
constexpr int RING = 3;                            // operand tiles K0, V0, K1, V1, ...
constexpr int RAW = 3;                             // their codes, loaded or on the way
constexpr int INFO = 4;                            // key tiles whose places and scales are known
constexpr float BF16_UP = 1024.0f;                 // on bf16 queries
constexpr int TMEM_O = 256;                        // S (and P) of tile t at 128 t, O at 256 + 128 t

template <int HD>
struct TcSmem {
  alignas(1024) uint8_t q[2][128 * HD * 2];        // [64-column half][row][128 bytes], swizzled
  alignas(1024) uint8_t kv[RING][TC_KEYS * HD * 2];// [64-column half][key][128 bytes], swizzled
  alignas(16) uint4 raw[RAW][TC_KEYS * HD / 16];   // in the order of the code threads
  // scales in the order a row thread reads them: 16 keys 16k .. lie as [t4][keys 2 t4, 2 t4 + 1,
  // 8 + 2 t4, 8 + 2 t4 + 1]
  alignas(16) float ks[INFO][TC_KEYS], lv[INFO][TC_KEYS], rv[INFO][TC_KEYS];
  long long place[INFO][TC_KEYS];                  // byte offset of a key's row in the pool, or -1
  float a[TC_ROWS], l[TC_ROWS], m[TC_ROWS], fold_m[TC_ROWS];
  unsigned long long full[RING], empty[RING], place_full[INFO], info_full[INFO], info_empty[INFO];
  unsigned long long s_full[2][2], p_full[2][2], o_full;   // [row tile][half & 1]
  uint32_t tmem;
  int abort;
  int seq, tile;                                   // this CTA's, from the lookup
};

// Bounded wait for the phase with parity par (about a second, or until another thread gave up); false:
// it has not come, and what it stands for must not be used as an address
__device__ __forceinline__ bool wait_bar(unsigned long long *b, uint32_t par, int *abort) {
  const uint32_t at = su32(b);
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(at), "r"(par)
        : "memory");
    if (ok) return true;
    if ((it & 63) == 0) {
      if (*reinterpret_cast<volatile int *>(abort)) return false;
      const uint64_t t = gtime();
      if (t0 == 0) t0 = t;
      else if (t - t0 > 1000000000ull) break;
    }
  }
  atomicOr(&g_chunk_tc_error, kErrWait);
  *reinterpret_cast<volatile int *>(abort) = 1;
  return false;
}

// kind::f16 with float32 sums: f16 x f16, M = 128, N = n; b_mn: B is MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// 128-byte swizzle, MN-major, two 64-column atoms side by side `lbo` bytes apart
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr, uint32_t lbo) {
  uint64_t d = (saddr & 0x3FFFFu) >> 4;
  d |= static_cast<uint64_t>(lbo >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}
// 32 columns of 16 TMEM lanes as fragments: v[4i], v[4i+1] row lane / 4 and columns 8i + 2 (lane % 4),
// + 1; v[4i+2], v[4i+3] row lane / 4 + 8
__device__ __forceinline__ void tm_ld(uint32_t at, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15},"
      " [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(at));
}
__device__ __forceinline__ void tm_st(uint32_t at, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          at),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
      "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
// 32 columns of 16 lanes: v[2i] row lane / 4, column 4i + lane % 4; v[2i+1] row lane / 4 + 8
__device__ __forceinline__ void tm_st_p(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// 32 columns of one row (lane)
__device__ __forceinline__ void tm_ld_row(uint32_t at, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
        "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(at));
}
// after tcgen05.wait::ld: no use of v moves above it
__device__ __forceinline__ void landed(float (&v)[16]) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                 "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
__device__ __forceinline__ void landed(float (&v)[32]) {
  landed(reinterpret_cast<float(&)[16]>(v[0]));
  landed(reinterpret_cast<float(&)[16]>(v[16]));
}
// two float32 at once
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void un(F2 x, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x.v));
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Half a key tile (64 keys) for 16 rows of a warp, a thread holding rows e = 0, 1 (lane / 4 and + 8) and
// columns 8i + 2 (lane % 4), + 1: scores at `st` to weights in their place.  ks holds ks qk_scale
// log2 e; UNIT: a = 1 in all rows.  The reference of a row's weights moves only when a weight
// outgrows it by 2^kRefMove, which a vote tells, so no row maximum is formed otherwise; then the sums at
// `ot` are rescaled, once the products before this half's are in (`next`, the barrier of the next
// half's scores, which follow them, with parity par; par < 0: there are none).
template <int HD, bool MASK, bool UNIT>
__device__ __forceinline__ void rows16(const float *ks, const float *lv, const float *rv, uint32_t st,
                                       uint32_t ot, unsigned long long *next, int par, int *abort,
                                       const float (&a)[2], float (&mref)[2], float (&l)[2],
                                       const int (&pos)[2], int key0, int causal, int window) {
  float x[2][16];
  tm_ld(st, x[0]);
  tm_ld(st + 32, x[1]);
  tmem_wait_ld();
  landed(x[0]);
  landed(x[1]);
  const F2 a0 = f2(a[0], a[0]), a1 = f2(a[1], a[1]);
  float b0 = mref[0] == kNegInf ? 0.0f : -mref[0], b1 = mref[1] == kNegInf ? 0.0f : -mref[1];
  const F2 n0 = f2(b0, b0), n1 = f2(b1, b1);
  float mx0 = kNegInf, mx1 = kNegInf;
#pragma unroll
  for (int k = 0; k < 4; ++k) {                    // 16 keys: column groups 2k and 2k + 1
    const float4 kk = *reinterpret_cast<const float4 *>(ks + k * 16);
    const float4 ll = *reinterpret_cast<const float4 *>(lv + k * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float *y = &x[k >> 1][((k & 1) * 2 + h) * 4];
      const F2 k2 = h ? f2(kk.z, kk.w) : f2(kk.x, kk.y), l2 = h ? f2(ll.z, ll.w) : f2(ll.x, ll.y);
      if (UNIT) {
        un(add2(fma2(f2(y[0], y[1]), k2, l2), n0), y[0], y[1]);
        un(add2(fma2(f2(y[2], y[3]), k2, l2), n1), y[2], y[3]);
      } else {
        un(add2(fma2(mul2(f2(y[0], y[1]), k2), a0, l2), n0), y[0], y[1]);
        un(add2(fma2(mul2(f2(y[2], y[3]), k2), a1, l2), n1), y[2], y[3]);
      }
      if (MASK) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + k * 16 + h * 8 + (i & 1), at = pos[i >> 1];
          const bool hide = (causal && key > at) || (window > 0 && key <= at - window);
          y[i] = hide ? kNegInf : y[i];
        }
      }
      mx0 = max3(mx0, y[0], y[1]);
      mx1 = max3(mx1, y[2], y[3]);
    }
  }
  const bool grow = fmaxf(mx0, mx1) > kRefMove || mref[0] == kNegInf || mref[1] == kNegInf;
  if (__any_sync(0xffffffffu, grow)) {
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    // maxima relative to the old references (0 where there was none yet)
    const bool g0 = mx0 > (mref[0] == kNegInf ? kNegInf : kRefMove);
    const bool g1 = mx1 > (mref[1] == kNegInf ? kNegInf : kRefMove);
    const float u0 = g0 ? __fsub_rn(kRefBelow, mx0) : 0.0f, u1 = g1 ? __fsub_rn(kRefBelow, mx1) : 0.0f;
    // (without a reference all sums are still zero)
    const float r0 = mref[0] == kNegInf ? 1.0f : ex2(u0), r1 = mref[1] == kNegInf ? 1.0f : ex2(u1);
    b0 = __fadd_rn(b0, u0);
    b1 = __fadd_rn(b1, u1);
    mref[0] = g0 ? -b0 : mref[0];
    mref[1] = g1 ? -b1 : mref[1];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i >> 4][i & 15] = __fadd_rn(x[i >> 4][i & 15], (i & 2) ? u1 : u0);
    l[0] = __fmul_rn(l[0], r0);
    l[1] = __fmul_rn(l[1], r1);
    if (par >= 0) {
      wait_bar(next, par, abort);
      __syncwarp();
      fence_after();
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float o[16];
        tm_ld(ot + c * 32, o);
        tmem_wait_ld();
        landed(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __fmul_rn(o[i], (i & 2) ? r1 : r0);
        tm_st(ot + c * 32, o);
      }
    }
  }
  F2 s0 = f2(0.0f, 0.0f), s1 = s0;
  uint32_t w[16];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float4 rr = *reinterpret_cast<const float4 *>(rv + k * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float *y = &x[k >> 1][((k & 1) * 2 + h) * 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = ex2(y[i]);
      const F2 r2 = h ? f2(rr.z, rr.w) : f2(rr.x, rr.y);
      s0 = fma2(f2(y[0], y[1]), r2, s0);
      s1 = fma2(f2(y[2], y[3]), r2, s1);
      w[(k * 2 + h) * 2] = pack_f16(y[0], y[1]);
      w[(k * 2 + h) * 2 + 1] = pack_f16(y[2], y[3]);
    }
  }
  tm_st_p(st, w);
  float u, v;
  un(s0, u, v);
  l[0] = __fadd_rn(l[0], __fadd_rn(u, v));
  un(s1, u, v);
  l[1] = __fadd_rn(l[1], __fadd_rn(u, v));
}

// The sums at `ot` of 16 rows of a warp (a thread: rows e = 0, 1, as in rows16) to the float32 sums of
// these rows, `to`, which are relative to the reference *from; first: there are none yet.  `next`, par: as
// there.  The products after it start from zero.
template <int HD>
__device__ __forceinline__ void fold16(uint32_t ot, float *const (&to)[2], float *const (&from)[2], bool first,
                                       unsigned long long *next, int par, int *abort,
                                       const float (&mref)[2]) {
  wait_bar(next, par, abort);
  __syncwarp();
  fence_after();
  float f[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float was = first ? kNegInf : *from[e];
    f[e] = was == kNegInf ? 0.0f : ex2(__fsub_rn(was, mref[e]));
  }
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 2; ++e) *from[e] = mref[e];   // (four lanes, the same value)
#pragma unroll 1
  for (int c = 0; c < HD / 32; ++c) {
    float o[16];
    float2 x[8];                                     // all loads before the stores
#pragma unroll
    for (int i = 0; i < 8; ++i) {                    // (no such row: null)
      x[i] = make_float2(0.0f, 0.0f);
      if (!first && to[i & 1]) x[i] = *reinterpret_cast<const float2 *>(to[i & 1] + c * 32 + (i >> 1) * 8);
    }
    __syncwarp();
    tm_ld(ot + c * 32, o);
    tmem_wait_ld();
    landed(o);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = __fmaf_rn(x[i].x, f[i & 1], o[2 * i]), b = __fmaf_rn(x[i].y, f[i & 1], o[2 * i + 1]);
      if (to[i & 1]) *reinterpret_cast<float2 *>(to[i & 1] + c * 32 + (i >> 1) * 8) = make_float2(a, b);
    }
    __syncwarp();
  }
}

__device__ __forceinline__ bool elect_one() {   // one lane of the converged warp
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}
// the row warps and the MMA warp: queries staged, TMEM allocated
__device__ __forceinline__ void start_sync() {
  asm volatile("bar.sync 3, %0;" ::"n"((ROW_WARPS + 1) * 32) : "memory");
}
__device__ __forceinline__ void asm_less_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
}

template <int HD>
__global__ void __launch_bounds__(TC_THREADS, 1) k_attn_tc(const Args p) {
  constexpr int HALVES = HD / 64;
  constexpr int HALF_BYTES = 128 * 128;            // 128 rows (or keys) of 64 f16
  constexpr uint32_t ID_S = idesc_f16(64, false), ID_O = idesc_f16(HD, true);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (an offset, not a rounded address: accesses stay shared-memory accesses)
  TcSmem<HD> &sm = *reinterpret_cast<TcSmem<HD> *>(smem_raw + ((0u - su32(smem_raw)) & 1023u));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // KV heads first: they share the tile's row arrays, and heavy tiles of a sequence start together
  const int kvh = blockIdx.x % p.kv_heads, tile_id = blockIdx.x / p.kv_heads;

  pdl_trigger();   // the few-row kernel may fill the SMs that this grid leaves
  if (warp == 0) {
    unsigned err = 0;
    int tile;
    const int s = find_tile(p, tile_id, lane, &err, tile);
    if (lane == 0) {
      sm.seq = s;
      sm.tile = tile;
      sm.abort = 0;
      for (int i = 0; i < RING; ++i) {
        mbar_init(&sm.full[i], LOADERS);
        mbar_init(&sm.empty[i], 1);
      }
      for (int i = 0; i < INFO; ++i) {
        mbar_init(&sm.place_full[i], 1);
        mbar_init(&sm.info_full[i], 1);
        mbar_init(&sm.info_empty[i], LOADERS + ROW_WARPS);
      }
      for (int i = 0; i < 2; ++i) {
        for (int b = 0; b < 2; ++b) {
          mbar_init(&sm.s_full[i][b], 1);
          mbar_init(&sm.p_full[i][b], ROW_WARPS / 2);
        }
      }
      mbar_init(&sm.o_full, 1);
      mbar_init_fence();
    }
    if (blockIdx.x == 0 && blockIdx.z == 0) {   // refusals, once a launch
      for (int x = lane; x < p.n_seqs; x += 32) load_seq(p, x, &err);
      if (err) atomicOr(&g_chunk_tc_error, err);
    }
  }
  __syncthreads();
  const int s = sm.seq;
  if (s < 0) return;
  unsigned none = 0;
  const Seq q = load_seq(p, s, &none);
  const int packed = q.n * p.group, m0 = sm.tile * TC_ROWS;
  const int rows = min(TC_ROWS, packed - m0);
  // packed row m0 + m: token t0 + (o0 + m) / group, head (o0 + m) % group; the quotient by a 16-bit
  // reciprocal is exact for o0 + m < 272 and group <= 16
  const int t0 = m0 / p.group, o0 = m0 - t0 * p.group;
  const uint32_t magic = (65535u + p.group) / p.group;
  auto token = [&](int m, int &g) {
    const int x = o0 + m, y = static_cast<int>((x * magic) >> 16);
    g = x - y * p.group;
    return t0 + y;
  };
  // key tiles [z0, z0 + nj) of this CTA; row tile t needs the first ht[t] of their halves
  int z0, nj, ht[2];
  {
    const int pf = q.pos0 + m0 / p.group, pl = q.pos0 + (m0 + rows - 1) / p.group;
    int lo, hi, z1;
    key_range(p, q, pf, pl, lo, hi);
    split_range(lo / TC_KEYS, (hi + TC_KEYS - 1) / TC_KEYS, p.splits, blockIdx.z, z0, z1);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int last = min(rows, 128 * (t + 1)) - 1;
      const int h = p.causal ? q.pos0 + (m0 + last) / p.group + 1 : q.kv;
      const int n = (h + 63) / 64 - 2 * z0;
      ht[t] = rows > 128 * t ? max(0, min(2 * (z1 - z0), n)) : 0;
    }
    nj = (max(ht[0], ht[1]) + 1) / 2;
  }

  // registers move from the other warps to those of the rows: 4 x 128 x 88 + 3 x 128 x 48 is
  // within the launch's 896 x 72
  if (warp < ROW_WARPS) {
    // ------------------------------------------------------------------ rows
    asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    // ---- queries as f16 in the operand layout and each row's a: 8 columns a thread at a time
    {
      constexpr int G8 = HD / 8, EACH = TC_ROWS * G8 / (ROW_WARPS * 32);
      uint4 raw[EACH];
      float qs[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int id = i * ROW_WARPS * 32 + threadIdx.x, m = id / G8;
        raw[i] = make_uint4(0, 0, 0, 0);
        qs[i] = 0.0f;
        if (m < rows) {
          int hg;
          const long r = q.first + token(m, hg);
          const int h = kvh * p.group + hg;
          const char *qp = p.q + r * p.q_rb;
          const long col = static_cast<long>(h) * HD + (id % G8) * 8;
          qs[i] = 1.0f;
          if (p.q_dt == Q3_DT_I8) {
            *reinterpret_cast<uint2 *>(&raw[i]) = *reinterpret_cast<const uint2 *>(qp + col);
            qs[i] = reinterpret_cast<const float *>(p.qs + r * p.qs_rb)[h];
          } else {
            raw[i] = *reinterpret_cast<const uint4 *>(qp + col * 2);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int id = i * ROW_WARPS * 32 + threadIdx.x, m = id / G8, d8 = id % G8;
        uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        if (p.q_dt == Q3_DT_I8) {
          const uint32_t lo = w[0] ^ 0x80808080u, hi = w[1] ^ 0x80808080u;
          w[0] = f16_pair(lo, 0x4140), w[1] = f16_pair(lo, 0x4342);
          w[2] = f16_pair(hi, 0x4140), w[3] = f16_pair(hi, 0x4342);
        } else if (p.q_dt == Q3_DT_BF16) {
          float mx = 0.0f, up = 1.0f, down = 1.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[k] << 16)),
                                 fabsf(__uint_as_float(w[k] & 0xffff0000u))));
#pragma unroll
          for (int o = 1; o < G8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          // rows of usual size, [2^-3, 2^5), take 2^10, which the keys' scales undo (a = 1 then): exact
          // in f16 down to 2^-24 of the maximum, as others are with a power of their own
          if (mx != 0.0f && !(mx >= 0.125f && mx < 32.0f)) {
            bf16_scale(mx, up, down);
            down = __fmul_rn(down, BF16_UP);
          } else {
            up = BF16_UP;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = pack_f16(__fmul_rn(__uint_as_float(w[k] << 16), up),
                            __fmul_rn(__uint_as_float(w[k] & 0xffff0000u), up));
          qs[i] = __fmul_rn(qs[i], down);
        }
        const int r = m & 127;
        *reinterpret_cast<uint4 *>(sm.q[m >> 7] + (d8 / 8) * HALF_BYTES + r * 128 +
                                   (((d8 % 8) ^ (r & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        if (d8 == 0) sm.a[m] = qs[i];
      }
    }
    fence_proxy_async();
    start_sync();
    fence_after();
    const uint32_t tmem = sm.tmem;
    // warp: tile t, lane quadrant qd, its 16 rows ps; thread: rows rb + 8 e + g
    const int t = warp >> 3, ps = (warp >> 2) & 1, qd = warp & 3, g = lane >> 2, t4 = lane & 3;
    float a[2], mref[2], l[2];
    int pos[2];
    const int rb = t * 128 + qd * 32 + ps * 16;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = rb + 8 * e + g;
      a[e] = sm.a[m];
      int hg;
      pos[e] = q.pos0 + token(min(m, rows - 1), hg);
      mref[e] = kNegInf;
      l[e] = 0.0f;
    }
    const bool unit = __all_sync(0xffffffffu, a[0] == 1.0f && a[1] == 1.0f);
    int unused;
    const int pmin = q.pos0 + token(min(rb, rows - 1), unused);
    const int pmax = q.pos0 + token(min(rb + 15, rows - 1), unused);
    const int mine = t ? ht[1] : ht[0];
    const uint32_t st = tmem + (static_cast<uint32_t>(qd * 32 + ps * 16) << 16) + t * 128;
    // float32 sums of packed row x of the tile
    auto sums_of = [&](int x) -> float * {
      int hx;
      const long r = q.first + token(x, hx);
      const long at = p.splits > 1 ? (static_cast<long>(blockIdx.x) * p.splits + blockIdx.z) * TC_ROWS + x
                                   : r * p.heads + kvh * p.group + hx;
      return p.part_o + at * HD;
    };
    for (int j0 = 0; j0 < nj; j0 += FOLD_TILES) {
      if (j0 && 2 * j0 < mine) {
        const int m = rb + g;
        float *const to[2] = {m < rows ? sums_of(m) + t4 * 2 : nullptr,
                              m + 8 < rows ? sums_of(m + 8) + t4 * 2 : nullptr};
        float *const from[2] = {sm.fold_m + m, sm.fold_m + m + 8};
        fold16<HD>(st + TMEM_O, to, from, j0 == FOLD_TILES, &sm.s_full[t][1], j0 & 1, &sm.abort, mref);
      }
#pragma unroll 1
      for (int j = j0; j < min(nj, j0 + FOLD_TILES); ++j) {
        const int in = j % INFO;
        wait_bar(&sm.info_full[in], (j / INFO) & 1, &sm.abort);
        const float *ks = sm.ks[in] + t4 * 4, *lv = sm.lv[in] + t4 * 4, *rv = sm.rv[in] + t4 * 4;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int h = 2 * j + b;
          if (h < mine) {
            wait_bar(&sm.s_full[t][b], j & 1, &sm.abort);
            __syncwarp();
            fence_after();
            const int key0 = z0 * TC_KEYS + h * 64, at = b * 64, par = h ? ((h + 1) >> 1) & 1 : -1;
            const bool masked = (p.causal && key0 + 63 > pmin) || (p.window > 0 && key0 <= pmax - p.window);
            if (masked)
              rows16<HD, true, false>(ks + at, lv + at, rv + at, st + at, st + TMEM_O,
                                      &sm.s_full[t][b ^ 1], par, &sm.abort, a, mref, l, pos,
                                      key0 + t4 * 2, p.causal, p.window);
            else if (unit)
              rows16<HD, false, true>(ks + at, lv + at, rv + at, st + at, st + TMEM_O,
                                      &sm.s_full[t][b ^ 1], par, &sm.abort, a, mref, l, pos,
                                      key0 + t4 * 2, p.causal, p.window);
            else
              rows16<HD, false, false>(ks + at, lv + at, rv + at, st + at, st + TMEM_O,
                                       &sm.s_full[t][b ^ 1], par, &sm.abort, a, mref, l, pos,
                                       key0 + t4 * 2, p.causal, p.window);
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_full[t][b]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.info_empty[in]);
      }
    }
    // ---- sums of the rows; then each thread half the columns of its own row
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float y = l[e];
      y = __fadd_rn(y, __shfl_xor_sync(0xffffffffu, y, 1));
      y = __fadd_rn(y, __shfl_xor_sync(0xffffffffu, y, 2));
      if (t4 == 0) {
        sm.l[rb + 8 * e + g] = y;
        sm.m[rb + 8 * e + g] = mref[e];
      }
    }
    asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");   // the eight warps of the tile
    // (the float32 sums of other warps' threads are visible behind it, too)
    if (nj > 0) wait_bar(&sm.o_full, 0, &sm.abort);
    fence_after();
    const int m = t * 128 + qd * 32 + lane;
    const bool have = m < rows;
    int hg;
    const long r = q.first + token(min(m, rows - 1), hg);
    const int h = kvh * p.group + hg;
    const uint32_t src = tmem + (static_cast<uint32_t>(qd * 32) << 16) + TMEM_O + t * 128;
    const float lsum = sm.l[m];
    // 32 columns of this lane's row
    const bool folded = mine > 2 * FOLD_TILES && have;
    const float ff = !folded || sm.fold_m[m] == kNegInf ? 0.0f : ex2(__fsub_rn(sm.fold_m[m], sm.m[m]));
    auto sums = [&](int c, float (&o)[32]) {
      tm_ld_row(src + c * 32, o);
      tmem_wait_ld();
      landed(o);
      if (folded) {
        const float4 *at = reinterpret_cast<const float4 *>(sums_of(m) + c * 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float4 x;   // (one at a time: 32 more registers are not there)
          asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];"
                       : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                       : "l"(at + i)
                       : "memory");
          o[4 * i] = __fmaf_rn(x.x, ff, o[4 * i]);
          o[4 * i + 1] = __fmaf_rn(x.y, ff, o[4 * i + 1]);
          o[4 * i + 2] = __fmaf_rn(x.z, ff, o[4 * i + 2]);
          o[4 * i + 3] = __fmaf_rn(x.w, ff, o[4 * i + 3]);
        }
      }
      __syncwarp();
    };
    // this warp's columns, 32 at a time (its chunks ps * OC ..), go through its part of the query
    // tile, which the products no longer read: a row's pieces then leave as whole lines
    constexpr int OC = HD / 64;
    uint8_t *stage = sm.q[0] + warp * 4096;        // (HD = 64: on into the ring, which is idle too)
    const int nr = min(32, rows - (t * 128 + qd * 32));
    auto flush = [&](const int bytes, char *to) {   // `bytes` a row; `to`: where this lane's row goes
      __syncwarp();
      const int per = bytes / 16;
      const unsigned long long mine_ = reinterpret_cast<unsigned long long>(to);
#pragma unroll 4
      for (int k = lane; k < 32 * per; k += 32) {
        const int row = k / per, c = k % per;
        const unsigned long long at = __shfl_sync(0xffffffffu, mine_, row);
        if (row < nr)
          *reinterpret_cast<uint4 *>(at + c * 16) =
              *reinterpret_cast<const uint4 *>(stage + row * bytes + ((c ^ (row & (per - 1))) * 16));
      }
      __syncwarp();
    };
    auto put = [&](const int bytes, const int c, const uint4 x) {   // 16-byte piece c of this lane's row
      *reinterpret_cast<uint4 *>(stage + lane * bytes + ((c ^ (lane & (bytes / 16 - 1))) * 16)) = x;
    };
    if (p.splits > 1) {
      const long at = (static_cast<long>(blockIdx.x) * p.splits + blockIdx.z) * TC_ROWS + m;
      if (mine > 0) {
#pragma unroll 1
        for (int c = ps * OC; c < ps * OC + OC; ++c) {
          Elems<float, 32> o;
          sums(c, o.e);
#pragma unroll
          for (int i = 0; i < 8; ++i) put(128, i, o.v[i]);
          flush(128, reinterpret_cast<char *>(p.part_o + at * HD + c * 32));
        }
      }
      if (have && ps == 0) {
        p.part_ml[at * 2] = mine > 0 ? sm.m[m] : kNegInf;
        p.part_ml[at * 2 + 1] = mine > 0 ? lsum : 0.0f;
      }
    } else if (mine > 0) {
      const float inv = inverse_sum(lsum);
      const bool i8 = p.o_dt == Q3_DT_I8;
      const int es = i8 ? 1 : 2;
      char *out = p.o + r * p.o_rb + (static_cast<long>(h) * HD + ps * OC * 32) * es;
      float scale = 0.0f;
      if (i8) {
        float mx = 0.0f;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          float o[32];
          sums(c, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fabsf(__fmul_rn(o[i], inv)));
        }
        scale = __fmul_rn(mx, kInv127);
        if (have && ps == 0) reinterpret_cast<float *>(p.os + r * p.os_rb)[h] = scale;
      }
#pragma unroll 1
      for (int c = 0; c < OC; ++c) {
        float o[32];
        sums(ps * OC + c, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __fmul_rn(o[i], inv);
        if (i8) {
          uint32_t w[8];
          quant_pack_absmax<32>(o, scale, w);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            put(32 * OC, c * 2 + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
        } else {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (p.o_dt == Q3_DT_F16) {
              w[i] = pack_f16(o[2 * i], o[2 * i + 1]);
            } else {
              const __nv_bfloat162 v = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
              w[i] = *reinterpret_cast<const uint32_t *>(&v);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            put(64 * OC, c * 4 + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
        }
      }
      flush(32 * OC * es, out);
    }
  } else if (asm_less_registers(), warp < INFO_WARP) {
    // ------------------------------------------------------------------ codes of K and V
    // Operand tile `item` (K and V in turn): a warp takes WR key rows in chunks of CR rows, 16 bytes
    // a lane, copied into places of its own (cp.async, RAW items ahead: the latency of L2 is
    // longer than an item takes), then widened into the operand layout.
    constexpr int WR = TC_KEYS / LOADERS, CR = HD == 128 ? 4 : 8, CHUNKS = WR / CR;
    const int lw = warp - ROW_WARPS, items = 2 * nj;
    // eight lanes take 4 chunks of two rows: their f16 chunks then lie in 8 different places of a
    // 128-byte line
    const int rowl = HD == 128 ? 2 * (lane >> 4) + ((lane >> 2) & 1) : lane >> 2;
    const int c = HD == 128 ? ((lane >> 3) & 1) * 4 + (lane & 3) : lane & 3;
    const long kcol = static_cast<long>(kvh) * HD + c * 16;
    const int row0 = lw * WR + rowl;
    const uint32_t to = static_cast<uint32_t>((c >> 2) * HALF_BYTES + row0 * 128);
    const int ch = (c & 3) * 2;
    uint4 *raw = sm.raw[0] + lw * 32 + lane;
    auto request = [&](int item) {
      if (item < items) {
        const int j = item >> 1, in = j % INFO;
        const bool known = wait_bar(&sm.place_full[in], (j / INFO) & 1, &sm.abort);
        const char *from = ((item & 1) ? p.v : p.k) + kcol;
        const uint32_t dst = su32(raw + (item % RAW) * (TC_KEYS * HD / 16));
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const long long at = known ? sm.place[in][row0 + i * CR] : -1;
          cp16(dst + i * LOADERS * 512, at >= 0 ? from + at : p.k, at >= 0);
        }
        __syncwarp();
        if (lane == 0 && (item & 1)) mbar_arrive(&sm.info_empty[in]);   // its places are read
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < RAW; ++i) request(i);
    for (int item = 0; item < items; ++item) {
      const int slot = item % RING;
      if (item >= RING) wait_bar(&sm.empty[slot], ((item / RING) - 1) & 1, &sm.abort);
      asm volatile("cp.async.wait_group %0;" ::"n"(RAW - 1) : "memory");
      uint8_t *dst = sm.kv[slot] + to;
      const uint4 *src = raw + (item % RAW) * (TC_KEYS * HD / 16);
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const uint4 x = src[i * LOADERS * 32];
        const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u,
                               x.w ^ 0x80808080u};
        uint4 lo, hi;
        lo.x = f16_pair(w[0], 0x4140), lo.y = f16_pair(w[0], 0x4342);
        lo.z = f16_pair(w[1], 0x4140), lo.w = f16_pair(w[1], 0x4342);
        hi.x = f16_pair(w[2], 0x4140), hi.y = f16_pair(w[2], 0x4342);
        hi.z = f16_pair(w[3], 0x4140), hi.w = f16_pair(w[3], 0x4342);
        const int r = row0 + i * CR;
        *reinterpret_cast<uint4 *>(dst + i * CR * 128 + ((ch ^ (r & 7)) * 16)) = lo;
        *reinterpret_cast<uint4 *>(dst + i * CR * 128 + (((ch + 1) ^ (r & 7)) * 16)) = hi;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.full[slot]);
      request(item + RAW);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == INFO_WARP) {
    // ------------------------------------------------------------------ places and scales
    // A lane has keys i*32 + lane of a tile.  Pages are looked up two tiles ahead; a tile's places
    // are published, and its scales requested, one tile ahead.
    const uint16_t *table = p.tables + static_cast<long>(s) * p.max_pages;
    const float scale = p.q_dt == Q3_DT_BF16 ? __fmul_rn(p.scale_log2, 1.0f / BF16_UP) : p.scale_log2;
    auto page_of = [&](int j, int (&pg)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = (z0 + j) * TC_KEYS + i * 32 + lane;
        pg[i] = j < nj && key < q.kv ? table[page_index(p, key)] : -1;
      }
    };
    struct Scales {
      bool have[4];
      float ks[4], vs[4];
    };
    auto publish = [&](int j, const int (&pg)[4], Scales &k) {
      if (j >= nj) return;
      const int in = j % INFO;
      if (j >= INFO) wait_bar(&sm.info_empty[in], ((j / INFO) - 1) & 1, &sm.abort);
      size_t so[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t key = (z0 + j) * TC_KEYS + i * 32 + lane, slot = page_slot(p, key);
        k.have[i] = pg[i] >= 0 && static_cast<uint32_t>(pg[i]) < p.num_pages;
        if (pg[i] >= 0 && !k.have[i]) atomicOr(&g_chunk_tc_error, kBadPage);
        sm.place[in][i * 32 + lane] = k.have[i] ? static_cast<long long>(pg[i]) * p.page_bytes +
                                                      static_cast<long long>(slot) * p.row_bytes
                                                : -1;
        so[i] = k.have[i] ? static_cast<size_t>(pg[i]) * p.scale_page_bytes +
                                static_cast<size_t>(slot) * p.scale_row_bytes + kvh * 4
                          : 0;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.place_full[in]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k.ks[i] = k.vs[i] = 0.0f;
        if (k.have[i]) {
          k.ks[i] = __ldg(reinterpret_cast<const float *>(p.ks + so[i]));
          k.vs[i] = __ldg(reinterpret_cast<const float *>(p.vs + so[i]));
        }
      }
    };
    int pg[4], pg1[4];
    Scales now;
    page_of(0, pg);
    page_of(1, pg1);
    publish(0, pg, now);
    for (int j = 0; j < nj; ++j) {
      const int in = j % INFO;
      Scales next;
      publish(j + 1, pg1, next);
      page_of(j + 2, pg1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = i * 32 + lane, k = key & 15;
        const int to = (key & ~15) + ((k & 7) >> 1) * 4 + (k >> 3) * 2 + (k & 1);
        const float v = fmaxf(now.vs[i], kVsMin);    // (NaN: fmaxf drops it ...
        sm.ks[in][to] = __fmul_rn(now.ks[i], scale);
        // ... and the rows that see it get NaN); a key that is not there: weight 0
        sm.lv[in][to] = !now.have[i] ? kNegInf : now.vs[i] != now.vs[i] ? now.vs[i] : lg2(v);
        sm.rv[in][to] = __fmul_rn(rcp(v), kSumScale);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.info_full[in]);
      now = next;
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------------ products
    tmem_alloc<512>(&sm.tmem);
    fence_before();
    start_sync();
    fence_after();
    if (elect_one()) {
      // descriptors: constant but for the start address (in 16-byte units) in the low bits
      const uint64_t qd[2] = {sdesc_sw128(su32(sm.q[0])), sdesc_sw128(su32(sm.q[1]))};
      const uint64_t kd = sdesc_sw128(su32(sm.kv[0]));
      const uint64_t vd = sdesc_mn(su32(sm.kv[0]), HALVES == 2 ? HALF_BYTES : 16);
      constexpr uint32_t SLOT = TC_KEYS * HD * 2 / 16, KEYS64 = 64 * 128 / 16;
      const uint32_t tmem = sm.tmem;
      auto scores = [&](const int t, int h) {   // S of half h = Q K8^T
        const uint64_t b = kd + static_cast<uint32_t>((h & ~1) % RING) * SLOT + (h & 1) * KEYS64;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t at = ((k / 4) * HALF_BYTES + (k % 4) * 32) / 16;
          mma_ss(tmem + t * 128 + (h & 1) * 64, qd[t] + at, b + at, ID_S, k != 0);
        }
      };
      auto values = [&](const int t, int h) {   // O += P V8 of half h
        const uint64_t b = vd + static_cast<uint32_t>((h | 1) % RING) * SLOT + (h & 1) * KEYS64;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_ts(tmem + TMEM_O + t * 128, tmem + t * 128 + (h & 1) * 64 + k * 8, b + k * (2048 / 16),
                 ID_O, h % (2 * FOLD_TILES) > 0 || k > 0);
      };
      auto ready = [&](int item) {
        wait_bar(&sm.full[item % RING], (item / RING) & 1, &sm.abort);
        fence_after();
      };
      if (nj > 0) {
        ready(0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (h < ht[t]) {
              scores(t, h);
              mma_commit(&sm.s_full[t][h]);
            }
        mma_commit(&sm.empty[0]);
      }
      for (int h = 0; h < 2 * nj; ++h) {
        const int j = h >> 1;                      // V of tile j, then K of tile j + 1
        if (!(h & 1)) ready(2 * j + 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (h < ht[t]) {
            wait_bar(&sm.p_full[t][h & 1], j & 1, &sm.abort);
            fence_after();
            values(t, h);
          }
          if (t == 0 && !(h & 1) && j + 1 < nj) ready(2 * j + 2);
          if (h < ht[t]) {
            // these scores overwrite the weights of half h: products of one thread run in order
            if (h + 2 < ht[t]) scores(t, h + 2);
            mma_commit(&sm.s_full[t][h & 1]);      // (after the last halves: their products are in)
          }
        }
        if (h & 1) {
          mma_commit(&sm.empty[(2 * j + 1) % RING]);
          if (j + 1 < nj) mma_commit(&sm.empty[(2 * j + 2) % RING]);
        }
      }
      if (nj > 0) {
        mma_commit(&sm.o_full);
        wait_bar(&sm.o_full, 0, &sm.abort);
      }
    }
    __syncwarp();
  }

  fence_before();
  __syncthreads();
  fence_after();
  if (warp == MMA_WARP) tmem_dealloc<512>(sm.tmem);
}

template <int HD>
static int launch(const Args &p, cudaStream_t s) {
  constexpr int smem = static_cast<int>(sizeof(TcSmem<HD>)) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(k_attn_tc<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      q3h::set_cuda_error(e);
      return Q3_ERR_CUDA;
    }
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  k_attn_tc<HD><<<dim3(p.tiles * p.kv_heads, 1, p.splits), TC_THREADS, smem, s>>>(p);
  return q3h::launch_status();
}

int launch_tc(const Args &p, int head_dim, cudaStream_t s) {
  return head_dim == 128 ? launch<128>(p, s) : launch<64>(p, s);
}

}  // namespace chunk
}  // namespace q3
