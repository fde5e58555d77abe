// Banded causal attention with an optional relative position bias, forward and backward.
//
// Query row i stands at position p_i = q_pos0 + i, key j at position j.
//   visible(i, j) = j <= p_i  and  j < Skv  and  (p_i - j < window  or  j < sinks)
//   x_ij = scale * q_i . k_j + table[h, bucket(p_i - j)]
//   P    = softmax of x over the visible keys (a row that sees none: P = 0)
//   O    = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P * (dP - D),  D_i = dO_i . O_i
//   dQ = scale dS K,  dK = scale dS^T Q,  dtable[h, b] = sum of dS_ij with bucket(p_i - j) = b
// Rows are kept by their maximum m and l = log2(sum 2^(x - m)), both in the base-2 exponent domain and apart
// from one another: with a bias of the type's lowest value in every place m + l would round l away.
#include "band_args.h"
#include "common.cuh"

#include <algorithm>
#include <atomic>
#include <climits>

namespace nmb {

constexpr float kBandLog2e = 1.4426950408889634f;
constexpr float kBiasLimit = 3.0e38f;  // finite biases stay finite after the change to base 2

__device__ __forceinline__ float table_at(const BandArgs& p, int h, int b) {
  const long long at = static_cast<long long>(h) * p.buckets + b;
  return p.table_fp32 ? static_cast<const float*>(p.table)[at]
                      : __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[at]);
}
// a table entry in the base-2 exponent domain; infinities and NaN stay
__device__ __forceinline__ float bias_log2(float x) {
  const float y = x * kBandLog2e;
  return isfinite(x) ? fminf(fmaxf(y, -kBiasLimit), kBiasLimit) : x;
}
__device__ __forceinline__ __nv_bfloat16* rest_row(const BandArgs& a, int b, int s, int h, int d) {
  return a.o_rest + ((static_cast<long long>(b) * a.rest_rows + s) * a.Hq + h) * d;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ T* band_row(T* ptr, const BandStride& st, int b, int s, int h) {
  return ptr + b * st.b + s * st.s + h * st.h;
}

// Division by a number that the launch fixes: multiply by a rounded-up reciprocal and shift (Granlund and Montgomery, 1994).
// All warps of a CTA work out where their next item lies, and a few divisions each of them cost an item 3000 clocks.
struct FastDiv {
  uint32_t mul, shift, d;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int quot(int n) const {  // 0 <= n < 2^31
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift);
  }
  __device__ __forceinline__ int quot(int n, int& rest) const {
    const int q = quot(n);
    rest = n - q * static_cast<int>(d);
    return q;
  }
};

// ------------------------------------------------------------- key tiles --
// The tiles of 128 keys that a tile of 128 query rows sees: [0, sink) and [lo, hi].
struct KeyTiles {
  int sink, lo, hi;
  __device__ __forceinline__ bool uses(int j) const { return j < sink || (j >= lo && j <= hi); }
  __device__ __forceinline__ int count() const { return sink + max(0, hi - lo + 1); }
};
constexpr int kNoTile = 1 << 28;

__device__ __forceinline__ KeyTiles key_tiles(const BandArgs& a, int q0) {
  KeyTiles r;
  const int pmin = a.q_pos0 + q0, pmax = a.q_pos0 + min(q0 + 128, a.Sq) - 1;
  const int first = max(0, pmin - a.window + 1), last = min(pmax, a.Skv - 1);
  const bool band = first <= last;
  r.lo = band ? first >> 7 : kNoTile;
  r.hi = band ? last >> 7 : -1;
  r.sink = min((min(a.sinks, min(pmax + 1, a.Skv)) + 127) >> 7, r.lo);
  return r;
}
// u-th tile of a list
__device__ __forceinline__ int tile_at(const KeyTiles& r, int u) { return u < r.sink ? u : r.lo + u - r.sink; }

__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// ------------------------------------------------------------------- bias --
// A head's biases by distance, in the base-2 domain, for distances -256 .. t_last + 255 (the ones that a tile whose
// smallest distance is below t_last can meet); t_last is the first distance of the last bucket.  Which bucket a distance
// falls into is worked out once per CTA.
constexpr int kLutFront = 256, kLutBack = 256;
__host__ __device__ __forceinline__ int lut_entries(int t_last) { return kLutFront + t_last + kLutBack; }

__host__ __device__ inline int lut_bytes(int t_last, int heads) { return (lut_entries(t_last) * (4 * heads + 1) + 15) / 16 * 16; }

__device__ __forceinline__ void build_bucket_map(const BandArgs& a, int t_last, uint8_t* map, int tid, int threads) {
  for (int n = tid; n < lut_entries(t_last); n += threads) {
    int lo = 0, hi = a.buckets - 1;  // the last bucket whose first distance is not beyond n
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (n - kLutFront >= a.limit[mid - 1]) lo = mid; else hi = mid - 1;
    }
    map[n] = static_cast<uint8_t>(lo);
  }
}
__device__ __forceinline__ void build_lut(const BandArgs& a, int h, int t_last, const uint8_t* map, float* lut, int tid, int threads) {
  for (int n = tid; n < lut_entries(t_last); n += threads) lut[n] = bias_log2(table_at(a, h, map[n]));
}

// ------------------------------------------------------------------ TMEM ---
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// The issuing warp runs its loops with all lanes together and lets one lane of them issue: addresses then are the same for
// the whole warp by construction, which is where the instruction wants them (uniform registers).  With the loops inside a
// branch of one lane every operand was moved there first and issuing, not the tensor core, set the pace (a step of two slots
// at d = 128: 4160 clocks to issue 32 products that take 2048).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(e));
  return e;
}
// Shared-memory operands: the low word of a descriptor (address and the stride between slabs of an MN-major operand) moves
// from product to product, the high word does not.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row stride 1024, version, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_k(uint32_t smem) { return ((smem & 0x3ffff) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t smem) { return ((smem & 0x3ffff) >> 4) | ((16384u >> 4) << 16); }

// (`one`: see commit_one)
template <bool kAccumulate>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t one) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "n"(kAccumulate ? 1 : 0), "n"(kDescHigh), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate, uint32_t one) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh), "r"(one)
      : "memory");
}
// A commit by the lanes with `one`, as a predicate instead of a branch around it.  Products and commits without branches, for
// the whole warp in one stream of instructions, took 1 to 3 percent off the forward kernel at D > 64 (one issuer, two slots) and
// added 1 to 2 percent elsewhere.
__device__ __forceinline__ void commit_one(uint64_t* bar, uint32_t one) {
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "}" ::"r"(smem_u32(bar)), "r"(one)
      : "memory");
}
// D[128 x 128] = A B^T over a depth of D, both K-major; one lane
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t one = 1) {
  mma_ss<false>(d, a_low, b_low, idesc, one);
#pragma unroll
  for (int k = 1; k < D / 16; ++k) {
    const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
    mma_ss<true>(d, a_low + off, b_low + off, idesc, one);
  }
}
// D[128 x n] (+)= A B over a depth of 16 kSteps, A bf16 in tensor memory (kPer steps side by side, the next kStride columns
// on), B MN-major; one lane
template <int kSteps, int kPer, int kStride>
__device__ __forceinline__ void mma_apply(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, bool first,
                                          uint32_t one = 1) {
  mma_ts(d, a_tmem, b_low, idesc, first ? 0u : 1u, one);
#pragma unroll
  for (int k = 1; k < kSteps; ++k) mma_ts(d, a_tmem + (k / kPer) * kStride + (k % kPer) * 8, b_low + k * (2048 >> 4), idesc, 1u, one);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Maxima that are NaN where one of the values is: a NaN among the scores of a row must not get lost.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x for two x, on the FMA pipe: x = n + f with n the nearest whole number (adding 1.5 * 2^23 leaves it in the low bits), 2^f
// by the polynomial of degree 4 with the smallest relative error on [-1/2, 1/2] (2.7e-6, found by exchange of extrema), 2^n
// added to the exponent.  x below -126 gives 2^-126.  The exponential unit does 16 a clock and SM, a tile of 128 x 128 weights
// 1024 clocks, as long as the tensor core takes for its products at d = 128; a part of the weights goes this way instead.
// A NaN comes out as 2^-126, unless kNan asks for a NaN: then 2^n is a factor, since what is added to a NaN's bits can make
// a number of it.  (Needed only where nothing else of the row's result shows the NaN.)
template <bool kNan>
__device__ __forceinline__ void exp2_pair_fma(uint64_t x2, float& y0, float& y1) {
  float x0, x1;
  unpack2(x2, x0, x1);
  const uint64_t x = kNan ? pack2(max2(x0, -126.f), max2(x1, -126.f)) : pack2(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t t = add2(x, pack2(12582912.f, 12582912.f));
  const uint64_t n = add2(t, pack2(-12582912.f, -12582912.f));
  const uint64_t f = fma2(n, pack2(-1.f, -1.f), x);
  uint64_t q = fma2(f, pack2(9.570102207362652e-3f, 9.570102207362652e-3f), pack2(5.591785907745361e-2f, 5.591785907745361e-2f));
  q = fma2(q, f, pack2(0.240247443318367f, 0.240247443318367f));
  q = fma2(q, f, pack2(0.6931217908859253f, 0.6931217908859253f));
  q = fma2(q, f, pack2(0.9999992847442627f, 0.9999992847442627f));
  float t0, t1, q0, q1;
  unpack2(t, t0, t1);
  if (kNan) {
    const uint64_t factor = pack2(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u),
                                  __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u));
    unpack2(mul2(q, factor), y0, y1);
    return;
  }
  unpack2(q, q0, q1);
  y0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23));
  y1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23));
}
// One pair in this many takes that way.
constexpr int kFmaPairs = 4;
template <bool kMix, bool kNan = false>
__device__ __forceinline__ void exp2_pair(int pair, uint64_t x2, float& y0, float& y1) {
  if (kMix && (pair % kFmaPairs) == kFmaPairs - 1) {
    exp2_pair_fma<kNan>(x2, y0, y1);
  } else {
    float x0, x1;
    unpack2(x2, x0, x1);
    y0 = ex2(x0);
    y1 = ex2(x1);
  }
}
// Weights 2^(s * mul + shift) of 32 scores, as bf16 pairs, and their sum.
template <bool kMix>
__device__ __forceinline__ void weights32(const uint32_t (&s)[32], uint64_t mul, uint64_t shift, uint64_t& sum, uint32_t (&pk)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float p0, p1;
    exp2_pair<kMix>(k, fma2(pack2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), mul, shift), p0, p1);
    sum = add2(sum, pack2(p0, p1));
    pk[k] = pack_bf16x2(p0, p1);
  }
}
// 32 bytes to a 32-byte aligned address: a whole sector per lane
__device__ __forceinline__ void st_global_32(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f,
                                             uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e),
               "r"(f), "r"(g), "r"(h)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 16 consecutive values of a row as bf16
__device__ __forceinline__ void store_bf16_16(__nv_bfloat16* dst, const uint32_t (&r)[16], float mul) {
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = pack_bf16x2(__uint_as_float(r[2 * k]) * mul, __uint_as_float(r[2 * k + 1]) * mul);
  st_global_32(dst, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Results of D = 64 leave through a swizzled tile in shared memory and one tile store: 32 bytes a lane, a line each, took an item
// 2600 clocks.  (Wider heads leave no room for the tile.)  Rows behind the last are cut off by the tensor map.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, const void* smem_src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// 16 values of row r from column c (a multiple of 16) on
__device__ __forceinline__ void stage_bf16_16(uint8_t* tile, int r, int c, const uint32_t (&v)[16], float mul) {
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = pack_bf16x2(__uint_as_float(v[2 * k]) * mul, __uint_as_float(v[2 * k + 1]) * mul);
  *reinterpret_cast<uint4*>(tile + swz128_offset(r, c / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(tile + swz128_offset(r, c / 8 + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
}
// Bounded wait: as mbar_wait, but asleep for up to kNapNs at a time after the first look.  (The first look takes about 50
// clocks, try_wait 80.)
constexpr uint32_t kNapNs = 10000;
__device__ __forceinline__ bool band_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int where) {
  if (mbar_test_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity), "r"(kNapNs)
        : "memory");
    if (done != 0) return true;
    if (*abort_flag != 0) return false;
    if (clock64() - t0 > kWaitBudgetCycles) {
      report_status(status, kMbarTimeout, where);
      *abort_flag = 1;
      return false;
    }
  }
}
// Several at once: their latencies overlap.
struct BandBar {
  uint64_t* bar;
  uint32_t parity;
};
__device__ __forceinline__ bool try_wait_all(const BandBar& a, const BandBar& b) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "and.pred p, p, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(ok)
      : "r"(smem_u32(a.bar)), "r"(a.parity), "r"(smem_u32(b.bar)), "r"(b.parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool try_wait_all(const BandBar& a, const BandBar& b, const BandBar& c) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q, r;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
      "and.pred p, p, q;\n\t"
      "and.pred p, p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(ok)
      : "r"(smem_u32(a.bar)), "r"(a.parity), "r"(smem_u32(b.bar)), "r"(b.parity), "r"(smem_u32(c.bar)), "r"(c.parity)
      : "memory");
  return ok != 0;
}
template <typename... Bars>
__device__ __forceinline__ bool band_wait_all(volatile int* abort_flag, int* status, int where, const Bars&... bars) {
  if (try_wait_all(bars...)) return true;
  return (band_wait(bars.bar, bars.parity, abort_flag, status, where) && ...);
}
// Which comes first: all of `bars` (0) or `other` (1); 2 on failure
template <class... Bars>
__device__ __forceinline__ int band_wait_first(volatile int* abort_flag, int* status, int where, BandBar other, const Bars&... bars) {
  if ((mbar_test_wait(bars.bar, bars.parity) && ...)) return 0;
  const long long t0 = clock64();
  while (true) {
    if (mbar_test_wait(other.bar, other.parity)) return 1;
    if ((mbar_test_wait(bars.bar, bars.parity) && ...)) return 0;
    if (*abort_flag != 0) return 2;
    if (clock64() - t0 > kWaitBudgetCycles) {
      report_status(status, kMbarTimeout, where);
      *abort_flag = 1;
      return 2;
    }
  }
}
// The compute warps' waits.  After one has failed the others are passed by and the loops run to their end on whatever is
// there: every warp comes to every named barrier, whichever of them gave up, and no warp waits at one for another that left.
#define NMB_BAND_WAIT(bar, parity, where)                                            \
  do {                                                                               \
    ok = ok && band_wait(bar, parity, abort_flag, a.status, where);                  \
    __syncwarp();                                                                    \
  } while (0)
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Items are sorted longest first; rounds alternate in direction so that no CTA gets the longest of every round.
__device__ __forceinline__ int item_of_round(int round) {
  const int g = gridDim.x, c = blockIdx.x;
  return round * g + ((round & 1) ? g - 1 - c : c);
}

// ---------------------------------------------------------------- forward --
// A CTA works on two query tiles ("slots") at a time against the same key tiles: two heads of a group where the group is
// even, else two neighbouring tiles of a head, else (few tiles in all) one, or a piece of one's keys.  While the softmax warps of one slot turn its
// scores into weights the tensor core works on the other's.  640 threads:
//   warps 0-7, 8-15  softmax of slot 0, 1: two threads per query row, 64 keys each, that agree on the maximum through shared
//                    memory.  One thread per row left two warps per scheduler, whose latencies nothing covered.
//   warp 16          TMA producer: Q per slot, K and V tiles in one ring
//   warps 17, 18     tcgen05.mma issuers.  At D = 64 one per slot: with one for both, each wait of one slot kept the other's
//                    products back.  At D > 64 the tensor core is what is scarce and one issues for both: products of two
//                    issuers take turns one by one, both slots then wait for them and work on weights at the same time, and
//                    nothing overlaps (326 against 265 us, 8192 positions, 16 heads of 128)
// TMEM: S of the slots at columns 0 and 128, O at 256 and 256 + D.  P (bf16), the A operand of P V, has columns of its own
// where there is room (D = 64: 384, 448): the next scores are then computed while this tile's weights are.  Else each half
// overwrites its own part of S.
// The CTA stays for all its items: loads and the first products of the next item run under the last steps of the one before.
constexpr int kBandThreads = 640;  // whole warpgroups: registers are handed from the last one to the others
constexpr int kComputeWarps = 16, kLoadWarp = 16, kMmaWarp = 17;  // kMmaWarp owns the TMEM; it and the next one issue
// 640 threads start with 96 registers each: 4 * 104 + 56 <= 5 * 96
#define NMB_BAND_FEW_REGISTERS asm volatile("setmaxnreg.dec.sync.aligned.u32 56;")
#define NMB_BAND_MORE_REGISTERS asm volatile("setmaxnreg.inc.sync.aligned.u32 104;")

struct BandFwdParams {
  CUtensorMap q_map, k_map, v_map, o_map, rest_map;
  BandArgs a;
  int pair;     // 0: one tile an item, 1: two neighbouring tiles, 2: two heads
  int n_qt;     // query tiles of a head
  int n_items;
  int t_last;   // first distance of the last bucket
  int pieces;   // parts of a tile's keys, with pair == 0 only: sums and statistics of each go to `part`
  float* part;  // per item: [128][D], then m [128] and l [128]
  FastDiv by_pieces;
  FastDiv by_hb, by_heads, by_group;  // heads (or pairs of them) times batches; heads (or pairs); query heads of a key head
};

template <int D>
struct BandFwdSmem {
  static constexpr int kSlabs = (D + 63) / 64;
  static constexpr int kTile = kSlabs * 16384;
  static constexpr int kStages = D == 64 ? 6 : 4;
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTile;
  static constexpr bool kStage = D == 64;  // results through shared memory: O and what was cut off of it, per slot
  static constexpr int kOut = kRing + kStages * kTile;
  static constexpr int kBar = kOut + (kStage ? 4 * kTile : 0);
  static constexpr int kNumBars = 2 * kStages + 16;
  static constexpr int kXch = kBar + ((kNumBars * 8 + 16 + 127) / 128) * 128;  // float [2][2 slots][2 halves][128]
  static constexpr int kLut = kXch + 4096;                                     // float [2][entries], then the map
};

template <int D>
constexpr int kFwdPart = 128 * D + 256;  // floats

struct FwdItem {
  int b, hk;
  int slot;  // of a piece; -1: the whole
  int h[2], q0[2];
  KeyTiles t[2], all;
};

template <bool kSplit>
__device__ __forceinline__ FwdItem fwd_item(const BandFwdParams& p, int item) {
  const BandArgs& a = p.a;
  FwdItem w;
  int rest, h, piece = 0;
  w.slot = -1;
  if (kSplit) {
    w.slot = item;
    item = p.by_pieces.quot(item, piece);
  }
  const int tiles = p.pair == 1 ? (p.n_qt + 1) / 2 : p.n_qt;
  const int tile = tiles - 1 - p.by_hb.quot(item, rest);
  w.b = p.by_heads.quot(rest, h);
  w.h[0] = p.pair == 2 ? 2 * h : h;
  w.h[1] = p.pair == 2 ? 2 * h + 1 : h;
  w.hk = p.by_group.quot(w.h[0]);
  w.q0[0] = (p.pair == 1 ? 2 * tile : tile) * 128;
  w.q0[1] = p.pair == 1 ? w.q0[0] + 128 : w.q0[0];
  w.t[0] = key_tiles(a, w.q0[0]);
  if (kSplit) {  // the first piece has the sinks too
    const int first = w.t[0].lo, n = w.t[0].hi - first + 1;
    if (n > 0) {
      w.t[0].lo = first + n * piece / p.pieces;
      w.t[0].hi = first + n * (piece + 1) / p.pieces - 1;
    }
    if (piece > 0) w.t[0].sink = 0;
  }
  if (p.pair == 0 || w.q0[1] >= a.Sq) {
    w.q0[1] = -1;
    w.t[1].sink = 0;
    w.t[1].lo = kNoTile;
    w.t[1].hi = -1;
  } else {
    w.t[1] = key_tiles(a, w.q0[1]);
  }
  w.all.lo = min(w.t[0].lo, w.t[1].lo);
  w.all.hi = max(w.t[0].hi, w.t[1].hi);
  w.all.sink = min(max(w.t[0].sink, w.t[1].sink), w.all.lo);
  return w;
}

template <int D, bool kExact, bool kSplit>
__global__ void __launch_bounds__(kBandThreads, 1) band_fwd_kernel(const __grid_constant__ BandFwdParams p) {
  using L = BandFwdSmem<D>;
  constexpr int NS = L::kSlabs, ST = L::kStages;
  constexpr bool kOwn = D == 64 && !kExact;  // P has its own columns
  constexpr int kIssuers = kOwn ? 2 : 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_full = bars;              // [ST]
  uint64_t* kv_empty = bars + ST;        // [ST]
  uint64_t* q_full = bars + 2 * ST;      // [2] per slot, as all that follow
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_full + 4;
  uint64_t* p_full = q_full + 6;
  uint64_t* o_full = q_full + 8;
  uint64_t* o_empty = q_full + 10;
  uint64_t* s_read = q_full + 12;        // only with P's own columns, as the next
  uint64_t* pv_done = q_full + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const BandArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entries = lut_entries(p.t_last);
  float* luts = reinterpret_cast<float*>(smem + L::kLut);
  uint8_t* map = reinterpret_cast<uint8_t*>(luts + 2 * entries);

  if ((smem_u32(smem) & 1023u) != 0) {  // swizzled operands need 1 KiB alignment
    if (threadIdx.x == 0) report_status(a.status, kBadArgument, 60);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], kIssuers);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 8);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 8);
      mbar_init(&s_read[t], 8);
      mbar_init(&pv_done[t], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) build_bucket_map(a, p.t_last, map, threadIdx.x, kBandThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns were allocated, so they begin at 0; said as a constant the addresses need no moves to uniform registers.
  constexpr uint32_t tmem = 0;
  if (threadIdx.x == 0 && *tmem_slot != 0) {
    report_status(a.status, kBadArgument, 75);
    *abort_flag = 1;
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&p.q_map);
    tma_prefetch_desc(&p.k_map);
    tma_prefetch_desc(&p.v_map);
  }
  pdl_enter();  // the set-up above touches no global memory
  if (warp >= kComputeWarps) {
    NMB_BAND_FEW_REGISTERS;
    if (warp == kLoadWarp) {
    // ------------------------------------------------------------ producer --
    if (lane == 0) {
      int pos = 0, n_q[2] = {0, 0};
      bool ok = true;
      for (int round = 0; ok; ++round) {
        const int item = item_of_round(round);
        if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
        if (item >= p.n_items) continue;
        const FwdItem w = fwd_item<kSplit>(p, item);
        auto load = [&](const CUtensorMap* m, int j) {
          const int st = pos % ST, use = pos / ST;
          if (use > 0 && !band_wait(&kv_empty[st], (use - 1) & 1, abort_flag, a.status, 61)) return false;
          mbar_expect_tx(&kv_full[st], L::kTile);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(smem + L::kRing + st * L::kTile + c * 16384, m, &kv_full[st], c * 64, j * 128, w.hk, w.b);
          ++pos;
          return true;
        };
        const int n = w.all.count();
        for (int t = 0; t < 2 && ok; ++t) {
          if (w.t[t].count() == 0) continue;
          if (n_q[t] > 0 && !band_wait(&q_empty[t], (n_q[t] - 1) & 1, abort_flag, a.status, 62)) {
            ok = false;
            break;
          }
          ++n_q[t];
          mbar_expect_tx(&q_full[t], L::kTile);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(smem + L::kQ + t * L::kTile + c * 16384, &p.q_map, &q_full[t], c * 64, w.q0[t], w.h[t], w.b);
        }
        for (int u = 0; u < n && ok; ++u) {
          const int j = tile_at(w.all, u);
          ok = load(&p.k_map, j) && load(&p.v_map, j);
        }
      }
    }
    } else if (warp >= kMmaWarp && warp < kMmaWarp + kIssuers) {
      // ------------------------------------------------------- MMA issuers --
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_o = make_idesc_bf16(128, D, false, true);
      constexpr int kMine = 2 / kIssuers;  // slots of an issuer
      const uint32_t ring = smem_u32(smem + L::kRing);
      const int t0 = kOwn ? warp - kMmaWarp : 0;
      const uint32_t chosen = elect_one();
      const bool branch = kOwn ? chosen != 0 : true;
      const uint32_t one = kOwn ? 1 : chosen;
      uint32_t base = 0, n_s[kMine] = {}, n_p[kMine] = {}, n_item[kMine] = {};
      bool ok = true;
      for (int round = 0; ok; ++round) {
        const int item = item_of_round(round);
        if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
        if (item >= p.n_items) continue;
        const FwdItem w = fwd_item<kSplit>(p, item);
        const int n = w.all.count();
        KeyTiles mine[kMine];
        int left[kMine];
        bool any[kMine], pending[kMine], first_s[kMine], first_pv[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          mine[i] = t0 + i == 0 ? w.t[0] : w.t[1];
          left[i] = mine[i].count();
          any[i] = left[i] > 0;
          pending[i] = false;
          first_s[i] = first_pv[i] = true;
        }
        auto v_bar = [&](int u) {
          const uint32_t pos = base + 2 * u + 1;
          return BandBar{&kv_full[pos % ST], (pos / ST) & 1};
        };
        auto k_bar = [&](int u) {
          const uint32_t pos = base + 2 * u;
          return BandBar{&kv_full[pos % ST], (pos / ST) & 1};
        };
        auto p_bar = [&](int i) { return BandBar{&p_full[t0 + i], n_p[i] & 1}; };
        // O += P V of tile u, whose V and P are there
        auto pv = [&](int i, int u, bool last) {
          const int t = t0 + i;
          tc_fence_after();
          if (branch) {
            const uint32_t b_low = desc_mn(ring + ((base + 2 * u + 1) % ST) * L::kTile);
            const uint32_t to = tmem + 256 + t * D, p_at = tmem + (kOwn ? 384 + t * 64 : t * 128);
            mma_apply<8, kOwn ? 8 : 4, 64>(to, p_at, b_low, idesc_o, first_pv[i], one);
            if (kExact) mma_apply<8, 4, 64>(to, p_at + 32, b_low, idesc_o, false, one);
            if (kOwn) commit_one(&pv_done[t], one);
            if (last) commit_one(&o_full[t], one);
          }
          ++n_p[i];
          first_pv[i] = false;
          pending[i] = false;
        };
        auto o_free = [&](int i) {  // the accumulator, for the first product of an item
          return !first_pv[i] || n_item[i] == 0 || band_wait(&o_empty[t0 + i], (n_item[i] - 1) & 1, abort_flag, a.status, 64);
        };
        // S = Q K^T; the first of an item waits for its queries
        auto scores = [&](int i, int u) {
          const int t = t0 + i;
          if (first_s[i] && !band_wait(&q_full[t], n_item[i] & 1, abort_flag, a.status, 67)) return false;
          first_s[i] = false;
          ++n_s[i];
          tc_fence_after();
          const bool last = --left[i] == 0;
          if (branch) {
            mma_scores<D>(tmem + t * 128, desc_k(smem_u32(smem + L::kQ + t * L::kTile)),
                          desc_k(ring + ((base + 2 * u) % ST) * L::kTile), idesc_s, one);
            commit_one(&s_full[t], one);
            if (last) commit_one(&q_empty[t], one);
          }
          return true;
        };
        auto release = [&](uint32_t pos) {
          if (branch) commit_one(&kv_empty[pos % ST], one);
        };
        for (int u = 0; u < n && ok; ++u) {
          const int j = tile_at(w.all, u);
          if (kOwn) {
            const bool use = mine[0].uses(j), was = pending[0];
            // P of the tile before may still be in the making: its product comes after these scores
            ok = n_s[0] == 0 ? band_wait(k_bar(u).bar, k_bar(u).parity, abort_flag, a.status, 66)
                             : band_wait_all(abort_flag, a.status, 66, k_bar(u), BandBar{&s_read[t0], (n_s[0] - 1) & 1});
            if (ok && use) ok = scores(0, u);
            if (ok) release(base + 2 * u);
            if (ok && was) {
              ok = o_free(0) && band_wait_all(abort_flag, a.status, 63, v_bar(u - 1), p_bar(0));
              if (ok) pv(0, u - 1, left[0] == 0 && !use);
            }
            if (ok && u > 0) {  // V of a tile that only the other slot works on: passed on once it is there, not before
              if (!was) ok = band_wait(v_bar(u - 1).bar, v_bar(u - 1).parity, abort_flag, a.status, 76);
              if (ok) release(base + 2 * u - 1);
            }
            pending[0] = use;
          } else {
            bool k_there = false, v_there = u == 0;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
              const bool use = mine[i].uses(j);
              if (ok && pending[i]) {
                ok = o_free(i) && (k_there && v_there ? band_wait(p_bar(i).bar, p_bar(i).parity, abort_flag, a.status, 65)
                                                      : band_wait_all(abort_flag, a.status, 65, k_bar(u), v_bar(u - 1), p_bar(i)));
                k_there = v_there = true;
                if (ok) pv(i, u - 1, left[i] == 0);
              }
              if (ok && use) {
                ok = (k_there || band_wait(k_bar(u).bar, k_bar(u).parity, abort_flag, a.status, 66)) && scores(i, u);
                k_there = true;
              }
              pending[i] = use;
            }
            ok = ok && (k_there || band_wait(k_bar(u).bar, k_bar(u).parity, abort_flag, a.status, 76)) &&
                 (v_there || band_wait(v_bar(u - 1).bar, v_bar(u - 1).parity, abort_flag, a.status, 76));
            if (ok) {
              release(base + 2 * u);
              if (u > 0) release(base + 2 * u - 1);
            }
          }
        }
        bool v_there = false;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          if (ok && pending[i]) {
            ok = o_free(i) && band_wait_all(abort_flag, a.status, 65, v_bar(n - 1), p_bar(i));
            v_there = true;
            if (ok) pv(i, n - 1, true);
          }
        }
        if (ok && n > 0) {
          if (!v_there) ok = band_wait(v_bar(n - 1).bar, v_bar(n - 1).parity, abort_flag, a.status, 76);
          if (ok) release(base + 2 * n - 1);
        }
        base += 2 * n;
#pragma unroll
        for (int i = 0; i < kMine; ++i) n_item[i] += any[i];
      }
    }
  } else {
    NMB_BAND_MORE_REGISTERS;
    // ------------------------------------------------- softmax + epilogue --
    const int t = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const int r = quad * 32 + lane;  // row in the tile == TMEM lane
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t t_s = t_row + t * 128 + half * 64, t_o = t_row + 256 + t * D + half * (D / 2);
    const uint32_t t_p = kOwn ? t_row + 384 + t * 64 + half * 32 : t_s;
    const float sl2 = a.scale * kBandLog2e;
    float* lut = luts + t * entries;
    float* xch = reinterpret_cast<float*>(smem + L::kXch) + t * 256 + r;
    int n_s = 0, n_item = 0, parity = 0;
    bool ok = true;
    // the other thread's value of this row
    auto other = [&](float mine) {
      float* x = xch + parity * 512;
      parity ^= 1;
      x[half * 128] = mine;
      named_sync(1 + t * 4 + quad, 64);
      return x[(half ^ 1) * 128];
    };
    for (int round = 0;; ++round) {
      const int item = item_of_round(round);
      if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
      if (item >= p.n_items) continue;
      const FwdItem w = fwd_item<kSplit>(p, item);
      const int q0 = t == 0 ? w.q0[0] : w.q0[1], h = t == 0 ? w.h[0] : w.h[1];
      const KeyTiles mine = t == 0 ? w.t[0] : w.t[1];
      if (q0 < 0) continue;
      const int row = q0 + r, pos = a.q_pos0 + row;
      const int pmin = a.q_pos0 + q0, pmax = pmin + 127;
      float far_bias = 0.f;
      if (a.table != nullptr) {
        named_sync(9 + t, 256);  // everyone has left the item before
        build_lut(a, h, p.t_last, map, lut, threadIdx.x & 255, 256);
        named_sync(9 + t, 256);
        far_bias = lut[entries - 1];
      }
      const int n = mine.count();
      float m = -INFINITY, l = 0.f;  // l: of this thread's keys
      for (int u = 0; u < n; ++u) {
        const int kv0 = tile_at(mine, u) * 128;
        NMB_BAND_WAIT(&s_full[t], n_s & 1, 68);
        ++n_s;
        tc_fence_after();
        uint32_t s[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32(t_s + c * 32, s[c]);
        tmem_ld_wait();
        if (kOwn) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_read[t]);
        }
        float mul = sl2, add = far_bias;
        // Biases that differ inside the tile, or that are too large to be added to the maximum instead of to the scores.
        const bool added = a.table != nullptr && (pmin - (kv0 + 127) < p.t_last || fabsf(far_bias) > 1e30f);
        if (added) {
          const float* at = lut + kLutFront + min(pos - kv0, p.t_last + kLutBack - 1) - half * 64;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) s[c][k] = __float_as_uint(fmaf(__uint_as_float(s[c][k]), sl2, at[-(c * 32 + k)]));
          mul = 1.f;
          add = 0.f;
        }
        // What this warp's rows see of each chunk of 32 keys: all (1), none (2), or some (0).
        const bool whole = kv0 + 127 <= pmin && kv0 + 127 < a.Skv && (kv0 > pmax - a.window || kv0 + 127 < a.sinks);
        uint32_t part[2] = {1, 1};
        if (!whole) {
          const int k0 = kv0 + half * 64;
          const int hi = min(pos, a.Skv - 1) - k0 + 1, lo = pos - a.window + 1 - k0, sk = a.sinks - k0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t see = low_bits(hi - c * 32) & (~low_bits(lo - c * 32) | low_bits(sk - c * 32));
            part[c] = __all_sync(0xffffffffu, see == ~0u) ? 1u : __all_sync(0xffffffffu, see == 0u) ? 2u : 0u;
            if (part[c] == 0) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((see >> k) & 1u)) s[c][k] = 0xff800000u;
            }
          }
        }
        float mx[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[c] = -INFINITY;
          if (part[c] != 2) {
            float m0 = __uint_as_float(s[c][0]), m1 = __uint_as_float(s[c][1]);
#pragma unroll
            for (int k = 2; k < 30; k += 4) {
              m0 = max3(m0, __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
              m1 = max3(m1, __uint_as_float(s[c][k + 2]), __uint_as_float(s[c][k + 3]));
            }
            mx[c] = max3(max2(m0, m1), __uint_as_float(s[c][30]), __uint_as_float(s[c][31]));
          }
        }
        float top = fmaf(max2(mx[0], mx[1]), mul, add);
        top = max2(top, other(top));
        // The maximum that weights are relative to moves only when it grew by more than 2^8: most tiles need no pass over O,
        // and the division by the sum at the end makes the result exact.  A row with a score of NaN or +inf is NaN from here
        // on: not all of its weights would be (a polynomial makes a quarter of them, which knows no NaN), but m is.
        const float m_new = !(top < INFINITY) ? NAN : top > m + 8.f ? top : m;
        const float alpha = m_new == m ? 1.f : ex2(m - m_new);  // m == -inf: 0
        const float shift = add - (m_new == -INFINITY ? 0.f : m_new);
        // The product of the tile before is done: with shared columns the scores came after it.
        if (kOwn && n_s > 1) NMB_BAND_WAIT(&pv_done[t], n_s & 1, 73);
        if (u > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[16];
            tmem_ld_32x16(t_o + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st_32x16(t_o + c * 16, o);
          }
        }
        const uint64_t mul_2 = pack2(mul, mul), shift_2 = pack2(shift, shift);
        uint64_t sum = pack2(0.f, 0.f);
        if constexpr (!kExact) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
            if (part[c] == 2) {
#pragma unroll
              for (int k = 0; k < 16; ++k) pk[k] = 0;
            } else if (part[c] == 1 && !added) {
              weights32<true>(s[c], mul_2, shift_2, sum, pk);
            } else {
              weights32<false>(s[c], mul_2, shift_2, sum, pk);
            }
            tmem_st_32x16(t_p + c * 16, pk);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float p0 = 0.f, p1 = 0.f;
              if (part[c] != 2) {
                unpack2(fma2(pack2(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1])), mul_2, shift_2), p0, p1);
                p0 = ex2(p0);
                p1 = ex2(p1);
              }
              sum = add2(sum, pack2(p0, p1));
              pk[k] = pack_bf16x2(p0, p1);
              s[c][k] = pack_bf16x2(p0 - __uint_as_float(pk[k] << 16), p1 - __uint_as_float(pk[k] & 0xffff0000u));
            }
            tmem_st_32x16(t_p + c * 16, pk);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) tmem_st_32x16(t_p + 32 + c * 16, *reinterpret_cast<const uint32_t(*)[16]>(s[c]));
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        float sum0, sum1;
        unpack2(sum, sum0, sum1);
        // nothing but scores of -inf so far: the polynomial's 2^-126 for them are no weights
        l = l * alpha + (m_new == -INFINITY ? 0.f : sum0 + sum1);
        m = m_new;
      }
      if (n > 0) {
        l += other(l);
        NMB_BAND_WAIT(&o_full[t], n_item & 1, 69);
        ++n_item;
        tc_fence_after();
      }
      if (kSplit) {
        float* part = p.part + static_cast<long long>(w.slot) * kFwdPart<D>;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[16];
          if (n > 0) {
            tmem_ld_32x16(t_o + c * 16, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = 0;
          }
          float* at = part + r * D + half * (D / 2) + c * 16;
          st_global_32(at, o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]);
          st_global_32(at + 8, o[8], o[9], o[10], o[11], o[12], o[13], o[14], o[15]);
        }
        if (half == 0) {
          part[128 * D + r] = m;
          part[128 * D + 128 + r] = l;
        }
        if (n > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_empty[t]);
        }
        continue;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;  // NaN stays
      __nv_bfloat16* out = band_row(a.o, a.o_st, w.b, row, h) + half * (D / 2);
      uint8_t* tile = smem + L::kOut + 2 * t * L::kTile;
      const bool some_rest = q0 < a.rest_rows;
      if (L::kStage) {
        if (quad == 0 && half == 0 && lane == 0) store_wait_read();  // the item before has left the tile
        named_sync(9 + t, 256);
      }
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[16];
        if (n > 0) {
          tmem_ld_32x16(t_o + c * 16, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * inv);
        if (L::kStage) {
          stage_bf16_16(tile, r, half * (D / 2) + c * 16, o, 1.f);
        } else if (row < a.Sq) {
          store_bf16_16(out + c * 16, o, 1.f);
        }
        if (some_rest) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float x = __uint_as_float(o[k]);
            o[k] = __float_as_uint(x - __bfloat162float(__float2bfloat16(x)));
          }
          if (L::kStage) {
            stage_bf16_16(tile + L::kTile, r, half * (D / 2) + c * 16, o, 1.f);
          } else if (row < a.rest_rows) {
            store_bf16_16(rest_row(a, w.b, row, h, D) + half * (D / 2) + c * 16, o, 1.f);
          }
        }
      }
      if (L::kStage) {
        fence_proxy_async_smem();
        named_sync(9 + t, 256);
        if (quad == 0 && half == 0 && lane == 0) {
          tma_store_4d(&p.o_map, tile, 0, q0, h, w.b);
          if (some_rest) tma_store_4d(&p.rest_map, tile + L::kTile, 0, q0, h, w.b);
          store_commit();
        }
      }
      if (n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[t]);
      }
      if (half == 0 && row < a.Sq && a.m != nullptr) {
        const long long stat = (static_cast<long long>(w.b) * a.Hq + h) * a.Sq + row;
        a.m[stat] = l == 0.f ? INFINITY : m;  // a row that sees nothing: 2^(x - m) is 0 in the backward pass
        a.l[stat] = l == 0.f ? 0.f : log2f(l);
      }
    }
    if (L::kStage) store_wait();
  }

  if (*abort_flag != 0) {  // let the loads in flight land
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// What the pieces of a query tile come to: a warp per row, the pieces in order.  A piece that saw no key has m = -inf, l = 0.
template <int D>
__global__ void __launch_bounds__(256) band_join_kernel(const __grid_constant__ BandFwdParams p) {
  pdl_enter();
  const BandArgs& a = p.a;
  const int lane = threadIdx.x & 31, at = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5), item = at >> 7, r = at & 127;
  int rest, h;
  const int row = (p.n_qt - 1 - p.by_hb.quot(item, rest)) * 128 + r, b = p.by_heads.quot(rest, h);
  if (row >= a.Sq) return;
  const float* part = p.part + static_cast<long long>(item) * p.pieces * kFwdPart<D>;
  float top = -INFINITY;
  for (int i = 0; i < p.pieces; ++i) top = max2(top, part[static_cast<long long>(i) * kFwdPart<D> + 128 * D + r]);
  float sum = 0.f, o[D / 32] = {};
  if (top != -INFINITY) {
    for (int i = 0; i < p.pieces; ++i) {
      const float* one = part + static_cast<long long>(i) * kFwdPart<D>;
      const float w = ex2(one[128 * D + r] - top);
      sum = fmaf(w, one[128 * D + 128 + r], sum);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) o[k] = fmaf(w, one[r * D + k * 32 + lane], o[k]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __nv_bfloat16* out = band_row(a.o, a.o_st, b, row, h);
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    const float x = o[k] * inv;
    const __nv_bfloat16 y = __float2bfloat16(x);
    out[k * 32 + lane] = y;
    if (row < a.rest_rows) rest_row(a, b, row, h, D)[k * 32 + lane] = __float2bfloat16(x - __bfloat162float(y));
  }
  if (lane == 0 && a.m != nullptr) {
    const long long stat = (static_cast<long long>(b) * a.Hq + h) * a.Sq + row;
    a.m[stat] = sum == 0.f ? INFINITY : top;
    a.l[stat] = sum == 0.f ? 0.f : log2f(sum);
  }
}

static int make_band_map(CUtensorMap* m, const __nv_bfloat16* ptr, const BandStride& t, int d, int S, int H, int B) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(S), static_cast<uint64_t>(H), static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {static_cast<uint64_t>(t.s) * 2, static_cast<uint64_t>(t.h) * 2,
                               static_cast<uint64_t>(t.b) * 2};
  const uint32_t box[4] = {64, 128, 1, 1};
  return make_tmap_bf16(m, ptr, 4, dims, strides, box);
}

// With kExact the weights go into O to twice bf16's digits: the head and what it cut off lie in the columns that the scores were
// in, and take a product each.  D comes from O, and a bias table's gradient is a sum over dS in which D's error does not cancel,
// but adds up where a bucket has much of the rows' weight, be it the last one or a wide or favoured one before it: with bf16
// weights it was 2.2 times as far from the exact one as its own rounding at 22 keys, up to 14 times over thousands (2 to 64
// buckets), 7.5 times with a table that favours one bucket; with both parts it is no further.  The second product is
// paid by every training step with a table (8192 x 16 heads, D = 128: 1258 -> 1348 us; 2 x 2048, D = 64: 160 -> 168 us).
// Without a table it is for dQ and dK where rows see few keys: over 64 and over 65 keys dQ is 1.05 and 1.06 times as far from
// the exact one as one rounding of the power of two below a value (two independent roundings come to 1.04; with D from bf16 weights
// and a bf16 output it was 1.09 over 32 keys, 1.17 over 8, 1.5 over 2), at 18.7 and 15.6 us forward (8 x 512, 16/8 heads, D = 64).
static bool exact_weights(const BandArgs& a) {
  if (a.m == nullptr) return false;
  const long long keys = std::min<long long>(a.Skv, static_cast<long long>(a.window) + a.sinks);
  return a.table != nullptr || keys <= 64;
}
template <int D>
static cudaError_t launch_band_fwd(const BandFwdParams& p, cudaStream_t s) {
  const BandArgs& a = p.a;
  const int lut = a.table == nullptr ? 0 : lut_bytes(p.t_last, 2);
  const bool exact = exact_weights(a);
  return launch_pdl(p.pieces > 1 ? (exact ? band_fwd_kernel<D, true, true> : band_fwd_kernel<D, false, true>)
                                 : (exact ? band_fwd_kernel<D, true, false> : band_fwd_kernel<D, false, false>), dim3(std::min(p.n_items, sm_count())), dim3(kBandThreads), BandFwdSmem<D>::kLut + lut, s, p);
}
template <int D>
static cudaError_t launch_band_join(const BandFwdParams& p, cudaStream_t s) {
  return launch_pdl(band_join_kernel<D>, dim3(static_cast<unsigned>(p.n_items / p.pieces * 16)), dim3(256), 0, s, p);
}
// Into how many pieces the keys of a query tile are cut where there are not half as many tiles as SMs, three or four key tiles to
// a piece at least: one row over 8192 keys, 16 heads of 128 (16/4 heads alike): 115 -> 25 us; over 1024 keys 18 -> 15 us.  The
// window's tiles alone are counted and cut, sinks stay with the first piece: one row with a window of 64 and 4096 sinks, 61 us.
// (As a variant of its own: the pieces cost the others 2 to 5 percent.)
constexpr int kSplitKeyTiles = 8;
static int fwd_pieces(const BandArgs& a) {
  const long long tiles = static_cast<long long>((a.Sq + 127) / 128) * a.Hq * a.B;
  if (tiles * 2 > sm_count()) return 1;
  const long long seen = std::min<long long>(std::min<long long>(a.Skv, static_cast<long long>(a.q_pos0) + a.Sq), a.window + 127ll);
  const int n = static_cast<int>((seen + 127) / 128);
  if (n < kSplitKeyTiles) return 1;
  return std::min(static_cast<int>(sm_count() / tiles), (n + 3) / 4);
}

// --------------------------------------------------------------- backward --
// Two large kernels and no atomics: a query tile's dQ and a key tile's dK, dV are each summed by one CTA in a fixed order, at the
// price of working the weights out twice (seven products of a tile pair instead of five).
//
// Statistics of the query rows that both read, per (batch, query head, query tile): 128 floats each of
//   c = (far bias - m) - l,  D,  m,  l        (rows behind the last: c = -inf, so that their weights are 0)
constexpr int kStatBlock = 512;  // floats

// 2^(s * mul + shift) of 32 scores in place (a NaN may get lost: D is one then, and with it dS)
template <bool kMix>
__device__ __forceinline__ void exps32(uint32_t (&s)[32], uint64_t mul, uint64_t shift) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float p0, p1;
    exp2_pair<kMix>(k, fma2(pack2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), mul, shift), p0, p1);
    s[2 * k] = __float_as_uint(p0);
    s[2 * k + 1] = __float_as_uint(p1);
  }
}
// the same with a shift per column, and NaN where a score or a shift is one: these weights also go into dV, without D
template <bool kMix>
__device__ __forceinline__ void exps32(uint32_t (&s)[32], uint64_t mul, const float* shift) {
#pragma unroll
  for (int k = 0; k < 16; k += 2) {
    const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(shift + 2 * k);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float p0, p1;
      exp2_pair<kMix, true>(k + i, fma2(pack2(__uint_as_float(s[2 * (k + i)]), __uint_as_float(s[2 * (k + i) + 1])), mul, i ? c.y : c.x), p0, p1);
      s[2 * (k + i)] = __float_as_uint(p0);
      s[2 * (k + i) + 1] = __float_as_uint(p1);
    }
  }
}

struct BandBwdParams {
  CUtensorMap q_map, k_map, v_map, do_map, dq_map, dk_map, dv_map;
  BandArgs a;
  float* stat;      // [B, Hq, n_qt, kStatBlock]
  float* part;      // fp32 dV, dK tiles of key tiles whose rows are split
  float* dtable_part;  // [B, Hq, n_qt, buckets]
  int n_qt, n_kt;
  int n_items;      // of this kernel
  int t_last;
  int sink_tiles;   // dK, dV: key tiles that hold sinks, their pieces, the pieces of the others
  int sink_pieces, pieces;
  int first_seen;   // the first of the others that a row sees
  FastDiv by_hqb, by_hq, by_group;                        // dQ: query heads times batches, query heads; query heads of a key head
  FastDiv by_hkvb, by_hkv, by_sink_pieces, by_pieces;     // dK, dV: the same of key heads, and the pieces
};

// ---- D and the column statistics ----
// A block per query tile; D / 8 lanes a row (16 bytes each of dO, O and what was cut off of it), a thread's rows in flight together.
// In the dQ kernel, a thread per quarter row, the same loads hit a line per lane and cost an item 4000 clocks.
template <int D>
__host__ __device__ constexpr int stat_blocks() { return D == 64 ? 1 : 2; }
template <int D>
__global__ void __launch_bounds__(256, 3) band_stat_kernel(const __grid_constant__ BandBwdParams p) {
  pdl_enter();
  const BandArgs& a = p.a;
  constexpr int kLanes = D == 64 ? 8 : 16;  // 12 of 16 at D = 96
  constexpr int kRowsAtOnce = 256 / kLanes, kStatRows = 4, kParts = stat_blocks<D>();
  const int sub = threadIdx.x / kLanes, part = threadIdx.x % kLanes;
  // heads run fastest: their rows lie next to one another in memory
  int rest_of, h;
  const int at_qt = p.by_hqb.quot(static_cast<int>(blockIdx.x), rest_of), b = p.by_hq.quot(rest_of, h);
  const int qt = at_qt / kParts, r0 = at_qt % kParts * (kRowsAtOnce * kStatRows) + sub;
  const long long tile = (static_cast<long long>(b) * a.Hq + h) * p.n_qt + qt;
  const bool mine = part * 8 < D;
  uint4 o[kStatRows], rest[kStatRows], g[kStatRows];
  float m[kStatRows], l[kStatRows];
#pragma unroll
  for (int i = 0; i < kStatRows; ++i) {
    const int row = qt * 128 + r0 + i * kRowsAtOnce;
    m[i] = INFINITY;
    l[i] = 0.f;
    if (part == 0 && row < a.Sq) {
      const long long at = (static_cast<long long>(b) * a.Hq + h) * a.Sq + row;
      m[i] = a.m[at];
      l[i] = a.l[at];
    }
    if (mine && row < a.Sq) {
      o[i] = *reinterpret_cast<const uint4*>(band_row(a.o, a.o_st, b, row, h) + part * 8);
      rest[i] = row < a.rest_rows ? *reinterpret_cast<const uint4*>(rest_row(a, b, row, h, D) + part * 8) : make_uint4(0, 0, 0, 0);
      g[i] = *reinterpret_cast<const uint4*>(band_row(a.dout, a.dout_st, b, row, h) + part * 8);
    } else {
      o[i] = rest[i] = g[i] = make_uint4(0, 0, 0, 0);
    }
  }
  const float far_bias = a.table == nullptr ? 0.f : bias_log2(table_at(a, h, a.buckets - 1));
  float* st = p.stat + tile * kStatBlock;
#pragma unroll
  for (int i = 0; i < kStatRows; ++i) {
    const uint32_t ow[4] = {o[i].x, o[i].y, o[i].z, o[i].w}, rw[4] = {rest[i].x, rest[i].y, rest[i].z, rest[i].w};
    const uint32_t gw[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = unpack_bf16x2(ow[k]), z = unpack_bf16x2(rw[k]), y = unpack_bf16x2(gw[k]);
      sum = fmaf(x.x + z.x, y.x, fmaf(x.y + z.y, y.y, sum));
    }
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const int r = r0 + i * kRowsAtOnce;
    if (part == 0) {
      st[r] = (far_bias - m[i]) - l[i];
      st[128 + r] = sum;
      st[256 + r] = m[i];
      st[384 + r] = l[i];
    }
  }
}

// The sixteen compute warps of the two kernels below work as one group on a tile of 128 x 128 weights, or (D = 64) as two
// groups on one half of its columns each, with tensor-memory columns, accumulators, barriers and an issuer of their own: while
// one group works out weights (16 exponentials a clock and SM: 512 clocks for its half) the other waits, loads and stores.  At
// D > 64 there are no columns for a second set of accumulators, and products with half the columns would take longer than the
// weights (59 clocks instead of 34 for a 128 x 64 x 16 product out of shared memory).
template <int D>
struct BandGroups {
  static constexpr int kGroups = D == 64 ? 2 : 1;
  static constexpr int kWidth = 128 / kGroups;               // columns of a group
  static constexpr int kWarps = kComputeWarps / kGroups;
  static constexpr int kQuarters = 4 / kGroups;              // of 32 columns, a thread's share of a row
};

// ---- dQ and the table's gradient ----
// A CTA works on one query tile: S = Q K^T and dP = dO V^T land in tensor memory, sixteen warps (four threads a row, 32 columns
// each) turn them into dS, which goes back as the A operand of dQ += dS K.  S and dP of the next tile are computed while
// dS of this one is.  TMEM: S 0, dP 128, dQ 256 (a second one for the second group at 256 + D), dS (two buffers) from 384.
//
// D = dO . O wants O with more bits than a bf16 result has: the error of its rounding is the same for all keys of a row, adds
// up where terms of dS cancel (few keys: 4.7e-3 of dQ's norm instead of 2.3e-3), and, summed over thousands of keys, is as large
// as the gradient of the last bucket (1.6e-2 of it).  So a forward pass that will be differentiated also keeps what the rounding
// cut off, as another bf16 value: of all rows with a bias, else of those that see few keys (the caller says up to which row).
//
// dtable: inside tiles that meet distances below t_last the sums along the diagonals (equal distance) are formed by passing a
// running sum from lane to lane, one row down per column; they are then added by bucket.  All other tiles belong to the last
// bucket as a whole.
template <int D>
struct BandDqSmem {
  static constexpr int kSlabs = (D + 63) / 64;
  static constexpr int kTile = kSlabs * 16384;
  static constexpr int kQStages = D == 64 ? 2 : 1;
  // K stays until dQ += dS K, V only until dP: where four tiles is all there is room for, three are for K (a ring of two
  // pairs left the loads of K exposed: 1640 of 4020 clocks a tile were spent waiting at d = 128)
  static constexpr int kStagesK = 3, kStagesV = D == 64 ? 3 : 1;
  static constexpr int kStages = kStagesK + kStagesV;
  static constexpr int kQ = 0;                     // Q, dO per stage
  static constexpr int kRing = 2 * kQStages * kTile;  // the stages of K, then those of V
  static constexpr bool kStage = D == 64;  // dQ through shared memory
  static constexpr int kOut = kRing + kStages * kTile;
  static constexpr int kStat = kOut + (kStage ? kTile : 0);  // per stage of Q
  static constexpr int kBar = kStat + kQStages * kStatBlock * 4;
  static constexpr int kNumBars = 2 * kStages + 2 * kQStages + 11;
  static constexpr int kLut = kBar + ((kNumBars * 8 + 16 + 127) / 128) * 128;  // float [entries], the map
  // behind them, where the table's gradient is wanted: float bins[16][128], diagonals[16][64]
  static constexpr int kBins = kComputeWarps * (kMaxBuckets + 64) * 4;
  // columns of a row that one of its four threads reads and writes; three do at D = 96
  static constexpr int kCols = D == 96 ? 32 : D / 4;
};

// The query tile of an item, longest first.
struct DqItem {
  int b, h, hk, q0;
  KeyTiles t;
};
__device__ __forceinline__ DqItem dq_item(const BandBwdParams& p, int item) {
  const BandArgs& a = p.a;
  DqItem w;
  int rest;
  w.q0 = (p.n_qt - 1 - p.by_hqb.quot(item, rest)) * 128;
  w.b = p.by_hq.quot(rest, w.h);
  w.hk = p.by_group.quot(w.h);
  w.t = key_tiles(a, w.q0);
  return w;
}

template <int D>
__global__ void __launch_bounds__(kBandThreads, 1) band_bwd_dq_kernel(const __grid_constant__ BandBwdParams p) {
  using L = BandDqSmem<D>;
  using G = BandGroups<D>;
  constexpr int NS = L::kSlabs, ST = L::kStages, SK = L::kStagesK, SV = L::kStagesV, QS = L::kQStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_full = bars;                // [SK + SV]
  uint64_t* kv_empty = bars + ST;          // [SK + SV]
  uint64_t* q_full = bars + 2 * ST;        // [QS]
  uint64_t* q_empty = q_full + QS;         // [QS] the issuers + the warps that read the statistics
  uint64_t* sdp_full = q_empty + QS;       // [groups], as all that follow
  uint64_t* sdp_read = sdp_full + 2;
  uint64_t* dq_full = sdp_full + 4;
  uint64_t* ds_full = sdp_full + 6;        // [groups][2]: one for even and one for odd steps, as the buffers of dS (with one, a
                                           // step could be over twice before it was looked at)
  uint64_t* dq_empty = sdp_full + 10;      // one for both
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const BandArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entries = lut_entries(p.t_last);
  float* lut = reinterpret_cast<float*>(smem + L::kLut);
  uint8_t* map = reinterpret_cast<uint8_t*>(lut + entries);
  float* bins = reinterpret_cast<float*>(smem + L::kLut + lut_bytes(p.t_last, 1));
  constexpr uint32_t kDp = 128, kDq = 256, kDs = 384;

  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_status(a.status, kBadArgument, 80);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], G::kGroups);  // the issuers
    }
    for (int s = 0; s < QS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], G::kGroups + kComputeWarps);
    }
    for (int g = 0; g < G::kGroups; ++g) {
      mbar_init(&sdp_full[g], 1);
      mbar_init(&sdp_read[g], G::kWarps);
      mbar_init(&dq_full[g], 1);
      mbar_init(&ds_full[2 * g], G::kWarps);
      mbar_init(&ds_full[2 * g + 1], G::kWarps);
    }
    mbar_init(dq_empty, kComputeWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) {
    build_bucket_map(a, p.t_last, map, threadIdx.x, kBandThreads);
    if (a.dtable != nullptr)
      for (int n = threadIdx.x; n < kComputeWarps * kMaxBuckets; n += kBandThreads) bins[n] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns were allocated, so they begin at 0; said as a constant the addresses need no moves to uniform registers.
  constexpr uint32_t tmem = 0;
  if (threadIdx.x == 0 && *tmem_slot != 0) {
    report_status(a.status, kBadArgument, 75);
    *abort_flag = 1;
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&p.q_map);
    tma_prefetch_desc(&p.k_map);
    tma_prefetch_desc(&p.v_map);
    tma_prefetch_desc(&p.do_map);
  }
  pdl_enter();
  const int rounds = (p.n_items + gridDim.x - 1) / gridDim.x;

  if (warp >= kComputeWarps) {
    NMB_BAND_FEW_REGISTERS;
    if (warp == kLoadWarp && lane == 0) {
      // ---------------------------------------------------------- producer --
      int pos = 0, n_item = 0;
      bool ok = true;
      for (int round = 0; round < rounds && ok; ++round) {
        const int item = item_of_round(round);
        if (item >= p.n_items) continue;
        const DqItem w = dq_item(p, item);
        const int n = w.t.count();
        if (n == 0) continue;
        const int qs = n_item % QS, use = n_item / QS;
        ++n_item;
        if (use > 0 && !band_wait(&q_empty[qs], (use - 1) & 1, abort_flag, a.status, 81)) break;
        const uint32_t stat_bytes = a.table == nullptr ? 1024 : 2048;
        mbar_expect_tx(&q_full[qs], 2 * L::kTile + stat_bytes);
        bulk_load(smem + L::kStat + qs * kStatBlock * 4,
                  p.stat + ((static_cast<long long>(w.b) * a.Hq + w.h) * p.n_qt + w.q0 / 128) * kStatBlock, stat_bytes, &q_full[qs]);
#pragma unroll
        for (int c = 0; c < NS; ++c) {
          uint8_t* dst = smem + L::kQ + 2 * qs * L::kTile + c * 16384;
          tma_load_4d(dst, &p.q_map, &q_full[qs], c * 64, w.q0, w.h, w.b);
          tma_load_4d(dst + L::kTile, &p.do_map, &q_full[qs], c * 64, w.q0, w.h, w.b);
        }
        auto load = [&](const CUtensorMap* m, int st, int use, int j) {
          if (use > 0 && !band_wait(&kv_empty[st], (use - 1) & 1, abort_flag, a.status, 82)) return false;
          mbar_expect_tx(&kv_full[st], L::kTile);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(smem + L::kRing + st * L::kTile + c * 16384, m, &kv_full[st], c * 64, j * 128, w.hk, w.b);
          return true;
        };
        for (int u = 0; u < n && ok; ++u, ++pos) {
          const int j = tile_at(w.t, u);
          ok = load(&p.k_map, pos % SK, pos / SK, j) && load(&p.v_map, SK + pos % SV, pos / SV, j);
        }
      }
    } else if (warp >= kMmaWarp && warp < kMmaWarp + G::kGroups) {
      // -------------------------------------------------------- MMA issuer --
      // In order: S and dP of a step once those of the step before have been read, then dQ of the step before.  Whoever sees S
      // and dP of a step therefore knows that dQ of the step before the last has been added, whose dS buffer is next.
      constexpr uint32_t idesc_s = make_idesc_bf16(128, G::kWidth, false, false);
      constexpr uint32_t idesc_dq = make_idesc_bf16(128, D, false, true);
      const int g = warp - kMmaWarp;
      const uint32_t ring = smem_u32(smem + L::kRing) + g * G::kWidth * 128;  // this group's rows of K and V
      const uint32_t t_s = tmem + g * G::kWidth, t_dq = tmem + kDq + g * D, t_ds = tmem + kDs + g * (G::kWidth / 2);
      const bool one = elect_one();
      uint32_t step = 0, n_item = 0;  // tiles and items begun
      bool prev_first = false, prev_last = false;
      uint32_t prev_item = 0;
      bool ok = true;
      // dQ += dS K of step s
      auto issue_dq = [&](uint32_t s, bool first, bool last, uint32_t item_no) {
        if (first && item_no > 0 && !band_wait(dq_empty, (item_no - 1) & 1, abort_flag, a.status, 83)) return false;
        if (!band_wait(&ds_full[2 * g + (s & 1)], (s >> 1) & 1, abort_flag, a.status, 84)) return false;
        tc_fence_after();
        const uint32_t st = s % SK;
        if (one) {
          mma_apply<G::kWidth / 16, 8, 0>(t_dq, t_ds + (s & 1) * 64, desc_mn(ring + st * L::kTile), idesc_dq, first);
          tc_commit(&kv_empty[st]);
          if (last) tc_commit(&dq_full[g]);
        }
        return true;
      };
      for (int round = 0; round < rounds && ok; ++round) {
        const int item = item_of_round(round);
        if (item >= p.n_items) continue;
        const DqItem w = dq_item(p, item);
        const int n = w.t.count();
        if (n == 0) continue;
        const uint32_t qs = n_item % QS;
        const uint32_t q_low = desc_k(smem_u32(smem + L::kQ + 2 * qs * L::kTile));
        for (int u = 0; u < n; ++u, ++step) {
          const uint32_t sk = step % SK, sv = SK + step % SV;
          const BandBar k_bar{&kv_full[sk], (step / SK) & 1}, v_bar{&kv_full[sv], (step / SV) & 1};
          ok = u > 0 || band_wait(&q_full[qs], (n_item / QS) & 1, abort_flag, a.status, 85);
          if (!ok) break;
          ok = step == 0 ? band_wait(k_bar.bar, k_bar.parity, abort_flag, a.status, 86)
                         : band_wait_all(abort_flag, a.status, 88, k_bar, BandBar{&sdp_read[g], (step - 1) & 1});
          if (!ok) break;
          tc_fence_after();
          if (one) mma_scores<D>(t_s, q_low, desc_k(ring + sk * L::kTile), idesc_s);
          ok = band_wait(v_bar.bar, v_bar.parity, abort_flag, a.status, 87);
          if (!ok) break;
          if (one) {
            mma_scores<D>(t_s + kDp, q_low + (L::kTile >> 4), desc_k(ring + sv * L::kTile), idesc_s);
            tc_commit(&sdp_full[g]);
            tc_commit(&kv_empty[sv]);
            if (u == n - 1) tc_commit(&q_empty[qs]);
          }
          if (step > 0) ok = issue_dq(step - 1, prev_first, prev_last, prev_item);
          if (!ok) break;
          prev_first = u == 0;
          prev_last = u == n - 1;
          prev_item = n_item;
        }
        ++n_item;
      }
      if (ok && step > 0) issue_dq(step - 1, prev_first, prev_last, prev_item);
    }
  } else {
    NMB_BAND_MORE_REGISTERS;
    // ------------------------------------------------------------ compute --
    const int quad = warp & 3, quarter = warp >> 2;
    const int r = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const int g = quarter / G::kQuarters;
    const bool has_cols = quarter * L::kCols < D;
    float* my_bins = bins + warp * kMaxBuckets;
    float* diag = bins + kComputeWarps * kMaxBuckets + warp * 64;
    const float sl2 = a.scale * kBandLog2e;
    const bool want_table = a.dtable != nullptr;
    int step = 0, n_item = 0;
    auto together = [&]() { named_sync(1, kComputeWarps * 32); };
    bool ok = true;
    for (int round = 0; round < rounds; ++round) {
      const int item = item_of_round(round);
      if (item >= p.n_items) continue;
      const DqItem w = dq_item(p, item);
      const int n = w.t.count();
      const int row = w.q0 + r, pos = a.q_pos0 + row, pmin = a.q_pos0 + w.q0;
      const bool valid = row < a.Sq;
      float far_bias = 0.f;
      if (a.table != nullptr) {
        together();  // everyone has left the item before
        build_lut(a, w.h, p.t_last, map, lut, threadIdx.x, kComputeWarps * 32);
        together();
        far_bias = lut[entries - 1];
      }
      float c_far = 0.f, delta = 0.f, m = 0.f, l = 0.f;
      if (n > 0) {
        const int qs = n_item % QS;
        NMB_BAND_WAIT(&q_full[qs], (n_item / QS) & 1, 89);
        const float* st = reinterpret_cast<const float*>(smem + L::kStat) + qs * kStatBlock + r;
        c_far = st[0];
        delta = st[128];
        m = st[256];  // these two are there and used with a table only
        l = st[384];
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[qs]);
      }
      float ds_far = 0.f;  // sum of dS in tiles that are all the last bucket's own
      for (int u = 0; u < n; ++u, ++step) {
        const int kv0 = tile_at(w.t, u) * 128, k0 = kv0 + quarter * 32;
        NMB_BAND_WAIT(&sdp_full[g], step & 1, 90);
        tc_fence_after();
        uint32_t s[32], dp[32];
        tmem_ld_32x32(t_row + quarter * 32, s);
        tmem_ld_32x32(t_row + kDp + quarter * 32, dp);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sdp_read[g]);
        const bool near = a.table != nullptr && pmin - (kv0 + 127) < p.t_last;
        const bool added = near || (a.table != nullptr && fabsf(far_bias) > 1e30f);
        const bool whole = kv0 + 127 <= pmin && kv0 + 127 < a.Skv && (pmin + 127 - kv0 < a.window || kv0 + 127 < a.sinks);
        // weights, in place of the scores
        if (!added && w.q0 + 128 <= a.Sq) {  // every row sees finite scores: no weight has to come out as 0
          exps32<true>(s, pack2(sl2, sl2), pack2(c_far, c_far));
        } else if (!added) {
          exps32<false>(s, pack2(sl2, sl2), pack2(c_far, c_far));
        } else {
          const float* at = lut + kLutFront + min(pos - kv0, p.t_last + kLutBack - 1) - quarter * 32;
#pragma unroll
          for (int k = 0; k < 32; ++k) s[k] = __float_as_uint(ex2((fmaf(__uint_as_float(s[k]), sl2, at[-k]) - m) - l));
        }
        if (!whole) {
          const uint32_t see = low_bits(min(pos, a.Skv - 1) - k0 + 1) & (~low_bits(pos - a.window + 1 - k0) | low_bits(a.sinks - k0));
          if (!__all_sync(0xffffffffu, see == ~0u)) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1u)) s[k] = 0;
          }
        }
        {
          uint32_t pk[16];
          const uint64_t minus = pack2(-delta, -delta);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float d0, d1;
            unpack2(mul2(pack2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])),
                         add2(pack2(__uint_as_float(dp[2 * k]), __uint_as_float(dp[2 * k + 1])), minus)), d0, d1);
            dp[2 * k] = __float_as_uint(d0);
            dp[2 * k + 1] = __float_as_uint(d1);
            pk[k] = pack_bf16x2(d0, d1);
          }
          tmem_st_32x16(t_row + kDs + (step & 1) * 64 + quarter * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[2 * g + (step & 1)]);
        if (want_table) {
          if (!near) {
            uint64_t sum = pack2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 32; k += 2) sum = add2(sum, pack2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])));
            float s0, s1;
            unpack2(sum, s0, s1);
            ds_far += s0 + s1;
          } else {
            // diagonal e holds distance base + e; lane 31 completes one of them per column, the others stay behind at the end
            const int base = pmin + quad * 32 - k0 - 31;
            float run = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float from = __shfl_up_sync(0xffffffffu, run, 1);
              run = (lane == 0 ? 0.f : from) + __uint_as_float(dp[k]);
              if (lane == 31) diag[31 + 31 - k] = run;
            }
            if (lane < 31) diag[lane] = run;
            __syncwarp();
#pragma unroll
            for (int e0 = 0; e0 < 64; e0 += 32) {
              const int e = e0 + lane;
              float v = e < 63 ? diag[e] : 0.f;
              const int bucket = map[kLutFront + base + min(e, 62)];
              // sums over runs of equal buckets; the last lane of a run adds its
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const float v2 = __shfl_up_sync(0xffffffffu, v, o);
                const int b2 = __shfl_up_sync(0xffffffffu, bucket, o);
                if (lane >= o && b2 == bucket) v += v2;
              }
              const int next = __shfl_down_sync(0xffffffffu, bucket, 1);
              if (lane == 31 || next != bucket) my_bins[bucket] += v;
              __syncwarp();
            }
          }
        }
      }
      if (n > 0) {
        NMB_BAND_WAIT(&dq_full[0], n_item & 1, 91);
        if (G::kGroups == 2) NMB_BAND_WAIT(&dq_full[1], n_item & 1, 91);
        ++n_item;
        tc_fence_after();
      }
      if (L::kStage) {
        if (threadIdx.x == 0) store_wait_read();  // the item before has left the tile
        together();
      }
      if (has_cols) {
        __nv_bfloat16* out = band_row(a.dq, a.dq_st, w.b, row, w.h) + quarter * L::kCols;
#pragma unroll
        for (int c = 0; c < L::kCols / 16; ++c) {
          uint32_t v[16];
          if (n > 0) {
            tmem_ld_32x16(t_row + kDq + quarter * L::kCols + c * 16, v);
            if (G::kGroups == 2) {
              uint32_t v2[16];
              tmem_ld_32x16(t_row + kDq + D + quarter * L::kCols + c * 16, v2);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) + __uint_as_float(v2[k]));
            } else {
              tmem_ld_wait();
            }
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = 0;
          }
          if (L::kStage) {
            stage_bf16_16(smem + L::kOut, r, quarter * L::kCols + c * 16, v, a.scale);
          } else if (valid) {
            store_bf16_16(out + c * 16, v, a.scale);
          }
        }
      }
      if (L::kStage) {
        fence_proxy_async_smem();
        together();
        if (threadIdx.x == 0) {
          tma_store_4d(&p.dq_map, smem + L::kOut, 0, w.q0, w.h, w.b);
          store_commit();
        }
      }
      if (n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_empty);
      }
      if (want_table) {
        const float last = warp_sum(ds_far);
        if (lane == 0) my_bins[a.buckets - 1] += last;
        together();
        for (int b = threadIdx.x; b < a.buckets; b += kComputeWarps * 32) {
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < kComputeWarps; ++k) {
            sum += bins[k * kMaxBuckets + b];
            bins[k * kMaxBuckets + b] = 0.f;
          }
          p.dtable_part[((static_cast<long long>(w.b) * a.Hq + w.h) * p.n_qt + w.q0 / 128) * a.buckets + b] = sum;
        }
        together();
      }
    }
    if (L::kStage) store_wait();
  }

  if (*abort_flag != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- dK and dV ----
// A CTA works on one key tile of one key head, over the query heads of the group and the query tiles that see it, or on a
// piece of them.  S^T = K Q^T and dP^T = V dO^T have keys as rows, so P^T and dS^T go straight back to tensor memory as A
// operands of dV += P^T dO and dK += dS^T Q; they overwrite what they came from, each thread its own columns.  TMEM: S^T 0,
// dP^T 128, dV 256, dK 256 + D; those of the second group at 384.
template <int D>
struct BandDkvSmem {
  static constexpr int kSlabs = (D + 63) / 64;
  static constexpr int kTile = kSlabs * 16384;
  static constexpr int kStages = D == 64 ? 3 : 2;    // Q, dO and the column statistics
  static constexpr int kKvStages = D == 64 ? 2 : 1;  // K, V
  static constexpr int kK = 0;
  static constexpr int kRing = 2 * kKvStages * kTile;
  static constexpr bool kStage = D == 64;  // dV, dK through shared memory
  static constexpr int kOut = kRing + 2 * kStages * kTile;
  static constexpr int kStat = kOut + (kStage ? 2 * kTile : 0);
  static constexpr int kBar = kStat + kStages * kStatBlock * 4;
  static constexpr int kNumBars = 4 * kStages + 2 * kKvStages + 11;
  static constexpr int kLut = kBar + ((kNumBars * 8 + 16 + 127) / 128) * 128;
  static constexpr int kCols = D == 96 ? 32 : D / 4;  // as in the dQ kernel
};

struct DkvItem {
  int b, hk, kv0;
  int slot;        // where a piece goes; -1: the whole tile
  int first_qt, per_head;
  int from, to;    // steps of this piece: step / per_head = head of the group, step % per_head = query tile
};
// The n-th of the key tiles without sinks.  The first that a row sees comes first: it has the most rows; tiles before it (which
// a shard's window has left behind) have none and come last.
__host__ __device__ __forceinline__ int other_tile(const BandBwdParams& p, int n) {
  const int seen = p.first_seen + n;
  return seen < p.n_kt ? seen : seen - p.n_kt + p.sink_tiles;
}
__device__ __forceinline__ DkvItem dkv_item(const BandBwdParams& p, int item) {
  const BandArgs& a = p.a;
  DkvItem w;
  const int sink_items = p.sink_tiles * p.sink_pieces * a.Hkv * a.B;
  const bool sink = item < sink_items;
  const int rank = sink ? item : item - sink_items, pieces = sink ? p.sink_pieces : p.pieces;
  int hb, piece;
  const int at = p.by_hkvb.quot(rank, hb);
  const int nth = (sink ? p.by_sink_pieces : p.by_pieces).quot(at, piece);
  const int tile = sink ? nth : other_tile(p, nth);
  w.slot = pieces == 1 ? -1 : sink ? rank : (p.sink_pieces > 1 ? sink_items : 0) + rank;
  w.b = p.by_hkv.quot(hb, w.hk);
  w.kv0 = tile * 128;
  const int first = max(0, w.kv0 - a.q_pos0);
  const int last = w.kv0 < a.sinks ? a.Sq - 1 : min(a.Sq - 1, min(w.kv0 + 127, a.Skv - 1) - a.q_pos0 + a.window - 1);
  w.first_qt = first >> 7;
  w.per_head = first <= last ? (last >> 7) - w.first_qt + 1 : 0;
  const int n = w.per_head * static_cast<int>(p.by_group.d);
  const int len = (sink ? p.by_sink_pieces : p.by_pieces).quot(n + pieces - 1);
  w.from = min(n, piece * len);
  w.to = min(n, w.from + len);
  return w;
}

// The steps of a CTA, one after the other through its items; items without steps are left out.
struct DkvWalk {
  int round, step;
  DkvItem w;
  __device__ __forceinline__ bool open(const BandBwdParams& p, int from_round) {
    const int rounds = (p.n_items + gridDim.x - 1) / gridDim.x;
    for (round = from_round; round < rounds; ++round) {
      const int item = item_of_round(round);
      if (item >= p.n_items) continue;
      w = dkv_item(p, item);
      step = w.from;
      if (w.from < w.to) return true;
    }
    return false;
  }
  __device__ __forceinline__ bool next(const BandBwdParams& p) {
    if (++step < w.to) return true;
    return open(p, round + 1);
  }
  __device__ __forceinline__ bool first() const { return step == w.from; }
  __device__ __forceinline__ bool last() const { return step == w.to - 1; }
};

template <int D>
__global__ void __launch_bounds__(kBandThreads, 1) band_bwd_dkv_kernel(const __grid_constant__ BandBwdParams p) {
  using L = BandDkvSmem<D>;
  using G = BandGroups<D>;
  constexpr int NS = L::kSlabs, ST = L::kStages, KS = L::kKvStages;
  constexpr uint32_t kDp = 128, kDv = 256, kDk = 256 + D;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;              // [ST]
  uint64_t* q_empty = bars + ST;        // [ST] the issuers + the warps that read the statistics
  uint64_t* do_full = bars + 2 * ST;    // [ST]
  uint64_t* do_empty = bars + 3 * ST;   // [ST] the issuers
  uint64_t* kv_full = bars + 4 * ST;    // [KS]
  uint64_t* kv_empty = kv_full + KS;    // [KS] the issuers
  uint64_t* s_full = kv_empty + KS;     // [groups], as all that follow
  uint64_t* dp_full = s_full + 2;
  uint64_t* p_full = s_full + 4;
  uint64_t* ds_full = s_full + 6;
  uint64_t* acc_full = s_full + 8;
  uint64_t* acc_empty = s_full + 10;    // one for both
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const BandArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entries = lut_entries(p.t_last);
  float* lut = reinterpret_cast<float*>(smem + L::kLut);
  uint8_t* map = reinterpret_cast<uint8_t*>(lut + entries);

  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) report_status(a.status, kBadArgument, 100);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], G::kGroups + kComputeWarps);
      mbar_init(&do_full[s], 1);
      mbar_init(&do_empty[s], G::kGroups);
    }
    for (int s = 0; s < KS; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], G::kGroups);
    }
    for (int g = 0; g < G::kGroups; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&dp_full[g], 1);
      mbar_init(&p_full[g], G::kWarps);
      mbar_init(&ds_full[g], G::kWarps);
      mbar_init(&acc_full[g], 1);
    }
    mbar_init(acc_empty, kComputeWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) build_bucket_map(a, p.t_last, map, threadIdx.x, kBandThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns were allocated, so they begin at 0; said as a constant the addresses need no moves to uniform registers.
  constexpr uint32_t tmem = 0;
  if (threadIdx.x == 0 && *tmem_slot != 0) {
    report_status(a.status, kBadArgument, 75);
    *abort_flag = 1;
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&p.q_map);
    tma_prefetch_desc(&p.k_map);
    tma_prefetch_desc(&p.v_map);
    tma_prefetch_desc(&p.do_map);
  }
  pdl_enter();
  const int group = static_cast<int>(p.by_group.d);

  if (warp >= kComputeWarps) {
    NMB_BAND_FEW_REGISTERS;
    if (warp == kLoadWarp && lane == 0) {
      // ---------------------------------------------------------- producer --
      const uint32_t stat_bytes = a.table == nullptr ? 1024 : 2048;
      DkvWalk x;
      int n = 0, n_item = 0;
      for (bool more = x.open(p, 0); more; more = x.next(p), ++n) {
        if (x.first()) {
          const int ks = n_item % KS, kuse = n_item / KS;
          if (kuse > 0 && !band_wait(&kv_empty[ks], (kuse - 1) & 1, abort_flag, a.status, 101)) break;
          ++n_item;
          mbar_expect_tx(&kv_full[ks], 2 * L::kTile);
#pragma unroll
          for (int c = 0; c < NS; ++c) {
            uint8_t* dst = smem + L::kK + 2 * ks * L::kTile + c * 16384;
            tma_load_4d(dst, &p.k_map, &kv_full[ks], c * 64, x.w.kv0, x.w.hk, x.w.b);
            tma_load_4d(dst + L::kTile, &p.v_map, &kv_full[ks], c * 64, x.w.kv0, x.w.hk, x.w.b);
          }
        }
        const int st = n % ST, use = n / ST;
        const int h = x.w.hk * group + x.step / x.w.per_head, qt = x.w.first_qt + x.step % x.w.per_head;
        uint8_t* const to_q = smem + L::kRing + 2 * st * L::kTile;
        auto load = [&](uint8_t* dst, const CUtensorMap* from, uint64_t* bar) {
#pragma unroll
          for (int c = 0; c < NS; ++c) tma_load_4d(dst + c * 16384, from, bar, c * 64, qt * 128, h, x.w.b);
        };
        // dO's place is free after dV, long before Q's is: what is loaded late is half as much
        if (use > 0 && !band_wait(&do_empty[st], (use - 1) & 1, abort_flag, a.status, 104)) break;
        mbar_expect_tx(&do_full[st], L::kTile);
        load(to_q + L::kTile, &p.do_map, &do_full[st]);
        if (use > 0 && !band_wait(&q_empty[st], (use - 1) & 1, abort_flag, a.status, 102)) break;
        mbar_expect_tx(&q_full[st], L::kTile + stat_bytes);
        load(to_q, &p.q_map, &q_full[st]);
        bulk_load(smem + L::kStat + st * kStatBlock * 4,
                  p.stat + ((static_cast<long long>(x.w.b) * a.Hq + h) * p.n_qt + qt) * kStatBlock, stat_bytes, &q_full[st]);
      }
    } else if (warp >= kMmaWarp && warp < kMmaWarp + G::kGroups) {
      // -------------------------------------------------------- MMA issuer --
      // For step n: dV with P^T, then S^T of the next step in its place; dK with dS^T, then dP^T of the next step.  The tensor
      // core has the products of one operand to work on while the compute warps make the other.  Where there is room for two
      // query tiles only, the next but one is loaded into this one's place after dK: dK goes before S^T when it can.
      constexpr uint32_t idesc_s = make_idesc_bf16(128, G::kWidth, false, false);
      constexpr uint32_t idesc_d = make_idesc_bf16(128, D, false, true);
      const int g = warp - kMmaWarp;
      const uint32_t kv = smem_u32(smem + L::kK), ring = smem_u32(smem + L::kRing) + g * G::kWidth * 128;  // this group's queries
      const uint32_t t_s = tmem + g * G::kWidth, t_dv = tmem + kDv + g * 128, t_dk = tmem + kDk + g * 128;
      const bool one = elect_one();
      DkvWalk x;
      uint32_t n = 0, n_item = 0;  // step, item of `x`
      bool more = x.open(p, 0);
      auto q_bar = [&](uint32_t i) { return BandBar{&q_full[i % ST], (i / ST) & 1}; };
      auto do_bar = [&](uint32_t i) { return BandBar{&do_full[i % ST], (i / ST) & 1}; };
      auto scores = [&](uint32_t i, uint32_t item) {
        if (one) {
          mma_scores<D>(t_s, desc_k(kv + 2 * (item % KS) * L::kTile), desc_k(ring + 2 * (i % ST) * L::kTile), idesc_s);
          tc_commit(&s_full[g]);
        }
      };
      auto dps = [&](uint32_t i, uint32_t item, bool last) {
        if (one) {
          mma_scores<D>(t_s + kDp, desc_k(kv + (2 * (item % KS) + 1) * L::kTile), desc_k(ring + (2 * (i % ST) + 1) * L::kTile), idesc_s);
          tc_commit(&dp_full[g]);
          if (last) tc_commit(&kv_empty[item % KS]);
        }
      };
      bool ok = more && band_wait_all(abort_flag, a.status, 103, BandBar{&kv_full[0], 0}, q_bar(0), do_bar(0));
      if (ok) {
        tc_fence_after();
        scores(0, 0);
        dps(0, 0, x.last());
      }
      while (ok && more) {
        DkvWalk y = x;
        const bool ahead = y.next(p), fresh = ahead && y.first(), y_last = ahead && y.last();
        const bool x_first = x.first(), x_last = x.last();
        const uint32_t n_item2 = n_item + fresh, sq = ring + 2 * (n % ST) * L::kTile;
        if (x_first && n_item > 0 && !band_wait(acc_empty, (n_item - 1) & 1, abort_flag, a.status, 108)) break;
        if (!band_wait(&p_full[g], n & 1, abort_flag, a.status, 109)) break;
        tc_fence_after();
        if (one) {
          mma_apply<G::kWidth / 16, 2, 32>(t_dv, t_s, desc_mn(sq + L::kTile), idesc_d, x_first);
          tc_commit(&do_empty[n % ST]);
        }
        const BandBar ds_bar{&ds_full[g], n & 1}, k_bar{&kv_full[n_item2 % KS], (n_item2 / KS) & 1};
        const int late = !ahead  ? 0
                         : fresh ? band_wait_first(abort_flag, a.status, 106, ds_bar, k_bar, q_bar(n + 1))
                                 : band_wait_first(abort_flag, a.status, 106, ds_bar, q_bar(n + 1));
        if (late == 2) break;
        if (late == 0) {
          if (ahead) {
            tc_fence_after();
            scores(n + 1, n_item2);
          }
          if (!band_wait(ds_bar.bar, ds_bar.parity, abort_flag, a.status, 111)) break;
        }
        tc_fence_after();
        if (one) {
          mma_apply<G::kWidth / 16, 2, 32>(t_dk, t_s + kDp, desc_mn(sq), idesc_d, x_first);
          tc_commit(&q_empty[n % ST]);
          if (x_last) tc_commit(&acc_full[g]);
        }
        if (ahead) {
          if (late == 1) {
            if (!band_wait_all(abort_flag, a.status, 107, k_bar, q_bar(n + 1))) break;
            tc_fence_after();
            scores(n + 1, n_item2);
          }
          if (!band_wait(do_bar(n + 1).bar, do_bar(n + 1).parity, abort_flag, a.status, 105)) break;
          tc_fence_after();
          dps(n + 1, n_item2, y_last);
        }
        x = y;
        more = ahead;
        n_item = n_item2;
        ++n;
      }
    }
  } else {
    NMB_BAND_MORE_REGISTERS;
    // ------------------------------------------------------------ compute --
    const int quad = warp & 3, quarter = warp >> 2;
    const int r = quad * 32 + lane;  // key of the tile == TMEM lane
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const int g = quarter / G::kQuarters;
    const bool has_cols = quarter * L::kCols < D;
    const float sl2 = a.scale * kBandLog2e;
    const int rounds = (p.n_items + gridDim.x - 1) / gridDim.x;
    int n = 0, n_item = 0;
    auto together = [&]() { named_sync(1, kComputeWarps * 32); };
    bool ok = true;
    for (int round = 0; round < rounds; ++round) {
      const int item = item_of_round(round);
      if (item >= p.n_items) continue;
      const DkvItem w = dkv_item(p, item);
      if (w.slot >= 0 && w.per_head == 0) continue;  // no row sees the tile, and none reads its pieces
      const int j = w.kv0 + r;
      int lut_h = -1;
      float far_bias = 0.f;
      const int per_head = max(w.per_head, 1);
      int h = w.hk * group + w.from / per_head, qt = w.first_qt + w.from % per_head - 1;
      for (int step = w.from; step < w.to; ++step, ++n) {
        if (++qt == w.first_qt + w.per_head) {
          qt = w.first_qt;
          ++h;
        }
        const int pmin = a.q_pos0 + qt * 128;
        const int st = n % ST;
        if (a.table != nullptr && h != lut_h) {
          together();  // everyone is done with the table of the head before
          build_lut(a, h, p.t_last, map, lut, threadIdx.x, kComputeWarps * 32);
          together();
          far_bias = lut[entries - 1];
          lut_h = h;
        }
        // the statistics come with Q and dO; the scores do after them
        NMB_BAND_WAIT(&q_full[st], (n / ST) & 1, 112);
        NMB_BAND_WAIT(&s_full[g], n & 1, 113);
        tc_fence_after();
        uint32_t s[32];
        tmem_ld_32x32(t_row + quarter * 32, s);
        tmem_ld_wait();
        const float* stat = reinterpret_cast<const float*>(smem + L::kStat) + st * kStatBlock + quarter * 32;
        const bool added = a.table != nullptr && (pmin - (w.kv0 + 127) < p.t_last || fabsf(far_bias) > 1e30f);
        const bool whole = w.kv0 + 127 <= pmin && w.kv0 + 127 < a.Skv && (pmin + 127 - w.kv0 < a.window || w.kv0 + 127 < a.sinks);
        if (!added && qt * 128 + 128 <= a.Sq) {  // as in the dQ kernel
          exps32<true>(s, pack2(sl2, sl2), stat);
        } else if (!added) {
          exps32<false>(s, pack2(sl2, sl2), stat);
        } else {
          const float* at = lut + kLutFront + min(pmin - j, p.t_last + 128) + quarter * 32;
#pragma unroll
          for (int k = 0; k < 32; ++k)
            s[k] = __float_as_uint(ex2((fmaf(__uint_as_float(s[k]), sl2, at[k]) - stat[256 + k]) - stat[384 + k]));
        }
        if (!whole) {
          const int c0 = quarter * 32, lo = j < a.Skv ? j - pmin : 128, hi = j < a.sinks ? 128 : j - pmin + a.window;
          const uint32_t see = low_bits(hi - c0) & ~low_bits(lo - c0);
          if (!__all_sync(0xffffffffu, see == ~0u)) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1u)) s[k] = 0;
          }
        }
        {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) pk[k] = pack_bf16x2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
          tmem_st_32x16(t_row + quarter * 32, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
        NMB_BAND_WAIT(&dp_full[g], n & 1, 115);
        tc_fence_after();
        uint32_t dp[32];
        tmem_ld_32x32(t_row + kDp + quarter * 32, dp);
        tmem_ld_wait();
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          const ulonglong2 dd = *reinterpret_cast<const ulonglong2*>(stat + 128 + 2 * k);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int e = 2 * (k + i);
            float d0, d1;
            unpack2(mul2(pack2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                         fma2(i ? dd.y : dd.x, pack2(-1.f, -1.f), pack2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])))), d0, d1);
            pk[k + i] = pack_bf16x2(d0, d1);
          }
        }
        tmem_st_32x16(t_row + kDp + quarter * 32, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ds_full[g]);
          mbar_arrive(&q_empty[st]);
        }
      }
      const bool any = w.from < w.to;
      if (any) {
        NMB_BAND_WAIT(&acc_full[0], n_item & 1, 117);
        if (G::kGroups == 2) NMB_BAND_WAIT(&acc_full[1], n_item & 1, 117);
        ++n_item;
        tc_fence_after();
      }
      const bool staged = L::kStage && w.slot < 0;
      if (staged) {
        if (threadIdx.x == 0) store_wait_read();  // the item before has left the tiles
        together();
      }
      if (has_cols) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          const float mul = which == 0 ? 1.f : a.scale;
          __nv_bfloat16* out = band_row(which == 0 ? a.dv : a.dk, which == 0 ? a.dv_st : a.dk_st, w.b, j, w.hk) + quarter * L::kCols;
          float* part = p.part + ((static_cast<long long>(w.slot) * 2 + which) * 128 + r) * D + quarter * L::kCols;
#pragma unroll
          for (int c = 0; c < L::kCols / 16; ++c) {
            uint32_t v[16];
            if (any) {
              const uint32_t at = t_row + (which == 0 ? kDv : kDk) + quarter * L::kCols + c * 16;
              tmem_ld_32x16(at, v);
              if (G::kGroups == 2) {
                uint32_t v2[16];
                tmem_ld_32x16(at + 128, v2);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) + __uint_as_float(v2[k]));
              } else {
                tmem_ld_wait();
              }
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) v[k] = 0;
            }
            if (w.slot >= 0) {
              st_global_32(part + c * 16, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
              st_global_32(part + c * 16 + 8, v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]);
            } else if (L::kStage) {
              stage_bf16_16(smem + L::kOut + which * L::kTile, r, quarter * L::kCols + c * 16, v, mul);
            } else if (j < a.Skv) {
              store_bf16_16(out + c * 16, v, mul);
            }
          }
        }
      }
      if (staged) {
        fence_proxy_async_smem();
        together();
        if (threadIdx.x == 0) {
          tma_store_4d(&p.dv_map, smem + L::kOut, 0, w.kv0, w.hk, w.b);
          tma_store_4d(&p.dk_map, smem + L::kOut + L::kTile, 0, w.kv0, w.hk, w.b);
          store_commit();
        }
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
      }
    }
    if (L::kStage) store_wait();
  }

  if (*abort_flag != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Steps (query tiles times heads) of a key tile, as in dkv_item.
__host__ __device__ __forceinline__ int dkv_steps(const BandArgs& a, int tile) {
  const int kv0 = tile * 128, first = max(0, kv0 - a.q_pos0);
  const int last = kv0 < a.sinks ? a.Sq - 1 : min(a.Sq - 1, min(kv0 + 127, a.Skv - 1) - a.q_pos0 + a.window - 1);
  return first <= last ? ((last >> 7) - (first >> 7) + 1) * (a.Hq / a.Hkv) : 0;
}

// What is left after them, in one launch.  The first `sum_blocks` blocks add the pieces of split key tiles, in order: eight
// values of a row per thread.  The others add the table's gradient, over batches and query tiles in a fixed order: a warp per
// (head, bucket).
__global__ void __launch_bounds__(256) band_finish_kernel(const __grid_constant__ BandBwdParams p, int sum_blocks) {
  pdl_enter();
  const BandArgs& a = p.a;
  if (static_cast<int>(blockIdx.x) >= sum_blocks) {
    const int at = (blockIdx.x - sum_blocks) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (at >= a.Hq * a.buckets) return;
    const int h = at / a.buckets, bucket = at % a.buckets;
    float acc = 0.f;
    for (int b = 0; b < a.B; ++b)
      for (int t = lane; t < p.n_qt; t += 32)
        acc += p.dtable_part[((static_cast<long long>(b) * a.Hq + h) * p.n_qt + t) * a.buckets + bucket];
    acc = warp_sum(acc);
    if (lane == 0) {
      if (a.dtable_fp32) {
        float* out = static_cast<float*>(a.dtable) + at;
        *out = acc;
      } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.dtable) + at;
        *out = __float2bfloat16(acc);
      }
    }
    return;
  }
  const int n_hb = a.Hkv * a.B, per_row = a.d / 8;
  const int sink_items = p.sink_tiles * p.sink_pieces * n_hb;
  const int first = p.sink_pieces > 1 ? 0 : p.sink_tiles, end = p.pieces > 1 ? p.n_kt : p.sink_tiles;
  long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int c8 = idx % per_row;
  idx /= per_row;
  const int r = idx % 128;
  idx /= 128;
  const int which = idx % 2;
  idx /= 2;
  const int hb = idx % n_hb, nth = first + static_cast<int>(idx / n_hb);
  if (nth >= end) return;
  const bool sink = nth < p.sink_tiles;
  const int j = (sink ? nth : other_tile(p, nth - p.sink_tiles)) * 128 + r;
  if (j >= a.Skv) return;
  const int pieces = dkv_steps(a, j >> 7) == 0 ? 0 : sink ? p.sink_pieces : p.pieces;
  const int slot0 = sink ? nth * pieces * n_hb + hb
                         : (p.sink_pieces > 1 ? sink_items : 0) + (nth - p.sink_tiles) * pieces * n_hb + hb;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < pieces; ++i) {
    const float4* src = reinterpret_cast<const float4*>(
        p.part + ((static_cast<long long>(slot0 + i * n_hb) * 2 + which) * 128 + r) * a.d + c8 * 8);
    const float4 u = src[0], v = src[1];
    x[0] += u.x; x[1] += u.y; x[2] += u.z; x[3] += u.w;
    x[4] += v.x; x[5] += v.y; x[6] += v.z; x[7] += v.w;
  }
  const float mul = which == 0 ? 1.f : a.scale;
  __nv_bfloat16* out = 
      band_row(which == 0 ? a.dv : a.dk, which == 0 ? a.dv_st : a.dk_st, hb / a.Hkv, j, hb % a.Hkv) + c8 * 8;
  *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(x[0] * mul, x[1] * mul), pack_bf16x2(x[2] * mul, x[3] * mul),
                                              pack_bf16x2(x[4] * mul, x[5] * mul), pack_bf16x2(x[6] * mul, x[7] * mul));
}

// Into how many pieces the steps of a key tile are cut.  Cutting costs the pieces' way through memory and a launch; not
// cutting leaves SMs idle when there are few key tiles and heads (grouped heads), or when the tiles that hold sinks, which
// every query sees, take many times as long as the others.  The estimate, in steps: what the most loaded of five of the SMs
// gets, with two steps for an item's beginning and end, D / 32 more for a piece (writing 128 KB of fp32 sums took as long
// as 2.6 steps at D = 128, and they are read again) and two for the launch that adds them up.  Over 300 shapes its choice was
// 0.4 percent behind the best one of all SMs' loads, never cutting 58 percent.
static void plan_pieces(BandBwdParams& p) {
  const BandArgs& a = p.a;
  const int sms = std::max(1, sm_count()), n_hb = a.Hkv * a.B, piece_cost = 2 + a.d / 32;
  constexpr int kMaxRounds = 16;  // looked at one by one; cutting gains nothing where there are more
  int longest = 1, longest_sink = 1;
  for (int t = 0; t < p.n_kt; ++t) {
    int& most = t < p.sink_tiles ? longest_sink : longest;
    most = std::max(most, dkv_steps(a, t));
  }
  const int others = p.n_kt - p.sink_tiles;
  p.pieces = p.sink_pieces = 1;
  long long best = LLONG_MAX;
  const long long looked_at = static_cast<long long>(kMaxRounds) * sms;
  for (int c : {1, 2, 3, 4, 6, 8, 12, 16}) {
    if (c > 1 && (c > longest || static_cast<long long>(others) * c * n_hb > looked_at)) break;
    const int piece = (longest + c - 1) / c;
    const int even = p.sink_tiles == 0 ? 1 : std::min(64, (longest_sink + std::max(piece, 4) - 1) / std::max(piece, 4));
    for (int cs : {1, even}) {
      const long long sink_items = static_cast<long long>(p.sink_tiles) * cs * n_hb;
      const long long items = sink_items + static_cast<long long>(others) * c * n_hb;
      if (cs > 1 && sink_items > looked_at) break;
      const int of_sink = (longest_sink + cs - 1) / cs + (cs > 1 ? piece_cost : 2), of_other = piece + (c > 1 ? piece_cost : 2);
      const int rounds = static_cast<int>(std::min<long long>((items + sms - 1) / sms, kMaxRounds));
      long long cost = 0;
      for (int part = 0; part < 5; ++part) {
        const int sm = part * (sms - 1) / 4;
        int load = 0;
        for (int round = 0; round < rounds; ++round) {
          const long long i = static_cast<long long>(round) * sms + ((round & 1) ? sms - 1 - sm : sm);
          if (i >= items) break;
          if (i < sink_items) load += of_sink;
          else if (const int steps = dkv_steps(a, other_tile(p, static_cast<int>((i - sink_items) / n_hb / c))))
            load += (steps + c - 1) / c + (c > 1 ? piece_cost : 2);
        }
        cost = std::max<long long>(cost, load);
      }
      const long long sinks_after = std::max<long long>(0, sink_items - looked_at), after = std::max<long long>(0, items - looked_at);
      cost += (sinks_after * of_sink + (after - sinks_after) * of_other) / sms;
      if (c > 1 || (cs > 1 && p.sink_tiles > 0)) cost += 2;
      if (cost < best) {
        best = cost;
        p.pieces = c;
        p.sink_pieces = cs;
      }
      if (even == 1) break;
    }
  }
}

struct BandScratch {
  long long stat, part, dtable, total;  // floats
};
static BandScratch plan_bwd(BandBwdParams& p, const BandArgs& a, const BandPlan* plan = nullptr) {
  p.a = a;
  p.n_qt = (a.Sq + 127) / 128;
  p.n_kt = (a.Skv + 127) / 128;
  p.t_last = a.buckets < 2 ? 0 : a.limit[a.buckets - 2];
  p.sink_tiles = a.window >= a.q_pos0 + a.Sq ? 0 : std::min((std::min(a.sinks, a.Skv) + 127) / 128, p.n_kt);
  p.first_seen = std::min(std::max(p.sink_tiles, std::max(0, a.q_pos0 - a.window + 1) >> 7), p.n_kt - (p.n_kt > p.sink_tiles));
  if (plan == nullptr) {
    plan_pieces(p);
  } else {
    p.sink_pieces = plan->sink_pieces;
    p.pieces = plan->pieces;
  }
  p.by_hqb = FastDiv(a.Hq * a.B);
  p.by_hq = FastDiv(a.Hq);
  p.by_group = FastDiv(a.Hq / a.Hkv);
  p.by_hkvb = FastDiv(a.Hkv * a.B);
  p.by_hkv = FastDiv(a.Hkv);
  p.by_sink_pieces = FastDiv(p.sink_pieces);
  p.by_pieces = FastDiv(p.pieces);
  const long long n_hb = static_cast<long long>(a.Hkv) * a.B;
  const long long slots = (p.sink_pieces > 1 ? p.sink_tiles * p.sink_pieces * n_hb : 0) +
                          (p.pieces > 1 ? (p.n_kt - p.sink_tiles) * p.pieces * n_hb : 0);
  BandScratch w;
  w.stat = static_cast<long long>(a.B) * a.Hq * p.n_qt * kStatBlock;
  w.part = slots * 256 * a.d;
  w.dtable = static_cast<long long>(a.B) * a.Hq * p.n_qt * a.buckets;
  w.total = w.stat + w.part + w.dtable;
  return w;
}

template <int D>
static cudaError_t launch_band_bwd(BandBwdParams& p, long long dq_items, long long dkv_items, bool split, cudaStream_t s) {
  const int lut = p.a.table == nullptr ? 0 : lut_bytes(p.t_last, 1);
  cudaError_t e = launch_pdl(band_stat_kernel<D>, dim3(static_cast<unsigned>(dq_items * stat_blocks<D>())), dim3(256), 0, s, p);
  if (e != cudaSuccess) return e;
  p.n_items = static_cast<int>(dq_items);
  e = launch_pdl(band_bwd_dq_kernel<D>, dim3(std::min(p.n_items, sm_count())), dim3(kBandThreads),
                             BandDqSmem<D>::kLut + lut + (p.a.dtable == nullptr ? 0 : BandDqSmem<D>::kBins), s, p);
  if (e != cudaSuccess) return e;
  p.n_items = static_cast<int>(dkv_items);
  e = launch_pdl(band_bwd_dkv_kernel<D>, dim3(std::min(p.n_items, sm_count())), dim3(kBandThreads),
                 BandDkvSmem<D>::kLut + lut, s, p);
  const int tiles = !split ? 0 : (p.pieces > 1 ? p.n_kt : p.sink_tiles) - (p.sink_pieces > 1 ? 0 : p.sink_tiles);
  const long long sum_blocks = static_cast<long long>(tiles) * p.a.Hkv * p.a.B * (D / 8);  // 2 * 128 rows of D / 8 octets, 256 a block
  const int table_blocks = p.a.dtable == nullptr ? 0 : (p.a.Hq * p.a.buckets + 7) / 8;
  if (e == cudaSuccess && sum_blocks + table_blocks > 0)
    e = launch_pdl(band_finish_kernel, dim3(static_cast<unsigned>(sum_blocks + table_blocks)), dim3(256), 0, s, p,
                   static_cast<int>(sum_blocks));
  return e;
}

}  // namespace nmb

using namespace nmb;

static std::atomic<long long> g_band_launches{0};

extern "C" long long nmb_band_launches() { return g_band_launches.load(); }

static int band_check(const BandArgs* a) {
  if (a->d != 64 && a->d != 96 && a->d != 128) return kBadArgument;
  if (a->B < 1 || a->Hkv < 1 || a->Hq % a->Hkv != 0 || a->Sq < 1 || a->Skv < 1) return kBadArgument;
  if (a->q_pos0 < 0 || a->window < 1 || a->sinks < 0 || !(a->scale > 0.f)) return kBadArgument;
  if (a->table != nullptr && (a->buckets < 2 || a->buckets > kMaxBuckets || a->limit[a->buckets - 2] > kMaxDistance)) return kBadArgument;
  auto aligned = [](const void* ptr, const BandStride& t, int bytes) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && t.b * 2 % bytes == 0 && t.s * 2 % bytes == 0 && t.h * 2 % bytes == 0;
  };
  // tile loads want 16 bytes; results are written in pieces of 32
  if (reinterpret_cast<uintptr_t>(a->o_rest) % 32 != 0) return kBadArgument;
  if (!aligned(a->q, a->q_st, 16) || !aligned(a->k, a->k_st, 16) || !aligned(a->v, a->v_st, 16) || !aligned(a->o, a->o_st, 32) ||
      !aligned(a->dout, a->dout_st, 16) || !aligned(a->dq, a->dq_st, 32) || !aligned(a->dk, a->dk_st, 32) ||
      !aligned(a->dv, a->dv_st, 32))
    return kBadArgument;
  return 0;
}

static int fwd_check(const BandArgs* a) {
  if (int bad = band_check(a)) return bad;
  if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->o == nullptr || (a->m == nullptr) != (a->l == nullptr)) return kBadArgument;
  if (a->rest_rows < 0 || a->rest_rows > a->Sq || (a->rest_rows > 0 && a->o_rest == nullptr)) return kBadArgument;
  return 0;
}
static int bwd_check(const BandArgs* a) {
  if (int bad = fwd_check(a)) return bad;
  if (a->m == nullptr || a->dout == nullptr || a->dq == nullptr || a->dk == nullptr || a->dv == nullptr || a->scratch == nullptr) return kBadArgument;
  if (a->dtable != nullptr && a->table == nullptr) return kBadArgument;
  return 0;
}

extern "C" int nmb_band_args_size() { return static_cast<int>(sizeof(BandArgs)); }

extern "C" long long nmb_band_bwd_scratch(const BandArgs* a) {
  if (band_check(a)) return 0;
  BandBwdParams p;
  return plan_bwd(p, *a).total;
}

extern "C" int nmb_band_configure() {
  cudaError_t e = cudaSuccess;
  auto opt_in = [&](const void* f, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  };
  const int lut = lut_bytes(kMaxDistance, 2);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<64, false, false>), BandFwdSmem<64>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<64, false, true>), BandFwdSmem<64>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<64, true, false>), BandFwdSmem<64>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<64, true, true>), BandFwdSmem<64>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<96, false, false>), BandFwdSmem<96>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<96, false, true>), BandFwdSmem<96>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<96, true, false>), BandFwdSmem<96>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<96, true, true>), BandFwdSmem<96>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<128, false, false>), BandFwdSmem<128>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<128, false, true>), BandFwdSmem<128>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<128, true, false>), BandFwdSmem<128>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<128, true, true>), BandFwdSmem<128>::kLut + lut);
  const int lut1 = lut_bytes(kMaxDistance, 1);
  opt_in(reinterpret_cast<const void*>(band_bwd_dq_kernel<64>), BandDqSmem<64>::kLut + lut1 + BandDqSmem<64>::kBins);
  opt_in(reinterpret_cast<const void*>(band_bwd_dq_kernel<96>), BandDqSmem<96>::kLut + lut1 + BandDqSmem<96>::kBins);
  opt_in(reinterpret_cast<const void*>(band_bwd_dq_kernel<128>), BandDqSmem<128>::kLut + lut1 + BandDqSmem<128>::kBins);
  opt_in(reinterpret_cast<const void*>(band_bwd_dkv_kernel<64>), BandDkvSmem<64>::kLut + lut1);
  opt_in(reinterpret_cast<const void*>(band_bwd_dkv_kernel<96>), BandDkvSmem<96>::kLut + lut1);
  opt_in(reinterpret_cast<const void*>(band_bwd_dkv_kernel<128>), BandDkvSmem<128>::kLut + lut1);
  return e == cudaSuccess ? 0 : 300 + e;
}

extern "C" long long nmb_band_fwd_scratch(const BandArgs* a) {
  if (band_check(a)) return 0;
  const int pieces = fwd_pieces(*a);
  return pieces == 1 ? 0 : static_cast<long long>((a->Sq + 127) / 128) * a->Hq * a->B * pieces * (128 * a->d + 256);
}

extern "C" int nmb_band_fwd(const BandArgs* a, void* stream) { return nmb_band_fwd_split(a, nullptr, stream); }

extern "C" int nmb_band_fwd_split(const BandArgs* a, float* scratch, void* stream) {
  if (int bad = fwd_check(a)) return bad;
  if (reinterpret_cast<uintptr_t>(scratch) % 32 != 0) return kBadArgument;
  (void)cudaGetLastError();
  BandFwdParams p;
  p.a = *a;
  if (make_band_map(&p.q_map, a->q, a->q_st, a->d, a->Sq, a->Hq, a->B)) return 101;
  if (make_band_map(&p.k_map, a->k, a->k_st, a->d, a->Skv, a->Hkv, a->B)) return 102;
  if (make_band_map(&p.v_map, a->v, a->v_st, a->d, a->Skv, a->Hkv, a->B)) return 103;
  if (make_band_map(&p.o_map, a->o, a->o_st, a->d, a->Sq, a->Hq, a->B)) return 105;
  if (a->rest_rows > 0) {
    const long long row = static_cast<long long>(a->Hq) * a->d;
    if (make_band_map(&p.rest_map, a->o_rest, BandStride{a->rest_rows * row, row, a->d}, a->d, a->rest_rows, a->Hq, a->B)) return 106;
  }
  p.n_qt = (a->Sq + 127) / 128;
  p.t_last = a->table == nullptr ? 0 : a->limit[a->buckets - 2];
  const long long tiles = static_cast<long long>(p.n_qt) * a->Hq * a->B;
  // One tile an item while every tile can have an SM of its own.  From there on pairs: with a window of 256 over 192 tiles 11.0 us
  // where single tiles take 12.9 (D = 64), over 256 tiles 13.6 and 17.6 (D = 96).  Causal rows over 8 to 16 key tiles would be
  // better off as single tiles up to about 300 (192 tiles 19.0 and 15.8 us, 256 tiles 32.9 and 27.9, 320 tiles 33.3 and 36.3): the
  // pairs are one round of long items there.
  p.pair = tiles <= sm_count() ? 0 : (a->Hq / a->Hkv) % 2 == 0 ? 2 : 1;
  p.pieces = scratch == nullptr ? 1 : fwd_pieces(*a);
  p.part = scratch;
  p.by_pieces = FastDiv(p.pieces);
  const long long items = p.pair == 0 ? tiles * p.pieces : p.pair == 2 ? tiles / 2 : static_cast<long long>((p.n_qt + 1) / 2) * a->Hq * a->B;
  if (items > (1 << 30)) return kTooLarge;
  p.n_items = static_cast<int>(items);
  const int heads = p.pair == 2 ? a->Hq / 2 : a->Hq;
  p.by_hb = FastDiv(heads * a->B);
  p.by_heads = FastDiv(heads);
  p.by_group = FastDiv(a->Hq / a->Hkv);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = a->d == 64 ? launch_band_fwd<64>(p, s) : a->d == 96 ? launch_band_fwd<96>(p, s) : launch_band_fwd<128>(p, s);
  if (e == cudaSuccess) ++g_band_launches;
  if (e == cudaSuccess && p.pieces > 1) {
    e = a->d == 64 ? launch_band_join<64>(p, s) : a->d == 96 ? launch_band_join<96>(p, s) : launch_band_join<128>(p, s);
    if (e == cudaSuccess) ++g_band_launches;
  }
  return e == cudaSuccess ? 0 : 400 + e;
}

extern "C" int nmb_band_bwd_plan(const BandArgs* a, BandPlan* plan) {
  if (int bad = band_check(a)) return bad;
  BandBwdParams p;
  plan->scratch = plan_bwd(p, *a).total;
  plan->sink_pieces = p.sink_pieces;
  plan->pieces = p.pieces;
  return 0;
}

extern "C" int nmb_band_bwd(const BandArgs* a, void* stream) {
  if (int bad = bwd_check(a)) return bad;
  BandPlan plan;
  if (int bad = nmb_band_bwd_plan(a, &plan)) return bad;
  return nmb_band_bwd_planned(a, &plan, stream);
}

extern "C" int nmb_band_bwd_planned(const BandArgs* a, const BandPlan* plan, void* stream) {
  if (int bad = bwd_check(a)) return bad;
  (void)cudaGetLastError();
  BandBwdParams p;
  const BandScratch w = plan_bwd(p, *a, plan);
  p.stat = a->scratch;
  p.part = p.stat + w.stat;
  p.dtable_part = p.part + w.part;
  if (make_band_map(&p.q_map, a->q, a->q_st, a->d, a->Sq, a->Hq, a->B)) return 101;
  if (make_band_map(&p.k_map, a->k, a->k_st, a->d, a->Skv, a->Hkv, a->B)) return 102;
  if (make_band_map(&p.v_map, a->v, a->v_st, a->d, a->Skv, a->Hkv, a->B)) return 103;
  if (make_band_map(&p.do_map, a->dout, a->dout_st, a->d, a->Sq, a->Hq, a->B)) return 104;
  if (make_band_map(&p.dq_map, a->dq, a->dq_st, a->d, a->Sq, a->Hq, a->B)) return 107;
  if (make_band_map(&p.dk_map, a->dk, a->dk_st, a->d, a->Skv, a->Hkv, a->B)) return 108;
  if (make_band_map(&p.dv_map, a->dv, a->dv_st, a->d, a->Skv, a->Hkv, a->B)) return 109;
  const long long n_hb = static_cast<long long>(a->Hkv) * a->B;
  const long long dq_items = static_cast<long long>(p.n_qt) * a->Hq * a->B;
  const long long dkv_items = (static_cast<long long>(p.sink_tiles) * p.sink_pieces +
                               static_cast<long long>(p.n_kt - p.sink_tiles) * p.pieces) * n_hb;
  if (dq_items > (1 << 30) || dkv_items > (1 << 30)) return kTooLarge;
  const bool split = (p.sink_pieces > 1 && p.sink_tiles > 0) || p.pieces > 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->d == 64 ? launch_band_bwd<64>(p, dq_items, dkv_items, split, s)
                      : a->d == 96 ? launch_band_bwd<96>(p, dq_items, dkv_items, split, s)
                                   : launch_band_bwd<128>(p, dq_items, dkv_items, split, s);
  if (e == cudaSuccess) g_band_launches += 3 + (split || a->dtable != nullptr);
  return e == cudaSuccess ? 0 : 500 + e;
}
