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
#include "common.cuh"

#include <algorithm>

namespace nmb {

constexpr float kBandLog2e = 1.4426950408889634f;
constexpr int kMaxBuckets = 128;
constexpr int kMaxDistance = 2048;
constexpr float kBiasLimit = 3.0e38f;  // finite biases stay finite after the change to base 2

struct BandStride {
  long long b, s, h;  // elements; head_dim is contiguous
};

// Arguments of both passes, laid out as in ops/band_attention.py: the pointers of a call, then what its shapes fix.
struct BandArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  const __nv_bfloat16* dout;
  __nv_bfloat16 *dq, *dk, *dv;
  float* m;              // [B, Hq, Sq]
  float* l;              // [B, Hq, Sq]
  float* scratch;        // nmb_band_bwd_scratch() floats, backward only
  const void* table;     // [Hq, buckets] bf16 or fp32; null without a bias
  void* dtable;          // [Hq, buckets]; null when it is not wanted
  int* status;
  int table_fp32, dtable_fp32, accumulate;  // accumulate: dtable is added to
  int pad;
  BandStride q_st, k_st, v_st, o_st, dout_st, dq_st, dk_st, dv_st;
  int B, Hq, Hkv, Sq, Skv, d;
  int q_pos0, window, sinks, buckets;
  float scale;
  int pad2;
  unsigned short limit[kMaxBuckets];  // first distance of bucket b + 1
};

__device__ __forceinline__ float table_at(const BandArgs& p, int h, int b) {
  const long long at = static_cast<long long>(h) * p.buckets + b;
  return p.table_fp32 ? static_cast<const float*>(p.table)[at]
                      : __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[at]);
}
// a table entry in the base-2 exponent domain
__device__ __forceinline__ float bias_log2(float x) {
  const float y = x * kBandLog2e;
  return isinf(x) ? x : fminf(fmaxf(y, -kBiasLimit), kBiasLimit);
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
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(e));
  return e != 0;
}
// Shared-memory operands: the low word of a descriptor (address and the stride between slabs of an MN-major operand) moves
// from product to product, the high word does not.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row stride 1024, version, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_k(uint32_t smem) { return ((smem & 0x3ffff) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t smem) { return ((smem & 0x3ffff) >> 4) | ((16384u >> 4) << 16); }

template <bool kAccumulate>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "n"(kAccumulate ? 1 : 0), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
// D[128 x 128] = A B^T over a depth of D, both K-major; one lane
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc) {
  mma_ss<false>(d, a_low, b_low, idesc);
#pragma unroll
  for (int k = 1; k < D / 16; ++k) {
    const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
    mma_ss<true>(d, a_low + off, b_low + off, idesc);
  }
}
// D[128 x n] (+)= A B over a depth of 128, A bf16 in tensor memory (its halves kHalf columns apart), B MN-major; one lane
template <int kHalf>
__device__ __forceinline__ void mma_apply(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, bool first) {
  mma_ts(d, a_tmem, b_low, idesc, first ? 0u : 1u);
#pragma unroll
  for (int k = 1; k < 8; ++k) mma_ts(d, a_tmem + (k >> 2) * kHalf + (k & 3) * 8, b_low + k * (2048 >> 4), idesc, 1u);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 bytes to a 32-byte aligned address: a whole sector per lane
__device__ __forceinline__ void st_global_32(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f,
                                             uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e),
               "r"(f), "r"(g), "r"(h)
               : "memory");
}
// 32 consecutive values of a row as bf16
__device__ __forceinline__ void store_bf16_32(__nv_bfloat16* dst, const uint32_t (&r)[32], float mul) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      w[k] = pack_bf16x2(__uint_as_float(r[q * 16 + 2 * k]) * mul, __uint_as_float(r[q * 16 + 2 * k + 1]) * mul);
    st_global_32(dst + q * 16, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
  }
}
// A wait of a whole warp: the same answer in every lane, so that the warp stays together for .aligned instructions.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, where));
}
// All warps that `bar` counts; like every wait, it ends when another role gave up.
__device__ __forceinline__ bool group_sync(uint64_t* bar, uint32_t& phase, volatile int* abort_flag, int* status, int where) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  const bool ok = warp_wait(bar, phase, abort_flag, status, where);
  phase ^= 1;
  return ok;
}

// Items are sorted longest first; rounds alternate in direction so that no CTA gets the longest of every round.
__device__ __forceinline__ int item_of_round(int round) {
  const int g = gridDim.x, c = blockIdx.x;
  return round * g + ((round & 1) ? g - 1 - c : c);
}

// ---------------------------------------------------------------- forward --
// A CTA works on two query tiles ("slots") at a time against the same key tiles: two heads of a group where the group is
// even, else two neighbouring tiles of a head, else (few tiles in all) one.  While the softmax warps of one slot turn its
// scores into weights the tensor core works on the other's.  384 threads:
//   warps 0-3, 4-7  softmax of slot 0, 1: a thread per query row
//   warp 8          TMA producer: Q per slot, K and V tiles in one ring
//   warp 9          TMEM owner, tcgen05.mma issuer
// TMEM: S of the slots at columns 0 and 128, O at 256 and 256 + D.  P (bf16) overwrites the first 64 columns of its S
// and is the A operand of P V from there.  The CTA stays for all its items: loads and the first products of the next item
// run under the last steps of the one before.
constexpr int kFwdThreads = 384;  // whole warpgroups: registers are handed from the last one to the first two

struct BandFwdParams {
  CUtensorMap q_map, k_map, v_map;
  BandArgs a;
  int pair;     // 0: one tile an item, 1: two neighbouring tiles, 2: two heads
  int n_qt;     // query tiles of a head
  int s_pad;    // rows of the statistics: n_qt * 128
  int n_items;
  int t_last;   // first distance of the last bucket
};

template <int D>
struct BandFwdSmem {
  static constexpr int kSlabs = (D + 63) / 64;
  static constexpr int kTile = kSlabs * 16384;
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTile;
  static constexpr int kBar = kRing + kStages * kTile;
  static constexpr int kNumBars = 2 * kStages + 14;
  static constexpr int kLut = kBar + ((kNumBars * 8 + 16 + 127) / 128) * 128;  // float [2][entries], then the map
};

struct FwdItem {
  int b, hk;
  int h[2], q0[2];
  KeyTiles t[2], all;
};

__device__ __forceinline__ FwdItem fwd_item(const BandFwdParams& p, int item) {
  const BandArgs& a = p.a;
  FwdItem w;
  const int heads = p.pair == 2 ? a.Hq / 2 : a.Hq;
  const int n_hb = heads * a.B;
  const int rest = item % n_hb;
  const int tiles = p.pair == 1 ? (p.n_qt + 1) / 2 : p.n_qt;
  const int tile = tiles - 1 - item / n_hb;
  w.b = rest / heads;
  const int h = rest % heads;
  w.h[0] = p.pair == 2 ? 2 * h : h;
  w.h[1] = p.pair == 2 ? 2 * h + 1 : h;
  w.hk = w.h[0] / (a.Hq / a.Hkv);
  w.q0[0] = (p.pair == 1 ? 2 * tile : tile) * 128;
  w.q0[1] = p.pair == 1 ? w.q0[0] + 128 : w.q0[0];
  w.t[0] = key_tiles(a, w.q0[0]);
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

template <int D>
__global__ void __launch_bounds__(kFwdThreads, 1) band_fwd_kernel(const __grid_constant__ BandFwdParams p) {
  using L = BandFwdSmem<D>;
  constexpr int NS = L::kSlabs, ST = L::kStages;
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
  uint64_t* sync_bar = q_full + 12;
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
      mbar_init(&kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 4);
      mbar_init(&sync_bar[t], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) build_bucket_map(a, p.t_last, map, threadIdx.x, kFwdThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_enter();  // the set-up above touches no global memory
  // 384 threads start with 168 registers each: 2 * 208 + 80 <= 3 * 168

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
    // ------------------------------------------------------------ producer --
    if (lane == 0) {
      tma_prefetch_desc(&p.q_map);
      tma_prefetch_desc(&p.k_map);
      tma_prefetch_desc(&p.v_map);
      int pos = 0, n_q[2] = {0, 0};
      bool ok = true;
      for (int round = 0; ok; ++round) {
        const int item = item_of_round(round);
        if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
        if (item >= p.n_items) continue;
        const FwdItem w = fwd_item(p, item);
        auto load = [&](const CUtensorMap* m, int j) {
          const int st = pos % ST, use = pos / ST;
          if (use > 0 && !mbar_wait(&kv_empty[st], (use - 1) & 1, abort_flag, a.status, 61)) return false;
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
          if (n_q[t] > 0 && !mbar_wait(&q_empty[t], (n_q[t] - 1) & 1, abort_flag, a.status, 62)) {
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
    } else if (warp == 9) {
      // -------------------------------------------------------- MMA issuer --
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_o = make_idesc_bf16(128, D, false, true);
      const uint32_t ring = smem_u32(smem + L::kRing);
      const bool one = elect_one();
      uint32_t base = 0;
      uint32_t n_p[2] = {0, 0}, n_item[2] = {0, 0};
      bool ok = true;
      for (int round = 0; ok; ++round) {
        const int item = item_of_round(round);
        if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
        if (item >= p.n_items) continue;
        const FwdItem w = fwd_item(p, item);
        const int n = w.all.count();
        int left[2] = {w.t[0].count(), w.t[1].count()};
        bool pending[2] = {false, false}, fresh[2] = {true, true};
        const bool any[2] = {left[0] > 0, left[1] > 0};
        // O += P V of tile u for slot t
        auto pv = [&](int t, int u) {
          const uint32_t pos = base + 2 * u + 1;
          if (!warp_wait(&kv_full[pos % ST], (pos / ST) & 1, abort_flag, a.status, 63)) return false;
          if (fresh[t] && n_item[t] > 0 && !warp_wait(&o_empty[t], (n_item[t] - 1) & 1, abort_flag, a.status, 64)) return false;
          if (!warp_wait(&p_full[t], n_p[t] & 1, abort_flag, a.status, 65)) return false;
          ++n_p[t];
          tc_fence_after();
          const uint32_t b_low = desc_mn(ring + (pos % ST) * L::kTile);
          const bool last = left[t] == 0, first = fresh[t];
          if (one) {
            mma_apply<32>(tmem + 256 + t * D, tmem + t * 128, b_low, idesc_o, first);
            if (last) tc_commit(&o_full[t]);
          }
          fresh[t] = false;
          pending[t] = false;
          return true;
        };
        for (int u = 0; u < n && ok; ++u) {
          const int j = tile_at(w.all, u);
          const uint32_t pos = base + 2 * u;
          if (!warp_wait(&kv_full[pos % ST], (pos / ST) & 1, abort_flag, a.status, 66)) {
            ok = false;
            break;
          }
          const uint32_t b_low = desc_k(ring + (pos % ST) * L::kTile);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && pending[t]) ok = pv(t, u - 1);
            if (ok && w.t[t].uses(j)) {
              // the first scores of an item (nothing was multiplied with V since) wait for its queries
              if (fresh[t] && !pending[t] && !warp_wait(&q_full[t], n_item[t] & 1, abort_flag, a.status, 67)) {
                ok = false;
              } else {
                tc_fence_after();
                const bool last = --left[t] == 0;
                if (one) {
                  mma_scores<D>(tmem + t * 128, desc_k(smem_u32(smem + L::kQ + t * L::kTile)), b_low, idesc_s);
                  tc_commit(&s_full[t]);
                  if (last) tc_commit(&q_empty[t]);
                }
                pending[t] = true;
              }
            }
          }
          if (ok && one) {
            tc_commit(&kv_empty[pos % ST]);
            if (u > 0) tc_commit(&kv_empty[(pos - 1) % ST]);
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && pending[t]) ok = pv(t, n - 1);
        if (ok && n > 0 && one) tc_commit(&kv_empty[(base + 2 * n - 1) % ST]);
        base += 2 * n;
#pragma unroll
        for (int t = 0; t < 2; ++t) n_item[t] += any[t];
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------- softmax + epilogue --
    const int t = warp >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;  // row in the tile == TMEM lane
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t t_s = t_row + t * 128, t_o = t_row + 256 + t * D;
    const float sl2 = a.scale * kBandLog2e;
    float* lut = luts + t * entries;
    int n_s = 0, n_item = 0;
    uint32_t sync_phase = 0;
    bool ok = true;
    for (int round = 0; ok; ++round) {
      const int item = item_of_round(round);
      if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
      if (item >= p.n_items) continue;
      const FwdItem w = fwd_item(p, item);
      const int q0 = w.q0[t], h = w.h[t];
      const KeyTiles mine = w.t[t];
      if (q0 < 0) continue;
      const int row = q0 + r, pos = a.q_pos0 + row;
      const int pmin = a.q_pos0 + q0, pmax = pmin + 127;
      float far_bias = 0.f;
      if (a.table != nullptr) {
        ok = group_sync(&sync_bar[t], sync_phase, abort_flag, a.status, 70);  // everyone has left the item before
        build_lut(a, h, p.t_last, map, lut, r, 128);
        ok = ok && group_sync(&sync_bar[t], sync_phase, abort_flag, a.status, 71);
        if (!ok) break;
        far_bias = lut[entries - 1];
      }
      const int n = mine.count();
      float m = -INFINITY, l = 0.f;
      for (int u = 0; u < n; ++u) {
        const int kv0 = tile_at(mine, u) * 128;
        if (!warp_wait(&s_full[t], n_s & 1, abort_flag, a.status, 68)) {
          ok = false;
          break;
        }
        ++n_s;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_s + c * 32, s[c]);
        tmem_ld_wait();
        float mul = sl2, add = far_bias;
        // Biases that differ inside the tile, or that are too large to be added to the maximum instead of to the scores.
        if (a.table != nullptr && (pmin - (kv0 + 127) < p.t_last || fabsf(far_bias) > 1e30f)) {
          const float* at = lut + kLutFront + min(pos - kv0, p.t_last + kLutBack - 1);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) s[c][k] = __float_as_uint(fmaf(__uint_as_float(s[c][k]), sl2, at[-(c * 32 + k)]));
          mul = 1.f;
          add = 0.f;
        }
        const bool whole = kv0 + 127 <= pmin && kv0 + 127 < a.Skv && (kv0 > pmax - a.window || kv0 + 127 < a.sinks);
        if (!whole) {
          const int hi = min(pos, a.Skv - 1) - kv0 + 1, lo = pos - a.window + 1 - kv0, sk = a.sinks - kv0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t see = low_bits(hi - c * 32) & (~low_bits(lo - c * 32) | low_bits(sk - c * 32));
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1u)) s[c][k] = 0xff800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
          for (int k = 1; k < 32; ++k) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][k]));
        }
        const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), mul, add);
        // The maximum that weights are relative to moves only when it grew by more than 2^8: most tiles need no pass over O,
        // and the division by the sum at the end makes the result exact.
        const float m_new = top > m + 8.f ? top : m;
        const float alpha = m_new == m ? 1.f : ex2(m - m_new);  // m == -inf: 0
        const float shift = add - (m_new == -INFINITY ? 0.f : m_new);
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float p0 = ex2(fmaf(__uint_as_float(s[c][2 * k]), mul, shift));
            const float p1 = ex2(fmaf(__uint_as_float(s[c][2 * k + 1]), mul, shift));
            sum0 += p0;
            sum1 += p1;
            pk[k] = pack_bf16x2(p0, p1);
          }
          tmem_st_32x16(t_s + c * 16, pk);
        }
        // the scores are complete, so is the product of the tile before: O may be rescaled
        if (u > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(t_o + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st_32x32(t_o + c * 32, o);
          }
        }
        l = l * alpha + (sum0 + sum1);
        m = m_new;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      const long long stat = (static_cast<long long>(w.b) * a.Hq + h) * a.Sq + row;
      __nv_bfloat16* out = band_row(a.o, a.o_st, w.b, row, h);
      if (n > 0) {
        if (!warp_wait(&o_full[t], n_item & 1, abort_flag, a.status, 69)) {
          ok = false;
          break;
        }
        ++n_item;
        tc_fence_after();
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_32x32(t_o + c * 32, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0;
        }
        if (row < a.Sq) store_bf16_32(out + c * 32, o, inv);
      }
      if (n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[t]);
      }
      if (row < a.Sq) {
        a.m[stat] = l > 0.f ? m : INFINITY;  // a row that sees nothing: 2^(x - m) is 0 in the backward pass
        a.l[stat] = l > 0.f ? log2f(l) : 0.f;
      }
    }
  }

  if (*abort_flag != 0) {  // let the loads in flight land
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

static int make_band_map(CUtensorMap* m, const __nv_bfloat16* ptr, const BandStride& t, int d, int S, int H, int B) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(S), static_cast<uint64_t>(H), static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {static_cast<uint64_t>(t.s) * 2, static_cast<uint64_t>(t.h) * 2,
                               static_cast<uint64_t>(t.b) * 2};
  const uint32_t box[4] = {64, 128, 1, 1};
  return make_tmap_bf16(m, ptr, 4, dims, strides, box);
}

template <int D>
static cudaError_t launch_band_fwd(const BandFwdParams& p, cudaStream_t s) {
  const int lut = p.a.table == nullptr ? 0 : lut_bytes(p.t_last, 2);
  return launch_pdl(band_fwd_kernel<D>, dim3(std::min(p.n_items, sm_count())), dim3(kFwdThreads), BandFwdSmem<D>::kLut + lut, s, p);
}

// --------------------------------------------------------------- backward --
// Two kernels and no atomics: a query tile's dQ and a key tile's dK, dV are each summed by one CTA in a fixed order, at the
// price of working the weights out twice (seven products of a tile pair instead of five).
//
// Column statistics passed from the first to the second, per (batch, query head, query tile): 128 floats each of
//   c = (far bias - m) - l,  D,  m,  l        (rows behind the last: c = -inf, so that their weights are 0)
constexpr int kBwdBandThreads = 384;
constexpr int kStatBlock = 512;  // floats

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

struct BandBwdParams {
  CUtensorMap q_map, k_map, v_map, do_map;
  BandArgs a;
  float* stat;      // [B, Hq, n_qt, kStatBlock]
  float* part;      // fp32 dV, dK tiles of key tiles whose rows are split
  float* dtable_part;  // [B, Hq, n_qt, buckets]
  int n_qt, n_kt;
  int n_items;      // of this kernel
  int t_last;
  int sink_tiles;   // dK, dV: key tiles that hold sinks, their pieces, the pieces of the others
  int sink_pieces, pieces;
};

// ---- dQ, D, and the table's gradient ----
// A CTA works on one query tile: S = Q K^T and dP = dO V^T land in tensor memory, eight warps (two threads a row, 64 columns
// each) turn them into dS, which goes back as the A operand of dQ += dS K.  S and dP of the next tile are computed while
// dS of this one is.  TMEM: S 0, dP 128, dQ 256, dS (two buffers) from 384.
//
// dtable: inside tiles that meet distances below t_last the sums along the diagonals (equal distance) are formed by passing a
// running sum from lane to lane, one row down per column; they are then added by bucket.  All other tiles belong to the last
// bucket.  Its sum over many keys is small against its terms' rounding: D comes from the output rounded to bf16 and is off by
// some e, which the rows' sums show (sum_j dS_ij is e times the sum of P, 1, instead of 0); e * P is taken off again.
template <int D>
struct BandDqSmem {
  static constexpr int kSlabs = (D + 63) / 64;
  static constexpr int kTile = kSlabs * 16384;
  static constexpr int kQStages = D == 64 ? 2 : 1;
  static constexpr int kStages = D == 64 ? 8 : 4;  // K and V tiles in turn
  static constexpr int kQ = 0;                     // Q, dO per stage
  static constexpr int kRing = 2 * kQStages * kTile;
  static constexpr int kBar = kRing + kStages * kTile;
  static constexpr int kNumBars = 2 * kStages + 2 * kQStages + 6;
  static constexpr int kXch = kBar + ((kNumBars * 8 + 16 + 127) / 128) * 128;  // float [2][2][128]
  static constexpr int kLut = kXch + 2048;                                     // float [entries], the map
  // behind them, where the table's gradient is wanted: float bins[8][128], diagonals[8][96]
  static constexpr int kBins = 8 * (kMaxBuckets + 96) * 4;
};

// The query tile of an item, longest first.
struct DqItem {
  int b, h, hk, q0;
  KeyTiles t;
};
__device__ __forceinline__ DqItem dq_item(const BandBwdParams& p, int item) {
  const BandArgs& a = p.a;
  DqItem w;
  const int n_hb = a.Hq * a.B;
  w.h = item % n_hb % a.Hq;
  w.b = item % n_hb / a.Hq;
  w.hk = w.h / (a.Hq / a.Hkv);
  w.q0 = (p.n_qt - 1 - item / n_hb) * 128;
  w.t = key_tiles(a, w.q0);
  return w;
}

template <int D>
__global__ void __launch_bounds__(kBwdBandThreads, 1) band_bwd_dq_kernel(const __grid_constant__ BandBwdParams p) {
  using L = BandDqSmem<D>;
  constexpr int NS = L::kSlabs, ST = L::kStages, QS = L::kQStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_full = bars;                // [ST]
  uint64_t* kv_empty = bars + ST;          // [ST]
  uint64_t* q_full = bars + 2 * ST;        // [QS]
  uint64_t* q_empty = q_full + QS;         // [QS] last product issued + 8 warps that read dO
  uint64_t* sdp_full = q_empty + QS;
  uint64_t* sdp_read = sdp_full + 1;
  uint64_t* ds_full = sdp_full + 2;
  uint64_t* dq_full = sdp_full + 3;
  uint64_t* dq_empty = sdp_full + 4;
  uint64_t* sync_bar = sdp_full + 5;
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
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < QS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 9);
    }
    mbar_init(sdp_full, 1);
    mbar_init(sdp_read, 8);
    mbar_init(ds_full, 8);
    mbar_init(dq_full, 1);
    mbar_init(dq_empty, 8);
    mbar_init(sync_bar, 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) {
    build_bucket_map(a, p.t_last, map, threadIdx.x, kBwdBandThreads);
    if (a.dtable != nullptr)
      for (int n = threadIdx.x; n < 8 * kMaxBuckets; n += kBwdBandThreads) bins[n] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_enter();
  const int rounds = (p.n_items + gridDim.x - 1) / gridDim.x;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8 && lane == 0) {
      // ---------------------------------------------------------- producer --
      tma_prefetch_desc(&p.q_map);
      tma_prefetch_desc(&p.do_map);
      tma_prefetch_desc(&p.k_map);
      tma_prefetch_desc(&p.v_map);
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
        if (use > 0 && !mbar_wait(&q_empty[qs], (use - 1) & 1, abort_flag, a.status, 81)) break;
        mbar_expect_tx(&q_full[qs], 2 * L::kTile);
#pragma unroll
        for (int c = 0; c < NS; ++c) {
          uint8_t* dst = smem + L::kQ + 2 * qs * L::kTile + c * 16384;
          tma_load_4d(dst, &p.q_map, &q_full[qs], c * 64, w.q0, w.h, w.b);
          tma_load_4d(dst + L::kTile, &p.do_map, &q_full[qs], c * 64, w.q0, w.h, w.b);
        }
        for (int u = 0; u < 2 * n; ++u, ++pos) {
          const int st = pos % ST, kuse = pos / ST, j = tile_at(w.t, u >> 1);
          if (kuse > 0 && !mbar_wait(&kv_empty[st], (kuse - 1) & 1, abort_flag, a.status, 82)) {
            ok = false;
            break;
          }
          mbar_expect_tx(&kv_full[st], L::kTile);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(smem + L::kRing + st * L::kTile + c * 16384, (u & 1) ? &p.v_map : &p.k_map, &kv_full[st], c * 64,
                        j * 128, w.hk, w.b);
        }
      }
    } else if (warp == 9) {
      // -------------------------------------------------------- MMA issuer --
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_dq = make_idesc_bf16(128, D, false, true);
      const uint32_t ring = smem_u32(smem + L::kRing);
      const bool one = elect_one();
      uint32_t step = 0, n_item = 0;  // tiles and items begun
      bool prev_first = false, prev_last = false;
      uint32_t prev_item = 0;
      bool ok = true;
      // dQ += dS K of step s
      auto issue_dq = [&](uint32_t s, bool first, bool last, uint32_t item_no) {
        if (first && item_no > 0 && !warp_wait(dq_empty, (item_no - 1) & 1, abort_flag, a.status, 83)) return false;
        if (!warp_wait(ds_full, s & 1, abort_flag, a.status, 84)) return false;
        tc_fence_after();
        const uint32_t st = 2 * s % ST;
        if (one) {
          mma_apply<32>(tmem + kDq, tmem + kDs + (s & 1) * 64, desc_mn(ring + st * L::kTile), idesc_dq, first);
          tc_commit(&kv_empty[st]);
          if (last) tc_commit(dq_full);
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
          const uint32_t pk = 2 * step, pv = pk + 1;
          ok = (u > 0 || warp_wait(&q_full[qs], (n_item / QS) & 1, abort_flag, a.status, 85)) &&
               warp_wait(&kv_full[pk % ST], (pk / ST) & 1, abort_flag, a.status, 86) &&
               warp_wait(&kv_full[pv % ST], (pv / ST) & 1, abort_flag, a.status, 87) &&
               (step == 0 || warp_wait(sdp_read, (step - 1) & 1, abort_flag, a.status, 88));
          if (!ok) break;
          tc_fence_after();
          if (one) {
            mma_scores<D>(tmem, q_low, desc_k(ring + (pk % ST) * L::kTile), idesc_s);
            mma_scores<D>(tmem + kDp, q_low + (L::kTile >> 4), desc_k(ring + (pv % ST) * L::kTile), idesc_s);
            tc_commit(sdp_full);
            tc_commit(&kv_empty[pv % ST]);
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------ compute --
    const int quad = warp & 3, half = warp >> 2;
    const int r = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float* xch = reinterpret_cast<float*>(smem + L::kXch);
    float* my_bins = bins + warp * kMaxBuckets;
    float* diag = bins + 8 * kMaxBuckets + warp * 96;
    const float sl2 = a.scale * kBandLog2e;
    const bool want_table = a.dtable != nullptr;
    int step = 0, n_item = 0, parity = 0;
    uint32_t sync_phase = 0;
    auto together = [&]() { return group_sync(sync_bar, sync_phase, abort_flag, a.status, 92); };
    bool ok = true;
    for (int round = 0; round < rounds && ok; ++round) {
      const int item = item_of_round(round);
      if (item >= p.n_items) continue;
      const DqItem w = dq_item(p, item);
      const int n = w.t.count();
      const int row = w.q0 + r, pos = a.q_pos0 + row, pmin = a.q_pos0 + w.q0;
      const bool valid = row < a.Sq;
      const long long at_row = (static_cast<long long>(w.b) * a.Hq + w.h) * a.Sq + row;
      const float m = valid ? a.m[at_row] : INFINITY;
      const float l = valid ? a.l[at_row] : 0.f;
      float far_bias = 0.f;
      if (a.table != nullptr) {
        if (!together()) break;  // everyone has left the item before
        build_lut(a, w.h, p.t_last, map, lut, threadIdx.x, 256);
      }
      // D: half a row of O and dO per thread
      float dsum = 0.f;
      if (n > 0) {
        constexpr int kChunks = D / 16;  // 16-byte chunks of half a row
        uint4 o[kChunks];
        const uint4* src = reinterpret_cast<const uint4*>(band_row(a.o, a.o_st, w.b, valid ? row : w.q0, w.h)) + half * kChunks;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) o[c] = src[c];
        const int qs = n_item % QS;
        if (!warp_wait(&q_full[qs], (n_item / QS) & 1, abort_flag, a.status, 89)) break;
        const uint8_t* sdo = smem + L::kQ + (2 * qs + 1) * L::kTile;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int ch = half * kChunks + c;
          const uint4 g = *reinterpret_cast<const uint4*>(sdo + (ch >> 3) * 16384 + swz128_offset(r, ch & 7));
          const uint32_t ow[4] = {o[c].x, o[c].y, o[c].z, o[c].w}, gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = unpack_bf16x2(ow[k]), y = unpack_bf16x2(gw[k]);
            dsum = fmaf(x.x, y.x, fmaf(x.y, y.y, dsum));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[qs]);
      }
      float* mine = xch + parity * 256;
      parity ^= 1;
      mine[half * 128 + r] = dsum;
      if (!together()) break;
      const float delta = valid ? mine[r] + mine[128 + r] : 0.f;
      if (a.table != nullptr) far_bias = lut[entries - 1];
      const float c_far = (far_bias - m) - l;
      if (half == 0) {
        float* st = p.stat + ((static_cast<long long>(w.b) * a.Hq + w.h) * p.n_qt + w.q0 / 128) * kStatBlock + r;
        st[0] = c_far;
        st[128] = delta;
        st[256] = m;
        st[384] = l;
      }
      float ds_all = 0.f, ds_far = 0.f, p_far = 0.f;
      for (int u = 0; u < n; ++u, ++step) {
        const int kv0 = tile_at(w.t, u) * 128;
        if (!warp_wait(sdp_full, step & 1, abort_flag, a.status, 90)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[2][32], dp[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tmem_ld_32x32(t_row + half * 64 + c * 32, s[c]);
          tmem_ld_32x32(t_row + kDp + half * 64 + c * 32, dp[c]);
        }
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sdp_read);
        const bool near = a.table != nullptr && pmin - (kv0 + 127) < p.t_last;
        const bool added = near || (a.table != nullptr && fabsf(far_bias) > 1e30f);
        const bool whole = kv0 + 127 <= pmin && kv0 + 127 < a.Skv && (pmin + 127 - kv0 < a.window || kv0 + 127 < a.sinks);
        // weights, in place of the scores
        if (!added) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) s[c][k] = __float_as_uint(ex2(fmaf(__uint_as_float(s[c][k]), sl2, c_far)));
        } else {
          const float* at = lut + kLutFront + min(pos - kv0, p.t_last + kLutBack - 1) - half * 64;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              s[c][k] = __float_as_uint(ex2((fmaf(__uint_as_float(s[c][k]), sl2, at[-(c * 32 + k)]) - m) - l));
        }
        if (!whole) {
          const int hi = min(pos, a.Skv - 1) - kv0 + 1, lo = pos - a.window + 1 - kv0, sk = a.sinks - kv0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int c0 = half * 64 + c * 32;
            const uint32_t see = low_bits(hi - c0) & (~low_bits(lo - c0) | low_bits(sk - c0));
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1u)) s[c][k] = 0;
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; ++k) dp[c][k] = __float_as_uint(__uint_as_float(s[c][k]) * (__uint_as_float(dp[c][k]) - delta));
#pragma unroll
          for (int k = 0; k < 16; ++k) pk[k] = pack_bf16x2(__uint_as_float(dp[c][2 * k]), __uint_as_float(dp[c][2 * k + 1]));
          tmem_st_32x16(t_row + kDs + (step & 1) * 64 + half * 32 + c * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full);
        if (want_table) {
          float sum = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) sum += __uint_as_float(dp[c][k]);
          ds_all += sum;
          const int far_from = pos - kv0 - p.t_last - half * 64;  // columns up to this one belong to the last bucket
          if (!near) {
            ds_far += sum;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int k = 0; k < 32; ++k) p_far += __uint_as_float(s[c][k]);
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int k = 0; k < 32; ++k) p_far += c * 32 + k <= far_from ? __uint_as_float(s[c][k]) : 0.f;
            // diagonal e holds distance base + e; lane 31 completes one of them per column, the others stay behind at the end
            const int base = pmin + quad * 32 - kv0 - half * 64 - 63;
            float run = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const float from = __shfl_up_sync(0xffffffffu, run, 1);
                run = (lane == 0 ? 0.f : from) + __uint_as_float(dp[c][k]);
                if (lane == 31) diag[31 + 63 - (c * 32 + k)] = run;
              }
            if (lane < 31) diag[lane] = run;
            __syncwarp();
#pragma unroll
            for (int e0 = 0; e0 < 96; e0 += 32) {
              const int e = e0 + lane;
              float v = e < 95 ? diag[e] : 0.f;
              const int bucket = map[kLutFront + base + min(e, 94)];
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
      if (!ok) break;
      __nv_bfloat16* out = band_row(a.dq, a.dq_st, w.b, row, w.h) + half * (D / 2);
      if (n > 0) {
        if (!warp_wait(dq_full, n_item & 1, abort_flag, a.status, 91)) break;
        ++n_item;
        tc_fence_after();
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[16];
        if (n > 0) {
          tmem_ld_32x16(t_row + kDq + half * (D / 2) + c * 16, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = 0;
        }
        if (valid) store_bf16_16(out + c * 16, v, a.scale);
      }
      if (n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_empty);
      }
      if (want_table) {
        float* other = xch + parity * 256;  // error of D per half row, its share of the last bucket
        other[half * 128 + r] = ds_all;
        if (!together()) break;
        const float off = other[r] + other[128 + r];
        const float last = warp_sum(ds_far - off * p_far);
        // the far part of tiles that were summed by diagonals is in the bins already, with its error: p_far covers it
        if (lane == 0) my_bins[a.buckets - 1] += last;
        if (!together()) break;
        parity ^= 1;
        for (int b = threadIdx.x; b < a.buckets; b += 256) {
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            sum += bins[k * kMaxBuckets + b];
            bins[k * kMaxBuckets + b] = 0.f;
          }
          p.dtable_part[((static_cast<long long>(w.b) * a.Hq + w.h) * p.n_qt + w.q0 / 128) * a.buckets + b] = sum;
        }
        if (!together()) break;
      }
    }
  }

  if (*abort_flag != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- dK and dV ----
// A CTA works on one key tile of one key head, over the query heads of the group and the query tiles that see it, or on a
// piece of them.  S^T = K Q^T and dP^T = V dO^T have keys as rows, so P^T and dS^T go straight back to tensor memory as A
// operands of dV += P^T dO and dK += dS^T Q.  TMEM: S^T 0, dP^T 128, dV 256, dK 256 + D; with D = 64 P^T and dS^T have
// columns of their own (384, 448), else they overwrite S^T and dP^T.
template <int D>
struct BandDkvSmem {
  static constexpr int kSlabs = (D + 63) / 64;
  static constexpr int kTile = kSlabs * 16384;
  static constexpr int kStages = D == 64 ? 4 : 2;  // Q, dO and the column statistics
  static constexpr int kK = 0;                     // K, V
  static constexpr int kRing = 2 * kTile;
  static constexpr int kStat = kRing + 2 * kStages * kTile;
  static constexpr int kBar = kStat + kStages * kStatBlock * 4;
  static constexpr int kNumBars = 2 * kStages + 11;
  static constexpr int kLut = kBar + ((kNumBars * 8 + 16 + 127) / 128) * 128;
};

struct DkvItem {
  int b, hk, kv0;
  int slot;        // where a piece goes; -1: the whole tile
  int first_qt, per_head;
  int from, to;    // steps of this piece: step / per_head = head of the group, step % per_head = query tile
};
__device__ __forceinline__ DkvItem dkv_item(const BandBwdParams& p, int item) {
  const BandArgs& a = p.a;
  DkvItem w;
  const int n_hb = a.Hkv * a.B;
  const int sink_items = p.sink_tiles * p.sink_pieces * n_hb;
  int tile, piece, pieces;
  if (item < sink_items) {
    pieces = p.sink_pieces;
    w.slot = item;
    tile = item / n_hb / pieces;
    piece = item / n_hb % pieces;
  } else {
    pieces = p.pieces;
    const int rest = item - sink_items;
    w.slot = (p.sink_pieces > 1 ? sink_items : 0) + rest;
    tile = p.sink_tiles + rest / n_hb / pieces;
    piece = rest / n_hb % pieces;
  }
  if (pieces == 1) w.slot = -1;
  w.hk = item % n_hb % a.Hkv;
  w.b = item % n_hb / a.Hkv;
  w.kv0 = tile * 128;
  const int first = max(0, w.kv0 - a.q_pos0);
  const int last = w.kv0 < a.sinks ? a.Sq - 1 : min(a.Sq - 1, min(w.kv0 + 127, a.Skv - 1) - a.q_pos0 + a.window - 1);
  w.first_qt = first >> 7;
  w.per_head = first <= last ? (last >> 7) - w.first_qt + 1 : 0;
  const int n = w.per_head * (a.Hq / a.Hkv);
  w.from = static_cast<int>(static_cast<long long>(n) * piece / pieces);
  w.to = static_cast<int>(static_cast<long long>(n) * (piece + 1) / pieces);
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
__global__ void __launch_bounds__(kBwdBandThreads, 1) band_bwd_dkv_kernel(const __grid_constant__ BandBwdParams p) {
  using L = BandDkvSmem<D>;
  constexpr int NS = L::kSlabs, ST = L::kStages;
  constexpr bool kOwn = D == 64;  // P^T and dS^T have their own columns
  constexpr uint32_t kDp = 128, kDv = 256, kDk = 256 + D, kP = kOwn ? 384 : 0, kDs = kOwn ? 448 : 128;
  constexpr uint32_t kHalf = kOwn ? 32 : 64;  // a warp that is ahead must not write over the half that another still reads
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;             // [ST]
  uint64_t* q_empty = bars + ST;       // [ST] dK of the step issued and done + 8 warps that read the statistics
  uint64_t* kv_full = bars + 2 * ST;
  uint64_t* kv_empty = kv_full + 1;
  uint64_t* s_full = kv_full + 2;
  uint64_t* s_read = kv_full + 3;
  uint64_t* dp_full = kv_full + 4;
  uint64_t* dp_read = kv_full + 5;
  uint64_t* p_full = kv_full + 6;
  uint64_t* ds_full = kv_full + 7;
  uint64_t* acc_full = kv_full + 8;
  uint64_t* acc_empty = kv_full + 9;
  uint64_t* sync_bar = kv_full + 10;
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
      mbar_init(&q_empty[s], 9);
    }
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(s_read, 8);
    mbar_init(dp_full, 1);
    mbar_init(dp_read, 8);
    mbar_init(p_full, 8);
    mbar_init(ds_full, 8);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 8);
    mbar_init(sync_bar, 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) build_bucket_map(a, p.t_last, map, threadIdx.x, kBwdBandThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_enter();
  const int group = a.Hq / a.Hkv;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8 && lane == 0) {
      // ---------------------------------------------------------- producer --
      tma_prefetch_desc(&p.q_map);
      tma_prefetch_desc(&p.do_map);
      tma_prefetch_desc(&p.k_map);
      tma_prefetch_desc(&p.v_map);
      const uint32_t stat_bytes = a.table == nullptr ? 1024 : 2048;
      DkvWalk x;
      int n = 0, n_item = 0;
      for (bool more = x.open(p, 0); more; more = x.next(p), ++n) {
        if (x.first()) {
          if (n_item > 0 && !mbar_wait(kv_empty, (n_item - 1) & 1, abort_flag, a.status, 101)) break;
          ++n_item;
          mbar_expect_tx(kv_full, 2 * L::kTile);
#pragma unroll
          for (int c = 0; c < NS; ++c) {
            tma_load_4d(smem + L::kK + c * 16384, &p.k_map, kv_full, c * 64, x.w.kv0, x.w.hk, x.w.b);
            tma_load_4d(smem + L::kK + L::kTile + c * 16384, &p.v_map, kv_full, c * 64, x.w.kv0, x.w.hk, x.w.b);
          }
        }
        const int st = n % ST, use = n / ST;
        if (use > 0 && !mbar_wait(&q_empty[st], (use - 1) & 1, abort_flag, a.status, 102)) break;
        const int h = x.w.hk * group + x.step / x.w.per_head, qt = x.w.first_qt + x.step % x.w.per_head;
        mbar_expect_tx(&q_full[st], 2 * L::kTile + stat_bytes);
#pragma unroll
        for (int c = 0; c < NS; ++c) {
          uint8_t* dst = smem + L::kRing + 2 * st * L::kTile + c * 16384;
          tma_load_4d(dst, &p.q_map, &q_full[st], c * 64, qt * 128, h, x.w.b);
          tma_load_4d(dst + L::kTile, &p.do_map, &q_full[st], c * 64, qt * 128, h, x.w.b);
        }
        bulk_load(smem + L::kStat + st * kStatBlock * 4,
                  p.stat + ((static_cast<long long>(x.w.b) * a.Hq + h) * p.n_qt + qt) * kStatBlock, stat_bytes, &q_full[st]);
      }
    } else if (warp == 9) {
      // -------------------------------------------------------- MMA issuer --
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_d = make_idesc_bf16(128, D, false, true);
      const uint32_t sk = smem_u32(smem + L::kK), ring = smem_u32(smem + L::kRing);
      const uint32_t k_low = desc_k(sk), v_low = desc_k(sk + L::kTile);
      const bool one = elect_one();
      DkvWalk x;
      uint32_t n = 0, n_item = 0;  // step, item of `x`
      bool more = x.open(p, 0);
      bool ok = more && warp_wait(kv_full, 0, abort_flag, a.status, 103) && warp_wait(&q_full[0], 0, abort_flag, a.status, 104);
      if (ok) {
        tc_fence_after();
        const bool last = x.last();
        if (one) {
          mma_scores<D>(tmem, k_low, desc_k(ring), idesc_s);
          tc_commit(s_full);
          mma_scores<D>(tmem + kDp, v_low, desc_k(ring + L::kTile), idesc_s);
          tc_commit(dp_full);
          if (last) tc_commit(kv_empty);
        }
      }
      while (ok && more) {
        DkvWalk y = x;
        const bool ahead = y.next(p), fresh = ahead && y.first(), y_last = ahead && y.last();
        const bool x_first = x.first(), x_last = x.last();
        const uint32_t n_item2 = n_item + fresh;
        const uint32_t sq = ring + 2 * (n % ST) * L::kTile, sq2 = ring + 2 * ((n + 1) % ST) * L::kTile;
        // S^T and dP^T of the next step
        auto next_s = [&]() {
          if (!ahead) return true;
          if (fresh && !warp_wait(kv_full, n_item2 & 1, abort_flag, a.status, 105)) return false;
          if (!warp_wait(&q_full[(n + 1) % ST], ((n + 1) / ST) & 1, abort_flag, a.status, 106)) return false;
          if (kOwn && !warp_wait(s_read, n & 1, abort_flag, a.status, 107)) return false;
          tc_fence_after();
          if (one) {
            mma_scores<D>(tmem, k_low, desc_k(sq2), idesc_s);
            tc_commit(s_full);
          }
          return true;
        };
        auto next_dp = [&]() {
          if (one) {
            mma_scores<D>(tmem + kDp, v_low, desc_k(sq2 + L::kTile), idesc_s);
            tc_commit(dp_full);
            if (y_last) tc_commit(kv_empty);
          }
        };
        if (kOwn && !next_s()) break;
        if (x_first && n_item > 0 && !warp_wait(acc_empty, (n_item - 1) & 1, abort_flag, a.status, 108)) break;
        if (!warp_wait(p_full, n & 1, abort_flag, a.status, 109)) break;
        tc_fence_after();
        if (one) mma_apply<kHalf>(tmem + kDv, tmem + kP, desc_mn(sq + L::kTile), idesc_d, x_first);
        if (!kOwn && !next_s()) break;
        if (kOwn && ahead) {
          if (!warp_wait(dp_read, n & 1, abort_flag, a.status, 110)) break;
          tc_fence_after();
          next_dp();
        }
        if (!warp_wait(ds_full, n & 1, abort_flag, a.status, 111)) break;
        tc_fence_after();
        if (one) {
          mma_apply<kHalf>(tmem + kDk, tmem + kDs, desc_mn(sq), idesc_d, x_first);
          tc_commit(&q_empty[n % ST]);
          if (x_last) tc_commit(acc_full);
        }
        if (!kOwn && ahead) next_dp();
        x = y;
        more = ahead;
        n_item = n_item2;
        ++n;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------ compute --
    const int quad = warp & 3, half = warp >> 2;
    const int r = quad * 32 + lane;  // key of the tile == TMEM lane
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float sl2 = a.scale * kBandLog2e;
    const int rounds = (p.n_items + gridDim.x - 1) / gridDim.x;
    int n = 0, n_item = 0;
    uint32_t sync_phase = 0;
    auto together = [&]() { return group_sync(sync_bar, sync_phase, abort_flag, a.status, 118); };
    bool ok = true;
    for (int round = 0; round < rounds && ok; ++round) {
      const int item = item_of_round(round);
      if (item >= p.n_items) continue;
      const DkvItem w = dkv_item(p, item);
      const int j = w.kv0 + r;
      int lut_h = -1;
      float far_bias = 0.f;
      for (int step = w.from; step < w.to; ++step, ++n) {
        const int h = w.hk * group + step / w.per_head, qt = w.first_qt + step % w.per_head;
        const int pmin = a.q_pos0 + qt * 128;
        const int st = n % ST;
        if (a.table != nullptr && h != lut_h) {
          ok = together();  // everyone is done with the table of the head before
          build_lut(a, h, p.t_last, map, lut, threadIdx.x, 256);
          ok = ok && together();
          if (!ok) break;
          far_bias = lut[entries - 1];
          lut_h = h;
        }
        // the statistics come with Q and dO; the scores do after them
        if (!warp_wait(&q_full[st], (n / ST) & 1, abort_flag, a.status, 112) ||
            !warp_wait(s_full, n & 1, abort_flag, a.status, 113)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32(t_row + half * 64 + c * 32, s[c]);
        tmem_ld_wait();
        if (kOwn) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_read);
        }
        const float* stat = reinterpret_cast<const float*>(smem + L::kStat) + st * kStatBlock + half * 64;
        const bool added = a.table != nullptr && (pmin - (w.kv0 + 127) < p.t_last || fabsf(far_bias) > 1e30f);
        const bool whole = w.kv0 + 127 <= pmin && w.kv0 + 127 < a.Skv && (pmin + 127 - w.kv0 < a.window || w.kv0 + 127 < a.sinks);
        if (!added) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              const float4 cc = *reinterpret_cast<const float4*>(stat + c * 32 + k);
              s[c][k] = __float_as_uint(ex2(fmaf(__uint_as_float(s[c][k]), sl2, cc.x)));
              s[c][k + 1] = __float_as_uint(ex2(fmaf(__uint_as_float(s[c][k + 1]), sl2, cc.y)));
              s[c][k + 2] = __float_as_uint(ex2(fmaf(__uint_as_float(s[c][k + 2]), sl2, cc.z)));
              s[c][k + 3] = __float_as_uint(ex2(fmaf(__uint_as_float(s[c][k + 3]), sl2, cc.w)));
            }
        } else {
          const float* at = lut + kLutFront + min(pmin - j, p.t_last + 128) + half * 64;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              s[c][k] = __float_as_uint(
                  ex2((fmaf(__uint_as_float(s[c][k]), sl2, at[c * 32 + k]) - stat[256 + c * 32 + k]) - stat[384 + c * 32 + k]));
        }
        if (!whole) {
          const int lo = j < a.Skv ? j - pmin : 128, hi = j < a.sinks ? 128 : j - pmin + a.window;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int c0 = half * 64 + c * 32;
            const uint32_t see = low_bits(hi - c0) & ~low_bits(lo - c0);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((see >> k) & 1u)) s[c][k] = 0;
          }
        }
        if (kOwn && !warp_wait(dp_full, n & 1, abort_flag, a.status, 114)) {  // P^T of the step before has been read
          ok = false;
          break;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) pk[k] = pack_bf16x2(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1]));
          tmem_st_32x16(t_row + kP + half * kHalf + c * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
        if (!kOwn && !warp_wait(dp_full, n & 1, abort_flag, a.status, 115)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t dp[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32(t_row + kDp + half * 64 + c * 32, dp[c]);
        tmem_ld_wait();
        if (kOwn) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(dp_read);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float4 dd = *reinterpret_cast<const float4*>(stat + 128 + c * 32 + k);
            s[c][k] = __float_as_uint(__uint_as_float(s[c][k]) * (__uint_as_float(dp[c][k]) - dd.x));
            s[c][k + 1] = __float_as_uint(__uint_as_float(s[c][k + 1]) * (__uint_as_float(dp[c][k + 1]) - dd.y));
            s[c][k + 2] = __float_as_uint(__uint_as_float(s[c][k + 2]) * (__uint_as_float(dp[c][k + 2]) - dd.z));
            s[c][k + 3] = __float_as_uint(__uint_as_float(s[c][k + 3]) * (__uint_as_float(dp[c][k + 3]) - dd.w));
          }
        if (kOwn && n > 0 && !warp_wait(&q_empty[(n - 1) % ST], ((n - 1) / ST) & 1, abort_flag, a.status, 116)) {
          ok = false;  // dS^T of the step before has been read
          break;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) pk[k] = pack_bf16x2(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1]));
          tmem_st_32x16(t_row + kDs + half * kHalf + c * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(ds_full);
          mbar_arrive(&q_empty[st]);
        }
      }
      if (!ok) break;
      const bool any = w.from < w.to;
      if (any) {
        if (!warp_wait(acc_full, n_item & 1, abort_flag, a.status, 117)) break;
        ++n_item;
        tc_fence_after();
      }
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float mul = which == 0 ? 1.f : a.scale;
        __nv_bfloat16* out = band_row(which == 0 ? a.dv : a.dk, which == 0 ? a.dv_st : a.dk_st, w.b, j, w.hk) + half * (D / 2);
        float* part = p.part + ((static_cast<long long>(w.slot) * 2 + which) * 128 + r) * D + half * (D / 2);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[16];
          if (any) {
            tmem_ld_32x16(t_row + (which == 0 ? kDv : kDk) + half * (D / 2) + c * 16, v);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = 0;
          }
          if (w.slot >= 0) {
            st_global_32(part + c * 16, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
            st_global_32(part + c * 16 + 8, v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]);
          } else if (j < a.Skv) {
            store_bf16_16(out + c * 16, v, mul);
          }
        }
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
      }
    }
  }

  if (*abort_flag != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
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
        *out = a.accumulate ? *out + acc : acc;
      } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.dtable) + at;
        *out = __float2bfloat16(a.accumulate ? __bfloat162float(*out) + acc : acc);
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
  const int hb = idx % n_hb, tile = first + static_cast<int>(idx / n_hb);
  if (tile >= end) return;
  const int j = tile * 128 + r;
  if (j >= a.Skv) return;
  const bool sink = tile < p.sink_tiles;
  const int pieces = sink ? p.sink_pieces : p.pieces;
  const int slot0 = sink ? tile * pieces * n_hb + hb
                         : (p.sink_pieces > 1 ? sink_items : 0) + (tile - p.sink_tiles) * pieces * n_hb + hb;
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

// Steps (query tiles times heads) of a key tile, as in dkv_item.
static int dkv_steps(const BandArgs& a, int tile) {
  const int kv0 = tile * 128, first = std::max(0, kv0 - a.q_pos0);
  const int last = kv0 < a.sinks ? a.Sq - 1 : std::min(a.Sq - 1, std::min(kv0 + 127, a.Skv - 1) - a.q_pos0 + a.window - 1);
  return first <= last ? ((last >> 7) - (first >> 7) + 1) * (a.Hq / a.Hkv) : 0;
}

// Into how many pieces the steps of a key tile are cut.  Cutting costs the pieces' way through memory and a launch; not
// cutting leaves SMs idle when there are few key tiles and heads (grouped heads), or when the tiles that hold sinks, which
// every query sees, take many times as long as the others.  The estimate, in steps: the sum over rounds of the longest item
// of each, with two steps for an item's beginning and end and two more for a piece.
static void plan_pieces(BandBwdParams& p) {
  const BandArgs& a = p.a;
  const int sms = sm_count(), n_hb = a.Hkv * a.B;
  p.sink_tiles = a.window >= a.q_pos0 + a.Sq ? 0 : std::min((std::min(a.sinks, a.Skv) + 127) / 128, p.n_kt);
  int longest = 1, longest_sink = 1;
  for (int t = 0; t < p.n_kt; ++t) {
    int& most = t < p.sink_tiles ? longest_sink : longest;
    most = std::max(most, dkv_steps(a, t));
  }
  const int others = p.n_kt - p.sink_tiles;
  double best = 1e30;
  for (int c : {1, 2, 3, 4, 6, 8, 12, 16}) {
    if (c > longest || (c > 1 && others == 0)) break;
    const int piece = (longest + c - 1) / c;
    const int cs = p.sink_tiles == 0 ? 1 : std::min(64, (longest_sink + std::max(piece, 4) - 1) / std::max(piece, 4));
    const long long sink_items = static_cast<long long>(p.sink_tiles) * cs * n_hb, items = sink_items + static_cast<long long>(others) * c * n_hb;
    double cost = (c > 1 || cs > 1) ? 4.0 : 0.0;
    for (long long i = 0; i < items; i += sms) {
      if (i < sink_items) cost += longest_sink / cs + (cs > 1 ? 4 : 2);
      else cost += (dkv_steps(a, p.sink_tiles + static_cast<int>((i - sink_items) / n_hb / c)) + c - 1) / c + (c > 1 ? 4 : 2);
    }
    if (cost < best) {
      best = cost;
      p.pieces = c;
      p.sink_pieces = cs;
    }
  }
}

struct BandScratch {
  long long stat, part, dtable, total;  // floats
};
static BandScratch plan_bwd(BandBwdParams& p, const BandArgs& a) {
  p.a = a;
  p.n_qt = (a.Sq + 127) / 128;
  p.n_kt = (a.Skv + 127) / 128;
  p.t_last = a.buckets < 2 ? 0 : a.limit[a.buckets - 2];
  plan_pieces(p);
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
  p.n_items = static_cast<int>(dq_items);
  cudaError_t e = launch_pdl(band_bwd_dq_kernel<D>, dim3(std::min(p.n_items, sm_count())), dim3(kBwdBandThreads),
                             BandDqSmem<D>::kLut + lut + (p.a.dtable == nullptr ? 0 : BandDqSmem<D>::kBins), s, p);
  if (e != cudaSuccess) return e;
  p.n_items = static_cast<int>(dkv_items);
  e = launch_pdl(band_bwd_dkv_kernel<D>, dim3(std::min(p.n_items, sm_count())), dim3(kBwdBandThreads),
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

static int band_check(const BandArgs* a) {
  if (a->d != 64 && a->d != 96 && a->d != 128) return kBadArgument;
  if (a->B < 1 || a->Hkv < 1 || a->Hq % a->Hkv != 0 || a->Sq < 1 || a->Skv < 1) return kBadArgument;
  if (a->q_pos0 < 0 || a->window < 1 || a->sinks < 0 || !(a->scale > 0.f)) return kBadArgument;
  if (a->table != nullptr && (a->buckets < 2 || a->buckets > kMaxBuckets || a->limit[a->buckets - 2] > kMaxDistance)) return kBadArgument;
  auto aligned = [](const void* ptr, const BandStride& t, int bytes) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && t.b * 2 % bytes == 0 && t.s * 2 % bytes == 0 && t.h * 2 % bytes == 0;
  };
  // tile loads want 16 bytes; results are written in pieces of 32
  if (!aligned(a->q, a->q_st, 16) || !aligned(a->k, a->k_st, 16) || !aligned(a->v, a->v_st, 16) || !aligned(a->o, a->o_st, 32) ||
      !aligned(a->dout, a->dout_st, 16) || !aligned(a->dq, a->dq_st, 32) || !aligned(a->dk, a->dk_st, 32) ||
      !aligned(a->dv, a->dv_st, 32))
    return kBadArgument;
  return 0;
}

extern "C" int nmb_band_args_size() { return static_cast<int>(sizeof(BandArgs)); }

// Floats of `scratch` that the backward pass of these arguments needs.
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
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<64>), BandFwdSmem<64>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<96>), BandFwdSmem<96>::kLut + lut);
  opt_in(reinterpret_cast<const void*>(band_fwd_kernel<128>), BandFwdSmem<128>::kLut + lut);
  const int lut1 = lut_bytes(kMaxDistance, 1);
  opt_in(reinterpret_cast<const void*>(band_bwd_dq_kernel<64>), BandDqSmem<64>::kLut + lut1 + BandDqSmem<64>::kBins);
  opt_in(reinterpret_cast<const void*>(band_bwd_dq_kernel<96>), BandDqSmem<96>::kLut + lut1 + BandDqSmem<96>::kBins);
  opt_in(reinterpret_cast<const void*>(band_bwd_dq_kernel<128>), BandDqSmem<128>::kLut + lut1 + BandDqSmem<128>::kBins);
  opt_in(reinterpret_cast<const void*>(band_bwd_dkv_kernel<64>), BandDkvSmem<64>::kLut + lut1);
  opt_in(reinterpret_cast<const void*>(band_bwd_dkv_kernel<96>), BandDkvSmem<96>::kLut + lut1);
  opt_in(reinterpret_cast<const void*>(band_bwd_dkv_kernel<128>), BandDkvSmem<128>::kLut + lut1);
  return e == cudaSuccess ? 0 : 300 + e;
}

extern "C" int nmb_band_fwd(const BandArgs* a, void* stream) {
  if (int bad = band_check(a)) return bad;
  (void)cudaGetLastError();
  BandFwdParams p;
  p.a = *a;
  if (make_band_map(&p.q_map, a->q, a->q_st, a->d, a->Sq, a->Hq, a->B)) return 101;
  if (make_band_map(&p.k_map, a->k, a->k_st, a->d, a->Skv, a->Hkv, a->B)) return 102;
  if (make_band_map(&p.v_map, a->v, a->v_st, a->d, a->Skv, a->Hkv, a->B)) return 103;
  p.n_qt = (a->Sq + 127) / 128;
  p.s_pad = p.n_qt * 128;
  p.t_last = a->table == nullptr ? 0 : a->limit[a->buckets - 2];
  const long long tiles = static_cast<long long>(p.n_qt) * a->Hq * a->B;
  // one tile an item while every tile can have an SM of its own
  p.pair = tiles <= sm_count() ? 0 : (a->Hq / a->Hkv) % 2 == 0 ? 2 : 1;
  const long long items = p.pair == 0 ? tiles : p.pair == 2 ? tiles / 2 : static_cast<long long>((p.n_qt + 1) / 2) * a->Hq * a->B;
  if (items > (1 << 30)) return kTooLarge;
  p.n_items = static_cast<int>(items);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->d == 64 ? launch_band_fwd<64>(p, s) : a->d == 96 ? launch_band_fwd<96>(p, s) : launch_band_fwd<128>(p, s);
  return e == cudaSuccess ? 0 : 400 + e;
}

extern "C" int nmb_band_bwd(const BandArgs* a, void* stream) {
  if (int bad = band_check(a)) return bad;
  (void)cudaGetLastError();
  BandBwdParams p;
  const BandScratch w = plan_bwd(p, *a);
  p.stat = a->scratch;
  p.part = p.stat + w.stat;
  p.dtable_part = p.part + w.part;
  if (make_band_map(&p.q_map, a->q, a->q_st, a->d, a->Sq, a->Hq, a->B)) return 101;
  if (make_band_map(&p.k_map, a->k, a->k_st, a->d, a->Skv, a->Hkv, a->B)) return 102;
  if (make_band_map(&p.v_map, a->v, a->v_st, a->d, a->Skv, a->Hkv, a->B)) return 103;
  if (make_band_map(&p.do_map, a->dout, a->dout_st, a->d, a->Sq, a->Hq, a->B)) return 104;
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
  return e == cudaSuccess ? 0 : 500 + e;
}
