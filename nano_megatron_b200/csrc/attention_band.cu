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

struct BandTensor {
  void* ptr;
  long long stride_b, stride_s, stride_h;  // elements; head_dim is contiguous
};

// Arguments of both passes, laid out as in ops/band_attention.py.
struct BandArgs {
  BandTensor q, k, v, o, dout, dq, dk, dv;
  float* m;              // [B, Hq, Sq]
  float* l;              // [B, Hq, Sq]
  float* delta;          // [B, Hq, Sq]
  const void* table;     // [Hq, buckets] bf16 or fp32; null without a bias
  void* dtable;          // [Hq, buckets]; null when it is not wanted
  float* dtable_part;    // scratch of the backward pass
  int* status;
  int table_fp32, dtable_fp32, accumulate;  // accumulate: dtable is added to
  int B, Hq, Hkv, Sq, Skv, d;
  int q_pos0, window, sinks, buckets;
  float scale;
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
__device__ __forceinline__ int bucket_of(const BandArgs& p, int distance) {
  int b = 0;
  while (b + 1 < p.buckets && distance >= p.limit[b]) ++b;
  return b;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ const __nv_bfloat16* band_row(const BandTensor& t, int b, int s, int h) {
  return static_cast<const __nv_bfloat16*>(t.ptr) + b * t.stride_b + s * t.stride_s + h * t.stride_h;
}
__device__ __forceinline__ float dot_row(const __nv_bfloat16* a, const float* x, int d) {
  float acc = 0.f;
  for (int c = 0; c < d; c += 2) {
    const float2 f = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(a + c));
    acc = fmaf(f.x, x[c], fmaf(f.y, x[c + 1], acc));
  }
  return acc;
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

inline int lut_bytes(int t_last, int heads) { return (lut_entries(t_last) * (4 * heads + 1) + 15) / 16 * 16; }

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
// D[tmem] (+)= A[tmem, 128 rows of bf16 pairs] * B[smem]
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
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
  static constexpr int kNumBars = 2 * kStages + 12;
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
    // ---------------------------------------------------------- MMA issuer --
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_o = make_idesc_bf16(128, D, false, true);
      const uint32_t ring = smem_u32(smem + L::kRing);
      int base = 0, n_p[2] = {0, 0}, n_item[2] = {0, 0};
      bool ok = true;
      for (int round = 0; ok; ++round) {
        const int item = item_of_round(round);
        if (round * static_cast<int>(gridDim.x) >= p.n_items) break;
        if (item >= p.n_items) continue;
        const FwdItem w = fwd_item(p, item);
        const int n = w.all.count();
        int left[2] = {w.t[0].count(), w.t[1].count()};
        bool pending[2] = {false, false}, fresh[2] = {true, true}, any[2] = {left[0] > 0, left[1] > 0};
        // O += P V of tile u for slot t
        auto pv = [&](int t, int u) {
          const int pos = base + 2 * u + 1;
          if (!mbar_wait(&kv_full[pos % ST], (pos / ST) & 1, abort_flag, a.status, 63)) return false;
          if (fresh[t] && n_item[t] > 0 && !mbar_wait(&o_empty[t], (n_item[t] - 1) & 1, abort_flag, a.status, 64)) return false;
          if (!mbar_wait(&p_full[t], n_p[t] & 1, abort_flag, a.status, 65)) return false;
          ++n_p[t];
          tc_fence_after();
          const uint32_t sv = ring + (pos % ST) * L::kTile;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc_mma_bf16_ts(tmem + 256 + t * D, tmem + t * 128 + k * 8, make_smem_desc(sv + k * 2048, 16384, 1024), idesc_o,
                           (fresh[t] && k == 0) ? 0u : 1u);
          fresh[t] = false;
          pending[t] = false;
          if (left[t] == 0) tc_commit(&o_full[t]);
          return true;
        };
        for (int u = 0; u < n && ok; ++u) {
          const int j = tile_at(w.all, u), pos = base + 2 * u;
          if (!mbar_wait(&kv_full[pos % ST], (pos / ST) & 1, abort_flag, a.status, 66)) {
            ok = false;
            break;
          }
          for (int t = 0; t < 2 && ok; ++t) {
            if (pending[t]) ok = pv(t, u - 1);
            if (!ok || !w.t[t].uses(j)) continue;
            if (fresh[t] && !pending[t] && !mbar_wait(&q_full[t], n_item[t] & 1, abort_flag, a.status, 67)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sk = ring + (pos % ST) * L::kTile, sq = smem_u32(smem + L::kQ + t * L::kTile);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
              tc_mma_bf16(tmem + t * 128, make_smem_desc(sq + off, 16, 1024), make_smem_desc(sk + off, 16, 1024), idesc_s,
                          k != 0 ? 1u : 0u);
            }
            tc_commit(&s_full[t]);
            pending[t] = true;
            if (--left[t] == 0) tc_commit(&q_empty[t]);
          }
          if (!ok) break;
          tc_commit(&kv_empty[pos % ST]);
          if (u > 0) tc_commit(&kv_empty[(pos - 1) % ST]);
        }
        for (int t = 0; t < 2 && ok; ++t)
          if (pending[t]) ok = pv(t, n - 1);
        if (ok && n > 0) tc_commit(&kv_empty[(base + 2 * n - 1) % ST]);
        base += 2 * n;
        for (int t = 0; t < 2; ++t) n_item[t] += any[t];
      }
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
        named_sync(1 + t, 128);  // everyone has left the item before
        build_lut(a, h, p.t_last, map, lut, r, 128);
        named_sync(1 + t, 128);
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
      __nv_bfloat16* out = const_cast<__nv_bfloat16*>(band_row(a.o, w.b, row, h));
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

static int make_band_map(CUtensorMap* m, const BandTensor& t, int d, int S, int H, int B) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(S), static_cast<uint64_t>(H), static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {static_cast<uint64_t>(t.stride_s) * 2, static_cast<uint64_t>(t.stride_h) * 2,
                               static_cast<uint64_t>(t.stride_b) * 2};
  const uint32_t box[4] = {64, 128, 1, 1};
  return make_tmap_bf16(m, t.ptr, 4, dims, strides, box);
}

template <int D>
static cudaError_t launch_band_fwd(const BandFwdParams& p, cudaStream_t s) {
  const int lut = p.a.table == nullptr ? 0 : lut_bytes(p.t_last, 2);
  return launch_pdl(band_fwd_kernel<D>, dim3(std::min(p.n_items, sm_count())), dim3(kFwdThreads), BandFwdSmem<D>::kLut + lut, s, p);
}

constexpr int kSimpleWarps = 4;

__device__ __forceinline__ bool band_visible(const BandArgs& p, int pos, int j) {
  return j <= pos && j < p.Skv && (pos - j < p.window || j < p.sinks);
}

// One warp per query row: D, dQ and the row's part of the table's gradient (per warp in shared memory, in key order).
__global__ void band_bwd_dq_kernel(const __grid_constant__ BandArgs p) {
  __shared__ float qs[kSimpleWarps][128], gs[kSimpleWarps][128], bins[kSimpleWarps][kMaxBuckets];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kSimpleWarps + warp;
  if (row >= static_cast<long long>(p.B) * p.Hq * p.Sq) return;
  const int i = row % p.Sq, h = (row / p.Sq) % p.Hq, b = row / p.Sq / p.Hq, hk = h / (p.Hq / p.Hkv);
  const __nv_bfloat16 *q = band_row(p.q, b, i, h), *g = band_row(p.dout, b, i, h), *o = band_row(p.o, b, i, h);
  float delta = 0.f;
  for (int c = lane; c < p.d; c += 32) {
    qs[warp][c] = __bfloat162float(q[c]);
    gs[warp][c] = __bfloat162float(g[c]);
    delta = fmaf(gs[warp][c], __bfloat162float(o[c]), delta);
  }
  for (int c = lane; c < kMaxBuckets; c += 32) bins[warp][c] = 0.f;
  delta = warp_sum(delta);
  __syncwarp();
  const int pos = p.q_pos0 + i;
  const int last = min(pos, p.Skv - 1), first = max(0, pos - p.window + 1);
  const float m = p.m[row], l = p.l[row];
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < 2; ++part) {
    const int lo = part == 0 ? 0 : first, hi = part == 0 ? min(min(p.sinks, first), last + 1) : last + 1;
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      float ds = 0.f;
      int bucket = 0;
      if (j < hi) {
        float x = dot_row(band_row(p.k, b, j, hk), qs[warp], p.d) * (p.scale * kBandLog2e);
        if (p.table != nullptr) {
          bucket = bucket_of(p, pos - j);
          x += bias_log2(table_at(p, h, bucket));
        }
        ds = exp2f((x - m) - l) * (dot_row(band_row(p.v, b, j, hk), gs[warp], p.d) - delta);
      }
      for (int t = 0; t < 32 && j0 + t < hi; ++t) {
        const float s = __shfl_sync(0xffffffffu, ds, t);
        const int bt = __shfl_sync(0xffffffffu, bucket, t);
        if (lane == 0) bins[warp][bt] += s;
        const __nv_bfloat16* k = band_row(p.k, b, j0 + t, hk);
        for (int c = 0; c < 4; ++c)
          if (c * 32 + lane < p.d) acc[c] = fmaf(s, __bfloat162float(k[c * 32 + lane]), acc[c]);
      }
    }
  }
  __nv_bfloat16* dq = const_cast<__nv_bfloat16*>(band_row(p.dq, b, i, h));
  for (int c = 0; c < 4; ++c)
    if (c * 32 + lane < p.d) dq[c * 32 + lane] = __float2bfloat16(acc[c] * p.scale);
  if (lane == 0) p.delta[row] = delta;
  __syncwarp();
  if (p.dtable != nullptr)
    for (int c = lane; c < p.buckets; c += 32) p.dtable_part[row * p.buckets + c] = bins[warp][c];
}

// One warp per key row of a key head: dK and dV over the rows of the group's query heads.
__global__ void band_bwd_dkv_kernel(const __grid_constant__ BandArgs p) {
  __shared__ float ks[kSimpleWarps][128], vs[kSimpleWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kSimpleWarps + warp;
  if (row >= static_cast<long long>(p.B) * p.Hkv * p.Skv) return;
  const int j = row % p.Skv, hk = (row / p.Skv) % p.Hkv, b = row / p.Skv / p.Hkv, group = p.Hq / p.Hkv;
  const __nv_bfloat16 *k = band_row(p.k, b, j, hk), *v = band_row(p.v, b, j, hk);
  for (int c = lane; c < p.d; c += 32) {
    ks[warp][c] = __bfloat162float(k[c]);
    vs[warp][c] = __bfloat162float(v[c]);
  }
  __syncwarp();
  float ak[4] = {0.f, 0.f, 0.f, 0.f}, av[4] = {0.f, 0.f, 0.f, 0.f};
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    for (int i0 = max(0, j - p.q_pos0); i0 < p.Sq; i0 += 32) {
      if (j >= p.sinks && p.q_pos0 + i0 - j >= p.window) break;
      const int i = i0 + lane;
      float w = 0.f, ds = 0.f;
      if (i < p.Sq && band_visible(p, p.q_pos0 + i, j)) {
        const long long at = (static_cast<long long>(b) * p.Hq + h) * p.Sq + i;
        float x = dot_row(band_row(p.q, b, i, h), ks[warp], p.d) * (p.scale * kBandLog2e);
        if (p.table != nullptr) x += bias_log2(table_at(p, h, bucket_of(p, p.q_pos0 + i - j)));
        w = exp2f((x - p.m[at]) - p.l[at]);
        ds = w * (dot_row(band_row(p.dout, b, i, h), vs[warp], p.d) - p.delta[at]);
      }
      for (int t = 0; t < 32 && i0 + t < p.Sq; ++t) {
        const float wt = __shfl_sync(0xffffffffu, w, t), st = __shfl_sync(0xffffffffu, ds, t);
        const __nv_bfloat16 *q = band_row(p.q, b, i0 + t, h), *g = band_row(p.dout, b, i0 + t, h);
        for (int c = 0; c < 4; ++c)
          if (c * 32 + lane < p.d) {
            ak[c] = fmaf(st, __bfloat162float(q[c * 32 + lane]), ak[c]);
            av[c] = fmaf(wt, __bfloat162float(g[c * 32 + lane]), av[c]);
          }
      }
    }
  }
  __nv_bfloat16* dk = const_cast<__nv_bfloat16*>(band_row(p.dk, b, j, hk));
  __nv_bfloat16* dv = const_cast<__nv_bfloat16*>(band_row(p.dv, b, j, hk));
  for (int c = 0; c < 4; ++c)
    if (c * 32 + lane < p.d) {
      dk[c * 32 + lane] = __float2bfloat16(ak[c] * p.scale);
      dv[c * 32 + lane] = __float2bfloat16(av[c]);
    }
}

// dtable[h, b] = sum over batches and the parts of a head, in a fixed order.
// dtable_part: [B, Hq, parts, buckets].
__global__ void band_dtable_kernel(const __grid_constant__ BandArgs p, int parts) {
  __shared__ float sums[256];
  const int h = blockIdx.x / p.buckets, bucket = blockIdx.x % p.buckets;
  float acc = 0.f;
  for (int b = 0; b < p.B; ++b)
    for (int t = threadIdx.x; t < parts; t += 256)
      acc += p.dtable_part[((static_cast<long long>(b) * p.Hq + h) * parts + t) * p.buckets + bucket];
  sums[threadIdx.x] = acc;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    if (p.dtable_fp32) {
      float* out = static_cast<float*>(p.dtable) + blockIdx.x;
      *out = p.accumulate ? *out + sums[0] : sums[0];
    } else {
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.dtable) + blockIdx.x;
      *out = __float2bfloat16(p.accumulate ? __bfloat162float(*out) + sums[0] : sums[0]);
    }
  }
}

}  // namespace nmb

using namespace nmb;

static int band_check(const BandArgs* a) {
  if (a->d != 64 && a->d != 96 && a->d != 128) return kBadArgument;
  if (a->B < 1 || a->Hkv < 1 || a->Hq % a->Hkv != 0 || a->Sq < 1 || a->Skv < 1) return kBadArgument;
  if (a->q_pos0 < 0 || a->window < 1 || a->sinks < 0 || !(a->scale > 0.f)) return kBadArgument;
  if (a->table != nullptr && (a->buckets < 2 || a->buckets > kMaxBuckets || a->limit[a->buckets - 2] > kMaxDistance)) return kBadArgument;
  for (const BandTensor* t : {&a->q, &a->k, &a->v, &a->o, &a->dout, &a->dq, &a->dk, &a->dv}) {
    const bool written = t == &a->o || t == &a->dq || t == &a->dk || t == &a->dv;  // 32-byte stores
    const int bytes = written ? 32 : 16;
    if (reinterpret_cast<uintptr_t>(t->ptr) % bytes != 0 || t->stride_b * 2 % bytes != 0 || t->stride_s * 2 % bytes != 0 ||
        t->stride_h * 2 % bytes != 0)
      return kBadArgument;
  }
  return 0;
}

extern "C" int nmb_band_args_size() { return static_cast<int>(sizeof(BandArgs)); }

// Floats of `dtable_part` that the backward pass of these arguments needs.
extern "C" long long nmb_band_dtable_part(int B, int Hq, int Sq, int buckets) {
  return static_cast<long long>(B) * Hq * Sq * buckets;
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
  return e == cudaSuccess ? 0 : 300 + e;
}

extern "C" int nmb_band_fwd(const BandArgs* a, void* stream) {
  if (int bad = band_check(a)) return bad;
  (void)cudaGetLastError();
  BandFwdParams p;
  p.a = *a;
  if (make_band_map(&p.q_map, a->q, a->d, a->Sq, a->Hq, a->B)) return 101;
  if (make_band_map(&p.k_map, a->k, a->d, a->Skv, a->Hkv, a->B)) return 102;
  if (make_band_map(&p.v_map, a->v, a->d, a->Skv, a->Hkv, a->B)) return 103;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long rows = static_cast<long long>(a->B) * a->Hq * a->Sq;
  const long long keys = static_cast<long long>(a->B) * a->Hkv * a->Skv;
  band_bwd_dq_kernel<<<static_cast<unsigned>((rows + kSimpleWarps - 1) / kSimpleWarps), kSimpleWarps * 32, 0, s>>>(*a);
  band_bwd_dkv_kernel<<<static_cast<unsigned>((keys + kSimpleWarps - 1) / kSimpleWarps), kSimpleWarps * 32, 0, s>>>(*a);
  if (a->dtable != nullptr) band_dtable_kernel<<<a->Hq * a->buckets, 256, 0, s>>>(*a, a->Sq);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + e;
}
