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

namespace nmb {

constexpr float kBandLog2e = 1.4426950408889634f;
constexpr int kMaxBuckets = 128;
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

constexpr int kSimpleWarps = 4;

// One warp per query row; lane t takes keys t, t + 32, ... of a row's visible ranges for the scores and columns
// t, t + 32, ... of the head for the sums.
__global__ void band_fwd_kernel(const __grid_constant__ BandArgs p) {
  __shared__ float qs[kSimpleWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kSimpleWarps + warp;
  if (row >= static_cast<long long>(p.B) * p.Hq * p.Sq) return;
  const int i = row % p.Sq, h = (row / p.Sq) % p.Hq, b = row / p.Sq / p.Hq, hk = h / (p.Hq / p.Hkv);
  const __nv_bfloat16* q = band_row(p.q, b, i, h);
  for (int c = lane; c < p.d; c += 32) qs[warp][c] = __bfloat162float(q[c]);
  __syncwarp();
  const int pos = p.q_pos0 + i;
  const int last = min(pos, p.Skv - 1);
  const int first = max(0, pos - p.window + 1);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < 2; ++part) {
    const int lo = part == 0 ? 0 : first, hi = part == 0 ? min(min(p.sinks, first), last + 1) : last + 1;
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j < hi) {
        x = dot_row(band_row(p.k, b, j, hk), qs[warp], p.d) * (p.scale * kBandLog2e);
        if (p.table != nullptr) x += bias_log2(table_at(p, h, bucket_of(p, pos - j)));
      }
      const float mn = fmaxf(m, warp_max(x));
      const float w = mn == -INFINITY ? 0.f : exp2f(x - mn);
      const float a = m == -INFINITY ? 0.f : exp2f(m - mn);
      l = l * a + warp_sum(w);
      m = mn;
      for (int k = 0; k < 4; ++k) acc[k] *= a;
      for (int t = 0; t < 32 && j0 + t < hi; ++t) {
        const float wt = __shfl_sync(0xffffffffu, w, t);
        const __nv_bfloat16* v = band_row(p.v, b, j0 + t, hk);
        for (int k = 0; k < 4; ++k)
          if (k * 32 + lane < p.d) acc[k] = fmaf(wt, __bfloat162float(v[k * 32 + lane]), acc[k]);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  __nv_bfloat16* o = const_cast<__nv_bfloat16*>(band_row(p.o, b, i, h));
  for (int k = 0; k < 4; ++k)
    if (k * 32 + lane < p.d) o[k * 32 + lane] = __float2bfloat16(acc[k] * inv);
  if (lane == 0) {
    p.m[row] = l > 0.f ? m : INFINITY;  // a row that sees nothing: 2^(x - m) is 0 in the backward pass
    p.l[row] = l > 0.f ? log2f(l) : 0.f;
  }
}

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
  if (a->table != nullptr && (a->buckets < 2 || a->buckets > kMaxBuckets)) return kBadArgument;
  return 0;
}

extern "C" int nmb_band_args_size() { return static_cast<int>(sizeof(BandArgs)); }

// Floats of `dtable_part` that the backward pass of these arguments needs.
extern "C" long long nmb_band_dtable_part(int B, int Hq, int Sq, int buckets) {
  return static_cast<long long>(B) * Hq * Sq * buckets;
}

extern "C" int nmb_band_fwd(const BandArgs* a, void* stream) {
  if (int bad = band_check(a)) return bad;
  (void)cudaGetLastError();
  const long long rows = static_cast<long long>(a->B) * a->Hq * a->Sq;
  band_fwd_kernel<<<static_cast<unsigned>((rows + kSimpleWarps - 1) / kSimpleWarps), kSimpleWarps * 32, 0,
                    static_cast<cudaStream_t>(stream)>>>(*a);
  const cudaError_t e = cudaGetLastError();
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
