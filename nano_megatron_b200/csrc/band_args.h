// Arguments of the banded attention's entry points (attention_band.cu), for callers that do not compile CUDA.
#pragma once

#include <cuda_bf16.h>

namespace nmb {

constexpr int kMaxBuckets = 128;
constexpr int kMaxDistance = 2048;

struct BandStride {
  long long b, s, h;  // elements; head_dim is contiguous
};

struct BandArgs {
  const __nv_bfloat16 *q, *k, *v;  // [B, Sq, Hq, d], [B, Skv, Hkv, d]
  __nv_bfloat16* o;
  __nv_bfloat16* o_rest;  // [B, rest_rows, Hq, d], dense: what rounding cut off of the first rows of o
  const __nv_bfloat16* dout;
  __nv_bfloat16 *dq, *dk, *dv;
  float* m;           // [B, Hq, Sq]; null, as l, for a forward pass without a backward one
  float* l;           // [B, Hq, Sq]
  float* scratch;     // nmb_band_bwd_scratch() floats, backward only
  const void* table;  // [Hq, buckets] bf16 or fp32; null without a bias
  void* dtable;       // [Hq, buckets]; null when it is not wanted
  int* status;
  BandStride q_st, k_st, v_st, o_st, dout_st, dq_st, dk_st, dv_st;
  int table_fp32, dtable_fp32;
  int B, Hq, Hkv, Sq, Skv, d;
  int q_pos0, window, sinks, buckets;
  float scale;
  int rest_rows;
  unsigned short limit[kMaxBuckets];  // first distance of bucket b + 1
};

// How the backward pass cuts key tiles that take long, and what it needs for that; of the sizes alone.
struct BandPlan {
  int sink_pieces, pieces;
  long long scratch;  // floats
};

}  // namespace nmb

extern "C" {
int nmb_band_args_size();
// Floats of `scratch` that the backward pass of these arguments needs.
long long nmb_band_bwd_scratch(const nmb::BandArgs* a);
int nmb_band_fwd(const nmb::BandArgs* a, void* stream);
// The same with the keys of a query tile cut into pieces where few tiles see many keys: floats of `scratch` that it takes then
// (0: not cut), and the call, which does without where `scratch` is null.
long long nmb_band_fwd_scratch(const nmb::BandArgs* a);
int nmb_band_fwd_split(const nmb::BandArgs* a, float* scratch, void* stream);
int nmb_band_bwd(const nmb::BandArgs* a, void* stream);
// The two steps of the backward pass for a caller that makes `scratch` in between.
int nmb_band_bwd_plan(const nmb::BandArgs* a, nmb::BandPlan* plan);
int nmb_band_bwd_planned(const nmb::BandArgs* a, const nmb::BandPlan* plan, void* stream);
// Kernels launched by the two so far.
long long nmb_band_launches();
}
