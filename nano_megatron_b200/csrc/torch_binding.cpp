// The banded attention as an autograd operator of PyTorch, in C++.
//
// A training step of a short sequence is over on the GPU before an autograd function written in Python has been called:
// one forward and backward pass took 180 us on the host (of which the autograd engine itself takes about 45), against 90 us
// on the GPU for 8 x 512 tokens.  Everything that a call does between the check of its arguments and the launch is here.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <array>
#include <map>
#include <mutex>
#include <vector>

#include "band_args.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int kMaxDevices = 64;
std::array<int*, kMaxDevices> g_status{};  // per device: the word that kernels write on a failed wait
std::mutex g_limits_mutex;
std::map<std::pair<int64_t, int64_t>, std::vector<unsigned short>> g_limits;  // (buckets, max distance): first distances

void band_device(int64_t device, int64_t status) {
  TORCH_CHECK(device >= 0 && device < kMaxDevices, "device index ", device, " out of range");
  g_status[device] = reinterpret_cast<int*>(status);
}

void band_limits(int64_t buckets, int64_t max_distance, at::IntArrayRef limits) {
  TORCH_CHECK(buckets >= 2 && buckets <= nmb::kMaxBuckets && static_cast<int64_t>(limits.size()) == buckets - 1,
              "expected ", buckets - 1, " first distances for ", buckets, " buckets");
  std::vector<unsigned short> v(limits.begin(), limits.end());
  std::lock_guard<std::mutex> lock(g_limits_mutex);
  g_limits[{buckets, max_distance}] = std::move(v);
}

// `t`, or a copy where the kernels cannot address it: tile loads want contiguous rows, strides of whole 16 bytes (none of them
// 0) and a start on one.
bool strides_fit(const Tensor& t) {
  if (t.stride(3) != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8 != 0)) return false;
  return true;
}
Tensor readable(const Tensor& t) {
  if (!strides_fit(t)) return t.clone(at::MemoryFormat::Contiguous);
  if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) return at::empty_strided(t.sizes(), t.strides(), t.options()).copy_(t);
  return t;
}
// A gradient buffer: laid out as the input where that is dense, so that it can become the leaf's gradient as it is.
Tensor gradient_of(const Tensor& t) {
  bool same = t.is_non_overlapping_and_dense() && t.stride(3) == 1;
  for (int i = 0; i < 3; ++i) same = same && (t.size(i) == 1 || t.stride(i) % 16 == 0);
  return same ? at::empty_strided(t.sizes(), t.strides(), t.options()) : at::empty(t.sizes(), t.options());
}

// The stride of a dimension of one may be anything; the tile loads get one that is valid.
nmb::BandStride strides(const Tensor& t) {
  const int64_t d = t.size(3);
  return {t.size(0) > 1 ? t.stride(0) : d, t.size(1) > 1 ? t.stride(1) : d, t.size(2) > 1 ? t.stride(2) : d};
}
template <typename T>
void place(T*& ptr, nmb::BandStride& st, const Tensor& t) {
  ptr = static_cast<T*>(const_cast<void*>(t.const_data_ptr()));
  st = strides(t);
}

nmb::BandArgs arguments(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& out, const Tensor& rest,
                        const Tensor& stats, double scale, int64_t window, int64_t sinks, int64_t start, int64_t max_distance) {
  nmb::BandArgs a{};
  place(a.q, a.q_st, q);
  place(a.k, a.k_st, k);
  place(a.v, a.v_st, v);
  place(a.o, a.o_st, out);
  if (stats.defined()) {
    a.o_rest = static_cast<__nv_bfloat16*>(const_cast<void*>(rest.const_data_ptr()));
    a.rest_rows = static_cast<int>(rest.size(1));
    a.m = stats.data_ptr<float>();
    a.l = a.m + stats.numel() / 2;
  }
  a.B = static_cast<int>(q.size(0));
  a.Sq = static_cast<int>(q.size(1));
  a.Hq = static_cast<int>(q.size(2));
  a.d = static_cast<int>(q.size(3));
  a.Skv = static_cast<int>(k.size(1));
  a.Hkv = static_cast<int>(k.size(2));
  a.q_pos0 = static_cast<int>(start);
  a.window = static_cast<int>(std::min<int64_t>(window, 1 << 30));
  a.sinks = static_cast<int>(std::min<int64_t>(sinks, a.Skv));
  a.scale = static_cast<float>(scale);
  a.status = g_status[q.device().index()];
  TORCH_CHECK(a.status != nullptr, "the kernels are not set up for ", q.device());
  if (table.defined()) {
    a.table = table.const_data_ptr();
    a.table_fp32 = table.scalar_type() == at::kFloat;
    a.buckets = static_cast<int>(table.size(1));
    std::lock_guard<std::mutex> lock(g_limits_mutex);
    const auto found = g_limits.find({table.size(1), max_distance});
    TORCH_CHECK(found != g_limits.end(), "no first distances for ", table.size(1), " buckets up to ", max_distance);
    std::copy(found->second.begin(), found->second.end(), a.limit);
  }
  return a;
}

void* current_stream(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

struct BandAttention : torch::autograd::Function<BandAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                        const std::optional<Tensor>& table_in, double scale, int64_t window, int64_t sinks, int64_t start,
                        int64_t max_distance, bool train) {
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in);
    const Tensor table = table_in.has_value() ? table_in->contiguous() : Tensor();
    const Tensor out = at::empty(q.sizes(), q.options());
    Tensor rest, stats;
    if (train) {
      // Rows that see kFewKeys or more do without: there the error of D is below a tenth of the other roundings' (it falls with
      // the root of their number).  A table's gradient is a sum over all rows, and wants them all.  Later rows see more keys until
      // the window or the keys end, then fewer: those that see few are the first ones and, where the keys end, the last ones.
      constexpr int64_t kFewKeys = 256;
      const int64_t rows = q.size(1), keys = k.size(1);
      auto few = [&](int64_t position) {
        const int64_t first = std::max<int64_t>(0, position - window + 1);
        const int64_t band = std::max<int64_t>(0, std::min(position, keys - 1) - first + 1);
        return band + std::min(sinks, std::min(first, keys)) < kFewKeys;
      };
      const int64_t kept = table.defined() || few(start + rows - 1) ? rows : std::min(rows, std::max<int64_t>(0, kFewKeys - start));
      rest = at::empty({q.size(0), kept, q.size(2), q.size(3)}, q.options());
      stats = at::empty({2, q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    }
    const nmb::BandArgs a = arguments(q, k, v, table, out, rest, stats, scale, window, sinks, start, max_distance);
    Tensor scratch;
    if (const long long floats = nmb_band_fwd_scratch(&a)) scratch = at::empty({floats}, q.options().dtype(at::kFloat));
    const int rc = nmb_band_fwd_split(&a, scratch.defined() ? scratch.data_ptr<float>() : nullptr, current_stream(q));
    TORCH_CHECK(rc == 0, "nmb_band_fwd_split: launcher returned ", rc);
    if (train) {
      ctx->save_for_backward({q, k, v, table, out, rest, stats});
      ctx->saved_data["numbers"] =  // all of them exact in a double
          std::vector<double>{scale, double(window), double(sinks), double(start), double(max_distance)};
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result = gradients(ctx, grads[0]);
    if (at::GradMode::is_enabled()) {
      // a backward pass that builds a graph: whoever differentiates through these gradients is told that they cannot
      const int n = result[3].defined() ? 4 : 3;
      variable_list some(result.begin(), result.begin() + n);
      for (auto& t : some) t = t.detach().requires_grad_();
      auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of the banded attention cannot be differentiated again", n);
      some = (*error)(std::move(some));
      std::copy(some.begin(), some.end(), result.begin());
    }
    return result;
  }

  static variable_list gradients(AutogradContext* ctx, const Tensor& dout_in) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &table = saved[3], &out = saved[4], &rest = saved[5], &stats = saved[6];
    variable_list result(10);
    const c10::cuda::CUDAGuard guard(q.device());
    const std::vector<double> n = ctx->saved_data["numbers"].toDoubleVector();
    const Tensor dout = dout_in.defined() ? readable(dout_in.is_contiguous() ? dout_in : dout_in.contiguous()) : at::zeros_like(out);
    nmb::BandArgs a = arguments(q, k, v, table, out, rest, stats, n[0], static_cast<int64_t>(n[1]),
                                static_cast<int64_t>(n[2]), static_cast<int64_t>(n[3]), static_cast<int64_t>(n[4]));
    Tensor dq, dk, dv;
    // q, k and v the slices of one packed projection: their gradients go to the slices of one buffer, and are joined
    // without a copy
    const int64_t hq = q.size(2), hkv = k.size(2), d = q.size(3), row = (hq + 2 * hkv) * d;
    const std::array<int64_t, 4> packed{q.size(1) * row, row, d, 1};
    const auto* at_q = static_cast<const char*>(q.const_data_ptr());
    if (q.size(1) == k.size(1) && q.strides() == at::IntArrayRef(packed) && k.strides() == q.strides() && v.strides() == q.strides() &&
        k.const_data_ptr() == at_q + 2 * hq * d && v.const_data_ptr() == at_q + 2 * (hq + hkv) * d) {
      const Tensor all = at::empty({q.size(0), q.size(1), hq + 2 * hkv, d}, q.options());
      dq = all.narrow(2, 0, hq);
      dk = all.narrow(2, hq, hkv);
      dv = all.narrow(2, hq + hkv, hkv);
    } else {
      dq = gradient_of(q);
      dk = gradient_of(k);
      dv = gradient_of(v);
    }
    place(a.dout, a.dout_st, dout);
    place(a.dq, a.dq_st, dq);
    place(a.dk, a.dk_st, dk);
    place(a.dv, a.dv_st, dv);
    if (table.defined() && ctx->needs_input_grad(3)) {
      result[3] = at::empty(table.sizes(), table.options());
      a.dtable = result[3].data_ptr();
      a.dtable_fp32 = a.table_fp32;
    }
    nmb::BandPlan plan;
    const int bad = nmb_band_bwd_plan(&a, &plan);
    TORCH_CHECK(bad == 0, "nmb_band_bwd_plan: returned ", bad);
    const Tensor scratch = at::empty({plan.scratch}, stats.options());
    a.scratch = scratch.data_ptr<float>();
    const int rc = nmb_band_bwd_planned(&a, &plan, current_stream(q));
    TORCH_CHECK(rc == 0, "nmb_band_bwd: launcher returned ", rc);
    result[0] = dq;
    result[1] = dk;
    result[2] = dv;
    return result;
  }
};

// Is this a call that the kernels take as it is?  All that the entry points in Python look at, for one look from here.
bool ready(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& table, double scale, int64_t window,
           int64_t sinks, int64_t start, int64_t max_distance) {
  constexpr int64_t kMaxPosition = int64_t{1} << 30, kIntMax = (int64_t{1} << 31) - 1;
  for (const Tensor* t : {&q, &k, &v})
    if (!t->defined() || !t->is_cuda() || t->layout() != at::kStrided || t->scalar_type() != at::kBFloat16 || t->dim() != 4 ||
        t->numel() == 0 || t->device() != q.device())
      return false;
  const int64_t d = q.size(3);
  if (k.sizes() != v.sizes() || q.size(0) != k.size(0) || d != k.size(3) || (d != 64 && d != 96 && d != 128) || q.size(2) % k.size(2) != 0)
    return false;
  constexpr double kScaleLimit = 0x1p126;  // held in fp32, times log2(e)
  if (!(scale >= 1.0 / kScaleLimit && scale <= kScaleLimit) || window < 1 || window > kIntMax || sinks < 0 || sinks > kIntMax || start < 0 ||
      start > kMaxPosition || start + q.size(1) > kMaxPosition || k.size(1) > kMaxPosition || g_status[q.device().index()] == nullptr)
    return false;
  if (!table.has_value()) return true;
  if (!table->defined() || table->dim() != 2 || table->layout() != at::kStrided || table->device() != q.device() ||
      table->size(0) != q.size(2) || (table->scalar_type() != at::kBFloat16 && table->scalar_type() != at::kFloat))
    return false;
  std::lock_guard<std::mutex> lock(g_limits_mutex);
  return g_limits.count({table->size(1), max_distance}) != 0;  // what is there has passed the checks
}

// Tensors without memory (fake ones, of a trace) and calls under a mode that records operators: the kernels would run on null
// addresses, or beside the record.
void refuse_tracing(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t.unsafeGetTensorImpl()->is_python_dispatch(),
                              "banded attention: the kernels cannot be traced; wrap the call in torch.compiler.disable");
}
void refuse_tracing() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  TORCH_CHECK_NOT_IMPLEMENTED(!Modes::get_mode(Key::FAKE).has_value() && !Modes::get_mode(Key::PROXY).has_value() &&
                                  !Modes::get_mode(Key::FUNCTIONAL).has_value(),
                              "banded attention: the kernels cannot be traced; wrap the call in torch.compiler.disable");
}

// None where the call is not one for the kernels, or not yet.
std::optional<Tensor> band_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& table, double scale,
                                     int64_t window, int64_t sinks, int64_t start, int64_t max_distance) {
  const int64_t d = q.defined() && q.dim() == 4 ? q.size(3) : 0;
  if (q.defined() && q.scalar_type() == at::kBFloat16 && (d == 64 || d == 96 || d == 128)) {  // others take the plain expression
    refuse_tracing();
    for (const Tensor* t : {&q, &k, &v}) refuse_tracing(*t);
    if (table.has_value()) refuse_tracing(*table);
  }
  if (!ready(q, k, v, table, scale, window, sinks, start, max_distance)) return std::nullopt;
  const bool train = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                                    (table.has_value() && table->requires_grad()));
  return BandAttention::apply(q, k, v, table, scale, window, sinks, start, max_distance, train);
}

}  // namespace

TORCH_LIBRARY(nmb, m) {
  m.def("band_device(int device, int status) -> ()", band_device);
  m.def("band_limits(int buckets, int max_distance, int[] limits) -> ()", band_limits);
  m.def(
      "band_attention(Tensor q, Tensor k, Tensor v, Tensor? table, float scale, int window, int sinks, int start, int max_distance) "
      "-> Tensor?",
      band_attention);
}
