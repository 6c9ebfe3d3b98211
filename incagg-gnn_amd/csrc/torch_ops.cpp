// Operator objects that `torch.ops.load_library` can load: the reference package finds
// `_relabel` and `_async` next to its __init__ and loads them
// (torch_geometric_autoscale/__init__.py:8-10); these two objects register the same five
// operators with the same schemas (csrc/async.cpp:44-48, csrc/relabel.cpp:40-42) and forward
// every call to the C ABI of libincagg_gnn.so.  Nothing is computed here: tensors are checked
// the way the reference asserts them (csrc/cuda/async_cuda.cu:20-59,119-137,
// csrc/cpu/relabel_cpu.cpp:9-16) and unwrapped into pointers and sizes.
//
// One source, three objects: -DINCAGG_OPS_RELABEL builds `_relabel`, -DINCAGG_OPS_ASYNC `_async`;
// -DINCAGG_OPS_TRAIN builds `_train_ops`, which has no counterpart in the reference: calls whose
// kernels are shorter than their host side would be in Python -- gradient lists (norm, clipping, the
// clipped Adam step: a list of ten took longer to walk than the GPU needs for the whole call) and
// the grouped linear layer with its autograd node.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>
#ifdef INCAGG_OPS_TRAIN
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#endif

#include <deque>
#include <mutex>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/incagg_gnn.h"

namespace {

using at::Tensor;

void check_status(int64_t rc) { TORCH_CHECK(rc >= 0, incagg_last_error()); }

template <typename T>
const T *ptr_or_null(const Tensor &t) {
  return t.numel() ? static_cast<const T *>(t.data_ptr()) : nullptr;
}

#ifdef INCAGG_OPS_RELABEL
using RelabelFn = int (*)(const int64_t *, int64_t, const int64_t *, const void *, int64_t,
                          const int64_t *, int64_t, int, int64_t *, int64_t *, void *, int64_t *,
                          int64_t *);

std::tuple<Tensor, Tensor, std::optional<Tensor>, Tensor> relabel(
    RelabelFn fn, Tensor rowptr, Tensor col, std::optional<Tensor> optional_value, Tensor idx,
    bool bipartite) {
  TORCH_CHECK(!rowptr.is_cuda(), "No GPU version supported: relabelling runs on the host");
  TORCH_CHECK(!col.is_cuda(), "Col tensor must be a CPU tensor");
  TORCH_CHECK(!idx.is_cuda(), "Index tensor must be a CPU tensor");
  Tensor value;
  if (optional_value.has_value()) {
    value = optional_value.value();
    TORCH_CHECK(!value.is_cuda(), "Value tensor must be a CPU tensor");
    TORCH_CHECK(value.dim() == 1, "Value tensor must be one-dimensional");
    value = value.contiguous();
  }
  TORCH_CHECK(rowptr.scalar_type() == at::kLong, "rowptr must be int64");
  TORCH_CHECK(col.scalar_type() == at::kLong, "col must be int64");
  TORCH_CHECK(idx.scalar_type() == at::kLong, "idx must be int64");
  TORCH_CHECK(rowptr.dim() == 1 && rowptr.numel() >= 1, "rowptr must be 1-D and non-empty");
  rowptr = rowptr.contiguous();
  col = col.contiguous();
  idx = idx.contiguous();
  const int64_t n_nodes = rowptr.numel() - 1, n_idx = idx.numel();
  const int64_t ub = incagg_relabel_bound(rowptr.data_ptr<int64_t>(), n_nodes,
                                          ptr_or_null<int64_t>(idx), n_idx);
  check_status(ub);
  Tensor out_rowptr = at::empty({2 * n_idx + 1 + ub}, rowptr.options());
  Tensor out_col = at::empty({ub}, col.options());
  Tensor out_n_id = at::empty({n_idx + ub}, idx.options());
  Tensor out_value;
  if (value.defined()) out_value = at::empty({ub}, value.options());
  int64_t counts[3] = {0, 0, 0};
  check_status(fn(rowptr.data_ptr<int64_t>(), n_nodes, ptr_or_null<int64_t>(col),
                  value.defined() ? ptr_or_null<void>(value) : nullptr,
                  value.defined() ? (int64_t)value.element_size() : 0, ptr_or_null<int64_t>(idx),
                  n_idx, bipartite ? 1 : 0, out_rowptr.data_ptr<int64_t>(),
                  const_cast<int64_t *>(ptr_or_null<int64_t>(out_col)),
                  out_value.defined() ? const_cast<void *>(ptr_or_null<void>(out_value)) : nullptr,
                  const_cast<int64_t *>(ptr_or_null<int64_t>(out_n_id)), counts));
  std::optional<Tensor> ret_value;
  if (out_value.defined()) ret_value = out_value.narrow(0, 0, counts[0]).clone();
  return std::make_tuple(out_rowptr.narrow(0, 0, counts[2]).clone(),
                         out_col.narrow(0, 0, counts[0]).clone(), ret_value,
                         out_n_id.narrow(0, 0, counts[1]).clone());
}

std::tuple<Tensor, Tensor, std::optional<Tensor>, Tensor> relabel_one_hop(
    Tensor rowptr, Tensor col, std::optional<Tensor> value, Tensor idx, bool bipartite) {
  return relabel(&incagg_relabel_one_hop, rowptr, col, value, idx, bipartite);
}

std::tuple<Tensor, Tensor, std::optional<Tensor>, Tensor> relabel_one_hop_within_batch(
    Tensor rowptr, Tensor col, std::optional<Tensor> value, Tensor idx, bool bipartite) {
  return relabel(&incagg_relabel_one_hop_within_batch, rowptr, col, value, idx, bipartite);
}
#endif  // INCAGG_OPS_RELABEL

#ifdef INCAGG_OPS_ASYNC
// Tensors of queued reads stay referenced until the matching synchronize(), which is what
// capturing them by value in the worker's closure does in the reference (async_cuda.cu:63).
std::mutex g_inflight_mutex;
std::deque<std::vector<Tensor>> g_inflight;

Tensor host_i64(const Tensor &t, const char *name) {
  TORCH_CHECK(!t.is_cuda(), name, " tensor must be a CPU tensor");
  TORCH_CHECK(t.dim() == 1, name, " tensor must be one-dimensional");
  return t.to(at::kLong).contiguous();
}

void *non_default_stream(const Tensor &on_device) {
  const auto idx = on_device.get_device();
  auto cur = c10::hip::getCurrentHIPStream(idx);
  TORCH_CHECK(cur != c10::hip::getDefaultHIPStream(idx),
              "Asynchronous read/write requires a non-default stream");
  return static_cast<void *>(cur.stream());
}

int64_t row_elements(const Tensor &t) { return t.numel() / std::max<int64_t>(t.size(0), 1); }

void read_async(Tensor src, std::optional<Tensor> optional_offset,
                std::optional<Tensor> optional_count, Tensor index, Tensor dst, Tensor buffer) {
  TORCH_CHECK(!src.is_cuda(), "Source tensor must be a CPU tensor");
  TORCH_CHECK(!index.is_cuda(), "Index tensor must be a CPU tensor");
  TORCH_CHECK(dst.is_cuda(), "Target tensor must be a GPU tensor");
  TORCH_CHECK(!buffer.is_cuda(), "Buffer tensor must be a CPU tensor");
  TORCH_CHECK(buffer.is_pinned(), "Buffer tensor must be pinned");
  TORCH_CHECK(src.is_contiguous(), "Source tensor must be contiguous");
  TORCH_CHECK(dst.is_contiguous(), "Target tensor must be contiguous");
  TORCH_CHECK(buffer.is_contiguous(), "Buffer tensor must be contiguous");
  TORCH_CHECK(index.dim() == 1, "Index tensor must be one-dimensional");
  TORCH_CHECK(src.dim() >= 1 && dst.dim() >= 1 && buffer.dim() >= 1, "tensors must have rows");
  Tensor offset, count;
  int64_t n_chunks = 0;
  if (optional_offset.has_value()) {
    TORCH_CHECK(src.is_pinned(), "Source tensor must be pinned");
    TORCH_CHECK(optional_count.has_value(), "Count tensor is undefined");
    offset = host_i64(optional_offset.value(), "Offset");
    count = host_i64(optional_count.value(), "Count");
    TORCH_CHECK(offset.numel() == count.numel(), "Size mismatch");
    n_chunks = offset.numel();
  }
  TORCH_CHECK(index.numel() == 0 || index.scalar_type() == at::kLong, "Index tensor must be int64");
  index = index.contiguous();
  TORCH_CHECK(src.scalar_type() == dst.scalar_type() && src.scalar_type() == buffer.scalar_type(),
              "Source, target and buffer must share one dtype");
  const int64_t row_elems = row_elements(src);
  TORCH_CHECK(row_elements(dst) == row_elems && row_elements(buffer) == row_elems,
              "Source, target and buffer rows must have the same size");
  void *stream = non_default_stream(dst);
  c10::DeviceGuard guard(dst.device());
  check_status(incagg_stage_read_async(
      ptr_or_null<void>(src), src.size(0), row_elems * (int64_t)src.element_size(),
      n_chunks ? offset.data_ptr<int64_t>() : nullptr,
      n_chunks ? count.data_ptr<int64_t>() : nullptr, n_chunks, ptr_or_null<int64_t>(index),
      index.numel(), const_cast<void *>(ptr_or_null<void>(dst)), dst.size(0),
      const_cast<void *>(ptr_or_null<void>(buffer)), buffer.size(0), stream));
  std::vector<Tensor> keep{src, index, dst, buffer};
  if (n_chunks) {
    keep.push_back(offset);
    keep.push_back(count);
  }
  std::lock_guard<std::mutex> lock(g_inflight_mutex);
  g_inflight.push_back(std::move(keep));
}

void synchronize() {
  const int rc = incagg_stage_synchronize();
  {
    std::lock_guard<std::mutex> lock(g_inflight_mutex);
    if (!g_inflight.empty()) g_inflight.pop_front();
  }
  check_status(rc);
}

void write_async(Tensor src, Tensor offset, Tensor count, Tensor dst) {
  TORCH_CHECK(src.is_cuda(), "Source tensor must be a GPU tensor");
  TORCH_CHECK(!dst.is_cuda(), "Target tensor must be a CPU tensor");
  TORCH_CHECK(dst.is_pinned(), "Target tensor must be pinned");
  TORCH_CHECK(src.is_contiguous(), "Source tensor must be contiguous");
  TORCH_CHECK(dst.is_contiguous(), "Target tensor must be contiguous");
  TORCH_CHECK(src.dim() >= 1 && dst.dim() >= 1, "tensors must have rows");
  offset = host_i64(offset, "Offset");
  count = host_i64(count, "Count");
  TORCH_CHECK(offset.numel() == count.numel(), "Size mismatch");
  TORCH_CHECK(src.scalar_type() == dst.scalar_type(), "Source and target must share one dtype");
  const int64_t row_elems = row_elements(src);
  TORCH_CHECK(row_elements(dst) == row_elems, "Source and target rows must have the same size");
  void *stream = non_default_stream(src);
  c10::DeviceGuard guard(src.device());
  check_status(incagg_stage_write_async(
      ptr_or_null<void>(src), src.size(0), row_elems * (int64_t)src.element_size(),
      ptr_or_null<int64_t>(offset), ptr_or_null<int64_t>(count), offset.numel(),
      const_cast<void *>(ptr_or_null<void>(dst)), dst.size(0), stream));
}
#endif  // INCAGG_OPS_ASYNC

#ifdef INCAGG_OPS_TRAIN
int64_t element_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return INCAGG_DTYPE_F32;
    case at::kBFloat16: return INCAGG_DTYPE_BF16;
    case at::kHalf: return INCAGG_DTYPE_F16;
    default: return -1;
  }
}

// The gradients as segments.  What is wanted of them does not depend on the order of their elements,
// so a transposed one is taken as it lies; those with gaps go in as copies (`dense`), which are
// written back behind the call when `scaled`.
struct Segments {
  std::vector<incagg_norm_segment> segs;
  std::vector<std::pair<size_t, Tensor>> dense;
  int64_t elements = 0;

  Segments(const std::vector<Tensor> &grads, bool scaled) {
    segs.reserve(grads.size());
    for (size_t i = 0; i < grads.size(); i++) {
      const Tensor &g = grads[i];
      TORCH_CHECK(g.is_cuda(), "gradients must live on the GPU: the norm and clipping kernels are "
                  "HIP only and there is no CPU implementation");
      const int64_t code = g.layout() == at::kStrided ? element_code(g) : -1;
      TORCH_CHECK_TYPE(code >= 0, "gradients must be dense float32, bfloat16 or float16, got ",
                       g.scalar_type());
      TORCH_CHECK_VALUE(g.device() == grads[0].device(), "all gradients must be on one device");
      void *p = g.numel() ? g.data_ptr() : nullptr;
      if (!g.unsafeGetTensorImpl()->is_non_overlapping_and_dense()) {
        if (scaled) {
          if (g.numel() > 1)
            for (int64_t st : g.strides())
              TORCH_CHECK(st != 0, "a gradient's elements overlap in memory (an expanded tensor)");
          for (const auto &d : dense)           // (the others' memory is compared by the call itself)
            TORCH_CHECK(grads[d.first].data_ptr() != p, "two gradients overlap in memory");
        }
        dense.emplace_back(i, g.detach().contiguous());
        p = dense.back().second.data_ptr();
      }
      segs.push_back({p, g.numel(), code});
      elements += g.numel();
    }
  }
};

struct Scratch {
  Tensor ws, norm;
  int64_t doubles;
  Scratch(int64_t n_segs, int64_t elements, const at::Device &device)
      : doubles(incagg_grad_norm_ws_doubles(n_segs, elements)) {
    check_status(doubles);
    const auto options = at::TensorOptions().device(device);
    ws = at::empty({doubles + 1}, options.dtype(at::kDouble));
    norm = at::empty({}, options.dtype(at::kFloat));
  }
  double *ptr() { return ws.data_ptr<double>(); }
};

void *current_stream(const at::Device &device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

Tensor grad_norm(std::vector<Tensor> grads, int64_t norm_type, double max_norm, bool clip) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  const Segments s(grads, clip);
  const at::Device device = grads[0].device();
  c10::DeviceGuard guard(device);
  const int64_t n = (int64_t)s.segs.size();
  Scratch scratch(n, s.elements, device);
  float *out = scratch.norm.data_ptr<float>();
  if (!clip) {
    check_status(incagg_grad_norm(s.segs.data(), n, (int)norm_type, scratch.ptr(), scratch.doubles,
                                  out, current_stream(device)));
    return scratch.norm;
  }
  check_status(incagg_grad_clip(s.segs.data(), n, (int)norm_type, max_norm, scratch.ptr(),
                                scratch.doubles, out, current_stream(device)));
  for (const auto &d : s.dense) grads[d.first].detach().copy_(d.second);
  return scratch.norm;
}

// hyper: lr, beta1, beta2, eps, weight_decay of every parameter group; group[i]: of tensor i.
Tensor adam_step_clipped(std::vector<Tensor> params, std::vector<Tensor> grads,
                         std::vector<Tensor> exp_avg, std::vector<Tensor> exp_avg_sq,
                         std::vector<Tensor> steps, std::vector<int64_t> group,
                         std::vector<double> hyper, double max_norm, at::Device device) {
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n &&
                    steps.size() == n && group.size() == n && hyper.size() % 5 == 0,
                    "one gradient, two moments, a step count and a group for every parameter");
  std::vector<incagg_adam_clip_segment> segs;
  std::vector<Tensor> keep;
  segs.reserve(n);
  int64_t elements = 0;
  auto state = [&](const Tensor &t, int64_t numel) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat && t.device() == device,
                     "parameters and state must be float32 on one device");
    TORCH_CHECK_VALUE(t.is_contiguous() && t.numel() == numel,
                      "parameters and state must be contiguous and of one size");
    return numel ? static_cast<float *>(t.data_ptr()) : nullptr;
  };
  for (size_t i = 0; i < n; i++) {
    Tensor g = grads[i];
    TORCH_CHECK_TYPE(g.layout() == at::kStrided && g.scalar_type() == at::kFloat &&
                     g.device() == device, "gradients must be float32 on the parameter's device");
    const int64_t numel = params[i].numel();
    TORCH_CHECK_VALUE(g.numel() == numel, "a gradient differs in size from its parameter");
    if (!g.is_contiguous()) {
      g = g.detach().contiguous();
      keep.push_back(g);
    }
    segs.push_back({state(params[i], numel), numel ? static_cast<const float *>(g.data_ptr()) : nullptr,
                    state(exp_avg[i], numel), state(exp_avg_sq[i], numel), state(steps[i], 1), numel,
                    group[i]});
    elements += numel;
  }
  c10::DeviceGuard guard(device);
  Scratch scratch((int64_t)n, elements, device);
  check_status(incagg_adam_step_clipped_f32(
      segs.data(), (int64_t)n, reinterpret_cast<const incagg_adam_hyper *>(hyper.data()),
      (int64_t)(hyper.size() / 5), max_norm, scratch.ptr(), scratch.doubles,
      scratch.norm.data_ptr<float>(), current_stream(device)));
  return scratch.norm;
}

std::tuple<Tensor, Tensor> group_rows(const Tensor &ids, int64_t n_groups) {
  TORCH_CHECK(ids.is_cuda(), "ids must live on the GPU: the grouping kernels are HIP only and there "
              "is no CPU implementation");
  const bool wide = ids.scalar_type() == at::kLong;
  TORCH_CHECK_TYPE((wide || ids.scalar_type() == at::kInt) && ids.dim() == 1 && ids.is_contiguous(),
                   "ids must be a contiguous 1-D int64 or int32 tensor");
  TORCH_CHECK_VALUE(n_groups >= 1 && n_groups <= incagg_group_rows_max_groups(),
                    "n_groups must be between 1 and ", incagg_group_rows_max_groups(), ", got ",
                    n_groups);
  const int64_t rows = ids.numel(), need = incagg_group_rows_ws_ints(rows, n_groups);
  check_status(need);
  const auto options = ids.options().dtype(at::kInt);
  Tensor order = at::empty({rows}, options), ptr = at::empty({n_groups + 1}, options), ws;
  if (need) ws = at::empty({need}, options);
  c10::DeviceGuard guard(ids.device());
  check_status(incagg_group_rows(
      ptr_or_null<void>(ids), wide ? 1 : 0, rows, n_groups, need ? ws.data_ptr<int32_t>() : nullptr,
      need, const_cast<int32_t *>(ptr_or_null<int32_t>(order)), ptr.data_ptr<int32_t>(),
      current_stream(ids.device())));
  return {order, ptr};
}

// ---- the grouped linear layer ------------------------------------------------------------------
// Rows as the C ABI takes them: unit stride, no two rows in one place (an expanded gradient).
Tensor plain_rows(const Tensor &t) {
  const bool unit = t.size(1) <= 1 || t.stride(1) == 1;
  const bool apart = t.size(0) <= 1 || t.stride(0) >= t.size(1);
  return unit && apart ? t : t.contiguous();
}

int64_t pitch_of(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }

// [rows, width] with `pitch` elements from row to row (0: width).
Tensor rows_empty(int64_t rows, int64_t width, int64_t pitch, const Tensor &like) {
  if (pitch <= width) return at::empty({rows, width}, like.options());
  return at::empty_strided({rows, width}, {pitch, 1}, like.options());
}

struct Groups {
  Tensor ptr, order;                    // order undefined: the rows lie sorted
  int64_t count() const { return ptr.numel() - 1; }
  const int32_t *ptr_data() const { return ptr.data_ptr<int32_t>(); }
  const int32_t *order_data() const {
    return order.defined() && order.numel() ? order.data_ptr<int32_t>() : nullptr;
  }
};

Tensor grouped_gemm(const Tensor &x_in, const Tensor &w_in, bool trans_w, const Tensor &bias_in,
                    const Groups &groups, int64_t pitch) {
  const Tensor x = plain_rows(x_in);
  const bool plain = w_in.stride(2) == 1 && w_in.stride(1) >= w_in.size(2);
  const Tensor w = plain ? w_in : w_in.contiguous();
  const Tensor bias = bias_in.defined() ? plain_rows(bias_in) : bias_in;
  const int64_t rows = x.size(0), k = x.size(1), n = w.size(trans_w ? 1 : 2);
  Tensor y = rows_empty(rows, n, pitch, x);
  c10::DeviceGuard guard(x.device());
  check_status(incagg_grouped_gemm(
      ptr_or_null<void>(x), pitch_of(x), w.data_ptr(), w.stride(1), w.stride(0), trans_w ? 1 : 0,
      bias.defined() ? bias.data_ptr() : nullptr, bias.defined() ? pitch_of(bias) : 0,
      groups.ptr_data(), groups.order_data(), groups.count(), rows, k, n, (int)element_code(x),
      const_cast<void *>(ptr_or_null<void>(y)), pitch_of(y), current_stream(x.device())));
  return y;
}

std::pair<Tensor, Tensor> grouped_tn(const Tensor &a_in, const Tensor &b_in, const Groups &groups,
                                     bool sums) {
  const Tensor a = plain_rows(a_in), b = plain_rows(b_in);
  const int64_t rows = a.size(0), m = a.size(1), n = b.size(1), g = groups.count();
  const int code = (int)element_code(a);
  const int64_t need = incagg_grouped_tn_ws_bytes(g, rows, m, n, code);
  check_status(need);
  Tensor d = at::empty({g, m, n}, a.options()), s, ws;
  if (sums) s = at::empty({g, m}, a.options());
  if (need) ws = at::empty({need}, a.options().dtype(at::kByte));
  c10::DeviceGuard guard(a.device());
  check_status(incagg_grouped_tn(
      ptr_or_null<void>(a), pitch_of(a), ptr_or_null<void>(b), pitch_of(b), groups.ptr_data(),
      groups.order_data(), g, rows, m, n, code, d.data_ptr(), m * n, sums ? s.data_ptr() : nullptr,
      need ? ws.data_ptr() : nullptr, need, current_stream(a.device())));
  return {d, s};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A backward pass that is recorded into a HIP graph must not meet a leaf whose accumulation node a
// graph of the default stream keeps alive: autograd would tie the recording to that stream, which
// ends the process.  An error instead, before anything of it runs.
void check_recording(const Tensor &leaf) {
  if (!leaf.requires_grad() || !leaf.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!node) return;
  const auto stream = node->stream();
  TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(leaf.device().index()).id(),
              "recording a backward pass while an earlier, eager graph of the same leaf is alive "
              "(a loss or output that is still referenced): delete it before the recording begins");
}

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w,
                        const std::optional<Tensor> &bias, const Tensor &ptr,
                        const std::optional<Tensor> &order, int64_t pitch_y, int64_t pitch_dx) {
    const Groups groups{ptr, order.value_or(Tensor())};
    ctx->save_for_backward({x, w, ptr, groups.order});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["pitch"] = pitch_dx;
    return grouped_gemm(x, w, true, bias.value_or(Tensor()), groups, pitch_y);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor x = saved[0], w = saved[1], dy = grads[0];
    const Groups groups{saved[2], saved[3]};
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const bool need_w = ctx->needs_input_grad(1), need_b = has_bias && ctx->needs_input_grad(2);
    variable_list out(7);
    {
      c10::DeviceGuard guard(x.device());
      if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
        check_recording(x);
        check_recording(w);
      }
    }
    {
      at::AutoGradMode no_graph(false);
      if (ctx->needs_input_grad(0))
        out[0] = grouped_gemm(dy, w, false, Tensor(), groups, ctx->saved_data["pitch"].toInt());
      if (need_w || need_b) {
        const auto d = grouped_tn(dy, x, groups, need_b);
        if (need_w) out[1] = d.first;
        if (need_b) out[2] = d.second;
      }
    }
    if (!at::GradMode::is_enabled()) return out;
    // a graph of the gradients was asked for: differentiating them again raises
    for (int i = 0; i < 3; i++) {
      if (!out[i].defined()) continue;
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "the grouped linear layer has no second derivatives", 1);
      Tensor t = out[i].detach();
      t.set_requires_grad(true);
      out[i] = (*error)({t})[0];
    }
    return out;
  }
};

Tensor grouped_linear(const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias,
                      const Tensor &ptr, const std::optional<Tensor> &order, int64_t n_rows,
                      int64_t pitch_y, int64_t pitch_dx) {
  TORCH_CHECK(x.is_cuda(), "x must live on the GPU: the grouped products are HIP only and there is "
              "no CPU implementation");
  TORCH_CHECK_TYPE(element_code(x) >= 0 && w.scalar_type() == x.scalar_type() &&
                   (!bias || bias->scalar_type() == x.scalar_type()),
                   "x, weight and bias must be of one dtype: float32, bfloat16 or float16");
  TORCH_CHECK_VALUE(x.device() == ptr.device() && w.device() == x.device() &&
                    (!bias || bias->device() == x.device()),
                    "x, weight, bias and groups must be on one device");
  const int64_t g = ptr.numel() - 1;
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == n_rows && x.size(1) >= 1, "x must be [", n_rows,
                    ", in], got ", x.sizes());
  TORCH_CHECK_VALUE(w.dim() == 3 && w.size(0) == g && w.size(1) >= 1 && w.size(2) == x.size(1),
                    "weight must be [", g, ", out, ", x.size(1), "], got ", w.sizes());
  TORCH_CHECK_VALUE(!bias || (bias->dim() == 2 && bias->size(0) == g && bias->size(1) == w.size(1)),
                    "bias must be [", g, ", ", w.size(1), "]");
  return GroupedLinear::apply(x, w, bias, ptr, order, pitch_y, pitch_dx);
}
#endif  // INCAGG_OPS_TRAIN

}  // namespace

#ifdef INCAGG_OPS_TRAIN
TORCH_LIBRARY(incagg_train, m) {
  m.def("grad_norm(Tensor[] grads, int norm_type, float max_norm, bool clip) -> Tensor", &grad_norm);
  m.def("adam_step_clipped(Tensor[] params, Tensor[] grads, Tensor[] exp_avg, Tensor[] exp_avg_sq, "
        "Tensor[] steps, int[] group, float[] hyper, float max_norm, Device device) -> Tensor",
        &adam_step_clipped);
  m.def("group_rows(Tensor ids, int n_groups) -> (Tensor, Tensor)", &group_rows);
  m.def("grouped_linear(Tensor x, Tensor weight, Tensor? bias, Tensor ptr, Tensor? order, int n_rows, "
        "int pitch_y, int pitch_dx) -> Tensor", &grouped_linear);
}
#else
// Both objects contribute to one namespace, hence fragments.
TORCH_LIBRARY_FRAGMENT(torch_geometric_autoscale, m) {
#ifdef INCAGG_OPS_RELABEL
  m.def("relabel_one_hop(Tensor rowptr, Tensor col, Tensor? value, Tensor idx, bool bipartite)"
        " -> (Tensor, Tensor, Tensor?, Tensor)", &relabel_one_hop);
  m.def("relabel_one_hop_within_batch(Tensor rowptr, Tensor col, Tensor? value, Tensor idx, "
        "bool bipartite) -> (Tensor, Tensor, Tensor?, Tensor)", &relabel_one_hop_within_batch);
#endif
#ifdef INCAGG_OPS_ASYNC
  m.def("synchronize() -> ()", &synchronize);
  m.def("read_async(Tensor src, Tensor? offset, Tensor? count, Tensor index, Tensor dst, "
        "Tensor buffer) -> ()", &read_async);
  m.def("write_async(Tensor src, Tensor offset, Tensor count, Tensor dst) -> ()", &write_async);
#endif
}
#endif
