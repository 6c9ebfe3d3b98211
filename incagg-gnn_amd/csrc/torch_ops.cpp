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
// the grouped linear layer with its autograd node.  It is a Python module of plain functions: through
// the operator registry a call costs 3 us more, and a list 0.2 us a tensor.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>
#ifdef INCAGG_OPS_TRAIN
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <c10/hip/HIPGraphsC10Utils.h>
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

Tensor grad_norm(const std::vector<Tensor> &grads, int64_t norm_type, double max_norm, bool clip) {
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

// A parameter with its gradient and state; group: its hyperparameters.
struct AdamTensor {
  Tensor p, g, m, v, step;
  int64_t group;
};

Tensor adam_step_clipped(const std::vector<AdamTensor> &tensors,
                         const std::vector<incagg_adam_hyper> &hyper, double max_norm,
                         at::Device device) {
  std::vector<incagg_adam_clip_segment> segs;
  std::vector<Tensor> keep;
  segs.reserve(tensors.size());
  int64_t elements = 0;
  auto state = [&](const Tensor &t, int64_t numel) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat && t.device() == device,
                     "parameters and state must be float32 on one device");
    TORCH_CHECK_VALUE(t.is_contiguous() && t.numel() == numel,
                      "parameters and state must be contiguous and of one size");
    return numel ? static_cast<float *>(t.data_ptr()) : nullptr;
  };
  for (const AdamTensor &t : tensors) {
    TORCH_CHECK_TYPE(t.g.layout() == at::kStrided && t.g.scalar_type() == at::kFloat &&
                     t.g.device() == device, "gradients must be float32 on the parameter's device");
    const int64_t numel = t.p.numel();
    TORCH_CHECK_VALUE(t.g.numel() == numel, "a gradient differs in size from its parameter");
    const Tensor *g = &t.g;
    if (!g->is_contiguous()) {
      keep.push_back(g->detach().contiguous());
      g = &keep.back();
    }
    segs.push_back({state(t.p, numel), numel ? static_cast<const float *>(g->data_ptr()) : nullptr,
                    state(t.m, numel), state(t.v, numel), state(t.step, 1), numel, t.group});
    elements += numel;
  }
  c10::DeviceGuard guard(device);
  const int64_t n = (int64_t)segs.size();
  Scratch scratch(n, elements, device);
  check_status(incagg_adam_step_clipped_f32(
      segs.data(), n, hyper.data(), (int64_t)hyper.size(), max_norm, scratch.ptr(), scratch.doubles,
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
  // (the stride of a dimension of one says nothing, and contiguous() leaves it as it is)
  const bool unit = w_in.size(2) <= 1 || w_in.stride(2) == 1;
  const bool apart = w_in.size(1) <= 1 || w_in.stride(1) >= w_in.size(2);
  const Tensor w = unit && apart ? w_in : w_in.contiguous();
  const int64_t ldw = w.size(1) > 1 ? w.stride(1) : w.size(2);
  const Tensor bias = bias_in.defined() ? plain_rows(bias_in) : bias_in;
  const int64_t rows = x.size(0), k = x.size(1), n = w.size(trans_w ? 1 : 2);
  Tensor y = rows_empty(rows, n, pitch, x);
  c10::DeviceGuard guard(x.device());
  check_status(incagg_grouped_gemm(
      ptr_or_null<void>(x), pitch_of(x), w.data_ptr(), ldw, w.stride(0), trans_w ? 1 : 0,
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
// ends the process.  An error instead, before anything of it runs.  Asked of the running node's edges,
// which lead to the accumulation nodes of all its inputs, the bias (which is not saved) among them.
void check_recording() {
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto &edge : node->next_edges()) {
    if (!dynamic_cast<torch::autograd::AccumulateGrad *>(edge.function.get())) continue;
    const auto stream = edge.function->stream();
    TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(stream->device_index()).id(),
                "recording a backward pass while an earlier, eager graph of the same leaf is alive "
                "(a loss or output that is still referenced): delete it before the recording begins");
  }
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
      if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
        check_recording();
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
  const bool recorded = x.requires_grad() || w.requires_grad() || (bias && bias->requires_grad());
  // (forward-mode derivatives are refused by the node, which has none)
  const bool dual = x._fw_grad(0).defined() || w._fw_grad(0).defined() ||
                    (bias && bias->_fw_grad(0).defined());
  if (!dual && !(recorded && at::GradMode::is_enabled()))
    return grouped_gemm(x, w, true, bias.value_or(Tensor()), {ptr, order.value_or(Tensor())}, pitch_y);
  return GroupedLinear::apply(x, w, bias, ptr, order, pitch_y, pitch_dx);
}

// ---- the Python module -------------------------------------------------------------------------
struct NoGil {
  PyThreadState *state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

PyObject *raised(PyObject *o) {
  if (!o) throw python_error();
  return o;
}
int64_t to_int(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double to_double(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
const Tensor &to_tensor(PyObject *o, const char *name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
std::optional<Tensor> to_optional(PyObject *o, const char *name) {
  if (o == Py_None) return std::nullopt;
  return to_tensor(o, name);
}
void need_args(Py_ssize_t n, Py_ssize_t want) {
  TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n);
}
// An entry of a dict, by a name that is made a string object once.
PyObject *entry(PyObject *dict, PyObject *key) {
  TORCH_CHECK_TYPE(PyDict_Check(dict), "parameter groups and states must be dicts");
  PyObject *v = PyDict_GetItemWithError(dict, key);
  if (!v && !PyErr_Occurred()) PyErr_SetObject(PyExc_KeyError, key);
  return raised(v);
}
PyObject *name_of(const char *name) { return raised(PyUnicode_InternFromString(name)); }

// (parameters: list, norm_type, max_norm, clip) -> norm, None without a gradient
PyObject *py_grad_norm(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 4);
  TORCH_CHECK_TYPE(PyList_Check(args[0]), "parameters must be a list");
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  std::vector<Tensor> grads;
  grads.reserve(n);
  for (Py_ssize_t i = 0; i < n; i++) {
    const Tensor &g = to_tensor(PyList_GET_ITEM(args[0], i), "a parameter").grad();
    if (g.defined()) grads.push_back(g);
  }
  if (grads.empty()) Py_RETURN_NONE;
  const int64_t norm_type = to_int(args[1]);
  const double max_norm = to_double(args[2]);
  const bool clip = args[3] == Py_True;
  Tensor norm;
  {
    NoGil unlocked;
    norm = grad_norm(grads, norm_type, max_norm, clip);
  }
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// Looks up the parameters' states in the optimizer's own mapping, every time: it belongs to the user,
// who may replace a state or reorder the parameters between two steps.  The entries usually stand in
// the order in which the parameters are asked for, so the next one is tried first: finding a tensor by
// its hash is a call into Python, a fifth of a small step for twenty of them.
class StateWalk {
  PyObject *states_;
  Py_ssize_t next_ = 0;

  // The next entry's state if the entry is this parameter's, which is passed then.
  PyObject *pass(PyObject *parameter) {
    if (!PyDict_CheckExact(states_)) return nullptr;
    Py_ssize_t at = next_;
    PyObject *key, *value;
    if (!PyDict_Next(states_, &at, &key, &value) || key != parameter) return nullptr;
    next_ = at;
    return value;
  }

 public:
  explicit StateWalk(PyObject *states) : states_(states) {}
  void skip(PyObject *parameter) { pass(parameter); }
  PyObject *of(PyObject *parameter) {             // (a new reference)
    if (PyObject *state = pass(parameter)) {
      Py_INCREF(state);
      return state;
    }
    return raised(PyObject_GetItem(states_, parameter));      // KeyError where there is none
  }
};

// (param_groups: list of dicts, state: mapping of the parameters to their state dicts, max_norm)
PyObject *py_adam_step_clipped(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  static PyObject *const k_params = name_of("params"), *const k_lr = name_of("lr"),
                  *const k_betas = name_of("betas"), *const k_eps = name_of("eps"),
                  *const k_decay = name_of("weight_decay"), *const k_m = name_of("exp_avg"),
                  *const k_v = name_of("exp_avg_sq"), *const k_step = name_of("step");
  need_args(n_args, 3);
  TORCH_CHECK_TYPE(PyList_Check(args[0]), "parameter groups must be a list");
  StateWalk states(args[1]);
  std::vector<incagg_adam_hyper> hyper;
  std::vector<AdamTensor> tensors;
  std::optional<at::Device> device;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); i++) {
    PyObject *group = PyList_GET_ITEM(args[0], i);
    PyObject *params = entry(group, k_params), *betas = entry(group, k_betas);
    TORCH_CHECK_TYPE(PyList_Check(params), "params must be a list");
    TORCH_CHECK_TYPE(PySequence_Check(betas) && PySequence_Size(betas) == 2, "betas must be a pair");
    THPObjectPtr b1(raised(PySequence_GetItem(betas, 0))), b2(raised(PySequence_GetItem(betas, 1)));
    hyper.push_back({to_double(entry(group, k_lr)), to_double(b1.get()), to_double(b2.get()),
                     to_double(entry(group, k_eps)), to_double(entry(group, k_decay))});
    for (Py_ssize_t j = 0; j < PyList_GET_SIZE(params); j++) {
      PyObject *parameter = PyList_GET_ITEM(params, j);
      const Tensor p = to_tensor(parameter, "a parameter"), g = p.grad();
      if (!device) device = p.device();
      if (!g.defined()) {
        states.skip(parameter);
        continue;
      }
      THPObjectPtr state(states.of(parameter));
      tensors.push_back({p, g, to_tensor(entry(state, k_m), "exp_avg"),
                         to_tensor(entry(state, k_v), "exp_avg_sq"),
                         to_tensor(entry(state, k_step), "step"), (int64_t)i});
    }
  }
  TORCH_CHECK_VALUE(device, "no parameters");
  const double max_norm = to_double(args[2]);
  Tensor norm;
  {
    NoGil unlocked;
    norm = adam_step_clipped(tensors, hyper, max_norm, *device);
  }
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// (ids, n_groups) -> order, ptr
PyObject *py_group_rows(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 2);
  const Tensor ids = to_tensor(args[0], "ids");
  const int64_t n_groups = to_int(args[1]);
  std::tuple<Tensor, Tensor> r;
  {
    NoGil unlocked;
    r = group_rows(ids, n_groups);
  }
  THPObjectPtr order(raised(THPVariable_Wrap(std::get<0>(r))));
  THPObjectPtr ptr(raised(THPVariable_Wrap(std::get<1>(r))));
  return PyTuple_Pack(2, order.get(), ptr.get());
  END_HANDLE_TH_ERRORS
}

// (x, weight, bias or None, ptr, order or None, n_rows, pitch_y, pitch_dx) -> y
PyObject *py_grouped_linear(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 8);
  const Tensor x = to_tensor(args[0], "x"), w = to_tensor(args[1], "weight");
  const std::optional<Tensor> bias = to_optional(args[2], "bias");
  const Tensor ptr = to_tensor(args[3], "ptr");
  const std::optional<Tensor> order = to_optional(args[4], "order");
  const int64_t n_rows = to_int(args[5]), pitch_y = to_int(args[6]), pitch_dx = to_int(args[7]);
  Tensor y;
  {
    NoGil unlocked;
    y = grouped_linear(x, w, bias, ptr, order, n_rows, pitch_y, pitch_dx);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

template <typename F> PyCFunction function(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef g_functions[] = {
    {"grad_norm", function(py_grad_norm), METH_FASTCALL, nullptr},
    {"adam_step_clipped", function(py_adam_step_clipped), METH_FASTCALL, nullptr},
    {"group_rows", function(py_group_rows), METH_FASTCALL, nullptr},
    {"grouped_linear", function(py_grouped_linear), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_train_ops", nullptr, -1, g_functions};
#endif  // INCAGG_OPS_TRAIN

}  // namespace

#ifdef INCAGG_OPS_TRAIN
extern "C" __attribute__((visibility("default"))) PyObject *PyInit__train_ops() {
  return PyModule_Create(&g_module);
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
