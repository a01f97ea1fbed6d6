// The Python side of include/tabby_decode.h on torch tensors (tabby_b200/decode.py documents the
// calls): checks of the arguments, outputs and workspaces from PyTorch's allocator, the tensors'
// current stream. In C++ because a decode step's small kernels take less time than the same
// checks and allocations take in Python (beam_step of 4 beams: 28 us a call there, 12 us here).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "tabby_decode.h"

namespace py = pybind11;
using at::Tensor;

namespace {

[[noreturn]] void value_error(const std::string &m) { throw py::value_error(m); }
[[noreturn]] void type_error(const std::string &m) { throw py::type_error(m); }

// Raises tabby_b200._lib.TabbyError for a failed call of the library.
void check(int status) {
  if (status == TABBY_OK) return;
  py::object error = py::module_::import("tabby_b200._lib").attr("TabbyError");
  py::object e = error(status, std::string(tabby_decode_last_error()));
  PyErr_SetObject(error.ptr(), e.ptr());
  throw py::error_already_set();
}

std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

// Type, shape (-1: any size) and device of an argument.
void need(const Tensor &x, const char *name, at::ScalarType type, at::IntArrayRef shape,
          at::Device device) {
  if (x.scalar_type() != type)
    type_error(std::string(name) + " must be " + c10::toString(type) + ", got " +
               c10::toString(x.scalar_type()));
  bool ok = x.dim() == (int64_t)shape.size();
  for (int64_t i = 0; ok && i < x.dim(); i++) ok = shape[i] < 0 || shape[i] == x.size(i);
  if (!ok)
    value_error(std::string(name) + " must have shape " + text(shape) + ", got " +
                text(x.sizes()));
  if (x.device() != device)
    value_error(std::string(name) + " must live on " + device.str() + ", got " +
                x.device().str());
}

at::Device cuda_device(const Tensor &x, const char *name) {
  if (!x.is_cuda()) value_error(std::string(name) + " must be a CUDA tensor");
  return x.device();
}

Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

// A tensor in the storage of `whole`, from element `first` on: outputs of one type share an
// allocation, without a view's bookkeeping. (Of several types they could not be saved together.)
Tensor part(const Tensor &whole, int64_t first, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(
      c10::TensorImpl::VIEW, c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

void *stream_of(at::Device device) {
  return c10::cuda::getCurrentCUDAStream(device.index()).stream();
}

int32_t size32(int64_t n, const char *what) {
  if (n > INT32_MAX || n < INT32_MIN)
    value_error(std::string(what) + " is out of range: " + std::to_string(n));
  return (int32_t)n;
}

// -1 for a type that the library does not know.
int32_t type_of(at::ScalarType t) {
  return t == at::kFloat ? TABBY_F32 : t == at::kBFloat16 ? TABBY_BF16
                                   : t == at::kHalf ? TABBY_F16 : -1;
}

py::tuple beam_step(Tensor logits, Tensor scores, std::optional<int64_t> n_out_or,
                    std::optional<Tensor> finished, int64_t eos) {
  const at::Device device = cuda_device(logits, "logits");
  if (logits.dim() != 3) value_error("logits must be [batch, beams, vocab]");
  const int32_t dtype = type_of(logits.scalar_type());
  if (dtype < 0) type_error("logits must be float32, bfloat16 or float16");
  const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  if (vocab > 1 && logits.stride(2) != 1) logits = logits.contiguous();
  need(scores, "scores", at::kFloat, {batch, beams}, device);
  scores = scores.contiguous();
  if (finished) {
    if (finished->scalar_type() != at::kByte)
      need(*finished, "finished", at::kBool, {batch, beams}, device);
    else
      need(*finished, "finished", at::kByte, {batch, beams}, device);
    finished = finished->contiguous();
  }
  const int64_t n_out = n_out_or.value_or(beams);
  size_t bytes = 0;
  check(tabby_beam_workspace_bytes(size32(batch, "batch"), size32(beams, "beams"),
                                   size32(vocab, "vocab"), size32(n_out, "n_out"), &bytes));
  const int64_t n = batch * n_out;
  Tensor next_scores = fresh({batch, n_out}, at::kFloat, device);
  const Tensor all = fresh({2 * n + batch}, at::kInt, device);
  Tensor parents = part(all, 0, {batch, n_out});
  Tensor tokens = part(all, n, {batch, n_out});
  Tensor status = part(all, 2 * n, {batch});
  Tensor ends = fresh({batch, n_out}, at::kBool, device);
  Tensor work = fresh({(int64_t)bytes}, at::kByte, device);
  check(tabby_beam_step_async(
      device.index(), logits.data_ptr(), dtype, logits.stride(0), logits.stride(1),
      (int32_t)batch, (int32_t)beams, (int32_t)vocab, scores.data_ptr<float>(),
      finished ? static_cast<const uint8_t *>(finished->data_ptr()) : nullptr,
      size32(eos, "eos_id"), (int32_t)n_out, next_scores.data_ptr<float>(),
      parents.data_ptr<int32_t>(), tokens.data_ptr<int32_t>(),
      static_cast<uint8_t *>(ends.data_ptr()), status.data_ptr<int32_t>(), work.data_ptr(), bytes,
      stream_of(device)));
  return py::make_tuple(next_scores, parents, tokens, ends, status);
}

// The layout of rows [rows, ...] of `size`-byte elements. With entries the shape is [rows, heads,
// entries, dim]; else the axes behind the first are merged where memory allows, and three may
// remain.
tabby_state_layout layout_of(at::IntArrayRef shape, at::IntArrayRef stride, int64_t size,
                             bool with_entries) {
  struct Axis {
    int64_t n, stride;
  };
  std::vector<Axis> axes;
  for (size_t i = 1; i < shape.size(); i++) axes.push_back({shape[i], stride[i]});
  if (with_entries) {
    if (axes.size() != 3) value_error("states with lengths must be [rows, heads, entries, dim]");
  } else {
    std::vector<Axis> merged;
    for (const Axis &a : axes) {
      if (a.n == 1) continue;
      if (!merged.empty() && merged.back().stride == a.n * a.stride)
        merged.back() = {merged.back().n * a.n, a.stride};
      else
        merged.push_back(a);
    }
    if (merged.empty() || merged.back().stride != 1) merged.push_back({1, 1});
    if (merged.size() > 3)
      value_error("a state's rows may have at most two strides beside the innermost");
    axes.assign(3 - merged.size(), {1, 0});
    axes.insert(axes.end(), merged.begin(), merged.end());
  }
  if (axes[2].n > 1 && axes[2].stride != 1)
    value_error("a state's innermost axis must be contiguous");
  tabby_state_layout l;
  l.row_stride = shape[0] > 1 ? stride[0] * size : 0;
  l.segment_stride = axes[0].stride * size;
  l.entry_stride = axes[1].stride * size;
  l.entry_bytes = axes[2].n * size;
  l.segments = size32(axes[0].n, "an axis of a state");
  l.entries = size32(axes[1].n, "an axis of a state");
  return l;
}

// Whether elements of a tensor share memory: taken from the smallest stride up, each must pass
// what the ones below it span. (The library's check of a layout, with the axis of a stack.)
bool overlaps(const Tensor &x) {
  std::vector<std::pair<int64_t, int64_t>> axes;  // stride, size
  for (int64_t i = 0; i < x.dim(); i++)
    if (x.size(i) > 1) axes.push_back({x.stride(i), x.size(i)});
  std::sort(axes.begin(), axes.end());
  int64_t span = 1;
  for (const auto &a : axes) {
    if (a.first < span) return true;
    span += a.first * (a.second - 1);
  }
  return false;
}

// States of one shape, type and strides.
struct Group {
  at::DimVector shape, stride;
  int64_t size;
  std::vector<void *> pointers;
};

// Groups of states with one layout each: of one tensor that stacks them or a sequence of them.
// Those without an element are left out and counted.
std::vector<Group> groups_of(const py::object &states, int64_t rows, at::Device device,
                             const std::string &name, int64_t *empty = nullptr) {
  std::vector<Group> groups;
  auto check_rows = [&](const Tensor &x, int64_t axis) {
    if (x.device() != device)
      value_error(name + " must live on " + device.str() + ", got " + x.device().str());
    if (x.dim() <= axis || x.size(axis) != rows)
      value_error(name + " must have " + std::to_string(rows) + " rows, got shape " +
                  text(x.sizes()));
  };
  if (THPVariable_Check(states.ptr())) {
    const Tensor &x = THPVariable_Unpack(states.ptr());
    check_rows(x, 1);
    if (x.numel() == 0) {
      if (empty) *empty = x.size(0);
      return groups;
    }
    if (overlaps(x)) value_error(name + " overlap");
    Group g;
    g.shape.assign(x.sizes().begin() + 1, x.sizes().end());
    g.stride.assign(x.strides().begin() + 1, x.strides().end());
    g.size = (int64_t)x.element_size();
    for (int64_t i = 0; i < x.size(0); i++)
      g.pointers.push_back(static_cast<char *>(x.data_ptr()) + i * x.stride(0) * g.size);
    groups.push_back(std::move(g));
    return groups;
  }
  for (py::handle h : states) {
    if (!THPVariable_Check(h.ptr())) type_error(name + " must be tensors");
    const Tensor &x = THPVariable_Unpack(h.ptr());
    check_rows(x, 0);
    if (x.numel() == 0) {
      if (empty) ++*empty;
      continue;
    }
    Group *at = nullptr;
    for (Group &g : groups)
      if (g.size == (int64_t)x.element_size() && at::IntArrayRef(g.shape) == x.sizes() &&
          at::IntArrayRef(g.stride) == x.strides())
        at = &g;
    if (!at) {
      groups.emplace_back();
      at = &groups.back();
      at->shape.assign(x.sizes().begin(), x.sizes().end());
      at->stride.assign(x.strides().begin(), x.strides().end());
      at->size = (int64_t)x.element_size();
    }
    at->pointers.push_back(x.data_ptr());
  }
  std::vector<void *> all;
  for (const Group &g : groups) all.insert(all.end(), g.pointers.begin(), g.pointers.end());
  std::sort(all.begin(), all.end());
  if (std::adjacent_find(all.begin(), all.end()) != all.end())
    value_error("one of the " + name + " is given twice");
  return groups;
}

void reorder_states(const py::object &states, Tensor parents, std::optional<Tensor> lengths) {
  const at::Device device = cuda_device(parents, "parents");
  need(parents, "parents", at::kInt, {-1, -1}, device);
  const int64_t batch = parents.size(0), beams = parents.size(1);
  parents = parents.contiguous();
  if (lengths) {
    need(*lengths, "lengths", at::kInt, {batch}, device);
    lengths = lengths->contiguous();
  }
  const std::vector<Group> groups = groups_of(states, batch * beams, device, "states");
  std::vector<tabby_state_layout> layouts;
  auto call = [&](const tabby_state_layout &l, void *const *pointers, int32_t n) {
    check(tabby_states_reorder_async(
        device.index(), pointers, n, &l, size32(batch, "batch"), size32(beams, "beams"),
        parents.data_ptr<int32_t>(), lengths ? lengths->data_ptr<int32_t>() : nullptr,
        stream_of(device)));
  };
  // All are checked before the first is moved: a call that raises has moved nothing.
  for (const Group &g : groups) {
    layouts.push_back(layout_of(g.shape, g.stride, g.size, lengths.has_value()));
    size32((int64_t)g.pointers.size(), "states");
    call(layouts.back(), nullptr, 0);
  }
  for (size_t i = 0; i < groups.size(); i++)
    call(layouts[i], groups[i].pointers.data(), (int32_t)groups[i].pointers.size());
}

// A tree's parents as [batch, nodes], a row of nodes for all.
Tensor trees(Tensor parents, int64_t batch, int64_t nodes, at::Device device) {
  if (parents.dim() == 1 && parents.size(0) == nodes) parents = parents.expand({batch, nodes});
  need(parents, "parents", at::kInt, {batch, nodes}, device);
  return nodes > 1 && parents.stride(1) != 1 ? parents.contiguous() : parents;
}

// Stride of an outer axis, 0 for an axis of one.
int64_t outer(const Tensor &x, int64_t axis) { return x.size(axis) > 1 ? x.stride(axis) : 0; }

// Rows of the last axis contiguous and 16-byte aligned.
bool fits(const Tensor &x) {
  return x.stride(3) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
         (outer(x, 0) | outer(x, 1) | outer(x, 2)) % 8 == 0;
}

Tensor tree_attention(Tensor q, const Tensor &k, const Tensor &v, Tensor lengths, Tensor parents,
                      std::optional<double> scale) {
  const at::Device device = cuda_device(q, "q");
  if (q.dim() != 4) value_error("q must be [batch, nodes, heads, dim]");
  if (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf)
    type_error("q must be bfloat16 or float16");
  const int64_t batch = q.size(0), nodes = q.size(1), heads = q.size(2), dim = q.size(3);
  need(k, "k_cache", q.scalar_type(), {batch, -1, -1, dim}, device);
  need(v, "v_cache", q.scalar_type(), k.sizes(), device);
  need(lengths, "lengths", at::kInt, {batch}, device);
  parents = trees(parents, batch, nodes, device);
  size_t bytes = 0;
  check(tabby_tree_workspace_bytes(size32(batch, "batch"), size32(nodes, "nodes"),
                                   size32(heads, "heads"), size32(k.size(1), "kv_heads"),
                                   size32(dim, "dim"), &bytes));
  if (!fits(q)) q = q.clone(at::MemoryFormat::Contiguous);
  if (!fits(k) || !fits(v))
    value_error("the caches' rows must be contiguous and 16-byte aligned");
  lengths = lengths.contiguous();
  Tensor out = fresh({batch, nodes, heads, dim}, q.scalar_type(), device);
  if (batch == 0) return out;
  Tensor work = fresh({(int64_t)bytes}, at::kByte, device);
  tabby_tree_attention_args a = {};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.q_batch_stride = outer(q, 0);
  a.q_node_stride = outer(q, 1);
  a.q_head_stride = outer(q, 2);
  a.k_batch_stride = outer(k, 0);
  a.k_head_stride = outer(k, 1);
  a.k_entry_stride = outer(k, 2);
  a.v_batch_stride = outer(v, 0);
  a.v_head_stride = outer(v, 1);
  a.v_entry_stride = outer(v, 2);
  a.out_batch_stride = outer(out, 0);
  a.out_node_stride = outer(out, 1);
  a.out_head_stride = outer(out, 2);
  a.lengths = lengths.data_ptr<int32_t>();
  a.parents = parents.data_ptr<int32_t>();
  a.parents_stride = outer(parents, 0);
  a.dtype = type_of(q.scalar_type());
  a.batch = (int32_t)batch;
  a.nodes = (int32_t)nodes;
  a.heads = (int32_t)heads;
  a.kv_heads = (int32_t)k.size(1);
  a.dim = (int32_t)dim;
  a.entries = size32(k.size(2), "entries");
  a.scale = (float)scale.value_or(1.0 / std::sqrt((double)dim));
  a.workspace = work.data_ptr();
  a.workspace_bytes = bytes;
  check(tabby_tree_attention_async(device.index(), &a, stream_of(device)));
  return out;
}

py::tuple tree_accept(const Tensor &sampled, Tensor tokens, Tensor parents, Tensor lengths,
                      const py::object &caches) {
  const at::Device device = cuda_device(tokens, "tokens");
  need(tokens, "tokens", at::kInt, {-1, -1}, device);
  const int64_t batch = tokens.size(0), nodes = tokens.size(1);
  need(sampled, "sampled", at::kInt, {batch, nodes}, device);
  parents = trees(parents, batch, nodes, device);
  need(lengths, "lengths", at::kInt, {batch}, device);
  tokens = tokens.contiguous();
  lengths = lengths.contiguous();
  int64_t empty = 0;
  const std::vector<Group> groups = groups_of(caches, batch, device, "caches", &empty);
  if (groups.size() > 1) value_error("the caches must share one layout");
  tabby_state_layout l = {};
  // (Without a cache no slot lies past the end: one without an entry is not the same.)
  if (empty > 0 && batch > 0) value_error("the caches must not be empty");
  if (!groups.empty()) l = layout_of(groups[0].shape, groups[0].stride, groups[0].size, true);
  const Tensor all = fresh({batch * (nodes + 3)}, at::kInt, device);
  Tensor path = part(all, 0, {batch, nodes});
  Tensor counts = part(all, batch * nodes, {batch});
  Tensor next_tokens = part(all, batch * (nodes + 1), {batch});
  Tensor next_lengths = part(all, batch * (nodes + 2), {batch});
  check(tabby_tree_accept_async(
      device.index(), sampled.data_ptr<int32_t>(), sampled.stride(0), sampled.stride(1),
      tokens.data_ptr<int32_t>(), parents.data_ptr<int32_t>(), outer(parents, 0),
      size32(batch, "batch"), size32(nodes, "nodes"), lengths.data_ptr<int32_t>(),
      path.data_ptr<int32_t>(), counts.data_ptr<int32_t>(), next_tokens.data_ptr<int32_t>(),
      next_lengths.data_ptr<int32_t>(), groups.empty() ? nullptr : groups[0].pointers.data(),
      groups.empty() ? 0 : size32((int64_t)groups[0].pointers.size(), "caches"),
      groups.empty() ? nullptr : &l, stream_of(device)));
  return py::make_tuple(path, counts, next_tokens, next_lengths);
}

py::tuple layout(const std::vector<int64_t> &shape, const std::vector<int64_t> &stride,
                 int64_t size, bool with_entries) {
  const tabby_state_layout l = layout_of(shape, stride, size, with_entries);
  return py::make_tuple(l.row_stride, l.segment_stride, l.entry_stride, l.entry_bytes, l.segments,
                        l.entries);
}

}  // namespace

PYBIND11_MODULE(tabby_decode_torch, m) {
  m.def("beam_step", &beam_step);
  m.def("reorder_states", &reorder_states);
  m.def("tree_attention", &tree_attention);
  m.def("tree_accept", &tree_accept);
  m.def("layout", &layout);
}
