// Host path of the Python backend in C++: argument checks, scratch, descriptor, launch and autograd of the operators that
// are called often and on small inputs, where the interpreter cost more than the kernels (an aggregation of 11,000 edges:
// 32 us per call through ctypes and a Python autograd function, 20 us of it kernels).
//
// The kernels stay behind the C ABI of libcxgnn_b200.so: this module opens the library it is told to (init) and calls its
// entry points. No CUDA code, no other state than the scratch buffers per stream and the transposed graphs.
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/autocast_mode.h>
#include <c10/core/Event.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <list>
#include <map>
#include <mutex>

#include "../../include/cxgnn_b200.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- the library -----------------------------------------------------------------------------------------------------
struct Lib {
  void *handle = nullptr;
#define CXG_FN(name) decltype(&::name) name = nullptr
  CXG_FN(cxg_last_error_string);
  CXG_FN(cxg_spmm_csr_workspace_size);
  CXG_FN(cxg_spmm_csr);
  CXG_FN(cxg_spmm_csr_rows_size);
  CXG_FN(cxg_spmm_csr_rows);
  CXG_FN(cxg_spmm_csr_backward);
  CXG_FN(cxg_csr_transpose_workspace_size);
  CXG_FN(cxg_csr_transpose);
  CXG_FN(cxg_gather_edges);
  CXG_FN(cxg_linear_f32_supported);
  CXG_FN(cxg_linear_f32);
  CXG_FN(cxg_dense_wgrad_f32_workspace_size);
  CXG_FN(cxg_dense_wgrad_f32);
  CXG_FN(cxg_column_sum_workspace_size);
  CXG_FN(cxg_column_sum);
  CXG_FN(cxg_gat_scores);
  CXG_FN(cxg_gat_fused_workspace_size);
  CXG_FN(cxg_gat_fused_forward);
  CXG_FN(cxg_gat_fused_backward_bias);
  CXG_FN(cxg_gat_att_grad_workspace_size);
  CXG_FN(cxg_gat_scores_backward_add);
  CXG_FN(cxg_head_mean_bias);
  CXG_FN(cxg_gat_pad_heads);
  CXG_FN(cxg_gat_unpad_heads);
  CXG_FN(cxg_gather_rows);
  CXG_FN(cxg_sample_batch_bounds);
  CXG_FN(cxg_sample_batch);
  CXG_FN(cxg_relation_pairs_workspace_size);
  CXG_FN(cxg_relation_pairs_count);
  CXG_FN(cxg_relation_pairs_fill);
  CXG_FN(cxg_rows8_pitch);
  CXG_FN(cxg_rows8_write);
  CXG_FN(cxg_rows8_write_at);
  CXG_FN(cxg_rows8_read);
  CXG_FN(cxg_rows8_aggregate_workspace_size);
  CXG_FN(cxg_rows8_aggregate);
  CXG_FN(cxg_rows8_wgrad_workspace_size);
  CXG_FN(cxg_rows8_wgrad);
  CXG_FN(cxg_residual_norm_max_width);
  CXG_FN(cxg_residual_norm_keeps);
  CXG_FN(cxg_residual_norm_forward);
  CXG_FN(cxg_residual_norm_backward_workspace_size);
  CXG_FN(cxg_residual_norm_backward);
#undef CXG_FN
} lib;

void init(const std::string &path) {
  lib.handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (lib.handle == nullptr) throw std::runtime_error(std::string("cannot open ") + path + ": " + dlerror());
#define CXG_FN(name)                                                                \
  lib.name = reinterpret_cast<decltype(&::name)>(dlsym(lib.handle, #name));         \
  if (lib.name == nullptr) throw std::runtime_error(std::string("no ") + #name + " in " + path)
  CXG_FN(cxg_last_error_string);
  CXG_FN(cxg_spmm_csr_workspace_size);
  CXG_FN(cxg_spmm_csr);
  CXG_FN(cxg_spmm_csr_rows_size);
  CXG_FN(cxg_spmm_csr_rows);
  CXG_FN(cxg_spmm_csr_backward);
  CXG_FN(cxg_csr_transpose_workspace_size);
  CXG_FN(cxg_csr_transpose);
  CXG_FN(cxg_gather_edges);
  CXG_FN(cxg_linear_f32_supported);
  CXG_FN(cxg_linear_f32);
  CXG_FN(cxg_dense_wgrad_f32_workspace_size);
  CXG_FN(cxg_dense_wgrad_f32);
  CXG_FN(cxg_column_sum_workspace_size);
  CXG_FN(cxg_column_sum);
  CXG_FN(cxg_gat_scores);
  CXG_FN(cxg_gat_fused_workspace_size);
  CXG_FN(cxg_gat_fused_forward);
  CXG_FN(cxg_gat_fused_backward_bias);
  CXG_FN(cxg_gat_att_grad_workspace_size);
  CXG_FN(cxg_gat_scores_backward_add);
  CXG_FN(cxg_head_mean_bias);
  CXG_FN(cxg_gat_pad_heads);
  CXG_FN(cxg_gat_unpad_heads);
  CXG_FN(cxg_gather_rows);
  CXG_FN(cxg_sample_batch_bounds);
  CXG_FN(cxg_sample_batch);
  CXG_FN(cxg_relation_pairs_workspace_size);
  CXG_FN(cxg_relation_pairs_count);
  CXG_FN(cxg_relation_pairs_fill);
  CXG_FN(cxg_rows8_pitch);
  CXG_FN(cxg_rows8_write);
  CXG_FN(cxg_rows8_write_at);
  CXG_FN(cxg_rows8_read);
  CXG_FN(cxg_rows8_aggregate_workspace_size);
  CXG_FN(cxg_rows8_aggregate);
  CXG_FN(cxg_rows8_wgrad_workspace_size);
  CXG_FN(cxg_rows8_wgrad);
  CXG_FN(cxg_residual_norm_max_width);
  CXG_FN(cxg_residual_norm_keeps);
  CXG_FN(cxg_residual_norm_forward);
  CXG_FN(cxg_residual_norm_backward_workspace_size);
  CXG_FN(cxg_residual_norm_backward);
#undef CXG_FN
}

[[noreturn]] void fail(const std::string &text) { throw std::runtime_error(text); }

void check(int rc, const char *what) {
  if (rc != 0) fail(std::string(what) + " failed with status " + std::to_string(rc) + ": " + lib.cxg_last_error_string());
}

const Tensor &cuda(const Tensor &t, const char *name) {
  if (!t.is_cuda()) fail(std::string(name) + " must be a CUDA tensor (this backend has no CPU path)");
  if (!t.is_contiguous()) fail(std::string(name) + " must be contiguous");
  return t;
}
const Tensor &of_type(const Tensor &t, const char *name, std::initializer_list<at::ScalarType> types) {
  cuda(t, name);
  for (auto s : types)
    if (t.scalar_type() == s) return t;
  fail(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + ", which this operator does not take");
}
const Tensor &feature(const Tensor &t, const char *name) { return of_type(t, name, {at::kFloat, at::kBFloat16}); }
const Tensor &index_of(const Tensor &t, const char *name) { return of_type(t, name, {at::kLong, at::kInt}); }
const Tensor &f32(const Tensor &t, const char *name) { return of_type(t, name, {at::kFloat}); }

// A tensor under forward-mode differentiation. The kernels know nothing of its tangent: torch's operators take it where
// there is one, and the operators of this module go through their autograd function, which refuses it.
bool has_tangent(const Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }

// Whether the pass has to go through the autograd function.
bool recorded(const Tensor &t) { return (t.requires_grad() && at::GradMode::is_enabled()) || has_tangent(t); }
bool recorded(const optional<Tensor> &t) { return t && recorded(*t); }
template <typename A, typename... B>
bool recorded(const A &a, const B &...b) {
  return recorded(a) || recorded(b...);
}

// Whether torch's own operator has to be called: transforms (vmap, functionalisation, fake tensors and other subclasses),
// forward-mode differentiation, tracing.
bool foreign(const Tensor &t) { return at::isTensorSubclassLike(t) || has_tangent(t); }
bool foreign(const optional<Tensor> &t) { return t && foreign(*t); }
template <typename... T>
bool for_torch(const T &...t) {
  return torch::jit::tracer::isTracing() || (foreign(t) || ...);
}

void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The capture that records what the stream is given, or none.
optional<unsigned long long> capture_of(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &status, &id));
  if (status == cudaStreamCaptureStatusNone) return c10::nullopt;
  return id;
}

// ---- scratch ---------------------------------------------------------------------------------------------------------
// One buffer per (device, stream), grown on demand; contents never carry over. `kind` names the entry point family that
// used it last (whose status word check_device_status can ask for). The launches of one call hand the buffer on to each
// other, so whoever uses it holds its lock until the last of them is issued: two threads may work on one stream (a backward
// runs on a thread of the autograd engine, without the interpreter's lock), and launches of another call in between would
// overwrite what the next kernel reads. A call that a graph capture records gets a buffer of its own out of the capture's
// memory: the graph runs it again when the stream's buffer has long been replaced, or is in use.
struct Scratch {
  std::mutex in_use;
  Tensor buf;
  std::string kind;
};
std::mutex scratch_lock;
std::map<std::pair<int, void *>, Scratch> scratch;

Scratch &scratch_of(int device, void *stream) {
  std::lock_guard<std::mutex> hold(scratch_lock);
  return scratch[{device, stream}];
}

// Takes the lock without keeping other threads from the interpreter meanwhile: the holder may be Python code.
std::unique_lock<std::mutex> lock_for_launches(std::mutex &m) {
  std::unique_lock<std::mutex> hold(m, std::try_to_lock);
  if (!hold.owns_lock()) {
    if (PyGILState_Check()) {
      py::gil_scoped_release others;
      hold.lock();
    } else {
      hold.lock();
    }
  }
  return hold;
}

// The stream's scratch buffer while this thread may use it.
struct Workspace {
  std::unique_lock<std::mutex> hold;
  Tensor buf;
  void *data() const { return buf.data_ptr(); }
  size_t bytes() const { return static_cast<size_t>(buf.numel()); }
};

Workspace workspace_on(int device, void *stream, int64_t bytes, const char *kind) {
  auto buffer = [&]() {
    return at::empty({std::max<int64_t>(bytes, 1 << 20)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
  };
  if (capture_of(static_cast<cudaStream_t>(stream))) {
    Workspace w;
    w.buf = buffer();
    return w;
  }
  Scratch &s = scratch_of(device, stream);
  Tensor grown;  // allocated without the lock
  for (;;) {
    Workspace w;
    w.hold = lock_for_launches(s.in_use);
    if (grown.defined() && (!s.buf.defined() || s.buf.numel() < grown.numel())) std::swap(s.buf, grown);
    if (s.buf.defined() && s.buf.numel() >= bytes) {
      if (s.kind != kind) s.kind = kind;
      w.buf = s.buf;
      return w;
    }
    w.hold.unlock();
    grown = buffer();
  }
}

// The same for Python: `with` the object, the buffer is the calling thread's until the block ends.
class HeldWorkspace {
 public:
  HeldWorkspace(int device, int64_t bytes, std::string kind) : device_(device), bytes_(bytes), kind_(std::move(kind)) {}
  Tensor enter() {
    w_ = workspace_on(device_, c10::cuda::getCurrentCUDAStream(device_).stream(), bytes_, kind_.c_str());
    return w_.buf;
  }
  void exit() { w_ = Workspace(); }

 private:
  int device_;
  int64_t bytes_;
  std::string kind_;
  Workspace w_;
};

// (buffer or None, kind) of the current stream
std::pair<optional<Tensor>, std::string> last_workspace(int device) {
  Scratch &s = scratch_of(device, c10::cuda::getCurrentCUDAStream(device).stream());
  const auto hold = lock_for_launches(s.in_use);
  return {s.buf.defined() ? optional<Tensor>(s.buf) : c10::nullopt, s.kind};
}

// ---- aggregation -----------------------------------------------------------------------------------------------------
int64_t rows_of(const Tensor &ptr, int64_t num_node) {
  const int64_t all = ptr.size(0) - 1;
  const int64_t n = num_node > 0 ? num_node : all;  // 0 means all rows
  if (n > all) fail("num_node " + std::to_string(n) + " exceeds the " + std::to_string(all) + " rows of ptr");
  return n;
}

cxg_spmm_desc describe(const Tensor &ptr, const Tensor &idx, int64_t n, int64_t heads, int64_t feat, at::ScalarType type,
                       int64_t reduce, int64_t flags, int64_t split) {
  cxg_spmm_desc d = {};
  d.ptr = ptr.data_ptr();
  d.idx = idx.data_ptr();
  d.n_dst = n;
  d.nnz = idx.size(0);
  d.feat = static_cast<int32_t>(feat);
  d.heads = static_cast<int32_t>(heads);
  d.dtype = type == at::kFloat ? CXG_F32 : CXG_BF16;
  d.ptr_bytes = static_cast<int32_t>(ptr.element_size());
  d.idx_bytes = static_cast<int32_t>(idx.element_size());
  d.reduce = static_cast<int32_t>(reduce);
  d.flags = static_cast<uint32_t>(flags);
  d.split_edges = static_cast<int32_t>(split);
  return d;
}

void run_spmm(cxg_spmm_desc &d, const Tensor &x) {
  size_t need = 0, copy = 0;
  check(lib.cxg_spmm_csr_workspace_size(d.n_dst, d.nnz, d.feat, d.heads, d.split_edges, &need), "cxg_spmm_csr_workspace_size");
  check(lib.cxg_spmm_csr_rows_size(&d, x.size(0), &copy), "cxg_spmm_csr_rows_size");
  Tensor rows;
  if (copy > 0) {
    try {
      rows = at::empty({static_cast<int64_t>(copy)}, x.options().dtype(at::kByte));
    } catch (const c10::OutOfMemoryError &) {  // x as it is, then
      copy = 0;
    }
  }
  void *st = stream_of(x);
  const Workspace ws = workspace_on(x.device().index(), st, static_cast<int64_t>(need), "spmm");
  check(lib.cxg_spmm_csr_rows(&d, x.size(0), copy > 0 ? rows.data_ptr() : nullptr, copy, ws.data(), ws.bytes(), st), "cxg_spmm_csr");
}

// y = A x for the first rows of the graph; x [N, F] or [N, H, F]
Tensor spmm(const Tensor &x, const Tensor &ptr, const Tensor &idx, int64_t num_node, const optional<Tensor> &edge_val,
            int64_t reduce, const optional<Tensor> &out, const optional<Tensor> &edge_mask, const optional<Tensor> &edge_rel,
            int64_t rel_stride, const optional<Tensor> &targets, int64_t flags, int64_t split) {
  feature(x, "x");
  index_of(ptr, "ptr");
  index_of(idx, "idx");
  const int64_t n = rows_of(ptr, num_node);
  if (x.dim() != 2 && x.dim() != 3) fail("x must be [N, F] or [N, H, F]");
  const int64_t heads = x.dim() == 3 ? x.size(1) : 1, feat = x.size(-1);
  if (edge_val) {
    f32(*edge_val, "edge_value");
    const int64_t vh = edge_val->dim() == 2 ? edge_val->size(1) : 1;
    if (vh != heads) fail("edge_value has " + std::to_string(vh) + " heads, x has " + std::to_string(heads));
  }
  if (x.size(0) > UINT32_MAX) flags |= CXG_SPMM_GENERIC_WALK;  // the default walk keeps source rows as 32-bit numbers
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = out ? *out : (x.dim() == 3 ? at::empty({n, heads, feat}, x.options()) : at::empty({n, feat}, x.options()));
  cxg_spmm_desc d = describe(ptr, idx, n, heads, feat, x.scalar_type(), reduce, flags, split);
  d.x = x.data_ptr();
  d.y = y.data_ptr();
  if (edge_val) d.edge_val = static_cast<const float *>(edge_val->data_ptr());
  if (edge_mask) d.edge_mask = static_cast<const uint8_t *>(edge_mask->data_ptr());
  if (edge_rel) d.edge_rel = static_cast<const int32_t *>(edge_rel->data_ptr());
  if (targets) d.targets = static_cast<const int64_t *>(targets->data_ptr());
  d.rel_stride = rel_stride;
  run_spmm(d, x);
  return y;
}

// ---- transposed graphs -----------------------------------------------------------------------------------------------
struct Transposed {
  Tensor t_ptr, t_idx, t_eid, inv_deg;
};

Transposed transpose(const Tensor &ptr, const Tensor &idx, int64_t num_node, int64_t n_src, bool want_eid) {
  index_of(ptr, "ptr");
  index_of(idx, "idx");
  const int64_t n = rows_of(ptr, num_node), nnz = idx.size(0);
  c10::cuda::CUDAGuard guard(ptr.device());
  Transposed t;
  t.t_ptr = at::empty({n_src + 1}, ptr.options().dtype(at::kLong));
  t.t_idx = at::empty({nnz}, idx.options());
  if (want_eid) t.t_eid = at::empty({nnz}, idx.options());
  t.inv_deg = at::empty({n}, ptr.options().dtype(at::kFloat));
  size_t need = 0;
  check(lib.cxg_csr_transpose_workspace_size(nnz, &need), "cxg_csr_transpose_workspace_size");
  void *st = stream_of(ptr);
  const Workspace ws = workspace_on(ptr.device().index(), st, static_cast<int64_t>(need), "");
  check(lib.cxg_csr_transpose(ptr.data_ptr(), idx.data_ptr(), static_cast<int>(ptr.element_size()),
                              static_cast<int>(idx.element_size()), n, n_src, nnz, t.t_ptr.data_ptr<int64_t>(),
                              t.t_idx.data_ptr(), want_eid ? t.t_eid.data_ptr() : nullptr, t.inv_deg.data_ptr<float>(),
                              ws.data(), ws.bytes(), st),
        "cxg_csr_transpose");
  return t;
}

// The stream that has built something for keeping, and an event behind that.
struct Built {
  c10::cuda::CUDAStream stream;
  std::shared_ptr<c10::Event> event;
  explicit Built(const c10::cuda::CUDAStream &s) : stream(s), event(std::make_shared<c10::Event>(c10::DeviceType::CUDA)) { event->record(s); }
  // Another stream waits for the build, and the memory for that stream. A stream under capture cannot wait for what lies in
  // front of the capture (`outside`): the host does.
  template <typename Tensors>
  void hand_to(const c10::cuda::CUDAStream &other, bool outside, const Tensors &tensors) const {
    if (outside) {
      c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
      event->synchronize();
    } else {
      event->block(other);
    }
    for (const Tensor &t : tensors) t.record_stream(other);
  }
};

// Tensors that the current stream has built and a cache of the Python side keeps.
class Kept {
 public:
  explicit Kept(std::vector<Tensor> tensors)
      : tensors_(std::move(tensors)), device_(tensors_.at(0).device().index()), built_(c10::cuda::getCurrentCUDAStream(device_)) {}
  // They are about to be used on the current stream. True: under a capture, whose replays use them again.
  bool take() const {
    const auto stream = c10::cuda::getCurrentCUDAStream(device_);
    const bool capturing = capture_of(stream.stream()).has_value();
    if (stream != built_.stream) built_.hand_to(stream, capturing, tensors_);
    return capturing;
  }

 private:
  std::vector<Tensor> tensors_;
  c10::DeviceIndex device_;
  Built built_;
};

// The last eight transposed graphs, by the tensors they came from. An entry keeps ptr and idx alive, so their addresses
// cannot be handed to another graph. What a graph capture has recorded is there for that capture alone.
struct CachedGraph {
  const void *ptr_data, *idx_data;
  int64_t n, n_src;
  uint32_t ptr_version, idx_version;
  int device;
  Tensor ptr, idx;
  Transposed t;
  Built built;
  optional<unsigned long long> capture;
  // 1 / in-degree of every transposed edge's destination, when a mean's gradient has asked for it
  Tensor weight;
  optional<Built> weight_built;
};
std::mutex graphs_lock;
std::list<CachedGraph> &graphs = *new std::list<CachedGraph>;  // not torn down at exit: events would outlive the driver
std::list<Transposed> &captured_graphs = *new std::list<Transposed>;  // those that captures have taken: replays read them
constexpr size_t kMostGraphs = 8;

Transposed transposed_graph(const Tensor &ptr, const Tensor &idx, int64_t n, int64_t n_src) {
  const uint32_t pv = ptr._version(), iv = idx._version();
  const auto stream = c10::cuda::getCurrentCUDAStream(ptr.device().index());
  const auto capture = capture_of(stream.stream());
  {
    std::lock_guard<std::mutex> hold(graphs_lock);
    for (const auto &g : graphs)
      if (g.ptr_data == ptr.data_ptr() && g.idx_data == idx.data_ptr() && g.n == n && g.n_src == n_src && g.ptr_version == pv &&
          g.idx_version == iv && g.device == ptr.device().index() && (!g.capture || g.capture == capture)) {
        const bool outside = capture && !g.capture;
        if (outside && std::none_of(captured_graphs.begin(), captured_graphs.end(), [&](const Transposed &c) { return c.t_idx.is_same(g.t.t_idx); }))
          captured_graphs.push_back(g.t);
        if (stream != g.built.stream)
          g.built.hand_to(stream, outside, std::initializer_list<Tensor>{g.t.t_ptr, g.t.t_idx, g.t.t_eid, g.t.inv_deg});
        return g.t;
      }
  }
  const Transposed t = transpose(ptr, idx, n, n_src, true);
  CachedGraph g{ptr.data_ptr(), idx.data_ptr(), n, n_src, pv, iv, ptr.device().index(), ptr, idx, t, Built(stream), capture,
                Tensor(), c10::nullopt};
  std::lock_guard<std::mutex> hold(graphs_lock);
  while (graphs.size() >= kMostGraphs) graphs.pop_front();
  graphs.push_back(std::move(g));
  return t;
}
void forget_graphs() {
  std::lock_guard<std::mutex> hold(graphs_lock);
  graphs.clear();
  captured_graphs.clear();
}
size_t count_graphs() {
  std::lock_guard<std::mutex> hold(graphs_lock);
  return graphs.size();
}

// The weights of a mean's gradient, per transposed edge: kept with the graph, on whichever stream they are wanted. All graphs'
// together take a gigabyte at most, like the plans of the relational layers: the weights of the oldest graphs make room, and
// those of a graph that alone has more are made for the call.
constexpr size_t kMostWeightBytes = size_t{1} << 30;

Tensor mean_weights(const Transposed &t) {
  auto make = [&]() {
    Tensor w = at::empty({t.t_idx.size(0)}, t.inv_deg.options());
    check(lib.cxg_gather_edges(t.inv_deg.data_ptr<float>(), t.t_idx.data_ptr(), static_cast<int>(t.t_idx.element_size()),
                               w.data_ptr<float>(), t.t_idx.size(0), 1, 1, stream_of(w)),
          "cxg_gather_edges");
    return w;
  };
  const auto stream = c10::cuda::getCurrentCUDAStream(t.t_idx.device().index());
  const size_t bytes = static_cast<size_t>(t.t_idx.size(0)) * sizeof(float);
  if (bytes > kMostWeightBytes || capture_of(stream.stream())) return make();  // what a graph capture records is not there for others
  std::lock_guard<std::mutex> hold(graphs_lock);
  for (auto &g : graphs)
    if (g.t.t_idx.is_same(t.t_idx)) {
      if (!g.weight.defined()) {
        size_t kept = 0;
        for (const auto &other : graphs) kept += other.weight.defined() ? other.weight.nbytes() : 0;
        for (auto &other : graphs)
          if (other.weight.defined() && kept + bytes > kMostWeightBytes) {
            kept -= other.weight.nbytes();
            other.weight = Tensor();
            other.weight_built.reset();
          }
        g.weight = make();
        g.weight_built.emplace(stream);
      } else if (stream != g.weight_built->stream) {
        g.weight_built->hand_to(stream, false, std::initializer_list<Tensor>{g.weight});
      }
      return g.weight;
    }
  return make();
}

// dX = A^T dY on the cached transposed graph, in dY's type
Tensor spmm_transposed(const Tensor &grad, const Tensor &ptr, const Tensor &idx, int64_t n, int64_t n_src,
                       const optional<Tensor> &edge_val, int64_t reduce, int64_t flags, int64_t split) {
  const Transposed t = transposed_graph(ptr, idx, n, n_src);
  Tensor dy = grad.size(0) == n ? grad : grad.narrow(0, 0, n);
  optional<Tensor> tv;
  // A mean's gradient: weights per edge instead of a pass over dY (two, and two more for bf16), except where the edges are many
  // more than the values (12.6 M edges, fp32: a weight costs 10 us at 18 columns and 29 at 128, the pass 8 and 45).
  const int64_t columns = dy.numel() / std::max<int64_t>(n, 1), passes = dy.scalar_type() == at::kFloat ? 2 : 5;
  if (reduce == CXG_MEAN && dy.dim() == 2 && !edge_val && 8 * t.t_idx.size(0) <= n * columns * passes) {
    tv = mean_weights(t);
  } else if (reduce == CXG_MEAN) {
    std::vector<int64_t> shape(dy.dim(), 1);
    shape[0] = n;
    const Tensor w = t.inv_deg.view(shape);
    dy = dy.scalar_type() == at::kFloat ? at::mul(dy, w) : at::mul(dy.to(at::kFloat), w).to(dy.scalar_type());
  }
  if (edge_val) {  // the edge values in transposed order
    const Tensor ev = edge_val->contiguous();
    tv = at::empty_like(ev);
    check(lib.cxg_gather_edges(ev.data_ptr<float>(), t.t_eid.data_ptr(), static_cast<int>(t.t_eid.element_size()),
                               tv->data_ptr<float>(), std::min(t.t_eid.size(0), ev.size(0)),
                               static_cast<int>(ev.dim() == 2 ? ev.size(1) : 1), 1, stream_of(ev)),
          "cxg_gather_edges");
  }
  return spmm(dy.contiguous(), t.t_ptr, t.t_idx, n_src, tv, CXG_SUM, c10::nullopt, c10::nullopt, c10::nullopt, 0, c10::nullopt,
              flags, split);
}

// Sum or mean aggregation with its gradients: x over the transposed graph (or, `scatter`, with atomics over the forward
// edges), the edge values by a second pass over the forward edges.
class SageFunction : public torch::autograd::Function<SageFunction> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &ptr, const Tensor &idx,
                        const optional<Tensor> &edge_val, int64_t num_node, int64_t reduce, int64_t flags, int64_t split,
                        bool scatter) {
    ctx->save_for_backward({x, ptr, idx, edge_val ? *edge_val : Tensor()});
    ctx->saved_data["n"] = num_node;
    ctx->saved_data["reduce"] = reduce;
    ctx->saved_data["flags"] = flags;
    ctx->saved_data["split"] = split;
    ctx->saved_data["scatter"] = scatter;
    return spmm(x, ptr, idx, num_node, edge_val, reduce, c10::nullopt, c10::nullopt, c10::nullopt, 0, c10::nullopt, flags, split);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &ptr = saved[1], &idx = saved[2];
    optional<Tensor> edge_val;
    if (saved[3].defined()) edge_val = saved[3];
    const Tensor g = grads[0].contiguous();
    const int64_t n = rows_of(ptr, ctx->saved_data["n"].toInt()), reduce = ctx->saved_data["reduce"].toInt();
    const int64_t flags = ctx->saved_data["flags"].toInt(), split = ctx->saved_data["split"].toInt();
    c10::cuda::CUDAGuard guard(g.device());
    Tensor dx, dval;
    bool need_dx = ctx->needs_input_grad(0);
    const bool need_dval = edge_val && ctx->needs_input_grad(3);
    if (need_dx && !ctx->saved_data["scatter"].toBool() && n > 0 && idx.size(0) > 0) {
      dx = spmm_transposed(g, ptr, idx, n, x.size(0), edge_val, reduce, flags, split);
      need_dx = false;
    }
    if (need_dx || need_dval) {
      cxg_spmm_desc d = describe(ptr, idx, n, g.dim() == 3 ? g.size(1) : 1, g.size(-1), g.scalar_type(), reduce, flags, split);
      Tensor xs;
      if (edge_val) d.edge_val = static_cast<const float *>(edge_val->data_ptr());
      if (need_dx) dx = at::zeros(x.sizes(), x.options().dtype(at::kFloat));
      if (need_dval) {
        dval = at::zeros(edge_val->sizes(), edge_val->options());
        xs = x.scalar_type() == g.scalar_type() ? x : x.to(g.scalar_type());
        d.x = xs.data_ptr();
      }
      check(lib.cxg_spmm_csr_backward(&d, g.data_ptr(), need_dx ? dx.data_ptr<float>() : nullptr,
                                      need_dval ? dval.data_ptr<float>() : nullptr, stream_of(g)),
            "cxg_spmm_csr_backward");
    }
    if (dx.defined() && dx.scalar_type() != x.scalar_type()) dx = dx.to(x.scalar_type());
    return {dx, Tensor(), Tensor(), dval, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor sage(const Tensor &x, const Tensor &ptr, const Tensor &idx, const optional<Tensor> &edge_val, int64_t num_node,
            int64_t reduce, int64_t flags, int64_t split, bool scatter) {
  if (recorded(x, edge_val))
    return SageFunction::apply(x, ptr, idx, edge_val, num_node, reduce, flags, split, scatter);
  return spmm(x, ptr, idx, num_node, edge_val, reduce, c10::nullopt, c10::nullopt, c10::nullopt, 0, c10::nullopt, flags, split);
}

Tensor gather_rows(const Tensor &x, const Tensor &rows) {
  if (for_torch(x, rows)) return x.index_select(0, rows);
  cuda(x, "x");
  of_type(rows, "rows", {at::kLong});
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty({rows.size(0), x.size(1)}, x.options());
  check(lib.cxg_gather_rows(x.data_ptr(), rows.data_ptr<int64_t>(), out.data_ptr(), rows.size(0),
                            x.size(1) * static_cast<int64_t>(x.element_size()), stream_of(x)),
        "cxg_gather_rows");
  return out;
}

// ---- linear transform ------------------------------------------------------------------------------------------------
bool aligned16(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// fp32 matrices that the tensor-core kernel takes as they are
bool dense_rows(const Tensor &t) {
  return t.dim() == 2 && t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() > 0 && aligned16(t);
}

// x [M, K] . w [N, K]^T (w_rows_k: w is [K, N]) + bias + add
Tensor linear_product(const Tensor &x, const Tensor &w, bool w_rows_k, const optional<Tensor> &bias, const optional<Tensor> &add) {
  const int64_t n = w_rows_k ? w.size(1) : w.size(0);
  Tensor y = at::empty({x.size(0), n}, x.options());
  check(lib.cxg_linear_f32(x.data_ptr<float>(), w.data_ptr<float>(), bias ? bias->data_ptr<float>() : nullptr,
                           add ? add->data_ptr<float>() : nullptr, y.data_ptr<float>(), x.size(0), static_cast<int>(x.size(1)),
                           static_cast<int>(n), w_rows_k ? 1 : 0, stream_of(x)),
        "cxg_linear_f32");
  return y;
}

// g [M, N]^T . x [M, K]
Tensor linear_weight_grad(const Tensor &g, const Tensor &x) {
  const int64_t m = x.size(0), n = g.size(1), k = x.size(1);
  if (!dense_rows(g) || !dense_rows(x) || n % 4 != 0 || k % 4 != 0) return at::mm(g.t(), x);
  Tensor dw = at::empty({n, k}, x.options());
  size_t need = 0;
  check(lib.cxg_dense_wgrad_f32_workspace_size(m, static_cast<int>(n), static_cast<int>(k), &need),
        "cxg_dense_wgrad_f32_workspace_size");
  void *st = stream_of(x);
  const Workspace ws = workspace_on(x.device().index(), st, static_cast<int64_t>(need), "");
  check(lib.cxg_dense_wgrad_f32(g.data_ptr<float>(), x.data_ptr<float>(), m, static_cast<int>(n), static_cast<int>(k),
                                dw.data_ptr<float>(), ws.data(), ws.bytes(), st),
        "cxg_dense_wgrad_f32");
  return dw;
}

Tensor rows_sum(const Tensor &g) {
  Tensor out = at::empty({g.size(1)}, g.options());
  size_t need = 0;
  check(lib.cxg_column_sum_workspace_size(static_cast<int>(g.size(1)), &need), "cxg_column_sum_workspace_size");
  void *st = stream_of(g);
  const Workspace ws = workspace_on(g.device().index(), st, static_cast<int64_t>(need), "");
  check(lib.cxg_column_sum(g.data_ptr(), CXG_F32, g.size(0), static_cast<int>(g.size(1)), out.data_ptr<float>(), ws.data(),
                           ws.bytes(), st),
        "cxg_column_sum");
  return out;
}

bool linear_fits(const Tensor &x, const Tensor &w) {
  return dense_rows(x) && dense_rows(w) && x.size(1) == w.size(1) && x.device() == w.device() &&
         lib.cxg_linear_f32_supported(x.size(0), static_cast<int>(x.size(1)), static_cast<int>(w.size(0))) == 1;
}

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const optional<Tensor> &bias,
                        const optional<Tensor> &add, bool same_bits) {
    ctx->save_for_backward({x, w});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["add"] = add.has_value();
    if (!same_bits) return linear_product(x, w, false, bias, add);
    const Tensor y = at::linear(x, w, bias);
    return add ? *add + y : y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    const Tensor g = grads[0].contiguous();
    c10::cuda::CUDAGuard guard(g.device());
    Tensor dx, dw, db;
    // the edges of the node are those of the tensors that were given
    const bool bias = ctx->saved_data["bias"].toBool(), need_db = bias && ctx->needs_input_grad(2);
    const bool need_add = ctx->saved_data["add"].toBool() && ctx->needs_input_grad(bias ? 3 : 2);
    if (at::GradMode::is_enabled()) {  // a graph of the backward itself is wanted
      if (ctx->needs_input_grad(0)) dx = at::mm(g, w);
      if (ctx->needs_input_grad(1)) dw = at::mm(g.t(), x);
      if (need_db) db = g.sum(0);
    } else {
      if (ctx->needs_input_grad(0))
        dx = dense_rows(g) && lib.cxg_linear_f32_supported(g.size(0), static_cast<int>(g.size(1)), static_cast<int>(w.size(1)))
                 ? linear_product(g, w, true, c10::nullopt, c10::nullopt)
                 : at::mm(g, w);
      if (ctx->needs_input_grad(1)) dw = linear_weight_grad(g, x);
      if (need_db) db = rows_sum(g);
    }
    return {dx, dw, db, need_add ? grads[0] : Tensor(), Tensor()};
  }
};

// x . w^T (+ bias) (+ add): the tensor-core kernel for fp32 matrices it takes, torch otherwise (CPU, other types, autocast,
// rows that are not whole 16-byte vectors). same_bits: where a gradient is recorded the product itself is torch's and only
// the gradients are the kernel's. In front of a ReLU (and of the LeakyReLU on a GAT layer's scores) another rounding, though
// a better one, puts the few values within rounding of zero on its other side, and each of them moves the gradients: those
// of a sampled batch by up to 3e-4 of their norm, those of a GAT layer by up to 2e-3.
Tensor linear(const Tensor &x, const Tensor &w, const optional<Tensor> &bias, const optional<Tensor> &add, bool same_bits) {
  const bool fits = !for_torch(x, w, bias, add) && linear_fits(x, w) && !at::autocast::is_autocast_enabled(at::kCUDA) &&
                    (!bias || (bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->device() == x.device() &&
                               bias->dim() == 1 && bias->size(0) == w.size(0)));
  const bool add_fits = add && dense_rows(*add) && add->size(0) == x.size(0) && add->size(1) == w.size(0) && add->device() == x.device();
  if (!fits || (add && !add_fits)) {
    const Tensor y = at::linear(x, w, bias);
    return add ? *add + y : y;
  }
  c10::cuda::CUDAGuard guard(x.device());
  if (recorded(x, w, bias, add)) return LinearFunction::apply(x, w, bias, add, same_bits);
  return linear_product(x, w, false, bias, add);
}

// ---- rows held in 8 bits ---------------------------------------------------------------------------------------------
const char *const kTransform = " does not take tensors of a transform (vmap, forward-mode differentiation, tracing)";

int code_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? CXG_F32 : CXG_BF16; }

// Whether the backward pass that a call records would lead from a graph capture into nodes of the default stream: those of a leaf
// that an eager graph still holds, or of a tensor that was computed outside the capture. torch's engine then makes that stream
// wait for a captured event, which breaks the capture and can end the process. (Any other stream joins the capture by that wait,
// and the engine joins it back: steps that were run on a side stream first may stay alive.)
void recorded_in_capture(const char *who, const Tensor &t) {
  if (!t.defined() || !t.requires_grad() || !at::GradMode::is_enabled()) return;
  const auto stream = c10::cuda::getCurrentCUDAStream(t.device().index());
  if (!capture_of(stream.stream())) return;
  const auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto of = node->stream();
  if (of && *of != stream.unwrap() && c10::cuda::CUDAStream(c10::cuda::CUDAStream::UNCHECKED, *of).stream() == nullptr)
    fail(std::string(who) + ": under capture, with gradients recorded, of a tensor whose graph belongs to the default stream and is still "
                            "alive: drop what was computed from it before the capture");
}
void recorded_in_capture(const char *who, const optional<Tensor> &t) {
  if (t) recorded_in_capture(who, *t);
}
template <typename... T>
void all_recorded_in_capture(const char *who, const T &...t) {
  (recorded_in_capture(who, t), ...);
}

// A copy of views that stand for the negative of what is stored.
Tensor as_stored(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

// A matrix of rows that lie any distance apart, each in one piece; a copy of any other.
Tensor row_matrix(const Tensor &t_in, const char *name) {
  const Tensor t = as_stored(t_in);
  if (!t.is_cuda()) fail(std::string(name) + " must be a CUDA tensor (this backend has no CPU path)");
  if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16)
    fail(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + ", which this operator does not take");
  if (t.dim() != 2 || t.size(1) == 0) fail(std::string(name) + " must be a matrix with at least one column");
  if (t.size(1) > (1 << 20)) fail(std::string(name) + " has more than 2^20 columns");
  const bool rows = t.stride(1) == 1 || t.size(1) == 1;
  return rows && (t.stride(0) >= t.size(1) || t.size(0) <= 1) ? t : t.contiguous();
}
int64_t row_step(const Tensor &t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

void same_device(const Tensor &a, const Tensor &b, const char *name) {
  if (a.device() != b.device()) fail(std::string(name) + " is on another device");
}

// codes [rows + 1, pitch], scales [rows + 1, pitch / 32]: the last row of zeros
struct Held {
  Tensor codes, scales;
  int64_t rows() const { return codes.size(0) - 1; }
};

Held held_like(int64_t rows, int64_t width, at::Device device) {
  const int64_t pitch = lib.cxg_rows8_pitch(static_cast<int>(width));
  const auto opt = at::TensorOptions().dtype(at::kByte).device(device);
  return {at::empty({rows + 1, pitch}, opt), at::empty({rows + 1, pitch / 32}, opt)};
}

Held quantize(const Tensor &x_in) {
  if (for_torch(x_in)) fail(std::string("quantize_rows") + kTransform);
  const Tensor x = row_matrix(x_in, "x");
  c10::cuda::CUDAGuard guard(x.device());
  Held h = held_like(x.size(0), x.size(1), x.device());
  check(lib.cxg_rows8_write(x.data_ptr(), code_of(x), row_step(x), x.size(0), static_cast<int>(x.size(1)), h.codes.data_ptr(),
                            h.scales.data_ptr(), 1, stream_of(x)),
        "cxg_rows8_write");
  return h;
}

// Rows of zeros.
Held held_zeros(int64_t rows, int64_t width, at::Device device) {
  if (rows < 0 || width <= 0 || width > (1 << 20)) fail("Rows8: bad sizes");
  if (!device.is_cuda()) fail("Rows8: the device must be a CUDA device (this backend has no CPU path)");
  c10::cuda::CUDAGuard guard(device);
  Held h = held_like(rows, width, device);
  h.codes.fill_(128);
  h.scales.zero_();
  return h;
}

// Rows of x over rows [0, n) of what is held, or over the rows that index names (claims: the words of cxg_rows8_write_at).
void quantize_into(const Tensor &x_in, const Tensor &codes, const Tensor &scales, int64_t width, const optional<Tensor> &index,
                   const optional<Tensor> &claims) {
  if (for_torch(x_in)) fail(std::string("quantize_rows") + kTransform);
  const Tensor x = row_matrix(x_in, "x");
  const int64_t rows = codes.size(0) - 1, n = x.size(0);
  same_device(codes, x, "x");
  if (x.size(1) != width) fail("quantize_rows: x has " + std::to_string(x.size(1)) + " columns, the rows have " + std::to_string(width));
  c10::cuda::CUDAGuard guard(x.device());
  void *st = stream_of(x);
  if (!index) {
    if (n > rows) fail("quantize_rows: x has " + std::to_string(n) + " rows, there are " + std::to_string(rows));
    check(lib.cxg_rows8_write(x.data_ptr(), code_of(x), row_step(x), n, static_cast<int>(width), codes.data_ptr(), scales.data_ptr(),
                              0, st),
          "cxg_rows8_write");
  } else {
    of_type(*index, "index", {at::kLong});
    same_device(codes, *index, "index");
    if (index->dim() != 1 || index->size(0) != n) fail("quantize_rows: index must name a row for every row of x");
    check(lib.cxg_rows8_write_at(x.data_ptr(), code_of(x), row_step(x), n, static_cast<int>(width), index->data_ptr<int64_t>(),
                                 codes.data_ptr(), scales.data_ptr(), rows, claims->data_ptr<int32_t>(), st),
          "cxg_rows8_write_at");
  }
  // a backward pass that was to read these rows hears of it (inference tensors cannot be kept for one and count no versions)
  for (const Tensor *t : {&codes, &scales})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

at::ScalarType row_type(const std::string &who, at::ScalarType t) {
  if (t != at::kFloat && t != at::kBFloat16) fail(who + ": dtype must be float32 or bfloat16");
  return t;
}

Tensor dequantize(const Tensor &codes, const Tensor &scales, int64_t width, const optional<Tensor> &index, at::ScalarType type,
                  int64_t num_rows) {
  row_type("dequantize_rows", type);
  c10::cuda::CUDAGuard guard(codes.device());
  const int64_t rows = codes.size(0) - 1;
  if (index) {
    of_type(*index, "index", {at::kLong});
    same_device(codes, *index, "index");
    if (index->dim() != 1) fail("dequantize_rows: index must be a vector");
  }
  if (num_rows < 0 || num_rows > rows) fail("dequantize_rows: " + std::to_string(num_rows) + " rows of " + std::to_string(rows));
  Tensor out = at::empty({index ? index->size(0) : num_rows, width}, codes.options().dtype(type));
  check(lib.cxg_rows8_read(codes.data_ptr(), scales.data_ptr(), rows, static_cast<int>(width),
                           index ? index->data_ptr<int64_t>() : nullptr, out.size(0), out.data_ptr(), code_of(out), width,
                           stream_of(codes)),
        "cxg_rows8_read");
  return out;
}

Tensor rows8_aggregate(const Tensor &codes, const Tensor &scales, int64_t width, const Tensor &ptr, const Tensor &idx,
                       int64_t num_node, bool mean, const optional<Tensor> &edge_value, at::ScalarType type, int64_t split) {
  row_type("rows8_aggregate", type);
  index_of(ptr, "ptr");
  index_of(idx, "idx");
  same_device(codes, ptr, "ptr");
  same_device(codes, idx, "idx");
  if (ptr.dim() != 1 || ptr.size(0) < 1 || idx.dim() != 1) fail("rows8_aggregate: ptr and idx must be vectors, ptr of at least one entry");
  const int64_t n = rows_of(ptr, num_node);
  if (edge_value) {
    if (mean) fail("rows8_aggregate: a mean takes no edge values");
    if (for_torch(*edge_value)) fail(std::string("rows8_aggregate") + kTransform);
    if (recorded(*edge_value)) fail("rows8_aggregate: there is no gradient for edge values");
    f32(*edge_value, "edge_value");
    same_device(codes, *edge_value, "edge_value");
    if (edge_value->numel() != idx.size(0)) fail("rows8_aggregate: one edge value per edge");
    if (edge_value->is_neg()) fail("rows8_aggregate: edge_value is a view that stands for its negative: resolve_neg() it first");
  }
  c10::cuda::CUDAGuard guard(codes.device());
  Tensor y = at::empty({n, width}, codes.options().dtype(type));
  size_t need = 0;
  check(lib.cxg_rows8_aggregate_workspace_size(idx.size(0), static_cast<int>(width), static_cast<int>(split), &need),
        "cxg_rows8_aggregate_workspace_size");
  void *st = stream_of(codes);
  const Workspace ws = workspace_on(codes.device().index(), st, static_cast<int64_t>(need), "spmm");
  check(lib.cxg_rows8_aggregate(codes.data_ptr(), scales.data_ptr(), codes.size(0) - 1, static_cast<int>(width), ptr.data_ptr(),
                                static_cast<int>(ptr.element_size()), idx.data_ptr(), static_cast<int>(idx.element_size()),
                                edge_value ? edge_value->data_ptr<float>() : nullptr, n, idx.size(0), mean ? CXG_MEAN : CXG_SUM,
                                static_cast<int>(split), y.data_ptr(), code_of(y), ws.data(), ws.bytes(), st),
        "cxg_rows8_aggregate");
  return y;
}

// (dy^T . rows [n, width], column sums of dy [n] or none), summed in fp32
std::pair<Tensor, Tensor> rows8_weight_grad(const Tensor &codes, const Tensor &scales, int64_t width, const Tensor &dy_in, bool bias,
                                            at::ScalarType type) {
  if (for_torch(dy_in)) fail(std::string("rows8_weight_grad") + kTransform);
  const Tensor dy = row_matrix(dy_in, "grad");
  same_device(codes, dy, "grad");
  const int64_t m = dy.size(0), n = dy.size(1);
  if (m > codes.size(0) - 1) fail("rows8_weight_grad: grad has " + std::to_string(m) + " rows, there are " + std::to_string(codes.size(0) - 1));
  c10::cuda::CUDAGuard guard(dy.device());
  const auto opt = dy.options().dtype(type);
  Tensor dw = at::empty({n, width}, opt), db = bias ? at::empty({n}, opt) : Tensor();
  size_t need = 0;
  check(lib.cxg_rows8_wgrad_workspace_size(m, static_cast<int>(width), static_cast<int>(n), &need), "cxg_rows8_wgrad_workspace_size");
  void *st = stream_of(dy);
  const Workspace ws = workspace_on(dy.device().index(), st, static_cast<int64_t>(need), "");
  check(lib.cxg_rows8_wgrad(codes.data_ptr(), scales.data_ptr(), m, static_cast<int>(width), dy.data_ptr(), code_of(dy), row_step(dy),
                            static_cast<int>(n), 0, dw.data_ptr(), bias ? db.data_ptr() : nullptr, code_of(dw), ws.data(), ws.bytes(),
                            st),
        "cxg_rows8_wgrad");
  return {dw, db};
}

// The result of a linear transform in the input's type: the tensor-core kernel for the fp32 matrices it takes, else torch's, or
// always torch's (of_torch).
Tensor plain_linear(const Tensor &x, const Tensor &w, const optional<Tensor> &bias, const optional<Tensor> &add, bool of_torch) {
  const bool add_fits = !add || (dense_rows(*add) && add->sizes() == at::IntArrayRef({x.size(0), w.size(0)}));
  if (!of_torch && linear_fits(x, w) && add_fits && (!bias || bias->is_contiguous())) return linear_product(x, w, false, bias, add);
  const Tensor y = at::linear(x, w, bias);
  return add ? *add + y : y;
}

// A linear transform whose backward pass reads its input in 8 bits.
class LinearKept8Function : public torch::autograd::Function<LinearKept8Function> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const optional<Tensor> &bias,
                        const optional<Tensor> &add, const optional<Tensor> &codes, const optional<Tensor> &scales, bool same_bits) {
    Held held;
    if (codes)
      held = {*codes, *scales};
    else if (w.requires_grad())  // nobody reads the rows otherwise
      held = quantize(x);
    ctx->save_for_backward({w, held.codes, held.scales});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["add"] = add.has_value();
    return plain_linear(x, w, bias, add, same_bits);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    if (at::GradMode::is_enabled()) fail("linear_kept8: the rows it keeps in 8 bits have no second derivative");
    const auto saved = ctx->get_saved_variables();
    const Tensor &w = saved[0];
    const Tensor g = as_stored(grads[0]).contiguous();
    c10::cuda::CUDAGuard guard(g.device());
    Tensor dx, dw, db;
    const bool bias = ctx->saved_data["bias"].toBool(), need_db = bias && ctx->needs_input_grad(2);
    const bool need_add = ctx->saved_data["add"].toBool() && ctx->needs_input_grad(bias ? 3 : 2);
    if (ctx->needs_input_grad(0))
      dx = dense_rows(g) && dense_rows(w) &&
                   lib.cxg_linear_f32_supported(g.size(0), static_cast<int>(g.size(1)), static_cast<int>(w.size(1)))
               ? linear_product(g, w, true, c10::nullopt, c10::nullopt)
               : at::mm(g, w);
    if (ctx->needs_input_grad(1)) {
      const auto grad = rows8_weight_grad(saved[1], saved[2], w.size(1), g, need_db, w.scalar_type());
      dw = grad.first;
      db = grad.second;
    } else if (need_db) {
      db = g.sum(0, false, at::kFloat).to(g.scalar_type());
    }
    return {dx, dw, db, need_add ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear_kept8(Tensor x, Tensor w, optional<Tensor> bias, optional<Tensor> add, const optional<Tensor> &codes,
                    const optional<Tensor> &scales, bool same_bits) {
  if (for_torch(x, w, bias, add)) fail(std::string("linear_kept8") + kTransform);
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    const auto type = row_type("linear_kept8 under autocast", at::autocast::get_autocast_dtype(at::kCUDA));
    x = x.to(type), w = w.to(type);
    if (bias) bias = bias->to(type);
    if (add) add = add->to(type);
  }
  for (const Tensor *t : {&x, &w}) {
    if (!t->is_cuda()) fail("linear_kept8: x and weight must be CUDA tensors (this backend has no CPU path)");
    if (t->dim() != 2 || t->size(1) == 0) fail("linear_kept8: x and weight must be matrices");
  }
  row_type("linear_kept8", x.scalar_type());
  if (w.scalar_type() != x.scalar_type() || (bias && bias->scalar_type() != x.scalar_type()) || (add && add->scalar_type() != x.scalar_type()))
    fail("linear_kept8: x, weight, bias and add must be of one type");
  if (w.size(1) != x.size(1) || w.size(0) == 0) fail("linear_kept8: weight must be [out, " + std::to_string(x.size(1)) + "]");
  if (bias && (bias->dim() != 1 || bias->size(0) != w.size(0))) fail("linear_kept8: bias must be [" + std::to_string(w.size(0)) + "]");
  if (add && (add->dim() != 2 || add->size(0) != x.size(0) || add->size(1) != w.size(0))) fail("linear_kept8: add must have the shape of the result");
  same_device(x, w, "weight");
  if (bias) same_device(x, *bias, "bias");
  if (add) same_device(x, *add, "add");
  if (codes) {
    same_device(x, *codes, "kept");
    if (codes->size(0) - 1 < x.size(0) || codes->size(1) != lib.cxg_rows8_pitch(static_cast<int>(x.size(1))))
      fail("linear_kept8: kept must hold the rows of x");
  }
  c10::cuda::CUDAGuard guard(x.device());
  x = as_stored(x), w = as_stored(w);
  if (bias) bias = as_stored(*bias);
  if (add) add = as_stored(*add);
  all_recorded_in_capture("linear_kept8", x, w, bias, add);
  c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::AutocastCUDA);
  if (recorded(x, w, bias, add))
    return LinearKept8Function::apply(x, w, bias, add, codes, scales, same_bits);
  return plain_linear(x, w, bias, add, false);
}

// ---- the step between two blocks of a residual network -----------------------------------------------------------------
struct ResidualOptions {
  bool post, next, layer, keep;
  double eps;
};

const float *param(const optional<Tensor> &t) { return t ? t->data_ptr<float>() : nullptr; }

cxg_residual_desc describe_residual(const Tensor &x, const optional<Tensor> &f, const optional<Tensor> &gate, const optional<Tensor> &scale,
                                    const optional<Tensor> &w2, const optional<Tensor> &b2, const optional<Tensor> &w1,
                                    const optional<Tensor> &b1, const ResidualOptions &o) {
  cxg_residual_desc d = {};
  d.x = x.data_ptr();
  if (f) d.f = f->data_ptr();
  if (gate) {
    d.gate = gate->data_ptr();
    d.gate_mode = gate->dim() == 2 && gate->size(1) == x.size(1) && x.size(1) > 1 ? CXG_GATE_VALUE : CXG_GATE_ROW;
  }
  d.scale = param(scale), d.post_weight = param(w2), d.post_bias = param(b2), d.next_weight = param(w1), d.next_bias = param(b1);
  d.n = x.size(0);
  d.width = static_cast<int32_t>(x.size(1));
  d.dtype = code_of(x);
  d.layer = o.layer, d.post = o.post, d.next = o.next;
  d.eps = static_cast<float>(o.eps);
  return d;
}

// {y (with f), h (with next), codes and scales of h (with keep)}
variable_list residual_forward(const Tensor &x, const optional<Tensor> &f, const optional<Tensor> &gate, const optional<Tensor> &scale,
                               const optional<Tensor> &w2, const optional<Tensor> &b2, const optional<Tensor> &w1,
                               const optional<Tensor> &b1, const ResidualOptions &o) {
  cxg_residual_desc d = describe_residual(x, f, gate, scale, w2, b2, w1, b1, o);
  variable_list out;
  if (f) {
    out.push_back(at::empty_like(x));
    d.y = out.back().data_ptr();
  }
  Tensor h;
  if (o.next) {
    h = at::empty_like(x);
    out.push_back(h);
    d.h = h.data_ptr();
  }
  Held held;
  bool with_h = false;
  if (o.keep) {
    held = held_like(x.size(0), x.size(1), x.device());
    d.codes = held.codes.data_ptr();
    with_h = d.n > 0 && lib.cxg_residual_norm_keeps(&d) == 1;
    d.codes = with_h ? held.codes.data_ptr() : nullptr;
    d.scales = with_h ? held.scales.data_ptr() : nullptr;
  }
  check(lib.cxg_residual_norm_forward(&d, stream_of(x)), "cxg_residual_norm_forward");
  if (o.keep) {
    if (!with_h)
      check(lib.cxg_rows8_write(h.data_ptr(), code_of(h), h.size(1), h.size(0), static_cast<int>(h.size(1)), held.codes.data_ptr(),
                                held.scales.data_ptr(), 1, stream_of(h)),
            "cxg_rows8_write");
    out.push_back(held.codes);
    out.push_back(held.scales);
  }
  return out;
}

class ResidualNormFunction : public torch::autograd::Function<ResidualNormFunction> {
 public:
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const optional<Tensor> &f, const optional<Tensor> &gate,
                               const optional<Tensor> &scale, const optional<Tensor> &w2, const optional<Tensor> &b2,
                               const optional<Tensor> &w1, const optional<Tensor> &b1, bool post, bool next, bool layer, double eps,
                               bool keep) {
    const ResidualOptions o{post, next, layer, keep, eps};
    variable_list out = residual_forward(x, f, gate, scale, w2, b2, w1, b1, o);
    auto or_none = [](const optional<Tensor> &t) { return t ? *t : Tensor(); };
    ctx->save_for_backward({x, or_none(f), or_none(gate), or_none(scale), or_none(w2), or_none(b2), or_none(w1), or_none(b1)});
    ctx->saved_data["options"] = std::vector<bool>{post, next, layer};
    ctx->saved_data["eps"] = eps;
    if (keep) ctx->mark_non_differentiable({out[out.size() - 2], out[out.size() - 1]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    if (at::GradMode::is_enabled()) fail("residual_norm: its backward pass has no derivative");
    const auto saved = ctx->get_saved_variables();
    auto given = [&](int i) { return saved[i].defined() ? optional<Tensor>(saved[i]) : c10::nullopt; };
    const auto flags = ctx->saved_data["options"].toBoolList();
    const ResidualOptions o{flags[0], flags[1], flags[2], false, ctx->saved_data["eps"].toDouble()};
    const Tensor &x = saved[0];
    const optional<Tensor> f = given(1);
    c10::cuda::CUDAGuard guard(x.device());
    cxg_residual_desc d = describe_residual(x, f, given(2), given(3), given(4), given(5), given(6), given(7), o);
    const int h_at = f ? 1 : 0;
    Tensor dy, dh;
    if (f && grads[0].defined()) dy = as_stored(grads[0]).contiguous();
    if (o.next && grads[h_at].defined()) dh = as_stored(grads[h_at]).contiguous();
    variable_list out(13);
    if (!dy.defined() && !dh.defined()) return out;
    d.dy = dy.defined() ? dy.data_ptr() : nullptr;
    d.dh = dh.defined() ? dh.data_ptr() : nullptr;
    // the edges of the node are those of the tensors that were given
    bool need[8];
    for (int i = 0, edge = 0; i < 8; ++i) need[i] = saved[i].defined() && ctx->needs_input_grad(edge++);
    void **into[3] = {&d.dx, &d.df, &d.dgate};
    for (int i = 0; i < 3; ++i)
      if (need[i]) {
        out[i] = at::empty_like(saved[i]);
        *into[i] = out[i].data_ptr();
      }
    Tensor sums = at::empty({5, x.size(1)}, x.options().dtype(at::kFloat));
    size_t bytes = 0;
    check(lib.cxg_residual_norm_backward_workspace_size(d.n, d.width, &bytes), "cxg_residual_norm_backward_workspace_size");
    void *st = stream_of(x);
    {
      const Workspace ws = workspace_on(x.device().index(), st, static_cast<int64_t>(bytes), "");
      check(lib.cxg_residual_norm_backward(&d, sums.data_ptr<float>(), ws.data(), ws.bytes(), st), "cxg_residual_norm_backward");
    }
    for (int i = 3; i < 8; ++i)
      if (need[i]) out[i] = sums.select(0, i - 3);
    return out;
  }
};

// A parameter as fp32 [width] (or one value for all columns), differentiably.
optional<Tensor> row_parameter(const optional<Tensor> &t, const Tensor &x, const char *name) {
  if (!t) return t;
  same_device(x, *t, name);
  if (!t->is_floating_point()) fail(std::string("residual_norm: ") + name + " must be of a floating-point type");
  Tensor v = t->to(at::kFloat);
  if (std::string(name) == "scale" && v.numel() == 1) v = v.reshape({1}).expand({x.size(1)});
  if (v.dim() != 1 || v.size(0) != x.size(1)) fail(std::string("residual_norm: ") + name + " must be [" + std::to_string(x.size(1)) + "]");
  return as_stored(v).contiguous();
}

std::vector<optional<Tensor>> residual_norm(const Tensor &x_in, const optional<Tensor> &f_in, const optional<Tensor> &gate_in,
                                            const optional<Tensor> &scale_in, bool post, const optional<Tensor> &post_weight,
                                            const optional<Tensor> &post_bias, bool next, const optional<Tensor> &next_weight,
                                            const optional<Tensor> &next_bias, bool layer, double eps, bool keep) {
  if (for_torch(x_in, f_in, gate_in, scale_in, post_weight, post_bias, next_weight, next_bias))
    fail(std::string("residual_norm") + kTransform);
  const bool autocast = at::autocast::is_autocast_enabled(at::kCUDA);
  auto rows = [&](Tensor t, const char *name) {
    if (!t.is_cuda()) fail(std::string(name) + " must be a CUDA tensor (this backend has no CPU path)");
    if (autocast && t.is_floating_point()) t = t.to(x_in.scalar_type());  // what a block returns may be of another type than x
    if (t.scalar_type() != x_in.scalar_type()) fail(std::string("residual_norm: ") + name + " must be of x's type");
    same_device(x_in, t, name);
    return as_stored(t).contiguous();
  };
  row_type("residual_norm", x_in.scalar_type());
  if (x_in.dim() != 2 || x_in.size(1) == 0) fail("residual_norm: x must be a matrix with at least one column");
  if (x_in.size(1) > lib.cxg_residual_norm_max_width())
    fail("residual_norm: rows of " + std::to_string(x_in.size(1)) + " values, at most " + std::to_string(lib.cxg_residual_norm_max_width()));
  if (!(eps >= 0)) fail("residual_norm: eps must not be negative");
  const Tensor x = rows(x_in, "x");
  optional<Tensor> f, gate;
  if (f_in) {
    f = rows(*f_in, "f");
    if (f->sizes() != x.sizes()) fail("residual_norm: f must have the shape of x");
  } else if (gate_in || scale_in || post_weight || post_bias || !next) {
    fail("residual_norm: without f there is the norm of x alone (no gate, scale or norm of f)");
  }
  if (!next && (next_weight || next_bias || keep)) fail("residual_norm: parameters or kept rows of a norm that is not asked for");
  if (!post && (post_weight || post_bias)) fail("residual_norm: parameters of a norm that is not asked for");
  if (gate_in) {
    gate = rows(*gate_in, "gate");
    const bool per_row = (gate->dim() == 1 || (gate->dim() == 2 && gate->size(1) == 1)) && gate->size(0) == x.size(0);
    if (!per_row && gate->sizes() != x.sizes()) fail("residual_norm: gate must have the shape of x, or one value per row");
  }
  c10::cuda::CUDAGuard guard(x.device());
  all_recorded_in_capture("residual_norm", x_in, f_in, gate_in, scale_in, post_weight, post_bias, next_weight, next_bias);
  const auto scale = row_parameter(scale_in, x, "scale"), w2 = row_parameter(post_weight, x, "post_weight"),
             b2 = row_parameter(post_bias, x, "post_bias"), w1 = row_parameter(next_weight, x, "next_weight"),
             b1 = row_parameter(next_bias, x, "next_bias");
  const bool norm_f = f && post;
  const variable_list out =
      recorded(x, f, gate, scale, w2, b2, w1, b1)
          ? ResidualNormFunction::apply(x, f, gate, scale, w2, b2, w1, b1, norm_f, next, layer, eps, keep)
          : residual_forward(x, f, gate, scale, w2, b2, w1, b1, ResidualOptions{norm_f, next, layer, keep, eps});
  std::vector<optional<Tensor>> all(4);
  size_t at = 0;
  all[0] = f ? out[at++] : x_in;
  if (next) all[1] = out[at++];
  if (keep) all[2] = out[at], all[3] = out[at + 1];
  return all;
}

// ---- SAGE layer ------------------------------------------------------------------------------------------------------
// into += g . w, or g . w into a new matrix
Tensor linear_input_grad(const Tensor &g, const Tensor &w, const Tensor &into) {
  const int n = static_cast<int>(g.size(1)), k = static_cast<int>(w.size(1));
  if (dense_rows(g) && lib.cxg_linear_f32_supported(g.size(0), n, k) && (!into.defined() || aligned16(into))) {
    const Tensor out = into.defined() ? into : at::empty({g.size(0), k}, g.options());
    check(lib.cxg_linear_f32(g.data_ptr<float>(), w.data_ptr<float>(), nullptr, into.defined() ? into.data_ptr<float>() : nullptr,
                             out.data_ptr<float>(), g.size(0), n, k, 1, stream_of(g)),
          "cxg_linear_f32");
    return out;
  }
  return into.defined() ? into.addmm_(g, w) : at::mm(g, w);
}

// mean(x) . wl^T + x[:n] . wr^T + bl, the mean taken before (`first`) or behind the product with wl. As one operator the
// gradient of x[:n] is added to that of the aggregation in place; as separate ones it was a matrix of zeros, a copy and a sum.
class SageLayerFunction : public torch::autograd::Function<SageLayerFunction> {
 public:
  static Tensor run(const Tensor &x, const Tensor &ptr, const Tensor &idx, const Tensor &wl, const Tensor &wr,
                    const optional<Tensor> &bl, int64_t n, bool first, int64_t flags, int64_t split, Tensor *mean, bool record) {
    auto aggregate = [&](const Tensor &t) {
      return spmm(t, ptr, idx, n, c10::nullopt, CXG_MEAN, c10::nullopt, c10::nullopt, c10::nullopt, 0, c10::nullopt, flags, split);
    };
    // the products of a recorded pass keep torch's rounding, as in `linear`
    auto product = [&](const Tensor &t) { return record ? at::linear(t, wl, bl) : linear_product(t, wl, false, bl, c10::nullopt); };
    Tensor out;
    if (first) {
      const Tensor m = aggregate(x);
      if (mean != nullptr) *mean = m;
      out = product(m);
    } else {
      out = aggregate(product(x));
    }
    if (record) return out.add_(at::linear(x.narrow(0, 0, n), wr));
    check(lib.cxg_linear_f32(x.data_ptr<float>(), wr.data_ptr<float>(), nullptr, out.data_ptr<float>(), out.data_ptr<float>(), n,
                             static_cast<int>(x.size(1)), static_cast<int>(wr.size(0)), 0, stream_of(x)),
          "cxg_linear_f32");
    return out;
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &ptr, const Tensor &idx, const Tensor &wl,
                        const Tensor &wr, const optional<Tensor> &bl, int64_t n, bool first, int64_t flags, int64_t split) {
    Tensor mean;
    const Tensor out = run(x, ptr, idx, wl, wr, bl, n, first, flags, split, &mean, true);
    ctx->save_for_backward({x, ptr, idx, wl, wr, mean});
    ctx->saved_data["bias"] = bl.has_value();
    ctx->saved_data["n"] = n;
    ctx->saved_data["first"] = first;
    ctx->saved_data["flags"] = flags;
    ctx->saved_data["split"] = split;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &ptr = saved[1], &idx = saved[2], &wl = saved[3], &wr = saved[4], &mean = saved[5];
    const int64_t n = ctx->saved_data["n"].toInt(), flags = ctx->saved_data["flags"].toInt(), split = ctx->saved_data["split"].toInt();
    const bool need_x = ctx->needs_input_grad(0), need_wl = ctx->needs_input_grad(3), need_wr = ctx->needs_input_grad(4);
    const bool need_bl = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(5);
    const Tensor g = grads[0].contiguous();
    c10::cuda::CUDAGuard guard(g.device());
    auto back = [&](const Tensor &t) { return spmm_transposed(t, ptr, idx, n, x.size(0), c10::nullopt, CXG_MEAN, flags, split); };
    Tensor dx, dwl, dwr, dbl;
    if (ctx->saved_data["first"].toBool()) {
      if (need_x) dx = back(linear_input_grad(g, wl, Tensor()));
      if (need_wl) dwl = linear_weight_grad(g, mean);
      if (need_bl) dbl = rows_sum(g);
    } else if (need_x || need_wl || need_bl) {
      const Tensor dh = back(g);
      if (need_x) dx = linear_input_grad(dh, wl, Tensor());
      if (need_wl) dwl = linear_weight_grad(dh, x);
      if (need_bl) dbl = rows_sum(dh);
    }
    if (need_x) linear_input_grad(g, wr, dx.narrow(0, 0, n));
    if (need_wr) dwr = linear_weight_grad(g, x.narrow(0, 0, n));
    return {dx, Tensor(), Tensor(), dwl, dwr, dbl, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// None when the operator does not cover the arguments.
optional<Tensor> sage_layer(const Tensor &x, const Tensor &ptr, const Tensor &idx, const Tensor &wl, const Tensor &wr,
                            const optional<Tensor> &bl, int64_t n, bool first, int64_t flags, int64_t split) {
  if (for_torch(x, wl, wr, bl) || n < 1 || !dense_rows(x) || x.size(0) < n || idx.size(0) < 1 || ptr.size(0) - 1 < n || wl.size(0) != wr.size(0) ||
      !linear_fits(x, wl) || !linear_fits(x, wr) ||
      !lib.cxg_linear_f32_supported(n, static_cast<int>(x.size(1)), static_cast<int>(wl.size(0))) ||
      at::autocast::is_autocast_enabled(at::kCUDA) ||
      (bl && (bl->scalar_type() != at::kFloat || !bl->is_contiguous() || bl->device() != x.device() || bl->numel() != wl.size(0))))
    return c10::nullopt;
  index_of(ptr, "ptr");
  index_of(idx, "idx");
  c10::cuda::CUDAGuard guard(x.device());
  if (recorded(x, wl, wr, bl)) return SageLayerFunction::apply(x, ptr, idx, wl, wr, bl, n, first, flags, split);
  return SageLayerFunction::run(x, ptr, idx, wl, wr, bl, n, first, flags, split, nullptr, false);
}

// ---- GAT layer -------------------------------------------------------------------------------------------------------
Tensor head_mean_bias(const Tensor &x, const optional<Tensor> &bias, int64_t heads, int64_t c) {
  Tensor out = at::empty({x.size(0), c}, x.options());
  check(lib.cxg_head_mean_bias(x.data_ptr<float>(), bias ? bias->data_ptr<float>() : nullptr, out.data_ptr<float>(), x.size(0),
                               static_cast<int>(heads), static_cast<int>(c), stream_of(x)),
        "cxg_head_mean_bias");
  return out;
}

// Attention scores, softmax, weighted neighbour sum, heads joined or averaged, bias: x [n_src, H, C] -> [n, H * C] or [n, C].
class GatFunction : public torch::autograd::Function<GatFunction> {
 public:
  static Tensor run(const Tensor &x, const Tensor &att_src, const Tensor &att_dst, const optional<Tensor> &bias, const Tensor &ptr,
                    const Tensor &idx, int64_t n, double slope, bool concat, variable_list *keep, Tensor *joined = nullptr) {
    const int64_t n_src = x.size(0), h = x.size(1), c = x.size(2);
    const int hi = static_cast<int>(h), ci = static_cast<int>(c);
    void *st = stream_of(x);
    const Tensor a_src = at::empty({n_src, h}, x.options()), a_dst = at::empty({n, h}, x.options());
    check(lib.cxg_gat_scores(x.data_ptr<float>(), att_src.data_ptr<float>(), att_dst.data_ptr<float>(), a_src.data_ptr<float>(),
                             a_dst.data_ptr<float>(), n_src, n, hi, ci, st),
          "cxg_gat_scores");
    const Tensor y = at::empty({n, h * c}, x.options()), top = at::empty({n, h}, x.options()), sum = at::empty({n, h}, x.options());
    size_t need = 0;
    check(lib.cxg_gat_fused_workspace_size(n, idx.size(0), hi, ci, &need), "cxg_gat_fused_workspace_size");
    {
      const Workspace ws = workspace_on(x.device().index(), st, static_cast<int64_t>(need), "");
      check(lib.cxg_gat_fused_forward(ptr.data_ptr(), idx.data_ptr(), static_cast<int>(ptr.element_size()),
                                      static_cast<int>(idx.element_size()), x.data_ptr<float>(), a_src.data_ptr<float>(),
                                      a_dst.data_ptr<float>(), y.data_ptr<float>(), top.data_ptr<float>(), sum.data_ptr<float>(), n,
                                      idx.size(0), hi, ci, static_cast<float>(slope), ws.data(),
                                      ws.bytes(), st),
            "cxg_gat_fused_forward");
    }
    if (keep != nullptr) *keep = {x, att_src, att_dst, ptr, idx, a_src, a_dst, y, top, sum};
    if (joined != nullptr) {
      *joined = y;
      return y;
    }
    if (concat) return bias ? head_mean_bias(y, bias, 1, h * c) : y;
    return head_mean_bias(y, bias, h, c);
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &att_src, const Tensor &att_dst,
                        const optional<Tensor> &bias, const Tensor &ptr, const Tensor &idx, int64_t n, double slope, bool concat) {
    variable_list keep;
    Tensor out = run(x, att_src, att_dst, bias, ptr, idx, n, slope, concat, &keep);
    if (concat && !bias) out = out.view(out.sizes());  // y itself is kept for the backward
    ctx->save_for_backward(keep);
    ctx->saved_data["slope"] = slope;
    ctx->saved_data["concat"] = concat;
    ctx->saved_data["bias"] = bias.has_value();
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &att_src = saved[1], &att_dst = saved[2], &ptr = saved[3], &idx = saved[4], &a_src = saved[5],
                 &a_dst = saved[6], &y = saved[7], &top = saved[8], &sum = saved[9];
    const int64_t n_src = x.size(0), h = x.size(1), c = x.size(2), n = y.size(0);
    const int hi = static_cast<int>(h), ci = static_cast<int>(c);
    c10::cuda::CUDAGuard guard(x.device());
    void *st = stream_of(x);
    const Tensor g = grads[0].contiguous();
    Tensor db;
    const bool concat = ctx->saved_data["concat"].toBool(), need_db = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
    // heads side by side: the columns of dy are the bias's, and the backward reads them anyway
    if (need_db) db = concat && n > 0 && n_src > 0 ? at::empty({h * c}, x.options()) : rows_sum(g);
    const Tensor dy =
        concat ? g : g.mul(1.0 / static_cast<double>(h)).unsqueeze(1).expand({n, h, c}).contiguous();
    const Transposed t = transposed_graph(ptr, idx, n, n_src);
    const Tensor dx = at::empty_like(x), d_src = at::empty_like(a_src), d_dst = at::empty_like(a_dst);
    const Tensor g_as = at::empty_like(att_src), g_ad = at::empty_like(att_dst);
    size_t need = 0, need_att = 0;
    check(lib.cxg_gat_fused_workspace_size(n, idx.size(0), hi, ci, &need), "cxg_gat_fused_workspace_size");
    check(lib.cxg_gat_att_grad_workspace_size(hi, ci, &need_att), "cxg_gat_att_grad_workspace_size");
    const Workspace ws = workspace_on(x.device().index(), st, static_cast<int64_t>(std::max(need, need_att)), "");
    check(lib.cxg_gat_fused_backward_bias(t.t_ptr.data_ptr(), t.t_idx.data_ptr(), static_cast<int>(t.t_ptr.element_size()),
                                     static_cast<int>(t.t_idx.element_size()), dy.data_ptr<float>(), y.data_ptr<float>(),
                                     x.data_ptr<float>(), a_src.data_ptr<float>(), a_dst.data_ptr<float>(), top.data_ptr<float>(),
                                     sum.data_ptr<float>(), dx.data_ptr<float>(), d_src.data_ptr<float>(), d_dst.data_ptr<float>(),
                                     n_src, n, t.t_idx.size(0), hi, ci, static_cast<float>(ctx->saved_data["slope"].toDouble()),
                                     nullptr, nullptr, static_cast<int>(ptr.element_size()),
                                     need_db && concat && n > 0 && n_src > 0 ? db.data_ptr<float>() : nullptr, ws.data(), ws.bytes(), st),
          "cxg_gat_fused_backward");
    check(lib.cxg_gat_scores_backward_add(x.data_ptr<float>(), d_src.data_ptr<float>(), d_dst.data_ptr<float>(),
                                          att_src.data_ptr<float>(), att_dst.data_ptr<float>(), dx.data_ptr<float>(),
                                          g_as.data_ptr<float>(), g_ad.data_ptr<float>(), n_src, n, hi, ci, ws.data(),
                                          ws.bytes(), st),
          "cxg_gat_scores_backward_add");
    return {dx, g_as, g_ad, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor gat_layer(const Tensor &x, const Tensor &att_src, const Tensor &att_dst, const optional<Tensor> &bias, const Tensor &ptr,
                 const Tensor &idx, int64_t num_dst, double slope, bool concat) {
  f32(x, "x");
  f32(att_src, "att_src");
  f32(att_dst, "att_dst");
  index_of(ptr, "ptr");
  index_of(idx, "idx");
  const int64_t n = rows_of(ptr, num_dst), h = x.size(1), c = x.size(2);
  if (x.dim() != 3 || att_src.numel() != h * c || att_dst.numel() != h * c || n > x.size(0))
    fail("gat_layer: x must be [n_src, H, C] with n_src >= num_dst, the attention vectors [H, C]");
  if (bias) {
    f32(*bias, "bias");
    if (bias->numel() != (concat ? h * c : c)) fail("gat_layer: the bias must have one value per output column");
  }
  c10::cuda::CUDAGuard guard(x.device());
  if (recorded(x, att_src, att_dst, bias))
    return GatFunction::apply(x, att_src, att_dst, bias, ptr, idx, n, slope, concat);
  return GatFunction::run(x, att_src, att_dst, bias, ptr, idx, n, slope, concat, nullptr);
}

// The whole layer in inference where its heads are not whole vectors (class counts): transformed with the heads padded, so that
// no vector lies across two of them (4 heads of 47, 2.3 M edges: 665 us without, see gat_weights for what the walk gains). None
// where it does not cover the arguments.
optional<Tensor> gat_layer_padded(const Tensor &x, const Tensor &w, const Tensor &att_src, const Tensor &att_dst,
                                  const optional<Tensor> &bias, const Tensor &ptr, const Tensor &idx, int64_t num_dst, int64_t heads,
                                  double slope, bool concat) {
  const int64_t c = w.dim() == 2 && heads > 0 ? w.size(0) / heads : 0, cp = (c + 3) / 4 * 4;
  // below eight columns the zeros are a third of a row and more
  if (c < 8 || cp == c || (heads & (heads - 1)) != 0 || heads > 8 || heads * cp > 512 || c * heads != w.size(0)) return c10::nullopt;
  if (for_torch(x, w, att_src, att_dst, bias) || recorded(x, w, att_src, att_dst, bias) || at::autocast::is_autocast_enabled(at::kCUDA) ||
      !linear_fits(x, w) || !lib.cxg_linear_f32_supported(x.size(0), static_cast<int>(x.size(1)), static_cast<int>(heads * cp)))
    return c10::nullopt;
  auto fits = [&](const Tensor &t, int64_t numel) {
    return t.is_cuda() && t.device() == x.device() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == numel;
  };
  if (!fits(att_src, heads * c) || !fits(att_dst, heads * c) || (bias && !fits(*bias, concat ? heads * c : c))) return c10::nullopt;
  index_of(ptr, "ptr");
  index_of(idx, "idx");
  const int64_t n = rows_of(ptr, num_dst);
  if (n < 1 || n > x.size(0)) return c10::nullopt;
  c10::cuda::CUDAGuard guard(x.device());
  const int hi = static_cast<int>(heads), ci = static_cast<int>(c), cpi = static_cast<int>(cp);
  const Tensor wp = at::empty({heads * cp, x.size(1)}, x.options()), att = at::empty({2, heads, cp}, x.options());
  check(lib.cxg_gat_pad_heads(w.data_ptr<float>(), att_src.data_ptr<float>(), att_dst.data_ptr<float>(), wp.data_ptr<float>(),
                              att.data_ptr<float>(), att.data_ptr<float>() + heads * cp, hi, ci, cpi, static_cast<int>(x.size(1)),
                              stream_of(x)),
        "cxg_gat_pad_heads");
  const Tensor h = linear_product(x, wp, false, c10::nullopt, c10::nullopt).view({x.size(0), heads, cp});
  Tensor y;
  GatFunction::run(h, att.select(0, 0), att.select(0, 1), c10::nullopt, ptr, idx, n, slope, concat, nullptr, &y);
  Tensor out = at::empty({n, concat ? heads * c : c}, x.options());
  check(lib.cxg_gat_unpad_heads(y.data_ptr<float>(), bias ? bias->data_ptr<float>() : nullptr, out.data_ptr<float>(), n, hi, ci, cpi,
                                concat ? 1 : 0, stream_of(x)),
        "cxg_gat_unpad_heads");
  return out;
}

// ---- relational layer ------------------------------------------------------------------------------------------------
// (relation, source and number of every position, first position of every source's list, the lists, position of every edge)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> relation_pairs(const Tensor &idx, const Tensor &etype, int64_t n_src,
                                                                          int64_t num_rel) {
  index_of(idx, "idx");
  index_of(etype, "edge types");
  const int64_t nnz = std::min(idx.size(0), etype.size(0));
  const int ib = static_cast<int>(idx.element_size()), rb = static_cast<int>(etype.element_size()), r = static_cast<int>(num_rel);
  c10::cuda::CUDAGuard guard(idx.device());
  const auto i64 = idx.options().dtype(at::kLong), i32 = idx.options().dtype(at::kInt);
  size_t need = 0;
  check(lib.cxg_relation_pairs_workspace_size(n_src, r, &need), "cxg_relation_pairs_workspace_size");
  // a buffer of its own: the second call continues in it behind the read-back
  const Tensor ws = at::empty({static_cast<int64_t>(need)}, idx.options().dtype(at::kByte)), sizes = at::empty({3}, i64);
  void *st = stream_of(idx);
  check(lib.cxg_relation_pairs_count(idx.data_ptr(), ib, etype.data_ptr(), rb, nnz, n_src, r, sizes.data_ptr<int64_t>(),
                                     ws.data_ptr(), need, st),
        "cxg_relation_pairs_count");
  Tensor host;
  {
    py::gil_scoped_release other_threads;
    host = sizes.cpu();
  }
  const int64_t *h = host.data_ptr<int64_t>();
  if (h[2] != 0)
    fail("edge types must lie in [0, " + std::to_string(num_rel) + ") and sources in [0, " + std::to_string(n_src) + ")");
  Tensor rel = at::empty({h[0]}, i64), src = at::empty({h[0]}, i64), pos = at::empty({h[0]}, i64), src_ptr = at::empty({n_src + 1}, i64),
         src_pos = at::empty({h[1]}, i32), edge_pos = at::empty({nnz}, i32);
  check(lib.cxg_relation_pairs_fill(idx.data_ptr(), ib, etype.data_ptr(), rb, nnz, n_src, r, rel.data_ptr<int64_t>(),
                                    src.data_ptr<int64_t>(), pos.data_ptr<int64_t>(), src_ptr.data_ptr<int64_t>(),
                                    src_pos.data_ptr<int32_t>(), edge_pos.data_ptr<int32_t>(), ws.data_ptr(), need, st),
        "cxg_relation_pairs_fill");
  return {rel, src, pos, src_ptr, src_pos, edge_pos};
}

// ---- neighbour sampling ----------------------------------------------------------------------------------------------
// The most a call may reserve for the nodes and edges a batch can reach; above it the hops are run one by one.
constexpr int64_t kMostSampled = 1 << 27;

bool sample_batch_fits(int64_t n_seeds, std::vector<int> fanouts, int64_t n_nodes, int64_t nnz) {
  int64_t nodes = 0, rows = 0, edges = 0;
  size_t bytes = 0;
  if (n_seeds < 1 || lib.cxg_sample_batch_bounds(n_seeds, fanouts.data(), static_cast<int>(fanouts.size()), n_nodes, nnz, &nodes,
                                                 &rows, &edges, &bytes) != 0)
    return false;
  return nodes + edges <= kMostSampled;
}

// (nodes, ptr, idx, nodes after every hop, edges after every hop): one host synchronisation, at the end, for the sizes.
std::tuple<Tensor, Tensor, Tensor, std::vector<int64_t>, std::vector<int64_t>> sample_batch(
    const Tensor &gptr, const Tensor &gidx, const Tensor &seeds, std::vector<int> fanouts, std::vector<uint64_t> hop_seeds,
    const Tensor &local_of, const Tensor &bitmap, const Tensor &host_sizes) {
  index_of(gptr, "graph_ptr");
  index_of(gidx, "graph_idx");
  of_type(seeds, "seeds", {at::kLong});
  const int hops = static_cast<int>(fanouts.size());
  const int64_t n_nodes = gptr.size(0) - 1, nnz = gidx.size(0);
  int64_t max_nodes = 0, max_rows = 0, max_edges = 0;
  size_t bytes = 0;
  check(lib.cxg_sample_batch_bounds(seeds.size(0), fanouts.data(), hops, n_nodes, nnz, &max_nodes, &max_rows, &max_edges, &bytes),
        "cxg_sample_batch_bounds");
  c10::cuda::CUDAGuard guard(seeds.device());
  const auto opt = seeds.options();
  Tensor nodes = at::empty({max_nodes}, opt), ptr = at::empty({max_rows + 1}, opt), idx = at::empty({max_edges}, opt);
  Tensor sizes = at::empty({2 * (hops + 1)}, opt);
  void *st = stream_of(seeds);
  {
    const Workspace ws = workspace_on(seeds.device().index(), st, static_cast<int64_t>(bytes), "");
    check(lib.cxg_sample_batch(gptr.data_ptr(), gidx.data_ptr(), static_cast<int>(gptr.element_size()),
                               static_cast<int>(gidx.element_size()), n_nodes, nnz, seeds.data_ptr<int64_t>(), seeds.size(0),
                               fanouts.data(), hops, hop_seeds.data(), local_of.data_ptr<int64_t>(),
                               reinterpret_cast<uint32_t *>(bitmap.data_ptr()), nodes.data_ptr<int64_t>(), ptr.data_ptr<int64_t>(),
                               idx.data_ptr<int64_t>(), sizes.data_ptr<int64_t>(), ws.data(), ws.bytes(), st),
          "cxg_sample_batch");
  }
  host_sizes.narrow(0, 0, sizes.size(0)).copy_(sizes, /*non_blocking=*/true);
  {
    py::gil_scoped_release other_threads;
    c10::cuda::getCurrentCUDAStream(seeds.device().index()).synchronize();
  }
  const int64_t *h = host_sizes.data_ptr<int64_t>();
  if (h[0] < 0) fail("sample_batch: seeds must be node ids in [0, " + std::to_string(n_nodes) + ")");
  std::vector<int64_t> known(h, h + hops + 1), edges(h + hops + 2, h + 2 * (hops + 1));
  const int64_t rows = known[hops - 1];
  return {nodes.narrow(0, 0, known[hops]), ptr.narrow(0, 0, rows + 1), idx.narrow(0, 0, edges[hops - 1]), known, edges};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("init", &init);
  py::class_<HeldWorkspace>(m, "Workspace")
      .def(py::init<int, int64_t, std::string>())
      .def("__enter__", &HeldWorkspace::enter)
      .def("__exit__", [](HeldWorkspace &w, const py::args &) { w.exit(); });
  m.def("last_workspace", &last_workspace);
  py::class_<Kept>(m, "Kept").def(py::init<std::vector<Tensor>>()).def("take", &Kept::take);
  m.def("capturing", [](int device) { return capture_of(c10::cuda::getCurrentCUDAStream(device).stream()).has_value(); });
  m.def("spmm", &spmm);
  m.def("sage", &sage);
  m.def("spmm_transposed", &spmm_transposed);
  m.def("transpose", [](const Tensor &ptr, const Tensor &idx, int64_t n, int64_t n_src, bool want_eid) {
    const Transposed t = transpose(ptr, idx, n, n_src, want_eid);
    return std::make_tuple(t.t_ptr, t.t_idx, want_eid ? optional<Tensor>(t.t_eid) : c10::nullopt, t.inv_deg);
  });
  m.def("transposed_graph", [](const Tensor &ptr, const Tensor &idx, int64_t n, int64_t n_src) {
    const Transposed t = transposed_graph(ptr, idx, n, n_src);
    return std::make_tuple(t.t_ptr, t.t_idx, t.t_eid, t.inv_deg);
  });
  m.def("forget_graphs", &forget_graphs);
  m.def("count_graphs", &count_graphs);
  m.def("gather_rows", &gather_rows);
  m.def("linear", &linear);
  m.def("gat_layer", &gat_layer);
  m.def("gat_layer_padded", &gat_layer_padded);
  m.def("sage_layer", &sage_layer);
  m.def("head_mean_bias", [](const Tensor &x, const optional<Tensor> &bias, int64_t heads, int64_t c) {
    f32(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    return head_mean_bias(x, bias, heads, c);
  });
  m.def("relation_pairs", &relation_pairs);
  m.def("rows8_pitch", [](int64_t width) { return lib.cxg_rows8_pitch(static_cast<int>(width)); });
  m.def("rows8_zeros", [](int64_t rows, int64_t width, at::Device device) {
    const Held h = held_zeros(rows, width, device);
    return std::make_pair(h.codes, h.scales);
  });
  m.def("rows8_quantize", [](const Tensor &x) {
    const Held h = quantize(x);
    return std::make_pair(h.codes, h.scales);
  });
  m.def("rows8_quantize_into", &quantize_into);
  m.def("rows8_dequantize", &dequantize);
  m.def("rows8_aggregate", &rows8_aggregate);
  m.def("rows8_weight_grad", [](const Tensor &codes, const Tensor &scales, int64_t width, const Tensor &dy, bool bias) {
    const auto g = rows8_weight_grad(codes, scales, width, dy, bias, at::kFloat);
    return std::make_pair(g.first, bias ? optional<Tensor>(g.second) : c10::nullopt);
  });
  m.def("linear_kept8", &linear_kept8);
  m.def("residual_norm", &residual_norm);
  m.def("sample_batch_fits", &sample_batch_fits);
  m.def("sample_batch", &sample_batch);
}
