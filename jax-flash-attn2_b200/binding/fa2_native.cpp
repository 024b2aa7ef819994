// CPython module between torch tensors and the C ABI of fa2_b200_lm.h: the operators for language models without the
// Python layer's cost per call.
//
// A call of a few microseconds on the GPU is bound by what the host does for it: reading shapes and strides, filling a
// parameter block field by field and crossing into autograd in Python takes 15 to 200 us, here 5 to 40. Each function takes
// exactly the calls that need nothing but a launch. For any other (an argument to be refused, a tensor to be copied first) it
// returns None, and the Python function of the same name goes on: it holds the checks with their messages and is the
// description of every operator. Nothing is computed here.
//
// The C ABI's functions are handed over as addresses (`bind`), so that this module works on whichever build of the library the
// package has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstdlib>
#include <cstring>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/autograd.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/fa2_b200_lm.h"

namespace {

using at::Tensor;

struct Abi {
  decltype(&fa2_document_layout_bytes) document_layout_bytes;
  decltype(&fa2_document_layout) document_layout;
  decltype(&fa2_fwd_workspace_bytes) fwd_workspace_bytes;
  decltype(&fa2_scored_bwd_workspace_bytes) scored_bwd_workspace_bytes;
  decltype(&fa2_scored_fwd) scored_fwd;
  decltype(&fa2_scored_bwd) scored_bwd;
  decltype(&fa2_paged_work_bytes) paged_work_bytes;
  decltype(&fa2_paged_plan) paged_plan;
  decltype(&fa2_paged_cache_write) paged_cache_write;
  decltype(&fa2_paged_workspace_bytes) paged_workspace_bytes;
  decltype(&fa2_paged_attention) paged_attention;
  decltype(&fa2_last_error) last_error;
} abi;
constexpr int kAbiFunctions = sizeof(Abi) / sizeof(void*);

// ---- arguments -------------------------------------------------------------------------------
bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }
// None becomes an undefined tensor; false if it is neither None nor a tensor.
bool optional_tensor(PyObject* o, Tensor* out) {
  if (o == Py_None) return true;
  if (!is_tensor(o)) return false;
  *out = tensor(o);
  return true;
}
// None becomes `fallback`; false if it is neither None nor a number.
bool optional_number(PyObject* o, double fallback, double* out) {
  *out = fallback;
  if (o == Py_None) return true;
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  *out = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool integer(PyObject* o, int64_t* out) {
  if (!PyLong_Check(o)) return false;
  *out = PyLong_AsLongLong(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return *out >= INT32_MIN && *out <= INT32_MAX;
}

int dtype_code(at::ScalarType t) { return t == at::kHalf ? FA2_FP16 : t == at::kBFloat16 ? FA2_BF16 : -1; }

fa2_strides strides_of(const Tensor& x) { return {x.stride(0), x.stride(1), x.stride(2)}; }

bool vector_of(const Tensor& x, at::ScalarType t, int64_t n, const at::Device& device) {
  return x.scalar_type() == t && x.dim() == 1 && x.size(0) == n && x.device() == device && x.is_contiguous();
}

bool softcap_ok(double cap) { return cap == 0.0 || (cap >= 1.0 / 1024 && cap <= 1024.0); }

void* stream_of(const Tensor& x) { return at::cuda::getCurrentCUDAStream(x.device().index()).stream(); }

Tensor bytes_like(const Tensor& x, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, x.options().dtype(at::kByte));
}

// `n` elements of type `t` from byte `at` of a fresh buffer, as a tensor of their own.
Tensor part_of(const Tensor& buffer, at::ScalarType t, int64_t at, int64_t n) {
  Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(),
                                                      c10::scalarTypeToTypeMeta(t));
  x.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(t)));
  x.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return x;
}

// Tells autograd of a write in place, so that a backward pass that saved `x` notices.
void written(const Tensor& x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

// ---- attention with changed scores -------------------------------------------------------------
struct Scored {
  Tensor slopes, layout, prefix, rest;
  double scale, softcap;
  bool causal;

  void fill(fa2_score_mod* m) const {
    *m = {};
    m->softcap = static_cast<float>(softcap);
    if (slopes.defined()) m->alibi_slopes = slopes.const_data_ptr<float>();
    if (prefix.defined()) m->prefix_lens = prefix.const_data_ptr<int32_t>();
    if (layout.defined()) m->document_layout = layout.const_data_ptr<int32_t>();
    if (rest.defined()) {
      m->o_rest = rest.data_ptr();
      m->o_rest_strides = strides_of(rest);
    }
  }
};

fa2_problem problem_of(const Tensor& q, const Tensor& k, const Scored& s) {
  fa2_problem p = {};
  p.batch = static_cast<int32_t>(q.size(0));
  p.seqlen_q = static_cast<int32_t>(q.size(1));
  p.seqlen_k = static_cast<int32_t>(k.size(1));
  p.heads_q = p.heads_q_global = static_cast<int32_t>(q.size(2));
  p.heads_kv = static_cast<int32_t>(k.size(2));
  p.head_dim = static_cast<int32_t>(q.size(3));
  p.dtype = dtype_code(q.scalar_type());
  p.causal = s.causal;
  p.softmax_scale = static_cast<float>(s.scale);
  return p;
}

// Output and lse; false if the library refused the call (nothing has been launched then).
bool forward_launch(const Tensor& q, const Tensor& k, const Tensor& v, const Scored& s, Tensor* out, Tensor* lse) {
  fa2_fwd_params a = {};
  a.p = problem_of(q, k, s);
  const fa2_problem& p = a.p;
  *out = at::empty(q.sizes(), q.options());
  const int64_t rows = (p.seqlen_q + 127) / 128 * 128;
  *lse = at::empty({p.batch, p.heads_q, rows}, q.options().dtype(at::kFloat));
  a.q = q.const_data_ptr(); a.q_strides = strides_of(q);
  a.k = k.const_data_ptr(); a.k_strides = strides_of(k);
  a.v = v.const_data_ptr(); a.v_strides = strides_of(v);
  a.o = out->data_ptr(); a.o_strides = strides_of(*out);
  a.lse = lse->data_ptr<float>();
  a.lse_stride_b = p.heads_q * rows;
  a.lse_stride_h = rows;
  Tensor workspace;
  if (const size_t n = abi.fwd_workspace_bytes(&p)) {
    workspace = bytes_like(q, n);
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = n;
  }
  fa2_score_mod m;
  s.fill(&m);
  return abi.scored_fwd(&a, &m, stream_of(q)) == FA2_OK;
}

// A cotangent may have any strides (expanded, transposed): the kernels want positive multiples of 8 and unit columns.
Tensor laid_out(const Tensor& x) {
  bool fine = x.stride(3) == 1 && reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) fine = fine && x.stride(i) > 0 && x.stride(i) % 8 == 0;
  return fine ? x : x.clone(at::MemoryFormat::Contiguous);
}

// The backward pass as a node of the autograd graph. Written out (torch::autograd::Function would do) because at a few
// hundred tokens autograd's work on the host is what a training step takes: lse and rest never leave the node.
struct ScoredBackward : torch::autograd::Node {
  torch::autograd::SavedVariable q, k, v, out, slopes, layout, prefix;
  Tensor lse, rest;
  double scale = 0, softcap = 0;
  bool causal = false;

  std::string name() const override { return "ScoredAttentionBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* x : {&q, &k, &v, &out, &slopes, &layout, &prefix}) x->reset_data();
    lse.reset();
    rest.reset();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!at::GradMode::is_enabled(), "scored_flash_attention has no second derivatives (create_graph=True)");
    torch::autograd::variable_list result(3);
    if (!grads[0].defined()) return result;
    const Tensor inputs[3] = {q.unpack(), k.unpack(), v.unpack()};
    const Tensor o = out.unpack(shared_from_this());
    Scored s;
    s.slopes = slopes.unpack();
    s.layout = layout.unpack();
    s.prefix = prefix.unpack();
    s.rest = rest;
    s.scale = scale;
    s.softcap = softcap;
    s.causal = causal;
    const at::AutoDispatchBelowADInplaceOrView no_autograd;
    const c10::cuda::CUDAGuard guard(o.device());
    const Tensor d_o = laid_out(grads[0]);
    fa2_bwd_params a = {};
    a.p = problem_of(inputs[0], inputs[1], s);
    const size_t n = abi.scored_bwd_workspace_bytes(&a.p);
    const Tensor workspace = bytes_like(o, n);
    for (int i = 0; i < 3; ++i) result[i] = at::empty(inputs[i].sizes(), o.options());
    a.q = inputs[0].const_data_ptr(); a.q_strides = strides_of(inputs[0]);
    a.k = inputs[1].const_data_ptr(); a.k_strides = strides_of(inputs[1]);
    a.v = inputs[2].const_data_ptr(); a.v_strides = strides_of(inputs[2]);
    a.o = o.const_data_ptr(); a.o_strides = strides_of(o);
    a.d_o = d_o.const_data_ptr(); a.do_strides = strides_of(d_o);
    a.lse = lse.const_data_ptr<float>();
    a.lse_stride_b = lse.stride(0);
    a.lse_stride_h = lse.stride(1);
    a.dq = result[0].data_ptr(); a.dq_strides = strides_of(result[0]);
    a.dk = result[1].data_ptr(); a.dk_strides = strides_of(result[1]);
    a.dv = result[2].data_ptr(); a.dv_strides = strides_of(result[2]);
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = n;
    const char* det = std::getenv("FA2_B200_DETERMINISTIC");
    a.deterministic = det && *det && !(det[0] == '0' && det[1] == 0);
    fa2_score_mod m;
    s.fill(&m);
    const int rc = abi.scored_bwd(&a, &m, stream_of(o));
    TORCH_CHECK(rc == FA2_OK, "fa2_b200 error ", rc, ": ", abi.last_error());
    return result;
  }
};

// The forward pass under autograd; false if the library refused the call.
bool forward_with_node(const Tensor& q, const Tensor& k, const Tensor& v, Scored* s, Tensor* out) {
  const std::shared_ptr<ScoredBackward> node(new ScoredBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
  {
    const at::AutoDispatchBelowADInplaceOrView no_autograd;
    // bf16: see o_rest in fa2_b200_lm.h
    if (q.scalar_type() == at::kBFloat16) node->rest = s->rest = at::empty(q.sizes(), q.options());
    if (!forward_launch(q, k, v, *s, out, &node->lse)) return false;
  }
  torch::autograd::set_history(*out, node);
  using torch::autograd::SavedVariable;
  node->q = SavedVariable(q, false);
  node->k = SavedVariable(k, false);
  node->v = SavedVariable(v, false);
  node->out = SavedVariable(*out, true);
  node->slopes = SavedVariable(s->slopes, false);
  node->layout = SavedVariable(s->layout, false);
  node->prefix = SavedVariable(s->prefix, false);
  node->scale = s->scale;
  node->softcap = s->softcap;
  node->causal = s->causal;
  return true;
}

// Whether a live autograd graph made on another stream ends in the leaf `x`: autograd would synchronise with that stream,
// which breaks a capture.
bool leaf_of_another_stream(const Tensor& x, const c10::Stream& now) {
  if (!x.requires_grad() || !x.is_leaf()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(x);
  if (!node) return false;
  const auto made_on = node->stream();
  return made_on.has_value() && *made_on != now;
}

// Raises if this call, under capture, would break it: leaves whose live graph belongs to another stream.
bool capture_refused(const Tensor& q, const Tensor& k, const Tensor& v) {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return false;
  const c10::Stream now = at::cuda::getCurrentCUDAStream(q.device().index());
  if (!leaf_of_another_stream(q, now) && !leaf_of_another_stream(k, now) && !leaf_of_another_stream(v, now)) return false;
  PyErr_SetString(PyExc_RuntimeError,
                  "a forward pass on another stream has a live autograd graph with the same leaf tensors: "
                  "drop its outputs (or detach them) before capturing this call into a CUDA graph");
  return true;
}

// (q, k, v)
PyObject* check_capture(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !is_tensor(args[0]) || !is_tensor(args[1]) || !is_tensor(args[2])) Py_RETURN_NONE;
  if (capture_refused(tensor(args[0]), tensor(args[1]), tensor(args[2]))) return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (q, k, v, softmax_scale, causal, softcap, alibi_slopes, document_ids, prefix_lens, layout)
PyObject* scored_flash_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !is_tensor(args[0]) || !is_tensor(args[1]) || !is_tensor(args[2])) Py_RETURN_NONE;
  const Tensor &q = tensor(args[0]), &k = tensor(args[1]), &v = tensor(args[2]);
  Scored s;
  Tensor ids;
  if (!optional_tensor(args[6], &s.slopes) || !optional_tensor(args[7], &ids) || !optional_tensor(args[8], &s.prefix) ||
      !optional_tensor(args[9], &s.layout))
    Py_RETURN_NONE;
  if (!q.is_cuda() || q.dim() != 4 || k.dim() != 4 || v.dim() != 4) Py_RETURN_NONE;
  const at::Device device = q.device();
  const int64_t batch = q.size(0), sq = q.size(1), heads = q.size(2), d = q.size(3);
  if (k.device() != device || v.device() != device || dtype_code(q.scalar_type()) < 0 ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.sizes() != v.sizes() ||
      k.size(0) != batch || k.size(3) != d || k.size(2) <= 0 || heads % k.size(2) != 0 || q.numel() == 0 || k.numel() == 0)
    Py_RETURN_NONE;
  if (q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1) Py_RETURN_NONE;
  double cap;
  if (!optional_number(args[3], 1.0 / std::sqrt(static_cast<double>(d)), &s.scale) || !optional_number(args[5], 0.0, &cap) ||
      !softcap_ok(cap))
    Py_RETURN_NONE;
  s.softcap = cap;
  const int causal = PyObject_IsTrue(args[4]);
  if (causal < 0) return nullptr;
  s.causal = causal;
  if (s.slopes.defined() && (!vector_of(s.slopes, at::kFloat, heads, device) || s.slopes.requires_grad())) Py_RETURN_NONE;
  if (s.prefix.defined() && (!causal || !vector_of(s.prefix, at::kInt, batch, device))) Py_RETURN_NONE;
  if (ids.defined() && (s.layout.defined() || ids.scalar_type() != at::kInt || ids.dim() != 2 || ids.size(0) != batch ||
                        ids.size(1) != sq || ids.device() != device || ids.stride(1) != 1 || ids.stride(0) < 0))
    Py_RETURN_NONE;
  if ((ids.defined() || s.layout.defined()) && k.size(1) != sq) Py_RETURN_NONE;
  const size_t layout_bytes = ids.defined() || s.layout.defined()
                                  ? abi.document_layout_bytes(static_cast<int32_t>(batch), static_cast<int32_t>(sq))
                                  : 0;
  // [batch, words per row]: the shape tells the layout of one batch and length from that of another
  const int64_t layout_words = static_cast<int64_t>(layout_bytes / 4) / batch;
  if (s.layout.defined() &&
      (s.layout.scalar_type() != at::kInt || s.layout.dim() != 2 || s.layout.size(0) != batch ||
       s.layout.size(1) != layout_words || s.layout.device() != device || !s.layout.is_contiguous()))
    Py_RETURN_NONE;

  const c10::cuda::CUDAGuard guard(device);
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  if (grad && capture_refused(q, k, v)) return nullptr;
  Tensor out;
  bool refused = false;
  {
    pybind11::gil_scoped_release no_gil;
    if (ids.defined()) {
      s.layout = at::empty({batch, layout_words}, q.options().dtype(at::kInt));
      refused = abi.document_layout(ids.const_data_ptr<int32_t>(), ids.stride(0), static_cast<int32_t>(batch),
                                    static_cast<int32_t>(sq), s.layout.data_ptr<int32_t>(), layout_bytes,
                                    stream_of(q)) != FA2_OK;
    }
    if (!refused) {
      if (grad) {
        refused = !forward_with_node(q, k, v, &s, &out);
      } else {
        Tensor lse;
        refused = !forward_launch(q, k, v, s, &out, &lse);
      }
    }
  }
  if (refused) Py_RETURN_NONE;   // the Python function repeats the call and raises the library's message
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---- paged cache -------------------------------------------------------------------------------
bool page_size_ok(int64_t p) { return p >= 8 && p <= (1 << 20) && (p & (p - 1)) == 0; }

// (context_lens, new_lens, block_table, free_pages, page_size, num_tokens, heads_q, heads_kv, free_start)
//   -> (cu_seqlens, seqlens_k, slot_map, positions, pages_taken, work)
PyObject* paged_step_plan(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    if (!is_tensor(args[i])) Py_RETURN_NONE;
  const Tensor &context = tensor(args[0]), &fresh = tensor(args[1]), &table = tensor(args[2]), &free = tensor(args[3]);
  int64_t page, tokens, heads_q, heads_kv;
  Tensor start;
  if (!integer(args[4], &page) || !integer(args[5], &tokens) || !integer(args[6], &heads_q) || !integer(args[7], &heads_kv) ||
      !optional_tensor(args[8], &start))
    Py_RETURN_NONE;
  if (!table.is_cuda() || table.scalar_type() != at::kInt || table.dim() != 2 || table.numel() == 0 || table.stride(1) != 1 ||
      !page_size_ok(page) || tokens < 0)
    Py_RETURN_NONE;
  const at::Device device = table.device();
  const int64_t requests = table.size(0), width = table.size(1);
  if ((requests > 1 && table.stride(0) < width) || !vector_of(context, at::kInt, requests, device) ||
      !vector_of(fresh, at::kInt, requests, device) || free.dim() != 1 || !vector_of(free, at::kInt, free.size(0), device))
    Py_RETURN_NONE;
  if (start.defined() && !vector_of(start, at::kInt, 1, device)) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(device);
  const size_t bytes = abi.paged_work_bytes(static_cast<int32_t>(requests), static_cast<int32_t>(tokens),
                                            static_cast<int32_t>(heads_q), static_cast<int32_t>(heads_kv));
  if (bytes == 0) Py_RETURN_NONE;
  // one buffer for all of it (an allocation takes longer on the host than a tensor on top of one): the work list, whose size is
  // a multiple of 16 bytes, the slots, and the int32 arrays
  const int64_t slots_at = static_cast<int64_t>((bytes + 15) / 16 * 16), cu_at = slots_at + 8 * tokens,
                lens_at = cu_at + 4 * (requests + 1), positions_at = lens_at + 4 * requests, taken_at = positions_at + 4 * tokens;
  const Tensor buffer = bytes_like(table, static_cast<size_t>(taken_at + 4));
  const Tensor work = part_of(buffer, at::kInt, 0, static_cast<int64_t>(bytes / 4)), slots = part_of(buffer, at::kLong, slots_at, tokens),
               cu = part_of(buffer, at::kInt, cu_at, requests + 1), lens = part_of(buffer, at::kInt, lens_at, requests),
               positions = part_of(buffer, at::kInt, positions_at, tokens), taken = part_of(buffer, at::kInt, taken_at, 1);
  fa2_paged_plan_params a = {};
  a.context_lens = context.const_data_ptr<int32_t>();
  a.new_lens = fresh.const_data_ptr<int32_t>();
  a.requests = static_cast<int32_t>(requests);
  a.block_table = table.data_ptr<int32_t>();
  a.table_stride = requests > 1 ? table.stride(0) : width;
  a.table_width = static_cast<int32_t>(width);
  a.free_pages = free.const_data_ptr<int32_t>();
  a.n_free = static_cast<int32_t>(free.size(0));
  if (start.defined()) a.free_start = start.const_data_ptr<int32_t>();
  a.page_size = static_cast<int32_t>(page);
  a.num_tokens = static_cast<int32_t>(tokens);
  a.heads_q = static_cast<int32_t>(heads_q);
  a.heads_kv = static_cast<int32_t>(heads_kv);
  a.cu_seqlens = cu.data_ptr<int32_t>();
  a.seqlens_k = lens.data_ptr<int32_t>();
  a.slot_map = slots.data_ptr<int64_t>();
  a.positions = positions.data_ptr<int32_t>();
  a.pages_taken = taken.data_ptr<int32_t>();
  a.work = work.data_ptr<int32_t>();
  a.work_bytes = bytes;
  if (abi.paged_plan(&a, stream_of(table)) != FA2_OK) Py_RETURN_NONE;
  written(table);
  PyObject* result = PyTuple_New(6);
  if (!result) return nullptr;
  const Tensor* parts[6] = {&cu, &lens, &slots, &positions, &taken, &work};
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(*parts[i]));
  return result;
  END_HANDLE_TH_ERRORS
}

bool caches_ok(const Tensor& k, const Tensor& v) {
  return k.is_cuda() && k.dim() == 4 && k.numel() > 0 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() &&
         k.device() == v.device() && dtype_code(k.scalar_type()) >= 0 && k.stride(3) == 1 && v.stride(3) == 1 &&
         page_size_ok(k.size(1)) && k.size(0) <= INT32_MAX;
}
fa2_paged_cache cache_of(const Tensor& x) { return {x.const_data_ptr(), x.stride(0), x.stride(1), x.stride(2)}; }

// (k, v, k_cache, v_cache, slot_map) -> True
PyObject* paged_cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  for (int i = 0; i < 5; ++i)
    if (!is_tensor(args[i])) Py_RETURN_NONE;
  const Tensor &k = tensor(args[0]), &v = tensor(args[1]), &kc = tensor(args[2]), &vc = tensor(args[3]), &slots = tensor(args[4]);
  if (!caches_ok(kc, vc) || k.dim() != 3 || k.sizes() != v.sizes() || k.size(1) != kc.size(2) || k.size(2) != kc.size(3) ||
      k.scalar_type() != kc.scalar_type() || v.scalar_type() != kc.scalar_type() || k.device() != kc.device() ||
      v.device() != kc.device() || k.stride(2) != 1 || v.stride(2) != 1 || k.size(0) > INT32_MAX ||
      !vector_of(slots, at::kLong, k.size(0), kc.device()))
    Py_RETURN_NONE;
  if (at::GradMode::is_enabled() && (k.requires_grad() || v.requires_grad() || kc.requires_grad() || vc.requires_grad()))
    Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(kc.device());
  fa2_paged_write_params a = {};
  a.k = k.const_data_ptr(); a.k_stride_t = k.stride(0); a.k_stride_h = k.stride(1);
  a.v = v.const_data_ptr(); a.v_stride_t = v.stride(0); a.v_stride_h = v.stride(1);
  a.k_cache = cache_of(kc);
  a.v_cache = cache_of(vc);
  a.slot_map = slots.const_data_ptr<int64_t>();
  a.tokens = static_cast<int32_t>(k.size(0));
  a.heads = static_cast<int32_t>(kc.size(2));
  a.head_dim = static_cast<int32_t>(kc.size(3));
  a.pages = static_cast<int32_t>(kc.size(0));
  a.page_size = static_cast<int32_t>(kc.size(1));
  if (abi.paged_cache_write(&a, stream_of(kc)) != FA2_OK) Py_RETURN_NONE;
  written(kc);
  written(vc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, block_table, work, plan's (num_tokens, heads_q, heads_kv, page_size), softmax_scale, softcap,
//  alibi_slopes, out, lse) -> out
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14) Py_RETURN_NONE;
  for (int i = 0; i < 5; ++i)
    if (!is_tensor(args[i])) Py_RETURN_NONE;
  const Tensor &q = tensor(args[0]), &kc = tensor(args[1]), &vc = tensor(args[2]), &table = tensor(args[3]), &work = tensor(args[4]);
  int64_t tokens, heads_q, heads_kv, page;
  double scale, cap;
  Tensor slopes, out, lse;
  if (!integer(args[5], &tokens) || !integer(args[6], &heads_q) || !integer(args[7], &heads_kv) || !integer(args[8], &page) ||
      !optional_tensor(args[11], &slopes) || !optional_tensor(args[12], &out) || !optional_tensor(args[13], &lse))
    Py_RETURN_NONE;
  if (!caches_ok(kc, vc) || q.dim() != 3 || q.size(0) != tokens || q.size(1) != heads_q || q.size(2) != kc.size(3) ||
      kc.size(2) != heads_kv || kc.size(1) != page || q.scalar_type() != kc.scalar_type() || q.device() != kc.device() ||
      work.device() != kc.device() || work.scalar_type() != at::kInt || q.stride(2) != 1)
    Py_RETURN_NONE;
  if (table.device() != kc.device() || table.scalar_type() != at::kInt || table.dim() != 2 || table.numel() == 0 ||
      table.stride(1) != 1)
    Py_RETURN_NONE;
  if (!optional_number(args[9], 1.0 / std::sqrt(static_cast<double>(kc.size(3))), &scale) ||
      !optional_number(args[10], 0.0, &cap) || !softcap_ok(cap))
    Py_RETURN_NONE;
  if (at::GradMode::is_enabled() && (q.requires_grad() || kc.requires_grad() || vc.requires_grad() ||
                                     (out.defined() && out.requires_grad()) || (lse.defined() && lse.requires_grad())))
    Py_RETURN_NONE;
  if (slopes.defined() && (!vector_of(slopes, at::kFloat, heads_q, q.device()) || slopes.requires_grad())) Py_RETURN_NONE;
  if (lse.defined() && (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != tokens || lse.size(1) != heads_q ||
                        lse.device() != q.device() || !lse.is_contiguous()))
    Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(q.device());
  if (!out.defined())
    out = at::empty(q.sizes(), q.options());
  else if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || out.device() != q.device() || out.stride(2) != 1)
    Py_RETURN_NONE;
  fa2_paged_attention_params a = {};
  a.q = q.const_data_ptr(); a.q_stride_t = q.stride(0); a.q_stride_h = q.stride(1);
  a.o = out.data_ptr(); a.o_stride_t = out.stride(0); a.o_stride_h = out.stride(1);
  if (lse.defined()) a.lse = lse.data_ptr<float>();
  a.k_cache = cache_of(kc);
  a.v_cache = cache_of(vc);
  a.tokens = static_cast<int32_t>(tokens);
  a.heads_q = static_cast<int32_t>(heads_q);
  a.heads_kv = static_cast<int32_t>(heads_kv);
  a.head_dim = static_cast<int32_t>(kc.size(3));
  a.dtype = dtype_code(q.scalar_type());
  a.pages = static_cast<int32_t>(kc.size(0));
  a.page_size = static_cast<int32_t>(page);
  a.block_table = table.const_data_ptr<int32_t>();
  a.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  a.table_width = static_cast<int32_t>(table.size(1));
  a.requests = static_cast<int32_t>(table.size(0));
  a.work = work.const_data_ptr<int32_t>();
  a.softmax_scale = static_cast<float>(scale);
  a.softcap = static_cast<float>(cap);
  if (slopes.defined()) a.alibi_slopes = slopes.const_data_ptr<float>();
  const size_t bytes = abi.paged_workspace_bytes(a.head_dim);
  if (bytes == 0) Py_RETURN_NONE;
  const Tensor workspace = bytes_like(q, bytes);
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = bytes;
  if (abi.paged_attention(&a, stream_of(q)) != FA2_OK) Py_RETURN_NONE;
  written(out);
  if (lse.defined()) written(lse);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (address, address, ...): the functions of Abi in order.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kAbiFunctions) {
    PyErr_Format(PyExc_ValueError, "%d addresses are wanted", kAbiFunctions);
    return nullptr;
  }
  void* addresses[kAbiFunctions];
  for (int i = 0; i < kAbiFunctions; ++i) {
    addresses[i] = PyLong_AsVoidPtr(args[i]);
    if (!addresses[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is null");
      return nullptr;
    }
  }
  std::memcpy(&abi, addresses, sizeof(abi));
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {{"bind", fast<bind>(), METH_FASTCALL, nullptr},
                         {"scored_flash_attention", fast<scored_flash_attention>(), METH_FASTCALL, nullptr},
                         {"check_capture", fast<check_capture>(), METH_FASTCALL, nullptr},
                         {"paged_step_plan", fast<paged_step_plan>(), METH_FASTCALL, nullptr},
                         {"paged_cache_write", fast<paged_cache_write>(), METH_FASTCALL, nullptr},
                         {"paged_attention", fast<paged_attention>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fa2_native", "torch tensors to the C ABI of fa2_b200_lm.h", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fa2_native() { return PyModule_Create(&module); }
