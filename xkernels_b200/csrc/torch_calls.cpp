// The call path of the small ops (router, routing sort, top-k reduce, losses and gradients) from Python: checks, output
// tensors and the C-ABI call in one native function.
//
// These ops often take 3 to 10 us on the device and a call through Python and ctypes 9 to 18 us of host time, which therefore
// was what a caller waited for.  A function here serves the plain call - ordinary contiguous CUDA tensors on the current
// device, arguments of the plain Python types, no dispatch or function mode - and returns None for any other, which the
// Python form then handles or refuses as it always has.  A failing C call returns its status.
// Time of a call in a loop of calls: topk_softmax (one row) 11.3 -> 5.9 us, moe_align_block_size (131072 slots) 17.9 -> 10.4,
// moe_sum_reduce (one token) 8.9 -> 3.9; the losses and gradients 12 to 25 -> 4 to 5.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/xkb200.h"

namespace {

decltype(&xkb_topk_softmax) g_topk_softmax;
decltype(&xkb_moe_align_block_size) g_align;
decltype(&xkb_moe_align_workspace_bytes) g_align_bytes;
decltype(&xkb_moe_sum_reduce) g_sum_reduce;
decltype(&xkb_token_logprobs) g_logprobs;
decltype(&xkb_token_logprobs_backward) g_logprobs_grad;
decltype(&xkb_moe_balance_loss) g_balance;
decltype(&xkb_moe_balance_loss_workspace_bytes) g_balance_bytes;
decltype(&xkb_moe_router_backward) g_router_grad;
decltype(&xkb_moe_sum_reduce_backward) g_sum_reduce_grad;

bool modes_active() {
  return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set();
}

// The tensor behind `obj` if it is a plain one, else nullptr.
const at::Tensor* plain(PyObject* obj, bool contiguous = true) {
  if (!THPVariable_CheckExact(obj)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || (contiguous && !t.is_contiguous()) || t.is_neg() ||
      t.is_conj() || t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                                              c10::DispatchKey::FuncTorchGradWrapper,
                                                              c10::DispatchKey::Functionalize})) ||
      t.get_device() != c10::cuda::current_device())
    return nullptr;
  return &t;
}

int code_of(at::ScalarType t) {   // -1: not a type of the library
  return t == at::kBFloat16 ? XKB_BF16 : t == at::kFloat ? XKB_F32 : t == at::kHalf ? XKB_F16 : -1;
}

bool plain_int(PyObject* obj, int64_t* value) {
  if (!PyLong_CheckExact(obj)) return false;
  int overflow = 0;
  *value = PyLong_AsLongLongAndOverflow(obj, &overflow);
  return overflow == 0;
}

// None, or a plain tensor of this type and shape (shape[1] < 0: a vector); false for anything else
bool optional(PyObject* obj, at::ScalarType type, int64_t rows, int64_t cols, const at::Tensor** out) {
  *out = nullptr;
  if (obj == Py_None) return true;
  const at::Tensor* t = plain(obj);
  if (t == nullptr || t->scalar_type() != type || t->dim() != (cols < 0 ? 1 : 2) || t->size(0) != rows ||
      (cols >= 0 && t->size(1) != cols))
    return false;
  *out = t;
  return true;
}
// the same with one element, whatever the dimensions
bool optional_scalar(PyObject* obj, at::ScalarType type, const at::Tensor** out) {
  *out = nullptr;
  if (obj == Py_None) return true;
  const at::Tensor* t = plain(obj);
  if (t == nullptr || t->scalar_type() != type || t->numel() != 1) return false;
  *out = t;
  return true;
}
template <typename T> const T* data(const at::Tensor* t) { return t == nullptr ? nullptr : static_cast<const T*>(t->const_data_ptr()); }

// A head's logits [M, V], rows of neighbouring columns, and the tokens [M] given for them.
const at::Tensor* head(PyObject* obj) {
  const at::Tensor* t = plain(obj, false);
  return t != nullptr && t->dim() == 2 && t->size(1) >= 1 && t->stride(1) == 1 && code_of(t->scalar_type()) >= 0 ? t : nullptr;
}
bool tokens_of(PyObject* obj, int64_t M, const at::Tensor** out) {
  return optional(obj, at::kLong, M, -1, out) || optional(obj, at::kInt, M, -1, out);
}
const at::Tensor* gating(PyObject* obj) {
  const at::Tensor* t = plain(obj);
  return t != nullptr && t->dim() == 2 && t->size(1) >= 1 && t->size(1) <= 1024 && code_of(t->scalar_type()) >= 0 ? t : nullptr;
}
const at::Tensor* chosen(PyObject* obj, int64_t M) {
  const at::Tensor* t = plain(obj);
  return t != nullptr && t->dim() == 2 && t->size(0) == M && t->size(1) <= 0x7fffffff && t->scalar_type() == at::kInt ? t : nullptr;
}
bool mask_of(PyObject* obj, int64_t M, const at::Tensor** out) {
  return optional(obj, at::kBool, M, -1, out) || optional(obj, at::kByte, M, -1, out);
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// a tuple of new references (nullptr: an error is set)
template <typename... Objects>
PyObject* tuple_of(Objects... objects) {
  PyObject* const all[] = {objects...};
  PyObject* t = PyTuple_New(sizeof...(objects));
  bool ok = t != nullptr;
  for (size_t i = 0; i < sizeof...(objects); ++i) {
    ok = ok && all[i] != nullptr;
    if (t != nullptr) PyTuple_SET_ITEM(t, (Py_ssize_t)i, all[i]);
    else Py_XDECREF(all[i]);
  }
  if (!ok) { Py_XDECREF(t); return nullptr; }
  return t;
}

// topk_softmax(gating [M, E], topk, renormalize) -> (weights, ids)
PyObject* topk_softmax(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t topk;
  if (n != 3 || modes_active() || !plain_int(args[1], &topk) || !PyBool_Check(args[2])) Py_RETURN_NONE;
  const at::Tensor* g = plain(args[0]);
  if (g == nullptr || g->dim() != 2 || code_of(g->scalar_type()) < 0) Py_RETURN_NONE;
  const int64_t M = g->size(0), E = g->size(1);
  if (topk < 1 || topk > E || E > 0x7fffffff) Py_RETURN_NONE;
  at::Tensor w = at::empty({M, topk}, g->options().dtype(at::kFloat));
  at::Tensor ids = at::empty({M, topk}, g->options().dtype(at::kInt));
  const int code = code_of(g->scalar_type()), renorm = args[2] == Py_True;
  void* const stream = stream_of(*g);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_topk_softmax(g->const_data_ptr(), code, static_cast<float*>(w.mutable_data_ptr()),
                          static_cast<int32_t*>(ids.mutable_data_ptr()), M, (int)E, (int)topk, renorm, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return tuple_of(THPVariable_Wrap(std::move(w)), THPVariable_Wrap(std::move(ids)));
  END_HANDLE_TH_ERRORS
}

// moe_align_block_size(topk_ids, block_size, num_experts) -> (sorted_ids, expert_ids, num_post), untruncated
PyObject* moe_align_block_size(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t block, E;
  if (n != 3 || modes_active() || !plain_int(args[1], &block) || !plain_int(args[2], &E)) Py_RETURN_NONE;
  const at::Tensor* ids = plain(args[0]);
  if (ids == nullptr || ids->scalar_type() != at::kInt) Py_RETURN_NONE;
  const int64_t numel = ids->numel();
  if (block < 1 || block > (1 << 20) || E < 0 || E > 1024 || numel >= (1ll << 30)) Py_RETURN_NONE;
  const int64_t max_pad = numel + (E + 1) * (block - 1), max_blocks = (max_pad + block - 1) / block;
  if (max_blocks == 0) Py_RETURN_NONE;
  const at::TensorOptions opt = ids->options();
  at::Tensor sorted = at::empty({max_pad}, opt), experts = at::empty({max_blocks}, opt), post = at::empty({1}, opt), ws;
  void* ws_ptr = nullptr;
  int64_t ws_bytes = 0;
  if (numel > 8192) {   // up to there the sort takes no scratch memory
    ws_bytes = (g_align_bytes(numel, (int)E) + 3) / 4 * 4;
    ws = at::empty({ws_bytes / 4}, opt);
    ws_ptr = ws.mutable_data_ptr();
  }
  void* const stream = stream_of(*ids);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_align(static_cast<const int32_t*>(ids->const_data_ptr()), numel, (int)E, (int)block, nullptr, 0,
                   static_cast<int32_t*>(sorted.mutable_data_ptr()), static_cast<int32_t*>(experts.mutable_data_ptr()),
                   static_cast<int32_t*>(post.mutable_data_ptr()), nullptr, ws_ptr, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return tuple_of(THPVariable_Wrap(std::move(sorted)), THPVariable_Wrap(std::move(experts)),
                  THPVariable_Wrap(std::move(post)));
  END_HANDLE_TH_ERRORS
}

// moe_sum_reduce(y [M, top_k, H], w [M, top_k] or None, routed_scaling_factor) -> [M, H]
PyObject* moe_sum_reduce(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || modes_active() || !PyFloat_CheckExact(args[2])) Py_RETURN_NONE;
  const at::Tensor* y = plain(args[0]);
  if (y == nullptr || y->dim() != 3 || (y->scalar_type() != at::kBFloat16 && y->scalar_type() != at::kFloat)) Py_RETURN_NONE;
  const int64_t M = y->size(0), top_k = y->size(1), H = y->size(2);
  if (top_k > 0x7fffffff) Py_RETURN_NONE;
  const at::Tensor* w = nullptr;
  if (args[1] != Py_None) {
    w = plain(args[1]);
    if (w == nullptr || w->dim() != 2 || w->size(0) != M || w->size(1) != top_k || w->get_device() != y->get_device() ||
        (w->scalar_type() != at::kBFloat16 && w->scalar_type() != at::kFloat))
      Py_RETURN_NONE;
  }
  at::Tensor out = at::empty({M, H}, y->options());
  const int y_code = code_of(y->scalar_type()), w_code = w == nullptr ? XKB_F32 : code_of(w->scalar_type());
  const float factor = (float)PyFloat_AS_DOUBLE(args[2]);
  void* const stream = stream_of(*y);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_sum_reduce(y->const_data_ptr(), y_code, w == nullptr ? nullptr : w->const_data_ptr(), w_code,
                        out.mutable_data_ptr(), y_code, M, (int)top_k, H, factor, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// An uninitialised tensor on the current device, of the allocator that at::empty uses, without the way through the dispatcher.  Host time of
// a call, at::empty / this: moe_sum_reduce_backward (two outputs) 5.2 / 4.5 us, token_logprobs 5.3 / 4.8, its gradient 4.5 / 4.1,
// moe_balance_loss 4.8 / 4.4; moe_router_backward 3.7 either way.
c10::Storage storage_of(int64_t bytes) {
  c10::Allocator* const from = c10::cuda::CUDACachingAllocator::get();
  return c10::Storage(c10::Storage::use_byte_size_t(), bytes, from->allocate(bytes), from, /*resizable=*/true);
}
at::Tensor tensor_on(c10::Storage&& storage, at::ScalarType type, at::IntArrayRef sizes, int64_t offset = 0) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(std::move(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                   c10::scalarTypeToTypeMeta(type));
  impl->set_sizes_contiguous(sizes);
  impl->set_storage_offset(offset);
  return at::Tensor(std::move(impl));
}
at::Tensor fresh(at::ScalarType type, at::IntArrayRef sizes) {
  return tensor_on(storage_of(c10::multiply_integers(sizes) * (int64_t)c10::elementSize(type)), type, sizes);
}

// Several small outputs are pieces of one allocation (an allocation takes as long as a short kernel): ordinary tensors over
// disjoint pieces of one storage, each on 16 bytes.
struct Pieces {
  c10::Storage base;
  int64_t at = 0;
  static int64_t room(int64_t elements) { return (elements * 4 + 15) / 16 * 16; }   // of 4-byte elements
  explicit Pieces(int64_t bytes) : base(storage_of(bytes)) {}
  at::Tensor take(at::ScalarType type, at::IntArrayRef sizes) {   // of 4-byte elements
    at::Tensor t = tensor_on(c10::Storage(base), type, sizes, at / 4);
    at += room(t.numel());
    return t;
  }
};

// token_logprobs(logits [M, V], token_ids [M], top_k) -> (logprobs, entropy, stats, top_logprobs, top_ids)
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t top_k;
  const at::Tensor* ids;
  if (n != 3 || modes_active() || !plain_int(args[2], &top_k)) Py_RETURN_NONE;
  const at::Tensor* x = head(args[0]);
  if (x == nullptr || args[1] == Py_None || !tokens_of(args[1], x->size(0), &ids)) Py_RETURN_NONE;
  const int64_t M = x->size(0), V = x->size(1);
  if (top_k < 0 || top_k > 64 || top_k > V) Py_RETURN_NONE;
  Pieces pieces(2 * Pieces::room(M) + Pieces::room(2 * M) + 2 * Pieces::room(M * top_k));
  at::Tensor lp = pieces.take(at::kFloat, {M}), entropy = pieces.take(at::kFloat, {M}), stats = pieces.take(at::kFloat, {M, 2}),
             top_lp = pieces.take(at::kFloat, {M, top_k}), top_ids = pieces.take(at::kInt, {M, top_k});
  const int code = code_of(x->scalar_type()), ids64 = ids->scalar_type() == at::kLong;
  void* const stream = stream_of(*x);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_logprobs(x->const_data_ptr(), code, x->stride(0), ids->const_data_ptr(), ids64, static_cast<float*>(lp.mutable_data_ptr()),
                      static_cast<float*>(entropy.mutable_data_ptr()), static_cast<float*>(stats.mutable_data_ptr()),
                      static_cast<float*>(top_lp.mutable_data_ptr()), static_cast<int32_t*>(top_ids.mutable_data_ptr()), M, V,
                      (int)top_k, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return tuple_of(THPVariable_Wrap(std::move(lp)), THPVariable_Wrap(std::move(entropy)), THPVariable_Wrap(std::move(stats)),
                  THPVariable_Wrap(std::move(top_lp)), THPVariable_Wrap(std::move(top_ids)));
  END_HANDLE_TH_ERRORS
}

// token_logprobs_backward(logits, token_ids, stats, entropy, grad_logprobs, grad_entropy, top_ids, grad_top_logprobs)
// -> [M, V]; rows that do not start on 16 bytes are the Python form's
PyObject* token_logprobs_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || modes_active() || (args[4] == Py_None && args[5] == Py_None && args[7] == Py_None)) Py_RETURN_NONE;
  const at::Tensor *ids, *stats, *entropy, *g_lp, *g_entropy, *top_ids = nullptr, *g_top = nullptr;
  const at::Tensor* x = head(args[0]);
  if (x == nullptr) Py_RETURN_NONE;
  const int64_t M = x->size(0), V = x->size(1), es = x->element_size();
  if (args[2] == Py_None || !tokens_of(args[1], M, &ids) || !optional(args[2], at::kFloat, M, 2, &stats) ||
      !optional(args[4], at::kFloat, M, -1, &g_lp) || !optional(args[5], at::kFloat, M, -1, &g_entropy) ||
      !optional(args[3], at::kFloat, M, -1, &entropy) || (g_lp != nullptr && ids == nullptr) || (g_entropy != nullptr && entropy == nullptr))
    Py_RETURN_NONE;
  int64_t top_k = 0;
  if (args[7] != Py_None) {
    g_top = plain(args[7]);
    if (g_top == nullptr || g_top->dim() != 2 || g_top->size(0) != M || g_top->size(1) > 64 || g_top->scalar_type() != at::kFloat ||
        args[6] == Py_None || !optional(args[6], at::kInt, M, g_top->size(1), &top_ids))
      Py_RETURN_NONE;
    top_k = g_top->size(1);
  }
  if (reinterpret_cast<uintptr_t>(x->const_data_ptr()) % 16 != 0 || (M > 1 && (x->stride(0) - V) * es % 16 != 0)) Py_RETURN_NONE;
  at::Tensor out = fresh(x->scalar_type(), {M, V});
  const int code = code_of(x->scalar_type()), ids64 = ids != nullptr && ids->scalar_type() == at::kLong;
  void* const stream = stream_of(*x);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_logprobs_grad(x->const_data_ptr(), code, x->stride(0), data<void>(ids), ids64, data<float>(stats),
                           g_entropy != nullptr ? data<float>(entropy) : nullptr, data<float>(g_lp), data<float>(g_entropy),
                           top_k != 0 ? data<int32_t>(top_ids) : nullptr, top_k != 0 ? data<float>(g_top) : nullptr, (int)top_k,
                           out.mutable_data_ptr(), V, M, V, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// moe_balance_loss(gating [M, E], topk_ids [M, top_k], token_mask [M] or None) -> (loss, counts, mean_probs, tokens)
PyObject* moe_balance_loss(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* mask;
  if (n != 3 || modes_active()) Py_RETURN_NONE;
  const at::Tensor* x = gating(args[0]);
  const at::Tensor* ids = x == nullptr ? nullptr : chosen(args[1], x->size(0));
  if (ids == nullptr || !mask_of(args[2], x->size(0), &mask)) Py_RETURN_NONE;
  const int64_t M = x->size(0), E = x->size(1), ws_bytes = g_balance_bytes(M, (int)E);
  Pieces pieces(2 * Pieces::room(1) + 2 * Pieces::room(E));
  at::Tensor loss = pieces.take(at::kFloat, {}), tokens = pieces.take(at::kInt, {}), counts = pieces.take(at::kInt, {E}),
             mean = pieces.take(at::kFloat, {E}), ws;
  if (ws_bytes > 0) ws = fresh(at::kByte, {ws_bytes});
  const int code = code_of(x->scalar_type()), top_k = (int)ids->size(1);
  void* const stream = stream_of(*x);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_balance(x->const_data_ptr(), code, data<int32_t>(ids), data<uint8_t>(mask), static_cast<float*>(loss.mutable_data_ptr()),
                     static_cast<int32_t*>(counts.mutable_data_ptr()), static_cast<float*>(mean.mutable_data_ptr()),
                     static_cast<int32_t*>(tokens.mutable_data_ptr()), M, (int)E, top_k, ws.defined() ? ws.mutable_data_ptr() : nullptr, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return tuple_of(THPVariable_Wrap(std::move(loss)), THPVariable_Wrap(std::move(counts)), THPVariable_Wrap(std::move(mean)),
                  THPVariable_Wrap(std::move(tokens)));
  END_HANDLE_TH_ERRORS
}

// moe_router_backward(gating, topk_ids, grad_weights, renormalize, counts, tokens, grad_loss, token_mask) -> [M, E]
PyObject* moe_router_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *g_w, *counts, *tokens, *g_loss, *mask;
  if (n != 8 || modes_active() || !PyBool_Check(args[3]) || (args[2] == Py_None && args[4] == Py_None)) Py_RETURN_NONE;
  const at::Tensor* x = gating(args[0]);
  const at::Tensor* ids = x == nullptr ? nullptr : chosen(args[1], x->size(0));
  if (ids == nullptr) Py_RETURN_NONE;
  const int64_t M = x->size(0), E = x->size(1);
  float scale = 1.f;
  PyObject* loss = args[6];
  if (PyFloat_CheckExact(loss)) {
    scale = (float)PyFloat_AS_DOUBLE(loss);
    loss = Py_None;
  }
  if (!optional(args[2], at::kFloat, M, ids->size(1), &g_w) || !optional(args[4], at::kInt, E, -1, &counts) ||
      !optional_scalar(args[5], at::kInt, &tokens) || !optional_scalar(loss, at::kFloat, &g_loss) || !mask_of(args[7], M, &mask) ||
      (counts == nullptr && (args[5] != Py_None || args[6] != Py_None)))
    Py_RETURN_NONE;
  at::Tensor out = fresh(x->scalar_type(), {M, E});
  const int code = code_of(x->scalar_type()), renorm = args[3] == Py_True, top_k = (int)ids->size(1);
  void* const stream = stream_of(*x);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_router_grad(x->const_data_ptr(), code, data<int32_t>(ids), data<float>(g_w), renorm, data<int32_t>(counts),
                         data<int32_t>(tokens), data<float>(g_loss), scale, data<uint8_t>(mask), out.mutable_data_ptr(), M, (int)E,
                         top_k, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// moe_sum_reduce_backward(grad_out [M, H], y [M, top_k, H], w or None, factor, need_grad_y, need_grad_w) -> (grad_y, grad_w)
PyObject* moe_sum_reduce_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || modes_active() || !PyFloat_CheckExact(args[3]) || !PyBool_Check(args[4]) || !PyBool_Check(args[5])) Py_RETURN_NONE;
  const at::Tensor *y = plain(args[1]), *w = nullptr, *go;
  if (y == nullptr || y->dim() != 3 || (y->scalar_type() != at::kBFloat16 && y->scalar_type() != at::kFloat)) Py_RETURN_NONE;
  const int64_t M = y->size(0), top_k = y->size(1), H = y->size(2);
  if (args[0] == Py_None || !optional(args[0], y->scalar_type(), M, H, &go) || top_k > 0x7fffffff ||
      !(optional(args[2], at::kFloat, M, top_k, &w) || optional(args[2], at::kBFloat16, M, top_k, &w)))
    Py_RETURN_NONE;
  const bool need_y = args[4] == Py_True, need_w = args[5] == Py_True && w != nullptr;
  at::Tensor gy, gw;
  if (need_y) gy = fresh(y->scalar_type(), {M, top_k, H});
  if (need_w) gw = fresh(w->scalar_type(), {M, top_k});
  const int code = code_of(y->scalar_type()), w_code = w == nullptr ? XKB_F32 : code_of(w->scalar_type());
  const float factor = (float)PyFloat_AS_DOUBLE(args[3]);
  void* const stream = stream_of(*y);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_sum_reduce_grad(go->const_data_ptr(), code, need_w ? y->const_data_ptr() : nullptr, data<void>(w), w_code,
                             need_y ? gy.mutable_data_ptr() : nullptr, need_w ? gw.mutable_data_ptr() : nullptr, M, (int)top_k, H,
                             factor, stream);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(status);
  PyObject* a = need_y ? THPVariable_Wrap(std::move(gy)) : Py_NewRef(Py_None);
  PyObject* b = need_w ? THPVariable_Wrap(std::move(gw)) : Py_NewRef(Py_None);
  return tuple_of(a, b);
  END_HANDLE_TH_ERRORS
}

// bind(...): the library's functions, as addresses, in the order of the pointers above
constexpr Py_ssize_t kFunctions = 10;
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kFunctions) { PyErr_SetString(PyExc_TypeError, "bind: another number of addresses expected"); return nullptr; }
  void* p[kFunctions];
  for (Py_ssize_t i = 0; i < kFunctions; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
      return nullptr;
    }
  }
  g_topk_softmax = reinterpret_cast<decltype(g_topk_softmax)>(p[0]);
  g_align = reinterpret_cast<decltype(g_align)>(p[1]);
  g_align_bytes = reinterpret_cast<decltype(g_align_bytes)>(p[2]);
  g_sum_reduce = reinterpret_cast<decltype(g_sum_reduce)>(p[3]);
  g_logprobs = reinterpret_cast<decltype(g_logprobs)>(p[4]);
  g_logprobs_grad = reinterpret_cast<decltype(g_logprobs_grad)>(p[5]);
  g_balance = reinterpret_cast<decltype(g_balance)>(p[6]);
  g_balance_bytes = reinterpret_cast<decltype(g_balance_bytes)>(p[7]);
  g_router_grad = reinterpret_cast<decltype(g_router_grad)>(p[8]);
  g_sum_reduce_grad = reinterpret_cast<decltype(g_sum_reduce_grad)>(p[9]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {method<topk_softmax>("topk_softmax"), method<moe_align_block_size>("moe_align_block_size"),
                           method<moe_sum_reduce>("moe_sum_reduce"), method<token_logprobs>("token_logprobs"),
                           method<token_logprobs_backward>("token_logprobs_backward"), method<moe_balance_loss>("moe_balance_loss"),
                           method<moe_router_backward>("moe_router_backward"),
                           method<moe_sum_reduce_backward>("moe_sum_reduce_backward"), method<bind>("bind"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls() { return PyModule_Create(&g_module); }
