// Host side of the calls that a decode step makes, in native code: argument checks, output allocation, stream
// and device lookup and the library call.  In Python the same steps took 12 to 20 us a call, several times the
// kernels of a small linear.  Every function returns None when it does not take the call (a dtype, shape or
// alignment of another path, tensors on different devices, a library error): the Python wrappers then go on
// to that path or raise the error.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/gemq_b200.h"

namespace {

using at::Tensor;

PyObject* none() { Py_RETURN_NONE; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

const Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

void* stream_of(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

Tensor empty_cuda(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) {
  return at::empty(sizes, at::TensorOptions().dtype(t).device(like.device()));
}

// plain(*args) -> whether the call is one that nobody but its caller looks at: kernels/_ops.py, plain_call, which asks
// here first.  A default device is a function mode: False, the Python form tells it from others.
PyObject* plain(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const auto& tls = c10::impl::tls_local_dispatch_key_set().included_;
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
      tls.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || torch::jit::tracer::isTracing())
    Py_RETURN_FALSE;
  const bool grad = c10::GradMode::is_enabled();
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_Check(a[i])) continue;
    const Tensor* t = tensor(a[i]);
    if (!t || (grad && t->requires_grad()) || t->_fw_grad(0).defined()) Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
}

// written(tensor) -> True: a kernel has written to it, which autograd is to know (torch.autograd.graph.increment_version, 0.3 us less).
PyObject* written(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1 || !THPVariable_Check(a[0])) return none();
  const Tensor& t = THPVariable_Unpack(a[0]);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  Py_RETURN_TRUE;
}

// linear(x, w_q, scales, zeros, nbits, group_size, bias | None, err_word_ptr, mode)
// x [..., K] fp16 / bf16 -> [..., N] of the same type.  mode: the caller's contract.
enum { kLayer = 0,      // any leading dimensions
       kRowsOp = 1,     // 2-D fp16
       kOneRowOp = 2,   // [1, K] fp16
       kGemmOp = 3 };   // 2-D; below 32 rows fp16
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) { PyErr_SetString(PyExc_TypeError, "linear takes 9 arguments"); return nullptr; }
  const Tensor *x = tensor(a[0]), *w = tensor(a[1]), *s = tensor(a[2]), *z = tensor(a[3]);
  if (!x || !w || !s || !z) return none();
  const Tensor* bias = nullptr;
  if (a[6] != Py_None && !(bias = tensor(a[6]))) return none();
  const long nbits = PyLong_AsLong(a[4]), G = PyLong_AsLong(a[5]);
  int32_t* err = static_cast<int32_t*>(PyLong_AsVoidPtr(a[7]));
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  const long mode = PyLong_AsLong(a[8]);
  if (!err || nbits < 1 || nbits > 4 || G != 128 || x->dim() < 1 || w->dim() != 2 || s->dim() != 2 || z->dim() != 2) return none();
  if (!x->is_cuda() || !half_type(*x) || (mode != kLayer && x->dim() != 2)) return none();
  const int64_t K = x->size(-1), N = w->size(1), eps = 32 / nbits;
  if (K <= 0 || K % 128 || K > 32768 || N <= 0 || N % 32 || x->numel() == 0) return none();
  const int64_t M = x->numel() / K;
  if (M > (1 << 30) || (mode == kOneRowOp && M != 1)) return none();
  if (M == 1 && x->scalar_type() == at::kHalf && gemq_one_row_streams(static_cast<int>(N), static_cast<int>(K))) return none();
  const bool gemm = mode == kLayer ? gemq_linear_takes_gemm(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(nbits))
                                   : mode == kGemmOp && M >= 32;
  if (mode != kLayer && !gemm && x->scalar_type() != at::kHalf) return none();
  const auto dev = x->device();
  if (w->scalar_type() != at::kInt || w->size(0) != (K + eps - 1) / eps || !w->is_contiguous() || w->device() != dev) return none();
  for (const Tensor* m : {s, z})
    if (m->scalar_type() != at::kHalf || m->size(0) != K / 128 || m->size(1) != N || !m->is_contiguous() || m->device() != dev)
      return none();
  // only what works on rows of one pitch; other strides are made contiguous by the Python path
  int64_t ldx = K;
  if (x->dim() == 2) {
    if (x->stride(1) != 1) return none();
    ldx = x->stride(0);
  } else if (!x->is_contiguous()) {
    return none();
  }
  if (ldx < K || ldx > (1 << 30)) { if (M > 1) return none(); ldx = K; }
  const void* wp = w->data_ptr();
  if (!aligned16(wp) || !aligned16(s->data_ptr()) || !aligned16(z->data_ptr())) return none();
  const bool bf = x->scalar_type() == at::kBFloat16;
  Tensor b;
  if (bias) {
    if (bias->dim() != 1 || bias->size(0) != N) return none();
    b = bias->scalar_type() == x->scalar_type() && bias->device() == dev && bias->is_contiguous()
            ? *bias : bias->to(dev, x->scalar_type()).contiguous();
  }
  c10::cuda::CUDAGuard guard(dev);
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = N;
  Tensor y = empty_cuda(shape, x->scalar_type(), *x);
  const void* bp = bias ? b.data_ptr() : nullptr;
  int rc;
  if (gemm) {
    if (ldx != K || !aligned16(x->data_ptr())) return none();
    const size_t parts = gemq_linear_gemm_scratch_bytes(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(nbits));
    Tensor scratch;
    if (parts) scratch = empty_cuda({static_cast<int64_t>(parts / 4)}, at::kFloat, *x);
    rc = gemq_linear_gemm(x->data_ptr(), nullptr, static_cast<const int32_t*>(wp), s->data_ptr(), z->data_ptr(), nullptr, nullptr,
                          nullptr, static_cast<int>(nbits), bp, y.data_ptr(), static_cast<int>(M), static_cast<int>(N),
                          static_cast<int>(K), 128, bf, err, parts ? scratch.data_ptr() : nullptr, parts, stream_of(*x));
    if (rc) return none();
  } else {
    rc = gemq_linear_rows(x->data_ptr(), static_cast<int>(ldx), bf, static_cast<const int32_t*>(wp), s->data_ptr(), z->data_ptr(),
                          bp, y.data_ptr(), static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(nbits),
                          128, err, stream_of(*x));
    if (rc) return none();
  }
  return THPVariable_Wrap(std::move(y));
}

// moe_decode(layer_ptr, x, scratch, hidden, top_k, route_mode): every row of x [..., hidden], fp16 or bf16 -> out like x
PyObject* moe_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) { PyErr_SetString(PyExc_TypeError, "moe_decode takes 6 arguments"); return nullptr; }
  const auto* L = static_cast<const gemq_moe_layer_t*>(PyLong_AsVoidPtr(a[0]));
  const Tensor *x = tensor(a[1]), *sc = tensor(a[2]);
  const long D = PyLong_AsLong(a[3]), A = PyLong_AsLong(a[4]), mode = PyLong_AsLong(a[5]);
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  if (!L || !x || !sc || !x->is_cuda() || !half_type(*x) || x->dim() < 1 || x->size(-1) != D || x->numel() == 0) return none();
  if (!sc->is_cuda() || sc->device() != x->device()) return none();
  c10::cuda::CUDAGuard guard(x->device());
  const bool bf = x->scalar_type() == at::kBFloat16;
  Tensor xh = (bf ? x->to(at::kHalf) : *x).contiguous();
  const int64_t T = x->numel() / D;
  Tensor out = empty_cuda(x->sizes(), at::kHalf, *x);
  // routing results: not returned, but part of the call's contract
  Tensor r = empty_cuda({T * A * 10}, at::kByte, *x);
  auto* idx = static_cast<int64_t*>(r.data_ptr());
  void* w = static_cast<char*>(r.data_ptr()) + T * A * 8;
  const int rc = gemq_moe_decode(L, xh.data_ptr(), out.data_ptr(), idx, w, static_cast<int>(T), 1, static_cast<int>(mode),
                                 sc->data_ptr(), static_cast<size_t>(sc->numel()), stream_of(*x));
  if (rc) return none();
  return THPVariable_Wrap(bf ? out.to(at::kBFloat16) : out);
}

// moe_prefill(layer_ptr, x, scratch | None, hidden, top_k, n_experts, route_mode, want_logits)
// -> (out, logits | None), logits [T, E] of x's type; None also when the scratch is too small, and under capture
// (the block then keeps the scratch for the graph).
PyObject* moe_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) { PyErr_SetString(PyExc_TypeError, "moe_prefill takes 8 arguments"); return nullptr; }
  const auto* L = static_cast<const gemq_moe_layer_t*>(PyLong_AsVoidPtr(a[0]));
  const Tensor *x = tensor(a[1]), *sc = tensor(a[2]);
  const long D = PyLong_AsLong(a[3]), A = PyLong_AsLong(a[4]), E = PyLong_AsLong(a[5]), mode = PyLong_AsLong(a[6]);
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  const bool want = a[7] == Py_True;
  if (!L || !x || !sc || !x->is_cuda() || !half_type(*x) || x->dim() < 1 || x->size(-1) != D || x->numel() == 0) return none();
  if (!x->is_contiguous() || !aligned16(x->data_ptr()) || sc->device() != x->device()) return none();
  const int64_t T = x->numel() / D;
  if (T > (1 << 24) || gemq_moe_prefill_scratch_bytes(L, static_cast<int>(T)) > static_cast<size_t>(sc->numel())) return none();
  c10::cuda::CUDAGuard guard(x->device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return none();
  Tensor out = empty_cuda(x->sizes(), x->scalar_type(), *x);
  Tensor logits;
  if (want) logits = empty_cuda({T, E}, x->scalar_type(), *x);
  Tensor r = empty_cuda({T * A * 10}, at::kByte, *x);
  auto* idx = static_cast<int64_t*>(r.data_ptr());
  void* w = static_cast<char*>(r.data_ptr()) + T * A * 8;
  const int rc = gemq_moe_prefill(L, x->data_ptr(), out.data_ptr(), idx, w, want ? logits.data_ptr() : nullptr,
                                  static_cast<int>(T), 2, static_cast<int>(mode), x->scalar_type() == at::kBFloat16, sc->data_ptr(),
                                  static_cast<size_t>(sc->numel()), stream_of(*x));
  if (rc) return none();
  PyObject* o = THPVariable_Wrap(std::move(out));
  PyObject* l = want ? THPVariable_Wrap(std::move(logits)) : none();
  PyObject* t = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return t;
}

// ---- latent attention: the calls of kernels/latent_attention.py where every check holds ----------------
// Strides of all but the last dimension, 0 where there is one of it; false where rows are not contiguous or off 16-byte boundaries.
bool row_strides(const Tensor& t, int64_t* s) {
  const int64_t n = t.dim() - 1;
  if (t.stride(n) != 1 || !aligned16(t.data_ptr())) return false;
  for (int64_t i = 0; i < n; ++i) {
    s[i] = t.size(i) == 1 ? 0 : t.stride(i);
    if (s[i] & 7) return false;
  }
  return true;
}
bool ints(const Tensor* t, at::ScalarType type, const c10::Device& dev, int64_t d0, int64_t d1 = -1) {
  return t && t->scalar_type() == type && t->device() == dev && t->is_contiguous() && t->dim() == (d1 < 0 ? 1 : 2) && t->size(0) == d0 &&
         (d1 < 0 || t->size(1) == d1);
}
// A cache [pages, page, rank + 64] -> rank, or 0
int64_t cache_rank(const Tensor* c, const Tensor& like, int64_t* page_stride) {
  if (!c || c->dim() != 3 || c->scalar_type() != like.scalar_type() || c->device() != like.device() || !half_type(*c)) return 0;
  const int64_t pages = c->size(0), page = c->size(1), rank = c->size(2) - 64;
  int64_t s[2];
  if (rank < 128 || rank > 512 || rank % 128 || pages <= 0 || pages * page >= (int64_t(1) << 31) || c->stride(1) != c->size(2)) return 0;
  if (pages > 1 && c->stride(0) < page * c->size(2)) return 0;
  if (!(page == 16 || page == 32 || (page > 0 && page % 64 == 0)) || !row_strides(*c, s)) return 0;
  *page_stride = s[0];
  return rank;
}
PyObject* pair(Tensor a, Tensor b) {
  PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b));
  PyObject* t = PyTuple_Pack(2, x, y);
  Py_DECREF(x);
  Py_DECREF(y);
  return t;
}
bool all_on_gpu(std::initializer_list<const Tensor*> v) {
  for (const Tensor* t : v)
    if (!t || !t->is_cuda() || t->device() != (*v.begin())->device()) return false;
  return true;
}

// latent_decode(err_word_ptr, q_latent, q_rope, cache, table, lens, scale[, prefix_table, prefix_lens, starts])
PyObject* latent_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7 && n != 10) return none();
  auto* err = static_cast<int32_t*>(PyLong_AsVoidPtr(a[0]));
  const Tensor *ql = tensor(a[1]), *qr = tensor(a[2]), *c = tensor(a[3]), *tb = tensor(a[4]), *ln = tensor(a[5]);
  const double scale = PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  if (!err || !all_on_gpu({ql, qr, c, tb, ln}) || ql->dim() != 4 || qr->dim() != 4 || tb->dim() != 2) return none();
  gemq_latent_decode_t A = {};
  const int64_t rank = cache_rank(c, *ql, &A.page_stride), B = ql->size(0), S = ql->size(1), H = ql->size(2);
  if (!rank || ql->size(3) != rank || B <= 0 || S <= 0 || H <= 0 || qr->size(0) != B || qr->size(1) != S || qr->size(2) != H || qr->size(3) != 64 ||
      qr->scalar_type() != ql->scalar_type() || B * S * H > (1 << 28))
    return none();
  const auto dev = ql->device();
  if (!row_strides(*ql, A.q_latent_stride) || !row_strides(*qr, A.q_rope_stride)) return none();
  if (!ints(tb, at::kInt, dev, B, tb->size(1)) || tb->size(1) <= 0 || !ints(ln, at::kInt, dev, B)) return none();
  if (n == 10) {
    const Tensor *pt = tensor(a[7]), *pl = tensor(a[8]), *st = tensor(a[9]);
    if (!pt || pt->dim() != 2 || pt->size(0) <= 0 || !ints(pt, at::kInt, dev, pt->size(0), pt->size(1)) || !ints(pl, at::kInt, dev, pt->size(0)) ||
        !ints(st, at::kInt, dev, pt->size(0) + 1) || pt->size(1) <= 0 || pt->size(0) > (1 << 24))
      return none();
    A.prefix_table = pt->data_ptr<int32_t>();
    A.prefix_pitch = static_cast<int32_t>(pt->size(1));
    A.prefix_lens = pl->data_ptr<int32_t>();
    A.starts = st->data_ptr<int32_t>();
    A.groups = static_cast<int32_t>(pt->size(0));
  }
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = empty_cuda({B, S, H, rank}, ql->scalar_type(), *ql), lse = empty_cuda({B, S, H}, at::kFloat, *ql);
  A.q_latent = ql->data_ptr();
  A.q_rope = qr->data_ptr();
  A.cache = c->data_ptr();
  A.n_pages = static_cast<int32_t>(c->size(0));
  A.page_size = static_cast<int32_t>(c->size(1));
  A.table = tb->data_ptr<int32_t>();
  A.table_pitch = static_cast<int32_t>(tb->size(1));
  A.lens = ln->data_ptr<int32_t>();
  A.batch = static_cast<int32_t>(B);
  A.steps = static_cast<int32_t>(S);
  A.heads = static_cast<int32_t>(H);
  A.rank = static_cast<int32_t>(rank);
  A.scale = static_cast<float>(scale);
  A.is_bf16 = ql->scalar_type() == at::kBFloat16;
  A.out = out.data_ptr();
  A.lse = lse.data_ptr<float>();
  A.err = err;
  const size_t bytes = gemq_latent_decode_scratch_bytes(&A);
  if (!bytes) return none();
  Tensor scratch = empty_cuda({static_cast<int64_t>(bytes)}, at::kByte, *ql);
  if (gemq_latent_decode(&A, scratch.data_ptr(), bytes, stream_of(*ql))) return none();
  return pair(std::move(out), std::move(lse));
}

// latent_prefill(err_word_ptr, q_nope, q_rope, kv, k_rope, cu_q, cu_k, scale[, causal])
PyObject* latent_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 && n != 9) return none();
  auto* err = static_cast<int32_t*>(PyLong_AsVoidPtr(a[0]));
  const Tensor *qn = tensor(a[1]), *qr = tensor(a[2]), *kv = tensor(a[3]), *kr = tensor(a[4]), *cq = tensor(a[5]), *ck = tensor(a[6]);
  const double scale = PyFloat_AsDouble(a[7]);
  const int causal = n == 9 ? PyObject_IsTrue(a[8]) : 1;
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  if (!err || !all_on_gpu({qn, qr, kv, kr, cq, ck}) || qn->dim() != 3 || qr->dim() != 3 || kv->dim() != 3 || kr->dim() != 2 || !half_type(*qn))
    return none();
  const int64_t Tq = qn->size(0), H = qn->size(1), Tk = kv->size(0);
  const auto type = qn->scalar_type();
  const auto dev = qn->device();
  if (Tq <= 0 || Tk <= 0 || H <= 0 || qn->size(2) != 128 || qr->size(0) != Tq || qr->size(1) != H || qr->size(2) != 64 || kv->size(1) != H ||
      kv->size(2) != 256 || kr->size(0) != Tk || kr->size(1) != 64 || qr->scalar_type() != type || kv->scalar_type() != type ||
      kr->scalar_type() != type || Tq >= (int64_t(1) << 31) || Tk >= (int64_t(1) << 31))
    return none();
  if (cq->dim() != 1 || cq->size(0) < 1 || !ints(cq, at::kInt, dev, cq->size(0)) || !ints(ck, at::kInt, dev, cq->size(0))) return none();
  gemq_latent_prefill_t A = {};
  if (!row_strides(*qn, A.q_nope_stride) || !row_strides(*qr, A.q_rope_stride) || !row_strides(*kv, A.kv_stride) ||
      !row_strides(*kr, &A.k_rope_stride))
    return none();
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = empty_cuda({Tq, H, 128}, type, *qn), lse = empty_cuda({Tq, H}, at::kFloat, *qn);
  A.q_nope = qn->data_ptr();
  A.q_rope = qr->data_ptr();
  A.kv = kv->data_ptr();
  A.k_rope = kr->data_ptr();
  A.cu_q = cq->data_ptr<int32_t>();
  A.cu_k = ck->data_ptr<int32_t>();
  A.batch = static_cast<int32_t>(cq->size(0) - 1);
  A.q_rows = static_cast<int32_t>(Tq);
  A.k_rows = static_cast<int32_t>(Tk);
  A.heads = static_cast<int32_t>(H);
  A.causal = causal;
  A.scale = static_cast<float>(scale);
  A.is_bf16 = type == at::kBFloat16;
  A.out = out.data_ptr();
  A.lse = lse.data_ptr<float>();
  A.err = err;
  if (gemq_latent_prefill(&A, stream_of(*qn))) return none();
  return pair(std::move(out), std::move(lse));
}

// latent_append(err_word_ptr, kv, q_rope, norm_weight, eps, inv_freq, positions, slots, cache[, rope_scale])
PyObject* latent_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9 && n != 10) return none();
  auto* err = static_cast<int32_t*>(PyLong_AsVoidPtr(a[0]));
  const Tensor *kv = tensor(a[1]), *q = tensor(a[2]), *w = tensor(a[3]), *f = tensor(a[5]), *pos = tensor(a[6]), *slots = tensor(a[7]),
               *c = tensor(a[8]);
  const double eps = PyFloat_AsDouble(a[4]), scale = n == 10 ? PyFloat_AsDouble(a[9]) : 1.0;
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  if (!err || !all_on_gpu({kv, q, w, f, pos, slots, c}) || kv->dim() != 2 || q->dim() != 3) return none();
  int64_t page_stride = 0, kv_stride = 0, q_stride[2];
  const int64_t rank = cache_rank(c, *kv, &page_stride), T = kv->size(0), H = q->size(1);
  const auto type = kv->scalar_type();
  const auto dev = kv->device();
  if (!rank || T <= 0 || T > (1 << 30) || H <= 0 || kv->size(1) != rank + 64 || q->size(0) != T || q->size(2) != 64 || q->scalar_type() != type)
    return none();
  if (!ints(w, type, dev, rank) || !aligned16(w->data_ptr()) || !ints(f, at::kFloat, dev, 32) || !ints(pos, at::kLong, dev, T) ||
      !ints(slots, at::kLong, dev, T) || !row_strides(*kv, &kv_stride) || !row_strides(*q, q_stride))
    return none();
  c10::cuda::CUDAGuard guard(dev);
  Tensor q_out = empty_cuda({T, H, 64}, type, *kv), rows = empty_cuda({T, rank + 64}, type, *kv);
  if (gemq_latent_append(kv->data_ptr(), kv_stride, q->data_ptr(), q_stride[0], q_stride[1], w->data_ptr(), static_cast<float>(eps),
                         f->data_ptr<float>(), static_cast<float>(scale), pos->data_ptr<int64_t>(), slots->data_ptr<int64_t>(), c->data_ptr(),
                         page_stride, static_cast<int>(c->size(0)), static_cast<int>(c->size(1)), rows.data_ptr(), q_out.data_ptr(),
                         static_cast<int>(T), static_cast<int>(H), static_cast<int>(rank), type == at::kBFloat16, err, stream_of(*kv)))
    return none();
  return pair(std::move(q_out), std::move(rows));
}

// copy_pages(err_word_ptr, cache [layers, pages, ..], src, dst) -> True where it was taken
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) return none();
  auto* err = static_cast<int32_t*>(PyLong_AsVoidPtr(a[0]));
  const Tensor *c = tensor(a[1]), *src = tensor(a[2]), *dst = tensor(a[3]);
  if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
  if (!err || !all_on_gpu({c, src, dst}) || c->dim() < 4 || c->numel() == 0 || src->dim() != 1 || src->size(0) <= 0 || src->size(0) >= (1ll << 31))
    return none();
  const auto dev = c->device();
  if (!ints(src, at::kLong, dev, src->size(0)) || !ints(dst, at::kLong, dev, src->size(0))) return none();
  int64_t bytes = static_cast<int64_t>(c->element_size());
  for (int64_t d = c->dim() - 1; d > 1; --d) {
    if (c->size(d) != 1 && c->stride(d) * static_cast<int64_t>(c->element_size()) != bytes) return none();
    bytes *= c->size(d);
  }
  const int64_t e = static_cast<int64_t>(c->element_size()), ls = c->stride(0) * e, ps = c->stride(1) * e;
  if (((bytes | ls | ps) & 15) || !aligned16(c->data_ptr()) || c->size(0) >= (1ll << 31) || c->size(1) >= (1ll << 31)) return none();
  c10::cuda::CUDAGuard guard(dev);
  if (gemq_copy_pages(c->data_ptr(), ls, ps, static_cast<int>(c->size(0)), static_cast<int>(c->size(1)), bytes, src->data_ptr<int64_t>(),
                      dst->data_ptr<int64_t>(), static_cast<int>(src->size(0)), err, stream_of(*c)))
    return none();
  Py_RETURN_TRUE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(self, a, n);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"plain", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<plain>)), METH_FASTCALL, nullptr},
    {"written", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<written>)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<linear>)), METH_FASTCALL, nullptr},
    {"moe_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<moe_decode>)), METH_FASTCALL, nullptr},
    {"moe_prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<moe_prefill>)), METH_FASTCALL, nullptr},
    {"latent_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<latent_decode>)), METH_FASTCALL, nullptr},
    {"latent_prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<latent_prefill>)), METH_FASTCALL, nullptr},
    {"latent_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<latent_append>)), METH_FASTCALL, nullptr},
    {"copy_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<copy_pages>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
