// The eager host path of the small calls (one linear, one norm, one
// activation): a decode step is bound by what the host does per call, about
// 9 us from Python of which the kernel launch is 3.  Each function here takes
// the module's tensors, makes the checks, allocates the outputs and calls the
// C entry point in one step; whatever is not the plain case (another type,
// layout or device, a tensor subclass, an active mode or transform, graph
// capture, a workspace that must grow, an argument the entry point refuses
// before it launches anything) returns None and the caller takes its Python
// path, which handles it or raises.  An error after a launch raises here: the
// call is never made a second time.  Figures stand at the callers.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <utility>
#include <vector>

#include "kbn_fp8.h"

namespace {

constexpr int64_t kGroup = 128;
constexpr float kQuantEps = 1e-10f;

// Nothing watches or replaces tensor operations on this thread.
bool plain_thread() {
    return !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
           at::impl::PythonTorchFunctionTLS::stack_len() == 0 &&
           !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// A torch.Tensor or Parameter itself (no subclass), strided, on a GPU.
const at::Tensor* plain_tensor(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

bool is(const at::Tensor& t, at::ScalarType type, int64_t dev, int64_t dim) {
    return t.scalar_type() == type && t.get_device() == dev && t.dim() == dim;
}

// The launch stream of device dev, which must be the current one and not be
// capturing a graph.
bool launch_stream(int64_t dev, hipStream_t& st) {
    if (c10::hip::current_device() != dev) return false;
    st = c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream();
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &cs) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return cs == hipStreamCaptureStatusNone;
}

at::Tensor empty_codes(const at::Tensor& like, int64_t rows, int64_t cols) {
    return at::empty({rows, cols}, like.options().dtype(at::kFloat8_e4m3fn).requires_grad(false));
}
at::Tensor empty_scales(const at::Tensor& like, int64_t rows, int64_t groups) {   // column-major
    return at::empty_strided({rows, groups}, {1, rows}, like.options().dtype(at::kFloat).requires_grad(false));
}

// An eager workspace of at least `bytes` for (device, stream), from the dict
// the Python side keeps ({(device, stream): uint8 tensor}); undefined if it
// has none that large.  The caller holds the tensor over its launch: another
// thread may put a larger one in its place once the GIL is released.
at::Tensor kept_workspace(PyObject* bufs, int64_t dev, hipStream_t st, int64_t bytes) {
    PyObject* key = Py_BuildValue("(LL)", (long long)dev, (long long)(intptr_t)st);
    if (!key) {
        PyErr_Clear();
        return {};
    }
    PyObject* buf = PyDict_GetItem(bufs, key);   // borrowed; no exception set
    Py_DECREF(key);
    const at::Tensor* t = buf ? plain_tensor(buf) : nullptr;
    return t && t->numel() >= bytes ? *t : at::Tensor();
}

// No GIL while it lives; taken again on every way out, an exception included
// (guarded below calls into Python).
struct NoGil {
    PyThreadState* s = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(s); }
};

// Failures of the torch calls (out of memory, say) surface from the Python path.
template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

// What a call that ended with `rc` != 0 gives.  1: an argument was refused and
// nothing was launched, so None, and the Python path refuses it too.  Anything
// else comes after a launch (the runtime's last error, which may be another
// call's): the launch may have run, and a fused add + norm run again would add
// twice, so the error is raised as the Python path raises it.
PyObject* failed(int rc, const char* what) {
    if (rc == 1) Py_RETURN_NONE;
    if (PyObject* lib = PyImport_ImportModule("kb_nano_amd._lib")) {
        PyObject* r = PyObject_CallMethod(lib, "check", "is", rc, what);   // raises KbnError
        Py_DECREF(lib);
        Py_XDECREF(r);
    }
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", what, rc);
    return nullptr;
}

// failed(code, name): the rule above, for tests
PyObject* failed_call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    const char* what = n == 2 ? PyUnicode_AsUTF8(args[1]) : nullptr;
    const long rc = what ? PyLong_AsLong(args[0]) : 0;
    if (!what || PyErr_Occurred()) return PyErr_Format(PyExc_TypeError, "failed(code, name)");
    return failed((int)rc, what);
}

// (codes, scales), made before the launch so that nothing but the launch can
// fail after it; empty with the Python error set if it cannot be made.
struct Ref {
    PyObject* p;
    ~Ref() { Py_XDECREF(p); }
    PyObject* take() { return std::exchange(p, nullptr); }
};
PyObject* pair(const at::Tensor& q, const at::Tensor& s) {
    Ref a{THPVariable_Wrap(q)}, b{THPVariable_Wrap(s)};
    return a.p && b.p ? PyTuple_Pack(2, a.p, b.p) : nullptr;
}

// norm(input, weight, eps, residual | None) -> (codes, scales) | None
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const bool add = args[3] != Py_None;
        const at::Tensor *x = plain_tensor(args[0]), *w = plain_tensor(args[1]), *r = add ? plain_tensor(args[3]) : nullptr;
        if (!x || !w || (add && !r) || !PyFloat_CheckExact(args[2]) || !plain_thread()) Py_RETURN_NONE;
        const int64_t dev = x->get_device();
        hipStream_t st;
        if (x->dim() < 1 || x->numel() == 0 || !is(*x, at::kBFloat16, dev, x->dim()) || !is(*w, at::kBFloat16, dev, 1) ||
            !x->is_contiguous() || !w->is_contiguous() || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const int64_t H = x->size(-1), T = x->numel() / H;
        if (w->size(0) != H || (add && (!is(*r, at::kBFloat16, dev, x->dim()) || !r->is_contiguous() ||
                                        r->sizes() != x->sizes())))
            Py_RETURN_NONE;
        const at::Tensor q = empty_codes(*x, T, H), s = empty_scales(*x, T, (H + kGroup - 1) / kGroup);
        Ref out{pair(q, s)};
        if (!out.p) return nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_rmsnorm_fp8_quant(x->data_ptr(), T, H, H, w->data_ptr(), add ? r->data_ptr() : nullptr, H, q.data_ptr(),
                                       H, (float*)s.data_ptr(), s.stride(0), s.stride(1), (float)PyFloat_AS_DOUBLE(args[2]),
                                       (void*)st);
        }
        if (rc) return failed(rc, add ? "fused_add_rmsnorm_fp8_quant" : "rmsnorm_fp8_quant");
        return out.take();
    });
}

// silu(input, ue8m0, eps) -> (codes, scales) | None
PyObject* silu(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 3) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor* x = plain_tensor(args[0]);
        if (!x || !PyFloat_CheckExact(args[2]) || !plain_thread()) Py_RETURN_NONE;
        const int ue8m0 = PyObject_IsTrue(args[1]);   // any object, as in Python: its truth value may raise
        if (ue8m0 < 0) return nullptr;
        const int64_t dev = x->get_device();
        hipStream_t st;
        if (!is(*x, at::kBFloat16, dev, 2) || x->numel() == 0 || x->stride(1) != 1 || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const int64_t M = x->size(0), Nh = x->size(1) / 2;
        if (M % kGroup || Nh % kGroup || x->size(1) % 2) Py_RETURN_NONE;
        const at::Tensor q = empty_codes(*x, M, Nh), s = empty_scales(*x, M, Nh / kGroup);
        Ref out{pair(q, s)};
        if (!out.p) return nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_silu_mul_quant_fp8(x->data_ptr(), M, Nh, x->stride(0), q.data_ptr(), Nh, (float*)s.data_ptr(), s.stride(0),
                                        s.stride(1), (float)PyFloat_AS_DOUBLE(args[2]), ue8m0, (void*)st);
        }
        if (rc) return failed(rc, "silu_mul_quant_fp8");
        return out.take();
    });
}

// Whether a shape's bf16-input GEMM is preferred, and its workspace: the
// thread's latest answers, as each asks for a plan.
struct Bf16aPlan {
    int64_t M = 0, N = 0, K = 0, dev = -1;
    bool preferred = false;
    int64_t ws = 0;
};
const Bf16aPlan& bf16a_plan(int64_t dev, int64_t M, int64_t N, int64_t K) {
    thread_local Bf16aPlan kept[64];
    Bf16aPlan& p = kept[(uint64_t)(M * 31 + N * 7 + K / 128 + dev) % 64];
    if (p.M != M || p.N != N || p.K != K || p.dev != dev) {
        p.preferred = kbn_fp8_gemm_bf16a_preferred(M, N, K) != 0;
        p.ws = p.preferred ? kbn_fp8_gemm_bf16a_workspace_bytes(M, N, K) : 0;
        p.M = M; p.N = N; p.K = K; p.dev = dev;
    }
    return p;
}

// linear(x, weight, weight_scale, a_buf | None, s_buf | None, o_buf | None,
//        prefill buffers | None, ue8m0, workspaces) -> output [M, N] | None
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 9) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = plain_tensor(args[0]), *w = plain_tensor(args[1]), *ws = plain_tensor(args[2]);
        if (!x || !w || !ws || !PyDict_CheckExact(args[8]) || !plain_thread()) Py_RETURN_NONE;
        const int64_t dev = x->get_device();
        hipStream_t st;
        if (!is(*x, at::kBFloat16, dev, 2) || !is(*w, at::kFloat8_e4m3fn, dev, 2) || !is(*ws, at::kFloat, dev, 2) ||
            x->numel() == 0 || w->numel() == 0 || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const int64_t M = x->size(0), K = x->size(1), N = w->size(0);
        if (w->size(1) != K || K % kGroup || ws->size(0) * kGroup < N || ws->size(1) * kGroup < K || x->stride(1) != 1 ||
            w->stride(1) != 1 || ws->stride(1) != 1)
            Py_RETURN_NONE;
        // the installed buffers that hold M rows: decode, else prefill
        const bool ue8m0 = PyObject_IsTrue(args[7]) == 1;
        const Bf16aPlan* direct = M <= 64 && ue8m0 ? &bf16a_plan(dev, M, N, K) : nullptr;
        if (direct && !direct->preferred) direct = nullptr;
        PyObject* const pf = args[6];
        PyObject *qo = args[3], *so = args[4], *oo = args[5];
        auto rows = [](PyObject* o) { const at::Tensor* t = plain_tensor(o); return t && t->dim() == 2 ? t->size(0) : -1; };
        PyObject* held[3] = {nullptr, nullptr, nullptr};   // attributes of pf
        struct Release {
            PyObject** h;
            ~Release() { for (int i = 0; i < 3; ++i) Py_XDECREF(h[i]); }
        } release{held};
        if (rows(direct ? oo : qo) < M) {
            if (pf == Py_None) Py_RETURN_NONE;
            const char* names[3] = {"a", "s", "o"};
            for (int i = 0; i < 3; ++i)
                if (!(held[i] = PyObject_GetAttrString(pf, names[i]))) {
                    PyErr_Clear();
                    Py_RETURN_NONE;
                }
            qo = held[0]; so = held[1]; oo = held[2];
        }
        const at::Tensor* o = plain_tensor(oo);
        if (!o || !is(*o, at::kBFloat16, dev, 2) || o->size(0) < M || o->size(1) != N || o->stride(1) != 1) Py_RETURN_NONE;
        int rc;
        if (direct) {
            const int64_t bytes = direct->ws;
            const at::Tensor buf = bytes ? kept_workspace(args[8], dev, st, bytes) : at::Tensor();
            if (bytes && !buf.defined()) Py_RETURN_NONE;
            void* const wsp = bytes ? buf.data_ptr() : nullptr;
            {
                NoGil no_gil;
                rc = kbn_fp8_gemm_bf16a(x->data_ptr(), x->stride(0), kQuantEps, w->data_ptr(), w->stride(0),
                                        (const float*)ws->data_ptr(), ws->stride(0), o->data_ptr(), o->stride(0), M, N, K, wsp,
                                        bytes, (void*)st);
            }
        } else {
            const at::Tensor *q = plain_tensor(qo), *s = plain_tensor(so);
            if (!q || !s || !is(*q, at::kFloat8_e4m3fn, dev, 2) || !is(*s, at::kFloat, dev, 2) || q->size(0) < M ||
                q->size(1) != K || q->stride(1) != 1 || s->size(0) < M || s->size(1) != K / kGroup)
                Py_RETURN_NONE;
            const int64_t bytes = kbn_fp8_gemm_nt_workspace_bytes(M, N, K, ue8m0);
            const at::Tensor buf = bytes ? kept_workspace(args[8], dev, st, bytes) : at::Tensor();
            if (bytes && !buf.defined()) Py_RETURN_NONE;
            void* const wsp = bytes ? buf.data_ptr() : nullptr;
            {
                NoGil no_gil;
                rc = kbn_fp8_linear_forward(x->data_ptr(), M, K, x->stride(0), q->data_ptr(), q->stride(0),
                                            (float*)s->data_ptr(), s->stride(0), s->stride(1), kQuantEps, 1, w->data_ptr(),
                                            w->stride(0), (const float*)ws->data_ptr(), ws->stride(0), o->data_ptr(),
                                            o->stride(0), N, ue8m0, wsp, bytes, (void*)st);
            }
        }
        if (rc) return failed(rc, direct ? "fp8_gemm_bf16a" : "fp8_linear_forward");
        if (o->size(0) == M) {
            Py_INCREF(oo);
            return oo;
        }
        return THPVariable_Wrap(o->narrow(0, 0, M));
    });
}

// ---- MXFP4 and the experts layer for few tokens

// The C entries' code of a value type; -1 for another type.
int value_code(at::ScalarType t) {
    return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : t == at::kFloat ? 2 : -1;
}
bool is_mx_scales(const at::Tensor& t, int64_t dev) {
    return (t.scalar_type() == at::kFloat8_e8m0fnu || t.scalar_type() == at::kByte) && t.get_device() == dev;
}

// A tensor as rows: contiguous, or two dimensions with contiguous rows.
struct Rows {
    int64_t n = 0, k = 0, ld = 0;
    bool ok = false;
};
Rows rows_of(const at::Tensor& t) {
    Rows r;
    if (t.dim() < 1 || t.numel() == 0) return r;
    r.k = t.size(-1);
    r.n = t.numel() / r.k;
    r.ok = t.is_contiguous() || (t.dim() == 2 && t.stride(1) == 1);
    r.ld = t.dim() == 2 && r.n > 1 ? t.stride(0) : r.k;
    return r;
}
std::vector<int64_t> with_last(const at::Tensor& like, int64_t last) {
    std::vector<int64_t> s = like.sizes().vec();
    s.back() = last;
    return s;
}
at::Tensor empty_like_rows(const at::Tensor& like, int64_t last, at::ScalarType type) {
    return at::empty(with_last(like, last), like.options().dtype(type).requires_grad(false));
}

// mx_quant(x) -> (codes, scales) | None
PyObject* mx_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 1) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor* x = plain_tensor(args[0]);
        if (!x || !plain_thread()) Py_RETURN_NONE;
        const int code = value_code(x->scalar_type());
        const Rows r = rows_of(*x);
        hipStream_t st;
        if (code < 0 || !r.ok || r.k % 32 || !launch_stream(x->get_device(), st)) Py_RETURN_NONE;
        const at::Tensor q = empty_like_rows(*x, r.k / 2, at::kByte), s = empty_like_rows(*x, r.k / 32, at::kFloat8_e8m0fnu);
        Ref out{pair(q, s)};
        if (!out.p) return nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_mxfp4_quant(x->data_ptr(), code, r.n, r.k, r.ld, q.data_ptr(), r.k / 2, s.data_ptr(), r.k / 32, (void*)st);
        }
        if (rc) return failed(rc, "mxfp4_quant");
        return out.take();
    });
}

// mx_dequant(codes, scales, value code) -> values | None
PyObject* mx_dequant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 3) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *q = plain_tensor(args[0]), *s = plain_tensor(args[1]);
        if (!q || !s || !PyLong_CheckExact(args[2]) || !plain_thread()) Py_RETURN_NONE;
        const long code = PyLong_AsLong(args[2]);
        const int64_t dev = q->get_device();
        const Rows r = rows_of(*q), t = rows_of(*s);
        hipStream_t st;
        if (code < 0 || code > 2 || q->scalar_type() != at::kByte || !is_mx_scales(*s, dev) || !r.ok || !t.ok || r.k % 16 ||
            t.k != r.k / 16 || s->dim() != q->dim() || s->sizes().slice(0, s->dim() - 1) != q->sizes().slice(0, q->dim() - 1) ||
            !launch_stream(dev, st))
            Py_RETURN_NONE;
        const at::Tensor out = empty_like_rows(*q, 2 * r.k, code == 0 ? at::kBFloat16 : code == 1 ? at::kHalf : at::kFloat);
        Ref o{THPVariable_Wrap(out)};
        if (!o.p) return nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_mxfp4_dequant(q->data_ptr(), r.ld, s->data_ptr(), t.ld, r.n, 2 * r.k, out.data_ptr(), (int)code, 2 * r.k, (void*)st);
        }
        if (rc) return failed(rc, "mxfp4_dequant");
        return o.take();
    });
}

// mx_linear(x, codes, scales) -> output | None
PyObject* mx_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 3) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = plain_tensor(args[0]), *w = plain_tensor(args[1]), *s = plain_tensor(args[2]);
        if (!x || !w || !s || !plain_thread()) Py_RETURN_NONE;
        const int code = value_code(x->scalar_type());
        const int64_t dev = x->get_device();
        const Rows r = rows_of(*x);
        hipStream_t st;
        if (code < 0 || !r.ok || r.k % kGroup || !is(*w, at::kByte, dev, 2) || w->numel() == 0 || w->size(1) * 2 != r.k ||
            w->stride(1) != 1 || !is_mx_scales(*s, dev) || s->dim() != 2 || s->size(0) != w->size(0) || s->size(1) != r.k / 32 ||
            s->stride(1) != 1 || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const int64_t N = w->size(0), ldw = N > 1 ? w->stride(0) : r.k / 2, lds = N > 1 ? s->stride(0) : r.k / 32;
        const at::Tensor out = empty_like_rows(*x, N, at::kBFloat16);
        Ref o{THPVariable_Wrap(out)};
        if (!o.p) return nullptr;
        // a buffer of the call's own: calls at once on one stream share nothing
        const int64_t bytes = kbn_mxfp4_linear_workspace_bytes(r.n, N, r.k, code);
        const at::Tensor ws = bytes ? at::empty({bytes}, w->options().requires_grad(false)) : at::Tensor();
        void* const wsp = bytes ? ws.data_ptr() : nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_mxfp4_linear(x->data_ptr(), code, r.ld, w->data_ptr(), ldw, s->data_ptr(), lds, out.data_ptr(), N, r.n, N, r.k,
                                  wsp, bytes, (void*)st);
        }
        if (rc) return failed(rc, "mxfp4_linear");
        return o.take();
    });
}

// few_experts(x, w13, w13 scales, w2, w2 scales, topk weights, topk ids) -> output | None
PyObject* few_experts(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor* t[7];
        for (int i = 0; i < 7; ++i)
            if (!(t[i] = plain_tensor(args[i])) || t[i]->numel() == 0) Py_RETURN_NONE;
        const at::Tensor &x = *t[0], &w13 = *t[1], &s13 = *t[2], &w2 = *t[3], &s2 = *t[4], &tw = *t[5], &ids = *t[6];
        const int64_t dev = x.get_device();
        hipStream_t st;
        if (!plain_thread() || x.dim() != 2 || w13.dim() != 3 || ids.dim() != 2) Py_RETURN_NONE;
        const int code = value_code(x.scalar_type());
        const bool fp8 = w13.scalar_type() == at::kFloat8_e4m3fn;
        const int64_t T = x.size(0), H = x.size(1), E = w13.size(0), N2 = w13.size(1), I = N2 / 2, topk = ids.size(1);
        const Rows r = rows_of(x);
        if ((code != 0 && code != 1) || !r.ok || T > 64 || H % kGroup || N2 % (2 * kGroup) ||
            (!fp8 && w13.scalar_type() != at::kByte) || w13.get_device() != dev || !is(w2, w13.scalar_type(), dev, 3) ||
            !is(tw, at::kFloat, dev, 2) || (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) ||
            ids.get_device() != dev || ids.size(0) != T || tw.sizes() != ids.sizes())
            Py_RETURN_NONE;
        const int64_t per = fp8 ? 1 : 2;   // values a byte
        auto shape = [](const at::Tensor& a, int64_t p, int64_t q, int64_t s) {
            return a.dim() == 3 && a.size(0) == p && a.size(1) == q && a.size(2) == s && a.is_contiguous();
        };
        if (!shape(w13, E, N2, H / per) || !shape(w2, E, H, I / per) || !tw.is_contiguous() || !ids.is_contiguous()) Py_RETURN_NONE;
        if (fp8) {
            if (!is(s13, at::kFloat, dev, 3) || !is(s2, at::kFloat, dev, 3) || !shape(s13, E, N2 / kGroup, H / kGroup) ||
                !shape(s2, E, H / kGroup, I / kGroup))
                Py_RETURN_NONE;
        } else if (!is_mx_scales(s13, dev) || !is_mx_scales(s2, dev) || !shape(s13, E, N2, H / 32) || !shape(s2, E, H, I / 32)) {
            Py_RETURN_NONE;
        }
        if (!launch_stream(dev, st)) Py_RETURN_NONE;
        const at::Tensor out = at::empty({T, H}, x.options().requires_grad(false));
        Ref o{THPVariable_Wrap(out)};
        if (!o.p) return nullptr;
        const int64_t bytes = kbn_few_token_experts_workspace_bytes(T, topk, I);
        if (bytes <= 0) Py_RETURN_NONE;
        const at::Tensor ws = at::empty({bytes}, x.options().dtype(at::kByte).requires_grad(false));
        void* const wsp = ws.data_ptr();
        int rc;
        {
            NoGil no_gil;
            rc = kbn_few_token_experts(x.data_ptr(), code, r.ld, w13.data_ptr(), s13.data_ptr(), w2.data_ptr(), s2.data_ptr(), fp8 ? 0 : 1,
                                       (const float*)tw.data_ptr(), ids.data_ptr(), (int)ids.element_size(), T, topk, E, H, I,
                                       out.data_ptr(), H, wsp, bytes, (void*)st);
        }
        if (rc) return failed(rc, "few_token_experts");
        return o.take();
    });
}

// ---- router, gated norms and adapters

constexpr int64_t kFarRows = 1 << 23;   // row strides from here on are copied by the Python path

// A Python int or float (no subclass) as a number; false for anything else.
bool int_of(PyObject* o, int64_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    v = PyLong_AsLongLongAndOverflow(o, &over);
    return over == 0;
}
bool number_of(PyObject* o, double& v) {
    int64_t i;
    if (PyFloat_CheckExact(o)) v = PyFloat_AS_DOUBLE(o);
    else if (int_of(o, i)) v = (double)i;
    else return false;
    return true;
}
// A tensor or None; false for anything else.
bool plain_or_none(PyObject* o, const at::Tensor*& t) {
    t = o == Py_None ? nullptr : plain_tensor(o);
    return t || o == Py_None;
}
bool is_vector(const at::Tensor& t, at::ScalarType type, int64_t dev, int64_t n) {
    return is(t, type, dev, 1) && t.size(0) == n && t.is_contiguous();
}

// router_gemm(x, weight) -> logits | None
PyObject* router_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = plain_tensor(args[0]), *w = plain_tensor(args[1]);
        if (!x || !w || !plain_thread()) Py_RETURN_NONE;
        const int xc = value_code(x->scalar_type()), wc = value_code(w->scalar_type());
        const int64_t dev = x->get_device();
        const Rows r = rows_of(*x), v = rows_of(*w);
        hipStream_t st;
        if (xc < 0 || (wc != xc && wc != 2) || !r.ok || !v.ok || w->dim() != 2 || w->get_device() != dev || v.k != r.k || r.k % 8 ||
            r.ld >= kFarRows || v.ld >= kFarRows || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const at::Tensor out = empty_like_rows(*x, v.n, at::kFloat);
        Ref o{THPVariable_Wrap(out)};
        if (!o.p) return nullptr;
        const int64_t bytes = kbn_moe_router_gemm_workspace_bytes(r.n, v.n, r.k, xc, wc);
        if (bytes < 0) Py_RETURN_NONE;
        const at::Tensor ws = bytes ? at::empty({bytes}, w->options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
        void* const wsp = bytes ? ws.data_ptr() : nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_moe_router_gemm(x->data_ptr(), xc, r.ld, w->data_ptr(), wc, v.ld, (float*)out.data_ptr(), v.n, r.n, v.n, r.k, wsp,
                                     bytes, (void*)st);
        }
        if (rc) return failed(rc, "moe_router_gemm");
        return o.take();
    });
}

// router_topk(logits, top_k, scoring, bias | None, num_groups, topk_groups, renormalize, scale, index dtype)
//   -> (weights, ids) | None
PyObject* router_topk(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 9) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *l = plain_tensor(args[0]), *bias = nullptr;
        int64_t k, G, kept;
        double scale;
        if (!l || !int_of(args[1], k) || !PyUnicode_CheckExact(args[2]) || !plain_or_none(args[3], bias) || !int_of(args[4], G) ||
            !int_of(args[5], kept) || !PyBool_Check(args[6]) || !number_of(args[7], scale) || !THPDtype_Check(args[8]) ||
            !plain_thread())
            Py_RETURN_NONE;
        const bool sigmoid = PyUnicode_CompareWithASCIIString(args[2], "sigmoid") == 0;
        if (!sigmoid && PyUnicode_CompareWithASCIIString(args[2], "softmax") != 0) Py_RETURN_NONE;
        const at::ScalarType it = ((THPDtype*)args[8])->scalar_type;
        const int code = value_code(l->scalar_type());
        const int64_t dev = l->get_device();
        const Rows r = rows_of(*l);
        hipStream_t st;
        if (code < 0 || !r.ok || k < 1 || k > 64 || (it != at::kInt && it != at::kLong) ||
            (bias && !is_vector(*bias, at::kFloat, dev, r.k)) || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const at::Tensor w = empty_like_rows(*l, k, at::kFloat), ids = empty_like_rows(*l, k, it);
        Ref out{pair(w, ids)};
        if (!out.p) return nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_moe_router_topk(l->data_ptr(), code, r.ld, bias ? (const float*)bias->data_ptr() : nullptr, r.n, r.k, k, sigmoid, G,
                                     kept, args[6] == Py_True, (float)scale, (float*)w.data_ptr(), ids.data_ptr(),
                                     (int)ids.element_size(), (void*)st);
        }
        if (rc) return failed(rc, "moe_router_topk");
        return out.take();
    });
}

// gated_norm(x, residual, weight, post_weight | None, gate | None, residual_scale, eps, rows, codes)
//   -> (normed | None, codes | None, scales | None, residual') | None
PyObject* gated_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 9) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = plain_tensor(args[0]), *r = plain_tensor(args[1]), *w = plain_tensor(args[2]), *post, *gate;
        double rs, eps;
        if (!x || !r || !w || !plain_or_none(args[3], post) || !plain_or_none(args[4], gate) || !number_of(args[5], rs) ||
            !number_of(args[6], eps) || !plain_thread())
            Py_RETURN_NONE;
        const int rows = PyObject_IsTrue(args[7]), codes = PyObject_IsTrue(args[8]);   // any object, as in Python
        if (rows < 0 || codes < 0) return nullptr;
        const at::ScalarType type = x->scalar_type();
        const int code = value_code(type);
        const int64_t dev = x->get_device();
        const Rows xr = rows_of(*x), rr = rows_of(*r);
        hipStream_t st;
        if (code < 0 || !xr.ok || !rr.ok || !is(*r, type, dev, x->dim()) || r->sizes() != x->sizes() || xr.k % 8 ||
            !is_vector(*w, type, dev, xr.k) || (post && !is_vector(*post, type, dev, xr.k)) || (!rows && !codes))
            Py_RETURN_NONE;
        const int64_t T = xr.n, H = xr.k;
        int64_t g_row = 0, g_col = 0;   // [H]; as x; or a column of one value a token
        if (gate) {
            if (gate->scalar_type() != type || gate->get_device() != dev) Py_RETURN_NONE;
            const Rows g = rows_of(*gate);
            if (!g.ok) Py_RETURN_NONE;
            if (gate->dim() == 1 && g.k == H) {
                g_col = 1;
            } else if (gate->dim() == x->dim() && gate->sizes() == x->sizes()) {
                g_col = 1;
                g_row = T > 1 ? g.ld : 0;
            } else if (gate->dim() == x->dim() && g.k == 1 && g.n == T &&
                       gate->sizes().slice(0, gate->dim() - 1) == x->sizes().slice(0, x->dim() - 1)) {
                g_row = T > 1 ? g.ld : 0;
            } else {
                Py_RETURN_NONE;
            }
        }
        if (!launch_stream(dev, st)) Py_RETURN_NONE;
        const int64_t groups = (H + kGroup - 1) / kGroup;
        const at::Tensor res = empty_like_rows(*x, H, type);
        at::Tensor out, q, s;
        Ref res_o{THPVariable_Wrap(res)}, out_o{nullptr}, q_o{nullptr}, s_o{nullptr};
        if (rows) {
            out = empty_like_rows(*x, H, type);
            out_o.p = THPVariable_Wrap(out);
        }
        if (codes) {
            q = empty_codes(*x, T, H);
            s = empty_scales(*x, T, groups);
            q_o.p = THPVariable_Wrap(q);
            s_o.p = THPVariable_Wrap(s);
        }
        if (!res_o.p || (rows && !out_o.p) || (codes && (!q_o.p || !s_o.p))) return nullptr;
        Ref all{PyTuple_Pack(4, rows ? out_o.p : Py_None, codes ? q_o.p : Py_None, codes ? s_o.p : Py_None, res_o.p)};
        if (!all.p) return nullptr;
        int rc;
        {
            NoGil no_gil;
            rc = kbn_gated_add_rmsnorm(x->data_ptr(), code, xr.ld, r->data_ptr(), rr.ld, w->data_ptr(), post ? post->data_ptr() : nullptr,
                                       gate ? gate->data_ptr() : nullptr, g_row, g_col, (float)rs, (float)eps, T, H, res.data_ptr(), H,
                                       rows ? out.data_ptr() : nullptr, H, codes ? q.data_ptr() : nullptr, H,
                                       codes ? (float*)s.data_ptr() : nullptr, codes ? s.stride(0) : 0, codes ? s.stride(1) : 0,
                                       (void*)st);
        }
        if (rc) return failed(rc, "gated_add_rmsnorm");
        return all.take();
    });
}

// lora_add(x, base, lora_a, lora_b, adapter_ids, scaling | None) -> a new output | None
PyObject* lora_add(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 6) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = plain_tensor(args[0]), *base = plain_tensor(args[1]), *a = plain_tensor(args[2]), *b = plain_tensor(args[3]),
                         *ids = plain_tensor(args[4]), *sc;
        if (!x || !base || !a || !b || !ids || !plain_or_none(args[5], sc) || !plain_thread()) Py_RETURN_NONE;
        const at::ScalarType type = x->scalar_type();
        const int code = value_code(type);
        const int64_t dev = x->get_device();
        const Rows xr = rows_of(*x), br = rows_of(*base);
        hipStream_t st;
        if ((code != 0 && code != 1) || !xr.ok || !br.ok || !is(*base, type, dev, x->dim()) || xr.n != br.n ||
            x->sizes().slice(0, x->dim() - 1) != base->sizes().slice(0, base->dim() - 1) || !is(*a, type, dev, 3) ||
            !is(*b, type, dev, 3) || !a->is_contiguous() || !b->is_contiguous() || xr.ld >= kFarRows / 2)
            Py_RETURN_NONE;
        const int64_t T = xr.n, K = xr.k, N = br.k, L = a->size(0), R = a->size(1);
        if (a->size(2) != K || b->size(0) != L || b->size(1) != N || b->size(2) != R || K % 8 || L < 1 ||
            (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || ids->get_device() != dev || ids->numel() != T ||
            !ids->is_contiguous() || (ids->dim() != 1 && ids->sizes() != x->sizes().slice(0, x->dim() - 1)) || (sc && !is_vector(*sc, at::kFloat, dev, L)) || !launch_stream(dev, st))
            Py_RETURN_NONE;
        const int64_t bytes = kbn_lora_add_workspace_bytes(T, K, L, R);
        if (bytes <= 0) Py_RETURN_NONE;
        const at::Tensor out = empty_like_rows(*base, N, type);
        Ref o{THPVariable_Wrap(out)};
        if (!o.p) return nullptr;
        const at::Tensor ws = at::empty({bytes}, x->options().dtype(at::kByte).requires_grad(false));   // of the call's own
        void* const wsp = ws.data_ptr();
        int rc;
        {
            NoGil no_gil;
            rc = kbn_lora_add(x->data_ptr(), code, xr.ld, base->data_ptr(), br.ld, a->data_ptr(), b->data_ptr(), ids->data_ptr(),
                              (int)ids->element_size(), sc ? (const float*)sc->data_ptr() : nullptr, T, N, K, L, R, out.data_ptr(), N,
                              wsp, bytes, (void*)st);
        }
        if (rc) return failed(rc, "lora_add");
        return o.take();
    });
}

PyMethodDef kMethods[] = {
    {"mx_quant", (PyCFunction)(void (*)())mx_quant, METH_FASTCALL, "MXFP4 quantization"},
    {"mx_dequant", (PyCFunction)(void (*)())mx_dequant, METH_FASTCALL, "the values of MXFP4 codes"},
    {"mx_linear", (PyCFunction)(void (*)())mx_linear, METH_FASTCALL, "rows through an MXFP4 weight"},
    {"few_experts", (PyCFunction)(void (*)())few_experts, METH_FASTCALL, "experts layer for few tokens"},
    {"router_gemm", (PyCFunction)(void (*)())router_gemm, METH_FASTCALL, "router logits"},
    {"router_topk", (PyCFunction)(void (*)())router_topk, METH_FASTCALL, "experts of each token"},
    {"gated_norm", (PyCFunction)(void (*)())gated_norm, METH_FASTCALL, "norms after and before a block, gate, residual"},
    {"lora_add", (PyCFunction)(void (*)())lora_add, METH_FASTCALL, "adapters added to a projection's output"},
    {"norm", (PyCFunction)(void (*)())norm, METH_FASTCALL, "RMSNorm (+ residual add) + 1x128 quant"},
    {"silu", (PyCFunction)(void (*)())silu, METH_FASTCALL, "SiLU*Mul + 1x128 quant"},
    {"linear", (PyCFunction)(void (*)())linear, METH_FASTCALL, "bf16 activations through an FP8 weight"},
    {"failed", (PyCFunction)(void (*)())failed_call, METH_FASTCALL, "what a call gives for an error code"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&kModule); }
