// The torch side of the gated projection and of gradient clipping: a Python module that takes tensors, checks them, asks the
// caching allocator for outputs and workspaces and calls the C ABI of libdiffputer_hip.so (include/diffputer.h) on torch's
// current stream, and the gated projection's autograd node.  Host code only; no torch type crosses into the library.
//
// Why not ctypes, as for the sampler: these calls are made once per layer and training step, and take 5 to 20 us on the GPU at
// small sizes.  Through ctypes and a Python autograd function a call took 13 us, a clipping of 14 tensors 24, forward and backward 113;
// here 5, 10 and 75, of which torch's own engine is about 54 (a graph of five inputs).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/Exception.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <optional>
#include <vector>

#include "../../include/diffputer.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject *g_error = nullptr, *g_oom = nullptr;                    // _lib.DiffputerError, torch.OutOfMemoryError

// an error of the library, raised as DiffputerError at the Python boundary (as RuntimeError from a backward pass)
struct LibraryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
    if (rc != DP_OK) throw LibraryError(std::string(what) + " failed (code " + std::to_string(rc) + "): " + dp_last_error());
}

// Forward-mode derivatives: the kernels read values only, so a tangent would be dropped without a word.  (torch itself raises where
// the call makes an autograd node.)
void refuse_tangent(const Tensor& t, const char* who) {
    if (t.defined() && t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        throw LibraryError(std::string(who) + " has no forward-mode derivatives (a tensor carries a tangent)");
}

// Tracers (torch.jit.trace, make_fx, fake and functional tensors) record torch's operations: of a call that would be the
// allocation of its output, and a traced function that returns memory which nothing has filled.  (torch.compile breaks its graph here.)
void refuse_trace(const char* who) {
    using Mode = c10::impl::TorchDispatchModeKey;
    bool on = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
    if (c10::impl::TorchDispatchModeTLS::any_modes_set())
        for (const Mode m : {Mode::PROXY, Mode::FAKE, Mode::FUNCTIONAL}) on = on || c10::impl::TorchDispatchModeTLS::get_mode(m).has_value();
    if (on) throw LibraryError(std::string(who) + " cannot be traced (torch.jit.trace, make_fx, fake tensors): its kernels are not torch operations");
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor bytes_like(const Tensor& t, size_t n) { return at::empty({(int64_t)n}, t.options().dtype(at::kByte).requires_grad(false)); }

// A call with a workspace of the size that is asked for right before it: where another thread's dp_tune comes in between and the
// call needs more, both are made again.
template <typename Size, typename Call> void with_workspace(const Tensor& like, const char* who, Size size, Call call) {
    for (int again = 8;; --again) {
        const size_t need = size();
        if (need == 0) check(DP_EINVAL, who);
        const Tensor ws = bytes_like(like, need);
        const int rc = call(ws.data_ptr(), need);
        if (rc == DP_EWORKSPACE && again) continue;
        return check(rc, who);
    }
}

int code_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? DP_DTYPE_F32 : t.scalar_type() == at::kBFloat16 ? DP_DTYPE_BF16 : -1; }

// ---- gated projection ----------------------------------------------------------------------------------------------------
// [rows, cols] with contiguous rows that do not overlap: `t` itself, or a copy (also of a tensor whose negation is a bit, which its
// memory does not show)
Tensor rows_of(const Tensor& t) {
    if (t.is_neg()) return t.resolve_neg().contiguous();
    if (t.is_contiguous() || ((t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) == 1))) return t;
    return t.contiguous();
}
int64_t ld_of(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }           // a single row's stride says nothing
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bias_of(const Tensor& t) { return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }

// the kernels take both weights with one row stride
void weights_of(Tensor& wg, Tensor& wu) {
    wg = rows_of(wg);
    wu = rows_of(wu);
    if (wg.size(0) > 1 && ld_of(wg) != ld_of(wu)) {
        wg = wg.contiguous();
        wu = wu.contiguous();
    }
}

Tensor forward_of(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int act, Tensor* pre) {
    const int64_t M = x.size(0), K = x.size(1), N = wg.size(0);
    const c10::DeviceGuard guard(x.device());
    Tensor h = at::empty({M, N}, x.options().requires_grad(false));
    if (pre) *pre = bytes_like(x, dp_gated_linear_pre_bytes(code_of(x), M, (int)N));
    if (M == 0) return h;
    const int dt = code_of(x);
    with_workspace(
        x, "dp_gated_linear", [&] { return dp_gated_linear_workspace_bytes(dt, x.data_ptr(), ld_of(x), wg.data_ptr(), wu.data_ptr(), ld_of(wg), M, (int)N, (int)K, 0); },
        [&](void* ws, size_t n) {
            return dp_gated_linear(dt, x.data_ptr(), ld_of(x), wg.data_ptr(), wu.data_ptr(), ld_of(wg), ptr(bg), ptr(bu), h.data_ptr(), N, pre ? pre->data_ptr() : nullptr, M, (int)N, (int)K, act,
                                   ws, n, stream_of(x));
        });
    return h;
}

// A leaf's accumulation node belongs to the stream on which its first graph was made, and lives as long as any graph of the leaf.  A
// backward pass under capture whose gradients go on to a node of another stream would have that stream wait, which is no part of
// the capture, and end the process: whether one of the node's gradients goes to such a node.
bool goes_elsewhere(const torch::autograd::Node& node, c10::DeviceIndex device) {
    const auto here = c10::hip::getCurrentHIPStream(device).id();
    for (const auto& edge : node.next_edges()) {
        if (!edge.function) continue;
        const auto stream = edge.function->stream();
        if (stream && stream->id() != here) return true;
    }
    return false;
}
// the capture that a stream is part of (a stream that was forked from a captured one is), 0 = none
unsigned long long capture_of(hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(stream, &status, &id) != hipSuccess) {
        (void)hipGetLastError();                                 // which the next launch would report as its own
        return 0;
    }
    return status == hipStreamCaptureStatusActive ? id : 0;
}
// whether this is captured and one of the node's gradients goes to a node of a stream outside the capture
bool leaves_capture(const torch::autograd::Node& node, c10::DeviceIndex device) {
    if (!goes_elsewhere(node, device)) return false;
    const auto here = c10::hip::getCurrentHIPStream(device);
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(here.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return false;
    const auto capture = capture_of(here.stream());
    for (const auto& edge : node.next_edges()) {
        if (!edge.function) continue;
        const auto stream = edge.function->stream();
        if (!stream || stream->id() == here.id()) continue;
        const hipStream_t other = c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *stream).stream();
        // (the null stream takes part in no capture, and may not be asked during one)
        if (!capture || !other || stream->device_index() != device || capture_of(other) != capture) return true;
    }
    return false;
}

struct GatedLinear : public torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const std::optional<Tensor>& b_gate,
                          const std::optional<Tensor>& b_up, int64_t act) {
        Tensor wg = w_gate, wu = w_up, pre;
        weights_of(wg, wu);
        const Tensor xr = rows_of(x), bg = b_gate ? bias_of(*b_gate) : Tensor(), bu = b_up ? bias_of(*b_up) : Tensor();
        const Tensor h = forward_of(xr, wg, wu, bg, bu, (int)act, &pre);
        ctx->save_for_backward({x, w_gate, w_up, pre});
        ctx->saved_data["act"] = act;
        ctx->saved_data["biases"] = (int64_t)((b_gate ? 1 : 0) + (b_up ? 2 : 0));
        return h;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const int64_t act = ctx->saved_data["act"].toInt(), biases = ctx->saved_data["biases"].toInt();
        refuse_trace("gated_linear's backward pass");
        for (const Tensor* t : {&saved[0], &saved[1], &saved[2], (const Tensor*)&grads[0]}) refuse_tangent(*t, "gated_linear's backward pass");
        const auto node = torch::autograd::get_current_node();
        if (node && leaves_capture(*node, saved[0].device().index()))
            throw LibraryError("gated_linear: this backward pass is captured while a graph of its inputs that was made on a stream outside the capture is alive; drop that graph before the capture");
        const Tensor x = rows_of(saved[0]), &pre = saved[3];
        Tensor wg = saved[1], wu = saved[2];
        weights_of(wg, wu);
        const int64_t M = x.size(0), K = x.size(1), N = wg.size(0);
        const c10::DeviceGuard guard(x.device());
        const Tensor dh = rows_of(grads[0]);
        const auto opt = x.options().requires_grad(false);
        int edge = 0;                                            // the node's edges are those of the tensors that were given
        auto out = [&](bool given, at::IntArrayRef size) { return given && ctx->needs_input_grad(edge++) ? at::empty(size, opt) : Tensor(); };
        Tensor dx = out(true, {M, K}), dwg = out(true, {N, K}), dwu = out(true, {N, K}), dbg = out(biases & 1, {N}), dbu = out(biases & 2, {N});
        const int dt = code_of(x), flags = (dx.defined() ? DP_GATED_DX : 0) | (dwg.defined() ? DP_GATED_DW_GATE : 0) | (dwu.defined() ? DP_GATED_DW_UP : 0) | DP_GATED_DB;
        with_workspace(
            x, "dp_gated_linear_bwd", [&] { return dp_gated_linear_workspace_bytes(dt, x.data_ptr(), ld_of(x), wg.data_ptr(), wu.data_ptr(), ld_of(wg), M, (int)N, (int)K, flags); },
            [&](void* ws, size_t n) {
                return dp_gated_linear_bwd(dt, x.data_ptr(), ld_of(x), wg.data_ptr(), wu.data_ptr(), ld_of(wg), pre.data_ptr(), dh.data_ptr(), ld_of(dh), ptr(dx), ptr(dwg), ptr(dwu), ptr(dbg), ptr(dbu),
                                           M, (int)N, (int)K, (int)act, ws, n, stream_of(x));
            });
        variable_list res = {dx, dwg, dwu, dbg, dbu, Tensor()};
        if (at::GradMode::is_enabled()) {                        // create_graph: first derivatives only, said when a second one is asked for
            variable_list given;
            for (auto& t : res)
                if (t.defined()) given.push_back(t.set_requires_grad(true));
            const auto error = std::make_shared<torch::autograd::DelayedError>("gated_linear has first derivatives only", (int64_t)given.size());
            given = (*error)(std::move(given));
            size_t k = 0;
            for (auto& t : res)
                if (t.defined()) t = given[k++];
        }
        return res;
    }
};

// what a Python argument is: a tensor, None (an undefined tensor), or neither
bool tensor_arg(PyObject* o, Tensor& t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    t = THPVariable_Unpack(o);
    return true;
}

// runs f; C++ exceptions become Python's
template <typename F> PyObject* guarded(F f) {
    try {
        return f();
    } catch (const LibraryError& e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(g_oom ? g_oom : PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// gated_linear(x, w_gate, w_up, b_gate, b_up, act) -> h, or None for arguments that it does not take (the caller says why)
PyObject* py_gated_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Tensor x, w[2], b[2];
        if (n != 6 || !tensor_arg(args[0], x) || !tensor_arg(args[1], w[0]) || !tensor_arg(args[2], w[1]) || !tensor_arg(args[3], b[0]) || !tensor_arg(args[4], b[1])) Py_RETURN_NONE;
        const long act = PyLong_AsLong(args[5]);
        if (act == -1 && PyErr_Occurred()) return nullptr;
        refuse_trace("gated_linear");
        for (const Tensor* t : {&x, &w[0], &w[1], &b[0], &b[1]}) refuse_tangent(*t, "gated_linear");
        if (!x.defined() || !w[0].defined() || !w[1].defined() || !x.is_cuda() || code_of(x) < 0 || x.dim() < 1 || w[0].dim() != 2 || w[1].sizes() != w[0].sizes()) Py_RETURN_NONE;
        const int64_t N = w[0].size(0), K = w[0].size(1);
        if (N < 1 || K < 1 || x.size(-1) != K) Py_RETURN_NONE;
        if (N > 1 << 20 || K > 1 << 20) throw LibraryError("gated_linear: N = " + std::to_string(N) + ", K = " + std::to_string(K) + ": both are limited to 2^20");
        bool grad = x.requires_grad();
        for (const Tensor* t : {&w[0], &w[1], &b[0], &b[1]}) {
            if (!t->defined()) continue;
            if (t->scalar_type() != x.scalar_type() || t->device() != x.device() || t->layout() != at::kStrided) Py_RETURN_NONE;
            grad = grad || t->requires_grad();
        }
        if (x.layout() != at::kStrided) Py_RETURN_NONE;
        for (const Tensor& t : b) {
            if (!t.defined()) continue;
            if (t.dim() != 1 || t.size(0) != N) Py_RETURN_NONE;
            if (!t.data_ptr()) throw LibraryError("gated_linear: a bias has no memory of its own (a wrapper of other tensors?)");     // a null pointer is no bias
        }
        const bool flat = x.dim() == 2;
        int64_t M = 1;
        for (int64_t d = 0; d + 1 < x.dim(); ++d) M *= x.size(d);
        const Tensor x2 = flat ? x : x.reshape({M, K});
        Tensor h;
        if (grad && at::GradMode::is_enabled()) {
            auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
            h = GatedLinear::apply(x2, w[0], w[1], opt(b[0]), opt(b[1]), (int64_t)act);
        } else {
            const at::NoGradGuard off;
            weights_of(w[0], w[1]);
            for (Tensor& t : b)
                if (t.defined()) t = bias_of(t);
            h = forward_of(rows_of(x2), w[0], w[1], b[0], b[1], (int)act, nullptr);
        }
        if (!flat) {
            auto size = x.sizes().vec();
            size.back() = N;
            h = h.reshape(size);
        }
        return THPVariable_Wrap(h);
    });
}

// ---- gradient norm and clipping ---------------------------------------------------------------------------------------------
// whether t's elements fill one range of memory, each place once (in any order of its dimensions)
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// grads(tensors, norm_type (DP_NORM_..), limit): limit None = the norm alone, else clipped in place -> norm; None for
// arguments that it does not take; the index of the first tensor that has to be passed as a dense one otherwise
PyObject* py_grads(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 3 || !PyList_Check(args[0])) Py_RETURN_NONE;
        const Py_ssize_t count = PyList_GET_SIZE(args[0]);
        const long kind = PyLong_AsLong(args[1]);
        if (kind == -1 && PyErr_Occurred()) return nullptr;
        const bool clip = args[2] != Py_None;
        const double limit = clip ? PyFloat_AsDouble(args[2]) : 0.0;
        if (clip && limit == -1.0 && PyErr_Occurred()) return nullptr;
        if (count < 1 || count > (1 << 24)) Py_RETURN_NONE;
        refuse_trace(clip ? "clip_grads" : "grad_norm");
        for (Py_ssize_t i = 0; i < count; ++i)
            if (THPVariable_Check(PyList_GET_ITEM(args[0], i))) refuse_tangent(THPVariable_Unpack(PyList_GET_ITEM(args[0], i)), clip ? "clip_grads" : "grad_norm");
        std::vector<void*> ptrs(count);
        std::vector<int64_t> numel(count);
        std::vector<int> dtypes(count);
        c10::Device dev(c10::kCPU);
        const Tensor* first = nullptr;
        for (Py_ssize_t i = 0; i < count; ++i) {
            PyObject* const o = PyList_GET_ITEM(args[0], i);
            if (!THPVariable_Check(o)) Py_RETURN_NONE;
            const Tensor& t = THPVariable_Unpack(o);
            if (i == 0) {
                first = &t;
                dev = t.device();
            }
            dtypes[i] = code_of(t);
            if (!t.is_cuda() || dtypes[i] < 0 || t.device() != dev || t.layout() != at::kStrided) Py_RETURN_NONE;
            if (!dense(t)) return PyLong_FromSsize_t(i);
            ptrs[i] = t.data_ptr();
            numel[i] = t.numel();
        }
        const at::NoGradGuard off;
        const c10::DeviceGuard guard(dev);
        const Tensor norm = at::empty({}, first->options().dtype(at::kFloat).requires_grad(false));
        const size_t need = dp_grad_workspace_bytes((int)count);
        const Tensor ws = bytes_like(*first, need);
        if (clip)                                                // written in place: a graph that kept one of them notices
            for (Py_ssize_t i = 0; i < count; ++i) {
                const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(args[0], i));
                if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
            }
        if (clip) check(dp_clip_grads((int)count, ptrs.data(), numel.data(), dtypes.data(), (int)kind, limit, (float*)norm.data_ptr(), ws.data_ptr(), need, stream_of(norm)), "dp_clip_grads");
        else check(dp_grad_norm((int)count, (const void* const*)ptrs.data(), numel.data(), dtypes.data(), (int)kind, (float*)norm.data_ptr(), ws.data_ptr(), need, stream_of(norm)), "dp_grad_norm");
        return THPVariable_Wrap(norm);
    });
}

PyObject* py_set_errors(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i) {
        PyObject*& to = i ? g_oom : g_error;
        Py_INCREF(args[i]);
        Py_XDECREF(to);
        to = args[i];
    }
    Py_RETURN_NONE;
}

PyObject* py_goes_elsewhere(PyObject*, PyObject* o) {
    return guarded([&]() -> PyObject* {
        Tensor t;
        if (!tensor_arg(o, t) || !t.defined() || !t.grad_fn()) Py_RETURN_NONE;
        return PyBool_FromLong(goes_elsewhere(*t.grad_fn(), t.device().index()));
    });
}

PyMethodDef g_methods[] = {
    {"goes_elsewhere", py_goes_elsewhere, METH_O, "whether a gradient of the node that made a tensor goes to a node of another stream than the current one"},
    {"gated_linear", (PyCFunction)(void (*)(void))py_gated_linear, METH_FASTCALL, "gated_linear(x, w_gate, w_up, b_gate, b_up, act)"},
    {"grads", (PyCFunction)(void (*)(void))py_grads, METH_FASTCALL, "grads(tensors, norm_type, limit)"},
    {"set_errors", (PyCFunction)(void (*)(void))py_set_errors, METH_FASTCALL, "classes of the library's errors and of the allocator's"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "dp_torch", "torch side of libdiffputer_hip.so", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dp_torch() { return PyModule_Create(&g_module); }
