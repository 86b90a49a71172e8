// The op's host path in native code: what hip.scan_forward / hip.scan_backward do for plain GPU tensors -- checks,
// layout, outputs, workspace, stream, launch -- in one call from Python. At [4, 256, 1024] fp32 those steps took 13.5 us
// forward and 16.8 us backward in Python, several times the scan itself (4.8 / 6.0 us), and take 4.6 and 5.4 us here,
// the launch included; a training step through the op 67 -> 38 us where the autograd engine's thread wakes at once,
// 141 -> 64 us where it does not and the two threads pass the interpreter lock back and forth.
//
// scan(gate, value) is the whole op, its autograd node included. The node saves gate and output as the Python one does (hooks
// on saved tensors, version checks and the release after a backward pass are the engine's own), and its backward pass takes
// no interpreter lock: the same step 72 -> 55 us where the engine's thread does not wake at once (two wake-ups are most of
// what is left), the forward pass alone 8.0 -> 5.9 us and without gradients 6.3 -> 3.8 us ([8, 256, 32]).
//
// scan(gate, value), forward(gate, value) and backward(gate, output, out_grad) return None for every call they do not cover,
// and the caller goes on with the Python path, which also raises the errors: tensor subclasses and modes, functorch and fake
// tensors, forward-mode gradients, tracing, mismatched arguments, empty tensors, and views that have to be copied first. The
// library's entry points are handed in as addresses by bind(), so that whichever build of it hip.py loaded is the one that
// runs.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <array>
#include <atomic>
#include <sstream>
#include <unordered_map>
#include <vector>

#include "scanscam_hip.h"
#include "scanscam_ops.h"

namespace {

decltype(&scanscam_scan_fwd_strided) fwd_rows = nullptr;
decltype(&scanscam_scan_bwd_strided) bwd_rows = nullptr;
decltype(&scanscam_scan_fwd_cl_strided) fwd_cl = nullptr;
decltype(&scanscam_scan_bwd_cl_strided) bwd_cl = nullptr;
decltype(&scanscam_workspace_bytes) ws_rows = nullptr;
decltype(&scanscam_workspace_bytes_cl) ws_cl = nullptr;
decltype(&scanscam_strerror) error_text = nullptr;

// What scan()'s backward pass calls for gradients that the native path does not cover (bind(); never released).
PyObject *python_backward = nullptr;
// Calls are left to the Python path while it checks waits or limits polls (hip.check_waits).
std::atomic<bool> left_to_python{false};

constexpr int kMaxDims = 16;

int dtype_code(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return SCANSCAM_F32;
    case at::kBFloat16: return SCANSCAM_BF16;
    case at::kHalf: return SCANSCAM_F16;
    case at::kDouble: return SCANSCAM_F64;
    default: return -1;
    }
}

// A strided GPU tensor with memory of its own and nothing on top of it that a plain pointer would bypass.
bool plain(const at::Tensor &t)
{
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet wrapped({K::Python, K::PythonTLSSnapshot, K::FuncTorchBatched, K::FuncTorchGradWrapper,
                                           K::FuncTorchVmapMode, K::Functionalize, K::Negative, K::Conjugate, K::ZeroTensor});
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(wrapped) && t.has_storage();
}

struct Call {
    std::array<at::Tensor, 5> t;  // forward: gate, value, out; backward: gate, output, out_grad, gate_grad, value_grad
    int inputs, outputs;
    int code;
    bool cl;                      // channels-last
    int64_t n0, n1, T, C;         // rows: n0 groups of n1 rows of T; channels-last: n0 batch elements of [T, C]
    bool dense;
    std::array<scanscam_strides, 5> st;

    bool row_view(const at::Tensor &x) const { return x.size(-1) == 1 || x.stride(-1) == 1; }
    bool cl_view(const at::Tensor &x) const { return x.size(-2) > 1 && x.stride(-2) == 1 && !row_view(x); }

    // Inputs that this path takes as they are.
    bool accept()
    {
        const at::Tensor &first = t[0];
        const int64_t dims = first.dim();
        code = dtype_code(first.scalar_type());
        if (code < 0 || dims < 2 || dims > kMaxDims || first.numel() == 0) return false;
        for (int i = 0; i < inputs; i++) {
            if (!plain(t[i])) return false;
            if (i > 0 && (t[i].device() != first.device() || t[i].scalar_type() != first.scalar_type() || t[i].sizes() != first.sizes()))
                return false;
        }
        T = first.size(-1);
        cl = cl_view(t[0]) && cl_view(t[1]);  // (the rule looks at gate and value, or gate and output)
        if (cl) {
            C = first.size(-2);
            for (int i = 2; i < inputs; i++)
                if (!cl_view(t[i])) return false;
        } else {
            for (int i = 0; i < inputs; i++)
                if (!row_view(t[i])) return false;
        }
        return true;
    }

    void allocate()
    {
        const at::Tensor &first = t[0];
        const auto options = at::TensorOptions().dtype(first.scalar_type()).device(first.device());
        std::array<int64_t, kMaxDims> sizes;
        const int64_t dims = first.dim();
        for (int64_t d = 0; d < dims; d++) sizes[d] = first.size(d);
        if (cl) std::swap(sizes[dims - 1], sizes[dims - 2]);
        for (int i = inputs; i < inputs + outputs; i++) {
            t[i] = at::empty(at::IntArrayRef(sizes.data(), dims), options);
            if (cl) t[i] = t[i].transpose(-1, -2);
        }
    }

    // The leading dimensions (all but the last `inner`) merged into as few levels as all tensors allow, into n0, n1 and
    // st; false if that takes more than `most` levels.
    bool merge(int inner, int most)
    {
        const int n = inputs + outputs;
        int64_t size[2] = {1, 1}, stride[2][5] = {};
        int levels = 0;
        for (int64_t d = 0; d < t[0].dim() - inner; d++) {
            const int64_t s = t[0].size(d);
            if (s == 1) continue;
            bool joins = levels > 0;
            for (int i = 0; i < n && joins; i++) joins = stride[levels - 1][i] == t[i].stride(d) * s;
            if (joins) {
                size[levels - 1] *= s;
            } else {
                if (levels == most) return false;
                size[levels++] = s;
            }
            for (int i = 0; i < n; i++) stride[levels - 1][i] = t[i].stride(d);
        }
        const int last = levels > 0 ? levels - 1 : 0;
        n0 = levels == 2 || inner == 2 ? size[0] : 1;
        n1 = inner == 2 ? 1 : size[last];
        for (int i = 0; i < n; i++) {
            if (inner == 2) st[i] = {stride[0][i], t[i].stride(-1)};
            else st[i] = {levels == 2 ? stride[0][i] : 0, stride[last][i]};
        }
        return true;
    }

    bool lay_out()
    {
        dense = false;
        if (cl) {
            const int64_t esize = (int64_t)t[0].element_size();
            for (int i = 0; i < inputs + outputs; i++)  // (further apart than the kernels address: copied first)
                if (t[i].stride(-1) >= (int64_t(1) << 31) / esize / 18 || C >= (int64_t(1) << 31) / esize) return false;
            return merge(2, 1);
        }
        dense = true;
        for (int i = 0; i < inputs; i++) dense = dense && t[i].is_contiguous();
        if (dense) {
            n0 = 1;
            n1 = t[0].numel() / T;
            return true;
        }
        return merge(1, 2);
    }

    size_t workspace_bytes() const
    {
        const int direction = inputs == 2 ? SCANSCAM_FORWARD : SCANSCAM_BACKWARD;
        if (!cl) return ws_rows(n0 * n1, T, code, direction);
        // The channels-last choice goes through a cost model: remembered, a pure function of the shape.
        struct Key {
            int64_t b, T, C;
            int what;
            bool operator==(const Key &o) const { return b == o.b && T == o.T && C == o.C && what == o.what; }
        };
        struct Hash {
            size_t operator()(const Key &k) const
            {
                return (size_t)((uint64_t)k.b * 0x9E3779B97F4A7C15ull ^ (uint64_t)k.T * 0xC2B2AE3D27D4EB4Full ^
                                (uint64_t)k.C * 0x165667B19E3779F9ull ^ (uint64_t)k.what);
            }
        };
        static thread_local std::unordered_map<Key, size_t, Hash> known;
        const Key key{n0, T, C, code * 2 + direction};
        const auto it = known.find(key);
        if (it != known.end()) return it->second;
        if (known.size() >= 4096) known.clear();
        const size_t n = ws_cl(n0, T, C, code, direction, nullptr);
        known.emplace(key, n);
        return n;
    }

    int launch()
    {
        const size_t bytes = workspace_bytes();
        at::Tensor ws;
        if (bytes != 0) ws = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(t[0].device()));
        void *w = bytes != 0 ? ws.data_ptr() : nullptr;
        void *stream = c10::hip::getCurrentHIPStream(t[0].device().index()).stream();
        void *p[5];
        for (int i = 0; i < inputs + outputs; i++) p[i] = t[i].data_ptr();
        auto s = [&](int i) { return dense ? nullptr : &st[i]; };
        if (inputs == 2)
            return cl ? fwd_cl(p[0], p[1], p[2], s(0), s(1), s(2), n0, T, C, code, w, bytes, stream, nullptr)
                      : fwd_rows(p[0], p[1], p[2], s(0), s(1), s(2), n0, n1, T, code, w, bytes, stream, nullptr);
        return cl ? bwd_cl(p[0], p[1], p[2], p[3], p[4], s(0), s(1), s(2), s(3), s(4), n0, T, C, code, w, bytes, stream, nullptr)
                  : bwd_rows(p[0], p[1], p[2], p[3], p[4], s(0), s(1), s(2), s(3), s(4), n0, n1, T, code, w, bytes, stream, nullptr);
    }
};

// A Python-level function or dispatch mode sees the calls of the Python path; leave them to it.
bool modes_active()
{
    return at::impl::PythonTorchFunctionTLS::stack_len() > 0 || c10::impl::TorchDispatchModeTLS::any_modes_set();
}

// Runs an accepted call; false if it is not covered after all. The library's errors are exceptions.
bool perform(Call &c)
{
    const c10::DeviceGuard guard(c.t[0].device());
    c.allocate();
    if (!c.lay_out()) return false;
    const int rc = c.launch();
    if (rc != SCANSCAM_OK)
        throw std::runtime_error(std::string("scanscam_scan_") + (c.inputs == 2 ? "fwd" : "bwd") + (c.cl ? "_cl" : "") + "_strided: " + error_text(rc));
    return true;
}

// The same for a call of which only the inputs are there, in c.t.
bool execute(Call &c) { return c.accept() && perform(c); }

PyObject *run(PyObject *const *args, Py_ssize_t nargs, int inputs, int outputs)
{
    HANDLE_TH_ERRORS
    if (nargs != inputs || !fwd_rows || modes_active()) Py_RETURN_NONE;
    Call c;
    c.inputs = inputs;
    c.outputs = outputs;
    for (int i = 0; i < inputs; i++) {
        if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
        c.t[i] = THPVariable_Unpack(args[i]);
    }
    bool covered;
    {
        pybind11::gil_scoped_release no_gil;
        covered = execute(c);
    }
    if (!covered) Py_RETURN_NONE;
    if (outputs == 1) return THPVariable_Wrap(std::move(c.t[2]));
    pybind11::object ga = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(c.t[3])));
    pybind11::object gb = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(c.t[4])));
    return PyTuple_Pack(2, ga.ptr(), gb.ptr());
    END_HANDLE_TH_ERRORS
}

using torch::autograd::variable_list;

variable_list backward_in_python(const at::Tensor &gate, const at::Tensor &output, const at::Tensor &out_grad)
{
    pybind11::gil_scoped_acquire gil;
    variable_list grads(2);
    pybind11::object args[3], result;
    const at::Tensor *t[3] = {&gate, &output, &out_grad};
    for (int i = 0; i < 3; i++) args[i] = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(*t[i]));
    result = pybind11::reinterpret_steal<pybind11::object>(
        PyObject_CallFunctionObjArgs(python_backward, args[0].ptr(), args[1].ptr(), args[2].ptr(), nullptr));
    if (!result) {
        python_error error;
        error.persist();
        throw error;
    }
    for (int i = 0; i < 2; i++) grads[i] = THPVariable_Unpack(PyTuple_GET_ITEM(result.ptr(), i));
    return grads;
}

struct ScanBackward : torch::autograd::Function<ScanBackward> {
    // `done`: the call, executed.
    static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &gate, const at::Tensor &, Call *done)
    {
        ctx->save_for_backward({gate, done->t[2]});
        return done->t[2];
    }
    static variable_list backward(torch::autograd::AutogradContext *ctx, variable_list out_grads)
    {
        RECORD_FUNCTION("ScanBackward", c10::ArrayRef<const c10::IValue>{});
        const variable_list saved = ctx->get_saved_variables();
        variable_list grads;
        Call c;
        c.inputs = 3;
        c.outputs = 2;
        c.t[0] = saved[0];
        c.t[1] = saved[1];
        c.t[2] = out_grads[0];
        if (!left_to_python && !modes_active() && execute(c)) grads = {c.t[3], c.t[4]};
        else grads = backward_in_python(saved[0], saved[1], out_grads[0]);
        grads.emplace_back();  // none for `done`
        return grads;
    }
};

// What Python sees of the node (output.grad_fn): the name and the attributes that a Python function's node has, on top of a
// C++ node's.
using ScanNode = torch::autograd::CppNode<ScanBackward>;

ScanNode *scan_node(PyObject *self) { return static_cast<ScanNode *>(reinterpret_cast<torch::autograd::THPCppFunction *>(self)->cdata.get()); }

PyObject *node_name(PyObject *, PyObject *) { return PyUnicode_FromString("ScanBackward"); }

PyObject *node_saved_tensors(PyObject *self, void *)
{
    HANDLE_TH_ERRORS
    const variable_list saved = scan_node(self)->ctx_.get_saved_variables();
    pybind11::tuple out(saved.size());
    for (size_t i = 0; i < saved.size(); i++) out[i] = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(saved[i]));
    return out.release().ptr();
    END_HANDLE_TH_ERRORS
}

PyObject *node_needs_input_grad(PyObject *self, void *)
{
    ScanNode *node = scan_node(self);
    return PyTuple_Pack(2, node->should_compute_output(0) ? Py_True : Py_False, node->should_compute_output(1) ? Py_True : Py_False);
}

PyMethodDef node_methods[] = {{"name", node_name, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyGetSetDef node_properties[] = {{"saved_tensors", node_saved_tensors, nullptr, nullptr, nullptr},
                                 {"needs_input_grad", node_needs_input_grad, nullptr, nullptr, nullptr},
                                 {nullptr, nullptr, nullptr, nullptr, nullptr}};
PyTypeObject node_type;

PyObject *scan(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 2 || !fwd_rows || left_to_python || modes_active() || torch::jit::tracer::isTracing() ||
        c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
        Py_RETURN_NONE;
    Call c;
    c.inputs = 2;
    c.outputs = 1;
    for (int i = 0; i < 2; i++) {
        if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
        c.t[i] = THPVariable_Unpack(args[i]);
        if (c.t[i]._fw_grad(/*level=*/0).defined()) Py_RETURN_NONE;
    }
    if (!c.accept()) Py_RETURN_NONE;
    bool covered;
    {
        pybind11::gil_scoped_release no_gil;
        RECORD_FUNCTION("Scan", c10::ArrayRef<const c10::IValue>{});
        {
            const at::AutoGradMode no_grad(false);
            covered = perform(c);
        }
        if (covered && at::GradMode::is_enabled() && (c.t[0].requires_grad() || c.t[1].requires_grad()))
            c.t[2] = ScanBackward::apply(c.t[0], c.t[1], &c);
    }
    if (!covered) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(c.t[2]));
    END_HANDLE_TH_ERRORS
}

PyObject *leave_to_python(PyObject *, PyObject *on)
{
    left_to_python = PyObject_IsTrue(on) == 1;
    Py_RETURN_NONE;
}

PyObject *forward(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return run(args, nargs, 2, 1); }
PyObject *backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) { return run(args, nargs, 3, 2); }

// bind(fwd_rows, bwd_rows, fwd_cl, bwd_cl, ws_rows, ws_cl, strerror, backward): addresses of the library's entry points, and
// the Python function (gate, output, out_grad) -> (gate_grad, value_grad). Returns the type of the autograd nodes.
PyObject *bind(PyObject *, PyObject *args)
{
    unsigned long long a[7];
    PyObject *callable;
    if (!PyArg_ParseTuple(args, "KKKKKKKO", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, &callable)) return nullptr;
    Py_INCREF(callable);
    python_backward = callable;
    bwd_rows = reinterpret_cast<decltype(bwd_rows)>(a[1]);
    fwd_cl = reinterpret_cast<decltype(fwd_cl)>(a[2]);
    bwd_cl = reinterpret_cast<decltype(bwd_cl)>(a[3]);
    ws_rows = reinterpret_cast<decltype(ws_rows)>(a[4]);
    ws_cl = reinterpret_cast<decltype(ws_cl)>(a[5]);
    error_text = reinterpret_cast<decltype(error_text)>(a[6]);
    fwd_rows = reinterpret_cast<decltype(fwd_rows)>(a[0]);
    static const bool registered = [] {
        // The type of a node whose class has none of its own.
        const std::shared_ptr<torch::autograd::Node> node(new ScanNode, torch::autograd::deleteNode);
        PyObject *plain_node = torch::autograd::functionToPyObject(node);
        node_type.tp_base = Py_TYPE(plain_node);
        Py_INCREF(node_type.tp_base);
        Py_DECREF(plain_node);
        torch::autograd::_initFunctionPyTypeObject(node_type, "ScanBackward", node_properties, node_methods);
        torch::autograd::registerCppFunction(typeid(ScanNode), &node_type);
        return true;
    }();
    (void)registered;
    Py_INCREF(&node_type);
    return reinterpret_cast<PyObject *>(&node_type);
}

// ---------------------------------------------------------------------------------------------------------------------------
// The operators of a state space layer. In Python the checks, the struct of arguments and the outputs took 13 to 20 us a call,
// against 3 to 6 us here (4 us of the kernel at one token); a forward and backward pass over 9 x 1 x 32 values took 142 us
// (norm), 145 (conv) and 222 (selective scan), and 64, 62 and 89 with nodes in C++ as for scan(). As above, None is returned for every
// call that is not covered (CPU tensors, mismatched arguments, views that have to be copied first), and the Python path goes on with it.
// ---------------------------------------------------------------------------------------------------------------------------
struct Operators {
    decltype(&scanscam_selective_fwd) selective = nullptr;
    decltype(&scanscam_selective_workspace_bytes) selective_workspace = nullptr;
    decltype(&scanscam_selective_step_fwd) selective_step = nullptr;
    decltype(&scanscam_conv_fwd) conv = nullptr;
    decltype(&scanscam_conv_step_fwd) conv_step = nullptr;
    decltype(&scanscam_norm_fwd) norm = nullptr;
    decltype(&scanscam_selective_bwd) selective_back = nullptr;
    decltype(&scanscam_selective_saved_bytes) selective_saved = nullptr;
    decltype(&scanscam_conv_bwd) conv_back = nullptr;
    decltype(&scanscam_conv_workspace_bytes) conv_workspace = nullptr;
    decltype(&scanscam_norm_bwd) norm_back = nullptr;
    decltype(&scanscam_norm_workspace_bytes) norm_workspace = nullptr;
} operators;

constexpr int64_t kMostStates = 256, kMostTaps = 8, kMostNormChannels = 32768;

// The arguments of one call, looked at one after the other; `ok` says whether it is covered so far.
// An output that the kernels write whole, without the dispatcher's part of at::empty() (0.8 us each against 0.45; modes and the tracer have been asked for).
at::Tensor output(at::IntArrayRef sizes, at::ScalarType type, at::Device device) { return at::detail::empty_cuda(sizes, type, device, std::nullopt); }

struct Arguments {
    PyObject *const *args;
    bool ok;
    bool gradients = false;  // an argument requires one
    at::Tensor first;        // the activations: what the others are compared with

    Arguments(PyObject *const *args, Py_ssize_t nargs, Py_ssize_t expected, int first_at) : args(args)
    {
        ok = nargs == expected && operators.norm && !left_to_python && !modes_active() && !torch::jit::tracer::isTracing() &&
             !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
        if (!ok) return;
        first = tensor(first_at);
        if (!ok || !first.defined()) {
            ok = false;
            return;
        }
        code();
    }
    // An argument that may be None (then undefined).
    at::Tensor tensor(int i)
    {
        if (!ok || args[i] == Py_None) return {};
        if (!THPVariable_CheckExact(args[i])) {
            ok = false;
            return {};
        }
        at::Tensor t = THPVariable_Unpack(args[i]);
        ok = plain(t) && !t._fw_grad(/*level=*/0).defined() && (!first.defined() || t.device() == first.device());
        if (at::GradMode::is_enabled() && t.requires_grad()) gradients = true;
        return t;
    }
    int code()
    {
        const int c = dtype_code(first.scalar_type());
        if (c < 0 || c == SCANSCAM_F64) ok = false;
        return c;
    }
    bool flag(int i)
    {
        const int v = PyObject_IsTrue(args[i]);
        if (v < 0) {
            PyErr_Clear();
            ok = false;
        }
        return v == 1;
    }
    int activation(int i)
    {
        if (args[i] == Py_None) return SCANSCAM_ACT_NONE;
        if (PyUnicode_Check(args[i]) && PyUnicode_CompareWithASCIIString(args[i], "silu") == 0) return SCANSCAM_ACT_SILU;
        ok = false;
        return 0;
    }
    // What one call takes; the Python path says so.
    void sizes(int64_t channels, int64_t tokens, int64_t sequences = 0)
    {
        if (channels > SCANSCAM_MOST_CHANNELS || tokens >= SCANSCAM_MOST_TOKENS || sequences >= SCANSCAM_MOST_TOKENS) ok = false;
    }
    void shape(const at::Tensor &t, at::IntArrayRef sizes)
    {
        if (t.defined() && t.sizes() != sizes) ok = false;
    }
    // [batch, T, ...] (lead 2) or [rows, ...] (lead 1) of the activations' type, unit-stride at the end.
    scanscam_tokens tokens(const at::Tensor &t, int lead)
    {
        scanscam_tokens k{};
        if (!ok || !t.defined()) return k;
        const int64_t token = t.size(lead - 1) > 1 ? t.stride(lead - 1) : 0;  // (a single token's distance to the next may be anything)
        if (t.scalar_type() != first.scalar_type() || (t.size(-1) != 1 && t.stride(-1) != 1) || token >= SCANSCAM_MOST_TOKEN_STRIDE) {
            ok = false;
            return k;
        }
        k.p = t.data_ptr();
        k.batch = lead == 2 ? t.stride(0) : 0;
        k.token = token;
        k.group = t.dim() > lead + 1 ? t.stride(lead) : 0;
        return k;
    }
    scanscam_param parameter(const at::Tensor &t)
    {
        scanscam_param k{};
        if (!ok || !t.defined()) return k;
        const int c = dtype_code(t.scalar_type());
        if (c < 0 || c == SCANSCAM_F64 || !t.is_contiguous()) ok = false;
        k.p = t.data_ptr();
        k.dtype = c;
        return k;
    }
    void *dense(const at::Tensor &t, at::ScalarType type)
    {
        if (!ok || !t.defined()) return nullptr;
        if (t.scalar_type() != type || !t.is_contiguous()) ok = false;
        return t.data_ptr();
    }
    const void *indices(const at::Tensor &t, int32_t *wide)
    {
        *wide = t.defined() && t.scalar_type() == at::kLong;
        return dense(t, *wide ? at::kLong : at::kInt);
    }
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const { return output(sizes, type, first.device()); }
    void *stream() const { return c10::hip::getCurrentHIPStream(first.device().index()).stream(); }
};

void check_launch(int rc, const char *what)
{
    if (rc != SCANSCAM_OK) throw std::runtime_error(std::string("scanscam_") + what + ": " + error_text(rc));
}

// The device that the tensors are on must be the current one when a call is made.
#define SCANSCAM_LAUNCH(call, what)                             \
    {                                                           \
        pybind11::gil_scoped_release no_gil;                    \
        const c10::DeviceGuard guard(in.first.device());        \
        check_launch(call, what);                               \
    }

using torch::autograd::AutogradContext;

// An argument that may be absent, as a node takes it: an undefined tensor has no metadata for the node to record, none at all is no input.
using Maybe = std::optional<at::Tensor>;
Maybe maybe(const at::Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }

// make_fx records ATen calls, of which a launch is none: it would take gradients for constants.
void check_unrecorded(const char *what)
{
    if (c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
        throw std::runtime_error(std::string(what) + ": make_fx cannot record this call, whose kernels are no ATen operators");
}

// What a node saves, with types and shapes (of each tensor its type and sizes, -1 where there is none): a hook on saved tensors may lay out
// what it gives back in its own way, but the kernels take addresses.
std::vector<int64_t> types_and_shapes(const variable_list &tensors)
{
    std::vector<int64_t> all;
    all.reserve(tensors.size() * 5);
    for (const at::Tensor &t : tensors) {
        all.push_back(t.defined() ? (int64_t)t.scalar_type() : -1);
        if (!t.defined()) continue;
        all.push_back(t.dim());
        for (const int64_t n : t.sizes()) all.push_back(n);
    }
    return all;
}
void keep(AutogradContext *ctx, variable_list &&tensors)
{
    ctx->saved_data["meta"] = types_and_shapes(tensors);
    ctx->save_for_backward(std::move(tensors));
}
// ... and what it gets back, for gradients of which one is `grad`.
variable_list returned(AutogradContext *ctx, const at::Tensor &grad, const char *what)
{
    variable_list tensors = ctx->get_saved_variables();
    bool same = types_and_shapes(tensors) == ctx->saved_data["meta"].toIntVector();
    for (const at::Tensor &t : tensors) same = same && (!t.defined() || (plain(t) && t.device() == grad.device()));
    if (!same) {
        std::ostringstream text;
        text << what << ": a tensor that was saved for the backward pass came back with another type or shape, or not on " << grad.device() << " as it was";
        throw std::runtime_error(text.str());
    }
    return tensors;
}

// What a backward call has of its own: outputs, a workspace, gradients as the library takes them.
struct Gradients {
    const at::Tensor &like;
    at::Tensor empty(const at::Tensor &t, at::ScalarType type) const
    {
        return t.defined() ? output(t.sizes(), type, like.device()) : at::Tensor();
    }
    at::Tensor empty(const at::Tensor &t) const { return t.defined() ? empty(t, t.scalar_type()) : at::Tensor(); }
    at::Tensor bytes(size_t n) const { return n != 0 ? output({(int64_t)n}, at::kByte, like.device()) : at::Tensor(); }
    // Zeros where there is no gradient; a copy where the last dimension is not unit-stride or tokens are too far apart.
    at::Tensor tokens(const at::Tensor &g) const { return g.defined() ? near(g) : at::zeros(like.sizes(), like.options()); }
    // What was saved, as the kernels take it: a hook on saved tensors may lay out what it gives back in its own way.
    static at::Tensor near(const at::Tensor &t)
    {
        return !t.defined() || ((t.size(-1) == 1 || t.stride(-1) == 1) && (t.size(1) <= 1 || t.stride(1) < SCANSCAM_MOST_TOKEN_STRIDE)) ? t : t.contiguous();
    }
    static at::Tensor dense(const at::Tensor &t) { return t.defined() ? t.contiguous() : t; }
    static scanscam_tokens view(const at::Tensor &t)
    {
        if (!t.defined()) return {};
        return {t.data_ptr(), t.stride(0), t.size(1) > 1 ? t.stride(1) : 0, t.dim() > 3 ? t.stride(2) : 0};
    }
    static scanscam_param parameter(const at::Tensor &t) { return t.defined() ? scanscam_param{t.data_ptr(), dtype_code(t.scalar_type()), 0} : scanscam_param{}; }
    template <typename T = void> static T *at(const at::Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }
    static at::Tensor as(at::Tensor &&g, const at::Tensor &t) { return g.defined() && g.scalar_type() != t.scalar_type() ? g.to(t.scalar_type()) : std::move(g); }
    void *stream() const { return c10::hip::getCurrentHIPStream(like.device().index()).stream(); }
};

// The gradients, which have none themselves: asking for one is an error, as with a Python function that is differentiable once.
variable_list once(variable_list &&grads, const variable_list &saved, const variable_list &from)
{
    if (!at::GradMode::is_enabled()) return std::move(grads);
    bool any = false;
    for (const variable_list *list : {&saved, &from})
        for (const at::Tensor &t : *list) any = any || (t.defined() && t.requires_grad());
    if (!any) return std::move(grads);
    variable_list given;
    for (const at::Tensor &t : grads)
        if (t.defined()) given.push_back(t.detach().set_requires_grad(true));
    const auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)given.size());
    variable_list marked = (*error)(std::move(given));
    size_t i = 0;
    for (at::Tensor &t : grads)
        if (t.defined()) t = marked[i++];
    return std::move(grads);
}

// The distance between rows where the leading dimensions merge into one level of rows with unit-stride channels, else -1.
int64_t row_stride(const at::Tensor &t)
{
    const int64_t channels = t.size(-1);
    if (t.is_contiguous()) return channels;
    if (channels != 1 && t.stride(-1) != 1) return -1;
    int64_t stride = channels, size = 1;
    bool any = false;
    for (int64_t d = t.dim() - 2; d >= 0; d--) {
        if (t.size(d) == 1) continue;
        if (!any) stride = t.stride(d);
        else if (t.stride(d) != stride * size) return -1;
        any = true;
        size *= t.size(d);
    }
    return stride;
}

struct NormBackward : torch::autograd::Function<NormBackward> {
    struct Done {
        at::Tensor y, sum, rstd;
    };
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const Maybe &residual, Done *done)
    {
        keep(ctx, {residual ? done->sum : x, weight, done->rstd});
        ctx->set_materialize_grads(false);
        ctx->saved_data["dtype"] = (int64_t)x.scalar_type();
        ctx->saved_data["residual"] = residual.has_value();
        return residual ? variable_list{done->y, done->sum} : variable_list{done->y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        check_unrecorded("rms_norm");
        const bool added = ctx->saved_data["residual"].toBool();
        at::Tensor gy = grads[0], gsum = added ? grads[1] : at::Tensor();
        if (!gy.defined() && !gsum.defined()) return {{}, {}, {}, {}};
        const variable_list saved = returned(ctx, gy.defined() ? gy : gsum, "rms_norm");
        const auto type = (at::ScalarType)ctx->saved_data["dtype"].toInt();
        // (the library takes rows of x at any distance, those of a sum dense)
        const at::Tensor kept = !added && row_stride(saved[0]) >= 0 ? saved[0] : saved[0].contiguous(), weight = Gradients::dense(saved[1]), rstd = Gradients::dense(saved[2]);
        const c10::DeviceGuard guard(kept.device());
        const Gradients make{kept};
        gy = gy.defined() ? gy.contiguous() : at::zeros(kept.sizes(), kept.options().dtype(type));
        if (gsum.defined()) gsum = gsum.contiguous();
        scanscam_norm a{};
        a.channels = kept.size(-1);
        a.rows = kept.numel() / a.channels;
        a.dtype = dtype_code(type);
        a.weight = Gradients::parameter(weight);
        a.rstd = Gradients::at<float>(rstd);
        a.x = kept.data_ptr();
        a.x_stride = row_stride(kept);
        at::Tensor gx = make.empty(kept, type), gresidual, gweight = make.empty(weight, at::kFloat);
        if (added) {
            a.residual = a.sum = kept.data_ptr();
            a.residual_dtype = dtype_code(kept.scalar_type());
            a.gsum = Gradients::at(gsum);
            gresidual = kept.scalar_type() == type ? gx : make.empty(kept);  // (where the types agree the two are the same values)
            if (kept.scalar_type() != type) a.gresidual = gresidual.data_ptr();
        }
        a.gy = gy.data_ptr();
        a.gx = gx.data_ptr();
        a.gweight = Gradients::at<float>(gweight);
        a.workspace_bytes = operators.norm_workspace(&a);
        const at::Tensor workspace = make.bytes(a.workspace_bytes);
        a.workspace = Gradients::at(workspace);
        check_launch(operators.norm_back(&a, make.stream()), "norm_bwd");
        return once({gx, Gradients::as(std::move(gweight), weight), gresidual, {}}, saved, grads);
    }
};

struct ConvBackward : torch::autograd::Function<ConvBackward> {
    struct Done {
        at::Tensor y, state, offsets;
        int activation;
    };
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const Maybe &bias, const Maybe &state, Done *done)
    {
        keep(ctx, {x, weight, bias.value_or(at::Tensor()), state.value_or(at::Tensor()), done->offsets});
        ctx->set_materialize_grads(false);
        ctx->saved_data["activation"] = (int64_t)done->activation;
        return done->state.defined() ? variable_list{done->y, done->state} : variable_list{done->y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        check_unrecorded("causal_conv");
        at::Tensor gstate_out = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!grads[0].defined() && !gstate_out.defined()) return {{}, {}, {}, {}, {}};
        const variable_list saved = returned(ctx, grads[0].defined() ? grads[0] : gstate_out, "causal_conv");
        const at::Tensor x = Gradients::near(saved[0]), weight = Gradients::dense(saved[1]), bias = Gradients::dense(saved[2]), state = Gradients::dense(saved[3]),
                         offsets = Gradients::dense(saved[4]);
        const c10::DeviceGuard guard(x.device());
        const Gradients make{x};
        const at::Tensor gy = make.tokens(grads[0]);
        if (gstate_out.defined()) gstate_out = gstate_out.contiguous();
        at::Tensor gx = make.empty(x), gweight = make.empty(weight, at::kFloat), gbias = make.empty(bias, at::kFloat);
        // (inputs of the node are counted without the absent ones)
        at::Tensor gstate = state.defined() && ctx->needs_input_grad(2 + bias.defined()) ? make.empty(state) : at::Tensor();
        scanscam_conv a{};
        a.batch = x.size(0);
        a.T = x.size(1);
        a.channels = x.size(2);
        a.K = weight.size(1);
        a.sequences = offsets.defined() ? offsets.numel() - 1 : a.batch;
        a.offsets = Gradients::at(offsets);
        a.offsets64 = offsets.defined() && offsets.scalar_type() == at::kLong;
        a.dtype = dtype_code(x.scalar_type());
        a.activation = (int32_t)ctx->saved_data["activation"].toInt();
        a.x = Gradients::view(x);
        a.weight = Gradients::parameter(weight);
        a.bias = Gradients::parameter(bias);
        a.state_in = Gradients::at(state);
        a.gy = Gradients::view(gy);
        a.gx = Gradients::view(gx);
        a.gweight = Gradients::at<float>(gweight);
        a.gbias = Gradients::at<float>(gbias);
        a.gstate_out = Gradients::at(gstate_out);
        a.gstate_in = Gradients::at(gstate);
        a.workspace_bytes = operators.conv_workspace(&a);
        const at::Tensor workspace = make.bytes(a.workspace_bytes);
        a.workspace = Gradients::at(workspace);
        check_launch(operators.conv_back(&a, make.stream()), "conv_bwd");
        return once({gx, Gradients::as(std::move(gweight), weight), Gradients::as(std::move(gbias), bias), gstate, {}}, saved, grads);
    }
};

struct SelectiveBackward : torch::autograd::Function<SelectiveBackward> {
    struct Done {
        at::Tensor y, state, saved, offsets;
        bool softplus;
    };
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &dt, const at::Tensor &A, const at::Tensor &B, const at::Tensor &C,
                                 const Maybe &D, const Maybe &z, const Maybe &bias, const Maybe &state, Done *done)
    {
        const at::Tensor none;
        keep(ctx, {x, dt, A, B, C, D.value_or(none), z.value_or(none), bias.value_or(none), state.value_or(none), done->offsets, done->saved});
        ctx->set_materialize_grads(false);
        ctx->saved_data["softplus"] = done->softplus;
        return done->state.defined() ? variable_list{done->y, done->state} : variable_list{done->y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        check_unrecorded("selective_scan");
        at::Tensor gstate_out = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!grads[0].defined() && !gstate_out.defined()) return variable_list(10);
        const variable_list kept = returned(ctx, grads[0].defined() ? grads[0] : gstate_out, "selective_scan");
        const auto near = [&](int i) { return Gradients::near(kept[i]); };
        const auto dense = [&](int i) { return Gradients::dense(kept[i]); };
        const at::Tensor x = near(0), dt = near(1), A = dense(2), B = near(3), C = near(4), D = dense(5), z = near(6), bias = dense(7), state = dense(8),
                         offsets = dense(9), saved = dense(10);
        const c10::DeviceGuard guard(x.device());
        const Gradients make{x};
        const at::Tensor gy = make.tokens(grads[0]);
        if (gstate_out.defined()) gstate_out = gstate_out.contiguous();
        at::Tensor gx = make.empty(x), gdt = make.empty(dt), gB = make.empty(B), gC = make.empty(C), gz = make.empty(z);
        at::Tensor gA = make.empty(A, at::kFloat), gD = make.empty(D, at::kFloat), gbias = make.empty(bias, at::kFloat);
        at::Tensor gstate = state.defined() && ctx->needs_input_grad(5 + D.defined() + z.defined() + bias.defined()) ? make.empty(state) : at::Tensor();
        scanscam_selective a{};
        a.batch = x.size(0);
        a.T = x.size(1);
        a.channels = x.size(2);
        a.N = A.size(1);
        a.groups = B.dim() == 4 ? B.size(2) : 1;
        a.sequences = offsets.defined() ? offsets.numel() - 1 : a.batch;
        a.offsets = Gradients::at(offsets);
        a.offsets64 = offsets.defined() && offsets.scalar_type() == at::kLong;
        a.dtype = dtype_code(x.scalar_type());
        a.softplus = ctx->saved_data["softplus"].toBool();
        a.x = Gradients::view(x);
        a.dt = Gradients::view(dt);
        a.B = Gradients::view(B);
        a.C = Gradients::view(C);
        a.z = Gradients::view(z);
        a.A = Gradients::parameter(A);
        a.D = Gradients::parameter(D);
        a.dt_bias = Gradients::parameter(bias);
        a.state_in = Gradients::at<float>(state);
        a.saved = Gradients::at(saved);
        a.gy = Gradients::view(gy);
        a.gx = Gradients::view(gx);
        a.gdt = Gradients::view(gdt);
        a.gB = Gradients::view(gB);
        a.gC = Gradients::view(gC);
        a.gz = Gradients::view(gz);
        a.gA = Gradients::at<float>(gA);
        a.gD = Gradients::at<float>(gD);
        a.gdt_bias = Gradients::at<float>(gbias);
        a.gstate_out = Gradients::at<float>(gstate_out);
        a.gstate_in = Gradients::at<float>(gstate);
        a.workspace_bytes = operators.selective_workspace(&a, SCANSCAM_BACKWARD);
        const at::Tensor workspace = make.bytes(a.workspace_bytes);
        a.workspace = Gradients::at(workspace);
        check_launch(operators.selective_back(&a, make.stream()), "selective_bwd");
        return once({gx, gdt, Gradients::as(std::move(gA), A), gB, gC, Gradients::as(std::move(gD), D), gz, Gradients::as(std::move(gbias), bias), gstate, {}}, kept, grads);
    }
};

// norm(x, weight, residual, eps, quant code): the tuple that rms_norm returns, or y alone.
PyObject *norm(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    Arguments in(args, nargs, 5, 0);
    if (!in.ok) Py_RETURN_NONE;
    const at::Tensor &x = in.first, weight = in.tensor(1), residual = in.tensor(2);
    const int64_t dims = x.dim();
    if (!in.ok || dims < 1 || x.numel() == 0 || x.size(-1) > kMostNormChannels || !weight.defined()) Py_RETURN_NONE;
    const int64_t channels = x.size(-1);
    in.shape(weight, {channels});
    in.shape(residual, x.sizes());
    scanscam_norm a{};
    a.rows = x.numel() / channels;
    a.channels = channels;
    in.sizes(channels, a.rows);
    a.x = x.data_ptr();
    a.x_stride = row_stride(x);
    if (a.x_stride < 0) in.ok = false;
    a.weight = in.parameter(weight);
    a.eps = (float)PyFloat_AsDouble(args[3]);
    a.dtype = in.code();
    const long quant = PyLong_AsLong(args[4]);
    if (in.gradients && quant != 0) Py_RETURN_NONE;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (quant != 0 && quant != SCANSCAM_I8 && quant != SCANSCAM_F8) Py_RETURN_NONE;
    a.out_dtype = quant != 0 ? (int)quant : a.dtype;
    at::Tensor sum, scale;
    if (residual.defined()) {
        a.residual_dtype = dtype_code(residual.scalar_type());
        if (a.residual_dtype < 0 || a.residual_dtype == SCANSCAM_F64) in.ok = false;
        a.residual = residual.data_ptr();
        a.residual_stride = row_stride(residual);
        if (a.residual_stride < 0) in.ok = false;
    }
    if (!in.ok) Py_RETURN_NONE;
    at::Tensor y = in.empty(x.sizes(), quant == SCANSCAM_I8 ? at::kChar : quant == SCANSCAM_F8 ? at::kFloat8_e4m3fn : x.scalar_type());
    a.y = y.data_ptr();
    if (residual.defined()) {
        sum = in.empty(x.sizes(), residual.scalar_type());
        a.sum = sum.data_ptr();
    }
    if (quant != 0) {
        scale = in.empty(x.sizes().slice(0, (size_t)dims - 1), at::kFloat);
        a.scale = static_cast<float *>(scale.data_ptr());
    }
    at::Tensor rstd;
    if (in.gradients) {
        rstd = in.empty({a.rows}, at::kFloat);
        a.rstd = static_cast<float *>(rstd.data_ptr());
    }
    SCANSCAM_LAUNCH(operators.norm(&a, in.stream()), "norm_fwd")
    if (in.gradients) {
        NormBackward::Done done{y, sum, rstd};
        variable_list out = NormBackward::apply(x, weight, maybe(residual), &done);
        y = out[0];
        if (residual.defined()) sum = out[1];
    }
    if (quant == 0 && !residual.defined()) return THPVariable_Wrap(std::move(y));
    pybind11::list out;
    for (at::Tensor *t : {&y, &scale, &sum})
        if (t->defined()) out.append(pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(*t))));
    return PyList_AsTuple(out.ptr());
    END_HANDLE_TH_ERRORS
}

PyObject *with_state(at::Tensor &&y, at::Tensor &&state)
{
    pybind11::object a = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(y)));
    if (!state.defined()) return a.release().ptr();
    pybind11::object b = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(state)));
    return PyTuple_Pack(2, a.ptr(), b.ptr());
}

// conv(x, weight, bias, activation, state, offsets, return_state)
PyObject *conv(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    Arguments in(args, nargs, 7, 0);
    if (!in.ok) Py_RETURN_NONE;
    const at::Tensor &x = in.first, weight = in.tensor(1), bias = in.tensor(2), state = in.tensor(4), offsets = in.tensor(5);
    if (!in.ok || x.dim() != 3 || x.numel() == 0 || !weight.defined() || weight.dim() != 2 || (offsets.defined() && (offsets.dim() != 1 || offsets.numel() < 2 || x.size(0) != 1)))
        Py_RETURN_NONE;
    scanscam_conv a{};
    a.batch = x.size(0);
    a.T = x.size(1);
    a.channels = x.size(2);
    a.K = weight.size(1);
    a.sequences = offsets.defined() ? offsets.numel() - 1 : a.batch;
    if (a.K < 1 || a.K > kMostTaps) Py_RETURN_NONE;
    in.sizes(a.channels, a.batch * a.T, a.sequences);
    in.shape(weight, {a.channels, a.K});
    in.shape(bias, {a.channels});
    in.shape(state, {a.sequences, a.K - 1, a.channels});
    a.offsets = in.indices(offsets, &a.offsets64);
    a.dtype = in.code();
    a.activation = in.activation(3);
    a.x = in.tokens(x, 2);
    a.weight = in.parameter(weight);
    a.bias = in.parameter(bias);
    a.state_in = in.dense(state, x.scalar_type());
    const bool keep = in.flag(6);
    if (!in.ok) Py_RETURN_NONE;
    at::Tensor y = in.empty(x.sizes(), x.scalar_type()), new_state;
    a.y = in.tokens(y, 2);
    if (keep) {
        new_state = in.empty({a.sequences, a.K - 1, a.channels}, x.scalar_type());
        a.state_out = new_state.data_ptr();
    }
    SCANSCAM_LAUNCH(operators.conv(&a, in.stream()), "conv_fwd")
    if (in.gradients) {
        ConvBackward::Done done{y, new_state, offsets, a.activation};
        variable_list out = ConvBackward::apply(x, weight, maybe(bias), maybe(state), &done);
        y = out[0];
        if (keep) new_state = out[1];
    }
    return with_state(std::move(y), std::move(new_state));
    END_HANDLE_TH_ERRORS
}

// conv_step(state, x, weight, bias, activation, slots)
PyObject *conv_step(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    Arguments in(args, nargs, 6, 1);
    if (!in.ok) Py_RETURN_NONE;
    const at::Tensor &x = in.first, state = in.tensor(0), weight = in.tensor(2), bias = in.tensor(3), slots = in.tensor(5);
    if (!in.ok || in.gradients || x.dim() != 2 || x.numel() == 0 || !state.defined() || state.dim() != 3 || !weight.defined() || weight.dim() != 2) Py_RETURN_NONE;
    scanscam_conv_step a{};
    a.rows = x.size(0);
    a.channels = x.size(1);
    a.K = weight.size(1);
    a.slots = state.size(0);
    if (a.K < 1 || a.K > kMostTaps || (!slots.defined() && a.slots != a.rows)) Py_RETURN_NONE;
    in.sizes(a.channels, a.rows);
    in.shape(weight, {a.channels, a.K});
    in.shape(bias, {a.channels});
    in.shape(state, {a.slots, a.K - 1, a.channels});
    in.shape(slots, {a.rows});
    a.slot = in.indices(slots, &a.slot64);
    a.dtype = in.code();
    a.activation = in.activation(4);
    a.x = in.tokens(x, 1);
    a.weight = in.parameter(weight);
    a.bias = in.parameter(bias);
    a.state = in.dense(state, x.scalar_type());
    if (!in.ok) Py_RETURN_NONE;
    at::Tensor y = in.empty(x.sizes(), x.scalar_type());
    a.y = in.tokens(y, 1);
    SCANSCAM_LAUNCH(operators.conv_step(&a, in.stream()), "conv_step_fwd")
    state.unsafeGetTensorImpl()->bump_version();  // (written in place)
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// What the selective scan's two forms have in common: x, dt, A, B, C, D, z, dt_bias from `at` on.
template <typename Args> bool selective_arguments(Arguments &in, int at, int lead, Args &a)
{
    const at::Tensor &x = in.first, dt = in.tensor(at + 1), A = in.tensor(at + 2), B = in.tensor(at + 3), C = in.tensor(at + 4), D = in.tensor(at + 5),
                     z = in.tensor(at + 6), bias = in.tensor(at + 7);
    if (!in.ok || x.dim() != lead + 1 || x.numel() == 0 || !dt.defined() || !A.defined() || !B.defined() || !C.defined() || A.dim() != 2 ||
        (B.dim() != lead + 1 && B.dim() != lead + 2))
        return false;
    a.channels = x.size(-1);
    a.N = A.size(1);
    a.groups = B.dim() == lead + 2 ? B.size(lead) : 1;
    if (a.N < 1 || a.N > kMostStates || a.groups < 1 || a.channels % a.groups != 0 || B.size(-1) != a.N) return false;
    if (a.groups * a.N >= SCANSCAM_MOST_TOKEN_STRIDE) return false;  // (gradients of B and C need a layout of their own)
    for (int d = 0; d < lead; d++)
        if (B.size(d) != x.size(d)) return false;
    in.shape(dt, x.sizes());
    in.shape(z, x.sizes());
    in.shape(A, {a.channels, a.N});
    in.shape(C, B.sizes());
    in.shape(D, {a.channels});
    in.shape(bias, {a.channels});
    a.dtype = in.code();
    a.x = in.tokens(x, lead);
    a.dt = in.tokens(dt, lead);
    a.B = in.tokens(B, lead);
    a.C = in.tokens(C, lead);
    a.z = in.tokens(z, lead);
    a.A = in.parameter(A);
    a.D = in.parameter(D);
    a.dt_bias = in.parameter(bias);
    return in.ok;
}

// selective(x, dt, A, B, C, D, z, dt_bias, softplus, state, offsets, return_state)
PyObject *selective(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    Arguments in(args, nargs, 12, 0);
    if (!in.ok) Py_RETURN_NONE;
    const at::Tensor &x = in.first, state = in.tensor(9), offsets = in.tensor(10);
    scanscam_selective a{};
    if (!in.ok || !selective_arguments(in, 0, 2, a) || (offsets.defined() && (offsets.dim() != 1 || offsets.numel() < 2 || x.size(0) != 1))) Py_RETURN_NONE;
    a.batch = x.size(0);
    a.T = x.size(1);
    a.sequences = offsets.defined() ? offsets.numel() - 1 : a.batch;
    in.sizes(a.channels, a.batch * a.T, a.sequences);
    in.shape(state, {a.sequences, a.channels, a.N});
    a.offsets = in.indices(offsets, &a.offsets64);
    a.state_in = static_cast<const float *>(in.dense(state, at::kFloat));
    a.softplus = in.flag(8);
    const bool keep = in.flag(11);
    if (!in.ok) Py_RETURN_NONE;
    at::Tensor y = in.empty(x.sizes(), x.scalar_type()), new_state, workspace;
    a.y = in.tokens(y, 2);
    if (keep) {
        new_state = in.empty({a.sequences, a.channels, a.N}, at::kFloat);
        a.state_out = static_cast<float *>(new_state.data_ptr());
    }
    at::Tensor saved;
    if (in.gradients) {
        saved = in.empty({(int64_t)operators.selective_saved(&a)}, at::kByte);
        a.saved = saved.data_ptr();
    }
    a.workspace_bytes = operators.selective_workspace(&a, SCANSCAM_FORWARD);
    if (a.workspace_bytes != 0) {
        workspace = in.empty({(int64_t)a.workspace_bytes}, at::kByte);
        a.workspace = workspace.data_ptr();
    }
    SCANSCAM_LAUNCH(operators.selective(&a, in.stream()), "selective_fwd")
    if (in.gradients) {
        SelectiveBackward::Done done{y, new_state, saved, offsets, a.softplus != 0};
        const auto given = [&](int i) { return args[i] == Py_None ? Maybe() : Maybe(THPVariable_Unpack(args[i])); };
        variable_list out = SelectiveBackward::apply(x, *given(1), *given(2), *given(3), *given(4), given(5), given(6), given(7), maybe(state), &done);
        y = out[0];
        if (keep) new_state = out[1];
    }
    return with_state(std::move(y), std::move(new_state));
    END_HANDLE_TH_ERRORS
}

// selective_step(state, x, dt, A, B, C, D, z, dt_bias, softplus, slots)
PyObject *selective_step(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    Arguments in(args, nargs, 11, 1);
    if (!in.ok) Py_RETURN_NONE;
    const at::Tensor &x = in.first, state = in.tensor(0), slots = in.tensor(10);
    scanscam_selective_step a{};
    if (!in.ok || !state.defined() || state.dim() != 3 || !selective_arguments(in, 1, 1, a) || in.gradients) Py_RETURN_NONE;
    a.rows = x.size(0);
    a.slots = state.size(0);
    if (!slots.defined() && a.slots != a.rows) Py_RETURN_NONE;
    in.sizes(a.channels, a.rows);
    in.shape(state, {a.slots, a.channels, a.N});
    in.shape(slots, {a.rows});
    a.slot = in.indices(slots, &a.slot64);
    a.softplus = in.flag(9);
    a.state = static_cast<float *>(in.dense(state, at::kFloat));
    if (!in.ok) Py_RETURN_NONE;
    at::Tensor y = in.empty(x.sizes(), x.scalar_type());
    a.y = in.tokens(y, 1);
    SCANSCAM_LAUNCH(operators.selective_step(&a, in.stream()), "selective_step_fwd")
    state.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// bind_operators(selective_fwd, selective_workspace_bytes, selective_step_fwd, conv_fwd, conv_step_fwd, norm_fwd, and of the backward calls
// selective_bwd, selective_saved_bytes, conv_bwd, conv_workspace_bytes, norm_bwd, norm_workspace_bytes): addresses.
PyObject *bind_operators(PyObject *, PyObject *args)
{
    unsigned long long p[12];
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7, p + 8, p + 9, p + 10, p + 11)) return nullptr;
    operators.selective_back = reinterpret_cast<decltype(operators.selective_back)>(p[6]);
    operators.selective_saved = reinterpret_cast<decltype(operators.selective_saved)>(p[7]);
    operators.conv_back = reinterpret_cast<decltype(operators.conv_back)>(p[8]);
    operators.conv_workspace = reinterpret_cast<decltype(operators.conv_workspace)>(p[9]);
    operators.norm_back = reinterpret_cast<decltype(operators.norm_back)>(p[10]);
    operators.norm_workspace = reinterpret_cast<decltype(operators.norm_workspace)>(p[11]);
    operators.selective = reinterpret_cast<decltype(operators.selective)>(p[0]);
    operators.selective_workspace = reinterpret_cast<decltype(operators.selective_workspace)>(p[1]);
    operators.selective_step = reinterpret_cast<decltype(operators.selective_step)>(p[2]);
    operators.conv = reinterpret_cast<decltype(operators.conv)>(p[3]);
    operators.conv_step = reinterpret_cast<decltype(operators.conv_step)>(p[4]);
    operators.norm = reinterpret_cast<decltype(operators.norm)>(p[5]);
    Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)> PyCFunction fast()
{
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {{"scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scan)), METH_FASTCALL, nullptr},
                         {"leave_to_python", leave_to_python, METH_O, nullptr},
                         {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
                         {"backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(backward)), METH_FASTCALL, nullptr},
                         {"bind", bind, METH_VARARGS, nullptr},
                         {"norm", fast<norm>(), METH_FASTCALL, nullptr},
                         {"conv", fast<conv>(), METH_FASTCALL, nullptr},
                         {"conv_step", fast<conv_step>(), METH_FASTCALL, nullptr},
                         {"selective", fast<selective>(), METH_FASTCALL, nullptr},
                         {"selective_step", fast<selective_step>(), METH_FASTCALL, nullptr},
                         {"bind_operators", bind_operators, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding()
{
    PyObject *m = PyModule_Create(&module);
    // The PyTorch it was compiled against, for hip.py to compare: its C++ API is not stable between versions.
    if (m && PyModule_AddStringConstant(m, "torch_version", SCANSCAM_TORCH_VERSION) != 0) Py_CLEAR(m);
    return m;
}
