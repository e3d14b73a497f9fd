// Host path of the Python package in native code: from a module call to the launch without the interpreter in between.
//
// A decode kernel runs for 3 ... 12 us, so what a call costs on the host decides how fast eager code decodes.  The same
// steps written in Python (views, checks, the output tensor, a ctypes call with sixteen arguments) took 8 ... 9 us a
// call, and an autograd node written in Python about 50 us per forward + backward.  Here: a layer's buffers are looked at
// on every call (dtype, shape, strides, device, address: about 0.1 us, so nothing about them has to be remembered), the
// output comes straight from the caching allocator, and the node that backward runs is a C++ node.
//
// The kernels are reached through function pointers of the C ABI (bind(), called once by hip_loader), so this file
// neither links the kernel library nor knows where it lies.  Anything a function here does not take - CPU tensors,
// tensor subclasses, buffers of another dtype or layout - it answers with None, and the Python code that it stands in
// front of deals with the call and raises what has to be raised.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/bitween_hip.h"

namespace {

using at::Tensor;

struct Library {
    decltype(&bw_qlinear_ws) qlinear = nullptr;
    decltype(&bw_qlinear_workspace_bytes) qlinear_ws_bytes = nullptr;
    decltype(&bw_cast_bf16_f16) cast = nullptr;
    decltype(&bw_qdgrad) qdgrad = nullptr;
    decltype(&bw_qdgrad_workspace_bytes) qdgrad_ws_bytes = nullptr;
    decltype(&bw_qdgrad_tile_rows) qdgrad_tile_rows = nullptr;
    decltype(&bw_quantize_pack_add) quantize = nullptr;
    decltype(&bw_dequantize) dequantize = nullptr;
    decltype(&bw_rotate_heads) rotate = nullptr;
    decltype(&bw_rotate_heads_grad) rotate_grad = nullptr;
    decltype(&bw_rotate_heads_grad_workspace_bytes) rotate_grad_ws_bytes = nullptr;
    decltype(&bw_cache_write) cache_write = nullptr;
    decltype(&bw_cache_read) cache_read = nullptr;
    decltype(&bw_cache_attention) attention = nullptr;
    decltype(&bw_cache_attention_workspace_bytes) attention_ws_bytes = nullptr;
} lib;

PyObject* g_check = nullptr;          // Python: check(status, entry point's name) raises for a status other than 0
PyObject* g_limits = nullptr;         // Python: the dict with the row limits of the fused input gradient

PyObject *s_fused_rows, *s_fused_large_rows;
PyObject *s_buffers, *s_qweight, *s_scale, *s_zero, *s_bias, *s_bits, *s_group;

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return BW_F16;
        case at::kBFloat16: return BW_BF16;
        case at::kFloat: return BW_F32;
        case at::kInt: return BW_I32;
        case at::kDouble: return BW_F64;
        default: return -1;
    }
}

at::ScalarType dtype_of(int code) {
    switch (code) {
        case BW_F16: return at::kHalf;
        case BW_BF16: return at::kBFloat16;
        case BW_F32: return at::kFloat;
        case BW_F64: return at::kDouble;
        default: return at::kInt;
    }
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline Tensor empty(at::IntArrayRef sizes, at::ScalarType t, const at::Device& dev) {
    return Tensor(at::detail::empty_cuda(sizes, t, dev, std::nullopt));
}

inline void* stream_of(at::DeviceIndex index) { return (void*)c10::hip::getCurrentHIPStream(index).stream(); }

// The device of a call made current, only where it is not already.
struct OnDevice {
    std::optional<c10::DeviceGuard> guard;
    explicit OnDevice(const at::Device& d) {
        if (c10::hip::current_device() != d.index()) guard.emplace(d);
    }
};

// The interpreter lock given up while a call allocates, plans and launches: a full queue or an allocator that goes to the driver would
// hold every other Python thread up.  Nothing between here and the end of its scope touches a Python object.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// The row limits as they are now (0 = not a number: no row runs fused); takes the interpreter lock where the thread does not hold it.
struct FusedRows {
    int64_t always = 0, large = 0;
    FusedRows() {
        const PyGILState_STATE state = PyGILState_Ensure();
        always = read(s_fused_rows);
        large = read(s_fused_large_rows);
        PyGILState_Release(state);
    }
    static int64_t read(PyObject* name) {
        PyObject* v = g_limits ? PyDict_GetItemWithError(g_limits, name) : nullptr;
        const long long rows = v && PyLong_Check(v) ? PyLong_AsLongLong(v) : 0;
        if (PyErr_Occurred()) PyErr_Clear();
        return rows < 0 ? 0 : rows;
    }
};

struct Layer {
    const void *qweight, *scale, *zero, *bias;
    int64_t n, k;
    int bits, group;
    at::DeviceIndex device;
};

// What the kernels ask of a layer's buffers; false = the general Python path has to look at them.
bool layer_of(const Tensor& qweight, const Tensor& scale, const Tensor& zero, const Tensor* bias, int64_t bits, int64_t group, Layer& l) {
    if (!lib.qlinear || (bits != 2 && bits != 4 && bits != 8) || group < 1) return false;
    if (!qweight.is_cuda() || !qweight.has_storage() || qweight.scalar_type() != at::kInt || qweight.dim() != 2 || !qweight.is_contiguous()) return false;
    const int64_t n = qweight.size(0), k = qweight.size(1) * (32 / bits);
    if (n < 1 || k < 1 || k % group) return false;
    for (const Tensor* t : {&scale, &zero})
        if (t->device() != qweight.device() || t->scalar_type() != at::kHalf || t->dim() != 2 || !t->is_contiguous() || t->size(0) != n ||
            t->size(1) != k / group)
            return false;
    if (bias && (bias->device() != qweight.device() || bias->scalar_type() != at::kHalf || bias->dim() != 1 || bias->size(0) != n ||
                 !bias->is_contiguous()))
        return false;
    l = {qweight.const_data_ptr(), scale.const_data_ptr(), zero.const_data_ptr(), bias ? bias->const_data_ptr() : nullptr,
         n, k, (int)bits, (int)group, qweight.device().index()};
    return true;
}

// x.to(float16) of a bfloat16 matrix [m, k] with row pitch ldx: the library's streaming kernel where the layout qualifies.
Tensor cast_to_f16(const Tensor& x, int64_t m, int64_t k, int64_t ldx, void* stream) {
    if (k % 8 == 0 && ldx % 8 == 0 && aligned16(x.const_data_ptr())) {
        Tensor y = empty({m, k}, at::kHalf, x.device());
        if (lib.cast(x.const_data_ptr(), m, k, ldx, y.mutable_data_ptr(), k, stream) == BW_OK) return y;
    }
    return x.to(at::kHalf).contiguous();
}

// y = x W16^T (+ bias); the result keeps x's leading dimensions.  An undefined tensor with status 0 = not taken here.
Tensor linear(const Layer& l, Tensor x, int& status, const char*& what) {
    status = 0;
    if (!x.is_cuda() || x.device().index() != l.device || x.dim() < 1 || x.size(-1) != l.k || x.numel() == 0) return {};
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = l.n;
    OnDevice on(x.device());
    at::ScalarType t = x.scalar_type();
    if (t != at::kHalf && t != at::kBFloat16) {
        x = x.to(at::kHalf);
        t = at::kHalf;
    }
    const int64_t m = x.numel() / l.k;
    int64_t ldx = l.k;
    if (!x.is_contiguous()) {
        if (x.dim() != 2) x = x.reshape({m, l.k});
        if (x.stride(1) == 1 && x.stride(0) >= l.k) ldx = x.stride(0);
        else x = x.contiguous();
    }
    if ((ldx * 2) % 16 || !aligned16(x.const_data_ptr())) {
        x = x.clone(at::MemoryFormat::Contiguous);
        ldx = l.k;
    }
    void* stream = stream_of(l.device);
    Tensor y = empty(shape, at::kHalf, x.device());
    what = "bw_qlinear_ws";
    auto launch = [&](int act) {
        const size_t bytes = lib.qlinear_ws_bytes(m, l.n, l.k, l.bits, l.group, act);
        Tensor ws;
        if (bytes) ws = empty({(int64_t)bytes}, at::kByte, x.device());
        return lib.qlinear(x.const_data_ptr(), act, m, l.k, ldx, (const int32_t*)l.qweight, l.scale, l.zero, l.bias, l.n, l.bits, l.group,
                           y.mutable_data_ptr(), l.n, bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream);
    };
    status = launch(t == at::kHalf ? BW_F16 : BW_BF16);
    if (t == at::kBFloat16 && (status == BW_EUNSUPPORTED || status == BW_EALIGN || status == BW_EWORKSPACE)) {
        x = cast_to_f16(x, m, l.k, ldx, stream);               // a shape or layout that wants float16 in memory
        ldx = l.k;
        status = launch(BW_F16);
    }
    return y;
}

// grad_x = grad_y @ W, W the dequantised weight in grad_y's dtype (bitween/modules.py:108-141).  float16 / bfloat16
// gradients run the fused kernel - up to `fused.always` rows always, up to `fused.large` where the library plans its
// 256 x 256 kernel - and dequantise + library GEMM beyond, which is faster there; so does a backward that is itself
// recorded (create_graph).
Tensor input_grad(const Tensor& go, const Tensor& qweight, const Tensor& scale, const Tensor& zero, int bits, int group, const FusedRows& fused) {
    const int64_t n = qweight.size(0), k = qweight.size(1) * (32 / bits);
    OnDevice on(go.device());
    void* stream = stream_of(go.device().index());
    const at::ScalarType t = go.scalar_type();
    const int64_t m = go.numel() / n;
    const bool recorded = c10::GradMode::is_enabled() && go.requires_grad();
    if ((t == at::kHalf || t == at::kBFloat16) && !recorded && m > 0 &&
        (m <= fused.always || (m <= fused.large && lib.qdgrad_tile_rows(m, n, k, bits, group) == 257))) {
        Tensor g = go;
        int64_t ldg = n;
        if (!g.is_contiguous()) {
            if (g.dim() != 2) g = g.reshape({m, n});
            if (g.stride(1) == 1 && g.stride(0) >= n) ldg = g.stride(0);
            else g = g.contiguous();
        }
        if (n >= 32) {
            c10::SmallVector<int64_t, 5> shape(go.sizes().begin(), go.sizes().end());
            shape.back() = k;
            Tensor gx = empty(shape, t, go.device());
            const size_t bytes = lib.qdgrad_ws_bytes(m, n, k, bits, group);
            Tensor ws;
            if (bytes) ws = empty({(int64_t)bytes}, at::kByte, go.device());
            const int st = lib.qdgrad(g.const_data_ptr(), dtype_code(t), m, n, ldg, (const int32_t*)qweight.const_data_ptr(),
                                      scale.const_data_ptr(), zero.const_data_ptr(), k, bits, group, gx.mutable_data_ptr(), k,
                                      bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream);
            if (st == BW_OK) return gx;
            TORCH_CHECK(st == BW_EUNSUPPORTED || st == BW_EALIGN, "bw_qdgrad failed (status ", st, ")");
        }
    }
    // W = scale * (q - zp) in float32, cast to grad_output's dtype: the float32 product is exact, so dequantising straight
    // to that dtype gives the same bits
    const at::ScalarType wt = (t == at::kHalf || t == at::kBFloat16 || t == at::kFloat) ? t : at::kFloat;
    Tensor w = empty({n, k}, wt, go.device());
    const int st = lib.dequantize((const int32_t*)qweight.const_data_ptr(), scale.const_data_ptr(), BW_F16, zero.const_data_ptr(), BW_F16, n, k,
                                  bits, group, w.mutable_data_ptr(), dtype_code(wt), k, stream);
    TORCH_CHECK(st == BW_OK, "bw_dequantize failed (status ", st, ")");
    return at::matmul(go, wt == t ? w : w.to(t));
}

// The node of a recorded forward, in the likeness of QuantizedLinearFunction's: its name, what it saves (x too, so that a change of x in
// place is noticed, and saved-tensor hooks see it) and the edges it has.
struct QuantizedLinearBackward : public torch::autograd::Node {
    enum { X, QWEIGHT, SCALE, ZERO, BIAS };
    torch::autograd::SavedVariable saved[5];
    bool has_bias = false;
    int bits = 0, group = 0;
    std::string name() const override { return "QuantizedLinearFunctionBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : saved) v.reset_data();
    }
    std::array<Tensor, 5> unpack() const {
        std::array<Tensor, 5> t;
        for (int i = 0; i < (has_bias ? 5 : 4); i++) t[i] = saved[i].unpack();
        return t;
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        const FusedRows fused;
        std::lock_guard<std::mutex> lock(mutex_);
        const auto t = unpack();
        torch::autograd::variable_list out(has_bias ? 5 : 4);
        if (!task_should_compute_output(0)) return out;
        const Tensor go = grads[0].defined() ? grads[0] : input_metadata(0).zeros_like();
        out[0] = input_grad(go, t[QWEIGHT].contiguous(), t[SCALE].contiguous(), t[ZERO].contiguous(), bits, group, fused);
        return out;
    }
};

QuantizedLinearBackward* node_of(PyObject* self) {
    return static_cast<QuantizedLinearBackward*>(reinterpret_cast<torch::autograd::THPCppFunction*>(self)->cdata.get());
}

PyObject* node_saved_tensors(PyObject* self, void*) {
    HANDLE_TH_ERRORS
    QuantizedLinearBackward* node = node_of(self);
    const auto t = node->unpack();
    PyObject* r = PyTuple_New(5);
    if (!r) return nullptr;
    for (int i = 0; i < 5; i++) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(t[i]));   // (an undefined tensor is None)
    return r;
    END_HANDLE_TH_ERRORS
}

PyObject* node_needs_input_grad(PyObject* self, void*) {
    QuantizedLinearBackward* node = node_of(self);
    PyObject* r = PyTuple_New(7);
    if (!r) return nullptr;
    for (uint32_t i = 0; i < 7; i++)
        PyTuple_SET_ITEM(r, i, PyBool_FromLong(i < node->num_outputs() && node->task_should_compute_output(i)));
    return r;
}

using namespace torch::autograd;                              // (the names of the next macro)
PyGetSetDef node_properties[] = {THP_FUNCTION_DEFAULT_PROPERTIES,
                                 {"saved_tensors", node_saved_tensors, nullptr, nullptr, nullptr},
                                 {"needs_input_grad", node_needs_input_grad, nullptr, nullptr, nullptr},
                                 {"bits", [](PyObject* self, void*) { return PyLong_FromLong(node_of(self)->bits); }, nullptr, nullptr, nullptr},
                                 {"group_size", [](PyObject* self, void*) { return PyLong_FromLong(node_of(self)->group); }, nullptr, nullptr, nullptr},
                                 {nullptr, nullptr, nullptr, nullptr, nullptr}};
PyTypeObject node_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---- Python side ----

// A plain tensor or parameter; subclasses have their own ideas of every operation and go through Python.
inline bool plain(PyObject* o) { return THPVariable_CheckExact(o); }
inline const Tensor& unpack(PyObject* o) { return THPVariable_Unpack(o); }

PyObject* none() { Py_RETURN_NONE; }

PyObject* checked(Tensor y, int status, const char* what) {
    if (status == 0) return y.defined() ? THPVariable_Wrap(std::move(y)) : none();
    PyObject* r = PyObject_CallFunction(g_check, "is", status, what);   // raises
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
    return nullptr;
}

// The C++ exceptions of torch as Python ones.
template <class F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    return f();
    END_HANDLE_TH_ERRORS
}

// The module's buffers as they are now; false = the general path (or, with a Python error set, none).
struct Module {
    Tensor qweight, scale, zero, bias;                         // held: the interpreter may run while a call is under way
    Layer layer;
};

bool module_of(PyObject* dict, Module& m) {
    PyObject* buffers = PyDict_GetItemWithError(dict, s_buffers);
    PyObject *bits = PyDict_GetItemWithError(dict, s_bits), *group = PyDict_GetItemWithError(dict, s_group);
    if (!buffers || !PyDict_Check(buffers) || !bits || !group || !PyLong_Check(bits) || !PyLong_Check(group)) return false;
    PyObject* names[4] = {s_qweight, s_scale, s_zero, s_bias};
    Tensor* out[4] = {&m.qweight, &m.scale, &m.zero, &m.bias};
    for (int i = 0; i < 4; i++) {
        PyObject* t = PyDict_GetItemWithError(buffers, names[i]);
        if (i == 3 && (!t || t == Py_None)) break;
        if (!t || !plain(t)) return false;
        *out[i] = unpack(t);
    }
    const long b = PyLong_AsLong(bits), g = PyLong_AsLong(group);
    return !PyErr_Occurred() && layer_of(m.qweight, m.scale, m.zero, m.bias.defined() ? &m.bias : nullptr, b, g, m.layer);
}

// forward(module.__dict__, x) -> y or None
PyObject* py_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 2 || !PyDict_Check(args[0]) || !plain(args[1])) return none();
        const Tensor x = unpack(args[1]);
        if (!x.is_cuda() || !x.has_storage()) return none();    // (no storage: a wrapper of vmap or torch.func)
        Module l;
        if (!module_of(args[0], l)) {
            if (PyErr_Occurred()) return nullptr;
            return none();
        }
        int status = 0;
        const char* what = "";
        const bool recorded = c10::GradMode::is_enabled() && x.requires_grad();
        if (recorded && x._fw_grad(0).defined()) return none();   // the Python function refuses forward-mode derivatives
        Tensor y;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            y = linear(l.layer, x, status, what);
        }
        if (recorded && status == 0 && y.defined()) {
            std::shared_ptr<QuantizedLinearBackward> node(new QuantizedLinearBackward(), torch::autograd::deleteNode);
            const Tensor* inputs[5] = {&x, &l.qweight, &l.scale, &l.zero, &l.bias};
            node->has_bias = l.bias.defined();
            node->set_next_edges(node->has_bias ? torch::autograd::collect_next_edges(x, l.qweight, l.scale, l.zero, l.bias)
                                                : torch::autograd::collect_next_edges(x, l.qweight, l.scale, l.zero));
            for (int i = 0; i < (node->has_bias ? 5 : 4); i++) node->saved[i] = torch::autograd::SavedVariable(*inputs[i], false);
            node->bits = l.layer.bits;
            node->group = l.layer.group;
            torch::autograd::set_history(y, node);
        }
        return checked(std::move(y), status, what);
    });
}

// matmul(x, qweight, scale, zero_point, bias, bits, group_size) -> y or None
PyObject* py_matmul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 7 || !PyLong_Check(args[5]) || !PyLong_Check(args[6])) return none();
        for (int i = 0; i < 5; i++)
            if (!plain(args[i]) && !(i == 4 && args[i] == Py_None)) return none();
        const Tensor x = unpack(args[0]);
        if (!x.has_storage() || (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)) return none();
        const Tensor qweight = unpack(args[1]), scale = unpack(args[2]), zero = unpack(args[3]), bias = args[4] == Py_None ? Tensor() : unpack(args[4]);
        const int64_t bits = PyLong_AsLong(args[5]), group = PyLong_AsLong(args[6]);
        if (PyErr_Occurred()) return nullptr;
        Layer l;
        if (!layer_of(qweight, scale, zero, bias.defined() ? &bias : nullptr, bits, group, l)) return none();
        int status = 0;
        const char* what = "";
        Tensor y;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            y = linear(l, x, status, what);
        }
        return checked(std::move(y), status, what);
    });
}

// input_grad(grad_output, qweight, scale, zero_point, bits, group_size) -> grad_input or None
PyObject* py_input_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 6 || !PyLong_Check(args[4]) || !PyLong_Check(args[5])) return none();
        for (int i = 0; i < 4; i++)
            if (!plain(args[i])) return none();
        const Tensor go = unpack(args[0]), qweight = unpack(args[1]), scale = unpack(args[2]), zero = unpack(args[3]);
        const int64_t bits = PyLong_AsLong(args[4]), group = PyLong_AsLong(args[5]);
        if (PyErr_Occurred()) return nullptr;
        Layer l;
        if (!go.is_cuda() || !go.has_storage() || !layer_of(qweight, scale, zero, nullptr, bits, group, l)) return none();
        if (go.dim() < 1 || go.size(-1) != l.n || !go.is_floating_point() || go.device().index() != l.device) return none();
        const FusedRows fused;
        Tensor gx;
        {
            Unlocked unlocked;
            gx = input_grad(go, qweight, scale, zero, l.bits, l.group, fused);
        }
        return THPVariable_Wrap(std::move(gx));
    });
}

// quantize(weight, delta or None, bits, group_size, math code with flags, scale code, zero-point code) -> (qweight, scale, zero_point) or None
PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 7 || !plain(args[0]) || !(args[1] == Py_None || plain(args[1]))) return none();
        Tensor w = unpack(args[0]), delta = args[1] == Py_None ? Tensor() : unpack(args[1]);
        const int64_t bits = PyLong_AsLong(args[2]), group = PyLong_AsLong(args[3]);
        const int math = (int)PyLong_AsLong(args[4]), sc = (int)PyLong_AsLong(args[5]), zc = (int)PyLong_AsLong(args[6]);
        if (PyErr_Occurred()) return nullptr;
        const int code = dtype_code(w.scalar_type());
        if (!lib.quantize || !w.is_cuda() || w.dim() != 2 || code < 0 || (bits != 2 && bits != 4 && bits != 8) || group < 1) return none();
        if (delta.defined() && (delta.device() != w.device() || delta.sizes() != w.sizes() || delta.scalar_type() != w.scalar_type())) return none();
        Tensor q, s, z;
        int st;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            if (w.stride(1) != 1) w = w.contiguous();
            if (delta.defined() && delta.stride(1) != 1) delta = delta.contiguous();
            const int64_t n = w.size(0), k = w.size(1);
            OnDevice on(w.device());
            q = empty({n, k / (32 / bits)}, at::kInt, w.device());
            s = empty({n, k / group}, dtype_of(sc), w.device());
            z = empty({n, k / group}, dtype_of(zc), w.device());
            st = lib.quantize(w.const_data_ptr(), delta.defined() ? delta.const_data_ptr() : nullptr, code, math, n, k, w.stride(0),
                              delta.defined() ? delta.stride(0) : 0, (int)bits, (int)group, (int32_t*)q.mutable_data_ptr(),
                              s.mutable_data_ptr(), sc, z.mutable_data_ptr(), zc, stream_of(w.device().index()));
        }
        if (st) return checked({}, st, "bw_quantize_pack");
        PyObject* r = PyTuple_New(3);
        if (!r) return nullptr;
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(q)));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(s)));
        PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(z)));
        return r;
    });
}

// dequantize(qweight, scale, zero_point, group_size, bits, output code) -> weight or None
PyObject* py_dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 6 || !plain(args[0]) || !plain(args[1]) || !plain(args[2])) return none();
        const int64_t group = PyLong_AsLong(args[3]), bits = PyLong_AsLong(args[4]);
        const int oc = (int)PyLong_AsLong(args[5]);
        if (PyErr_Occurred()) return nullptr;
        Tensor q = unpack(args[0]), s = unpack(args[1]), z = unpack(args[2]), w;
        const int sc = dtype_code(s.scalar_type()), zc = dtype_code(z.scalar_type());
        if (!lib.dequantize || !q.is_cuda() || s.device() != q.device() || z.device() != q.device() || q.scalar_type() != at::kInt || q.dim() != 2 ||
            sc < 0 || zc < 0 || (bits != 2 && bits != 4 && bits != 8) || group < 1)
            return none();
        const int64_t n = q.size(0), k = q.size(1) * (32 / bits);
        if (s.numel() < n * (k / group) || z.numel() < n * (k / group)) return none();
        int st;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            q = q.contiguous();
            s = s.contiguous();
            z = z.contiguous();
            OnDevice on(q.device());
            w = empty({n, k}, dtype_of(oc), q.device());
            st = lib.dequantize((const int32_t*)q.const_data_ptr(), s.const_data_ptr(), sc, z.const_data_ptr(), zc, n, k, (int)bits, (int)group,
                                w.mutable_data_ptr(), oc, k, stream_of(q.device().index()));
        }
        return checked(std::move(w), st, "bw_dequantize");
    });
}

// ---- rotation, cache and attention of a decode step ----

// A tensor [..., heads, dim] of 16-bit values as rows of tokens: base address, distance of two tokens and of two heads in elements.  A
// layout that the kernels do not read (leading dimensions that are no single stride, pieces that do not start at 16 bytes) is copied.
struct Rows {
    Tensor held;
    const void* data = nullptr;
    int64_t row = 0, head = 0;
    Rows() = default;
    Rows(const Tensor& t, int64_t tokens) {
        const int64_t heads = t.size(-2), dim = t.size(-1);
        held = t.dim() == 3 ? t : t.reshape({tokens, heads, dim});
        const bool one_token = tokens <= 1, one_head = heads <= 1;
        if (held.stride(2) != 1 || (!one_token && held.stride(0) % 8) || (!one_head && held.stride(1) % 8) || !aligned16(held.const_data_ptr()))
            held = held.clone(at::MemoryFormat::Contiguous);
        data = held.const_data_ptr();
        row = one_token ? 0 : held.stride(0);                   // (the stride of a single row may be anything)
        head = one_head ? 0 : held.stride(1);
    }
};

// Forward-mode derivatives are refused, with and without grad mode: a result without its tangent would be wrong without a word.
void check_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs) TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

inline bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
inline bool on_gpu(const Tensor& t, const Tensor& like) { return t.is_cuda() && t.has_storage() && t.device() == like.device(); }

// [..., heads, dim] with the leading dimensions of `lead`
bool heads_of(const Tensor& t, at::IntArrayRef lead) {
    return t.dim() == (int64_t)lead.size() + 2 && t.sizes().slice(0, lead.size()).equals(lead) && t.size(-1) > 0 && t.size(-2) > 0;
}

struct Rotation {
    bw_heads heads;
    int act;
    Tensor weights[2];                                          // the queries' and the keys', as the kernels read them
};

bool rotation_of(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions, const Tensor& qw, const Tensor& kw,
                 double eps, Rotation& r) {
    if (!lib.rotate || !q.is_cuda() || !q.has_storage() || !half_type(q.scalar_type()) || k.scalar_type() != q.scalar_type()) return false;
    for (const Tensor* t : {&k, &cos, &sin, &positions})
        if (!on_gpu(*t, q)) return false;
    if (positions.scalar_type() != at::kLong || !positions.is_contiguous() || !heads_of(q, positions.sizes()) || !heads_of(k, positions.sizes())) return false;
    const int64_t dim = q.size(-1);
    if (k.size(-1) != dim || q.size(-2) > 65535 || k.size(-2) > 65535 || dim > 65535) return false;
    for (const Tensor* t : {&cos, &sin})
        if (t->scalar_type() != at::kFloat || t->dim() != 2 || !t->is_contiguous() || !aligned16(t->const_data_ptr())) return false;
    if (!cos.sizes().equals(sin.sizes()) || cos.size(0) < 1 || cos.size(1) < 1 || 2 * cos.size(1) > dim) return false;
    at::ScalarType wt = q.scalar_type();
    for (const Tensor* t : {&qw, &kw})
        if (t->defined()) {
            if (!on_gpu(*t, q) || t->dim() != 1 || t->size(0) != dim) return false;
            wt = t->scalar_type();
        }
    if (wt != q.scalar_type() && wt != at::kFloat) return false;
    if (qw.defined() && kw.defined() && qw.scalar_type() != kw.scalar_type()) return false;
    r.weights[0] = qw;
    r.weights[1] = kw;
    for (Tensor& w : r.weights)
        if (w.defined() && (!w.is_contiguous() || !aligned16(w.const_data_ptr()))) {
            c10::AutoGradMode off(false);
            OnDevice on(q.device());
            w = w.clone(at::MemoryFormat::Contiguous);
        }
    r.act = dtype_code(q.scalar_type());
    r.heads = {positions.numel(), (int)q.size(-2), (int)k.size(-2), (int)dim, (int)(2 * cos.size(1)), (const float*)cos.const_data_ptr(),
               (const float*)sin.const_data_ptr(), cos.size(0), (const int64_t*)positions.const_data_ptr(), qw.defined() ? r.weights[0].const_data_ptr() : nullptr,
               kw.defined() ? r.weights[1].const_data_ptr() : nullptr, dtype_code(wt), (float)eps};
    return true;
}

struct RotateHeadsBackward : public torch::autograd::Node {
    enum { Q, K, QW, KW, COS, SIN, POSITIONS };
    torch::autograd::SavedVariable saved[7];
    c10::SmallVector<int64_t, 5> q_sizes, k_sizes;
    at::ScalarType type = at::kHalf;
    double eps = 0;
    std::string name() const override { return "RotateHeadsBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : saved) v.reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list out(4);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        Tensor t[7];
        for (int i = 0; i < 7; i++) t[i] = saved[i].unpack();
        const Tensor gq = grads[0].defined() ? grads[0] : input_metadata(0).zeros_like(), gk = grads[1].defined() ? grads[1] : input_metadata(1).zeros_like();
        OnDevice on(gq.device());
        {
            c10::AutoGradMode off(false);
            Rotation r;
            TORCH_CHECK(rotation_of(gq, gk, t[COS], t[SIN], t[POSITIONS], t[QW], t[KW], eps, r), "bw_rotate_heads_grad: the gradients or what the forward saved have changed");
            const int64_t tokens = r.heads.tokens;
            const Rows rgq(gq, tokens), rgk(gk, tokens);
            Rows rq, rk;
            if (t[QW].defined()) rq = Rows(t[Q], tokens);
            if (t[KW].defined()) rk = Rows(t[K], tokens);
            out[0] = empty(q_sizes, type, gq.device());
            out[1] = empty(k_sizes, type, gq.device());
            for (int i : {2, 3})
                if (t[i].defined() && task_should_compute_output(i)) out[i] = empty(t[i].sizes(), t[i].scalar_type(), gq.device());
            Tensor ws;
            size_t bytes = 0;
            if (out[2].defined() || out[3].defined()) bytes = lib.rotate_grad_ws_bytes(&r.heads);
            if (bytes) ws = empty({(int64_t)bytes}, at::kByte, gq.device());
            const int st = lib.rotate_grad(&r.heads, r.act, rgq.data, rgq.row, rgq.head, rgk.data, rgk.row, rgk.head, rq.data, rq.row, rq.head, rk.data, rk.row,
                                           rk.head, out[0].mutable_data_ptr(), out[1].mutable_data_ptr(), out[2].defined() ? out[2].mutable_data_ptr() : nullptr,
                                           out[3].defined() ? out[3].mutable_data_ptr() : nullptr, bytes ? ws.mutable_data_ptr() : nullptr, bytes,
                                           stream_of(gq.device().index()));
            TORCH_CHECK(st == BW_OK, "bw_rotate_heads_grad failed (status ", st, ")");
        }
        for (int i : {0, 1})
            if (!task_should_compute_output(i)) out[i] = Tensor();
        if (c10::GradMode::is_enabled()) {                      // create_graph: these gradients have no derivative of their own
            for (auto& v : out)
                if (v.defined()) {
                    auto error = std::make_shared<torch::autograd::DelayedError>("rotate_heads has no second derivative", 1);
                    v = error->apply({v.detach().requires_grad_(true)})[0];
                }
        }
        return out;
    }
};

// Autograd runs a leaf's accumulation on the stream where its node was made.  A node that an eager graph keeps alive on another stream would
// be waited for inside the capture, which a capture cannot do: refused here, while nothing is recorded yet.
void check_capture(std::initializer_list<const Tensor*> inputs, at::DeviceIndex index) {
    const auto stream = c10::hip::getCurrentHIPStream(index);
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    for (const Tensor* t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto on = node->stream();
        TORCH_CHECK(!on || *on == stream.unwrap(), "rotate_heads: a graph recorded on another stream still holds the gradient accumulation of an input of this "
                    "captured call; drop that graph (its outputs) before the capture");
    }
}

// rotate_heads(q, k, cos, sin, positions, q_weight or None, k_weight or None, eps) -> (q, k) or None
PyObject* py_rotate_heads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        if (nargs != 8) return none();
        for (int i = 0; i < 7; i++)
            if (!plain(args[i]) && !(i >= 5 && args[i] == Py_None)) return none();
        const double eps = PyFloat_AsDouble(args[7]);
        if (PyErr_Occurred()) return nullptr;
        const Tensor q = unpack(args[0]), k = unpack(args[1]), cos = unpack(args[2]), sin = unpack(args[3]), positions = unpack(args[4]);
        const Tensor qw = args[5] == Py_None ? Tensor() : unpack(args[5]), kw = args[6] == Py_None ? Tensor() : unpack(args[6]);
        Rotation r;
        if (!rotation_of(q, k, cos, sin, positions, qw, kw, eps, r)) return none();
        check_tangents("rotate_heads", {&q, &k, &qw, &kw, &cos, &sin});
        bool recorded = false;
        for (const Tensor* t : {&q, &k, &qw, &kw}) recorded |= t->defined() && t->requires_grad();
        recorded &= c10::GradMode::is_enabled();
        if (c10::GradMode::is_enabled()) {
            if (cos.requires_grad() || sin.requires_grad()) return none();
        }
        if (recorded) check_capture({&q, &k, &qw, &kw}, q.device().index());
        Tensor q_out, k_out;
        int status = 0;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            OnDevice on(q.device());
            q_out = empty(q.sizes(), q.scalar_type(), q.device());
            k_out = empty(k.sizes(), q.scalar_type(), q.device());
            if (r.heads.tokens > 0) {
                const Rows rq(q, r.heads.tokens), rk(k, r.heads.tokens);
                status = lib.rotate(&r.heads, r.act, rq.data, rq.row, rq.head, rk.data, rk.row, rk.head, q_out.mutable_data_ptr(), k_out.mutable_data_ptr(),
                                    stream_of(q.device().index()));
            }
        }
        if (status) return checked({}, status, "bw_rotate_heads");
        if (recorded) {
            std::shared_ptr<RotateHeadsBackward> node(new RotateHeadsBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(q, k, qw, kw));
            const Tensor none_, *keep[7] = {qw.defined() ? &q : &none_, kw.defined() ? &k : &none_, &qw, &kw, &cos, &sin, &positions};
            for (int i = 0; i < 7; i++) node->saved[i] = torch::autograd::SavedVariable(*keep[i], false);
            node->q_sizes = q.sizes();
            node->k_sizes = k.sizes();
            node->type = q.scalar_type();
            node->eps = eps;
            torch::autograd::set_history(torch::autograd::variable_list{q_out, k_out}, node);
        }
        PyObject* p = PyTuple_New(2);
        if (!p) return nullptr;
        PyTuple_SET_ITEM(p, 0, THPVariable_Wrap(std::move(q_out)));
        PyTuple_SET_ITEM(p, 1, THPVariable_Wrap(std::move(k_out)));
        return p;
    });
}

// The cache that six arguments name: keys, values, key_meta or None, value_meta or None, bits, group size.
struct Cache {
    Tensor keys, values, key_meta, value_meta;
    bw_cache c = {};
};

bool cache_of(PyObject* const* args, Cache& h) {
    if (!lib.attention || !plain(args[0]) || !plain(args[1]) || !PyLong_Check(args[4]) || !PyLong_Check(args[5])) return false;
    const int64_t bits = PyLong_AsLong(args[4]), group = PyLong_AsLong(args[5]);
    if (PyErr_Occurred() || (bits != 16 && bits != 8 && bits != 4)) return false;
    h.keys = unpack(args[0]);
    h.values = unpack(args[1]);
    if (!h.keys.is_cuda() || !h.keys.has_storage() || h.keys.dim() != 4 || !on_gpu(h.values, h.keys) || !h.values.sizes().equals(h.keys.sizes()) ||
        h.values.scalar_type() != h.keys.scalar_type() || !h.keys.is_contiguous() || !h.values.is_contiguous())
        return false;
    for (int i = 0; i < 4; i++)
        if (h.keys.size(i) < 1 || h.keys.size(i) >= (int64_t)1 << 31) return false;
    int64_t dim = h.keys.size(3);
    if (bits == 16) {
        if (!half_type(h.keys.scalar_type()) || args[2] != Py_None || args[3] != Py_None) return false;
    } else {
        dim = dim * 32 / bits;
        if (h.keys.scalar_type() != at::kInt || !plain(args[2]) || !plain(args[3]) || group < 1 || group > dim || dim % group) return false;
        h.key_meta = unpack(args[2]);
        h.value_meta = unpack(args[3]);
        const int64_t want[5] = {h.keys.size(0), h.keys.size(1), dim / group, h.keys.size(2), 2};
        for (const Tensor* t : {&h.key_meta, &h.value_meta})
            if (!on_gpu(*t, h.keys) || t->scalar_type() != at::kHalf || !t->sizes().equals(want) || !t->is_contiguous()) return false;
    }
    h.c = {h.keys.data_ptr(), h.values.data_ptr(), bits == 16 ? nullptr : h.key_meta.data_ptr(), bits == 16 ? nullptr : h.value_meta.data_ptr(),
           h.keys.size(0), (int)h.keys.size(1), (int)h.keys.size(2), (int)dim, (int)bits, (int)group, bits == 16 ? dtype_code(h.keys.scalar_type()) : BW_F16};
    return true;
}

bool slots_of(PyObject* o, const Tensor& like, Tensor& slots) {
    if (!plain(o)) return false;
    slots = unpack(o);
    return on_gpu(slots, like) && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous();
}

// Two contiguous tensors of one size that share memory.
inline bool overlap(const Tensor& a, const Tensor& b) {
    const auto *x = (const char*)a.const_data_ptr(), *y = (const char*)b.const_data_ptr();
    return x < y + b.nbytes() && y < x + a.nbytes();
}

inline bool wants_grad(const Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }
// A cache that asks for gradients, which neither its reader nor its writer gives (the Python functions refuse it).
inline bool wants_grad(const Cache& h) {
    for (const Tensor* t : {&h.keys, &h.values, &h.key_meta, &h.value_meta})
        if (t->defined() && wants_grad(*t)) return true;
    return false;
}

// cache_write(k, v, slots, keys, values, key_meta, value_meta, bits, group_size) -> True or None
PyObject* py_cache_write(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        Cache h;
        Tensor slots;
        if (nargs != 9 || !plain(args[0]) || !plain(args[1]) || !cache_of(args + 3, h) || !slots_of(args[2], h.keys, slots)) {
            if (PyErr_Occurred()) return nullptr;
            return none();
        }
        Tensor k = unpack(args[0]), v = unpack(args[1]);
        for (const Tensor* t : {&k, &v})
            if (!on_gpu(*t, h.keys) || !half_type(t->scalar_type()) || t->dim() != 3 || t->size(0) != slots.size(0) || t->size(1) != h.c.kv_heads ||
                t->size(2) != h.c.dim || wants_grad(*t))
                return none();
        if (k.scalar_type() != v.scalar_type() || (h.c.bits == 16 && k.scalar_type() != h.keys.scalar_type())) return none();
        check_tangents("write_cache", {&k, &v, &h.keys, &h.values, &h.key_meta, &h.value_meta});
        if (wants_grad(h) || overlap(h.keys, h.values) || (h.key_meta.defined() && overlap(h.key_meta, h.value_meta))) return none();
        int status = 0;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            for (const Tensor* t : {&h.keys, &h.values, &h.key_meta, &h.value_meta})       // written in place: what autograd saved of them is stale
                if (t->defined()) torch::autograd::impl::bump_version(*t);
            const int64_t tokens = slots.size(0);
            if (tokens > 0) {
                OnDevice on(k.device());
                for (Tensor* t : {&k, &v})                      // rows of this very cache: they may be written before they are read
                    if (t->is_alias_of(h.keys) || t->is_alias_of(h.values)) *t = t->clone();
                const Rows rk(k, tokens), rv(v, tokens);
                status = lib.cache_write(&h.c, dtype_code(k.scalar_type()), tokens, rk.data, rk.row, rk.head, rv.data, rv.row, rv.head,
                                         (const int64_t*)slots.const_data_ptr(), stream_of(k.device().index()));
            }
        }
        if (status) return checked({}, status, "bw_cache_write");
        Py_RETURN_TRUE;
    });
}

// cache_read(slots, keys, values, key_meta, value_meta, bits, group_size, output code) -> (k, v) or None
PyObject* py_cache_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        Cache h;
        Tensor slots;
        if (nargs != 8 || !cache_of(args + 1, h) || !slots_of(args[0], h.keys, slots)) {
            if (PyErr_Occurred()) return nullptr;
            return none();
        }
        const int code = (int)PyLong_AsLong(args[7]);
        if (PyErr_Occurred()) return nullptr;
        if ((code != BW_F16 && code != BW_BF16) || (h.c.bits == 16 && code != h.c.dtype) || wants_grad(h)) return none();
        check_tangents("read_cache", {&h.keys, &h.values, &h.key_meta, &h.value_meta});
        Tensor k, v;
        int status = 0;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            OnDevice on(slots.device());
            const int64_t tokens = slots.size(0);
            k = empty({tokens, h.c.kv_heads, h.c.dim}, dtype_of(code), slots.device());
            v = empty({tokens, h.c.kv_heads, h.c.dim}, dtype_of(code), slots.device());
            if (tokens > 0)
                status = lib.cache_read(&h.c, code, tokens, (const int64_t*)slots.const_data_ptr(), k.mutable_data_ptr(), v.mutable_data_ptr(),
                                        stream_of(slots.device().index()));
        }
        if (status) return checked({}, status, "bw_cache_read");
        PyObject* p = PyTuple_New(2);
        if (!p) return nullptr;
        PyTuple_SET_ITEM(p, 0, THPVariable_Wrap(std::move(k)));
        PyTuple_SET_ITEM(p, 1, THPVariable_Wrap(std::move(v)));
        return p;
    });
}

// cache_attention(q, page_table, lengths, keys, values, key_meta, value_meta, bits, group_size, scale) -> out or None
PyObject* py_cache_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject* {
        Cache h;
        if (nargs != 10 || !plain(args[0]) || !plain(args[1]) || !plain(args[2]) || !cache_of(args + 3, h)) {
            if (PyErr_Occurred()) return nullptr;
            return none();
        }
        const Tensor q = unpack(args[0]), table = unpack(args[1]), lengths = unpack(args[2]);
        const double scale = PyFloat_AsDouble(args[9]);
        if (PyErr_Occurred()) return nullptr;
        for (const Tensor* t : {&q, &table, &lengths})
            if (!on_gpu(*t, h.keys)) return none();
        if (!half_type(q.scalar_type()) || (h.c.bits == 16 && q.scalar_type() != h.keys.scalar_type()) || q.dim() != 3 || q.size(2) != h.c.dim ||
            q.size(1) < 1 || q.size(1) > 65535 || q.size(1) % h.c.kv_heads || wants_grad(q) || wants_grad(h))
            return none();
        const int64_t batch = q.size(0);
        if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != batch || table.size(1) < 1 || (table.size(1) > 1 && table.stride(1) != 1) ||
            lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != batch || !lengths.is_contiguous())
            return none();
        check_tangents("cache_attention", {&q, &h.keys, &h.values, &h.key_meta, &h.value_meta});
        Tensor out;
        int status = 0;
        {
            Unlocked unlocked;
            c10::AutoGradMode off(false);
            OnDevice on(q.device());
            out = empty({batch, q.size(1), q.size(2)}, q.scalar_type(), q.device());
            if (batch > 0) {
                const Rows rq(q, batch);
                const size_t bytes = lib.attention_ws_bytes(&h.c, batch, (int)q.size(1), table.size(1));
                Tensor ws;
                if (bytes) ws = empty({(int64_t)bytes}, at::kByte, q.device());
                status = lib.attention(&h.c, dtype_code(q.scalar_type()), rq.data, batch, (int)q.size(1), rq.row, rq.head,
                                       (const int32_t*)table.const_data_ptr(), table.size(1), batch > 1 ? table.stride(0) : table.size(1),
                                       (const int32_t*)lengths.const_data_ptr(), (float)scale, out.mutable_data_ptr(), bytes ? ws.mutable_data_ptr() : nullptr,
                                       bytes, stream_of(q.device().index()));
            }
        }
        return checked(std::move(out), status, "bw_cache_attention");
    });
}

// bind({entry point name: address}, check, dict with the fused gradient's row limits): once, after the kernel library is loaded
PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject *table, *check, *limits;
    if (!PyArg_ParseTuple(args, "O!OO!", &PyDict_Type, &table, &check, &PyDict_Type, &limits)) return nullptr;
    bool ok = true;
    auto get = [&](auto& fn, const char* name) {
        PyObject* v = PyDict_GetItemString(table, name);
        void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
        if (!p) ok = false;
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(p);
    };
    Library l;
    get(l.qlinear, "bw_qlinear_ws");
    get(l.qlinear_ws_bytes, "bw_qlinear_workspace_bytes");
    get(l.cast, "bw_cast_bf16_f16");
    get(l.qdgrad, "bw_qdgrad");
    get(l.qdgrad_ws_bytes, "bw_qdgrad_workspace_bytes");
    get(l.qdgrad_tile_rows, "bw_qdgrad_tile_rows");
    get(l.quantize, "bw_quantize_pack_add");
    get(l.dequantize, "bw_dequantize");
    const bool linears = ok;                                    // a table may hold the linears' entry points alone: the others' functions then give None
    get(l.rotate, "bw_rotate_heads");
    get(l.rotate_grad, "bw_rotate_heads_grad");
    get(l.rotate_grad_ws_bytes, "bw_rotate_heads_grad_workspace_bytes");
    get(l.cache_write, "bw_cache_write");
    get(l.cache_read, "bw_cache_read");
    get(l.attention, "bw_cache_attention");
    get(l.attention_ws_bytes, "bw_cache_attention_workspace_bytes");
    if (PyErr_Occurred()) return nullptr;
    if (!ok) l.rotate = nullptr, l.attention = nullptr;
    if (!linears) {
        PyErr_SetString(PyExc_RuntimeError, "bind: an entry point is missing");
        return nullptr;
    }
    lib = l;
    Py_INCREF(check);
    Py_XSETREF(g_check, check);
    Py_INCREF(limits);
    Py_XSETREF(g_limits, limits);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"forward", (PyCFunction)(void*)py_forward, METH_FASTCALL, nullptr},
    {"matmul", (PyCFunction)(void*)py_matmul, METH_FASTCALL, nullptr},
    {"input_grad", (PyCFunction)(void*)py_input_grad, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void*)py_quantize, METH_FASTCALL, nullptr},
    {"dequantize", (PyCFunction)(void*)py_dequantize, METH_FASTCALL, nullptr},
    {"rotate_heads", (PyCFunction)(void*)py_rotate_heads, METH_FASTCALL, nullptr},
    {"cache_write", (PyCFunction)(void*)py_cache_write, METH_FASTCALL, nullptr},
    {"cache_read", (PyCFunction)(void*)py_cache_read, METH_FASTCALL, nullptr},
    {"cache_attention", (PyCFunction)(void*)py_cache_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_bw_host", "Native host path of bitween_amd", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__bw_host() {
    s_fused_rows = PyUnicode_InternFromString("FUSED_DGRAD_MAX_ROWS");
    s_fused_large_rows = PyUnicode_InternFromString("FUSED_DGRAD_LARGE_MAX_ROWS");
    s_buffers = PyUnicode_InternFromString("_buffers");
    s_qweight = PyUnicode_InternFromString("qweight");
    s_scale = PyUnicode_InternFromString("scale");
    s_zero = PyUnicode_InternFromString("zero_point");
    s_bias = PyUnicode_InternFromString("bias");
    s_bits = PyUnicode_InternFromString("bits");
    s_group = PyUnicode_InternFromString("group_size");
    HANDLE_TH_ERRORS
    torch::autograd::_initFunctionPyTypeObject(node_type, "QuantizedLinearFunctionBackward", node_properties, nullptr);
    torch::autograd::registerCppFunction(typeid(QuantizedLinearBackward), &node_type);
    return PyModule_Create(&module_def);
    END_HANDLE_TH_ERRORS
}
