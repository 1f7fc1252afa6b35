// rf_pyblocks.cpp -- native host path of the residual-block operators and of the
// vocabulary loss (CPython module rollfast_amd._lib._rfblocks).
//
// Each function checks its tensors, allocates the outputs and calls the C
// entry (include/rfadam8.h), in one to two microseconds where the same steps
// from Python take eight to fifteen.  What is not the plain case (another
// device than the current one, a layout to copy, an argument to refuse) makes
// a function return None; rollfast_amd.blocks (or losses) then checks and lays out the
// arguments and calls again with `shape`, the outputs' shape, which says that
// every tensor is rows [rows, cols] in order.
//
// What the backward pass keeps lies in one byte tensor (an arena), in the order
//   codes of each kept row tensor, their exponents, 16-byte alignment,
//   f32 statistics [rows] each: post rstd, post mean, next rstd, next mean
// with only those that the norms have; rollfast_amd.blocks lays out the same.
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstdint>
#include <string>
#include <vector>

#include <ATen/ATen.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include "rfadam8.h"

namespace {

struct Entries {
    decltype(&rf_checkpoint_store) checkpoint_store;
    decltype(&rf_checkpoint_load) checkpoint_load;
    decltype(&rf_gated_forward) gated_forward;
    decltype(&rf_gated_backward) gated_backward;
    decltype(&rf_norm_forward) norm_forward;
    decltype(&rf_norm_backward_workspace) norm_backward_workspace;
    decltype(&rf_norm_backward) norm_backward;
    decltype(&rf_linear_weight_grad_workspace) weight_grad_workspace;
    decltype(&rf_linear_weight_grad) weight_grad;
    decltype(&rf_linear_cross_entropy_workspace) cross_entropy_workspace;
    decltype(&rf_linear_cross_entropy) cross_entropy;
    decltype(&rf_last_error) last_error;
};
Entries g_lib{};
PyObject* g_raw_stream = nullptr;  // torch._C._cuda_getCurrentRawStream
PyObject* g_parameter = nullptr;   // torch.nn.Parameter

struct Refused {};  // a Python error is set

int32_t code_of(at::ScalarType t)
{
    return t == at::kFloat ? RF_F32 : t == at::kBFloat16 ? RF_BF16 : t == at::kHalf ? RF_F16 : -1;
}

// set_entries(dict of addresses, raw stream function, Parameter type)
PyObject* py_set_entries(PyObject*, PyObject* args)
{
    PyObject *d, *stream, *parameter;
    if (!PyArg_ParseTuple(args, "O!OO", &PyDict_Type, &d, &stream, &parameter)) return nullptr;
    struct { const char* name; void** at; } const all[] = {
        {"rf_checkpoint_store", (void**)&g_lib.checkpoint_store},
        {"rf_checkpoint_load", (void**)&g_lib.checkpoint_load},
        {"rf_gated_forward", (void**)&g_lib.gated_forward},
        {"rf_gated_backward", (void**)&g_lib.gated_backward},
        {"rf_norm_forward", (void**)&g_lib.norm_forward},
        {"rf_norm_backward_workspace", (void**)&g_lib.norm_backward_workspace},
        {"rf_norm_backward", (void**)&g_lib.norm_backward},
        {"rf_linear_weight_grad_workspace", (void**)&g_lib.weight_grad_workspace},
        {"rf_linear_weight_grad", (void**)&g_lib.weight_grad},
        {"rf_linear_cross_entropy_workspace", (void**)&g_lib.cross_entropy_workspace},
        {"rf_linear_cross_entropy", (void**)&g_lib.cross_entropy},
        {"rf_last_error", (void**)&g_lib.last_error},
    };
    for (const auto& e : all) {
        PyObject* const v = PyDict_GetItemString(d, e.name);
        if (!v) return PyErr_Format(PyExc_KeyError, "%s", e.name);
        *e.at = PyLong_AsVoidPtr(v);
        if (!*e.at) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "%s is null", e.name);
    }
    Py_XDECREF(g_raw_stream);
    Py_XDECREF(g_parameter);
    g_raw_stream = Py_NewRef(stream);
    g_parameter = Py_NewRef(parameter);
    Py_RETURN_NONE;
}

// Raises what rollfast_amd._lib.check raises.
void check(rf_status status, const char* what)
{
    if (status == RF_OK) return;
    PyObject* const type = status == RF_ERR_INVALID       ? PyExc_ValueError
                           : status == RF_ERR_UNSUPPORTED ? PyExc_NotImplementedError
                                                          : PyExc_RuntimeError;
    PyErr_Format(type, "%s: %s", what, g_lib.last_error());
    throw Refused{};
}

// The call's device, stream, rows and output shape.
struct Call {
    bool trusted = false, fine = true;  // trusted: laid out by blocks.py
    int64_t rows = 0, cols = 0;
    std::vector<int64_t> shape;
    c10::Device device{c10::DeviceType::CUDA, 0};
    void* stream = nullptr;

    // The first tensor of a call, and `shape` (None, or a tuple).
    at::Tensor first(PyObject* o, PyObject* given)
    {
        trusted = given != Py_None;
        if (!THPVariable_Check(o)) return no();
        if (!trusted && !plain(o)) return no();
        const at::Tensor t = THPVariable_Unpack(o);
        if (!t.is_cuda() || code_of(t.scalar_type()) < 0) return no();
        device = t.device();
        const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
        if (guard.getDevice().index() != device.index()) return no();
        if (trusted) {
            const Py_ssize_t n = PyTuple_Check(given) ? PyTuple_GET_SIZE(given) : 0;
            for (Py_ssize_t i = 0; i < n; ++i) shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(given, i)));
            if (PyErr_Occurred()) throw Refused{};
        } else {
            shape = t.sizes().vec();
        }
        if (shape.empty() || shape.back() < 1) return no();
        cols = shape.back();
        rows = 1;
        for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
        return t;
    }

    static bool plain(PyObject* o) { return THPVariable_CheckExact(o) || (PyObject*)Py_TYPE(o) == g_parameter; }

    at::Tensor no()
    {
        fine = false;
        return {};
    }

    // Another tensor of the call that has these rows and columns; dtype -1: any of the three.
    at::Tensor rows_like(PyObject* o, int64_t columns, int32_t dtype, const void** p, int64_t* stride)
    {
        if (!fine || !THPVariable_Check(o) || (!trusted && !plain(o))) return no();
        const at::Tensor t = THPVariable_Unpack(o);
        const int32_t code = code_of(t.scalar_type());
        if (!t.is_cuda() || t.device() != device || code < 0 || (dtype >= 0 && code != dtype)) return no();
        if (!trusted) {  // the call's shape but for the last dimension
            if (t.dim() != (int64_t)shape.size() || t.size(-1) != columns) return no();
            for (size_t i = 0; i + 1 < shape.size(); ++i)
                if (t.size((int64_t)i) != shape[i]) return no();
        }
        return as_rows(t, columns, p, stride);
    }

    at::Tensor as_rows(const at::Tensor& t, int64_t columns, const void** p, int64_t* stride)
    {
        if (t.is_contiguous()) {
            if (t.numel() != rows * columns) return no();
            *stride = columns;
        } else if (t.dim() == 2 && t.size(0) == rows && t.size(1) == columns && (columns == 1 || t.stride(1) == 1)) {
            *stride = t.stride(0);
        } else {
            return no();
        }
        *p = t.data_ptr();
        return t;
    }

    // A parameter vector [cols], or None.
    at::Tensor vector(PyObject* o, const void** p, int32_t* dtype)
    {
        if (o == Py_None) return {};
        if (!fine || !THPVariable_Check(o) || (!trusted && !plain(o))) return no();
        const at::Tensor t = THPVariable_Unpack(o);
        const int32_t code = code_of(t.scalar_type());
        if (!t.is_cuda() || t.device() != device || code < 0 || t.dim() != 1 || t.size(0) != cols || !t.is_contiguous())
            return no();
        *p = t.data_ptr();
        *dtype = code;
        return t;
    }

    // The gate: [cols], or the shape with ones after the dimensions it varies over.
    at::Tensor gate(PyObject* o, const void** p, int32_t* dtype, int64_t* gates)
    {
        if (o == Py_None) return {};
        if (!fine || !THPVariable_Check(o) || (!trusted && !plain(o))) return no();
        const at::Tensor t = THPVariable_Unpack(o);
        const int32_t code = code_of(t.scalar_type());
        if (!t.is_cuda() || t.device() != device || code < 0 || !t.is_contiguous() || t.dim() < 1 || t.size(-1) != cols)
            return no();
        const int64_t lead = t.dim() - 1;
        *gates = 1;
        if (lead) {
            if (lead != (int64_t)shape.size() - 1) return no();
            int64_t vary = lead;
            while (vary > 0 && t.size(vary - 1) == 1) --vary;
            for (int64_t i = 0; i < vary; ++i) {
                if (t.size(i) != shape[(size_t)i]) return no();
                *gates *= t.size(i);
            }
        }
        if (*gates == 0) return t;  // no rows
        *p = t.data_ptr();
        *dtype = code;
        return t;
    }

    // Whether a tensor that the forward pass kept is where and what it was: since then
    // a parameter's `data` may have been replaced, or a saved-tensor hook have given
    // back another tensor.
    bool kept(const at::Tensor& t, at::ScalarType type) const
    {
        return t.is_cuda() && t.device() == device && t.scalar_type() == type;
    }
    bool kept_bytes(const at::Tensor& t, int64_t n) const
    {
        return kept(t, at::kByte) && t.is_contiguous() && t.numel() == n;
    }

    at::TensorOptions options(at::ScalarType t) const { return at::TensorOptions().dtype(t).device(device); }
    at::Tensor empty(at::ScalarType t) const { return at::empty(shape, options(t)); }
    at::Tensor bytes(int64_t n) const { return at::empty({n}, options(at::kByte)); }

    // Right before the C entry.
    void enter()
    {
        PyObject* const index = PyLong_FromLong(device.index());
        PyObject* const v = index ? PyObject_CallOneArg(g_raw_stream, index) : nullptr;
        Py_XDECREF(index);
        if (!v) throw Refused{};
        stream = PyLong_AsVoidPtr(v);
        Py_DECREF(v);
        if (PyErr_Occurred()) throw Refused{};
    }
};

template <typename F> void call(Call& c, const char* what, F f)
{
    c.enter();
    rf_status s;
    Py_BEGIN_ALLOW_THREADS
    s = f(c.stream);
    Py_END_ALLOW_THREADS
    check(s, what);
}

int64_t pitch_of(int64_t cols) { return (cols + 31) / 32 * 32; }

PyObject* wrap(const at::Tensor& t)
{
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

template <size_t N> PyObject* pack(const std::array<at::Tensor, N>& t)
{
    PyObject* const out = PyTuple_New(N);
    if (!out) return nullptr;
    for (size_t i = 0; i < N; ++i) {
        PyObject* const o = wrap(t[i]);
        if (!o) {
            Py_DECREF(out);
            return nullptr;
        }
        PyTuple_SET_ITEM(out, i, o);
    }
    return out;
}

// A checkpoint of its own tensors (one that the caller gets).
struct Kept {
    at::Tensor codes, exponents;
    explicit Kept(const Call& c)
        : codes(at::empty({c.rows, pitch_of(c.cols)}, c.options(at::kChar))),
          exponents(at::empty({c.rows, pitch_of(c.cols) / 32}, c.options(at::kByte)))
    {
    }
    int8_t* c() const { return (int8_t*)codes.data_ptr(); }
    uint8_t* e() const { return (uint8_t*)exponents.data_ptr(); }
};

// The arena of a call: `kept` checkpoints, then `stats` rows of f32.
struct Arena {
    int64_t code_bytes, exponent_bytes, stats_at, rows;
    int kept;
    Arena(int64_t rows, int64_t cols, int kept)
        : code_bytes(rows * pitch_of(cols)), exponent_bytes(code_bytes / 32),
          stats_at((kept * (code_bytes + exponent_bytes) + 15) / 16 * 16), rows(rows), kept(kept)
    {
    }
    int64_t size(int stats) const { return stats_at + stats * rows * 4; }
    int8_t* codes(void* p, int i) const { return (int8_t*)p + i * code_bytes; }
    uint8_t* exponents(void* p, int i) const { return (uint8_t*)p + kept * code_bytes + i * exponent_bytes; }
    float* stats(void* p, int i) const { return (float*)((char*)p + stats_at) + i * rows; }
};

#define RFB_BEGIN HANDLE_TH_ERRORS try {
#define RFB_END                 \
    }                           \
    catch (const Refused&)      \
    {                           \
        return nullptr;         \
    }                           \
    END_HANDLE_TH_ERRORS

// checkpoint_store(x, shape) -> (codes, exponents) or None
PyObject* py_checkpoint_store(PyObject*, PyObject* args)
{
    PyObject *x, *shape;
    if (!PyArg_ParseTuple(args, "OO", &x, &shape)) return nullptr;
    RFB_BEGIN
    Call c;
    const at::Tensor t = c.first(x, shape);
    const void* p = nullptr;
    int64_t stride = 0;
    if (c.fine) c.as_rows(t, c.cols, &p, &stride);
    if (!c.fine) Py_RETURN_NONE;
    const Kept k(c);
    call(c, "checkpoint_activations", [&](void* s) {
        return g_lib.checkpoint_store(p, code_of(t.scalar_type()), c.rows, c.cols, stride, k.c(), k.e(), s);
    });
    return pack<2>({k.codes, k.exponents});
    RFB_END
}

// checkpoint_load(codes, exponents, shape, dtype) -> tensor or None (another device)
PyObject* py_checkpoint_load(PyObject*, PyObject* args)
{
    PyObject *co, *eo, *shape, *dtype;
    if (!PyArg_ParseTuple(args, "OOO!O", &co, &eo, &PyTuple_Type, &shape, &dtype)) return nullptr;
    RFB_BEGIN
    const at::Tensor codes = THPVariable_Unpack(co), exps = THPVariable_Unpack(eo);
    const at::ScalarType type = ((THPDtype*)dtype)->scalar_type;
    const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
    Call c;
    c.device = codes.device();
    if (guard.getDevice().index() != c.device.index()) Py_RETURN_NONE;
    c.rows = 1;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) {
        c.shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)));
        if (i + 1 < PyTuple_GET_SIZE(shape)) c.rows *= c.shape.back();
    }
    if (PyErr_Occurred()) return nullptr;
    c.cols = c.shape.back();
    const at::Tensor out = c.empty(type);
    call(c, "restore_activations", [&](void* s) {
        return g_lib.checkpoint_load((const int8_t*)codes.data_ptr(), (const uint8_t*)exps.data_ptr(), c.rows, c.cols,
                                     code_of(type), out.data_ptr(), s);
    });
    return THPVariable_Wrap(out);
    RFB_END
}

// weight_grad(dy, shape, codes, exponents, cols, out, accumulate, dtype) -> out or None
PyObject* py_weight_grad(PyObject*, PyObject* args)
{
    PyObject *dyo, *shape, *co, *eo, *oo, *dtype;
    long long cols;
    int accumulate;
    if (!PyArg_ParseTuple(args, "OOOOLOpO", &dyo, &shape, &co, &eo, &cols, &oo, &accumulate, &dtype)) return nullptr;
    RFB_BEGIN
    Call c;
    const at::Tensor dy = c.first(dyo, shape);
    rf_weight_grad a{};
    if (c.fine) c.as_rows(dy, c.cols, &a.dy, &a.dy_stride);
    if (!c.fine || a.dy_stride >= (1ll << 24)) Py_RETURN_NONE;
    const at::Tensor codes = THPVariable_Unpack(co), exps = THPVariable_Unpack(eo);
    const at::Tensor out = oo != Py_None ? THPVariable_Unpack(oo)
                                         : at::empty({c.cols, cols}, c.options(dtype == Py_None ? dy.scalar_type()
                                                                                   : ((THPDtype*)dtype)->scalar_type));
    a.rows = c.rows;
    a.outs = c.cols;
    a.cols = cols;
    a.dy_dtype = code_of(dy.scalar_type());
    a.out_dtype = code_of(out.scalar_type());
    a.codes = (const int8_t*)codes.data_ptr();
    a.exponents = (const uint8_t*)exps.data_ptr();
    a.out = out.data_ptr();
    a.accumulate = accumulate;
    int64_t size = 0;
    check(g_lib.weight_grad_workspace(&a, &size), "linear_weight_grad");
    at::Tensor space;  // memory of the current stream: reused only behind this call's work
    if (size) space = c.bytes(size);
    call(c, "linear_weight_grad",
         [&](void* s) { return g_lib.weight_grad(&a, size ? space.data_ptr() : nullptr, size, s); });
    // a write that autograd must notice where it has kept `out` (inference tensors have no version)
    if (oo != Py_None && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return oo != Py_None ? Py_NewRef(oo) : THPVariable_Wrap(out);
    RFB_END
}

// cross_entropy(hidden, weight, targets, dloss, ignore_index, z_loss, reduction, grad)
//   -> (loss, or with a reduction the reduced one; dhidden; dweight) or None
//   reduction: RF_REDUCE_*, + RF_GRADS_F32 for gradients in f32
PyObject* py_cross_entropy(PyObject*, PyObject* args)
{
    PyObject *ho, *wo, *to, *dlo;
    long long ignore_index;
    float z_loss;
    int reduction, grad;
    if (!PyArg_ParseTuple(args, "OOOOLfip", &ho, &wo, &to, &dlo, &ignore_index, &z_loss, &reduction, &grad)) return nullptr;
    RFB_BEGIN
    Call c;
    const at::Tensor hidden = c.first(ho, Py_None);
    rf_cross_entropy a{};
    if (c.fine) c.as_rows(hidden, c.cols, &a.hidden_rows, &a.hidden_stride);
    // another plain tensor of the call's device, contiguous, of the targets' shape
    auto per_token = [&](PyObject* o) -> at::Tensor {
        if (!c.fine || !THPVariable_Check(o) || !Call::plain(o)) return c.no();
        const at::Tensor t = THPVariable_Unpack(o);
        if (t.device() != c.device || t.dim() + 1 != (int64_t)c.shape.size() || !t.is_contiguous()) return c.no();
        for (int64_t i = 0; i < t.dim(); ++i)
            if (t.size(i) != c.shape[(size_t)i]) return c.no();
        return t;
    };
    const at::Tensor targets = per_token(to);
    if (!c.fine || (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt)) Py_RETURN_NONE;
    if (dlo != Py_None) {
        const at::Tensor dloss = per_token(dlo);
        if (!c.fine || dloss.scalar_type() != at::kFloat) Py_RETURN_NONE;
        a.dloss = (const float*)dloss.data_ptr();
    }
    if (!THPVariable_Check(wo) || !Call::plain(wo)) Py_RETURN_NONE;
    const at::Tensor weight = THPVariable_Unpack(wo);
    if (weight.device() != c.device || weight.scalar_type() != hidden.scalar_type() || weight.dim() != 2 || weight.size(1) != c.cols ||
        weight.size(0) < 1 || (weight.stride(1) != 1 && c.cols > 1))
        Py_RETURN_NONE;
    a.tokens = c.rows;
    a.vocab = weight.size(0);
    a.hidden = c.cols;
    a.dtype = code_of(hidden.scalar_type());
    a.target_bits = targets.scalar_type() == at::kLong ? 64 : 32;
    a.weight = weight.data_ptr();
    a.weight_stride = weight.stride(0);
    a.targets = targets.data_ptr();
    a.ignore_index = ignore_index;
    a.z_loss = z_loss;
    a.reduction = reduction;
    std::array<at::Tensor, 3> out;
    const at::Tensor loss = at::empty(targets.sizes(), c.options(at::kFloat));
    a.loss = (float*)loss.data_ptr();
    const bool reduced = (reduction & ~RF_GRADS_F32) != RF_REDUCE_NONE;
    out[0] = reduced ? at::empty({}, c.options(at::kFloat)) : loss;
    if (reduced) a.total = (float*)out[0].data_ptr();
    if (grad) {
        const at::ScalarType type = reduction & RF_GRADS_F32 ? at::kFloat : hidden.scalar_type();
        out[1] = c.empty(type);
        out[2] = at::empty(weight.sizes(), c.options(type));
        a.dhidden = out[1].data_ptr();
        a.dweight = out[2].data_ptr();
    }
    const char* const what = grad ? "linear_cross_entropy_grad" : "linear_cross_entropy";
    int64_t size = 0;
    check(g_lib.cross_entropy_workspace(&a, &size), what);
    const at::Tensor space = c.bytes(size);  // memory of the current stream: reused only behind this call's work
    call(c, what, [&](void* s) { return g_lib.cross_entropy(&a, space.data_ptr(), size, s); });
    return pack<3>(out);
    RFB_END
}

// gated_forward(gate, up, shape, activation, save, output) -> (h, arena, codes, exponents) or None
//   up None: gate holds both halves.  save: 0 nothing, 1 8-bit, 2 the inputs.
PyObject* py_gated_forward(PyObject*, PyObject* args)
{
    PyObject *go, *uo, *shape;
    int act, save, output;
    if (!PyArg_ParseTuple(args, "OOOiip", &go, &uo, &shape, &act, &save, &output)) return nullptr;
    RFB_BEGIN
    Call c;
    const at::Tensor gate = c.first(go, shape);
    if (!c.fine) Py_RETURN_NONE;
    rf_gated a{};
    a.dtype = code_of(gate.scalar_type());
    a.activation = act;
    if (uo == Py_None) {
        if (c.cols % 2) Py_RETURN_NONE;
        c.as_rows(gate, c.cols, &a.gate, &a.gate_stride);
        c.cols /= 2;
        c.shape.back() = c.cols;
        a.up = (const char*)a.gate + c.cols * gate.element_size();
        a.up_stride = a.gate_stride;
    } else {
        c.as_rows(gate, c.cols, &a.gate, &a.gate_stride);
        c.rows_like(uo, c.cols, a.dtype, &a.up, &a.up_stride);
    }
    if (!c.fine) Py_RETURN_NONE;
    a.rows = c.rows;
    a.cols = c.cols;
    const at::Tensor h = c.empty(gate.scalar_type());
    a.h = h.data_ptr();
    at::Tensor arena;
    if (save == 1) {
        const Arena l(c.rows, c.cols, 2);
        arena = c.bytes(l.size(0));
        void* const p = arena.data_ptr();
        a.gate_codes = l.codes(p, 0);
        a.up_codes = l.codes(p, 1);
        a.gate_exponents = l.exponents(p, 0);
        a.up_exponents = l.exponents(p, 1);
    }
    at::Tensor codes, exps;
    if (output) {
        const Kept k(c);
        codes = k.codes;
        exps = k.exponents;
        a.h_codes = k.c();
        a.h_exponents = k.e();
    }
    call(c, "gated_activation", [&](void* s) { return g_lib.gated_forward(&a, s); });
    return pack<4>({h, arena, codes, exps});
    RFB_END
}

// gated_backward(dh, shape, activation, fused, arena, gate, up) -> (dgate, dup), or one tensor, or None
//   arena None: gate and up are the saved rows.
PyObject* py_gated_backward(PyObject*, PyObject* args)
{
    PyObject *dho, *shape, *ao, *go, *uo;
    int act, fused;
    if (!PyArg_ParseTuple(args, "OOipOOO", &dho, &shape, &act, &fused, &ao, &go, &uo)) return nullptr;
    RFB_BEGIN
    Call c;
    const at::Tensor dh = c.first(dho, shape);
    rf_gated a{};
    if (c.fine) c.as_rows(dh, c.cols, &a.dh, &a.dh_stride);
    if (!c.fine) Py_RETURN_NONE;
    a.rows = c.rows;
    a.cols = c.cols;
    a.dtype = code_of(dh.scalar_type());
    a.activation = act;
    at::Tensor keep[2];
    if (ao != Py_None) {
        keep[0] = THPVariable_Unpack(ao);
        const Arena l(c.rows, c.cols, 2);
        if (!c.kept_bytes(keep[0], l.size(0))) Py_RETURN_NONE;
        void* const p = keep[0].data_ptr();
        a.gate_codes = l.codes(p, 0);
        a.up_codes = l.codes(p, 1);
        a.gate_exponents = l.exponents(p, 0);
        a.up_exponents = l.exponents(p, 1);
    } else {
        keep[0] = THPVariable_Unpack(go);
        keep[1] = THPVariable_Unpack(uo);
        if (!c.kept(keep[0], dh.scalar_type()) || !c.kept(keep[1], dh.scalar_type())) Py_RETURN_NONE;
        c.as_rows(keep[0], c.cols, &a.gate, &a.gate_stride);
        c.as_rows(keep[1], c.cols, &a.up, &a.up_stride);
        if (!c.fine) Py_RETURN_NONE;
    }
    at::Tensor dgate, dup;
    if (fused) {
        std::vector<int64_t> both = c.shape;
        both.back() *= 2;
        dgate = at::empty(both, c.options(dh.scalar_type()));
        a.dgate = dgate.data_ptr();
        a.dup = (char*)a.dgate + c.cols * dgate.element_size();
        a.dgate_stride = a.dup_stride = 2 * c.cols;
    } else {
        dgate = c.empty(dh.scalar_type());
        dup = c.empty(dh.scalar_type());
        a.dgate = dgate.data_ptr();
        a.dup = dup.data_ptr();
        a.dgate_stride = a.dup_stride = c.cols;
    }
    call(c, "gated_activation_grad", [&](void* s) { return g_lib.gated_backward(&a, s); });
    if (fused) return THPVariable_Wrap(dgate);
    return pack<2>({dgate, dup});
    RFB_END
}

int stats_of(int32_t kind) { return kind == RF_NORM_RMS ? 1 : kind == RF_NORM_LAYER ? 2 : 0; }

// norm_forward(x, branch, shape, (weight, bias, gate, next_weight, next_bias), post, next, post_eps, next_eps,
//              branch_scale, residual_scale, dtype, save, output)
//   -> (out, y, arena, gates, codes, exponents) or None.  x: the residual, or with post absent the input.
//   dtype: y's where there is no branch, or None.
PyObject* py_norm_forward(PyObject*, PyObject* args)
{
    PyObject *xo, *bo, *shape, *wo, *bias, *gate, *w2, *b2, *dtype;
    int post, next, save, output;
    rf_norm a{};
    if (!PyArg_ParseTuple(args, "OOO(OOOOO)iiffffOip", &xo, &bo, &shape, &wo, &bias, &gate, &w2, &b2, &post, &next,
                          &a.post_eps, &a.next_eps, &a.branch_scale, &a.residual_scale, &dtype, &save, &output))
        return nullptr;
    RFB_BEGIN
    Call c;
    const at::Tensor x = c.first(xo, shape);
    if (!c.fine) Py_RETURN_NONE;
    a.dtype = code_of(x.scalar_type());
    a.post = post;
    a.next = next;
    at::ScalarType y_type = x.scalar_type();
    const void* p = nullptr;
    c.as_rows(x, c.cols, &p, &a.residual_stride);
    at::Tensor branch;
    if (post) {
        a.residual = p;
        branch = c.rows_like(bo, c.cols, -1, &a.branch, &a.branch_stride);
        if (!c.fine) Py_RETURN_NONE;
        y_type = branch.scalar_type();
    } else {
        a.hidden = const_cast<void*>(p);
        a.hidden_stride = a.residual_stride;
        if (dtype != Py_None) y_type = ((THPDtype*)dtype)->scalar_type;
    }
    a.branch_dtype = code_of(y_type);
    c.vector(wo, &a.weight, &a.weight_dtype);
    c.vector(bias, &a.bias, &a.bias_dtype);
    c.gate(gate, &a.gate, &a.gate_dtype, &a.gates);
    c.vector(w2, &a.next_weight, &a.next_weight_dtype);
    c.vector(b2, &a.next_bias, &a.next_bias_dtype);
    if (!c.fine) Py_RETURN_NONE;
    a.rows = c.rows;
    a.cols = c.cols;
    at::Tensor out, y, arena, codes, exps;
    if (post) {
        out = c.empty(x.scalar_type());
        a.hidden = out.data_ptr();
        a.hidden_stride = c.cols;
    }
    if (next) {
        y = c.empty(y_type);
        a.y = y.data_ptr();
    }
    if (save) {
        const Arena l(c.rows, c.cols, save == 1 ? (post != 0) + (next != 0) : 0);
        const int post_stats = stats_of(post), next_stats = stats_of(next);
        arena = c.bytes(l.size(post_stats + next_stats));
        void* const q = arena.data_ptr();
        if (save == 1) {
            if (post) {
                a.branch_codes = l.codes(q, 0);
                a.branch_exponents = l.exponents(q, 0);
            }
            if (next) {
                a.hidden_codes = l.codes(q, post ? 1 : 0);
                a.hidden_exponents = l.exponents(q, post ? 1 : 0);
            }
        }
        if (post_stats) a.post_rstd = l.stats(q, 0);
        if (post_stats == 2) a.post_mean = l.stats(q, 1);
        if (next_stats) a.next_rstd = l.stats(q, post_stats);
        if (next_stats == 2) a.next_mean = l.stats(q, post_stats + 1);
    }
    if (output) {
        const Kept k(c);
        codes = k.codes;
        exps = k.exponents;
        a.y_codes = k.c();
        a.y_exponents = k.e();
    }
    call(c, post ? "postnorm_residual" : "prenorm", [&](void* s) { return g_lib.norm_forward(&a, s); });
    PyObject* const t = pack<6>({out, y, arena, at::Tensor(), codes, exps});
    if (t) {
        PyObject* const n = PyLong_FromLongLong(a.gates);
        if (!n) {
            Py_DECREF(t);
            return nullptr;
        }
        Py_DECREF(PyTuple_GET_ITEM(t, 3));
        PyTuple_SET_ITEM(t, 3, n);
    }
    return t;
    RFB_END
}

// norm_backward(dhidden, dy, shape, vectors, (gates, post, next, branch_scale, residual_scale, save), dtype,
//               branch dtype, arena, branch, hidden)
//   -> (dresidual, dbranch, dweight, dbias, dgate, dnext_weight, dnext_bias) or None
PyObject* py_norm_backward(PyObject*, PyObject* args)
{
    PyObject *dho, *dyo, *shape, *v[5], *dtype, *branch_dtype, *ao, *bo, *ho;
    int post, next, save;
    long long gates;
    rf_norm a{};
    if (!PyArg_ParseTuple(args, "OOO(OOOOO)(Liiffi)OOOOO", &dho, &dyo, &shape, &v[0], &v[1], &v[2], &v[3], &v[4], &gates,
                          &post, &next, &a.branch_scale, &a.residual_scale, &save, &dtype, &branch_dtype, &ao, &bo, &ho))
        return nullptr;
    RFB_BEGIN
    Call c;
    const at::ScalarType type = ((THPDtype*)dtype)->scalar_type, u_type = ((THPDtype*)branch_dtype)->scalar_type;
    a.dtype = code_of(type);
    a.branch_dtype = code_of(u_type);
    a.post = post;
    a.next = next;
    a.gates = gates;
    // the first of the two gradients gives the call its shape
    const at::Tensor t = c.first(next ? dyo : dho, shape);
    if (!c.fine || t.scalar_type() != (next ? u_type : type)) Py_RETURN_NONE;
    if (next) c.as_rows(t, c.cols, &a.dy, &a.dy_stride);
    else c.as_rows(t, c.cols, &a.dhidden, &a.dhidden_stride);
    if (next && dho != Py_None) c.rows_like(dho, c.cols, a.dtype, &a.dhidden, &a.dhidden_stride);
    if (!c.fine) Py_RETURN_NONE;
    a.rows = c.rows;
    a.cols = c.cols;
    const at::Tensor arena = THPVariable_Unpack(ao);
    const Arena l(c.rows, c.cols, save == 1 ? (post != 0) + (next != 0) : 0);
    const int post_stats = stats_of(post), next_stats = stats_of(next);
    if (!c.kept_bytes(arena, l.size(post_stats + next_stats))) Py_RETURN_NONE;
    void* const q = arena.data_ptr();
    at::Tensor branch, hidden;
    if (save == 1) {
        if (post) {
            a.branch_codes = l.codes(q, 0);
            a.branch_exponents = l.exponents(q, 0);
        }
        if (next) {
            a.hidden_codes = l.codes(q, post ? 1 : 0);
            a.hidden_exponents = l.exponents(q, post ? 1 : 0);
        }
    } else {
        const void* p = nullptr;
        if (post) branch = THPVariable_Unpack(bo);
        if (next) hidden = THPVariable_Unpack(ho);
        if ((post && !c.kept(branch, u_type)) || (next && !c.kept(hidden, type))) Py_RETURN_NONE;
        if (post) c.as_rows(branch, c.cols, &a.branch, &a.branch_stride);
        if (next) c.as_rows(hidden, c.cols, &p, &a.hidden_stride);
        a.hidden = const_cast<void*>(p);
        if (!c.fine) Py_RETURN_NONE;
    }
    if (post_stats) a.post_rstd = l.stats(q, 0);
    if (post_stats == 2) a.post_mean = l.stats(q, 1);
    if (next_stats) a.next_rstd = l.stats(q, post_stats);
    if (next_stats == 2) a.next_mean = l.stats(q, post_stats + 1);
    struct { const void** p; int32_t* dtype; void** grad; } const vectors[5] = {
        {&a.weight, &a.weight_dtype, &a.dweight},
        {&a.bias, &a.bias_dtype, &a.dbias},
        {&a.gate, &a.gate_dtype, &a.dgate},
        {&a.next_weight, &a.next_weight_dtype, &a.dnext_weight},
        {&a.next_bias, &a.next_bias_dtype, &a.dnext_bias}};
    std::array<at::Tensor, 7> g;
    for (int i = 0; i < 5; ++i) {
        if (v[i] == Py_None) continue;
        const at::Tensor w = THPVariable_Unpack(v[i]);
        const int64_t size = (i == 2 ? gates : 1) * c.cols;
        if (!c.kept(w, w.scalar_type()) || !w.is_contiguous() || w.numel() != size) Py_RETURN_NONE;
        g[2 + i] = at::empty(w.sizes(), c.options(w.scalar_type()));
        if (!w.numel()) continue;
        *vectors[i].p = w.data_ptr();
        *vectors[i].dtype = code_of(w.scalar_type());
        *vectors[i].grad = g[2 + i].data_ptr();
    }
    g[0] = c.empty(type);
    a.dresidual = g[0].data_ptr();
    if (post) {
        g[1] = c.empty(u_type);
        a.dbranch = g[1].data_ptr();
    }
    const char* const what = post ? "postnorm_residual_grad" : "prenorm_grad";
    int64_t size = 0;
    check(g_lib.norm_backward_workspace(&a, &size), what);
    at::Tensor space;  // memory of the current stream: reused only behind this call's work
    if (size) space = c.bytes(size);
    call(c, what, [&](void* s) { return g_lib.norm_backward(&a, size ? space.data_ptr() : nullptr, size, s); });
    return pack<7>(g);
    RFB_END
}

PyMethodDef methods[] = {
    {"set_entries", py_set_entries, METH_VARARGS, "addresses of the C entries, the raw stream function, Parameter"},
    {"checkpoint_store", py_checkpoint_store, METH_VARARGS, "(codes, exponents), or None"},
    {"checkpoint_load", py_checkpoint_load, METH_VARARGS, "the values, or None"},
    {"weight_grad", py_weight_grad, METH_VARARGS, "out, or None"},
    {"cross_entropy", py_cross_entropy, METH_VARARGS, "(loss, dhidden, dweight), or None"},
    {"gated_forward", py_gated_forward, METH_VARARGS, "(h, arena, codes, exponents), or None"},
    {"gated_backward", py_gated_backward, METH_VARARGS, "(dgate, dup) or one tensor, or None"},
    {"norm_forward", py_norm_forward, METH_VARARGS, "(out, y, arena, gates, codes, exponents), or None"},
    {"norm_backward", py_norm_backward, METH_VARARGS, "the gradients, or None"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rfblocks", "native host path of the residual-block operators", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__rfblocks(void) { return PyModule_Create(&module); }
