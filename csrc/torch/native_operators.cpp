// native_operators.cpp - the short way from Python to the operators of a mixture-of-experts layer: routing with its gradient, 4-bit
// quantisation and products.  Rules as in native_calls.cpp: None for whatever is not known for certain, an HcclResult for a launch
// that failed, entry points by address, no interpreter lock around them.
//
// The gradient of the routing is a C++ node: backward passes run on the autograd engine's thread without the interpreter.
#include "plain.h"

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include "released.h"

namespace {

using namespace hcomm_torch;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using QuantizeFn = int (*)(const void *, int, const float *, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, const int32_t *, int, void *, void *, void *);
using DequantizeFn = int (*)(const void *, const void *, int64_t, int64_t, int64_t, const int32_t *, int, void *, int, void *);
using GemmFn = int (*)(const void *, const void *, const void *, const void *, void *, int, int, int, int64_t, const int32_t *, int, void *);
using GemmSwigluFn = int (*)(const void *, const void *, const void *, const void *, const void *, const void *, void *, int, int, int, int64_t, const int32_t *, int, void *);
using RouteFn = int (*)(const void *, int, int64_t, int, int, int, int, int, float, const float *, const uint8_t *, int32_t *, float *, int32_t *, float *, float, float *, void *, void *);
using RouteBackwardFn = int (*)(const void *, int, int64_t, int, int, int, int, int, float, const uint8_t *, const int32_t *, const float *, const int32_t *, float, const float *, void *,
                                int64_t, void *);
using ScratchFn = uint64_t (*)(int, int);

// The distance of a dimension's neighbours; of a dimension of one, whatever it says, the width.
int64_t Pitch(const Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : std::max(t.stride(dim), t.size(-1)); }
// offsets: None, or a contiguous int32 vector of 2 to 1025 entries.  false: neither.
bool Offsets(PyObject *o, int dev, const Tensor **t, int *experts)
{
    *t = nullptr; *experts = 0;
    if (o == Py_None) return true;
    *t = Plain(o, dev);
    if (!*t || (*t)->scalar_type() != at::kInt || (*t)->dim() != 1 || !(*t)->is_contiguous() || (*t)->size(0) < 2 || (*t)->size(0) > 1025) return false;
    *experts = (int)(*t)->size(0) - 1;
    return true;
}
int64_t ScaleTiles(int64_t batch, int64_t rows, int64_t cols, int experts)
{
    const int64_t tileRows = experts ? rows / 128 + std::min<int64_t>(rows, experts) : batch * ((rows + 127) / 128);
    return tileRows * ((cols + 127) / 128);
}

// fp4_quantize(entry, x, scales or None, offsets or None) -> (values, scales), an error code, or None
PyObject *Quantize(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 4) Py_RETURN_NONE;
    const int dev = Device();
    const Tensor *x = dev < 0 ? nullptr : Plain(args[1], dev), *xs = nullptr, *offsets;
    int experts;
    void *entry;
    if (!x || !Offsets(args[3], dev, &offsets, &experts) || !Address(args[0], &entry)) Py_RETURN_NONE;
    const bool fp8 = x->scalar_type() == at::kFloat8_e4m3fn;
    const int type = fp8 ? (int)HCCL_DATA_TYPE_FP8E4M3 : x->scalar_type() == at::kDouble ? -1 : TypeCode(x->scalar_type());
    const int64_t dims = x->dim();
    if (!(fp8 || type == HCCL_DATA_TYPE_FP32 || type == HCCL_DATA_TYPE_FP16 || type == HCCL_DATA_TYPE_BFP16) || dims < 2 || dims > 3 || (dims == 3 && (fp8 || offsets))) Py_RETURN_NONE;
    const int64_t rows = x->size(-2), cols = x->size(-1), batch = dims == 3 ? x->size(0) : 1;
    if (x->numel() == 0 || cols % (fp8 ? 128 : 32) || x->stride(-1) != 1) Py_RETURN_NONE;
    int64_t scalePitch = 0;
    if (fp8) {
        xs = Plain(args[2], dev);
        if (!xs || xs->scalar_type() != at::kFloat || xs->dim() != 2 || xs->size(0) != rows || xs->size(1) != cols / 128 || (xs->size(1) > 1 && xs->stride(1) != 1)) Py_RETURN_NONE;
        scalePitch = Pitch(*xs, 0);
    } else if (args[2] != Py_None) Py_RETURN_NONE;
    const auto bytes = x->options().dtype(at::kByte).requires_grad(false);
    Tensor values = dims == 3 ? at::empty({batch, rows, cols / 2}, bytes) : at::empty({rows, cols / 2}, bytes);
    Tensor tiles = at::empty({ScaleTiles(batch, rows, cols, experts), 512}, bytes);
    const auto fn = (QuantizeFn)entry;
    const void *px = x->data_ptr();
    const float *ps = xs ? (const float *)xs->data_ptr() : nullptr;
    const int32_t *po = offsets ? (const int32_t *)offsets->data_ptr() : nullptr;
    void *pv = values.data_ptr(), *pt = tiles.data_ptr(), *stream = StreamOf(dev);
    const int64_t batchPitch = dims == 3 ? Pitch(*x, 0) : 0, rowPitch = Pitch(*x, -2);
    const int rc = Released([=] { return fn(px, type, ps, batch, rows, cols, batchPitch, rowPitch, scalePitch, po, experts, pv, pt, stream); });
    if (rc) return PyLong_FromLong(rc);
    PyObject *pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(values)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(tiles)));
    return pair;
    END_HANDLE_TH_ERRORS
}

struct Operand { const Tensor *values, *scales; int64_t batch, rows, cols; };
// Two arguments as a quantised matrix (or several): contiguous bytes whose sizes belong together.
bool Quantised(PyObject *values, PyObject *scales, int dev, int experts, Operand *o)
{
    o->values = Plain(values, dev); o->scales = o->values ? Plain(scales, dev) : nullptr;
    if (!o->scales || o->values->scalar_type() != at::kByte || o->scales->scalar_type() != at::kByte || !o->values->is_contiguous() || !o->scales->is_contiguous()) return false;
    const int64_t dims = o->values->dim();
    if (dims < 2 || dims > 3 || (experts && dims != 2)) return false;
    o->batch = dims == 3 ? o->values->size(0) : 1;
    o->rows = o->values->size(-2); o->cols = 2 * o->values->size(-1);
    return o->cols % 32 == 0 && o->cols <= INT32_MAX && o->rows <= INT32_MAX && o->scales->numel() == 512 * ScaleTiles(o->batch, o->rows, o->cols, experts);
}

// fp4_dequantize(entry, values, scales, offsets or None, type code, dtype) -> the result, an error code, or None
PyObject *Dequantize(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 5) Py_RETURN_NONE;
    const int dev = Device();
    const Tensor *offsets;
    int experts;
    Operand q;
    void *entry;
    if (dev < 0 || !Offsets(args[3], dev, &offsets, &experts) || !Quantised(args[1], args[2], dev, experts, &q) || !Address(args[0], &entry)) Py_RETURN_NONE;
    const long type = PyLong_AsLong(args[4]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const auto dtype = type == HCCL_DATA_TYPE_FP32 ? at::kFloat : type == HCCL_DATA_TYPE_FP16 ? at::kHalf : type == HCCL_DATA_TYPE_BFP16 ? at::kBFloat16 : at::kByte;
    if (dtype == at::kByte || q.values->numel() == 0) Py_RETURN_NONE;
    const auto options = q.values->options().dtype(dtype).requires_grad(false);
    Tensor out = q.values->dim() == 3 ? at::empty({q.batch, q.rows, q.cols}, options) : at::empty({q.rows, q.cols}, options);
    const auto fn = (DequantizeFn)entry;
    const void *pv = q.values->data_ptr(), *ps = q.scales->data_ptr();
    const int32_t *po = offsets ? (const int32_t *)offsets->data_ptr() : nullptr;
    void *to = out.data_ptr(), *stream = StreamOf(dev);
    const int64_t batch = q.batch, rows = q.rows, cols = q.cols;
    const int rc = Released([=] { return fn(pv, ps, batch, rows, cols, po, experts, to, (int)type, stream); });
    if (rc) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// fp4_gemm(entry, a values, a scales, offsets or None, out or None, b values, b scales[, the same of the up projection])
// -> the result, an error code, or None
PyObject *Gemm(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 7 && n != 9) Py_RETURN_NONE;
    const bool gated = n == 9;
    const int dev = Device();
    const Tensor *offsets;
    int experts;
    Operand a, b, u;
    void *entry;
    if (dev < 0 || !Offsets(args[3], dev, &offsets, &experts) || !Quantised(args[1], args[2], dev, experts, &a) || !Quantised(args[5], args[6], dev, 0, &b) ||
        (gated && !Quantised(args[7], args[8], dev, 0, &u)) || !Address(args[0], &entry))
        Py_RETURN_NONE;
    const int64_t dims = experts ? 3 : 2;
    if (a.values->dim() != 2 || b.values->dim() != dims || b.cols != a.cols || (experts && b.batch != experts) || (gated && u.values->sizes() != b.values->sizes())) Py_RETURN_NONE;
    const int64_t m = a.rows, w = b.rows, k = a.cols;
    constexpr int64_t kMost = INT32_MAX - 256;          // of a product, as the entry points have it
    if (m == 0 || w == 0 || k == 0 || m > kMost || w > kMost || k > kMost) Py_RETURN_NONE;
    Tensor made;
    const Tensor *out = &made;
    if (args[4] == Py_None) made = at::empty({m, w}, a.values->options().dtype(at::kBFloat16).requires_grad(false));
    else if (!(out = Plain(args[4], dev)) || out->scalar_type() != at::kBFloat16 || out->dim() != 2 || out->size(0) != m || out->size(1) != w || (w > 1 && out->stride(1) != 1) ||
             (m > 1 && out->stride(0) < w))
        Py_RETURN_NONE;
    const void *av = a.values->data_ptr(), *as = a.scales->data_ptr(), *bv = b.values->data_ptr(), *bs = b.scales->data_ptr();
    const void *uv = gated ? u.values->data_ptr() : nullptr, *us = gated ? u.scales->data_ptr() : nullptr;
    const int32_t *po = offsets ? (const int32_t *)offsets->data_ptr() : nullptr;
    void *to = out->data_ptr(), *stream = StreamOf(dev);
    const int64_t ld = Pitch(*out, 0);
    const int rc = Released([=] {
        return gated ? ((GemmSwigluFn)entry)(av, as, bv, bs, uv, us, to, (int)m, (int)w, (int)k, ld, po, experts, stream)
                     : ((GemmFn)entry)(av, as, bv, bs, to, (int)m, (int)w, (int)k, ld, po, experts, stream);
    });
    if (rc) return PyLong_FromLong(rc);
    if (args[4] != Py_None) return Py_NewRef(args[4]);
    return THPVariable_Wrap(std::move(made));
    END_HANDLE_TH_ERRORS
}

struct RouteCall {
    RouteFn forward;
    RouteBackwardFn backward;
    ScratchFn scratch;
    int topk, scoring, renormalize;
    float scale, balance;
    bool lossWanted;            // balance as it was given is not 0, though as a float it may be
    const Tensor *bias, *valid;
};
struct Routed {
    Tensor idx, gates, counts, loss;
    int rc;
};
Routed Forward(const RouteCall &c, const Tensor &x)
{
    const int64_t t = x.size(0), e = x.size(1);
    const auto ints = x.options().dtype(at::kInt).requires_grad(false), floats = x.options().dtype(at::kFloat).requires_grad(false);
    Routed r{at::empty({t, c.topk}, ints), at::empty({t, c.topk}, floats), at::empty({e + 1}, ints), Tensor(), 0};
    if (c.lossWanted) r.loss = at::empty({}, floats);
    const int64_t bytes = (int64_t)c.scratch((int)t, (int)e);
    Tensor scratch;
    if (bytes) scratch = at::empty({bytes / 4}, ints);
    r.rc = c.forward(x.data_ptr(), TypeCode(x.scalar_type()), Pitch(x, 0), (int)t, (int)e, c.topk, c.scoring, c.renormalize, c.scale, c.bias ? (const float *)c.bias->data_ptr() : nullptr,
                     c.valid ? (const uint8_t *)c.valid->data_ptr() : nullptr, (int32_t *)r.idx.data_ptr(), (float *)r.gates.data_ptr(), (int32_t *)r.counts.data_ptr(), nullptr, c.balance,
                     r.loss.defined() ? (float *)r.loss.data_ptr() : nullptr, bytes ? scratch.data_ptr() : nullptr, StreamOf(x.get_device()));
    return r;
}

// The routing in the autograd graph: inputs of the node are the gradients of gates and loss, its output that of the logits.
struct RouteNode : public torch::autograd::Node {
    SavedVariable x, valid, idx, counts;
    RouteBackwardFn backward;
    int topk, scoring, renormalize;
    float scale, balance;

    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        Tensor dgates = grads[0], dloss = grads.size() > 1 ? grads[1] : Tensor();
        if (!task_should_compute_output(0) || (!dgates.defined() && !dloss.defined())) return {Tensor()};
        const bool again = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        const Tensor l = x.unpack(), v = valid.unpack(), i = idx.unpack(), n = counts.unpack();
        if (dgates.defined()) dgates = dgates.contiguous();
        Tensor dx = at::empty({l.size(0), l.size(1)}, l.options().requires_grad(false));
        const int rc = backward(l.data_ptr(), TypeCode(l.scalar_type()), Pitch(l, 0), (int)l.size(0), (int)l.size(1), topk, scoring, renormalize, scale,
                                v.defined() ? (const uint8_t *)v.data_ptr() : nullptr, (const int32_t *)i.data_ptr(), dgates.defined() ? (const float *)dgates.data_ptr() : nullptr,
                                (const int32_t *)n.data_ptr(), balance, dloss.defined() ? (const float *)dloss.data_ptr() : nullptr, dx.data_ptr(), l.size(1), StreamOf(l.get_device()));
        TORCH_CHECK(rc == 0, "HcommMoeRouteBackward failed with ", rc);
        if (again) {        // a gradient of the gradient is not offered: asking for it is an error, not a silent zero
            dx.set_requires_grad(true);
            auto error = std::make_shared<torch::autograd::DelayedError>("route: the backward pass is not differentiable", 1);
            dx = (*error)({dx})[0];
        }
        return {dx};
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(); valid.reset_data(); idx.reset_data(); counts.reset_data();
    }
    std::string name() const override { return "RouteBackward"; }
};
Routed ForwardWithGraph(const RouteCall &c, const Tensor &x)
{
    Routed r;
    {
        at::AutoGradMode off(false);
        r = Forward(c, x);
    }
    if (r.rc) return r;
    std::shared_ptr<RouteNode> node(new RouteNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->x = SavedVariable(x, false);
    node->valid = SavedVariable(c.valid ? *c.valid : Tensor(), false);
    node->idx = SavedVariable(r.idx, false);
    node->counts = SavedVariable(r.counts, false);
    node->backward = c.backward;
    node->topk = c.topk; node->scoring = c.scoring; node->renormalize = c.renormalize;
    node->scale = c.scale; node->balance = c.balance;
    torch::autograd::set_history(r.gates, node);
    if (r.loss.defined()) torch::autograd::set_history(r.loss, node);
    return r;
}

// moe_route(entry, backward entry, scratch size entry, logits, topk, scoring, renormalize, scale, bias or None, valid or None, balance)
// -> (choices, gates, counts with the number of tokens behind them, loss or None), an error code, or None
PyObject *Route(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 11) Py_RETURN_NONE;
    const int dev = Device();
    const Tensor *x = dev < 0 ? nullptr : Plain(args[3], dev);
    if (!x || x->dim() != 2 || (x->scalar_type() != at::kFloat && x->scalar_type() != at::kHalf && x->scalar_type() != at::kBFloat16)) Py_RETURN_NONE;
    if (x->_fw_grad(0).defined()) Py_RETURN_NONE;       // forward mode, which the general way refuses
    void *f, *b, *s;
    if (!Address(args[0], &f) || !Address(args[1], &b) || !Address(args[2], &s)) Py_RETURN_NONE;
    const long topk = PyLong_AsLong(args[4]);           // whole: 2^32 + 2 is not 2
    if (topk < 1 || topk > 16) { PyErr_Clear(); Py_RETURN_NONE; }
    RouteCall c{(RouteFn)f, (RouteBackwardFn)b, (ScratchFn)s, (int)topk, (int)PyLong_AsLong(args[5]), (int)PyLong_AsLong(args[6]),
                (float)PyFloat_AsDouble(args[7]), (float)PyFloat_AsDouble(args[10]), PyFloat_AsDouble(args[10]) != 0, nullptr, nullptr};
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const int64_t t = x->size(0), e = x->size(1);
    if (t < 1 || t > INT32_MAX || e < 1 || e > 1024 || topk > e || (e > 1 && x->stride(1) != 1) || (t > 1 && x->stride(0) < e)) Py_RETURN_NONE;
    if (args[8] != Py_None) {
        c.bias = Plain(args[8], dev);
        if (!c.bias || c.scoring != 1 || c.bias->scalar_type() != at::kFloat || c.bias->dim() != 1 || c.bias->size(0) != e || !c.bias->is_contiguous()) Py_RETURN_NONE;
    }
    if (args[9] != Py_None) {
        c.valid = Plain(args[9], dev);
        if (!c.valid || c.valid->scalar_type() != at::kBool || c.valid->dim() != 1 || c.valid->size(0) != t || !c.valid->is_contiguous()) Py_RETURN_NONE;
    }
    Tensor idx, gates, counts, loss;
    int rc = 0;
    {
        pybind11::gil_scoped_release unlocked;
        Routed r = x->requires_grad() && at::GradMode::is_enabled() ? ForwardWithGraph(c, *x) : Forward(c, *x);
        idx = std::move(r.idx); gates = std::move(r.gates); counts = std::move(r.counts); loss = std::move(r.loss);
        rc = r.rc;
        if (!rc) counts = counts.narrow(0, 0, e);
    }
    if (rc) return PyLong_FromLong(rc);
    PyObject *tuple = PyTuple_New(4);
    if (!tuple) return nullptr;
    PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(idx)));
    PyTuple_SET_ITEM(tuple, 1, THPVariable_Wrap(std::move(gates)));
    PyTuple_SET_ITEM(tuple, 2, THPVariable_Wrap(std::move(counts)));
    PyTuple_SET_ITEM(tuple, 3, loss.defined() ? THPVariable_Wrap(std::move(loss)) : Py_NewRef(Py_None));
    return tuple;
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"fp4_quantize", (PyCFunction)(void *)Quantize, METH_FASTCALL, nullptr},
    {"fp4_dequantize", (PyCFunction)(void *)Dequantize, METH_FASTCALL, nullptr},
    {"fp4_gemm", (PyCFunction)(void *)Gemm, METH_FASTCALL, nullptr},
    {"moe_route", (PyCFunction)(void *)Route, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

namespace hcomm_torch {
bool AddNativeOperators(PyObject *module) { return PyModule_AddFunctions(module, kMethods) == 0; }
}  // namespace hcomm_torch
