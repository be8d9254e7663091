// Calls of the sequence, gated and 4-bit operators from Python without ctypes: one token through a layer takes a few
// microseconds on the GPU, and marshalling it in Python takes three times as long.  The functions here take tensors, check
// where they live, allocate the results and call the C ABI (include/srt_matmul_api.h) on torch's current stream; the public
// functions with their documentation are in linear_recurrent.py, dense.py and int4.py.
//
// Only torch's tensors, allocator and streams are used; nothing is computed here.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <optional>
#include <utility>

#include "srt_matmul_api.h"

namespace {

PyObject* g_error_class = nullptr;              // MatmulError(code, text)
PyObject* g_memory_class = nullptr;             // torch.OutOfMemoryError

struct PythonError {};                          // a Python exception is set

const at::Tensor* tensor_or_null(PyObject* o, const char* what)
{
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", what);
        throw PythonError{};
    }
    return &THPVariable_Unpack(o);
}

const at::Tensor& tensor(PyObject* o, const char* what)
{
    const at::Tensor* t = tensor_or_null(o, what);
    if (!t) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", what);
        throw PythonError{};
    }
    return *t;
}

// all tensors (null is skipped) on the CUDA device of the first
void on_one_device(std::initializer_list<const at::Tensor*> tensors)
{
    const at::Tensor& first = **tensors.begin();
    if (!first.is_cuda()) {
        PyErr_SetString(PyExc_ValueError, "device tensors expected");
        throw PythonError{};
    }
    for (const at::Tensor* t : tensors)
        if (t && t->device() != first.device()) {
            PyErr_Format(PyExc_ValueError, "tensors on different devices: %s and %s", first.device().str().c_str(), t->device().str().c_str());
            throw PythonError{};
        }
}

bool truth(PyObject* o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError{};
    return v != 0;
}

srtDataType data_type(const at::Tensor& t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return real32F;
    case at::kHalf: return real16F;
    case at::kBFloat16: return real16BF;
    default: return srtUnknownType;
    }
}

// a tensor as the C ABI takes it, for the duration of a call
struct Arg {
    void* p = nullptr;
    srtTensorDescriptor d;
    const srtTensorDescriptor* desc = nullptr;
    Arg(const at::Tensor* t)
    {
        if (!t) return;
        static_assert(sizeof(size_t) == sizeof(int64_t), "sizes and strides are passed in place");
        p = t->data_ptr();
        d.type = data_type(*t);
        d.rank = static_cast<uint32_t>(t->dim());
        d.order = srtOrderRow;
        d.count = d.spanCount = static_cast<size_t>(t->numel());
        d.shape = reinterpret_cast<const size_t*>(t->sizes().data());
        d.strides = d.logicalStrides = reinterpret_cast<const size_t*>(t->strides().data());
        desc = &d;
    }
    Arg(const at::Tensor& t) : Arg(&t) {}
    Arg(const Arg&) = delete;
};

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device)
{
    return at::detail::empty_cuda(sizes, type, device, std::nullopt);
}

// two matrices in one allocation, both starting on 16 bytes: a dense [2 x rows x cols] tensor where that is one
std::pair<at::Tensor, at::Tensor> empty_pair(int64_t rows, int64_t cols, at::ScalarType type, const at::Device& device)
{
    const int64_t unit = 16 / static_cast<int64_t>(c10::elementSize(type)), apart = (rows * cols + unit - 1) / unit * unit;
    const at::Tensor whole = empty({apart + rows * cols}, type, device);
    const auto part = [&](int64_t offset) {
        auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
        impl->set_storage_offset(offset);
        const int64_t sizes[2] = {rows, cols};
        impl->set_sizes_contiguous(sizes);
        return at::Tensor(std::move(impl));
    };
    return {part(0), part(apart)};
}

// the device made current where it is not, and torch's current stream there
struct Queue {
    c10::cuda::OptionalCUDAGuard guard;
    cudaStream_t stream;
    explicit Queue(const at::Tensor& t)
    {
        if (c10::cuda::current_device() != t.device().index()) guard.set_device(t.device());
        stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
    }
};

void check(cudaError_t rc)
{
    if (rc == cudaSuccess) return;
    PyObject* e = PyObject_CallFunction(g_error_class, "is", static_cast<int>(rc), srtMatmulGetLastErrorString());
    if (e) {
        PyErr_SetObject(g_error_class, e);
        Py_DECREF(e);
    }
    throw PythonError{};
}

const int32_t* lengths_pointer(const at::Tensor* t, int64_t batch)
{
    if (!t) return nullptr;
    if (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != batch || (batch > 1 && t->stride(0) != 1)) {
        PyErr_Format(PyExc_ValueError, "lengths must be a contiguous int32 tensor of %lld elements", static_cast<long long>(batch));
        throw PythonError{};
    }
    return t->data_ptr<int32_t>();
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

PyObject* pack(std::initializer_list<const at::Tensor*> tensors)
{
    PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    Py_ssize_t i = 0;
    for (const at::Tensor* t : tensors) {
        PyObject* o = t && t->defined() ? wrap(*t) : Py_NewRef(Py_None);
        PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
}

// runs f, which may throw PythonError or a C++ exception, and turns either into a Python exception
template <typename F> PyObject* guarded(Py_ssize_t n, Py_ssize_t expected, F f)
{
    if (n != expected) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", expected, n);
        return nullptr;
    }
    try {
        return f();
    } catch (const PythonError&) {
    } catch (const c10::Error& e) {
        // out of memory keeps torch's own class, which callers catch
        PyErr_SetString(dynamic_cast<const c10::OutOfMemoryError*>(&e) ? g_memory_class : PyExc_RuntimeError,
                        e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

void sequence_rank(const at::Tensor& t)
{
    if (t.dim() == 2 || t.dim() == 3) return;
    PyErr_SetString(PyExc_ValueError, "update must be [batch, steps, channels], or [batch, channels] for one step");
    throw PythonError{};
}

// (update, forget, input, output, initial, lengths, keep, last) -> (hidden, last) or (hidden, last, states)
PyObject* recurrence(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 8, [&]() -> PyObject* {
        const at::Tensor& update = tensor(a[0], "update");
        const at::Tensor& forget = tensor(a[1], "forget");
        const at::Tensor *input = tensor_or_null(a[2], "input"), *output = tensor_or_null(a[3], "output"), *initial = tensor_or_null(a[4], "initial"),
                         *lengths = tensor_or_null(a[5], "lengths"), *given = tensor_or_null(a[7], "last");
        const bool keep = truth(a[6]);
        on_one_device({&update, &forget, input, output, initial, lengths, given});
        sequence_rank(update);
        const int64_t batch = update.size(0), channels = update.size(-1), steps = update.dim() == 3 ? update.size(1) : 1;
        const int32_t* const n_steps = lengths_pointer(lengths, batch);
        Queue q(update);
        const at::Tensor hidden = empty(update.sizes(), update.scalar_type(), update.device());
        const at::Tensor last = given ? *given : empty({batch, channels}, at::kFloat, update.device());
        at::Tensor states;
        if (keep) states = empty({batch, (steps + SRT_GATED_RECURRENCE_CHUNK - 1) / SRT_GATED_RECURRENCE_CHUNK, channels}, at::kFloat, update.device());
        const Arg u(update), f(forget), i(input), o(output), c(initial), h(hidden), l(last), s(keep ? &states : nullptr);
        // (a kept tensor without elements has no address, and is given all the same)
        check(srtGatedRecurrence(u.p, u.desc, f.p, f.desc, i.p, i.desc, o.p, o.desc, c.p, c.desc, n_steps, h.p, h.desc, l.p, l.desc, s.p, s.desc, q.stream));
        return keep ? pack({&hidden, &last, &states}) : pack({&hidden, &last});
    });
}

// (outGrad, update, forget, input, output, states, lengths, lastGrad, dUpdate, dForget, dInput, dOutput) -> the four and dInitial; the
// four gradients are all given or all None
PyObject* recurrence_backward(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 12, [&]() -> PyObject* {
        const at::Tensor& grad = tensor(a[0], "out_grad");
        const at::Tensor& update = tensor(a[1], "update");
        const at::Tensor& forget = tensor(a[2], "forget");
        const at::Tensor *input = tensor_or_null(a[3], "input"), *output = tensor_or_null(a[4], "output");
        const at::Tensor& states = tensor(a[5], "states");
        const at::Tensor *lengths = tensor_or_null(a[6], "lengths"), *last_grad = tensor_or_null(a[7], "last_grad");
        const at::Tensor* given[4] = {tensor_or_null(a[8], "out"), tensor_or_null(a[9], "out"), tensor_or_null(a[10], "out"), tensor_or_null(a[11], "out")};
        on_one_device({&update, &grad, &forget, input, output, &states, lengths, last_grad, given[0], given[1], given[2], given[3]});
        sequence_rank(update);
        const int64_t batch = update.size(0), channels = update.size(-1);
        const int32_t* const n_steps = lengths_pointer(lengths, batch);
        Queue q(update);
        at::Tensor out[4];
        const bool wanted[4] = {true, true, input != nullptr, output != nullptr};
        const bool allocate = !given[0] && !given[1] && !given[2] && !given[3];
        for (int k = 0; k < 4; ++k) {
            if (!wanted[k]) continue;
            if (allocate) out[k] = empty(update.sizes(), update.scalar_type(), update.device());
            else if (given[k]) out[k] = *given[k];
        }
        const at::Tensor initial_grad = empty({batch, channels}, at::kFloat, update.device());
        const Arg g(grad), lg(last_grad), u(update), f(forget), i(input), o(output), s(states);
        auto opt = [](const at::Tensor& t) { return t.defined() ? &t : nullptr; };
        const Arg du(opt(out[0])), df(opt(out[1])), di(opt(out[2])), dout(opt(out[3])), dc(initial_grad);
        check(srtGatedRecurrenceBackward(g.p, g.desc, lg.p, lg.desc, u.p, u.desc, f.p, f.desc, i.p, i.desc, o.p, o.desc, s.p, s.desc, n_steps, du.p, du.desc,
                                         df.p, df.desc, di.p, di.desc, dout.p, dout.desc, dc.p, dc.desc, q.stream));
        return pack({&out[0], &out[1], &out[2], &out[3], &initial_grad});
    });
}

// (x, wGate, wUp, biasGate, biasUp, activation, keep) -> y or (y, gate, up).  A product that is not one launch needs gate and up
// whether they are kept or not.
PyObject* gated(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 7, [&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "input");
        const at::Tensor& wg = tensor(a[1], "weight_gate");
        const at::Tensor& wu = tensor(a[2], "weight_up");
        const at::Tensor *bg = tensor_or_null(a[3], "bias_gate"), *bu = tensor_or_null(a[4], "bias_up");
        const auto act = static_cast<srtActivationType>(PyLong_AsLong(a[5]));
        const bool keep = truth(a[6]);
        on_one_device({&x, &wg, &wu, bg, bu});
        if (x.dim() != 2 || wg.dim() != 2) {
            PyErr_SetString(PyExc_ValueError, "matrices expected");
            throw PythonError{};
        }
        Queue q(x);
        const int64_t shape[2] = {x.size(0), wg.size(1)};
        const at::Tensor y = empty(shape, x.scalar_type(), x.device());
        const Arg ax(x), ag(wg), au(wu), bga(bg), bua(bu), ay(y);
        auto call = [&](const at::Tensor* gate, const at::Tensor* up) {
            const Arg kg(gate), ku(up);
            return srtMatmulGated(ax.p, ax.desc, ag.p, ag.desc, au.p, au.desc, bga.p, bga.desc, bua.p, bua.desc, act, kg.p, kg.desc, ku.p, ku.desc, ay.p, ay.desc, q.stream);
        };
        cudaError_t rc = cudaErrorNotSupported;
        if (!keep) rc = call(nullptr, nullptr);
        at::Tensor gate, up;
        if (rc == cudaErrorNotSupported) {
            gate = empty(shape, x.scalar_type(), x.device());
            up = empty(shape, x.scalar_type(), x.device());
            rc = call(&gate, &up);
        }
        check(rc);
        return keep ? pack({&y, &gate, &up}) : wrap(y);
    });
}

// (x, outGrad, wGate, wUp, gate, up, biasGate, biasUp, activation) -> gradients of x, wGate, wUp, biasGate and biasUp (None where the
// bias is None)
PyObject* gated_backward(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 9, [&]() -> PyObject* {
        const at::Tensor &x = tensor(a[0], "input"), &grad = tensor(a[1], "out_grad"), &wg = tensor(a[2], "weight_gate"), &wu = tensor(a[3], "weight_up"),
                         &gate = tensor(a[4], "saved"), &up = tensor(a[5], "saved");
        const at::Tensor *bg = tensor_or_null(a[6], "bias_gate"), *bu = tensor_or_null(a[7], "bias_up");
        const auto act = static_cast<srtActivationType>(PyLong_AsLong(a[8]));
        on_one_device({&x, &grad, &wg, &wu, &gate, &up, bg, bu});
        if (x.dim() != 2 || wg.dim() != 2) {
            PyErr_SetString(PyExc_ValueError, "matrices expected");
            throw PythonError{};
        }
        Queue q(x);
        const at::ScalarType type = x.scalar_type();
        const int64_t rows = x.size(0), inner = x.size(1), cols = wg.size(1);
        // the matrices of a pair lie behind each other: batched products
        const auto [dgate, dup] = empty_pair(rows, cols, type, x.device());
        const auto [dwg, dwu] = empty_pair(inner, cols, type, x.device());
        const at::Tensor dx = empty({rows, inner}, type, x.device());
        at::Tensor dbg, dbu, dx2;
        if (bg) dbg = empty(bg->sizes(), type, x.device());
        if (bu) dbu = empty(bu->sizes(), type, x.device());
        auto opt = [](const at::Tensor& t) { return t.defined() ? &t : nullptr; };
        const Arg ay(grad), ax(x), ag(wg), au(wu), kg(gate), ku(up), dg(dgate), du(dup), ox(dx), og(dwg), ou(dwu), sg(opt(dbg)), su(opt(dbu));
        auto call = [&] {
            const Arg ox2(opt(dx2));
            return srtMatmulGatedBackward(ay.p, ay.desc, ax.p, ax.desc, ag.p, ag.desc, au.p, au.desc, kg.p, kg.desc, ku.p, ku.desc, act, dg.p, dg.desc, du.p, du.desc,
                                          ox.p, ox.desc, ox2.p, ox2.desc, og.p, og.desc, ou.p, ou.desc, sg.p, sg.desc, su.p, su.desc, q.stream);
        };
        cudaError_t rc = cudaErrorNotSupported;
        if (type != at::kFloat) rc = call();
        if (rc == cudaErrorNotSupported) {                       // an input gradient in two products needs a place for the second
            dx2 = empty({rows, inner}, type, x.device());
            rc = call();
        }
        check(rc);
        return pack({&dx, &dwg, &dwu, &dbg, &dbu});
    });
}

// (x, address of the weight's srtInt4Matrix, address of a second one or 0, a tensor of the weights, columns, bias, second bias,
// activation) -> y
PyObject* int4(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 8, [&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "x");
        const auto* w0 = static_cast<const srtInt4Matrix*>(PyLong_AsVoidPtr(a[1]));
        const auto* w1 = static_cast<const srtInt4Matrix*>(PyLong_AsVoidPtr(a[2]));
        const at::Tensor& packed = tensor(a[3], "packed");
        const int64_t cols = PyLong_AsLongLong(a[4]);
        const at::Tensor *b0 = tensor_or_null(a[5], "bias"), *b1 = tensor_or_null(a[6], "bias");
        const auto act = static_cast<srtActivationType>(PyLong_AsLong(a[7]));
        on_one_device({&x, &packed, b0, b1});
        if (x.dim() != 2) {
            PyErr_SetString(PyExc_ValueError, "a matrix expected");
            throw PythonError{};
        }
        Queue q(x);
        const at::Tensor y = empty({x.size(0), cols}, x.scalar_type(), x.device());
        const Arg ax(x), ab0(b0), ab1(b1), ay(y);
        check(w1 ? srtMatmulGatedInt4(ax.p, ax.desc, w0, w1, ab0.p, ab0.desc, ab1.p, ab1.desc, act, ay.p, ay.desc, q.stream)
                 : srtMatmulInt4(ax.p, ax.desc, w0, ab0.p, ab0.desc, act, ay.p, ay.desc, q.stream));
        return wrap(y);
    });
}

PyObject* set_error_classes(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 2, [&]() -> PyObject* {
        Py_XDECREF(g_error_class);
        Py_XDECREF(g_memory_class);
        g_error_class = Py_NewRef(a[0]);
        g_memory_class = Py_NewRef(a[1]);
        Py_RETURN_NONE;
    });
}

PyMethodDef kMethods[] = {
    {"recurrence", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(recurrence)), METH_FASTCALL, nullptr},
    {"recurrence_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(recurrence_backward)), METH_FASTCALL, nullptr},
    {"gated", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated)), METH_FASTCALL, nullptr},
    {"gated_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated_backward)), METH_FASTCALL, nullptr},
    {"int4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(int4)), METH_FASTCALL, nullptr},
    {"set_error_classes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_error_classes)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
