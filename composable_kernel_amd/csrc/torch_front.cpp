// The short way from a torch call to the library, for the fp8 operators.
//
// A small call is bound by the host: of the 11 us that rmsnorm_fp8 of one row took from Python, its kernel runs 3; three output
// tensors cost 4 there and 2 here, reading and checking the operands 4 and under 1.  This module takes the plain calls: plain
// torch.Tensor operands of the right types and shapes on the current device, contiguous or (the row operands) strided by rows, while
// nothing records, transforms or fakes the calls of this thread.  It answers None to everything else -- what has to be copied,
// converted or refused goes the long way in torch_ops.py, which says why, and what is recorded or transformed goes to the
// registered operators.  Outputs come from torch's caching allocator, the launch goes to the current stream of the operands' device.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include "wqgemm.h"

namespace {

// the library is loaded by the caller (capi.py); these are its entry points, handed over once by bind()
int (*quantize)(const wqgemm_quant*, void*)               = nullptr;
int (*launch)(const wqgemm_problem*, void*, void*)        = nullptr;
size_t (*workspace_bytes)(const wqgemm_problem*)          = nullptr;
const char* (*last_error)()                               = nullptr;
PyObject* error_type                                      = nullptr;

bool current_device_is(c10::Device d)
{
    return d.is_cuda() && c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice().index() == d.index();
}

// A dispatch mode (fake tensors, a tracer's proxies), a functorch transform or torch.jit.trace stands between this thread's calls and
// the kernels: it has to see the registered operator, not the allocations of its outputs.
bool intercepted()
{
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet k({K::Python, K::PythonTLSSnapshot, K::PythonDispatcher, K::PreDispatch, K::Tracer, K::Functionalize,
                                     K::FuncTorchDynamicLayerFrontMode, K::FuncTorchDynamicLayerBackMode, K::FuncTorchVmapMode,
                                     K::FuncTorchBatched, K::FuncTorchGradWrapper});
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    return c10::impl::TorchDispatchModeTLS::any_modes_set() || (tls.included_ - tls.excluded_).has_any(k);
}

// rows of `cols` contiguous elements: (rows, distance between them), or false where the layout cannot be read as such
bool as_rows(const at::Tensor& t, int64_t cols, int64_t& rows, int64_t& ld)
{
    if(t.is_contiguous())
        rows = t.numel() / cols, ld = cols;
    else if(t.dim() == 2 && (t.stride(1) == 1 || cols == 1) && t.size(0) > 1 && t.stride(0) >= cols)
        rows = t.size(0), ld = t.stride(0);
    else
        return false;
    return rows > 0 && rows <= INT32_MAX && ld <= INT32_MAX;
}

// a plain torch.Tensor (no subclass) on device d (any GPU if d is null) that needs no gradient and carries no tangent
const at::Tensor* plain(PyObject* o, const c10::Device* d)
{
    if(!THPVariable_CheckExact(o))
        return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if(!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || (d && t.device() != *d) || t.is_conj() || t.is_neg() ||
       (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined())
        return nullptr;
    return &t;
}

// other Python threads run while memory is allocated and the kernel is launched: either may wait for the device
struct WithoutGil
{
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

// the raw handle of the device's current stream, from the function that the caller passes; false with an exception set, or if it is none
bool current_stream(PyObject* f, c10::Device d, void*& stream)
{
    if(!PyCallable_Check(f))
        return false;
    PyObject* index = PyLong_FromLong(d.index());
    PyObject* raw   = index ? PyObject_CallOneArg(f, index) : nullptr;
    Py_XDECREF(index);
    if(!raw)
        return false;
    stream = PyLong_AsVoidPtr(raw);
    Py_DECREF(raw);
    return !PyErr_Occurred();
}

int dtype_of(at::ScalarType s) { return s == at::kHalf ? (int)WQ_F16 : s == at::kBFloat16 ? (int)WQ_BF16 : -1; }

PyObject* raise(int status)
{
    if(PyObject* args = Py_BuildValue("(is)", status, last_error()))
    {
        PyErr_SetObject(error_type, args);
        Py_DECREF(args);
    }
    return nullptr;
}

// quantized(op, x, x2 | None, weight | None, activation, eps, group_k, stream of a device) -> (q, scale, residual_out | None), or None
PyObject* quantized(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if(n != 8 || !quantize)
        return PyErr_Format(PyExc_TypeError, "quantized takes 8 arguments, after bind()");
    HANDLE_TH_ERRORS // (what torch throws here, out of memory first of all, arrives as the exception that its own functions raise)
    {
        wqgemm_quant d{};
        d.op         = (int32_t)PyLong_AsLong(a[0]);
        d.activation = (int32_t)PyLong_AsLong(a[4]);
        const double eps = PyFloat_AsDouble(a[5]);
        const long group = PyLong_AsLong(a[6]);
        void* stream     = nullptr;
        if(PyErr_Occurred())
        {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        const at::Tensor* x = plain(a[1], nullptr);
        if(intercepted() || !x || x->dim() < 1 || (group != 128 && group != 0) || !(eps >= 0) || !current_device_is(x->device()))
            Py_RETURN_NONE;
        const c10::Device dev = x->device();
        const int64_t K       = x->size(-1);
        int64_t rows, ld;
        d.dtype = dtype_of(x->scalar_type());
        if(d.dtype < 0 || K < 1 || K > INT32_MAX || !as_rows(*x, K, rows, ld))
            Py_RETURN_NONE;
        d.M = (int32_t)rows, d.K = (int32_t)K, d.group_k = (int32_t)group, d.ldx = (int32_t)ld, d.x = x->data_ptr(), d.eps = (float)eps;
        if(a[2] != Py_None)
        {
            const at::Tensor* x2 = plain(a[2], &dev);
            if(!x2 || x2->scalar_type() != x->scalar_type() || x2->sizes() != x->sizes() || !as_rows(*x2, K, rows, ld))
                Py_RETURN_NONE;
            d.x2 = x2->data_ptr(), d.ldx2 = (int32_t)ld;
        }
        if(a[3] != Py_None)
        {
            const at::Tensor* w = plain(a[3], &dev);
            if(!w || w->dim() != 1 || w->size(0) != K || !w->is_contiguous() || (w->scalar_type() != x->scalar_type() && w->scalar_type() != at::kFloat))
                Py_RETURN_NONE;
            d.weight = w->data_ptr(), d.weight_dtype = w->scalar_type() == at::kFloat ? (int)WQ_F32 : d.dtype;
        }
        if(!current_stream(a[7], dev, stream))
            return PyErr_Occurred() ? nullptr : (Py_INCREF(Py_None), Py_None);
        const int64_t groups = group ? (K + 127) / 128 : 1;
        c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
        at::Tensor q, scale, out;
        int rc;
        {
            const WithoutGil section;
            q = at::empty(shape, x->options().dtype(at::kFloat8_e4m3fn));
            if(d.op == WQ_QUANT_RMSNORM && d.x2)
                out = at::empty(shape, x->options()), d.residual_out = out.data_ptr(), d.ld_residual_out = (int32_t)K;
            shape.back() = groups;
            scale        = at::empty(shape, x->options().dtype(at::kFloat));
            d.q = q.data_ptr(), d.scale = scale.data_ptr<float>(), d.ldq = (int32_t)K, d.ld_scale = (int32_t)groups;
            rc = quantize(&d, stream);
        }
        if(rc != WQ_OK)
            return raise(rc);
        PyObject* r = PyTuple_New(3);
        if(!r)
            return nullptr;
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(q)));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scale)));
        PyTuple_SET_ITEM(r, 2, out.defined() ? THPVariable_Wrap(std::move(out)) : (Py_INCREF(Py_None), Py_None));
        return r;
    }
    END_HANDLE_TH_ERRORS
}

// linear(x, x_scale, weight, weight_scale, bias | None, epilogue, out_dtype, stream of a device) -> y, or None
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if(n != 8 || !launch)
        return PyErr_Format(PyExc_TypeError, "linear takes 8 arguments, after bind()");
    HANDLE_TH_ERRORS
    {
        const at::Tensor* x = plain(a[0], nullptr);
        if(intercepted() || !x || x->dim() < 1 || x->scalar_type() != at::kFloat8_e4m3fn || !current_device_is(x->device()) || !THPDtype_Check(a[6]))
            Py_RETURN_NONE;
        const c10::Device dev         = x->device();
        const at::Tensor *xs = plain(a[1], &dev), *w = plain(a[2], &dev), *ws = plain(a[3], &dev);
        const at::ScalarType out_type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
        const long epilogue           = PyLong_AsLong(a[5]);
        void* stream                  = nullptr;
        if(PyErr_Occurred())
        {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        const bool with_bias = epilogue == WQ_EPI_ADD || epilogue == WQ_EPI_ADD_FASTGELU;
        if(!xs || !w || !ws || dtype_of(out_type) < 0 || (a[4] == Py_None) == with_bias || w->dim() != 2 || w->scalar_type() != at::kFloat8_e4m3fn ||
           xs->scalar_type() != at::kFloat || ws->scalar_type() != at::kFloat || ws->dim() != 2 || xs->dim() != x->dim())
            Py_RETURN_NONE;
        const int64_t N = w->size(0), K = w->size(1), kb = (K + 127) / 128;
        if(N < 1 || K < 1 || N > INT32_MAX || K > INT32_MAX || x->size(-1) != K || xs->size(-1) != kb || ws->size(0) != (N + 127) / 128 ||
           ws->size(1) != kb || xs->sizes().slice(0, xs->dim() - 1) != x->sizes().slice(0, x->dim() - 1))
            Py_RETURN_NONE;
        wqgemm_problem p{};
        int64_t rows, ld, ignored;
        if(!as_rows(*x, K, rows, ld))
            Py_RETURN_NONE;
        p.M = (int32_t)rows, p.N = (int32_t)N, p.K = (int32_t)K, p.lda = (int32_t)ld, p.a = x->data_ptr();
        if(!as_rows(*w, K, ignored, ld))
            Py_RETURN_NONE;
        p.ldb = (int32_t)ld, p.b = w->data_ptr();
        if(!as_rows(*xs, kb, ignored, ld))
            Py_RETURN_NONE;
        p.ld_a_scale = (int32_t)ld, p.a_block_scale = xs->data_ptr();
        if(!as_rows(*ws, kb, ignored, ld))
            Py_RETURN_NONE;
        p.ld_b_scale = (int32_t)ld, p.b_block_scale = ws->data_ptr();
        if(with_bias)
        {
            const at::Tensor* bias = plain(a[4], &dev);
            if(!bias || bias->dim() != 1 || bias->size(0) != N || bias->scalar_type() != out_type || !bias->is_contiguous())
                Py_RETURN_NONE;
            p.d0 = bias->data_ptr();
        }
        if(!current_stream(a[7], dev, stream))
            return PyErr_Occurred() ? nullptr : (Py_INCREF(Py_None), Py_None);
        c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
        shape.back()   = N;
        p.a_dtype = p.b_dtype = p.scale_dtype = WQ_F8_E4M3FN;
        p.c_dtype  = dtype_of(out_type);
        p.a_layout = p.c_layout = WQ_ROW_MAJOR, p.b_layout = WQ_COL_MAJOR;
        p.ldc = (int32_t)N, p.epilogue = (int32_t)epilogue, p.k_batch = 1, p.flags = WQ_FLAG_BF16_RTN;
        p.scale_block_m = 1, p.scale_block_n = p.scale_block_k = 128;
        at::Tensor y;
        int rc;
        {
            const WithoutGil section;
            y   = at::empty(shape, x->options().dtype(out_type));
            p.c = y.data_ptr();
            at::Tensor scratch;
            if(const size_t bytes = workspace_bytes(&p))
                scratch = at::empty({(int64_t)bytes}, x->options().dtype(at::kByte));
            rc = launch(&p, scratch.defined() ? scratch.data_ptr() : nullptr, stream);
        }
        if(rc != WQ_OK)
            return raise(rc);
        return THPVariable_Wrap(std::move(y));
    }
    END_HANDLE_TH_ERRORS
}

// direct(tensor | None, ...) -> whether a call with these tensors goes to the device as it stands: nothing intercepts it, none is a subclass
PyObject* direct(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    bool yes = !intercepted();
    for(Py_ssize_t i = 0; i < n; ++i)
        yes = yes && (a[i] == Py_None || THPVariable_CheckExact(a[i]));
    return PyBool_FromLong(yes);
}

// bind(quantize, launch, workspace_bytes, last_error, error type): addresses of the library's functions
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if(n != 5)
        return PyErr_Format(PyExc_TypeError, "bind takes 5 arguments");
    void* f[4];
    for(int i = 0; i < 4; ++i)
        if(!(f[i] = PyLong_AsVoidPtr(a[i])))
            return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "null address");
    quantize        = (int (*)(const wqgemm_quant*, void*))f[0];
    launch          = (int (*)(const wqgemm_problem*, void*, void*))f[1];
    workspace_bytes = (size_t (*)(const wqgemm_problem*))f[2];
    last_error      = (const char* (*)())f[3];
    Py_INCREF(a[4]);
    Py_XSETREF(error_type, a[4]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"quantized", (PyCFunction)(void (*)(void))quantized, METH_FASTCALL, nullptr},
                         {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
                         {"direct", (PyCFunction)(void (*)(void))direct, METH_FASTCALL, nullptr},
                         {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__torch_front(void) { return PyModule_Create(&module); }
