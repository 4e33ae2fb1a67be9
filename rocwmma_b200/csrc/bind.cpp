// Python binding of the entry points that a decoding step calls once per layer or more: 4-bit
// block-scaled operands and embedding.  Checks the tensors, allocates what the caller does not
// give, and calls the C ABI on the tensors' device and stream.  The same in Python over ctypes took
// 9 to 12 us a call, about three times what the launch itself takes and more than the kernels
// do on small inputs.
//
// The functions are called by rocwmma_b200/api.py, which documents them; arguments are
// positional, None stands for a default.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "rocwmma_b200.h"
#include "row_overlap.h"

namespace
{
    struct Refused // a ValueError
    {
        std::string what;
    };
    struct PythonError // one that Python has set already
    {
    };
    struct Status // one of the library's codes
    {
        int         code;
        const char* where;
    };
    [[noreturn]] void refuse(std::string what)
    {
        throw Refused{std::move(what)};
    }

    // ---- arguments -----------------------------------------------------------------------------
    int64_t integer(PyObject* o)
    {
        const long long v = PyLong_AsLongLong(o);
        if(v == -1 && PyErr_Occurred())
            throw PythonError{};
        return v;
    }
    uint32_t size32(PyObject* o, const char* what)
    {
        const int64_t v = integer(o);
        if(v < 0 || v > 0xffffffffll)
            refuse(std::string(what) + ": " + std::to_string(v) + " is no 32-bit size");
        return uint32_t(v);
    }
    int code(PyObject* o)
    {
        const int64_t v = integer(o);
        return v < 0 || v > 1000 ? 1000 : int(v); // no such type, layout or format
    }
    // A leading dimension; None or 0: the natural one.
    uint64_t stride(PyObject* o, uint64_t natural, const char* what)
    {
        if(o == Py_None)
            return natural;
        const int64_t v = integer(o);
        if(v < 0)
            refuse(std::string(what) + " is negative");
        return v == 0 ? natural : uint64_t(v);
    }
    double number(PyObject* o)
    {
        const double v = PyFloat_AsDouble(o);
        if(v == -1.0 && PyErr_Occurred())
            throw PythonError{};
        return v;
    }
    bool truth(PyObject* o)
    {
        const int v = PyObject_IsTrue(o);
        if(v < 0)
            throw PythonError{};
        return v != 0;
    }
    const at::Tensor& tensor(PyObject* o, const char* what)
    {
        if(!THPVariable_Check(o))
            refuse(std::string(what) + " must be a tensor");
        return THPVariable_Unpack(o);
    }
    const at::Tensor* tensorOrNone(PyObject* o, const char* what)
    {
        return o == Py_None ? nullptr : &tensor(o, what);
    }

    // The one device that all given tensors are on.
    c10::Device deviceOf(std::initializer_list<const at::Tensor*> tensors)
    {
        const at::Tensor* first = nullptr;
        for(const at::Tensor* t : tensors)
        {
            if(!t)
                continue;
            if(!t->is_cuda())
                refuse("device tensors required (this library has no CPU path)");
            if(first && t->device() != first->device())
                refuse("tensors on several devices");
            first = first ? first : t;
        }
        return first->device();
    }

    // Makes the tensors' device and the stream (None: that device's current one) current, so that
    // new tensors may be used on the stream at once.
    struct Place
    {
        c10::cuda::CUDAGuard                      device;
        std::optional<c10::cuda::CUDAStreamGuard> guard;
        void*                                     stream;
        Place(c10::Device d, PyObject* handle) : device(d)
        {
            if(handle == Py_None)
                stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
            else
            {
                stream = PyLong_AsVoidPtr(handle);
                if(!stream && PyErr_Occurred())
                    throw PythonError{};
                guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), d.index()));
            }
        }
    };

    std::optional<at::ScalarType> valueType(int code)
    {
        switch(code)
        {
        case B200WMMA_F16:
            return at::kHalf;
        case B200WMMA_BF16:
            return at::kBFloat16;
        case B200WMMA_F32:
            return at::kFloat;
        }
        return std::nullopt;
    }
    int valueCode(const at::Tensor& t, const char* what)
    {
        switch(t.scalar_type())
        {
        case at::kHalf:
            return B200WMMA_F16;
        case at::kBFloat16:
            return B200WMMA_BF16;
        case at::kFloat:
            return B200WMMA_F32;
        default:
            refuse(std::string(what) + ": float16, bfloat16 or float32 expected");
        }
    }
    // A contiguous tensor of the type that holds what a call reads or writes of it.
    void holds(const at::Tensor& t, const char* what, at::ScalarType type, unsigned __int128 count)
    {
        if(t.scalar_type() != type)
            refuse(std::string(what) + ": " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(type));
        if(!t.is_contiguous())
            refuse(std::string(what) + ": must be contiguous");
        if(count > (unsigned __int128)(t.numel()))
            refuse(std::string(what) + ": " + std::to_string(t.numel()) + " elements are too few");
    }
    // Elements of `rows` rows of `length`, `ld` apart.
    unsigned __int128 extent(uint64_t rows, uint64_t length, uint64_t ld)
    {
        return rows ? (unsigned __int128)(rows - 1u) * ld + length : 0u;
    }
    at::Tensor empty(std::initializer_list<int64_t> shape, at::ScalarType type, c10::Device device)
    {
        return at::empty(at::IntArrayRef(shape), at::TensorOptions().dtype(type).device(device));
    }
    void finish(int status, const char* where)
    {
        if(status != B200WMMA_OK)
            throw Status{status, where};
    }
    PyObject* wrap(at::Tensor t)
    {
        return THPVariable_Wrap(std::move(t));
    }

    // ---- 4-bit block-scaled operands -----------------------------------------------------------
    void operandHolds(int fmt, uint32_t rows, uint32_t k, const at::Tensor& codes, const at::Tensor& scales, uint64_t ld)
    {
        holds(codes, "codes", at::kByte, extent(rows, b200wmma_mx_pitch(k), ld));
        holds(scales, "scales", at::kByte, b200wmma_mx_scale_bytes(fmt, rows, k));
    }

    // fmt, in_t, rows, k, x, layout, exponent, ldx, ldq, codes, scales, stream
    PyObject* quantize(PyObject* const* a)
    {
        const int         fmt = code(a[0]), type = code(a[1]), layout = code(a[5]);
        const uint32_t    rows = size32(a[2], "rows"), k = size32(a[3], "k");
        const at::Tensor& x   = tensor(a[4], "x");
        const bool        columns = layout == B200WMMA_COL_MAJOR;
        const int64_t     exponent = integer(a[6]);
        const uint64_t    ldx = stride(a[7], columns ? rows : k, "ldx"), ldq = stride(a[8], b200wmma_mx_pitch(k), "ldq");
        const at::Tensor *codesIn = tensorOrNone(a[9], "codes"), *scalesIn = tensorOrNone(a[10], "scales");
        const c10::Device device = deviceOf({&x, codesIn, scalesIn});
        const auto        want   = valueType(type);
        if(!want)
            finish(B200WMMA_ERR_UNSUPPORTED, "b200wmma_mx_quantize");
        holds(x, "x", *want, columns ? extent(k, rows, ldx) : extent(rows, k, ldx));
        Place      place(device, a[11]);
        at::Tensor codes  = codesIn ? *codesIn : empty({int64_t(rows * ldq)}, at::kByte, device);
        at::Tensor scales = scalesIn ? *scalesIn : empty({int64_t(b200wmma_mx_scale_bytes(fmt, rows, k))}, at::kByte, device);
        operandHolds(fmt, rows, k, codes, scales, ldq);
        finish(b200wmma_mx_quantize(fmt, type, rows, k, x.data_ptr(), ldx, layout,
                                    exponent < -1000 || exponent > 1000 ? 1000 : int(exponent), codes.data_ptr(), ldq,
                                    scales.data_ptr(), place.stream),
               "b200wmma_mx_quantize");
        PyObject* c = wrap(std::move(codes));
        PyObject* s = wrap(std::move(scales));
        PyObject* t = c && s ? PyTuple_Pack(2, c, s) : nullptr;
        Py_XDECREF(c);
        Py_XDECREF(s);
        return t;
    }

    // fmt, out_t, rows, k, codes, scales, exponent, ldq, ldo, out, stream
    PyObject* dequantize(PyObject* const* a)
    {
        const int         fmt = code(a[0]), type = code(a[1]);
        const uint32_t    rows = size32(a[2], "rows"), k = size32(a[3], "k");
        const at::Tensor &codes = tensor(a[4], "codes"), &scales = tensor(a[5], "scales");
        const int64_t     exponent = integer(a[6]);
        const uint64_t    ldq = stride(a[7], b200wmma_mx_pitch(k), "ldq"), ldo = stride(a[8], k, "ldo");
        const at::Tensor* outIn  = tensorOrNone(a[9], "out");
        const c10::Device device = deviceOf({&codes, &scales, outIn});
        const auto        want   = valueType(type);
        if(!want)
            finish(B200WMMA_ERR_UNSUPPORTED, "b200wmma_mx_dequantize");
        operandHolds(fmt, rows, k, codes, scales, ldq);
        Place      place(device, a[10]);
        at::Tensor out = outIn ? *outIn : empty({int64_t(rows * ldo)}, *want, device);
        holds(out, "out", *want, extent(rows, k, ldo));
        finish(b200wmma_mx_dequantize(fmt, type, rows, k, codes.data_ptr(), ldq, scales.data_ptr(),
                                      exponent < -1000 || exponent > 1000 ? 1000 : int(exponent), out.data_ptr(), ldo,
                                      place.stream),
               "b200wmma_mx_dequantize");
        return wrap(std::move(out));
    }

    // fmt, out_t, m, n, k, A codes, A scales, B codes, B scales, c, alpha, beta, lda, ldb, ldc, ldd, out, stream
    PyObject* gemm(PyObject* const* a)
    {
        const int         fmt = code(a[0]), type = code(a[1]);
        const uint32_t    m = size32(a[2], "m"), n = size32(a[3], "n"), k = size32(a[4], "k");
        const at::Tensor &ac = tensor(a[5], "codes of A"), &as = tensor(a[6], "scales of A");
        const at::Tensor &bc = tensor(a[7], "codes of B"), &bs = tensor(a[8], "scales of B");
        const double      alpha = number(a[10]), beta = number(a[11]);
        const at::Tensor *c = beta != 0.0 ? tensorOrNone(a[9], "c") : nullptr, *outIn = tensorOrNone(a[16], "out");
        const uint64_t    pitch = b200wmma_mx_pitch(k);
        const uint64_t    lda = stride(a[12], pitch, "lda"), ldb = stride(a[13], pitch, "ldb");
        const uint64_t    ldc = stride(a[14], n, "ldc"), ldd = stride(a[15], n, "ldd");
        if(ldc > 0xffffffffull || ldd > 0xffffffffull)
            refuse("ldc and ldd are 32-bit sizes");
        const c10::Device device = deviceOf({&ac, &as, &bc, &bs, c, outIn});
        const auto        want   = valueType(type);
        if(!want)
            finish(B200WMMA_ERR_UNSUPPORTED, "b200wmma_mx_gemm");
        operandHolds(fmt, m, k, ac, as, lda);
        operandHolds(fmt, n, k, bc, bs, ldb);
        if(c)
            holds(*c, "c", *want, extent(m, n, ldc));
        Place      place(device, a[17]);
        at::Tensor d = outIn ? *outIn : empty({int64_t(m * ldd)}, *want, device);
        holds(d, "out", *want, extent(m, n, ldd));
        finish(b200wmma_mx_gemm(fmt, type, m, n, k, ac.data_ptr(), as.data_ptr(), bc.data_ptr(), bs.data_ptr(),
                                c ? c->data_ptr() : nullptr, d.data_ptr(), lda, ldb, uint32_t(ldc), uint32_t(ldd), alpha,
                                beta, place.stream),
               "b200wmma_mx_gemm");
        return wrap(std::move(d));
    }

    // ---- embedding -----------------------------------------------------------------------------
    // ids as outer x inner tokens.
    struct Tokens
    {
        int64_t        outer, inner, idsOuter, idsInner;
        int            bytes;
        const int64_t* first;
    };
    Tokens tokensOf(const at::Tensor& ids, const at::Tensor* first)
    {
        Tokens t{};
        if(ids.scalar_type() == at::kLong)
            t.bytes = 8;
        else if(ids.scalar_type() == at::kInt)
            t.bytes = 4;
        else
            refuse("ids must be int32 or int64");
        if(first
           && (ids.dim() != 2 || first->scalar_type() != at::kLong || !first->is_contiguous() || first->dim() != 1
               || first->size(0) != ids.size(1) + 1))
            refuse("with first, ids are [outer, inner] and first inner + 1 int64 row numbers");
        t.first = first ? first->data_ptr<int64_t>() : nullptr;
        if(ids.dim() == 2)
        {
            t.outer    = ids.size(0);
            t.inner    = ids.size(1);
            t.idsOuter = ids.stride(0);
            t.idsInner = ids.stride(1);
        }
        else if(ids.dim() == 1)
        {
            t.outer    = ids.size(0);
            t.inner    = 1;
            t.idsOuter = ids.stride(0);
        }
        else
        {
            if(!ids.is_contiguous())
                refuse("ids of this shape must be contiguous");
            t.outer    = ids.numel();
            t.inner    = 1;
            t.idsOuter = 1;
        }
        return t;
    }
    // Distances of the rows of t [*ids.shape, dim] along outer and inner.
    void rowsOf(const at::Tensor& t, const at::Tensor& ids, int64_t dim, const char* what, int64_t& outer, int64_t& inner)
    {
        bool ok = t.dim() == ids.dim() + 1 && t.size(-1) == dim;
        for(int64_t i = 0; ok && i < ids.dim(); ++i)
            ok = t.size(i) == ids.size(i);
        if(!ok)
            refuse(std::string(what) + " must have the shape of ids and a row of " + std::to_string(dim) + " behind it");
        if(dim > 1 && t.stride(-1) != 1)
            refuse(std::string("the rows of ") + what + " must be contiguous");
        outer = dim;
        inner = 0;
        if(ids.dim() == 1 || ids.dim() == 2)
        {
            outer = t.stride(0);
            inner = ids.dim() == 2 ? t.stride(1) : 0;
        }
        else if(!t.is_contiguous())
            refuse(std::string(what) + " must be contiguous for ids of this shape");
    }
    void isTable(const at::Tensor& t, const char* what)
    {
        if(t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1))
            refuse(std::string(what) + " must be [rows, dim] with contiguous rows");
    }
    uint32_t width(int64_t dim)
    {
        return dim > 0xffffffffll ? 0xffffffffu : uint32_t(dim);
    }

    // table, ids, scale, first, out_t, out, stream
    PyObject* embedding(PyObject* const* a)
    {
        const at::Tensor &table = tensor(a[0], "table"), &ids = tensor(a[1], "ids");
        const double      scale = number(a[2]);
        const at::Tensor *first = tensorOrNone(a[3], "first"), *outIn = tensorOrNone(a[5], "out");
        isTable(table, "table");
        const c10::Device device = deviceOf({&table, &ids, first, outIn});
        const Tokens      t      = tokensOf(ids, first);
        const int64_t     rows = table.size(0), dim = table.size(1);
        const int         tableCode = valueCode(table, "table");
        const int         outCode   = a[4] == Py_None ? tableCode : code(a[4]);
        const auto        want      = valueType(outCode);
        if(!outIn && !want)
            finish(B200WMMA_ERR_UNSUPPORTED, "b200wmma_embedding");
        Place      place(device, a[6]);
        at::Tensor out;
        if(outIn)
            out = *outIn;
        else
        {
            c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
            shape.push_back(dim);
            out = at::empty(shape, at::TensorOptions().dtype(*want).device(device));
        }
        int64_t outOuter, outInner;
        rowsOf(out, ids, dim, "out", outOuter, outInner);
        if(b200wmma::rowsOverlap(uint64_t(t.outer), uint64_t(outOuter), uint64_t(t.inner), uint64_t(outInner), uint64_t(dim)))
            refuse("the rows of out must not overlap");
        const int outType = valueCode(out, "out");
        if(t.outer && t.inner)
            finish(b200wmma_embedding(tableCode, outType, uint64_t(rows), width(dim), uint64_t(t.outer), width(t.inner),
                                      table.data_ptr(), uint64_t(rows > 1 ? table.stride(0) : dim), ids.data_ptr(), t.bytes,
                                      uint64_t(t.idsOuter), uint64_t(t.idsInner), t.first, out.data_ptr(), uint64_t(outOuter),
                                      uint64_t(outInner), scale, place.stream),
                   "b200wmma_embedding");
        return wrap(std::move(out));
    }

    // grad, ids, rows, out_t, scale, first, out, accumulate, workspace, stream
    PyObject* embeddingGrad(PyObject* const* a)
    {
        const at::Tensor &grad = tensor(a[0], "grad"), &ids = tensor(a[1], "ids");
        const int64_t     rows  = integer(a[2]);
        const double      scale = number(a[4]);
        const at::Tensor *first = tensorOrNone(a[5], "first"), *outIn = tensorOrNone(a[6], "out");
        const bool        accumulate = truth(a[7]);
        const at::Tensor* workIn     = tensorOrNone(a[8], "workspace");
        if(accumulate && !outIn)
            refuse("accumulate needs out");
        if(rows < 0 || grad.dim() == 0)
            refuse("grad must be [*ids.shape, dim], rows a size");
        const c10::Device device = deviceOf({&grad, &ids, first, outIn, workIn});
        const Tokens      t      = tokensOf(ids, first);
        const int64_t     dim    = grad.size(-1);
        int64_t           gradOuter, gradInner;
        rowsOf(grad, ids, dim, "grad", gradOuter, gradInner);
        const int  gradCode = valueCode(grad, "grad");
        const auto want     = valueType(a[3] == Py_None ? gradCode : code(a[3]));
        if(!outIn && !want)
            finish(B200WMMA_ERR_UNSUPPORTED, "b200wmma_embedding_grad");
        Place      place(device, a[9]);
        at::Tensor out = outIn ? *outIn : empty({rows, dim}, *want, device);
        isTable(out, "out");
        if(out.size(0) != rows || out.size(1) != dim)
            refuse("out must be [rows, dim]");
        if(rows > 1 && out.stride(0) < dim)
            refuse("out must not hold a row twice");
        const int outCode = valueCode(out, "out");
        if(t.outer && t.inner)
        {
            const uint64_t need = b200wmma_embedding_grad_workspace(uint64_t(rows), width(dim), uint64_t(t.outer), width(t.inner));
            if(workIn && (workIn->scalar_type() != at::kByte || !workIn->is_contiguous()))
                refuse("workspace must be a contiguous uint8 tensor");
            const at::Tensor work = workIn ? *workIn : empty({int64_t(need)}, at::kByte, device);
            finish(b200wmma_embedding_grad(gradCode, outCode, uint64_t(rows), width(dim), uint64_t(t.outer), width(t.inner),
                                           grad.data_ptr(), uint64_t(gradOuter), uint64_t(gradInner), ids.data_ptr(), t.bytes,
                                           uint64_t(t.idsOuter), uint64_t(t.idsInner), t.first, out.data_ptr(),
                                           uint64_t(rows > 1 ? out.stride(0) : dim), scale, accumulate, work.data_ptr(),
                                           uint64_t(work.numel()), place.stream),
                   "b200wmma_embedding_grad");
        }
        else if(!accumulate)
            out.zero_();
        return wrap(std::move(out));
    }

    // ---- module --------------------------------------------------------------------------------
    PyObject* raise = nullptr; // rocwmma_b200._lib.check(status, where)

    template <PyObject* (*F)(PyObject* const*), Py_ssize_t COUNT>
    PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t count)
    {
        if(count != COUNT)
        {
            PyErr_Format(PyExc_TypeError, "%zd arguments expected", COUNT);
            return nullptr;
        }
        try
        {
            return F(args);
        }
        catch(PythonError const&)
        {
        }
        catch(Refused const& r)
        {
            PyErr_SetString(PyExc_ValueError, r.what.c_str());
        }
        catch(Status const& s)
        {
            PyObject* r = PyObject_CallFunction(raise, "is", s.code, s.where);
            if(r) // it raises
                PyErr_SetString(PyExc_RuntimeError, s.where);
            Py_XDECREF(r);
        }
        catch(...) // torch's own, such as no memory left
        {
            torch::translate_exception_to_python(std::current_exception());
        }
        return nullptr;
    }
    template <PyObject* (*F)(PyObject* const*), Py_ssize_t COUNT>
    PyMethodDef method(const char* name)
    {
        return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<F, COUNT>)), METH_FASTCALL, nullptr};
    }
    PyMethodDef methods[] = {method<quantize, 12>("mx_quantize"),
                             method<dequantize, 11>("mx_dequantize"),
                             method<gemm, 18>("mx_gemm"),
                             method<embedding, 7>("embedding"),
                             method<embeddingGrad, 10>("embedding_grad"),
                             {nullptr, nullptr, 0, nullptr}};
    PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
} // namespace

PyMODINIT_FUNC PyInit__bind()
{
    PyObject* lib = PyImport_ImportModule("rocwmma_b200._lib");
    if(!lib)
        return nullptr;
    raise = PyObject_GetAttrString(lib, "check");
    Py_DECREF(lib);
    return raise ? PyModule_Create(&module) : nullptr;
}
