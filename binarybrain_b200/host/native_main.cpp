// CPython module `binarybrain_b200._native`: the bbcu_* operators of libbbcu_b200.so as functions on torch tensors.
//
// The operators take about 2 us of host time per kernel; called through ctypes with the current stream looked up in Python they took
// 6-9 us more, which is what bounded small networks (the training step of a 1024-420-70 MLP: 134 us of kernels in 390 us).
// Here a call parses its arguments straight into the C signature: tensors give their data pointer, None is a null pointer, numbers
// pass as they are, and a trailing stream argument that is left out is torch's current stream.  A status other than 0 raises
// binarybrain_b200.abi.BbcuError.  The functions are looked up in the library that binarybrain_b200.abi has loaded.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <exception>
#include <tuple>
#include <type_traits>
#include <utility>

#include "bbcu_b200.h"

namespace {

void *g_library = nullptr;

// the library handle of binarybrain_b200.abi (loads it on first use); false with a Python error set
bool bind_library()
{
    if (g_library) return true;
    PyObject *abi = PyImport_ImportModule("binarybrain_b200.abi");
    if (!abi) return false;
    PyObject *lib = PyObject_CallMethod(abi, "lib", nullptr);
    Py_DECREF(abi);
    if (!lib) return false;
    PyObject *handle = PyObject_GetAttrString(lib, "_handle");
    Py_DECREF(lib);
    if (!handle) return false;
    g_library = PyLong_AsVoidPtr(handle);
    Py_DECREF(handle);
    return g_library != nullptr;
}

PyObject *raise_status(const char *name, int status)
{
    using Text = const char *(*)(int);
    Text text = reinterpret_cast<Text>(dlsym(g_library, "bbcu_b200_error_string"));
    PyObject *abi = PyImport_ImportModule("binarybrain_b200.abi");
    if (!abi) return nullptr;
    PyObject *cls = PyObject_GetAttrString(abi, "BbcuError");
    Py_DECREF(abi);
    if (!cls) return nullptr;
    PyObject *e = PyObject_CallFunction(cls, "sis", name, status, text ? text(status) : "");
    if (e) { PyErr_SetObject(cls, e); Py_DECREF(e); }
    Py_DECREF(cls);
    return nullptr;
}

// one argument of type T; false with a Python error set when the object does not fit
template <class T> bool parse(PyObject *o, T &v)
{
    if constexpr (std::is_pointer_v<T>) {
        if (o == Py_None) { v = nullptr; return true; }
        if (THPVariable_Check(o)) {
            // an operator that may write through the pointer needs the tensor's own memory: mutable_data_ptr() gives a lazily cloned
            // tensor its copy, where const_data_ptr() would have the operator write into the tensor it was cloned from
            const at::Tensor &t = THPVariable_Unpack(o);
            try {
                if constexpr (std::is_const_v<std::remove_pointer_t<T>>) v = static_cast<T>(t.const_data_ptr());
                else v = static_cast<T>(t.mutable_data_ptr());
            } catch (const std::exception &e) {
                PyErr_SetString(PyExc_RuntimeError, e.what());
                return false;
            }
            return true;
        }
        v = reinterpret_cast<T>(PyLong_AsVoidPtr(o));
    } else if constexpr (std::is_floating_point_v<T>) {
        v = static_cast<T>(PyFloat_AsDouble(o));
    } else {
        const long long n = PyLong_AsLongLong(o);
        if (n == -1 && PyErr_Occurred()) return false;
        v = static_cast<T>(n);
        if (static_cast<long long>(v) != n) { PyErr_Format(PyExc_OverflowError, "%lld does not fit the argument", n); return false; }
        return true;
    }
    return !PyErr_Occurred();
}

template <class F> struct Operator;
template <class... A> struct Operator<int(A...)> {
    using Fn = int (*)(A...);
    static constexpr Py_ssize_t kArgs = sizeof...(A);
    using Args = std::tuple<A...>;
    static constexpr bool kStream = std::is_same_v<std::tuple_element_t<kArgs - 1, Args>, bbcu_stream_t>;

    template <std::size_t... I> static bool parse_all(PyObject *const *o, Py_ssize_t n, Args &a, std::index_sequence<I...>)
    {
        return (((Py_ssize_t)I >= n || parse(o[I], std::get<I>(a))) && ...);
    }
    static PyObject *call(Fn &fn, const char *name, PyObject *const *o, Py_ssize_t n)
    {
        if (!fn) {
            if (!bind_library()) return nullptr;
            fn = reinterpret_cast<Fn>(dlsym(g_library, name));
            if (!fn) { PyErr_Format(PyExc_AttributeError, "the library lacks %s", name); return nullptr; }
        }
        if (n != kArgs && !(kStream && n == kArgs - 1)) {
            PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, kArgs - kStream, n);
            return nullptr;
        }
        Args a{};
        if (!parse_all(o, n, a, std::make_index_sequence<sizeof...(A)>())) return nullptr;
        int status = 0;
        try {
            if constexpr (kStream) {
                if (n == kArgs - 1) std::get<kArgs - 1>(a) = reinterpret_cast<bbcu_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
            }
            Py_BEGIN_ALLOW_THREADS
            status = std::apply(fn, a);
            Py_END_ALLOW_THREADS
        } catch (const std::exception &e) {
            PyErr_SetString(PyExc_RuntimeError, e.what());
            return nullptr;
        }
        if (status != 0) return raise_status(name, status);
        Py_RETURN_NONE;
    }
};

// A new uninitialised tensor on the device of `like`: empty_f32 / empty_i32(like, rows, cols), vector_f32(like, n), scalar_f64(like)
template <int DIM> PyObject *empty(at::ScalarType type, PyObject *const *o, Py_ssize_t n)
{
    constexpr Py_ssize_t want = DIM + 1;
    if (n != want || !THPVariable_Check(o[0])) { PyErr_SetString(PyExc_TypeError, "expected (tensor, size...)"); return nullptr; }
    int64_t size[2] = {0, 0};
    for (Py_ssize_t i = 1; i < n; ++i)
        if (!parse(o[i], size[i - 1])) return nullptr;
    try {
        const at::Tensor &like = THPVariable_Unpack(o[0]);
        return THPVariable_Wrap(at::empty(at::IntArrayRef(size, (size_t)DIM), at::TensorOptions().dtype(type).device(like.device())));
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject *empty_f32(PyObject *, PyObject *const *o, Py_ssize_t n)  { return empty<2>(at::kFloat, o, n); }
PyObject *empty_i32(PyObject *, PyObject *const *o, Py_ssize_t n)  { return empty<2>(at::kInt, o, n); }
PyObject *vector_f32(PyObject *, PyObject *const *o, Py_ssize_t n) { return empty<1>(at::kFloat, o, n); }
PyObject *scalar_f64(PyObject *, PyObject *const *o, Py_ssize_t n) { return empty<0>(at::kDouble, o, n); }

#define BB200_OPERATORS(X)                                                                                                                    \
    X(bbcu_fp32_StochasticLut6_Forward) X(bbcu_bit_fp32_StochasticLut6_Forward) X(bbcu_bit_bit_fp32_StochasticLut6_Forward)                   \
    X(bbcu_fp32_StochasticLut6_Backward) X(bbcu_bit_fp32_StochasticLut6_Backward) X(bbcu_fp32_DifferentiableLut6_ForwardTrainingRows)         \
    X(bbcu_bit_fp32_DifferentiableLut6_ForwardTraining) X(bbcu_fp32_DifferentiableLut6_ForwardInference)                                      \
    X(bbcu_bit_fp32_DifferentiableLut6_ForwardInference) X(bbcu_fp32_DifferentiableLut6_Backward) X(bbcu_bit_fp32_DifferentiableLut6_Backward) \
    X(bbcu_fp32_DifferentiableLut6_ForwardStats) X(bbcu_fp32_DifferentiableLut6_ForwardNormalize) X(bbcu_fp32_DifferentiableLut6_BackwardStats) \
    X(bbcu_fp32_DifferentiableLut6_BackwardStatsFromOutput) X(bbcu_fp32_DifferentiableLut6_BackwardApply)                                     \
    X(bbcu_fp32_StochasticBatchNormalization_ForwardTraining) X(bbcu_fp32_StochasticBatchNormalization_ReForward)                             \
    X(bbcu_fp32_StochasticBatchNormalization_ForwardInference) X(bbcu_fp32_StochasticBatchNormalization_Backward)                             \
    X(bbcu_bit_BinaryLut6_Forward) X(bbcu_bit_BinaryLut6_Forward_Lop3Immediate) X(bbcu_host_bit_BinaryLut6_Forward)                           \
    X(bbcu_fp32_Vector_clamp) X(bbcu_fp32_OptimizerAdam) X(bbcu_fp32_OptimizerAdamUpdate) X(bbcu_fp32_LossSoftmaxCrossEntropyMean)             \
    X(bbcu_fp32_LossMeanSquaredError)                                                                                                         \
    X(bbcu_fp32_Reduce_Forward) X(bbcu_fp32_Reduce_Backward) X(bbcu_bit_fp32_RealToBinary_Forward) X(bbcu_bit_fp32_BinaryToReal_Forward)      \
    X(bbcu_fp32_BinaryToReal_Forward) X(bbcu_fp32_BinaryToReal_Backward) X(bbcu_fp32_Im2Col_Forward) X(bbcu_bit_Im2Col_Forward)               \
    X(bbcu_fp32_Im2Col_Backward) X(bbcu_fp32_Col2Im_Forward) X(bbcu_bit_Col2Im_Forward) X(bbcu_fp32_Col2Im_Backward)                          \
    X(bbcu_fp32_MaxPooling_Forward) X(bbcu_bit_MaxPooling_Forward) X(bbcu_fp32_MaxPooling_Backward) X(bbcu_bit_fp32_MaxPooling_Backward)     \
    X(bbcu_fp32_LayerNormalization_Forward) X(bbcu_bf16_LayerNormalization_Forward) X(bbcu_fp32_LayerNormalization_Backward)                  \
    X(bbcu_bf16_LayerNormalization_Backward) X(bbcu_fp32_QuantizeInt8_Frames) X(bbcu_bf16_QuantizeInt8_Frames)                                \
    X(bbcu_fp32_QuantizeInt8_Channels) X(bbcu_int8_fp32_DenseAffine_Forward) X(bbcu_int8_bf16_DenseAffine_Forward)                            \
    X(bbcu_fp32_LossDistillation) X(bbcu_bf16_LossDistillation)

#define BB200_DEFINE(name)                                                          \
    PyObject *py_##name(PyObject *, PyObject *const *o, Py_ssize_t n)               \
    {                                                                               \
        static Operator<decltype(name)>::Fn fn = nullptr;                           \
        return Operator<decltype(name)>::call(fn, #name, o, n);                     \
    }
BB200_OPERATORS(BB200_DEFINE)
#undef BB200_DEFINE

// ---- a layer's training step on fp32 frames: the tensors that are not given are made here and the sizes are read off the tensors, which in Python took
// 1.5 us a call (the optimizer step of a small MLP is some 65 us of host time)

template <class F> F *bound(F *&fn, const char *name)
{
    if (fn || !bind_library()) return fn;
    fn = reinterpret_cast<F *>(dlsym(g_library, name));
    if (!fn) PyErr_Format(PyExc_AttributeError, "the library lacks %s", name);
    return fn;
}

// the tensor in `o`, which has to have `dims` dimensions at least; null with a Python error set
const at::Tensor *tensor_of(PyObject *o, int64_t dims, const char *name)
{
    if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "%s: expected a tensor", name); return nullptr; }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.dim() < dims) { PyErr_Format(PyExc_IndexError, "%s: expected %d dimensions", name, (int)dims); return nullptr; }
    return &t;
}

// a flag, or any number that int() takes
bool parse_flag(PyObject *o, int &v)
{
    if (PyLong_Check(o)) return parse(o, v);
    PyObject *n = PyNumber_Long(o);
    if (!n) return false;
    const bool ok = parse(n, v);
    Py_DECREF(n);
    return ok;
}

// an fp32 output: memory of the given tensor, the given address, or, for None, a new tensor beside `like`; false with a Python error set
struct Output {
    PyObject *given;
    at::Tensor made;
    float *data = nullptr;

    bool take(PyObject *o, const at::Tensor &like, at::IntArrayRef size)
    {
        given = o;
        if (o != Py_None) return parse(o, data);
        made = at::empty(size, at::TensorOptions().dtype(at::kFloat).device(like.device()));
        data = static_cast<float *>(made.mutable_data_ptr());
        return true;
    }
    PyObject *result() const { return given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(made); }
};

// train_forward(x, y, idx, W, mean, rstd, running_mean, running_var, gamma, beta, momentum, bias, frames, lut_binarize, binary) -> (y, mean, rstd)
PyObject *train_forward(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    static decltype(&bbcu_fp32_DifferentiableLut6_ForwardTrainingRows) fn = nullptr;
    if (n != 15) { PyErr_SetString(PyExc_TypeError, "train_forward takes 15 arguments"); return nullptr; }
    float gamma, beta, momentum, bias, *running_mean, *running_var;
    const float *x, *W;
    const int *index;
    int frames, lut_binarize, binary;
    try {
        const at::Tensor *xt = tensor_of(o[0], 2, "x"), *idx = xt ? tensor_of(o[2], 1, "idx") : nullptr;
        if (!idx || !parse(o[0], x) || !parse(o[2], index) || !parse(o[3], W) || !parse(o[6], running_mean) || !parse(o[7], running_var) ||
            !parse(o[8], gamma) || !parse(o[9], beta) || !parse(o[10], momentum) || !parse(o[11], bias) || !parse(o[12], frames) ||
            !parse_flag(o[13], lut_binarize) || !parse_flag(o[14], binary) || !bound(fn, "bbcu_fp32_DifferentiableLut6_ForwardTrainingRows")) return nullptr;
        const int64_t rows = xt->size(0), stride = xt->size(1), nodes = idx->size(0);
        if (rows > INT_MAX || stride > INT_MAX || nodes > INT_MAX) { PyErr_SetString(PyExc_OverflowError, "a size does not fit the operator"); return nullptr; }
        Output y, mean, rstd;
        if (!y.take(o[1], *xt, {nodes, stride}) || !mean.take(o[4], *xt, {nodes}) || !rstd.take(o[5], *xt, {nodes})) return nullptr;
        const auto stream = reinterpret_cast<bbcu_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
        int status = 0;
        Py_BEGIN_ALLOW_THREADS
        status = fn(x, y.data, index, W, mean.data, rstd.data, running_mean, running_var, gamma, beta, momentum, bias, (int)rows, (int)nodes, frames, (int)stride,
                    lut_binarize, binary, stream);
        Py_END_ALLOW_THREADS
        if (status != 0) return raise_status("bbcu_fp32_DifferentiableLut6_ForwardTrainingRows", status);
        PyObject *r = PyTuple_New(3);
        if (!r) return nullptr;
        PyTuple_SET_ITEM(r, 0, y.result());
        PyTuple_SET_ITEM(r, 1, mean.result());
        PyTuple_SET_ITEM(r, 2, rstd.result());
        return r;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// train_backward(x, dy, dx, idx, W, dW, mean, rstd, gamma, beta, bias, n_in, frames, lut_binarize, binary) -> dx; dmean and dvar go to scratch
PyObject *train_backward(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    static decltype(&bbcu_fp32_DifferentiableLut6_Backward) fn = nullptr;
    if (n != 15) { PyErr_SetString(PyExc_TypeError, "train_backward takes 15 arguments"); return nullptr; }
    float gamma, beta, bias, *dW;
    const float *x, *dy, *W, *mean, *rstd;
    const int *index;
    int n_in, frames, lut_binarize, binary;
    try {
        const at::Tensor *xt = tensor_of(o[0], 2, "x"), *dyt = xt ? tensor_of(o[1], 2, "dy") : nullptr, *idx = dyt ? tensor_of(o[3], 1, "idx") : nullptr;
        if (!idx || !parse(o[0], x) || !parse(o[1], dy) || !parse(o[3], index) || !parse(o[4], W) || !parse(o[5], dW) || !parse(o[6], mean) ||
            !parse(o[7], rstd) || !parse(o[8], gamma) || !parse(o[9], beta) || !parse(o[10], bias) || !parse(o[11], n_in) || !parse(o[12], frames) ||
            !parse_flag(o[13], lut_binarize) || !parse_flag(o[14], binary) || !bound(fn, "bbcu_fp32_DifferentiableLut6_Backward")) return nullptr;
        const int64_t stride = dyt->size(1), nodes = idx->size(0);
        if (xt->size(1) != stride) { PyErr_SetString(PyExc_AssertionError, "x and dy differ in their stride"); return nullptr; }
        if (stride > INT_MAX || nodes > INT_MAX) { PyErr_SetString(PyExc_OverflowError, "a size does not fit the operator"); return nullptr; }
        Output dx, scratch;
        if (!dx.take(o[2], *dyt, {n_in, stride}) || !scratch.take(Py_None, *dyt, {2 * nodes})) return nullptr;
        const auto stream = reinterpret_cast<bbcu_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
        int status = 0;
        Py_BEGIN_ALLOW_THREADS
        status = fn(x, dy, dx.data, nullptr, index, nullptr, W, dW, mean, rstd, scratch.data, scratch.data + nodes, gamma, beta, bias, 0, n_in, (int)nodes, frames,
                    (int)stride, 0, 0, lut_binarize, binary, stream);
        Py_END_ALLOW_THREADS
        if (status != 0) return raise_status("bbcu_fp32_DifferentiableLut6_Backward", status);
        return dx.result();
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// ---- operators over the nodes of a frame: checks, new tensors and the call in one, as for the training step above (a call on one frame is some 5 us of
// device time; the checks and allocations in Python took 8)

bool refuse(const char *name, const char *what) { PyErr_Format(PyExc_ValueError, "%s: %s", name, what); return false; }

// the size as the operators take it
bool fits(int64_t n, int &v)
{
    if (n < 0 || n > INT_MAX) { PyErr_SetString(PyExc_OverflowError, "a size does not fit the operator"); return false; }
    v = (int)n;
    return true;
}

// The device of a call's tensors: that of the first one, and the current one, since that is whose stream and scratch the operators take.
struct Place {
    int index = -1;

    bool take(const at::Tensor &t, const char *name)
    {
        if (!t.is_cuda()) return refuse(name, "expected a CUDA tensor (the bbcu_* operators have no CPU path)");
        const int at = t.device().index();
        if (index < 0) index = at;
        if (at == index) return true;
        PyErr_Format(PyExc_ValueError, "%s: expected a tensor on cuda:%d, as the others of the call, got cuda:%d", name, index, at);
        return false;
    }
    // before anything is allocated or launched
    bool here() const
    {
        const int current = c10::cuda::current_device();
        if (current == index) return true;
        PyErr_Format(PyExc_ValueError, "the tensors are on cuda:%d, the current device is cuda:%d", index, current);
        return false;
    }
    bool stream(bbcu_stream_t &s) const
    {
        if (!here()) return false;
        s = reinterpret_cast<bbcu_stream_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream());
        return true;
    }
};

// A buffer of at least `frames` columns that are next to each other, rows any distance apart; `rows` < 0: any number.
struct Frames {
    Place &place;
    PyObject *given = nullptr;
    at::Tensor made;
    const at::Tensor *t = nullptr;
    int stride = 0;

    explicit Frames(Place &place) : place(place) {}
    bool check(PyObject *o, const char *name, int64_t frames, int64_t rows)
    {
        if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "%s: expected a tensor", name); return false; }
        given = o;
        t = &THPVariable_Unpack(o);
        if (!place.take(*t, name)) return false;
        if (t->dim() != 2 || t->size(1) < frames || (t->size(1) > 1 && t->stride(1) != 1) || (t->size(0) > 1 && t->stride(0) < frames))
            return refuse(name, "expected [nodes, frame_stride] of at least the frames asked for, the frames of a node next to each other");
        if (rows >= 0 && t->size(0) != rows) { PyErr_Format(PyExc_ValueError, "%s: expected %lld rows, got %lld", name, (long long)rows, (long long)t->size(0)); return false; }
        return fits(t->size(0) > 1 ? t->stride(0) : t->size(1), stride);
    }
    // fp32 or bf16, or of the same type as `like`
    bool take(PyObject *o, const char *name, int64_t frames, const at::Tensor *like, int64_t rows)
    {
        if (!check(o, name, frames, rows)) return false;
        if (t->scalar_type() != at::kFloat && t->scalar_type() != at::kBFloat16) return refuse(name, "expected dtype float32 or bfloat16");
        if (like && t->scalar_type() != like->scalar_type()) return refuse(name, "expected the dtype of the other frames");
        return true;
    }
    // an output: the given buffer, or for None a new one whose rows are padded to 32 bytes
    bool output(PyObject *o, const char *name, int64_t frames, at::ScalarType type, const at::Tensor &like, int64_t rows)
    {
        if (o != Py_None) {
            if (!take(o, name, frames, nullptr, rows)) return false;
            return t->scalar_type() == type || refuse(name, "expected the dtype of the other frames");
        }
        if (!place.here()) return false;
        const int64_t unit = type == at::kFloat ? 8 : 16;
        made = at::empty({rows, (frames + unit - 1) / unit * unit}, at::TensorOptions().dtype(type).device(like.device()));
        t = &made;
        return fits(made.size(1), stride);
    }
    bool fp32() const { return t->scalar_type() == at::kFloat; }
    template <class P> P in() const { return static_cast<P>(t->const_data_ptr()); }
    template <class P> P out() const { return static_cast<P>(t->mutable_data_ptr()); }
    PyObject *result() const { return given ? Py_NewRef(given) : THPVariable_Wrap(made); }
};

// fp32 numbers of nodes or frames: given, or for None absent (input) or new (output)
struct Numbers {
    Place &place;
    PyObject *given = nullptr;
    at::Tensor made;
    float *data = nullptr;

    explicit Numbers(Place &place) : place(place) {}
    bool check(PyObject *o, const char *name, int64_t size, bool written)
    {
        if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "%s: expected a tensor", name); return false; }
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!place.take(t, name)) return false;
        if (t.scalar_type() != at::kFloat || t.numel() < size || !t.is_contiguous()) {
            PyErr_Format(PyExc_ValueError, "%s: expected a contiguous float32 tensor of %lld values", name, (long long)size);
            return false;
        }
        data = written ? static_cast<float *>(t.mutable_data_ptr()) : const_cast<float *>(static_cast<const float *>(t.const_data_ptr()));
        given = o;
        return true;
    }
    bool input(PyObject *o, const char *name, int64_t size) { return o == Py_None || check(o, name, size, false); }
    bool output(PyObject *o, const char *name, int64_t size, const at::Tensor &like)
    {
        if (o != Py_None) return check(o, name, size, true);
        if (!place.here()) return false;
        made = at::empty({size}, at::TensorOptions().dtype(at::kFloat).device(like.device()));
        data = static_cast<float *>(made.mutable_data_ptr());
        return true;
    }
    PyObject *result() const { return given ? Py_NewRef(given) : THPVariable_Wrap(made); }
};

// rows of 8-bit integers
const at::Tensor *int8_rows(PyObject *o, const char *name, Place &place)
{
    if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "%s: expected a tensor", name); return nullptr; }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!place.take(t, name)) return nullptr;
    if (t.scalar_type() != at::kChar || t.dim() != 2 || !t.is_contiguous()) { refuse(name, "expected a contiguous int8 CUDA tensor [rows, inputs]"); return nullptr; }
    return &t;
}

PyObject *tuple_of(PyObject *a, PyObject *b, PyObject *c = nullptr)
{
    PyObject *r = a && b ? (c ? PyTuple_Pack(3, a, b, c) : PyTuple_Pack(2, a, b)) : nullptr;
    Py_XDECREF(a); Py_XDECREF(b); Py_XDECREF(c);
    return r;
}

// the operator of the frames' type, looked up once; a status, or INT_MIN with a Python error set
#define BB200_CALL_OF_TYPE(fp32, name32, name16, T32, T16, ...)                                            \
    [&] {                                                                                                  \
        static decltype(&name32) fn32 = nullptr;                                                           \
        static decltype(&name16) fn16 = nullptr;                                                           \
        if (fp32 ? !bound(fn32, #name32) : !bound(fn16, #name16)) return INT_MIN;                          \
        int status = 0;                                                                                    \
        Py_BEGIN_ALLOW_THREADS                                                                             \
        if (fp32) { using T = T32; status = fn32(__VA_ARGS__); } else { using T = T16; status = fn16(__VA_ARGS__); } \
        Py_END_ALLOW_THREADS                                                                               \
        if (status != 0) { raise_status(fp32 ? #name32 : #name16, status); return INT_MIN; }               \
        return 0;                                                                                          \
    }()

#define BB200_GUARDED(name, args)                                                                           \
    PyObject *name(PyObject *, PyObject *const *o, Py_ssize_t n)                                            \
    {                                                                                                       \
        if (n != args) { PyErr_SetString(PyExc_TypeError, #name " takes " #args " arguments"); return nullptr; } \
        try {                                                                                               \
            return name##_body(o);                                                                          \
        } catch (const std::exception &e) {                                                                 \
            PyErr_SetString(PyExc_RuntimeError, e.what());                                                  \
            return nullptr;                                                                                 \
        }                                                                                                   \
    }

// layer_norm_forward(x, frames, gamma, beta, eps, y, mean, rstd) -> (y, mean, rstd)
PyObject *layer_norm_forward_body(PyObject *const *o)
{
    int frames, nodes;
    float eps;
    Place place;
    bbcu_stream_t stream;
    Frames x(place), y(place);
    Numbers gamma(place), beta(place), mean(place), rstd(place);
    if (!parse(o[1], frames) || !parse(o[4], eps) || !x.take(o[0], "x", frames, nullptr, -1) || !fits(x.t->size(0), nodes) || !gamma.input(o[2], "gamma", nodes) ||
        !beta.input(o[3], "beta", nodes) || !y.output(o[5], "y", frames, x.t->scalar_type(), *x.t, nodes) || !mean.output(o[6], "mean", frames, *x.t) ||
        !rstd.output(o[7], "rstd", frames, *x.t)) return nullptr;
    if (!place.stream(stream) || BB200_CALL_OF_TYPE(x.fp32(), bbcu_fp32_LayerNormalization_Forward, bbcu_bf16_LayerNormalization_Forward, float, bbcu_bf16_t, x.in<const T *>(), y.out<T *>(),
                           gamma.data, beta.data, mean.data, rstd.data, eps, nodes, frames, x.stride, y.stride, stream)) return nullptr;
    return tuple_of(y.result(), mean.result(), rstd.result());
}
BB200_GUARDED(layer_norm_forward, 8)

// layer_norm_backward(x, dy, mean, rstd, frames, gamma, dx, dgamma, dbeta) -> (dx, dgamma, dbeta)
PyObject *layer_norm_backward_body(PyObject *const *o)
{
    int frames, nodes;
    Place place;
    bbcu_stream_t stream;
    Frames x(place), dy(place), dx(place);
    Numbers gamma(place), mean(place), rstd(place), dgamma(place), dbeta(place);
    if (!parse(o[4], frames) || !x.take(o[0], "x", frames, nullptr, -1) || !fits(x.t->size(0), nodes) || !dy.take(o[1], "dy", frames, x.t, nodes) ||
        !gamma.input(o[5], "gamma", nodes) || !mean.check(o[2], "mean", frames, false) || !rstd.check(o[3], "rstd", frames, false)) return nullptr;
    if ((o[7] == Py_None) != (o[8] == Py_None)) { refuse("dgamma and dbeta", "both or neither"); return nullptr; }
    const int accumulate = o[7] != Py_None;
    if (!dgamma.output(o[7], "dgamma", nodes, *x.t) || !dbeta.output(o[8], "dbeta", nodes, *x.t) ||
        !dx.output(o[6], "dx", frames, x.t->scalar_type(), *x.t, nodes)) return nullptr;
    if (!place.stream(stream) || BB200_CALL_OF_TYPE(x.fp32(), bbcu_fp32_LayerNormalization_Backward, bbcu_bf16_LayerNormalization_Backward, float, bbcu_bf16_t, x.in<const T *>(), dy.in<const T *>(),
                           dx.out<T *>(), gamma.data, mean.data, rstd.data, dgamma.data, dbeta.data, accumulate, nodes, frames, x.stride, dy.stride, dx.stride,
                           stream)) return nullptr;
    return tuple_of(dx.result(), dgamma.result(), dbeta.result());
}
BB200_GUARDED(layer_norm_backward, 9)

// quantize_int8(x, frames) -> (q, scale)
PyObject *quantize_int8_body(PyObject *const *o)
{
    int frames, nodes;
    Place place;
    bbcu_stream_t stream;
    Frames x(place);
    Numbers scale(place);
    if (!parse(o[1], frames) || !x.take(o[0], "x", frames, nullptr, -1) || !fits(x.t->size(0), nodes) || !scale.output(Py_None, "scale", frames, *x.t)) return nullptr;
    const int row = (int)std::min<int64_t>(((int64_t)nodes + 15) / 16 * 16, INT_MAX / 16 * 16);
    at::Tensor q = at::empty({frames, row}, at::TensorOptions().dtype(at::kChar).device(x.t->device()));
    if (!place.stream(stream) || BB200_CALL_OF_TYPE(x.fp32(), bbcu_fp32_QuantizeInt8_Frames, bbcu_bf16_QuantizeInt8_Frames, float, bbcu_bf16_t, x.in<const T *>(),
                           static_cast<signed char *>(q.mutable_data_ptr()), scale.data, nodes, frames, x.stride, row, stream)) return nullptr;
    return tuple_of(THPVariable_Wrap(q), scale.result());
}
BB200_GUARDED(quantize_int8, 2)

// int8_dense_forward(q, scale, W, w_scale, n_in, bias, y, bf16) -> y; n_in None: the length of q's rows; bf16: the type of a new y
PyObject *int8_dense_forward_body(PyObject *const *o)
{
    int frames, nodes, n_in, q_stride, w_stride, bf16;
    Place place;
    bbcu_stream_t stream;
    Frames y(place);
    Numbers scale(place), w_scale(place), bias(place);
    const at::Tensor *q = int8_rows(o[0], "q", place), *W = q ? int8_rows(o[2], "W", place) : nullptr;
    if (!W || !fits(q->size(0), frames) || !fits(W->size(0), nodes) || !fits(q->size(1), q_stride) || !fits(W->size(1), w_stride) || !parse_flag(o[7], bf16) ||
        !scale.check(o[1], "scale", frames, false) || !w_scale.check(o[3], "w_scale", nodes, false) || !bias.input(o[5], "bias", nodes)) return nullptr;
    n_in = q_stride;
    if (o[4] != Py_None && !parse(o[4], n_in)) return nullptr;
    if (o[6] != Py_None ? !y.take(o[6], "y", frames, nullptr, nodes) : !y.output(Py_None, "y", frames, bf16 ? at::kBFloat16 : at::kFloat, *q, nodes)) return nullptr;
    if (!place.stream(stream) || BB200_CALL_OF_TYPE(y.fp32(), bbcu_int8_fp32_DenseAffine_Forward, bbcu_int8_bf16_DenseAffine_Forward, float, bbcu_bf16_t,
                           static_cast<const signed char *>(q->const_data_ptr()), scale.data, static_cast<const signed char *>(W->const_data_ptr()), w_scale.data,
                           bias.data, y.out<T *>(), n_in, nodes, frames, q_stride, w_stride, y.stride, stream)) return nullptr;
    return y.result();
}
BB200_GUARDED(int8_dense_forward, 8)

// distillation_loss(z, t, index, frames, temperature, t_lse, weight, batch_size, dz, loss_buf) -> (dz, loss, loss_buf)
PyObject *distillation_loss_body(PyObject *const *o)
{
    int frames, classes, top;
    float temperature;
    double batch;
    Place place;
    bbcu_stream_t stream;
    Frames z(place), t(place), index(place), dz(place);
    Numbers t_lse(place), weight(place), loss_buf(place);
    if (!parse(o[3], frames) || !parse(o[4], temperature) || !z.take(o[0], "z", frames, nullptr, -1) || !fits(z.t->size(0), classes) ||
        !t.take(o[1], "t", frames, z.t, -1) || !fits(t.t->size(0), top) || !index.check(o[2], "index", frames, top)) return nullptr;
    if (index.t->scalar_type() != at::kInt) { refuse("index", "expected dtype int32"); return nullptr; }
    if (!t_lse.input(o[5], "t_lse", frames) || !weight.input(o[6], "weight", frames) || !dz.output(o[8], "dz", frames, z.t->scalar_type(), *z.t, classes) ||
        !loss_buf.output(o[9], "loss_buf", frames, *z.t)) return nullptr;
    batch = frames;
    if (o[7] != Py_None && !parse(o[7], batch)) return nullptr;
    const double reduction = 1.0 / (batch > 1.0 ? batch : 1.0);
    at::Tensor loss = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(z.t->device()));
    float *const loss_data = static_cast<float *>(loss.mutable_data_ptr());
    if (!place.stream(stream) || BB200_CALL_OF_TYPE(z.fp32(), bbcu_fp32_LossDistillation, bbcu_bf16_LossDistillation, float, bbcu_bf16_t, z.in<const T *>(), dz.out<T *>(), t.in<const T *>(),
                           index.in<const int *>(), t_lse.data, weight.data, loss_buf.data, loss_data, temperature, (float)reduction, reduction, classes, top, frames,
                           z.stride, dz.stride, t.stride, index.stride, stream)) return nullptr;
    return tuple_of(dz.result(), THPVariable_Wrap(loss), loss_buf.result());
}
BB200_GUARDED(distillation_loss, 10)

#define BB200_METHOD(name, function) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)), METH_FASTCALL, nullptr},
#define BB200_OPERATOR_METHOD(name) BB200_METHOD(#name, py_##name)
PyMethodDef g_methods[] = {
    BB200_OPERATORS(BB200_OPERATOR_METHOD)
    BB200_METHOD("empty_f32", empty_f32) BB200_METHOD("empty_i32", empty_i32) BB200_METHOD("vector_f32", vector_f32) BB200_METHOD("scalar_f64", scalar_f64)
    BB200_METHOD("train_forward", train_forward) BB200_METHOD("train_backward", train_backward)
    BB200_METHOD("layer_norm_forward", layer_norm_forward) BB200_METHOD("layer_norm_backward", layer_norm_backward) BB200_METHOD("quantize_int8", quantize_int8)
    BB200_METHOD("int8_dense_forward", int8_dense_forward) BB200_METHOD("distillation_loss", distillation_loss)
    {nullptr, nullptr, 0, nullptr}};
#undef BB200_METHOD

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", "bbcu_* operators on torch tensors", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}   // namespace

PyMODINIT_FUNC PyInit__native()
{
    PyObject *m = PyModule_Create(&g_module);
    if (!m) return nullptr;
    if (PyModule_AddIntConstant(m, "SMALL_NODE_FRAMES", BBCU_B200_SMALL_NODE_FRAMES) || PyModule_AddIntConstant(m, "SMALL_FRAMES", BBCU_B200_SMALL_FRAMES)) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
