// The operator calls on torch CUDA tensors, as a CPython extension (module catccos_b200._torch_calls).
//
// catccos_b200/capi.py declares the calls; what they do per call is here: unpack the tensors, fill the tiling record,
// take the current stream, allocate the outputs, call the C ABI (include/catccos_b200.h).  Host time of a call, launch
// included: 8.8 us (mx_gemm) to 14 (mx_quant) with these steps in Python and ctypes, more than the kernels of the small
// problems take; 2.9 to 4.2 us here.
//
// The C ABI's functions are not linked but bound by address (bind()), so that they are those of the library that capi.py
// has loaded.  Every function returns the C ABI's code (alone, or first in a tuple with the outputs).
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstring>
#include <initializer_list>

#include "../../include/catccos_b200.h"

namespace {

#define BOUND(name) decltype(&catccos_b200_##name) name##_fn = nullptr
BOUND(mx_quant);
BOUND(mx_quant_fp4);
BOUND(mx_gemm);
BOUND(mx_gemm_quant_out);
BOUND(mx_quant_scatter_packed);
BOUND(mxfp8_matmul_reduce_scatter);
BOUND(add_rms_norm_mx_quant);
BOUND(moe_route);
BOUND(moe_row_plan);
BOUND(mx_grouped_gemm_typed);
BOUND(moe_combine);
BOUND(mx_fp4_matvec_typed);
BOUND(mx_quant_matmul_static);
BOUND(mx_quant_allgather);
BOUND(mx_quant_allgather_matmul);
BOUND(fp8_mx_allgather_matmul);
BOUND(fp4_mx_allgather_matmul);
#undef BOUND

struct Error {};  // a Python exception is set

const at::Tensor& tensor(PyObject* o)
{
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expected a torch tensor, got %s", Py_TYPE(o)->tp_name);
        throw Error{};
    }
    return THPVariable_Unpack(o);
}

struct Rows {
    const at::Tensor& t;
    uint32_t rows, cols;
};

Rows matrix(PyObject* o)
{
    const at::Tensor& t = tensor(o);
    if (t.dim() != 2) {
        PyErr_Format(PyExc_ValueError, "expected a matrix, got %d dimensions", (int)t.dim());
        throw Error{};
    }
    return {t, (uint32_t)t.size(0), (uint32_t)t.size(1)};
}

// columns of the product: b_scales is [k / 64, n, 2]
uint32_t product_columns(PyObject* b_scales)
{
    const at::Tensor& t = tensor(b_scales);
    if (t.dim() < 2) {
        PyErr_SetString(PyExc_IndexError, "b_scales is [k / 64, n, 2]");
        throw Error{};
    }
    return (uint32_t)t.size(1);
}

void* pointer(PyObject* tensor_object) { return tensor(tensor_object).data_ptr(); }

// An address as ctypes takes one: a number, None, or a pointer object with a `value` (ctypes.c_void_p).
void* address(PyObject* o)
{
    if (o == Py_None) {
        return nullptr;
    }
    if (PyLong_Check(o)) {
        void* p = PyLong_AsVoidPtr(o);
        if (p == nullptr && PyErr_Occurred()) {
            throw Error{};
        }
        return p;
    }
    PyObject* value = PyObject_GetAttrString(o, "value");
    if (value == nullptr || !(value == Py_None || PyLong_Check(value))) {
        Py_XDECREF(value);
        PyErr_Format(PyExc_TypeError, "expected an address, got %s", Py_TYPE(o)->tp_name);
        throw Error{};
    }
    void* p = value == Py_None ? nullptr : PyLong_AsVoidPtr(value);
    Py_DECREF(value);
    if (p == nullptr && PyErr_Occurred()) {
        throw Error{};
    }
    return p;
}

uint32_t count(PyObject* number)
{
    const long v = PyLong_AsLong(number);
    if (v == -1 && PyErr_Occurred()) {
        throw Error{};
    }
    return (uint32_t)v;
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

at::Tensor bytes_like(const at::Tensor& x, int64_t rows, int64_t cols)
{
    return at::detail::empty_cuda({rows, cols}, at::kByte, x.device(), std::nullopt);
}

// The reference drivers' default tile fields (main.cpp:105-118), with the problem shape filled in.
catccos_b200_tiling_t tiling(uint32_t m, uint32_t k, uint32_t n, uint32_t world)
{
    catccos_b200_tiling_t t;
    memset(&t, 0, sizeof(t));
    t.m = m;
    t.k = k;
    t.n = n;
    t.m0 = 128;
    t.k0 = 256;
    t.n0 = 256;
    t.commTileM = 64;
    t.commInterval = 3;
    t.commNpuSplit = 2;
    t.commDataSplit = 16;
    t.commBlockM = 64;
    t.rankSize = world;
    t.topK = 1;
    return t;
}

// Launches may wait for room in the stream's queue: other Python threads run meanwhile.  The lock is back before an
// exception leaves.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

template <typename F>
PyObject* released(F&& call)
{
    int rc;
    {
        Unlocked unlocked;
        rc = call();
    }
    return PyLong_FromLong(rc);
}

PyObject* with_outputs(PyObject* code, const at::Tensor& a, const at::Tensor& b)
{
    PyObject* out = PyTuple_New(3);
    PyTuple_SET_ITEM(out, 0, code);
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(a));
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(b));
    return out;
}

template <typename F>
PyObject* guarded(const char* name, Py_ssize_t want, Py_ssize_t n, bool bound, F&& body)
{
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, n);
        return nullptr;
    }
    if (!bound) {
        PyErr_Format(PyExc_RuntimeError, "%s is not bound to the library", name);
        return nullptr;
    }
    try {
        return body();
    } catch (const Error&) {
        return nullptr;
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());  // torch.OutOfMemoryError and the like
        return nullptr;
    }
}

void assert_activations(const at::Tensor& x)
{
    if (!x.is_cuda() || !x.is_contiguous() || x.element_size() != 2) {
        PyErr_SetString(PyExc_AssertionError, "expected a contiguous CUDA tensor of 16-bit values");
        throw Error{};
    }
}

// ---- calls that check what they are given: element types, shapes, one device (which becomes the current one) -----------------
[[noreturn]] void refuse(const char* what, const char* wanted)
{
    PyErr_Format(PyExc_ValueError, "%s: expected %s", what, wanted);
    throw Error{};
}

float real(PyObject* number)
{
    const double v = PyFloat_AsDouble(number);
    if (v == -1.0 && PyErr_Occurred()) {
        throw Error{};
    }
    return (float)v;
}

int64_t whole(PyObject* number, const char* what)
{
    const long long v = PyLong_AsLongLong(number);
    if (v == -1 && PyErr_Occurred()) {
        throw Error{};
    }
    if (v < 0 || v > 0x7FFFFFFFll) {
        refuse(what, "a number from 0 to 2^31 - 1");
    }
    return v;
}

// A CUDA tensor on `like`'s device (any, without one), of one of the types, contiguous.
const at::Tensor& plain(PyObject* o, const char* what, const char* wanted, std::initializer_list<at::ScalarType> types, int dims,
                        const at::Tensor* like = nullptr, bool contiguous = true)
{
    const at::Tensor& t = tensor(o);
    bool ok = t.is_cuda() && (dims < 0 || t.dim() == dims) && (!contiguous || t.is_contiguous()) &&
              (like == nullptr || t.device() == like->device());
    bool type = false;
    for (at::ScalarType s : types) {
        type = type || t.scalar_type() == s;
    }
    if (!ok || !type) {
        refuse(what, wanted);
    }
    for (int64_t s : t.sizes()) {
        if (s > 0x7FFFFFFFll) {
            refuse(what, "sizes below 2^31");
        }
    }
    return t;
}

// Two outputs of a call.  Small ones lie in one allocation, the second behind the first: taking a block from the caching allocator
// costs 0.8 us, a quarter of a small call's time on the host.  Large ones are apart, so that neither keeps the other's memory.
struct Pair {
    at::Tensor first, second;
    Pair(const at::Tensor& like, at::IntArrayRef shape1, at::ScalarType type1, at::IntArrayRef shape2, at::ScalarType type2)
    {
        constexpr size_t kTogether = 1u << 20;
        const size_t size1 = (size_t)c10::multiply_integers(shape1) * c10::elementSize(type1), at2 = (size1 + 255) / 256 * 256;
        const size_t size2 = (size_t)c10::multiply_integers(shape2) * c10::elementSize(type2);
        if (at2 + size2 > kTogether) {
            first = at::detail::empty_cuda(shape1, type1, like.device(), std::nullopt);
            second = at::detail::empty_cuda(shape2, type2, like.device(), std::nullopt);
            return;
        }
        const at::Tensor whole = at::detail::empty_cuda({(int64_t)(at2 + size2)}, at::kByte, like.device(), std::nullopt);
        first = part(whole, 0, shape1, type1);
        second = part(whole, at2, shape2, type2);
    }

private:
    static at::Tensor part(const at::Tensor& whole, size_t byte, at::IntArrayRef shape, at::ScalarType type)
    {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_storage_offset((int64_t)(byte / c10::elementSize(type)));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        return t;
    }
};

// The result's tensor: the one that is given, checked, or a new one.
at::Tensor result(PyObject* given, const char* wanted, std::initializer_list<at::ScalarType> types, const at::Tensor& like, int64_t rows,
                  int64_t cols, at::ScalarType type)
{
    if (given == Py_None) {
        return at::detail::empty_cuda({rows, cols}, type, like.device(), std::nullopt);
    }
    const at::Tensor& out = plain(given, "out", wanted, types, 2, &like);
    if (out.size(0) != rows || out.size(1) != cols) {
        refuse("out", wanted);
    }
    return out;
}

// torch.bfloat16, torch.float16, or None for the first
at::ScalarType half_type(PyObject* dtype)
{
    if (dtype == Py_None) {
        return at::kBFloat16;
    }
    const at::ScalarType type = THPDtype_Check(dtype) ? reinterpret_cast<THPDtype*>(dtype)->scalar_type : at::kFloat;
    if (type != at::kBFloat16 && type != at::kHalf) {
        refuse("out_dtype", "torch.bfloat16 or torch.float16");
    }
    return type;
}

// The type of 8-bit codes as the C ABI numbers it, where the tensor says it: bytes may be either, the option tells (-1).
int code_type(const at::Tensor& t)
{
    return t.scalar_type() == at::kFloat8_e4m3fn ? 0 : (t.scalar_type() == at::kFloat8_e5m2 ? 1 : -1);
}

PyObject* with_output(PyObject* code, PyObject* given, const at::Tensor& made)
{
    PyObject* out = PyTuple_New(2);
    PyTuple_SET_ITEM(out, 0, code);
    if (given != Py_None) {
        Py_INCREF(given);
    }
    PyTuple_SET_ITEM(out, 1, given != Py_None ? given : THPVariable_Wrap(made));
    return out;
}

void* data_or_null(PyObject* o) { return o == Py_None ? nullptr : tensor(o).data_ptr(); }

// The tensors' device for the rest of a call, and its current stream.
struct OnDevice {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit OnDevice(const at::Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

constexpr auto kBf16 = at::kBFloat16, kF16 = at::kHalf, kF32 = at::kFloat, kI32 = at::kInt, kU8 = at::kByte;

#define CALL(name, nargs) \
    PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(#name, nargs, n, name##_fn != nullptr, [&]() -> PyObject* {
#define END_CALL }); }

CALL(mx_quant, 1)
    const Rows x = matrix(a[0]);
    assert_activations(x.t);
    const at::Tensor codes = bytes_like(x.t, x.rows, x.cols), scales = bytes_like(x.t, x.rows, x.cols / 32);
    void *st = stream(), *in = x.t.data_ptr(), *c = codes.data_ptr(), *s = scales.data_ptr();
    return with_outputs(released([&] { return mx_quant_fn(st, in, x.rows, x.cols, c, s); }), codes, scales);
END_CALL

CALL(mx_quant_fp4, 1)
    const Rows x = matrix(a[0]);
    assert_activations(x.t);
    const at::Tensor packed = bytes_like(x.t, x.rows, x.cols / 2), scales = bytes_like(x.t, x.rows, x.cols / 32);
    void *st = stream(), *in = x.t.data_ptr(), *c = packed.data_ptr(), *s = scales.data_ptr();
    return with_outputs(released([&] { return mx_quant_fp4_fn(st, in, x.rows, x.cols, c, s); }), packed, scales);
END_CALL

// a, a_scales, b, b_scales, out
CALL(mx_gemm, 5)
    const Rows x = matrix(a[0]);
    const uint32_t cols = product_columns(a[3]);
    void *st = stream(), *ac = x.t.data_ptr(), *as = pointer(a[1]), *b = pointer(a[2]), *bs = pointer(a[3]), *c = pointer(a[4]);
    return released([&] { return mx_gemm_fn(st, ac, as, b, bs, c, x.rows, cols, x.cols); });
END_CALL

// a, a_scales, b, b_scales
CALL(mx_gemm_quant_out, 4)
    const Rows x = matrix(a[0]);
    const uint32_t cols = product_columns(a[3]);
    const at::Tensor codes = bytes_like(x.t, x.rows, cols), scales = bytes_like(x.t, x.rows, cols / 32);
    void *st = stream(), *ac = x.t.data_ptr(), *as = pointer(a[1]), *b = pointer(a[2]), *bs = pointer(a[3]);
    void *c = codes.data_ptr(), *s = scales.data_ptr();
    return with_outputs(released([&] { return mx_gemm_quant_out_fn(st, ac, as, b, bs, c, s, x.rows, cols, x.cols); }), codes, scales);
END_CALL

// x, expanded_row_idx, packed_out, top_k
CALL(mx_quant_scatter_packed, 4)
    const Rows x = matrix(a[0]);
    const uint32_t top_k = count(a[3]);
    void *st = stream(), *in = x.t.data_ptr(), *idx = pointer(a[1]), *out = pointer(a[2]);
    return released([&] { return mx_quant_scatter_packed_fn(st, in, (const int32_t*)idx, out, x.rows, x.cols, top_k); });
END_CALL

// a, a_scales, b, b_scales, d, symm, world
CALL(mxfp8_matmul_reduce_scatter, 7)
    const Rows x = matrix(a[0]);
    const catccos_b200_tiling_t t = tiling(x.rows, x.cols, product_columns(a[3]), count(a[6]));
    void *st = stream(), *ac = x.t.data_ptr(), *as = pointer(a[1]), *b = pointer(a[2]), *bs = pointer(a[3]), *d = pointer(a[4]);
    void* symm = address(a[5]);
    return released([&] { return mxfp8_matmul_reduce_scatter_fn(st, ac, b, as, bs, d, symm, &t, 0); });
END_CALL

// a_bf16, b, b_scales, c
CALL(mx_quant_matmul_static, 4)
    const Rows x = matrix(a[0]);
    const uint32_t cols = product_columns(a[2]);
    void *st = stream(), *in = x.t.data_ptr(), *b = pointer(a[1]), *bs = pointer(a[2]), *c = pointer(a[3]);
    return released([&] { return mx_quant_matmul_static_fn(st, in, b, bs, c, x.rows, cols, x.cols); });
END_CALL

// x, out_codes, out_scales, symm, world
CALL(mx_quant_allgather, 5)
    const Rows x = matrix(a[0]);
    const catccos_b200_tiling_t t = tiling(x.rows, 1, x.cols, count(a[4]));  // the quantised axis is `n` for this operator
    void *st = stream(), *in = x.t.data_ptr(), *c = pointer(a[1]), *s = pointer(a[2]), *symm = address(a[3]);
    return released([&] { return mx_quant_allgather_fn(st, in, c, s, symm, &t, 0); });
END_CALL

// a_bf16, b, b_scales, c, symm, world
CALL(mx_quant_allgather_matmul, 6)
    const Rows x = matrix(a[0]);
    const catccos_b200_tiling_t t = tiling(x.rows, x.cols, product_columns(a[2]), count(a[5]));
    void *st = stream(), *in = x.t.data_ptr(), *b = pointer(a[1]), *bs = pointer(a[2]), *c = pointer(a[3]), *symm = address(a[4]);
    return released([&] { return mx_quant_allgather_matmul_fn(st, in, b, bs, c, symm, &t, 0); });
END_CALL

// a, a_scales, b, b_scales, c, symm, world
CALL(fp8_mx_allgather_matmul, 7)
    const Rows x = matrix(a[0]);
    const catccos_b200_tiling_t t = tiling(x.rows, x.cols, product_columns(a[3]), count(a[6]));
    void *st = stream(), *ac = x.t.data_ptr(), *as = pointer(a[1]), *b = pointer(a[2]), *bs = pointer(a[3]), *c = pointer(a[4]);
    void* symm = address(a[5]);
    return released([&] { return fp8_mx_allgather_matmul_fn(st, ac, b, as, bs, c, symm, &t, 0); });
END_CALL

// a_packed [m, k / 2], a_scales, b_packed, b_scales, c, symm, world
CALL(fp4_mx_allgather_matmul, 7)
    const Rows x = matrix(a[0]);
    const catccos_b200_tiling_t t = tiling(x.rows, x.cols * 2, product_columns(a[3]), count(a[6]));
    void *st = stream(), *ac = x.t.data_ptr(), *as = pointer(a[1]), *b = pointer(a[2]), *bs = pointer(a[3]), *c = pointer(a[4]);
    void* symm = address(a[5]);
    return released([&] { return fp4_mx_allgather_matmul_fn(st, ac, b, as, bs, c, symm, &t, 0); });
END_CALL

// x, residual, weight, eps, residual_out, norm_out
CALL(add_rms_norm_mx_quant, 6)
    const char* same = "a contiguous bf16 CUDA matrix of x's shape on x's device";
    const at::Tensor& x = plain(a[0], "x", "a contiguous bf16 CUDA matrix", {kBf16}, 2);
    const int64_t rows = x.size(0), n = x.size(1);
    PyObject* residual_out = a[4] == Py_None ? a[1] : a[4];
    if (a[1] == Py_None && a[4] != Py_None) {
        refuse("residual_out", "None where residual is None");
    }
    PyObject* others[3] = {a[1], residual_out, a[5]};
    const char* names[3] = {"residual", "residual_out", "norm_out"};
    for (int i = 0; i < 3; ++i) {
        if (others[i] != Py_None && plain(others[i], names[i], same, {kBf16}, 2, &x).sizes() != x.sizes()) {
            refuse(names[i], same);
        }
    }
    if (plain(a[2], "weight", "a contiguous bf16 CUDA vector on x's device", {kBf16}, 1, &x).size(0) != n) {
        refuse("weight", "one value for each column of x");
    }
    const float eps = real(a[3]);
    const OnDevice on(x);
    const Pair out(x, {rows, n}, kU8, {rows, n / 32}, kU8);
    const at::Tensor &codes = out.first, &scales = out.second;
    void *in = x.data_ptr(), *r = data_or_null(a[1]), *w = pointer(a[2]), *ro = data_or_null(residual_out), *no = data_or_null(a[5]);
    void *c = codes.data_ptr(), *s = scales.data_ptr();
    return with_outputs(released([&] { return add_rms_norm_mx_quant_fn(on.stream, in, r, w, eps, (uint32_t)rows, (uint32_t)n, ro, no, c, s); }),
                        codes, scales);
END_CALL

// logits, bias, top_k, groups, top_groups, group_best, score, renormalize, scale
CALL(moe_route, 9)
    const at::Tensor& l = plain(a[0], "logits", "a contiguous fp32 or bf16 CUDA matrix", {kF32, kBf16}, 2);
    const int64_t tokens = l.size(0), experts = l.size(1);
    if (a[1] != Py_None &&
        plain(a[1], "bias", "a contiguous fp32 CUDA vector on the logits' device", {kF32}, 1, &l).size(0) != experts) {
        refuse("bias", "one value for each expert");
    }
    const int64_t top_k = whole(a[2], "top_k"), groups = whole(a[3], "groups"), top_groups = whole(a[4], "top_groups"),
                  group_best = whole(a[5], "group_best"), score = whole(a[6], "score"), renormalize = whole(a[7], "renormalize");
    const float scale = real(a[8]);
    const OnDevice on(l);
    // a top_k that the library refuses is not allocated for
    const int64_t k = top_k <= experts ? top_k : 0;
    const Pair out(l, {tokens, k}, kI32, {tokens, k}, kF32);
    const at::Tensor &ids = out.first, &weights = out.second;
    void *in = l.data_ptr(), *b = data_or_null(a[1]), *i = ids.data_ptr(), *w = weights.data_ptr();
    return with_outputs(released([&] {
                            return moe_route_fn(on.stream, in, l.scalar_type() == kBf16 ? 1 : 0, (const float*)b, (uint32_t)tokens,
                                                (uint32_t)experts, (uint32_t)top_k, (uint32_t)groups, (uint32_t)top_groups,
                                                (uint32_t)group_best, (int)score, (int)renormalize, scale, (int32_t*)i, (float*)w);
                        }),
                        ids, weights);
END_CALL

// ids, experts, first_expert
CALL(moe_row_plan, 3)
    const at::Tensor& ids = plain(a[0], "ids", "a contiguous int32 CUDA tensor", {kI32}, -1);
    const int64_t experts = whole(a[1], "experts"), first = whole(a[2], "first_expert");
    if (ids.numel() > 0x7FFFFFFFll) {
        refuse("ids", "fewer than 2^31 routes");
    }
    const OnDevice on(ids);
    // as many experts as the library takes are allocated for
    const Pair out(ids, ids.sizes(), kI32, {experts <= 1024 ? experts + 1 : 1}, kI32);
    const at::Tensor &index = out.first, &offsets = out.second;
    void *in = ids.data_ptr(), *i = index.data_ptr(), *o = offsets.data_ptr();
    const uint32_t routes = (uint32_t)ids.numel();
    return with_outputs(released([&] { return moe_row_plan_fn(on.stream, (const int32_t*)in, routes, (uint32_t)experts, (int32_t)first, (int32_t*)i, (int32_t*)o); }),
                        index, offsets);
END_CALL

// a, a_scales, b, b_scales, offsets, out, out_dtype
CALL(mx_grouped_gemm_typed, 7)
    const auto codes = {kU8, at::kFloat8_e4m3fn, at::kFloat8_e5m2};
    const at::Tensor& x = plain(a[0], "a_codes", "a CUDA matrix of 8-bit codes, its columns next to one another", codes, 2, nullptr, false);
    const at::Tensor& xs = plain(a[1], "a_scales", "a CUDA matrix of bytes on a_codes' device, its columns next to one another",
                                 {kU8, at::kFloat8_e8m0fnu}, 2, &x, false);
    const at::Tensor& b = plain(a[2], "b", "contiguous 8-bit codes [experts, K, N] on a_codes' device", codes, 3, &x);
    const at::Tensor& bs = plain(a[3], "b_scales", "contiguous bytes [experts, K / 64, N, 2] on a_codes' device", {kU8, at::kFloat8_e8m0fnu}, 4, &x);
    const at::Tensor& offsets = plain(a[4], "offsets", "a contiguous int32 vector on a_codes' device", {kI32}, 1, &x);
    const int64_t rows = x.size(0), k = x.size(1), experts = b.size(0), n = b.size(2);
    if ((k > 1 && x.stride(1) != 1) || (k >= 64 && xs.stride(1) != 1) || x.stride(0) < 0 || xs.stride(0) < 0) {
        refuse("a_codes, a_scales", "columns next to one another");
    }
    if (xs.size(0) != rows || xs.size(1) != k / 32 || b.size(1) != k || bs.size(0) != experts || bs.size(1) != k / 64 || bs.size(2) != n ||
        bs.size(3) != 2 || offsets.size(0) != experts + 1) {
        refuse("mx_grouped_gemm", "a [rows, K], a_scales [rows, K / 32], b [experts, K, N], b_scales [experts, K / 64, N, 2], "
                                  "offsets [experts + 1]");
    }
    const OnDevice on(x);
    const at::Tensor out = result(a[5], "a contiguous bf16 or fp16 matrix [rows, N] on a_codes' device", {kBf16, kF16}, x, rows, n, half_type(a[6]));
    // one row has no distance to the next
    const size_t step = rows > 1 ? (size_t)x.stride(0) : (size_t)(k + 15) / 16 * 16, scale_step = rows > 1 ? (size_t)xs.stride(0) : (size_t)(k / 32 + 3) / 4 * 4;
    const int a_type = code_type(x), b_type = code_type(b), c_type = out.scalar_type() == kF16 ? 1 : 0;
    void *ac = x.data_ptr(), *as = xs.data_ptr(), *bc = b.data_ptr(), *bf = bs.data_ptr(), *o = offsets.data_ptr(), *c = out.data_ptr();
    return with_output(released([&] {
                           return mx_grouped_gemm_typed_fn(on.stream, ac, step, as, scale_step, bc, bf, (const int32_t*)o, c,
                                                           (uint32_t)rows, (uint32_t)experts, (uint32_t)n, (uint32_t)k, a_type, b_type,
                                                           c_type);
                       }),
                       a[5], out);
END_CALL

// expert_out, row_index, weights, shared, out
CALL(moe_combine, 5)
    const at::Tensor& y = plain(a[0], "expert_out", "a contiguous bf16 or fp16 CUDA matrix", {kBf16, kF16}, 2);
    const at::ScalarType type = y.scalar_type();
    const at::Tensor& index = plain(a[1], "row_index", "a contiguous int32 matrix on expert_out's device", {kI32}, 2, &y);
    const at::Tensor& w = plain(a[2], "weights", "a contiguous fp32 matrix on expert_out's device", {kF32}, 2, &y);
    const int64_t tokens = index.size(0), n = y.size(1);
    if (w.sizes() != index.sizes()) {
        refuse("moe_combine", "row_index and weights [tokens, top_k]");
    }
    const char* wanted = "a contiguous matrix [tokens, n] of expert_out's type and device";
    const OnDevice on(y);
    const at::Tensor out = result(a[4], wanted, {type}, y, tokens, n, type);
    if (a[3] != Py_None && plain(a[3], "shared", wanted, {type}, 2, &y).sizes() != out.sizes()) {
        refuse("shared", wanted);
    }
    void *in = y.data_ptr(), *i = index.data_ptr(), *g = w.data_ptr(), *s = data_or_null(a[3]), *o = out.data_ptr();
    const uint32_t top_k = (uint32_t)index.size(1), rows = (uint32_t)y.size(0);
    return with_output(released([&] {
                           return moe_combine_fn(on.stream, in, rows, (const int32_t*)i, (const float*)g, s, o, (uint32_t)tokens,
                                                 (uint32_t)n, top_k, type == kF16 ? 1 : 0);
                       }),
                       a[4], out);
END_CALL

// x, w, w_scales, ids, out, out_dtype
CALL(mx_fp4_matvec_typed, 6)
    const bool many = a[3] != Py_None;
    const at::Tensor& x = plain(a[0], "x", "a contiguous bf16 CUDA matrix", {kBf16}, 2);
    const at::Tensor& w = plain(a[1], "w", "contiguous packed codes [K, N / 2], with ids [experts, K, N / 2], on x's device", {kU8}, many ? 3 : 2, &x);
    const at::Tensor& ws = plain(a[2], "w_scales", "contiguous bytes [K / 64, N, 2], with ids [experts, K / 64, N, 2], on x's device",
                                 {kU8, at::kFloat8_e8m0fnu}, many ? 4 : 3, &x);
    const int64_t x_rows = x.size(0), k = x.size(1), experts = many ? w.size(0) : 1, n = 2 * w.size(-1);
    const int64_t rows = many ? plain(a[3], "ids", "a contiguous int32 tensor on x's device", {kI32}, -1, &x).numel() : x_rows;
    if (w.size(-2) != k || ws.size(-3) != k / 64 || ws.size(-2) != n || ws.size(-1) != 2 || (many && ws.size(0) != experts) ||
        rows > 0x7FFFFFFFll) {
        refuse("mx_fp4_matvec", "x [rows, K], w [.., K, N / 2], w_scales [.., K / 64, N, 2]");
    }
    const OnDevice on(x);
    const at::Tensor out = result(a[4], "a contiguous bf16 or fp16 matrix [rows or ids, N] on x's device", {kBf16, kF16}, x, rows, n, half_type(a[5]));
    const int c_type = out.scalar_type() == kF16 ? 1 : 0;
    void *in = x.data_ptr(), *wp = w.data_ptr(), *sp = ws.data_ptr(), *i = data_or_null(a[3]), *o = out.data_ptr();
    return with_output(released([&] {
                           return mx_fp4_matvec_typed_fn(on.stream, in, wp, sp, (const int32_t*)i, o, (uint32_t)rows, (uint32_t)x_rows,
                                                         (uint32_t)experts, (uint32_t)n, (uint32_t)k, c_type);
                       }),
                       a[4], out);
END_CALL

// bind(name, address): which function of the loaded library a call goes to
PyObject* bind(PyObject*, PyObject* args)
{
    const char* name = nullptr;
    unsigned long long at = 0;
    if (!PyArg_ParseTuple(args, "sK", &name, &at)) {
        return nullptr;
    }
#define BIND(fn)                                          \
    if (strcmp(name, "catccos_b200_" #fn) == 0) {         \
        fn##_fn = reinterpret_cast<decltype(fn##_fn)>(at); \
        Py_RETURN_TRUE;                                   \
    }
    BIND(mx_quant)
    BIND(mx_quant_fp4)
    BIND(mx_gemm)
    BIND(mx_gemm_quant_out)
    BIND(mx_quant_scatter_packed)
    BIND(mxfp8_matmul_reduce_scatter)
    BIND(add_rms_norm_mx_quant)
    BIND(moe_route)
    BIND(moe_row_plan)
    BIND(mx_grouped_gemm_typed)
    BIND(moe_combine)
    BIND(mx_fp4_matvec_typed)
    BIND(mx_quant_matmul_static)
    BIND(mx_quant_allgather)
    BIND(mx_quant_allgather_matmul)
    BIND(fp8_mx_allgather_matmul)
    BIND(fp4_mx_allgather_matmul)
#undef BIND
    Py_RETURN_FALSE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    METHOD(mx_quant),
    METHOD(mx_quant_fp4),
    METHOD(mx_gemm),
    METHOD(mx_gemm_quant_out),
    METHOD(mx_quant_scatter_packed),
    METHOD(mxfp8_matmul_reduce_scatter),
    METHOD(add_rms_norm_mx_quant),
    METHOD(moe_route),
    METHOD(moe_row_plan),
    METHOD(mx_grouped_gemm_typed),
    METHOD(moe_combine),
    METHOD(mx_fp4_matvec_typed),
    METHOD(mx_quant_matmul_static),
    METHOD(mx_quant_allgather),
    METHOD(mx_quant_allgather_matmul),
    METHOD(fp8_mx_allgather_matmul),
    METHOD(fp4_mx_allgather_matmul),
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
#undef METHOD

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls(void) { return PyModule_Create(&module); }
