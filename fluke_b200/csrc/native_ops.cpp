// native_ops.cpp -- the tensor side of fluke_b200.ops: argument checks, output allocation and the
// call of the C entry point in one step per operator (extension module fluke_b200._native).
//
// A small launch costs the GPU two or three microseconds; the same call through ctypes costs the
// host eight to ten (attribute look-ups for the checks, one Python call per data pointer,
// torch.empty, conversion of up to eleven arguments). Here the arguments are read from the
// tensors directly and the output comes from the CUDA allocator without the dispatcher.
//
// The functions take exactly the positional arguments that ops.py passes. The entry points are those
// of the library that fluke_b200.lib has loaded: bind() receives their addresses, so both share one
// copy of its state (stream setting, last error, prepared weights). The interpreter lock is
// released around every entry point.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include <fluke/fluke.h>

namespace {

#define FLUKE_NATIVE_FUNCTIONS(X) \
    X(fluke_rmsnorm_gpu) X(fluke_rmsnorm_quant_int8_gpu) X(fluke_rmsnorm_quant_fp8_gpu) X(fluke_quant_int8_gpu) \
    X(fluke_quant_fp8_gpu) X(fluke_dequant_fp8_transpose_gpu) X(fluke_dequant_int8_transpose_gpu) X(fluke_rotary_emb_gpu) \
    X(fluke_silu_mul_gpu) X(fluke_flstm_step_gpu) X(fluke_qkv_rotary_i8_gpu) X(fluke_gated_mlp_i8_gpu) \
    X(fluke_qkv_rotary_fp8_gpu) X(fluke_gated_mlp_fp8_gpu) X(fluke_qkv_rotary_fp8_plain_gpu) \
    X(fluke_gated_mlp_fp8_plain_gpu) X(fluke_gemm_i8_gpu) X(fluke_gemm_fp8_gpu) X(fluke_down_proj_i8_gpu) \
    X(fluke_down_proj_fp8_gpu) X(fluke_factored_lstm_step_i8_gpu) X(fluke_factored_lstm_step_fp8_gpu) X(fluke_last_error) \
    X(fluke_fp4_scale_bytes) X(fluke_quant_mxfp4_gpu) X(fluke_quant_nvfp4_gpu) X(fluke_dequant_mxfp4_gpu) X(fluke_dequant_nvfp4_gpu) \
    X(fluke_gemm_mxfp4_gpu) X(fluke_gemm_nvfp4_gpu) X(fluke_gated_mlp_mxfp4_gpu) X(fluke_gated_mlp_nvfp4_gpu) X(fluke_rmsnorm_block_gpu) \
    X(fluke_linear_gpu) X(fluke_linear_recurrence_gpu) X(fluke_linear_recurrence_backward_gpu)

struct Entry {
#define X(name) decltype(&::name) name = nullptr;
    FLUKE_NATIVE_FUNCTIONS(X)
#undef X
} L;

struct Failed {};  // a Python error is set

const at::Tensor &tensor(PyObject *o) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "fluke_b200.ops needs torch tensors, got %s", Py_TYPE(o)->tp_name);
        throw Failed();
    }
    return THPVariable_Unpack(o);
}
// An input: on the GPU and contiguous, or None.
const at::Tensor *input(PyObject *o) {
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o);
    if (!t.is_cuda()) {
        PyErr_SetString(PyExc_RuntimeError, "fluke_b200.ops needs CUDA tensors (there is no CPU fallback)");
        throw Failed();
    }
    if (!t.is_contiguous()) {
        PyErr_SetString(PyExc_RuntimeError, "fluke_b200.ops needs contiguous tensors");
        throw Failed();
    }
    return &t;
}
const at::Tensor &required(PyObject *o) {
    const at::Tensor *t = input(o);
    if (!t) tensor(o);  // raises
    return *t;
}
// The same with the dimensions that the operator's sizes are read from.
const at::Tensor &required(PyObject *o, int64_t dims) {
    const at::Tensor &t = required(o);
    if (t.dim() != dims) {
        PyErr_Format(PyExc_ValueError, "fluke_b200.ops: a tensor of %lld dimensions where %lld are needed", (long long)t.dim(), (long long)dims);
        throw Failed();
    }
    return t;
}
void *ptr(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
void *ptr(const at::Tensor &t) { return t.data_ptr(); }
// Numbers and addresses are taken as ctypes takes them for the same C arguments: an int of any size
// by its low bits (the stride of a dimension of one element may be anything), a ctypes integer by its value,
// an address also as a ctypes pointer or array; a real number as float() converts it.
int integer(PyObject *o) {
    if (PyLong_Check(o)) return int(PyLong_AsUnsignedLongMask(o));
    PyObject *v = PyIndex_Check(o) ? PyNumber_Index(o) : PyObject_GetAttrString(o, "value");
    if (!v || !PyLong_Check(v)) {
        Py_XDECREF(v);
        PyErr_Format(PyExc_TypeError, "fluke_b200.ops: an integer is needed, got %s", Py_TYPE(o)->tp_name);
        throw Failed();
    }
    const int r = int(PyLong_AsUnsignedLongMask(v));
    Py_DECREF(v);
    return r;
}
void *address(PyObject *o) {
    if (o == Py_None) return nullptr;
    if (PyLong_Check(o)) return reinterpret_cast<void *>(uintptr_t(PyLong_AsUnsignedLongLongMask(o)));
    PyObject *ctypes = PyImport_ImportModule("ctypes");
    PyObject *type = ctypes ? PyObject_GetAttrString(ctypes, "c_void_p") : nullptr;
    PyObject *cast = type ? PyObject_CallMethod(ctypes, "cast", "OO", o, type) : nullptr;
    PyObject *v = cast ? PyObject_GetAttrString(cast, "value") : nullptr;
    void *p = v && v != Py_None ? PyLong_AsVoidPtr(v) : nullptr;
    const bool ok = v && !PyErr_Occurred();
    Py_XDECREF(v);
    Py_XDECREF(cast);
    Py_XDECREF(type);
    Py_XDECREF(ctypes);
    if (!ok) throw Failed();
    return p;
}
float real(PyObject *o) {
    if (PyFloat_Check(o)) return float(PyFloat_AS_DOUBLE(o));
    PyObject *v = PyNumber_Float(o);
    if (!v) throw Failed();
    const double r = PyFloat_AS_DOUBLE(v);
    Py_DECREF(v);
    return float(r);
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Failed();
    return v != 0;
}

// A new tensor on `like`'s device. On the current device (nearly always) without the device guard and the
// initialisation check of at::detail::empty_cuda: 0.40 instead of 0.53 us.
at::Tensor empty_on(const at::Tensor &like, at::IntArrayRef size, at::ScalarType type) {
    const at::Device device = like.device();
    if (device.index() != c10::cuda::current_device()) return at::detail::empty_cuda(size, type, device, c10::nullopt);
    return at::detail::empty_generic(size, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type,
                                     c10::nullopt);
}
// `o` as the output tensor, or a new one when it is None.
at::Tensor output(PyObject *o, const at::Tensor &like, at::IntArrayRef size, at::ScalarType type) {
    return o == Py_None ? empty_on(like, size, type) : tensor(o);
}

template <typename F>
auto unlocked(F f) {
    struct Release {
        PyThreadState *s = PyEval_SaveThread();
        ~Release() { PyEval_RestoreThread(s); }
    } r;
    return f();
}
void check(int rc, const char *what) {
    if (rc == 0) return;
    PyErr_SetString(PyExc_RuntimeError, (std::string(what) + " failed: rc=" + std::to_string(rc) + " " + L.fluke_last_error()).c_str());
    throw Failed();
}

PyObject *wrap(const at::Tensor &t) { return THPVariable_Wrap(t); }
PyObject *wrap(const at::Tensor &a, const at::Tensor &b) {
    PyObject *x = wrap(a), *y = wrap(b), *r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
}

using Args = PyObject *const *;

// Turns C++ errors into Python ones and checks the argument count.
template <PyObject *(*F)(Args), int N>
PyObject *entry(PyObject *, Args a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
        return nullptr;
    }
    if (!L.fluke_last_error) {
        PyErr_SetString(PyExc_RuntimeError, "fluke_b200._native: no library bound");
        return nullptr;
    }
    try {
        return F(a);
    } catch (const Failed &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ---- memory-bound kernels ------------------------------------------------------------------------

// x, residual, weight, alpha, eps, out
PyObject *rmsnorm(Args a) {
    const at::Tensor &x = required(a[0]);
    const at::Tensor *res = input(a[1]), *w = input(a[2]);
    const float alpha = real(a[3]), eps = real(a[4]);
    at::Tensor out = output(a[5], x, x.sizes(), x.scalar_type());
    unlocked([&] { L.fluke_rmsnorm_gpu(ptr(x), ptr(res), ptr(w), ptr(out), int(x.size(0)), int(x.size(1)), alpha, eps); });
    return wrap(out);
}

// x, weight, residual, residual_scale, alpha, eps, fp8
PyObject *rmsnorm_quant(Args a) {
    const at::Tensor &x = required(a[0]);
    const at::Tensor *w = input(a[1]), *res = input(a[2]), *scale = input(a[3]);
    const float alpha = real(a[4]), eps = real(a[5]);
    auto fn = truth(a[6]) ? L.fluke_rmsnorm_quant_fp8_gpu : L.fluke_rmsnorm_quant_int8_gpu;
    unlocked([&] { fn(ptr(x), ptr(w), ptr(res), ptr(scale), int(x.size(0)), int(x.size(1)), alpha, eps); });
    return PyTuple_Pack(2, a[2], a[3]);
}

// x, out, scale, fp8
PyObject *quant(Args a) {
    const at::Tensor &x = required(a[0]);
    const bool fp8 = truth(a[3]);
    at::Tensor out = output(a[1], x, x.sizes(), fp8 ? at::kByte : at::kChar);
    at::Tensor scale = output(a[2], x, {x.size(0)}, at::kFloat);
    auto fn = fp8 ? L.fluke_quant_fp8_gpu : L.fluke_quant_int8_gpu;
    unlocked([&] { fn(ptr(x), ptr(out), ptr(scale), int(x.size(0)), int(x.size(1))); });
    return wrap(out, scale);
}

// x, scale, fp8
PyObject *dequant_transpose(Args a) {
    const at::Tensor &x = required(a[0], 3);
    const float scale = real(a[1]);
    auto fn = truth(a[2]) ? L.fluke_dequant_fp8_transpose_gpu : L.fluke_dequant_int8_transpose_gpu;
    const int64_t t = x.size(0), n = x.size(1), c = x.size(2);
    at::Tensor out = empty_on(x, {n, t, c}, at::kHalf);
    unlocked([&] { fn(ptr(x), ptr(out), int(t), int(n), int(c), scale); });
    return wrap(out);
}

// x address, sin, cos, batch, seq_len, heads, head_dim, width, stride_batch, stride_seq, stride_head
PyObject *rotary_emb(Args a) {
    void *x = address(a[0]);
    const at::Tensor *sin = input(a[1]), *cos = input(a[2]);
    int v[8];
    for (int i = 0; i < 8; ++i) v[i] = integer(a[3 + i]);
    unlocked([&] { L.fluke_rotary_emb_gpu(x, ptr(sin), ptr(cos), v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]); });
    Py_RETURN_NONE;
}

// qkv, sin, cos, width
PyObject *rotary_qkv(Args a) {
    const at::Tensor &qkv = required(a[0], 5);
    const at::Tensor *sin = input(a[1]), *cos = input(a[2]);
    const int width = integer(a[3]);
    // The q and k heads lie side by side: one call rotates both. The strides follow from the sizes: those of
    // a contiguous tensor say nothing in a dimension of one element, and with one head q and k are two.
    const int64_t heads = qkv.size(3), head_dim = qkv.size(4), position = qkv.size(2) * heads * head_dim;
    unlocked([&] {
        L.fluke_rotary_emb_gpu(ptr(qkv), ptr(sin), ptr(cos), int(qkv.size(0)), int(qkv.size(1)), 2 * int(heads), int(head_dim),
                               width, int(qkv.size(1) * position), int(position), int(head_dim));
    });
    Py_INCREF(a[0]);
    return a[0];
}

// x
PyObject *silu_mul(Args a) {
    const at::Tensor &x = required(a[0]);
    const int64_t m = x.size(0), h = x.size(1) / 2;
    at::Tensor out = empty_on(x, {m, h}, x.scalar_type());
    unlocked([&] { L.fluke_silu_mul_gpu(ptr(x), ptr(out), int(m), int(h)); });
    return wrap(out);
}

// scratch, ih_t, cell, hh_next
PyObject *flstm_step(Args a) {
    const at::Tensor *scratch = input(a[0]), *ih = input(a[1]);
    const at::Tensor &cell = required(a[2]);
    at::Tensor out = output(a[3], cell, cell.sizes(), cell.scalar_type());
    unlocked([&] { L.fluke_flstm_step_gpu(ptr(scratch), ptr(ih), ptr(cell), ptr(out), int(cell.size(0)), int(cell.size(1))); });
    return wrap(out);
}

// ---- fused transformer kernels -------------------------------------------------------------------

// backend, a, w, scale_a, scale_b, sin, cos, seqlen, out, kind (0 int8, 1 fp8 pre-shuffled, 2 fp8 row-major), columns
PyObject *qkv_rotary(Args a) {
    void *backend = address(a[0]);
    const at::Tensor &x = required(a[1]);
    const at::Tensor *w = input(a[2]), *sa = input(a[3]), *sb = input(a[4]), *sin = input(a[5]), *cos = input(a[6]);
    const int seqlen = integer(a[7]), kind = integer(a[9]), m = int(x.size(0));
    at::Tensor out = output(a[8], x, {m, integer(a[10])}, at::kHalf);
    check(unlocked([&] {
              if (kind == 0)
                  return L.fluke_qkv_rotary_i8_gpu(static_cast<const fluke_int8_backend_t *>(backend), ptr(out), ptr(x), ptr(w),
                                                   ptr(sa), ptr(sb), ptr(sin), ptr(cos), m, seqlen);
              auto fn = kind == 1 ? L.fluke_qkv_rotary_fp8_gpu : L.fluke_qkv_rotary_fp8_plain_gpu;
              return fn(static_cast<const fluke_fp8_backend_t *>(backend), ptr(out), ptr(x), ptr(w), ptr(sa), ptr(sb), ptr(sin),
                        ptr(cos), m, seqlen);
          }),
          kind == 0 ? "fluke_qkv_rotary_i8_gpu" : "fluke_qkv_rotary_fp8_gpu");
    return wrap(out);
}

// backend, a, gate, up, scale_a, scale_gate, scale_up, out, kind (as above), columns
PyObject *gated_mlp(Args a) {
    void *backend = address(a[0]);
    const at::Tensor &x = required(a[1]);
    const at::Tensor *gate = input(a[2]), *up = input(a[3]), *sa = input(a[4]), *sg = input(a[5]), *su = input(a[6]);
    const int kind = integer(a[8]), m = int(x.size(0));
    at::Tensor out = output(a[7], x, {m, integer(a[9])}, at::kHalf);
    check(unlocked([&] {
              if (kind == 0)
                  return L.fluke_gated_mlp_i8_gpu(static_cast<const fluke_int8_backend_t *>(backend), ptr(out), ptr(x), ptr(gate),
                                                  ptr(up), ptr(sa), ptr(sg), ptr(su), m);
              auto fn = kind == 1 ? L.fluke_gated_mlp_fp8_gpu : L.fluke_gated_mlp_fp8_plain_gpu;
              return fn(static_cast<const fluke_fp8_backend_t *>(backend), ptr(out), ptr(x), ptr(gate), ptr(up), ptr(sa), ptr(sg),
                        ptr(su), m);
          }),
          kind == 0 ? "fluke_gated_mlp_i8_gpu" : "fluke_gated_mlp_fp8_gpu");
    return wrap(out);
}

// ---- plain GEMMs and the LSTM step ---------------------------------------------------------------

// a, b, scale_a, scale_b, const_scale_a
PyObject *gemm_i8(Args a) {
    const at::Tensor &x = required(a[0], 2), &w = required(a[1]);
    const at::Tensor *sa = input(a[2]), *sb = input(a[3]);
    const float csa = real(a[4]);
    const int m = int(x.size(0)), k = int(x.size(1)), n = int(w.size(0));
    at::Tensor out = empty_on(x, {m, n}, at::kHalf);
    check(unlocked([&] { return L.fluke_gemm_i8_gpu(ptr(out), ptr(x), ptr(w), ptr(sa), csa, ptr(sb), m, n, k); }), "fluke_gemm_i8_gpu");
    return wrap(out);
}

// a, b, scale_a, scale_b
PyObject *gemm_fp8(Args a) {
    const at::Tensor &x = required(a[0], 2), &w = required(a[1]);
    const at::Tensor *sa = input(a[2]), *sb = input(a[3]);
    const int m = int(x.size(0)), k = int(x.size(1)), n = int(w.size(0));
    at::Tensor out = empty_on(x, {m, n}, at::kHalf);
    check(unlocked([&] { return L.fluke_gemm_fp8_gpu(ptr(out), ptr(x), ptr(w), ptr(sa), ptr(sb), m, n, k); }), "fluke_gemm_fp8_gpu");
    return wrap(out);
}

// a, w, scale_a, scale_b, out, fp8
PyObject *down_proj(Args a) {
    const at::Tensor &x = required(a[0], 2), &w = required(a[1]);
    const at::Tensor *sa = input(a[2]), *sb = input(a[3]);
    const bool fp8 = truth(a[5]);
    const int m = int(x.size(0)), k = int(x.size(1)), n = int(w.size(0));
    at::Tensor out = output(a[4], x, {m, n}, at::kHalf);
    const int ld = int(out.stride(0));
    auto fn = fp8 ? L.fluke_down_proj_fp8_gpu : L.fluke_down_proj_i8_gpu;
    check(unlocked([&] { return fn(ptr(out), ld, ptr(x), ptr(w), ptr(sa), ptr(sb), m, n, k); }),
          fp8 ? "fluke_down_proj_fp8_gpu" : "fluke_down_proj_i8_gpu");
    return wrap(out);
}

// A, W4, bias4, c, h_out, fp8_export_name
PyObject *lstm_step(Args a) {
    const at::Tensor &x = required(a[0], 2), &w4 = required(a[1]), &b4 = required(a[2]), &c = required(a[3]);
    const int b = int(x.size(0)), kc = int(x.size(1)), h = int(c.size(1));
    at::Tensor out = output(a[4], x, {b, h}, at::kChar);
    const char *w = static_cast<const char *>(ptr(w4));
    const float *bias = static_cast<const float *>(ptr(b4));
    const size_t ws = size_t(h) * kc * 2;
    auto fn = truth(a[5]) ? L.fluke_factored_lstm_step_fp8_gpu : L.fluke_factored_lstm_step_i8_gpu;
    check(unlocked([&] {
              return fn(ptr(x), w, w + ws, w + 2 * ws, w + 3 * ws, bias, bias + h, bias + 2 * h, bias + 3 * h, ptr(c), ptr(out), b, h, kc);
          }),
          "fluke_factored_lstm_step_i8_gpu");
    return wrap(out);
}

// ---- microscaled 4-bit floating point -------------------------------------------------------------

template <typename... A>
[[noreturn]] void refuse(const char *format, A... a) {
    PyErr_Format(PyExc_ValueError, format, a...);
    throw Failed();
}
int small(int64_t v, const char *what) {
    if (v > INT32_MAX) refuse("fluke_b200.ops: %s of %lld", what, (long long)v);
    return int(v);
}
// 0 f16, 1 bf16 (FLUKE_F16, FLUKE_BF16)
int activation_type(at::ScalarType t) {
    if (t != at::kHalf && t != at::kBFloat16) refuse("fluke_b200.ops: float16 or bfloat16 is needed, got %s", c10::toString(t));
    return t == at::kBFloat16;
}
at::ScalarType out_type(PyObject *o) {
    if (!THPDtype_Check(o)) {
        PyErr_Format(PyExc_TypeError, "fluke_b200.ops: a torch.dtype is needed, got %s", Py_TYPE(o)->tp_name);
        throw Failed();
    }
    const at::ScalarType t = reinterpret_cast<THPDtype *>(o)->scalar_type;
    activation_type(t);
    return t;
}
// An argument that must have this type, these sizes and `like`'s device.
void expect(const at::Tensor &t, const char *what, at::ScalarType type, at::IntArrayRef size, const at::Tensor &like) {
    if (t.scalar_type() != type) refuse("fluke_b200.ops: %s is %s, %s is needed", what, c10::toString(t.scalar_type()), c10::toString(type));
    if (t.device() != like.device()) refuse("fluke_b200.ops: %s is on another device", what);
    bool same = t.dim() == int64_t(size.size());
    for (size_t i = 0; same && i < size.size(); ++i) same = t.size(i) == size[i];
    if (!same) refuse("fluke_b200.ops: %s has the wrong shape", what);
}
// A quantised matrix: codes [rows, cols / 2], block scales, and row scales in nvfp4.
struct Fp4 {
    const at::Tensor &codes, &scale;
    const at::Tensor *row;
    int rows, cols;
};
Fp4 fp4_matrix(PyObject *codes, PyObject *scale, PyObject *row, bool nv, const char *what, const at::Tensor *like) {
    const at::Tensor &c = required(codes, 2), &s = required(scale);
    const at::Tensor *r = nv ? &required(row) : nullptr;
    if (!nv && row != Py_None) refuse("fluke_b200.ops: row scales of %s, mxfp4 has none", what);
    const int64_t rows = c.size(0), cols = 2 * c.size(1), block = nv ? 16 : 32;
    if (!like) like = &c;
    expect(c, what, at::kByte, c.sizes(), *like);
    expect(s, "a block scale", at::kByte, {(rows + 127) / 128, (cols / block + 3) / 4, 512}, *like);
    if (nv) expect(*r, "a row scale", at::kFloat, {rows}, *like);
    if (cols % 32 != 0 || cols == 0) refuse("fluke_b200.ops: %s has %lld columns, a multiple of 32 is needed", what, (long long)cols);
    return {c, s, r, small(rows, "rows"), small(cols, "columns")};
}
at::Tensor new_scale(const at::Tensor &like, int64_t rows, int64_t cols, bool nv) {
    return empty_on(like, {(rows + 127) / 128, (cols / (nv ? 16 : 32) + 3) / 4, 512}, at::kByte);
}
// The calls run on the tensors' device, whichever is current.
template <typename F>
int on_device(const at::Tensor &like, F f) {
    c10::cuda::OptionalCUDAGuard guard;
    if (like.device().index() != c10::cuda::current_device()) guard.set_device(like.device());
    return unlocked(f);
}
PyObject *wrap_all(std::initializer_list<const at::Tensor *> list) {
    Py_ssize_t n = 0;
    for (auto t : list) n += t != nullptr;
    PyObject *r = PyTuple_New(n);
    Py_ssize_t i = 0;
    for (auto t : list) {
        if (!r || !t) continue;
        PyObject *o = wrap(*t);
        if (!o) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

// x, nv
PyObject *quant_fp4(Args a) {
    const at::Tensor &x = required(a[0], 2);
    const bool nv = truth(a[1]);
    const int type = activation_type(x.scalar_type()), m = small(x.size(0), "rows"), k = small(x.size(1), "columns");
    if (k % 32 != 0 || k == 0) refuse("fluke_b200.ops: %d columns, a multiple of 32 is needed", k);
    at::Tensor codes = empty_on(x, {m, k / 2}, at::kByte), scale = new_scale(x, m, k, nv), row;
    if (nv) row = empty_on(x, {m}, at::kFloat);
    check(on_device(x, [&] {
              return nv ? L.fluke_quant_nvfp4_gpu(ptr(x), ptr(codes), ptr(scale), ptr(row), m, k, type)
                        : L.fluke_quant_mxfp4_gpu(ptr(x), ptr(codes), ptr(scale), m, k, type);
          }),
          nv ? "fluke_quant_nvfp4_gpu" : "fluke_quant_mxfp4_gpu");
    return wrap_all({&codes, &scale, nv ? &row : nullptr});
}

// codes, scale, row_scale (mxfp4: None), dtype, nv
PyObject *dequant_fp4(Args a) {
    const bool nv = truth(a[4]);
    const Fp4 q = fp4_matrix(a[0], a[1], a[2], nv, "the codes", nullptr);
    const at::ScalarType dtype = out_type(a[3]);
    const int type = activation_type(dtype);
    at::Tensor out = empty_on(q.codes, {q.rows, q.cols}, dtype);
    check(on_device(q.codes, [&] {
              return nv ? L.fluke_dequant_nvfp4_gpu(ptr(q.codes), ptr(q.scale), ptr(q.row), ptr(out), q.rows, q.cols, type)
                        : L.fluke_dequant_mxfp4_gpu(ptr(q.codes), ptr(q.scale), ptr(out), q.rows, q.cols, type);
          }),
          nv ? "fluke_dequant_nvfp4_gpu" : "fluke_dequant_mxfp4_gpu");
    return wrap(out);
}

// a: codes, scale, row scale (mxfp4: None); b the same; up the same (not gated: three times None); dtype, nv, gated
PyObject *gemm_fp4(Args v) {
    const bool nv = truth(v[10]), gated = truth(v[11]);
    const at::ScalarType dtype = out_type(v[9]);
    const int type = activation_type(dtype);
    const Fp4 a = fp4_matrix(v[0], v[1], v[2], nv, "a", nullptr), b = fp4_matrix(v[3], v[4], v[5], nv, gated ? "gate" : "b", &a.codes);
    const Fp4 u = gated ? fp4_matrix(v[6], v[7], v[8], nv, "up", &a.codes) : b;
    const int m = a.rows, n = b.rows, k = a.cols;
    if (b.cols != k || u.cols != k) refuse("fluke_b200.ops: the matrices have %d, %d and %d columns", k, b.cols, u.cols);
    if (u.rows != n) refuse("fluke_b200.ops: gate has %d rows, up %d", n, u.rows);
    if (n % 8 != 0 || n == 0) refuse("fluke_b200.ops: a weight of %d rows, a multiple of 8 is needed", n);
    at::Tensor out = empty_on(a.codes, {m, n}, dtype);
    check(on_device(a.codes, [&] {
              if (gated)
                  return nv ? L.fluke_gated_mlp_nvfp4_gpu(ptr(out), ptr(a.codes), ptr(a.scale), ptr(a.row), ptr(b.codes), ptr(b.scale), ptr(b.row),
                                                          ptr(u.codes), ptr(u.scale), ptr(u.row), m, n, k, type)
                            : L.fluke_gated_mlp_mxfp4_gpu(ptr(out), ptr(a.codes), ptr(a.scale), ptr(b.codes), ptr(b.scale), ptr(u.codes),
                                                          ptr(u.scale), m, n, k, type);
              return nv ? L.fluke_gemm_nvfp4_gpu(ptr(out), ptr(a.codes), ptr(a.scale), ptr(a.row), ptr(b.codes), ptr(b.scale), ptr(b.row), m, n, k,
                                                 type)
                        : L.fluke_gemm_mxfp4_gpu(ptr(out), ptr(a.codes), ptr(a.scale), ptr(b.codes), ptr(b.scale), m, n, k, type);
          }),
          gated ? "fluke_gated_mlp_fp4_gpu" : "fluke_gemm_fp4_gpu");
    return wrap(out);
}

// x, residual, post_weight, gate, pre_weight, alpha, eps, seqlen, format (0: 16 bits), residual_out or None
PyObject *rmsnorm_block(Args a) {
    const at::Tensor &x = required(a[0], 2), &res = required(a[1]);
    const at::Tensor *post = input(a[2]), *gate = input(a[3]), *pre = input(a[4]);
    const int format = pre ? integer(a[8]) : 0, m = small(x.size(0), "rows"), k = small(x.size(1), "columns"), seqlen = integer(a[7]);
    const at::ScalarType type = x.scalar_type();
    if (k % 32 != 0 || k == 0) refuse("fluke_b200.ops: %d columns, a multiple of 32 is needed", k);
    if (seqlen < 0) refuse("fluke_b200.ops: a seqlen of %d", seqlen);
    fluke_rmsnorm_block_t b = {};
    b.dtype = activation_type(type);
    expect(res, "residual", type, {m, k}, x);
    if (post) expect(*post, "post_weight", type, {k}, x);
    if (pre) expect(*pre, "pre_weight", type, {k}, x);
    if (gate) {
        if (seqlen > 0) expect(*gate, "gate", type, {(int64_t(m) + seqlen - 1) / seqlen, k}, x);
        else if (gate->dim() == 1) expect(*gate, "gate", type, {k}, x);
        else expect(*gate, "gate", type, {1, k}, x);
    }
    at::Tensor stream = output(a[9], x, {m, k}, type), out, scale, row;
    if (a[9] != Py_None) {
        required(a[9]);
        expect(stream, "residual_out", type, {m, k}, x);
    }
    const bool fp4 = format == FLUKE_FP4_MX || format == FLUKE_FP4_NV, by_row = format != 0 && format != FLUKE_FP4_MX;
    if (pre) out = format == 0 ? empty_on(x, {m, k}, type) : fp4 ? empty_on(x, {m, k / 2}, at::kByte) : empty_on(x, {m, k}, format == FLUKE_ROW_INT8 ? at::kChar : at::kByte);
    if (fp4) scale = new_scale(x, m, k, format == FLUKE_FP4_NV);
    if (by_row) row = empty_on(x, {m}, at::kFloat);
    b.n_tokens = m; b.hidden_dim = k; b.seqlen = gate ? seqlen : 0;
    b.x = ptr(x); b.residual = ptr(res); b.post_weight = ptr(post); b.gate = ptr(gate); b.pre_weight = ptr(pre);
    b.alpha = real(a[5]); b.eps = real(a[6]);
    b.residual_out = ptr(stream);
    b.out_format = format;
    if (pre) b.out = ptr(out);
    if (fp4) b.scale = ptr(scale);
    if (by_row) b.row_scale = ptr(row);
    check(on_device(x, [&] { return L.fluke_rmsnorm_block_gpu(&b); }), "fluke_rmsnorm_block_gpu");
    return wrap_all({&stream, pre ? &out : nullptr, fp4 ? &scale : nullptr, by_row ? &row : nullptr});
}

// ---- 16-bit product with an epilogue, gated linear recurrence --------------------------------------

// A tensor on the GPU whose last dimension is dense, with this many dimensions.
const at::Tensor &rows_of(PyObject *o, const char *what, int64_t dims) {
    const at::Tensor &t = tensor(o);
    if (!t.is_cuda()) {
        PyErr_SetString(PyExc_RuntimeError, "fluke_b200.ops needs CUDA tensors (there is no CPU fallback)");
        throw Failed();
    }
    if (t.dim() != dims) refuse("fluke_b200.ops: %s has %lld dimensions, %lld are needed", what, (long long)t.dim(), (long long)dims);
    if (t.size(dims - 1) > 1 && t.stride(dims - 1) != 1) refuse("fluke_b200.ops: the rows of %s are not dense", what);
    return t;
}
// Distance between rows; one row has any.
long long pitch(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// x, weight, bias, activation, residual, alpha, out
PyObject *linear(Args a) {
    const at::Tensor &x = rows_of(a[0], "x", 2), &w = required(a[1], 2);
    const at::Tensor *bias = input(a[2]), *res = a[4] == Py_None ? nullptr : &rows_of(a[4], "residual", 2);
    const at::ScalarType type = x.scalar_type();
    fluke_linear_t l = {};
    l.dtype = activation_type(type);
    l.M = small(x.size(0), "rows"); l.K = small(x.size(1), "columns"); l.N = small(w.size(0), "columns");
    if (l.K % 8 != 0 || l.K == 0) refuse("fluke_b200.ops: rows of %d values, a multiple of 8 is needed", l.K);
    if (l.N % 8 != 0 || l.N == 0) refuse("fluke_b200.ops: a weight of %d rows, a multiple of 8 is needed", l.N);
    expect(w, "weight", type, {l.N, l.K}, x);
    if (bias) expect(*bias, "bias", type, {l.N}, x);
    if (res) expect(*res, "residual", type, {l.M, l.N}, x);
    at::Tensor out;
    if (a[6] == Py_None) {
        out = empty_on(x, {l.M, l.N}, type);
    } else {
        out = rows_of(a[6], "out", 2);
        expect(out, "out", type, {l.M, l.N}, x);
    }
    l.activation = integer(a[3]);
    l.x = ptr(x); l.weight = ptr(w); l.bias = ptr(bias); l.residual = ptr(res); l.out = ptr(out);
    l.ld_x = pitch(x); l.ld_residual = res ? pitch(*res) : 0; l.ld_out = pitch(out);
    l.alpha = real(a[5]);
    check(on_device(x, [&] { return L.fluke_linear_gpu(&l); }), "fluke_linear_gpu");
    return wrap(out);
}

// Strides of a tensor [T, B, H]; a dimension of one element has any.
long long step_of(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(2); }
long long chunk_of(const at::Tensor &t) { return t.size(1) > 1 ? t.stride(1) : t.size(2); }
// A new tensor [T, B, H] with the leading dimensions in `like`'s order.
at::Tensor new_steps(const at::Tensor &like) {
    const int64_t t = like.size(0), b = like.size(1), h = like.size(2);
    if (t > 1 && b > 1 && like.stride(1) > like.stride(0)) return empty_on(like, {b, t, h}, like.scalar_type()).transpose(0, 1);
    return empty_on(like, {t, b, h}, like.scalar_type());
}
const at::Tensor *state_of(PyObject *o, const char *what, const at::Tensor &like) {
    const at::Tensor *t = input(o);
    if (t) expect(*t, what, at::kFloat, {like.size(1), like.size(2)}, like);
    return t;
}
const at::Tensor *lengths_of(PyObject *o, const at::Tensor &like) {
    const at::Tensor *t = input(o);
    if (t) expect(*t, "lengths", at::kInt, {like.size(1)}, like);
    return t;
}
template <typename R>
void steps_of(R &r, const at::Tensor &gate, const at::Tensor &value) {
    r.dtype = activation_type(gate.scalar_type());
    r.T = small(gate.size(0), "steps"); r.B = small(gate.size(1), "chunks"); r.H = small(gate.size(2), "channels");
    if (r.H % 2 != 0) refuse("fluke_b200.ops: %d channels, an even number is needed", r.H);
    expect(value, "value", gate.scalar_type(), gate.sizes(), gate);
    r.gate = ptr(gate); r.value = ptr(value);
    r.gate_step = step_of(gate); r.gate_chunk = chunk_of(gate);
    r.value_step = step_of(value); r.value_chunk = chunk_of(value);
}

// gate, value, h0, lengths, reverse, save, out, h_last
PyObject *linear_recurrence(Args a) {
    const at::Tensor &gate = rows_of(a[0], "gate", 3), &value = rows_of(a[1], "value", 3);
    fluke_linear_recurrence_t r = {};
    steps_of(r, gate, value);
    const at::Tensor *h0 = state_of(a[2], "h0", gate), *lengths = lengths_of(a[3], gate);
    const bool save = truth(a[5]);
    at::Tensor out, last, states;
    if (a[6] == Py_None) {
        out = new_steps(value);
    } else {
        out = rows_of(a[6], "out", 3);
        expect(out, "out", gate.scalar_type(), gate.sizes(), gate);
    }
    if (a[7] == Py_None) last = empty_on(gate, {r.B, r.H}, at::kFloat);
    else {
        state_of(a[7], "h_last", gate);
        last = tensor(a[7]);
    }
    if (save) states = empty_on(gate, {(int64_t(r.T) + 15) / 16, r.B, r.H}, at::kFloat);
    r.reverse = truth(a[4]);
    r.out = ptr(out); r.out_step = step_of(out); r.out_chunk = chunk_of(out);
    r.lengths = ptr(lengths); r.h0 = ptr(h0); r.h_last = ptr(last);
    r.states = save ? ptr(states) : nullptr;
    check(on_device(gate, [&] { return L.fluke_linear_recurrence_gpu(&r); }), "fluke_linear_recurrence_gpu");
    return wrap_all({&out, &last, save ? &states : nullptr});
}

// grad, gate, value, states, grad_last, lengths, reverse
PyObject *linear_recurrence_backward(Args a) {
    const at::Tensor &grad = rows_of(a[0], "grad", 3), &gate = rows_of(a[1], "gate", 3), &value = rows_of(a[2], "value", 3), &states = required(a[3]);
    fluke_linear_recurrence_grad_t r = {};
    steps_of(r, gate, value);
    expect(grad, "grad", gate.scalar_type(), gate.sizes(), gate);
    expect(states, "states", at::kFloat, {(int64_t(r.T) + 15) / 16, r.B, r.H}, gate);
    const at::Tensor *grad_last = state_of(a[4], "grad_last", gate), *lengths = lengths_of(a[5], gate);
    at::Tensor dg = new_steps(gate), dv = new_steps(value), dh = empty_on(gate, {r.B, r.H}, at::kFloat);
    r.reverse = truth(a[6]);
    r.grad = ptr(grad); r.grad_step = step_of(grad); r.grad_chunk = chunk_of(grad);
    r.grad_gate = ptr(dg); r.grad_gate_step = step_of(dg); r.grad_gate_chunk = chunk_of(dg);
    r.grad_value = ptr(dv); r.grad_value_step = step_of(dv); r.grad_value_chunk = chunk_of(dv);
    r.lengths = ptr(lengths); r.states = ptr(states); r.grad_last = ptr(grad_last); r.grad_h0 = ptr(dh);
    check(on_device(gate, [&] { return L.fluke_linear_recurrence_backward_gpu(&r); }), "fluke_linear_recurrence_backward_gpu");
    return wrap_all({&dg, &dv, &dh});
}

// {name: address} of the loaded library's entry points
PyObject *bind(PyObject *, PyObject *dict) {
    Entry e;
    if (!PyDict_Check(dict)) return PyErr_Format(PyExc_TypeError, "bind() takes a dict of addresses");
#define X(name)                                                                                     \
    {                                                                                               \
        PyObject *v = PyDict_GetItemString(dict, #name);                                            \
        void *p = v ? PyLong_AsVoidPtr(v) : nullptr;                                                \
        if (!p) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_KeyError, "%s", #name);      \
        e.name = reinterpret_cast<decltype(e.name)>(p);                                             \
    }
    FLUKE_NATIVE_FUNCTIONS(X)
#undef X
    L = e;
    Py_RETURN_NONE;
}

PyObject *names(PyObject *, PyObject *) {
    PyObject *list = PyList_New(0);
#define X(name)                                         \
    if (list) {                                         \
        PyObject *s = PyUnicode_FromString(#name);      \
        if (s) PyList_Append(list, s);                  \
        Py_XDECREF(s);                                  \
    }
    FLUKE_NATIVE_FUNCTIONS(X)
#undef X
    return list;
}

#define FAST(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr}, {"names", names, METH_NOARGS, nullptr},
    FAST(rmsnorm, 6), FAST(rmsnorm_quant, 7), FAST(quant, 4), FAST(dequant_transpose, 3), FAST(rotary_emb, 11), FAST(rotary_qkv, 4),
    FAST(silu_mul, 1), FAST(flstm_step, 4), FAST(qkv_rotary, 11), FAST(gated_mlp, 10), FAST(gemm_i8, 5), FAST(gemm_fp8, 4),
    FAST(down_proj, 6), FAST(lstm_step, 6), FAST(quant_fp4, 2), FAST(dequant_fp4, 5), FAST(gemm_fp4, 12), FAST(rmsnorm_block, 10),
    FAST(linear, 7), FAST(linear_recurrence, 8), FAST(linear_recurrence_backward, 7), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__native() { return PyModule_Create(&module); }
