// The launchers of include/llm_amd/kernels.h as functions of a CPython module (_launchers), called
// with the arguments of the Python wrappers of the same names: torch tensors (or raw addresses, or
// None), numbers and a stream. A call checks and unwraps its arguments, takes the current stream,
// launches with the GIL released and raises LlmError if the library recorded an error.
//
// Most launchers run 2-10 us on the GPU, less than the Python bindings needed to prepare one call:
// several Python attribute calls per tensor, ctypes conversions, the stream object, two calls for the
// error. Host time of a call, launches included: rmsnorm_forward 9.6 -> 3.4 us; the four calls of an
// attention block (five launches) 47.0 -> 15.8 us, so that at Qwen3-0.6B's widths and 260 positions a
// block takes 16.8 us instead of 40.8 (15.3 on the GPU); a small LM head with its argmax 19.6 -> 8.8.
//
// A call takes only what it recognises: exact torch tensors (no subclass) on the GPU, contiguous, of
// a 16-bit type where bf16 is expected; exact ints and floats in range. For anything else it returns
// False without having launched, and the Python wrapper goes its general way, which converts what it
// accepts and reports what it refuses.
#include <Python.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <limits.h>
#include <stddef.h>

#include <initializer_list>
#include <type_traits>
#include <utility>

#include "llm_amd/kernels.h"
#include "llm_amd/paged.h"

namespace {

PyObject *g_error = nullptr;  // LlmError, set by init

union Arg {
    void *p;
    int i;
    float f;
    size_t z;
};

// The device pointer of a tensor, a raw address or None.
bool take_pointer(PyObject *o, bool bits16, void *&out) {
    if (o == Py_None) {
        out = nullptr;
        return true;
    }
    if (PyLong_CheckExact(o)) {
        out = (void *)PyLong_AsUnsignedLongLongMask(o);
        return !PyErr_Occurred();
    }
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous()) return false;
    if (bits16 && t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kShort &&
        t.scalar_type() != at::kUInt16)
        return false;
    out = t.data_ptr();
    return true;
}

// A stream address, an object with one (torch.cuda.Stream), or None: torch's current stream.
bool take_stream(PyObject *o, void *&out) {
    if (o == Py_None) {
        out = c10::hip::getCurrentHIPStream().stream();
        return true;
    }
    if (PyLong_CheckExact(o)) {
        out = (void *)PyLong_AsUnsignedLongLongMask(o);
        return !PyErr_Occurred();
    }
    PyObject *address = PyObject_GetAttrString(o, "cuda_stream");
    if (!address) return false;
    const bool ok = PyLong_CheckExact(address);
    if (ok) out = (void *)PyLong_AsUnsignedLongLongMask(address);
    Py_DECREF(address);
    return ok && !PyErr_Occurred();
}

template <class T>
bool take(PyObject *o, Arg &a) {
    if constexpr (std::is_same_v<T, hipStream_t>) {
        return take_stream(o, a.p);
    } else if constexpr (std::is_pointer_v<T>) {
        return take_pointer(o, std::is_same_v<std::remove_cv_t<std::remove_pointer_t<T>>, bf16>, a.p);
    } else if constexpr (std::is_same_v<T, float>) {
        if (!PyFloat_CheckExact(o)) return false;
        a.f = (float)PyFloat_AS_DOUBLE(o);
        return true;
    } else {
        if (!PyLong_CheckExact(o)) return false;
        int overflow = 0;
        const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
        if (overflow) return false;
        if constexpr (std::is_same_v<T, size_t>) {
            a.z = (size_t)v;
            return v >= 0;
        } else {
            static_assert(std::is_same_v<T, int>, "argument type");
            a.i = (int)v;
            return v >= INT_MIN && v <= INT_MAX;
        }
    }
}

template <class T>
T value(const Arg &a) {
    if constexpr (std::is_pointer_v<T>)
        return (T)a.p;
    else if constexpr (std::is_same_v<T, float>)
        return a.f;
    else if constexpr (std::is_same_v<T, size_t>)
        return a.z;
    else
        return a.i;
}

// Workspace of the attention launchers: a tensor `att` holds the floats they need. (att is argument
// AT; the head count, head_dim and max_seq are arguments H, D and S.)
template <int AT, int H, int D, int S>
bool att_large_enough(PyObject *const *args, const Arg *v) {
    if (!THPVariable_CheckExact(args[AT])) return true;  // a raw address, checked by the library
    const at::Tensor &t = THPVariable_Unpack(args[AT]);
    return (size_t)t.numel() >= attention_workspace_floats(v[H].i, v[D].i, v[S].i);
}
bool no_check(PyObject *const *, const Arg *) { return true; }

// Launches with the GIL released; True, or LlmError if the library recorded an error.
template <class Launch>
PyObject *launched(Launch launch) {
    Py_BEGIN_ALLOW_THREADS
    launch();
    Py_END_ALLOW_THREADS
    if (const char *message = llm_last_error()) {
        PyErr_SetString(g_error, message);
        llm_clear_error();
        return nullptr;
    }
    Py_RETURN_TRUE;
}

template <class... T, size_t... I>
PyObject *launch(void (*fn)(T...), bool (*check)(PyObject *const *, const Arg *),
                 PyObject *const *args, Py_ssize_t n, std::index_sequence<I...>) {
    if (n != (Py_ssize_t)sizeof...(T)) Py_RETURN_FALSE;
    Arg v[sizeof...(T)];
    bool ok = false;
    try {
        ok = (take<T>(args[I], v[I]) && ...) && check(args, v);
    } catch (...) {  // the general way reports it
        ok = false;
    }
    if (!ok) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    return launched([&] { fn(value<T>(v[I])...); });
}

template <auto FN, auto CHECK, class... T>
PyObject *call(void (*)(T...), PyObject *const *args, Py_ssize_t n) {
    return launch<T...>(FN, CHECK, args, n, std::index_sequence_for<T...>{});
}

template <auto FN, auto CHECK = no_check>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return call<FN, CHECK>(FN, args, n);
}

// ---- the operators over pages: tensors alone, whose sizes and strides are read here ----

// A tensor on the current device.
const at::Tensor *tensor_here(PyObject *o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.get_device() != c10::hip::current_device())
        return nullptr;
    return &t;
}

bool bits16(const at::Tensor &t) {
    return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kShort || t.scalar_type() == at::kUInt16;
}

// A contiguous tensor of this shape and type (null where the type does not matter), or None.
template <class P>
bool take_dense(PyObject *o, const at::ScalarType *type, std::initializer_list<int64_t> shape, P *&out) {
    out = nullptr;
    if (o == Py_None) return true;
    const at::Tensor *t = tensor_here(o);
    if (!t || (type && t->scalar_type() != *type) || !t->is_contiguous() ||
        t->sizes() != at::IntArrayRef(shape.begin(), shape.size()))
        return false;
    out = (P *)t->data_ptr();
    return true;
}

constexpr at::ScalarType INT32 = at::kInt, FLOAT32 = at::kFloat, FLOAT64 = at::kDouble;

bool take_norm(PyObject *o, int dim, const bf16 *&out) {
    out = nullptr;
    if (o == Py_None) return true;
    const at::Tensor *t = tensor_here(o);
    return t && bits16(*t) && take_dense(o, nullptr, {dim}, out);
}

// Rows [n, heads, dim] of whole heads, contiguous within a row.
bool take_rows(PyObject *o, int64_t n, int64_t heads, int64_t dim, bf16 *&out, int64_t &stride) {
    const at::Tensor *t = tensor_here(o);
    if (!t || !bits16(*t) || t->dim() != 3 || t->size(0) != n || t->size(1) != heads || t->size(2) != dim ||
        t->stride(2) != 1 || (heads > 1 && t->stride(1) != dim))
        return false;
    out = (bf16 *)t->data_ptr();
    stride = n > 1 ? t->stride(0) : heads * dim;
    return true;
}

// key_cache, value_cache, page_table, q_start, kv_len
bool take_batch(PyObject *const *o, PagedBatch &b) {
    const at::Tensor *k = tensor_here(o[0]), *v = tensor_here(o[1]), *table = tensor_here(o[2]);
    if (!k || !v || !table || !bits16(*k) || !bits16(*v) || k->dim() != 4 || k->sizes() != v->sizes() ||
        k->strides() != v->strides() || k->stride(3) != 1 || table->dim() != 2)
        return false;
    int64_t strides[3];
    for (int i = 0; i < 3; i++) strides[i] = k->size(i) > 1 ? k->stride(i) : 0;
    const int64_t seqs = table->size(0), pages = table->size(1);
    if (k->size(0) > INT_MAX || k->size(1) > INT_MAX || k->size(2) > INT_MAX || k->size(3) > INT_MAX ||
        seqs > INT_MAX || pages > INT_MAX)
        return false;
    b = {(bf16 *)k->data_ptr(), (bf16 *)v->data_ptr(), strides[0], strides[1], strides[2], nullptr, nullptr, nullptr,
         (int)seqs, (int)k->size(0), (int)k->size(1), (int)pages, (int)k->size(2), (int)k->size(3)};
    return take_dense(o[2], &INT32, {seqs, pages}, b.page_table) && take_dense(o[3], &INT32, {seqs + 1}, b.q_start) &&
           take_dense(o[4], &INT32, {seqs}, b.kv_len);
}

// What `take` accepts of a call's arguments is launched; everything else, and what throws, goes the
// general way.
template <class Take, class Launch>
PyObject *take_and_launch(Take take_all, Launch launch) {
    bool ok = false;
    try {
        ok = take_all();
    } catch (...) {
        ok = false;
    }
    if (!ok) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    return launched(launch);
}

PyObject *native_qk_norm_rope_paged(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    bf16 *q_out, *q, *k, *v;
    const bf16 *qn, *kn;
    const double *inv_freq;
    PagedBatch b;
    Arg eps, scale, stream;
    int64_t n = 0, heads = 0, half = 0, strides[4];
    return take_and_launch(
        [&] {
            if (n_args != 16 || !take_batch(o + 7, b)) return false;
            const at::Tensor *rows = tensor_here(o[1]), *freq = tensor_here(o[6]);
            if (!rows || rows->dim() != 3 || !freq || freq->dim() != 1) return false;
            n = rows->size(0), heads = rows->size(1), half = freq->size(0);
            return n < INT_MAX && heads < INT_MAX && half < INT_MAX / 2 &&
                   take_rows(o[0], n, heads, b.head_dim, q_out, strides[0]) &&
                   take_rows(o[1], n, heads, b.head_dim, q, strides[1]) &&
                   take_rows(o[2], n, b.n_kv_heads, b.head_dim, k, strides[2]) &&
                   take_rows(o[3], n, b.n_kv_heads, b.head_dim, v, strides[3]) && take_norm(o[4], b.head_dim, qn) &&
                   take_norm(o[5], b.head_dim, kn) && take_dense(o[6], &FLOAT64, {half}, inv_freq) &&
                   take<float>(o[12], eps) && take<float>(o[13], scale) && PyBool_Check(o[14]) &&
                   take<hipStream_t>(o[15], stream);
        },
        [&] {
            qk_norm_rope_paged(q_out, q, k, v, qn, kn, inv_freq, &b, (int)n, (int)heads, 2 * (int)half,
                               o[14] == Py_True, eps.f, scale.f, strides[0], strides[1], strides[2], strides[3],
                               (hipStream_t)stream.p);
        });
}

PyObject *native_attention_paged_forward(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    bf16 *out, *q;
    float *ws = nullptr;
    PagedBatch b;
    Arg scale, max_q, max_kv, window, stream;
    int64_t n = 0, heads = 0, strides[2];
    return take_and_launch(
        [&] {
            if (n_args != 13 || !take_batch(o + 2, b)) return false;
            const at::Tensor *rows = tensor_here(o[1]);
            if (!rows || rows->dim() != 3) return false;
            n = rows->size(0), heads = rows->size(1);
            if (n >= INT_MAX || heads >= INT_MAX || !take_rows(o[0], n, heads, b.head_dim, out, strides[0]) ||
                !take_rows(o[1], n, heads, b.head_dim, q, strides[1]) || !take<float>(o[8], scale) ||
                !take<int>(o[9], max_q) || !take<int>(o[10], max_kv) || !take<int>(o[11], window) ||
                !take<hipStream_t>(o[12], stream))
                return false;
            if (llm_last_error()) return false;  // from an earlier call: the general way reports it
            const size_t need = attention_paged_workspace_floats((int)n, b.n_seqs, (int)heads, b.n_kv_heads,
                                                                 b.head_dim, max_q.i, max_kv.i);
            if (llm_last_error()) {  // the general way meets and reports it again
                llm_clear_error();
                return false;
            }
            size_t have = 0;
            if (o[7] != Py_None) {
                const at::Tensor *t = tensor_here(o[7]);
                if (!t || t->scalar_type() != at::kFloat || !t->is_contiguous()) return false;
                ws = (float *)t->data_ptr();
                have = (size_t)t->numel();
            }
            return have >= need;
        },
        [&] {
            attention_paged_forward(out, q, &b, ws, (int)n, (int)heads, max_q.i, max_kv.i, window.i, scale.f,
                                    strides[0], strides[1], (hipStream_t)stream.p);
        });
}

PyObject *native_logits_penalty_forward(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    bf16 *out = nullptr, *logits = nullptr;
    const int *tokens, *prompt_len, *token_len, *bias_tokens, *bias_len;
    const float *repetition, *frequency, *presence, *bias;
    const uint32_t *allowed;
    int64_t rows = 0, vocab = 0, strides[2], wide[3];
    Arg stream;
    return take_and_launch(
        [&] {
            if (n_args != 13) return false;
            for (int i = 0; i < 2; i++) {
                const at::Tensor *t = tensor_here(o[i]);
                if (!t || !bits16(*t) || t->dim() != 2 || (t->size(1) > 1 && t->stride(1) != 1) ||
                    (i && (t->size(0) != rows || t->size(1) != vocab)))
                    return false;
                rows = t->size(0), vocab = t->size(1);
                strides[i] = rows > 1 ? t->stride(0) : vocab;
                (i ? logits : out) = (bf16 *)t->data_ptr();
            }
            const int at[3] = {2, 8, 11};
            for (int i = 0; i < 3; i++) {
                const at::Tensor *t = o[at[i]] == Py_None ? nullptr : tensor_here(o[at[i]]);
                if (o[at[i]] != Py_None && (!t || t->dim() != 2)) return false;
                wide[i] = t ? t->size(1) : 0;
                if (wide[i] > INT_MAX) return false;
                if (i == 2 && t && t->scalar_type() != at::kInt && t->scalar_type() != at::kUInt32) return false;
            }
            return rows <= INT_MAX && vocab > 0 && vocab <= INT_MAX && take_dense(o[2], &INT32, {rows, wide[0]}, tokens) &&
                   take_dense(o[3], &INT32, {rows}, prompt_len) && take_dense(o[4], &INT32, {rows}, token_len) &&
                   take_dense(o[5], &FLOAT32, {rows}, repetition) && take_dense(o[6], &FLOAT32, {rows}, frequency) &&
                   take_dense(o[7], &FLOAT32, {rows}, presence) &&
                   take_dense(o[8], &INT32, {rows, wide[1]}, bias_tokens) &&
                   take_dense(o[9], &FLOAT32, {rows, wide[1]}, bias) && take_dense(o[10], &INT32, {rows}, bias_len) &&
                   take_dense(o[11], nullptr, {rows, wide[2]}, allowed) && take<hipStream_t>(o[12], stream);
        },
        [&] {
            logits_penalty_forward(out, logits, tokens, prompt_len, token_len, repetition, frequency, presence,
                                   bias_tokens, bias, bias_len, allowed, (int)rows, (int)vocab, (int)wide[0],
                                   (int)wide[1], (int)wide[2], strides[0], strides[1], (hipStream_t)stream.p);
        });
}

PyObject *init(PyObject *, PyObject *error) {
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    Py_RETURN_NONE;
}

#define LAUNCHER(NAME, ...) \
    {#NAME, (PyCFunction)(void *)entry<NAME, ##__VA_ARGS__>, METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    LAUNCHER(embedding_forward),
    LAUNCHER(rmsnorm_forward),
    LAUNCHER(gemv_forward),
    LAUNCHER(gemv_residual_forward),
    LAUNCHER(qkv_forward),
    LAUNCHER(gate_up_forward),
    LAUNCHER(rmsnorm_qkv_forward),
    LAUNCHER(rmsnorm_gemv_forward),
    LAUNCHER(rmsnorm_gate_up_forward),
    LAUNCHER(qk_norm_rope_forward),
    LAUNCHER(qk_norm_rope_rows),
    LAUNCHER(attention_forward, att_large_enough<4, 5, 7, 9>),
    LAUNCHER(attention_forward_noalloc),
    LAUNCHER(qk_norm_rope_attention_forward, att_large_enough<8, 10, 12, 15>),
    LAUNCHER(argmax_forward),
    LAUNCHER(sample_forward),
    LAUNCHER(swiglu_forward),
    {"qk_norm_rope_paged", (PyCFunction)(void *)native_qk_norm_rope_paged, METH_FASTCALL, nullptr},
    {"attention_paged_forward", (PyCFunction)(void *)native_attention_paged_forward, METH_FASTCALL, nullptr},
    {"logits_penalty_forward", (PyCFunction)(void *)native_logits_penalty_forward, METH_FASTCALL, nullptr},
    {"init", init, METH_O, "The exception class of library errors."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launchers", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__launchers(void) {
    PyObject *m = PyModule_Create(&module);
    // the torch whose tensors this reads: the package leaves the module alone under another
    if (m && PyModule_AddStringConstant(m, "TORCH_VERSION", TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
