// native.cpp -- the Python front's way into the C ABI: CPython functions that take torch tensors,
// read their device addresses and the current stream, and make the call.
//
// What bounds it: an eager decode step is a handful of launches of a few microseconds each, so what the
// host spends in front of a launch is on the critical path.  Through ctypes an attend call of nine
// arguments cost 7 us before its first launch (tensor attribute look-ups, c_void_p objects, a Stream object,
// argument conversion); here the conversion of a call is a fraction of a microsecond.
//
// Every wrapper returns the C function's code as an int; ops.py turns a non-zero one into an exception.
// Integers wrap like ctypes' unsigned types do, None is a null pointer, a tensor has to be
// contiguous and on a CUDA device.  The interpreter lock is not held during a call that may block (a launch into a full
// queue, the synchronise at the end of `clear`): other Python threads go on, and a stream that waits for one of them
// gets there.  What torch throws on the way (a tensor without storage, no device) becomes the
// Python exception that torch itself would raise.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstring>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/tc_attn.h"

namespace {

tc_stream currentStream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// ---- one argument ---------------------------------------------------------------------------
bool toPointer(PyObject *o, void **out) {
    if (o == Py_None) {
        *out = nullptr;
        return true;
    }
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "tensor or None expected, got %s", Py_TYPE(o)->tp_name);
        return false;
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || !t.is_contiguous()) {
        PyErr_SetString(PyExc_AssertionError, "device-resident contiguous tensor required");
        return false;
    }
    *out = t.data_ptr();
    return true;
}
// the address alone (the batch descriptor's fields: layout is the caller's business there)
bool toAddress(PyObject *o, const void **out) {
    *out = nullptr;
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "tensor or None expected, got %s", Py_TYPE(o)->tp_name);
        return false;
    }
    *out = THPVariable_Unpack(o).data_ptr();
    return true;
}
template <typename T>
bool toArg(PyObject *o, T *out) {
    if constexpr (std::is_same_v<T, tc_kv_session *> || std::is_same_v<T, const tc_kv_session *>) {
        *out = static_cast<tc_kv_session *>(PyLong_AsVoidPtr(o));
    } else if constexpr (std::is_pointer_v<T>) {
        void *p = nullptr;
        if (!toPointer(o, &p)) return false;
        *out = static_cast<T>(p);
    } else if constexpr (std::is_floating_point_v<T>) {
        *out = static_cast<T>(PyFloat_AsDouble(o));
    } else {
        *out = static_cast<T>(PyLong_AsUnsignedLongLongMask(o));
    }
    return PyErr_Occurred() == nullptr;
}

// The C call itself, without the interpreter lock.
template <typename F>
auto unlocked(F &&call) {
    PyThreadState *const state = PyEval_SaveThread();
    const auto rc = call();
    PyEval_RestoreThread(state);
    return rc;
}

// ---- a C function int f(args..., tc_stream) as a Python function f(args...) -------------------
template <auto Fn>
struct Wrap;
template <typename... A, int (*Fn)(A...)>
struct Wrap<Fn> {
    static constexpr size_t kArgs = sizeof...(A) - 1;  // the stream is the current one
    template <size_t... I>
    static PyObject *call(PyObject *const *args, std::index_sequence<I...>) {
        std::tuple<A...> v;
        if (!(toArg(args[I], &std::get<I>(v)) && ...)) return nullptr;
        std::get<kArgs>(v) = currentStream();
        return PyLong_FromLong(unlocked([&] { return std::apply(Fn, v); }));
    }
    static PyObject *py(PyObject *, PyObject *const *args, Py_ssize_t n) {
        HANDLE_TH_ERRORS
        if (static_cast<size_t>(n) != kArgs) {
            PyErr_Format(PyExc_TypeError, "%zu arguments expected, got %zd", kArgs, n);
            return nullptr;
        }
        return call(args, std::make_index_sequence<kArgs>());
        END_HANDLE_TH_ERRORS
    }
};

// ---- the calls that need more than that -----------------------------------------------------------

// attend(session, slot, q, k, v, out, pos, dev_pos, graph_capture): the rows of the call are q's
PyObject *attend(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) {
        PyErr_SetString(PyExc_TypeError, "attend: 9 arguments expected");
        return nullptr;
    }
    tc_kv_session *s;
    uint32_t slot, pos;
    float *q, *out;
    const float *k, *v;
    const uint32_t *dev;
    int graph;
    if (!toArg(a[0], &s) || !toArg(a[1], &slot) || !toArg(a[2], &q) || !toArg(a[3], &k) || !toArg(a[4], &v) ||
        !toArg(a[5], &out) || !toArg(a[6], &pos) || !toArg(a[7], &dev))
        return nullptr;
    graph = PyObject_IsTrue(a[8]);
    if (graph < 0) return nullptr;
    if (a[2] == Py_None) {
        PyErr_SetString(PyExc_TypeError, "attend: q is required");
        return nullptr;
    }
    const uint32_t rows = static_cast<uint32_t>(THPVariable_Unpack(a[2]).size(0));
    const tc_stream st = currentStream();
    return PyLong_FromLong(unlocked([&] { return tc_kv_session_attend(s, slot, q, k, v, out, rows, pos, dev, graph, st); }));
    END_HANDLE_TH_ERRORS
}

// begin(session, n) -> position, or -code
PyObject *begin(PyObject *, PyObject *const *a, Py_ssize_t n) {
    tc_kv_session *s;
    uint32_t rows, pos = 0;
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "begin: 2 arguments expected");
        return nullptr;
    }
    if (!toArg(a[0], &s) || !toArg(a[1], &rows)) return nullptr;
    const int rc = tc_kv_session_begin(s, rows, &pos);
    return PyLong_FromLongLong(rc == TC_OK ? static_cast<long long>(pos) : -static_cast<long long>(rc));
}

// decode_i8_batch(q, k8, v8, ks, vs, out, pAcc, pM, pL, lens, rowBase, nextK8, nextV8, tickets, appendK,
//                 appendV, rowsPerSeq, totalRows, batch, nHeads, nKV, hd, maxLen, numChunks, invSqrt,
//                 partialsOnly, flags, prefetchRows) -> chunk slots used, or -code
PyObject *decodeI8Batch(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 28) {
        PyErr_SetString(PyExc_TypeError, "decode_i8_batch: 28 arguments expected");
        return nullptr;
    }
    const void *p[16];
    for (int i = 0; i < 16; ++i)
        if (!toAddress(a[i], &p[i])) return nullptr;
    tc_decode_i8_batch d;
    memset(&d, 0, sizeof(d));
    uint32_t used = 0;
    auto f = [&](int i) { return const_cast<float *>(static_cast<const float *>(p[i])); };
    d.q = f(0);
    d.k8 = static_cast<const int8_t *>(p[1]), d.v8 = static_cast<const int8_t *>(p[2]);
    d.ks = f(3), d.vs = f(4);
    d.out = f(5);
    d.pAcc = f(6), d.pM = f(7), d.pL = f(8);
    d.lens = static_cast<const uint32_t *>(p[9]);
    d.rowBase = static_cast<const uint64_t *>(p[10]);
    d.nextK8 = static_cast<const int8_t *>(p[11]), d.nextV8 = static_cast<const int8_t *>(p[12]);
    d.mergeTickets = const_cast<uint32_t *>(static_cast<const uint32_t *>(p[13]));
    d.appendK = f(14), d.appendV = f(15);
    if (!toArg(a[16], &d.rowsPerSeq) || !toArg(a[17], &d.totalRows) || !toArg(a[18], &d.batch) ||
        !toArg(a[19], &d.nHeads) || !toArg(a[20], &d.nKV) || !toArg(a[21], &d.hd) || !toArg(a[22], &d.maxLen) ||
        !toArg(a[23], &d.numChunks) || !toArg(a[24], &d.invSqrt) || !toArg(a[25], &d.partialsOnly) ||
        !toArg(a[26], &d.flags) || !toArg(a[27], &d.prefetchRows))
        return nullptr;
    d.chunksUsed = &used;
    const tc_stream st = currentStream();
    const int rc = unlocked([&] { return tc_attn_decode_i8_batch(&d, st); });
    return PyLong_FromLongLong(rc == TC_OK ? static_cast<long long>(used) : -static_cast<long long>(rc));
    END_HANDLE_TH_ERRORS
}

// The paged cache of a call, from its tensors: pools [pages][rows][kv heads][head_dim], tables int32 [batch][pages per sequence], and
// `like`, whose first dimension is the call's tokens.  What a layout or a type would make wrong is refused here; sizes are the library's to check.
bool pagedTensor(PyObject *o, const char *name, at::ScalarType type, int64_t dims, const at::Tensor **out, const at::Device *dev = nullptr) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: tensor expected, got %s", name, Py_TYPE(o)->tp_name);
        return false;
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || !t.is_contiguous()) {
        PyErr_Format(PyExc_AssertionError, "%s: device-resident contiguous tensor required", name);
        return false;
    }
    if (t.scalar_type() != type || t.dim() != dims) {
        PyErr_Format(PyExc_ValueError, "%s: %s of %lld dimensions expected", name, c10::toString(type), static_cast<long long>(dims));
        return false;
    }
    if (dev != nullptr && t.device() != *dev) {
        PyErr_Format(PyExc_ValueError, "%s: not on the device of the cache", name);
        return false;
    }
    *out = &t;
    return true;
}
struct Paged {
    tc_paged_kv c;
    at::Device dev = at::Device(at::kCUDA);
    bool fail(const char *text) {
        PyErr_SetString(PyExc_ValueError, text);
        return false;
    }
    bool same(const at::Tensor &t, std::initializer_list<int64_t> sizes, const char *name) {
        if (t.sizes() != at::IntArrayRef(sizes.begin(), sizes.size())) {
            PyErr_Format(PyExc_ValueError, "%s: another shape expected", name);
            return false;
        }
        return true;
    }
    // kc, vc, ks, vs, pages, lens, starts
    bool take(PyObject *const *a) {
        memset(&c, 0, sizeof(c));
        const at::Tensor *kc, *vc, *pages, *lens, *t;
        if (!THPVariable_Check(a[0])) return fail("the cache is a tensor");
        const auto type = THPVariable_Unpack(a[0]).scalar_type();
        if (type != at::kHalf && type != at::kChar) return fail("the cache is fp16 or int8");
        if (!pagedTensor(a[0], "k cache", type, 4, &kc)) return false;
        dev = kc->device();
        if (dev.index() != c10::cuda::current_device()) return fail("the cache is not on the current device");
        if (!pagedTensor(a[1], "v cache", type, 4, &vc, &dev) || !pagedTensor(a[4], "pages", at::kInt, 2, &pages, &dev) ||
            !pagedTensor(a[5], "lens", at::kInt, 1, &lens, &dev))
            return false;
        if (vc->sizes() != kc->sizes()) return fail("k and v caches of different shapes");
        if (lens->size(0) != pages->size(0)) return fail("lens and pages of different batches");
        for (const auto *x : {kc, pages})
            for (const int64_t n : x->sizes())
                if (n > 0x7fffffffll) return fail("a dimension of the cache is too long");
        c.kvI8 = type == at::kChar;
        if (c.kvI8) {
            for (int i = 2; i < 4; ++i) {
                if (!pagedTensor(a[i], i == 2 ? "ks" : "vs", at::kFloat, 3, &t, &dev) || !same(*t, {kc->size(0), kc->size(1), kc->size(2)}, "scales")) return false;
                (i == 2 ? c.ks : c.vs) = static_cast<float *>(t->data_ptr());
            }
        } else if (a[2] != Py_None || a[3] != Py_None) {
            return fail("scales belong to an int8 cache");
        }
        if (a[6] != Py_None) {
            if (!pagedTensor(a[6], "starts", at::kInt, 1, &t, &dev) || !same(*t, {lens->size(0) + 1}, "starts")) return false;
            c.starts = static_cast<const uint32_t *>(t->data_ptr());
        }
        c.k = kc->data_ptr(), c.v = vc->data_ptr();
        c.pages = static_cast<const int32_t *>(pages->data_ptr());
        c.lens = static_cast<const uint32_t *>(lens->data_ptr());
        c.numPages = static_cast<uint32_t>(kc->size(0)), c.pageRows = static_cast<uint32_t>(kc->size(1));
        c.nKV = static_cast<uint32_t>(kc->size(2)), c.hd = static_cast<uint32_t>(kc->size(3));
        c.batch = static_cast<uint32_t>(pages->size(0)), c.pagesPerSeq = static_cast<uint32_t>(pages->size(1));
        return true;
    }
    // a token array [tokens][heads (0: any)][hd]; the first one says how many tokens there are
    bool rows(PyObject *o, const char *name, at::ScalarType type, int64_t heads, bool first, const at::Tensor **out) {
        if (!pagedTensor(o, name, type, 3, out, &dev)) return false;
        const at::Tensor &t = **out;
        if (t.size(0) > 0x7fffffffll || t.size(1) > 0x7fffffffll) return fail("too many tokens or heads");
        if (first) c.tokens = static_cast<uint32_t>(t.size(0));
        return same(t, {first ? t.size(0) : static_cast<int64_t>(c.tokens), heads ? heads : t.size(1), static_cast<int64_t>(c.hd)}, name);
    }
    static bool halfOrFloat(PyObject *o, at::ScalarType *type) {
        *type = THPVariable_Check(o) ? THPVariable_Unpack(o).scalar_type() : at::kFloat;
        if (*type == at::kHalf || *type == at::kFloat) return true;
        PyErr_SetString(PyExc_ValueError, "f32 or fp16 expected");
        return false;
    }
};

// paged_write(kc, vc, ks, vs, pages, lens, starts, k, v, q, q_out, cosT, sinT)
PyObject *pagedWrite(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13) {
        PyErr_SetString(PyExc_TypeError, "paged_write: 13 arguments expected");
        return nullptr;
    }
    Paged p;
    const at::Tensor *k, *v, *q = nullptr, *qOut = nullptr, *cosT = nullptr, *sinT = nullptr;
    at::ScalarType outType = at::kFloat;
    if (!p.take(a) || !p.rows(a[7], "k", at::kFloat, p.c.nKV, true, &k) || !p.rows(a[8], "v", at::kFloat, p.c.nKV, false, &v)) return nullptr;
    if (a[9] != Py_None &&
        (!p.rows(a[9], "q", at::kFloat, 0, false, &q) || !Paged::halfOrFloat(a[10], &outType) || !p.rows(a[10], "q_out", outType, q->size(1), false, &qOut)))
        return nullptr;
    if ((a[11] == Py_None) != (a[12] == Py_None)) return p.fail("cosT and sinT come together"), nullptr;
    if (a[11] != Py_None) {
        if (!pagedTensor(a[11], "cosT", at::kFloat, 2, &cosT, &p.dev) || !pagedTensor(a[12], "sinT", at::kFloat, 2, &sinT, &p.dev) ||
            !p.same(*cosT, {cosT->size(0), static_cast<int64_t>(p.c.hd / 2)}, "cosT") || !p.same(*sinT, {cosT->size(0), cosT->size(1)}, "sinT"))
            return nullptr;
        if (cosT->size(0) > 0x7fffffffll) return p.fail("too many table rows"), nullptr;
    }
    auto f = [](const at::Tensor *t) { return t != nullptr ? static_cast<float *>(t->data_ptr()) : nullptr; };
    const tc_stream st = currentStream();
    return PyLong_FromLong(unlocked([&] {
        return tc_paged_kv_write(&p.c, f(k), f(v), f(q), qOut != nullptr ? qOut->data_ptr() : nullptr, outType == at::kHalf,
                                 q != nullptr ? static_cast<uint32_t>(q->size(1)) : 0u, f(cosT), f(sinT),
                                 cosT != nullptr ? static_cast<uint32_t>(cosT->size(0)) : 0u, st);
    }));
    END_HANDLE_TH_ERRORS
}

// paged_read(kc, vc, ks, vs, pages, lens, starts, k_out, v_out)
PyObject *pagedRead(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) {
        PyErr_SetString(PyExc_TypeError, "paged_read: 9 arguments expected");
        return nullptr;
    }
    Paged p;
    const at::Tensor *k, *v;
    at::ScalarType type;
    if (!p.take(a) || !Paged::halfOrFloat(a[7], &type) || !p.rows(a[7], "k_out", type, p.c.nKV, true, &k) ||
        !p.rows(a[8], "v_out", type, p.c.nKV, false, &v))
        return nullptr;
    const tc_stream st = currentStream();
    return PyLong_FromLong(unlocked([&] { return tc_paged_kv_read(&p.c, k->data_ptr(), v->data_ptr(), type == at::kHalf, st); }));
    END_HANDLE_TH_ERRORS
}

// attn_paged(kc, vc, ks, vs, pages, lens, starts, q, out, workspace, max_tokens, invSqrt)
PyObject *attnPaged(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12) {
        PyErr_SetString(PyExc_TypeError, "attn_paged: 12 arguments expected");
        return nullptr;
    }
    Paged p;
    const at::Tensor *q, *out, *ws;
    at::ScalarType type;
    uint32_t maxTokens;
    float invSqrt;
    if (!p.take(a) || !Paged::halfOrFloat(a[7], &type) || !p.rows(a[7], "q", type, 0, true, &q) || !p.rows(a[8], "out", type, q->size(1), false, &out) ||
        !pagedTensor(a[9], "workspace", at::kFloat, 1, &ws, &p.dev) || !toArg(a[10], &maxTokens))
        return nullptr;
    if (a[11] == Py_None) invSqrt = 1.0f / std::sqrt(static_cast<float>(p.c.hd));
    else if (!toArg(a[11], &invSqrt)) return nullptr;
    const tc_stream st = currentStream();
    return PyLong_FromLong(unlocked([&] {
        return tc_attn_paged(&p.c, q->data_ptr(), out->data_ptr(), type == at::kHalf, static_cast<uint32_t>(q->size(1)), maxTokens, invSqrt, ws->data_ptr(),
                             static_cast<size_t>(ws->numel()) * 4, st);
    }));
    END_HANDLE_TH_ERRORS
}

#define TC_FAST(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
#define TC_WRAP(name, fn) TC_FAST(name, Wrap<fn>::py)
PyMethodDef kMethods[] = {
        TC_FAST("attend", attend),
        TC_FAST("begin", begin),
        TC_FAST("decode_i8_batch", decodeI8Batch),
        TC_FAST("paged_write", pagedWrite),
        TC_FAST("paged_read", pagedRead),
        TC_FAST("attn_paged", attnPaged),
        TC_WRAP("clear", tc_kv_session_clear),
        TC_WRAP("kv_append", tc_kv_append),
        TC_WRAP("kv_append_rope", tc_kv_append_rope),
        TC_WRAP("rope_q", tc_rope_q),
        TC_WRAP("kv_quantize_i8", tc_kv_quantize_i8),
        TC_WRAP("kv_quantize_i8_batch", tc_kv_quantize_i8_batch),
        TC_WRAP("decode_i8", tc_attn_decode_i8),
        TC_WRAP("decode_i8_noalloc", tc_attn_decode_i8_noalloc),
        TC_WRAP("decode_kv", tc_attn_decode_kv),
        TC_WRAP("merge_partials", tc_attn_merge_partials),
        TC_WRAP("merge_gathered", tc_attn_merge_gathered),
        TC_WRAP("prefill_f16", tc_attn_prefill_f16),
        TC_WRAP("prefill_f16_kv8", tc_attn_prefill_f16_kv8),
        TC_WRAP("prefill_f16_kvhalf", tc_attn_prefill_f16_kvhalf),
        TC_WRAP("prefill_f16_i8", tc_attn_prefill_f16_i8),
        TC_WRAP("prefill_kv", tc_attn_prefill_kv),
        TC_WRAP("prefill_i8", tc_attn_prefill_i8),
        TC_WRAP("qk_norm_rope", tc_qk_norm_rope),
        TC_WRAP("sigmoid_gate", tc_attn_sigmoid_gate),
        {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", "Calls into libtc_attn.so with torch tensors.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
