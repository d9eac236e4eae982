// ops_module.cpp -- tie_b200._ops, the part of the Python binding of the operators
// over device memory that runs at every call: it reads the tensors (through the
// exchange interface that torch.Tensor publishes, no copies and no references kept),
// checks what the C entry points cannot see, and calls them. The same checks written
// in Python took 5 to 7 us a call, as long as the smaller operators run.
//
// Every function returns the entry point's status; what it refuses itself is a
// ValueError. tie_b200/ops.py has the signatures and their meaning.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/dlpack.h>

#include <climits>
#include <cmath>
#include <cstdint>

#include "tie_b200.h"

namespace {

constexpr int kHeadDim = 64;

PyTypeObject* tensor_type = nullptr;
const DLPackExchangeAPI* api = nullptr;
// the entry points, from the library that the package has loaded
decltype(&tie_page_plan) page_plan_fn = nullptr;
decltype(&tie_kv_store) kv_store_fn = nullptr;
decltype(&tie_attention_paged) attention_paged_fn = nullptr;
decltype(&tie_beam_select) beam_select_fn = nullptr;
decltype(&tie_kv_reorder) kv_reorder_fn = nullptr;
decltype(&tie_kv_store_q8) kv_store_q8_fn = nullptr;
decltype(&tie_kv_load) kv_load_fn = nullptr;
decltype(&tie_attention_shared) attention_shared_fn = nullptr;
decltype(&tie_quantize_q4) quantize_q4_fn = nullptr;
decltype(&tie_dequantize_q4) dequantize_q4_fn = nullptr;
decltype(&tie_matvec_q4) matvec_q4_fn = nullptr;
decltype(&tie_q4_bytes) q4_bytes_fn = nullptr;

// Thrown after a Python error has been set.
struct Refused {};

[[noreturn]] void wrong(const char* name, const char* what) {
    PyErr_Format(PyExc_ValueError, "%s: %s wanted", name, what);
    throw Refused{};
}

// One argument that is a tensor; its numbers live as long as the call's arguments.
struct Tensor {
    DLTensor t;
    const char* name;
    Tensor(const char* n, PyObject* o) : name(n) {
        if (!PyObject_TypeCheck(o, tensor_type)) wrong(n, "a torch tensor is");
        if (api->dltensor_from_py_object_no_sync(o, &t) != 0) {
            PyErr_Clear();
            wrong(n, "a dense torch tensor is");
        }
    }
    int device() const { return t.device.device_type == kDLCUDA ? t.device.device_id : -1; }
    bool is(uint8_t code, int bits) const { return t.dtype.code == code && t.dtype.bits == bits && t.dtype.lanes == 1; }
    int64_t numel() const {
        int64_t n = 1;
        for (int i = 0; i < t.ndim; ++i) n *= t.shape[i];
        return n;
    }
    bool contiguous() const {
        if (!t.strides) return true;
        int64_t want = 1;
        for (int i = t.ndim - 1; i >= 0; --i) {
            if (t.shape[i] == 0) return true;
            if (t.shape[i] != 1 && t.strides[i] != want) return false;
            want *= t.shape[i];
        }
        return true;
    }
    void* data() const { return static_cast<char*>(t.data) + t.byte_offset; }
};

int as_int(const char* name, PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw Refused{};
        PyErr_Clear();
        wrong(name, "an integer of 32 bits is");
    }
    if (v < INT_MIN || v > INT_MAX) wrong(name, "an integer of 32 bits is");
    return (int)v;
}
int as_int(const char* name, int64_t v) {
    if (v > INT_MAX) wrong(name, "fewer than 2^31 elements are");
    return (int)v;
}

// a contiguous int32 (or float32) tensor of at least n elements on `device`
template <typename E>
E* vector_of(const char* name, PyObject* o, int64_t n, int device) {
    const Tensor x(name, o);
    constexpr bool ints = sizeof(E) == 4 && E(0.5) == E(0);
    if (!x.is(ints ? (uint8_t)kDLInt : (uint8_t)kDLFloat, 32) || x.numel() < n || x.device() != device || !x.contiguous()) {
        PyErr_Format(PyExc_ValueError, "%s: a contiguous %s tensor of %lld elements on device %d is wanted", name,
                     ints ? "int32" : "float32", (long long)n, device);
        throw Refused{};
    }
    return static_cast<E*>(x.data());
}
int32_t* ints(const char* name, PyObject* o, int64_t n, int device) { return vector_of<int32_t>(name, o, n, device); }
int32_t* ints_or_none(const char* name, PyObject* o, int64_t n, int device) {
    return o == Py_None ? nullptr : ints(name, o, n, device);
}

// a float32 matrix of `width` columns whose rows are contiguous
struct Rows {
    float* p;
    int64_t rows;
    int ld;
    Rows(const char* name, PyObject* o, int64_t width, int device) {
        const Tensor x(name, o);
        if (!x.is(kDLFloat, 32) || x.t.ndim != 2 || x.device() != device) wrong(name, "a float32 matrix on the pool's device is");
        rows = x.t.shape[0];
        const int64_t w = x.t.shape[1], one = x.t.strides ? x.t.strides[1] : 1;
        int64_t step = x.t.strides ? x.t.strides[0] : w;
        if (w != width || (one != 1 && w > 1)) wrong(name, "one width with contiguous rows is");
        // (a row alone has no next one, so its stride means nothing, and two of them need not agree; one of a width that is
        // not whole groups of 4 keeps a stride that may be)
        if (rows <= 1 && (step < w || w % 4 == 0)) step = w;
        p = static_cast<float*>(x.data());
        ld = as_int(name, step);
        as_int(name, rows);
    }
};

// a pool's two tensors
struct Pool {
    void *k, *v;
    int format, n_pages, heads, layers, device;
    size_t layer_stride;
    // levels: 8-bit pages are taken too (with scales, below)
    Pool(PyObject* ko, PyObject* vo, bool levels = false) {
        const Tensor a("k_pages", ko), b("v_pages", vo);
        bool same = a.t.ndim == b.t.ndim && a.t.dtype.code == b.t.dtype.code && a.t.dtype.bits == b.t.dtype.bits &&
                    a.device() >= 0 && a.device() == b.device() && a.contiguous() && b.contiguous();
        for (int i = 0; same && i < a.t.ndim; ++i) same = a.t.shape[i] == b.t.shape[i];
        if (!same) wrong("k_pages and v_pages", "one shape, type and CUDA device, contiguous, are");
        if (a.is(kDLFloat, 32)) format = TIE_KV_F32;
        else if (a.is(kDLBfloat, 16)) format = TIE_KV_BF16;
        else if (levels && a.is(kDLInt, 8)) format = TIE_KV_INT8;
        else wrong("k_pages, v_pages", levels ? "float32, bfloat16 or int8 is" : "float32 or bfloat16 is");
        const int64_t* s = a.t.shape + (a.t.ndim == 4);
        if ((a.t.ndim != 3 && a.t.ndim != 4) || s[1] != KV_CACHE_PAGE_ROWS || s[2] % kHeadDim)
            wrong("k_pages, v_pages", "[n_pages, 16, n_kv_head * 64] is");
        layers = a.t.ndim == 4 ? as_int("k_pages", a.t.shape[0]) : 1;
        n_pages = as_int("k_pages", s[0]);
        heads = as_int("k_pages", s[2] / kHeadDim);
        layer_stride = (size_t)(s[0] * s[1] * s[2]);
        device = a.device();
        k = a.data();
        v = b.data();
    }
    void one_layer() const {
        if (layers != 1) wrong("k_pages, v_pages", "one layer is");
    }
};

// the scales of a pool in 8 bits, or none for one that is not
struct Scales {
    float *k = nullptr, *v = nullptr;
    Scales(const Pool& pool, PyObject* ko, PyObject* vo) {
        pool.one_layer();
        if (pool.format != TIE_KV_INT8) {
            if (ko != Py_None || vo != Py_None) wrong("k_scales, v_scales", "int8 pages are");
            return;
        }
        k = one(pool, "k_scales", ko);
        v = one(pool, "v_scales", vo);
    }
    static float* one(const Pool& pool, const char* name, PyObject* o) {
        if (o == Py_None) wrong(name, "a scale per row and head (int8 pages) is");
        const Tensor x(name, o);
        if (!x.is(kDLFloat, 32) || x.t.ndim != 3 || x.t.shape[0] != pool.n_pages || x.t.shape[1] != pool.heads ||
            x.t.shape[2] != KV_CACHE_PAGE_ROWS || !x.contiguous() || x.device() != pool.device)
            wrong(name, "a contiguous float32 [n_pages, n_kv_head, 16] on the pool's device is");
        return static_cast<float*>(x.data());
    }
};

struct Table {
    int32_t* p;
    int n_seq, width, device;
    // any: on the device that the table itself is on
    Table(PyObject* o, int on, bool any = false, const char* name = "page_table") {
        const Tensor x(name, o);
        device = x.device();
        if (!x.is(kDLInt, 32) || x.t.ndim != 2 || !x.contiguous() || device < 0 || (!any && device != on))
            wrong(name, "a contiguous int32 [n_seq, pages_per_seq] on the pool's device is");
        p = static_cast<int32_t*>(x.data());
        n_seq = as_int(name, x.t.shape[0]);
        width = as_int(name, x.t.shape[1]);
    }
};

struct Workspace {
    void* p;
    size_t bytes;
    Workspace(PyObject* o, int device) {
        const Tensor x("workspace", o);
        if (!x.contiguous() || x.device() != device) wrong("workspace", "a contiguous tensor on the pool's device is");
        p = x.data();
        bytes = (size_t)x.numel() * (x.t.dtype.bits * x.t.dtype.lanes / 8);
    }
};

// the stream given, or torch's current one of the device
void* stream_of(PyObject* o, int device) {
    if (o != Py_None) {
        const unsigned long long v = PyLong_AsUnsignedLongLong(o);
        if (v == (unsigned long long)-1 && PyErr_Occurred()) throw Refused{};
        return reinterpret_cast<void*>((uintptr_t)v);
    }
    void* st = nullptr;
    if (api->current_work_stream(kDLCUDA, device, &st) != 0) throw Refused{};
    return st;
}

// Runs body() (which returns a status) as a Python function of exactly n arguments.
template <typename Body>
PyObject* guarded(Py_ssize_t given, Py_ssize_t n, const Body& body) {
    if (!api) {
        PyErr_SetString(PyExc_RuntimeError, "tie_b200._ops: init() has not been called");
        return nullptr;
    }
    if (given != n) {
        PyErr_Format(PyExc_TypeError, "%zd arguments are wanted, not %zd", n, given);
        return nullptr;
    }
    try {
        return PyLong_FromLong(body());
    } catch (const Refused&) {
        return nullptr;
    }
}

// The call itself: other Python threads may run meanwhile.
template <typename Call>
long unlocked(const Call& call) {
    model_status rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call();
    Py_END_ALLOW_THREADS
    return (long)rc;
}

// ctx_lens, new_lens, page_table, n_pages, row_start, seq_of, pos_of, slot_of, status,
// free_pages, n_free, n_free_out, stream
PyObject* page_plan(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 13, [&] {
        const Table table(v[2], 0, true);
        const int d = table.device, n_pages = as_int("n_pages", v[3]);
        const int rows = as_int("seq_of", Tensor("seq_of", v[5]).numel());
        int32_t *ctx = ints("ctx_lens", v[0], table.n_seq, d), *fresh = ints("new_lens", v[1], table.n_seq, d);
        int32_t* start = ints("row_start", v[4], (int64_t)table.n_seq + 1, d);
        int32_t *seq = ints("seq_of", v[5], rows, d), *pos = ints("pos_of", v[6], rows, d);
        int32_t *slot = ints("slot_of", v[7], rows, d), *status = ints("status", v[8], 1, d);
        int32_t* pages = ints_or_none("free_pages", v[9], 0, d);
        const int max_free = pages || v[9] != Py_None ? as_int("free_pages", Tensor("free_pages", v[9]).numel()) : 0;
        int32_t *n_free = ints_or_none("n_free", v[10], 1, d), *out = ints_or_none("n_free_out", v[11], 1, d);
        void* st = stream_of(v[12], d);
        return unlocked([&] {
            return page_plan_fn(ctx, fresh, table.n_seq, table.p, table.width, n_pages, pages, max_free, n_free, out, start,
                                seq, pos, slot, rows, status, st);
        });
    });
}

// k, v, slots, k_pages, v_pages, stream
PyObject* kv_store(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 6, [&] {
        const Pool pool(v[3], v[4]);
        pool.one_layer();
        const int64_t w = (int64_t)pool.heads * kHeadDim;
        const Rows a("k", v[0], w, pool.device), b("v", v[1], w, pool.device);
        if (a.rows != b.rows || a.ld != b.ld) wrong("k and v", "one shape and row stride is");
        int32_t* slots = ints("slots", v[2], a.rows, pool.device);
        void* st = stream_of(v[5], pool.device);
        return unlocked([&] {
            return kv_store_fn(a.p, b.p, a.ld, slots, (int)a.rows, pool.k, pool.v, pool.format, pool.n_pages, pool.heads, st);
        });
    });
}

// q, k_pages, v_pages, page_table, row_start, ctx_lens, max_new, out, workspace, scale,
// status, stream
PyObject* attention_paged(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        const Pool pool(v[1], v[2]);
        pool.one_layer();
        const int d = pool.device;
        const Table table(v[3], d);
        const Tensor qt("q", v[0]);
        const int64_t w = qt.t.ndim == 2 ? qt.t.shape[1] : -1;
        if (w < 0 || w % kHeadDim) wrong("q and out", "one shape [rows, n_head * 64] is");
        const Rows q("q", v[0], w, d), out("out", v[7], w, d);
        if (q.rows != out.rows) wrong("q and out", "one shape [rows, n_head * 64] is");
        int32_t* start = ints("row_start", v[4], (int64_t)table.n_seq + 1, d);
        int32_t* ctx = ints("ctx_lens", v[5], table.n_seq, d);
        const int max_new = as_int("max_new", v[6]);
        const Workspace ws(v[8], d);
        const double scale = PyFloat_AsDouble(v[9]);
        if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
        int32_t* status = ints_or_none("status", v[10], 1, d);
        void* st = stream_of(v[11], d);
        return unlocked([&] {
            return attention_paged_fn(q.p, q.ld, (int)(w / kHeadDim), pool.k, pool.v, pool.format, pool.n_pages, pool.heads,
                                      table.p, table.width, start, ctx, table.n_seq, max_new, (int)q.rows, (float)scale,
                                      out.p, out.ld, ws.p, ws.bytes, status, st);
        });
    });
}

// logits, scores, beams, next_ids, parent, scores_out, workspace, done, done_out, eos_id, stream
PyObject* beam_select(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        const Tensor lt("logits", v[0]);
        const int d = lt.device(), beams = as_int("beams", v[2]), eos = as_int("eos_id", v[9]);
        if (lt.t.ndim != 2 || beams <= 0 || lt.t.shape[0] % beams || d < 0)
            wrong("logits", "n_req * beams rows on a CUDA device are");
        const Rows logits("logits", v[0], lt.t.shape[1], d);
        const int vocab = as_int("logits", lt.t.shape[1]);
        float *scores = vector_of<float>("scores", v[1], logits.rows, d), *sout = vector_of<float>("scores_out", v[5], logits.rows, d);
        int32_t *next = ints("next_ids", v[3], logits.rows, d), *parent = ints("parent", v[4], logits.rows, d);
        int32_t *done = ints_or_none("done", v[7], logits.rows, d), *dout = ints_or_none("done_out", v[8], logits.rows, d);
        const Workspace ws(v[6], d);
        void* st = stream_of(v[10], d);
        return unlocked([&] {
            return beam_select_fn(logits.p, logits.ld, scores, done, (int)(logits.rows / beams), beams, vocab, eos, next,
                                  parent, sout, dout, ws.p, ws.bytes, st);
        });
    });
}

// k_pages, v_pages, page_table, parent, first, length, beams, stream
PyObject* kv_reorder(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const Pool pool(v[0], v[1]);
        const int d = pool.device, beams = as_int("beams", v[6]);
        const Table table(v[2], d);
        if (beams <= 0 || table.n_seq % beams) wrong("page_table", "n_req * beams sequences are");
        const int req = table.n_seq / beams;
        int32_t* parent = ints("parent", v[3], table.n_seq, d);
        int32_t *first = ints("first", v[4], req, d), *length = ints("length", v[5], req, d);
        void* st = stream_of(v[7], d);
        return unlocked([&] {
            return kv_reorder_fn(pool.k, pool.v, pool.format, pool.layers, pool.layer_stride, pool.n_pages, pool.heads,
                                 table.p, table.width, parent, first, length, req, beams, st);
        });
    });
}

// k, v, slots, k_pages, v_pages, k_scales, v_scales, stream
PyObject* kv_store_q8(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const Pool pool(v[3], v[4], true);
        if (pool.format != TIE_KV_INT8) wrong("k_pages, v_pages", "int8 is");
        const Scales sc(pool, v[5], v[6]);
        const int64_t w = (int64_t)pool.heads * kHeadDim;
        const Rows a("k", v[0], w, pool.device), b("v", v[1], w, pool.device);
        if (a.rows != b.rows || a.ld != b.ld) wrong("k and v", "one shape and row stride is");
        int32_t* slots = ints("slots", v[2], a.rows, pool.device);
        void* st = stream_of(v[7], pool.device);
        return unlocked([&] {
            return kv_store_q8_fn(a.p, b.p, a.ld, slots, (int)a.rows, pool.k, pool.v, sc.k, sc.v, pool.n_pages, pool.heads, st);
        });
    });
}

// slots, k_pages, v_pages, k_out, v_out, k_scales, v_scales, stream
PyObject* kv_load(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const Pool pool(v[1], v[2], true);
        const Scales sc(pool, v[5], v[6]);
        const int64_t w = (int64_t)pool.heads * kHeadDim;
        const Rows a("k_out", v[3], w, pool.device), b("v_out", v[4], w, pool.device);
        if (a.rows != b.rows || a.ld != b.ld) wrong("k_out and v_out", "one shape and row stride is");
        int32_t* slots = ints("slots", v[0], a.rows, pool.device);
        void* st = stream_of(v[7], pool.device);
        return unlocked([&] {
            return kv_load_fn(slots, (int)a.rows, pool.k, pool.v, sc.k, sc.v, pool.format, pool.n_pages, pool.heads, a.p, b.p,
                              a.ld, st);
        });
    });
}

// q, k_pages, v_pages, page_table, row_start, ctx_lens, max_new, out, workspace, k_scales, v_scales,
// prefix_table, prefix_lens, group_start, scale, status, stream
PyObject* attention_shared(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 17, [&] {
        const Pool pool(v[1], v[2], true);
        const Scales sc(pool, v[9], v[10]);
        const int d = pool.device;
        const Table table(v[3], d);
        const Tensor qt("q", v[0]);
        const int64_t w = qt.t.ndim == 2 ? qt.t.shape[1] : -1;
        if (w < 0 || w % kHeadDim) wrong("q and out", "one shape [rows, n_head * 64] is");
        const Rows q("q", v[0], w, d), out("out", v[7], w, d);
        if (q.rows != out.rows) wrong("q and out", "one shape [rows, n_head * 64] is");
        int32_t* start = ints("row_start", v[4], (int64_t)table.n_seq + 1, d);
        int32_t* ctx = ints("ctx_lens", v[5], table.n_seq, d);
        const int max_new = as_int("max_new", v[6]);
        const Workspace ws(v[8], d);
        int32_t *prefix = nullptr, *lens = nullptr, *groups = nullptr;
        int n_group = 0, prefix_width = 0;
        if (v[11] != Py_None) {
            const Table t(v[11], d, false, "prefix_table");
            prefix = t.p;
            prefix_width = t.width;
            n_group = t.n_seq;
            if (n_group <= 0) wrong("prefix_table", "a row for each group is");
            lens = ints("prefix_lens", v[12], n_group, d);
            groups = ints("group_start", v[13], (int64_t)n_group + 1, d);
        } else if (v[12] != Py_None || v[13] != Py_None) {
            wrong("prefix_table", "a table beside prefix_lens and group_start is");
        }
        const double scale = PyFloat_AsDouble(v[14]);
        if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
        int32_t* status = ints_or_none("status", v[15], 1, d);
        void* st = stream_of(v[16], d);
        return unlocked([&] {
            return attention_shared_fn(q.p, q.ld, (int)(w / kHeadDim), pool.k, pool.v, sc.k, sc.v, pool.format, pool.n_pages,
                                       pool.heads, table.p, table.width, start, ctx, table.n_seq, max_new, (int)q.rows, prefix,
                                       prefix_width, lens, groups, n_group, (float)scale, out.p, out.ld, ws.p, ws.bytes, status,
                                       st);
        });
    });
}

// The levels and scales of 4-bit weights of n rows of k.
struct Q4 {
    void *packed, *scales;
    int n, k, group, device;
    Q4(PyObject* po, PyObject* so, PyObject* go, int64_t columns) {
        const Tensor p("packed", po), s("scales", so);
        group = as_int("group", go);
        if (group != 32 && group != 64 && group != 128) wrong("group", "32, 64 or 128 is");
        device = p.device();
        k = as_int("k", columns);
        if (p.t.ndim != 2 || !p.is(kDLUInt, 8) || !p.contiguous() || device < 0 || k <= 0 || p.t.shape[0] <= 0 ||
            (size_t)p.t.shape[1] != q4_bytes_fn(1, k))
            wrong("packed", "a contiguous uint8 [n, 64 ceil(k / 128)] on a CUDA device is");
        n = as_int("packed", p.t.shape[0]);
        if (s.t.ndim != 2 || !s.is(kDLBfloat, 16) || !s.contiguous() || s.device() != device || s.t.shape[0] != n ||
            s.t.shape[1] != (k + (int64_t)group - 1) / group)
            wrong("scales", "a contiguous bfloat16 [n, ceil(k / group)] beside packed is");
        packed = p.data();
        scales = s.data();
    }
};
int64_t columns_of(const char* name, PyObject* o) {
    const Tensor x(name, o);
    if (x.t.ndim != 2) wrong(name, "a float32 matrix is");
    return x.t.shape[1];
}

// w, packed, scales, group, stream
PyObject* quantize_q4(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 5, [&] {
        const Q4 z(v[1], v[2], v[3], columns_of("w", v[0]));
        const Rows w("w", v[0], z.k, z.device);
        if (w.rows != z.n) wrong("w and packed", "one number of rows is");
        void* st = stream_of(v[4], z.device);
        return unlocked([&] { return quantize_q4_fn(w.p, w.ld, z.n, z.k, z.group, z.packed, z.scales, st); });
    });
}

// packed, scales, group, w, stream
PyObject* dequantize_q4(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 5, [&] {
        const Q4 z(v[0], v[1], v[2], columns_of("w", v[3]));
        const Rows w("w", v[3], z.k, z.device);
        if (w.rows != z.n) wrong("w and packed", "one number of rows is");
        void* st = stream_of(v[4], z.device);
        return unlocked([&] { return dequantize_q4_fn(z.packed, z.scales, z.n, z.k, z.group, w.p, w.ld, st); });
    });
}

// x, packed, scales, group, y, bias, residual, gelu, stream
PyObject* matvec_q4(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 9, [&] {
        const Q4 z(v[1], v[2], v[3], columns_of("x", v[0]));
        const Rows x("x", v[0], z.k, z.device), y("y", v[4], z.n, z.device);
        if (x.rows != y.rows) wrong("x and y", "one number of rows is");
        float* bias = v[5] == Py_None ? nullptr : vector_of<float>("bias", v[5], z.n, z.device);
        float* residual = nullptr;
        int ldr = 0;
        if (v[6] != Py_None) {
            const Rows r("residual", v[6], z.n, z.device);
            if (r.rows != y.rows) wrong("residual and y", "one shape is");
            residual = r.p;
            ldr = r.ld;
        }
        const int gelu = PyObject_IsTrue(v[7]);
        if (gelu < 0) throw Refused{};
        void* st = stream_of(v[8], z.device);
        return unlocked([&] {
            return matvec_q4_fn(x.p, x.ld, (int)x.rows, z.packed, z.scales, z.n, z.k, z.group, bias, residual, ldr, gelu, y.p,
                                y.ld, st);
        });
    });
}

// torch.Tensor, its exchange interface, the addresses of the entry points in the order below
PyObject* init(PyObject*, PyObject* const* v, Py_ssize_t n) {
    constexpr Py_ssize_t kFns = 12;
    if (n != 2 + kFns || !PyType_Check(v[0])) {
        PyErr_SetString(PyExc_TypeError, "torch.Tensor, its exchange interface and the entry points' addresses are wanted");
        return nullptr;
    }
    const auto* got = static_cast<const DLPackExchangeAPI*>(PyCapsule_GetPointer(v[1], "dlpack_exchange_api"));
    if (!got) return nullptr;
    if (got->header.version.major != DLPACK_MAJOR_VERSION || !got->dltensor_from_py_object_no_sync ||
        !got->current_work_stream) {
        PyErr_SetString(PyExc_ImportError, "tie_b200._ops was built for another version of torch's tensors");
        return nullptr;
    }
    void* at[kFns];
    for (int i = 0; i < kFns; ++i)
        if (!(at[i] = PyLong_AsVoidPtr(v[2 + i]))) return PyErr_Occurred() ? nullptr : (PyErr_SetString(PyExc_ValueError, "address"), nullptr);
    page_plan_fn = reinterpret_cast<decltype(page_plan_fn)>(at[0]);
    kv_store_fn = reinterpret_cast<decltype(kv_store_fn)>(at[1]);
    attention_paged_fn = reinterpret_cast<decltype(attention_paged_fn)>(at[2]);
    beam_select_fn = reinterpret_cast<decltype(beam_select_fn)>(at[3]);
    kv_reorder_fn = reinterpret_cast<decltype(kv_reorder_fn)>(at[4]);
    kv_store_q8_fn = reinterpret_cast<decltype(kv_store_q8_fn)>(at[5]);
    kv_load_fn = reinterpret_cast<decltype(kv_load_fn)>(at[6]);
    attention_shared_fn = reinterpret_cast<decltype(attention_shared_fn)>(at[7]);
    quantize_q4_fn = reinterpret_cast<decltype(quantize_q4_fn)>(at[8]);
    dequantize_q4_fn = reinterpret_cast<decltype(dequantize_q4_fn)>(at[9]);
    matvec_q4_fn = reinterpret_cast<decltype(matvec_q4_fn)>(at[10]);
    q4_bytes_fn = reinterpret_cast<decltype(q4_bytes_fn)>(at[11]);
    Py_INCREF(v[0]);
    tensor_type = reinterpret_cast<PyTypeObject*>(v[0]);
    api = got;
    Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }
PyMethodDef methods[] = {{"init", fast(init), METH_FASTCALL, nullptr},
                         {"page_plan", fast(page_plan), METH_FASTCALL, nullptr},
                         {"kv_store", fast(kv_store), METH_FASTCALL, nullptr},
                         {"attention_paged", fast(attention_paged), METH_FASTCALL, nullptr},
                         {"beam_select", fast(beam_select), METH_FASTCALL, nullptr},
                         {"kv_reorder", fast(kv_reorder), METH_FASTCALL, nullptr},
                         {"kv_store_q8", fast(kv_store_q8), METH_FASTCALL, nullptr},
                         {"kv_load", fast(kv_load), METH_FASTCALL, nullptr},
                         {"attention_shared", fast(attention_shared), METH_FASTCALL, nullptr},
                         {"quantize_q4", fast(quantize_q4), METH_FASTCALL, nullptr},
                         {"dequantize_q4", fast(dequantize_q4), METH_FASTCALL, nullptr},
                         {"matvec_q4", fast(matvec_q4), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", "Argument checks and calls of tie_b200.ops", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
