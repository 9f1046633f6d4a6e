// Python binding of the paged KV cache's entry points for the plain case: exact tensors,
// dense, of the right types and shapes, on the current device. From Python the checks of a
// call's tensors and the conversion of its twenty arguments take two to three times as long
// as the launch, and a decode step makes three such calls a layer. Anything that is not
// plain gives None, and the caller's own checks say what is wrong or make the call; a call
// that is made gives its result, or its status where it is not FL_OK.
//
// The entry points' addresses come from bind(): the library is whichever the package loaded.
// built_for says which fl355.h and which torch this was compiled with; with any others it must
// not be bound.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>

#include <algorithm>

#include <limits.h>

#include "fl355.h"

namespace {

decltype(&fl_paged_kv_store) p_store;
decltype(&fl_paged_kv_load) p_load;
decltype(&fl_attn_prep_paged) p_prep;
decltype(&fl_attention_prefill_paged_work_bytes) p_prefill_bytes;
decltype(&fl_attention_prefill_paged) p_prefill;
decltype(&fl_attn_decode_paged_work_bytes) p_decode_bytes;
decltype(&fl_attn_decode_paged) p_decode;
decltype(&fl_attn_prep_axes) p_prep_axes;
decltype(&fl_paged_kv_copy) p_copy;
decltype(&fl_paged_kv_keep) p_keep;
decltype(&fl_gdn_tree_normed) p_gdn_tree;
decltype(&fl_gdn_tree_commit) p_gdn_commit;
decltype(&fl_attn_tree_paged_work_bytes) p_tree_bytes;
decltype(&fl_attn_tree_paged) p_tree;

constexpr int64_t HEAD_DIM = 256, KV8_ROW = HEAD_DIM + HEAD_DIM / 32 * 2;   // bytes of an int8 head row

// The arguments of a call, taken in order; `ok` falls once one is not plain.
struct Args {
    PyObject* const* a;
    bool ok = true;
    int dev = -1;

    PyObject* next() { return *a++; }
    int64_t integer() {
        PyObject* o = next();
        if (!PyLong_CheckExact(o)) return ok = false, 0;
        int over = 0;
        const long long v = PyLong_AsLongLongAndOverflow(o, &over);
        ok = ok && over == 0;
        return v;
    }
    int integer32() {
        const int64_t v = integer();
        ok = ok && v >= INT_MIN && v <= INT_MAX;
        return (int)v;
    }
    int boolean() {
        PyObject* o = next();
        ok = ok && (o == Py_True || o == Py_False);
        return o == Py_True;
    }
    float real() {
        PyObject* o = next();
        if (!PyFloat_CheckExact(o)) return ok = false, 0.f;
        return (float)PyFloat_AS_DOUBLE(o);
    }
    // a dense tensor on the current device (null: not plain)
    const at::Tensor* dense(PyObject* o, at::ScalarType type, int64_t dim) {
        const at::Tensor* t = THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
        if (!t || t->scalar_type() != type || t->dim() != dim || !t->is_cuda() || t->get_device() != dev ||
            !t->is_contiguous())
            return ok = false, nullptr;
        return t;
    }
    const at::Tensor* dense(at::ScalarType type, int64_t dim) { return dense(next(), type, dim); }
};

// kpool, vpool, pages
struct Pools {
    const at::Tensor *k, *v, *pages;
    int q8 = 0, n_pages = 0, max_pages = 0;
    long long stride = 0;

    Pools(Args& a) {
        PyObject *ko = a.next(), *vo = a.next(), *po = a.next();
        k = THPVariable_CheckExact(ko) ? &THPVariable_Unpack(ko) : nullptr;
        q8 = k && k->scalar_type() == at::kChar;
        k = a.dense(ko, q8 ? at::kChar : at::kHalf, q8 ? 1 : 4);
        v = a.dense(vo, q8 ? at::kChar : at::kHalf, q8 ? 1 : 4);
        pages = THPVariable_CheckExact(po) ? &THPVariable_Unpack(po) : nullptr;
        if (!pages || pages->scalar_type() != at::kInt || pages->dim() != 2 || !pages->is_cuda() ||
            pages->get_device() != a.dev)
            a.ok = false;
    }
    // the rest, once the sizes are known
    bool fit(int64_t B, int64_t page_size, int64_t n_kv, int64_t head_dim) {
        if (page_size < 1 || n_kv < 1 || page_size > INT_MAX || n_kv > INT_MAX || head_dim != HEAD_DIM)
            return false;
        if (k->sizes() != v->sizes()) return false;
        int64_t n;
        if (q8) {
            if (page_size * n_kv > INT_MAX) return false;
            const int64_t unit = page_size * n_kv * KV8_ROW;
            n = k->numel() / unit;
            if (n * unit != k->numel()) return false;
        } else {
            n = k->size(0);
            if (k->size(1) != page_size || k->size(2) != n_kv || k->size(3) != head_dim) return false;
        }
        if (n > INT_MAX || pages->size(0) != B || pages->size(1) > INT_MAX ||
            (pages->stride(1) != 1 && pages->size(1) != 1))
            return false;
        n_pages = (int)n;
        max_pages = (int)pages->size(1);
        stride = B > 1 ? pages->stride(0) : max_pages;
        return true;
    }
};

// starts, pos0: the number of sequences, -1 where they do not fit
struct Packed {
    const at::Tensor *starts, *pos0;
    Packed(Args& a) : starts(a.dense(at::kInt, 1)), pos0(a.dense(at::kInt, 1)) {}
    int64_t count() const { return starts->numel() == pos0->numel() + 1 ? pos0->numel() : -1; }
};

at::Tensor half_rows(at::IntArrayRef sizes, int dev) {
    return at::empty(sizes, at::TensorOptions().dtype(at::kHalf).device(at::kCUDA, dev));
}

// work, given or made: its pointer and size (`made` keeps it)
bool work_of(PyObject* o, Args& a, size_t need, at::Tensor& made, void*& p, size_t& bytes) {
    if (o != Py_None) {
        const at::Tensor* t = a.dense(o, at::kByte, 1);
        if (!t) return false;
        p = t->data_ptr();
        bytes = (size_t)t->numel();
        return true;
    }
    p = nullptr;
    bytes = need;
    if (need == 0) return true;
    made = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, a.dev));
    p = made.data_ptr();
    return true;
}

// f() while other Python threads run
template <class F>
auto released(F f) {
    decltype(f()) r;
    Py_BEGIN_ALLOW_THREADS r = f();
    Py_END_ALLOW_THREADS return r;
}

#define PLAIN(x) \
    if (!(x)) Py_RETURN_NONE
#define MADE(rc) \
    if (rc) return PyLong_FromLong(rc)

// (dev, stream, k, v, starts, pos0, kpool, vpool, pages, page_size, n_kv, head_dim)
PyObject* kv_store(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == 12);
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const at::Tensor *k = a.dense(at::kHalf, 3), *v = a.dense(at::kHalf, 3);
    const Packed s(a);
    Pools c(a);
    const int64_t page_size = a.integer(), n_kv = a.integer(), head_dim = a.integer();
    PLAIN(a.ok && s.count() >= 0 && c.fit(s.count(), page_size, n_kv, head_dim));
    const int64_t N = k->size(0), row = n_kv * head_dim;
    PLAIN(N > 0 && N <= INT_MAX && k->sizes() == v->sizes() && k->size(1) == n_kv && k->size(2) == head_dim);
    const int rc = released([&] {
        return p_store(k->data_ptr(), v->data_ptr(), row, row, c.k->data_ptr(), c.v->data_ptr(), c.q8,
                       c.n_pages, (int)page_size, (const int*)c.pages->data_ptr(), c.max_pages, c.stride,
                       (const int*)s.starts->data_ptr(), (const int*)s.pos0->data_ptr(), (int)s.count(),
                       (int)N, (int)n_kv, (int)head_dim, stream);
    });
    MADE(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (dev, stream, starts, pos0, kpool, vpool, pages, T, page_size, n_kv, head_dim): (k, v), new
PyObject* kv_load(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == 11);
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const Packed s(a);
    Pools c(a);
    const int64_t T = a.integer(), page_size = a.integer(), n_kv = a.integer(), head_dim = a.integer();
    PLAIN(a.ok && T > 0 && T <= INT_MAX && s.count() >= 0 && c.fit(s.count(), page_size, n_kv, head_dim));
    const at::Tensor both = half_rows({2, T, n_kv, head_dim}, a.dev);
    const at::Tensor k = both.select(0, 0), v = both.select(0, 1);
    const int64_t row = n_kv * head_dim;
    const int rc = released([&] {
        return p_load(c.k->data_ptr(), c.v->data_ptr(), c.q8, c.n_pages, (int)page_size,
                      (const int*)c.pages->data_ptr(), c.max_pages, c.stride,
                      (const int*)s.starts->data_ptr(), (const int*)s.pos0->data_ptr(), k.data_ptr(),
                      v.data_ptr(), row, row, 1, (int)s.count(), (int)T, (int)n_kv, (int)head_dim, stream);
    });
    MADE(rc);
    PyObject *kp = THPVariable_Wrap(k), *vp = THPVariable_Wrap(v);
    PyObject* out = kp && vp ? PyTuple_Pack(2, kp, vp) : nullptr;
    Py_XDECREF(kp);
    Py_XDECREF(vp);
    return out;
    END_HANDLE_TH_ERRORS
}

// host ints of a list or tuple; false where it is neither, or holds anything else
bool ints(PyObject* o, int* out, Py_ssize_t most, Py_ssize_t& n) {
    const bool list = PyList_CheckExact(o);
    if (!list && !PyTuple_CheckExact(o)) return false;
    n = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
    if (n > most) return false;
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* x = list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i);
        if (!PyLong_CheckExact(x)) return false;
        int over = 0;
        const long long v = PyLong_AsLongLongAndOverflow(x, &over);
        if (over || v < 0 || v > INT_MAX) return false;
        out[i] = (int)v;
    }
    return true;
}

// (dev, stream, qg, k, v, wq, wk, q_out or None, starts, pos0, kpool, vpool, pages, page_size,
//  n_q, n_kv, head_dim, rope_dim, theta, eps), AXES: and (positions, the pairs' axes)
template <bool AXES>
PyObject* prep_of(PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == (AXES ? 22 : 20));
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const at::Tensor *qg = a.dense(at::kHalf, 3), *k = a.dense(at::kHalf, 3), *v = a.dense(at::kHalf, 3);
    const at::Tensor *wq = a.dense(at::kFloat, 1), *wk = a.dense(at::kFloat, 1);
    PyObject* qo = a.next();
    const at::Tensor* q_out = qo == Py_None ? nullptr : a.dense(qo, at::kHalf, 3);
    const Packed s(a);
    Pools c(a);
    const int64_t page_size = a.integer(), n_q = a.integer(), n_kv = a.integer(), head_dim = a.integer();
    const int rope_dim = a.integer32();
    const float theta = a.real(), eps = a.real();
    const at::Tensor* at = nullptr;
    int axis[HEAD_DIM / 2];
    if (AXES) {
        at = a.dense(at::kInt, 2);
        Py_ssize_t pairs = 0;
        PLAIN(ints(a.next(), axis, HEAD_DIM / 2, pairs) && pairs * 2 == rope_dim);
    }
    PLAIN(a.ok && s.count() >= 0 && c.fit(s.count(), page_size, n_kv, head_dim));
    const int64_t N = qg->size(0), pitch = qg->size(2);
    PLAIN(N > 0 && N <= INT_MAX && n_q <= INT_MAX && pitch <= INT_MAX && qg->size(1) == n_q &&
          k->sizes() == v->sizes() && k->size(0) == N && k->size(1) == n_kv && k->size(2) == head_dim &&
          wq->numel() >= head_dim && wk->numel() >= head_dim);
    PLAIN(!q_out || (q_out->size(0) == N && q_out->size(1) == n_q && q_out->size(2) <= INT_MAX));
    PLAIN(!AXES || (at->size(1) == N && at->size(0) <= INT_MAX));
    const int rc = released([&] {
        auto call = [&](auto f, auto... more) {
            return f(qg->data_ptr(), (int)pitch, k->data_ptr(), v->data_ptr(), (const float*)wq->data_ptr(),
                     (const float*)wk->data_ptr(), q_out ? q_out->data_ptr() : nullptr,
                     q_out ? (int)q_out->size(2) : 0, c.k->data_ptr(), c.v->data_ptr(), c.q8, c.n_pages,
                     (int)page_size, (const int*)c.pages->data_ptr(), c.max_pages, c.stride,
                     (const int*)s.starts->data_ptr(), (const int*)s.pos0->data_ptr(), more...,
                     (int)s.count(), (int)N, (int)n_q, (int)n_kv, (int)head_dim, rope_dim, theta, eps, stream);
        };
        if constexpr (AXES) return call(p_prep_axes, (const int*)at->data_ptr(), (int)at->size(0), (const int*)axis);
        else return call(p_prep);
    });
    MADE(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}
PyObject* prep(PyObject*, PyObject* const* args, Py_ssize_t n) { return prep_of<false>(args, n); }
PyObject* prep_axes(PyObject*, PyObject* const* args, Py_ssize_t n) { return prep_of<true>(args, n); }

// The pools of several layers, alike: two lists or tuples of tensors, or two tensors.
struct LayerPools {
    void *k[FL_POOL_MAX], *v[FL_POOL_MAX];
    int layers = 0, q8 = 0;
    const at::Tensor* first = nullptr;

    LayerPools(Args& a) {
        const int nk = take(a, k), nv = take(a, v);
        layers = nk;
        a.ok = a.ok && nk == nv;
    }
    // pages of the pools, -1 where they are none of these sizes
    int64_t pages(int64_t page_size, int64_t n_kv, int64_t head_dim) const {
        if (page_size < 1 || n_kv < 1 || page_size > INT_MAX || n_kv > INT_MAX || head_dim != HEAD_DIM ||
            page_size * n_kv > INT_MAX)
            return -1;
        if (!q8) {
            const bool fit = first->size(1) == page_size && first->size(2) == n_kv && first->size(3) == head_dim;
            return fit && first->size(0) <= INT_MAX ? first->size(0) : -1;
        }
        const int64_t unit = page_size * n_kv * KV8_ROW, n = first->numel() / unit;
        return n * unit == first->numel() && n <= INT_MAX ? n : -1;
    }

  private:
    int take(Args& a, void** to) {
        PyObject* o = a.next();
        if (THPVariable_CheckExact(o)) return one(a, o, to) ? 1 : -1;
        const bool list = PyList_CheckExact(o);
        const Py_ssize_t n = list ? PyList_GET_SIZE(o) : PyTuple_CheckExact(o) ? PyTuple_GET_SIZE(o) : 0;
        if (n < 1 || n > FL_POOL_MAX) return a.ok = false, -1;
        for (Py_ssize_t i = 0; i < n; ++i)
            if (!one(a, list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i), to + i)) return -1;
        return (int)n;
    }
    bool one(Args& a, PyObject* o, void** to) {
        if (!first) q8 = THPVariable_CheckExact(o) && THPVariable_Unpack(o).scalar_type() == at::kChar;
        const at::Tensor* t = a.dense(o, q8 ? at::kChar : at::kHalf, q8 ? 1 : 4);
        if (!t) return false;
        if (!first) first = t;
        else if (t->sizes() != first->sizes()) return a.ok = false;
        *to = t->data_ptr();
        return true;
    }
};

// (dev, stream, kpools, vpools, src, dst, page_size, n_kv, head_dim)
PyObject* kv_copy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == 9);
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const LayerPools c(a);
    const at::Tensor *src = a.dense(at::kInt, 1), *dst = a.dense(at::kInt, 1);
    const int64_t page_size = a.integer(), n_kv = a.integer(), head_dim = a.integer();
    PLAIN(a.ok);
    const int64_t pages = c.pages(page_size, n_kv, head_dim);
    PLAIN(pages >= 0 && src->numel() == dst->numel() && src->numel() <= INT_MAX);
    const int rc = released([&] {
        return p_copy(c.k, c.v, c.layers, c.q8, (int)pages, (int)page_size, (const int*)src->data_ptr(),
                      (const int*)dst->data_ptr(), (int)src->numel(), (int)n_kv, (int)head_dim, stream);
    });
    MADE(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (dev, stream, kpools, vpools, pages, pos0, path, page_size, n_kv, head_dim)
PyObject* kv_keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == 10);
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const LayerPools c(a);
    const at::Tensor *table = a.dense(at::kInt, 2), *pos0 = a.dense(at::kInt, 1), *path = a.dense(at::kInt, 2);
    const int64_t page_size = a.integer(), n_kv = a.integer(), head_dim = a.integer();
    PLAIN(a.ok);
    const int64_t pages = c.pages(page_size, n_kv, head_dim), B = pos0->numel();
    PLAIN(pages >= 0 && B > 0 && B <= INT_MAX && table->size(0) == B && path->size(0) == B &&
          table->size(1) <= INT_MAX && path->size(1) <= INT_MAX);
    const int rc = released([&] {
        return p_keep(c.k, c.v, c.layers, c.q8, (int)pages, (int)page_size, (const int*)table->data_ptr(),
                      (int)table->size(1), table->size(1), (const int*)pos0->data_ptr(),
                      (const int*)path->data_ptr(), (int)B, (int)path->size(1), (int)n_kv, (int)head_dim, stream);
    });
    MADE(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (dev, stream, q, kpool, vpool, pages, Ts, pos0s, page_size, window, sinks, gated, z or None,
//  work or None, n_kv, scale): z
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == 16);
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const at::Tensor* q = a.dense(at::kHalf, 3);
    Pools c(a);
    int Ts[FL_PAGED_MAX_SEQS_PREFILL], p0s[FL_PAGED_MAX_SEQS_PREFILL];
    Py_ssize_t B = 0, Bp = 0;
    PyObject *ts = a.next(), *ps = a.next();
    PLAIN(ints(ts, Ts, FL_PAGED_MAX_SEQS_PREFILL, B) && ints(ps, p0s, FL_PAGED_MAX_SEQS_PREFILL, Bp));
    const int64_t page_size = a.integer();
    const int window = a.integer32(), sinks = a.integer32(), gated = a.boolean();
    PyObject *zo = a.next(), *wo = a.next();
    const int64_t n_kv = a.integer();
    const float scale = a.real();
    PLAIN(a.ok && B > 0 && B == Bp && c.fit(B, page_size, n_kv, HEAD_DIM));
    const int64_t N = q->size(0), n_q = q->size(1), pitch = q->size(2);
    int64_t total = 0;
    for (Py_ssize_t b = 0; b < B; ++b) total += Ts[b];
    PLAIN(total > 0 && total <= N && n_q <= INT_MAX && pitch <= INT_MAX);
    at::Tensor z;
    if (zo == Py_None) {
        PLAIN(total == N);   // (else its last rows are zeros)
    } else {
        const at::Tensor* t = a.dense(zo, at::kHalf, 3);
        PLAIN(t && t->size(0) >= total && t->size(1) == n_q && t->size(2) <= INT_MAX);
        z = *t;
    }
    // (this makes the call's plan, up to milliseconds of host work)
    const size_t need = wo != Py_None ? 0 : released([&] {
        return p_prefill_bytes(Ts, p0s, (int)B, (int)n_q, (int)n_kv, (int)HEAD_DIM, window, sinks, c.q8);
    });
    at::Tensor made;
    void* work;
    size_t bytes;
    PLAIN(work_of(wo, a, need, made, work, bytes));
    if (zo == Py_None) z = half_rows({N, n_q, HEAD_DIM}, a.dev);
    const int rc = released([&] {
        return p_prefill(q->data_ptr(), (int)pitch, c.k->data_ptr(), c.v->data_ptr(), c.q8, c.n_pages,
                         (int)page_size, (const int*)c.pages->data_ptr(), c.max_pages, c.stride, Ts, p0s,
                         (int)B, (int)n_q, (int)n_kv, (int)HEAD_DIM, scale, window, sinks, gated,
                         z.data_ptr(), (int)z.size(2), work, bytes, stream);
    });
    MADE(rc);
    if (zo == Py_None) return THPVariable_Wrap(std::move(z));
    Py_INCREF(zo);
    return zo;
    END_HANDLE_TH_ERRORS
}

// (dev, stream, qg, kpool, vpool, pages, pos0, TREE: parents, page_size, window, sinks, gate, z or
//  None, work or None, n_kv, scale): z
template <bool TREE>
PyObject* decode_of(PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{args};
    PLAIN(n == (TREE ? 16 : 15));
    a.dev = a.integer32();
    const auto stream = (fl_stream_t)a.integer();
    const at::Tensor* qg = a.dense(at::kHalf, 4);
    Pools c(a);
    const at::Tensor* pos0 = a.dense(at::kInt, 1);
    const at::Tensor* parents = TREE ? a.dense(at::kInt, 2) : nullptr;
    const int64_t page_size = a.integer();
    const int window = a.integer32(), sinks = a.integer32(), gate = a.boolean();
    PyObject *zo = a.next(), *wo = a.next();
    const int64_t n_kv = a.integer();
    const float scale = a.real();
    PLAIN(a.ok);
    const int64_t B = qg->size(0), T = qg->size(1), n_q = qg->size(2), pitch = qg->size(3);
    PLAIN(B <= FL_PAGED_MAX_SEQS && T <= INT_MAX && n_q <= INT_MAX && pitch <= INT_MAX &&
          pos0->numel() == B && c.fit(B, page_size, n_kv, HEAD_DIM));
    PLAIN(!TREE || (parents->size(0) == B && parents->size(1) == T));
    at::Tensor z;
    if (zo != Py_None) {
        const at::Tensor* t = a.dense(zo, at::kHalf, 4);
        PLAIN(t && t->size(0) == B && t->size(1) == T && t->size(2) == n_q && t->size(3) <= INT_MAX);
        z = *t;
    }
    const size_t need = wo != Py_None ? 0
                                      : (TREE ? p_tree_bytes : p_decode_bytes)((int)B, (int)T, (int)n_q, (int)n_kv,
                                                                               (int)HEAD_DIM);
    PLAIN(wo != Py_None || need > 0);   // (sizes that the call refuses)
    at::Tensor made;
    void* work;
    size_t bytes;
    PLAIN(work_of(wo, a, need, made, work, bytes));
    if (zo == Py_None) z = half_rows({B, T, n_q, HEAD_DIM}, a.dev);
    const int rc = released([&] {
        auto call = [&](auto f, auto... more) {
            return f(qg->data_ptr(), (int)pitch, c.k->data_ptr(), c.v->data_ptr(), c.q8, c.n_pages,
                     (int)page_size, (const int*)c.pages->data_ptr(), c.max_pages, c.stride,
                     (const int*)pos0->data_ptr(), more..., (int)B, (int)T, (int)n_q, (int)n_kv, (int)HEAD_DIM,
                     scale, window, sinks, gate, z.data_ptr(), (int)z.size(3), work, bytes, stream);
        };
        if constexpr (TREE) return call(p_tree, (const int*)parents->data_ptr());
        else return call(p_decode);
    });
    MADE(rc);
    if (zo == Py_None) return THPVariable_Wrap(std::move(z));
    Py_INCREF(zo);
    return zo;
    END_HANDLE_TH_ERRORS
}
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) { return decode_of<false>(args, n); }
PyObject* tree(PyObject*, PyObject* const* args, Py_ssize_t n) { return decode_of<true>(args, n); }

// A list or tuple of dense tensors, one a sequence: their pointers, and the fewest elements of one.
struct Buffers {
    void* p[FL_MAX_SEQS];
    int n = 0;
    int64_t least = INT64_MAX;

    Buffers(Args& a, at::ScalarType type) {
        PyObject* o = a.next();
        const bool list = PyList_CheckExact(o);
        const Py_ssize_t size = list ? PyList_GET_SIZE(o) : PyTuple_CheckExact(o) ? PyTuple_GET_SIZE(o) : 0;
        if (size < 1 || size > FL_MAX_SEQS) {
            a.ok = false;
            return;
        }
        for (Py_ssize_t i = 0; i < size; ++i) {
            PyObject* x = list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i);
            const at::Tensor* t = THPVariable_CheckExact(x) ? &THPVariable_Unpack(x) : nullptr;
            if (!t || !a.dense(x, type, t->dim())) {
                a.ok = false;
                return;
            }
            p[i] = t->data_ptr();
            least = std::min(least, t->numel());
        }
        n = (int)size;
    }
};

// What the two GDN calls of a tree round share: x, S, a, b, A_log, dt_bias
struct GdnTree {
    const at::Tensor* x;
    Buffers S;
    const at::Tensor *a, *b, *A, *dt;
    int pos0[FL_MAX_SEQS];
    const at::Tensor* conv_w = nullptr;
    int64_t n_k = 0, n_v = 0, K = 0, V = 0, B = 0, T = 0;

    GdnTree(Args& g)
        : x(g.dense(at::kHalf, 3)), S(g, at::kFloat), a(g.dense(at::kFloat, 3)), b(g.dense(at::kFloat, 3)),
          A(g.dense(at::kFloat, 1)), dt(g.dense(at::kFloat, 1)) {}
    // pos0s, conv_w
    void more(Args& g) {
        Py_ssize_t n = 0;
        g.ok = ints(g.next(), pos0, FL_MAX_SEQS, n) && g.ok && n == S.n;
        conv_w = g.dense(at::kHalf, 2);
    }
    void sizes(Args& g) { n_k = g.integer(), n_v = g.integer(), K = g.integer(), V = g.integer(); }
    bool fit(const Buffers& frames) {
        for (int64_t d : {n_k, n_v, K, V})
            if (d < 1 || d > 4096) return false;
        const int64_t dim = 2 * n_k * K + n_v * V;
        B = S.n, T = x->size(1);
        return x->size(0) == B && T >= 1 && T <= INT_MAX && x->size(2) >= dim && x->size(2) <= INT_MAX &&
               S.least >= n_v * V * K && a->sizes() == b->sizes() && a->size(0) == B && a->size(1) == T &&
               a->size(2) >= n_v && a->size(2) <= INT_MAX && A->numel() >= n_v && dt->numel() >= n_v &&
               conv_w->numel() >= 4 * dim && frames.n == S.n && frames.least >= 3 * dim;
    }
};

// (dev, stream, x, S, a, b, A_log, dt_bias, z, norm_w, parents, y or None, pos0s, conv_w, cst_in, n_k, n_v,
//  K, V, out_scale, l2eps, norm_eps): y
PyObject* gdn_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args g{args};
    PLAIN(n == 22);
    g.dev = g.integer32();
    const auto stream = (fl_stream_t)g.integer();
    GdnTree c(g);
    PyObject* zo = g.next();
    const at::Tensor* z = THPVariable_CheckExact(zo) ? &THPVariable_Unpack(zo) : nullptr;
    PLAIN(z && (z->dim() == 3 || z->dim() == 4));
    z = g.dense(zo, at::kHalf, z->dim());
    const at::Tensor *norm_w = g.dense(at::kFloat, 1), *parents = g.dense(at::kInt, 2);
    PyObject* yo = g.next();
    c.more(g);
    const Buffers frames(g, at::kHalf);
    c.sizes(g);
    const float out_scale = g.real(), l2eps = g.real(), norm_eps = g.real();
    PLAIN(g.ok && c.fit(frames));
    const int64_t width = c.n_v * c.V;
    PLAIN(z->size(0) == c.B && z->size(1) == c.T && z->numel() == c.B * c.T * width &&
          norm_w->numel() >= c.V && parents->size(0) == c.B && parents->size(1) == c.T);
    at::Tensor y;
    if (yo != Py_None) {
        const at::Tensor* t = g.dense(yo, at::kHalf, 3);
        PLAIN(t && t->size(0) == c.B && t->size(1) == c.T && t->size(2) == width);
        y = *t;
    } else {
        y = half_rows({c.B, c.T, width}, g.dev);
    }
    const int rc = released([&] {
        return p_gdn_tree(c.x->data_ptr(), (int)c.x->size(2), c.conv_w->data_ptr(), frames.p, c.pos0,
                          (const int*)parents->data_ptr(), (const float*)c.a->data_ptr(),
                          (const float*)c.b->data_ptr(), (int)c.a->size(2), (const float*)c.A->data_ptr(),
                          (const float*)c.dt->data_ptr(), (const float* const*)c.S.p, z->data_ptr(), (int)width,
                          (const float*)norm_w->data_ptr(), y.data_ptr(), (int)width, (int)c.B, (int)c.T,
                          (int)c.n_k, (int)c.n_v, (int)c.K, (int)c.V, out_scale, l2eps, norm_eps, stream);
    });
    MADE(rc);
    if (yo == Py_None) return THPVariable_Wrap(std::move(y));
    Py_INCREF(yo);
    return yo;
    END_HANDLE_TH_ERRORS
}

// (dev, stream, x, S, a, b, A_log, dt_bias, path, S_out, pos0s, conv_w, cst_in, cst_out, n_k, n_v, K, V, l2eps)
PyObject* gdn_commit(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args g{args};
    PLAIN(n == 19);
    g.dev = g.integer32();
    const auto stream = (fl_stream_t)g.integer();
    GdnTree c(g);
    const at::Tensor* path = g.dense(at::kInt, 2);
    const Buffers S_out(g, at::kFloat);
    c.more(g);
    const Buffers frames(g, at::kHalf), frames_out(g, at::kHalf);
    c.sizes(g);
    const float l2eps = g.real();
    PLAIN(g.ok && c.fit(frames));
    PLAIN(path->size(0) == c.B && path->size(1) <= INT_MAX && S_out.n == c.S.n &&
          S_out.least >= c.n_v * c.V * c.K && frames_out.n == c.S.n &&
          frames_out.least >= 3 * (2 * c.n_k * c.K + c.n_v * c.V));
    const int rc = released([&] {
        return p_gdn_commit(c.x->data_ptr(), (int)c.x->size(2), c.conv_w->data_ptr(), frames.p, frames_out.p,
                            c.pos0, (const int*)path->data_ptr(), (const float*)c.a->data_ptr(),
                            (const float*)c.b->data_ptr(), (int)c.a->size(2), (const float*)c.A->data_ptr(),
                            (const float*)c.dt->data_ptr(), (const float* const*)c.S.p, (float* const*)S_out.p,
                            (int)c.B, (int)c.T, (int)path->size(1), (int)c.n_k, (int)c.n_v, (int)c.K, (int)c.V,
                            l2eps, stream);
    });
    MADE(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// the entry points' addresses, in the order of the declarations above
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    void** const to[] = {(void**)&p_store, (void**)&p_load, (void**)&p_prep, (void**)&p_prefill_bytes,
                         (void**)&p_prefill, (void**)&p_decode_bytes, (void**)&p_decode,
                         (void**)&p_prep_axes, (void**)&p_copy, (void**)&p_keep, (void**)&p_gdn_tree,
                         (void**)&p_gdn_commit, (void**)&p_tree_bytes, (void**)&p_tree};
    if (n != (Py_ssize_t)(sizeof(to) / sizeof(to[0]))) {
        PyErr_SetString(PyExc_TypeError, "bind: one address an entry point");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < n; ++i) {
        *to[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
    {"kv_store", (PyCFunction)(void (*)())kv_store, METH_FASTCALL, nullptr},
    {"kv_load", (PyCFunction)(void (*)())kv_load, METH_FASTCALL, nullptr},
    {"prep", (PyCFunction)(void (*)())prep, METH_FASTCALL, nullptr},
    {"prefill", (PyCFunction)(void (*)())prefill, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction)(void (*)())decode, METH_FASTCALL, nullptr},
    {"prep_axes", (PyCFunction)(void (*)())prep_axes, METH_FASTCALL, nullptr},
    {"kv_copy", (PyCFunction)(void (*)())kv_copy, METH_FASTCALL, nullptr},
    {"kv_keep", (PyCFunction)(void (*)())kv_keep, METH_FASTCALL, nullptr},
    {"gdn_tree", (PyCFunction)(void (*)())gdn_tree, METH_FASTCALL, nullptr},
    {"gdn_commit", (PyCFunction)(void (*)())gdn_commit, METH_FASTCALL, nullptr},
    {"tree", (PyCFunction)(void (*)())tree, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fl355_paged", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_fl355_paged() {
    PyObject* m = PyModule_Create(&module);
    PyObject* built_for = m ? Py_BuildValue("(ss)", FL_HEADER_DIGEST, BUILT_WITH_TORCH) : nullptr;
    if (built_for && PyModule_AddObject(m, "built_for", built_for) == 0) return m;
    Py_XDECREF(built_for);
    Py_XDECREF(m);
    return nullptr;
}
