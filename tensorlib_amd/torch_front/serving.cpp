// The serving operators' Python front end: torch tensors in, checked, results and workspaces out of torch's allocator, one
// call of the C ABI each.  HipDevice's methods of the same names call these with their device's number first.
//
// Why native: the kernels behind a decode step take 3 to 10 us, and a call with the same checks in Python over ctypes took 9 to
// 12 us of the host.  It takes 4 to 5 here: the launch 3.1, torch's allocator 0.8, the rest for some twenty checks.
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "tensorlib_amd.h"

namespace {

PyObject* g_error = nullptr;        // tensorlib_amd.TensorLibError

// Sets a Python exception and leaves the call.
[[noreturn]] void fail(PyObject* type, const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    PyErr_SetString(type, text);
    throw python_error();
}

// One call of the library, without the interpreter's lock: a launch waits when the queue is full.
template <class F, class... A>
void call(const char* what, F entry, A... args) {
    PyThreadState* thread = PyEval_SaveThread();
    const int status = entry(args...);
    PyEval_RestoreThread(thread);
    if (status != TL_OK) fail(g_error, "%s failed (%d): %s", what, status, tl_last_error());
}

// One call's arguments, positional: the device's number, then the method's.
struct Args {
    PyObject* const* v;
    int64_t ordinal;

    Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t expected, const char* what) : v(args), ordinal(0) {
        if (n != expected) fail(PyExc_TypeError, "%s takes %zd arguments, got %zd", what, expected, n);
        ordinal = integer(0, "ordinal");
    }
    bool none(int i) const { return v[i] == Py_None; }
    long long integer(int i, const char* name) const {
        const long long x = PyLong_AsLongLong(v[i]);
        if (x == -1 && PyErr_Occurred()) fail(PyExc_TypeError, "%s must be an integer", name);
        return x;
    }
    int int32(int i, const char* name) const {
        const long long x = integer(i, name);
        if (x < INT32_MIN || x > INT32_MAX) fail(PyExc_ValueError, "%s %lld is out of range", name, x);
        return (int)x;
    }
    double number(int i, const char* name) const {
        const double x = PyFloat_AsDouble(v[i]);
        if (x == -1.0 && PyErr_Occurred()) fail(PyExc_TypeError, "%s must be a number", name);
        return x;
    }
    // TL_ROTARY_HALF or TL_ROTARY_INTERLEAVED.
    int layout(int i) const {
        if (PyUnicode_Check(v[i])) {
            if (PyUnicode_CompareWithASCIIString(v[i], "half") == 0) return TL_ROTARY_HALF;
            if (PyUnicode_CompareWithASCIIString(v[i], "interleaved") == 0) return TL_ROTARY_INTERLEAVED;
        }
        PyErr_Format(PyExc_ValueError, "unknown layout %R, one of 'half', 'interleaved'", v[i]);
        throw python_error();
    }
    // The library launches on the current device.
    void on_device() const {
        const int64_t current = c10::hip::current_device();
        if (current != ordinal) fail(g_error, "the current device is cuda:%lld, this device is cuda:%lld", (long long)current, (long long)ordinal);
    }
    // Results and workspaces come from torch's allocator, which hands memory out in the order of torch's current stream: the
    // library must enqueue on that one.
    void may_allocate() const {
        on_device();
        if (tl_get_stream() != (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)ordinal).stream())
            fail(g_error, "the library stream is not torch's current stream; call bind_stream(torch.cuda.current_stream()) first");
    }
    // A tensor of this device with the given type and number of dimensions.
    const at::Tensor& tensor(int i, const char* name, at::ScalarType type, int64_t dims) const {
        const at::Tensor& t = any_type(i, name);
        if (t.scalar_type() != type) fail(PyExc_TypeError, "%s must be %s, got %s", name, c10::toString(type), c10::toString(t.scalar_type()));
        if (t.dim() != dims) fail(PyExc_ValueError, "%s must have %lld dimensions, got %lld", name, (long long)dims, (long long)t.dim());
        return t;
    }
    const at::Tensor& any_type(int i, const char* name) const {
        if (!THPVariable_Check(v[i])) fail(g_error, "%s must be a CUDA(HIP) tensor; there is no CPU path", name);
        const at::Tensor& t = THPVariable_Unpack(v[i]);
        if (!t.is_cuda()) fail(g_error, "%s must be a CUDA(HIP) tensor; there is no CPU path", name);
        if (t.get_device() != ordinal) fail(PyExc_ValueError, "%s is on cuda:%lld, this device is cuda:%lld", name, (long long)t.get_device(), (long long)ordinal);
        if (t.layout() != c10::kStrided) fail(PyExc_ValueError, "%s must be a dense tensor", name);
        return t;
    }
    // The same, contiguous.
    const at::Tensor& dense(int i, const char* name, at::ScalarType type, int64_t dims) const {
        const at::Tensor& t = tensor(i, name, type, dims);
        if (!t.is_contiguous()) fail(PyExc_ValueError, "%s must be contiguous", name);
        return t;
    }
    const at::Tensor& vector(int i, const char* name, at::ScalarType type, int64_t n) const {
        const at::Tensor& t = dense(i, name, type, 1);
        if (t.size(0) != n) fail(PyExc_ValueError, "%s must have %lld elements, got %lld", name, (long long)n, (long long)t.size(0));
        return t;
    }
    // [rows, heads, dim] halves whose heads lie next to each other; rows may be apart.  -1: any extent.
    const at::Tensor& head_rows(int i, const char* name, int64_t rows, int64_t heads, int64_t dim) const {
        const at::Tensor& t = tensor(i, name, at::kHalf, 3);
        const int64_t n = t.size(0), h = t.size(1), d = t.size(2);
        if ((rows >= 0 && n != rows) || (heads >= 0 && h != heads) || (dim >= 0 && d != dim))
            fail(PyExc_ValueError, "%s must have shape [%s, %s, %s] (-1: any), got [%lld, %lld, %lld]", name, std::to_string(rows).c_str(), std::to_string(heads).c_str(),
                 std::to_string(dim).c_str(), (long long)n, (long long)h, (long long)d);
        if ((t.stride(2) != 1 && d > 1) || (t.stride(1) != d && h > 1) || (t.stride(0) < h * d && n > 1))
            fail(PyExc_ValueError, "%s: the heads of a row must be dense and rows must not overlap, got strides [%lld, %lld, %lld]", name, (long long)t.stride(0),
                 (long long)t.stride(1), (long long)t.stride(2));
        return t;
    }
    // Keys and values as [pages, positions, kv heads, dim] with the same strides.
    tl_kv_pages kv_pages(int i) const {
        const at::Tensor &k = tensor(i, "k_pages", at::kHalf, 4), &t = tensor(i + 1, "v_pages", at::kHalf, 4);
        if (k.sizes() != t.sizes() || k.strides() != t.strides() || (k.stride(3) != 1 && k.size(3) > 1))
            fail(PyExc_ValueError, "k_pages and v_pages need equal shapes, equal strides and dense heads");
        for (int64_t d = 0; d < 4; ++d)
            if (k.size(d) > INT32_MAX) fail(PyExc_ValueError, "k_pages is too large");
        return {k.data_ptr(), t.data_ptr(), (size_t)k.stride(0), (size_t)k.stride(1), (size_t)k.stride(2), (int)k.size(0), (int)k.size(1),
                 (int)k.size(2), (int)k.size(3)};
    }
};

int size32(int64_t n, const char* name) {
    if (n > INT32_MAX) fail(PyExc_ValueError, "%s is too large", name);
    return (int)n;
}
template <class T>
T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// The results of one call, as parts of one allocation: six of their own were 4 us.  Parts start 256 bytes apart.
class Results {
    at::Tensor whole_;
    int64_t used_ = 0;
    static int64_t rounded(int64_t words) { return (words + 63) & ~(int64_t)63; }

public:
    Results(const at::Tensor& like, std::initializer_list<int64_t> words) {
        int64_t n = 0;
        for (int64_t w : words) n += rounded(w);
        whole_ = at::empty({n}, like.options().dtype(at::kInt));
    }
    at::Tensor part(c10::IntArrayRef shape, at::ScalarType type = at::kInt) {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole_.storage()), whole_.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        t.unsafeGetTensorImpl()->set_storage_offset(used_ * (int64_t)(sizeof(int) / t.element_size()));
        used_ += rounded(t.numel());      // of at most one word each
        return t;
    }
};

// A workspace of the caller or, where that is None, `need` bytes from torch's allocator.
struct Workspace {
    at::Tensor held;
    void* p = nullptr;
    size_t bytes = 0;
    Workspace(const Args& a, int i, size_t need, const at::Tensor& like) {
        if (!a.none(i)) {
            const at::Tensor& t = a.dense(i, "workspace", at::kByte, 1);
            p = t.data_ptr();
            bytes = (size_t)t.numel();
        } else if (need) {
            held = at::empty({(int64_t)need}, like.options().dtype(at::kByte));
            p = held.data_ptr();
            bytes = need;
        }
    }
};

PyObject* pack(std::initializer_list<at::Tensor> tensors) {
    THPObjectPtr result(PyTuple_New((Py_ssize_t)tensors.size()));
    if (!result) throw python_error();
    Py_ssize_t i = 0;
    for (const at::Tensor& t : tensors) {
        PyObject* o = THPVariable_Wrap(t);
        if (!o) throw python_error();
        PyTuple_SET_ITEM(result.get(), i++, o);
    }
    return result.release();
}

// Puts one call, which allocates nothing, in line with torch's current stream where the library enqueues on another one: behind
// what was enqueued there so far, since that made the tensors, and ahead of what comes, since that reads them or has their
// memory again once they are freed.  A capture on the library's stream has an order of its own; one on torch's alone would go
// without the call.
class InLine {
    hipStream_t library_, torch_;
    bool apart_;

    static void check(hipError_t e) {
        if (e == hipSuccess) return;
        (void)hipGetLastError();           // reported here, not by the next call
        fail(g_error, "ordering the library stream and torch's current stream failed: %s", hipGetErrorString(e));
    }
    static bool capturing(hipStream_t s) {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        if (s) check(hipStreamIsCapturing(s, &status));       // the null stream never is
        return status != hipStreamCaptureStatusNone;
    }
    static void follow(hipStream_t later, hipStream_t earlier) {
        hipEvent_t event;
        check(hipEventCreateWithFlags(&event, hipEventDisableTiming));
        hipError_t e = hipEventRecord(event, earlier);
        if (e == hipSuccess) e = hipStreamWaitEvent(later, event, 0);
        (void)hipEventDestroy(event);      // what waits for it goes on doing so
        check(e);
    }

public:
    explicit InLine(const Args& a) {
        a.on_device();
        library_ = static_cast<hipStream_t>(tl_get_stream());
        torch_ = c10::hip::getCurrentHIPStream((c10::DeviceIndex)a.ordinal).stream();
        apart_ = library_ != torch_ && !capturing(library_);
        if (!apart_) return;
        if (capturing(torch_))
            fail(g_error, "torch's current stream is being captured and the library stream is another; call bind_stream(torch.cuda.current_stream()) first");
        follow(library_, torch_);
    }
    void done() const {
        if (apart_) follow(torch_, library_);
    }
};

// (ordinal, x, positions, freq, layout, magnitude, out or None)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 7, "rotary");
    const at::Tensor& x = a.head_rows(1, "x", -1, -1, -1);
    const int64_t rows = x.size(0), h = x.size(1), d = x.size(2);
    const at::Tensor &positions = a.vector(2, "positions", at::kInt, rows), &freq = a.dense(3, "freq", at::kDouble, 1);
    a.may_allocate();
    const at::Tensor out = a.none(6) ? at::empty({rows, h, d}, x.options()) : a.head_rows(6, "out", rows, h, d);
    call("tl_rotary_f16", tl_rotary_f16, out.data_ptr(), (size_t)out.stride(0), x.data_ptr(), (size_t)x.stride(0), ptr<int>(positions),
         ptr<double>(freq),
         size32(2 * freq.numel(), "freq"), a.layout(4), (float)a.number(5, "magnitude"), size32(rows, "x"), size32(h, "x"), size32(d, "x"));
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// (ordinal, q, k, v, positions, seq_ids or None, freq, k_pages, v_pages, tables, layout, magnitude, q_out or None)
PyObject* rotary_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 13, "rotary_paged");
    const tl_kv_pages cache = a.kv_pages(7);
    const at::Tensor& q = a.head_rows(1, "q", -1, -1, cache.head_dim);
    const int64_t rows = q.size(0), h = q.size(1);
    const at::Tensor& k = a.head_rows(2, "k", rows, cache.n_kv_heads, cache.head_dim);
    const at::Tensor& v = a.head_rows(3, "v", rows, cache.n_kv_heads, cache.head_dim);
    const at::Tensor &positions = a.vector(4, "positions", at::kInt, rows), &freq = a.dense(6, "freq", at::kDouble, 1);
    const at::Tensor& tables = a.dense(9, "tables", at::kInt, 2);
    const int* seq_ids = a.none(5) ? nullptr : ptr<int>(a.vector(5, "seq_ids", at::kInt, rows));
    a.may_allocate();
    const at::Tensor out = a.none(12) ? at::empty({rows, h, cache.head_dim}, q.options()) : a.head_rows(12, "q_out", rows, h, cache.head_dim);
    if (!out.is_contiguous()) fail(PyExc_ValueError, "q_out must be contiguous");
    call("tl_rotary_kv_pages_f16", tl_rotary_kv_pages_f16, out.data_ptr(), q.data_ptr(), (size_t)q.stride(0), k.data_ptr(), (size_t)k.stride(0),
         v.data_ptr(), (size_t)v.stride(0), ptr<int>(positions), seq_ids,
         ptr<double>(freq), size32(2 * freq.numel(), "freq"), a.layout(10), (float)a.number(11, "magnitude"), size32(rows, "q"),
         size32(h, "q"), &cache, ptr<int>(tables), (size_t)tables.size(1), size32(tables.size(0), "tables"));
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// (ordinal, q, k_pages, v_pages, tables, lens, scale or None, max_len or None, out or None, workspace or None)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 10, "paged_attention");
    const tl_kv_pages cache = a.kv_pages(2);
    const at::Tensor& q = a.head_rows(1, "q", -1, -1, cache.head_dim);
    const int64_t b = q.size(0);
    const int h = size32(q.size(1), "q"), seqs = size32(b, "q");
    const at::Tensor &tables = a.dense(4, "tables", at::kInt, 2), &lens = a.vector(5, "lens", at::kInt, b);
    const int64_t width = tables.size(1);
    if (tables.size(0) != b) fail(PyExc_ValueError, "tables must have %lld rows, got %lld", (long long)b, (long long)tables.size(0));
    int max_len;
    if (a.none(7)) max_len = (int)std::min<int64_t>(width * cache.page_size, INT32_MAX);
    else if ((max_len = a.int32(7, "max_len")) < 0) fail(PyExc_ValueError, "max_len %d is out of range", max_len);
    const float scale = a.none(6) ? 1.0f / std::sqrt((float)cache.head_dim) : (float)a.number(6, "scale");
    a.may_allocate();
    const at::Tensor out = a.none(8) ? at::empty({b, h, cache.head_dim}, q.options()) : a.head_rows(8, "out", b, h, cache.head_dim);
    if (!out.is_contiguous()) fail(PyExc_ValueError, "out must be contiguous");
    const Workspace ws(a, 9, a.none(9) ? tl_paged_attention_workspace_of_call(seqs, h, cache.n_kv_heads, cache.head_dim, max_len) : 0, q);
    call("tl_paged_attention_f16", tl_paged_attention_f16, out.data_ptr(), q.data_ptr(), (size_t)q.stride(0), &cache, ptr<int>(tables), (size_t)width,
         ptr<int>(lens), seqs, h, max_len, scale, ws.p, ws.bytes);
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// tables [rows, width], lens [rows], refs [pages] at arguments i, i + 1, i + 2.
struct PageState {
    const at::Tensor &tables, &lens, &refs;
    int rows, width, pages;
    PageState(const Args& a, int i)
        : tables(a.dense(i, "tables", at::kInt, 2)), lens(a.vector(i + 1, "lens", at::kInt, tables.size(0))), refs(a.dense(i + 2, "refs", at::kInt,
                 1)),
          rows(size32(tables.size(0), "tables")), width(size32(tables.size(1), "tables")), pages(size32(refs.size(0), "refs")) {}
};

// (ordinal, tables, lens, refs, parents, page_size) -> (tables, lens, refs, copy_src, copy_dst, missing)
PyObject* pages_fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 6, "pages_fork");
    const PageState s(a, 1);
    const at::Tensor& parents = a.vector(4, "parents", at::kInt, s.rows);
    a.may_allocate();
    Results r(s.tables, {(int64_t)s.rows * s.width, s.rows, s.pages, s.rows, s.rows, 1});
    const at::Tensor tables = r.part({s.rows, s.width}), lens = r.part({s.rows}), refs = r.part({s.pages}), src = r.part({s.rows}), dst =
             r.part({s.rows}), missing = r.part({1});
    call("tl_pages_fork", tl_pages_fork, ptr<int>(s.tables), ptr<int>(s.lens), ptr<int>(s.refs), ptr<int>(parents), ptr<int>(tables), ptr<int>(lens),
         ptr<int>(refs), ptr<int>(src), ptr<int>(dst),
         ptr<int>(missing), s.rows, s.width, s.pages, a.int32(5, "page_size"));
    return pack({tables, lens, refs, src, dst, missing});
    END_HANDLE_TH_ERRORS
}

// (ordinal, tables, lens, refs, add, page_size) -> missing
PyObject* pages_extend(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 6, "pages_extend");
    const PageState s(a, 1);
    const at::Tensor& add = a.vector(4, "add", at::kInt, s.rows);
    a.may_allocate();
    const at::Tensor missing = at::empty({1}, s.lens.options());
    call("tl_pages_extend", tl_pages_extend, ptr<int>(s.tables), ptr<int>(s.lens), ptr<int>(s.refs), ptr<int>(add), ptr<int>(missing), s.rows,
         s.width, s.pages, a.int32(5, "page_size"));
    return THPVariable_Wrap(missing);
    END_HANDLE_TH_ERRORS
}

// (ordinal, tables, lens, refs, rows, page_size)
PyObject* pages_free(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 6, "pages_free");
    const PageState s(a, 1);
    const at::Tensor& rows = a.vector(4, "rows", at::kBool, s.rows);
    const InLine line(a);
    call("tl_pages_free", tl_pages_free, ptr<int>(s.tables), ptr<int>(s.lens), ptr<int>(s.refs), ptr<uint8_t>(rows), s.rows, s.width, s.pages,
         a.int32(5, "page_size"));
    line.done();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// (ordinal, tables, refs) -> (tables, refs, remap, copy_src, copy_dst, count)
PyObject* pages_compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 3, "pages_compact");
    const at::Tensor &tables = a.dense(1, "tables", at::kInt, 2), &refs = a.dense(2, "refs", at::kInt, 1);
    const int rows = size32(tables.size(0), "tables"), width = size32(tables.size(1), "tables"), pages = size32(refs.size(0), "refs");
    a.may_allocate();
    Results r(tables, {(int64_t)rows * width, pages, pages, pages, pages, 1});
    const at::Tensor new_tables = r.part({rows, width}), new_refs = r.part({pages}), remap = r.part({pages}), src = r.part({pages});
    const at::Tensor dst = r.part({pages}), count = r.part({1});
    call("tl_pages_compact", tl_pages_compact, ptr<int>(tables), ptr<int>(refs), ptr<int>(new_tables), ptr<int>(new_refs), ptr<int>(remap),
         ptr<int>(src), ptr<int>(dst), ptr<int>(count), rows, width, pages);
    return pack({new_tables, new_refs, remap, src, dst, count});
    END_HANDLE_TH_ERRORS
}

// (ordinal, pool, src, dst, count or None)
PyObject* pages_copy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 5, "pages_copy");
    const at::Tensor& pool = a.any_type(1, "pool");
    if (pool.dim() < 3) fail(PyExc_ValueError, "pool must be [planes, pages, ...page]");
    const int64_t item = (int64_t)pool.element_size();
    int64_t page_bytes = item;
    for (int64_t d = pool.dim() - 1; d >= 2; --d) {
        if (pool.stride(d) * item != page_bytes && pool.size(d) > 1) fail(PyExc_ValueError, "a page of the pool must be contiguous");
        page_bytes *= pool.size(d);
    }
    const at::Tensor& src = a.dense(2, "src", at::kInt, 1);
    const at::Tensor& dst = a.vector(3, "dst", at::kInt, src.size(0));
    const int* count = a.none(4) ? nullptr : ptr<int>(a.vector(4, "count", at::kInt, 1));
    const InLine line(a);
    call("tl_pages_copy", tl_pages_copy, pool.data_ptr(), (size_t)(pool.stride(0) * item), (size_t)(pool.stride(1) * item), (size_t)page_bytes,
         size32(pool.size(0), "pool"), size32(pool.size(1), "pool"), ptr<int>(src), ptr<int>(dst), count, size32(src.size(0), "src"));
    line.done();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// (ordinal, logits, scores, n_beams, finished or None, end_token, n_select or None, workspace or None) -> (scores, tokens, parents)
PyObject* beam_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 8, "beam_select");
    const at::Tensor& logits = a.tensor(1, "logits", at::kHalf, 2);
    const int64_t rows = logits.size(0);
    const int vocab = size32(logits.size(1), "logits"), beams = a.int32(3, "n_beams");
    if (beams < 1 || rows % beams || (logits.stride(1) != 1 && vocab > 1) || (logits.stride(0) < vocab && rows > 1))
        fail(PyExc_ValueError, "logits must be [requests * %d, vocab] with dense rows, got [%lld, %d], strides [%lld, %lld]", beams, (long long)rows, vocab,
             (long long)logits.stride(0), (long long)logits.stride(1));
    const at::Tensor& scores = a.vector(2, "scores", at::kFloat, rows);
    const uint8_t* finished = a.none(4) ? nullptr : ptr<uint8_t>(a.vector(4, "finished", at::kBool, rows));
    const int batch = size32(rows / beams, "logits"), best = a.none(6) ? beams : a.int32(6, "n_select");
    const int64_t results = best > 0 ? (int64_t)batch * best : 0;
    a.may_allocate();
    Results r(scores, {results, results, results});
    const at::Tensor new_scores = r.part({results}, at::kFloat), tokens = r.part({results}), parents = r.part({results});
    const Workspace ws(a, 7, a.none(7) ? tl_beam_select_workspace(batch, beams, vocab, best) : 0, scores);
    call("tl_beam_select_f16", tl_beam_select_f16, ptr<float>(new_scores), ptr<int>(tokens), ptr<int>(parents), logits.data_ptr(),
         (size_t)logits.stride(0), ptr<float>(scores), finished, batch, beams, vocab, best, a.int32(5, "end_token"), ws.p, ws.bytes);
    return pack({new_scores, tokens, parents});
    END_HANDLE_TH_ERRORS
}

// (ordinal, history, lens, finished or None, parents, tokens, end_token) -> (history, lens, finished)
PyObject* beam_advance(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a(args, n, 7, "beam_advance");
    const at::Tensor& history = a.dense(1, "history", at::kInt, 2);
    const int rows = size32(history.size(0), "history"), width = size32(history.size(1), "history");
    const at::Tensor &lens = a.vector(2, "lens", at::kInt, rows), &parents = a.dense(4, "parents", at::kInt, 1);
    const uint8_t* finished = a.none(3) ? nullptr : ptr<uint8_t>(a.vector(3, "finished", at::kBool, rows));
    const int out = size32(parents.size(0), "parents");
    const at::Tensor& tokens = a.vector(5, "tokens", at::kInt, out);
    a.may_allocate();
    Results r(history, {(int64_t)out * width, out, out});
    const at::Tensor new_history = r.part({out, width}), new_lens = r.part({out}), new_finished = r.part({out}, at::kBool);
    call("tl_beam_advance", tl_beam_advance, ptr<int>(new_history), ptr<int>(new_lens), ptr<uint8_t>(new_finished), ptr<int>(history), ptr<int>(lens),
         finished, ptr<int>(parents), ptr<int>(tokens), rows, out, width, a.int32(6, "end_token"));
    return pack({new_history, new_lens, new_finished});
    END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {METHOD(rotary),        METHOD(rotary_paged), METHOD(paged_attention), METHOD(pages_fork), METHOD(pages_extend),
         METHOD(pages_free),
                           METHOD(pages_compact), METHOD(pages_copy),   METHOD(beam_select),     METHOD(beam_advance), {nullptr, nullptr, 0,
                           nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "tensorlib_torch_front", "Checked calls of the serving operators on torch tensors", -1, g_methods,
         nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_tensorlib_torch_front() {
    PyObject* lib = PyImport_ImportModule("tensorlib_amd._lib");
    if (!lib) return nullptr;
    g_error = PyObject_GetAttrString(lib, "TensorLibError");
    Py_DECREF(lib);
    return g_error ? PyModule_Create(&g_module) : nullptr;
}
