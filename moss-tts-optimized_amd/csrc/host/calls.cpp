// The operators of a batch as Python calls them, for the calls that need nothing said about them: arguments are checked,
// outputs and workspaces allocated and the C entry called without the interpreter, which took most of a call's time (one sequence's
// decode 16.8 -> 9.0 us, of which its two kernels are 8.8; adjust of 512 rows 11.8 -> 5.1, a written token read back 26.7 -> 8.3).
//
// Every function returns None for a call that it does not take (a wrong argument, another current device, no memory), before
// anything is launched: the Python function of the same name, which called it, then checks again and says what is wrong, or
// makes the call itself.  What is accepted here is accepted there.  An entry's error is raised by the function that raises
// it for Python's calls.
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <tuple>

#include "moss_hip.h"

namespace {

#define MOSS_ENTRIES(X)                                                                                                       \
    X(moss_paged_qk_rope) X(moss_paged_qk_rope_fp8) X(moss_paged_gather) X(moss_paged_gather_fp8)                             \
    X(moss_paged_decode_workspace_bytes) X(moss_paged_decode_attention) X(moss_paged_decode_attention_fp8)                    \
    X(moss_paged_shared_workspace_bytes) X(moss_paged_shared_decode_attention) X(moss_paged_shared_decode_attention_fp8)      \
    X(moss_paged_prompt_workspace_bytes) X(moss_paged_prompt_workspace_bytes_fp8) X(moss_paged_prompt_attention)              \
    X(moss_paged_prompt_attention_fp8) X(moss_adjust_rows)
struct Entries {
#define X(name) decltype(&::name) name;
    MOSS_ENTRIES(X)
#undef X
} lib;
PyObject* check;  // check(code, name) raises what an entry's error stands for
struct Raised {};  // an exception of Python's is set

typedef long long ll;
struct Span {
    const char *first, *end;
};
bool apart(const Span& a, const Span& b) { return a.end <= b.first || b.end <= a.first; }

// ---------------------------------------------------------------- arguments
struct Arg {  // a tensor on device `index`, or not `ok`
    const at::Tensor* t = nullptr;
    Arg(PyObject* o, int index) {
        if (!THPVariable_CheckExact(o)) return;  // a subclass makes its outputs by itself
        const at::Tensor& x = THPVariable_Unpack(o);
        if (x.defined() && x.is_cuda() && x.layout() == at::kStrided && x.get_device() == index) t = &x;
    }
    bool ok() const { return t != nullptr; }
    char* at() const { return static_cast<char*>(t->data_ptr()); }
    bool is(at::ScalarType s) const { return t->scalar_type() == s; }
    int dim() const { return (int)t->dim(); }
    ll size(int i) const { return t->sizes()[i]; }
    ll stride(int i) const { return t->strides()[i]; }
    Span all() const { return Span{at(), at() + t->numel() * t->element_size()}; }  // of a contiguous one
    // one value each of `n`, contiguous
    bool list(at::ScalarType s, ll n) const { return ok() && is(s) && t->numel() == n && t->is_contiguous(); }
};
bool none(PyObject* o) { return o == Py_None; }
int device_of(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return -1;
    const at::Tensor& x = THPVariable_Unpack(o);
    return x.defined() && x.is_cuda() ? (int)x.get_device() : -1;
}
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool number(PyObject* o, double& v) {  // not a truth value
    if (PyFloat_CheckExact(o)) v = PyFloat_AS_DOUBLE(o);
    else if (PyLong_CheckExact(o)) v = PyLong_AsDouble(o);
    else return false;
    if (PyErr_Occurred()) return PyErr_Clear(), false;
    return std::isfinite(v);
}
int kind_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : -1; }

struct Spans {
    Span s[24];
    int n = 0;
    void add(const Span& x) { s[n++] = x; }
    bool apart_from(const Span& x) const {
        for (int i = 0; i < n; ++i)
            if (!apart(s[i], x)) return false;
        return true;
    }
};

struct Region {
    char *first, *end;
    ll step, page;  // bytes from a page to the next, of a page
};
struct Cache {
    ll pages, kh, rows, d, strides[4];  // strides of keys, values and their scales, in elements
    Region regions[4];
    at::Tensor held[2];  // the scales: other threads may run before the launch, and a list of them may change
    int n;               // 2, or 4 in 8 bits
    bool eight() const { return n == 4; }
    bool of(PyObject* keys, PyObject* values, PyObject* scales, at::ScalarType type, int index) {
        n = none(scales) ? 2 : 4;
        PyObject* parts[4] = {keys, values, nullptr, nullptr};
        if (n == 4) {
            if (!(PyTuple_CheckExact(scales) || PyList_CheckExact(scales)) || PySequence_Fast_GET_SIZE(scales) != 2) return false;
            parts[2] = PySequence_Fast_GET_ITEM(scales, 0), parts[3] = PySequence_Fast_GET_ITEM(scales, 1);
            type = at::kFloat8_e4m3fn;
        }
        for (int i = 0; i < n; ++i) {
            const Arg a(parts[i], index);
            const int dims = i < 2 ? 4 : 3;
            if (!a.ok() || a.dim() != dims || !a.is(i < 2 ? type : at::kByte)) return false;
            if (i == 0) {
                pages = a.size(0), kh = a.size(1), rows = a.size(2), d = a.size(3);
                if (pages <= 0 || pages > INT_MAX || kh <= 0 || kh > 1024 || rows < 16 || rows > 4096 || rows & (rows - 1) ||
                    (d != 64 && d != 128))
                    return false;
            } else if (a.size(0) != pages || a.size(1) != kh || a.size(2) != rows || (i < 2 && a.size(3) != d)) {
                return false;
            }
            const ll row = i < 2 ? d : 1, wide = a.t->element_size(), page = kh * rows * row;
            if (a.stride(dims - 1) != 1 || (i < 2 && a.stride(2) != d) || (kh > 1 && a.stride(1) != rows * row)) return false;
            const ll step = pages == 1 ? page : a.stride(0);
            if (step < page || step % (n == 4 ? 16 : 8) || !aligned(a.at())) return false;
            strides[i] = step;
            regions[i] = Region{a.at(), a.at() + wide * ((pages - 1) * step + page), wide * step, wide * page};
            if (i >= 2) held[i - 2] = *a.t;
        }
        return true;
    }
    void spans(Spans& s) const {
        for (int i = 0; i < n; ++i) s.add(Span{regions[i].first, regions[i].end});
    }
    bool written_apart() const {
        for (int i = 0; i < n; ++i)
            for (int j = i + 1; j < n; ++j) {
                const Region &a = regions[i], &b = regions[j];
                if (a.end <= b.first || b.end <= a.first) continue;
                if (a.step != b.step) return false;
                const ll at = ((b.first - a.first) % a.step + a.step) % a.step;
                if (at < a.page || at > a.step - b.page) return false;
            }
        return true;
    }
};

struct Batch {
    int b, w;
    ll stride;
    char *table, *lengths, *starts;
    bool of(PyObject* table_, PyObject* lengths_, PyObject* starts_, ll rows, int index) {
        const Arg t(table_, index), l(lengths_, index);
        if (!t.ok() || t.dim() != 2 || !t.is(at::kInt)) return false;
        const ll many = t.size(0), wide = t.size(1);
        if (many <= 0 || many > 65535 || wide <= 0 || wide > (1ll << 30) / rows) return false;
        stride = many == 1 ? wide : t.stride(0);
        if ((wide > 1 && t.stride(1) != 1) || stride < wide || !l.list(at::kInt, many)) return false;
        b = (int)many, w = (int)wide, table = t.at(), lengths = l.at(), starts = nullptr;
        if (!none(starts_)) {
            const Arg s(starts_, index);
            if (!s.list(at::kInt, many + 1)) return false;
            starts = s.at();
        }
        return true;
    }
    void spans(Spans& s) const {
        s.add(Span{table, table + 4 * ((b - 1) * stride + w)});
        s.add(Span{lengths, lengths + 4ll * b});
        if (starts) s.add(Span{starts, starts + 4ll * b + 4});
    }
};

// Rows of queries [tokens, heads, head dim], or of qkv [tokens, width].
struct Query {
    ll tokens, heads, d, stride;
    char* at;
    Span span;
    bool of(const Arg& q) {
        if (q.dim() != 3 || q.t->numel() == 0) return false;
        tokens = q.size(0), heads = q.size(1), d = q.size(2), at = q.at();
        stride = tokens == 1 ? heads * d : q.stride(0);
        if ((d > 1 && q.stride(2) != 1) || (heads > 1 && q.stride(1) != d)) return false;
        span = Span{at, at + 2 * ((tokens - 1) * stride + heads * d)};
        return stride >= heads * d && stride % 8 == 0 && aligned(at) && heads <= 1024;
    }
};

bool scale_of(PyObject* o, ll d, double& v) {
    if (none(o)) return v = std::pow((double)d, -0.5), true;
    return number(o, v) && std::fabs((float)v) < 0x1p127f;
}

// A new tensor.  Device memory may have to be found for it, which can take long: other Python threads run meanwhile.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, int index) {
    Unlocked now;
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, index));
}

// An output or workspace: a new one, or the caller's, of this shape and apart from the rest.
bool output(PyObject* given, at::IntArrayRef shape, at::ScalarType type, int index, const Spans& rest, at::Tensor& made, char*& at,
            Span& span) {
    if (none(given)) {
        made = fresh(shape, type, index);
        at = static_cast<char*>(made.data_ptr());
        span = Span{at, at + made.numel() * made.element_size()};
        return true;
    }
    const Arg a(given, index);
    if (!a.ok() || !a.is(type) || !a.t->is_contiguous() || a.t->sizes() != shape) return false;
    at = a.at(), span = a.all();
    return aligned(at) && rest.apart_from(span);
}
bool workspace(PyObject* given, ll bytes, int index, const Spans& rest, const Span& out, at::Tensor& made, char*& at) {
    if (none(given)) {
        at = nullptr;
        if (bytes) {
            made = fresh({bytes / 4}, at::kFloat, index);
            at = static_cast<char*>(made.data_ptr());
        }
        return true;
    }
    const Arg a(given, index);
    if (!a.ok() || !a.is(at::kFloat) || !a.t->is_contiguous() || 4 * a.t->numel() < bytes) return false;
    at = a.at();
    return aligned(at) && rest.apart_from(a.all()) && apart(out, a.all());
}
PyObject* result(PyObject* given, const at::Tensor& made) {
    if (none(given)) return THPVariable_Wrap(made);
    Py_INCREF(given);
    return given;
}

bool current(int index) { return index >= 0 && c10::hip::current_device() == index; }
void* stream(int index) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)index).stream(); }

// A C entry's launches, without the interpreter's lock.
template <typename F, typename... A>
void launch(const char* name, F f, A... a) {
    int code;
    Py_BEGIN_ALLOW_THREADS;
    code = f(a...);
    Py_END_ALLOW_THREADS;
    if (code == 0) return;
    PyObject* r = PyObject_CallFunction(check, "is", code, name);
    if (r) PyErr_Format(PyExc_RuntimeError, "%s: error %d", name, code), Py_DECREF(r);
    throw Raised();
}
// ... over a cache in either form: what comes before it, the cache, what comes behind.
template <typename F16, typename F8, typename... A, typename... B>
void launch_over(const Cache& c, const char* name, F16 f16, F8 f8, const std::tuple<A...>& before, const std::tuple<B...>& behind) {
    auto all = [&](auto f, auto... cache) {
        std::apply([&](auto... a) { std::apply([&](auto... b) { launch(name, f, a..., cache..., b...); }, behind); }, before);
    };
    const Region* r = c.regions;
    if (c.eight())
        all(f8, (void*)r[0].first, (void*)r[1].first, (void*)r[2].first, (void*)r[3].first, c.strides[0], c.strides[1],
            c.strides[2], c.strides[3], (int)c.pages, (int)c.rows);
    else
        all(f16, (void*)r[0].first, (void*)r[1].first, c.strides[0], c.strides[1], (int)c.pages, (int)c.rows);
}
#define MOSS_OVER(c, name) c, c.eight() ? #name "_fp8" : #name, lib.name, lib.name##_fp8

// ---------------------------------------------------------------- the functions
// decode(q, keys, values, scales, table, lengths, groups, shared, scale, out, ws); groups and shared None: nothing shared
PyObject* decode(PyObject* const* v) {
    const int index = device_of(v[0]);
    if (!current(index)) return nullptr;
    const Arg q(v[0], index);
    Query x;
    Cache c;
    Batch b;
    double scale;
    if (!q.ok() || kind_of(*q.t) < 0 || !x.of(q) || !c.of(v[1], v[2], v[3], q.t->scalar_type(), index) ||
        !b.of(v[4], v[5], Py_None, c.rows, index) || x.tokens != b.b || x.d != c.d || x.heads % c.kh || !scale_of(v[8], c.d, scale))
        return nullptr;
    const bool runs = !none(v[6]);
    const Arg groups(v[6], index), shared(v[7], index);
    if (runs && (!groups.list(at::kInt, b.b) || !shared.list(at::kInt, b.b))) return nullptr;
    Spans s;
    s.add(x.span);
    c.spans(s);
    b.spans(s);
    if (runs) s.add(groups.all()), s.add(shared.all());
    const int qh = (int)x.heads, kh = (int)c.kh, d = (int)c.d, kind = kind_of(*q.t);
    at::Tensor made, made_ws;
    char *out, *ws;
    Span span;
    if (!output(v[9], {x.tokens, x.heads * x.d}, q.t->scalar_type(), index, s, made, out, span)) return nullptr;
    const ll bytes = (runs ? lib.moss_paged_shared_workspace_bytes : lib.moss_paged_decode_workspace_bytes)(b.b, b.w, (int)c.rows, qh, kh, d);
    if (!workspace(v[10], bytes, index, s, span, made_ws, ws)) return nullptr;
    const auto before = std::make_tuple((const void*)x.at, x.stride);
    void* st = stream(index);
    if (runs)
        launch_over(MOSS_OVER(c, moss_paged_shared_decode_attention), before,
                    std::make_tuple((const void*)b.table, b.stride, (const void*)b.lengths, (const void*)groups.at(),
                                    (const void*)shared.at(), b.b, b.w, qh, kh, d, (float)scale, (void*)out, (void*)ws, bytes, kind, st));
    else
        launch_over(MOSS_OVER(c, moss_paged_decode_attention), before,
                    std::make_tuple((const void*)b.table, b.stride, (const void*)b.lengths, b.b, b.w, qh, kh, d, (float)scale, (void*)out,
                                    (void*)ws, bytes, kind, st));
    return result(v[9], made);
}

// prompt(q, keys, values, scales, table, lengths, starts, scale, out, ws)
PyObject* prompt(PyObject* const* v) {
    const int index = device_of(v[0]);
    if (!current(index) || none(v[6])) return nullptr;
    const Arg q(v[0], index);
    Query x;
    Cache c;
    Batch b;
    double scale;
    if (!q.ok() || kind_of(*q.t) < 0 || !x.of(q) || !c.of(v[1], v[2], v[3], q.t->scalar_type(), index) ||
        !b.of(v[4], v[5], v[6], c.rows, index) || x.tokens > 1 << 20 || x.d != c.d || x.heads % c.kh || !scale_of(v[7], c.d, scale))
        return nullptr;
    Spans s;
    s.add(x.span);
    c.spans(s);
    b.spans(s);
    const int T = (int)x.tokens, qh = (int)x.heads, kh = (int)c.kh, d = (int)c.d;
    at::Tensor made, made_ws;
    char *out, *ws;
    Span span;
    if (!output(v[8], {x.tokens, x.heads * x.d}, q.t->scalar_type(), index, s, made, out, span)) return nullptr;
    // what the cache's form takes at best, or the caller's, which the 16-bit form's is enough for
    const auto size = c.eight() && none(v[9]) ? lib.moss_paged_prompt_workspace_bytes_fp8 : lib.moss_paged_prompt_workspace_bytes;
    ll bytes = size(b.b, b.w, (int)c.rows, T, qh, kh, d);
    if (!workspace(v[9], bytes, index, s, span, made_ws, ws)) return nullptr;
    if (!none(v[9])) bytes = 4 * THPVariable_Unpack(v[9]).numel();
    launch_over(MOSS_OVER(c, moss_paged_prompt_attention), std::make_tuple((const void*)x.at, x.stride),
                std::make_tuple((const void*)b.table, b.stride, (const void*)b.lengths, (const void*)b.starts, b.b, b.w, T, qh, kh, d,
                                (float)scale, (void*)out, (void*)ws, bytes, kind_of(*q.t), stream(index)));
    return result(v[8], made);
}

// qk_rope(qkv, q_weight, k_weight, cos, sin, keys, values, scales, table, lengths, starts, eps, out)
PyObject* qk_rope(PyObject* const* v) {
    const int index = device_of(v[0]);
    if (!current(index)) return nullptr;
    const Arg qkv(v[0], index);
    if (!qkv.ok() || kind_of(*qkv.t) < 0 || qkv.dim() != 2 || qkv.t->numel() == 0) return nullptr;
    const at::ScalarType type = qkv.t->scalar_type();
    const ll tokens = qkv.size(0), width = qkv.size(1), stride = tokens == 1 ? width : qkv.stride(0);
    if ((width > 1 && qkv.stride(1) != 1) || stride < width || stride % 8 || !aligned(qkv.at()) || tokens >= 1 << 24) return nullptr;
    Cache c;
    Batch b;
    double eps;
    if (!c.of(v[5], v[6], v[7], type, index) || !b.of(v[8], v[9], v[10], c.rows, index) || !number(v[11], eps) || !(eps >= 0))
        return nullptr;
    const ll qh = width / c.d - 2 * c.kh;
    if (width % c.d || qh <= 0 || qh > 1024 || qh % c.kh || (!b.starts && tokens != b.b)) return nullptr;
    const Arg cos(v[3], index), sin(v[4], index);
    if (!cos.ok() || !sin.ok() || cos.dim() != 2 || !(cos.is(at::kFloat) || cos.is(type)) || !sin.is(cos.t->scalar_type()) ||
        sin.t->sizes() != cos.t->sizes() || cos.size(1) != c.d || cos.size(0) <= 0 || cos.size(0) > INT_MAX || !cos.t->is_contiguous() ||
        !sin.t->is_contiguous() || !aligned(cos.at()) || !aligned(sin.at()))
        return nullptr;
    Spans s;
    const Span span{qkv.at(), qkv.at() + 2 * ((tokens - 1) * stride + width)};
    c.spans(s);
    if (!s.apart_from(span) || !c.written_apart()) return nullptr;
    const void* weights[2] = {nullptr, nullptr};
    if (none(v[1]) != none(v[2])) return nullptr;
    if (!none(v[1]))
        for (int i = 0; i < 2; ++i) {
            const Arg w(v[1 + i], index);
            if (!w.list(type, c.d) || !aligned(w.at())) return nullptr;
            weights[i] = w.at();
            s.add(w.all());
        }
    s.add(span), s.add(cos.all()), s.add(sin.all());
    b.spans(s);
    at::Tensor made;
    char* out;
    Span written;
    if (!output(v[12], {tokens, qh, c.d}, type, index, s, made, out, written)) return nullptr;
    launch_over(MOSS_OVER(c, moss_paged_qk_rope),
                std::make_tuple((const void*)qkv.at(), stride, weights[0], weights[1], (const void*)cos.at(), (const void*)sin.at(),
                                (int)cos.is(at::kFloat), (int)cos.size(0), (void*)out),
                std::make_tuple((const void*)b.table, b.stride, (const void*)b.lengths, (const void*)b.starts, b.b, b.w, (int)tokens,
                                (int)qh, (int)c.kh, (int)c.d, (float)eps, kind_of(*qkv.t), stream(index)));
    return result(v[12], made);
}

// gather(keys, values, scales, table, lengths, starts, tokens, out): in the type of out, a 16-bit cache's own, or bf16
PyObject* gather(PyObject* const* v) {
    const int index = device_of(v[0]);
    if (!current(index) || none(v[5]) || !PyLong_CheckExact(v[6])) return nullptr;
    const ll tokens = PyLong_AsLongLong(v[6]);
    if (PyErr_Occurred()) return PyErr_Clear(), nullptr;
    if (tokens <= 0 || tokens >= 1 << 24) return nullptr;
    const bool given = !none(v[7]);
    PyObject* outs[2] = {Py_None, Py_None};
    if (given) {
        if (!PyTuple_CheckExact(v[7]) || PyTuple_GET_SIZE(v[7]) != 2) return nullptr;  // a list may change meanwhile
        for (int i = 0; i < 2; ++i)
            if (device_of(outs[i] = PyTuple_GET_ITEM(v[7], i)) != index) return nullptr;  // one of them alone: refused
    }
    at::ScalarType type = none(v[2]) ? THPVariable_Unpack(v[0]).scalar_type() : at::kBFloat16;
    if (given && !none(v[2])) type = THPVariable_Unpack(outs[0]).scalar_type();
    const int kind = type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : -1;
    Cache c;
    Batch b;
    if (kind < 0 || !c.of(v[0], v[1], v[2], type, index) || !b.of(v[3], v[4], v[5], c.rows, index)) return nullptr;
    Spans s;
    c.spans(s);
    b.spans(s);
    at::Tensor made[2];
    char* at[2];
    for (int i = 0; i < 2; ++i) {
        Span span;
        if (!output(outs[i], {tokens, c.kh, c.d}, type, index, s, made[i], at[i], span)) return nullptr;
        if (given) s.add(span);
    }
    const auto behind = std::make_tuple((const void*)b.table, b.stride, (const void*)b.lengths, (const void*)b.starts, b.b, b.w, (int)tokens,
                                        (int)c.kh, (int)c.d, (void*)at[0], (void*)at[1], kind, stream(index));
    PyObject* pair = PyTuple_New(2);
    if (!pair) return PyErr_Clear(), nullptr;
    try {
        launch_over(MOSS_OVER(c, moss_paged_gather), std::make_tuple(), behind);
    } catch (const Raised&) {
        Py_DECREF(pair);
        throw;
    }
    for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(pair, i, result(outs[i], made[i]));
    return pair;
}

// [rows, n] or [1, n], or a row for all.
struct Rows {
    char* at = nullptr;
    ll stride = 0, n = 0;
    bool of(PyObject* o, at::ScalarType type, ll rows, int index, Spans& s) {
        const Arg a(o, index);
        if (!a.ok() || !a.is(type) || a.dim() != 2 || (a.size(0) != 1 && a.size(0) != rows) || a.size(1) <= 0) return false;
        n = a.size(1), stride = a.size(0) == 1 ? 0 : a.stride(0), at = a.at();
        if ((n > 1 && a.stride(1) != 1) || (stride != 0 && stride < n)) return false;
        s.add(Span{at, at + 4 * ((rows - 1) * stride + n)});
        return true;
    }
};

// adjust(logits, tokens, lengths, prompt, repetition, presence, frequency, bias_ids, bias, mask, out)
PyObject* adjust(PyObject* const* v) {
    const int index = device_of(v[0]);
    if (!current(index)) return nullptr;
    const Arg x(v[0], index);
    if (!x.ok() || x.dim() != 2 || x.t->numel() == 0) return nullptr;
    const at::ScalarType type = x.t->scalar_type();
    const int kind = type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : type == at::kFloat ? 2 : -1;
    const ll rows = x.size(0), entries = x.size(1), wide = x.t->element_size(), stride = rows == 1 ? entries : x.stride(0);
    if (kind < 0 || rows > 1 << 21 || entries > 1 << 19 || rows * entries > 1ll << 38 || (entries > 1 && x.stride(1) != 1) || stride < entries) return nullptr;
    Spans s;
    const bool history = !none(v[1]);
    char *tokens = nullptr, *counts[2] = {nullptr, nullptr}, *settings[3] = {nullptr, nullptr, nullptr};
    ll token_row = 0, token_step = 0, width = 0, token_bytes = 8;
    if (history) {
        const Arg t(v[1], index);
        if (!t.ok() || !(t.is(at::kLong) || t.is(at::kInt)) || t.dim() != 2 || t.size(0) != rows || t.size(1) <= 0 || t.size(1) > 1 << 30)
            return nullptr;
        tokens = t.at(), token_row = t.stride(0), token_step = t.stride(1), width = t.size(1), token_bytes = t.t->element_size();
        s.add(Span{tokens, tokens + token_bytes * ((rows - 1) * token_row + (width - 1) * token_step + 1)});
    }
    for (int i = 0; i < 2; ++i)
        if (!none(v[2 + i])) {
            const Arg t(v[2 + i], index);
            if (!history || !t.list(at::kInt, rows)) return nullptr;
            counts[i] = t.at();
            s.add(t.all());
        }
    float values[3];
    for (int i = 0; i < 3; ++i) {
        double value = i == 0 ? 1.0 : 0.0;
        if (THPVariable_Check(v[4 + i])) {
            const Arg t(v[4 + i], index);
            if (!history || !t.list(at::kFloat, rows)) return nullptr;
            settings[i] = t.at();
            s.add(t.all());
            value = 0.0;
        } else if (!number(v[4 + i], value) || (!history && value != (i == 0 ? 1.0 : 0.0)) || (i == 0 && !((float)value > 0.f)) ||
                   !std::isfinite((float)value)) {
            return nullptr;
        }
        values[i] = (float)value;
    }
    if (none(v[7]) != none(v[8])) return nullptr;
    Rows ids, bias, mask;
    if (!none(v[7]) && (!ids.of(v[7], at::kInt, rows, index, s) || !bias.of(v[8], at::kFloat, rows, index, s) || ids.n != bias.n || ids.n >= 1 << 16))
        return nullptr;
    if (!none(v[9]) && (!mask.of(v[9], at::kInt, rows, index, s) || 32 * mask.n < entries)) return nullptr;
    at::Tensor made;
    char* out;
    ll out_stride = entries;
    if (none(v[10])) {
        made = fresh({rows, entries}, type, index);
        out = static_cast<char*>(made.data_ptr());
    } else {
        const Arg o(v[10], index);
        if (!o.ok() || !o.is(type) || o.t->sizes() != x.t->sizes() || (entries > 1 && o.stride(1) != 1)) return nullptr;
        if (rows > 1) out_stride = o.stride(0);
        out = o.at();
        if (out_stride < entries) return nullptr;
        if (out != x.at() || out_stride != stride) s.add(Span{x.at(), x.at() + wide * ((rows - 1) * stride + entries)});
        if (!s.apart_from(Span{out, out + wide * ((rows - 1) * out_stride + entries)})) return nullptr;
    }
    launch("moss_adjust_rows", lib.moss_adjust_rows, (const void*)x.at(), kind, (int)rows, stride, (int)entries, (const void*)tokens,
           (int)token_bytes, token_row, token_step, (int)width, (const void*)counts[0], (const void*)counts[1],
           (const void*)settings[0], values[0], (const void*)settings[1], values[1], (const void*)settings[2], values[2],
           (const void*)ids.at, ids.stride, (const void*)bias.at, bias.stride, (int)bias.n, (const void*)mask.at, mask.stride, (void*)out,
           out_stride, stream(index));
    return result(v[10], made);
}

// ---------------------------------------------------------------- the module
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    PyObject* r = nullptr;
    if (n == N) {
        try {
            r = F(args);
        } catch (const Raised&) {
            return nullptr;
        } catch (const std::exception&) {  // out of memory and the like: the Python function meets it again, and says so
            r = nullptr;
        }
    }
    if (r) return r;
    PyErr_Clear();
    Py_RETURN_NONE;
}

// init(handle of the loaded library, check)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !PyCallable_Check(args[1])) return PyErr_Format(PyExc_TypeError, "a handle and a function required");
    void* at = PyLong_AsVoidPtr(args[0]);
    if (PyErr_Occurred()) return nullptr;
#define X(name)                                                                               \
    lib.name = reinterpret_cast<decltype(&::name)>(dlsym(at, #name));                         \
    if (!lib.name) return PyErr_Format(PyExc_RuntimeError, "the library has no %s", #name);
    MOSS_ENTRIES(X)
#undef X
    Py_INCREF(args[1]);
    Py_XDECREF(check);
    check = args[1];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"init", (PyCFunction)(void*)init, METH_FASTCALL, ""},
                         {"decode", (PyCFunction)(void*)call<decode, 11>, METH_FASTCALL, ""},
                         {"prompt", (PyCFunction)(void*)call<prompt, 10>, METH_FASTCALL, ""},
                         {"qk_rope", (PyCFunction)(void*)call<qk_rope, 13>, METH_FASTCALL, ""},
                         {"gather", (PyCFunction)(void*)call<gather, 8>, METH_FASTCALL, ""},
                         {"adjust", (PyCFunction)(void*)call<adjust, 11>, METH_FASTCALL, ""},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_moss_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__moss_calls() {
    PyObject* m = PyModule_Create(&module);
    // what reads tensors by the headers of one torch reads another's wrongly: the loader compares
    if (m && PyModule_AddStringConstant(m, "built_for", MOSS_BUILT_FOR) < 0) Py_CLEAR(m);
    return m;
}
