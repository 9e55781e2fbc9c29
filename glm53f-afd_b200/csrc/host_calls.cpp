// The host side of the per-layer launches, natively: what kernel.ChainBatch and core.decode_batch do between the caller
// and the C ABI -- unwrap the views, check every extent against the geometry, pick the stream, launch.
//
// A decode step makes one such call per layer.  In Python the checks and the foreign call of 33 arguments take about
// 20 us (chain) and 15 us (core) a layer, several times what the kernel of a small batch runs for (4 us at one slot):
// the GPU waits for the host.  Here a call is 2 to 4 us, most of it the launch itself.
//
// Every function answers -1 when the call is not the plain accepted one: a check fails, an argument is of a type it
// does not know, a subclass, a tensor on the CPU.  Nothing has been enqueued then and the caller runs the Python code,
// which holds the same checks and raises the errors.  Any other answer is the launcher's status.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "glm53f_kda.h"
#include "glm53f_proj.h"

namespace {

constexpr int64_t kD = 128, kWindow = 3;

// Interned attribute names.
struct Names {
    PyObject *t, *buf, *offset, *stride, *weights, *heads, *conv_w, *a_log, *dt_bias, *norm_w, *eps, *lower, *p, *b_off, *a, *g, *conv, *state, *state_out,
        *out, *saves, *kind, *rows, *k, *v, *b, *fast, *cu_rows, *conv_off, *state_off, *stream, *cuda_stream;
} N;

// The exact Python types the fast path knows (set once by bind()).
PyObject *T_buffer = nullptr, *T_view = nullptr, *T_weights = nullptr, *T_saves = nullptr, *T_chain = nullptr, *T_meta = nullptr, *T_stream = nullptr;

struct Miss {};  // thrown to leave for the Python path

struct Ref {  // an owned reference
    PyObject* o;
    explicit Ref(PyObject* x) : o(x) {
        if (o == nullptr) throw Miss{};
    }
    Ref(const Ref&) = delete;
    Ref& operator=(const Ref&) = delete;
    ~Ref() { Py_DECREF(o); }
};
inline PyObject* get(PyObject* o, PyObject* name) { return PyObject_GetAttr(o, name); }
inline int64_t to_i64(PyObject* o) {
    if (!PyLong_CheckExact(o)) throw Miss{};
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Miss{};
    return v;
}
inline int64_t get_i64(PyObject* o, PyObject* name) {
    Ref r(get(o, name));
    return to_i64(r.o);
}
inline double get_f64(PyObject* o, PyObject* name) {
    Ref r(get(o, name));
    if (!PyFloat_CheckExact(r.o)) throw Miss{};
    return PyFloat_AS_DOUBLE(r.o);
}
inline void is_exactly(PyObject* o, PyObject* type) {
    if (reinterpret_cast<PyObject*>(Py_TYPE(o)) != type) throw Miss{};
}
// A launch without the interpreter's lock, as a foreign call makes it: a full launch queue blocks the caller, and what it waits for
// may be a host function that needs the lock.  Everything Python has been read by then.
template <typename F>
int unlocked(F&& launch) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = launch();
    Py_END_ALLOW_THREADS
    return rc;
}

inline const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) throw Miss{};
    return THPVariable_Unpack(o);
}

// The tensors whose addresses a launch takes, held until it is out: another thread may let go of them meanwhile.
struct Held {
    PyObject* o[24];
    int n = 0;
    PyObject* add(PyObject* x) {
        if (n == 24) throw Miss{};
        Py_INCREF(x);
        return o[n++] = x;
    }
    ~Held() {
        while (n > 0) Py_DECREF(o[--n]);
    }
};

struct Buffer {  // a DeviceBuffer: address and bytes
    unsigned char* ptr;
    int64_t bytes;
};
inline Buffer buffer(PyObject* o, Held& held) {
    is_exactly(o, T_buffer);
    Ref t(get(o, N.t));
    const at::Tensor& x = tensor(held.add(t.o));
    if (!x.is_cuda()) throw Miss{};
    const int64_t n = x.numel();
    return {n != 0 ? static_cast<unsigned char*>(x.data_ptr()) : nullptr, n};
}
inline Buffer get_buffer(PyObject* o, PyObject* name, Held& held) {
    Ref r(get(o, name));
    return buffer(r.o, held);
}
// a * b + c, exactly.
inline int64_t mul_add(int64_t a, int64_t b, int64_t c) {
    int64_t r;
    if (__builtin_mul_overflow(a, b, &r) || __builtin_add_overflow(r, c, &r)) throw Miss{};
    return r;
}
// Elements [offset, offset + n) of `size` bytes lie inside the buffer.
inline void region(const Buffer& b, int64_t size, int64_t offset, int64_t n) {
    if (offset < 0 || mul_add(offset, 1, n) > b.bytes / size) throw Miss{};
}

struct Rows {
    glm53f_bf16* ptr;
    int64_t stride;
};
// A RowView of bf16 rows whose columns [lo, hi) lie inside its buffer for `rows` rows.
inline Rows rows_of(PyObject* owner, PyObject* name, int64_t rows, int64_t lo, int64_t hi, Held& held) {
    Ref v(get(owner, name));
    is_exactly(v.o, T_view);
    const Buffer b = get_buffer(v.o, N.buf, held);
    const int64_t offset = get_i64(v.o, N.offset), stride = get_i64(v.o, N.stride);
    if (rows > 0 && (mul_add(offset, 1, lo) < 0 || mul_add(rows - 1, stride, mul_add(offset, 1, hi)) > b.bytes / 2)) throw Miss{};
    return {reinterpret_cast<glm53f_bf16*>(b.ptr) + offset, stride};
}

inline glm53f_stream_t stream_of(PyObject* s) {
    is_exactly(s, T_stream);
    Ref given(get(s, N.stream));
    if (given.o == Py_None) return reinterpret_cast<glm53f_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
    Ref raw(get(given.o, N.cuda_stream));
    return reinterpret_cast<glm53f_stream_t>(static_cast<uintptr_t>(to_i64(raw.o)));
}

// chain_batch(ChainBatch, BatchMeta, Stream, bf16_state) -> status, or -1.  kernel.ChainBatch._launch_as holds the checks
// in the order they raise.
int chain_batch(PyObject* cb, PyObject* meta, PyObject* stream, bool bf16) {
    is_exactly(cb, T_chain);
    is_exactly(meta, T_meta);
    // (requests, rows, then per kind of offset: least, greatest, least distance between two), kept by BatchMeta.set
    Ref fast(get(meta, N.fast));
    if (!PyTuple_CheckExact(fast.o) || PyTuple_GET_SIZE(fast.o) != 8) throw Miss{};
    int64_t m[8];
    for (int i = 0; i < 8; ++i) m[i] = to_i64(PyTuple_GET_ITEM(fast.o, i));
    const int64_t batch = m[0], total = m[1];
    Held held;
    Ref w(get(cb, N.weights));
    is_exactly(w.o, T_weights);
    const int64_t heads = get_i64(w.o, N.heads), es = bf16 ? 2 : 4;
    if (heads < 1 || heads > 65535 || batch < 1) throw Miss{};
    const int64_t channels = 3 * heads * kD, width = heads * kD, state_len = heads * kD * kD;
    const int64_t b_off = get_i64(cb, N.b_off);
    const int64_t b_end = mul_add(b_off, 1, heads);
    const Rows p = rows_of(cb, N.p, total, b_off < 0 ? b_off : 0, b_end > channels ? b_end : channels, held);
    const Rows a = rows_of(cb, N.a, total, 0, width, held), g = rows_of(cb, N.g, total, 0, width, held), out = rows_of(cb, N.out, total, 0, width, held);
    if (total > 1 && out.stride < width) throw Miss{};
    const Buffer conv = get_buffer(cb, N.conv, held), state = get_buffer(cb, N.state, held);
    region(conv, 2, m[2], kWindow * channels);
    region(conv, 2, m[3], kWindow * channels);
    region(state, es, m[5], state_len);
    region(state, es, m[6], state_len);
    if (m[7] < state_len) throw Miss{};
    void* state_out = nullptr;
    {
        Ref so(get(cb, N.state_out));
        Ref kind(get(so.o, N.kind));
        if (!PyUnicode_CheckExact(kind.o)) throw Miss{};
        if (PyUnicode_CompareWithASCIIString(kind.o, "in_place") == 0) state_out = state.ptr;
        else if (PyUnicode_CompareWithASCIIString(kind.o, "skip") != 0) throw Miss{};
    }
    void *ks = nullptr, *vs = nullptr, *gs = nullptr, *bs = nullptr;
    {
        Ref s(get(cb, N.saves));
        if (s.o != Py_None) {
            is_exactly(s.o, T_saves);
            if (get_i64(s.o, N.heads) != heads || get_i64(s.o, N.rows) < total) throw Miss{};
            ks = get_buffer(s.o, N.k, held).ptr;
            vs = get_buffer(s.o, N.v, held).ptr;
            gs = get_buffer(s.o, N.g, held).ptr;
            bs = get_buffer(s.o, N.b, held).ptr;
        }
    }
    const auto* cu = reinterpret_cast<const int32_t*>(get_buffer(meta, N.cu_rows, held).ptr);
    const auto* conv_off = reinterpret_cast<const int64_t*>(get_buffer(meta, N.conv_off, held).ptr);
    const auto* state_off = reinterpret_cast<const int64_t*>(get_buffer(meta, N.state_off, held).ptr);
    const auto* conv_w = reinterpret_cast<const glm53f_bf16*>(get_buffer(w.o, N.conv_w, held).ptr);
    const auto* a_log = reinterpret_cast<const float*>(get_buffer(w.o, N.a_log, held).ptr);
    const auto* dt_bias = reinterpret_cast<const float*>(get_buffer(w.o, N.dt_bias, held).ptr);
    const auto* norm_w = reinterpret_cast<const glm53f_bf16*>(get_buffer(w.o, N.norm_w, held).ptr);
    const float eps = (float)get_f64(w.o, N.eps), lower = (float)get_f64(w.o, N.lower);
    const glm53f_stream_t st = stream_of(stream);
    auto launch = [&](auto fn, auto* s_in, auto* s_out) {
        return unlocked([&] {
            return fn((int32_t)heads, (int32_t)batch, cu, p.ptr, p.stride, b_off, a.ptr, a.stride, g.ptr, g.stride, reinterpret_cast<const glm53f_bf16*>(conv.ptr),
                      conv_off, conv_w, s_in, s_out, state_off, a_log, dt_bias, norm_w, eps, lower, out.ptr, out.stride, static_cast<float*>(ks),
                      static_cast<glm53f_bf16*>(vs), static_cast<float*>(gs), static_cast<float*>(bs), st);
        });
    };
    if (bf16) return launch(glm53f_kda_chain_batch_bf16state, reinterpret_cast<const glm53f_bf16*>(state.ptr), static_cast<glm53f_bf16*>(state_out));
    return launch(glm53f_kda_chain_batch, reinterpret_cast<const float*>(state.ptr), static_cast<float*>(state_out));
}

// A contiguous CUDA tensor of the kind's element type with at least n elements.
enum Kind { kBf16, kF32, kI32, kI64 };
template <typename T>
T* need(PyObject* o, Kind kind, int64_t n) {
    const at::Tensor& t = tensor(o);
    const auto d = t.scalar_type();
    const bool ok = kind == kBf16  ? d == at::kBFloat16 || d == at::kShort || d == at::kUInt16
                    : kind == kF32 ? d == at::kFloat
                    : kind == kI32 ? d == at::kInt
                                   : d == at::kLong;
    if (!ok || !t.is_cuda() || !t.is_contiguous() || t.numel() < n) throw Miss{};
    return static_cast<T*>(t.data_ptr());
}

// core_decode(heads, rows, cu_rows, q, k, v, g, beta, state, state_off, state_out, flags, gate, norm_w, eps, out, saves,
// max_state_off) -> status, or -1.  core.decode_batch holds the checks in the order they raise.
int core_decode(PyObject* const* a) {
    const int64_t heads = to_i64(a[0]), rows = to_i64(a[1]), flags = to_i64(a[11]);
    if (heads < 1 || heads > 65535 || rows < 0 || rows > 0x7fffffff || flags < 0 || flags > 0x7fffffff) throw Miss{};
    const int64_t n = rows * heads * kD;
    const auto* cu = need<const int32_t>(a[2], kI32, 2);
    const int64_t batch = tensor(a[2]).numel() - 1;
    if (batch > 65535) throw Miss{};
    const auto *q = need<const glm53f_bf16>(a[3], kBf16, n), *k = need<const glm53f_bf16>(a[4], kBf16, n), *v = need<const glm53f_bf16>(a[5], kBf16, n);
    const auto* g = need<const float>(a[6], kF32, n);
    const auto* beta = need<const float>(a[7], kF32, rows * heads);
    const auto* off = need<const int64_t>(a[9], kI64, batch);
    const at::Tensor& state = tensor(a[8]);
    const auto sd = state.scalar_type();
    if (!state.is_cuda()) throw Miss{};
    const int32_t kind = sd == at::kFloat ? 0 : sd == at::kBFloat16 || sd == at::kShort || sd == at::kUInt16 ? 1 : -1;
    if (kind < 0) throw Miss{};
    if (a[17] != Py_None && state.numel() < mul_add(to_i64(a[17]), 1, heads * kD * kD)) throw Miss{};
    void* so = nullptr;
    if (PyUnicode_Check(a[10])) so = state.data_ptr();
    else if (a[10] != Py_None) {
        const at::Tensor& t = tensor(a[10]);
        if (!t.is_cuda() || t.scalar_type() != sd || t.numel() < state.numel()) throw Miss{};
        so = t.data_ptr();
    }
    const glm53f_bf16 *gate = nullptr, *norm_w = nullptr;
    if (a[12] != Py_None) {
        gate = need<const glm53f_bf16>(a[12], kBf16, n);
        norm_w = need<const glm53f_bf16>(a[13], kBf16, kD);
    } else if (a[13] != Py_None) {
        norm_w = static_cast<const glm53f_bf16*>(tensor(a[13]).data_ptr());
    }
    if (!PyFloat_CheckExact(a[14])) throw Miss{};
    const float eps = (float)PyFloat_AS_DOUBLE(a[14]);
    auto* out = need<glm53f_bf16>(a[15], kBf16, n);
    const auto st = reinterpret_cast<glm53f_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
    const void* si = state.data_ptr();
    // (the caller's frame holds the tensors)
    if (a[16] == Py_None)
        return unlocked([&] {
            return glm53f_kda_core_decode_batch((int32_t)heads, (int32_t)batch, cu, q, k, v, g, beta, si, so, off, kind, (int32_t)flags, gate, norm_w, eps, out, st);
        });
    if (!PyTuple_CheckExact(a[16]) || PyTuple_GET_SIZE(a[16]) != 4) throw Miss{};
    auto* ks = need<float>(PyTuple_GET_ITEM(a[16], 0), kF32, n);
    auto* vs = need<glm53f_bf16>(PyTuple_GET_ITEM(a[16], 1), kBf16, n);
    auto* gs = need<float>(PyTuple_GET_ITEM(a[16], 2), kF32, n);
    auto* bs = need<float>(PyTuple_GET_ITEM(a[16], 3), kF32, rows * heads);
    return unlocked([&] {
        return glm53f_kda_core_verify_batch((int32_t)heads, (int32_t)batch, cu, q, k, v, g, beta, si, so, off, kind, (int32_t)flags, gate, norm_w, eps, out, ks, vs,
                                            gs, bs, st);
    });
}

// ---- linear.py, spec.py and proj.fused: the modules hold the same checks, with their errors ---------------------------------------
inline int here() { return c10::cuda::current_device(); }
inline const at::Tensor& on_device(PyObject* o, int dev) {
    const at::Tensor& t = tensor(o);
    if (!t.is_cuda() || t.get_device() != dev) throw Miss{};
    return t;
}
template <typename T>
T* need_here(PyObject* o, Kind kind, int64_t n, int dev) {
    on_device(o, dev);
    return need<T>(o, kind, n);
}
inline bool is_bf16(const at::Tensor& t) {
    const auto d = t.scalar_type();
    return d == at::kBFloat16 || d == at::kShort || d == at::kUInt16;
}
// `rows` rows of heads x 128 bf16 values: [rows][heads x 128] or [rows][heads][128], rows any multiple of eight elements apart.
inline Rows head_rows(PyObject* o, int64_t rows, int64_t heads, int dev) {
    const at::Tensor& t = on_device(o, dev);
    const int64_t width = heads * kD;
    if (!is_bf16(t) || t.dim() < 2 || t.dim() > 3 || t.size(0) < rows) throw Miss{};
    if (t.dim() == 2 ? t.size(1) != width || t.stride(1) != 1 : t.size(1) != heads || t.size(2) != kD || t.stride(2) != 1 || (heads > 1 && t.stride(1) != kD)) throw Miss{};
    const int64_t stride = t.size(0) > 1 ? t.stride(0) : width;
    auto* at = static_cast<glm53f_bf16*>(t.data_ptr());
    if (stride % 8 || stride < width || (reinterpret_cast<uintptr_t>(at) & 15)) throw Miss{};
    return {at, stride};
}

// lin(prefill, heads, qk_heads, rows, max_len, cu_rows, q, k, v, g, state, state_off, keep, state_out, scale, out, workspace, max_state_off)
int lin(PyObject* const* a) {
    const bool prefill = a[0] == Py_True;
    const int64_t heads = to_i64(a[1]), qk = to_i64(a[2]), rows = to_i64(a[3]), max_len = to_i64(a[4]);
    if (heads < 1 || heads > 65535 || qk < 1 || heads % qk || rows < 1 || rows > 0x7fffffff || max_len < 0 || max_len > rows) throw Miss{};
    const int dev = here();
    const auto* cu = need_here<const int32_t>(a[5], kI32, 2, dev);
    const int64_t batch = tensor(a[5]).numel() - 1;
    if (batch > 65535) throw Miss{};
    const Rows q = head_rows(a[6], rows, qk, dev), k = head_rows(a[7], rows, qk, dev), v = head_rows(a[8], rows, heads, dev);
    const at::Tensor& g = on_device(a[9], dev);
    if (g.scalar_type() != at::kFloat || g.numel() == 0) throw Miss{};
    int64_t g_stride = 0;
    if (g.dim() == 1) {
        if (g.size(0) != heads || (heads > 1 && g.stride(0) != 1)) throw Miss{};
    } else {
        if (g.dim() != 2 || g.size(0) < rows || g.size(1) != heads || (heads > 1 && g.stride(1) != 1)) throw Miss{};
        g_stride = g.size(0) > 1 ? g.stride(0) : heads;
        if (g_stride < heads) throw Miss{};
    }
    const at::Tensor& state = on_device(a[10], dev);
    const bool f32 = state.scalar_type() == at::kFloat;
    if ((!f32 && !is_bf16(state)) || !state.is_contiguous()) throw Miss{};
    const auto* off = need_here<const int64_t>(a[11], kI64, batch, dev);
    const auto* keep = a[12] == Py_None ? nullptr : need_here<const int32_t>(a[12], kI32, batch, dev);
    if (a[17] != Py_None) {
        const int64_t most = to_i64(a[17]);
        if (most < 0 || state.numel() < mul_add(most, 1, heads * kD * kD)) throw Miss{};
    }
    void *si = state.data_ptr(), *so = nullptr;
    if (PyUnicode_Check(a[13])) {
        so = si;
    } else if (a[13] != Py_None) {
        const at::Tensor& t = on_device(a[13], dev);
        if (t.scalar_type() != state.scalar_type() || t.numel() < state.numel() || !t.is_contiguous()) throw Miss{};
        so = t.data_ptr();
        const auto x = reinterpret_cast<uintptr_t>(si), y = reinterpret_cast<uintptr_t>(so);
        if (x != y && y < x + state.nbytes() && x < y + t.nbytes()) throw Miss{};
    }
    double scale = 0.08838834764831845;
    if (a[14] != Py_None) {
        if (!PyFloat_CheckExact(a[14])) throw Miss{};
        scale = PyFloat_AS_DOUBLE(a[14]);
    }
    const Rows out = a[15] == Py_None ? Rows{nullptr, 0} : head_rows(a[15], rows, heads, dev);
    const auto st = reinterpret_cast<glm53f_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
    const auto* gp = static_cast<const float*>(g.data_ptr());
    if (!prefill) {
        if (so == nullptr && out.ptr == nullptr) throw Miss{};
        return unlocked([&] {
            return glm53f_kda_lin_decode_batch((int32_t)heads, (int32_t)qk, (int32_t)batch, cu, keep, q.ptr, q.stride, k.ptr, k.stride, v.ptr, v.stride, gp, g_stride,
                                               si, so, off, f32 ? 0 : 1, (float)scale, out.ptr, out.stride, st);
        });
    }
    if (so == nullptr || out.ptr == nullptr) throw Miss{};
    void* ws = nullptr;
    int64_t bytes = 0;
    if (a[16] != Py_None) {
        const at::Tensor& w = on_device(a[16], dev);
        if (!w.is_contiguous()) throw Miss{};
        bytes = (int64_t)w.nbytes();
        ws = bytes != 0 ? w.data_ptr() : nullptr;
    }
    return unlocked([&] {
        return glm53f_kda_lin_prefill_varlen((int32_t)heads, (int32_t)qk, (int32_t)batch, cu, (int32_t)rows, (int32_t)max_len, q.ptr, q.stride, k.ptr, k.stride, v.ptr,
                                             v.stride, gp, g_stride, si, so, off, f32 ? 0 : 1, (float)scale, out.ptr, out.stride, ws, bytes, st);
    });
}

// accept(cu_rows, tokens, target, u, keep, next, probabilities, draft, temperature)
int accept(PyObject* const* a) {
    const int dev = here();
    const auto* cu = need_here<const int32_t>(a[0], kI32, 2, dev);
    const int64_t batch = tensor(a[0]).numel() - 1;
    const auto* tokens = need_here<const int32_t>(a[1], kI32, 1, dev);
    const int64_t rows = tensor(a[1]).numel();
    if (batch > 0xffffff || (a[6] != Py_True && a[6] != Py_False)) throw Miss{};
    const bool probabilities = a[6] == Py_True;
    auto matrix = [&](PyObject* o, int64_t vocab, int64_t& ld) -> const at::Tensor& {
        const at::Tensor& t = on_device(o, dev);
        if (t.dim() != 2 || t.size(0) < rows || t.size(1) < 1 || t.size(1) > 0x7fffffff || (vocab > 0 && t.size(1) != vocab) || (t.size(1) > 1 && t.stride(1) != 1))
            throw Miss{};
        ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
        if (ld < t.size(1)) throw Miss{};
        return t;
    };
    int64_t ld = 0, draft_ld = 0;
    const at::Tensor& target = matrix(a[2], 0, ld);
    const int64_t vocab = target.size(1);
    const bool f32 = target.scalar_type() == at::kFloat;
    if (!f32 && (probabilities || target.scalar_type() != at::kBFloat16)) throw Miss{};
    const float *draft = nullptr, *temperature = nullptr;
    if (a[7] != Py_None) {
        const at::Tensor& d = matrix(a[7], vocab, draft_ld);
        if (d.scalar_type() != at::kFloat) throw Miss{};
        draft = static_cast<const float*>(d.data_ptr());
    }
    if (a[8] != Py_None) {
        if (probabilities) throw Miss{};
        temperature = need_here<const float>(a[8], kF32, batch, dev);
    }
    const auto* u = need_here<const float>(a[3], kF32, rows, dev);
    auto *keep = need_here<int32_t>(a[4], kI32, batch, dev), *next = need_here<int32_t>(a[5], kI32, batch, dev);
    const auto st = reinterpret_cast<glm53f_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
    const void* tp = target.data_ptr();
    const int32_t kind = probabilities ? GLM53F_KDA_PROBABILITIES : f32 ? GLM53F_KDA_LOGITS_F32 : GLM53F_KDA_LOGITS_BF16;
    return unlocked([&] { return glm53f_kda_accept_batch((int32_t)batch, cu, (int32_t)vocab, tp, kind, ld, tokens, draft, draft_ld, temperature, u, keep, next, st); });
}

// proj_fused(x, ldx, x_gstride, w, n, k, ldw, groups, w_gstride, rows, out, ldo, o_gstride, out_f32, x_offset, out_offset, bias, activation, residual, ldr, r_gstride,
// residual_offset)
int proj_fused(PyObject* const* a) {
    const int dev = here();
    const at::Tensor &x = on_device(a[0], dev), &w = on_device(a[3], dev), &out = on_device(a[10], dev);
    const int64_t ldx = to_i64(a[1]), xg = to_i64(a[2]), n = to_i64(a[4]), k = to_i64(a[5]), ldw = to_i64(a[6]), groups = to_i64(a[7]), wg = to_i64(a[8]),
                  rows = to_i64(a[9]), ldo = to_i64(a[11]), og = to_i64(a[12]), x_offset = to_i64(a[14]), o_offset = to_i64(a[15]), act = to_i64(a[17]);
    const bool f32 = a[13] == Py_True;
    if (!f32 && a[13] != Py_False) throw Miss{};
    for (int64_t v : {ldx, xg, n, k, ldw, groups, wg, rows, ldo, og, x_offset, o_offset})
        if (v < 0 || v > 0x3fffffffffll) throw Miss{};
    if (groups < 1 || rows < 1 || n < 1 || k < 1 || groups > 0xffff || rows > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff) throw Miss{};
    auto fits = [&](const at::Tensor& t, int64_t offset, int64_t gs, int64_t r, int64_t ld, int64_t width) {
        return mul_add(groups - 1, gs, mul_add(r - 1, ld, mul_add(offset, 1, width))) <= t.numel();
    };
    if (!is_bf16(x) || !is_bf16(w) || (f32 ? out.scalar_type() != at::kFloat : out.element_size() != 2)) throw Miss{};
    if (!fits(x, x_offset, xg, rows, ldx, k) || !fits(w, 0, wg, n, ldw, k) || !fits(out, o_offset, og, rows, ldo, n)) throw Miss{};
    glm53f_proj_epilogue e{};
    if (act < GLM53F_PROJ_NONE || act > GLM53F_PROJ_SIGMOID) throw Miss{};
    e.activation = (int32_t)act;
    if (a[16] != Py_None) {
        const at::Tensor& b = on_device(a[16], dev);
        e.bias_f32 = b.scalar_type() == at::kFloat;
        if ((!e.bias_f32 && !is_bf16(b)) || !b.is_contiguous() || b.numel() != groups * n) throw Miss{};
        e.bias = b.data_ptr();
        e.bias_gstride = n;
    }
    if (a[18] != Py_None) {
        const at::Tensor& r = on_device(a[18], dev);
        e.ldr = a[19] == Py_None ? ldo : to_i64(a[19]);
        e.r_gstride = a[20] == Py_None ? og : to_i64(a[20]);
        const int64_t offset = to_i64(a[21]);
        if (f32 ? r.scalar_type() != at::kFloat : !is_bf16(r)) throw Miss{};
        if (offset < 0 || e.ldr < n || e.r_gstride < 0 || !fits(r, offset, e.r_gstride, rows, e.ldr, n)) throw Miss{};
        e.residual = static_cast<const unsigned char*>(r.data_ptr()) + offset * r.element_size();
    }
    const glm53f_proj_job job{static_cast<const uint16_t*>(x.data_ptr()) + x_offset, ldx, xg, static_cast<const uint16_t*>(w.data_ptr()), ldw, wg, (int32_t)groups,
                              (int32_t)rows, (int32_t)n, (int32_t)k, static_cast<unsigned char*>(out.data_ptr()) + o_offset * out.element_size(), f32 ? 1 : 0, ldo, og};
    const auto st = reinterpret_cast<glm53f_stream_t>(c10::cuda::getCurrentCUDAStream().stream());
    return unlocked([&] { return glm53f_kda_proj_bf16_fused(&job, &e, st); });
}

template <typename F>
PyObject* answer(F&& f) {
    long code = -1;
    try {
        code = f();
    } catch (const Miss&) {
        PyErr_Clear();
        code = -1;
    } catch (const std::exception&) {
        PyErr_Clear();
        code = -1;
    }
    return PyLong_FromLong(code);
}

PyObject* py_chain_batch(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return answer([&] { return n == 4 && T_chain != nullptr ? chain_batch(args[0], args[1], args[2], args[3] == Py_True) : -1; });
}
PyObject* py_core_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return answer([&] { return n == 18 ? core_decode(args) : -1; });
}
PyObject* py_lin(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return answer([&] { return n == 18 ? lin(args) : -1; });
}
PyObject* py_accept(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return answer([&] { return n == 9 ? accept(args) : -1; });
}
PyObject* py_proj_fused(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return answer([&] { return n == 22 ? proj_fused(args) : -1; });
}
// raw_stream(Stream) -> the CUDA stream's address, or None for a stream it does not know.
PyObject* py_raw_stream(PyObject*, PyObject* s) {
    try {
        return PyLong_FromVoidPtr(stream_of(s));
    } catch (const std::exception&) {
    } catch (const Miss&) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}
// bind(DeviceBuffer, RowView, Weights, Saves, ChainBatch, BatchMeta, Stream): the types the fast path accepts, exactly.
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "bind takes seven types");
        return nullptr;
    }
    PyObject** slots[7] = {&T_buffer, &T_view, &T_weights, &T_saves, &T_chain, &T_meta, &T_stream};
    for (int i = 0; i < 7; ++i) {
        Py_INCREF(args[i]);
        Py_XDECREF(*slots[i]);
        *slots[i] = args[i];
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_bind)), METH_FASTCALL, nullptr},
    {"chain_batch", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_chain_batch)), METH_FASTCALL, nullptr},
    {"raw_stream", py_raw_stream, METH_O, nullptr},
    {"core_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_core_decode)), METH_FASTCALL, nullptr},
    {"lin", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_lin)), METH_FASTCALL, nullptr},
    {"accept", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_accept)), METH_FASTCALL, nullptr},
    {"proj_fused", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_proj_fused)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Native host path of the per-layer launches.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
#define NAME(field, text) N.field = PyUnicode_InternFromString(text)
    NAME(t, "t"); NAME(buf, "buf"); NAME(offset, "offset"); NAME(stride, "stride"); NAME(weights, "weights"); NAME(heads, "heads"); NAME(conv_w, "conv_w");
    NAME(a_log, "a_log"); NAME(dt_bias, "dt_bias"); NAME(norm_w, "norm_w"); NAME(eps, "eps"); NAME(lower, "lower"); NAME(p, "p"); NAME(b_off, "b_off");
    NAME(a, "a"); NAME(g, "g"); NAME(conv, "conv"); NAME(state, "state"); NAME(state_out, "state_out"); NAME(out, "out"); NAME(saves, "saves");
    NAME(kind, "kind"); NAME(rows, "rows"); NAME(k, "k"); NAME(v, "v"); NAME(b, "b"); NAME(fast, "_extent"); NAME(cu_rows, "cu_rows");
    NAME(conv_off, "conv_off"); NAME(state_off, "state_off"); NAME(stream, "stream"); NAME(cuda_stream, "cuda_stream");
#undef NAME
    PyObject* m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", HOST_BUILT_FOR) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
