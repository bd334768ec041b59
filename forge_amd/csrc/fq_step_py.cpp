// fq_step_py.cpp -- forge_amd._step: the host side of forge_amd/step.py, from tensors
// to the C ABI of include/forge_step.h.  Checks of arguments, outputs' allocation and the call
// in one native function each: of small calls' time the host's part is the
// larger (rotation of one token: 9.9 us a call through Python checks and ctypes, kernel 2.4).
//
// step.py documents the functions; the last argument of each is the stream.  The C ABI's
// calls go to the current device, which is the tensors' while one runs.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <optional>
#include <string>

#include "../../include/forge_step.h"

namespace {

struct Refused {
    std::string what;
};
[[noreturn]] void refuse(const std::string& what) { throw Refused{what}; }

const char* type_name(at::ScalarType t) {
    return t == at::kInt ? "int32" : t == at::kLong ? "int64" : t == at::kFloat ? "fp32" : "other";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

// Makes a device the current one, and the one before again at its end.  (Nothing to do
// where there is one device: 0.13 us of a call's 5.)
struct On {
    std::optional<c10::DeviceGuard> guard;
    explicit On(c10::Device d) {
        static const bool several = c10::impl::VirtualGuardImpl(d.type()).deviceCount() > 1;
        if (several) guard.emplace(d);
    }
};

// The address of a contiguous tensor of that type and shape on device dev; NULL for None.
void* vec(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef shape, int64_t dev) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_cuda() || t.get_device() != dev ||
        !t.is_contiguous()) {
        std::string s;
        for (int64_t n : shape) s += (s.empty() ? "" : ", ") + std::to_string(n);
        refuse(std::string(name) + " must be a contiguous " + type_name(type) + " tensor of shape [" + s +
               "] on cuda:" + std::to_string(dev));
    }
    return t.data_ptr();
}
void* required(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef shape, int64_t dev) {
    if (o == Py_None) refuse(std::string(name) + " must be a tensor");
    return vec(o, name, type, shape, dev);
}

int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw 0;
    return v;
}
int narrow_int(PyObject* o, const char* name) {
    const int64_t v = integer(o);
    if (v < INT32_MIN || v > INT32_MAX) refuse(std::string(name) + " is out of range");
    return (int)v;
}
int to_int(int64_t v, const char* name) {
    if (v > INT32_MAX) refuse(std::string(name) + " is too large");
    return (int)v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw 0;
    return v;
}

struct Table {
    int32_t* p;
    int cols;
    int64_t stride;
};
Table table(PyObject* o, const char* name, int64_t rows, int64_t dev) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() != 2 || t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != dev ||
        t.size(0) != rows || t.size(1) < 1 || (t.stride(1) != 1 && t.size(1) != 1) ||
        (t.stride(0) < t.size(1) && rows > 1))
        refuse(std::string(name) + " must be an int32 block table of " + std::to_string(rows) +
               " rows on cuda:" + std::to_string(dev));
    return {static_cast<int32_t*>(t.data_ptr()), to_int(t.size(1), name), std::max(t.stride(0), t.size(1))};
}

struct Cache {
    uint32_t type;
    void *k, *v;
    float *ks, *vs;  // of caches of 8 bits
    int blocks, block_size, heads, D;
    int64_t sb, st, sh;
};
// A cache's elements or codes, and its scales (None in 16 bits).
struct Halves {
    PyObject *data, *scales;
};
Halves halves(PyObject* o) {
    if (!PyTuple_Check(o)) return {o, Py_None};
    if (PyTuple_GET_SIZE(o) != 2) refuse("a cache of 8 bits is (codes, scales)");
    return {PyTuple_GET_ITEM(o, 0), PyTuple_GET_ITEM(o, 1)};
}
Cache cache(PyObject* ko, PyObject* vo, const std::string& name, int64_t dev) {
    const Halves kh = halves(ko), vh = halves(vo);
    const at::Tensor &k = tensor(kh.data, "k_cache"), &v = tensor(vh.data, "v_cache");
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides() ||
        k.scalar_type() != v.scalar_type() || !k.is_cuda() || k.get_device() != dev || !v.is_cuda() ||
        v.get_device() != dev)
        refuse(name + ": caches must be 4D [blocks, block size, kv heads, D], alike, on cuda:" +
               std::to_string(dev));
    const bool codes = kh.scales != Py_None || vh.scales != Py_None;
    if (codes ? k.scalar_type() != at::kChar : k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16)
        refuse(name + ": caches must be fp16 or bf16, or Cache8 of int8 codes and scales");
    if (k.stride(3) != 1 && k.size(3) != 1) refuse(name + ": a cached head must be contiguous");
    Cache c{codes ? FQ_TYPE_I8 : k.scalar_type() == at::kHalf ? FQ_TYPE_F16 : FQ_TYPE_BF16, k.data_ptr(), v.data_ptr(),
            nullptr, nullptr, to_int(k.size(0), "k_cache"), to_int(k.size(1), "k_cache"), to_int(k.size(2), "k_cache"),
            to_int(k.size(3), "k_cache"), k.stride(0), k.stride(1), k.stride(2)};
    if (codes) {
        const std::array<int64_t, 3> shape{k.size(0), k.size(2), k.size(1) / 16};
        c.ks = static_cast<float*>(required(kh.scales, "k_cache's scales", at::kFloat, shape, dev));
        c.vs = static_cast<float*>(required(vh.scales, "v_cache's scales", at::kFloat, shape, dev));
    }
    return c;
}

void check(int status, const char* what) {
    if (status == FQ_OK) return;
    PyObject* lib = PyImport_ImportModule("forge_amd._lib");  // FqError and its text
    if (lib) {
        PyObject* r = PyObject_CallMethod(lib, "check", "is", status, what);
        Py_XDECREF(r);
        Py_DECREF(lib);
    }
    throw 0;
}

void* stream(PyObject* o) {
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw 0;
    return p;
}

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
    PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
    if (!t) throw 0;
    Py_ssize_t i = 0;
    for (const at::Tensor& x : ts) {
        PyObject* o;
        if (x.defined()) {
            o = THPVariable_Wrap(x);
        } else {
            o = Py_None;
            Py_INCREF(o);
        }
        if (!o) {
            Py_DECREF(t);
            throw 0;
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

// Runs f, turning what it throws into a Python error.
template <class F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F&& f) {
    if (have != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are wanted", have, want);
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_RuntimeError, r.what.c_str());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "forge_amd._step: failed");
    }
    return nullptr;
}

// plan(lengths, new_tokens, block_table, free_blocks, block_size, n_tokens, parents, stream)
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const at::Tensor& lengths = tensor(a[0], "plan_step: lengths");
        if (!lengths.is_cuda() || lengths.dim() != 1)
            refuse("plan_step: lengths must be a 1D device tensor");
        const int64_t B = lengths.size(0), dev = lengths.get_device();
        const On on(lengths.device());
        const int N = narrow_int(a[5], "plan_step: n_tokens");
        if (N < 0) refuse("plan_step: n_tokens must not be negative");
        auto* ln = static_cast<int32_t*>(required(a[0], "plan_step: lengths", at::kInt, {B}, dev));
        auto* nw = static_cast<int32_t*>(required(a[1], "plan_step: new_tokens", at::kInt, {B}, dev));
        const Table t = table(a[2], "plan_step: block_table", B, dev);
        const int64_t F = tensor(a[3], "plan_step: free_blocks").numel();
        auto* fr = static_cast<int32_t*>(required(a[3], "plan_step: free_blocks", at::kInt, {F}, dev));
        auto* pa = static_cast<int32_t*>(vec(a[6], "plan_step: parents", at::kInt, {N}, dev));
        at::Tensor masks;
        if (a[6] != Py_None) masks = at::empty({N}, lengths.options().dtype(at::kLong));
        const at::Tensor out = at::empty({B + 3 + 2 * (int64_t)N}, lengths.options());  // one allocation
        auto* o = static_cast<int32_t*>(out.data_ptr());
        check(fq_plan_step(ln, nw, pa, to_int(B, "plan_step: lengths"), N, narrow_int(a[4], "plan_step: block_size"), t.p,
                           t.cols, t.stride, fr, to_int(F, "plan_step: free_blocks"), o, o + B + 3, o + B + 3 + N,
                           masks.defined() ? static_cast<uint64_t*>(masks.data_ptr()) : nullptr, o + B + 1, stream(a[7])),
              "plan_step");
        return tuple_of({out.narrow(0, 0, B + 1), out.narrow(0, B + 3, N), out.narrow(0, B + 3 + N, N), masks,
                         out.narrow(0, B + 1, 2)});
    });
}

// rope(qkv, positions, slots, table, k_cache, v_cache, bias, q_weight, k_weight, eps, interleaved, stream)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        const at::Tensor& x = tensor(a[0], "qk_norm_rope: qkv");
        if (x.dim() != 2 || !x.is_cuda() || x.scalar_type() != at::kFloat || (x.stride(1) != 1 && x.size(1) != 1))
            refuse("qk_norm_rope: qkv must be a 2D fp32 device tensor of contiguous rows");
        const int64_t N = x.size(0), width = x.size(1), dev = x.get_device();
        const On on(x.device());
        const Cache c = cache(a[4], a[5], "qk_norm_rope", dev);
        const int64_t hq = c.D ? width / c.D - 2 * (int64_t)c.heads : 0;
        if (hq < 1 || width % c.D || c.heads < 1 || hq % c.heads)
            refuse("qk_norm_rope: rows of " + std::to_string(width) + " do not hold heads of " +
                   std::to_string(c.D) + " for " + std::to_string(c.heads) + " kv heads");
        const at::Tensor& t = tensor(a[3], "qk_norm_rope: table");
        if (t.dim() != 2 || t.scalar_type() != at::kFloat || !t.is_contiguous() || !t.is_cuda() ||
            t.get_device() != dev)
            refuse("qk_norm_rope: table must be a contiguous fp32 [positions, rot] on cuda:" +
                   std::to_string(dev));
        const auto f32 = [&](PyObject* o, const char* name, int64_t len) {
            return static_cast<const float*>(vec(o, name, at::kFloat, {len}, dev));
        };
        const float* bias = f32(a[6], "qk_norm_rope: bias", width);
        const float* qw = f32(a[7], "qk_norm_rope: q_weight", c.D);
        const float* kw = f32(a[8], "qk_norm_rope: k_weight", c.D);
        auto* pos = static_cast<int32_t*>(required(a[1], "qk_norm_rope: positions", at::kInt, {N}, dev));
        auto* slots = static_cast<int32_t*>(required(a[2], "qk_norm_rope: slots", at::kInt, {N}, dev));
        const int inter = PyObject_IsTrue(a[10]);
        if (inter < 0) throw 0;
        at::Tensor q = at::empty({N, hq, c.D}, x.options());
        const float* xp = static_cast<const float*>(x.data_ptr());
        const int64_t ld = N > 1 ? x.stride(0) : width;
        const int rows = to_int(N, "qk_norm_rope: qkv"), heads = to_int(hq, "qk_norm_rope: qkv");
        const int rot = to_int(t.size(1), "qk_norm_rope: table"), known = to_int(t.size(0), "qk_norm_rope: table");
        const float* tp = static_cast<const float*>(t.data_ptr());
        float* qp = static_cast<float*>(q.data_ptr());
        const float eps = (float)number(a[9]);
        check(c.type == FQ_TYPE_I8
                  ? fq_qk_norm_rope8(xp, ld, rows, heads, c.heads, c.D, rot, inter, bias, qw, kw, eps, pos, slots, tp,
                                     known, qp, static_cast<int8_t*>(c.k), static_cast<int8_t*>(c.v), c.ks, c.vs,
                                     c.blocks, c.block_size, c.sb, c.st, c.sh, stream(a[11]))
                  : fq_qk_norm_rope(xp, ld, rows, heads, c.heads, c.D, rot, inter, bias, qw, kw, eps, pos, slots, tp,
                                    known, qp, c.type, c.k, c.v, c.blocks, c.block_size, c.sb, c.st, c.sh, stream(a[11])),
              "qk_norm_rope");
        return THPVariable_Wrap(q);
    });
}

// attention(q, k_cache, v_cache, block_table, lengths, cu, masks, max_new, scale, window, sinks, stream)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        const at::Tensor& q = tensor(a[0], "tree_attention: q");
        if (q.dim() != 3 || !q.is_cuda() || q.scalar_type() != at::kFloat)
            refuse("tree_attention: q must be a 3D fp32 device tensor");
        const int64_t N = q.size(0), hq = q.size(1), D = q.size(2), dev = q.get_device();
        const On on(q.device());
        if ((q.stride(2) != 1 && D != 1) || (hq != 1 && q.stride(1) != D))
            refuse("tree_attention: a token's queries must be contiguous");
        const Cache c = cache(a[1], a[2], "tree_attention", dev);
        if (c.D != D || c.heads < 1 || hq % c.heads)
            refuse("tree_attention: " + std::to_string(hq) + " heads of " + std::to_string(D) + " do not share " +
                   std::to_string(c.heads) + " kv heads of " + std::to_string(c.D));
        const int64_t B = tensor(a[4], "tree_attention: lengths").numel();
        auto* ln = static_cast<int32_t*>(required(a[4], "tree_attention: lengths", at::kInt, {B}, dev));
        auto* cu = static_cast<int32_t*>(required(a[5], "tree_attention: cu", at::kInt, {B + 1}, dev));
        auto* masks = static_cast<uint64_t*>(vec(a[6], "tree_attention: masks", at::kLong, {N}, dev));
        const Table t = table(a[3], "tree_attention: block_table", B, dev);
        const int64_t hint = a[7] == Py_None ? (B ? (N + B - 1) / B : 0) : std::min(integer(a[7]), N);
        const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)D) : number(a[8]);
        const int64_t window = a[9] == Py_None ? 0 : integer(a[9]), sinks = integer(a[10]);
        if (a[9] != Py_None && window < 1) refuse("tree_attention: a window has a token at least");
        if (sinks < 0 || (sinks && !window)) refuse("tree_attention: sinks are the first tokens beside a window");
        at::Tensor out = at::empty({N, hq, D}, q.options());
        check(fq_window_attention(static_cast<const float*>(q.data_ptr()), N > 1 ? q.stride(0) : hq * D, ln, cu, masks,
                                  to_int(B, "tree_attention: lengths"), to_int(N, "tree_attention: q"),
                                  to_int(std::max<int64_t>(hint, -1), "tree_attention: max_new"),
                                  to_int(hq, "tree_attention: q"), c.heads, c.D, (float)scale,
                                  (int)std::min<int64_t>(window, INT32_MAX), (int)std::min<int64_t>(sinks, INT32_MAX),
                                  c.type, c.k, c.v, c.ks, c.vs, c.blocks, c.block_size, c.sb, c.st, c.sh, t.p, t.cols,
                                  t.stride, static_cast<float*>(out.data_ptr()), stream(a[11])),
              "tree_attention");
        return THPVariable_Wrap(out);
    });
}

// logprobs(logits, targets, top, stream)
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&] {
        const at::Tensor& x = tensor(a[0], "token_logprobs: logits");
        const auto st = x.scalar_type();
        if (x.dim() != 2 || !x.is_cuda() || (st != at::kFloat && st != at::kHalf && st != at::kBFloat16) ||
            (x.stride(1) != 1 && x.size(1) != 1))
            refuse("token_logprobs: logits must be a 2D fp32, fp16 or bf16 device tensor of contiguous rows");
        const int64_t M = x.size(0), V = x.size(1), dev = x.get_device(), top = integer(a[2]);
        const On on(x.device());
        if (top < 0 || top > std::min<int64_t>(64, V))
            refuse("token_logprobs: top must be at most " + std::to_string(std::min<int64_t>(64, V)));
        const auto f32 = x.options().dtype(at::kFloat);
        at::Tensor lp, tl, tt;
        int32_t* targets = nullptr;
        int64_t J = 0;
        if (a[1] != Py_None) {
            const at::Tensor& t = tensor(a[1], "token_logprobs: targets");
            if (t.dim() != 1 && t.dim() != 2) refuse("token_logprobs: targets must be [M] or [M, J]");
            J = t.dim() == 1 ? 1 : t.size(1);
            const int64_t shape[2] = {M, J};
            targets = static_cast<int32_t*>(
                vec(a[1], "token_logprobs: targets", at::kInt, at::IntArrayRef(shape, (size_t)t.dim()), dev));
            lp = at::empty(t.sizes(), f32);
        }
        at::Tensor entropy = at::empty({M}, f32);
        if (top) {
            tl = at::empty({M, top}, f32);
            tt = at::empty({M, top}, f32.dtype(at::kInt));
        }
        const auto p = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
        check(fq_token_logprobs(x.data_ptr(), st == at::kFloat ? FQ_TYPE_F32 : st == at::kHalf ? FQ_TYPE_F16 : FQ_TYPE_BF16,
                                M > 1 ? x.stride(0) : V, to_int(M, "token_logprobs: logits"),
                                to_int(V, "token_logprobs: logits"), targets, to_int(J, "token_logprobs: targets"), (int)top,
                                static_cast<float*>(p(lp)), static_cast<float*>(p(entropy)),
                                static_cast<float*>(p(tl)), static_cast<int32_t*>(p(tt)), stream(a[3])),
              "token_logprobs");
        return tuple_of({lp, entropy, tl, tt});
    });
}

// read(k_cache, v_cache, block_table, starts, n_tokens, type, first, stream)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const at::Tensor& starts = tensor(a[3], "read_cache: starts");
        if (!starts.is_cuda() || starts.dim() != 1 || starts.size(0) < 2)
            refuse("read_cache: starts must be a 1D device tensor of two and more");
        const int64_t B = starts.size(0) - 1, dev = starts.get_device();
        const On on(starts.device());
        const Cache c = cache(a[0], a[1], "read_cache", dev);
        if (c.type != FQ_TYPE_I8) refuse("read_cache: caches must be Cache8 of int8 codes and scales");
        const Table t = table(a[2], "read_cache: block_table", B, dev);
        auto* st = static_cast<int32_t*>(required(a[3], "read_cache: starts", at::kInt, {B + 1}, dev));
        auto* first = static_cast<int32_t*>(vec(a[6], "read_cache: first", at::kInt, {B}, dev));
        const int N = narrow_int(a[4], "read_cache: n_tokens");
        if (N < 0) refuse("read_cache: n_tokens must not be negative");
        const uint32_t type = (uint32_t)integer(a[5]);
        const auto options = starts.options().dtype(type == FQ_TYPE_F32 ? at::kFloat
                                                    : type == FQ_TYPE_F16 ? at::kHalf : at::kBFloat16);
        at::Tensor k = at::empty({N, c.heads, c.D}, options), v = at::empty({N, c.heads, c.D}, options);
        check(fq_read_cache8(static_cast<int8_t*>(c.k), static_cast<int8_t*>(c.v), c.ks, c.vs, c.blocks, c.block_size,
                             c.heads, c.D, c.sb, c.st, c.sh, t.p, t.cols, t.stride, st, first,
                             to_int(B, "read_cache: starts"), N, type, k.data_ptr(), v.data_ptr(), stream(a[7])),
              "read_cache");
        return tuple_of({k, v});
    });
}

// keep(k_cache, v_cache, block_table, lengths, cu, path, accepted, stream)
PyObject* keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const at::Tensor& lengths = tensor(a[3], "keep_accepted: lengths");
        if (!lengths.is_cuda() || lengths.dim() != 1) refuse("keep_accepted: lengths must be a 1D device tensor");
        const int64_t B = lengths.size(0), dev = lengths.get_device();
        const On on(lengths.device());
        const Cache c = cache(a[0], a[1], "keep_accepted", dev);
        const Table t = table(a[2], "keep_accepted: block_table", B, dev);
        auto* ln = static_cast<int32_t*>(required(a[3], "keep_accepted: lengths", at::kInt, {B}, dev));
        auto* cu = static_cast<int32_t*>(required(a[4], "keep_accepted: cu", at::kInt, {B + 1}, dev));
        const int64_t N = tensor(a[5], "keep_accepted: path").numel();
        auto* path = static_cast<int32_t*>(required(a[5], "keep_accepted: path", at::kInt, {N}, dev));
        auto* acc = static_cast<int32_t*>(required(a[6], "keep_accepted: accepted", at::kInt, {B}, dev));
        check(fq_keep_accepted(c.type, c.k, c.v, c.ks, c.vs, c.blocks, c.block_size, c.heads, c.D, c.sb, c.st, c.sh,
                               t.p, t.cols, t.stride, ln, cu, path, acc, to_int(B, "keep_accepted: lengths"),
                               to_int(N, "keep_accepted: path"), stream(a[7])),
              "keep_accepted");
        Py_RETURN_NONE;
    });
}

// verify(logits, tokens, cu, uniforms, parents, draft_probs, temperature, stream)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const at::Tensor& x = tensor(a[0], "verify_draft: logits");
        const auto st = x.scalar_type();
        if (x.dim() != 2 || !x.is_cuda() || (st != at::kFloat && st != at::kHalf && st != at::kBFloat16) ||
            (x.stride(1) != 1 && x.size(1) != 1))
            refuse("verify_draft: logits must be a 2D fp32, fp16 or bf16 device tensor of contiguous rows");
        const int64_t N = x.size(0), V = x.size(1), dev = x.get_device();
        const On on(x.device());
        const int64_t B = tensor(a[2], "verify_draft: cu").numel() - 1;
        if (B < 1) refuse("verify_draft: cu must have two numbers and more");
        auto* tokens = static_cast<int32_t*>(required(a[1], "verify_draft: tokens", at::kInt, {N}, dev));
        auto* cu = static_cast<int32_t*>(required(a[2], "verify_draft: cu", at::kInt, {B + 1}, dev));
        auto* u = static_cast<float*>(required(a[3], "verify_draft: uniforms", at::kFloat, {N}, dev));
        auto* parents = static_cast<int32_t*>(vec(a[4], "verify_draft: parents", at::kInt, {N}, dev));
        auto* temperature = static_cast<float*>(vec(a[6], "verify_draft: temperature", at::kFloat, {B}, dev));
        const float* q = nullptr;
        int64_t ldq = V;
        if (a[5] != Py_None) {
            const at::Tensor& d = tensor(a[5], "verify_draft: draft_probs");
            if (d.dim() != 2 || !d.is_cuda() || d.get_device() != dev || d.scalar_type() != at::kFloat ||
                d.size(0) != N || d.size(1) != V || (d.stride(1) != 1 && V != 1))
                refuse("verify_draft: draft_probs must be fp32 [" + std::to_string(N) + ", " + std::to_string(V) +
                       "] of contiguous rows on cuda:" + std::to_string(dev));
            if (parents) refuse("verify_draft: draft_probs come with chains, not with parents");
            q = static_cast<const float*>(d.data_ptr());
            if (N > 1) ldq = d.stride(0);
        }
        const at::Tensor out = at::empty({2 * B + N}, x.options().dtype(at::kInt));  // one allocation
        auto* o = static_cast<int32_t*>(out.data_ptr());
        check(fq_verify_draft(x.data_ptr(), st == at::kFloat ? FQ_TYPE_F32 : st == at::kHalf ? FQ_TYPE_F16 : FQ_TYPE_BF16,
                              N > 1 ? x.stride(0) : V, to_int(V, "verify_draft: logits"), tokens, cu,
                              to_int(B, "verify_draft: cu"), to_int(N, "verify_draft: logits"), parents, u, q, ldq,
                              temperature, o, o + 2 * B, o + B, stream(a[7])),
              "verify_draft");
        return tuple_of({out.narrow(0, 0, B), out.narrow(0, 2 * B, N), out.narrow(0, B, B)});
    });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<plan>("plan"), method<rope>("rope"), method<attention>("attention"),
                         method<logprobs>("logprobs"), method<read>("read"), method<keep>("keep"),
                         method<verify>("verify"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "forge_amd._step", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step() { return PyModule_Create(&module); }
