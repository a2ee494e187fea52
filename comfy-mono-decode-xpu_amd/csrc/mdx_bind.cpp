// mdx._bind: the paged cache's calls and verify_drafts from Python without a Python-level check of every operand. The module
// checks torch tensors (type, shape, strides, device), takes outputs and workspaces from torch's allocator and calls libmdx's C
// entry points on the current stream of the tensors' device. These calls are a few microseconds of GPU work in a serving loop
// that captures no graph: with the checks in Python a call of attn_paged took 14.5 us of host time, two thirds of them
// outside the launches.
//
// The entry points come as addresses from mdx._lib (init), so that one loaded libmdx serves both bindings. Every C++
// exception becomes a Python one. Built into mdx/_bind.so by build.py.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/mdx.h"

namespace {

struct Entries {
    decltype(&mdx_last_error) last_error;
    decltype(&mdx_page_fork_workspace) fork_workspace;
    decltype(&mdx_page_fork) fork;
    decltype(&mdx_page_commit_workspace) commit_workspace;
    decltype(&mdx_page_commit) commit;
    decltype(&mdx_attn_paged_workspace) paged_workspace;
    decltype(&mdx_attn_paged) paged;
    decltype(&mdx_attn_blocks_workspace) blocks_workspace;
    decltype(&mdx_attn_blocks) blocks;
    decltype(&mdx_verify_drafts_workspace) verify_workspace;
    decltype(&mdx_verify_drafts) verify;
    decltype(&mdx_attn_window_workspace) window_workspace;
    decltype(&mdx_attn_window) window;
    decltype(&mdx_attn_mass_workspace) mass_workspace;
    decltype(&mdx_attn_mass) mass;
    decltype(&mdx_page_evict_workspace) evict_workspace;
    decltype(&mdx_page_evict) evict;
} g;
constexpr int ENTRIES = 17;
PyObject* g_error = nullptr;  // _lib.MdxError

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(bool ok, const char* what) {
    if (!ok) throw Refused(what);
}

bool given(PyObject* o) { return o != Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused(std::string(name) + " must be a tensor on the ROCm device");
    return THPVariable_Unpack(o);
}
// (of device d; the first operand names it)
const at::Tensor& on(PyObject* o, const char* name, c10::Device d) {
    const at::Tensor& t = tensor(o, name);
    if (t.device() != d) throw Refused(std::string(name) + " must be a tensor on the same ROCm device");
    return t;
}
c10::Device rocm_device(const at::Tensor& t) {
    check(t.is_cuda(), "expected tensors on the ROCm device");
    return t.device();
}

void ints(const at::Tensor& t, const char* name, at::IntArrayRef shape) {
    if (t.scalar_type() != at::kInt || t.sizes() != shape || !t.is_contiguous()) {
        std::string s = std::string(name) + ": contiguous int32 [";
        for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
        throw Refused(s + "]");
    }
}

int64_t number(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused("");
    return v;
}

int32_t code_of(const at::Tensor& t) {
    return t.scalar_type() == at::kBFloat16 ? MDX_DT_BF16 : t.scalar_type() == at::kHalf ? MDX_DT_F16 : -1;
}

void* data(const at::Tensor& t) { return t.data_ptr(); }

// A call on the device's current stream, with that device as the current one (a launch belongs to it).
template <class F>
void call(const char* name, c10::Device d, F f) {
    c10::hip::OptionalHIPGuard guard;
    if (c10::hip::current_device() != d.index()) guard.set_index(d.index());
    if (f(static_cast<void*>(c10::hip::getCurrentHIPStream(d.index()).stream())) != MDX_OK)
        throw Refused(std::string(name) + ": " + g.last_error());
}

at::Tensor scratch(size_t bytes, c10::Device d) {
    return at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(d));
}

template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Refused& e) {
        if (!PyErr_Occurred()) PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown exception");
    }
    return nullptr;
}

#define EXPECT(n, name)                                                   \
    if (nargs != n) {                                                     \
        PyErr_SetString(PyExc_TypeError, name " takes " #n " arguments"); \
        return nullptr;                                                   \
    }

// ---- the cache's bookkeeping ----
struct Pool {
    c10::Device d;
    int64_t L, Hk, P, T, D, B, W, ts;
    int32_t dt;
    void *kv, *ksum, *table, *length, *refs;
};
Pool pool(PyObject* const* a) {  // kv, ksum, table, length, refs
    const at::Tensor& kv = tensor(a[0], "kv");
    const c10::Device d = rocm_device(kv);
    const auto s = kv.sizes();
    const int32_t dt = code_of(kv);
    check(dt >= 0 && s.size() == 6 && s[1] == 2 && kv.is_contiguous(),
          "kv: contiguous bf16 / fp16 [layers, 2, kv_heads, pages, page rows, head_dim]");
    Pool p{d, s[0], s[2], s[3], s[4], s[5], 0, 0, 0, dt, data(kv), nullptr, nullptr, nullptr, nullptr};
    if (given(a[1])) {
        const at::Tensor& ksum = on(a[1], "ksum", d);
        check(ksum.scalar_type() == kv.scalar_type() && ksum.sizes() == at::IntArrayRef({p.L, p.Hk, p.P, p.D}) && ksum.is_contiguous(),
              "ksum: contiguous [layers, kv_heads, pages, head_dim] of the cache's type");
        p.ksum = data(ksum);
    }
    const at::Tensor& table = on(a[2], "table", d);
    check(table.scalar_type() == at::kInt && table.dim() == 2 && table.stride(1) == 1 && table.stride(0) >= table.size(1),
          "table: int32 [sequences, W], rows contiguous");
    p.B = table.size(0), p.W = table.size(1), p.ts = table.stride(0), p.table = data(table);
    const at::Tensor &length = on(a[3], "length", d), &refs = on(a[4], "refs", d);
    ints(length, "length", {p.B});
    ints(refs, "refs", {p.P});
    p.length = data(length), p.refs = data(refs);
    return p;
}
void* slots_of(PyObject* o, const Pool& p, int64_t rows, int64_t room) {
    if (!given(o)) return nullptr;
    const at::Tensor& t = on(o, "slots", p.d);
    check(t.scalar_type() == at::kLong && t.sizes() == at::IntArrayRef({rows, room}) && t.is_contiguous(), "slots: contiguous int64 [rows, room]");
    return data(t);
}

// kv, ksum, table, length, refs, dst, src, room, share, slots -> status
PyObject* page_fork(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(10, "page_fork")
    return guarded([&]() -> PyObject* {
        const Pool p = pool(a);
        const at::Tensor &dst = on(a[5], "dst", p.d), &src = on(a[6], "src", p.d);
        const int64_t M = dst.numel(), room = number(a[7]);
        ints(dst, "dst", {M});
        ints(src, "src", {M});
        const int share = PyObject_IsTrue(a[8]);
        check(share >= 0, "");
        void* slots = slots_of(a[9], p, M, room);
        at::Tensor status = at::empty({M}, at::TensorOptions().dtype(at::kInt).device(p.d));
        if (M > 0) {
            const size_t n = g.fork_workspace(M, p.W);
            at::Tensor ws = scratch(n, p.d);
            call("mdx_page_fork", p.d, [&](void* st) {
                return g.fork(p.kv, p.ksum, p.L, p.Hk, p.P, p.T, p.D, static_cast<int32_t*>(p.table), p.ts, p.B, p.W,
                              static_cast<int32_t*>(p.length), static_cast<int32_t*>(p.refs), dst.data_ptr<int32_t>(),
                              src.data_ptr<int32_t>(), M, room, share, static_cast<int64_t*>(slots), status.data_ptr<int32_t>(), data(ws), n,
                              st);
            });
        }
        return THPVariable_Wrap(std::move(status));
    });
}

// kv, ksum, table, length, refs, count, path, room, new_length, slots -> status
PyObject* page_commit(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(10, "page_commit")
    return guarded([&]() -> PyObject* {
        const Pool p = pool(a);
        const at::Tensor& count = on(a[5], "count", p.d);
        ints(count, "count", {p.B});
        const int32_t* path = nullptr;
        int64_t R = 0;
        if (given(a[6])) {
            const at::Tensor& t = on(a[6], "path", p.d);
            R = t.dim() ? t.size(-1) : 0;
            ints(t, "path", {p.B, R});
            path = t.data_ptr<int32_t>();
        }
        const int64_t room = number(a[7]);
        void* new_length = p.length;
        if (given(a[8])) {
            const at::Tensor& t = on(a[8], "new_length", p.d);
            ints(t, "new_length", {p.B});
            new_length = data(t);
        }
        void* slots = slots_of(a[9], p, p.B, room);
        at::Tensor status = at::empty({p.B}, at::TensorOptions().dtype(at::kInt).device(p.d));
        const size_t n = g.commit_workspace(p.B, p.W);
        at::Tensor ws = scratch(n, p.d);
        call("mdx_page_commit", p.d, [&](void* st) {
            return g.commit(p.kv, p.ksum, p.dt, p.L, p.Hk, p.P, p.T, p.D, static_cast<int32_t*>(p.table), p.ts, p.B, p.W,
                            static_cast<const int32_t*>(p.length), static_cast<int32_t*>(new_length), static_cast<int32_t*>(p.refs),
                            count.data_ptr<int32_t>(), path, R, room, static_cast<int64_t*>(slots), status.data_ptr<int32_t>(), data(ws),
                            n, st);
        });
        return THPVariable_Wrap(std::move(status));
    });
}

// ---- attention ----
struct Attn {
    c10::Device d;
    const at::Tensor &q, &key, &value, &table, &length;
    const int64_t* mask;
    at::Tensor out;
    int32_t dt;
    int64_t B, S, H, Hk, D, P, T, W, ts;
};
Attn attn(PyObject* q_, PyObject* key_, PyObject* value_, PyObject* table_, PyObject* length_, PyObject* mask_, PyObject* out_) {
    const at::Tensor& q = tensor(q_, "q");
    const c10::Device d = rocm_device(q);
    const at::Tensor &key = on(key_, "key", d), &value = on(value_, "value", d), &table = on(table_, "table", d), &length = on(length_, "length", d);
    const int32_t dt = code_of(q);
    check(dt >= 0 && key.scalar_type() == q.scalar_type() && value.scalar_type() == q.scalar_type(), "q, key and value: bf16 or fp16, one type");
    check(q.dim() == 4 && q.stride(3) == 1, "q: [sequences, rows, heads, head_dim], the last dim contiguous");
    const int64_t B = q.size(0), S = q.size(1), H = q.size(2), D = q.size(3);
    check(key.dim() == 4 && key.size(3) == D && value.sizes() == key.sizes() && key.stride(3) == 1 && value.stride(3) == 1,
          "key / value: [kv_heads, pages, page rows, head_dim], the last dim contiguous");
    const int64_t Hk = key.size(0);
    check(Hk >= 1 && H % Hk == 0, "query heads: a multiple of the kv heads");
    check(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && table.stride(1) == 1 && table.stride(0) >= table.size(1),
          "table: int32 [sequences, W], rows contiguous");
    ints(length, "length", {B});
    const int64_t* mask = nullptr;
    if (given(mask_)) {
        const at::Tensor& m = on(mask_, "mask", d);
        check(m.scalar_type() == at::kLong && m.sizes() == at::IntArrayRef({B, S}) && m.is_contiguous() && S <= 64,
              "mask: contiguous int64 [sequences, rows], at most 64 rows");
        mask = m.data_ptr<int64_t>();
    }
    at::Tensor out;
    if (given(out_)) {
        out = on(out_, "out", d);
        check(out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() && out.is_contiguous(), "out: contiguous, q's shape and type");
    } else {
        out = at::empty(q.sizes(), at::TensorOptions().dtype(q.scalar_type()).device(d));
    }
    return Attn{d, q, key, value, table, length, mask, out, dt, B, S, H, Hk, D, key.size(1), key.size(2), table.size(1), table.stride(0)};
}
float scale_of(PyObject* o, int64_t D) {
    if (!given(o)) return float(1.0 / std::sqrt(double(D)));
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused("");
    return float(v);
}
PyObject* same_or_new(PyObject* o, at::Tensor t) {
    if (given(o)) {
        Py_INCREF(o);
        return o;
    }
    return THPVariable_Wrap(std::move(t));
}

// q, key, value, table, length, mask, scale, out -> out
PyObject* attn_paged(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(8, "attn_paged")
    return guarded([&]() -> PyObject* {
        Attn x = attn(a[0], a[1], a[2], a[3], a[4], a[5], a[7]);
        const float scale = scale_of(a[6], x.D);
        if (x.B > 0 && x.S > 0) {
            const size_t n = g.paged_workspace(x.B, x.S, x.H, x.Hk, x.D, x.T, x.W);
            at::Tensor ws;
            if (n) ws = scratch(n, x.d);
            call("mdx_attn_paged", x.d, [&](void* st) {
                return g.paged(data(x.q), x.q.stride(0), x.q.stride(1), x.q.stride(2), data(x.key), x.key.stride(0), x.key.stride(1),
                               x.key.stride(2), data(x.value), x.value.stride(0), x.value.stride(1), x.value.stride(2), x.dt,
                               x.table.data_ptr<int32_t>(), x.ts, x.length.data_ptr<int32_t>(), x.mask, data(x.out), x.B, x.S, x.H, x.Hk,
                               x.D, x.P, x.T, x.W, scale, n ? data(ws) : nullptr, n, st);
            });
        }
        return same_or_new(a[7], x.out);
    });
}

// q, key, value, ksum, table, length, blocks, sink, local, mask, scale, out, sel -> (out, sel)
PyObject* attn_blocks(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(13, "attn_blocks")
    return guarded([&]() -> PyObject* {
        Attn x = attn(a[0], a[1], a[2], a[4], a[5], a[9], a[11]);
        const at::Tensor& ksum = on(a[3], "ksum", x.d);
        check(ksum.scalar_type() == x.q.scalar_type() && ksum.sizes() == at::IntArrayRef({x.Hk, x.P, x.D}) && ksum.stride(2) == 1,
              "ksum: [kv_heads, pages, head_dim] of the cache's type");
        const int64_t blocks = number(a[6]), sink = number(a[7]), local = number(a[8]);
        check(blocks >= 0 && sink >= 0 && local >= 0 && blocks <= 65536 && sink <= 65536 && local <= 65536 && blocks + sink + local >= 1 &&
                  blocks + sink + local <= 65536,
              "1..65536 selected blocks");
        const int64_t most = blocks + sink + local;
        const float scale = scale_of(a[10], x.D);
        at::Tensor sel;
        if (given(a[12])) {
            sel = on(a[12], "sel", x.d);
            ints(sel, "sel", {x.B, x.S, x.Hk, most});
        } else {
            sel = at::empty({x.B, x.S, x.Hk, most}, at::TensorOptions().dtype(at::kInt).device(x.d));
        }
        if (x.B > 0 && x.S > 0) {
            const size_t n = g.blocks_workspace(x.B, x.S, x.H, x.Hk, x.D, x.W, most);
            at::Tensor ws = scratch(n, x.d);
            call("mdx_attn_blocks", x.d, [&](void* st) {
                return g.blocks(data(x.q), x.q.stride(0), x.q.stride(1), x.q.stride(2), data(x.key), x.key.stride(0), x.key.stride(1),
                                x.key.stride(2), data(x.value), x.value.stride(0), x.value.stride(1), x.value.stride(2), data(ksum),
                                ksum.stride(0), ksum.stride(1), x.dt, x.table.data_ptr<int32_t>(), x.ts, x.length.data_ptr<int32_t>(),
                                x.mask, data(x.out), sel.data_ptr<int32_t>(), blocks, sink, local, x.B, x.S, x.H, x.Hk, x.D, x.P, x.T, x.W,
                                scale, data(ws), n, st);
            });
        }
        PyObject* o = same_or_new(a[11], x.out);
        PyObject* s = o ? same_or_new(a[12], sel) : nullptr;
        PyObject* both = s ? PyTuple_Pack(2, o, s) : nullptr;
        Py_XDECREF(o);
        Py_XDECREF(s);
        return both;
    });
}

// a window's length (None: everything)
int64_t window_of(PyObject* o) {
    const int64_t window = given(o) ? number(o) : int64_t(1) << 30;
    check(window >= 1 && window <= (int64_t(1) << 30), "window: 1..2^30 tokens, or None");
    return window;
}

// q, key, value, table, length, window, sinks, mask, scale, out, lse -> (out, lse)
PyObject* attn_window(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(11, "attn_window")
    return guarded([&]() -> PyObject* {
        Attn x = attn(a[0], a[1], a[2], a[3], a[4], a[7], a[9]);
        const int64_t window = window_of(a[5]), sinks = number(a[6]);
        check(sinks >= 0 && sinks <= (int64_t(1) << 30), "sinks: 0..2^30 tokens");
        const float scale = scale_of(a[8], x.D);
        at::Tensor lse;
        if (given(a[10])) {
            lse = on(a[10], "lse", x.d);
            check(lse.scalar_type() == at::kFloat && lse.sizes() == at::IntArrayRef({x.B, x.S, x.H}) && lse.is_contiguous(),
                  "lse: contiguous float32 [sequences, rows, heads]");
        } else {
            lse = at::empty({x.B, x.S, x.H}, at::TensorOptions().dtype(at::kFloat).device(x.d));
        }
        if (x.B > 0 && x.S > 0) {
            const size_t n = g.window_workspace(x.B, x.S, x.H, x.Hk, x.D, x.T, x.W, window, sinks);
            at::Tensor ws;
            if (n) ws = scratch(n, x.d);
            call("mdx_attn_window", x.d, [&](void* st) {
                return g.window(data(x.q), x.q.stride(0), x.q.stride(1), x.q.stride(2), data(x.key), x.key.stride(0), x.key.stride(1),
                                x.key.stride(2), data(x.value), x.value.stride(0), x.value.stride(1), x.value.stride(2), x.dt,
                                x.table.data_ptr<int32_t>(), x.ts, x.length.data_ptr<int32_t>(), x.mask, data(x.out), lse.data_ptr<float>(),
                                window, sinks, x.B, x.S, x.H, x.Hk, x.D, x.P, x.T, x.W, scale, n ? data(ws) : nullptr, n, st);
            });
        }
        PyObject* o = same_or_new(a[9], x.out);
        PyObject* l = o ? same_or_new(a[10], lse) : nullptr;
        PyObject* both = l ? PyTuple_Pack(2, o, l) : nullptr;
        Py_XDECREF(o);
        Py_XDECREF(l);
        return both;
    });
}

// q, key, table, length, lse, prior, count, path, window, sinks, scale, out -> out
PyObject* attn_mass(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(12, "attn_mass")
    return guarded([&]() -> PyObject* {
        const at::Tensor& q = tensor(a[0], "q");
        const c10::Device d = rocm_device(q);
        const at::Tensor &key = on(a[1], "key", d), &table = on(a[2], "table", d), &length = on(a[3], "length", d), &lse = on(a[4], "lse", d);
        const int32_t dt = code_of(q);
        check(dt >= 0 && key.scalar_type() == q.scalar_type(), "q and key: bf16 or fp16, one type");
        check(q.dim() == 4 && q.stride(3) == 1, "q: [sequences, rows, heads, head_dim], the last dim contiguous");
        const int64_t B = q.size(0), S = q.size(1), H = q.size(2), D = q.size(3);
        check(key.dim() == 4 && key.size(3) == D && key.stride(3) == 1, "key: [kv_heads, pages, page rows, head_dim], the last dim contiguous");
        const int64_t Hk = key.size(0), P = key.size(1), T = key.size(2);
        check(Hk >= 1 && H % Hk == 0, "query heads: a multiple of the kv heads");
        check(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && table.stride(1) == 1 && table.stride(0) >= table.size(1),
              "table: int32 [sequences, W], rows contiguous");
        const int64_t W = table.size(1);
        ints(length, "length", {B});
        check(lse.scalar_type() == at::kFloat && lse.sizes() == at::IntArrayRef({B, S, H}) && lse.is_contiguous(),
              "lse: contiguous float32 [sequences, rows, heads]");
        const int32_t *count = nullptr, *path = nullptr;
        if (given(a[6])) {
            const at::Tensor& t = on(a[6], "count", d);
            ints(t, "count", {B});
            count = t.data_ptr<int32_t>();
        }
        if (given(a[7])) {
            const at::Tensor& t = on(a[7], "path", d);
            ints(t, "path", {B, S});
            path = t.data_ptr<int32_t>();
        }
        const int64_t window = window_of(a[8]), sinks = number(a[9]);
        check(sinks >= 0 && sinks <= (int64_t(1) << 30), "sinks: 0..2^30 tokens");
        const float scale = scale_of(a[10], D);
        auto sums = [&](const at::Tensor& t, const char* what) {
            check(t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(0) == B && t.size(1) == Hk && t.size(2) >= 1 && t.stride(2) == 1, what);
        };
        const float* prior = nullptr;
        int64_t pb = 0, ph = 0, N = W * T;
        if (given(a[5])) {
            const at::Tensor& t = on(a[5], "prior", d);
            sums(t, "prior: float32 [sequences, kv_heads, places], rows contiguous");
            prior = t.data_ptr<float>();
            pb = t.stride(0), ph = t.stride(1), N = t.size(2);
        }
        at::Tensor out;
        if (given(a[11])) {
            out = on(a[11], "out", d);
            sums(out, "out: float32 [sequences, kv_heads, places], rows contiguous");
            check(!prior || out.size(2) == N, "prior and out: as many places");
            N = out.size(2);
        } else {
            out = at::zeros({B, Hk, N}, at::TensorOptions().dtype(at::kFloat).device(d));
        }
        if (B > 0 && S == 0) {  // the prior sums: a row that does not count
            const auto of = [&](at::ScalarType type) { return at::TensorOptions().dtype(type).device(d); };
            const at::Tensor none = at::zeros({B}, of(at::kInt)), row = at::empty({B, 1, H, D}, of(q.scalar_type())), sum = at::empty({B, 1, H}, of(at::kFloat));
            call("mdx_attn_mass", d, [&](void* st) {
                return g.mass(data(row), H * D, H * D, D, data(key), key.stride(0), key.stride(1), key.stride(2), dt, table.data_ptr<int32_t>(),
                              table.stride(0), length.data_ptr<int32_t>(), sum.data_ptr<float>(), prior, pb, ph, none.data_ptr<int32_t>(), nullptr,
                              window, sinks, out.data_ptr<float>(), out.stride(0), out.stride(1), N, B, 1, H, Hk, D, P, T, W, scale, nullptr, 0, st);
            });
        } else if (B > 0) {
            const size_t n = path ? 0 : g.mass_workspace(B, S, H, Hk, D, T, W, N);
            at::Tensor ws;
            if (n) ws = scratch(n, d);
            call("mdx_attn_mass", d, [&](void* st) {
                return g.mass(data(q), q.stride(0), q.stride(1), q.stride(2), data(key), key.stride(0), key.stride(1), key.stride(2), dt,
                              table.data_ptr<int32_t>(), table.stride(0), length.data_ptr<int32_t>(), lse.data_ptr<float>(), prior, pb, ph, count,
                              path, window, sinks, out.data_ptr<float>(), out.stride(0), out.stride(1), N, B, S, H, Hk, D, P, T, W, scale,
                              n ? data(ws) : nullptr, n, st);
            });
        }
        return same_or_new(a[11], out);
    });
}

// kv, ksum, table, length, refs, mass, dst, src, keep, sinks, recent, room, slots -> (status, kept)
PyObject* page_evict(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(13, "page_evict")
    return guarded([&]() -> PyObject* {
        const Pool p = pool(a);
        const at::Tensor &mass = on(a[5], "mass", p.d), &dst = on(a[6], "dst", p.d), &src = on(a[7], "src", p.d);
        check(mass.scalar_type() == at::kFloat && mass.dim() == 4 && mass.size(0) == p.L && mass.size(1) == p.B && mass.size(2) == p.Hk &&
                  mass.is_contiguous(),
              "mass: contiguous float32 [layers, sequences, kv_heads, places]");
        const int64_t M = dst.numel(), keep = number(a[8]), sinks = number(a[9]), recent = number(a[10]), room = number(a[11]);
        ints(dst, "dst", {M});
        ints(src, "src", {M});
        const int64_t cap = int64_t(1) << 29;
        check(keep >= 0 && sinks >= 0 && recent >= 0 && keep <= cap && sinks <= cap && recent <= cap && keep + sinks + recent >= 1,
              "1..2^29 kept tokens of each kind");
        const int64_t most = keep + sinks + recent;
        check(M * p.L * p.Hk * most < (int64_t(1) << 31), "too many pairs times heads times kept tokens for one call");
        void* slots = slots_of(a[12], p, M, room);
        const auto kind = at::TensorOptions().dtype(at::kInt).device(p.d);
        at::Tensor status = at::empty({M}, kind), kept = at::empty({M, p.L, p.Hk, most}, kind);
        if (M > 0) {
            const size_t n = g.evict_workspace(M, p.W, p.L, p.Hk, most);
            at::Tensor ws = scratch(n, p.d);
            call("mdx_page_evict", p.d, [&](void* st) {
                return g.evict(p.kv, p.ksum, p.dt, p.L, p.Hk, p.P, p.T, p.D, static_cast<int32_t*>(p.table), p.ts, p.B, p.W,
                               static_cast<int32_t*>(p.length), static_cast<int32_t*>(p.refs), mass.data_ptr<float>(), mass.size(3),
                               dst.data_ptr<int32_t>(), src.data_ptr<int32_t>(), M, keep, sinks, recent, room, static_cast<int64_t*>(slots),
                               status.data_ptr<int32_t>(), kept.data_ptr<int32_t>(), data(ws), n, st);
            });
        }
        PyObject *s = THPVariable_Wrap(std::move(status)), *k = s ? THPVariable_Wrap(std::move(kept)) : nullptr;
        PyObject* both = k ? PyTuple_Pack(2, s, k) : nullptr;
        Py_XDECREF(s);
        Py_XDECREF(k);
        return both;
    });
}

// ---- a step's answers ----
// logits, tokens, uniform, draft, parent, temperature -> (count, path, next)
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    EXPECT(6, "verify_drafts")
    return guarded([&]() -> PyObject* {
        const at::Tensor& logits = tensor(a[0], "logits");
        const c10::Device d = rocm_device(logits);
        const int32_t dt = logits.scalar_type() == at::kFloat ? MDX_DT_F32 : code_of(logits);
        check(dt >= 0 && logits.dim() == 3 && logits.size(2) >= 1 && logits.stride(2) == 1,
              "logits: bf16, fp16 or fp32 [sequences, rows, vocabulary], rows contiguous");
        const int64_t B = logits.size(0), R = logits.size(1), V = logits.size(2);
        const at::Tensor &tokens = on(a[1], "tokens", d), &uniform = on(a[2], "uniform", d);
        check(tokens.scalar_type() == at::kLong && tokens.sizes() == at::IntArrayRef({B, R}) && tokens.is_contiguous(),
              "tokens: contiguous int64 [sequences, rows]");
        check(uniform.scalar_type() == at::kDouble && uniform.sizes() == at::IntArrayRef({B, R + 1}) && uniform.is_contiguous(),
              "uniform: contiguous float64 [sequences, rows + 1]");
        const void* draft = nullptr;
        int64_t db = 0, dr = 0;
        if (given(a[3])) {
            const at::Tensor& t = on(a[3], "draft", d);
            check(R >= 1 && t.scalar_type() == logits.scalar_type() && t.sizes() == at::IntArrayRef({B, R - 1, V}) && t.stride(2) == 1,
                  "draft: [sequences, rows - 1, vocabulary] of the logits' type, rows contiguous");
            check(!given(a[4]), "drafts with probabilities: a chain (no parents)");
            if (R > 1) draft = data(t), db = t.stride(0), dr = t.stride(1);
        }
        const int32_t* parent = nullptr;
        if (given(a[4])) {
            const at::Tensor& t = on(a[4], "parent", d);
            ints(t, "parent", {B, R});
            parent = t.data_ptr<int32_t>();
        }
        const float* heats = nullptr;
        double heat = 0;
        if (THPVariable_Check(a[5])) {
            const at::Tensor& t = on(a[5], "temperature", d);
            check(t.scalar_type() == at::kFloat && t.sizes() == at::IntArrayRef({B}) && t.is_contiguous(), "temperature: a number, or contiguous float32 [sequences]");
            heats = t.data_ptr<float>();
        } else {
            heat = PyFloat_AsDouble(a[5]);
            if (heat == -1.0 && PyErr_Occurred()) throw Refused("");
        }
        const auto kind = at::TensorOptions().device(d);
        at::Tensor count = at::empty({B}, kind.dtype(at::kInt)), path = at::empty({B, R}, kind.dtype(at::kInt)), next = at::empty({B}, kind.dtype(at::kLong));
        if (B > 0) {
            const size_t n = g.verify_workspace(B, R, V, draft != nullptr);
            at::Tensor ws = scratch(n, d);
            call("mdx_verify_drafts", d, [&](void* st) {
                return g.verify(data(logits), logits.stride(0), logits.stride(1), draft, db, dr, dt, tokens.data_ptr<int64_t>(), parent,
                                uniform.data_ptr<double>(), heats, float(heat), count.data_ptr<int32_t>(), path.data_ptr<int32_t>(),
                                next.data_ptr<int64_t>(), B, R, V, data(ws), n, st);
            });
        }
        PyObject* o[3] = {THPVariable_Wrap(std::move(count)), THPVariable_Wrap(std::move(path)), THPVariable_Wrap(std::move(next))};
        PyObject* all = o[0] && o[1] && o[2] ? PyTuple_Pack(3, o[0], o[1], o[2]) : nullptr;
        for (PyObject* x : o) Py_XDECREF(x);
        return all;
    });
}

// init(the entry points' addresses in the order of Entries, error class)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != ENTRIES + 1) {
        PyErr_SetString(PyExc_TypeError, "init takes the entry points and the error class");
        return nullptr;
    }
    void* p[ENTRIES];
    for (int i = 0; i < ENTRIES; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "null entry point");
            return nullptr;
        }
    }
    int i = 0;
    g.last_error = reinterpret_cast<decltype(g.last_error)>(p[i++]);
    g.fork_workspace = reinterpret_cast<decltype(g.fork_workspace)>(p[i++]);
    g.fork = reinterpret_cast<decltype(g.fork)>(p[i++]);
    g.commit_workspace = reinterpret_cast<decltype(g.commit_workspace)>(p[i++]);
    g.commit = reinterpret_cast<decltype(g.commit)>(p[i++]);
    g.paged_workspace = reinterpret_cast<decltype(g.paged_workspace)>(p[i++]);
    g.paged = reinterpret_cast<decltype(g.paged)>(p[i++]);
    g.blocks_workspace = reinterpret_cast<decltype(g.blocks_workspace)>(p[i++]);
    g.blocks = reinterpret_cast<decltype(g.blocks)>(p[i++]);
    g.verify_workspace = reinterpret_cast<decltype(g.verify_workspace)>(p[i++]);
    g.verify = reinterpret_cast<decltype(g.verify)>(p[i++]);
    g.window_workspace = reinterpret_cast<decltype(g.window_workspace)>(p[i++]);
    g.window = reinterpret_cast<decltype(g.window)>(p[i++]);
    g.mass_workspace = reinterpret_cast<decltype(g.mass_workspace)>(p[i++]);
    g.mass = reinterpret_cast<decltype(g.mass)>(p[i++]);
    g.evict_workspace = reinterpret_cast<decltype(g.evict_workspace)>(p[i++]);
    g.evict = reinterpret_cast<decltype(g.evict)>(p[i++]);
    Py_XINCREF(a[ENTRIES]);
    Py_XDECREF(g_error);
    g_error = a[ENTRIES];
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&f))
PyMethodDef methods[] = {{"init", FAST(init), METH_FASTCALL, nullptr},
                         {"page_fork", FAST(page_fork), METH_FASTCALL, nullptr},
                         {"page_commit", FAST(page_commit), METH_FASTCALL, nullptr},
                         {"attn_paged", FAST(attn_paged), METH_FASTCALL, nullptr},
                         {"attn_blocks", FAST(attn_blocks), METH_FASTCALL, nullptr},
                         {"attn_window", FAST(attn_window), METH_FASTCALL, nullptr},
                         {"attn_mass", FAST(attn_mass), METH_FASTCALL, nullptr},
                         {"page_evict", FAST(page_evict), METH_FASTCALL, nullptr},
                         {"verify_drafts", FAST(verify_drafts), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
