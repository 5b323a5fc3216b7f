// ff_host.cpp - the host half of the cached-decoding calls (framefusion_amd/cache.py, rotary.py) as one crossing each: every check of the
// arguments, the outputs and the workspace, one call of the C ABI on PyTorch's current stream.
//
// A decoding step makes dozens of these calls and a kernel of one token takes 3 us, so what the host adds is what such a call costs:
// with the checks in Python and ctypes a write took 8.2 us of host time, an attention 14.7 us.  Nothing is kept from call to call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <sstream>
#include <string>

#include "ff_source_hash.h"
#include "framefusion_hip.h"

// what this module was built from, readable from the file
extern "C" __attribute__((visibility("default"), used)) const char ff_host_stamp[] = "FFSRCHASH:" FF_SOURCE_HASH;

namespace {

PyObject* g_error = nullptr;                 // framefusion_amd._lib.FrameFusionHipError

struct Refused { std::string what; };

template <class... A> [[noreturn]] void refuse(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw Refused{s.str()};
}
void check(int rc, const char* what) {
    if (rc) {
        const char* m = ff_error_string(rc);
        refuse(what, " failed: [", rc, "] ", m ? m : "?");
    }
}

// what a module function does with its exceptions: a refusal is FrameFusionHipError, torch's own are translated as everywhere
#define FF_CALL HANDLE_TH_ERRORS try {
#define FF_END                                            \
    }                                                     \
    catch (const Refused& r) {                            \
        PyErr_SetString(g_error, r.what.c_str());         \
        return nullptr;                                   \
    }                                                     \
    END_HANDLE_TH_ERRORS

// (its values lie in its memory: a sign that PyTorch keeps beside it, zeros that have none, are made so)
at::Tensor tensor(PyObject* o, const char* what, const char* name) {
    if (!THPVariable_Check(o)) refuse(what, ": ", name, " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.is_neg()) return t.resolve_neg();
    if (t._is_zerotensor()) return t.clone();
    if (t.numel() && !t.const_data_ptr()) refuse(what, ": ", name, " has no memory of its own (a wrapper around other tensors, or one of the meta device)");
    return t;
}
// what is written in place, or read where it lies
const at::Tensor& held(PyObject* o, const char* what, const char* name) {
    if (!THPVariable_Check(o)) refuse(what, ": ", name, " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.is_neg() || t._is_zerotensor()) refuse(what, ": ", name, " must be a tensor of values that lie in memory (no negative bit, no zeros without memory)");
    return t;
}
// whether a derivative is asked for with respect to `t`, backward or (a tangent beside it) forward
bool differentiable(const at::Tensor& t) { return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined(); }

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return FF_F32;
        case at::kBFloat16: return FF_BF16;
        case at::kHalf: return FF_F16;
        default: return -1;
    }
}
// the device must be a GPU (the last of a call's checks)
void on_gpu(const at::Tensor& t, const char* what) {
    if (!t.is_cuda())
        refuse(what, ": framefusion_amd runs on MI355X only (got a ", t.device().str(),
               " tensor); there is no CPU path in the product - the CPU oracle lives in oracle/ for tests.");
}
ff_stream_t stream_of(const at::Tensor& t) { return (ff_stream_t)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

struct Cache {
    ff_cache_t c{};
    at::Device device{at::kCPU};
    at::ScalarType own;                      // of the keys
    at::Tensor table, start;
};

// the head of every call on a cache: (keys, values, key_scales, value_scales), its table and start
Cache parse(PyObject* cache, PyObject* table_o, PyObject* start_o, int64_t n, at::ScalarType dtype, const char* what) {
    // (the caller's own tuple holds the tensors while the call runs: what an iterator made would be gone before the launch)
    if (!(PyTuple_Check(cache) || PyList_Check(cache)) || PySequence_Fast_GET_SIZE(cache) != 4)
        refuse(what, ": a cache is the four tensors (keys, values, key_scales, value_scales)");
    PyObject** items = PySequence_Fast_ITEMS(cache);
    const at::Tensor &keys = held(items[0], what, "keys"), &values = held(items[1], what, "values");
    Cache out;
    out.device = keys.device();
    out.own = keys.scalar_type();
    const int code = code_of(dtype);
    int store = code_of(out.own);
    if (out.own == at::kFloat8_e4m3fn) store = FF_STORE_E4M3;
    if (out.own == at::kByte) store = FF_STORE_E2M1;
    if (store < 0 || keys.dim() != 4 || values.sizes() != keys.sizes() || values.scalar_type() != out.own || values.device() != out.device ||
        !keys.is_contiguous() || !values.is_contiguous())
        refuse(what, ": keys and values of a cache must be alike and contiguous, [pages, kv_heads, page_size, head_dim]");
    if (differentiable(keys) || differentiable(values)) refuse(what, " has no gradient (serving only): call it under torch.no_grad()");
    if (code < 0) refuse(what, ": a cache serves float32, bfloat16 and float16, not ", c10::toString(dtype));
    ff_cache_t& c = out.c;
    c.n_pages = keys.size(0);
    c.kv_heads = keys.size(1);
    c.page_size = keys.size(2);
    c.dh = keys.size(3);
    if (store == code) {
        if (items[2] != Py_None || items[3] != Py_None) refuse(what, ": a cache in ", c10::toString(dtype), " holds no scales");
    } else {
        if (store != FF_STORE_E4M3 && store != FF_STORE_E2M1)
            refuse(what, ": a cache in ", c10::toString(out.own), " serves that type alone, not ", c10::toString(dtype));
        if (store == FF_STORE_E2M1) c.dh *= 2;
        const int64_t want[4] = {c.n_pages, c.kv_heads, c.page_size, c.dh / 32};
        uint8_t* scales[2];
        for (int i = 0; i < 2; ++i) {
            if (!THPVariable_Check(items[2 + i])) refuse(what, ": a cache of codes needs its scales");
            const at::Tensor& s = held(items[2 + i], what, "scales");
            if (s.sizes() != at::IntArrayRef(want, 4) || s.scalar_type() != at::kByte || !s.is_contiguous() || s.device() != out.device)
                refuse(what, ": a cache of codes needs contiguous uint8 scales ", at::IntArrayRef(want, 4));
            scales[i] = (uint8_t*)s.data_ptr();
        }
        c.key_scales = scales[0];
        c.value_scales = scales[1];
    }
    const at::Tensor &table = out.table = tensor(table_o, what, "table"), &start = out.start = tensor(start_o, what, "start");
    if (table.dim() != 2 || table.scalar_type() != at::kInt || start.dim() != 1 || start.scalar_type() != at::kInt || start.size(0) != table.size(0) ||
        table.device() != out.device || start.device() != out.device || !table.is_contiguous() || !start.is_contiguous())
        refuse(what, ": table must be int32 [B, width] and start int32 [B], contiguous, on the cache's device");
    c.keys = keys.data_ptr();
    c.values = values.data_ptr();
    c.table = (const int32_t*)table.data_ptr();
    c.start = (const int32_t*)start.data_ptr();
    c.store = store;
    c.table_width = table.size(1);
    c.B = table.size(0);
    c.n = n;
    c.dtype = code;
    on_gpu(keys, what);
    return out;
}

// strides of batch, head and token of `t` [B, heads, n, dh], which becomes a contiguous copy if the kernels cannot read it in
// place (16-byte pieces of whole rows; the stride of a dimension of one is never used)
at::Tensor rows(const at::Tensor& t, int64_t* st) {
    const int64_t per = 16 / t.element_size();
    bool fine = t.stride(3) == 1 && ((uintptr_t)t.data_ptr() & 15) == 0;
    for (int i = 0; i < 3; ++i) {
        st[i] = t.size(i) > 1 ? t.stride(i) : 0;
        fine = fine && st[i] % per == 0;
    }
    if (fine) return t;
    at::Tensor copy = t.clone(at::MemoryFormat::Contiguous);
    for (int i = 0; i < 3; ++i) st[i] = copy.stride(i);
    return copy;
}

// A tracer records the allocation of a call's outputs and nothing of what fills them: what it made would return whatever the memory
// holds.  (torch.compile leaves these calls out of its graphs by itself.)
void not_traced(const char* what) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    if (torch::jit::tracer::isTracing() ||
        (Modes::any_modes_set() && (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL))))
        refuse(what, " cannot be traced: torch.jit.trace, make_fx and fake or functional tensors do not see what it computes");
}
// the head of every call
void begin(Py_ssize_t n, Py_ssize_t want, const char* what) {
    if (n != want) refuse(what, ": ", want, " arguments");
    not_traced(what);
}

// not_traced(what): for the calls that go through ctypes
PyObject* py_not_traced(PyObject*, PyObject* what) {
    FF_CALL
    const char* name = PyUnicode_AsUTF8(what);
    if (!name) throw python_error();
    not_traced(name);
    Py_RETURN_NONE;
    FF_END
}

// write(cache, key, value, table, start)
PyObject* py_write(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    FF_CALL
    begin(nargs, 5, "cache_write");
    const at::Tensor key = tensor(args[1], "cache_write", "key"), value = tensor(args[2], "cache_write", "value");
    if (differentiable(key) || differentiable(value)) refuse("cache_write has no gradient (serving only): call it under torch.no_grad()");
    Cache cache = parse(args[0], args[3], args[4], key.dim() == 4 ? key.size(2) : 0, key.scalar_type(), "cache_write");
    const ff_cache_t& c = cache.c;
    const int64_t want[4] = {c.B, c.kv_heads, c.n, c.dh};
    if (key.sizes() != at::IntArrayRef(want, 4) || value.sizes() != key.sizes() || value.scalar_type() != key.scalar_type() ||
        key.device() != cache.device || value.device() != cache.device)
        refuse("cache_write: key and value must be ", at::IntArrayRef(want, 4), " of one dtype on the cache's device, got ", key.sizes(), " and ", value.sizes());
    if (key.numel() == 0) Py_RETURN_NONE;
    const c10::DeviceGuard guard(cache.device);
    ff_cache_rows_t a{};
    a.cache = c;
    const at::Tensor k = rows(key, &a.k_batch), v = rows(value, &a.v_batch);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.stream = stream_of(key);
    check(ff_cache_write(&a), "ff_cache_write");
    Py_RETURN_NONE;
    FF_END
}

// read(cache, table, start, count, dtype or None) -> (key, value)
PyObject* py_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    FF_CALL
    begin(nargs, 5, "cache_read");
    const int64_t count = PyLong_AsLongLong(args[3]);
    if (count == -1 && PyErr_Occurred()) throw python_error();
    if (count < 0) refuse("cache_read: count must not be negative");
    at::ScalarType dtype;
    if (args[4] == Py_None) {
        // the cache's own type, or bfloat16 for one of codes
        PyObject* first = PySequence_GetItem(args[0], 0);
        if (!first) throw python_error();
        dtype = THPVariable_Check(first) ? THPVariable_Unpack(first).scalar_type() : at::kBFloat16;
        Py_DECREF(first);
        if (code_of(dtype) < 0) dtype = at::kBFloat16;
    } else {
        if (!THPDtype_Check(args[4])) refuse("cache_read: dtype must be a torch.dtype");
        dtype = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    }
    Cache cache = parse(args[0], args[1], args[2], count, dtype, "cache_read");
    const ff_cache_t& c = cache.c;
    const c10::DeviceGuard guard(cache.device);
    const at::Tensor both = at::empty({2, c.B, c.kv_heads, count, c.dh}, at::TensorOptions().dtype(dtype).device(cache.device));
    at::Tensor key = both.select(0, 0), value = both.select(0, 1);
    if (key.numel()) {
        ff_cache_rows_t a{};
        a.cache = c;
        a.k = key.data_ptr();
        a.v = value.data_ptr();
        a.k_token = a.v_token = c.dh;
        a.k_head = a.v_head = count * c.dh;
        a.k_batch = a.v_batch = c.kv_heads * count * c.dh;
        a.stream = stream_of(key);
        check(ff_cache_read(&a), "ff_cache_read");
    }
    PyObject *k = THPVariable_Wrap(std::move(key)), *v = THPVariable_Wrap(std::move(value));
    return Py_BuildValue("(NN)", k, v);
    FF_END
}

// keep(cache, table, start, accepted)
PyObject* py_keep(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    FF_CALL
    begin(nargs, 4, "cache_keep");
    PyObject* first = PySequence_GetItem(args[0], 0);
    if (!first) throw python_error();
    at::ScalarType dtype = THPVariable_Check(first) ? THPVariable_Unpack(first).scalar_type() : at::kBFloat16;
    Py_DECREF(first);
    if (code_of(dtype) < 0) dtype = at::kBFloat16;
    Cache cache = parse(args[0], args[1], args[2], 0, dtype, "cache_keep");
    const at::Tensor accepted = tensor(args[3], "cache_keep", "accepted");
    if (accepted.scalar_type() != at::kInt || accepted.dim() != 2 || accepted.size(0) != cache.c.B || accepted.device() != cache.device ||
        !accepted.is_contiguous())
        refuse("cache_keep: accepted must be a contiguous int32 [B, m] on the cache's device");
    if (accepted.numel() == 0) Py_RETURN_NONE;
    const c10::DeviceGuard guard(cache.device);
    check(ff_cache_keep(&cache.c, (const int32_t*)accepted.data_ptr(), accepted.size(1), stream_of(accepted)), "ff_cache_keep");
    Py_RETURN_NONE;
    FF_END
}

// attention(query, cache, table, start, mask or None, scale or None) -> [B, H, n, dh]
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    FF_CALL
    const char* what = "cache_attention";
    begin(nargs, 6, what);
    const at::Tensor query = tensor(args[0], what, "query");
    if (differentiable(query)) refuse("cache_attention has no gradient (serving only): call it under torch.no_grad()");
    if (query.dim() != 4) refuse("cache_attention: query must be [B, H, n, head_dim], got ", query.sizes());
    const int64_t B = query.size(0), H = query.size(1), n = query.size(2), dh = query.size(3);
    at::Tensor mask;
    if (args[4] != Py_None) {
        mask = tensor(args[4], what, "mask");
        const bool shared = mask.dim() == 2, fits = shared ? mask.size(0) == n && mask.size(1) == n
                                                           : mask.dim() == 3 && mask.size(0) == B && mask.size(1) == n && mask.size(2) == n;
        if (mask.scalar_type() != at::kBool || mask.device() != query.device() || !fits)
            refuse("cache_attention: mask must be bool [", n, ", ", n, "] or [", B, ", ", n, ", ", n, "], got ", c10::toString(mask.scalar_type()), " ", mask.sizes());
    }
    if (dh != 32 && dh != 64 && dh != 128 && dh != 256) refuse("cache_attention: head_dim must be 32, 64, 128 or 256, got ", dh);
    double scale = 1.0 / std::sqrt((double)dh);
    if (args[5] != Py_None) {
        scale = PyFloat_AsDouble(args[5]);
        if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    }
    Cache cache = parse(args[1], args[2], args[3], n, query.scalar_type(), what);
    const ff_cache_t& c = cache.c;
    if (B != c.B || dh != c.dh || H < 1 || c.kv_heads < 1 || H % c.kv_heads || query.device() != cache.device)
        refuse("cache_attention: query ", query.sizes(), " does not fit a table of ", c.B, " sequences and ", c.kv_heads, " heads of ", c.dh);
    const c10::DeviceGuard guard(cache.device);
    const at::Tensor out = at::empty({B, n, H, dh}, query.options());
    if (B && n) {
        ff_cache_attention_t a{};
        a.cache = c;
        const at::Tensor q = rows(query, &a.q_batch);
        if (mask.defined()) {
            mask = mask.contiguous();
            a.mask = (const uint8_t*)mask.data_ptr();
            a.mask_batch = mask.dim() == 3 ? n * n : 0;
        }
        a.q = q.data_ptr();
        a.out = out.data_ptr();
        a.H = H;
        a.o_batch = n * H * dh;
        a.o_head = dh;
        a.o_token = H * dh;
        a.scale = scale;
        a.stream = stream_of(query);
        a.ws_bytes = ff_cache_attention_workspace_bytes(&a);
        at::Tensor ws;
        if (a.ws_bytes) {
            ws = at::empty({(int64_t)a.ws_bytes}, query.options().dtype(at::kByte));
            a.ws = ws.data_ptr();
        }
        check(ff_cache_attention(&a), "ff_cache_attention");
    }
    return THPVariable_Wrap(out.transpose(1, 2));
    FF_END
}

// rotary(query, key, cos, sin, sections or None, interleaved, transpose) -> (query, key): the call without autograd
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    FF_CALL
    const char* what = "apply_rotary";
    begin(nargs, 7, what);
    at::Tensor query = tensor(args[0], what, "query"), key = tensor(args[1], what, "key"), cos = tensor(args[2], what, "cos"), sin = tensor(args[3], what, "sin");
    const bool interleaved = PyObject_IsTrue(args[5]) == 1, transpose = PyObject_IsTrue(args[6]) == 1;
    if (query.dim() != 4 || key.dim() != 4 || query.size(0) != key.size(0) || query.size(2) != key.size(2) || query.size(3) != key.size(3))
        refuse("apply_rotary: query ", query.sizes(), " and key ", key.sizes(), " must be [B, H, L, dh] and [B, H_kv, L, dh]");
    const at::ScalarType dtype = query.scalar_type();
    const at::Device device = query.device();
    if (code_of(dtype) < 0 || key.scalar_type() != dtype)
        refuse("apply_rotary: dtypes ", c10::toString(dtype), " / ", c10::toString(key.scalar_type()), " must be the same of float32, bfloat16, float16");
    if ((cos.scalar_type() != dtype && cos.scalar_type() != at::kFloat) || sin.scalar_type() != cos.scalar_type() || sin.sizes() != cos.sizes())
        refuse("apply_rotary: cos and sin must have one shape and the inputs' dtype or float32");
    if (key.device() != device || cos.device() != device || sin.device() != device) refuse("apply_rotary: all tensors must be on one device");
    ff_rotary_t a{};
    a.B = query.size(0);
    a.H = query.size(1);
    a.L = query.size(2);
    a.dh = query.size(3);
    a.H_kv = key.size(1);
    if (args[4] != Py_None) {
        PyObject* seq = PySequence_Fast(args[4], "apply_rotary: sections must be three integers");
        if (!seq) throw python_error();
        struct Release { PyObject* p; ~Release() { Py_DECREF(p); } } release{seq};
        int64_t s[3] = {0, 0, 0};
        bool fits = PySequence_Fast_GET_SIZE(seq) == 3;
        for (int i = 0; fits && i < 3; ++i) {
            s[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
            if (s[i] == -1 && PyErr_Occurred()) throw python_error();
            fits = s[i] > 0 && s[i] < (1 << 20);
        }
        if (!fits || cos.dim() != 4 || cos.size(0) != 3 || 2 * (s[0] + s[1] + s[2]) != cos.size(3) || interleaved)
            refuse("apply_rotary: sections need tables [3, B, L, 2 * their sum] in the half layout, got ", cos.sizes());
        a.sec0 = s[0];
        a.sec1 = s[1];
    } else if (cos.dim() != 3) {
        refuse("apply_rotary: tables must be [B or 1, L, rot] (or [3, ...] with sections), got ", cos.sizes());
    }
    a.rot = cos.size(-1);
    if ((cos.size(-3) != 1 && cos.size(-3) != a.B) || cos.size(-2) != a.L || a.rot % 2 || a.rot < 2 || a.rot > a.dh)
        refuse("apply_rotary: tables ", cos.sizes(), " do not fit query ", query.sizes());
    if (cos.requires_grad() || sin.requires_grad() || differentiable(cos) || differentiable(sin))
        refuse("apply_rotary: the tables are constants, they have no gradient");
    if (query._fw_grad(0).defined() || key._fw_grad(0).defined()) refuse("apply_rotary: tangents go through the autograd function");
    on_gpu(query, what);
    const c10::DeviceGuard guard(device);
    const at::AutoDispatchBelowADInplaceOrView below;          // (the caller has dealt with autograd)
    if (cos.stride(-1) != 1 || sin.strides() != cos.strides()) {
        cos = cos.contiguous();
        sin = sin.contiguous();
    }
    if (query.stride(3) != 1) query = query.contiguous();
    if (key.stride(3) != 1) key = key.contiguous();
    // outputs in the inputs' own order where they are dense
    at::Tensor q_out = at::empty_like(query), k_out = at::empty_like(key);
    if (q_out.stride(3) != 1) q_out = at::empty_like(query, at::MemoryFormat::Contiguous);
    if (k_out.stride(3) != 1) k_out = at::empty_like(key, at::MemoryFormat::Contiguous);
    if (a.B && a.L) {
        a.q = query.data_ptr();
        a.k = key.data_ptr();
        a.q_out = q_out.data_ptr();
        a.k_out = k_out.data_ptr();
        a.cos = cos.data_ptr();
        a.sin = sin.data_ptr();
        a.dtype = code_of(dtype);
        a.table_dtype = code_of(cos.scalar_type());
        const at::Tensor* t[4] = {&query, &key, &q_out, &k_out};
        int64_t* st[4] = {&a.q_batch, &a.k_batch, &a.qo_batch, &a.ko_batch};
        for (int i = 0; i < 4; ++i)
            for (int d = 0; d < 3; ++d) st[i][d] = t[i]->stride(d);
        a.t_axis = cos.dim() == 4 ? cos.stride(0) : 0;
        a.t_batch = cos.size(-3) > 1 ? cos.stride(-3) : 0;
        a.t_token = cos.stride(-2);
        a.interleaved = interleaved;
        a.transpose = transpose;
        a.stream = stream_of(query);
        check(ff_rotary_apply(&a), "ff_rotary_apply");
    }
    PyObject *q = THPVariable_Wrap(std::move(q_out)), *k = THPVariable_Wrap(std::move(k_out));
    return Py_BuildValue("(NN)", q, k);
    FF_END
}

PyMethodDef g_methods[] = {
    {"not_traced", py_not_traced, METH_O, "not_traced(what): raises while a tracer records"},
    {"write", (PyCFunction)(void (*)(void))py_write, METH_FASTCALL, "write(cache, key, value, table, start)"},
    {"read", (PyCFunction)(void (*)(void))py_read, METH_FASTCALL, "read(cache, table, start, count, dtype) -> (key, value)"},
    {"keep", (PyCFunction)(void (*)(void))py_keep, METH_FASTCALL, "keep(cache, table, start, accepted)"},
    {"attention", (PyCFunction)(void (*)(void))py_attention, METH_FASTCALL, "attention(query, cache, table, start, mask, scale) -> out"},
    {"rotary", (PyCFunction)(void (*)(void))py_rotary, METH_FASTCALL, "rotary(query, key, cos, sin, sections, interleaved, transpose) -> (query, key)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", "checks, outputs and launches of the cached-decoding calls", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    // the structures below are passed to the library as they are: both must come from the same sources
    const size_t mine[4] = {sizeof(ff_rotary_t), sizeof(ff_cache_t), sizeof(ff_cache_rows_t), sizeof(ff_cache_attention_t)};
    bool same = std::string(ff_source_hash()) == ff_host_stamp + 10;
    for (int i = 0; i < 4; ++i) same = same && ff_abi_sizeof(6 + i) == mine[i];
    if (!same) {
        PyErr_Format(PyExc_ImportError, "_host.so was built from other sources (%s) than the library beside it (%s)", ff_host_stamp + 10, ff_source_hash());
        return nullptr;
    }
    PyObject* lib = PyImport_ImportModule("framefusion_amd._lib");
    if (!lib) return nullptr;
    g_error = PyObject_GetAttrString(lib, "FrameFusionHipError");
    Py_DECREF(lib);
    if (!g_error) return nullptr;
    return PyModule_Create(&g_module);
}
