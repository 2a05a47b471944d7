// torch_op.cpp — the Python call surface of op.py in native code: torch tensors to b200_tensor descriptors, output and
// workspace from torch's caching allocator, one planned launch through the C-ABI.
//
// A decode step of a small model is a few launches of 4-8 us each, so what a call costs on the host decides the step:
// the same work in Python (about sixty attribute reads and ctypes objects per call, the operator planned twice) took
// 27-33 us per call, this module 4 us, most of it the kernel launch and the output allocation.  A 6-layer step of Whisper
// base.en (12 calls) 400 -> 58 us and, as vector calls without a Python function in front, 54 us; a 30-layer Q8_0 decoder
// step (60 calls) 1604 -> 492 us before its kernels became faster.
#include <Python.h>

#include <exception>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDADevice.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b200_fattn.h"

namespace {

// Interned names of the arguments, compared by pointer first (keyword names of call sites are interned).
enum Key { kScale, kMaxBias, kSoftcap, kKvType, kCausal, kNPast, kKvLen, kQv, kR, kRelposF32, kBiasU, kBiasV, kKvIndex, kQLen, kOut,
           kWorkspace, kStream, kQ, kK, kV, kMask, kKeys };
const char* const kKeyNames[kKeys] = {"scale", "max_bias", "softcap", "kv_type", "causal", "n_past", "kv_len", "q_v", "r",
                                      "relpos_bias_f32", "pos_bias_u", "pos_bias_v", "kv_index", "q_len", "out", "workspace", "stream",
                                      "q", "k", "v", "mask"};
PyObject* g_keys[kKeys];

struct Kwargs {
    PyObject* v[kKeys] = {};   // borrowed; null = absent, or None where that is a value (a number has to be one)
    // `values`: those of the keyword names, behind the positional arguments of a vector call
    bool parse(PyObject* names, PyObject* const* values) {
        const Py_ssize_t n = names ? PyTuple_GET_SIZE(names) : 0;
        for (Py_ssize_t j = 0; j < n; j++) {
            PyObject* name = PyTuple_GET_ITEM(names, j);
            int hit = -1;
            for (int i = 0; i < kKeys && hit < 0; i++)
                if (name == g_keys[i]) hit = i;
            for (int i = 0; i < kKeys && hit < 0; i++)
                if (PyUnicode_Compare(name, g_keys[i]) == 0) hit = i;
            if (PyErr_Occurred()) return false;
            const bool number = hit == kScale || hit == kMaxBias || hit == kSoftcap || hit == kNPast;
            if (hit >= 0) v[hit] = values[j] == Py_None && !number ? nullptr : values[j];   // other names are ignored, as they always were
        }
        return true;
    }
    // q, k, v, mask: by position or by name
    bool operands(PyObject* const* a, Py_ssize_t n, const char* where, PyObject* (&op)[4]) const {
        if (n > 4) {
            PyErr_Format(PyExc_TypeError, "%s() takes from 3 to 4 positional arguments but %zd were given", where, n);
            return false;
        }
        for (int i = 0; i < 4; i++) {
            if (i < n && v[kQ + i]) {
                PyErr_Format(PyExc_TypeError, "%s() got multiple values for argument '%s'", where, kKeyNames[kQ + i]);
                return false;
            }
            op[i] = i < n ? a[i] : v[kQ + i];
            if (!op[i] && i < 3) {
                PyErr_Format(PyExc_TypeError, "%s() missing required argument '%s'", where, kKeyNames[kQ + i]);
                return false;
            }
        }
        return true;
    }
    bool number(Key k, double dflt, double* out) const {
        if (!v[k]) return *out = dflt, true;
        PyObject* f = PyNumber_Float(v[k]);   // float(x): texts as well
        if (!f) return false;
        *out = PyFloat_AS_DOUBLE(f);
        Py_DECREF(f);
        return true;
    }
    bool integer(Key k, long* out) const {
        if (!v[k]) return *out = 0, true;
        PyObject* i = PyNumber_Long(v[k]);
        if (!i) return false;
        *out = PyLong_AsLong(i);
        Py_DECREF(i);
        return !(*out == -1 && PyErr_Occurred());
    }
    bool truth(Key k, int32_t* out) const {
        const int t = v[k] ? PyObject_IsTrue(v[k]) : 0;
        *out = t;
        return t >= 0;
    }
};

const at::Tensor* tensor_of(PyObject* o, const char* what) {
    if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
    PyErr_Format(PyExc_TypeError, "%s is a torch tensor, not %s", what, Py_TYPE(o)->tp_name);
    return nullptr;
}

// torch order (slowest first) -> ggml order; absent dimensions get the strides of the full extent.
bool describe(const at::Tensor& x, long type, b200_tensor* t) {
    const auto st = x.scalar_type();
    if (type < 0) {
        if (st == at::kFloat) type = B200_TYPE_F32;
        else if (st == at::kHalf) type = B200_TYPE_F16;
        else {
            PyErr_Format(PyExc_KeyError, "torch.%s", c10::toString(st));
            return false;
        }
    }
    const int nd = (int)x.dim();
    if (nd > 4) {
        PyErr_SetString(PyExc_ValueError, "at most 4 dimensions");
        return false;
    }
    const int64_t block = type == B200_TYPE_Q8_0 ? 34 : (type == B200_TYPE_Q4_0 ? 18 : 0);   // bytes of 32 values
    if (block && (st != at::kByte || nd == 0 || x.stride(-1) != 1)) {
        PyErr_Format(PyExc_ValueError, "%s tensors are uint8 with a contiguous last axis", block == 34 ? "Q8_0" : "Q4_0");
        return false;
    }
    const int64_t es = x.element_size();
    t->data = x.data_ptr();
    t->type = (int32_t)type;
    t->reserved = 0;
    for (int i = 0; i < 4; i++) t->ne[i] = 1, t->nb[i] = 0;
    for (int i = 0; i < nd; i++) {
        t->ne[i] = x.size(nd - 1 - i);
        t->nb[i] = (uint64_t)(x.stride(nd - 1 - i) * es);
    }
    if (block) t->ne[0] = t->ne[0] / block * 32, t->nb[0] = (uint64_t)block;
    if (nd == 0) t->nb[0] = (uint64_t)es;
    for (int i = nd > 1 ? nd : 1; i < 4; i++) t->nb[i] = t->nb[i - 1] * (uint64_t)(block && i == 1 ? t->ne[0] / 32 : t->ne[i - 1]);
    return true;
}

// Address of an index table: a torch tensor's, that of any other object with data_ptr(), or a numpy array's.
bool address_of(PyObject* o, const int32_t** out) {
    if (THPVariable_Check(o)) {
        *out = (const int32_t*)THPVariable_Unpack(o).data_ptr();
        return true;
    }
    PyObject* data = nullptr;
    if (PyObject_HasAttrString(o, "data_ptr")) {
        data = PyObject_CallMethod(o, "data_ptr", nullptr);
    } else {
        PyObject* ct = PyObject_GetAttrString(o, "ctypes");
        data = ct ? PyObject_GetAttrString(ct, "data") : nullptr;
        Py_XDECREF(ct);
    }
    if (!data) return false;
    *out = (const int32_t*)PyLong_AsVoidPtr(data);
    Py_DECREF(data);
    return !PyErr_Occurred();
}

bool last_extent(PyObject* o, int32_t* out) {
    if (THPVariable_Check(o)) {
        *out = (int32_t)THPVariable_Unpack(o).size(-1);
        return true;
    }
    PyObject* shape = PyObject_GetAttrString(o, "shape");
    const Py_ssize_t n = shape ? PySequence_Length(shape) : -1;
    PyObject* last = n > 0 ? PySequence_GetItem(shape, n - 1) : nullptr;
    Py_XDECREF(shape);
    if (!last) return false;
    *out = (int32_t)PyLong_AsLong(last);
    Py_DECREF(last);
    return !PyErr_Occurred();
}

// Stream handle: None (the caller picks), an integer, a ctypes pointer, or an object that has one for ctypes (`_as_parameter_`:
// torch.cuda.Stream).
bool stream_of(PyObject* o, void** out) {
    if (PyLong_Check(o)) {
        *out = PyLong_AsVoidPtr(o);
        return !PyErr_Occurred();
    }
    if (PyObject* as = PyObject_GetAttrString(o, "_as_parameter_")) {
        const bool ok = PyLong_Check(as) || PyObject_HasAttrString(as, "value");
        if (!ok) PyErr_SetString(PyExc_TypeError, "stream is an integer, a ctypes pointer or a torch.cuda.Stream");
        const bool got = ok && stream_of(as, out);
        Py_DECREF(as);
        return got;
    }
    PyErr_Clear();
    PyObject* value = PyObject_GetAttrString(o, "value");
    if (!value) return false;
    *out = value == Py_None ? nullptr : PyLong_AsVoidPtr(value);
    Py_DECREF(value);
    return !PyErr_Occurred();
}

PyObject* raise_code(int rc, const char* where) {
    PyObject* mod = PyImport_ImportModule("crispasr_b200");
    PyObject* cls = mod ? PyObject_GetAttrString(mod, "B200Error") : nullptr;
    PyObject* err = cls ? PyObject_CallFunction(cls, "is", rc, where) : nullptr;
    if (err) PyErr_SetObject(cls, err);
    Py_XDECREF(err);
    Py_XDECREF(cls);
    Py_XDECREF(mod);
    return nullptr;
}

struct Operands {
    b200_tensor q, k, v, mask, dst, qv, r, bu, bv;
    bool has_mask = false;
    b200_fattn_params params;
    b200_fattn_ext ext;
    const b200_tensor* mask_p() const { return has_mask ? &mask : nullptr; }

    bool fill(PyObject* q_, PyObject* k_, PyObject* v_, PyObject* mask_, const Kwargs& kw) {
        if (!kw.v[kScale]) {
            PyErr_SetString(PyExc_KeyError, "scale");
            return false;
        }
        long kv_type = -1, n_past = 0;
        if (kw.v[kKvType] && !kw.integer(kKvType, &kv_type)) return false;
        const at::Tensor *tk = tensor_of(k_, "k"), *tv = tk ? tensor_of(v_, "v") : nullptr;
        if (!tv || !describe(THPVariable_Unpack(q_), -1, &q) || !describe(*tk, kv_type, &k) || !describe(*tv, kv_type, &v)) return false;
        if (mask_ && mask_ != Py_None) {
            const at::Tensor* tm = tensor_of(mask_, "mask");
            if (!tm || !describe(*tm, -1, &mask)) return false;
            has_mask = true;
        }
        double scale, max_bias, softcap;
        if (!kw.number(kScale, 0.0, &scale) || !kw.number(kMaxBias, 0.0, &max_bias) || !kw.number(kSoftcap, 0.0, &softcap)) return false;
        params = b200_fattn_params{(float)scale, (float)max_bias, (float)softcap, 0};
        ext = b200_fattn_ext{};
        const struct { Key key; b200_tensor* t; const b200_tensor** slot; const char* name; } opt[4] = {
            {kQv, &qv, &ext.q_v, "q_v"}, {kR, &r, &ext.r, "r"}, {kBiasU, &bu, &ext.pos_bias_u, "pos_bias_u"}, {kBiasV, &bv, &ext.pos_bias_v, "pos_bias_v"}};
        for (const auto& o : opt)
            if (kw.v[o.key]) {
                const at::Tensor* t = tensor_of(kw.v[o.key], o.name);
                if (!t || !describe(*t, -1, o.t)) return false;
                *o.slot = o.t;
            }
        if (!kw.truth(kCausal, &ext.causal) || !kw.integer(kNPast, &n_past) || !kw.truth(kRelposF32, &ext.relpos_bias_f32)) return false;
        ext.n_past = (int32_t)n_past;
        if (kw.v[kKvLen] && !address_of(kw.v[kKvLen], &ext.kv_len)) return false;
        if (kw.v[kKvIndex] && (!address_of(kw.v[kKvIndex], &ext.kv_index) || !last_extent(kw.v[kKvIndex], &ext.kv_index_stride))) return false;
        return !kw.v[kQLen] || address_of(kw.v[kQLen], &ext.q_len);
    }
};

// While it lives, tensors made here come from the pool of the stream that a launch goes to: a block of the current stream's pool may still be in
// use by that stream's earlier work, and would be handed out again while the launch is in flight.
struct PoolOf {
    c10::cuda::OptionalCUDAStreamGuard on_stream;
    PoolOf(void* stream, c10::Device device) {
        const cudaStream_t st = stream == (void*)cudaStreamLegacy ? nullptr : (cudaStream_t)stream;
        if (st != c10::cuda::getCurrentCUDAStream(device.index()).stream()) on_stream.reset_stream(c10::cuda::getStreamFromExternal(st, device.index()));
    }
};

struct Scratch {
    at::Tensor buf;
    c10::Device device;
    void* given;
    size_t given_bytes;
    void* stream;   // the launch's
    std::exception_ptr error;   // what the allocator raised: it must not pass through the C entry point, the caller gets it behind that
};
void* scratch_alloc(void* user, size_t bytes) {
    Scratch* s = (Scratch*)user;
    if (s->given && s->given_bytes >= bytes) return s->given;
    try {
        const PoolOf pool(s->stream, s->device);
        s->buf = at::detail::empty_cuda({(int64_t)bytes}, at::kByte, s->device, std::nullopt);
    } catch (...) {
        s->error = std::current_exception();
        return nullptr;
    }
    return s->buf.data_ptr();
}

const char kLaunchDoc[] =
    "flash_attn_ext(q, k, v, mask=None, *, out=None, workspace=None, stream=None, **kw)\n--\n\n"
    "Device tensors in, device tensor out; asynchronous on `stream` (default: torch's current stream).\n"
    "`workspace` (uint8 device tensor) is allocated here, for `stream`, when the launch needs one and none is given; the\n"
    "result comes from the current stream's pool, as any tensor made here would.";

PyObject* launch_py(PyObject*, PyObject* const* a, Py_ssize_t n, PyObject* names) {
    HANDLE_TH_ERRORS
    Kwargs kw;
    PyObject* in[4];
    if (!kw.parse(names, a + n) || !kw.operands(a, n, "flash_attn_ext", in)) return nullptr;
    const at::Tensor* q = tensor_of(in[0], "q");
    if (!q) return nullptr;
    if (!q->is_cuda()) {
        PyErr_SetString(PyExc_ValueError, "flash_attn_ext takes CUDA tensors; use flash_attn_ext_host for host buffers");
        return nullptr;
    }
    const c10::cuda::CUDAGuard guard(q->device());
    PyObject* out = kw.v[kOut];
    at::Tensor made;
    if (!out) {
        if (q->dim() != 4) {
            PyErr_SetString(PyExc_ValueError, "q is (B, H, Tq, hd)");
            return nullptr;
        }
        made = at::detail::empty_cuda({q->size(0), q->size(2), q->size(1), q->size(3)}, at::kFloat, q->device(), std::nullopt);
    }
    const at::Tensor* dst = out ? tensor_of(out, "out") : &made;
    Operands op;
    if (!dst || !op.fill(in[0], in[1], in[2], in[3], kw) || !describe(*dst, -1, &op.dst)) return nullptr;
    Scratch ws{at::Tensor(), q->device(), nullptr, 0, nullptr, nullptr};
    if (kw.v[kWorkspace]) {
        const at::Tensor* w = tensor_of(kw.v[kWorkspace], "workspace");
        if (!w) return nullptr;
        ws.given = w->data_ptr(), ws.given_bytes = (size_t)w->numel();
    }
    void* st = nullptr;
    if (!kw.v[kStream]) st = c10::cuda::getCurrentCUDAStream(q->device().index()).stream();
    else if (!stream_of(kw.v[kStream], &st)) return nullptr;
    ws.stream = st;
    int rc;
    Py_BEGIN_ALLOW_THREADS   // a full launch queue blocks: other host threads go on meanwhile
    rc = b200_fattn_launch_alloc(&op.q, &op.k, &op.v, op.mask_p(), &op.dst, &op.params, &op.ext, scratch_alloc, &ws, st);
    Py_END_ALLOW_THREADS
    if (ws.error) std::rethrow_exception(ws.error);   // torch.OutOfMemoryError, as from any other allocation
    if (rc) return raise_code(rc, "b200_fattn_launch");
    if (!out) return THPVariable_Wrap(std::move(made));
    Py_INCREF(out);
    return out;
    END_HANDLE_TH_ERRORS
}

const char kHostDoc[] =
    "flash_attn_ext_host(q, k, v, mask=None, *, out=None, **kw)\n--\n\n"
    "Host (CPU, ideally pinned) tensors in, host tensor out: H2D, compute, D2H inside one C call.";

PyObject* forward_host_py(PyObject*, PyObject* const* a, Py_ssize_t n, PyObject* names) {
    HANDLE_TH_ERRORS
    Kwargs kw;
    PyObject* in[4];
    if (!kw.parse(names, a + n) || !kw.operands(a, n, "flash_attn_ext_host", in)) return nullptr;
    const at::Tensor* q = tensor_of(in[0], "q");
    if (!q) return nullptr;
    PyObject* out = kw.v[kOut];
    at::Tensor made;
    if (!out) {
        if (q->dim() != 4) {
            PyErr_SetString(PyExc_ValueError, "q is (B, H, Tq, hd)");
            return nullptr;
        }
        made = at::empty({q->size(0), q->size(2), q->size(1), q->size(3)}, q->options().dtype(at::kFloat));
    }
    const at::Tensor* dst = out ? tensor_of(out, "out") : &made;
    Operands op;
    if (!dst || !op.fill(in[0], in[1], in[2], in[3], kw) || !describe(*dst, -1, &op.dst)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = b200_fattn_forward_host(&op.q, &op.k, &op.v, op.mask_p(), &op.dst, &op.params, &op.ext);
    Py_END_ALLOW_THREADS
    if (rc) return raise_code(rc, "b200_fattn_forward_host");
    if (!out) return THPVariable_Wrap(std::move(made));
    Py_INCREF(out);
    return out;
    END_HANDLE_TH_ERRORS
}

// A layer's index or a row's; one that passes 32 bits is no other's.
bool index_of(PyObject* o, const char* what, int32_t* out) {
    const long i = PyLong_AsLong(o);
    if (i == -1 && PyErr_Occurred()) return false;
    if (i != (int32_t)i) {
        PyErr_Format(PyExc_OverflowError, "%s is a 32-bit number", what);
        return false;
    }
    *out = (int32_t)i;
    return true;
}

// (cache address, layer, k_new, v_new, pos, pos0, stream)
PyObject* kv_append_py(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "kv_append takes 7 arguments");
        return nullptr;
    }
    HANDLE_TH_ERRORS
    b200_kv_cache* kv = (b200_kv_cache*)PyLong_AsVoidPtr(a[0]);
    int32_t layer = 0, pos0 = 0;
    if (PyErr_Occurred() || !index_of(a[1], "layer", &layer)) return nullptr;
    PyObject* p0 = PyNumber_Long(a[5]);   // int(pos0): floats as well
    if (!p0) return nullptr;
    const bool ok = index_of(p0, "pos0", &pos0);
    Py_DECREF(p0);
    if (!ok) return nullptr;
    const at::Tensor *k = tensor_of(a[2], "k_new"), *v = k ? tensor_of(a[3], "v_new") : nullptr;
    b200_tensor tk, tv;
    if (!v || !describe(*k, -1, &tk) || !describe(*v, -1, &tv)) return nullptr;
    const int32_t* pos = nullptr;
    if (a[4] != Py_None && !PyObject_HasAttrString(a[4], "data_ptr")) {   // (read by the kernel: a numpy array has no device address)
        PyErr_Format(PyExc_TypeError, "pos is a torch tensor, not %s", Py_TYPE(a[4])->tp_name);
        return nullptr;
    }
    if (a[4] != Py_None && !address_of(a[4], &pos)) return nullptr;
    if (a[6] == Py_None && !k->is_cuda()) {
        PyErr_SetString(PyExc_ValueError, "kv_append takes CUDA tensors");
        return nullptr;
    }
    void* st = nullptr;
    if (a[6] == Py_None) st = c10::cuda::getCurrentCUDAStream(k->device().index()).stream();
    else if (!stream_of(a[6], &st)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = b200_kv_append(kv, layer, &tk, &tv, pos, pos0, st);
    Py_END_ALLOW_THREADS
    if (rc) return raise_code(rc, "b200_kv_append");
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// ---- norm, rotation and append; reading rows back ----------------------------------------------------------------------------

// The arguments of the rotation's calls; all by keyword, unknown names are an error.
enum RopeKey { rQNorm, rKNorm, rEps, rDims, rBase, rScale, rNeox, rPos, rPos0, rNRows, rOut, rKOut, rStream, rKeys };
const char* const kRopeNames[rKeys] = {"q_norm", "k_norm", "eps", "rope_dims", "rope_base", "rope_scale", "neox", "pos", "pos0", "n_rows", "out", "k_out", "stream"};
PyObject *g_rope_keys[rKeys], *g_handle, *g_value;

// An int32 table on the device of `like`, one entry per stream.
bool table_of(PyObject* o, const char* what, const at::Tensor& like, int64_t streams, const int32_t** out) {
    const at::Tensor* t = tensor_of(o, what);
    if (!t) return false;
    if (t->scalar_type() != at::kInt || t->device() != like.device() || t->numel() != streams || !t->is_contiguous()) {
        PyErr_Format(PyExc_ValueError, "%s is a contiguous int32 tensor of %lld entries on the rows' device", what, (long long)streams);
        return false;
    }
    *out = (const int32_t*)t->data_ptr();
    return true;
}

bool rows_of(PyObject* o, const char* what, const at::Tensor* like, const at::Tensor** out) {
    const at::Tensor* t = tensor_of(o, what);
    if (!t) return false;
    if (!t->is_cuda() || (like && t->device() != like->device())) {
        PyErr_Format(PyExc_ValueError, like ? "%s is on another device than the other rows" : "%s is a CUDA tensor", what);
        return false;
    }
    if (t->dim() != 4) {
        PyErr_Format(PyExc_ValueError, "%s is (streams, heads, rows, head_dim)", what);
        return false;
    }
    *out = t;
    return true;
}

struct RopeCall {
    PyObject* v[rKeys] = {};   // borrowed
    b200_rope_params params{0, B200_ROPE_NEOX, 10000.0f, 1.0f, 1e-6f, 0};
    b200_tensor norm[2];
    const b200_tensor* norm_p[2] = {nullptr, nullptr};
    const int32_t *pos = nullptr, *n_rows = nullptr;
    int32_t pos0 = 0;
    void* stream = nullptr;

    bool parse(PyObject* names, PyObject* const* values, const char* where) {
        const Py_ssize_t n = names ? PyTuple_GET_SIZE(names) : 0;
        for (Py_ssize_t j = 0; j < n; j++) {
            PyObject* name = PyTuple_GET_ITEM(names, j);
            int hit = -1;
            for (int i = 0; i < rKeys && hit < 0; i++)
                if (name == g_rope_keys[i]) hit = i;
            for (int i = 0; i < rKeys && hit < 0; i++)
                if (PyUnicode_Compare(name, g_rope_keys[i]) == 0) hit = i;
            if (PyErr_Occurred()) return false;
            if (hit < 0) {
                PyErr_Format(PyExc_TypeError, "%s() got an unexpected keyword argument '%U'", where, name);
                return false;
            }
            v[hit] = values[j] == Py_None ? nullptr : values[j];
        }
        return true;
    }
    bool number(RopeKey k, float* out) const {
        if (!v[k]) return true;
        const double d = PyFloat_AsDouble(v[k]);
        if (d == -1.0 && PyErr_Occurred()) return false;
        *out = (float)d;
        return true;
    }
    bool integer(RopeKey k, int32_t* out) const {
        if (!v[k]) return true;
        const long i = PyLong_AsLong(v[k]);
        if (i == -1 && PyErr_Occurred()) return false;
        if (i != (int32_t)i) {
            PyErr_Format(PyExc_OverflowError, "%s is a 32-bit number", kRopeNames[k]);
            return false;
        }
        *out = (int32_t)i;
        return true;
    }
    // What the call says beside its rows; `like`: (streams, heads, rows, head_dim).
    bool fill(const at::Tensor& like) {
        params.n_dims = (int32_t)like.size(3);
        if (!number(rEps, &params.eps) || !number(rBase, &params.freq_base) || !number(rScale, &params.freq_scale) || !integer(rDims, &params.n_dims) ||
            !integer(rPos0, &pos0))
            return false;
        if (v[rNeox]) {
            const int t = PyObject_IsTrue(v[rNeox]);
            if (t < 0) return false;
            params.mode = t ? B200_ROPE_NEOX : B200_ROPE_NORM;
        }
        for (int x = 0; x < 2; x++) {
            const RopeKey key = x ? rKNorm : rQNorm;
            if (!v[key]) continue;
            const at::Tensor* w = tensor_of(v[key], kRopeNames[key]);
            if (!w) return false;
            if (w->device() != like.device()) {
                PyErr_Format(PyExc_ValueError, "%s is on another device than the rows", kRopeNames[key]);
                return false;
            }
            if (!describe(*w, -1, &norm[x])) return false;
            norm_p[x] = &norm[x];
        }
        if (v[rPos] && !table_of(v[rPos], "pos", like, like.size(0), &pos)) return false;
        if (v[rNRows] && !table_of(v[rNRows], "n_rows", like, like.size(0), &n_rows)) return false;
        if (!v[rStream]) stream = c10::cuda::getCurrentCUDAStream(like.device().index()).stream();
        else if (!stream_of(v[rStream], &stream)) return false;
        return true;
    }
    // The rows that a call writes: given, or made here (after fill: the stream is known).
    const at::Tensor* output(RopeKey k, const at::Tensor& like, at::ScalarType type, at::Tensor* made) const {
        const at::Tensor* out = made;
        if (v[k]) return rows_of(v[k], kRopeNames[k], &like, &out) ? out : nullptr;
        const PoolOf pool(stream, like.device());
        *made = at::detail::empty_cuda(like.sizes(), type, like.device(), std::nullopt);
        return out;
    }
};

const char kQkRopeDoc[] =
    "qk_norm_rope(q, k=None, *, q_norm=None, k_norm=None, eps=1e-6, rope_dims=head_dim, rope_base=10000.0, rope_scale=1.0, neox=True,\n"
    "             pos=None, pos0=0, n_rows=None, out=None, k_out=None, stream=None)\n--\n\n"
    "Norm of every head (where a weight is given) and rotation by position of q (streams, heads, rows, head_dim) and k (streams,\n"
    "kv heads, rows, head_dim), F32 or F16: (rotated q, rotated k or None), of q's type unless `out` and `k_out` say otherwise (they may\n"
    "be q and k).  Row i of stream s is at position pos[s] + i (`pos` an int32 CUDA tensor, else `pos0` for all); rows at or\n"
    "beyond n_rows[s] (an int32 CUDA tensor) are zeros.  Asynchronous on `stream` (default: torch's current stream), from whose pool the results are: a caller that\n"
    "uses them on another stream orders the two and says so to the allocator (record_stream).";

PyObject* qk_norm_rope_py(PyObject*, PyObject* const* a, Py_ssize_t n, PyObject* names) {
    HANDLE_TH_ERRORS
    if (n < 1 || n > 2) {
        PyErr_SetString(PyExc_TypeError, "qk_norm_rope() takes 1 or 2 positional arguments (q, k)");
        return nullptr;
    }
    RopeCall call;
    const at::Tensor *q = nullptr, *k = nullptr;
    if (!call.parse(names, a + n, "qk_norm_rope") || !rows_of(a[0], "q", nullptr, &q)) return nullptr;
    if (n > 1 && a[1] != Py_None && !rows_of(a[1], "k", q, &k)) return nullptr;
    if (!k && call.v[rKOut]) {
        PyErr_SetString(PyExc_ValueError, "k_out without k");
        return nullptr;
    }
    const c10::cuda::CUDAGuard guard(q->device());
    if (!call.fill(*q)) return nullptr;
    b200_tensor tq, tk, to, tko;
    at::Tensor made, made_k;
    const at::Tensor *out = nullptr, *k_out = nullptr;
    if (!describe(*q, -1, &tq) || (k && !describe(*k, -1, &tk)) || !(out = call.output(rOut, *q, q->scalar_type(), &made)) || !describe(*out, -1, &to)) return nullptr;
    if (k && (!(k_out = call.output(rKOut, *k, out->scalar_type(), &made_k)) || !describe(*k_out, -1, &tko))) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = b200_qk_norm_rope(&tq, k ? &tk : nullptr, call.norm_p[0], call.norm_p[1], &call.params, call.pos, call.pos0, call.n_rows, &to, k ? &tko : nullptr, call.stream);
    Py_END_ALLOW_THREADS
    if (rc) return raise_code(rc, "b200_qk_norm_rope");
    PyObject* first = THPVariable_Wrap(*out);
    PyObject* second = k ? THPVariable_Wrap(*k_out) : Py_NewRef(Py_None);
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

// The address in a KvCache object (its `_h`, a ctypes pointer; null after close()).
bool cache_of(PyObject* self, b200_kv_cache** out) {
    PyObject* h = PyObject_GetAttr(self, g_handle);
    PyObject* value = h ? PyObject_GetAttr(h, g_value) : nullptr;
    Py_XDECREF(h);
    if (!value) return false;
    *out = value == Py_None ? nullptr : (b200_kv_cache*)PyLong_AsVoidPtr(value);
    Py_DECREF(value);
    return !PyErr_Occurred();
}

const char kAppendRopeDoc[] =
    "append_rope(self, layer, q, k_new, v_new, *, q_norm=None, k_norm=None, eps=1e-6, rope_dims=head_dim, rope_base=10000.0, rope_scale=1.0,\n"
    "            neox=True, pos=None, pos0=0, n_rows=None, out=None, stream=None)\n--\n\n"
    "Norm (where a weight is given) and rotation of q (n_streams, heads, n_new, hd; or None) and k_new (n_streams, n_kv, n_new, hd), and\n"
    "k_new and v_new into the cache.  All float32 or all float16 CUDA tensors.  Row i of stream s is at position pos[s] + i, which is\n"
    "also its place in the cache; the other arguments, and the order of streams, as in qk_norm_rope.  Returns the\n"
    "rotated q, float16 unless `out` says otherwise.";

// A method of KvCache: called with the object in front.
PyObject* kv_append_rope_py(PyObject*, PyObject* const* a, Py_ssize_t n, PyObject* names) {
    HANDLE_TH_ERRORS
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "append_rope() takes 4 positional arguments (layer, q, k_new, v_new)");
        return nullptr;
    }
    b200_kv_cache* kv = nullptr;
    if (!cache_of(a[0], &kv)) return nullptr;
    int32_t layer = 0;
    if (!index_of(a[1], "layer", &layer)) return nullptr;
    RopeCall call;
    const at::Tensor *q = nullptr, *k = nullptr, *v = nullptr;
    if (!call.parse(names, a + n, "append_rope") || !rows_of(a[3], "k_new", nullptr, &k) || !rows_of(a[4], "v_new", k, &v)) return nullptr;
    if (a[2] != Py_None && !rows_of(a[2], "q", k, &q)) return nullptr;
    if (call.v[rKOut] || (!q && call.v[rOut])) {
        PyErr_SetString(PyExc_TypeError, call.v[rKOut] ? "append_rope() has no k_out: k goes into the cache" : "append_rope() got out without q");
        return nullptr;
    }
    const c10::cuda::CUDAGuard guard(k->device());
    if (!call.fill(*k)) return nullptr;
    b200_tensor tq, tk, tv, to;
    at::Tensor made;
    const at::Tensor* out = nullptr;
    if (!describe(*k, -1, &tk) || !describe(*v, -1, &tv)) return nullptr;
    if (q && (!describe(*q, -1, &tq) || !(out = call.output(rOut, *q, at::kHalf, &made)) || !describe(*out, -1, &to))) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = b200_kv_append_rope(kv, layer, q ? &tq : nullptr, &tk, &tv, call.norm_p[0], call.norm_p[1], &call.params, call.pos, call.pos0, call.n_rows,
                             q ? &to : nullptr, call.stream);
    Py_END_ALLOW_THREADS
    if (rc) return raise_code(rc, "b200_kv_append_rope");
    if (!q) Py_RETURN_NONE;
    return THPVariable_Wrap(*out);
    END_HANDLE_TH_ERRORS
}

int device_of_cache(const void* p) { return at::cuda::getDeviceFromPtr(const_cast<void*>(p)).index(); }

// (cache address, cache object, layer, n_rows): the views of kv_view as torch tensors that keep the cache object alive
PyObject* kv_tensors_py(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "kv_tensors takes 4 arguments");
        return nullptr;
    }
    HANDLE_TH_ERRORS
    const b200_kv_cache* kv = (const b200_kv_cache*)PyLong_AsVoidPtr(a[0]);
    int32_t layer = 0;
    const long rows = PyLong_AsLong(a[3]);
    if (PyErr_Occurred() || !index_of(a[2], "layer", &layer)) return nullptr;
    b200_tensor t[2];
    const int rc = b200_kv_view(kv, layer, rows, &t[0], &t[1]);
    if (rc) return raise_code(rc, "b200_kv_view");
    PyObject* views[2];
    for (int i = 0; i < 2; i++) {
        const bool f16 = t[i].type == B200_TYPE_F16;
        const int64_t es = f16 ? 2 : 1, width = f16 ? t[i].ne[0] : t[i].ne[0] / 32 * (int64_t)t[i].nb[0];
        const int64_t sizes[4] = {t[i].ne[3], t[i].ne[2], t[i].ne[1], width};
        const int64_t strides[4] = {(int64_t)t[i].nb[3] / es, (int64_t)t[i].nb[2] / es, (int64_t)t[i].nb[1] / es, 1};
        PyObject* owner = Py_NewRef(a[1]);
        views[i] = THPVariable_Wrap(at::from_blob(
            t[i].data, sizes, strides,
            [owner](void*) {
                if (!Py_IsInitialized()) return;
                const PyGILState_STATE gil = PyGILState_Ensure();
                Py_DECREF(owner);
                PyGILState_Release(gil);
            },
            at::TensorOptions().dtype(f16 ? at::kHalf : at::kByte).device(at::kCUDA, (c10::DeviceIndex)device_of_cache(t[i].data))));
    }
    PyObject* both = views[0] && views[1] ? PyTuple_Pack(2, views[0], views[1]) : nullptr;
    Py_XDECREF(views[0]);
    Py_XDECREF(views[1]);
    return both;
    END_HANDLE_TH_ERRORS
}

const char kReadDoc[] =
    "read(self, layer, n_rows, pos=None, pos0=0, dtype=None, out=None, stream=None)\n--\n\n"
    "Rows pos[s] .. pos[s] + n_rows - 1 of every stream (`pos` an int32 CUDA tensor, else `pos0` for all) as values: (K, V), each\n"
    "(n_streams, n_kv, n_rows, hd) float16, or float32 if `dtype` says so, or the pair `out`.  Rows outside the cache are\n"
    "zeros.  Asynchronous on `stream` (default: torch's current stream), from whose pool the results are.";

// A method of KvCache: called with the object in front.
PyObject* kv_read_py(PyObject*, PyObject* const* in, Py_ssize_t n, PyObject* names) {
    HANDLE_TH_ERRORS
    enum { kLayer, kRows, kPos, kPos0, kDtype, kOutPair, kOn, kArgs };
    static const char* const arg_names[kArgs] = {"layer", "n_rows", "pos", "pos0", "dtype", "out", "stream"};
    PyObject* a[kArgs] = {};
    if (n < 1 || n > kArgs + 1) {
        PyErr_SetString(PyExc_TypeError, "read() takes from 2 to 7 arguments");
        return nullptr;
    }
    for (Py_ssize_t i = 1; i < n; i++) a[i - 1] = in[i];
    for (Py_ssize_t j = 0; j < (names ? PyTuple_GET_SIZE(names) : 0); j++) {
        int hit = -1;
        for (int i = 0; i < kArgs && hit < 0; i++)
            if (PyUnicode_CompareWithASCIIString(PyTuple_GET_ITEM(names, j), arg_names[i]) == 0) hit = i;
        if (hit < 0 || a[hit]) {
            PyErr_Format(PyExc_TypeError, hit < 0 ? "read() got an unexpected keyword argument '%U'" : "read() got multiple values for argument '%U'",
                         PyTuple_GET_ITEM(names, j));
            return nullptr;
        }
        a[hit] = in[n + j];
    }
    if (!a[kLayer] || !a[kRows]) {
        PyErr_SetString(PyExc_TypeError, "read() needs layer and n_rows");
        return nullptr;
    }
    for (PyObject*& x : a)
        if (x == Py_None) x = nullptr;
    b200_kv_cache* kv = nullptr;
    if (!cache_of(in[0], &kv)) return nullptr;
    const long layer = a[kLayer] ? PyLong_AsLong(a[kLayer]) : -1, rows = a[kRows] ? PyLong_AsLong(a[kRows]) : -1, pos0 = a[kPos0] ? PyLong_AsLong(a[kPos0]) : 0;
    if (PyErr_Occurred()) return nullptr;
    if (pos0 != (int32_t)pos0 || layer != (int32_t)layer) {
        PyErr_SetString(PyExc_OverflowError, "layer and pos0 are 32-bit numbers");
        return nullptr;
    }
    at::ScalarType type = at::kHalf;
    if (a[kDtype]) {
        if (!THPDtype_Check(a[kDtype]) || ((type = ((THPDtype*)a[kDtype])->scalar_type) != at::kHalf && type != at::kFloat)) {
            PyErr_SetString(PyExc_ValueError, "dtype is torch.float16 or torch.float32");
            return nullptr;
        }
    }
    b200_tensor view[2], t[2];
    int rc = b200_kv_view(kv, (int)layer, rows, &view[0], &view[1]);
    if (rc) return raise_code(rc, "b200_kv_view");
    const c10::Device device(at::kCUDA, (c10::DeviceIndex)device_of_cache(view[0].data));
    const c10::cuda::CUDAGuard guard(device);
    const int64_t sizes[4] = {view[0].ne[3], view[0].ne[2], rows, view[0].ne[0]};
    void* st = nullptr;
    if (!a[kOn]) st = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    else if (!stream_of(a[kOn], &st)) return nullptr;
    at::Tensor out[2];
    if (!a[kOutPair]) {
        const PoolOf pool(st, device);
        for (at::Tensor& o : out) o = at::detail::empty_cuda(sizes, type, device, std::nullopt);
    } else {
        if (!PyTuple_Check(a[kOutPair]) || PyTuple_GET_SIZE(a[kOutPair]) != 2) {
            PyErr_SetString(PyExc_TypeError, "out is a pair of tensors");
            return nullptr;
        }
        for (int i = 0; i < 2; i++) {
            const at::Tensor* o = nullptr;
            if (!rows_of(PyTuple_GET_ITEM(a[kOutPair], i), "out", nullptr, &o)) return nullptr;
            if (o->device() != device || o->size(2) != rows) {
                PyErr_SetString(PyExc_ValueError, "out has n_rows rows and is on the cache's device");
                return nullptr;
            }
            out[i] = *o;
        }
    }
    if (!describe(out[0], -1, &t[0]) || !describe(out[1], -1, &t[1])) return nullptr;
    const int32_t* pos = nullptr;
    if (a[kPos] && !table_of(a[kPos], "pos", out[0], sizes[0], &pos)) return nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = b200_kv_read(kv, (int)layer, &t[0], &t[1], pos, (int32_t)pos0, st);
    Py_END_ALLOW_THREADS
    if (rc) return raise_code(rc, "b200_kv_read");
    PyObject* first = THPVariable_Wrap(out[0]);
    PyObject* second = THPVariable_Wrap(out[1]);
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

PyObject* as_method_py(PyObject*, PyObject* function) { return PyInstanceMethod_New(function); }

PyMethodDef kMethods[] = {
    {"flash_attn_ext", (PyCFunction)(void (*)(void))launch_py, METH_FASTCALL | METH_KEYWORDS, kLaunchDoc},
    {"flash_attn_ext_host", (PyCFunction)(void (*)(void))forward_host_py, METH_FASTCALL | METH_KEYWORDS, kHostDoc},
    {"kv_append", (PyCFunction)(void (*)(void))kv_append_py, METH_FASTCALL, "rows of a KV cache"},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope_py, METH_FASTCALL | METH_KEYWORDS, kQkRopeDoc},
    {"kv_append_rope", (PyCFunction)(void (*)(void))kv_append_rope_py, METH_FASTCALL | METH_KEYWORDS, kAppendRopeDoc},
    {"kv_tensors", (PyCFunction)(void (*)(void))kv_tensors_py, METH_FASTCALL, "views of a KV cache"},
    {"kv_read", (PyCFunction)(void (*)(void))kv_read_py, METH_FASTCALL | METH_KEYWORDS, kReadDoc},
    {"method", as_method_py, METH_O, "the function as one that binds to an object as a method (a built-in function does not)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_op", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_op(void) {
    for (int i = 0; i < kKeys; i++)
        if (!(g_keys[i] = PyUnicode_InternFromString(kKeyNames[i]))) return nullptr;
    if (!(g_handle = PyUnicode_InternFromString("_h")) || !(g_value = PyUnicode_InternFromString("value"))) return nullptr;
    for (int i = 0; i < rKeys; i++)
        if (!(g_rope_keys[i] = PyUnicode_InternFromString(kRopeNames[i]))) return nullptr;
    return PyModule_Create(&kModule);
}
