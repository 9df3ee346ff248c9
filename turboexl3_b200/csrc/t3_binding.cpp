// The Python face of the hot calls (module `_call`): linear, the routed chain and the plugin table's matmul on host arrays,
// argument checks, output and workspace allocation and the launch in one native call. Through ctypes a one-row linear spent
// 15 us on the host around a 7 us kernel (attribute reads, argument conversion, two Python-level allocations).
//
// Every function returns None when an argument is not what the engine takes: the Python side then names the refusal. A
// status of the C ABI other than T3_OK comes back as an int.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/t3.h"
#include "../../include/t3_table.h"

namespace {

PyObject *s_trellis, *s_suh, *s_svh, *s_gate, *s_up, *s_down, *s_codebook, *s_window_bits, *s_w, *s_scale;

// an attribute whose holder keeps it alive (instances of the package's dataclasses)
struct Attr {
    PyObject* p;
    Attr(PyObject* o, PyObject* name) : p(PyObject_GetAttr(o, name)) {}
    ~Attr() { Py_XDECREF(p); }
};

const at::Tensor* tensor(PyObject* o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.is_contiguous() ? &t : nullptr;
}

int act_dtype(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return T3_F32;
        case at::kHalf: return T3_F16;
        case at::kBFloat16: return T3_BF16;
        default: return -1;
    }
}
bool is_codes(const at::Tensor& t) { return t.scalar_type() == at::kUInt16 || t.scalar_type() == at::kShort; }
bool is_half(const at::Tensor& t) { return t.scalar_type() == at::kHalf; }
bool is_index(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32; }

bool decode_of(PyObject* o, t3_decode& dec) {
    Attr cb(o, s_codebook), wb(o, s_window_bits);
    if (!cb.p || !wb.p) return false;
    dec.codebook = (int)PyLong_AsLong(cb.p);
    dec.window_bits = (int)PyLong_AsLong(wb.p);
    return !PyErr_Occurred();
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

PyObject* finish(int status, at::Tensor& y) {
    if (status != T3_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(y));
}

// linear(x, trellis, suh, svh, dec)
PyObject* call_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 5) Py_RETURN_NONE;
    const at::Tensor *x = tensor(args[0]), *t = tensor(args[1]), *suh = tensor(args[2]), *svh = tensor(args[3]);
    if (!x || !t || !suh || !svh || x->dim() < 1 || t->dim() != 3) Py_RETURN_NONE;
    const int64_t in = t->size(0) * 16, out = t->size(1) * 16, n = t->size(2);
    const int dt = act_dtype(*x);
    if (x->size(-1) != in || suh->numel() != in || svh->numel() != out || dt < 0 || !is_codes(*t) || !is_half(*suh) || !is_half(*svh) ||
        in == 0 || in > INT32_MAX || out > INT32_MAX)
        Py_RETURN_NONE;
    const int64_t rows = x->numel() / in;
    t3_decode dec;
    if (rows < 1 || !decode_of(args[4], dec)) {
        if (PyErr_Occurred()) return nullptr;
        Py_RETURN_NONE;
    }
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = out;
    at::Tensor y = empty(shape, x->scalar_type(), *x), ws;
    const size_t bytes = t3_linear_workspace_bytes((size_t)rows, (int)in, (int)out, (int)n);
    if (bytes) ws = empty({(int64_t)bytes}, at::kByte, *x);
    void* stream = stream_of(*x);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = t3_linear(x->data_ptr(), dt, (size_t)rows, t->data_ptr(), suh->data_ptr(), svh->data_ptr(), (int)in, (int)out, (int)n, dec,
                       y.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(status, y);
    END_HANDLE_TH_ERRORS
}

// One projection of a bank: trellis [E, in / 16, out / 16, n], suh [E, in], svh [E, out]
bool proj_of(PyObject* bank, PyObject* name, t3_proj& p, int64_t (&dims)[4]) {
    Attr proj(bank, name);
    if (!proj.p) return false;
    Attr to(proj.p, s_trellis), so(proj.p, s_suh), vo(proj.p, s_svh);
    if (!to.p || !so.p || !vo.p) return false;
    const at::Tensor *t = tensor(to.p), *suh = tensor(so.p), *svh = tensor(vo.p);
    if (!t || !suh || !svh || t->dim() != 4 || suh->dim() != 2 || svh->dim() != 2 || !is_codes(*t) || !is_half(*suh) || !is_half(*svh))
        return false;
    for (int i = 0; i < 4; ++i) dims[i] = t->size(i);
    dims[1] *= 16, dims[2] *= 16;
    if (suh->size(0) != dims[0] || suh->size(1) != dims[1] || svh->size(0) != dims[0] || svh->size(1) != dims[2]) return false;
    p = {t->data_ptr(), suh->data_ptr(), svh->data_ptr()};
    return true;
}

// moe(x, bank, inds, scores, dec, limit, clamp_at, shared or None, event handle or 0)
PyObject* call_moe(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 9) Py_RETURN_NONE;
    const at::Tensor *x = tensor(args[0]), *inds = tensor(args[2]), *scores = tensor(args[3]);
    if (!x || !inds || !scores || x->dim() != 3 || inds->dim() != 3 || x->size(0) != inds->size(0) || x->size(1) != inds->size(1) ||
        !inds->sizes().equals(scores->sizes()))
        Py_RETURN_NONE;
    const int64_t topk = inds->size(2), hidden = x->size(2), rows = x->size(0) * x->size(1);
    const int dt = act_dtype(*x), sdt = act_dtype(*scores);
    if (topk <= 0 || topk > T3_REDUCE_MAX_TOPK || hidden % 128 || dt < 0 || sdt < 0 || !is_index(*inds)) Py_RETURN_NONE;
    t3_bank bank = {};
    int64_t g[4], u[4], d[4];
    if (!proj_of(args[1], s_gate, bank.gate, g) || !proj_of(args[1], s_up, bank.up, u) || !proj_of(args[1], s_down, bank.down, d)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const int64_t inter = g[2];
    if (g[1] != hidden || u[1] != hidden || u[2] != inter || d[1] != inter || d[2] != hidden || u[0] != g[0] || d[0] != g[0] || inter % 128)
        Py_RETURN_NONE;
    bank.experts = (int)g[0], bank.hidden = (int)hidden, bank.inter = (int)inter;
    bank.n_gate = (int)g[3], bank.n_up = (int)u[3], bank.n_down = (int)d[3];
    t3_decode dec;
    if (!decode_of(args[4], dec)) return nullptr;
    const long limit = PyLong_AsLong(args[5]), clamp_at = PyLong_AsLong(args[6]);
    const at::Tensor* shared = nullptr;
    if (args[7] != Py_None) {
        shared = tensor(args[7]);
        if (!shared || shared->scalar_type() != x->scalar_type() || shared->numel() != x->numel()) Py_RETURN_NONE;
    }
    void* event = PyLong_AsVoidPtr(args[8]);
    if (PyErr_Occurred()) return nullptr;
    const size_t bytes = t3_moe_workspace_bytes((size_t)rows, (int)topk, &bank);
    at::Tensor ws = empty({(int64_t)(bytes ? bytes : 1)}, at::kByte, *x), y = empty(x->sizes(), x->scalar_type(), *x);
    void* stream = stream_of(*x);
    int status;
    Py_BEGIN_ALLOW_THREADS
    if (shared && event)
        status = t3_moe_with_shared_after(x->data_ptr(), dt, (size_t)rows, &bank, inds->data_ptr(), scores->data_ptr(), sdt, (int)topk, dec,
                                          shared->data_ptr(), event, y.data_ptr(), ws.data_ptr(), bytes, stream);
    else if (shared)
        status = t3_moe_with_shared(x->data_ptr(), dt, (size_t)rows, &bank, inds->data_ptr(), scores->data_ptr(), sdt, (int)topk, dec,
                                    shared->data_ptr(), y.data_ptr(), ws.data_ptr(), bytes, stream);
    else
        status = t3_moe_swiglu(x->data_ptr(), dt, (size_t)rows, &bank, inds->data_ptr(), scores->data_ptr(), sdt, (int)topk, dec,
                               (uint32_t)limit, (int)clamp_at, y.data_ptr(), ws.data_ptr(), bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(status, y);
    END_HANDLE_TH_ERRORS
}

// ---- 8-bit layers and routing: every tensor on x's device, which need not be the current one ----

bool is_e4m3(const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn; }
bool is_f32(const at::Tensor& t) { return t.scalar_type() == at::kFloat; }

// route(logits, topk, scoring, bias or None, groups, group_topk, renormalise, scale)
PyObject* call_route(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 8) Py_RETURN_NONE;
    const at::Tensor *x = tensor(args[0]), *bias = nullptr;
    if (!x || x->dim() < 1 || act_dtype(*x) < 0) Py_RETURN_NONE;
    const int64_t experts = x->size(-1);
    if (args[3] != Py_None) {
        bias = tensor(args[3]);
        if (!bias || !is_f32(*bias) || bias->numel() != experts || bias->device() != x->device()) Py_RETURN_NONE;
    }
    const long topk = PyLong_AsLong(args[1]), scoring = PyLong_AsLong(args[2]), groups = PyLong_AsLong(args[4]),
               group_topk = PyLong_AsLong(args[5]), renormalise = PyObject_IsTrue(args[6]);
    const double scale = PyFloat_AsDouble(args[7]);
    if (PyErr_Occurred()) return nullptr;
    if (experts < 1 || experts > T3_ROUTE_EXPERTS_MAX || x->numel() < 1 || topk < 1 || topk > T3_REDUCE_MAX_TOPK || groups < 1 || groups > 32 ||
        group_topk < 1 || group_topk > 32)
        Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(x->device());
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = topk;
    at::Tensor inds = empty(shape, at::kInt, *x), scores = empty(shape, at::kFloat, *x);
    void* stream = stream_of(*x);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = t3_route(x->data_ptr(), act_dtype(*x), (size_t)(x->numel() / experts), (int)experts, (int)topk, (int)scoring,
                      bias ? bias->data_ptr() : nullptr, (int)groups, (int)group_topk, (int)renormalise, (float)scale, inds.data_ptr(),
                      scores.data_ptr(), stream);
    Py_END_ALLOW_THREADS
    if (status != T3_OK) return PyLong_FromLong(status);
    PyObject* i = THPVariable_Wrap(std::move(inds));
    PyObject* s = THPVariable_Wrap(std::move(scores));
    return Py_BuildValue("(NN)", i, s);
    END_HANDLE_TH_ERRORS
}

// quantize_fp8(x)
PyObject* call_quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 1) Py_RETURN_NONE;
    const at::Tensor* x = tensor(args[0]);
    if (!x || x->dim() < 1 || act_dtype(*x) < 0 || x->numel() < 1 || x->size(-1) % 128 != 0 || x->size(-1) > INT32_MAX) Py_RETURN_NONE;
    const int64_t in = x->size(-1);
    const c10::cuda::CUDAGuard guard(x->device());
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    at::Tensor q = empty(shape, at::kFloat8_e4m3fn, *x);
    shape.back() = in / 128;
    at::Tensor scale = empty(shape, at::kFloat, *x);
    void* stream = stream_of(*x);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = t3_quantize_fp8(x->data_ptr(), act_dtype(*x), (size_t)(x->numel() / in), (int)in, q.data_ptr(), scale.data_ptr(), stream);
    Py_END_ALLOW_THREADS
    if (status != T3_OK) return PyLong_FromLong(status);
    PyObject* a = THPVariable_Wrap(std::move(q));
    PyObject* b = THPVariable_Wrap(std::move(scale));
    return Py_BuildValue("(NN)", a, b);
    END_HANDLE_TH_ERRORS
}

// linear_fp8(x, w, w_scale, x_scale or None, out_dtype: a t3_dtype, or -1 for x's)
PyObject* call_linear_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 5) Py_RETURN_NONE;
    const at::Tensor *x = tensor(args[0]), *w = tensor(args[1]), *ws = tensor(args[2]), *xs = nullptr;
    if (!x || !w || !ws || x->dim() < 1 || w->dim() != 2 || ws->dim() != 2 || !is_e4m3(*w) || !is_f32(*ws)) Py_RETURN_NONE;
    const int64_t in = w->size(1), out = w->size(0);
    const bool given = is_e4m3(*x);
    int dt = given ? T3_E4M3 : act_dtype(*x), ydt = (int)PyLong_AsLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    if (ydt < 0) ydt = given ? T3_BF16 : dt;
    if (dt < 0 || ydt > T3_BF16 || in < 1 || in > INT32_MAX || out < 1 || out > INT32_MAX || in % 128 != 0 || x->size(-1) != in || x->numel() < 1 ||
        ws->size(0) != (out + 127) / 128 || ws->size(1) != in / 128 || w->device() != x->device() || ws->device() != x->device())
        Py_RETURN_NONE;
    if ((args[3] != Py_None) != given) Py_RETURN_NONE;
    if (given) {
        xs = tensor(args[3]);
        if (!xs || !is_f32(*xs) || xs->numel() != x->numel() / 128 || xs->dim() != x->dim() || xs->size(-1) != in / 128 ||
            xs->device() != x->device())
            Py_RETURN_NONE;
    }
    const int64_t rows = x->numel() / in;
    const c10::cuda::CUDAGuard guard(x->device());
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = out;
    at::Tensor y = empty(shape, ydt == T3_F32 ? at::kFloat : ydt == T3_F16 ? at::kHalf : at::kBFloat16, *x), scratch;
    const size_t bytes = given ? 0 : t3_linear_fp8_workspace_bytes((size_t)rows, (int)in, (int)out, dt);
    if (bytes) scratch = empty({(int64_t)bytes}, at::kByte, *x);
    void* stream = stream_of(*x);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = t3_linear_fp8(x->data_ptr(), dt, xs ? xs->data_ptr() : nullptr, (size_t)rows, w->data_ptr(), ws->data_ptr(), (int)in, (int)out,
                           y.data_ptr(), ydt, bytes ? scratch.data_ptr() : nullptr, bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(status, y);
    END_HANDLE_TH_ERRORS
}

// One projection of an 8-bit bank: w e4m3 [E, out, in], scale f32 [E, out / 128, in / 128]
bool fp8_proj_of(PyObject* bank, PyObject* name, const at::Device& device, t3_fp8_proj& p, int64_t (&dims)[3]) {
    Attr proj(bank, name);
    if (!proj.p) return false;
    Attr wo(proj.p, s_w), so(proj.p, s_scale);
    if (!wo.p || !so.p) return false;
    const at::Tensor *w = tensor(wo.p), *s = tensor(so.p);
    if (!w || !s || w->dim() != 3 || s->dim() != 3 || !is_e4m3(*w) || !is_f32(*s) || w->device() != device || s->device() != device) return false;
    for (int i = 0; i < 3; ++i) dims[i] = w->size(i);
    if (dims[1] % 128 != 0 || dims[2] % 128 != 0 || s->size(0) != dims[0] || s->size(1) != dims[1] / 128 || s->size(2) != dims[2] / 128) return false;
    p = {w->data_ptr(), s->data_ptr()};
    return true;
}

// moe_fp8(x, bank, inds, scores, shared or None)
PyObject* call_moe_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 5) Py_RETURN_NONE;
    const at::Tensor *x = tensor(args[0]), *inds = tensor(args[2]), *scores = tensor(args[3]), *shared = nullptr;
    if (!x || !inds || !scores || x->dim() != 3 || inds->dim() != 3 || x->size(0) != inds->size(0) || x->size(1) != inds->size(1) ||
        !inds->sizes().equals(scores->sizes()) || inds->device() != x->device() || scores->device() != x->device())
        Py_RETURN_NONE;
    const int64_t topk = inds->size(2), hidden = x->size(2), rows = x->size(0) * x->size(1);
    const int dt = act_dtype(*x), sdt = act_dtype(*scores);
    if (topk <= 0 || topk > T3_REDUCE_MAX_TOPK || rows < 1 || dt < 0 || sdt < 0 || !is_index(*inds)) Py_RETURN_NONE;
    t3_fp8_bank bank = {};
    int64_t g[3], u[3], d[3];
    if (!fp8_proj_of(args[1], s_gate, x->device(), bank.gate, g) || !fp8_proj_of(args[1], s_up, x->device(), bank.up, u) ||
        !fp8_proj_of(args[1], s_down, x->device(), bank.down, d)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (g[0] < 1 || g[0] > T3_FP8_EXPERTS_MAX || g[2] != hidden || u[0] != g[0] || u[1] != g[1] || u[2] != hidden || d[0] != g[0] ||
        d[1] != hidden || d[2] != g[1] || hidden > INT32_MAX || g[1] > INT32_MAX)
        Py_RETURN_NONE;
    bank.experts = (int)g[0], bank.hidden = (int)hidden, bank.inter = (int)g[1];
    if (args[4] != Py_None) {
        shared = tensor(args[4]);
        if (!shared || shared->scalar_type() != x->scalar_type() || shared->numel() != x->numel() || shared->device() != x->device()) Py_RETURN_NONE;
    }
    const c10::cuda::CUDAGuard guard(x->device());
    const size_t bytes = t3_moe_fp8_workspace_bytes((size_t)rows, (int)topk, &bank);
    at::Tensor ws = empty({(int64_t)(bytes ? bytes : 1)}, at::kByte, *x), y = empty(x->sizes(), x->scalar_type(), *x);
    void* stream = stream_of(*x);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = t3_moe_fp8(x->data_ptr(), dt, (size_t)rows, &bank, inds->data_ptr(), scores->data_ptr(), sdt, (int)topk,
                        shared ? shared->data_ptr() : nullptr, y.data_ptr(), ws.data_ptr(), bytes, stream);
    Py_END_ALLOW_THREADS
    return finish(status, y);
    END_HANDLE_TH_ERRORS
}

struct Buffer {
    Py_buffer view = {};
    bool held = false;
    bool get(PyObject* o, int flags) { return held = PyObject_GetBuffer(o, &view, flags) == 0; }
    ~Buffer() {
        if (held) PyBuffer_Release(&view);
    }
};

// table_matmul(weight, x, y, stream, dtype): the plugin table's matmul on two host buffers. True, or None where the caller has
// to take the general path (other dtypes, a refusal to be named).
PyObject* call_table_matmul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 5) Py_RETURN_NONE;
    Buffer w, x, y;
    if (!w.get(args[0], PyBUF_SIMPLE) || w.view.len != (Py_ssize_t)sizeof(t3_weight) || !x.get(args[1], PyBUF_ND) ||
        !y.get(args[2], PyBUF_ND | PyBUF_WRITABLE) || x.view.ndim < 1 || x.view.ndim > 8 || y.view.ndim != x.view.ndim) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    void* stream = PyLong_AsVoidPtr(args[3]);
    const int dtype = (int)PyLong_AsLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    t3_array xa = {}, ya = {};
    for (int k = 0; k < 2; ++k) {
        t3_array& a = k ? ya : xa;
        const Py_buffer& v = k ? y.view : x.view;
        a.data = v.buf;
        a.dtype = dtype;
        a.ndim = v.ndim;
        for (int i = 0; i < v.ndim; ++i) a.shape[i] = v.shape[i];
    }
    static const auto matmul = t3_table()->matmul;
    t3_verdict verdict;
    Py_BEGIN_ALLOW_THREADS
    verdict = matmul(static_cast<const t3_weight*>(w.view.buf), &xa, stream, &ya);
    Py_END_ALLOW_THREADS
    if (verdict.kind != T3_VERDICT_OK) Py_RETURN_NONE;
    Py_RETURN_TRUE;
}

PyMethodDef methods[] = {
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_linear)), METH_FASTCALL, nullptr},
    {"moe", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_moe)), METH_FASTCALL, nullptr},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_route)), METH_FASTCALL, nullptr},
    {"quantize_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_quantize_fp8)), METH_FASTCALL, nullptr},
    {"linear_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_linear_fp8)), METH_FASTCALL, nullptr},
    {"moe_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_moe_fp8)), METH_FASTCALL, nullptr},
    {"table_matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_table_matmul)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call(void) {
    s_trellis = PyUnicode_InternFromString("trellis"), s_suh = PyUnicode_InternFromString("suh"), s_svh = PyUnicode_InternFromString("svh");
    s_gate = PyUnicode_InternFromString("gate"), s_up = PyUnicode_InternFromString("up"), s_down = PyUnicode_InternFromString("down");
    s_codebook = PyUnicode_InternFromString("codebook"), s_window_bits = PyUnicode_InternFromString("window_bits");
    s_w = PyUnicode_InternFromString("w"), s_scale = PyUnicode_InternFromString("scale");
    return PyModule_Create(&module);
}
