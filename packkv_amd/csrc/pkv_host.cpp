// The host side of the calls that a decode loop repeats, in native code: the checks, the argument block and the result
// tensors of ops.attn_decode, AttnPlan's step, ops.window_append, ops.dense_view, the four matrix-vector ops, and ops.norm_rotary,
// window_append_rotary, attn_chunk, sample, add_rms_norm, fp8_quantize, fp8_linear and fp8_gated.
//
// A decode step is two such calls around 12 us of GPU time, and in Python their checks and ctypes' conversions take 6 to
// 12 us each besides the launch.  Every function here serves the usual call and gives up on any other before it has done
// anything (it returns None): ops.py then goes on with the general code, which copies what has to be copied and
// words what has to be refused.  So nothing is refused here, and what is served meets every condition the general code checks.
// Host time in us a call, general code -> here: attn_decode 15.5 -> 7.8 (two launches in it), window_append 7.3 -> 3.2 (one), the
// cache's attend 8.8 -> 4.3, fused_kq with its wait 16.2 -> 11.5.  Whole passes of one tree without and with this file: a request of 509
// tokens and 24 steps in two layers 1562 -> 1089, a prompt of 3001 tokens and six steps that return the dense tensors 294 -> 192, the four
// matrix-vector ops over 65536 tokens 101 -> 86.  Without it, or with one that was built for another torch, the general code serves.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/packkv.h"

namespace {

struct Library {                   // libpackkv_hip.so, as _lib.py has loaded it
    decltype(&pkv_attn_decode) attn_decode = nullptr;
    decltype(&pkv_window_append) window_append = nullptr;
    decltype(&pkv_dense_view) dense_view = nullptr;
    decltype(&pkv_kq_mat_vec_mul) kq = nullptr;
    decltype(&pkv_wv_mat_vec_mul) wv = nullptr;
    decltype(&pkv_fused_kq) fused_kq = nullptr;
    decltype(&pkv_fused_wv) fused_wv = nullptr;
    decltype(&pkv_norm_rotary) norm_rotary = nullptr;
    decltype(&pkv_attn_chunk_workspace) chunk_workspace = nullptr;
    decltype(&pkv_attn_chunk) attn_chunk = nullptr;
    decltype(&pkv_sample_workspace) sample_workspace = nullptr;
    decltype(&pkv_sample) sample = nullptr;
    decltype(&pkv_add_rms_norm) add_rms_norm = nullptr;
    decltype(&pkv_fp8_quantize) fp8_quantize = nullptr;
    decltype(&pkv_fp8_product) fp8_product = nullptr;
} lib;

// A plain torch.Tensor (a subclass, or a mode that wants to see the calls, gets the general code).
const at::Tensor *tensor(PyObject *o) { return o && THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }
bool modes() { return at::impl::torch_function_mode_enabled(); }

// The tensor's memory is addressable and lies on device `dev`.
bool there(const at::Tensor &t, int dev) { return t.is_cuda() && t.get_device() == dev && t.has_storage() && t.layout() == at::kStrided; }
bool dense(const at::Tensor &t, int dev) { return there(t, dev) && t.is_contiguous(); }
bool half(const at::Tensor &t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
int code(const at::Tensor &t) { return t.scalar_type() == at::kHalf ? PKV_F16 : PKV_BF16; }
template <typename T> T *at_ptr(const at::Tensor &t) { return reinterpret_cast<T *>(t.data_ptr()); }

// The current device where `t` lies on it, else -1, which is no tensor's.  (HIP is not asked about a tensor on the host: there may
// be no GPU, and the general code has the words for that.)
int here(const at::Tensor *t) {
    if (!t || !t->is_cuda()) return -1;
    const int dev = c10::hip::current_device();
    return t->get_device() == dev ? dev : -1;
}
pkv_stream_t stream(int dev) { return (pkv_stream_t)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

// An int argument (a plain Python int within 32 bits).
bool integer(PyObject *o, int *out) {
    if (!o || !PyLong_CheckExact(o)) return false;
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(o, &over);
    if (over || v < INT_MIN || v > INT_MAX) return false;
    *out = (int)v;
    return true;
}

// The library may wait or allocate: other threads go on meanwhile.  `f` calls it and nothing else: no address is taken in there (a lazily
// cloned tensor gets its memory then, and may throw), no Python object touched.
template <typename F> int call(F &&f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

// K's and V's side of a compressed cache, dicts as ops.attn_decode takes them, into `a`.  `batch` 0: from the parameters.
struct Cache {
    int tokens = 0, heads = 0, batch = 0;
    const at::Tensor *like = nullptr;
};
bool cache_args(PyObject *k, PyObject *v, int dev, int batch, pkv_attn_args &a, Cache &c) {
    if (!PyDict_CheckExact(k) || !PyDict_CheckExact(v)) return false;
    const at::Tensor *t[2][4];
    static PyObject *const names[4] = {PyUnicode_InternFromString("stream"), PyUnicode_InternFromString("info"), PyUnicode_InternFromString("scale"),
                                       PyUnicode_InternFromString("zero")};
    static PyObject *const s_bits = PyUnicode_InternFromString("bits"), *const s_tokens = PyUnicode_InternFromString("tokens"),
                    *const s_heads = PyUnicode_InternFromString("heads");
    int bits[2], tokens[2];
    for (int i = 0; i < 2; i++) {
        PyObject *d = i ? v : k;
        for (int f = 0; f < 4; f++) {
            t[i][f] = tensor(PyDict_GetItem(d, names[f]));
            if (!t[i][f] || !dense(*t[i][f], dev)) return false;
        }
        if (t[i][2]->dim() != 2 || t[i][3]->dim() != 2 || t[i][3]->sizes() != t[i][2]->sizes()) return false;
        if (t[i][0]->scalar_type() != at::kByte || t[i][1]->scalar_type() != at::kUInt32) return false;
        if (!integer(PyDict_GetItem(d, s_bits), &bits[i])) return false;
        PyObject *n = PyDict_GetItem(d, s_tokens);
        if (!n) tokens[i] = (int)t[i][2]->size(1);
        else if (!integer(n, &tokens[i])) return false;
    }
    const at::Tensor &scale = *t[0][2];
    if (t[1][2]->sizes() != scale.sizes() || tokens[0] != tokens[1] || tokens[0] < 128 || tokens[0] > scale.size(1) || scale.size(1) > INT_MAX) return false;
    if (scale.size(0) < 1 || (batch && scale.size(0) != batch)) return false;
    c.batch = batch ? batch : (int)scale.size(0);
    c.tokens = tokens[0];
    const int64_t rows = tokens[0] / 64, k_blocks = t[0][1]->numel() / 2, v_blocks = t[1][1]->numel() / 2;
    PyObject *h = PyDict_GetItem(k, s_heads);
    if (!h) c.heads = (int)(k_blocks / rows / c.batch);
    else if (!integer(h, &c.heads)) return false;
    const int64_t blocks = rows * c.batch * c.heads;      // (V: half as many rows of twice the blocks)
    if (c.heads < 1 || k_blocks < blocks || v_blocks < blocks) return false;
    for (int i = 0; i < 2; i++)
        for (int f = 2; f < 4; f++)
            if (t[i][f]->scalar_type() != scale.scalar_type()) return false;
    c.like = &scale;
    a.k_stream = at_ptr<uint8_t>(*t[0][0]); a.k_info = at_ptr<uint32_t>(*t[0][1]); a.k_scale = at_ptr<void>(*t[0][2]); a.k_zero = at_ptr<void>(*t[0][3]);
    a.v_stream = at_ptr<uint8_t>(*t[1][0]); a.v_info = at_ptr<uint32_t>(*t[1][1]); a.v_scale = at_ptr<void>(*t[1][2]); a.v_zero = at_ptr<void>(*t[1][3]);
    a.k_bytes = (uint64_t)t[0][0]->numel();
    a.v_bytes = (uint64_t)t[1][0]->numel();
    a.k_bits = bits[0]; a.v_bits = bits[1];
    a.par_stride = (int)scale.size(1);
    return true;
}

// The 16-bit windows [batch, heads, cap, 128] and the rows in use (None: all).
bool window_args(const at::Tensor *k, const at::Tensor *v, PyObject *rows, int dev, const Cache &c, at::ScalarType type, pkv_attn_args &a) {
    if (!k || !v || !dense(*k, dev) || !dense(*v, dev) || k->dim() != 4 || v->sizes() != k->sizes() || k->scalar_type() != type || v->scalar_type() != type) return false;
    if (k->size(0) != c.batch || k->size(1) != c.heads || k->size(3) != 128 || k->size(2) > INT_MAX) return false;
    a.T_w = (int)k->size(2);
    if (rows != Py_None && !integer(rows, &a.T_w)) return false;
    if (a.T_w < 1 || a.T_w > k->size(2)) return false;
    a.win_stride = (int)k->size(2);
    a.k_win = at_ptr<void>(*k);
    a.v_win = at_ptr<void>(*v);
    return true;
}

PyObject *status(int rc) { return PyLong_FromLong(rc); }

// attn_decode(q, k, v, k_win, v_win, sm_scale, win_len) -> the result, a status that is not zero, or None
PyObject *attn_decode(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *q = n == 7 && !modes() ? tensor(o[0]) : nullptr;
    const int dev = here(q);
    if (dev < 0 || !dense(*q, dev) || !half(*q) || q->dim() != 3 || q->size(2) != 128) Py_RETURN_NONE;
    pkv_attn_args a{};
    Cache c;
    c.batch = (int)q->size(0);
    if (q->size(0) < 1 || q->size(0) > INT_MAX || q->size(1) > INT_MAX) Py_RETURN_NONE;
    if (o[1] != Py_None) {
        if (!cache_args(o[1], o[2], dev, c.batch, a, c) || c.like->scalar_type() != q->scalar_type()) Py_RETURN_NONE;
        if ((reinterpret_cast<uintptr_t>(a.k_stream) | reinterpret_cast<uintptr_t>(a.v_stream)) % 16) Py_RETURN_NONE;
    } else if (o[2] != Py_None) {
        Py_RETURN_NONE;
    }
    if (o[3] != Py_None) {
        const at::Tensor *kw = tensor(o[3]);
        if (o[1] == Py_None && kw && kw->dim() == 4) c.heads = (int)kw->size(1);
        if (!window_args(kw, tensor(o[4]), o[6], dev, c, q->scalar_type(), a)) Py_RETURN_NONE;
    } else if (o[1] == Py_None || o[4] != Py_None) {
        Py_RETURN_NONE;
    }
    a.sm_scale = 0.08838834764831845f;                     // 128 ** -0.5
    if (o[5] != Py_None) {
        if (!PyFloat_CheckExact(o[5])) Py_RETURN_NONE;
        a.sm_scale = (float)PyFloat_AS_DOUBLE(o[5]);
    }
    at::Tensor out = at::empty(q->sizes(), q->options());
    a.q = at_ptr<void>(*q);
    a.out = at_ptr<void>(out);
    a.B = c.batch; a.Hq = (int)q->size(1); a.Hkv = c.heads; a.T_c = c.tokens;
    a.dtype = code(*q);
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.attn_decode(&a, nullptr, s); });
    return rc ? status(rc) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// plan_step(address of the plan's arguments, its device, window rows, q) -> the result in q's shape, a status that is not zero, or
// None.  q [B, Hq, 128] or [B, Hq, 1, 128] like the plan's.
PyObject *plan_step(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *q = n == 4 && !modes() ? tensor(o[3]) : nullptr;
    int plan_dev = -1, rows = 0;
    const int dev = here(q);
    if (dev < 0 || !PyLong_CheckExact(o[0]) || !integer(o[1], &plan_dev) || !integer(o[2], &rows) || plan_dev != dev || !dense(*q, dev)) Py_RETURN_NONE;
    // (a copy: the plan's own q, out and rows stay what its owner has set, and keeps alive)
    pkv_attn_args a = *(const pkv_attn_args *)PyLong_AsVoidPtr(o[0]);
    const int64_t d = q->dim();
    if ((d != 3 && (d != 4 || q->size(2) != 1)) || q->size(0) != a.B || q->size(1) != a.Hq || q->size(d - 1) != 128 ||
        !half(*q) || code(*q) != a.dtype || a.flags || rows < 1 || rows > a.win_stride) Py_RETURN_NONE;
    at::Tensor out = at::empty(q->sizes(), q->options());
    a.q = at_ptr<void>(*q);
    a.out = at_ptr<void>(out);
    a.T_w = rows;
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.attn_decode(&a, nullptr, s); });
    return rc ? status(rc) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// window_append(k_new, v_new, cos, sin, k_win, v_win, win_pos) -> status or None
PyObject *window_append(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || modes()) Py_RETURN_NONE;
    const at::Tensor *k = tensor(o[0]), *v = tensor(o[1]), *kw = tensor(o[4]), *vw = tensor(o[5]);
    const int dev = here(k);
    int pos = 0;
    if (dev < 0 || !v || !kw || !vw || !there(*k, dev) || !there(*v, dev) || !dense(*kw, dev) || !dense(*vw, dev) || !integer(o[6], &pos)) Py_RETURN_NONE;
    const auto type = k->scalar_type();
    if (k->dim() != 4 || k->size(3) != 128 || v->sizes() != k->sizes() || !half(*k) || v->scalar_type() != type || k->strides() != v->strides() ||
        k->stride(3) != 1 || kw->dim() != 4 || vw->sizes() != kw->sizes() || kw->size(0) != k->size(0) || kw->size(1) != k->size(1) ||
        kw->size(3) != 128 || kw->scalar_type() != type || vw->scalar_type() != type) Py_RETURN_NONE;
    const int64_t B = k->size(0), H = k->size(1), rows = k->size(2), cap = kw->size(2);
    if (B > INT_MAX || H > INT_MAX || rows > INT_MAX || cap > INT_MAX) Py_RETURN_NONE;
    const void *cos_p = nullptr, *sin_p = nullptr;
    int64_t rot = 0;
    if (o[2] != Py_None) {
        const at::Tensor *cos = tensor(o[2]), *sin = tensor(o[3]);
        const int64_t shape[3] = {B, rows, 128};
        if (!cos || !sin || !there(*cos, dev) || !there(*sin, dev) || cos->sizes() != at::IntArrayRef(shape, 3) || sin->sizes() != cos->sizes() ||
            cos->scalar_type() != type || sin->scalar_type() != type || cos->strides() != sin->strides() || cos->stride(2) != 1 ||
            (rows > 1 && cos->stride(1) != 128)) Py_RETURN_NONE;
        cos_p = at_ptr<void>(*cos);
        sin_p = at_ptr<void>(*sin);
        rot = B > 1 ? cos->stride(0) : 0;
    }
    const void *const k_p = at_ptr<void>(*k), *const v_p = at_ptr<void>(*v);
    void *const kw_p = at_ptr<void>(*kw), *const vw_p = at_ptr<void>(*vw);
    const int64_t sb = k->stride(0), sh = k->stride(1), st = k->stride(2);
    const int dtype = code(*k);
    const pkv_stream_t s = stream(dev);
    return status(call([&] { return lib.window_append(k_p, v_p, cos_p, sin_p, dtype, (int)B, (int)H, (int)rows, sb, sh, st, rot, kw_p, vw_p, pos, (int)cap, s); }));
    END_HANDLE_TH_ERRORS
}

// dense_view(k, v, k_win, v_win, win_len) -> (K, V), a status that is not zero, or None
PyObject *dense_view(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || modes() || !PyDict_CheckExact(o[0])) Py_RETURN_NONE;
    const int dev = here(tensor(PyDict_GetItemString(o[0], "scale")));
    pkv_attn_args a{};
    Cache c;
    if (dev < 0 || !cache_args(o[0], o[1], dev, 0, a, c) || !half(*c.like)) Py_RETURN_NONE;
    if (o[2] != Py_None && !window_args(tensor(o[2]), tensor(o[3]), o[4], dev, c, c.like->scalar_type(), a)) Py_RETURN_NONE;
    a.B = c.batch; a.Hkv = c.heads; a.T_c = c.tokens;
    a.dtype = code(*c.like);
    at::Tensor k = at::empty({c.batch, c.heads, (int64_t)c.tokens + a.T_w, 128}, c.like->options()), v = at::empty_like(k);
    void *const k_p = at_ptr<void>(k), *const v_p = at_ptr<void>(v);
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.dense_view(&a, k_p, v_p, s); });
    if (rc) return status(rc);
    PyObject *both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(k)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(v)));
    return both;
    END_HANDLE_TH_ERRORS
}

// A timed op: milliseconds, a status that is not zero, or None.
template <typename F> PyObject *timed(F &&f) {
    float ms = 0.f;
    const int rc = call([&] { return f(&ms); });
    return rc ? status(rc) : PyFloat_FromDouble((double)ms);
}

// mat_vec(is_k, stream, info, x, out, ctx_len, hidden_dim, ctx_blk, hid_blk, bits, interleaved)
PyObject *mat_vec(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11 || modes()) Py_RETURN_NONE;
    const bool is_k = o[0] == Py_True;
    const at::Tensor *stm = tensor(o[1]), *info = tensor(o[2]), *x = tensor(o[3]), *out = tensor(o[4]);
    const int dev = here(x);
    int i[5];
    for (int j = 0; j < 5; j++)
        if (!integer(o[5 + j], &i[j])) Py_RETURN_NONE;
    if (dev < 0 || !stm || !info || !out || !there(*stm, dev) || !there(*info, dev) || !there(*x, dev) || !there(*out, dev) || !half(*x) ||
        (!is_k && out->scalar_type() != at::kFloat) || (o[10] != Py_True && o[10] != Py_False)) Py_RETURN_NONE;
    const uint64_t bytes = (uint64_t)stm->numel() * (uint64_t)stm->element_size();
    const uint8_t *const stm_p = at_ptr<uint8_t>(*stm);
    const uint32_t *const info_p = at_ptr<uint32_t>(*info);
    const void *const x_p = at_ptr<void>(*x);
    void *const out_p = at_ptr<void>(*out);
    const int dtype = code(*x), interleaved = o[10] == Py_True;
    const pkv_stream_t s = stream(dev);
    if (is_k) return timed([&](float *ms) { return lib.kq(stm_p, bytes, info_p, x_p, out_p, i[0], i[1], i[2], i[3], i[4], dtype, interleaved, ms, s); });
    return timed([&](float *ms) { return lib.wv(stm_p, bytes, info_p, x_p, (float *)out_p, i[0], i[1], i[2], i[3], i[4], dtype, ms, s); });
    END_HANDLE_TH_ERRORS
}

// fused(is_k, out, x, zero, scale, t): ops.fused_kq(out, x = q, zero, scale, t) or ops.fused_wv(out, x = w, zero, scale, t = term1)
PyObject *fused(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || modes()) Py_RETURN_NONE;
    const bool is_k = o[0] == Py_True;
    const at::Tensor *out = tensor(o[1]), *x = tensor(o[2]), *zero = tensor(o[3]), *scale = tensor(o[4]), *t = tensor(o[5]);
    const int dev = here(x);
    if (dev < 0 || !out || !zero || !scale || !t || !dense(*out, dev) || !dense(*x, dev) || !dense(*zero, dev) || !dense(*scale, dev) || !dense(*t, dev) ||
        !half(*x)) Py_RETURN_NONE;
    if (out->dim() != 2 || x->dim() != 2 || t->dim() != 2 || zero->dim() != 1 || scale->dim() != 1) Py_RETURN_NONE;
    const int64_t M = x->size(0), K = x->size(1), T = t->size(1), columns = is_k ? T : K;
    if (t->size(0) != M || zero->size(0) != columns || scale->size(0) != columns || out->size(0) != M || out->size(1) != T ||
        (!is_k && t->scalar_type() != x->scalar_type()) || M > INT_MAX || K > INT_MAX || T > INT_MAX) Py_RETURN_NONE;
    void *const out_p = at_ptr<void>(*out);
    const void *const x_p = at_ptr<void>(*x), *const zero_p = at_ptr<void>(*zero), *const scale_p = at_ptr<void>(*scale), *const t_p = at_ptr<void>(*t);
    const int dtype = code(*x);
    const pkv_stream_t s = stream(dev);
    return timed([&](float *ms) { return (is_k ? lib.fused_kq : lib.fused_wv)(out_p, x_p, zero_p, scale_p, t_p, (int)M, (int)K, (int)T, dtype, ms, s); });
    END_HANDLE_TH_ERRORS
}

// Element strides of batch, head and token of x [B, H, n, 128]; dimensions of one element have none.
void row_strides(const at::Tensor &x, int64_t out[3]) {
    for (int i = 0; i < 3; i++) out[i] = x.size(i) > 1 ? x.stride(i) : 0;
}
bool whole_rows(const at::Tensor &x, int dev) { return there(x, dev) && x.dim() == 4 && x.size(3) == 128 && x.stride(3) == 1; }
bool real(PyObject *o, float *out) {
    if (!o || !PyFloat_CheckExact(o)) return false;
    *out = (float)PyFloat_AS_DOUBLE(o);
    return true;
}
// The position axis of each frequency (ops._frequency_axes) from sections, a tuple or None.
bool frequency_axes(PyObject *sections, PyObject *interleaved, pkv_rotary_args &a) {
    a.n_axes = 1;
    if (sections == Py_None) return true;                  // (all zeroes)
    if (!PyTuple_CheckExact(sections) || (interleaved != Py_True && interleaved != Py_False)) return false;
    const int A = (int)PyTuple_GET_SIZE(sections);
    int width[4], sum = 0;
    if (A < 1 || A > 4) return false;
    for (int i = 0; i < A; i++) {
        if (!integer(PyTuple_GET_ITEM(sections, i), &width[i]) || width[i] < 0 || width[i] > 64) return false;
        sum += width[i];
    }
    if (sum != 64) return false;
    a.n_axes = A;
    if (interleaved == Py_True) {
        for (int i = 1; i < A; i++)
            for (int j = 0; j < width[i]; j++) {
                if (i + A * j >= 64) return false;
                a.axis[i + A * j] = (uint8_t)i;
            }
        return true;
    }
    for (int i = 0, at = 0; i < A; i++)
        for (int j = 0; j < width[i]; j++) a.axis[at++] = (uint8_t)i;
    return true;
}
// What ops.norm_rotary and ops.window_append_rotary share: o = q, k, positions, inv_freq, q_norm, k_norm, eps, sections, interleaved.
bool rotary_args(PyObject *const *o, const at::Tensor *&q, const at::Tensor *&k, int &dev, pkv_rotary_args &a) {
    q = tensor(o[0]);
    k = tensor(o[1]);
    const at::Tensor *pos = tensor(o[2]), *freq = tensor(o[3]), *w[2] = {tensor(o[4]), tensor(o[5])};
    dev = here(q);
    if (dev < 0 || !k || !pos || !freq || !whole_rows(*q, dev) || !whole_rows(*k, dev) || !half(*q) || k->scalar_type() != q->scalar_type()) return false;
    const int64_t B = q->size(0), n = q->size(2);
    if (B < 1 || n < 1 || B > INT_MAX || n > INT_MAX || q->size(1) < 1 || k->size(1) < 1 || q->size(1) > INT_MAX || k->size(1) > INT_MAX ||
        k->size(0) != B || k->size(2) != n) return false;
    if (!dense(*freq, dev) || freq->scalar_type() != at::kFloat || freq->dim() != 1 || freq->size(0) != 64) return false;
    for (int i = 0; i < 2; i++)
        if (o[4 + i] != Py_None && (!w[i] || !dense(*w[i], dev) || w[i]->dim() != 1 || w[i]->size(0) != 128 || w[i]->scalar_type() != q->scalar_type())) return false;
    if (!real(o[6], &a.eps) || !frequency_axes(o[7], o[8], a)) return false;
    if (!there(*pos, dev) || (pos->scalar_type() != at::kLong && pos->scalar_type() != at::kInt)) return false;
    const int64_t shape[3] = {o[7] == Py_None ? 1 : a.n_axes, B, n}, d = pos->dim();
    if (d > (o[7] == Py_None ? 2 : 3)) return false;
    for (int64_t i = 0; i < d; i++) {                      // broadcast from the right
        const int64_t size = pos->size(d - 1 - i);
        if (size != shape[2 - i] && size != 1) return false;
        a.pos_stride[2 - i] = size > 1 ? pos->stride(d - 1 - i) : 0;
    }
    a.pos_bytes = pos->scalar_type() == at::kLong ? 8 : 4;
    a.q = at_ptr<void>(*q);
    a.k = at_ptr<void>(*k);
    a.positions = at_ptr<void>(*pos);
    a.inv_freq = at_ptr<float>(*freq);
    a.q_norm = w[0] ? at_ptr<void>(*w[0]) : nullptr;
    a.k_norm = w[1] ? at_ptr<void>(*w[1]) : nullptr;
    row_strides(*q, a.q_stride);
    row_strides(*k, a.k_stride);
    a.dtype = code(*q);
    a.B = (int)B; a.Hq = (int)q->size(1); a.Hkv = (int)k->size(1); a.n = (int)n;
    return true;
}

// norm_rotary(q, k, positions, inv_freq, q_norm, k_norm, eps, sections, interleaved) -> (q, k), a status that is not zero, or None
PyObject *norm_rotary(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *q, *k;
    int dev;
    pkv_rotary_args a{};
    if (n != 9 || modes() || !rotary_args(o, q, k, dev, a)) Py_RETURN_NONE;
    at::Tensor q_out = at::empty(q->sizes(), q->options()), k_out = at::empty(k->sizes(), k->options());
    a.q_out = at_ptr<void>(q_out);
    a.k_out = at_ptr<void>(k_out);
    row_strides(q_out, a.q_out_stride);
    row_strides(k_out, a.k_out_stride);
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.norm_rotary(&a, s); });
    if (rc) return status(rc);
    PyObject *both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(q_out)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(k_out)));
    return both;
    END_HANDLE_TH_ERRORS
}

// window_append_rotary(... as norm_rotary, v, k_win, v_win, win_pos) -> q, a status that is not zero, or None
PyObject *window_append_rotary(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *q, *k;
    int dev, pos;
    pkv_rotary_args a{};
    if (n != 13 || modes() || !rotary_args(o, q, k, dev, a) || !integer(o[12], &pos)) Py_RETURN_NONE;
    const at::Tensor *v = tensor(o[9]), *kw = tensor(o[10]), *vw = tensor(o[11]);
    const auto type = q->scalar_type();
    if (!v || !kw || !vw || !whole_rows(*v, dev) || v->sizes() != k->sizes() || v->scalar_type() != type || !dense(*kw, dev) || !dense(*vw, dev) || kw->dim() != 4 ||
        vw->sizes() != kw->sizes() || kw->size(0) != a.B || kw->size(1) != a.Hkv || kw->size(3) != 128 || kw->scalar_type() != type || vw->scalar_type() != type ||
        pos < 0 || (int64_t)pos + a.n > kw->size(2)) Py_RETURN_NONE;
    at::Tensor q_out = at::empty(q->sizes(), q->options());
    a.q_out = at_ptr<void>(q_out);
    row_strides(q_out, a.q_out_stride);
    a.v = at_ptr<void>(*v);
    row_strides(*v, a.v_stride);
    a.k_out = at_ptr<uint16_t>(*kw) + 128 * (int64_t)pos;
    a.v_out = at_ptr<uint16_t>(*vw) + 128 * (int64_t)pos;
    for (int i = 0; i < 3; i++) a.k_out_stride[i] = a.v_out_stride[i] = kw->stride(i);
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.norm_rotary(&a, s); });
    return rc ? status(rc) : THPVariable_Wrap(std::move(q_out));
    END_HANDLE_TH_ERRORS
}

// attn_chunk(q, k, v, k_win, v_win, sm_scale, win_len, starts, causal) -> the result, a status that is not zero, or None
PyObject *attn_chunk(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *q = n == 9 && !modes() ? tensor(o[0]) : nullptr;
    const int dev = here(q);
    if (dev < 0 || !whole_rows(*q, dev) || !half(*q) || q->numel() == 0 || q->size(0) > INT_MAX || q->size(1) > INT_MAX || q->size(2) > INT_MAX ||
        (o[8] != Py_True && o[8] != Py_False)) Py_RETURN_NONE;
    pkv_attn_args in{};
    Cache c;
    c.batch = (int)q->size(0);
    if (o[1] != Py_None) {
        if (!cache_args(o[1], o[2], dev, c.batch, in, c) || c.like->scalar_type() != q->scalar_type() || c.tokens % 128 ||
            (reinterpret_cast<uintptr_t>(in.k_stream) | reinterpret_cast<uintptr_t>(in.v_stream)) % 16) Py_RETURN_NONE;
    } else if (o[2] != Py_None) {
        Py_RETURN_NONE;
    }
    if (o[3] != Py_None) {
        const at::Tensor *kw = tensor(o[3]);
        if (o[1] == Py_None && kw && kw->dim() == 4) c.heads = (int)kw->size(1);
        if (!window_args(kw, tensor(o[4]), o[6], dev, c, q->scalar_type(), in) ||
            (reinterpret_cast<uintptr_t>(in.k_win) | reinterpret_cast<uintptr_t>(in.v_win)) % 16) Py_RETURN_NONE;
    } else if (o[1] == Py_None || o[4] != Py_None) {
        Py_RETURN_NONE;
    }
    pkv_chunk_args a{};
    a.sm_scale = 0.08838834764831845f;                     // 128 ** -0.5
    if (o[5] != Py_None && !real(o[5], &a.sm_scale)) Py_RETURN_NONE;
    if (o[7] != Py_None) {
        const at::Tensor *starts = tensor(o[7]);
        if (!starts || !dense(*starts, dev) || starts->scalar_type() != at::kInt || starts->dim() != 1 || starts->size(0) != c.batch) Py_RETURN_NONE;
        a.starts = at_ptr<int32_t>(*starts);
    }
    a.causal = o[8] == Py_True;
    if (c.heads < 1 || q->size(1) % c.heads || (a.causal && q->size(2) > (int64_t)c.tokens + in.T_w)) Py_RETURN_NONE;
    at::Tensor out = at::empty_like(*q);
    row_strides(*q, a.q_stride);
    row_strides(out, a.out_stride);
    a.q = at_ptr<void>(*q);
    a.out = at_ptr<void>(out);
    uint64_t off = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out);
    for (int i = 0; i < 3; i++) off |= 2u * (uint64_t)(a.q_stride[i] | a.out_stride[i]);
    if (off % 16 || out.stride(3) != 1) Py_RETURN_NONE;
    a.k_stream = in.k_stream; a.k_info = in.k_info; a.v_stream = in.v_stream; a.v_info = in.v_info;
    a.k_bytes = in.k_bytes; a.v_bytes = in.v_bytes;
    a.k_scale = in.k_scale; a.k_zero = in.k_zero; a.v_scale = in.v_scale; a.v_zero = in.v_zero;
    a.k_win = in.k_win; a.v_win = in.v_win;
    a.B = c.batch; a.Hq = (int)q->size(1); a.Hkv = c.heads; a.n = (int)q->size(2);
    a.T_c = c.tokens; a.T_w = in.T_w;
    a.k_bits = in.k_bits; a.v_bits = in.v_bits; a.dtype = code(*q); a.par_stride = in.par_stride; a.win_stride = in.win_stride;
    const uint64_t need = lib.chunk_workspace(&a);
    at::Tensor space;
    if (need) space = at::empty({(int64_t)need}, q->options().dtype(at::kByte));
    void *const space_p = need ? at_ptr<void>(space) : nullptr;
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.attn_chunk(&a, space_p, need, s); });
    return rc ? status(rc) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// sample(logits, u, temperature, top_k, top_p, min_p, want_logprob) -> tokens, or (tokens, log-probabilities); a status that is not
// zero; or None
PyObject *sample(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *x = n == 7 && !modes() ? tensor(o[0]) : nullptr, *u = x ? tensor(o[1]) : nullptr;
    const int dev = here(x);
    if (dev < 0 || !u || !there(*x, dev) || x->dim() != 2 || x->size(0) < 1 || x->size(0) > INT_MAX || x->size(1) < 1 || x->size(1) > 1 << 20 || x->stride(1) != 1 ||
        (!half(*x) && x->scalar_type() != at::kFloat) || (o[6] != Py_True && o[6] != Py_False)) Py_RETURN_NONE;
    const int64_t rows = x->size(0);
    const auto row_tensor = [&](const at::Tensor *t, at::ScalarType type) {
        return t && dense(*t, dev) && t->scalar_type() == type && t->dim() == 1 && t->size(0) == rows;
    };
    if (!row_tensor(u, at::kFloat)) Py_RETURN_NONE;
    pkv_sample_args a{};
    const float **const at_[3] = {&a.temperature, &a.top_p, &a.min_p};
    float *const all[3] = {&a.temperature_all, &a.top_p_all, &a.min_p_all};
    PyObject *const given[3] = {o[2], o[4], o[5]};
    for (int i = 0; i < 3; i++) {
        const at::Tensor *t = tensor(given[i]);
        if (t) {
            if (!row_tensor(t, at::kFloat)) Py_RETURN_NONE;
            *at_[i] = at_ptr<float>(*t);
        } else if (!real(given[i], all[i]) || !(PyFloat_AS_DOUBLE(given[i]) >= 0.0) || (i && PyFloat_AS_DOUBLE(given[i]) > 1.0)) {
            Py_RETURN_NONE;                                // (as given, not as rounded)
        }
    }
    const at::Tensor *k = tensor(o[3]);
    if (k) {
        if (!row_tensor(k, at::kInt)) Py_RETURN_NONE;
        a.top_k = at_ptr<int32_t>(*k);
    } else if (!integer(o[3], &a.top_k_all) || a.top_k_all < 0) {
        Py_RETURN_NONE;
    }
    at::Tensor token = at::empty({rows}, x->options().dtype(at::kLong)), logprob;
    if (o[6] == Py_True) logprob = at::empty({rows}, x->options().dtype(at::kFloat));
    a.logits = at_ptr<void>(*x);
    a.u = at_ptr<float>(*u);
    a.token = at_ptr<int64_t>(token);
    a.logprob = o[6] == Py_True ? at_ptr<float>(logprob) : nullptr;
    a.row_stride = rows > 1 ? x->stride(0) : 0;
    a.dtype = half(*x) ? code(*x) : PKV_F32;
    a.rows = (int)rows; a.vocab = (int)x->size(1);
    const uint64_t need = lib.sample_workspace(&a);
    at::Tensor space;
    if (need) space = at::empty({(int64_t)need}, x->options().dtype(at::kByte));
    void *const space_p = need ? at_ptr<void>(space) : nullptr;
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.sample(&a, space_p, need, s); });
    if (rc) return status(rc);
    if (o[6] != Py_True) return THPVariable_Wrap(std::move(token));
    PyObject *both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(token)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(logprob)));
    return both;
    END_HANDLE_TH_ERRORS
}

// Rows of [..., width] that lie one behind the other from a 16-byte boundary on.
bool rows16(const at::Tensor &x, int dev) {
    return dense(x, dev) && x.dim() >= 1 && x.numel() > 0 && x.size(-1) % 16 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}
// The 8-bit form's memory for [lead, width], `rows` rows in all (ops._fp8_empty), as a dict.
struct Eight {
    at::Tensor codes, scale;
};
Eight eight_empty(at::IntArrayRef lead, int64_t rows, int64_t width, int64_t block, const at::TensorOptions &like) {
    const int64_t down = (rows + block - 1) / block;
    c10::SmallVector<int64_t, 6> shape(lead.begin(), lead.end()), sizes, strides;
    shape.push_back(width);
    if (block == 1) sizes.append(lead.begin(), lead.end());
    else sizes.push_back(down);
    strides.resize(sizes.size());
    int64_t step = 1;
    for (size_t i = sizes.size(); i-- > 0; step *= sizes[i]) strides[i] = step;
    sizes.push_back((width + 127) / 128);
    strides.push_back(down);
    return Eight{at::empty(shape, like.dtype(at::kFloat8_e4m3fn)), at::empty_strided(sizes, strides, like.dtype(at::kFloat))};
}
PyObject *const s_codes() { static PyObject *const s = PyUnicode_InternFromString("codes"); return s; }
PyObject *const s_scale() { static PyObject *const s = PyUnicode_InternFromString("scale"); return s; }
PyObject *eight_dict(Eight &&e) {
    PyObject *d = PyDict_New(), *c = THPVariable_Wrap(std::move(e.codes)), *s = THPVariable_Wrap(std::move(e.scale));
    if (!d || !c || !s || PyDict_SetItem(d, s_codes(), c) || PyDict_SetItem(d, s_scale(), s)) Py_CLEAR(d);
    Py_XDECREF(c);
    Py_XDECREF(s);
    return d;
}

// add_rms_norm(x, weight, eps, residual, fp8) -> the norm (a tensor or the 8-bit form's dict), with a residual (norm, sum); a status
// that is not zero; or None
PyObject *add_rms_norm(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *x = n == 5 && !modes() ? tensor(o[0]) : nullptr, *w = x ? tensor(o[1]) : nullptr, *res = x ? tensor(o[3]) : nullptr;
    const int dev = here(x);
    if (dev < 0 || !w || !half(*x) || !rows16(*x, dev) || !rows16(*w, dev) || w->dim() != 1 || w->size(0) != x->size(-1) || w->scalar_type() != x->scalar_type() ||
        (o[4] != Py_True && o[4] != Py_False)) Py_RETURN_NONE;
    if (o[3] != Py_None && (!res || !rows16(*res, dev) || res->sizes() != x->sizes() || res->scalar_type() != x->scalar_type())) Py_RETURN_NONE;
    pkv_norm_args a{};
    const int64_t width = x->size(-1), rows = x->numel() / width;
    if (!real(o[2], &a.eps) || width > 65536 || rows >= 1 << 22) Py_RETURN_NONE;
    at::Tensor y, sum;
    Eight e;
    a.x = at_ptr<void>(*x);
    a.weight = at_ptr<void>(*w);
    a.x_stride = width;
    if (res) {
        sum = at::empty(x->sizes(), x->options());
        a.residual = at_ptr<void>(*res);
        a.sum = at_ptr<void>(sum);
        a.residual_stride = a.sum_stride = width;
    }
    if (o[4] == Py_True) {
        e = eight_empty(x->sizes().slice(0, x->dim() - 1), rows, width, 1, x->options());
        a.codes = at_ptr<uint8_t>(e.codes);
        a.scale = at_ptr<float>(e.scale);
        a.codes_stride = width;
        a.scale_stride[0] = 1;
        a.scale_stride[1] = rows;
    } else {
        y = at::empty(x->sizes(), x->options());
        a.out = at_ptr<void>(y);
        a.out_stride = width;
    }
    a.dtype = code(*x); a.rows = (int)rows; a.width = (int)width;
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.add_rms_norm(&a, s); });
    if (rc) return status(rc);
    PyObject *norm = o[4] == Py_True ? eight_dict(std::move(e)) : THPVariable_Wrap(std::move(y));
    if (!res || !norm) return norm;
    PyObject *both = PyTuple_New(2);
    if (!both) {
        Py_DECREF(norm);
        return nullptr;
    }
    PyTuple_SET_ITEM(both, 0, norm);
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(sum)));
    return both;
    END_HANDLE_TH_ERRORS
}

// fp8_quantize(x, block, heads) -> the 8-bit form's dict, a status that is not zero, or None
PyObject *fp8_quantize(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *x = n == 3 && !modes() ? tensor(o[0]) : nullptr;
    const int dev = here(x);
    pkv_fp8_quantize_args a{};
    if (dev < 0 || !half(*x) || !integer(o[1], &a.block) || (a.block != 1 && (a.block != 128 || x->dim() != 2 || o[2] == Py_True)) ||
        (o[2] != Py_True && o[2] != Py_False)) Py_RETURN_NONE;
    int64_t rows, width;
    c10::SmallVector<int64_t, 6> lead;
    if (o[2] == Py_True) {
        if (!whole_rows(*x, dev) || x->numel() == 0) Py_RETURN_NONE;
        int64_t st[3];
        row_strides(*x, st);
        if ((reinterpret_cast<uintptr_t>(x->data_ptr()) | 2u * (uint64_t)(st[0] | st[1] | st[2])) % 16) Py_RETURN_NONE;
        lead = {x->size(0), x->size(2)};
        rows = x->size(0) * x->size(2);
        width = x->size(1) * 128;
        a.x_stride[0] = st[0]; a.x_stride[1] = st[2]; a.x_stride[2] = st[1];
        a.per_batch = x->size(2) > INT_MAX ? 0 : (int)x->size(2);
    } else {
        if (!rows16(*x, dev)) Py_RETURN_NONE;
        lead.append(x->sizes().begin(), x->sizes().end() - 1);
        width = x->size(-1);
        rows = x->numel() / width;
        a.x_stride[1] = width; a.x_stride[2] = 128;
        a.per_batch = rows > INT_MAX ? 0 : (int)rows;
    }
    if (rows > INT_MAX || width > INT_MAX) Py_RETURN_NONE;
    Eight e = eight_empty(lead, rows, width, a.block, x->options());
    a.x = at_ptr<void>(*x);
    a.codes = at_ptr<uint8_t>(e.codes);
    a.scale = at_ptr<float>(e.scale);
    a.codes_stride = width;
    a.scale_stride[0] = 1;
    a.scale_stride[1] = (rows + a.block - 1) / a.block;
    a.dtype = code(*x); a.rows = (int)rows; a.width = (int)width;
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.fp8_quantize(&a, s); });
    return rc ? status(rc) : eight_dict(std::move(e));
    END_HANDLE_TH_ERRORS
}

// fp8_product(x, w, bias, dtype, gated): ops.fp8_linear, or with gated ops.fp8_gated -> the result, a status that is not zero, or None
PyObject *fp8_product(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || modes() || !PyDict_CheckExact(o[0]) || !PyDict_CheckExact(o[1]) || !THPDtype_Check(o[3]) || (o[4] != Py_True && o[4] != Py_False)) Py_RETURN_NONE;
    const at::Tensor *xc = tensor(PyDict_GetItem(o[0], s_codes())), *xs = tensor(PyDict_GetItem(o[0], s_scale())), *wc = tensor(PyDict_GetItem(o[1], s_codes())),
                     *ws = tensor(PyDict_GetItem(o[1], s_scale())), *bias = tensor(o[2]);
    const int dev = here(xc);
    const at::ScalarType type = reinterpret_cast<THPDtype *>(o[3])->scalar_type;
    const bool gated = o[4] == Py_True;
    if (dev < 0 || !xs || !wc || !ws || (type != at::kHalf && type != at::kBFloat16) || !rows16(*xc, dev) || !rows16(*wc, dev) || !there(*xs, dev) || !there(*ws, dev) ||
        xc->scalar_type() != at::kFloat8_e4m3fn || wc->scalar_type() != at::kFloat8_e4m3fn || xs->scalar_type() != at::kFloat || ws->scalar_type() != at::kFloat)
        Py_RETURN_NONE;
    const int64_t width = xc->size(-1), rows = xc->numel() / width, blocks = (width + 127) / 128, d = xc->dim();
    if (wc->dim() != 2 || ws->dim() != 2 || wc->size(1) != width || xs->dim() != d || xs->size(d - 1) != blocks || ws->size(1) != blocks ||
        ws->size(0) != (wc->size(0) + 127) / 128 || width > 1 << 20 || rows > 1 << 24 || wc->size(0) > 1 << 24 || (gated && wc->size(0) % 32)) Py_RETURN_NONE;
    for (int64_t i = 0; i < d - 1; i++)                    // one stride for all rows of scales
        if (xs->size(i) != xc->size(i) || (i + 1 < d - 1 && xs->stride(i) != xs->stride(i + 1) * xs->size(i + 1))) Py_RETURN_NONE;
    const int64_t cols = gated ? wc->size(0) / 2 : wc->size(0);
    pkv_fp8_product_args a{};
    if (o[2] != Py_None) {
        if (!bias || !dense(*bias, dev) || bias->dim() != 1 || bias->size(0) != cols || bias->scalar_type() != type) Py_RETURN_NONE;
        a.bias = at_ptr<void>(*bias);
    }
    c10::SmallVector<int64_t, 6> shape(xc->sizes().begin(), xc->sizes().end() - 1);
    shape.push_back(cols);
    at::Tensor out = at::empty(shape, xc->options().dtype(type));
    a.x = at_ptr<uint8_t>(*xc); a.w = at_ptr<uint8_t>(*wc); a.x_scale = at_ptr<float>(*xs); a.w_scale = at_ptr<float>(*ws);
    a.out = at_ptr<void>(out);
    a.x_stride = a.w_stride = width;
    a.out_stride = cols;
    a.x_scale_stride[0] = rows > 1 ? xs->stride(d - 2) : 0; a.x_scale_stride[1] = xs->stride(d - 1);
    a.w_scale_stride[0] = ws->size(0) > 1 ? ws->stride(0) : 0; a.w_scale_stride[1] = ws->stride(1);
    if (a.x_scale_stride[0] > 1 << 20 || a.w_scale_stride[0] > 1 << 20) Py_RETURN_NONE;
    a.dtype = type == at::kHalf ? PKV_F16 : PKV_BF16;
    a.rows = (int)rows; a.width = (int)width; a.cols = (int)cols; a.gated = gated;
    const pkv_stream_t s = stream(dev);
    const int rc = call([&] { return lib.fp8_product(&a, s); });
    return rc ? status(rc) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(addresses of attn_decode, window_append, dense_view, kq, wv, fused_kq, fused_wv, norm_rotary, attn_chunk_workspace, attn_chunk,
// sample_workspace, sample, add_rms_norm, fp8_quantize, fp8_product)
PyObject *bind(PyObject *, PyObject *const *o, Py_ssize_t n) {
    void *p[15];
    if (n != 15) {
        PyErr_SetString(PyExc_TypeError, "fifteen addresses");
        return nullptr;
    }
    for (int i = 0; i < 15; i++) {
        p[i] = PyLong_AsVoidPtr(o[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    lib.attn_decode = (decltype(lib.attn_decode))p[0];
    lib.window_append = (decltype(lib.window_append))p[1];
    lib.dense_view = (decltype(lib.dense_view))p[2];
    lib.kq = (decltype(lib.kq))p[3];
    lib.wv = (decltype(lib.wv))p[4];
    lib.fused_kq = (decltype(lib.fused_kq))p[5];
    lib.fused_wv = (decltype(lib.fused_wv))p[6];
    lib.norm_rotary = (decltype(lib.norm_rotary))p[7];
    lib.chunk_workspace = (decltype(lib.chunk_workspace))p[8];
    lib.attn_chunk = (decltype(lib.attn_chunk))p[9];
    lib.sample_workspace = (decltype(lib.sample_workspace))p[10];
    lib.sample = (decltype(lib.sample))p[11];
    lib.add_rms_norm = (decltype(lib.add_rms_norm))p[12];
    lib.fp8_quantize = (decltype(lib.fp8_quantize))p[13];
    lib.fp8_product = (decltype(lib.fp8_product))p[14];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"attn_decode", (PyCFunction)(void (*)(void))attn_decode, METH_FASTCALL, nullptr},
    {"plan_step", (PyCFunction)(void (*)(void))plan_step, METH_FASTCALL, nullptr},
    {"window_append", (PyCFunction)(void (*)(void))window_append, METH_FASTCALL, nullptr},
    {"dense_view", (PyCFunction)(void (*)(void))dense_view, METH_FASTCALL, nullptr},
    {"mat_vec", (PyCFunction)(void (*)(void))mat_vec, METH_FASTCALL, nullptr},
    {"fused", (PyCFunction)(void (*)(void))fused, METH_FASTCALL, nullptr},
    {"norm_rotary", (PyCFunction)(void (*)(void))norm_rotary, METH_FASTCALL, nullptr},
    {"window_append_rotary", (PyCFunction)(void (*)(void))window_append_rotary, METH_FASTCALL, nullptr},
    {"attn_chunk", (PyCFunction)(void (*)(void))attn_chunk, METH_FASTCALL, nullptr},
    {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, nullptr},
    {"add_rms_norm", (PyCFunction)(void (*)(void))add_rms_norm, METH_FASTCALL, nullptr},
    {"fp8_quantize", (PyCFunction)(void (*)(void))fp8_quantize, METH_FASTCALL, nullptr},
    {"fp8_product", (PyCFunction)(void (*)(void))fp8_product, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch", PKV_TORCH_VERSION)) Py_CLEAR(m);
    return m;
}
