// The calls a decode step makes per layer, marshalled from torch tensors in C++ (Python module lean_vllm_b200._calls).
//
// Reading the shapes, strides, types and addresses of ten tensors and checking them takes Python 10 us a call, several
// times the kernels' own time for one token; here it takes 1 us. Each function takes the plain case -- no explicit
// stream, output or peers, tensors on the current device, everything as documented -- and returns the output, or the
// library's error code as an int. Anything else it leaves to the Python wrapper (None), which repeats the checks and
// raises what is to be raised, or marshals the rarer arguments: there is one set of rules, and it is that one.
// The library itself stays a plain C one: its entry points come as addresses (bind).

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "kvx.h"

namespace {

decltype(&kvx_attention) g_attention = nullptr;
decltype(&kvx_rotate_store) g_rotate_store = nullptr;

int type_of(const at::Tensor &t) {
    return t.scalar_type() == at::kBFloat16 ? KVX_BF16 : t.scalar_type() == at::kHalf ? KVX_FP16 : -1;
}

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// An optional tensor: false for anything but None or a tensor.
bool optional(PyObject *o, const at::Tensor **out) {
    *out = nullptr;
    if (o == Py_None) return true;
    *out = tensor(o);
    return *out != nullptr;
}

bool integer(PyObject *o, int64_t low, int64_t high, int64_t *out) {
    if (!PyLong_Check(o)) return false;
    *out = PyLong_AsLongLong(o);
    if (*out == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return *out >= low && *out <= high;
}

bool number(PyObject *o, double *out) {
    if (PyFloat_Check(o)) *out = PyFloat_AS_DOUBLE(o);
    else if (PyLong_Check(o)) *out = PyLong_AsDouble(o);
    else return false;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

// Whether a gradient would be lost here, which the wrapper refuses.
bool loses_gradient(std::initializer_list<const at::Tensor *> tensors) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const at::Tensor *t : tensors)
        if (t && t->requires_grad()) return true;
    return false;
}

// A contiguous tensor of `type` on CUDA device `device`.
bool plain(const at::Tensor &t, at::ScalarType type, int device) {
    return t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.is_contiguous();
}

bool index_type(const at::Tensor &t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

bool on_current(const at::Tensor &t, int *device) {
    if (!t.is_cuda()) return false;
    *device = t.get_device();
    return c10::cuda::current_device() == *device;
}

PyObject *finished(int rc, const at::Tensor &out) { return rc == KVX_OK ? THPVariable_Wrap(out) : PyLong_FromLong(rc); }

PyObject *finished(int rc) {
    if (rc != KVX_OK) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
}

constexpr int64_t kInt32 = 0x7fffffff;

// attention(query, k_cache, v_cache, block_tables, kv_lens, scale, q_starts, max_q_len, max_kv_len, softcap, window,
//           slopes, prefix_lens, shared_table, shared_len, workspace address, workspace device, flags, status)
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != 19 || !g_attention) Py_RETURN_NONE;
    const at::Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *tables = tensor(args[3]),
                     *lens = tensor(args[4]), *starts, *slopes, *prefixes, *shared;
    int device;
    if (!q || !k || !v || !tables || !lens || !optional(args[6], &starts) || !optional(args[11], &slopes) ||
        !optional(args[12], &prefixes) || !optional(args[13], &shared) || !on_current(*q, &device) ||
        loses_gradient({q, k, v, slopes}))
        Py_RETURN_NONE;
    int64_t max_q, max_kv = 0, window, shared_len, work, work_device, flags, status;
    double scale = 0, softcap;
    if (!integer(args[7], -kInt32, kInt32, &max_q) || !integer(args[10], -kInt32, kInt32, &window) ||
        !integer(args[14], 0, kInt32, &shared_len) || !integer(args[15], 0, INT64_MAX, &work) ||
        !integer(args[16], 0, kInt32, &work_device) || !integer(args[17], 0, kInt32, &flags) ||
        !integer(args[18], 0, INT64_MAX, &status) || !number(args[9], &softcap) || work_device != device ||
        (args[5] != Py_None && !number(args[5], &scale)) ||
        (args[8] != Py_None && !integer(args[8], -kInt32, kInt32, &max_kv)))
        Py_RETURN_NONE;
    const int type = type_of(*q);
    if (type < 0 || q->dim() != 3 || k->dim() != 4 || tables->dim() != 2 || k->sizes() != v->sizes() ||
        k->strides() != v->strides() || k->stride(3) != 1 || q->stride(2) != 1 || k->size(3) != q->size(2) ||
        k->size(2) < 1 || q->size(1) % k->size(2) != 0 || k->scalar_type() != q->scalar_type() ||
        v->scalar_type() != q->scalar_type() || !k->is_cuda() || !v->is_cuda() || k->get_device() != device ||
        v->get_device() != device || !tables->is_cuda() || tables->get_device() != device ||
        tables->scalar_type() != at::kInt || (tables->size(1) > 1 && tables->stride(1) != 1))
        Py_RETURN_NONE;
    const int64_t batch = tables->size(0), tokens = q->size(0), heads = q->size(1), dim = q->size(2);
    if (!plain(*lens, at::kInt, device) || lens->dim() != 1 || lens->size(0) != batch ||
        (starts ? !plain(*starts, at::kInt, device) || starts->dim() != 1 || starts->size(0) != batch + 1
                : tokens != batch) ||
        (slopes && (!plain(*slopes, at::kFloat, device) || slopes->dim() != 1 || slopes->size(0) != heads)) ||
        (prefixes && (!plain(*prefixes, at::kInt, device) || prefixes->dim() != 1 || prefixes->size(0) != batch)) ||
        (shared && (!plain(*shared, at::kInt, device) || shared->dim() != 1)))
        Py_RETURN_NONE;
    for (const int64_t x : {batch, tokens, heads, dim, k->size(0), k->size(1), tables->size(1), shared ? shared->numel() : 0})
        if (x > kInt32) Py_RETURN_NONE;

    const at::Tensor out = at::empty(q->sizes(), q->options());
    kvx_attention_args a{};
    a.query = q->data_ptr();
    a.q_token_stride = 2 * q->stride(0);
    a.q_head_stride = 2 * q->stride(1);
    a.out = out.data_ptr();
    a.out_token_stride = 2 * heads * dim;
    a.out_head_stride = 2 * dim;
    a.k_cache = reinterpret_cast<uint64_t>(k->data_ptr());
    a.v_cache = reinterpret_cast<uint64_t>(v->data_ptr());
    a.block_stride = 2 * k->stride(0);
    a.token_stride = 2 * k->stride(1);
    a.head_stride = 2 * k->stride(2);
    a.block_tables = static_cast<const int32_t *>(tables->data_ptr());
    a.table_stride = tables->stride(0);
    a.kv_lens = static_cast<const int32_t *>(lens->data_ptr());
    a.q_starts = starts ? static_cast<const int32_t *>(starts->data_ptr()) : nullptr;
    a.slopes = slopes ? static_cast<const float *>(slopes->data_ptr()) : nullptr;
    a.prefix_lens = prefixes ? static_cast<const int32_t *>(prefixes->data_ptr()) : nullptr;
    a.shared_table = shared ? static_cast<const int32_t *>(shared->data_ptr()) : nullptr;
    a.workspace = reinterpret_cast<void *>(work);
    a.status = reinterpret_cast<int32_t *>(status);
    a.shared_len = (int32_t)shared_len;
    a.shared_blocks = shared ? (int32_t)shared->numel() : 0;
    a.block_size = (int32_t)k->size(1);
    a.num_blocks = (int32_t)k->size(0);
    a.max_blocks = (int32_t)tables->size(1);
    a.batch = (int32_t)batch;
    a.num_tokens = (int32_t)tokens;
    a.q_heads = (int32_t)heads;
    a.kv_heads = (int32_t)k->size(2);
    a.head_dim = (int32_t)dim;
    a.dtype = type;
    a.max_q_len = (int32_t)max_q;
    a.max_kv_len = (int32_t)(args[8] == Py_None ? std::min(tables->size(1) * k->size(1), kInt32) : max_kv);
    a.window = (int32_t)window;
    a.scale = args[5] == Py_None ? 1.f / std::sqrt((float)dim) : (float)scale;
    a.softcap = (float)softcap;
    return finished(g_attention(&a, (int)flags, c10::cuda::getCurrentCUDAStream(device).stream()), out);
}

// Slots and positions of the rows, and destination 0.
bool fill_step(const at::Tensor &slots, const at::Tensor &positions, const at::Tensor &table, PyObject *interleaved,
               int64_t tokens, int device, kvx_rotate_args &a, kvx_store_dest &d) {
    if (!index_type(slots) || !index_type(positions) || !plain(slots, slots.scalar_type(), device) ||
        !plain(positions, positions.scalar_type(), device) || slots.numel() != tokens || positions.numel() != tokens ||
        !plain(table, at::kFloat, device) || table.dim() != 2 || table.size(0) > kInt32 || table.size(1) > kInt32 ||
        !PyBool_Check(interleaved) || tokens > kInt32)
        return false;
    d.slot_mapping = slots.data_ptr();
    d.slot_bytes = (int32_t)slots.element_size();
    a.positions = positions.data_ptr();
    a.position_bytes = (int32_t)positions.element_size();
    a.table = static_cast<const float *>(table.data_ptr());
    a.num_positions = (int32_t)table.size(0);
    a.rotary_dim = (int32_t)table.size(1);
    a.interleaved = interleaved == Py_True;
    a.num_tokens = (int32_t)tokens;
    return true;
}

// Rows [tokens][heads][dim], or [tokens][dim] as one head, with their norm's weight if any.
bool fill_rows(const at::Tensor &x, const at::Tensor *weight, int64_t norm_dim, int64_t rotary_first, at::ScalarType type,
               int device, kvx_rotate_rows &r) {
    const int64_t dim = x.size(-1);
    if (x.scalar_type() != type || !x.is_cuda() || x.get_device() != device || x.stride(-1) != 1 || dim > kInt32 ||
        x.size(1) > kInt32 || (weight && (!plain(*weight, type, device) || weight->numel() != norm_dim)))
        return false;
    const bool heads = x.dim() == 3;
    r.rows = x.data_ptr();
    r.token_stride = 2 * x.stride(0);
    r.head_stride = heads ? 2 * x.stride(1) : 0;
    r.num_heads = heads ? (int32_t)x.size(1) : 1;
    r.dim = (int32_t)dim;
    r.norm_dim = weight ? (int32_t)norm_dim : 0;
    r.rotary_first = (int32_t)rotary_first;
    r.weight = weight ? weight->data_ptr() : nullptr;
    return true;
}

void fill_output(const at::Tensor &out, kvx_rotate_args &a) {
    a.query_out = out.data_ptr();
    a.out_token_stride = 2 * out.stride(0);
    a.out_head_stride = 2 * out.stride(1);
}

// rotate_store(query, key, value, k_cache, v_cache, slots, positions, table, interleaved, q_weight, k_weight, eps, flags,
//              status)
PyObject *rotate_store(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != 14 || !g_rotate_store) Py_RETURN_NONE;
    const at::Tensor *t[8], *q_weight, *k_weight;
    for (int i = 0; i < 8; ++i)
        if (!(t[i] = tensor(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &k_cache = *t[3], &v_cache = *t[4];
    int device;
    int64_t flags, status;
    double eps;
    if (!optional(args[9], &q_weight) || !optional(args[10], &k_weight) || !number(args[11], &eps) ||
        !integer(args[12], 0, 0xffffffffll, &flags) || !integer(args[13], 0, INT64_MAX, &status) || !on_current(q, &device) ||
        loses_gradient({&q, &k, &v, q_weight, k_weight, t[7]}))
        Py_RETURN_NONE;
    const int type = type_of(q);
    if (type < 0 || q.dim() != 3 || k.dim() != 3 || k_cache.dim() != 4 || k.sizes() != v.sizes() ||
        k_cache.sizes() != v_cache.sizes() || k_cache.strides() != v_cache.strides() || k_cache.stride(3) != 1 ||
        k_cache.size(2) != k.size(1) || k_cache.size(3) != k.size(2) || q.size(0) != k.size(0) || q.size(2) != k.size(2) ||
        k_cache.scalar_type() != q.scalar_type() || v_cache.scalar_type() != q.scalar_type() || !k_cache.is_cuda() ||
        !v_cache.is_cuda() || k_cache.get_device() != device || v_cache.get_device() != device ||
        k_cache.size(0) > kInt32 || k_cache.size(1) > kInt32)
        Py_RETURN_NONE;
    kvx_rotate_args a{};
    kvx_store_dest d{};
    const int64_t dim = k.size(2);
    if (!fill_step(*t[5], *t[6], *t[7], args[8], k.size(0), device, a, d) || a.rotary_dim > dim ||
        !fill_rows(q, q_weight, dim, 0, q.scalar_type(), device, a.query) ||
        !fill_rows(k, k_weight, dim, 0, q.scalar_type(), device, a.key) ||
        !fill_rows(v, nullptr, 0, 0, q.scalar_type(), device, a.value))
        Py_RETURN_NONE;
    const at::Tensor out = at::empty(q.sizes(), q.options());
    fill_output(out, a);
    a.dtype = type;
    a.eps = (float)eps;
    d.k_cache = reinterpret_cast<uint64_t>(k_cache.data_ptr());
    d.v_cache = reinterpret_cast<uint64_t>(v_cache.data_ptr());
    d.block_stride = 2 * k_cache.stride(0);
    d.token_stride = 2 * k_cache.stride(1);
    d.head_stride = 2 * k_cache.stride(2);
    d.block_size = (int32_t)k_cache.size(1);
    d.num_blocks = (int32_t)k_cache.size(0);
    d.num_heads = a.key.num_heads;
    return finished(g_rotate_store(&a, &d, 1, reinterpret_cast<int32_t *>(status), (int)flags,
                                   c10::cuda::getCurrentCUDAStream(device).stream()),
                    out);
}

// rotate_latents(latent, cache, slots, positions, table, interleaved, query_pe, weight, eps, flags, status); True without
// queries.
PyObject *rotate_latents(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != 11 || !g_rotate_store) Py_RETURN_NONE;
    const at::Tensor *t[5], *pe, *weight;
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = tensor(args[i]))) Py_RETURN_NONE;
    const at::Tensor &latent = *t[0], &cache = *t[1];
    int device;
    int64_t flags, status;
    double eps;
    if (!optional(args[6], &pe) || !optional(args[7], &weight) || !number(args[8], &eps) ||
        !integer(args[9], 0, 0xffffffffll, &flags) || !integer(args[10], 0, INT64_MAX, &status) ||
        !on_current(latent, &device) || loses_gradient({&latent, pe, weight, t[4]}))
        Py_RETURN_NONE;
    const int type = type_of(latent);
    if (type < 0 || latent.dim() != 2 || cache.dim() != 3 || cache.size(2) != latent.size(1) || cache.stride(2) != 1 ||
        cache.stride(1) != latent.size(1) || cache.scalar_type() != latent.scalar_type() || !cache.is_cuda() ||
        cache.get_device() != device || cache.size(0) > kInt32 || cache.size(1) > kInt32)
        Py_RETURN_NONE;
    kvx_rotate_args a{};
    kvx_store_dest d{};
    const int64_t dim = latent.size(1);
    if (!fill_step(*t[2], *t[3], *t[4], args[5], latent.size(0), device, a, d) || a.rotary_dim > dim) Py_RETURN_NONE;
    const int64_t rank = dim - a.rotary_dim;
    if (!fill_rows(latent, weight, rank, rank, latent.scalar_type(), device, a.key)) Py_RETURN_NONE;
    at::Tensor out;
    if (pe) {
        if (pe->dim() != 3 || pe->size(0) != latent.size(0) || pe->size(2) != a.rotary_dim ||
            !fill_rows(*pe, nullptr, 0, 0, latent.scalar_type(), device, a.query))
            Py_RETURN_NONE;
        out = at::empty(pe->sizes(), pe->options());
        fill_output(out, a);
    }
    a.dtype = type;
    a.eps = (float)eps;
    d.k_cache = reinterpret_cast<uint64_t>(cache.data_ptr());
    d.block_stride = 2 * cache.stride(0);
    d.token_stride = 2 * dim;
    d.block_size = (int32_t)cache.size(1);
    d.num_blocks = (int32_t)cache.size(0);
    d.num_heads = 1;
    const int rc = g_rotate_store(&a, &d, 1, reinterpret_cast<int32_t *>(status), (int)flags,
                                  c10::cuda::getCurrentCUDAStream(device).stream());
    return pe ? finished(rc, out) : finished(rc);
}

// bind(address of kvx_attention, address of kvx_rotate_store)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
    int64_t attention_at, rotate_at;
    if (n != 2 || !integer(args[0], 1, INT64_MAX, &attention_at) || !integer(args[1], 1, INT64_MAX, &rotate_at)) {
        PyErr_SetString(PyExc_TypeError, "bind takes the addresses of kvx_attention and kvx_rotate_store");
        return nullptr;
    }
    g_attention = reinterpret_cast<decltype(g_attention)>(attention_at);
    g_rotate_store = reinterpret_cast<decltype(g_rotate_store)>(rotate_at);
    Py_RETURN_NONE;
}

// No C++ exception leaves a call: one can only come ahead of the launch (an allocation that failed, say), and the Python
// wrapper then meets it in its own way.
template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    try {
        return F(self, args, n);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyCFunction method() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<F>));
}

PyMethodDef g_methods[] = {{"attention", method<attention>(), METH_FASTCALL, nullptr},
                           {"rotate_store", method<rotate_store>(), METH_FASTCALL, nullptr},
                           {"rotate_latents", method<rotate_latents>(), METH_FASTCALL, nullptr},
                           {"bind", method<bind>(), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) {
    PyObject *module = PyModule_Create(&g_module);
    if (module && PyModule_AddStringConstant(module, "torch_version", KVX_TORCH_VERSION) != 0) Py_CLEAR(module);
    return module;
}
