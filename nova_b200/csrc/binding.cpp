// Python binding of the serving operators (nova_b200._fast): argument checks,
// output allocation and the C call in one function each.  Through ctypes a call
// takes about 10 us of host time, longer than the kernels of a small step run;
// here it is 4 to 7, of which the launch is most.
//
// Every function raises ValueError for arguments that do not fit, before
// anything is launched, and works on its tensors' device, whichever is current:
// a stream handle alone does not say which device it belongs to.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdexcept>
#include <string>

#include "../../include/nova_b200.h"

namespace {

using at::Tensor;
constexpr int64_t D = 128, PAGE = 64;

struct Refused : std::runtime_error {   // -> ValueError
    using std::runtime_error::runtime_error;
};

[[noreturn]] void refuse(const std::string& what) { throw Refused(what); }

std::string shape_of(const Tensor& t) {
    std::string s = std::string(c10::toString(t.scalar_type())) + " [";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "] on " + t.device().str();
}

// The plan's side: PagePlan._handle / LoraPlan._handle are capsules over one of
// these (written by Python as consecutive int64), named after the plan's class.
struct PageHandle {
    static constexpr const char* name = "nova_b200.PagePlan";
    const nova_paged_plan_info* info;
    int64_t buffer, workspace, workspace_bytes, device, stream;
};
struct LoraHandle {
    static constexpr const char* name = "nova_b200.LoraPlan";
    int64_t tiles, workspace, workspace_bytes, device, stream;
    int64_t n_tiles, tile_rows, tokens, adapters, top_rank;
};

PyObject* handle_name;     // "_handle"
PyObject* other_name;      // "_on_other_stream"

template <typename H>
const H& handle_of(PyObject* plan) {
    PyObject* h = PyObject_GetAttr(plan, handle_name);
    if (!h) throw std::domain_error("");                      // the Python error is set
    const bool host = PyLong_Check(h), mine = !host && PyCapsule_IsValid(h, H::name);
    const void* p = mine ? PyCapsule_GetPointer(h, H::name) : nullptr;
    Py_DECREF(h);                                             // the plan holds it, and what it points at
    if (host) refuse("the plan is not on a CUDA device");
    if (!mine) refuse(std::string("the plan must be a ") + H::name + ", got " + Py_TYPE(plan)->tp_name);
    return *static_cast<const H*>(p);
}

// The current stream; where it is not the plan's own, the plan tells the allocator.
void* stream_for(PyObject* plan, int64_t device, int64_t own) {
    void* s = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream();
    if (reinterpret_cast<int64_t>(s) != own) {
        PyObject* r = PyObject_CallMethodNoArgs(plan, other_name);
        if (!r) throw std::domain_error("");
        Py_DECREF(r);
    }
    return s;
}

const Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

bool on(const Tensor& t, int64_t device) { return t.is_cuda() && t.get_device() == device; }

void want(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, int64_t device) {
    if (t.scalar_type() != type || t.sizes() != shape || !on(t, device)) {
        std::string s;
        for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
        refuse(std::string(name) + " must be " + c10::toString(type) + " [" + s + "] on cuda:" + std::to_string(device) +
               ", got " + shape_of(t));
    }
}
void want_contiguous(const Tensor& t, const char* name) {
    if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
}

void done(int rc, const char* what) {
    if (rc == NOVA_OK) return;
    const std::string msg = std::string(what) + ": " + nova_last_error();
    if (rc == NOVA_ERR_CUDA) throw std::runtime_error(msg);
    refuse(msg);
}

struct Cache {
    int64_t pages, buffers;
    const void *codes, *scales, *tails;
};
Cache cache(PyObject* const* a, const PageHandle& h) {
    const Tensor &codes = tensor(a[0], "codes"), &scales = tensor(a[1], "scales"), &tails = tensor(a[2], "tails");
    const int64_t heads = h.info->kv_heads;
    const int64_t pages = codes.dim() == 5 ? codes.size(0) : 0, buffers = tails.dim() == 5 ? tails.size(0) : 0;
    want(codes, "codes", at::kByte, {pages, heads, 2, PAGE, D}, h.device);
    want(scales, "scales", at::kHalf, {pages, heads, 4, D}, h.device);
    want(tails, "tails", at::kHalf, {buffers, heads, 2, PAGE, D}, h.device);
    want_contiguous(codes, "codes");
    want_contiguous(scales, "scales");
    want_contiguous(tails, "tails");
    return {pages, buffers, codes.const_data_ptr(), scales.const_data_ptr(), tails.const_data_ptr()};
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, int64_t device) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, c10::DeviceIndex(device)));
}

double number(PyObject* o, double otherwise) {
    if (o == Py_None) return otherwise;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw std::domain_error("");
    return v;
}

// (qkv, codes, scales, tails, plan, q_norm_weight, k_norm_weight, eps, cos, sin, out)
PyObject* qkv_append(PyObject* const* a) {
    const PageHandle& h = handle_of<PageHandle>(a[4]);
    const c10::cuda::CUDAGuard guard(c10::DeviceIndex(h.device));
    const nova_paged_plan_info& info = *h.info;
    const Cache c = cache(a + 1, h);
    const Tensor& qkv = tensor(a[0], "qkv");
    want(qkv, "qkv", at::kHalf, {info.tokens, (info.q_heads + 2 * info.kv_heads) * D}, h.device);
    if (qkv.stride(1) != 1) refuse("qkv needs a contiguous last dimension");
    nova_paged_append_args p{};
    p.qkv = qkv.const_data_ptr();
    p.qkv_stride = info.tokens > 1 ? qkv.stride(0) : qkv.size(1);
    const char* names[2] = {"q_norm_weight", "k_norm_weight"};
    const void** to[2] = {&p.q_norm_weight, &p.k_norm_weight};
    for (int i = 0; i < 2; ++i)
        if (const Tensor* w = optional(a[5 + i], names[i])) {
            want(*w, names[i], at::kHalf, {D}, h.device);
            want_contiguous(*w, names[i]);
            *to[i] = w->const_data_ptr();
        }
    p.eps = number(a[7], 1e-6);
    const Tensor *cos = optional(a[8], "cos"), *sin = optional(a[9], "sin");
    if (!cos != !sin) refuse("cos and sin go together");
    if (cos) {
        p.rope_len = cos->dim() == 2 ? cos->size(0) : 0;
        want(*cos, "cos", at::kHalf, {p.rope_len, D}, h.device);
        want(*sin, "sin", at::kHalf, {p.rope_len, D}, h.device);
        want_contiguous(*cos, "cos");
        want_contiguous(*sin, "sin");
        p.cos = cos->const_data_ptr();
        p.sin = sin->const_data_ptr();
    }
    const Tensor* given = optional(a[10], "out");
    const Tensor out = given ? *given : empty({info.tokens, info.q_heads, D}, at::kHalf, h.device);
    if (given) {
        want(out, "out", at::kHalf, {info.tokens, info.q_heads, D}, h.device);
        if (out.stride(2) != 1 || (info.q_heads > 1 && out.stride(1) != D)) refuse("out needs contiguous rows");
    }
    p.q_out = out.mutable_data_ptr();
    p.q_t_stride = info.tokens > 1 ? out.stride(0) : info.q_heads * D;
    p.codes = const_cast<void*>(c.codes);
    p.scales = const_cast<void*>(c.scales);
    p.tails = const_cast<void*>(c.tails);
    p.num_pages = c.pages;
    p.num_tails = c.buffers;
    p.plan = reinterpret_cast<const int32_t*>(h.buffer);
    done(nova_paged_append(&p, &info, stream_for(a[4], h.device, h.stream)), "nova_paged_append");
    return THPVariable_Wrap(out);
}

// (codes, scales, tails, plan)
PyObject* paged_read(PyObject* const* a) {
    const PageHandle& h = handle_of<PageHandle>(a[3]);
    const c10::cuda::CUDAGuard guard(c10::DeviceIndex(h.device));
    const Cache c = cache(a, h);
    const Tensor k = empty({h.info->read_rows, h.info->kv_heads, D}, at::kHalf, h.device);
    const Tensor v = empty({h.info->read_rows, h.info->kv_heads, D}, at::kHalf, h.device);
    done(nova_paged_read(c.codes, c.scales, c.tails, c.pages, c.buffers, reinterpret_cast<const int32_t*>(h.buffer), h.info,
                         k.mutable_data_ptr(), v.mutable_data_ptr(), stream_for(a[3], h.device, h.stream)),
         "nova_paged_read");
    PyObject *pk = THPVariable_Wrap(k), *pv = THPVariable_Wrap(v);
    PyObject* r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return r;
}

// (q, codes, scales, tails, plan, window, scale, out, lse_out)
PyObject* paged_attention(PyObject* const* a) {
    const PageHandle& h = handle_of<PageHandle>(a[4]);
    const c10::cuda::CUDAGuard guard(c10::DeviceIndex(h.device));
    const nova_paged_plan_info& info = *h.info;
    const Cache c = cache(a + 1, h);
    const Tensor& q = tensor(a[0], "q");
    want(q, "q", at::kHalf, {info.tokens, info.q_heads, D}, h.device);
    nova_paged_attn_args p{};
    const int64_t window = PyLong_AsLongLong(a[5]);
    if (window == -1 && PyErr_Occurred()) throw std::domain_error("");
    while (p.sched < info.n_windows && info.sched[p.sched].window != window) ++p.sched;
    if (p.sched == info.n_windows) refuse("window " + std::to_string(window) + " is not one of the plan's");
    const Tensor* given = optional(a[7], "out");
    const Tensor out = given ? *given : empty({info.tokens, info.q_heads, D}, at::kHalf, h.device);
    if (given) want(out, "out", at::kHalf, {info.tokens, info.q_heads, D}, h.device);
    if (q.stride(2) != 1 || out.stride(2) != 1) refuse("q and out need a contiguous last dimension");
    if (const Tensor* lse = optional(a[8], "lse_out")) {
        want(*lse, "lse_out", at::kFloat, {info.tokens, info.q_heads}, h.device);
        want_contiguous(*lse, "lse_out");
        p.lse = lse->mutable_data_ptr();
    }
    p.q = q.const_data_ptr();
    const bool tokens = info.tokens > 1, heads = info.q_heads > 1;   // a dimension of one has a stride that says nothing
    p.q_t_stride = tokens ? q.stride(0) : 0;
    p.q_h_stride = heads ? q.stride(1) : 0;
    p.codes = c.codes;
    p.scales = c.scales;
    p.tails = c.tails;
    p.num_pages = c.pages;
    p.num_tails = c.buffers;
    p.out = out.mutable_data_ptr();
    p.o_t_stride = tokens ? out.stride(0) : 0;
    p.o_h_stride = heads ? out.stride(1) : 0;
    p.scale = number(a[6], 0.08838834764831845);
    p.plan = reinterpret_cast<const int32_t*>(h.buffer);
    p.workspace = reinterpret_cast<void*>(h.workspace);
    p.workspace_bytes = h.workspace_bytes;
    done(nova_paged_attention(&p, &info, stream_for(a[4], h.device, h.stream)), "nova_paged_attention");
    return THPVariable_Wrap(out);
}

// (x, base, a, b, plan, scaling, out)
PyObject* lora_add(PyObject* const* o) {
    const LoraHandle& h = handle_of<LoraHandle>(o[4]);
    const c10::cuda::CUDAGuard guard(c10::DeviceIndex(h.device));
    const Tensor &x = tensor(o[0], "x"), &base = tensor(o[1], "base"), &a = tensor(o[2], "a"), &b = tensor(o[3], "b");
    if (x.dim() != 2 || base.dim() != 2 || a.dim() != 3) refuse("x and base must be 2-D, a and b 3-D");
    const int64_t k = x.size(1), n = base.size(1), r = a.size(1);
    want(x, "x", at::kHalf, {h.tokens, k}, h.device);
    want(base, "base", at::kHalf, {h.tokens, n}, h.device);
    want(a, "a", at::kHalf, {h.adapters, r, k}, h.device);
    want(b, "b", at::kHalf, {h.adapters, n, r}, h.device);
    if (h.top_rank > r) refuse("the plan has rank " + std::to_string(h.top_rank) + ", the weights hold " + std::to_string(r));
    want_contiguous(a, "a");
    want_contiguous(b, "b");
    nova_lora_args p{};
    if (const Tensor* s = optional(o[5], "scaling")) {
        want(*s, "scaling", at::kFloat, {h.adapters}, h.device);
        want_contiguous(*s, "scaling");
        p.scaling = s->const_data_ptr();
    }
    const Tensor* given = optional(o[6], "out");
    const Tensor out = given ? *given : empty({h.tokens, n}, at::kHalf, h.device);
    if (given) want(out, "out", at::kHalf, {h.tokens, n}, h.device);
    if (x.stride(1) != 1 || base.stride(1) != 1 || out.stride(1) != 1) refuse("x, base and out need a contiguous last dimension");
    const bool many = h.tokens > 1;             // a single row's stride says nothing
    p.x = x.const_data_ptr();
    p.x_stride = many ? x.stride(0) : k;
    p.base = base.const_data_ptr();
    p.base_stride = many ? base.stride(0) : n;
    p.out = out.mutable_data_ptr();
    p.out_stride = many ? out.stride(0) : n;
    p.a = a.const_data_ptr();
    p.b = b.const_data_ptr();
    p.tiles = reinterpret_cast<const int32_t*>(h.tiles);
    p.n_tiles = h.n_tiles;
    p.tile_rows = h.tile_rows;
    p.tokens = h.tokens;
    p.k = k;
    p.n = n;
    p.adapters = h.adapters;
    p.max_rank = r;
    p.top_rank = h.top_rank;
    p.workspace = reinterpret_cast<void*>(h.workspace);
    p.workspace_bytes = h.workspace_bytes;
    done(nova_lora_add(&p, stream_for(o[4], h.device, h.stream)), "nova_lora_add");
    return THPVariable_Wrap(out);
}

// (logits, history, repetition, frequency, presence, LogitBias._handle or None, allowed, allowed_row, out)
PyObject* adjust_logits(PyObject* const* a) {
    const Tensor& logits = tensor(a[0], "logits");
    const at::ScalarType type = logits.scalar_type();
    if (!logits.is_cuda() || logits.dim() != 2 || (type != at::kHalf && type != at::kFloat) || logits.stride(1) != 1)
        refuse("logits must be CUDA float16 or float32 [rows, vocab] with a contiguous last dimension, got " + shape_of(logits));
    const int64_t rows = logits.size(0), vocab = logits.size(1), device = logits.get_device();
    const c10::cuda::CUDAGuard guard(c10::DeviceIndex(device));
    nova_logits_args p{};
    p.rows = rows;
    p.vocab = vocab;
    p.logits = logits.const_data_ptr();
    p.logits_stride = rows > 1 ? logits.stride(0) : vocab;
    p.logits_fp32 = type == at::kFloat;
    const Tensor* history = optional(a[1], "history");
    if (history) {
        want(*history, "history", at::kShort, {rows, vocab}, device);
        if (history->stride(1) != 1) refuse("history needs a contiguous last dimension");
        p.history = history->const_data_ptr();
        p.history_stride = rows > 1 ? history->stride(0) : vocab;
    }
    const char* names[3] = {"repetition", "frequency", "presence"};
    const void** to[3] = {&p.repetition, &p.frequency, &p.presence};
    for (int i = 0; i < 3; ++i)
        if (const Tensor* t = optional(a[2 + i], names[i])) {
            want(*t, names[i], at::kFloat, {rows}, device);
            want_contiguous(*t, names[i]);
            if (!history) refuse(std::string(names[i]) + " needs a history");
            *to[i] = t->const_data_ptr();
        }
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device));
    if (a[5] != Py_None) {                      // LogitBias._handle: rows, vocab, number of biases, stream, buffer
        long long v[4];
        PyObject* held;
        if (!PyTuple_Check(a[5])) refuse("bias must be a LogitBias");
        if (!PyArg_ParseTuple(a[5], "LLLLO", v, v + 1, v + 2, v + 3, &held)) throw std::domain_error("");
        const Tensor& list = tensor(held, "the bias list");
        if (v[0] != rows || v[1] != vocab || !on(list, device))
            refuse("bias is for [" + std::to_string(v[0]) + ", " + std::to_string(v[1]) + "] logits on " +
                   list.device().str() + ", got " + shape_of(logits));
        if (v[2] > 0) {                         // offsets, then tokens, then values; no biases: no pointers
            p.bias_off = static_cast<const int32_t*>(list.const_data_ptr());
            p.bias_token = p.bias_off + (list.numel() - 2 * v[2]);
            p.bias_value = p.bias_token + v[2];
            // a stream other than the list's own reads it: the allocator must know
            if (reinterpret_cast<int64_t>(stream.stream()) != v[3]) list.record_stream(stream.unwrap());
        }
    }
    const Tensor *allowed = optional(a[6], "allowed"), *which = optional(a[7], "allowed_row");
    if (allowed) {
        const int64_t words = (vocab + 31) / 32;
        if (allowed->scalar_type() != at::kInt || allowed->dim() != 2 || !on(*allowed, device) || allowed->size(0) < 1 ||
            allowed->size(1) < words || allowed->stride(1) != 1 ||
            (allowed->size(0) > 1 && allowed->stride(0) < allowed->size(1)))
            refuse("allowed must be int32 [masks, " + std::to_string(words) + "] with rows of their own on the logits' device, got " +
                   shape_of(*allowed));
        p.allowed = allowed->const_data_ptr();
        p.n_masks = allowed->size(0);
        p.mask_stride = p.n_masks > 1 ? allowed->stride(0) : allowed->size(1);
        if (which) {
            want(*which, "allowed_row", at::kInt, {rows}, device);
            want_contiguous(*which, "allowed_row");
            p.allowed_row = static_cast<const int32_t*>(which->const_data_ptr());
        } else if (p.n_masks != rows) {
            refuse(std::to_string(p.n_masks) + " masks for " + std::to_string(rows) + " rows need allowed_row");
        }
    } else if (which) {
        refuse("allowed_row needs allowed");
    }
    const Tensor* given = optional(a[8], "out");
    const Tensor out = given ? *given : empty({rows, vocab}, type, device);
    if (given) {
        want(out, "out", type, {rows, vocab}, device);
        if (out.stride(1) != 1) refuse("out needs a contiguous last dimension");
    }
    p.out = out.mutable_data_ptr();
    p.out_stride = rows > 1 ? out.stride(0) : vocab;
    done(nova_adjust_logits(&p, stream.stream()), "nova_adjust_logits");
    return THPVariable_Wrap(out);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments are needed, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const std::domain_error&) {        // a Python error that is set already
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define ENTRY(name, n) \
    { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<name, n>)), METH_FASTCALL, nullptr }

PyMethodDef methods[] = {ENTRY(qkv_append, 11), ENTRY(paged_read, 4), ENTRY(paged_attention, 9), ENTRY(lora_add, 7),
                         ENTRY(adjust_logits, 9), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "Binding of the serving operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fast() {
    handle_name = PyUnicode_InternFromString("_handle");
    other_name = PyUnicode_InternFromString("_on_other_stream");
    return handle_name && other_name ? PyModule_Create(&module) : nullptr;
}
