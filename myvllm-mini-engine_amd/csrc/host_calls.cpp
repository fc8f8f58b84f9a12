// Native call path of the Python entry points.
//
// A small decode or prefill call runs 4-10 us on the GPU; checking its
// tensors, allocating its output and workspace and marshalling two dozen
// arguments in Python costs more than that.  These functions do the same for
// the plain form of a call -- ordinary dense CUDA tensors on the current
// device, no caller-supplied buffers, no host-synchronising validation -- and
// return None for anything else, also for everything the entry points refuse:
// the Python code then runs its checks in full and raises what it always
// raised.  Nothing is kept between calls.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "mvme_fp4.h"
#include "mvme_long.h"
#include "mvme_paged.h"

namespace {

// Entry points of libmvme_paged, bound once by the loader.
struct Library {
    decltype(&mvme_last_error) last_error;
    decltype(&mvme_paged_attention_workspace_size) decode_workspace;
    decltype(&mvme_paged_attention) decode;
    decltype(&mvme_paged_attention_decode_write) decode_write;
    decltype(&mvme_paged_prefill_workspace_size) prefill_workspace;
    decltype(&mvme_paged_prefill_attention) prefill;
    decltype(&mvme_prefill_attention_workspace_size) dense_workspace;
    decltype(&mvme_prefill_attention) dense;
    decltype(&mvme_write_kv_cache_slots) write_slots;
    decltype(&mvme_linear_rows) linear;
    decltype(&mvme_qk_norm_rope_write_kv) rope;
    decltype(&mvme_fp4_record_bytes) fp4_record;
    decltype(&mvme_fp4_write_slots) fp4_write_slots;
    decltype(&mvme_fp4_write_batch) fp4_write_batch;
    decltype(&mvme_fp4_gather_slots) fp4_gather_slots;
    decltype(&mvme_fp4_paged_attention_workspace_size) fp4_decode_workspace;
    decltype(&mvme_fp4_paged_attention) fp4_decode;
    decltype(&mvme_fp4_paged_prefill_workspace_size) fp4_prefill_workspace;
    decltype(&mvme_fp4_paged_prefill_attention) fp4_prefill;
    decltype(&mvme_copy_pages) copy_pages;
    decltype(&mvme_compact_pages) compact_pages;
    decltype(&mvme_paged_attention_shared_prefix_workspace_size) shared_workspace;
    decltype(&mvme_paged_attention_shared_prefix) shared_prefix;
    decltype(&mvme_paged_attention_weights_workspace_size) weights_workspace;
    decltype(&mvme_paged_attention_weights) decode_weights;
    decltype(&mvme_prefill_attention_weights_workspace_size) prefill_weights_workspace;
    decltype(&mvme_prefill_attention_weights) prefill_weights;
    decltype(&mvme_evict_kv_cache) evict;
} lib;
PyObject* current_raw_stream = nullptr;  // torch's getter: device index -> hipStream_t

constexpr int64_t kMaxCapacity = 1048576;
constexpr int64_t kMaxBatchHeads = 2147483647;

// The tensor behind an exact torch.Tensor / Parameter with dense CUDA storage
// of the process's current device; nullptr for anything else (subclasses,
// functorch wrappers, fake or sparse tensors).
const at::Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
    if (t.unsafeGetTensorImpl()->is_python_dispatch() || t.is_conj() || t.is_neg()) return nullptr;
    return &t;
}

// Ordinary eager state: no function or dispatch mode wants to see the calls
// that the Python path would make.
bool eager() { return !at::impl::torch_function_mode_enabled() && !c10::impl::dispatch_mode_enabled(); }

bool as_int(PyObject* o, int64_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}

bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? MVME_FP16 : MVME_BF16; }
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
bool on_current_device(const at::Tensor& t) {
    return c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index() == t.device().index();
}

// torch's current stream on the tensor's device; false with an error set.
bool stream_of(const at::Tensor& t, void*& stream) {
    PyObject* index = PyLong_FromLong(t.device().index());
    PyObject* raw = index ? PyObject_CallOneArg(current_raw_stream, index) : nullptr;
    Py_XDECREF(index);
    if (!raw) return false;
    stream = PyLong_AsVoidPtr(raw);
    Py_DECREF(raw);
    return !PyErr_Occurred();
}

at::Tensor bytes_like(const at::Tensor& t, size_t bytes) {
    return at::empty({static_cast<int64_t>(bytes)}, t.options().dtype(at::kByte).requires_grad(false));
}

PyObject* raise_status(const char* name, int status) {
    const char* message = lib.last_error();
    PyErr_Format(PyExc_RuntimeError, "%s: %s (status %d)", name, message ? message : "", status);
    return nullptr;
}

// Token stride of [T, H, D] rows the kernels can read in place, or -1.
int64_t row_stride(const at::Tensor& t) {
    const int64_t tokens = t.size(0), heads = t.size(1), dim = t.size(2);
    if ((dim != 1 && t.stride(2) != 1) || (heads != 1 && t.stride(1) != dim)) return -1;
    if (tokens <= 1) return heads * dim;
    return t.stride(0) >= heads * dim ? t.stride(0) : -1;
}

// What decode needs of the cache, the tables and the lengths beside a query
// of [batch, q_heads, head_dim] (which may be a strided view).
struct DecodeShape {
    int64_t batch, q_heads, kv_heads, head_dim, num_blocks, block, width;
};
bool decode_shape(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                  const at::Tensor& lens, int64_t block, DecodeShape& s) {
    if (q.dim() != 3 || k.dim() != 4 || v.dim() != 4 || tables.dim() != 2 || lens.dim() != 1) return false;
    const auto device = q.device();
    if (k.device() != device || v.device() != device || tables.device() != device || lens.device() != device) return false;
    if (!half_type(q) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
        tables.scalar_type() != at::kLong || lens.scalar_type() != at::kLong)
        return false;
    if (!k.is_contiguous() || !v.is_contiguous() || !tables.is_contiguous() || !lens.is_contiguous()) return false;
    if (v.sizes() != k.sizes()) return false;
    s = {q.size(0), q.size(1), k.size(2), q.size(2), k.size(0), block, tables.size(1)};
    if (s.batch <= 0 || s.q_heads <= 0 || s.num_blocks <= 0 || s.kv_heads <= 0 || block <= 0 || k.size(1) != block ||
        k.size(3) != s.head_dim || s.q_heads % s.kv_heads != 0)
        return false;
    switch (s.head_dim) {
        case 16: case 32: case 64: case 80: case 96: case 128: case 192: case 256: break;
        default: return false;
    }
    return tables.size(0) == s.batch && s.width > 0 && lens.size(0) == s.batch && block <= kMaxCapacity &&
           s.width <= kMaxCapacity / block && s.batch <= kMaxBatchHeads / s.q_heads;
}

// decode(query, key_cache, value_cache, block_tables, context_lens, block_size, partition_tokens)
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, partition = 0;
    if (n != 7 || !as_int(args[5], block) || !as_int(args[6], partition)) Py_RETURN_NONE;
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &tables = *t[3], &lens = *t[4];
    DecodeShape s;
    if (!eager() || !on_current_device(q) || !decode_shape(q, k, v, tables, lens, block, s) || !q.is_contiguous())
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const size_t need = lib.decode_workspace(s.batch, s.q_heads, s.kv_heads, s.head_dim, block, s.width, partition);
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.decode(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                        static_cast<const int64_t*>(tables.data_ptr()), static_cast<const int64_t*>(lens.data_ptr()),
                        s.batch, s.q_heads, s.kv_heads, s.head_dim, s.num_blocks, block, s.width, partition,
                        dtype_code(q), ws, need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_paged_attention", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// decode_write(query, key_cache, value_cache, block_tables, context_lens, block_size, new_key, new_value,
//              q_weight, k_weight, cos, sin, eps, partition_tokens): the fused form with norm and RoPE
// (or, with None for the four, the plain write) for rows the one launch can read in place.
PyObject* decode_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, partition = 0;
    if (n != 14 || !as_int(args[5], block) || !as_int(args[13], partition) || !PyFloat_CheckExact(args[12]))
        Py_RETURN_NONE;
    const bool rope = args[8] != Py_None;
    const double eps = PyFloat_AS_DOUBLE(args[12]);
    const at::Tensor* t[12] = {};
    for (int i = 0; i < 12; ++i) {
        if (i == 5 || (i >= 8 && !rope)) continue;
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    }
    // Without q_weight the Python path does not look at the other three.
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &tables = *t[3], &lens = *t[4], &nk = *t[6], &nv = *t[7];
    DecodeShape s;
    if (!eager() || !on_current_device(q) || !decode_shape(q, k, v, tables, lens, block, s)) Py_RETURN_NONE;
    switch (s.head_dim) {
        case 16: case 32: case 64: case 128: case 256: break;
        default: Py_RETURN_NONE;
    }
    const auto device = q.device();
    for (const at::Tensor* r : {&nk, &nv})
        if (r->dim() != 3 || r->size(0) != s.batch || r->size(1) != s.kv_heads || r->size(2) != s.head_dim ||
            r->scalar_type() != q.scalar_type() || r->device() != device || !aligned16(*r))
            Py_RETURN_NONE;
    const int64_t qs = rope ? row_stride(q) : s.q_heads * s.head_dim, ks = row_stride(nk), vs = row_stride(nv);
    if ((!rope && !q.is_contiguous()) || qs < 0 || ks < 0 || vs < 0 || qs % 8 || ks % 8 || vs % 8 || !aligned16(q) ||
        !aligned16(k) || !aligned16(v))
        Py_RETURN_NONE;
    if (rope) {
        for (int i = 8; i < 10; ++i)
            if (t[i]->scalar_type() != q.scalar_type() || t[i]->dim() != 1 || t[i]->size(0) != s.head_dim ||
                !t[i]->is_contiguous() || t[i]->device() != device || !aligned16(*t[i]))
                Py_RETURN_NONE;
        for (int i = 10; i < 12; ++i)
            if (t[i]->dim() != 2 || t[i]->size(0) != s.batch || t[i]->size(1) * 2 != s.head_dim ||
                !t[i]->is_contiguous() || t[i]->scalar_type() != q.scalar_type() || t[i]->device() != device ||
                !aligned16(*t[i]))
                Py_RETURN_NONE;
    }
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const size_t need = lib.decode_workspace(s.batch, s.q_heads, s.kv_heads, s.head_dim, block, s.width, partition);
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    auto ptr = [&](int i) -> const void* { return rope ? t[i]->data_ptr() : nullptr; };
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.decode_write(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                              static_cast<const int64_t*>(tables.data_ptr()),
                              static_cast<const int64_t*>(lens.data_ptr()), s.batch, s.q_heads, s.kv_heads, s.head_dim,
                              s.num_blocks, block, s.width, partition, dtype_code(q), nk.data_ptr(), nv.data_ptr(), ks,
                              vs, ptr(8), ptr(9), ptr(10), ptr(11), static_cast<float>(eps), qs, nullptr, ws, need,
                              stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_paged_attention_decode_write", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// prefill(q, key_cache, value_cache, cu_seqlens_q, query_starts, block_tables, context_lens, block_size, chunk_tokens)
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, chunk = 0;
    if (n != 9 || !as_int(args[7], block) || !as_int(args[8], chunk)) Py_RETURN_NONE;
    const at::Tensor* t[7];
    for (int i = 0; i < 7; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &cu = *t[3], &starts = *t[4], &tables = *t[5], &lens = *t[6];
    if (!eager() || !on_current_device(q)) Py_RETURN_NONE;
    if (q.dim() != 3 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(1) != block || block <= 0 || k.numel() <= 0 ||
        !k.is_contiguous() || !v.is_contiguous() || !q.is_contiguous() || !half_type(q) ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        Py_RETURN_NONE;
    const int64_t tokens = q.size(0), q_heads = q.size(1), head_dim = q.size(2), kv_heads = k.size(2);
    if (tokens <= 0 || q_heads <= 0 || head_dim != k.size(3) || head_dim > 1024 || q_heads % kv_heads != 0) Py_RETURN_NONE;
    if (cu.dim() != 1 || starts.dim() != 1 || lens.dim() != 1 || tables.dim() != 2) Py_RETURN_NONE;
    const int64_t seqs = starts.size(0), width = tables.size(1);
    if (tables.size(0) != seqs || lens.size(0) != seqs || cu.size(0) != seqs + 1) Py_RETURN_NONE;
    for (int i = 1; i < 7; ++i) {
        if (t[i]->device() != q.device()) Py_RETURN_NONE;
        if (i >= 3 && (t[i]->scalar_type() != at::kLong || !t[i]->is_contiguous())) Py_RETURN_NONE;
    }
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const size_t need = lib.prefill_workspace(seqs, tokens, q_heads, kv_heads, head_dim, block, width, chunk,
                                              dtype_code(q));
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.prefill(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         static_cast<const int64_t*>(cu.data_ptr()), static_cast<const int64_t*>(starts.data_ptr()),
                         static_cast<const int64_t*>(tables.data_ptr()), static_cast<const int64_t*>(lens.data_ptr()),
                         seqs, tokens, q_heads, kv_heads, head_dim, k.size(0), block, width, chunk, dtype_code(q), ws,
                         need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_paged_prefill_attention", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// dense(q, k, v, query_start): [batch, heads, tokens, head_dim] views whose layout needs no copy, head
// dims of the MFMA path.
PyObject* dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t start = 0;
    if (n != 4 || !as_int(args[3], start)) Py_RETURN_NONE;
    const at::Tensor* t[3];
    for (int i = 0; i < 3; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2];
    if (!eager() || !on_current_device(q) || q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() ||
        v.strides() != k.strides() || !half_type(q) || k.scalar_type() != q.scalar_type() ||
        v.scalar_type() != q.scalar_type() || k.device() != q.device() || v.device() != q.device())
        Py_RETURN_NONE;
    const int64_t batch = q.size(0), q_heads = q.size(1), tokens = q.size(2), d = q.size(3);
    const int64_t kv_heads = k.size(1), kv_tokens = k.size(2);
    if (batch <= 0 || q_heads <= 0 || tokens <= 0 || d <= 0 || d % 8 != 0 || d > 256 || kv_heads <= 0 ||
        q_heads % kv_heads != 0 || k.size(0) != batch || k.size(3) != d || start < 0 || start > kMaxCapacity ||
        start + tokens > kv_tokens || start + tokens > kMaxCapacity)
        Py_RETURN_NONE;
    // (batch, head, token) strides as the kernels read them: 0 for dimensions of size 1.
    int64_t st[3][3];
    for (int i = 0; i < 3; ++i) {
        if (t[i]->stride(3) != 1 || !aligned16(*t[i])) Py_RETURN_NONE;
        for (int j = 0; j < 3; ++j) {
            st[i][j] = t[i]->size(j) > 1 ? t[i]->stride(j) : 0;
            if (st[i][j] % 8 != 0) Py_RETURN_NONE;
        }
    }
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty({batch, tokens, q_heads, d}, q.options().requires_grad(false)).transpose(1, 2);
    int64_t so[3];
    for (int j = 0; j < 3; ++j) so[j] = out.size(j) > 1 ? out.stride(j) : 0;
    const size_t need = lib.dense_workspace(batch, tokens, q_heads, kv_heads, d, start, dtype_code(q));
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.dense(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), batch, q_heads, kv_heads, tokens,
                       kv_tokens, d, start, st[0][0], st[0][1], st[0][2], st[1][0], st[1][1], st[1][2], so[0], so[1],
                       so[2], dtype_code(q), ws, need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_prefill_attention", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// write_slots(key_cache, value_cache, slot_mapping, key, value): True when the rows were written.
PyObject* write_slots(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) Py_RETURN_NONE;
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &kc = *t[0], &vc = *t[1], &slots = *t[2], &key = *t[3], &value = *t[4];
    if (!eager() || !on_current_device(kc) || kc.dim() != 4 || vc.sizes() != kc.sizes() || kc.numel() <= 0 ||
        !kc.is_contiguous() || !vc.is_contiguous() || key.dim() != 3 || value.sizes() != key.sizes() ||
        key.size(1) != kc.size(2) || key.size(2) != kc.size(3) || slots.dim() != 1 || slots.size(0) != key.size(0) ||
        key.size(0) <= 0 || slots.scalar_type() != at::kLong || !slots.is_contiguous() || !half_type(kc))
        Py_RETURN_NONE;
    for (int i = 1; i < 5; ++i)
        if (t[i]->device() != kc.device() || (i != 2 && t[i]->scalar_type() != kc.scalar_type())) Py_RETURN_NONE;
    const int64_t ks = row_stride(key), vs = row_stride(value);
    if (ks < 0 || vs < 0) Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(kc, stream)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.write_slots(kc.data_ptr(), vc.data_ptr(), kc.size(0), kc.size(1), kc.size(2), kc.size(3),
                             static_cast<const int64_t*>(slots.data_ptr()), key.data_ptr(), value.data_ptr(),
                             key.size(0), ks, vs, dtype_code(kc), stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_write_kv_cache_slots", status);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// linear(x, weight, bias or None) for x of [..., in_features] with dense rows.
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) Py_RETURN_NONE;
    const at::Tensor *x = plain(args[0]), *w = plain(args[1]);
    const at::Tensor* bias = args[2] == Py_None ? nullptr : plain(args[2]);
    if (!x || !w || (args[2] != Py_None && !bias) || !eager() || !on_current_device(*x)) Py_RETURN_NONE;
    if (x->dim() != 2 || w->dim() != 2 || !half_type(*x) || w->scalar_type() != x->scalar_type() ||
        w->device() != x->device() || !w->is_contiguous())
        Py_RETURN_NONE;
    const int64_t rows = x->size(0), in = x->size(1), out_features = w->size(0);
    if (rows < 1 || rows > 64 || w->size(1) != in || in <= 0 || in % 32 != 0 || out_features <= 0 ||
        out_features % 16 != 0 || x->stride(1) != 1 || x->stride(0) < in || x->stride(0) % 8 != 0 || !aligned16(*x) ||
        !aligned16(*w))
        Py_RETURN_NONE;
    if (bias && (bias->dim() != 1 || bias->size(0) != out_features || bias->scalar_type() != x->scalar_type() ||
                 !bias->is_contiguous() || bias->device() != x->device()))
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(*x, stream)) return nullptr;
    at::Tensor out = at::empty({rows, out_features}, x->options().requires_grad(false));
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.linear(out.data_ptr(), x->data_ptr(), w->data_ptr(), bias ? bias->data_ptr() : nullptr, rows, in,
                        out_features, x->stride(0), dtype_code(*x), stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_linear_rows", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// rope_slots(q, k, v, q_weight, k_weight, cos, sin, key_cache, value_cache, slot_mapping, eps): the
// rotated queries of the slot-mapping (prefill) form.
PyObject* rope_slots(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11 || !PyFloat_CheckExact(args[10])) Py_RETURN_NONE;
    const double eps = PyFloat_AS_DOUBLE(args[10]);
    const at::Tensor* t[10];
    for (int i = 0; i < 10; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &cos = *t[5], &sin = *t[6], &kc = *t[7], &vc = *t[8];
    if (!eager() || !on_current_device(q) || !half_type(q) || q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() ||
        kc.dim() != 4 || vc.sizes() != kc.sizes() || kc.numel() <= 0 || !kc.is_contiguous() || !vc.is_contiguous())
        Py_RETURN_NONE;
    // What the entry point and the library refuse as too small stays with the Python checks.
    const float eps32 = static_cast<float>(eps);
    if (!(eps32 > 0.f) || !(eps32 < HUGE_VALF)) Py_RETURN_NONE;
    const int64_t tokens = q.size(0), q_heads = q.size(1), d = q.size(2), kv_heads = k.size(1);
    if (tokens <= 0 || k.size(0) != tokens || k.size(2) != d || kv_heads <= 0 || q_heads < kv_heads ||
        q_heads % kv_heads != 0 || d % 2 != 0 || d <= 0 || d > 512 || kc.size(2) != kv_heads || kc.size(3) != d)
        Py_RETURN_NONE;
    for (int i = 1; i < 10; ++i) {
        if (t[i]->device() != q.device()) Py_RETURN_NONE;
        if (i < 9 && t[i]->scalar_type() != q.scalar_type()) Py_RETURN_NONE;
    }
    for (int i = 3; i < 5; ++i)
        if (t[i]->dim() != 1 || t[i]->size(0) != d || !t[i]->is_contiguous()) Py_RETURN_NONE;
    if (cos.dim() != 2 || sin.sizes() != cos.sizes() || cos.size(0) != tokens || cos.size(1) * 2 != d ||
        !cos.is_contiguous() || !sin.is_contiguous())
        Py_RETURN_NONE;
    const at::Tensor& slots = *t[9];
    if (slots.dim() != 1 || slots.size(0) != tokens || slots.scalar_type() != at::kLong || !slots.is_contiguous())
        Py_RETURN_NONE;
    const int64_t qs = row_stride(q), ks = row_stride(k), vs = row_stride(v);
    if (qs < 0 || ks < 0 || vs < 0) Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.rope(out.data_ptr(), kc.data_ptr(), vc.data_ptr(), kc.size(0), kc.size(1), kv_heads, d,
                      static_cast<const int64_t*>(slots.data_ptr()), nullptr, 0, nullptr, q.data_ptr(), k.data_ptr(),
                      v.data_ptr(), qs, ks, vs, t[3]->data_ptr(), t[4]->data_ptr(), cos.data_ptr(), sin.data_ptr(),
                      tokens, q_heads, eps32, dtype_code(q), stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_qk_norm_rope_write_kv", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// The packed 4-bit cache and the page operators.
// ---------------------------------------------------------------------------
// What the entry points ask of a packed layer's caches.
bool packed_caches(const at::Tensor& k, const at::Tensor& v, int64_t block, int64_t dim) {
    if (k.dim() != 3 || v.sizes() != k.sizes() || k.numel() <= 0 || k.scalar_type() != at::kByte ||
        v.scalar_type() != at::kByte || !k.is_contiguous() || !v.is_contiguous() || v.device() != k.device() ||
        !aligned16(k) || !aligned16(v))
        return false;
    const int64_t record = lib.fp4_record(block, dim);
    return record > 0 && k.size(2) == record;
}

bool index_list(const at::Tensor& t, const at::Tensor& beside) {
    return t.scalar_type() == at::kLong && t.is_contiguous() && t.device() == beside.device();
}
const int64_t* indices(const at::Tensor& t) { return static_cast<const int64_t*>(t.data_ptr()); }

// fp4_decode(query, key_cache, value_cache, block_tables, context_lens, block_size, partition_tokens)
PyObject* fp4_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, partition = 0;
    if (n != 7 || !as_int(args[5], block) || !as_int(args[6], partition)) Py_RETURN_NONE;
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &tables = *t[3], &lens = *t[4];
    if (!eager() || !on_current_device(q) || q.dim() != 3 || !half_type(q) || !q.is_contiguous() || q.numel() <= 0 ||
        !aligned16(q) || k.device() != q.device() || !packed_caches(k, v, block, q.size(2)) || partition < 0)
        Py_RETURN_NONE;
    const int64_t batch = q.size(0), q_heads = q.size(1), kv_heads = k.size(1), d = q.size(2);
    if (q_heads % kv_heads != 0 || (d != 32 && d != 64 && d != 96 && d != 128 && d != 192 && d != 256)) Py_RETURN_NONE;
    if (tables.dim() != 2 || tables.size(0) != batch || tables.size(1) <= 0 || tables.size(1) > kMaxCapacity / block ||
        lens.dim() != 1 || lens.size(0) != batch || !index_list(tables, q) || !index_list(lens, q))
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const size_t need = lib.fp4_decode_workspace(batch, q_heads, kv_heads, d, block, tables.size(1), partition);
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.fp4_decode(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), indices(tables), indices(lens),
                            batch, q_heads, kv_heads, d, k.size(0), block, tables.size(1), partition, dtype_code(q), ws,
                            need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_fp4_paged_attention", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// fp4_prefill(q, key_cache, value_cache, cu_seqlens_q, query_starts, block_tables, context_lens, block_size, chunk_tokens)
PyObject* fp4_prefill(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, chunk = 0;
    if (n != 9 || !as_int(args[7], block) || !as_int(args[8], chunk)) Py_RETURN_NONE;
    const at::Tensor* t[7];
    for (int i = 0; i < 7; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &cu = *t[3], &starts = *t[4], &tables = *t[5], &lens = *t[6];
    if (!eager() || !on_current_device(q) || q.dim() != 3 || !half_type(q) || !q.is_contiguous() || q.numel() <= 0 ||
        !aligned16(q) || k.device() != q.device() || !packed_caches(k, v, block, q.size(2)) || chunk < 0)
        Py_RETURN_NONE;
    const int64_t tokens = q.size(0), q_heads = q.size(1), kv_heads = k.size(1), d = q.size(2);
    if (q_heads % kv_heads != 0 || (d != 32 && d != 64 && d != 96 && d != 128 && d != 192 && d != 256)) Py_RETURN_NONE;
    if (cu.dim() != 1 || starts.dim() != 1 || lens.dim() != 1 || tables.dim() != 2) Py_RETURN_NONE;
    const int64_t seqs = starts.size(0), width = tables.size(1);
    if (seqs <= 0 || tables.size(0) != seqs || lens.size(0) != seqs || cu.size(0) != seqs + 1 || width <= 0 ||
        width > kMaxCapacity / block)
        Py_RETURN_NONE;
    for (int i = 3; i < 7; ++i)
        if (!index_list(*t[i], q)) Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const size_t need = lib.fp4_prefill_workspace(seqs, tokens, q_heads, kv_heads, d, block, width, chunk);
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.fp4_prefill(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), indices(cu), indices(starts),
                             indices(tables), indices(lens), seqs, tokens, q_heads, kv_heads, d, k.size(0), block, width,
                             chunk, dtype_code(q), ws, need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_fp4_paged_prefill_attention", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// Rows [tokens, kv_heads, head_dim] for a packed cache, and their token strides.
bool packed_rows(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& key, const at::Tensor& value,
                 int64_t block, int64_t& key_stride, int64_t& value_stride) {
    if (!eager() || !on_current_device(kc) || key.dim() != 3 || value.sizes() != key.sizes() || !half_type(key) ||
        value.scalar_type() != key.scalar_type() || key.device() != kc.device() || value.device() != kc.device() ||
        key.size(0) <= 0 || !packed_caches(kc, vc, block, key.size(2)) || key.size(1) != kc.size(1))
        return false;
    key_stride = row_stride(key);
    value_stride = row_stride(value);
    return key_stride >= 0 && value_stride >= 0;
}

// fp4_write_slots(key_cache, value_cache, slot_mapping, key, value, block_size): True when the rows were written.
PyObject* fp4_write_slots(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, ks = 0, vs = 0;
    if (n != 6 || !as_int(args[5], block)) Py_RETURN_NONE;
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &kc = *t[0], &vc = *t[1], &slots = *t[2], &key = *t[3], &value = *t[4];
    if (!packed_rows(kc, vc, key, value, block, ks, vs) || slots.dim() != 1 || slots.size(0) != key.size(0) ||
        !index_list(slots, kc))
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(kc, stream)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.fp4_write_slots(kc.data_ptr(), vc.data_ptr(), kc.size(0), block, kc.size(1), key.size(2),
                                 indices(slots), key.data_ptr(), value.data_ptr(), key.size(0), ks, vs, dtype_code(key),
                                 stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_fp4_write_slots", status);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// fp4_write_batch(key_cache, value_cache, block_tables, token_offsets, key, value, block_size): True when written.
PyObject* fp4_write_batch(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, ks = 0, vs = 0;
    if (n != 7 || !as_int(args[6], block)) Py_RETURN_NONE;
    const at::Tensor* t[6];
    for (int i = 0; i < 6; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &kc = *t[0], &vc = *t[1], &tables = *t[2], &offsets = *t[3], &key = *t[4], &value = *t[5];
    if (!packed_rows(kc, vc, key, value, block, ks, vs) || tables.dim() != 2 || tables.size(0) != key.size(0) ||
        tables.size(1) <= 0 || offsets.dim() != 1 || offsets.size(0) != key.size(0) || !index_list(tables, kc) ||
        !index_list(offsets, kc))
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(kc, stream)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.fp4_write_batch(kc.data_ptr(), vc.data_ptr(), kc.size(0), block, kc.size(1), key.size(2),
                                 indices(tables), tables.size(1), indices(offsets), key.data_ptr(), value.data_ptr(),
                                 key.size(0), ks, vs, dtype_code(key), stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_fp4_write_batch", status);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// fp4_gather_slots(key_cache, value_cache, slot_mapping, block_size, head_dim, dtype): (key, value) rows.
PyObject* fp4_gather_slots(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, dim = 0;
    if (n != 6 || !as_int(args[3], block) || !as_int(args[4], dim) || !THPDtype_Check(args[5])) Py_RETURN_NONE;
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    const at::Tensor* t[3];
    for (int i = 0; i < 3; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &kc = *t[0], &vc = *t[1], &slots = *t[2];
    if ((type != at::kHalf && type != at::kBFloat16) || !eager() || !on_current_device(kc) ||
        !packed_caches(kc, vc, block, dim) || slots.dim() != 1 || slots.size(0) <= 0 || !index_list(slots, kc))
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(kc, stream)) return nullptr;
    const int64_t tokens = slots.size(0), heads = kc.size(1);
    at::Tensor rows = at::empty({2, tokens, heads, dim}, kc.options().dtype(type).requires_grad(false));
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.fp4_gather_slots(rows.data_ptr(), static_cast<char*>(rows.data_ptr()) + tokens * heads * dim * 2,
                                  kc.data_ptr(), vc.data_ptr(), kc.size(0), block, heads, dim, indices(slots), tokens,
                                  type == at::kHalf ? MVME_FP16 : MVME_BF16, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_fp4_gather_slots", status);
    PyObject* key = THPVariable_Wrap(rows.select(0, 0));
    PyObject* value = key ? THPVariable_Wrap(rows.select(0, 1)) : nullptr;
    PyObject* both = value ? PyTuple_Pack(2, key, value) : nullptr;
    Py_XDECREF(key);
    Py_XDECREF(value);
    return both;
    END_HANDLE_TH_ERRORS
}

// move_pages(cache, src_pages, dst_pages, block_tables or None, page_dim): True when the pages were moved.
PyObject* move_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t dim = 0;
    if (n != 5 || !as_int(args[4], dim)) Py_RETURN_NONE;
    const at::Tensor *cache = plain(args[0]), *src = plain(args[1]), *dst = plain(args[2]);
    const at::Tensor* tables = args[3] == Py_None ? nullptr : plain(args[3]);
    if (!cache || !src || !dst || (args[3] != Py_None && !tables) || !eager() || !on_current_device(*cache))
        Py_RETURN_NONE;
    if (dim < 0 || dim >= cache->dim() || !cache->is_contiguous() || cache->numel() <= 0) Py_RETURN_NONE;
    if (src->dim() != 1 || dst->sizes() != src->sizes() || src->size(0) <= 0 || src->size(0) > cache->size(dim) ||
        !index_list(*src, *cache) || !index_list(*dst, *cache) || (tables && !index_list(*tables, *cache)))
        Py_RETURN_NONE;
    int64_t planes = 1;
    for (int64_t i = 0; i < dim; ++i) planes *= cache->size(i);
    const int64_t pages = cache->size(dim);
    const int64_t bytes = cache->numel() / (planes * pages) * static_cast<int64_t>(cache->element_size());
    void* stream = nullptr;
    if (!stream_of(*cache, stream)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = tables ? lib.compact_pages(cache->data_ptr(), planes, pages, bytes, indices(*src), indices(*dst),
                                        src->size(0), static_cast<int64_t*>(tables->data_ptr()), tables->numel(), stream)
                    : lib.copy_pages(cache->data_ptr(), planes, pages, bytes, indices(*src), indices(*dst),
                                     src->size(0), stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status(tables ? "mvme_compact_pages" : "mvme_copy_pages", status);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Operators for long contexts.
// ---------------------------------------------------------------------------
// Whether the memory of two contiguous tensors meets.
bool meet(const at::Tensor& a, const at::Tensor& b) {
    const auto begin = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
    const auto end = [&](const at::Tensor& t) { return begin(t) + t.numel() * t.element_size(); };
    return a.numel() > 0 && b.numel() > 0 && begin(a) < end(b) && begin(b) < end(a);
}

// fp32 [lines..., at least `capacity`], beside a tensor.
bool weight_rows(const at::Tensor& w, const at::Tensor& beside, int64_t capacity) {
    return w.scalar_type() == at::kFloat && w.is_contiguous() && w.device() == beside.device() &&
           w.size(w.dim() - 1) >= capacity;
}

// A decode call's plain arguments whose caches the operators of this part take.
bool long_decode(const at::Tensor* const* t, int64_t block, DecodeShape& s) {
    return eager() && on_current_device(*t[0]) && decode_shape(*t[0], *t[1], *t[2], *t[3], *t[4], block, s) &&
           t[0]->is_contiguous() && aligned16(*t[0]) && aligned16(*t[1]) && aligned16(*t[2]);
}

// shared_prefix(query, key_cache, value_cache, block_tables, context_lens, block_size, group_offsets, prefix_lens)
PyObject* shared_prefix(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0;
    if (n != 8 || !as_int(args[5], block)) Py_RETURN_NONE;
    const at::Tensor* t[8] = {};
    for (int i = 0; i < 8; ++i)
        if (i != 5 && !(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &offsets = *t[6], &prefixes = *t[7];
    DecodeShape s;
    if (!long_decode(t, block, s)) Py_RETURN_NONE;
    if (offsets.dim() != 1 || prefixes.dim() != 1 || offsets.size(0) != prefixes.size(0) + 1 || prefixes.size(0) > s.batch ||
        !index_list(offsets, q) || !index_list(prefixes, q))
        Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const int64_t groups = prefixes.size(0);
    const size_t need = lib.shared_workspace(s.batch, s.q_heads, s.kv_heads, s.head_dim, groups, block, s.width, 0);
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.shared_prefix(out.data_ptr(), q.data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), indices(*t[3]),
                               indices(*t[4]), indices(offsets), indices(prefixes), s.batch, groups, s.q_heads, s.kv_heads,
                               s.head_dim, s.num_blocks, block, s.width, 0, dtype_code(q), ws, need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_paged_attention_shared_prefix", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// decode_weights(query, key_cache, value_cache, block_tables, context_lens, block_size, weights)
PyObject* decode_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0;
    if (n != 7 || !as_int(args[5], block)) Py_RETURN_NONE;
    const at::Tensor* t[7] = {};
    for (int i = 0; i < 7; ++i)
        if (i != 5 && !(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &w = *t[6];
    DecodeShape s;
    if (!long_decode(t, block, s)) Py_RETURN_NONE;
    if (w.dim() != 3 || w.size(0) != s.batch || w.size(1) != s.kv_heads || !weight_rows(w, q, s.width * block)) Py_RETURN_NONE;
    for (int i = 0; i < 5; ++i)
        if (meet(w, *t[i])) Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    const size_t need = lib.weights_workspace(s.batch, s.q_heads, s.kv_heads, s.head_dim, block, s.width);
    at::Tensor workspace;
    if (need) workspace = bytes_like(q, need);
    void* ws = need ? workspace.data_ptr() : nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.decode_weights(out.data_ptr(), q.data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), indices(*t[3]),
                                indices(*t[4]), static_cast<float*>(w.data_ptr()), w.size(2), s.batch, s.q_heads,
                                s.kv_heads, s.head_dim, s.num_blocks, block, s.width, dtype_code(q), ws, need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_paged_attention_weights", status);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// prefill_weights(q, key_cache, cu_seqlens_q, query_starts, block_tables, context_lens, block_size, weights): True when
// the weights were added.
PyObject* prefill_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0;
    if (n != 8 || !as_int(args[6], block)) Py_RETURN_NONE;
    const at::Tensor* t[8] = {};
    for (int i = 0; i < 8; ++i)
        if (i != 6 && !(t[i] = plain(args[i]))) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &cu = *t[2], &starts = *t[3], &tables = *t[4], &lens = *t[5], &w = *t[7];
    if (!eager() || !on_current_device(q) || q.dim() != 3 || !half_type(q) || !q.is_contiguous() || q.numel() <= 0 ||
        !aligned16(q) || k.dim() != 4 || k.numel() <= 0 || k.device() != q.device() || k.scalar_type() != q.scalar_type() ||
        !k.is_contiguous() || !aligned16(k) || block <= 0 || block > kMaxCapacity || k.size(1) != block)
        Py_RETURN_NONE;
    const int64_t tokens = q.size(0), q_heads = q.size(1), d = q.size(2), kv_heads = k.size(2);
    if (k.size(3) != d || q_heads % kv_heads != 0) Py_RETURN_NONE;
    switch (d) {
        case 16: case 32: case 64: case 80: case 96: case 128: case 192: case 256: break;
        default: Py_RETURN_NONE;
    }
    if (cu.dim() != 1 || starts.dim() != 1 || lens.dim() != 1 || tables.dim() != 2) Py_RETURN_NONE;
    const int64_t seqs = starts.size(0), width = tables.size(1);
    if (seqs <= 0 || tables.size(0) != seqs || lens.size(0) != seqs || cu.size(0) != seqs + 1 || width <= 0 ||
        width > kMaxCapacity / block)
        Py_RETURN_NONE;
    for (int i = 2; i < 6; ++i)
        if (!index_list(*t[i], q)) Py_RETURN_NONE;
    if (w.dim() != 3 || w.size(0) != seqs || w.size(1) != kv_heads || !weight_rows(w, q, width * block)) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (meet(w, *t[i])) Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(q, stream)) return nullptr;
    const size_t need = lib.prefill_weights_workspace(seqs, tokens, q_heads, kv_heads, d, block, width);
    at::Tensor workspace = bytes_like(q, need);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.prefill_weights(q.data_ptr(), k.data_ptr(), indices(cu), indices(starts), indices(tables), indices(lens),
                                 static_cast<float*>(w.data_ptr()), w.size(2), seqs, tokens, q_heads, kv_heads, d,
                                 k.size(0), block, width, dtype_code(q), workspace.data_ptr(), need, stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_prefill_attention_weights", status);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// evict(key_cache, value_cache, weights, block_tables, context_lens, block_size, keep, first or None, recent): the three
// new tensors.
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t block = 0, keep = 0, recent = 0;
    if (n != 9 || !as_int(args[5], block) || !as_int(args[6], keep) || !as_int(args[8], recent)) Py_RETURN_NONE;
    const at::Tensor* t[6] = {};
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
    if (args[7] != Py_None && !(t[5] = plain(args[7]))) Py_RETURN_NONE;
    const at::Tensor &k = *t[0], &v = *t[1], &w = *t[2], &tables = *t[3], &lens = *t[4];
    if (!eager() || !on_current_device(k) || (k.dim() != 4 && k.dim() != 5) || v.sizes() != k.sizes() || k.numel() <= 0 ||
        !half_type(k) || v.scalar_type() != k.scalar_type() || v.device() != k.device() || !k.is_contiguous() ||
        !v.is_contiguous() || !aligned16(k) || !aligned16(v))
        Py_RETURN_NONE;
    const int64_t lead = k.dim() - 4, layers = lead ? k.size(0) : 1;
    const int64_t kv_heads = k.size(lead + 2), d = k.size(lead + 3);
    if (block <= 0 || block > kMaxCapacity || k.size(lead + 1) != block || d % 8 != 0 || d > 1024 || keep <= 0 || recent < 0)
        Py_RETURN_NONE;
    if (tables.dim() != 2 || lens.dim() != 1 || tables.size(0) <= 0 || tables.size(1) <= 0 || lens.size(0) != tables.size(0) ||
        tables.size(1) > kMaxCapacity / block || !index_list(tables, k) || !index_list(lens, k))
        Py_RETURN_NONE;
    const int64_t batch = tables.size(0), width = tables.size(1);
    if (t[5] && (t[5]->dim() != 1 || t[5]->size(0) != batch || !index_list(*t[5], k))) Py_RETURN_NONE;
    if (w.dim() != lead + 3 || (lead && w.size(0) != layers) || w.size(lead) != batch || w.size(lead + 1) != kv_heads ||
        !weight_rows(w, k, width * block) || meet(k, v))
        Py_RETURN_NONE;
    for (int i = 2; i < 6; ++i)
        if (t[i] && (meet(k, *t[i]) || meet(v, *t[i]))) Py_RETURN_NONE;
    void* stream = nullptr;
    if (!stream_of(k, stream)) return nullptr;
    const int64_t row = w.size(lead + 2), columns = keep < row ? keep : row;
    auto shape = w.sizes().vec();
    shape.back() = columns;
    at::Tensor kept = at::empty(shape, lens.options()), new_lens = at::empty(lens.sizes(), lens.options());
    at::Tensor new_weights = at::empty(w.sizes(), w.options().requires_grad(false));
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = lib.evict(k.data_ptr(), v.data_ptr(), static_cast<const float*>(w.data_ptr()),
                       static_cast<float*>(new_weights.data_ptr()), row, static_cast<int64_t*>(kept.data_ptr()),
                       static_cast<int64_t*>(new_lens.data_ptr()), indices(tables), indices(lens),
                       t[5] ? indices(*t[5]) : nullptr, layers, batch, kv_heads, d, k.size(lead), block, width, columns,
                       recent, dtype_code(k), stream);
    Py_END_ALLOW_THREADS
    if (status != MVME_OK) return raise_status("mvme_evict_kv_cache", status);
    PyObject* made[3] = {THPVariable_Wrap(std::move(kept)), THPVariable_Wrap(std::move(new_lens)),
                         THPVariable_Wrap(std::move(new_weights))};
    PyObject* all = made[0] && made[1] && made[2] ? PyTuple_Pack(3, made[0], made[1], made[2]) : nullptr;
    for (PyObject* o : made) Py_XDECREF(o);
    return all;
    END_HANDLE_TH_ERRORS
}

// bind(raw_stream_getter, (address, ...)): the library's entry points in the order of Library.
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *getter = nullptr, *addresses = nullptr;
    if (!PyArg_ParseTuple(args, "OO!", &getter, &PyTuple_Type, &addresses)) return nullptr;
    constexpr Py_ssize_t kCount = sizeof(Library) / sizeof(void*);
    if (PyTuple_GET_SIZE(addresses) != kCount) {
        PyErr_SetString(PyExc_ValueError, "wrong number of entry points");
        return nullptr;
    }
    void* found[kCount];
    for (Py_ssize_t i = 0; i < kCount; ++i) {
        found[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i));
        if (PyErr_Occurred()) return nullptr;
        if (!found[i]) {
            PyErr_SetString(PyExc_ValueError, "null entry point");
            return nullptr;
        }
    }
    static_assert(sizeof(Library) == sizeof(found), "one address per member");
    memcpy(&lib, found, sizeof(lib));
    Py_INCREF(getter);
    Py_XSETREF(current_raw_stream, getter);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(decode), METH_FASTCALL, nullptr},
    {"decode_write", reinterpret_cast<PyCFunction>(decode_write), METH_FASTCALL, nullptr},
    {"prefill", reinterpret_cast<PyCFunction>(prefill), METH_FASTCALL, nullptr},
    {"dense", reinterpret_cast<PyCFunction>(dense), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(linear), METH_FASTCALL, nullptr},
    {"rope_slots", reinterpret_cast<PyCFunction>(rope_slots), METH_FASTCALL, nullptr},
    {"write_slots", reinterpret_cast<PyCFunction>(write_slots), METH_FASTCALL, nullptr},
    {"fp4_decode", reinterpret_cast<PyCFunction>(fp4_decode), METH_FASTCALL, nullptr},
    {"fp4_prefill", reinterpret_cast<PyCFunction>(fp4_prefill), METH_FASTCALL, nullptr},
    {"fp4_write_slots", reinterpret_cast<PyCFunction>(fp4_write_slots), METH_FASTCALL, nullptr},
    {"fp4_write_batch", reinterpret_cast<PyCFunction>(fp4_write_batch), METH_FASTCALL, nullptr},
    {"fp4_gather_slots", reinterpret_cast<PyCFunction>(fp4_gather_slots), METH_FASTCALL, nullptr},
    {"move_pages", reinterpret_cast<PyCFunction>(move_pages), METH_FASTCALL, nullptr},
    {"shared_prefix", reinterpret_cast<PyCFunction>(shared_prefix), METH_FASTCALL, nullptr},
    {"decode_weights", reinterpret_cast<PyCFunction>(decode_weights), METH_FASTCALL, nullptr},
    {"prefill_weights", reinterpret_cast<PyCFunction>(prefill_weights), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(evict), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "mvme_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mvme_host(void) { return PyModule_Create(&module); }
