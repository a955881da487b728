// Python entry points of the ops that run between the launches of a decode loop (attn_prompt, kv4_*, token_logprobs): their
// argument checks and the call into librptc_hip.so in one step.  A small call of these is bound by the host: with
// the checks in Python and the call through ctypes attn_prompt took 12.0 us of host time and token_logprobs 5.9; now all six
// take 2.9 to 3.2, nearly all of it the launch.
// rptc_kernels/__init__.py holds the documented functions; it hands over the addresses of the library it loaded.
#include <cmath>
#include <cstring>
#include <string>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/rptc_hip.h"

namespace {

struct {
    decltype(&rptc_status_string) status_string;
    decltype(&rptc_attn_prompt_workspace_bytes) attn_prompt_workspace_bytes;
    decltype(&rptc_attn_prompt) attn_prompt;
    decltype(&rptc_kv4_append) kv4_append;
    decltype(&rptc_kv4_read) kv4_read;
    decltype(&rptc_kv4_rope_append) kv4_rope_append;
    decltype(&rptc_kv4_attn_decode_workspace_bytes) kv4_attn_decode_workspace_bytes;
    decltype(&rptc_kv4_attn_decode) kv4_attn_decode;
    decltype(&rptc_token_logprobs) token_logprobs;
} api;
constexpr int kFunctions = 9;
static_assert(sizeof(api) == kFunctions * sizeof(void *), "setup() fills it in this order");
PyObject *raw_stream;                       // device index -> the current stream's handle

[[noreturn]] void refuse(const std::string &message) { throw std::runtime_error(message); }

void require(bool ok, const char *message)
{
    if (__builtin_expect(!ok, 0)) refuse(message);
}

void status(int rc)
{
    if (rc) refuse("rptc_kernels: " + std::string(api.status_string(rc)) + " (status " + std::to_string(rc) + ")");
}

const at::Tensor &tensor(PyObject *o, const char *name)
{
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a torch.Tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
    return t;
}

void same_device(const at::Tensor &t, const at::Device &device) { require(t.device() == device, "all tensors must be on the same device"); }

const at::Tensor &contiguous(PyObject *o, const char *name)
{
    const at::Tensor &t = tensor(o, name);
    if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
    return t;
}

const char *type_name(at::ScalarType type)
{
    switch (type) {
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kFloat: return "float32";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    default: return "another type";
    }
}

// [tokens, heads, hd], any token and head strides, the head dimension contiguous
struct Rows {
    uint16_t *p;
    int64_t n, heads, hd, token, head;
};

Rows rows_of(PyObject *o, const char *name, at::ScalarType type, const at::Device *device)
{
    const at::Tensor &t = tensor(o, name);
    if (t.dim() != 3) refuse(std::string(name) + ".dim() == 3 ([tokens, heads, head_dim])");
    if (t.scalar_type() != type) refuse(std::string(name) + " must be " + type_name(type));
    if (device) same_device(t, *device);
    if (t.stride(2) != 1) refuse(std::string(name) + " must be contiguous along the head dimension");
    Rows r = {static_cast<uint16_t *>(t.data_ptr()), t.size(0), t.size(1), t.size(2), t.stride(0), t.stride(1)};
    // the stride of a dimension of one element means nothing: any valid one will do
    if (r.n <= 1) r.token = r.hd;
    if (r.heads <= 1) r.head = r.hd;
    return r;
}

bool alike(const Rows &a, const Rows &b) { return a.n == b.n && a.heads == b.heads && a.hd == b.hd; }

void *vector_of(PyObject *o, const char *name, at::ScalarType type, int64_t count, const at::Device &device)
{
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != count)
        refuse(std::string(name) + " must be a 1-D " + type_name(type) + " tensor of " + std::to_string(count) + " elements");
    if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
    same_device(t, device);
    return t.data_ptr();
}

float scale_of(PyObject *o, int64_t hd)
{
    if (o == Py_None) return (float)std::pow((double)hd, -0.5);
    const double s = PyFloat_AsDouble(o);
    if (s == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)s;
}

bool truth(PyObject *o)
{
    const int t = PyObject_IsTrue(o);
    if (t < 0) throw python_error();
    return t != 0;
}

// fn(stream, ms) on the device's current stream; elapsed ms (0.0 when not timed)
template <class F>
PyObject *run_on(const at::Device &device, bool timed, F fn)
{
    PyObject *index = PyLong_FromLong(device.index());
    if (!index) throw python_error();
    PyObject *handle = PyObject_CallFunctionObjArgs(raw_stream, index, nullptr);
    Py_DECREF(index);
    if (!handle) throw python_error();
    void *stream = PyLong_AsVoidPtr(handle);
    Py_DECREF(handle);
    if (!stream && PyErr_Occurred()) throw python_error();
    float ms = 0.f;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(stream, timed ? &ms : nullptr);
    Py_END_ALLOW_THREADS
    status(rc);
    return PyFloat_FromDouble(ms);
}

// An op's workspace from torch's allocator, so it is this call's own on the current stream and in a graph being captured.
struct Workspace {
    at::Tensor t;
    void *p = nullptr;
    int64_t bytes;
    Workspace(int64_t need, const at::Device &device) : bytes(need)
    {
        if (need < 0) status((int)need);
        if (need == 0) return;
        t = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(device));
        p = t.data_ptr();
    }
};

PyObject *zero() { return PyFloat_FromDouble(0.0); }

void expect(Py_ssize_t got, Py_ssize_t want)
{
    if (got != want) refuse("wrong number of arguments");
}

PyObject *attn_prompt(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 12);
    PyObject *const *a = args;              // q k v out q_start k_start k_len causal scale lse max_k timed
    const at::ScalarType type = THPVariable_Check(a[0]) ? THPVariable_Unpack(a[0]).scalar_type() : at::kFloat;
    require(type == at::kHalf || type == at::kBFloat16, "q must be an fp16 or bf16 tensor");
    const Rows q = rows_of(a[0], "q", type, nullptr);
    const at::Device device = THPVariable_Unpack(a[0]).device();
    const Rows k = rows_of(a[1], "k", type, &device), v = rows_of(a[2], "v", type, &device), out = rows_of(a[3], "out", type, &device);
    require(alike(out, q), "out.shape == q.shape");
    require(alike(v, k) && k.hd == q.hd, "v.shape == k.shape, k.size(2) == q.size(2)");
    require(q.hd == 32 || q.hd == 64 || q.hd == 128 || q.hd == 256, "the head dimension must be 32, 64, 128 or 256");
    require(k.heads >= 1 && q.heads >= 1 && q.heads % k.heads == 0, "heads must be a multiple of kv_heads");
    int64_t seqs = 1;
    const int32_t *q_start = nullptr, *k_start = nullptr, *k_len = nullptr;
    if (a[4] != Py_None) {
        seqs = THPVariable_Check(a[4]) ? THPVariable_Unpack(a[4]).numel() - 1 : 0;
        require(seqs >= 1, "q_start must hold at least two entries");
        q_start = static_cast<const int32_t *>(vector_of(a[4], "q_start", at::kInt, seqs + 1, device));
    }
    require((a[5] == Py_None) == (a[6] == Py_None), "k_start and k_len go together");
    if (a[5] != Py_None) {
        k_start = static_cast<const int32_t *>(vector_of(a[5], "k_start", at::kInt, seqs, device));
        k_len = static_cast<const int32_t *>(vector_of(a[6], "k_len", at::kInt, seqs, device));
    } else {
        require(!q_start || k.n == q.n, "without k_start the keys lie as the queries do: k.size(0) == q.size(0)");
    }
    float *lse = nullptr;
    if (a[9] != Py_None) {
        const at::Tensor &t = contiguous(a[9], "lse");
        require(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == q.n && t.size(1) == q.heads, "lse must be float32 [Tq, heads]");
        same_device(t, device);
        lse = static_cast<float *>(t.data_ptr());
    }
    int64_t max_k = k.n;
    if (a[10] != Py_None) {
        max_k = PyLong_AsLongLong(a[10]);
        if (max_k == -1 && PyErr_Occurred()) throw python_error();
    }
    const bool causal = truth(a[7]), timed = truth(a[11]);
    const float scale = scale_of(a[8], q.hd);
    if (q.n == 0) return zero();
    const c10::DeviceGuard guard(device);
    const Workspace ws(api.attn_prompt_workspace_bytes(seqs, q.n, k.n, max_k, q.heads, k.heads, q.hd), device);
    const rptc_prompt_strides st = {q.token, q.head, k.token, k.head, v.token, v.head, out.token, out.head};
    return run_on(device, timed, [&](void *stream, float *ms) {
        return api.attn_prompt(q.p, k.p, v.p, out.p, lse, q_start, k_start, k_len, seqs, q.n, k.n, max_k, q.heads, k.heads, q.hd, &st, scale,
                               causal, type == at::kHalf ? RPTC_F16 : RPTC_BF16, ws.p, ws.bytes, stream, ms);
    });
    END_HANDLE_TH_ERRORS
}

// a pair of 4-bit caches
struct Caches {
    uint8_t *k, *v;
    int64_t seqs, kv_heads, max_len;
    at::Device device;
};

Caches caches_of(PyObject *ko, PyObject *vo, int64_t hd)
{
    const char *names[2] = {"k_cache", "v_cache"};
    PyObject *const os[2] = {ko, vo};
    for (int i = 0; i < 2; i++) {
        const at::Tensor &t = contiguous(os[i], names[i]);
        if (t.scalar_type() != at::kByte || t.dim() != 4) refuse(std::string(names[i]) + " must be uint8 [seqs, kv_heads, positions, row bytes]");
    }
    const at::Tensor &k = THPVariable_Unpack(ko), &v = THPVariable_Unpack(vo);
    require(k.sizes() == v.sizes() && k.device() == v.device(), "k_cache and v_cache must be alike");
    require(hd == 32 || hd == 64 || hd == 128 || hd == 256, "the head dimension must be 32, 64, 128 or 256");
    require(k.size(3) == hd / 2 + hd / 8, "the cache's rows must have kv4_row_bytes(head dimension) bytes");
    return {static_cast<uint8_t *>(k.data_ptr()), static_cast<uint8_t *>(v.data_ptr()), k.size(0), k.size(1), k.size(2), k.device()};
}

int64_t head_dim_of(PyObject *o, const char *message)
{
    require(THPVariable_Check(o) && THPVariable_Unpack(o).dim() == 3, message);
    return THPVariable_Unpack(o).size(2);
}

struct CacheRows {
    Caches c;
    Rows k, v;
};

CacheRows cache_rows(PyObject *ko, PyObject *vo, PyObject *kc, PyObject *vc)
{
    const int64_t hd = head_dim_of(ko, "k must be [tokens, kv_heads, head_dim]");
    const Caches c = caches_of(kc, vc, hd);
    const Rows k = rows_of(ko, "k", at::kHalf, &c.device), v = rows_of(vo, "v", at::kHalf, &c.device);
    require(alike(v, k), "v.shape == k.shape");
    require(k.heads == c.kv_heads, "the cache must have as many heads as k and v");
    return {c, k, v};
}

PyObject *kv4_append(PyObject *, PyObject *const *a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 7);                       // k v k_cache v_cache pos q_start timed
    const CacheRows r = cache_rows(a[0], a[1], a[2], a[3]);
    const Caches &c = r.c;
    const auto *pos = static_cast<const int64_t *>(vector_of(a[4], "pos", at::kLong, c.seqs, c.device));
    const int32_t *q_start = nullptr;
    if (a[5] != Py_None) q_start = static_cast<const int32_t *>(vector_of(a[5], "q_start", at::kInt, c.seqs + 1, c.device));
    else require(c.seqs >= 1 && r.k.n % c.seqs == 0, "without q_start the rows must divide evenly: k.size(0) % k_cache.size(0) == 0");
    const bool timed = truth(a[6]);
    if (r.k.n == 0 || c.max_len == 0) return zero();
    const c10::DeviceGuard guard(c.device);
    return run_on(c.device, timed, [&](void *stream, float *ms) {
        return api.kv4_append(r.k.p, r.v.p, c.k, c.v, pos, q_start, c.seqs, r.k.n, c.kv_heads, r.k.hd, c.max_len, r.k.token, r.k.head, r.v.token,
                              r.v.head, stream, ms);
    });
    END_HANDLE_TH_ERRORS
}

PyObject *kv4_read(PyObject *, PyObject *const *a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 5);                       // k_cache v_cache k v timed
    const CacheRows r = cache_rows(a[2], a[3], a[0], a[1]);
    const Caches &c = r.c;
    require(c.seqs >= 1 && r.k.n % c.seqs == 0 && r.k.n / c.seqs <= c.max_len,
            "k must hold the same number of rows for every sequence, at most the cache's positions");
    const bool timed = truth(a[4]);
    if (r.k.n == 0) return zero();
    require(r.k.token && r.k.head && r.v.token && r.v.head, "k and v must not repeat elements");
    const c10::DeviceGuard guard(c.device);
    return run_on(c.device, timed, [&](void *stream, float *ms) {
        return api.kv4_read(c.k, c.v, r.k.p, r.v.p, c.seqs, r.k.n / c.seqs, c.kv_heads, r.k.hd, c.max_len, r.k.token, r.k.head, r.v.token,
                            r.v.head, stream, ms);
    });
    END_HANDLE_TH_ERRORS
}

PyObject *kv4_rope_append(PyObject *, PyObject *const *a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 8);                       // qkv cos sin pos q_out k_cache v_cache timed
    const int order[4] = {0, 1, 2, 4};
    const char *names[4] = {"qkv", "cos", "sin", "q_out"};
    for (int i = 0; i < 4; i++)
        if (contiguous(a[order[i]], names[i]).scalar_type() != at::kHalf) refuse(std::string(names[i]) + " must be fp16");
    const at::Tensor &qkv = THPVariable_Unpack(a[0]), &cos = THPVariable_Unpack(a[1]), &sin = THPVariable_Unpack(a[2]), &q = THPVariable_Unpack(a[4]);
    require(q.dim() == 3 && qkv.dim() == 2, "q_out must be [seqs, heads, head_dim], qkv [seqs, (heads + 2 kv_heads) * head_dim]");
    const int64_t seqs = q.size(0), heads = q.size(1), hd = q.size(2);
    const Caches c = caches_of(a[5], a[6], hd);
    require(c.seqs == seqs && qkv.size(0) == seqs && qkv.size(1) == (heads + 2 * c.kv_heads) * hd,
            "qkv must be [seqs, (heads + 2 kv_heads) * head_dim], the caches hold as many sequences");
    require(c.kv_heads >= 1 && heads >= 1 && heads % c.kv_heads == 0, "heads must be a multiple of kv_heads");
    require(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(0) >= c.max_len && cos.size(1) == hd / 2,
            "cos and sin must be [positions, head_dim / 2] with as many positions as the cache");
    const auto *pos = static_cast<const int64_t *>(vector_of(a[3], "pos", at::kLong, seqs, c.device));
    same_device(qkv, c.device);
    same_device(cos, c.device);
    same_device(sin, c.device);
    same_device(q, c.device);
    const bool timed = truth(a[7]);
    if (seqs == 0 || c.max_len == 0) return zero();
    const c10::DeviceGuard guard(c.device);
    return run_on(c.device, timed, [&](void *stream, float *ms) {
        return api.kv4_rope_append(static_cast<const uint16_t *>(qkv.data_ptr()), static_cast<const uint16_t *>(cos.data_ptr()),
                                   static_cast<const uint16_t *>(sin.data_ptr()), pos, static_cast<uint16_t *>(q.data_ptr()), c.k, c.v, seqs,
                                   heads, c.kv_heads, hd, c.max_len, stream, ms);
    });
    END_HANDLE_TH_ERRORS
}

PyObject *kv4_attn_decode(PyObject *, PyObject *const *a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 7);                       // q k_cache v_cache pos out scale timed
    const int64_t hd = head_dim_of(a[0], "q must be [seqs, heads, head_dim]");
    const Caches c = caches_of(a[1], a[2], hd);
    const Rows q = rows_of(a[0], "q", at::kHalf, &c.device);
    require(q.head == hd, "q must have contiguous heads");
    const at::Tensor &out = contiguous(a[4], "out");
    require(out.scalar_type() == at::kHalf && out.dim() == 3 && out.size(0) == q.n && out.size(1) == q.heads && out.size(2) == hd &&
                out.device() == c.device, "out must be fp16, of the shape of q and on its device");
    require(c.seqs == q.n, "k_cache.size(0) == q.size(0)");
    require(c.kv_heads >= 1 && q.heads >= 1 && q.heads % c.kv_heads == 0, "heads must be a multiple of kv_heads");
    const auto *pos = static_cast<const int64_t *>(vector_of(a[3], "pos", at::kLong, q.n, c.device));
    const float scale = scale_of(a[5], hd);
    const bool timed = truth(a[6]);
    if (q.n == 0 || c.max_len == 0) return zero();
    const c10::DeviceGuard guard(c.device);
    const Workspace ws(api.kv4_attn_decode_workspace_bytes(q.n, q.heads, c.kv_heads, hd, c.max_len), c.device);
    return run_on(c.device, timed, [&](void *stream, float *ms) {
        return api.kv4_attn_decode(q.p, c.k, c.v, pos, static_cast<uint16_t *>(out.data_ptr()), q.n, q.heads, c.kv_heads, hd, c.max_len, q.token,
                                   scale, ws.p, ws.bytes, stream, ms);
    });
    END_HANDLE_TH_ERRORS
}

PyObject *token_logprobs(PyObject *, PyObject *const *a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 7);                       // logits tokens logprob entropy top_ids top_logprobs timed
    const at::Tensor &x = tensor(a[0], "logits");
    const at::ScalarType type = x.scalar_type();
    require(x.dim() == 2 && (type == at::kHalf || type == at::kBFloat16 || type == at::kFloat), "logits must be fp16, bf16 or float32 [rows, vocab]");
    const int64_t rows = x.size(0), vocab = x.size(1);
    require(vocab >= 1, "the vocabulary must not be empty");
    require(vocab == 1 || x.stride(1) == 1, "logits must be contiguous along the vocabulary");
    require(a[2] != Py_None || a[3] != Py_None || a[4] != Py_None || a[5] != Py_None, "at least one output is needed");
    require(a[2] == Py_None || a[1] != Py_None, "logprob needs tokens");
    const at::Device device = x.device();
    const int64_t *tokens = nullptr;
    float *logprob = nullptr, *entropy = nullptr, *top_logprobs = nullptr;
    int64_t *top_ids = nullptr, top = 0;
    if (a[1] != Py_None) tokens = static_cast<const int64_t *>(vector_of(a[1], "tokens", at::kLong, rows, device));
    if (a[2] != Py_None) logprob = static_cast<float *>(vector_of(a[2], "logprob", at::kFloat, rows, device));
    if (a[3] != Py_None) entropy = static_cast<float *>(vector_of(a[3], "entropy", at::kFloat, rows, device));
    for (int i = 4; i < 6; i++) {
        if (a[i] == Py_None) continue;
        const char *name = i == 4 ? "top_ids" : "top_logprobs";
        const at::ScalarType want = i == 4 ? at::kLong : at::kFloat;
        const at::Tensor &t = contiguous(a[i], name);
        if (t.scalar_type() != want || t.dim() != 2 || t.size(0) != rows) refuse(std::string(name) + " must be " + type_name(want) + " [rows, k]");
        same_device(t, device);
        require(top == 0 || top == t.size(1), "top_ids and top_logprobs must have the same shape");
        top = t.size(1);
        require(top >= 1 && top <= 64 && top <= vocab, "1 <= k <= 64, k <= vocabulary");
        if (i == 4) top_ids = static_cast<int64_t *>(t.data_ptr());
        else top_logprobs = static_cast<float *>(t.data_ptr());
    }
    const bool timed = truth(a[6]);
    if (rows == 0) return zero();
    const c10::DeviceGuard guard(device);
    return run_on(device, timed, [&](void *stream, float *ms) {
        return api.token_logprobs(x.data_ptr(), type == at::kHalf ? RPTC_F16 : type == at::kBFloat16 ? RPTC_BF16 : RPTC_F32, tokens, logprob, entropy,
                                  top_ids, top_logprobs, rows, vocab, rows > 1 ? x.stride(0) : vocab, top, stream, ms);
    });
    END_HANDLE_TH_ERRORS
}

// setup(addresses of the library's functions in the order of `api`, the function that names a device's current stream)
PyObject *setup(PyObject *, PyObject *const *a, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    expect(count, 2);
    require(PyTuple_Check(a[0]) && PyTuple_GET_SIZE(a[0]) == kFunctions && PyCallable_Check(a[1]), "setup(addresses, raw_stream)");
    void *p[kFunctions];
    for (int i = 0; i < kFunctions; i++) {
        p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i));
        if (!p[i]) {
            if (PyErr_Occurred()) throw python_error();
            refuse("a function of the library has no address");
        }
    }
    memcpy(&api, p, sizeof(api));
    Py_INCREF(a[1]);
    Py_XDECREF(raw_stream);
    raw_stream = a[1];
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define RPTC_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {RPTC_METHOD(setup), RPTC_METHOD(attn_prompt), RPTC_METHOD(kv4_append), RPTC_METHOD(kv4_read), RPTC_METHOD(kv4_rope_append),
                         RPTC_METHOD(kv4_attn_decode), RPTC_METHOD(token_logprobs), {nullptr, nullptr, 0, nullptr}};
#undef RPTC_METHOD
PyModuleDef module = {PyModuleDef_HEAD_INIT, "rptc_bindings", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_rptc_bindings(void) { return PyModule_Create(&module); }
