// Native call sites of the rotary, 4-bit cache and scoring operators (rotary.py, kv4.py, scores.py): argument checks, outputs,
// workspaces, the current stream and the autograd nodes in one native call.  Done in Python - a dozen checks, torch.empty, ctypes with
// some twenty arguments, a Python autograd node - the host side of a call took 27 - 41 us (177 us with its gradient).
//
// Wrong arguments raise ValueError, CPU tensors and failed launches RuntimeError, tensors with a forward-mode tangent NotImplementedError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <limits.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ternaspmm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return 0;
        case at::kHalf: return 1;
        case at::kFloat: return 2;
        default: return -1;
    }
}

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// (no call has a forward-mode derivative: a tangent that it dropped would count as zero)
const Tensor& tensor_arg(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " is a tensor, not ", Py_TYPE(o)->tp_name);
    const Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name, " has a tangent: no forward-mode derivative here");
    return t;
}
// One that the calls treat as given: tables and caches have no gradient, and one that is asked for is not dropped silently.
const Tensor& constant_arg(PyObject* o, const char* name) {
    const Tensor& t = tensor_arg(o, name);
    TORCH_CHECK(!wants_grad(t), name, " requires a gradient: the calls have none for it");
    return t;
}
OptTensor optional_constant(PyObject* o, const char* name) { return o == Py_None ? OptTensor() : OptTensor(constant_arg(o, name)); }
OptTensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? OptTensor() : OptTensor(tensor_arg(o, name)); }

long long int_arg(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    (void)name;
    return v;
}

void on_gpu(const Tensor& t, const char* what) { TORCH_CHECK(t.is_cuda(), what, " needs CUDA tensors: the B200 library has no CPU path"); }

void launched(int status, const char* what) {
    TORCH_CHECK_VALUE(status != 1 && status != 2, what, status == 1 ? ": more than a launch takes" : ": pointers off their boundaries");
    TORCH_CHECK(status == 0, what, ": status ", status);
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
template <typename T> T* as(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T> T* as(const OptTensor& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

// (a dimension of one element has no stride: what torch keeps there can be any number)
int64_t stride_of(const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; }
struct Strides {
    long long v[3];
    explicit Strides(const Tensor& t) : v{stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)} {}
};

// What a kernel reads is memory: a tensor that torch marks as the negative of its memory (imaginary parts of conjugates, as gradients come) is written out.
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// t with contiguous heads whose rows start on multiples of `bytes`
Tensor rows_on(const Tensor& given, int bytes) {
    const Tensor t = plain(given);
    const int64_t step = bytes / t.element_size();
    const bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0 && stride_of(t, 0) % step == 0 &&
                    stride_of(t, 1) % step == 0 && stride_of(t, 2) % step == 0;
    if (ok) return t;
    const Tensor r = t.contiguous();
    return r.data_ptr() == t.data_ptr() ? t.clone(at::MemoryFormat::Contiguous) : r;   // (contiguous, but off the boundary)
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const OptTensor& t) {
    if (t && t->defined()) return THPVariable_Wrap(*t);
    Py_RETURN_NONE;
}

// ---------------------------------------------------------------------------------------------------- rotate

struct RotaryArgs {
    Tensor cos, sin, positions;
    bool half, inverse;
};

variable_list rotate_launch(Tensor q, OptTensor k, const RotaryArgs& r) {
    const c10::cuda::CUDAGuard guard(q.device());
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), K = k ? k->size(2) : 0;
    // whole pairs start on their boundaries where pairs are neighbours
    q = rows_on(q, (r.half ? 1 : 2) * q.element_size());
    if (k) k = rows_on(*k, (r.half ? 1 : 2) * k->element_size());
    variable_list out = {at::empty({B, T, H, D}, q.options())};
    if (k) out.push_back(at::empty({B, T, K, D}, q.options()));
    if (B == 0 || T == 0 || H + K == 0 || D == 0) return out;
    TORCH_CHECK_VALUE(H > 0 && std::max({B, T, H, K}) <= INT_MAX, "rotate: sizes ", q.sizes());
    const Strides qs(q), ks(k ? *k : q);
    const bool shared = r.positions.dim() == 1;
    launched(ternaspmm_rotate(ptr(q), qs.v, (int)H, ptr(out[0]), ptr(k), ks.v, (int)K, k ? ptr(out[1]) : nullptr, type_code(q), as<float>(r.cos),
                              as<float>(r.sin), (int)r.cos.size(0), (int)r.cos.size(1) * 2, r.half, r.inverse, as<long long>(r.positions),
                              shared ? 0 : r.positions.stride(0), r.positions.stride(-1), (int)B, (int)T, (int)D,
                              c10::cuda::getCurrentCUDAStream().stream()),
             "ternaspmm_rotate");
    return out;
}

variable_list rotate_any(const Tensor& q, const OptTensor& k, const RotaryArgs& r);

struct Rotate : torch::autograd::Function<Rotate> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                                 bool half, bool inverse) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({cos, sin, positions});
        ctx->saved_data["half"] = half;
        ctx->saved_data["inverse"] = inverse;
        at::AutoDispatchBelowADInplaceOrView below;
        return rotate_launch(q, k, {cos, sin, positions, half, inverse});
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const RotaryArgs r = {saved[0], saved[1], saved[2], ctx->saved_data["half"].toBool(), !ctx->saved_data["inverse"].toBool()};
        variable_list out(7);
        const bool with_k = grads.size() > 1 && grads[1].defined() && ctx->needs_input_grad(1), with_q = grads[0].defined() && ctx->needs_input_grad(0);
        if (with_q) {              // (by the differentiable call: a second derivative is one more rotation)
            const variable_list g = rotate_any(grads[0], with_k ? OptTensor(grads[1]) : OptTensor(), r);
            out[0] = g[0];
            if (with_k) out[1] = g[1];
        } else if (with_k) {
            out[1] = rotate_any(grads[1], OptTensor(), r)[0];
        }
        return out;
    }
};

variable_list rotate_any(const Tensor& q, const OptTensor& k, const RotaryArgs& r) {
    if (wants_grad(q) || (k && wants_grad(*k))) return Rotate::apply(q, k, r.cos, r.sin, r.positions, r.half, r.inverse);
    return rotate_launch(q, k, r);
}

// rotate(q, k or None, cos, sin, half, positions)
PyObject* py_rotate(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 6, "rotate(q, k, cos, sin, half, positions)");
    const Tensor &q = tensor_arg(args[0], "q"), &cos = constant_arg(args[2], "cos"), &sin = constant_arg(args[3], "sin"), &pos = tensor_arg(args[5], "positions");
    const OptTensor k = optional_arg(args[1], "k");
    on_gpu(q, "rotate");
    TORCH_CHECK_VALUE(q.dim() == 4 && type_code(q) >= 0 && q.size(3) % 2 == 0, "q is bf16, fp16 or fp32 [B, T, H, D] with an even D, not ", q.scalar_type(), " ",
                      q.sizes());
    TORCH_CHECK_VALUE(!k || (k->dim() == 4 && k->scalar_type() == q.scalar_type() && k->device() == q.device() && k->size(0) == q.size(0) &&
                             k->size(1) == q.size(1) && k->size(3) == q.size(3)),
                      "k is ", q.scalar_type(), " [B, T, Hkv, D] beside q ", q.sizes(), ", not ", k ? k->scalar_type() : q.scalar_type(), " ", k ? k->sizes() : q.sizes());
    TORCH_CHECK_VALUE(pos.scalar_type() == at::kLong && pos.device() == q.device() &&
                          (pos.dim() == 1 ? pos.size(0) == q.size(1) : pos.dim() == 2 && pos.size(0) == q.size(0) && pos.size(1) == q.size(1)),
                      "positions are int64 [T] or [B, T] on ", q.device(), ", not ", pos.scalar_type(), " ", pos.sizes());
    TORCH_CHECK_VALUE(cos.size(1) * 2 <= q.size(3) && cos.device() == q.device() && cos.size(0) <= INT_MAX, "the table rotates ", cos.size(1) * 2, " values on ",
                      cos.device(), ", a head has ", q.size(3), " on ", q.device());
    const variable_list out = rotate_any(q, k, {cos, sin, pos, args[4] == Py_True, false});
    return Py_BuildValue("NN", wrap(out[0]), k ? wrap(out[1]) : wrap(OptTensor()));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------- 4-bit cache

// The tensors of a KV4Cache (checked when it was made), args[0 .. 3].
struct Cache {
    const Tensor &k_codes, &k_scales, &v_codes, &v_scales;
    int64_t batch, kv_heads, max_len, head_dim;
    explicit Cache(PyObject* const* args)
        : k_codes(tensor_arg(args[0], "k_codes")), k_scales(constant_arg(args[1], "k_scales")), v_codes(tensor_arg(args[2], "v_codes")),
          v_scales(constant_arg(args[3], "v_scales")), batch(k_codes.size(0)), kv_heads(k_codes.size(1)), max_len(k_codes.size(2)),
          head_dim(2 * k_codes.size(3)) {
        TORCH_CHECK_VALUE(std::max({batch, kv_heads, max_len}) <= INT_MAX, "cache of ", k_codes.sizes());
    }
};

void check_rows(const Cache& c, const char* name, const Tensor& x, int64_t heads) {
    on_gpu(x, name);
    TORCH_CHECK(!wants_grad(x), name, " requires a gradient: the 4-bit cache has none");
    TORCH_CHECK_VALUE(x.dim() == 4 && x.scalar_type() == at::kBFloat16 && x.device() == c.k_codes.device() && x.size(0) == c.batch && x.size(3) == c.head_dim &&
                          x.size(2) > 0 && x.size(1) <= INT_MAX && x.size(2) <= INT_MAX && (heads < 0 || x.size(2) == heads),
                      name, ": bf16 [", c.batch, ", T, ", heads < 0 ? std::string("heads") : std::to_string(heads), ", ", c.head_dim, "] on ", c.k_codes.device(),
                      " wanted, not ", x.scalar_type(), " ", x.sizes(), " on ", x.device());
}

void check_places(const Cache& c, const Tensor& start, const OptTensor& counts) {
    auto ok = [&](const Tensor& t, bool one) {
        return t.scalar_type() == at::kLong && t.dim() == 1 && (t.size(0) == c.batch || (one && t.size(0) == 1)) && t.is_contiguous() && t.device() == c.k_codes.device();
    };
    TORCH_CHECK_VALUE(ok(start, true), "start is contiguous int64 [", c.batch, "] or [1] on ", c.k_codes.device(), ", not ", start.scalar_type(), " ", start.sizes());
    TORCH_CHECK_VALUE(!counts || ok(*counts, false), "counts are contiguous int64 [", c.batch, "] on ", c.k_codes.device(), ", not ",
                      counts ? counts->scalar_type() : at::kLong, " ", counts ? counts->sizes() : start.sizes());
}

// kv4_append(cache x 4, k, v, start, counts, q, cos, sin, half)
PyObject* py_kv4_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 12, "kv4_append(k_codes, k_scales, v_codes, v_scales, k, v, start, counts, q, cos, sin, half)");
    const Cache c(args);
    const Tensor &k0 = tensor_arg(args[4], "k"), &v0 = tensor_arg(args[5], "v"), &start = tensor_arg(args[6], "start");
    const OptTensor counts = optional_arg(args[7], "counts"), q0 = optional_arg(args[8], "q"), cos = optional_constant(args[9], "cos"), sin = optional_constant(args[10], "sin");
    check_rows(c, "k", k0, c.kv_heads);
    check_rows(c, "v", v0, c.kv_heads);
    TORCH_CHECK_VALUE(v0.size(1) == k0.size(1), "k and v have one shape, not ", k0.sizes(), " and ", v0.sizes());
    check_places(c, start, counts);
    TORCH_CHECK_VALUE(!cos || (cos->size(1) * 2 <= c.head_dim && cos->device() == k0.device() && cos->size(0) <= INT_MAX), "the table rotates ",
                      cos ? cos->size(1) * 2 : 0, " values on ", cos ? cos->device() : k0.device(), ", a head has ", c.head_dim, " on ", k0.device());
    if (q0) {
        TORCH_CHECK_VALUE(cos, "queries are only passed to be rotated: table is missing");
        check_rows(c, "q", *q0, -1);
        TORCH_CHECK_VALUE(q0->size(1) == k0.size(1), q0->size(1), " queries beside ", k0.size(1), " keys");
    }
    const c10::cuda::CUDAGuard guard(k0.device());
    OptTensor out;
    if (q0) out = at::empty(q0->sizes(), q0->options());
    const int64_t T = k0.size(1);
    if (T) {
        const Tensor k = rows_on(k0, 8), v = rows_on(v0, 8), q = q0 ? rows_on(*q0, 8) : k;
        const Strides ks(k), vs(v), qs(q);
        launched(ternaspmm_kv4_append(ptr(c.k_codes), ptr(c.k_scales), ptr(c.v_codes), ptr(c.v_scales), (int)c.max_len, as<ternaspmm_bf16>(k), ks.v, as<ternaspmm_bf16>(v),
                                      vs.v, q0 ? as<ternaspmm_bf16>(q) : nullptr, qs.v, as<ternaspmm_bf16>(out), as<float>(cos), as<float>(sin),
                                      cos ? (int)cos->size(0) : 0, cos ? (int)cos->size(1) * 2 : 0, args[11] == Py_True, as<long long>(start), start.size(0) > 1,
                                      as<long long>(counts), (int)c.batch, (int)T, q0 ? (int)q.size(2) : 0, (int)c.kv_heads, (int)c.head_dim,
                                      c10::cuda::getCurrentCUDAStream().stream()),
                 "kv4_append");
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// kv4_read(cache x 4, start, tokens, counts)
PyObject* py_kv4_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 7, "kv4_read(k_codes, k_scales, v_codes, v_scales, start, tokens, counts)");
    const Cache c(args);
    const Tensor& start = tensor_arg(args[4], "start");
    const long long T = int_arg(args[5], "tokens");
    const OptTensor counts = optional_arg(args[6], "counts");
    TORCH_CHECK_VALUE(T >= 0 && T <= INT_MAX, T, " tokens");
    on_gpu(c.k_codes, "kv4_read");
    check_places(c, start, counts);
    const c10::cuda::CUDAGuard guard(c.k_codes.device());
    const auto options = c.k_codes.options().dtype(at::kBFloat16);
    const Tensor k = at::empty({c.batch, T, c.kv_heads, c.head_dim}, options), v = at::empty_like(k);
    if (T)
        launched(ternaspmm_kv4_read(ptr(c.k_codes), ptr(c.k_scales), ptr(c.v_codes), ptr(c.v_scales), (int)c.max_len, as<long long>(start), start.size(0) > 1,
                                    as<long long>(counts), as<ternaspmm_bf16>(k), as<ternaspmm_bf16>(v), (int)c.batch, (int)T, (int)c.kv_heads, (int)c.head_dim,
                                    c10::cuda::getCurrentCUDAStream().stream()),
                 "kv4_read");
    return Py_BuildValue("NN", wrap(k), wrap(v));
    END_HANDLE_TH_ERRORS
}

// kv4_attend(q, cache x 4, start, counts, window, scale or None)
PyObject* py_kv4_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 9, "kv4_attend(q, k_codes, k_scales, v_codes, v_scales, start, counts, window, scale)");
    const Tensor& q0 = tensor_arg(args[0], "q");
    const Cache c(args + 1);
    const Tensor& start = tensor_arg(args[5], "start");
    const OptTensor counts = optional_arg(args[6], "counts");
    const long long window = int_arg(args[7], "window");
    const double scale = args[8] == Py_None ? 1.0 / std::sqrt((double)c.head_dim) : PyFloat_AsDouble(args[8]);
    if (PyErr_Occurred()) throw python_error();
    check_rows(c, "q", q0, -1);
    check_places(c, start, counts);
    const int64_t B = c.batch, T = q0.size(1), H = q0.size(2);
    TORCH_CHECK_VALUE(H % c.kv_heads == 0, H, " query heads over ", c.kv_heads, " key heads");
    TORCH_CHECK_VALUE(window >= 0 && window <= INT_MAX && (float)scale > 0.f && scale <= 1e6, "window ", window, ", scale ", scale);
    const c10::cuda::CUDAGuard guard(q0.device());
    const Tensor out = at::empty(q0.sizes(), q0.options());
    if (T) {
        const Tensor q = rows_on(q0, 16);
        const long long need = ternaspmm_kv4_attend_workspace((int)B, (int)T, (int)H, (int)c.kv_heads, (int)c.head_dim, (int)c.max_len);
        TORCH_CHECK_VALUE(need >= 0, "kv4_attend: sizes ", q0.sizes(), " over a cache of ", c.max_len);
        OptTensor work;                // of this call alone: calls on other streams and captured graphs have their own
        if (need) work = at::empty({need}, q0.options().dtype(at::kByte));
        const Strides qs(q);
        launched(ternaspmm_kv4_attend(as<ternaspmm_bf16>(q), qs.v, ptr(c.k_codes), ptr(c.k_scales), ptr(c.v_codes), ptr(c.v_scales), (int)c.max_len,
                                      as<long long>(start), start.size(0) > 1, as<long long>(counts), (int)window, (float)scale, as<ternaspmm_bf16>(out), (int)B,
                                      (int)T, (int)H, (int)c.kv_heads, (int)c.head_dim, ptr(work), need, c10::cuda::getCurrentCUDAStream().stream()),
                 "kv4_attend");
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------- log probabilities

// Logits as rows [N, V] of contiguous elements, any distance apart.
Tensor logit_rows(const Tensor& given) {
    const Tensor x = plain(given);
    const int64_t V = x.size(-1);
    Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / V, V});
    return (V == 1 || r.stride(1) == 1) && (r.size(0) <= 1 || r.stride(0) >= V) ? r : r.contiguous();
}
long long row_step(const Tensor& rows) { return std::max<int64_t>(rows.stride(0), rows.size(1)); }

struct Scores {
    Tensor stats, top_logprob, top_token;
};

Scores scores_launch(const Tensor& logits, const Tensor& targets, int64_t top) {
    const c10::cuda::CUDAGuard guard(logits.device());
    Scores s;
    const Tensor rows = logit_rows(logits), ids = targets.reshape({-1}).contiguous();
    const int64_t N = rows.size(0), V = rows.size(1);
    TORCH_CHECK_VALUE(N <= INT_MAX && V <= INT_MAX, "logits of ", logits.sizes());
    s.stats = at::empty({4, N}, logits.options().dtype(at::kFloat));
    auto shape = targets.sizes().vec();
    shape.push_back(top);
    if (top) s.top_logprob = at::empty(shape, s.stats.options()), s.top_token = at::empty(shape, targets.options());
    float* stats = as<float>(s.stats);
    if (N) {
        const long long need = ternaspmm_token_logprobs_workspace((int)N, (int)V, type_code(logits), (int)top);
        TORCH_CHECK_VALUE(need >= 0, "token_logprobs: ", N, " rows of ", V, " logits (2^19 at most; 2^23 rows where a row is longer than 32 KB)");
        const Tensor work = at::empty({need}, logits.options().dtype(at::kByte));   // of this call alone
        launched(ternaspmm_token_logprobs(ptr(rows), row_step(rows), type_code(logits), as<long long>(ids), (int)N, (int)V, (int)top, stats, stats + N,
                                          stats + 2 * N, top ? as<float>(s.top_logprob) : nullptr, top ? as<long long>(s.top_token) : nullptr, ptr(work), need,
                                          c10::cuda::getCurrentCUDAStream().stream()),
                 "ternaspmm_token_logprobs");
    }
    return s;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t top) {
        ctx->set_materialize_grads(false);
        at::AutoDispatchBelowADInplaceOrView below;
        Scores s = scores_launch(logits, targets, top);
        const auto shape = targets.sizes();
        // (results of their own: a program may write to them before the backward pass)
        variable_list out = {s.stats[0].reshape(shape).clone(), s.stats[1].reshape(shape).clone()};
        // (the caller's own targets: a view made here would not share the counter by which torch notices that they have changed since)
        ctx->save_for_backward({logits, targets, s.stats});
        if (top) {
            out.push_back(s.top_logprob), out.push_back(s.top_token);
            ctx->mark_non_differentiable({s.top_logprob, s.top_token});
        }
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(3);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        TORCH_CHECK(!at::GradMode::is_enabled(), "token_logprobs is differentiable once: no gradient of its gradient (create_graph)");
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &stats = saved[2];
        const c10::cuda::CUDAGuard guard(logits.device());
        const Tensor rows = logit_rows(logits), ids = saved[1].reshape({-1}).contiguous();
        const int64_t N = rows.size(0), V = rows.size(1);
        const Tensor grad = at::empty({N, V}, rows.options());
        OptTensor g[2];
        for (int i = 0; i < 2; ++i)
            if (grads[i].defined()) g[i] = plain(grads[i]).contiguous();
        float* s = as<float>(stats);
        if (N)
            launched(ternaspmm_token_logprobs_grad(ptr(rows), row_step(rows), type_code(rows), as<long long>(ids), (int)N, (int)V, s + 2 * N, s + N, as<float>(g[0]),
                                                   as<float>(g[1]), ptr(grad), c10::cuda::getCurrentCUDAStream().stream()),
                     "ternaspmm_token_logprobs_grad");
        out[0] = grad.reshape(logits.sizes());
        return out;
    }
};

// token_logprobs(logits, targets, top) -> (logprob, entropy, top_logprob or None, top_token or None)
PyObject* py_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 3, "token_logprobs(logits, targets, top)");
    const Tensor &x = tensor_arg(args[0], "logits"), &t = tensor_arg(args[1], "targets");
    const long long top = int_arg(args[2], "top");
    on_gpu(x, "token_logprobs");
    TORCH_CHECK_VALUE(type_code(x) >= 0 && x.dim() >= 1 && x.size(-1) >= 1, "logits are bf16, fp16 or fp32 [..., V], not ", x.scalar_type(), " ", x.sizes());
    TORCH_CHECK_VALUE(t.scalar_type() == at::kLong && t.sizes() == x.sizes().slice(0, x.dim() - 1) && t.device() == x.device(), "targets are int64 ",
                      x.sizes().slice(0, x.dim() - 1), " on ", x.device(), ", not ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
    TORCH_CHECK_VALUE(top >= 0 && top <= 32 && top <= x.size(-1), "top is at most 32 and the vocabulary ", x.size(-1), ", not ", top);
    if (wants_grad(x)) {
        const variable_list r = TokenLogprobs::apply(x, t, (int64_t)top);
        return Py_BuildValue("NNNN", wrap(r[0]), wrap(r[1]), top ? wrap(r[2]) : wrap(OptTensor()), top ? wrap(r[3]) : wrap(OptTensor()));
    }
    const Scores s = scores_launch(x, t, top);
    return Py_BuildValue("NNNN", wrap(s.stats[0].reshape(t.sizes())), wrap(s.stats[1].reshape(t.sizes())), wrap(OptTensor(s.top_logprob)), wrap(OptTensor(s.top_token)));
    END_HANDLE_TH_ERRORS
}

#define TSP_METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}

}  // namespace

PyMethodDef operator_methods[] = {TSP_METHOD("rotate", py_rotate),         TSP_METHOD("kv4_append", py_kv4_append),
                                  TSP_METHOD("kv4_read", py_kv4_read),     TSP_METHOD("kv4_attend", py_kv4_attend),
                                  TSP_METHOD("token_logprobs", py_token_logprobs), {nullptr, nullptr, 0, nullptr}};
