// Tensor-level and autograd side of the operators whose host cost counts: layer norm, rotary positions, 16-bit cross
// attention. A training step of theirs is a few microseconds of device work for small tensors; as Python functions the same
// checks, allocations and autograd bookkeeping cost 147 us a step on the host (22 us forward, the rest in the backward, which
// runs on a thread of its own with cold caches), so they are done here. Checks raise RuntimeError, a status of libq8_hip
// raises q8_kernels_amd._lib.Q8Error, in a backward too. Everything runs on the current stream of the tensors' device; nothing synchronises.
//
// Host code only, compiled against torch; the kernels are reached through the C ABI (include/q8_hip.h).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <array>
#include <optional>

#include "../../include/q8_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A status becomes a Python error here, which torch carries through its engine's threads as it is (a C++ exception of this module
// would reach the caller of a backward as a RuntimeError without the status). The error belongs to the thread that made the call.
void check(int64_t status) {
    if (status >= 0) return;
    const char* last = q8_last_error();
    const std::string text = last && last[0] ? last : q8_strerror((int)status);
    const pybind11::gil_scoped_acquire gil;
    const pybind11::object type = pybind11::module_::import("q8_kernels_amd._lib").attr("Q8Error");
    PyErr_SetObject(type.ptr(), type((int)status, text).ptr());
    python_error error;
    error.persist();
    throw error;
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return Q8_BF16;
        case at::kHalf: return Q8_F16;
        case at::kFloat: return Q8_F32;
        default: return -1;
    }
}
OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
q8_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void require_gpu(const Tensor& t, const char* name) { TORCH_CHECK(t.is_cuda(), name, " must be a CUDA (HIP) tensor"); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Forward-mode derivatives are not formed: a dual tensor would lose its tangent without a word where nothing requires a gradient
// (where something does, torch's autograd refuses it).
void no_tangents(std::initializer_list<const Tensor*> inputs, const char* who) {
    for (const Tensor* t : inputs) TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), who, ": forward-mode derivatives are not formed");
}

// A leaf whose eager graph still lives keeps the stream that graph was built on for its gradients. If that is the default
// stream, a backward captured on another one would make it wait inside the capture, which ends the process from the engine's
// thread: refused here, before anything is recorded.
void no_eager_graph(const Tensor& x, std::initializer_list<const Tensor*> inputs, const char* who) {
    const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
    if (stream == nullptr) return;  // the default stream is never captured
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    for (const Tensor* t : inputs) {
        if (!wants_grad(*t) || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto own = node ? node->stream() : std::nullopt;
        TORCH_CHECK(!own || own->id() != 0, who, ": an eager graph of the same leaf still lives on the default stream; drop its results before capturing a backward");
    }
}

// gradients of gradients are not formed: where the caller records this backward, using its results again raises
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto fn = std::make_shared<torch::autograd::DelayedError>("this operator's gradient is not differentiable", (int64_t)grads.size());
    return (*fn)(std::move(grads));
}

// ---- layer norm ------------------------------------------------------------------------------------------------

// [rows, dim] with unit last stride and rows that do not overlap: in place where the strides allow it
Tensor as_rows(const Tensor& x) {
    Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) r = r.contiguous();
    return r;
}

// the parameters, contiguous, and their type's code: both float32 or both of x's type
int norm_params(const Tensor& x, Tensor& w, Tensor& b, const char* who) {
    std::optional<at::ScalarType> type;
    for (Tensor* t : {&w, &b}) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->device() == x.device(), who, ": weight and bias must be on ", x.device());
        TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), who, ": weight and bias must have shape [", x.size(-1), "], got ", t->sizes());
        TORCH_CHECK((t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type()) && (!type || *type == t->scalar_type()), who,
                    ": weight and bias must both be float32 or both of x's type ", x.scalar_type());
        type = t->scalar_type();
        if (!t->is_contiguous()) *t = t->contiguous();
    }
    return !type || *type == at::kFloat ? Q8_F32 : type_of(x);
}

// stats: NULL, or what the mean and the reciprocal deviation of every row go to: two tensors, or one of both
Tensor norm_forward(const Tensor& x, Tensor w, Tensor b, double eps, std::array<Tensor, 2>* stats, bool together = false) {
    require_gpu(x, "x");
    const int dt = type_of(x);
    TORCH_CHECK(dt >= 0, "layer_norm: x must be bfloat16, float16 or float32, got ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: x must have a last dimension of one element or more");
    TORCH_CHECK(x.size(-1) <= 32768, "layer_norm: last dimension of ", x.size(-1), " elements (at most 32768)");
    const int wd = norm_params(x, w, b, "layer_norm");
    const c10::DeviceGuard guard(x.device());
    const Tensor r = as_rows(x);
    Tensor y = at::empty(x.sizes(), x.options());
    float *mean = nullptr, *rstd = nullptr;
    if (stats && together) {
        (*stats)[0] = at::empty({2, r.size(0)}, x.options().dtype(at::kFloat));
        mean = (float*)ptr((*stats)[0]);
        rstd = mean + r.size(0);
    } else if (stats) {
        for (Tensor& t : *stats) t = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
        mean = (float*)ptr((*stats)[0]);
        rstd = (float*)ptr((*stats)[1]);
    }
    check(q8_layernorm(ptr(r), dt, r.stride(0), ptr(w), ptr(b), wd, ptr(y), mean, rstd, r.size(0), (int)r.size(1), (float)eps, stream_of(x)));
    return y;
}

std::array<Tensor, 3> norm_backward(const Tensor& grad, const Tensor& x, Tensor w, Tensor b, const float* mean, const float* rstd,
                                    std::array<bool, 3> needs) {
    const char* who = "layer_norm_backward";
    require_gpu(x, "x");
    TORCH_CHECK(type_of(x) >= 0 && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 32768, who, ": x is not one that the forward takes");
    TORCH_CHECK(grad.sizes() == x.sizes() && grad.scalar_type() == x.scalar_type() && grad.device() == x.device(), who, ": grad must match x");
    const int wd = norm_params(x, w, b, who);
    const c10::DeviceGuard guard(x.device());
    const Tensor r = as_rows(x), g = as_rows(grad);
    Tensor dx, dw, db, work;
    if (needs[0]) dx = at::empty(x.sizes(), x.options());
    if (needs[1] && w.defined()) dw = at::empty(w.sizes(), w.options());
    if (needs[2] && b.defined()) db = at::empty(b.sizes(), b.options());
    int64_t size = 0;
    if (dw.defined() || db.defined()) {
        size = q8_layernorm_backward_workspace(r.size(0), (int)r.size(1));
        check(size);
        work = at::empty({size}, x.options().dtype(at::kByte));
    }
    check(q8_layernorm_backward(ptr(g), g.stride(0), ptr(r), type_of(x), r.stride(0), ptr(w), wd, mean, rstd, ptr(dx),
                                ptr(dw), ptr(db), ptr(work), size, r.size(0), (int)r.size(1), stream_of(x)));
    return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
        const Tensor w = or_none(weight), b = or_none(bias);
        std::array<Tensor, 2> stats;
        Tensor y = norm_forward(x, w, b, eps, &stats, true);
        ctx->save_for_backward({x, w, b, stats[0]});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const auto s = ctx->get_saved_variables();
        // (needs_input_grad counts the tensors that were given)
        const bool w = s[1].defined(), b = s[2].defined();
        const float* mean = (const float*)ptr(s[3]);
        auto d = norm_backward(grads[0], s[0], s[1], s[2], mean, mean + s[3].size(1),
                               {ctx->needs_input_grad(0), w && ctx->needs_input_grad(1), b && ctx->needs_input_grad(w ? 2 : 1)});
        return once({d[0], d[1], d[2], Tensor()});
    }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const Tensor w = or_none(weight), b = or_none(bias);
    no_tangents({&x, &w, &b}, "layer_norm");
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) {
        require_gpu(x, "x");
        no_eager_graph(x, {&x, &w, &b}, "layer_norm");
        return LayerNorm::apply(x, given(w), given(b), eps);
    }
    return norm_forward(x, w, b, eps, nullptr);
}

// ---- rotary positions --------------------------------------------------------------------------------------------

// t's memory order with unit last stride, uninitialised
Tensor like(const Tensor& t) {
    Tensor out = at::empty_like(t);
    return out.stride(-1) == 1 ? out : at::empty(t.sizes(), t.options());
}

std::array<Tensor, 2> rotary(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, bool half, double factor, bool backward) {
    const Tensor x = q.defined() ? q : k;
    TORCH_CHECK(x.defined(), "rotary: q or k is needed");
    for (const Tensor* t : {&q, &k}) {
        if (!t->defined()) continue;
        require_gpu(*t, "q and k");
        TORCH_CHECK(t->dim() == 4 && type_of(*t) >= 0, "rotary: q and k must be [B, heads, T, D] in bfloat16, float16 or float32");
        TORCH_CHECK(t->scalar_type() == x.scalar_type() && t->device() == x.device() && t->size(0) == x.size(0) && t->size(2) == x.size(2) &&
                        t->size(3) == x.size(3),
                    "rotary: q and k must agree in type, device, batch, tokens and head size");
        TORCH_CHECK(t->size(1) <= 65536 && t->size(3) <= 512, "rotary: ", t->size(1), " heads of ", t->size(3), " elements (at most 65536 and 512)");
    }
    const int64_t batch = x.size(0), tokens = x.size(2);
    TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kDouble && inv_freq.device() == x.device() && inv_freq.size(0) <= 256,
                "rotary: inv_freq must be float64 [R / 2] on ", x.device());
    const c10::DeviceGuard guard(x.device());
    inv_freq = inv_freq.contiguous();
    int bits = 0;
    int64_t row = 0;
    if (positions.defined()) {
        const bool wide = positions.scalar_type() == at::kLong;
        TORCH_CHECK((wide || positions.scalar_type() == at::kInt) && positions.device() == x.device(), "rotary: positions must be int32 or int64 on ", x.device());
        const bool rows = positions.dim() == 2 && (positions.size(0) == batch || positions.size(0) == 1) && positions.size(1) == tokens;
        TORCH_CHECK(rows || (positions.dim() == 1 && positions.size(0) == tokens), "rotary: positions must be [", tokens, "] or [", batch, ", ", tokens,
                    "], got ", positions.sizes());
        bits = wide ? 64 : 32;
        if (tokens > 1 && positions.stride(-1) != 1) positions = positions.contiguous();
        if (positions.dim() == 2 && positions.size(0) > 1) {
            row = positions.stride(0);
            if (row > 0 && row < tokens) {
                positions = positions.contiguous();
                row = tokens;
            }
        }
    }
    Tensor q_out, k_out;
    if (q.defined()) {
        if (q.stride(3) != 1) q = q.contiguous();
        q_out = like(q);
    }
    if (k.defined()) {
        if (k.stride(3) != 1) k = k.contiguous();
        k_out = like(k);
    }
    auto strides = [](const Tensor& t) { return t.defined() ? t.strides().data() : nullptr; };
    check(q8_rotary(ptr(q), strides(q), ptr(q_out), strides(q_out), q.defined() ? (int)q.size(1) : 0, ptr(k), strides(k), ptr(k_out), strides(k_out),
                    k.defined() ? (int)k.size(1) : 0, type_of(x), ptr(positions), bits, row, (const double*)ptr(inv_freq), 2 * (int)inv_freq.size(0), half,
                    (float)factor, backward, batch, tokens, (int)x.size(3), stream_of(x)));
    return {q_out, k_out};
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& key, const OptTensor& pos, const Tensor& inv_freq, bool half,
                                 double factor) {
        const Tensor k = or_none(key), positions = or_none(pos);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, inv_freq});
        ctx->saved_data["half"] = half;
        ctx->saved_data["factor"] = factor;
        auto out = rotary(q, k, positions, inv_freq, half, factor, false);
        if (!k.defined()) return {out[0]};
        return {out[0], out[1]};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const auto s = ctx->get_saved_variables();
        Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), gk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor();
        std::array<Tensor, 2> d;
        if (gq.defined() || gk.defined()) d = rotary(gq, gk, s[0], s[1], ctx->saved_data["half"].toBool(), ctx->saved_data["factor"].toDouble(), true);
        return once({d[0], d[1], Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

std::array<Tensor, 2> apply_rotary(const Tensor& q, const OptTensor& key, const OptTensor& positions, const Tensor& inv_freq, bool half, double factor) {
    const Tensor k = or_none(key), p = or_none(positions);
    no_tangents({&q, &k, &inv_freq}, "rotary");
    TORCH_CHECK(!at::GradMode::is_enabled() || !inv_freq.requires_grad(), "rotary: no gradient of inv_freq is formed");
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k))) {
        require_gpu(q, "q and k");
        no_eager_graph(q, {&q, &k}, "rotary");
        auto out = Rotary::apply(q, given(k), given(p), inv_freq, half, factor);
        return {out[0], out.size() > 1 ? out[1] : Tensor()};
    }
    return rotary(q, k, p, inv_freq, half, factor, false);
}

// ---- 16-bit cross attention ------------------------------------------------------------------------------------------

// t itself where its rows are 16-byte chunks that the kernels can address, else a contiguous copy
Tensor chunks(const Tensor& t) {
    bool fine = t.stride(3) == 1 && (t.size(2) <= 1 || t.stride(2) < (1 << 24)) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) fine = fine && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
    return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct Keys {
    Tensor lens, mask;
    int64_t row = 0;
};

Keys attn_check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens, const Tensor& mask, const char* who) {
    for (const Tensor* t : {&q, &k, &v}) {
        require_gpu(*t, "q, k and v");
        TORCH_CHECK(t->dim() == 4, who, ": q, k and v must be [B, heads, tokens, D], got ", t->sizes());
        TORCH_CHECK((t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kHalf) && t->scalar_type() == q.scalar_type() && t->device() == q.device(),
                    who, ": q, k and v must be bfloat16 or float16, all of one type, on one device");
        for (int i = 1; i < 4; ++i) TORCH_CHECK(t->size(i) <= 0x3fffffff, who, ": ", t->sizes(), " is too large");
    }
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3), who, ": q ", q.sizes(), " does not go with k ", k.sizes(), " and v ",
                v.sizes());
    const int64_t b = k.size(0), n = k.size(2);
    Keys out{lens, mask};
    if (lens.defined()) {
        TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == b && lens.device() == q.device(), who, ": kv_lens must be int32 [", b,
                    "] on ", q.device());
        out.lens = lens.contiguous();
    }
    if (mask.defined()) {
        TORCH_CHECK(mask.scalar_type() == at::kBool && mask.dim() == 2 && mask.size(0) == b && mask.size(1) == n && mask.device() == q.device(), who,
                    ": key_mask must be bool [", b, ", ", n, "] on ", q.device());
        if (n > 1 && mask.stride(1) != 1) out.mask = mask.contiguous();
        out.row = out.mask.stride(0);
    }
    return out;
}

// {o, lse, o_low}: the last two with stats, for a backward (o_low: what the rounding of o left off, [B, H, M, D] contiguous)
std::array<Tensor, 3> attn_forward(Tensor q, Tensor k, Tensor v, double scale, const Tensor& lens, const Tensor& mask, bool stats, bool rest) {
    const Keys keys = attn_check(q, k, v, lens, mask, "cross_attention");
    const int64_t b = q.size(0);
    const int h = (int)q.size(1), hk = (int)k.size(1), m = (int)q.size(2), n = (int)k.size(2), d = (int)q.size(3);
    const c10::DeviceGuard guard(q.device());
    const int64_t size = q8_cross_attn_workspace(b, h, hk, m, n, d);
    check(size);
    q = chunks(q), k = chunks(k), v = chunks(v);
    Tensor o = like(q), lse, low, work;
    if (rest) low = at::empty(q.sizes(), q.options().dtype(at::kChar));
    if (stats) lse = at::empty({b, h, m}, q.options().dtype(at::kFloat));
    if (size) work = at::empty({size}, q.options().dtype(at::kByte));
    if (rest)
        check(q8_cross_attn_train(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(), ptr(o), o.strides().data(), ptr(low),
                                  (float*)ptr(lse), (const int32_t*)ptr(keys.lens), (const uint8_t*)ptr(keys.mask), keys.row, type_of(q), (float)scale, b, h, hk,
                                  m, n, d, ptr(work), size, stream_of(q)));
    else
        check(q8_cross_attn(ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(), ptr(o), o.strides().data(), (float*)ptr(lse),
                            (const int32_t*)ptr(keys.lens), (const uint8_t*)ptr(keys.mask), keys.row, type_of(q), (float)scale, b, h, hk, m, n, d, ptr(work),
                            size, stream_of(q)));
    return {o, lse, low};
}

// low: the forward's o_low, or undefined: it is formed again
std::array<Tensor, 3> attn_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor o, const Tensor& low, const Tensor& lse, double scale,
                                    const Tensor& lens, const Tensor& mask) {
    const char* who = "cross_attention_backward";
    const Keys keys = attn_check(q, k, v, lens, mask, who);
    const int64_t b = q.size(0);
    const int h = (int)q.size(1), hk = (int)k.size(1), m = (int)q.size(2), n = (int)k.size(2), d = (int)q.size(3);
    for (const Tensor* t : {&grad, &o})
        TORCH_CHECK(t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type() && t->device() == q.device(), who, ": grad and o must match q");
    TORCH_CHECK(lse.sizes() == q.sizes().slice(0, 3) && lse.scalar_type() == at::kFloat && lse.device() == q.device() && lse.is_contiguous(), who,
                ": lse must be the forward's");
    if (low.defined())
        TORCH_CHECK(low.sizes() == q.sizes() && low.scalar_type() == at::kChar && low.device() == q.device() && low.is_contiguous(), who,
                    ": o_low must be the forward's");
    const c10::DeviceGuard guard(q.device());
    const int64_t size = low.defined() ? q8_cross_attn_train_backward_workspace(b, h, hk, m, n, d) : q8_cross_attn_backward_workspace(b, h, hk, m, n, d);
    check(size);
    q = chunks(q), k = chunks(k), v = chunks(v), o = chunks(o), grad = chunks(grad);
    Tensor dq = like(q), dk = like(k), dv = like(v), work;
    if (size) work = at::empty({size}, q.options().dtype(at::kByte));
    if (low.defined())
        check(q8_cross_attn_train_backward(ptr(grad), grad.strides().data(), ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(),
                                           ptr(o), o.strides().data(), ptr(low), (const float*)ptr(lse), ptr(dq), dq.strides().data(), ptr(dk),
                                           dk.strides().data(), ptr(dv), dv.strides().data(), (const int32_t*)ptr(keys.lens), (const uint8_t*)ptr(keys.mask),
                                           keys.row, type_of(q), (float)scale, b, h, hk, m, n, d, ptr(work), size, stream_of(q)));
    else
        check(q8_cross_attn_backward(ptr(grad), grad.strides().data(), ptr(q), q.strides().data(), ptr(k), k.strides().data(), ptr(v), v.strides().data(), ptr(o),
                                     o.strides().data(), (const float*)ptr(lse), ptr(dq), dq.strides().data(), ptr(dk), dk.strides().data(), ptr(dv),
                                     dv.strides().data(), (const int32_t*)ptr(keys.lens), (const uint8_t*)ptr(keys.mask), keys.row, type_of(q), (float)scale, b,
                                     h, hk, m, n, d, ptr(work), size, stream_of(q)));
    return {dq, dk, dv};
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale, const OptTensor& kv_lens,
                          const OptTensor& key_mask) {
        const Tensor lens = or_none(kv_lens), mask = or_none(key_mask);
        auto out = attn_forward(q, k, v, scale, lens, mask, true, true);
        ctx->save_for_backward({q, k, v, out[0], out[2], out[1], lens, mask});
        ctx->saved_data["scale"] = scale;
        return out[0];
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const auto s = ctx->get_saved_variables();
        auto d = attn_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble(), s[6], s[7]);
        return once({d[0], d[1], d[2], Tensor(), Tensor(), Tensor()});
    }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> softmax_scale, const OptTensor& kv_lens,
                       const OptTensor& key_mask) {
    const double scale = softmax_scale.has_value() ? *softmax_scale : q.dim() && q.size(-1) ? 1.0 / std::sqrt((double)q.size(-1)) : 1.0;
    const Tensor lens = or_none(kv_lens), mask = or_none(key_mask);
    no_tangents({&q, &k, &v}, "cross_attention");
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v))) {
        require_gpu(q, "q, k and v");
        no_eager_graph(q, {&q, &k, &v}, "cross_attention");
        return CrossAttention::apply(q, k, v, scale, given(lens), given(mask));
    }
    return attn_forward(q, k, v, scale, lens, mask, false, false)[0];
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    namespace py = pybind11;
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (python_error& e) {
            e.restore();
        }
    });
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_forward", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, bool stats) {
        std::array<Tensor, 2> s;
        Tensor y = norm_forward(x, or_none(w), or_none(b), eps, stats ? &s : nullptr);
        return std::vector<OptTensor>{y, given(s[0]), given(s[1])};
    });
    m.def("layer_norm_backward", [](const Tensor& g, const Tensor& x, const OptTensor& w, const OptTensor& b, const Tensor& mean, const Tensor& rstd,
                                    std::array<bool, 3> needs) {
        for (const Tensor* t : {&mean, &rstd})
            TORCH_CHECK(x.dim() >= 1 && t->scalar_type() == at::kFloat && t->sizes() == x.sizes().slice(0, x.dim() - 1) && t->device() == x.device() &&
                            t->is_contiguous(), "layer_norm_backward: mean and rstd must be the forward's");
        auto r = norm_backward(g, x, or_none(w), or_none(b), (const float*)ptr(mean), (const float*)ptr(rstd), needs);
        return std::vector<OptTensor>{given(r[0]), given(r[1]), given(r[2])};
    });
    m.def("apply_rotary", [](const Tensor& q, const OptTensor& k, const OptTensor& p, const Tensor& f, bool half, double factor) {
        auto r = apply_rotary(q, k, p, f, half, factor);
        return std::make_pair(r[0], given(r[1]));
    });
    m.def("rotary", [](const OptTensor& q, const OptTensor& k, const OptTensor& p, const Tensor& f, bool half, double factor, bool backward) {
        auto r = rotary(or_none(q), or_none(k), or_none(p), f, half, factor, backward);
        return std::vector<OptTensor>{given(r[0]), given(r[1])};
    });
    m.def("cross_attention", &cross_attention);
    m.def("cross_attention_forward",
          [](const Tensor& q, const Tensor& k, const Tensor& v, double scale, const OptTensor& lens, const OptTensor& mask, bool stats, bool rest) {
              auto r = attn_forward(q, k, v, scale, or_none(lens), or_none(mask), stats || rest, rest);
              std::vector<OptTensor> out{r[0], given(r[1])};
              if (rest) out.push_back(r[2]);
              return out;
          });
    m.def("cross_attention_backward", [](const Tensor& g, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, double scale,
                                         const OptTensor& lens, const OptTensor& mask, const OptTensor& low) {
        auto r = attn_backward(g, q, k, v, o, or_none(low), lse, scale, or_none(lens), or_none(mask));
        return std::vector<Tensor>{r[0], r[1], r[2]};
    });
}
