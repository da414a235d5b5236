// The calls that a training or generation step makes most, from Python into the kernels without a detour:
// allocation, launch and autograd bookkeeping in native code.  A call of a few microseconds on the GPU used
// to spend 40 to 140 us of the host's time in Python autograd Functions and ctypes.
//
// Every function serves the plain form of its call and returns None for any other -- unusual layouts, types,
// devices, and everything that has to be refused --, for which the Python modules keep their general path with its
// checks and messages.  The kernels are those of include/neox_fused.h.  Nothing is kept between calls: what a
// backward pass needs is saved through autograd, under its version checks and saved-tensor hooks.
#include <torch/extension.h>
#include <torch/version.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/neox_fused.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int status) {
    if (status == NEOX_OK) return;
    const char* message = neox_fused_last_error();
    throw std::runtime_error(*message ? message : neox_fused_strerror(status));
}

bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
int32_t code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kHalf: return NEOX_F16;
        case at::kBFloat16: return NEOX_BF16;
        case at::kFloat: return NEOX_F32;
        default: throw std::runtime_error("Only fp16 and bf16 are supported");
    }
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool fits_int32(int64_t n) { return n >= 0 && n <= INT32_MAX; }
bool records(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
// a tensor whose memory this code may look at
bool on_gpu(const Tensor& t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj(); }
// ... and that a call may be served for: one with a forward-mode tangent goes to the Python autograd Functions,
// which refuse it (a result computed here would have lost the tangent)
bool plain(const Tensor& t) { return on_gpu(t) && !t._fw_grad(/*level=*/0).defined(); }

// ---- softmax ---------------------------------------------------------------------------------------
enum Kind : int64_t { kCausal = -1, kMasked = -2 };  // a window width otherwise

struct SoftmaxCall {
    double scale;
    int64_t kind;
    const Tensor* mask;    // kMasked
    const Tensor* slopes;  // kCausal, optional
    double p;              // kCausal: attention dropout, 0 = none
    int64_t seed, offset;
};

// probabilities, and the dropped ones (undefined without dropout); x is contiguous [b, np, sq, sk]
std::tuple<Tensor, Tensor> softmax_forward(const Tensor& x, const SoftmaxCall& c) {
    const c10::DeviceGuard guard(x.device());
    const auto b = (int32_t)x.size(0), np = (int32_t)x.size(1), sq = (int32_t)x.size(2), sk = (int32_t)x.size(3);
    Tensor y = at::empty_like(x), dropped;
    const auto scale = (float)c.scale;
    const void* in = x.const_data_ptr();
    void *out = y.mutable_data_ptr(), *stream = stream_of(x);
    const float* slopes = c.slopes ? static_cast<const float*>(c.slopes->const_data_ptr()) : nullptr;
    if (c.kind == kMasked) {
        check(neox_masked_softmax_fwd(out, in, static_cast<const uint8_t*>(c.mask->const_data_ptr()), scale, b, np, sq, sk,
                                      (int32_t)c.mask->size(0), code(x), stream));
    } else if (c.kind >= 0) {
        check(neox_sliding_window_softmax_fwd(out, in, scale, (int64_t)b * np, sq, sk, (int32_t)c.kind, code(x), stream));
    } else if (c.p != 0) {
        dropped = at::empty_like(x);
        check(neox_causal_softmax_dropout_fwd(dropped.mutable_data_ptr(), out, in, slopes, nullptr, 0, scale, (float)c.p,
                                              (uint64_t)c.seed, (uint64_t)c.offset, nullptr, b, np, sq, sk, code(x), stream));
    } else if (slopes) {
        check(neox_causal_softmax_alibi_fwd(out, in, slopes, scale, b, np, sq, sk, code(x), stream));
    } else {
        check(neox_causal_softmax_fwd(out, in, scale, (int64_t)b * np, sq, sk, code(x), stream));
    }
    return {y, dropped};
}

class Softmax : public torch::autograd::Function<Softmax> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const SoftmaxCall& c) {
        auto [y, dropped] = softmax_forward(x, c);
        ctx->save_for_backward({y});
        ctx->saved_data["scale"] = c.scale;
        ctx->saved_data["kind"] = c.kind;
        if (c.p != 0) {
            ctx->saved_data["p"] = c.p;
            ctx->saved_data["seed"] = c.seed;
            ctx->saved_data["offset"] = c.offset;
        }
        return dropped.defined() ? dropped : y;
    }

    // d(input), written into the incoming gradient when that is contiguous
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor y = ctx->get_saved_variables()[0].contiguous();
        const Tensor g = grads[0].contiguous();
        if (g.sizes() != y.sizes() || g.scalar_type() != y.scalar_type() || g.device() != y.device() || !on_gpu(g))
            throw std::runtime_error("output_grads and softmax_results must have the same dtype and shape");
        const c10::DeviceGuard guard(g.device());
        const auto scale = (float)ctx->saved_data["scale"].toDouble();
        const int64_t kind = ctx->saved_data["kind"].toInt();
        const int64_t batches = g.size(0) * g.size(1);
        const auto sq = (int32_t)g.size(2), sk = (int32_t)g.size(3);
        void *dx = g.mutable_data_ptr(), *stream = stream_of(g);
        const void* probs = y.const_data_ptr();
        const auto p = ctx->saved_data.find("p");
        if (kind == kMasked) {
            check(neox_masked_softmax_bwd(dx, dx, probs, scale, batches * sq, sk, code(g), stream));
        } else if (kind >= 0) {
            check(neox_sliding_window_softmax_bwd(dx, dx, probs, scale, batches, sq, sk, (int32_t)kind, code(g), stream));
        } else if (p != ctx->saved_data.end()) {
            check(neox_causal_softmax_dropout_bwd(dx, dx, probs, scale, (float)p->second.toDouble(),
                                                  (uint64_t)ctx->saved_data["seed"].toInt(),
                                                  (uint64_t)ctx->saved_data["offset"].toInt(), nullptr, batches, sq, sk,
                                                  code(g), stream));
        } else {
            check(neox_causal_softmax_bwd(dx, dx, probs, scale, batches, sq, sk, code(g), stream));
        }
        return {g, Tensor()};
    }
};

bool plain_scores(const Tensor& x) {
    return plain(x) && half_type(x) && x.dim() == 4 && x.numel() > 0 && x.is_contiguous() && fits_int32(x.size(0)) &&
           fits_int32(x.size(1)) && fits_int32(x.size(2)) && fits_int32(x.size(3));
}

Tensor run_softmax(const Tensor& x, const SoftmaxCall& c) {
    if (records(x)) return Softmax::apply(x, c);
    auto [y, dropped] = softmax_forward(x, c);
    return dropped.defined() ? dropped : y;
}

// whether causal_softmax serves these scores (and slopes): asked before random numbers are drawn for it
bool causal_takes(const Tensor& x, const std::optional<Tensor>& slopes) {
    return plain_scores(x) && (!slopes || (plain(*slopes) && slopes->device() == x.device() && slopes->scalar_type() == at::kFloat &&
                                           slopes->numel() == x.size(1) && slopes->is_contiguous() && !slopes->requires_grad()));
}

// causal (window < 0) or sliding-window scores [b, np, sq, sk]; slopes: fp32 [np]; p, seed, offset: dropout
std::optional<Tensor> causal_softmax(const Tensor& x, double scale, int64_t window, const std::optional<Tensor>& slopes,
                                     double p, uint64_t seed, uint64_t offset) {
    if (!causal_takes(x, slopes)) return std::nullopt;
    if (window >= 0 && (slopes || p != 0 || !fits_int32(window))) return std::nullopt;
    return run_softmax(x, {scale, window >= 0 ? window : (int64_t)kCausal, nullptr, slopes ? &*slopes : nullptr, p, (int64_t)seed,
                           (int64_t)offset});
}

// scores [b, np, sq, sk] under a mask tensor [1 or b, 1, sq, sk]
std::optional<Tensor> masked_softmax(const Tensor& x, const Tensor& mask, double scale) {
    if (!plain_scores(x) || !on_gpu(mask) || mask.device() != x.device() || mask.dim() != 4 || !mask.is_contiguous() ||
        (mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) ||
        (mask.size(0) != 1 && mask.size(0) != x.size(0)) || mask.size(1) != 1 || mask.size(2) != x.size(2) ||
        mask.size(3) != x.size(3))
        return std::nullopt;
    return run_softmax(x, {scale, kMasked, &mask, nullptr, 0, 0, 0});
}

// ---- rotary embedding ------------------------------------------------------------------------------
struct Tables {
    Tensor cos, sin;  // rows of d_rot values; sin undefined: cos holds angles
    int64_t d_rot, offset;
};

void rope_launch(const Tensor& out_q, const Tensor* out_k, const Tensor& q, const Tensor* k, const Tables& t, int64_t d,
                 bool backward) {
    const c10::DeviceGuard guard(q.device());
    auto strides = [](const Tensor& x) { return x.strides().data(); };
    const int64_t row = t.cos.size(0) > 1 ? t.cos.stride(0) : t.d_rot;
    const auto s = (int32_t)q.size(0), b = (int32_t)q.size(1), hq = (int32_t)q.size(2), hk = k ? (int32_t)k->size(2) : 0;
    void* oq = out_q.mutable_data_ptr();
    void* ok = k ? out_k->mutable_data_ptr() : nullptr;
    const void* kp = k ? k->const_data_ptr() : nullptr;
    const int64_t *ks = k ? strides(*k) : nullptr, *oks = k ? strides(*out_k) : nullptr;
    if (!t.sin.defined()) {
        check(neox_rope_apply_freqs(oq, ok, q.const_data_ptr(), kp, static_cast<const float*>(t.cos.const_data_ptr()), s, b,
                                    hq, hk, (int32_t)t.d_rot, (int32_t)d, strides(q), ks, strides(out_q), oks, row,
                                    (int32_t)t.offset, code(q), backward, stream_of(q)));
    } else {
        check(neox_rope_apply(oq, ok, q.const_data_ptr(), kp, t.cos.const_data_ptr(), t.sin.const_data_ptr(), s, b, hq, hk,
                              (int32_t)t.d_rot, (int32_t)d, strides(q), ks, strides(out_q), oks, row, (int32_t)t.offset,
                              code(q), code(t.cos), backward, stream_of(q)));
    }
}

void save_tables(AutogradContext* ctx, const Tables& t) {
    if (t.sin.defined()) ctx->save_for_backward({t.cos, t.sin});
    else ctx->save_for_backward({t.cos});
    ctx->saved_data["d_rot"] = t.d_rot;
    ctx->saved_data["offset"] = t.offset;
}
// The saved tables, for a gradient g [s, ..]: a saved-tensor hook may have given back another tensor than the forward
// pass left with it, so everything the kernel takes for granted is looked at again.
Tables saved_tables(AutogradContext* ctx, const Tensor& g) {
    variable_list v = ctx->get_saved_variables();
    const int64_t d_rot = ctx->saved_data["d_rot"].toInt(), offset = ctx->saved_data["offset"].toInt();
    for (Tensor& t : v) {
        if (!on_gpu(t) || t.device() != g.device())
            throw std::runtime_error("the saved cos/sin tables or angles must be on the device of the gradient");
        if (t.dim() != 4 || t.size(1) != 1 || t.size(2) != 1 || t.size(3) != d_rot || t.size(0) < offset + g.size(0))
            throw std::runtime_error("the saved cos/sin tables or angles have another shape than in the forward pass");
        if (t.scalar_type() != v[0].scalar_type() ||
            (t.scalar_type() != at::kFloat && (v.size() == 1 || t.scalar_type() != g.scalar_type())))
            throw std::runtime_error("the saved cos/sin tables must be float32 or have the dtype of the gradient, angles float32");
        t = t.contiguous();
    }
    return {v[0], v.size() > 1 ? v[1] : Tensor(), d_rot, offset};
}
Tensor dense_last(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// q and k rotated into new tensors, one launch
std::tuple<Tensor, Tensor> rotary_pair(const Tensor& q, const Tensor& k, const Tables& t, bool backward) {
    Tensor oq = at::empty(q.sizes(), q.options()), ok = at::empty(k.sizes(), k.options());
    rope_launch(oq, &ok, q, &k, t, t.d_rot, backward);
    return {oq, ok};
}

class Rotary : public torch::autograd::Function<Rotary> {
public:
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tables& t) {
        save_tables(ctx, t);
        auto [oq, ok] = rotary_pair(q, k, t, false);
        return {oq, ok};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        auto [dq, dk] = rotary_pair(dense_last(grads[0]), dense_last(grads[1]), saved_tables(ctx, grads[0]), true);
        return {dq, dk, Tensor()};
    }
};

// one tensor's whole heads; transposed: the memory of the result is [b, s, h, d]
Tensor rope_whole(const Tensor& x, const Tables& t, bool transposed, bool backward) {
    Tensor out = transposed ? at::empty({x.size(1), x.size(0), x.size(2), x.size(3)}, x.options()).transpose(0, 1)
                            : at::empty(x.sizes(), x.options());
    rope_launch(out, nullptr, x, nullptr, t, x.size(3), backward);
    return out;
}

class Rope : public torch::autograd::Function<Rope> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tables& t, bool transposed) {
        save_tables(ctx, t);
        ctx->saved_data["transposed"] = transposed;
        return rope_whole(x, t, transposed, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return {rope_whole(dense_last(grads[0]), saved_tables(ctx, grads[0]), ctx->saved_data["transposed"].toBool(), true), Tensor(),
                Tensor()};
    }
};

// strides that count from the tensor's first element upwards, and extents the kernels count in 32 bits
bool plain_heads(const Tensor& x) {
    return plain(x) && half_type(x) && x.dim() == 4 && x.numel() > 0 && x.stride(3) == 1 && fits_int32(x.size(0)) &&
           fits_int32(x.size(1)) && fits_int32(x.size(2)) && fits_int32(x.size(3));
}
// a table [n, 1, 1, d_rot] of dense rows in memory order, with the rows offset .. offset + s
bool plain_table(const Tensor& t, const Tensor& x, int64_t d_rot, int64_t rows) {
    return plain(t) && t.device() == x.device() && t.dim() == 4 && t.size(1) == 1 && t.size(2) == 1 && t.size(3) == d_rot &&
           t.size(0) >= rows && t.is_contiguous() && !t.requires_grad();
}

// q, k [s, b, h, d_rot] -> rotated, or None
std::optional<std::tuple<Tensor, Tensor>> rotary(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
                                                 int64_t offset) {
    if (!plain_heads(q) || !plain_heads(k) || q.scalar_type() != k.scalar_type() || q.device() != k.device() ||
        q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.size(3) != k.size(3) || q.size(3) % 2 != 0 || offset < 0 ||
        !fits_int32(offset + q.size(0)))
        return std::nullopt;
    const int64_t d_rot = q.size(3);
    if (!plain_table(cos, q, d_rot, offset + q.size(0)) || !plain_table(sin, q, d_rot, offset + q.size(0)) ||
        cos.scalar_type() != sin.scalar_type() || cos.size(0) != sin.size(0) ||
        (cos.scalar_type() != at::kFloat && cos.scalar_type() != q.scalar_type()))
        return std::nullopt;
    const Tables t{cos, sin, d_rot, offset};
    if (records(q) || records(k)) {
        variable_list out = Rotary::apply(q, k, t);
        return std::make_tuple(out[0], out[1]);
    }
    return rotary_pair(q, k, t, false);
}

// x [s, b, h, d], rotated over the first dims by angles (sin absent) or by tables [s, 1, 1, d_rot], or None
std::optional<Tensor> rope(const Tensor& x, const Tensor& cos, const std::optional<Tensor>& sin, bool transposed) {
    if (!plain_heads(x) || cos.dim() != 4) return std::nullopt;
    const int64_t d_rot = cos.size(3);
    if (d_rot > x.size(3) || d_rot < 2 || d_rot % 2 != 0 || cos.size(0) != x.size(0) || !plain_table(cos, x, d_rot, x.size(0)))
        return std::nullopt;
    if (sin ? (sin->dim() != 4 || sin->size(0) != x.size(0) || !plain_table(*sin, x, d_rot, x.size(0)) ||
               cos.scalar_type() != sin->scalar_type() ||
               (cos.scalar_type() != at::kFloat && cos.scalar_type() != x.scalar_type()))
            : cos.scalar_type() != at::kFloat)
        return std::nullopt;
    const Tables t{cos, sin ? *sin : Tensor(), d_rot, 0};
    if (records(x)) return Rope::apply(x, t, transposed);
    return rope_whole(x, t, transposed, false);
}

// ---- attention over windows and pages ---------------------------------------------------------------
// a 16-bit tensor [.., heads, d] that the attention kernels read as it lies (as whole_pieces in _lib.py)
bool in_pieces(const Tensor& x, int64_t per_piece = 8) {
    if (x.stride(-1) != 1 || reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 != 0) return false;
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
        if (x.size(i) > 1 && (x.stride(i) % per_piece != 0 || x.stride(i) < 0 || x.stride(i) >= (int64_t)1 << 31)) return false;
    return x.size(-2) == 1 || x.stride(-2) >= x.size(-1);
}
// the strides of all axes but the dense last one; an axis of one element counts as 0
struct RowStrides {
    int64_t of[3] = {0, 0, 0};
    RowStrides(const Tensor& x, int64_t axes) {
        for (int64_t i = 0; i < axes; ++i) of[i] = x.size(i) > 1 ? x.stride(i) : 0;
    }
    operator const int64_t*() const { return of; }
};
template <typename T>
T* pointer_or_null(const std::optional<Tensor>& t) {
    return t ? static_cast<T*>(const_cast<void*>(t->const_data_ptr())) : nullptr;
}

struct WindowCall {
    double scale;
    int64_t window, sinks;
    const std::optional<Tensor>& lengths;
};

// the output, and for a backward pass what its rounding took away and the rows' logarithms
std::tuple<Tensor, Tensor, Tensor> window_forward(const Tensor& q, const Tensor& k, const Tensor& v, const WindowCall& c, bool for_backward) {
    const c10::DeviceGuard guard(q.device());
    const auto sq = (int32_t)q.size(0), b = (int32_t)q.size(1), h = (int32_t)q.size(2), d = (int32_t)q.size(3);
    Tensor out = at::empty(q.sizes(), q.options()), low, lse;
    if (for_backward) {
        low = at::empty(q.sizes(), q.options());
        lse = at::empty({(int64_t)b * h * sq}, q.options().dtype(at::kFloat));
    }
    check(neox_window_attention_fwd(out.mutable_data_ptr(), for_backward ? low.mutable_data_ptr() : nullptr,
                                    for_backward ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), pointer_or_null<const int32_t>(c.lengths),
                                    b, sq, (int32_t)k.size(0), h, (int32_t)k.size(2), d, RowStrides(q, 3), RowStrides(k, 3),
                                    RowStrides(v, 3), RowStrides(out, 3), (float)c.scale, (int32_t)c.window, (int32_t)c.sinks, code(q),
                                    stream_of(q)));
    return {out, low, lse};
}

// Hands on the gradients of a backward pass that is itself recorded (create_graph), as results of the tensors they were
// computed from: the kernels have no second derivative, and asking for one has to fail and not to leave a term out.
class OnlyOnce : public torch::autograd::Function<OnlyOnce> {
public:
    static variable_list forward(AutogradContext*, const Tensor& dq, const Tensor& dk, const Tensor& dv, const Tensor&, const Tensor&, const Tensor&,
                                 const Tensor&) {
        return {dq, dk, dv};
    }
    static variable_list backward(AutogradContext*, variable_list) { throw std::runtime_error("window_attention has no second derivative"); }
};

class WindowAttention : public torch::autograd::Function<WindowAttention> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const WindowCall& c) {
        auto [out, low, lse] = window_forward(q, k, v, c, true);
        ctx->save_for_backward({q, k, v, out, low, lse, c.lengths ? *c.lengths : Tensor()});
        ctx->saved_data["scale"] = c.scale;
        ctx->saved_data["window"] = c.window;
        ctx->saved_data["sinks"] = c.sinks;
        return out;
    }
    // A saved-tensor hook may have given back other tensors than were left with it: everything the kernels take for
    // granted is looked at again.
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list v = ctx->get_saved_variables();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        Tensor g = grads[0];
        const Tensor sources[] = {v[0], v[1], v[2], g};
        const Tensor lengths = v[6];
        v.resize(6);
        for (const Tensor& t : v)
            if (!on_gpu(t) || t.device() != g.device()) throw std::runtime_error("the saved tensors must be on the device of the gradient");
        const Tensor &q0 = v[0], &k0 = v[1], &v0 = v[2], &out0 = v[3], &low0 = v[4];
        const Tensor lse = v[5].contiguous();
        if (q0.dim() != 4 || k0.dim() != 4 || k0.sizes() != v0.sizes() || out0.sizes() != q0.sizes() ||
            low0.sizes() != q0.sizes() || low0.scalar_type() != q0.scalar_type() || g.sizes() != q0.sizes() ||
            k0.size(1) != q0.size(1) || k0.size(3) != q0.size(3) || !half_type(q0) || !on_gpu(g) || g.scalar_type() != q0.scalar_type() ||
            k0.scalar_type() != q0.scalar_type() || v0.scalar_type() != q0.scalar_type() || out0.scalar_type() != q0.scalar_type() ||
            lse.scalar_type() != at::kFloat || lse.numel() != q0.size(0) * q0.size(1) * q0.size(2))
            throw std::runtime_error("the gradient and the saved tensors must have the shapes and dtypes of the forward pass");
        if (lengths.defined() && (!on_gpu(lengths) || lengths.device() != g.device() || lengths.scalar_type() != at::kInt ||
                                  lengths.numel() != q0.size(1) || !lengths.is_contiguous()))
            throw std::runtime_error("the saved key lengths have changed");
        auto readable = [](const Tensor& t) { return in_pieces(t) ? t : t.clone(at::MemoryFormat::Contiguous); };
        const Tensor q = readable(q0), k = readable(k0), val = readable(v0), out = out0.contiguous(), low = low0.contiguous();
        g = readable(g);
        const c10::DeviceGuard guard(q.device());
        const auto sq = (int32_t)q.size(0), b = (int32_t)q.size(1), h = (int32_t)q.size(2), d = (int32_t)q.size(3);
        const auto sk = (int32_t)k.size(0), h_kv = (int32_t)k.size(2);
        const auto window = (int32_t)ctx->saved_data["window"].toInt(), sinks = (int32_t)ctx->saved_data["sinks"].toInt();
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(k.sizes(), k.options());
        int64_t bytes = 0;
        check(neox_window_attention_bwd_workspace(&bytes, b, sq, sk, h, h_kv, d, window, sinks));
        const Tensor workspace = at::empty({bytes}, q.options().dtype(at::kByte));
        check(neox_window_attention_bwd(
            dq.mutable_data_ptr(), dk.mutable_data_ptr(), dv.mutable_data_ptr(), workspace.mutable_data_ptr(), bytes, g.const_data_ptr(),
            out.const_data_ptr(), low.const_data_ptr(), static_cast<const float*>(lse.const_data_ptr()), q.const_data_ptr(), k.const_data_ptr(),
            val.const_data_ptr(), lengths.defined() ? static_cast<const int32_t*>(lengths.const_data_ptr()) : nullptr, b, sq, sk, h, h_kv, d,
            RowStrides(dq, 3), RowStrides(dk, 3), RowStrides(dv, 3), RowStrides(g, 3), RowStrides(out, 3), RowStrides(q, 3),
            RowStrides(k, 3), RowStrides(val, 3), (float)ctx->saved_data["scale"].toDouble(), window, sinks, code(q), stream_of(q)));
        if (records(sources[0]) || records(sources[1]) || records(sources[2]) || records(sources[3])) {
            const variable_list once = OnlyOnce::apply(dq, dk, dv, sources[0], sources[1], sources[2], sources[3]);
            return {once[0], once[1], once[2], Tensor()};
        }
        return {dq, dk, dv, Tensor()};
    }
};

bool int_list(const Tensor& t, const Tensor& like, int64_t n) {
    return on_gpu(t) && t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
bool attention_heads(const Tensor& x) { return plain_heads(x) && x.size(3) % 8 == 0 && x.size(3) <= 256 && in_pieces(x); }

// q [sq, b, h, d], k, v [sk, b, h_kv, d]; window < 0: none; lengths int32 [b] -> [sq, b, h, d], or None
std::optional<Tensor> window_attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale, int64_t window, int64_t sinks,
                                       const std::optional<Tensor>& lengths) {
    if (!attention_heads(q) || !attention_heads(k) || !attention_heads(v) || k.device() != q.device() || v.device() != q.device() ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.sizes() != v.sizes() || k.size(1) != q.size(1) ||
        k.size(3) != q.size(3) || q.size(2) % k.size(2) != 0 || window > INT32_MAX || window < -1 || !fits_int32(sinks) ||
        (lengths && !int_list(*lengths, q, q.size(1))))
        return std::nullopt;
    const WindowCall c{scale, window, sinks, lengths};
    if (records(q) || records(k) || records(v)) return WindowAttention::apply(q, k, v, c);
    return std::get<0>(window_forward(q, k, v, c, false));
}

// The tensors of a PagedKVCache, which has looked at them; `like` is a 16-bit tensor of the call.
struct Cache {
    const Tensor &k, &v;
    const std::optional<Tensor>&k_scale, &v_scale;
    int32_t dtype(const Tensor& like) const {
        switch (k.scalar_type()) {
            case at::kChar: return NEOX_I8;
            case at::kFloat8_e4m3fn: return NEOX_F8;
            case at::kFloat4_e2m1fn_x2: return NEOX_F4;
            default: return code(like);
        }
    }
    bool coded() const { return k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == at::kFloat4_e2m1fn_x2; }
    int64_t dim() const { return k.size(3) * (k.scalar_type() == at::kFloat4_e2m1fn_x2 ? 2 : 1); }
    bool goes_with(const Tensor& like) const {
        return half_type(like) && (k_scale ? coded() : k.scalar_type() == like.scalar_type()) && k.device() == like.device() && k.dim() == 4 &&
               like.size(-1) == dim();
    }
};
RowStrides scale_strides(const std::optional<Tensor>& t) { return t ? RowStrides(*t, 3) : RowStrides(Tensor(), 0); }

bool slot_list(const Tensor& t, const Tensor& like) {
    return on_gpu(t) && t.device() == like.device() && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1 &&
           t.numel() > 0 && t.is_contiguous();
}

// k, v [tokens, heads, d] into slots [tokens]; whether that was done
bool cache_write(const Tensor& kc, const Tensor& vc, const std::optional<Tensor>& ks, const std::optional<Tensor>& vs, const Tensor& k,
                 const Tensor& v, const Tensor& slots) {
    const Cache cache{kc, vc, ks, vs};
    if (!on_gpu(k) || !on_gpu(v) || k.dim() != 3 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || v.device() != k.device() ||
        !cache.goes_with(k) || k.size(1) != kc.size(2) || !slot_list(slots, k) || slots.size(0) != k.size(0) || !in_pieces(k) || !in_pieces(v))
        return false;
    const c10::DeviceGuard guard(k.device());
    check(neox_cache_write(kc.mutable_data_ptr(), vc.mutable_data_ptr(), pointer_or_null<void>(ks), pointer_or_null<void>(vs),
                           k.const_data_ptr(), v.const_data_ptr(), slots.const_data_ptr(), slots.scalar_type() == at::kLong, k.size(0),
                           (int32_t)k.size(1), (int32_t)k.size(2), kc.size(0), (int32_t)kc.size(1), RowStrides(kc, 3), RowStrides(vc, 3),
                           scale_strides(ks), scale_strides(vs), RowStrides(k, 2), RowStrides(v, 2), code(k), cache.dtype(k), stream_of(k)));
    return true;
}

// the slots' keys and values in fp16 or bf16, or None
std::optional<std::tuple<Tensor, Tensor>> cache_read(const Tensor& kc, const Tensor& vc, const std::optional<Tensor>& ks,
                                                     const std::optional<Tensor>& vs, const Tensor& slots, at::ScalarType dtype) {
    if (!slot_list(slots, kc) || (dtype != at::kHalf && dtype != at::kBFloat16) || (!ks && dtype != kc.scalar_type())) return std::nullopt;
    const Cache cache{kc, vc, ks, vs};
    const c10::DeviceGuard guard(kc.device());
    Tensor k = at::empty({slots.size(0), kc.size(2), cache.dim()}, kc.options().dtype(dtype)), v = at::empty_like(k);
    check(neox_cache_read(k.mutable_data_ptr(), v.mutable_data_ptr(), kc.const_data_ptr(), vc.const_data_ptr(), pointer_or_null<const void>(ks),
                          pointer_or_null<const void>(vs), slots.const_data_ptr(), slots.scalar_type() == at::kLong, slots.size(0),
                          (int32_t)kc.size(2), (int32_t)cache.dim(), kc.size(0), (int32_t)kc.size(1), RowStrides(k, 2), RowStrides(v, 2),
                          RowStrides(kc, 3), RowStrides(vc, 3), scale_strides(ks), scale_strides(vs), code(k), cache.dtype(k), stream_of(k)));
    return std::make_tuple(k, v);
}

// q [tokens, h, d] over the pages of a cache -> [tokens, h, d], or None; max_context None: what the table has room for
std::optional<Tensor> paged_attention(const Tensor& q, const Tensor& kc, const Tensor& vc, const std::optional<Tensor>& ks,
                                      const std::optional<Tensor>& vs, const Tensor& table, const Tensor& starts, const Tensor& lengths,
                                      int64_t max_query, std::optional<int64_t> longest, double scale, int64_t window, int64_t sinks) {
    const Cache cache{kc, vc, ks, vs};
    if (!on_gpu(q) || q.dim() != 3 || q.numel() == 0 || !cache.goes_with(q) || q.size(1) % kc.size(2) != 0 || !fits_int32(q.size(0)) ||
        !in_pieces(q) || lengths.dim() != 1 || !int_list(lengths, q, lengths.size(0)) || !int_list(starts, q, lengths.size(0) + 1) ||
        !on_gpu(table) || table.device() != q.device() || table.scalar_type() != at::kInt || table.dim() != 2 ||
        table.size(0) != lengths.size(0) || table.size(0) < 1 || table.size(1) < 1 || table.stride(1) != 1 || table.stride(0) < 0 ||
        !fits_int32(table.size(1)) || !fits_int32(max_query) || window > INT32_MAX || window < -1 || !fits_int32(sinks))
        return std::nullopt;
    const int64_t max_context = longest.value_or(table.size(1) * kc.size(1));
    if (!fits_int32(max_context)) return std::nullopt;
    const c10::DeviceGuard guard(q.device());
    const auto tokens = (int32_t)q.size(0), h = (int32_t)q.size(1), d = (int32_t)q.size(2), b = (int32_t)lengths.size(0), h_kv = (int32_t)kc.size(2);
    Tensor out = at::empty(q.sizes(), q.options()), workspace;
    int64_t bytes = 0;
    check(neox_paged_attention_workspace(&bytes, b, tokens, (int32_t)max_query, (int32_t)max_context, h, h_kv, d, (int32_t)window, (int32_t)sinks));
    if (bytes) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
    check(neox_paged_attention(out.mutable_data_ptr(), bytes ? workspace.mutable_data_ptr() : nullptr, bytes, q.const_data_ptr(),
                               kc.const_data_ptr(), vc.const_data_ptr(), pointer_or_null<const void>(ks), pointer_or_null<const void>(vs),
                               static_cast<const int32_t*>(table.const_data_ptr()), static_cast<const int32_t*>(starts.const_data_ptr()),
                               static_cast<const int32_t*>(lengths.const_data_ptr()), b, tokens, (int32_t)max_query, (int32_t)max_context, h,
                               h_kv, d, kc.size(0), (int32_t)kc.size(1), (int32_t)table.size(1), table.size(0) > 1 ? table.stride(0) : 0,
                               RowStrides(out, 2), RowStrides(q, 2), RowStrides(kc, 3), RowStrides(vc, 3), scale_strides(ks),
                               scale_strides(vs), (float)scale, (int32_t)window, (int32_t)sinks, code(q), cache.dtype(q), stream_of(q)));
    return out;
}

// ---- the pages of caches ---------------------------------------------------------------------------
// The tensors of a PagePool, which has looked at them, and the numbers of a call, one for each sequence.
bool pool_list(const Tensor& t, const Tensor& lengths) { return int_list(t, lengths, lengths.size(0)); }
int64_t row_stride(const Tensor& table) { return table.size(0) > 1 ? table.stride(0) : 0; }
int32_t* words(const Tensor& t) { return static_cast<int32_t*>(t.mutable_data_ptr()); }

// `count` elements of `type`, `offset` of them behind the start of t's memory
Tensor part_of(const Tensor& t, at::ScalarType type, int64_t offset, int64_t count) {
    Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), c10::scalarTypeToTypeMeta(type));
    part.unsafeGetTensorImpl()->set_sizes_contiguous({count});
    part.unsafeGetTensorImpl()->set_storage_offset(offset);
    return part;
}

// starts, positions, slots and whether granted, or None
std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> pages_extend(const Tensor& table, const Tensor& lengths, const Tensor& free, const Tensor& left,
                                                                       const Tensor& tokens, int64_t page_size, int64_t max_tokens) {
    if (!pool_list(tokens, lengths) || max_tokens < 0 || max_tokens >= 1 << 30) return std::nullopt;
    const c10::DeviceGuard guard(table.device());
    const int64_t n = lengths.size(0);
    // one allocation: 64-bit words, 32-bit ones, the workspace, bytes (four of them and views of one took 2 us more of the host)
    const int64_t words64 = max_tokens, words32 = 2 * (n + 1) + max_tokens;
    const Tensor all = at::empty({words64 + (words32 + 1) / 2 + (n + 7) / 8}, lengths.options().dtype(at::kLong));
    auto* const base = static_cast<int64_t*>(all.mutable_data_ptr());
    auto* const base32 = reinterpret_cast<int32_t*>(base + words64);
    Tensor starts = part_of(all, at::kInt, 2 * words64, n + 1), positions = part_of(all, at::kInt, 2 * words64 + n + 1, max_tokens);
    Tensor slots = part_of(all, at::kLong, 0, max_tokens), granted = part_of(all, at::kBool, 8 * (words64 + (words32 + 1) / 2), n);
    check(neox_pages_extend(base32, base32 + n + 1, base, static_cast<uint8_t*>(granted.mutable_data_ptr()), base32 + n + 1 + max_tokens, words(table),
                            words(lengths), words(free), words(left), words(tokens), (int32_t)n, (int32_t)table.size(1), row_stride(table),
                            (int32_t)free.size(0), (int32_t)page_size, (int32_t)max_tokens, stream_of(table)));
    return std::make_tuple(starts, positions, slots, granted);
}

// whether that was done
bool pages_truncate(const Tensor& table, const Tensor& lengths, const Tensor& free, const Tensor& left, const Tensor& keep, int64_t page_size) {
    if (!pool_list(keep, lengths)) return false;
    const c10::DeviceGuard guard(table.device());
    check(neox_pages_truncate(words(table), words(lengths), words(free), words(left), words(keep), (int32_t)lengths.size(0), (int32_t)table.size(1),
                              row_stride(table), (int32_t)free.size(0), (int32_t)page_size, stream_of(table)));
    return true;
}

}  // namespace

// The interpreter is not held while a launch waits for room in its queue.  An exception that a saved-tensor hook
// raises (activation checkpointing ends its recomputation with one) comes back as what it is.
PYBIND11_MODULE(neox_torch, m) {
    namespace py = pybind11;
    using torch::wrap_pybind_function_no_gil;
    m.attr("abi_version") = NEOX_FUSED_ABI_VERSION;  // what this was compiled against, for the loader to compare
    m.attr("torch_version") = TORCH_VERSION;
    m.def("causal_softmax", wrap_pybind_function_no_gil(causal_softmax), py::arg("x"), py::arg("scale"), py::arg("window") = -1,
          py::arg("slopes") = std::optional<Tensor>(), py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0);
    m.def("causal_takes", wrap_pybind_function_no_gil(causal_takes), py::arg("x"), py::arg("slopes") = std::optional<Tensor>());
    m.def("masked_softmax", wrap_pybind_function_no_gil(masked_softmax), py::arg("x"), py::arg("mask"), py::arg("scale"));
    m.def("rotary", wrap_pybind_function_no_gil(rotary), py::arg("q"), py::arg("k"), py::arg("cos"), py::arg("sin"),
          py::arg("offset"));
    m.def("window_attention", wrap_pybind_function_no_gil(window_attention), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("scale"),
          py::arg("window"), py::arg("sinks"), py::arg("lengths"));
    m.def("cache_write", wrap_pybind_function_no_gil(cache_write));
    m.def("cache_read", wrap_pybind_function_no_gil(cache_read));
    m.def("paged_attention", wrap_pybind_function_no_gil(paged_attention));
    m.def("pages_extend", wrap_pybind_function_no_gil(pages_extend));
    m.def("pages_truncate", wrap_pybind_function_no_gil(pages_truncate));
    m.def("rope", wrap_pybind_function_no_gil(rope), py::arg("x"), py::arg("cos"), py::arg("sin"), py::arg("transposed"));
}
