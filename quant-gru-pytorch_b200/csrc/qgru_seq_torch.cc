// qgru_seq_torch.cc - torch binding of the sequence operators (linear attention, residual norm) over the C ABI of include/qgru.h.
//
// These calls are a few microseconds of GPU time where a token or a frame at a time goes through a stack of layers, and in Python
// their checks, argument blocks and autograd nodes took several times that: a step of one token 25 us, a norm with its gradient
// 123 us.  Arguments are checked here, tensors allocated by torch, and everything is queued on the current stream of their device.
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>

#include "qgru.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A status other than QGRU_OK and QGRU_ERR_BAD_ARG (which is a ValueError): raised as _cabi.QgruError.
struct Failure : std::runtime_error {
    int status;
    std::string where, detail;
    Failure(int s, const char *w, const char *d)
        : std::runtime_error(std::string(w) + ": " + qgru_status_string(s) + (*d ? " (" + std::string(d) + ")" : "")), status(s), where(w), detail(d) {}
};
void check(int status, const char *where) {
    if (status == QGRU_OK) return;
    const char *detail = qgru_seq_last_error();
    TORCH_CHECK_VALUE(status != QGRU_ERR_BAD_ARG, where, ": ", *detail ? detail : "bad argument");
    throw Failure(status, where, detail);
}

bool taken(const Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
void *ptr(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
int index_of(const Tensor &t) { return t.get_device(); }
void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
Tensor block(size_t bytes, const Tensor &like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }

std::optional<Tensor> some(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// t, or a dense copy where its last stride is not 1 or its rows could be fetched in 16-byte pieces but for where they lie.
Tensor readable(const Tensor &t) {
    if (t.numel() == 0) return t;
    const int64_t per = 16 / t.element_size(), last = t.dim() - 1;
    bool ok = t.stride(last) == 1;
    if (ok && t.size(last) % per == 0) {
        ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
        for (int64_t i = 0; ok && i < last; ++i) ok = t.stride(i) % per == 0;
    }
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
// A tensor saved for the backward, as it was: kernels go by its sizes and type.
constexpr const char *HOOKED = "a saved-tensor hook has returned another type, shape or device than it was given";
void check_saved(const Tensor &t, at::ScalarType type, at::IntArrayRef sizes, const Tensor &like) {
    TORCH_CHECK(t.defined() && t.scalar_type() == type && t.sizes() == sizes && t.device() == like.device(), HOOKED);
}
// What a backward computes has no gradient of its own: whoever differentiates it is told.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor &g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    return (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int)grads.size()))(std::move(grads));
}

// There is no forward-mode derivative: results without one would be taken for constants.
void check_tangents(std::initializer_list<const Tensor *> inputs) {
    for (const Tensor *t : inputs) TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "the sequence operators have no forward-mode derivative: an input has a tangent");
}

// The node that adds to a leaf's gradient lives as long as any graph of the leaf, with the stream that it was made on.  Where that is
// the default stream, a backward inside a capture on another one would have it wait for the captured work, which CUDA forbids and
// autograd does not survive.  Refused before anything is recorded.
void check_capture(std::initializer_list<const Tensor *> leaves) {
    for (const Tensor *t : leaves) {
        if (!t->defined() || !t->is_cuda() || !t->requires_grad() || !t->is_leaf()) continue;
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(t->get_device()).stream(), &capture) != cudaSuccess || capture == cudaStreamCaptureStatusNone) return;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto made_on = node ? node->stream() : std::nullopt;
        TORCH_CHECK(!made_on || *made_on != c10::cuda::getDefaultCUDAStream(t->get_device()).unwrap(),
                    "a graph of the same leaves that was made on the default stream still lives: release it (its outputs and losses) before the backward pass is captured");
    }
}

// ------------------------------------------------------------------------------------- linear attention
struct Sizes {
    int64_t T, B, H, Hk, Dk, Dv;
};

// Shapes and types; the log decay as [*lead, H].
Tensor check_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &decay, int64_t lead) {
    for (const auto &[name, t] : {std::pair<const char *, const Tensor &>("q", q), {"k", k}, {"v", v}}) {
        TORCH_CHECK_VALUE(t.is_cuda() && taken(t), name, " must be a CUDA tensor of float32 or bfloat16");
        TORCH_CHECK_VALUE(t.dim() == lead + 2, name, " must have ", lead + 2, " dimensions, got shape ", t.sizes());
    }
    TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.device() == q.device(), "k must be a ", q.scalar_type(), " tensor on ", q.device());
    TORCH_CHECK_VALUE(k.sizes() == q.sizes(), "k must have shape ", q.sizes(), ", got ", k.sizes());
    TORCH_CHECK_VALUE(v.scalar_type() == q.scalar_type() && v.device() == q.device() && v.sizes().slice(0, lead) == q.sizes().slice(0, lead), "v must be a ",
                      q.scalar_type(), " tensor on ", q.device(), " that begins with ", q.sizes().slice(0, lead), ", got ", v.sizes());
    const int64_t H = v.size(lead), Hk = q.size(lead);
    TORCH_CHECK_VALUE(H > 0 && Hk > 0 && q.size(lead + 1) > 0 && v.size(lead + 1) > 0, "heads and head sizes must be positive");
    TORCH_CHECK_VALUE(H % Hk == 0, H, " heads cannot share ", Hk, " heads of q and k");
    TORCH_CHECK_VALUE(decay.device() == q.device() && (decay.scalar_type() == at::kFloat || decay.scalar_type() == q.scalar_type()),
                      "log_decay must be a float32 or ", q.scalar_type(), " tensor on ", q.device());
    if (decay.dim() == 1 && decay.size(0) == H) {
        std::vector<int64_t> to(v.sizes().begin(), v.sizes().begin() + lead + 1);
        return decay.expand(to);
    }
    TORCH_CHECK_VALUE(decay.sizes() == v.sizes().slice(0, lead + 1), "log_decay must have shape [", H, "] or ", v.sizes().slice(0, lead + 1), ", got ", decay.sizes());
    return decay;
}
qgru_seq_tensor place(const Tensor &t, bool batch_first) {
    return {ptr(t), t.stride(batch_first ? 1 : 0), t.stride(batch_first ? 0 : 1), t.stride(2)};
}
qgru_attention head(const Sizes &n, const Tensor &q, const Tensor &decay, double scale) {
    qgru_attention a{};
    a.device = index_of(q);
    a.T = (int)n.T;
    a.B = (int)n.B;
    a.H = (int)n.H;
    a.Hk = (int)n.Hk;
    a.Dk = (int)n.Dk;
    a.Dv = (int)n.Dv;
    a.bf16 = q.scalar_type() == at::kBFloat16;
    a.decay_bf16 = decay.scalar_type() == at::kBFloat16;
    a.scale = (float)scale;
    return a;
}
Sizes sizes_of(const Tensor &q, const Tensor &v, bool batch_first) {
    const Sizes n{q.size(batch_first ? 1 : 0), q.size(batch_first ? 0 : 1), v.size(2), q.size(2), q.size(3), v.size(3)};
    for (const int64_t x : {n.T, n.B, n.H, n.Dk, n.Dv}) TORCH_CHECK_VALUE(x < (1ll << 31), "a dimension of ", x, " is too long");
    return n;
}

// out, state and, with `keep`, what the backward reads
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor &q0, const Tensor &k0, const Tensor &v0, const Tensor &decay, const Tensor &state0,
                                                     const Tensor &lengths, double scale, bool batch_first, bool keep) {
    const Tensor q = readable(q0), k = readable(k0), v = readable(v0);
    const Sizes n = sizes_of(q, v, batch_first);
    qgru_attention a = head(n, q, decay, scale);
    a.keep = keep;
    a.q = place(q, batch_first);
    a.k = place(k, batch_first);
    a.v = place(v, batch_first);
    a.decay = place(decay, batch_first);
    Tensor out = at::empty(v.sizes(), v.options()), state = at::empty({n.B, n.H, n.Dk, n.Dv}, q.options().dtype(at::kFloat));
    a.lengths = static_cast<const int32_t *>(ptr(lengths));
    a.state0 = static_cast<const float *>(ptr(state0));
    a.state = static_cast<float *>(ptr(state));
    a.out = place(out, batch_first);
    size_t states_bytes = 0, ws_bytes = 0;
    check(qgru_attention_sizes(&a, &states_bytes, &ws_bytes, nullptr), "qgru_attention_sizes");
    Tensor states = block(states_bytes, q), ws = block(ws_bytes, q);
    a.states = ptr(states);
    a.workspace = ptr(ws);
    a.states_bytes = states_bytes;
    a.workspace_bytes = ws_bytes;
    check(qgru_attention_forward(&a, stream_of(q)), "qgru_attention_forward");
    return {out, state, states};
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &decay, const std::optional<Tensor> &first,
                                 const std::optional<Tensor> &count, double scale, bool batch_first) {
        const Tensor state0 = first ? *first : Tensor(), lengths = count ? *count : Tensor();
        auto [out, state, states] = attention_forward(q, k, v, decay, state0, lengths, scale, batch_first, true);
        ctx->save_for_backward({q, k, v, decay, lengths, states});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["batch_first"] = batch_first;
        ctx->saved_data["states"] = (int64_t)(states.defined() ? states.numel() : 0);
        ctx->saved_data["has_state"] = state0.defined();
        ctx->saved_data["has_lengths"] = lengths.defined();
        ctx->saved_data["shape"] = std::vector<int64_t>{q.size(0), q.size(1), q.size(2), q.size(3), v.size(2), v.size(3)};
        ctx->saved_data["type"] = (int64_t)q.scalar_type();
        ctx->saved_data["decay_type"] = (int64_t)decay.scalar_type();
        ctx->set_materialize_grads(false);
        return {out, state};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list got(8);
        if (!grads[0].defined() && !grads[1].defined()) return got;
        {
            const at::NoGradGuard off;
            const bool batch_first = ctx->saved_data["batch_first"].toBool();
            const std::vector<int64_t> d = ctx->saved_data["shape"].toIntVector();
            const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
            const Tensor &like = grads[0].defined() ? grads[0] : grads[1], &decay = saved[3];
            for (int i = 0; i < 2; ++i) check_saved(saved[i], type, {d[0], d[1], d[2], d[3]}, like);
            check_saved(saved[2], type, {d[0], d[1], d[4], d[5]}, like);
            check_saved(decay, (at::ScalarType)ctx->saved_data["decay_type"].toInt(), {d[0], d[1], d[4]}, like);
            if (ctx->saved_data["has_lengths"].toBool()) check_saved(saved[4], at::kInt, {d[batch_first ? 0 : 1]}, like);
            const Tensor q = readable(saved[0]), k = readable(saved[1]), v = readable(saved[2]), lengths = saved[4].defined() ? saved[4].contiguous() : Tensor();
            Tensor states = saved[5];
            const int64_t states_size = ctx->saved_data["states"].toInt();
            if (states_size) {
                check_saved(states, at::kByte, {states_size}, like);
                if (!states.is_contiguous() || reinterpret_cast<uintptr_t>(states.data_ptr()) % 256) states = states.clone(at::MemoryFormat::Contiguous);
            }
            const Sizes n = sizes_of(q, v, batch_first);
            qgru_attention a = head(n, q, decay, ctx->saved_data["scale"].toDouble());
            a.keep = 1;
            const Tensor dout = grads[0].defined() ? readable(grads[0]) : at::zeros(v.sizes(), v.options());
            const Tensor dstate = grads[1].defined() ? grads[1].contiguous() : Tensor();
            a.q = place(q, batch_first);
            a.k = place(k, batch_first);
            a.v = place(v, batch_first);
            a.decay = place(decay, batch_first);
            a.dout = place(dout, batch_first);
            size_t states_bytes = 0, ws_bytes = 0;
            check(qgru_attention_sizes(&a, &states_bytes, nullptr, &ws_bytes), "qgru_attention_sizes");
            const Tensor ws = block(ws_bytes, q);
            const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
            const Tensor dg = at::empty(decay.sizes(), decay.options());
            const Tensor dstate0 = ctx->saved_data["has_state"].toBool() && ctx->needs_input_grad(4) ? at::empty({n.B, n.H, n.Dk, n.Dv}, q.options().dtype(at::kFloat)) : Tensor();
            a.lengths = static_cast<const int32_t *>(ptr(lengths));
            a.dstate = static_cast<const float *>(ptr(dstate));
            a.dstate0 = static_cast<float *>(ptr(dstate0));
            a.states = ptr(states);
            a.workspace = ptr(ws);
            a.states_bytes = states_bytes;
            a.workspace_bytes = ws_bytes;
            a.dq = place(dq, batch_first);
            a.dk = place(dk, batch_first);
            a.dv = place(dv, batch_first);
            a.ddecay = place(dg, batch_first);
            check(qgru_attention_backward(&a, stream_of(q)), "qgru_attention_backward");
            got[0] = dq;
            got[1] = dk;
            got[2] = dv;
            got[3] = dg;
            got[4] = dstate0;
        }
        return once(std::move(got));
    }
};

std::tuple<Tensor, Tensor> linear_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const std::optional<Tensor> &initial_state,
                                            const std::optional<Tensor> &lengths, std::optional<double> scale, bool batch_first) {
    const Tensor decay = check_attention(q, k, v, log_decay, 2);
    const int64_t B = q.size(batch_first ? 0 : 1);
    Tensor state0, n;
    if (initial_state) {
        const std::vector<int64_t> want{B, v.size(2), q.size(3), v.size(3)};
        TORCH_CHECK_VALUE(initial_state->scalar_type() == at::kFloat && initial_state->device() == q.device() && initial_state->sizes() == want,
                          "initial_state must be a float32 tensor of shape ", want, " on ", q.device(), ", got ", initial_state->sizes());
        state0 = initial_state->contiguous();
    }
    if (lengths) {
        TORCH_CHECK_VALUE(lengths->scalar_type() == at::kInt && lengths->device() == q.device() && lengths->dim() == 1 && lengths->size(0) == B,
                          "lengths must be an int32 tensor of shape [", B, "] on ", q.device());
        n = lengths->contiguous();
    }
    const double s = scale ? *scale : 1.0 / std::sqrt((double)q.size(3));
    check_tangents({&q, &k, &v, &decay, &state0});
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || decay.requires_grad() || (state0.defined() && state0.requires_grad()))) {
        check_capture({&q, &k, &v, &log_decay, &state0});
        const variable_list r = LinearAttention::apply(q, k, v, decay, some(state0), some(n), s, batch_first);
        return {r[0], r[1]};
    }
    auto [out, state, states] = attention_forward(q, k, v, decay, state0, n, s, batch_first, false);
    return {out, state};
}

Tensor linear_attention_step(const Tensor &q0, const Tensor &k0, const Tensor &v0, const Tensor &log_decay, const Tensor &state, std::optional<double> scale) {
    const Tensor decay = check_attention(q0, k0, v0, log_decay, 1);
    TORCH_CHECK(!at::GradMode::is_enabled() || !(q0.requires_grad() || k0.requires_grad() || v0.requires_grad() || decay.requires_grad() || state.requires_grad()),
                "linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention with T = 1");
    check_tangents({&q0, &k0, &v0, &decay, &state});
    const Sizes n{1, q0.size(0), v0.size(1), q0.size(1), q0.size(2), v0.size(2)};
    const std::vector<int64_t> want{n.B, n.H, n.Dk, n.Dv};
    TORCH_CHECK_VALUE(state.scalar_type() == at::kFloat && state.device() == q0.device() && state.sizes() == want, "state must be a float32 tensor of shape ", want, " on ",
                      q0.device(), ", got ", state.sizes());
    const int64_t bs = state.stride(0), hs = state.stride(1), one = n.Dk * n.Dv;
    const bool dense = (state.stride(3) == 1 || n.Dv == 1) && (state.stride(2) == n.Dv || n.Dk == 1);
    const bool apart = (n.H == 1 || hs >= one) && (n.B == 1 || bs >= one) && (n.H == 1 || n.B == 1 || bs >= n.H * hs || hs >= n.B * bs);
    TORCH_CHECK_VALUE(n.B == 0 || (dense && apart), "a head's state must be dense and the states must not overlap, got strides ", state.strides());
    const Tensor q = readable(q0), k = readable(k0), v = readable(v0), out = at::empty({n.B, n.H, n.Dv}, q.options());
    qgru_attention a = head(n, q, decay, scale ? *scale : 1.0 / std::sqrt((double)n.Dk));
    a.state = static_cast<float *>(ptr(state));
    const auto at = [](const Tensor &t) { return qgru_seq_tensor{ptr(t), 0, t.stride(0), t.stride(1)}; };
    a.q = at(q);
    a.k = at(k);
    a.v = at(v);
    a.decay = at(decay);
    a.out = at(out);
    state.unsafeGetTensorImpl()->bump_version();           // (raises where the state must not be written)
    check(qgru_attention_step(&a, bs, hs, stream_of(q)), "qgru_attention_step");
    return out;
}

// ------------------------------------------------------------------------------------- norm
void check_norm(const Tensor &x, const Tensor &weight, const Tensor &residual) {
    TORCH_CHECK_VALUE(x.is_cuda() && taken(x), "x must be a CUDA tensor of float32 or bfloat16");
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "x must have at least one feature, got shape ", x.sizes());
    TORCH_CHECK_VALUE(weight.device() == x.device() && taken(weight), "weight must be a tensor of float32 or bfloat16 on ", x.device());
    TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1), "weight must have shape [", x.size(-1), "], got ", weight.sizes());
    if (residual.defined())
        TORCH_CHECK_VALUE(residual.device() == x.device() && residual.scalar_type() == x.scalar_type() && residual.sizes() == x.sizes(), "residual must be a ",
                          x.scalar_type(), " tensor of shape ", x.sizes(), " on ", x.device());
}
// A tensor as rows: features next to each other (a copy where its strides do not allow a view).
Tensor rows_of(const Tensor &t) {
    const int64_t d = t.size(-1), n = t.numel() / d;
    if (t.dim() == 2 && t.stride(1) == 1) return t;
    const Tensor r = t.reshape({n, d});
    return r.stride(1) == 1 || d == 1 ? r : r.contiguous();
}
qgru_norm norm_head(const Tensor &rows, const Tensor &weight) {
    TORCH_CHECK_VALUE(rows.size(1) < (1ll << 31), "a row of ", rows.size(1), " is too long");
    qgru_norm n{};
    n.device = index_of(rows);
    n.bf16 = rows.scalar_type() == at::kBFloat16;
    n.weight_bf16 = weight.scalar_type() == at::kBFloat16;
    n.cols = (int)rows.size(1);
    n.rows = rows.size(0);
    n.weight = ptr(weight);
    return n;
}
qgru_norm norm_inputs(const Tensor &x, const Tensor &weight, const Tensor &residual, const Tensor &h, double eps) {
    qgru_norm n = norm_head(x, weight);
    n.eps = (float)eps;
    n.x = ptr(x);
    n.x_stride = x.stride(0);
    if (residual.defined()) {
        n.residual = ptr(residual);
        n.residual_stride = residual.stride(0);
        n.h_out = ptr(h);
        n.h_stride = n.cols;
    }
    return n;
}
// y, h (undefined without a residual), rstd where wanted
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps, bool keep) {
    const Tensor x2 = rows_of(x), w = weight.contiguous(), r2 = residual.defined() ? rows_of(residual) : Tensor();
    Tensor y = at::empty(x.sizes(), x.options()), h = residual.defined() ? at::empty(x.sizes(), x.options()) : Tensor();
    Tensor rstd = keep ? at::empty({x2.size(0)}, x.options().dtype(at::kFloat)) : Tensor();
    qgru_norm n = norm_inputs(x2, w, r2, h, eps);
    n.y = ptr(y);
    n.y_stride = n.cols;
    n.rstd = static_cast<float *>(ptr(rstd));
    check(qgru_norm_forward(&n, stream_of(x)), "qgru_norm_forward");
    return {y, h, rstd};
}
struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const std::optional<Tensor> &residual, double eps) {
        auto [y, h, rstd] = norm_forward(x, weight, residual ? *residual : Tensor(), eps, true);
        ctx->save_for_backward({h.defined() ? h : x, weight, rstd});
        ctx->saved_data["residual"] = h.defined();
        ctx->saved_data["weight_type"] = (int64_t)weight.scalar_type();
        ctx->set_materialize_grads(false);
        if (!h.defined()) return {y};
        return {y, h};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const bool residual = ctx->saved_data["residual"].toBool();
        const Tensor dy = grads[0], dh = residual ? grads[1] : Tensor();
        variable_list got(4);
        if (!dy.defined()) {                    // only the stream goes on
            got[0] = dh;
            if (residual) got[2] = dh;
            return got;
        }
        {
            const at::NoGradGuard off;
            check_saved(saved[0], dy.scalar_type(), dy.sizes(), dy);
            check_saved(saved[1], (at::ScalarType)ctx->saved_data["weight_type"].toInt(), {dy.size(-1)}, dy);
            check_saved(saved[2], at::kFloat, {dy.numel() / dy.size(-1)}, dy);
            const Tensor h2 = rows_of(saved[0]), weight = saved[1].contiguous(), rstd = saved[2].contiguous(), dy2 = rows_of(dy), dh2 = dh.defined() ? rows_of(dh) : Tensor();
            const Tensor dx = at::empty(saved[0].sizes(), saved[0].options()), dw = ctx->needs_input_grad(1) ? at::empty(weight.sizes(), weight.options()) : Tensor();
            qgru_norm n = norm_head(h2, weight);
            n.rstd = static_cast<float *>(ptr(rstd));
            const size_t bytes = dw.defined() ? qgru_norm_workspace(n.device, n.rows, n.cols) : 0;
            const Tensor ws = block(bytes, h2);
            check(qgru_norm_backward(&n, ptr(h2), h2.stride(0), ptr(dy2), dy2.stride(0), ptr(dh2), dh2.defined() ? dh2.stride(0) : 0, ptr(dx), n.cols, ptr(dw), ptr(ws), bytes,
                                     stream_of(h2)),
                  "qgru_norm_backward");
            got[0] = dx;
            got[1] = dw;
            if (residual) got[2] = dx;
        }
        return once(std::move(got));
    }
};

py::object rms_norm(const Tensor &x, const Tensor &weight, const std::optional<Tensor> &residual, double eps) {
    const Tensor r = residual ? *residual : Tensor();
    check_norm(x, weight, r);
    check_tangents({&x, &weight, &r});
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (r.defined() && r.requires_grad()))) {
        check_capture({&x, &weight, &r});
        const variable_list got = RmsNorm::apply(x, weight, some(r), eps);
        return got.size() == 1 ? py::cast(got[0]) : py::make_tuple(got[0], got[1]);
    }
    auto [y, h, rstd] = norm_forward(x, weight, r, eps, false);
    return h.defined() ? py::make_tuple(y, h) : py::cast(y);
}

py::object rms_norm_q8(const Tensor &x, const Tensor &weight, const std::optional<Tensor> &residual, double eps, std::optional<double> scale, int64_t zero_point, int64_t bits,
                       bool is_unsigned) {
    const Tensor r = residual ? *residual : Tensor();
    check_norm(x, weight, r);
    TORCH_CHECK(!at::GradMode::is_enabled() || !r.defined() || !(x.requires_grad() || r.requires_grad()),
                "rms_norm_q8 has no gradient, and the stream that it returns would end the residual's: call it under torch.no_grad()");
    if (r.defined()) check_tangents({&x, &r});
    const at::NoGradGuard off;
    const Tensor x2 = rows_of(x), w = weight.contiguous(), r2 = r.defined() ? rows_of(r) : Tensor(), h = r.defined() ? at::empty(x.sizes(), x.options()) : Tensor();
    const Tensor q = at::empty(x.sizes(), x.options().dtype(scale && is_unsigned ? at::kByte : at::kChar));
    const Tensor scales = scale ? Tensor() : at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    qgru_norm n = norm_inputs(x2, w, r2, h, eps);
    n.q8 = ptr(q);
    n.scales = static_cast<float *>(ptr(scales));
    if (scale) {
        n.q8_scale = (float)*scale;
        TORCH_CHECK_VALUE(n.q8_scale > 0.f && std::isfinite(n.q8_scale) && bits >= 1 && bits <= 8, "scale must be positive and bits between 1 and 8, got ", *scale, " and ", bits);
        TORCH_CHECK_VALUE(zero_point > -(1 << 24) && zero_point < 1 << 24, "zero_point ", zero_point, " is out of range");
        n.q8_zero_point = (int)zero_point;
        n.q8_lo = is_unsigned ? 0 : -(1 << (bits - 1));
        n.q8_hi = is_unsigned ? (1 << bits) - 1 : (1 << (bits - 1)) - 1;
    }
    check(qgru_norm_forward(&n, stream_of(x)), "qgru_norm_forward");
    if (scale) return h.defined() ? py::make_tuple(q, h) : py::cast(q);
    return h.defined() ? py::make_tuple(q, scales, h) : py::make_tuple(q, scales);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure &e) {
            const py::object type = py::module_::import("quant_gru_pytorch_b200._cabi").attr("QgruError");
            const py::object error = type(e.status, e.where, e.detail);
            PyErr_SetObject(type.ptr(), error.ptr());
        }
    });
    m.def("linear_attention", &linear_attention);
    m.def("linear_attention_step", &linear_attention_step);
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_q8", &rms_norm_q8);
}
