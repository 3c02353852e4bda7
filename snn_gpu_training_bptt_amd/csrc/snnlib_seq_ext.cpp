// The token-layer operators of module `snnlib`: embedding, group norm with an activation, gated delta rule.
//
//   embed_fp(tokens, weight, scale) -> out
//   embed_bp(tokens, grad_out, vocab, scale) -> grad_weight
//   gn_act_fp(x, weight_gn, bias_gn, groups, eps_gn, act) -> [mean, rstd, y]
//   gn_act_bp(x, weight_gn, bias_gn, mean, rstd, groups, act, grad_y) -> [grad_x, grad_weight_gn, grad_bias_gn]
//   gated_delta_fp(q, k, v, g, beta, state, lengths, scale, for_backward) -> [o, state_out, saved]
//   gated_delta_bp(q, k, v, g, beta, state, lengths, scale, saved, grad_o, grad_state_out)
//                  -> [grad_q, grad_k, grad_v, grad_g, grad_beta, grad_state]
//   gated_delta_step(q, k, v, g, beta, state, scale, state_out) -> o
//
// and, differentiable, embed(tokens, weight, scale), gn_act(x, weight_gn, bias_gn, groups, eps_gn, act) and
// gated_delta(q, k, v, g, beta, state, lengths, scale) -> (o, state_out).  Their autograd functions are here and not in
// Python, unlike the fire layers': on a few thousand tokens the kernels of a forward and backward are over in 16 us, and
// two Python frames and the wait for the interpreter in the backward's thread cost 4 us more than these (embedding of 1665
// tokens in a loop: 38 us a pass, 34 here, 16 without autograd).
//
// As in snnlib_ext.cpp: this file validates tensors, allocates outputs and workspaces and forwards raw device
// pointers to the C ABI (include/snnlib_seq.h) on the current stream of the tensors' device; it holds no device
// code and no fallback.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <string>
#include <vector>

#include "snnlib_seq.h"

namespace {

using torch::Tensor;
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

// What would come out wrong without an error.  A tracer records the allocation of an output and not the kernel that fills
// it: the graph would return whatever the memory holds.  And the kernels know nothing of tangents: an operand that carries
// one would give a result without, a derivative of zero.
void check_eager(const char* op, std::initializer_list<const Tensor*> operands) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                "snnlib.", op, ": cannot be recorded by torch.jit.trace or make_fx");
    for (const Tensor* t : operands)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "snnlib.", op,
                    ": forward-mode derivatives are not supported");
}

void check_on_gpu(const Tensor& t, const char* op, const char* name) {
    TORCH_CHECK(t.defined(), "snnlib.", op, ": ", name, " is undefined");
    TORCH_CHECK(t.is_cuda(), "snnlib.", op, ": ", name,
                " must live on a ROCm GPU (this build has no CPU path), got device ", t.device());
    // a fake tensor's address is its offset alone, and a kernel would follow it
    TORCH_CHECK(t.numel() == 0 || t.storage().data() != nullptr, "snnlib.", op, ": ", name, " has no memory (a fake tensor)");
}

int storage_dtype(const Tensor& t, const char* op, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return SNNLIF_DTYPE_F32;
        case at::kDouble: return SNNLIF_DTYPE_F64;
        case at::kBFloat16: return SNNLIF_DTYPE_BF16;
        default:
            TORCH_CHECK(false, "snnlib.", op, ": unsupported dtype ", t.scalar_type(), " of ", name,
                        " (supported: float32, float64, bfloat16)");
    }
    return -1;
}

void check_like(const Tensor& t, const Tensor& like, const char* op, const char* name, const char* like_name) {
    check_on_gpu(t, op, name);
    TORCH_CHECK(t.device() == like.device(), "snnlib.", op, ": ", name, " (", t.device(), ") must be on the device of ",
                like_name, " (", like.device(), ")");
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), "snnlib.", op, ": ", name, " (", t.scalar_type(),
                ") must have the dtype of ", like_name, " (", like.scalar_type(), ")");
}

void check_rc(int rc, const char* op) {
    TORCH_CHECK(rc == SNNLIF_OK, "snnlib.", op, ": ", snnlif_strerror(rc), " (code ", rc, ")");
}

void* current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

Tensor dense(const Tensor& t) { return t.contiguous(); }

// A workspace from the caching allocator: it goes back on return and stays valid for the work already queued,
// because later users are ordered on the same stream.
Tensor workspace_of(size_t bytes, const Tensor& like) {
    return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// ---- embedding ----------------------------------------------------------------------------------

int token_dtype(const Tensor& tokens, const char* op) {
    check_on_gpu(tokens, op, "tokens");
    TORCH_CHECK(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "snnlib.", op,
                ": tokens must be int64 or int32, got ", tokens.scalar_type());
    return tokens.scalar_type() == at::kLong ? SNNSEQ_TOKEN_I64 : SNNSEQ_TOKEN_I32;
}

Tensor embed_fp(Tensor tokens, Tensor weight, double scale) {
    const char* op = "embed_fp";
    check_eager(op, {&weight});
    const int tdtype = token_dtype(tokens, op);
    check_on_gpu(weight, op, "weight");
    TORCH_CHECK(weight.device() == tokens.device(), "snnlib.", op, ": weight (", weight.device(),
                ") must be on the device of tokens (", tokens.device(), ")");
    const int dtype = storage_dtype(weight, op, "weight");
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0, "snnlib.", op,
                ": weight must be [vocab, cout] with at least one row, got ", weight.sizes());
    const DeviceGuard guard(weight.device());
    Tensor ids = dense(tokens);
    Tensor table = weight.size(1) > 1 && weight.stride(1) != 1 ? dense(weight) : weight;  // rows may lie apart
    std::vector<int64_t> sizes = tokens.sizes().vec();
    sizes.push_back(weight.size(1));
    Tensor out = torch::empty(sizes, weight.options());
    check_rc(snnseq_embed_fp(ids.data_ptr(), table.data_ptr(), out.data_ptr(), dtype, tdtype, ids.numel(),
                             table.size(0), table.size(1), table.stride(0), scale, current_stream()),
             op);
    return out;
}

Tensor embed_bp(Tensor tokens, Tensor grad_out, int64_t vocab, double scale) {
    const char* op = "embed_bp";
    check_eager(op, {&grad_out});
    const int tdtype = token_dtype(tokens, op);
    check_on_gpu(grad_out, op, "grad_out");
    TORCH_CHECK(grad_out.device() == tokens.device(), "snnlib.", op, ": grad_out (", grad_out.device(),
                ") must be on the device of tokens (", tokens.device(), ")");
    const int dtype = storage_dtype(grad_out, op, "grad_out");
    TORCH_CHECK(vocab > 0, "snnlib.", op, ": vocab must be positive, got ", vocab);
    TORCH_CHECK(grad_out.dim() == tokens.dim() + 1 &&
                    grad_out.sizes().slice(0, tokens.dim()) == tokens.sizes(),
                "snnlib.", op, ": grad_out must be [", tokens.sizes(), ", cout], got ", grad_out.sizes());
    const DeviceGuard guard(grad_out.device());
    Tensor ids = dense(tokens), g = dense(grad_out);
    const int64_t C = g.size(-1);
    Tensor grad_weight = torch::empty({vocab, C}, g.options());
    const size_t ws_bytes = snnseq_embed_bp_workspace_bytes(dtype, ids.numel(), vocab, C);
    Tensor workspace = workspace_of(ws_bytes, g);
    check_rc(snnseq_embed_bp(ids.data_ptr(), g.data_ptr(), grad_weight.data_ptr(), dtype, tdtype, ids.numel(), vocab, C,
                             scale, workspace.data_ptr(), ws_bytes, current_stream()),
             op);
    return grad_weight;
}

// ---- group norm with an activation --------------------------------------------------------------

int act_code(const std::string& act, const char* op) {
    if (act == "none") return SNNSEQ_ACT_NONE;
    if (act == "relu") return SNNSEQ_ACT_RELU;
    if (act == "silu") return SNNSEQ_ACT_SILU;
    if (act == "gelu") return SNNSEQ_ACT_GELU;
    TORCH_CHECK(false, "snnlib.", op, ": unknown activation '", act, "' (none, relu, silu, gelu)");
    return -1;
}

struct GnOperands {
    int64_t S, P, C;
    int dtype;
    Tensor x, weight, bias;
};

GnOperands gn_operands(const Tensor& x, const Tensor& weight_gn, const Tensor& bias_gn, int64_t groups,
                       const char* op) {
    check_on_gpu(x, op, "x");
    GnOperands o;
    o.dtype = storage_dtype(x, op, "x");
    TORCH_CHECK(x.dim() >= 3, "snnlib.", op, ": x must be shaped [T, B, ..., C], got ", x.sizes());
    o.C = x.size(-1);
    o.S = x.size(0) * x.size(1);
    o.P = 1;
    for (int64_t d = 2; d + 1 < x.dim(); ++d) o.P *= x.size(d);
    TORCH_CHECK(groups > 0 && o.C % groups == 0, "snnlib.", op, ": groups (", groups,
                ") must divide the channels (", o.C, ")");
    TORCH_CHECK(o.S == 0 || (o.P > 0 && o.C > 0), "snnlib.", op, ": no values per group in a tensor shaped ",
                x.sizes());
    for (const auto& p : {std::make_pair(&weight_gn, "weight_gn"), std::make_pair(&bias_gn, "bias_gn")}) {
        check_like(*p.first, x, op, p.second, "x");
        TORCH_CHECK(p.first->dim() == 1 && p.first->size(0) == o.C, "snnlib.", op, ": ", p.second,
                    " must have one value per channel (", o.C, "), got ", p.first->sizes());
    }
    o.x = dense(x);
    o.weight = dense(weight_gn);
    o.bias = dense(bias_gn);
    return o;
}

std::vector<Tensor> gn_act_fp(Tensor x, Tensor weight_gn, Tensor bias_gn, int64_t groups, double eps_gn,
                              const std::string& act) {
    const char* op = "gn_act_fp";
    check_eager(op, {&x, &weight_gn, &bias_gn});
    const int code = act_code(act, op);
    TORCH_CHECK(eps_gn >= 0, "snnlib.", op, ": eps_gn must not be negative, got ", eps_gn);
    check_on_gpu(x, op, "x");
    const DeviceGuard guard(x.device());
    const GnOperands o = gn_operands(x, weight_gn, bias_gn, groups, op);
    Tensor y = torch::empty(o.x.sizes(), o.x.options());
    const auto stat = o.x.options().dtype(o.dtype == SNNLIF_DTYPE_F64 ? at::kDouble : at::kFloat);
    Tensor mean = torch::empty({o.x.size(0), o.x.size(1), groups}, stat);
    Tensor rstd = torch::empty({o.x.size(0), o.x.size(1), groups}, stat);
    const size_t ws_bytes = snnseq_gn_act_workspace_bytes(o.dtype, o.S, o.P, o.C, groups, 0);
    Tensor workspace;
    if (ws_bytes > 0) workspace = workspace_of(ws_bytes, o.x);
    check_rc(snnseq_gn_act_fp(o.x.data_ptr(), o.weight.data_ptr(), o.bias.data_ptr(), y.data_ptr(), mean.data_ptr(),
                              rstd.data_ptr(), o.dtype, o.S, o.P, o.C, groups, eps_gn, code,
                              ws_bytes ? workspace.data_ptr() : nullptr, ws_bytes, current_stream()),
             op);
    return {mean, rstd, y};
}

std::vector<Tensor> gn_act_bp(Tensor x, Tensor weight_gn, Tensor bias_gn, Tensor mean, Tensor rstd, int64_t groups,
                              const std::string& act, Tensor grad_y) {
    const char* op = "gn_act_bp";
    check_eager(op, {&x, &weight_gn, &bias_gn, &mean, &rstd, &grad_y});
    const int code = act_code(act, op);
    check_on_gpu(x, op, "x");
    const DeviceGuard guard(x.device());
    const GnOperands o = gn_operands(x, weight_gn, bias_gn, groups, op);
    check_like(grad_y, x, op, "grad_y", "x");
    TORCH_CHECK(grad_y.sizes() == x.sizes(), "snnlib.", op, ": grad_y ", grad_y.sizes(), " and x ", x.sizes(),
                " must have the same shape");
    const auto stat = o.dtype == SNNLIF_DTYPE_F64 ? at::kDouble : at::kFloat;
    for (const auto& p : {std::make_pair(&mean, "mean"), std::make_pair(&rstd, "rstd")}) {
        check_on_gpu(*p.first, op, p.second);
        TORCH_CHECK(p.first->device() == x.device() && p.first->scalar_type() == stat &&
                        p.first->numel() == o.S * groups,
                    "snnlib.", op, ": ", p.second, " must be what gn_act_fp returned for this x");
    }
    Tensor m = dense(mean), r = dense(rstd), g = dense(grad_y);
    Tensor grad_x = torch::empty(o.x.sizes(), o.x.options());
    // an empty batch contributes nothing to the parameter gradients; otherwise every channel is written
    Tensor grad_weight = o.S == 0 ? torch::zeros({o.C}, o.x.options()) : torch::empty({o.C}, o.x.options());
    Tensor grad_bias = torch::empty_like(grad_weight);
    if (o.S == 0) grad_bias.zero_();
    const size_t ws_bytes = snnseq_gn_act_workspace_bytes(o.dtype, o.S, o.P, o.C, groups, 1);
    Tensor workspace = workspace_of(ws_bytes, o.x);
    check_rc(snnseq_gn_act_bp(o.x.data_ptr(), o.weight.data_ptr(), o.bias.data_ptr(), m.data_ptr(), r.data_ptr(),
                              g.data_ptr(), grad_x.data_ptr(), grad_weight.data_ptr(), grad_bias.data_ptr(), o.dtype,
                              o.S, o.P, o.C, groups, code, workspace.data_ptr(), ws_bytes, current_stream()),
             op);
    return {grad_x, grad_weight, grad_bias};
}

bool records(std::initializer_list<const Tensor*> tensors);   // whether autograd would record an operator on these

// ---- gated delta rule ---------------------------------------------------------------------------

using MaybeTensor = c10::optional<Tensor>;

struct DeltaOperands {
    snnseq_delta call;
    Tensor q, k, v, g, beta, state, lengths;   // what the call points into
    bool has_state = false;
};

// Rows of values must be dense; any other layout is taken as it lies.
Tensor dense_rows(const Tensor& t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }

void strides_of(const Tensor& t, int64_t (&strides)[3]) {
    const int64_t d = t.dim();
    strides[0] = d == 4 ? t.stride(0) : 0;
    strides[1] = t.stride(d - 3);
    strides[2] = t.stride(d - 2);
}

// rank 4: [T, B, H, D] operands; rank 3: one step, [B, H, D].
DeltaOperands delta_operands(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                             const MaybeTensor& state, const MaybeTensor& lengths, double scale, int64_t rank,
                             const char* op) {
    const char* shape = rank == 4 ? "[T, B, heads, D]" : "[B, heads, D]";
    check_on_gpu(q, op, "q");
    TORCH_CHECK(q.scalar_type() == at::kFloat || q.scalar_type() == at::kBFloat16, "snnlib.", op,
                ": only float32 and bfloat16 are supported, got ", q.scalar_type());
    check_like(k, q, op, "k", "q");
    check_like(v, q, op, "v", "q");
    TORCH_CHECK(q.dim() == rank && v.dim() == rank, "snnlib.", op, ": q, k and v must be shaped ", shape, ", got ",
                q.sizes(), ", ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK(q.sizes() == k.sizes(), "snnlib.", op, ": q ", q.sizes(), " and k ", k.sizes(), " must have the same shape");
    TORCH_CHECK(v.sizes().slice(0, rank - 2) == q.sizes().slice(0, rank - 2), "snnlib.", op, ": v ", v.sizes(),
                " must share the time steps and batch entries of q ", q.sizes());
    const int64_t Hk = q.size(-2), Hv = v.size(-2), Dk = q.size(-1), Dv = v.size(-1), B = q.size(rank - 3);
    TORCH_CHECK(Hk > 0 && Hv > 0 && Hv % Hk == 0, "snnlib.", op, ": the heads of v (", Hv,
                ") must be a multiple of the heads of q and k (", Hk, ")");
    TORCH_CHECK(Dk > 0 && Dk <= SNNSEQ_MAX_KEY, "snnlib.", op, ": keys of 1 to ", SNNSEQ_MAX_KEY,
                " values are supported, got ", Dk);
    TORCH_CHECK(Dv > 0 && Dv <= SNNSEQ_MAX_VALUE, "snnlib.", op, ": values of 1 to ", SNNSEQ_MAX_VALUE,
                " values are supported, got ", Dv);
    TORCH_CHECK(B * Hv <= SNNSEQ_MAX_HEADS, "snnlib.", op, ": at most ", SNNSEQ_MAX_HEADS,
                " batch entries times heads, got ", B * Hv);
    for (const auto& p : {std::make_pair(&g, "g"), std::make_pair(&beta, "beta")}) {
        check_on_gpu(*p.first, op, p.second);
        TORCH_CHECK(p.first->device() == q.device(), "snnlib.", op, ": ", p.second, " must be on the device of q");
        TORCH_CHECK(p.first->scalar_type() == at::kFloat, "snnlib.", op, ": ", p.second, " must be float32, got ",
                    p.first->scalar_type());
        TORCH_CHECK(p.first->sizes() == v.sizes().slice(0, rank - 1), "snnlib.", op, ": ", p.second,
                    " must have one value per row of v (", v.sizes().slice(0, rank - 1), "), got ", p.first->sizes());
    }
    DeltaOperands o;
    o.q = dense_rows(q);
    o.k = dense_rows(k);
    o.v = dense_rows(v);
    o.g = dense(g);
    o.beta = dense(beta);
    if (state.has_value() && state->defined()) {
        check_on_gpu(*state, op, "state");
        TORCH_CHECK(state->device() == q.device() && state->scalar_type() == at::kFloat && state->dim() == 4 &&
                        state->size(0) == B && state->size(1) == Hv && state->size(2) == Dk && state->size(3) == Dv,
                    "snnlib.", op, ": state must be float32 [B, heads of v, Dk, Dv] on the device of q, got ",
                    state->scalar_type(), " ", state->sizes());
        o.state = dense(*state);
        o.has_state = true;
    }
    if (lengths.has_value() && lengths->defined()) {
        check_on_gpu(*lengths, op, "lengths");
        TORCH_CHECK(lengths->device() == q.device() && lengths->scalar_type() == at::kInt && lengths->dim() == 1 &&
                        lengths->size(0) == B,
                    "snnlib.", op, ": lengths must be int32 [B] on the device of q, got ", lengths->scalar_type(), " ",
                    lengths->sizes());
        o.lengths = dense(*lengths);
    }
    snnseq_delta& c = o.call;
    c = snnseq_delta{};
    c.T = rank == 4 ? q.size(0) : 1;
    c.B = B; c.Hk = Hk; c.Hv = Hv; c.Dk = Dk; c.Dv = Dv;
    strides_of(o.q, c.q_strides);
    strides_of(o.k, c.k_strides);
    strides_of(o.v, c.v_strides);
    c.scale = scale;
    c.q = o.q.data_ptr(); c.k = o.k.data_ptr(); c.v = o.v.data_ptr();
    c.g = o.g.data_ptr<float>(); c.beta = o.beta.data_ptr<float>();
    c.state = o.has_state ? o.state.data_ptr<float>() : nullptr;
    c.lengths = o.lengths.defined() ? o.lengths.data_ptr<int32_t>() : nullptr;
    c.dtype = q.scalar_type() == at::kFloat ? SNNLIF_DTYPE_F32 : SNNLIF_DTYPE_BF16;
    return o;
}

std::vector<Tensor> gated_delta_fp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, MaybeTensor state,
                                   MaybeTensor lengths, double scale, bool for_backward) {
    const char* op = "gated_delta_fp";
    const Tensor initial = state.value_or(Tensor());
    check_eager(op, {&q, &k, &v, &g, &beta, &initial});
    check_on_gpu(q, op, "q");
    const DeviceGuard guard(q.device());
    const DeltaOperands d = delta_operands(q, k, v, g, beta, state, lengths, scale, 4, op);
    Tensor o = torch::empty(v.sizes(), v.options());
    Tensor state_out = torch::empty({d.call.B, d.call.Hv, d.call.Dk, d.call.Dv}, d.g.options());
    const size_t bytes = snnseq_gated_delta_saved_bytes(&d.call, for_backward);
    Tensor saved = workspace_of(bytes, o);
    check_rc(snnseq_gated_delta_fp(&d.call, o.data_ptr(), state_out.data_ptr<float>(), saved.data_ptr(), bytes,
                                   for_backward, current_stream()),
             op);
    if (!for_backward) saved = Tensor();
    return {o, state_out, saved};
}

std::vector<Tensor> gated_delta_bp(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, MaybeTensor state,
                                   MaybeTensor lengths, double scale, Tensor saved, Tensor grad_o,
                                   MaybeTensor grad_state_out) {
    const char* op = "gated_delta_bp";
    const Tensor initial = state.value_or(Tensor()), grad_last = grad_state_out.value_or(Tensor());
    check_eager(op, {&q, &k, &v, &g, &beta, &initial, &grad_o, &grad_last});
    check_on_gpu(q, op, "q");
    const DeviceGuard guard(q.device());
    const DeltaOperands d = delta_operands(q, k, v, g, beta, state, lengths, scale, 4, op);
    check_like(grad_o, q, op, "grad_o", "q");
    TORCH_CHECK(grad_o.sizes() == v.sizes(), "snnlib.", op, ": grad_o ", grad_o.sizes(), " and v ", v.sizes(),
                " must have the same shape");
    check_on_gpu(saved, op, "saved");
    TORCH_CHECK(saved.device() == q.device() && saved.scalar_type() == at::kByte && saved.is_contiguous() &&
                    static_cast<size_t>(saved.numel()) == snnseq_gated_delta_saved_bytes(&d.call, 1),
                "snnlib.", op, ": saved must be what gated_delta_fp returned for these operands");
    Tensor go = dense_rows(grad_o), gs;
    if (grad_last.defined()) {
        gs = grad_last;
        check_on_gpu(gs, op, "grad_state_out");
        TORCH_CHECK(gs.device() == q.device() && gs.scalar_type() == at::kFloat && gs.dim() == 4 &&
                        gs.size(0) == d.call.B && gs.size(1) == d.call.Hv && gs.size(2) == d.call.Dk &&
                        gs.size(3) == d.call.Dv,
                    "snnlib.", op, ": grad_state_out must be shaped and typed as the state, got ", gs.scalar_type(), " ",
                    gs.sizes());
        gs = dense(gs);
    }
    Tensor grad_q = torch::empty(q.sizes(), q.options()), grad_k = torch::empty(q.sizes(), q.options());
    Tensor grad_v = torch::empty(v.sizes(), v.options());
    Tensor grad_g = torch::empty(g.sizes(), d.g.options()), grad_beta = torch::empty(g.sizes(), d.g.options());
    Tensor grad_state;
    if (d.has_state) grad_state = torch::empty(d.state.sizes(), d.state.options());
    int64_t strides[3];
    strides_of(go, strides);
    const size_t bytes = snnseq_gated_delta_bp_workspace_bytes(&d.call);
    Tensor workspace = workspace_of(bytes, q);
    check_rc(snnseq_gated_delta_bp(&d.call, saved.data_ptr(), static_cast<size_t>(saved.numel()), go.data_ptr(), strides,
                                   gs.defined() ? gs.data_ptr<float>() : nullptr, grad_q.data_ptr(), grad_k.data_ptr(),
                                   grad_v.data_ptr(), grad_g.data_ptr<float>(), grad_beta.data_ptr<float>(),
                                   d.has_state ? grad_state.data_ptr<float>() : nullptr, workspace.data_ptr(), bytes,
                                   current_stream()),
             op);
    return {grad_q, grad_k, grad_v, grad_g, grad_beta, grad_state};
}

Tensor gated_delta_step(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor state, double scale,
                        MaybeTensor state_out) {
    const char* op = "gated_delta_step";
    const Tensor result = state_out.value_or(Tensor());
    TORCH_CHECK(!records({&q, &k, &v, &g, &beta, &state, &result}), "snnlib.", op, ": a step is not differentiable: call it "
                "with gradients off, or use gated_delta");
    check_eager(op, {&q, &k, &v, &g, &beta, &state, &result});
    check_on_gpu(q, op, "q");
    check_on_gpu(state, op, "state");
    const DeviceGuard guard(q.device());
    const DeltaOperands d = delta_operands(q, k, v, g, beta, state, c10::nullopt, scale, 3, op);
    if (result.defined()) check_on_gpu(result, op, "state_out");
    Tensor out = result.defined() ? result : state;
    TORCH_CHECK(state.is_contiguous() && out.is_contiguous() && out.device() == q.device() &&
                    out.scalar_type() == at::kFloat && out.sizes() == state.sizes(),
                "snnlib.", op, ": the state is updated in place, or into state_out: both must be dense float32 ",
                state.sizes());
    if (out.data_ptr() != state.data_ptr()) {
        const char *a = static_cast<char*>(state.data_ptr()), *b = static_cast<char*>(out.data_ptr());
        const int64_t bytes = state.numel() * 4;
        TORCH_CHECK(a + bytes <= b || b + bytes <= a, "snnlib.", op, ": state_out must be state or not overlap it");
    }
    Tensor o = torch::empty(v.sizes(), v.options());
    check_rc(snnseq_gated_delta_step(&d.call, o.data_ptr(), out.data_ptr<float>(), current_stream()), op);
    // a graph that kept the tensor for its backward has to notice
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return o;
}

// ---- autograd -----------------------------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool records(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Gradients come from kernels autograd knows nothing of: differentiating them in turn is an error, not a zero.
variable_list differentiable_once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list defined;
    for (const Tensor& g : grads)
        if (g.defined()) {
            defined.push_back(g.detach());
            defined.back().set_requires_grad(true);
        }
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        "the gradients of the token layers cannot be differentiated again", static_cast<int64_t>(defined.size()));
    const variable_list out = (*error)(std::move(defined));
    size_t next = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = out[next++];
    return grads;
}

struct EmbedFunction : torch::autograd::Function<EmbedFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& weight, double scale) {
        Tensor out = embed_fp(tokens, weight, scale);
        ctx->save_for_backward({tokens});
        ctx->saved_data["vocab"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor tokens = ctx->get_saved_variables()[0];
        return differentiable_once({Tensor(), embed_bp(tokens, grads[0], ctx->saved_data["vocab"].toInt(),
                                                       ctx->saved_data["scale"].toDouble()),
                                    Tensor()});
    }
};

Tensor embed(const Tensor& tokens, const Tensor& weight, double scale) {
    return records({&weight}) ? EmbedFunction::apply(tokens, weight, scale) : embed_fp(tokens, weight, scale);
}

struct GnActFunction : torch::autograd::Function<GnActFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight_gn, const Tensor& bias_gn,
                          int64_t groups, double eps_gn, const std::string& act) {
        std::vector<Tensor> r = gn_act_fp(x, weight_gn, bias_gn, groups, eps_gn, act);
        ctx->save_for_backward({x, weight_gn, bias_gn, r[0], r[1]});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return r[2];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const std::vector<Tensor> g = gn_act_bp(s[0], s[1], s[2], s[3], s[4], ctx->saved_data["groups"].toInt(),
                                                ctx->saved_data["act"].toStringRef(), grads[0]);
        return differentiable_once({g[0], g[1], g[2], Tensor(), Tensor(), Tensor()});
    }
};

Tensor gn_act(const Tensor& x, const Tensor& weight_gn, const Tensor& bias_gn, int64_t groups, double eps_gn,
              const std::string& act) {
    if (records({&x, &weight_gn, &bias_gn})) return GnActFunction::apply(x, weight_gn, bias_gn, groups, eps_gn, act);
    return gn_act_fp(x, weight_gn, bias_gn, groups, eps_gn, act)[2];
}

// Unlike the fire layers this one keeps what its forward computed on the way -- the state before every chunk of 64 steps
// and the rows added to it: the state passes are bound by latency, running the forward's again would cost a third
// of the backward, and the memory is there.
struct GatedDeltaFunction : torch::autograd::Function<GatedDeltaFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                 const Tensor& beta, const MaybeTensor& state, const MaybeTensor& lengths, double scale) {
        ctx->set_materialize_grads(false);
        std::vector<Tensor> r = gated_delta_fp(q, k, v, g, beta, state, lengths, scale, true);
        ctx->save_for_backward({q, k, v, g, beta, state.value_or(Tensor()), lengths.value_or(Tensor()), r[2]});
        ctx->saved_data["scale"] = scale;
        return {r[0], r[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(8);
        const variable_list s = ctx->get_saved_variables();
        const Tensor& v = s[2];
        const Tensor grad_o = grads[0].defined() ? grads[0] : torch::zeros({v.size(3)}, v.options()).expand(v.sizes());
        std::vector<Tensor> g = gated_delta_bp(s[0], s[1], v, s[3], s[4], s[5], s[6], ctx->saved_data["scale"].toDouble(),
                                               s[7], grad_o, grads[1]);
        return differentiable_once({g[0], g[1], g[2], g[3], g[4], g[5], Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor> gated_delta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                       const Tensor& beta, const MaybeTensor& state, const MaybeTensor& lengths,
                                       double scale) {
    const Tensor initial = state.value_or(Tensor());
    if (records({&q, &k, &v, &g, &beta, &initial})) {
        const variable_list r = GatedDeltaFunction::apply(q, k, v, g, beta, state, lengths, scale);
        return {r[0], r[1]};
    }
    const std::vector<Tensor> r = gated_delta_fp(q, k, v, g, beta, state, lengths, scale, false);
    return {r[0], r[1]};
}

}  // namespace

void bind_token_layers(pybind11::module_& m) {
    m.attr("__seq_abi_version__") = snnseq_abi_version();
    const auto release = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("embed", &embed, "embedding lookup with a scale, differentiable", release);
    m.def("gn_act", &gn_act, "group norm with an activation, channels last, differentiable", release);
    m.def("gated_delta", &gated_delta, "gated delta rule over a sequence, differentiable: (o, state_out)", release);
    m.def("embed_fp", &embed_fp, "embedding lookup with a scale");
    m.def("embed_bp", &embed_bp, "gradient of the embedding table, by sorted tokens");
    m.def("gn_act_fp", &gn_act_fp, "group norm with an activation, channels last: [mean, rstd, y]");
    m.def("gn_act_bp", &gn_act_bp, "its backward: [grad_x, grad_weight_gn, grad_bias_gn]");
    m.def("gated_delta_fp", &gated_delta_fp, "gated delta rule over a sequence: [o, state_out, saved]",
          pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("g"), pybind11::arg("beta"),
          pybind11::arg("state"), pybind11::arg("lengths"), pybind11::arg("scale"), pybind11::arg("for_backward") = true);
    m.def("gated_delta_bp", &gated_delta_bp, "its backward: [grad_q, grad_k, grad_v, grad_g, grad_beta, grad_state]");
    m.def("gated_delta_step", &gated_delta_step, "gated delta rule, one time step: o, the state updated");
}
