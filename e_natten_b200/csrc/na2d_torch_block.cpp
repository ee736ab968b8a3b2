// group_norm, rotary and attention on PyTorch tensors: argument checks, layouts, allocation, the calls of the C ABI and the autograd
// functions.  A call that needs no gradient goes straight to the library.
//
// A call that something looks into (a trace, a dispatch mode) goes through PyTorch's dispatcher as an operator of the library e_natten_b200:
// whoever records calls sees one, with its arguments, and can make it again.  What the functions here do for themselves is not seen; a
// trace of them would be the allocation of their results and nothing else.  Ordinary calls do without the dispatcher.
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <torch/library.h>

#include <cstring>
#include <tuple>
#include <vector>

#include "na2d_torch_call.h"

namespace na2d_torch {
namespace {

namespace ag = torch::autograd;

// The library functions, as loaded by _lib.py.
struct Abi {
    int (*attention_forward)(const na2d_attention_args*) = nullptr;
    int (*attention_backward)(const na2d_attention_args*) = nullptr;
    size_t (*attention_workspace)(const na2d_attention_args*, int) = nullptr;
    int (*norm_forward)(const na2d_norm_args*) = nullptr;
    int (*norm_backward)(const na2d_norm_args*) = nullptr;
    size_t (*norm_workspace)(const na2d_norm_args*, int) = nullptr;
    int (*rotary)(const na2d_rotary_args*) = nullptr;
    int (*rotary_table)(const double*, const double*, int64_t, int, int, double, float*, int, void*) = nullptr;
    int (*poll)(int, void*) = nullptr;
} abi;

void bind_block_abi(uintptr_t attention_forward, uintptr_t attention_backward, uintptr_t attention_workspace, uintptr_t norm_forward,
                    uintptr_t norm_backward, uintptr_t norm_workspace, uintptr_t rotary, uintptr_t rotary_table, uintptr_t poll) {
    abi.attention_forward = reinterpret_cast<decltype(abi.attention_forward)>(attention_forward);
    abi.attention_backward = reinterpret_cast<decltype(abi.attention_backward)>(attention_backward);
    abi.attention_workspace = reinterpret_cast<decltype(abi.attention_workspace)>(attention_workspace);
    abi.norm_forward = reinterpret_cast<decltype(abi.norm_forward)>(norm_forward);
    abi.norm_backward = reinterpret_cast<decltype(abi.norm_backward)>(norm_backward);
    abi.norm_workspace = reinterpret_cast<decltype(abi.norm_workspace)>(norm_workspace);
    abi.rotary = reinterpret_cast<decltype(abi.rotary)>(rotary);
    abi.rotary_table = reinterpret_cast<decltype(abi.rotary_table)>(rotary_table);
    abi.poll = reinterpret_cast<decltype(abi.poll)>(poll);
}

// ---- operators of the dispatcher ------------------------------------------------------------------------------------
using AttentionForward = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, double, bool, int64_t);
using AttentionBackward = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                              const MaybeTensor&, double, bool, int64_t, bool, bool);
using Norm = Tensor(const Tensor&, const MaybeTensor&, const MaybeTensor&, int64_t, double, int64_t);
using NormForward = std::tuple<Tensor, Tensor>(const Tensor&, const MaybeTensor&, const MaybeTensor&, int64_t, double, int64_t);
using NormBackward = std::vector<Tensor>(const Tensor&, const MaybeTensor&, const MaybeTensor&, const Tensor&, const Tensor&, int64_t, double,
                                         int64_t, bool, bool, bool);
using Turn = std::vector<Tensor>(const Tensor&, const MaybeTensor&, const Tensor&, const MaybeTensor&, bool, bool);
using Table = Tensor(const Tensor&, const Tensor&, double);

// ---- attention -----------------------------------------------------------------------------------------------------------
struct AttentionCall {
    double scale;
    bool causal;
    int path;
};

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v) {
    check_map(q, "q");
    check_like(k, q, "k", "q");
    check_like(v, q, "v", "q");
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "q, k and v must be (B, heads, T, C); got ", q.sizes(), " and ", k.sizes());
    TORCH_CHECK_VALUE(k.sizes().equals(v.sizes()), "k and v must have the same shape; got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(q.size(0) == k.size(0) && q.size(3) == k.size(3), "q and k must have the same batch size and head dim; got ", q.sizes(),
                      " and ", k.sizes());
    TORCH_CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "the number of key heads must divide the number of query heads; got ",
                      k.size(1), " and ", q.size(1));
}
// Lengths as the kernels read them: int32, dense.
Tensor lengths_of(const Tensor& lengths, const Tensor& q, const Tensor& k) {
    if (!lengths.defined()) return lengths;
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == q.size(0) && lengths.device() == q.device() &&
                          (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong),
                      "key_lengths must be an int32 or int64 tensor of (B,) on q's device");
    check_plain(lengths, "key_lengths");
    if (lengths.scalar_type() == at::kLong) return lengths.clamp(0, k.size(2)).to(at::kInt);
    return lengths.contiguous();
}
na2d_attention_args attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const AttentionCall& call) {
    na2d_attention_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.B = extent(q.size(0), "batch"); a.N = extent(q.size(1), "heads"); a.Nk = extent(k.size(1), "key heads");
    a.Tq = extent(q.size(2), "query tokens"); a.Tk = extent(k.size(2), "key tokens"); a.C = extent(q.size(3), "head dim");
    a.dtype = dtype_of(q);
    a.path = call.path;
    a.device = q.device().index();
    a.causal = call.causal;
    a.scale = (float)call.scale;
    a.stream = stream_of(q);
    a.q = heads_of(q); a.k = heads_of(k); a.v = heads_of(v);
    a.key_lengths = lengths.defined() ? lengths.data_ptr<int>() : nullptr;
    return a;
}

// Checked operands of tokens -> o, lse.
std::tuple<Tensor, Tensor> attention_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& lengths,
                                             const AttentionCall& call) {
    const Tensor q = in_place_or_copy(q_in), k = in_place_or_copy(k_in), v = in_place_or_copy(v_in);
    const auto rows = at::DimVector(q.sizes().begin(), q.sizes().end() - 1);
    if (q.numel() == 0 || k.numel() == 0)                // no key: every row sees nothing
        return {at::zeros(q.sizes(), q.options()), at::full(rows, -std::numeric_limits<double>::infinity(), q.options().dtype(at::kFloat))};
    Tensor o = at::empty(q.sizes(), q.options()), lse = at::empty(rows, q.options().dtype(at::kFloat));
    na2d_attention_args a = attention_args(q, k, v, lengths, call);
    a.o = dense_heads(o);
    a.lse = lse.data_ptr<float>();
    check(abi.poll(a.device, nullptr));                  // a wait that gave up in a kernel of an earlier call surfaces here, without a sync
    const Tensor workspace = scratch(abi.attention_workspace(&a, 0), q);
    if (workspace.defined()) {
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = workspace.numel();
    }
    check(abi.attention_forward(&a));
    return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> attention_backward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& o_in,
                                                      const Tensor& lse_in, const Tensor& d_o_in, const Tensor& lengths_in,
                                                      const AttentionCall& call, bool need_dq, bool need_dkdv) {
    // (hooks on saved tensors may hand back other ones than were saved)
    check_attention(q_in, k_in, v_in);
    const Tensor lengths = lengths_of(lengths_in, q_in, k_in);
    check_like(o_in, q_in, "o", "q");
    check_like(d_o_in, q_in, "the gradient of o", "q");
    TORCH_CHECK_VALUE(o_in.sizes().equals(q_in.sizes()) && d_o_in.sizes().equals(q_in.sizes()), "o and its gradient must have q's shape");
    const auto rows = at::DimVector(q_in.sizes().begin(), q_in.sizes().end() - 1);
    TORCH_CHECK_VALUE(lse_in.sizes().equals(rows) && lse_in.scalar_type() == at::kFloat && lse_in.device() == q_in.device(),
                      "lse must hold a float32 for each row of q, on its device");
    if (q_in.numel() == 0 || k_in.numel() == 0)
        return {need_dq ? at::zeros(q_in.sizes(), q_in.options()) : Tensor(), need_dkdv ? at::zeros(k_in.sizes(), k_in.options()) : Tensor(),
                need_dkdv ? at::zeros(k_in.sizes(), k_in.options()) : Tensor()};
    const Tensor q = in_place_or_copy(q_in), k = in_place_or_copy(k_in), v = in_place_or_copy(v_in), o = in_place_or_copy(o_in),
                 d_o = in_place_or_copy(d_o_in), lse = lse_in.contiguous();
    Tensor d_q, d_k, d_v, delta = at::empty(rows, lse.options());
    na2d_attention_args a = attention_args(q, k, v, lengths, call);
    a.o = heads_of(o);
    a.d_o = heads_of(d_o);
    a.lse = lse.data_ptr<float>();
    a.delta = delta.data_ptr<float>();
    if (need_dq) {
        d_q = at::empty(q.sizes(), q.options());
        a.d_q = dense_heads(d_q);
    }
    if (need_dkdv) {
        d_k = at::empty(k.sizes(), k.options());
        d_v = at::empty(k.sizes(), k.options());
        a.d_k = dense_heads(d_k);
        a.d_v = dense_heads(d_v);
    }
    check(abi.poll(a.device, nullptr));
    const Tensor workspace = scratch(abi.attention_workspace(&a, 1), q);
    if (workspace.defined()) {
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = workspace.numel();
    }
    check(abi.attention_backward(&a));
    return {d_q, d_k, d_v};
}

// The operators' kernels: arguments as whoever calls them has them.
std::tuple<Tensor, Tensor> attention_forward_op(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& lengths, double scale,
                                                bool causal, int64_t path) {
    check_attention(q, k, v);
    return attention_forward(q, k, v, lengths_of(lengths.value_or(Tensor()), q, k), {scale, causal, (int)path});
}
std::vector<Tensor> attention_backward_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& d_o,
                                          const MaybeTensor& lengths, double scale, bool causal, int64_t path, bool need_dq, bool need_dkdv) {
    auto [d_q, d_k, d_v] = attention_backward(q, k, v, o, lse, d_o, lengths.value_or(Tensor()), {scale, causal, (int)path}, need_dq, need_dkdv);
    return !need_dkdv ? std::vector<Tensor>{d_q} : need_dq ? std::vector<Tensor>{d_q, d_k, d_v} : std::vector<Tensor>{d_k, d_v};
}

struct Attention : ag::Function<Attention> {
    static ag::variable_list forward(ag::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                     const MaybeTensor& lengths_in, double scale, bool causal, int64_t path) {
        const Tensor lengths = lengths_in.value_or(Tensor());
        Tensor o, lse;
        if (goes_through({q, k, v, lengths})) {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(o, lse) = operator_of<AttentionForward>("e_natten_b200::attention").call(q, k, v, lengths_in, scale, causal, path);
        } else {
            std::tie(o, lse) = attention_forward(q, k, v, lengths, {scale, causal, (int)path});
        }
        ctx->save_for_backward({q, k, v, o, lse, lengths});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["path"] = path;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);               // lse's gradient would be a buffer of zeros, filled at each backward
        return {o, lse};
    }
    static ag::variable_list backward(ag::AutogradContext* ctx, const ag::variable_list& grads) {
        check_once("attention");
        const auto s = ctx->get_saved_variables();
        const Tensor d_o = grads[0].defined() ? grads[0] : at::zeros(s[0].sizes(), s[0].options());
        const bool need_dq = ctx->needs_input_grad(0), need_dk = ctx->needs_input_grad(1), need_dv = ctx->needs_input_grad(2);
        const AttentionCall call{ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(), (int)ctx->saved_data["path"].toInt()};
        Tensor d_q, d_k, d_v;
        if (goes_through({s[0], s[1], s[2], s[3], s[4], d_o, s[5]})) {
            const auto found = operator_of<AttentionBackward>("e_natten_b200::attention_backward")
                                   .call(s[0], s[1], s[2], s[3], s[4], d_o, maybe(s[5]), call.scale, call.causal, call.path, need_dq, need_dk || need_dv);
            if (need_dq) d_q = found.front();
            if (need_dk || need_dv) std::tie(d_k, d_v) = std::make_tuple(found[found.size() - 2], found.back());
        } else {
            std::tie(d_q, d_k, d_v) = attention_backward(s[0], s[1], s[2], s[3], s[4], d_o, s[5], call, need_dq, need_dk || need_dv);
        }
        return {d_q, need_dk ? d_k : Tensor(), need_dv ? d_v : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& lengths, double scale, bool causal,
                                              int64_t path) {
    if (wants_grad({q, k, v})) {
        check_attention(q, k, v);
        const auto out = Attention::apply(q, k, v, maybe(lengths_of(lengths.value_or(Tensor()), q, k)), scale, causal, path);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return operator_of<AttentionForward>("e_natten_b200::attention").call(q, k, v, lengths, scale, causal, path);
}

std::tuple<Tensor, Tensor> attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, double scale, bool causal,
                                     const MaybeTensor& lengths_in, int64_t path) {
    check_map(q_in, "q");
    const Tensor q = tokens(q_in, "q"), k = tokens(k_in, "k"), v = tokens(v_in, "v");
    check_attention(q, k, v);
    const Tensor lengths = lengths_of(lengths_in.value_or(Tensor()), q, k);
    Tensor o, lse;
    if (goes_through({q, k, v, lengths})) {
        std::tie(o, lse) = operator_of<AttentionForward>("e_natten_b200::attention").call(q, k, v, maybe(lengths), scale, causal, path);
    } else if (wants_grad({q, k, v})) {
        const auto out = Attention::apply(q, k, v, maybe(lengths), scale, causal, path);
        o = out[0];
        lse = out[1];
    } else {
        std::tie(o, lse) = attention_forward(q, k, v, lengths, {scale, causal, (int)path});
    }
    if (q_in.dim() == 5) return {o.unflatten(2, {q_in.size(2), q_in.size(3)}), lse.unflatten(2, {q_in.size(2), q_in.size(3)})};
    return {o, lse};
}

// ---- group normalisation ----------------------------------------------------------------------------------------------------
struct NormCall {
    int64_t groups;
    double eps;
    int64_t activation;
};

// (B, P, C), C contiguous.
Tensor pixels(const Tensor& t) {
    Tensor x = t.dim() == 2 ? t.unsqueeze(1) : t.flatten(1, -2);
    const auto s = x.strides();
    const bool ready = (s[2] == 1 || x.size(2) == 1) && (s[1] > 0 || x.size(1) <= 1) && (s[0] > 0 || x.size(0) <= 1);
    return ready ? x : x.contiguous();
}
na2d_pixels pixels_of(const Tensor& x) { return {x.data_ptr(), at_least_one(x.stride(0)), at_least_one(x.stride(1))}; }
void check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, const NormCall& call) {
    check_map(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 2, "x must be (B, ..., C); got ", x.sizes());
    TORCH_CHECK_VALUE(call.groups > 0 && x.size(-1) > 0 && x.size(-1) % call.groups == 0, "num_groups must be positive and divide ", x.size(-1),
                      " channels; got ", call.groups);
    const Tensor* first = nullptr;
    for (const Tensor* p : {&weight, &bias}) {
        if (!p->defined()) continue;
        TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == x.size(-1) && p->device() == x.device() &&
                              (p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type()),
                          "weight and bias must be (C,), on x's device, float32 or of x's dtype");
        TORCH_CHECK_VALUE(!first || p->scalar_type() == first->scalar_type(), "weight and bias must have one dtype");
        check_plain(*p, "weight and bias");
        first = p;
    }
}
na2d_norm_args norm_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& stats, const NormCall& call) {
    na2d_norm_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.B = extent(x.size(0), "batch");
    a.C = extent(x.size(2), "channels");
    a.P = x.size(1);
    a.groups = (int)call.groups;
    a.dtype = dtype_of(x);
    a.param_dtype = weight.defined() ? dtype_of(weight) : bias.defined() ? dtype_of(bias) : NA2D_F32;
    a.activation = (int)call.activation;
    a.device = x.device().index();
    a.eps = (float)call.eps;
    a.stream = stream_of(x);
    a.x = pixels_of(x);
    a.weight = weight.defined() ? weight.data_ptr() : nullptr;
    a.bias = bias.defined() ? bias.data_ptr() : nullptr;
    a.mean = stats.data_ptr<float>();
    a.rstd = a.mean + x.size(0) * call.groups;
    return a;
}
Tensor dense_param(const Tensor& p) { return p.defined() ? p.contiguous() : p; }

// Checked arguments -> y, (2, B, groups) means and reciprocal deviations.
std::tuple<Tensor, Tensor> norm_forward(const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, const NormCall& call) {
    const Tensor weight = dense_param(weight_in), bias = dense_param(bias_in);
    Tensor y = at::empty(x_in.sizes(), x_in.options()), stats = at::empty({2, x_in.size(0), call.groups}, x_in.options().dtype(at::kFloat));
    if (x_in.numel() == 0) return {y, stats};
    const Tensor x = pixels(x_in);
    na2d_norm_args a = norm_args(x, weight, bias, stats, call);
    a.y = y.data_ptr();
    check(abi.poll(a.device, nullptr));                  // (the two passes wait for one another)
    const Tensor workspace = scratch(abi.norm_workspace(&a, 0), x);
    if (workspace.defined()) {
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = workspace.numel();
    }
    check(abi.norm_forward(&a));
    return {y, stats};
}

// d_x, d_weight, d_bias, those that are wanted.
std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, const Tensor& stats,
                                                 const Tensor& d_y_in, const NormCall& call, bool need_x, bool need_w, bool need_b) {
    const Tensor weight = dense_param(weight_in), bias = dense_param(bias_in);
    check_norm(x_in, weight, bias, call);
    check_like(d_y_in, x_in, "the gradient of y", "x");
    TORCH_CHECK_VALUE(d_y_in.sizes().equals(x_in.sizes()), "the gradient of y must have x's shape");
    TORCH_CHECK_VALUE(stats.is_contiguous() && stats.scalar_type() == at::kFloat && stats.device() == x_in.device() &&
                          stats.numel() == 2 * x_in.size(0) * call.groups,
                      "the saved statistics must be what the forward saved");
    Tensor d_x, d_w, d_b;
    need_w = need_w && weight.defined();
    need_b = need_b && bias.defined();
    if (need_x) d_x = at::empty(x_in.sizes(), x_in.options());
    if (x_in.numel() == 0) {
        if (need_w) d_w = at::zeros_like(weight);
        if (need_b) d_b = at::zeros_like(bias);
        return {d_x, d_w, d_b};
    }
    if (need_w) d_w = at::empty(weight.sizes(), weight.options());
    if (need_b) d_b = at::empty(bias.sizes(), bias.options());
    const Tensor x = pixels(x_in), d_y = pixels(d_y_in);
    na2d_norm_args a = norm_args(x, weight, bias, stats, call);
    a.d_y = pixels_of(d_y);
    a.d_x = d_x.defined() ? d_x.data_ptr() : nullptr;
    a.d_weight = need_w ? d_w.data_ptr() : nullptr;
    a.d_bias = need_b ? d_b.data_ptr() : nullptr;
    check(abi.poll(a.device, nullptr));
    const Tensor workspace = scratch(abi.norm_workspace(&a, 1), x);
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = workspace.numel();
    check(abi.norm_backward(&a));
    return {d_x, d_w, d_b};
}

// The operators' kernels.
std::tuple<Tensor, Tensor> norm_forward_op(const Tensor& x, const MaybeTensor& weight_in, const MaybeTensor& bias_in, int64_t groups, double eps,
                                           int64_t activation) {
    const Tensor weight = weight_in.value_or(Tensor()), bias = bias_in.value_or(Tensor());
    check_norm(x, weight, bias, {groups, eps, activation});
    return norm_forward(x, weight, bias, {groups, eps, activation});
}
Tensor norm_op(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, int64_t groups, double eps, int64_t activation) {
    return std::get<0>(norm_forward_op(x, weight, bias, groups, eps, activation));
}
std::vector<Tensor> norm_backward_op(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, const Tensor& stats, const Tensor& d_y,
                                     int64_t groups, double eps, int64_t activation, bool need_x, bool need_w, bool need_b) {
    const auto [d_x, d_w, d_b] = norm_backward(x, weight.value_or(Tensor()), bias.value_or(Tensor()), stats, d_y, {groups, eps, activation}, need_x,
                                               need_w, need_b);
    std::vector<Tensor> found;
    for (const Tensor& t : {d_x, d_w, d_b})
        if (t.defined()) found.push_back(t);
    return found;
}

struct GroupNorm : ag::Function<GroupNorm> {
    static Tensor forward(ag::AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight_in, const MaybeTensor& bias_in, int64_t groups,
                          double eps, int64_t activation) {
        const Tensor weight = weight_in.value_or(Tensor()), bias = bias_in.value_or(Tensor());
        Tensor y, stats;
        if (goes_through({x, weight, bias})) {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(y, stats) = operator_of<NormForward>("e_natten_b200::group_norm_forward").call(x, weight_in, bias_in, groups, eps, activation);
        } else {
            std::tie(y, stats) = norm_forward(x, weight, bias, {groups, eps, activation});
        }
        ctx->save_for_backward({x, weight, bias, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["activation"] = activation;
        return y;
    }
    static ag::variable_list backward(ag::AutogradContext* ctx, const ag::variable_list& grads) {
        check_once("group_norm");
        const auto s = ctx->get_saved_variables();
        const NormCall call{ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["activation"].toInt()};
        const bool need_x = ctx->needs_input_grad(0), need_w = s[1].defined() && ctx->needs_input_grad(1),
                   need_b = s[2].defined() && ctx->needs_input_grad(s[1].defined() ? 2 : 1);
        Tensor d_x, d_w, d_b;
        if (goes_through({s[0], s[1], s[2], s[3], grads[0]})) {
            const auto found = operator_of<NormBackward>("e_natten_b200::group_norm_backward")
                                   .call(s[0], maybe(s[1]), maybe(s[2]), s[3], grads[0], call.groups, call.eps, call.activation, need_x, need_w, need_b);
            auto next = found.begin();
            if (need_x) d_x = *next++;
            if (need_w) d_w = *next++;
            if (need_b) d_b = *next++;
        } else {
            std::tie(d_x, d_w, d_b) = norm_backward(s[0], s[1], s[2], s[3], grads[0], call, need_x, need_w, need_b);
        }
        return {d_x, d_w, d_b, Tensor(), Tensor(), Tensor()};
    }
};

Tensor norm_autograd(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, int64_t groups, double eps, int64_t activation) {
    if (wants_grad({x, weight.value_or(Tensor()), bias.value_or(Tensor())})) {
        check_norm(x, weight.value_or(Tensor()), bias.value_or(Tensor()), {groups, eps, activation});
        return GroupNorm::apply(x, weight, bias, groups, eps, activation);
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return operator_of<Norm>("e_natten_b200::group_norm").call(x, weight, bias, groups, eps, activation);
}

Tensor group_norm(const Tensor& x, int64_t groups, const MaybeTensor& weight_in, const MaybeTensor& bias_in, double eps, int64_t activation) {
    const Tensor weight = weight_in.value_or(Tensor()), bias = bias_in.value_or(Tensor());
    const NormCall call{groups, eps, activation};
    check_norm(x, weight, bias, call);
    if (goes_through({x, weight, bias}))
        return operator_of<Norm>("e_natten_b200::group_norm").call(x, maybe(weight), maybe(bias), groups, eps, activation);
    if (wants_grad({x, weight, bias})) return GroupNorm::apply(x, maybe(weight), maybe(bias), groups, eps, activation);
    return std::get<0>(norm_forward(x, weight, bias, call));
}

// ---- rotary positions ----------------------------------------------------------------------------------------------------------
// What turns x (B, heads, T, C): a table and, or not, the tokens' rows of it.
void check_turn(const Tensor& x, const Tensor& table, const Tensor& index) {
    TORCH_CHECK_VALUE(table.dim() == 3 && table.size(2) == 2 && table.scalar_type() == at::kFloat && table.device() == x.device(),
                      "table must be a float32 tensor of (rows, pairs, 2) on q's device (rotary_table makes one)");
    check_plain(table, "table");
    TORCH_CHECK_VALUE(table.size(1) > 0 && 2 * table.size(1) <= x.size(3), "table turns ", 2 * table.size(1), " channels of a head dim of ",
                      x.size(3));
    if (!index.defined()) {
        TORCH_CHECK_VALUE(table.size(0) >= x.size(2), "table has ", table.size(0), " rows for ", x.size(2), " tokens");
        return;
    }
    const int64_t rows = x.size(0) * x.size(2);
    TORCH_CHECK_VALUE((index.scalar_type() == at::kInt || index.scalar_type() == at::kLong) && index.device() == x.device() && index.dim() >= 2 &&
                          index.size(0) == x.size(0) && index.numel() == rows,
                      "index must be an int32 or int64 tensor with a table row for each token of each batch entry, on q's device");
    check_plain(index, "index");
    TORCH_CHECK_VALUE(table.size(0) > 0 || rows == 0, "table has no rows");
}

// The rows (B, heads, T, C) of q and k turned; either may be undefined.
std::tuple<Tensor, Tensor> turn(const Tensor& q_in, const Tensor& k_in, const Tensor& table, const Tensor& index, bool interleaved, bool inverse) {
    const Tensor &first_in = q_in.defined() ? q_in : k_in, second_in = q_in.defined() ? k_in : Tensor();
    const Tensor first = in_place_or_copy(first_in);
    Tensor out_first = at::empty(first.sizes(), first.options()), out_second, second;
    const bool two = second_in.defined();
    if (two) {
        second = in_place_or_copy(second_in);
        out_second = at::empty(second.sizes(), second.options());
    }
    na2d_rotary_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.B = extent(first.size(0), "batch");
    a.T = extent(first.size(2), "tokens");
    a.C = extent(first.size(3), "head dim");
    a.dims = extent(2 * table.size(1), "rotated channels");
    a.dtype = dtype_of(first);
    a.interleaved = interleaved;
    a.inverse = inverse;
    a.device = first.device().index();
    a.stream = stream_of(first);
    a.table = table.data_ptr<float>();
    a.table_rows = table.size(0);
    if (index.defined()) {
        a.index = index.data_ptr();
        a.index_64 = index.scalar_type() == at::kLong;
    }
    auto put = [&](const Tensor& in, Tensor& out, na2d_heads& side, void*& to, int& heads) {
        heads = extent(in.size(1), "heads");
        side = heads_of(in);
        to = out.data_ptr();
    };
    const bool any_first = first.numel() != 0, any_second = two && second.numel() != 0;
    if (any_first) put(first, out_first, a.q, a.out_q, a.N);
    if (any_second) put(second, out_second, any_first ? a.k : a.q, any_first ? a.out_k : a.out_q, any_first ? a.Nk : a.N);
    if (any_first || any_second) check(abi.rotary(&a));
    return q_in.defined() ? std::make_tuple(out_first, out_second) : std::make_tuple(Tensor(), out_first);
}

// q and k of one call, or their gradients.
void check_turned(const Tensor& q, const Tensor& k) {
    check_map(q, "q");
    TORCH_CHECK_VALUE(q.dim() == 4, "q must be (B, heads, T, C); got ", q.sizes());
    if (!k.defined()) return;
    check_like(k, q, "k", "q");
    TORCH_CHECK_VALUE(k.dim() == 4 && k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.size(3) == q.size(3),
                      "q and k may differ in their number of heads only; got ", q.sizes(), " and ", k.sizes());
}
// The operator's kernel.
std::vector<Tensor> turn_op(const Tensor& q, const MaybeTensor& k_in, const Tensor& table, const MaybeTensor& index_in, bool interleaved, bool inverse) {
    const Tensor k = k_in.value_or(Tensor()), index = index_in.value_or(Tensor());
    check_turned(q, k);
    check_turn(q, table, index);
    const auto [out_q, out_k] = turn(q, k, table.contiguous(), index.defined() ? index.contiguous() : index, interleaved, inverse);
    return k.defined() ? std::vector<Tensor>{out_q, out_k} : std::vector<Tensor>{out_q};
}
// The same for whoever may look into the call; either of q and k may be undefined.
std::tuple<Tensor, Tensor> turn_through(const Tensor& q, const Tensor& k, const Tensor& table, const Tensor& index, bool interleaved, bool inverse) {
    if (!goes_through({q, k, table, index})) return turn(q, k, table, index, interleaved, inverse);
    const bool two = q.defined() && k.defined();
    at::AutoDispatchBelowADInplaceOrView below;
    const auto out = operator_of<Turn>("e_natten_b200::rotary")
                         .call(q.defined() ? q : k, two ? MaybeTensor(k) : MaybeTensor(), table, maybe(index), interleaved, inverse);
    return two ? std::make_tuple(out[0], out[1]) : q.defined() ? std::make_tuple(out[0], Tensor()) : std::make_tuple(Tensor(), out[0]);
}

struct Rotary : ag::Function<Rotary> {
    static ag::variable_list forward(ag::AutogradContext* ctx, const Tensor& q, const MaybeTensor& k_in, const Tensor& table,
                                     const MaybeTensor& index_in, bool interleaved, bool inverse) {
        const Tensor k = k_in.value_or(Tensor()), index = index_in.value_or(Tensor());
        auto [out_q, out_k] = turn_through(q, k, table, index, interleaved, inverse);
        ctx->save_for_backward({table, index});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        if (!k.defined()) return {out_q};
        return {out_q, out_k};
    }
    static ag::variable_list backward(ag::AutogradContext* ctx, const ag::variable_list& grads) {
        check_once("rotary");
        const auto s = ctx->get_saved_variables();
        const Tensor g_q = ctx->needs_input_grad(0) ? grads[0] : Tensor();
        const Tensor g_k = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor();
        Tensor d_q, d_k;
        if (g_q.defined() || g_k.defined()) {
            if (g_q.defined()) check_map(g_q, "the gradient of q");
            if (g_k.defined()) check_map(g_k, "the gradient of k");
            check_turn(g_q.defined() ? g_q : g_k, s[0], s[1]);              // (hooks may hand back other tensors than were saved)
            const Tensor table = s[0].contiguous(), index = s[1].defined() ? s[1].contiguous() : s[1];
            std::tie(d_q, d_k) = turn_through(g_q, g_k, table, index, ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool());
        }
        return {d_q, d_k, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::vector<Tensor> turn_autograd(const Tensor& q, const MaybeTensor& k, const Tensor& table, const MaybeTensor& index, bool interleaved, bool inverse) {
    if (wants_grad({q, k.value_or(Tensor())})) {
        check_turned(q, k.value_or(Tensor()));
        check_turn(q, table, index.value_or(Tensor()));
        return Rotary::apply(q, k, table.contiguous(), index ? MaybeTensor(index->contiguous()) : index, interleaved, inverse);
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return operator_of<Turn>("e_natten_b200::rotary").call(q, k, table, index, interleaved, inverse);
}

std::tuple<Tensor, MaybeTensor> rotary(const Tensor& q_in, const MaybeTensor& k_in, const Tensor& table_in, const MaybeTensor& index_in,
                                       bool interleaved) {
    check_map(q_in, "q");
    const Tensor q = tokens(q_in, "q"), k = k_in ? tokens(*k_in, "k") : Tensor();
    check_turned(q, k);
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && table_in.requires_grad()), "rotary has no gradient for its table");
    const Tensor index_of = index_in.value_or(Tensor());
    check_turn(q, table_in, index_of);
    const Tensor table = table_in.contiguous(), index = index_of.defined() ? index_of.contiguous() : index_of;
    Tensor out_q, out_k;
    if (goes_through({q, k, table, index})) {
        const auto out = operator_of<Turn>("e_natten_b200::rotary").call(q, maybe(k), table, maybe(index), interleaved, false);
        out_q = out[0];
        if (k.defined()) out_k = out[1];
    } else if (wants_grad({q, k})) {
        const auto out = Rotary::apply(q, maybe(k), table, maybe(index), interleaved, false);
        out_q = out[0];
        if (k.defined()) out_k = out[1];
    } else {
        std::tie(out_q, out_k) = turn(q, k, table, index, interleaved, false);
    }
    auto shaped = [](const Tensor& t, const Tensor& like) { return like.dim() == 5 ? t.unflatten(2, {like.size(2), like.size(3)}) : t; };
    return {shaped(out_q, q_in), k_in ? MaybeTensor(shaped(out_k, *k_in)) : MaybeTensor()};
}

// positions (P, axes), frequencies (axes, pairs), float64 -> (P, axes * pairs, 2)
Tensor table_op(const Tensor& positions_in, const Tensor& frequencies_in, double magnitude) {
    const Tensor positions = positions_in.contiguous(), frequencies = frequencies_in.contiguous();
    for (const Tensor* t : {&positions, &frequencies}) check_plain(*t, "positions and frequencies");
    TORCH_CHECK_VALUE(positions.is_cuda() && frequencies.device() == positions.device() && positions.scalar_type() == at::kDouble &&
                          frequencies.scalar_type() == at::kDouble && positions.dim() == 2 && frequencies.dim() == 2 &&
                          positions.size(1) == frequencies.size(0),
                      "positions must be (P, axes), frequencies (axes, pairs), both float64 on one CUDA device");
    Tensor table = at::empty({positions.size(0), frequencies.numel(), 2}, positions.options().dtype(at::kFloat));
    if (table.numel() != 0)
        check(abi.rotary_table(positions.data_ptr<double>(), frequencies.data_ptr<double>(), positions.size(0), extent(positions.size(1), "axes"),
                               extent(frequencies.size(1), "pairs"), magnitude, table.data_ptr<float>(), positions.device().index(),
                               stream_of(positions)));
    return table;
}
Tensor rotary_table(const Tensor& positions, const Tensor& frequencies, double magnitude) {
    if (goes_through({positions, frequencies})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return operator_of<Table>("e_natten_b200::rotary_table").call(positions, frequencies, magnitude);
    }
    return table_op(positions, frequencies, magnitude);
}

// The operators.  `*_forward` and `*_backward` are what the others are made of, for whoever looks in below autograd; they have no gradient.
TORCH_LIBRARY(e_natten_b200, m) {
    m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? key_lengths, float scale, bool causal, int path) -> (Tensor, Tensor)");
    m.def("attention_backward(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor d_o, Tensor? key_lengths, float scale, bool causal, "
          "int path, bool need_dq, bool need_dkdv) -> Tensor[]");
    m.def("group_norm(Tensor x, Tensor? weight, Tensor? bias, int groups, float eps, int activation) -> Tensor");
    m.def("group_norm_forward(Tensor x, Tensor? weight, Tensor? bias, int groups, float eps, int activation) -> (Tensor, Tensor)");
    m.def("group_norm_backward(Tensor x, Tensor? weight, Tensor? bias, Tensor stats, Tensor d_y, int groups, float eps, int activation, "
          "bool need_dx, bool need_dweight, bool need_dbias) -> Tensor[]");
    m.def("rotary(Tensor q, Tensor? k, Tensor table, Tensor? index, bool interleaved, bool inverse) -> Tensor[]");
    m.def("rotary_table(Tensor positions, Tensor frequencies, float magnitude) -> Tensor");
}
TORCH_LIBRARY_IMPL(e_natten_b200, CUDA, m) {
    m.impl("attention", &attention_forward_op);
    m.impl("attention_backward", &attention_backward_op);
    m.impl("group_norm", &norm_op);
    m.impl("group_norm_forward", &norm_forward_op);
    m.impl("group_norm_backward", &norm_backward_op);
    m.impl("rotary", &turn_op);
    m.impl("rotary_table", &table_op);
}
TORCH_LIBRARY_IMPL(e_natten_b200, Autograd, m) {
    m.impl("attention", &attention_autograd);
    m.impl("group_norm", &norm_autograd);
    m.impl("rotary", &turn_autograd);
}

}  // namespace

void add_block_operators(pybind11::module_& m) {
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("bind_block_abi", &bind_block_abi);
    m.def("attention", &attention, release());
    m.def("group_norm", &group_norm, release());
    m.def("rotary", &rotary, release());
    m.def("rotary_table", &rotary_table, release());
}

}  // namespace na2d_torch
