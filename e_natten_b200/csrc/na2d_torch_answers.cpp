// prefix_attention, beam_select and beam_reorder on PyTorch tensors: argument checks, layouts, allocation, the calls of the C ABI and the
// autograd function.  As in na2d_torch_block.cpp, calls that something looks into go through PyTorch's dispatcher as operators.
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <torch/library.h>

#include <algorithm>
#include <cstring>
#include <tuple>
#include <vector>

#include "na2d_torch_call.h"

namespace na2d_torch {
namespace {

namespace ag = torch::autograd;

// The library functions, as loaded by _lib.py.
struct Abi {
    int (*prefix_forward)(const na2d_prefix_attention_args*) = nullptr;
    int (*prefix_backward)(const na2d_prefix_attention_args*) = nullptr;
    size_t (*prefix_workspace)(const na2d_prefix_attention_args*, int) = nullptr;
    int (*select)(const na2d_beam_select_args*) = nullptr;
    size_t (*select_workspace)(const na2d_beam_select_args*) = nullptr;
    int (*reorder)(const na2d_beam_reorder_args*) = nullptr;
    int (*poll)(int, void*) = nullptr;
} abi;

void bind_answers_abi(uintptr_t prefix_forward, uintptr_t prefix_backward, uintptr_t prefix_workspace, uintptr_t select, uintptr_t select_workspace,
                      uintptr_t reorder, uintptr_t poll) {
    abi.prefix_forward = reinterpret_cast<decltype(abi.prefix_forward)>(prefix_forward);
    abi.prefix_backward = reinterpret_cast<decltype(abi.prefix_backward)>(prefix_backward);
    abi.prefix_workspace = reinterpret_cast<decltype(abi.prefix_workspace)>(prefix_workspace);
    abi.select = reinterpret_cast<decltype(abi.select)>(select);
    abi.select_workspace = reinterpret_cast<decltype(abi.select_workspace)>(select_workspace);
    abi.reorder = reinterpret_cast<decltype(abi.reorder)>(reorder);
    abi.poll = reinterpret_cast<decltype(abi.poll)>(poll);
}

// ---- operators of the dispatcher ------------------------------------------------------------------------------------
using PrefixForward = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&,
                                                 const MaybeTensor&, const MaybeTensor&, double, bool, int64_t);
using PrefixBackward = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, const Tensor&,
                                           const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, double, bool, int64_t, bool, bool, bool);
using Select = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, int64_t, const MaybeTensor&, int64_t);
using Reordered = Tensor(const Tensor&, const Tensor&, const MaybeTensor&);

bool is_whole(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

// ---- attention over a prefix --------------------------------------------------------------------------------------------
struct PrefixCall {
    double scale;
    bool causal;
    int path;
};
// (k and v undefined: no own keys; lengths undefined: all)
struct PrefixOperands {
    Tensor q, pk, pv, k, v, lengths, prefix_lengths;
};

void check_keys(const Tensor& k, const Tensor& v, const Tensor& q, const char* k_name, const char* v_name) {
    check_like(k, q, k_name, "q");
    check_like(v, q, v_name, "q");
    TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes().equals(v.sizes()) && k.size(3) == q.size(3), k_name, " and ", v_name,
                      " must be (entries, key heads, T, C) of the same shape, with q's head dim; got ", k.sizes(), " and ", v.sizes());
}
void check_prefix(const PrefixOperands& x) {
    check_map(x.q, "q");
    TORCH_CHECK_VALUE(x.q.dim() == 4, "q must be (B, heads, T, C); got ", x.q.sizes());
    check_keys(x.pk, x.pv, x.q, "prefix_k", "prefix_v");
    TORCH_CHECK_VALUE(x.pk.size(0) > 0 && x.q.size(0) % x.pk.size(0) == 0, "the number of prefixes must divide the batch size; got ", x.pk.size(0), " and ",
                      x.q.size(0));
    TORCH_CHECK_VALUE(x.pk.size(1) > 0 && x.q.size(1) % x.pk.size(1) == 0, "the number of key heads must divide the number of query heads; got ",
                      x.pk.size(1), " and ", x.q.size(1));
    TORCH_CHECK_VALUE(x.k.defined() == x.v.defined(), "k and v come together");
    if (!x.k.defined()) {
        TORCH_CHECK_VALUE(!x.lengths.defined(), "key_lengths without k and v");
        return;
    }
    check_keys(x.k, x.v, x.q, "k", "v");
    TORCH_CHECK_VALUE(x.k.size(0) == x.q.size(0) && x.k.size(1) == x.pk.size(1), "k and v must have q's batch size and the prefix's key heads; got ",
                      x.k.sizes(), " for q ", x.q.sizes(), " and prefix_k ", x.pk.sizes());
}
// Lengths as the kernels read them: int32, dense.
Tensor lengths_of(const Tensor& lengths, int64_t count, int64_t most, const Tensor& q, const char* name) {
    if (!lengths.defined()) return lengths;
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == count && lengths.device() == q.device() && is_whole(lengths), name,
                      " must be an int32 or int64 tensor of (", count, ",) on q's device");
    check_plain(lengths, name);
    if (lengths.scalar_type() == at::kLong) return lengths.clamp(0, most).to(at::kInt);
    return lengths.contiguous();
}
// Checked, with lengths of int32.
PrefixOperands checked(const Tensor& q, const Tensor& pk, const Tensor& pv, const MaybeTensor& k, const MaybeTensor& v, const MaybeTensor& lengths,
                       const MaybeTensor& prefix_lengths) {
    PrefixOperands x{q, pk, pv, k.value_or(Tensor()), v.value_or(Tensor()), lengths.value_or(Tensor()), prefix_lengths.value_or(Tensor())};
    check_prefix(x);
    if (x.k.defined()) x.lengths = lengths_of(x.lengths, q.size(0), x.k.size(2), q, "key_lengths");
    x.prefix_lengths = lengths_of(x.prefix_lengths, pk.size(0), pk.size(2), q, "prefix_lengths");
    return x;
}
// What the kernels take: strides in place or copied; a prefix of no keys as one of which none is there; no own keys as none.
PrefixOperands ready(const PrefixOperands& given) {
    PrefixOperands x = given;
    if (x.k.defined() && x.k.size(2) == 0) x.k = x.v = x.lengths = Tensor();
    if (x.pk.size(2) == 0) {
        x.pk = x.pv = at::zeros({x.pk.size(0), x.pk.size(1), 1, x.pk.size(3)}, x.pk.options());
        x.prefix_lengths = at::zeros({x.pk.size(0)}, x.pk.options().dtype(at::kInt));
    }
    for (Tensor* t : {&x.q, &x.pk, &x.pv, &x.k, &x.v})
        if (t->defined()) *t = in_place_or_copy(*t);
    return x;
}
na2d_prefix_attention_args prefix_args(const PrefixOperands& x, const Tensor& lse, const PrefixCall& call) {
    na2d_prefix_attention_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.B = extent(x.q.size(0), "batch"); a.S = extent(x.pk.size(0), "prefixes");
    a.N = extent(x.q.size(1), "heads"); a.Nk = extent(x.pk.size(1), "key heads");
    a.Tq = extent(x.q.size(2), "query tokens"); a.P = extent(x.pk.size(2), "prefix tokens"); a.C = extent(x.q.size(3), "head dim");
    a.dtype = dtype_of(x.q);
    a.path = call.path;
    a.device = x.q.device().index();
    a.causal = call.causal;
    a.scale = (float)call.scale;
    a.stream = stream_of(x.q);
    a.q = heads_of(x.q); a.prefix_k = heads_of(x.pk); a.prefix_v = heads_of(x.pv);
    if (x.k.defined()) {
        a.Tk = extent(x.k.size(2), "key tokens");
        a.k = heads_of(x.k); a.v = heads_of(x.v);
        a.key_lengths = x.lengths.defined() ? x.lengths.data_ptr<int>() : nullptr;
    }
    a.prefix_lengths = x.prefix_lengths.defined() ? x.prefix_lengths.data_ptr<int>() : nullptr;
    a.lse = lse.data_ptr<float>();
    return a;
}
void give_workspace(na2d_prefix_attention_args& a, Tensor& workspace, const Tensor& like, int backward) {
    workspace = scratch(abi.prefix_workspace(&a, backward), like);
    if (!workspace.defined()) return;                    // (a call that will be refused)
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = workspace.numel();
}
at::DimVector rows_of(const Tensor& q) { return at::DimVector(q.sizes().begin(), q.sizes().end() - 1); }

// Checked operands -> o, lse.
std::tuple<Tensor, Tensor> prefix_forward(const PrefixOperands& given, const PrefixCall& call) {
    const auto rows = rows_of(given.q);
    const auto stats = given.q.options().dtype(at::kFloat);
    const bool any_key = given.pk.size(2) > 0 || (given.k.defined() && given.k.size(2) > 0);
    if (given.q.numel() == 0 || !any_key)
        return {at::zeros(given.q.sizes(), given.q.options()), at::full(rows, -std::numeric_limits<double>::infinity(), stats)};
    const PrefixOperands x = ready(given);
    Tensor o = at::empty(x.q.sizes(), x.q.options()), lse = at::empty(rows, stats), workspace;
    na2d_prefix_attention_args a = prefix_args(x, lse, call);
    a.o = dense_heads(o);
    check(abi.poll(a.device, nullptr));                  // a wait that gave up in a kernel of an earlier call surfaces here, without a sync
    give_workspace(a, workspace, x.q, 0);
    check(abi.prefix_forward(&a));
    return {o, lse};
}

// Which gradients are wanted, and those.
struct Wanted {
    bool q, prefix, own;
};
struct PrefixGrads {
    Tensor q, pk, pv, k, v;
};
PrefixGrads prefix_backward(const PrefixOperands& given, const Tensor& o_in, const Tensor& lse_in, const Tensor& d_o_in, const PrefixCall& call,
                            const Wanted& want) {
    check_like(o_in, given.q, "o", "q");
    check_like(d_o_in, given.q, "the gradient of o", "q");
    TORCH_CHECK_VALUE(o_in.sizes().equals(given.q.sizes()) && d_o_in.sizes().equals(given.q.sizes()), "o and its gradient must have q's shape");
    TORCH_CHECK_VALUE(lse_in.sizes().equals(rows_of(given.q)) && lse_in.scalar_type() == at::kFloat && lse_in.device() == given.q.device(),
                      "lse must hold a float32 for each row of q, on its device");
    const bool own = want.own && given.k.defined();
    auto empty = [](const Tensor& t) { return t.numel() ? at::empty(t.sizes(), t.options()) : at::zeros(t.sizes(), t.options()); };
    PrefixGrads d;
    const bool any_key = given.pk.size(2) > 0 || (given.k.defined() && given.k.size(2) > 0);
    if (given.q.numel() == 0 || !any_key) {
        if (want.q) d.q = at::zeros(given.q.sizes(), given.q.options());
        if (want.prefix) d.pk = at::zeros(given.pk.sizes(), given.pk.options()), d.pv = at::zeros(given.pk.sizes(), given.pk.options());
        if (own) d.k = at::zeros(given.k.sizes(), given.k.options()), d.v = at::zeros(given.k.sizes(), given.k.options());
        return d;
    }
    if (want.q) d.q = empty(given.q);
    if (want.prefix) d.pk = empty(given.pk), d.pv = empty(given.pv);
    if (own) d.k = empty(given.k), d.v = empty(given.v);
    const PrefixOperands x = ready(given);
    const Tensor o = in_place_or_copy(o_in), d_o = in_place_or_copy(d_o_in), lse = lse_in.contiguous();
    Tensor workspace;
    na2d_prefix_attention_args a = prefix_args(x, lse, call);
    a.o = heads_of(o);
    a.d_o = heads_of(d_o);
    if (want.q) a.d_q = dense_heads(d.q);
    if (want.prefix && d.pk.numel()) a.d_prefix_k = dense_heads(d.pk), a.d_prefix_v = dense_heads(d.pv);
    if (own && d.k.numel()) a.d_k = dense_heads(d.k), a.d_v = dense_heads(d.v);
    if (!a.d_q.ptr && !a.d_prefix_k.ptr && !a.d_k.ptr) return d;
    check(abi.poll(a.device, nullptr));
    give_workspace(a, workspace, x.q, 1);
    check(abi.prefix_backward(&a));
    return d;
}

// The operators' kernels.
std::tuple<Tensor, Tensor> prefix_forward_op(const Tensor& q, const Tensor& pk, const Tensor& pv, const MaybeTensor& k, const MaybeTensor& v,
                                             const MaybeTensor& lengths, const MaybeTensor& prefix_lengths, double scale, bool causal, int64_t path) {
    return prefix_forward(checked(q, pk, pv, k, v, lengths, prefix_lengths), {scale, causal, (int)path});
}
std::vector<Tensor> prefix_backward_op(const Tensor& q, const Tensor& pk, const Tensor& pv, const MaybeTensor& k, const MaybeTensor& v, const Tensor& o,
                                       const Tensor& lse, const Tensor& d_o, const MaybeTensor& lengths, const MaybeTensor& prefix_lengths, double scale,
                                       bool causal, int64_t path, bool need_dq, bool need_dprefix, bool need_dkdv) {
    const PrefixGrads d = prefix_backward(checked(q, pk, pv, k, v, lengths, prefix_lengths), o, lse, d_o, {scale, causal, (int)path},
                                          {need_dq, need_dprefix, need_dkdv});
    std::vector<Tensor> found;
    for (const Tensor& t : {d.q, d.pk, d.pv, d.k, d.v})
        if (t.defined()) found.push_back(t);
    return found;
}

struct PrefixAttention : ag::Function<PrefixAttention> {
    static ag::variable_list forward(ag::AutogradContext* ctx, const Tensor& q, const Tensor& pk, const Tensor& pv, const MaybeTensor& k,
                                     const MaybeTensor& v, const MaybeTensor& lengths, const MaybeTensor& prefix_lengths, double scale, bool causal,
                                     int64_t path) {
        const PrefixOperands x{q, pk, pv, k.value_or(Tensor()), v.value_or(Tensor()), lengths.value_or(Tensor()), prefix_lengths.value_or(Tensor())};
        Tensor o, lse;
        if (goes_through({q, pk, pv, x.k, x.v, x.lengths, x.prefix_lengths})) {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(o, lse) = operator_of<PrefixForward>("e_natten_b200::prefix_attention").call(q, pk, pv, k, v, lengths, prefix_lengths, scale, causal, path);
        } else {
            std::tie(o, lse) = prefix_forward(x, {scale, causal, (int)path});
        }
        ctx->save_for_backward({q, pk, pv, x.k, x.v, o, lse, x.lengths, x.prefix_lengths});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["path"] = path;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);
        return {o, lse};
    }
    static ag::variable_list backward(ag::AutogradContext* ctx, const ag::variable_list& grads) {
        check_once("prefix_attention");
        const auto s = ctx->get_saved_variables();
        const Tensor d_o = grads[0].defined() ? grads[0] : at::zeros(s[0].sizes(), s[0].options());
        const bool own = s[3].defined(), need_pk = ctx->needs_input_grad(1), need_pv = ctx->needs_input_grad(2),
                   need_k = own && ctx->needs_input_grad(3), need_v = own && ctx->needs_input_grad(4);
        const Wanted want{ctx->needs_input_grad(0), need_pk || need_pv, need_k || need_v};
        const PrefixCall call{ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(), (int)ctx->saved_data["path"].toInt()};
        PrefixGrads d;
        if (goes_through({s[0], s[1], s[2], s[3], s[4], s[5], s[6], d_o, s[7], s[8]})) {
            const auto found = operator_of<PrefixBackward>("e_natten_b200::prefix_attention_backward")
                                   .call(s[0], s[1], s[2], maybe(s[3]), maybe(s[4]), s[5], s[6], d_o, maybe(s[7]), maybe(s[8]), call.scale, call.causal,
                                         call.path, want.q, want.prefix, want.own);
            auto next = found.begin();
            if (want.q) d.q = *next++;
            if (want.prefix) d.pk = *next++, d.pv = *next++;
            if (want.own) d.k = *next++, d.v = *next++;
        } else {
            // (hooks on saved tensors may hand back other ones than were saved)
            d = prefix_backward(checked(s[0], s[1], s[2], maybe(s[3]), maybe(s[4]), maybe(s[7]), maybe(s[8])), s[5], s[6], d_o, call, want);
        }
        return {d.q, need_pk ? d.pk : Tensor(), need_pv ? d.pv : Tensor(), need_k ? d.k : Tensor(), need_v ? d.v : Tensor(),
                Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> prefix_autograd(const Tensor& q, const Tensor& pk, const Tensor& pv, const MaybeTensor& k, const MaybeTensor& v,
                                           const MaybeTensor& lengths, const MaybeTensor& prefix_lengths, double scale, bool causal, int64_t path) {
    if (wants_grad({q, pk, pv, k.value_or(Tensor()), v.value_or(Tensor())})) {
        const PrefixOperands x = checked(q, pk, pv, k, v, lengths, prefix_lengths);
        const auto out = PrefixAttention::apply(q, pk, pv, k, v, maybe(x.lengths), maybe(x.prefix_lengths), scale, causal, path);
        return {out[0], out[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return operator_of<PrefixForward>("e_natten_b200::prefix_attention").call(q, pk, pv, k, v, lengths, prefix_lengths, scale, causal, path);
}

std::tuple<Tensor, Tensor> prefix_attention(const Tensor& q_in, const Tensor& pk_in, const Tensor& pv_in, const MaybeTensor& k_in,
                                            const MaybeTensor& v_in, double scale, bool causal, const MaybeTensor& lengths,
                                            const MaybeTensor& prefix_lengths, int64_t path) {
    check_map(q_in, "q");
    const Tensor q = tokens(q_in, "q"), pk = tokens(pk_in, "prefix_k"), pv = tokens(pv_in, "prefix_v");
    const MaybeTensor k = k_in ? MaybeTensor(tokens(*k_in, "k")) : k_in, v = v_in ? MaybeTensor(tokens(*v_in, "v")) : v_in;
    const PrefixOperands x = checked(q, pk, pv, k, v, lengths, prefix_lengths);
    Tensor o, lse;
    if (goes_through({q, pk, pv, x.k, x.v, x.lengths, x.prefix_lengths})) {
        std::tie(o, lse) = operator_of<PrefixForward>("e_natten_b200::prefix_attention")
                               .call(q, pk, pv, k, v, maybe(x.lengths), maybe(x.prefix_lengths), scale, causal, path);
    } else if (wants_grad({q, pk, pv, x.k, x.v})) {
        const auto out = PrefixAttention::apply(q, pk, pv, k, v, maybe(x.lengths), maybe(x.prefix_lengths), scale, causal, path);
        o = out[0];
        lse = out[1];
    } else {
        std::tie(o, lse) = prefix_forward(x, {scale, causal, (int)path});
    }
    if (q_in.dim() == 5) return {o.unflatten(2, {q_in.size(2), q_in.size(3)}), lse.unflatten(2, {q_in.size(2), q_in.size(3)})};
    return {o, lse};
}

// ---- beam search ------------------------------------------------------------------------------------------------------------
// (a tangent would stay behind, or be dropped, without a word)
void check_no_gradient(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && t.requires_grad()) && !t._fw_grad(0).defined(), name, " has no gradient");
}
std::tuple<Tensor, Tensor, Tensor> select_op(const Tensor& logits_in, const Tensor& scores_in, int64_t count, const MaybeTensor& finished_in, int64_t end) {
    check_map(logits_in, "logits");
    TORCH_CHECK_VALUE(logits_in.dim() == 3 && logits_in.size(1) > 0 && logits_in.size(2) > 0, "logits must be (B, beams, words); got ", logits_in.sizes());
    const int64_t B = logits_in.size(0), K = logits_in.size(1), V = logits_in.size(2);
    TORCH_CHECK_VALUE(scores_in.dim() == 2 && scores_in.size(0) == B && scores_in.size(1) == K && scores_in.scalar_type() == at::kFloat &&
                          scores_in.device() == logits_in.device(),
                      "scores must be a float32 tensor of (B, beams) on logits' device");
    check_plain(scores_in, "scores");
    TORCH_CHECK_VALUE(count > 0, "count must be positive; got ", count);
    TORCH_CHECK_VALUE(end >= 0 && end < V, "end must be one of ", V, " words; got ", end);
    Tensor finished;
    if (finished_in) {
        TORCH_CHECK_VALUE(finished_in->dim() == 2 && finished_in->size(0) == B && finished_in->size(1) == K && finished_in->scalar_type() == at::kBool &&
                              finished_in->device() == logits_in.device(),
                          "finished must be a bool tensor of (B, beams) on logits' device");
        check_plain(*finished_in, "finished");
        finished = finished_in->contiguous();
    }
    const auto whole = logits_in.options().dtype(at::kLong);
    Tensor out_scores = at::empty({B, count}, scores_in.options()), parents = at::empty({B, count}, whole), words = at::empty({B, count}, whole);
    if (B == 0) return {out_scores, parents, words};
    const auto s = logits_in.strides();
    const bool in_place = (s[2] == 1 || V == 1) && (s[0] > 0 || B == 1) && (s[1] > 0 || K == 1);
    const Tensor logits = in_place ? logits_in : logits_in.contiguous(), scores = scores_in.contiguous();
    na2d_beam_select_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.B = extent(B, "batch"); a.K = extent(K, "beams"); a.V = extent(V, "words"); a.count = extent(count, "count");
    a.dtype = dtype_of(logits);
    a.device = logits.device().index();
    a.end = end;
    a.stream = stream_of(logits);
    a.logits = logits.data_ptr();
    a.stride_b = at_least_one(logits.stride(0));
    a.stride_k = at_least_one(logits.stride(1));
    a.scores = scores.data_ptr<float>();
    a.finished = finished.defined() ? reinterpret_cast<const uint8_t*>(finished.data_ptr<bool>()) : nullptr;
    a.out_scores = out_scores.data_ptr<float>();
    a.out_parents = parents.data_ptr<int64_t>();
    a.out_words = words.data_ptr<int64_t>();
    const Tensor workspace = scratch(abi.select_workspace(&a), logits);
    if (workspace.defined()) {
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = workspace.numel();
    }
    check(abi.select(&a));
    return {out_scores, parents, words};
}
std::tuple<Tensor, Tensor, Tensor> select(const Tensor& logits, const Tensor& scores, int64_t count, const MaybeTensor& finished, int64_t end) {
    check_map(logits, "logits");
    check_no_gradient(logits, "beam_select");
    check_no_gradient(scores, "beam_select");
    if (goes_through({logits, scores, finished.value_or(Tensor())})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return operator_of<Select>("e_natten_b200::beam_select").call(logits, scores, count, finished, end);
    }
    return select_op(logits, scores, count, finished, end);
}

// A cache of `entries` entries as rows, but for where it is; false where its rows cannot be told apart.
bool rows_of_cache(const Tensor& t, int64_t entries, na2d_cache* c) {
    const int64_t esize = t.element_size();
    if (t.dim() == 4 && (t.stride(3) == 1 || t.size(3) == 1)) {
        // strides that nest: sorted, each is at least what lies within it
        std::vector<std::pair<int64_t, int64_t>> dims;
        for (int64_t i = 0; i < 3; ++i)
            if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
        std::sort(dims.begin(), dims.end());
        int64_t within = t.size(3);
        for (const auto& [stride, size] : dims) {
            if (stride < within) return false;
            within = stride * size;
        }
        c->stride_e = t.size(0) > 1 ? t.stride(0) * esize : 0;
        c->stride_h = t.size(1) > 1 ? t.stride(1) * esize : 0;
        c->stride_t = t.size(2) > 1 ? t.stride(2) * esize : 0;
        c->heads = extent(t.size(1), "heads");
        c->tokens = extent(t.size(2), "tokens");
        c->row_bytes = t.size(3) * esize;
        return true;
    }
    if (!t.is_contiguous()) return false;
    c->heads = c->tokens = 1;
    c->row_bytes = t.numel() / entries * esize;
    c->stride_e = c->row_bytes;
    c->stride_h = c->stride_t = 0;
    return true;
}

// All that a call is refused for but what the library refuses; the rows of the caches that have any, without their places.
std::vector<na2d_cache> check_reorder(at::TensorList caches, const Tensor& parents_in, const MaybeTensor& lengths_in) {
    TORCH_CHECK_VALUE(parents_in.is_cuda() && parents_in.layout() == at::kStrided, "parents: e_natten_b200 runs on CUDA tensors only (there is no CPU path)");
    TORCH_CHECK_VALUE(parents_in.dim() == 2 && parents_in.size(1) > 0 && is_whole(parents_in), "parents must be an int32 or int64 tensor of (B, beams)");
    check_plain(parents_in, "parents");
    const int64_t B = parents_in.size(0), K = parents_in.size(1), entries = B * K;
    if (lengths_in) {
        TORCH_CHECK_VALUE(lengths_in->numel() == entries && is_whole(*lengths_in) && lengths_in->device() == parents_in.device() && lengths_in->dim() > 0 &&
                              lengths_in->dim() < 3,
                          "lengths must be an int32 or int64 tensor with a length for each of ", entries, " entries, on parents' device");
        check_plain(*lengths_in, "lengths");
    }
    std::vector<na2d_cache> rows;
    for (const Tensor& t : caches) {
        TORCH_CHECK_VALUE(t.is_cuda() && t.layout() == at::kStrided && t.device() == parents_in.device(), "caches must be on parents' device");
        check_plain(t, "caches");
        TORCH_CHECK_VALUE(!t.is_conj(), "caches: a lazily conjugated tensor is not supported");
        TORCH_CHECK_VALUE(t.dim() > 0 && t.size(0) == entries, "caches must have an entry for each of ", B, " x ", K, " beams; got ", t.sizes());
        TORCH_CHECK_VALUE(!lengths_in || t.dim() == 4, "with lengths, caches must be (entries, heads, tokens, channels); got ", t.sizes());
        if (t.numel() == 0) continue;
        na2d_cache c;
        std::memset(&c, 0, sizeof(c));
        TORCH_CHECK_VALUE(rows_of_cache(t, entries, &c), "caches must be contiguous, or (entries, heads, tokens, channels) with contiguous channels "
                          "and no element twice; got sizes ", t.sizes(), " and strides ", t.strides());
        rows.push_back(c);
    }
    return rows;
}
void reorder_in_place(at::TensorList caches, const Tensor& parents_in, const MaybeTensor& lengths_in) {
    std::vector<na2d_cache> rows = check_reorder(caches, parents_in, lengths_in);
    const int64_t B = parents_in.size(0), K = parents_in.size(1), entries = B * K;
    const Tensor parents = parents_in.contiguous(), lengths = lengths_in ? lengths_in->contiguous() : Tensor();
    auto next = rows.begin();
    for (const Tensor& t : caches)
        if (t.numel()) (next++)->ptr = t.data_ptr();
    for (const Tensor& t : caches)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    if (rows.empty()) return;
    // Caches move as if one after the other: those whose memory is not apart (the keys and values of one tensor, a cache twice) go into
    // different launches, in their order.
    std::vector<std::pair<char*, char*>> span;
    std::vector<size_t> turn;
    size_t turns = 0;
    for (const na2d_cache& c : rows) {
        char* first = static_cast<char*>(c.ptr);
        char* last = first + (entries - 1) * c.stride_e + (c.heads - 1) * c.stride_h + (c.tokens - 1) * c.stride_t + c.row_bytes;
        size_t own = 0;
        for (size_t i = 0; i < span.size(); ++i)
            if (first < span[i].second && span[i].first < last) own = std::max(own, turn[i] + 1);
        span.emplace_back(first, last);
        turn.push_back(own);
        turns = std::max(turns, own + 1);
    }
    na2d_beam_reorder_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.B = extent(B, "batch"); a.K = extent(K, "beams");
    a.parents = parents.data_ptr();
    a.parents_64 = parents.scalar_type() == at::kLong;
    if (lengths.defined()) {
        a.lengths = lengths.data_ptr();
        a.lengths_64 = lengths.scalar_type() == at::kLong;
    }
    a.device = parents.device().index();
    a.stream = stream_of(parents);
    for (size_t now = 0; now < turns; ++now) {
        std::vector<na2d_cache> some;
        for (size_t i = 0; i < rows.size(); ++i)
            if (turn[i] == now) some.push_back(rows[i]);
        a.caches = (int)some.size();
        a.cache = some.data();
        check(abi.reorder(&a));
    }
}
// x, or a copy of it where it lies in the storage of a cache, which moves while x is read.
Tensor apart_from(const std::vector<Tensor>& caches, const Tensor& x) {
    for (const Tensor& t : caches)
        if (x.has_storage() && t.has_storage() && x.is_alias_of(t)) return x.clone();
    return x;
}
void reorder(const std::vector<Tensor>& caches, const Tensor& parents_in, const MaybeTensor& lengths_in) {
    const Tensor parents = apart_from(caches, parents_in);
    const MaybeTensor lengths = lengths_in ? MaybeTensor(apart_from(caches, *lengths_in)) : lengths_in;
    TORCH_CHECK_VALUE(parents.is_cuda(), "parents: e_natten_b200 runs on CUDA tensors only (there is no CPU path)");
    // (a function mode sees no calls of the dispatcher, and the operator, a cache of its own and a copy back, costs several times as much)
    bool through = recorded() || any_special({parents, lengths.value_or(Tensor())});
    for (const Tensor& t : caches) {
        TORCH_CHECK_VALUE(t.is_cuda(), "caches must be on parents' device");
        check_no_gradient(t, "beam_reorder");
        through = through || any_special({t});
    }
    if (!through) return reorder_in_place(caches, parents, lengths);
    check_reorder(caches, parents, lengths);             // all of them, before the first one moves
    auto below = [](auto&& f) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return f();
    };
    for (Tensor t : caches) {
        const Tensor moved = below([&] { return operator_of<Reordered>("e_natten_b200::beam_reordered").call(t, parents, lengths); });
        // (not below: autograd counts the cache's version there; an inference tensor has none)
        if (t.is_inference()) below([&] { return t.copy_(moved); });
        else t.copy_(moved);
    }
}
// The operator: a cache of its own.  (Whoever records calls follows what copy_ changes; an operator without a result is dropped from a trace.)
Tensor reordered_op(const Tensor& cache, const Tensor& parents, const MaybeTensor& lengths) {
    TORCH_CHECK_VALUE(cache.is_cuda() && cache.device() == parents.device(), "caches must be on parents' device");
    Tensor mine = cache.clone();
    reorder_in_place({mine}, parents, lengths);
    return mine;
}

TORCH_LIBRARY_FRAGMENT(e_natten_b200, m) {
    m.def("prefix_attention(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor? k, Tensor? v, Tensor? key_lengths, Tensor? prefix_lengths, "
          "float scale, bool causal, int path) -> (Tensor, Tensor)");
    m.def("prefix_attention_backward(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor? k, Tensor? v, Tensor o, Tensor lse, Tensor d_o, "
          "Tensor? key_lengths, Tensor? prefix_lengths, float scale, bool causal, int path, bool need_dq, bool need_dprefix, bool need_dkdv) "
          "-> Tensor[]");
    m.def("beam_select(Tensor logits, Tensor scores, int count, Tensor? finished, int end) -> (Tensor, Tensor, Tensor)");
    m.def("beam_reordered(Tensor cache, Tensor parents, Tensor? lengths) -> Tensor");
}
TORCH_LIBRARY_IMPL(e_natten_b200, CUDA, m) {
    m.impl("prefix_attention", &prefix_forward_op);
    m.impl("prefix_attention_backward", &prefix_backward_op);
    m.impl("beam_select", &select_op);
    m.impl("beam_reordered", &reordered_op);
}
TORCH_LIBRARY_IMPL(e_natten_b200, Autograd, m) {
    m.impl("prefix_attention", &prefix_autograd);
}

}  // namespace

void add_answer_operators(pybind11::module_& m) {
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("bind_answers_abi", &bind_answers_abi);
    m.def("prefix_attention", &prefix_attention, release());
    m.def("beam_select", &select, release());
    m.def("beam_reorder", &reorder, release());
}

}  // namespace na2d_torch
