// The operators of asr_amd/Models/transformer_ops.py on their C entry points: outputs and workspaces from torch's allocator,
// the current stream of the tensors' device, and the autograd nodes.  Native because the calls are short: a training call of
// a few hundred frames keeps the GPU busy for 20 to 40 us, and nodes in Python took 70 to 140 us of host time.  Arguments have
// been checked by the Python functions; what the C entry points refuse raises with their message.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/asr_amd.h"

namespace {
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc) { TORCH_CHECK(rc == 0, "asr_amd: ", asr_last_error(), " (code ", rc, ")"); }

int type_of(const Tensor &t) {
    switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK(false, "asr_amd: tensors must be float32, bfloat16 or float16");
    }
}
int size(const Tensor &t, int i) {
    TORCH_CHECK(t.size(i) <= INT32_MAX, "asr_amd: an axis of ", t.size(i), " is too long");
    return (int)t.size(i);
}
// the tensors' device as the current one, and its current stream
struct Here {
    c10::DeviceGuard guard;
    void *stream;
    explicit Here(const Tensor &t) : guard(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
};
template <typename T = void>
T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }
Tensor floats(const Tensor &like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bytes(const Tensor &like, int64_t n) { return at::empty({n}, like.options().dtype(at::kByte)); }
Tensor heads(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
// Whether a call is a node of a graph.  Tangents raise with and without one: past the node they would be dropped in silence.  So
// does a trace, which would record the allocations and not the kernels.
bool wanted(std::initializer_list<const Tensor *> ts) {
    TORCH_CHECK(!torch::jit::tracer::isTracing(), "asr_amd: the encoder-layer operators cannot be traced: a trace holds torch's own operations only");
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
        for (const Tensor *t : ts)
            TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                                        "asr_amd: the encoder-layer operators have no forward-mode derivatives");
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
Tensor or_none(const optional<Tensor> &t) { return t ? *t : Tensor(); }
optional<Tensor> or_null(const Tensor &t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

// The operators have first derivatives only.  Where a graph of the gradients is asked for, they come with this node behind
// them: it depends on all that they depend on, and says so when somebody goes through it.
struct SecondDerivative : torch::autograd::Node {
    variable_list apply(variable_list &&) override {
        TORCH_CHECK_NOT_IMPLEMENTED(false, "asr_amd: an encoder-layer operator was differentiated twice; it has first derivatives only");
    }
};
// `compute` without a graph of its own; grads: the upstream gradients; the first four of `saved` are the inputs
template <typename F>
variable_list first_order(const variable_list &grads, const variable_list &saved, F compute) {
    variable_list out;
    {
        at::AutoGradMode off(false);
        out = compute();
    }
    if (!at::GradMode::is_enabled()) return out;
    torch::autograd::edge_list from;
    auto add = [&](const Tensor &t) {
        if (t.defined() && t.requires_grad()) from.push_back(torch::autograd::impl::gradient_edge(t));
    };
    for (const Tensor &g : grads) add(g);
    for (int i = 0; i < 4; ++i) add(saved[i]);
    std::shared_ptr<SecondDerivative> node(new SecondDerivative(), torch::autograd::deleteNode);
    node->set_next_edges(std::move(from));
    for (Tensor &t : out)
        if (t.defined()) torch::autograd::set_history(t, node);
    return out;
}

// ------------------------------------------------------------------------------------------ norm and rotation --
asr_rope_args rope_args(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const Tensor &pos, int64_t rot, double base, double eps) {
    asr_rope_args a{};
    TORCH_CHECK(q.size(2) && k.size(2), "asr_amd.qk_norm_rope: ", q.size(2), " query heads and ", k.size(2), " key heads: both or none");
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.wq = ptr<float>(wq);
    a.wk = ptr<float>(wk);
    a.pos = ptr<int64_t>(pos);
    a.q_sb = q.stride(0), a.q_st = q.stride(1), a.q_sh = q.stride(2);
    a.k_sb = k.stride(0), a.k_st = k.stride(1), a.k_sh = k.stride(2);
    a.pos_sb = pos.defined() && pos.dim() == 2 ? pos.stride(0) : 0;
    a.B = size(q, 0), a.T = size(q, 1), a.H = size(q, 2), a.Hk = size(k, 2), a.D = size(q, 3);
    a.rot = (int)rot;
    a.dtype = type_of(q);
    a.eps = (float)eps;
    a.base = base;
    return a;
}
std::tuple<Tensor, Tensor> rope_fwd(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const optional<Tensor> &pos, int64_t rot,
                                    double base, double eps) {
    Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    if (qo.numel() || ko.numel()) {
        asr_rope_args a = rope_args(q, k, wq, wk, or_none(pos), rot, base, eps);
        a.q_out = qo.data_ptr();
        a.k_out = ko.data_ptr();
        Here here(q);
        check(asr_qk_norm_rope_fwd(&a, here.stream));
    }
    return {qo, ko};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> rope_bwd(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const optional<Tensor> &pos,
                                                    int64_t rot, double base, double eps, const Tensor &gq0, const Tensor &gk0) {
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    if (!q.numel() && !k.numel()) return {dq, dk, at::zeros_like(wq), at::zeros_like(wk)};
    const Tensor gq = heads(gq0), gk = heads(gk0), dwq = floats(wq, wq.sizes()), dwk = floats(wk, wk.sizes());
    const Tensor ws = floats(wq, {asr_qk_norm_rope_ws_floats(size(q, 3))});
    asr_rope_args a = rope_args(q, k, wq, wk, or_none(pos), rot, base, eps);
    a.gq = gq.data_ptr();
    a.gk = gk.data_ptr();
    a.q_out = dq.data_ptr();
    a.k_out = dk.data_ptr();
    a.dwq = ptr<float>(dwq);
    a.dwk = ptr<float>(dwk);
    a.ws = ptr<float>(ws);
    a.gq_sb = gq.stride(0), a.gq_st = gq.stride(1), a.gq_sh = gq.stride(2);
    a.gk_sb = gk.stride(0), a.gk_st = gk.stride(1), a.gk_sh = gk.stride(2);
    Here here(q);
    check(asr_qk_norm_rope_bwd(&a, here.stream));
    return {dq, dk, dwq, dwk};
}
struct Rope : torch::autograd::Function<Rope> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const optional<Tensor> &pos,
                                 int64_t rot, double base, double eps) {
        ctx->save_for_backward({q, k, wq, wk, or_none(pos)});
        ctx->saved_data["rot"] = rot;
        ctx->saved_data["base"] = base;
        ctx->saved_data["eps"] = eps;
        auto [qo, ko] = rope_fwd(q, k, wq, wk, pos, rot, base, eps);
        return {qo, ko};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        const variable_list s = ctx->get_saved_variables();
        return first_order(g, s, [&]() -> variable_list {
            auto [dq, dk, dwq, dwk] = rope_bwd(s[0], s[1], s[2], s[3], or_null(s[4]), ctx->saved_data["rot"].toInt(), ctx->saved_data["base"].toDouble(),
                                               ctx->saved_data["eps"].toDouble(), g[0], g[1]);
            return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor()};
        });
    }
};
std::tuple<Tensor, Tensor> rope(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const optional<Tensor> &pos, int64_t rot, double base,
                                double eps) {
    if (!wanted({&q, &k, &wq, &wk})) return rope_fwd(q, k, wq, wk, pos, rot, base, eps);
    const variable_list o = Rope::apply(q, k, wq, wk, pos, rot, base, eps);
    return {o[0], o[1]};
}

// -------------------------------------------------------------------------- attention with a bucketed bias --
struct AttnOptions {
    int64_t edges;                       // address of the host's list of edges, which stays
    bool causal;
    double scale;
};
asr_bucket_attention_args attn_args(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lengths, const Tensor &keep,
                                    const Tensor &offset, const AttnOptions &o, bool train) {
    asr_bucket_attention_args a{};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.table = ptr<float>(table);
    a.edges_host = reinterpret_cast<const int32_t *>(o.edges);
    a.lengths = ptr<int32_t>(lengths);
    a.offset = ptr<int32_t>(offset);
    a.keep = static_cast<const uint8_t *>(ptr<>(keep));
    a.q_sb = q.stride(0), a.q_st = q.stride(1), a.q_sh = q.stride(2);
    a.k_sb = k.stride(0), a.k_st = k.stride(1), a.k_sh = k.stride(2);
    a.v_sb = v.stride(0), a.v_st = v.stride(1), a.v_sh = v.stride(2);
    a.B = size(q, 0), a.Tq = size(q, 1), a.Tk = size(k, 1), a.H = size(q, 2), a.Hk = size(k, 2), a.D = size(q, 3);
    a.nb = table.defined() ? size(table, 0) : o.causal ? 2 : 4;
    a.causal = o.causal;
    a.dtype = type_of(q);
    a.train = train;
    a.scale = (float)o.scale;
    return a;
}
void attn_call(asr_bucket_attention_args &a, const Tensor &q, bool backward) {
    Here here(q);
    const int64_t n = asr_bucket_attention_ws_bytes(&a, backward);
    if (n < 0) check(-1);
    const Tensor ws = n ? bytes(q, n) : Tensor();
    a.ws = ptr(ws);
    check(backward ? asr_bucket_attention_bwd(&a, here.stream) : asr_bucket_attention_fwd(&a, here.stream));
}
// out, and for training the row statistics and the output in float32 (out itself where it is)
variable_list attn_fwd_(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lengths, const Tensor &keep, const Tensor &offset,
                        const AttnOptions &o, bool train) {
    Tensor out = at::empty(q.sizes(), q.options()), lse, out32;
    if (!out.numel() || !k.size(1)) return {out.zero_(), lse, out32};
    asr_bucket_attention_args a = attn_args(q, k, v, table, lengths, keep, offset, o, train);
    a.out = out.data_ptr();
    if (train) {
        lse = floats(q, {q.size(0), q.size(2), q.size(1)});
        out32 = q.scalar_type() == at::kFloat ? out : floats(q, q.sizes());
        a.lse = ptr<float>(lse);
        a.out32 = ptr<float>(out32);
    }
    attn_call(a, q, false);
    return {out, lse, out32};
}
variable_list attn_bwd_(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lengths, const Tensor &keep, const Tensor &offset,
                        const Tensor &lse, const Tensor &out32, const AttnOptions &o, const Tensor &g0) {
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options()), dt;
    if (table.defined()) dt = floats(table, table.sizes());
    if (!q.numel() || !k.size(1)) {
        for (Tensor *t : {&dq, &dk, &dv, &dt})
            if (t->defined()) t->zero_();
        return {dq, dk, dv, dt};
    }
    const Tensor g = heads(g0);
    asr_bucket_attention_args a = attn_args(q, k, v, table, lengths, keep, offset, o, true);
    a.g = g.data_ptr();
    a.g_sb = g.stride(0), a.g_st = g.stride(1), a.g_sh = g.stride(2);
    a.out = out32.data_ptr();
    a.out32 = ptr<float>(out32);
    a.lse = ptr<float>(lse);
    a.dq = dq.data_ptr();
    a.dk = dk.data_ptr();
    a.dv = dv.data_ptr();
    a.dtable = ptr<float>(dt);
    attn_call(a, q, true);
    return {dq, dk, dv, dt};
}
struct Attention : torch::autograd::Function<Attention> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const optional<Tensor> &table,
                                 const optional<Tensor> &lengths, const optional<Tensor> &keep, const optional<Tensor> &offset, int64_t edges, bool causal,
                                 double scale) {
        const Tensor t = or_none(table), n = or_none(lengths), m = or_none(keep), p = or_none(offset);
        const variable_list o = attn_fwd_(q, k, v, t, n, m, p, {edges, causal, scale}, true);
        ctx->save_for_backward({q, k, v, t, n, m, p, o[1], o[2]});
        ctx->saved_data["edges"] = edges;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        return {o[0]};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        const variable_list s = ctx->get_saved_variables();
        return first_order(g, s, [&] {
            variable_list d = attn_bwd_(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8],
                                        {ctx->saved_data["edges"].toInt(), ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble()}, g[0]);
            d.resize(10);
            return d;
        });
    }
};
Tensor attention(const Tensor &q, const Tensor &k, const Tensor &v, const optional<Tensor> &table, const optional<Tensor> &lengths, const optional<Tensor> &keep,
                 const optional<Tensor> &offset, int64_t edges, bool causal, double scale) {
    const Tensor t = or_none(table);
    if (wanted({&q, &k, &v, &t})) return Attention::apply(q, k, v, table, lengths, keep, offset, edges, causal, scale)[0];
    return attn_fwd_(q, k, v, t, or_none(lengths), or_none(keep), or_none(offset), {edges, causal, scale}, false)[0];
}
std::tuple<Tensor, optional<Tensor>, optional<Tensor>> attn_fwd(const Tensor &q, const Tensor &k, const Tensor &v, const optional<Tensor> &table,
                                                               const optional<Tensor> &lengths, const optional<Tensor> &keep,
                                                               const optional<Tensor> &offset, int64_t edges, bool causal, double scale, bool train) {
    const variable_list o = attn_fwd_(q, k, v, or_none(table), or_none(lengths), or_none(keep), or_none(offset), {edges, causal, scale}, train);
    return {o[0], or_null(o[1]), or_null(o[2])};
}
std::tuple<Tensor, Tensor, Tensor, optional<Tensor>> attn_bwd(const Tensor &q, const Tensor &k, const Tensor &v, const optional<Tensor> &table,
                                                              const optional<Tensor> &lengths, const optional<Tensor> &keep, const optional<Tensor> &offset,
                                                              const optional<Tensor> &lse, const optional<Tensor> &out32, int64_t edges, bool causal,
                                                              double scale, const Tensor &g) {
    const variable_list d = attn_bwd_(q, k, v, or_none(table), or_none(lengths), or_none(keep), or_none(offset), or_none(lse), or_none(out32),
                                      {edges, causal, scale}, g);
    return {d[0], d[1], d[2], or_null(d[3])};
}

// --------------------------------------------------------------------------------------------- gated feed-forward --
void ff_call(asr_gated_ff_args &a, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act, bool backward) {
    a.x = x.data_ptr();
    a.wg = wg.data_ptr();
    a.wu = wu.data_ptr();
    a.wd = wd.data_ptr();
    a.M = x.size(0);
    a.d = size(x, 1), a.f = size(wg, 0), a.n = size(wd, 0);
    a.dtype = type_of(x);
    a.act = (int)act;
    Here here(x);
    const int64_t n = asr_gated_ff_ws_bytes(&a, backward);
    if (n < 0) check(-1);
    const Tensor ws = bytes(x, n);
    a.ws = ws.data_ptr();
    check(backward ? asr_gated_ff_bwd(&a, here.stream) : asr_gated_ff_fwd(&a, here.stream));
}
Tensor ff_fwd(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act) {
    Tensor y = at::empty({x.size(0), wd.size(0)}, x.options());
    if (!y.size(0)) return y;
    asr_gated_ff_args a{};
    a.y = y.data_ptr();
    ff_call(a, x, wg, wu, wd, act, false);
    return y;
}
// gradients of x and the three weights; none where `need` says so (the two first weights' come together)
variable_list ff_bwd_(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act, const Tensor &dy0, const std::array<bool, 4> &need) {
    if (!x.size(0)) return {at::zeros_like(x), at::zeros_like(wg), at::zeros_like(wu), at::zeros_like(wd)};
    const bool gate = need[1] || need[2];
    const Tensor dy = dy0.contiguous();
    auto like = [](const Tensor &t, bool on) { return on ? at::empty(t.sizes(), t.options()) : Tensor(); };
    Tensor dx = like(x, need[0]), dwg = like(wg, gate), dwu = like(wu, gate), dwd = like(wd, need[3]);
    asr_gated_ff_args a{};
    a.dy = dy.data_ptr();
    a.dx = ptr(dx);
    a.dwg = ptr(dwg);
    a.dwu = ptr(dwu);
    a.dwd = ptr(dwd);
    ff_call(a, x, wg, wu, wd, act, true);
    return {dx, dwg, dwu, dwd};
}
struct GatedFF : torch::autograd::Function<GatedFF> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act) {
        ctx->save_for_backward({x, wg, wu, wd});
        ctx->saved_data["act"] = act;
        return ff_fwd(x, wg, wu, wd, act);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        const variable_list s = ctx->get_saved_variables();
        return first_order(g, s, [&] {
            variable_list d = ff_bwd_(s[0], s[1], s[2], s[3], ctx->saved_data["act"].toInt(), g[0],
                                      {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)});
            d.resize(5);
            return d;
        });
    }
};
Tensor ff(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act) {
    return wanted({&x, &wg, &wu, &wd}) ? GatedFF::apply(x, wg, wu, wd, act) : ff_fwd(x, wg, wu, wd, act);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> ff_bwd(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act, const Tensor &dy) {
    const variable_list d = ff_bwd_(x, wg, wu, wd, act, dy, {true, true, true, true});
    return {d[0], d[1], d[2], d[3]};
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("rope", &rope);
    m.def("rope_fwd", &rope_fwd);
    m.def("rope_bwd", &rope_bwd);
    m.def("attention", &attention);
    m.def("attn_fwd", &attn_fwd);
    m.def("attn_bwd", &attn_bwd);
    m.def("ff", &ff);
    m.def("ff_fwd", &ff_fwd);
    m.def("ff_bwd", &ff_bwd);
}
