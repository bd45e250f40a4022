// The token operators as C++ autograd nodes over the C ABI (as host_ext.cpp does for the conv block): attention with a relative position bias, the gated residual
// between two norms, distillation from top logits.  Their kernels take 10 to 100 us at the framework's token counts; a Python autograd.Function around them took
// 120 to 200 us a forward + backward.  Arguments are checked by the callers in passion_amd/ops.py; here: allocation, device, stream, the calls.
// Nothing is kept between calls: workspaces are tensors of the call, so streams, captured graphs and threads share nothing.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "passion_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptT = std::optional<at::Tensor>;

struct Abi {
    decltype(&passion_rel_attn_workspace_floats) rel_ws = nullptr;
    decltype(&passion_rel_attn_fwd) rel_fwd = nullptr;
    decltype(&passion_rel_attn_bwd) rel_bwd = nullptr;
    decltype(&passion_residual_norm_part_floats) rn_part = nullptr;
    decltype(&passion_residual_norm_fwd) rn_fwd = nullptr;
    decltype(&passion_residual_norm_bwd) rn_bwd = nullptr;
    decltype(&passion_topk_distill_fwd) ds_fwd = nullptr;
    decltype(&passion_topk_distill_bwd) ds_bwd = nullptr;
} g;

inline void* cur_stream() { return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream().stream()); }
inline int code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? PASSION_BF16 : PASSION_F32; }
inline void check(int64_t rc, const char* what) { TORCH_CHECK(rc >= 0, what, " failed with code ", rc); }
inline void* ptr(const OptT& t) { return t && t->defined() ? t->data_ptr() : nullptr; }
inline void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* fptr(const OptT& t) { return static_cast<float*>(ptr(t)); }
inline float* fptr(const at::Tensor& t) { return static_cast<float*>(ptr(t)); }
inline bool wants(const OptT& t) { return t && t->requires_grad(); }
inline void bound(const void* f) { TORCH_CHECK(f, "passion_amd host extension is not bound to libpassion_hip.so"); }
// The kernels are launched outside torch's dispatcher: what follows calls there instead of the autograd node would go on without them (a tangent lost, a trace or an exported
// graph that holds the allocation of the result and nothing else).  Such calls are refused
inline bool refused(const at::Tensor& t) { return t.defined() && (t._fw_grad(/*level=*/0).defined() || t.unsafeGetTensorImpl()->is_python_dispatch()); }
inline bool refused(const OptT& t) { return t && refused(*t); }
template <typename... Ts> void eager_only(const char* what, const Ts&... ts) {
    using Mode = c10::impl::TorchDispatchModeKey;
    TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " can not be traced: its kernels are no torch operators");
    for (const Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL})
        TORCH_CHECK(!c10::impl::TorchDispatchModeTLS::get_mode(m), what, " can not be traced: its kernels are no torch operators");
    TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode), what, " does not support torch.func transforms");
    TORCH_CHECK(!(refused(ts) || ...), what, " takes plain tensors: no forward-mode derivatives, no tensor subclasses that dispatch to Python");
}
inline void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "this operator has no second derivative"); }
inline OptT opt(const at::Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
// as the kernels read a whole tensor: dense and on a 16-byte point
inline at::Tensor dense(const at::Tensor& t) {
    at::Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}

// ---------------------------------------------------------------------------------------------------------------- rel_attention
// geo: grid (3), q_start, table rows
struct RelCall {
    int dt, B, Nq, Nk, H, Hkv, D, nb;
    int geo[4];
    int64_t sq[3], sk[3], sv[3];
    RelCall(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::IntArrayRef gm) {
        dt = code(q);
        B = (int)q.size(0); Nq = (int)q.size(1); Nk = (int)k.size(1); H = (int)q.size(2); Hkv = (int)k.size(2); D = (int)q.size(3);
        for (int i = 0; i < 4; ++i) geo[i] = (int)gm[i];
        nb = (int)gm[4];
        for (int i = 0; i < 3; ++i) { sq[i] = q.stride(i); sk[i] = k.stride(i); sv[i] = v.stride(i); }
    }
    at::Tensor workspace(const at::Tensor& q, int backward, bool table, bool buckets) const {
        const int64_t n = g.rel_ws(dt, backward, B, Nq, Nk, H, Hkv, D, geo[0], geo[1], geo[2], geo[3], table, buckets, nb);
        check(n, "passion_rel_attn_workspace_floats");
        return n ? at::empty({n}, q.options().dtype(at::kFloat)) : at::Tensor();
    }
};

at::Tensor rel_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& table, const OptT& buckets, const OptT& mask, at::IntArrayRef geo,
                       double scale, at::Tensor* lse) {
    const c10::DeviceGuard guard(q.device());
    const RelCall c(q, k, v, geo);
    at::Tensor out = at::empty(q.sizes(), q.options());
    if (lse) *lse = at::empty({c.B, c.H, c.Nq}, q.options().dtype(at::kFloat));
    if (out.numel() == 0 || c.Nk == 0) return out.zero_();
    const at::Tensor ws = c.workspace(q, 0, table.has_value(), buckets.has_value());
    check(g.rel_fwd(q.data_ptr(), c.sq, k.data_ptr(), c.sk, v.data_ptr(), c.sv, c.dt, c.B, c.Nq, c.Nk, c.H, c.Hkv, c.D, c.geo[0], c.geo[1], c.geo[2], c.geo[3], ptr(table),
                    table ? code(*table) : 0, static_cast<const int*>(ptr(buckets)), c.nb, static_cast<const uint8_t*>(ptr(mask)), (float)scale, out.data_ptr(),
                    lse ? fptr(*lse) : nullptr, fptr(ws), cur_stream()),
          "passion_rel_attn_fwd");
    return out;
}

struct RelNode : public torch::autograd::Function<RelNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& table, const OptT& buckets, const OptT& mask,
                                 std::vector<int64_t> geo, double scale) {
        at::Tensor lse;
        const at::Tensor out = rel_forward(q, k, v, table, buckets, mask, geo, scale, &lse);
        ctx->save_for_backward({q, k, v, table.value_or(at::Tensor()), buckets.value_or(at::Tensor()), mask.value_or(at::Tensor()), out, lse});
        ctx->saved_data["geo"] = std::move(geo);
        ctx->saved_data["scale"] = scale;
        return {out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const variable_list s = ctx->get_saved_variables();
        const at::Tensor &q = s[0], &k = s[1], &v = s[2];
        const OptT table = opt(s[3]), buckets = opt(s[4]), mask = opt(s[5]);
        const c10::DeviceGuard guard(q.device());
        const std::vector<int64_t> geo = ctx->saved_data["geo"].toIntVector();
        const RelCall c(q, k, v, geo);
        at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options()), dt;
        if (table && ctx->needs_input_grad(3)) dt = at::empty(table->sizes(), table->options());
        if (q.numel() == 0 || c.Nk == 0) {
            dq.zero_(); dk.zero_(); dv.zero_();
            if (dt.defined()) dt.zero_();
        } else {
            const at::Tensor dout = dense(grads[0]);
            const at::Tensor ws = c.workspace(q, dt.defined() ? 1 : 2, table.has_value(), buckets.has_value());
            check(g.rel_bwd(q.data_ptr(), c.sq, k.data_ptr(), c.sk, v.data_ptr(), c.sv, c.dt, c.B, c.Nq, c.Nk, c.H, c.Hkv, c.D, c.geo[0], c.geo[1], c.geo[2], c.geo[3], ptr(table),
                            table ? code(*table) : 0, static_cast<const int*>(ptr(buckets)), c.nb, static_cast<const uint8_t*>(ptr(mask)),
                            (float)ctx->saved_data["scale"].toDouble(), s[6].data_ptr(), dout.data_ptr(), fptr(s[7]), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ptr(dt),
                            fptr(ws), cur_stream()),
                  "passion_rel_attn_bwd");
        }
        return {dq, dk, dv, dt, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

at::Tensor rel_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& table, const OptT& buckets, const OptT& mask, std::vector<int64_t> geo,
                         double scale) {
    bound(reinterpret_cast<const void*>(g.rel_fwd));
    eager_only("rel_attention", q, k, v, table, buckets, mask);
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || wants(table)))
        return RelNode::apply(q, k, v, table, buckets, mask, std::move(geo), scale)[0];
    return rel_forward(q, k, v, table, buckets, mask, geo, scale, nullptr);
}

// ---------------------------------------------------------------------------------------------------------------- residual_norm
// meta: post, pre, gate mode, B, N; eps: post, pre
variable_list rn_forward(const at::Tensor& x, const at::Tensor& h, const OptT& gate, const OptT& scale, const OptT& w1, const OptT& b1, const OptT& w2, const OptT& b2,
                         at::IntArrayRef m, const std::vector<double>& eps, at::Tensor* stat) {
    const c10::DeviceGuard guard(x.device());
    at::Tensor r = at::empty(x.sizes(), x.options()), y;
    if (m[1]) y = at::empty(h.sizes(), h.options());
    if (stat) *stat = at::empty({m[3] * m[4], 4}, x.options().dtype(at::kFloat));
    if (x.numel())
        check(g.rn_fwd(x.data_ptr(), code(x), h.data_ptr(), code(h), fptr(w1), fptr(b1), (int)m[0], (float)eps[0], ptr(gate), (int)m[2], gate ? code(*gate) : 0, fptr(scale),
                       fptr(w2), fptr(b2), (int)m[1], (float)eps[1], (int)m[3], (int)m[4], (int)x.size(-1), r.data_ptr(), ptr(y), stat ? fptr(*stat) : nullptr, cur_stream()),
              "passion_residual_norm_fwd");
    if (y.defined()) return {r, y};
    return {r};
}

struct RnNode : public torch::autograd::Function<RnNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& h, const OptT& gate, const OptT& scale, const OptT& w1, const OptT& b1, const OptT& w2,
                                 const OptT& b2, std::vector<int64_t> meta, std::vector<double> eps) {
        at::Tensor stat;
        variable_list out = rn_forward(x, h, gate, scale, w1, b1, w2, b2, meta, eps, &stat);
        auto t = [](const OptT& o) { return o.value_or(at::Tensor()); };
        ctx->save_for_backward({x, h, t(gate), t(scale), t(w1), t(b1), t(w2), stat});
        meta.push_back(b2.has_value());
        ctx->saved_data["meta"] = std::move(meta);
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        variable_list res(10);
        const variable_list s = ctx->get_saved_variables();
        const at::Tensor &x = s[0], &h = s[1], &gate = s[2];
        const std::vector<int64_t> m = ctx->saved_data["meta"].toIntVector();
        at::Tensor dr = grads[0], dy = m[1] ? grads[1] : at::Tensor();
        if (!dr.defined() && !dy.defined()) return res;
        const c10::DeviceGuard guard(x.device());
        if (dr.defined()) dr = dense(dr);
        if (dy.defined()) dy = dense(dy);
        const int64_t C = x.size(-1);
        const auto f32 = x.options().dtype(at::kFloat);
        res[0] = at::empty(x.sizes(), x.options());
        res[1] = at::empty(h.sizes(), h.options());
        // edges exist for the tensors that are there: x, h, then the optional ones in order
        int edge = 2;
        const bool there[6] = {gate.defined(), s[3].defined(), s[4].defined(), s[5].defined(), s[6].defined(), m[5] != 0};
        at::Tensor cols = at::empty({5, C}, f32);
        for (int i = 0; i < 6; ++i) {
            if (!there[i]) continue;
            if (ctx->needs_input_grad(edge)) res[2 + i] = i ? cols[i - 1] : at::empty(gate.sizes(), gate.options());
            ++edge;
        }
        if (!x.numel()) {
            for (int i = 2; i < 8; ++i) if (res[i].defined()) res[i].zero_();
            return res;
        }
        const at::Tensor part = at::empty({g.rn_part((int)m[3], (int)m[4], (int)C)}, f32);
        check(g.rn_bwd(x.data_ptr(), code(x), h.data_ptr(), code(h), fptr(s[4]), fptr(s[5]), (int)m[0], ptr(gate), (int)m[2], gate.defined() ? code(gate) : 0, fptr(s[3]),
                       fptr(s[6]), (int)m[1], fptr(s[7]), ptr(dr), ptr(dy), (int)m[3], (int)m[4], (int)C, res[0].data_ptr(), res[1].data_ptr(), ptr(res[2]), fptr(res[4]),
                       fptr(res[5]), fptr(res[6]), fptr(res[7]), fptr(res[3]), fptr(part), cur_stream()),
              "passion_residual_norm_bwd");
        return res;
    }
};

variable_list residual_norm(const at::Tensor& x, const at::Tensor& h, const OptT& gate, const OptT& scale, const OptT& w1, const OptT& b1, const OptT& w2, const OptT& b2,
                            std::vector<int64_t> meta, std::vector<double> eps) {
    bound(reinterpret_cast<const void*>(g.rn_fwd));
    eager_only("residual_norm", x, h, gate, scale, w1, b1, w2, b2);
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || h.requires_grad() || wants(gate) || wants(scale) || wants(w1) || wants(b1) || wants(w2) || wants(b2)))
        return RnNode::apply(x, h, gate, scale, w1, b1, w2, b2, std::move(meta), std::move(eps));
    return rn_forward(x, h, gate, scale, w1, b1, w2, b2, meta, eps, nullptr);
}

// ---------------------------------------------------------------------------------------------------------------- topk_distill
at::Tensor ds_forward(const at::Tensor& s, const at::Tensor& tv, const at::Tensor& ti, double temp, at::Tensor* lse) {
    const c10::DeviceGuard guard(s.device());
    const int64_t R = s.size(0);
    at::Tensor loss = at::empty({R}, s.options().dtype(at::kFloat));
    if (lse) *lse = at::empty({R, 2}, s.options().dtype(at::kFloat));
    if (R)
        check(g.ds_fwd(s.data_ptr(), code(s), tv.data_ptr(), code(tv), ti.data_ptr(), ti.scalar_type() == at::kLong, R, (int)s.size(1), (int)tv.size(1), (float)temp, fptr(loss),
                       lse ? fptr(*lse) : nullptr, cur_stream()),
              "passion_topk_distill_fwd");
    return loss;
}

struct DsNode : public torch::autograd::Function<DsNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& s, const at::Tensor& tv, const at::Tensor& ti, double temp) {
        at::Tensor lse;
        const at::Tensor loss = ds_forward(s, tv, ti, temp, &lse);
        ctx->save_for_backward({s, tv, ti, lse});
        ctx->saved_data["temp"] = temp;
        return {loss};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const variable_list v = ctx->get_saved_variables();
        const at::Tensor &s = v[0], &tv = v[1], &ti = v[2];
        const c10::DeviceGuard guard(s.device());
        at::Tensor d = at::empty(s.sizes(), s.options());
        if (s.size(0)) {
            const at::Tensor go = grads[0].contiguous();
            check(g.ds_bwd(s.data_ptr(), code(s), tv.data_ptr(), code(tv), ti.data_ptr(), ti.scalar_type() == at::kLong, s.size(0), (int)s.size(1), (int)tv.size(1),
                           (float)ctx->saved_data["temp"].toDouble(), fptr(v[3]), fptr(go), d.data_ptr(), cur_stream()),
                  "passion_topk_distill_bwd");
        }
        return {d, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

at::Tensor topk_distill(const at::Tensor& s, const at::Tensor& tv, const at::Tensor& ti, double temp) {
    bound(reinterpret_cast<const void*>(g.ds_fwd));
    eager_only("topk_distill", s, tv, ti);
    if (at::GradMode::is_enabled() && s.requires_grad()) return DsNode::apply(s, tv, ti, temp)[0];
    return ds_forward(s, tv, ti, temp, nullptr);
}

void bind_token_ops(const std::vector<uint64_t>& a) {
    TORCH_CHECK(a.size() == 8, "bind_token_ops: eight addresses");
    g.rel_ws = reinterpret_cast<decltype(g.rel_ws)>(a[0]);
    g.rel_fwd = reinterpret_cast<decltype(g.rel_fwd)>(a[1]);
    g.rel_bwd = reinterpret_cast<decltype(g.rel_bwd)>(a[2]);
    g.rn_part = reinterpret_cast<decltype(g.rn_part)>(a[3]);
    g.rn_fwd = reinterpret_cast<decltype(g.rn_fwd)>(a[4]);
    g.rn_bwd = reinterpret_cast<decltype(g.rn_bwd)>(a[5]);
    g.ds_fwd = reinterpret_cast<decltype(g.ds_fwd)>(a[6]);
    g.ds_bwd = reinterpret_cast<decltype(g.ds_bwd)>(a[7]);
}

}  // namespace

void register_token_ops(pybind11::module_& m) {
    m.def("bind_token_ops", &bind_token_ops, "addresses of the token operators' C-ABI entry points");
    m.def("rel_attention", &rel_attention);
    m.def("residual_norm", &residual_norm);
    m.def("topk_distill", &topk_distill);
}
