// The post-training operators of paperkiln_amd.ops and paperkiln_amd.blockops on torch tensors: argument checks, output and workspace allocation, the C ABI
// call and, for the two that stand inside a model, the autograd node. As in torch_ops.cpp Python keeps the signatures. Every call runs on the device of its
// tensors and on that device's current stream; outputs and workspaces come from torch's allocator on that stream.
#include <ATen/MemoryOverlap.h>

#include <cmath>

#include "op_args.h"

namespace pk_torch {
namespace {

// ---- per-head norms with rotation ----

constexpr const char* QK = "qk_norm_rope";
struct QkOptions {
    double theta, eps;
    int rotary;
    bool halves;
};
pk_tensor4 heads(const Tensor& x, const char* what) {
    if (x.dim() != 4 || (x.stride(3) != 1 && x.numel() != 0)) refuse(QK, std::string(what) + ": expected a [B,T,H,dk] tensor with contiguous head_dim");
    return pk_tensor4{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}
pk_qk_shape qk_shape(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& pos, const QkOptions& o) {
    on_gpu(QK, q);
    if (q.dim() != 4 || k.dim() != 4 || k.size(0) != q.size(0) || k.size(1) != q.size(1) || k.size(3) != q.size(3))
        refuse(QK, "shape mismatch: q is [B,T,Hq,dk], k [B,T,Hkv,dk]");
    if (k.scalar_type() != q.scalar_type()) refuse(QK, "dtype mismatch");
    if (k.device() != q.device()) refuse(QK, "k must live on the device of the other tensors");
    vector_of(QK, "wq", wq, at::kFloat, q.size(3), q);
    vector_of(QK, "wk", wk, at::kFloat, q.size(3), q);
    pk_qk_shape s{};
    s.B = narrow(QK, q.size(0)), s.T = narrow(QK, q.size(1)), s.Hq = narrow(QK, q.size(2)), s.Hkv = narrow(QK, k.size(2)), s.dk = narrow(QK, q.size(3));
    s.rotary = o.rotary, s.halves = o.halves, s.dtype = dtype_code(q.scalar_type()), s.eps = static_cast<float>(o.eps), s.theta = o.theta;
    if (pos.device() != q.device()) refuse(QK, "pos must live on the device of the other tensors");
    if (pos.scalar_type() != at::kInt) refuse(QK, "pos must be int32");
    const bool per_token = pos.dim() == 1 && pos.size(0) == s.T, per_row = pos.dim() == 2 && pos.size(1) == s.T && (pos.size(0) == s.B || pos.size(0) == 1);
    if (!per_token && !per_row) refuse(QK, "shape mismatch: pos is [T] or [B,T]");
    if (s.T > 1 && pos.stride(-1) != 1) refuse(QK, "pos must be contiguous along the tokens");
    s.pos_stride_b = per_token || pos.size(0) == 1 ? 0 : pos.stride(0);
    return s;
}
void like(const Tensor& y, const Tensor& x, const char* what) {
    if (y.sizes() != x.sizes() || y.scalar_type() != x.scalar_type() || y.device() != x.device()) refuse(QK, std::string("shape mismatch: ") + what);
}
void place(const Tensor& y, const Tensor& x) {
    like(y, x, "out");
    at::assert_no_internal_overlap(y);
}
std::pair<Tensor, Tensor> qk_fwd(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& pos, const QkOptions& o,
                                 const std::vector<Tensor>& out) {
    const pk_qk_shape s = qk_shape(q, k, wq, wk, pos, o);
    c10::DeviceGuard on(q.device());
    at::AutoDispatchBelowAutograd below;
    Tensor yq = out.empty() ? new_tensor(q.sizes(), q.scalar_type(), q) : out[0], yk = out.empty() ? new_tensor(k.sizes(), k.scalar_type(), q) : out[1];
    place(yq, q), place(yk, k);
    const pk_tensor4 q4 = heads(q, "q"), k4 = heads(k, "k"), yq4 = heads(yq, "out"), yk4 = heads(yk, "out");
    check(pk_qk_norm_rope_fwd(&s, &q4, &k4, wq.const_data_ptr<float>(), wk.const_data_ptr<float>(), pos.const_data_ptr<int>(), &yq4, &yk4, stream()));
    for (const Tensor& t : out) changed(t);
    return {std::move(yq), std::move(yk)};
}
std::vector<Tensor> qk_bwd(Tensor dyq, Tensor dyk, const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& pos,
                           const QkOptions& o, const std::vector<Tensor>& out) {
    const pk_qk_shape s = qk_shape(q, k, wq, wk, pos, o);
    c10::DeviceGuard on(q.device());
    at::AutoDispatchBelowAutograd below;
    like(dyq, q, "dyq"), like(dyk, k, "dyk");
    if (dyq.stride(3) != 1) dyq = dyq.contiguous();
    if (dyk.stride(3) != 1) dyk = dyk.contiguous();
    Tensor dq = out.empty() ? new_tensor(q.sizes(), q.scalar_type(), q) : out[0], dk = out.empty() ? new_tensor(k.sizes(), k.scalar_type(), q) : out[1];
    place(dq, q), place(dk, k);
    Tensor dwq = new_tensor(wq.sizes(), at::kFloat, q), dwk = new_tensor(wk.sizes(), at::kFloat, q);
    const int64_t bytes = static_cast<int64_t>(pk_qk_norm_rope_bwd_workspace_bytes(&s));
    Tensor ws = new_tensor({bytes > 16 ? bytes : 16}, at::kByte, q);
    const pk_tensor4 gq = heads(dyq, "dyq"), gk = heads(dyk, "dyk"), q4 = heads(q, "q"), k4 = heads(k, "k"), dq4 = heads(dq, "out"), dk4 = heads(dk, "out");
    check(pk_qk_norm_rope_bwd(&s, &gq, &gk, &q4, &k4, wq.const_data_ptr<float>(), wk.const_data_ptr<float>(), pos.const_data_ptr<int>(), &dq4, &dk4,
                              dwq.data_ptr<float>(), dwk.data_ptr<float>(), ws.data_ptr(), static_cast<size_t>(ws.numel()), stream()));
    for (const Tensor& t : out) changed(t);
    return {std::move(dq), std::move(dk), std::move(dwq), std::move(dwk)};
}

// Keeps the inputs only: the backward forms 1/rms again.
struct QkNormRopeBackward : public Node {
    SavedVariable q, k, wq, wk, pos;
    QkOptions options{};

    explicit QkNormRopeBackward(torch::autograd::edge_list&& next) : Node(std::move(next)) {}
    std::string name() const override { return "QkNormRopeBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        q.reset_data(), k.reset_data(), wq.reset_data(), wk.reset_data(), pos.reset_data();
    }
    variable_list apply(variable_list&& in) override {
        first_order(QK);
        recordable(QK, *this);
        Tensor tq, tk, twq, twk, tp;
        {
            const std::lock_guard<std::mutex> lock(mutex_);
            tq = q.unpack(), tk = k.unpack(), twq = wq.unpack(), twk = wk.unpack(), tp = pos.unpack();
        }
        auto g = qk_bwd(in[0].defined() ? in[0] : at::zeros_like(tq), in[1].defined() ? in[1] : at::zeros_like(tk), tq, tk, twq, twk, tp, options, {});
        return {std::move(g[0]), std::move(g[1]), std::move(g[2]), std::move(g[3])};
    }
};
std::pair<Tensor, Tensor> qk(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& pos, const QkOptions& o) {
    for (const Tensor* x : {&q, &k, &wq, &wk}) no_tangent(QK, *x);
    auto y = qk_fwd(q, k, wq, wk, pos, o, {});
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || wq.requires_grad() || wk.requires_grad())) {
        auto node = std::shared_ptr<QkNormRopeBackward>(new QkNormRopeBackward(torch::autograd::collect_next_edges(q, k, wq, wk)), torch::autograd::deleteNode);
        torch::autograd::set_history(y.first, node);
        torch::autograd::set_history(y.second, node);
        node->q = SavedVariable(q, false), node->k = SavedVariable(k, false), node->wq = SavedVariable(wq, false), node->wk = SavedVariable(wk, false);
        node->pos = SavedVariable(pos, false);
        node->options = o;
    }
    return y;
}

// ---- token log-probabilities and the losses on them ----

constexpr const char* LP = "token_logprobs";
std::pair<Tensor, Tensor> logprobs_fwd(const Tensor& logits, const Tensor& targets, double scale) {
    const Logits m = matrix(LP, "logits", logits);
    vector_of(LP, "targets", targets, at::kInt, m.rows, logits);
    c10::DeviceGuard on(logits.device());
    at::AutoDispatchBelowAutograd below;
    Tensor logp = new_tensor({m.rows}, at::kFloat, logits), lse = new_tensor({m.rows}, at::kFloat, logits);
    Tensor ws;
    const size_t bytes = pk_token_logprobs_workspace_bytes(m.rows, m.vocab, m.dtype);
    if (bytes) ws = new_tensor({static_cast<int64_t>(bytes)}, at::kByte, logits);
    check(pk_token_logprobs_fwd(logits.const_data_ptr(), m.ld, targets.const_data_ptr<int>(), m.rows, m.vocab, static_cast<float>(scale), logp.data_ptr<float>(),
                                lse.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr, bytes, m.dtype, stream()));
    return {std::move(logp), std::move(lse)};
}
Tensor logprobs_bwd(const Tensor& logits, const Tensor& targets, const Tensor& lse, const Tensor& dlogp, double scale, const Tensor& out) {
    const Logits m = matrix(LP, "logits", logits);
    vector_of(LP, "targets", targets, at::kInt, m.rows, logits);
    vector_of(LP, "lse", lse, at::kFloat, m.rows, logits);
    vector_of(LP, "dlogp", dlogp, at::kFloat, m.rows, logits);
    c10::DeviceGuard on(logits.device());
    at::AutoDispatchBelowAutograd below;
    Tensor d = gradient_of(LP, logits, out);
    const Logits g = matrix(LP, "out", d);
    check(pk_token_logprobs_bwd(logits.const_data_ptr(), m.ld, targets.const_data_ptr<int>(), lse.const_data_ptr<float>(), dlogp.const_data_ptr<float>(), m.rows,
                                m.vocab, static_cast<float>(scale), d.data_ptr(), g.ld, m.dtype, stream()));
    if (out.defined()) changed(out);
    return d;
}
struct TokenLogprobsBackward : public Node {
    SavedVariable logits, targets, lse;
    double scale = 1.0;

    explicit TokenLogprobsBackward(torch::autograd::edge_list&& next) : Node(std::move(next)) {}
    std::string name() const override { return "TokenLogprobsBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data(), targets.reset_data(), lse.reset_data();
    }
    variable_list apply(variable_list&& in) override {
        first_order(LP);
        recordable(LP, *this);
        Tensor x, t, l;
        {
            const std::lock_guard<std::mutex> lock(mutex_);
            x = logits.unpack(), t = targets.unpack(), l = lse.unpack();
        }
        return {logprobs_bwd(x, t, l, in[0].defined() ? in[0].contiguous() : at::zeros_like(l), scale, Tensor())};
    }
};
Tensor logprobs(const Tensor& logits, const Tensor& targets, double scale) {
    no_tangent(LP, logits);
    auto [logp, lse] = logprobs_fwd(logits, targets, scale);
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        auto node = std::shared_ptr<TokenLogprobsBackward>(new TokenLogprobsBackward(torch::autograd::collect_next_edges(logits)), torch::autograd::deleteNode);
        torch::autograd::set_history(logp, node);
        node->logits = SavedVariable(logits, false), node->targets = SavedVariable(targets, false), node->lse = SavedVariable(lse, false);
        node->scale = scale;
    }
    return logp;
}

std::vector<Tensor> policy(const Tensor& logits, const Tensor& targets, const Tensor& old, const Tensor& ref, const Tensor& adv, const Tensor& weights,
                           const pk_policy_config& c, const Tensor& out) {
    constexpr const char* who = "policy_loss";
    const Logits m = matrix(who, "logits", logits);
    vector_of(who, "targets", targets, at::kInt, m.rows, logits);
    vector_of(who, "old_logp", old, at::kFloat, m.rows, logits);
    vector_of(who, "advantages", adv, at::kFloat, m.rows, logits);
    vector_of(who, "weights", weights, at::kFloat, m.rows, logits);
    if (ref.defined()) vector_of(who, "ref_logp", ref, at::kFloat, m.rows, logits);
    c10::DeviceGuard on(logits.device());
    at::AutoDispatchBelowAutograd below;
    Tensor d = gradient_of(who, logits, out), logp = new_tensor({m.rows}, at::kFloat, logits), rows = new_tensor({m.rows}, at::kDouble, logits),
           loss = new_tensor({}, at::kFloat, logits), ws;
    const size_t bytes = pk_policy_loss_workspace_bytes(m.rows, m.vocab, m.dtype);
    if (bytes) ws = new_tensor({static_cast<int64_t>(bytes)}, at::kByte, logits);
    const Logits g = matrix(who, "out", d);
    check(pk_policy_loss(&c, logits.const_data_ptr(), m.ld, targets.const_data_ptr<int>(), old.const_data_ptr<float>(),
                         ref.defined() ? ref.const_data_ptr<float>() : nullptr, adv.const_data_ptr<float>(), weights.const_data_ptr<float>(), m.rows, m.vocab,
                         d.data_ptr(), g.ld, logp.data_ptr<float>(), rows.data_ptr<double>(), loss.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr, bytes, m.dtype, stream()));
    if (out.defined()) changed(out);
    return {std::move(loss), std::move(d), std::move(logp)};
}

std::vector<Tensor> preference(const Tensor& logits, const Tensor& targets, const Tensor& starts, const Tensor& ref, const pk_preference_config& c,
                               const Tensor& out) {
    constexpr const char* who = "preference_loss";
    const Logits m = matrix(who, "logits", logits);
    vector_of(who, "targets", targets, at::kInt, m.rows, logits);
    vector_of(who, "ref_logp", ref, at::kFloat, m.rows, logits);
    if (starts.numel() < 3 || starts.numel() % 2 == 0) refuse(who, "shape mismatch: seq_start has 2 * pairs + 1 values");
    vector_of(who, "seq_start", starts, at::kInt, starts.numel(), logits);
    const int64_t pairs = (starts.numel() - 1) / 2, bytes = static_cast<int64_t>(pk_preference_loss_workspace_bytes(m.rows, pairs));
    c10::DeviceGuard on(logits.device());
    at::AutoDispatchBelowAutograd below;
    Tensor d = gradient_of(who, logits, out), logp = new_tensor({m.rows}, at::kFloat, logits), margins = new_tensor({pairs}, at::kFloat, logits),
           loss = new_tensor({}, at::kFloat, logits), ws = new_tensor({bytes}, at::kByte, logits);
    const Logits g = matrix(who, "out", d);
    check(pk_preference_loss(&c, logits.const_data_ptr(), m.ld, targets.const_data_ptr<int>(), starts.const_data_ptr<int>(), pairs, ref.const_data_ptr<float>(),
                             m.rows, m.vocab, d.data_ptr(), g.ld, logp.data_ptr<float>(), margins.data_ptr<float>(), loss.data_ptr<float>(), ws.data_ptr(),
                             static_cast<size_t>(bytes), m.dtype, stream()));
    if (out.defined()) changed(out);
    return {std::move(loss), std::move(d), std::move(margins), std::move(logp)};
}

// ---- AdamW over a list ----

constexpr const char* ADAMW = "adamw_many_";
using Refs = std::vector<const Tensor*>;  // the caller's own tensors: hundreds of them, so the call keeps the interpreter lock rather than a reference to each
struct Lists {
    Refs p, g, m, v, ms, vs, copy;  // g: null where a parameter has no gradient; ms, vs, copy: empty where not asked for
};
void dense(const char* what, const Tensor& t, const Tensor& p, int64_t n, at::ScalarType type) {
    if (t.device() != p.device()) refuse(ADAMW, std::string(what) + " must live on the device of the parameters");
    if (t.scalar_type() != type) refuse(ADAMW, std::string("dtype mismatch: ") + what + " of " + at::toString(t.scalar_type()) + ", expected " + at::toString(type));
    if (t.numel() != n) refuse(ADAMW, std::string("shape mismatch: ") + what);
    if (!t.is_contiguous()) refuse(ADAMW, std::string(what) + " must be contiguous");
}
Tensor adamw_many(const Lists& l, pk_adamw_config c) {
    const size_t count = l.p.size();
    const bool bits8 = !l.ms.empty() || !l.vs.empty();
    for (const auto* x : {&l.g, &l.m, &l.v})
        if (x->size() != count) refuse(ADAMW, "shape mismatch: as many gradients and states as parameters are wanted");
    for (const auto* x : {&l.ms, &l.vs})
        if (bits8 && x->size() != count) refuse(ADAMW, "shape mismatch: as many scales as parameters are wanted");
    if (!l.copy.empty() && l.copy.size() != count) refuse(ADAMW, "shape mismatch: as many copies as parameters are wanted");
    c.state_bits = bits8 ? 8 : 32;
    if (count == 0) {
        if (c.max_norm > 0.0f) refuse(ADAMW, "a clip needs parameters");
        return Tensor();
    }
    on_gpu(ADAMW, *l.p[0]);
    const Tensor& first = *l.p[0];
    at::ScalarType g_type = at::kFloat;
    for (const Tensor* g : l.g)
        if (g) {
            g_type = g->scalar_type();
            break;
        }
    c.grad_dtype = dtype_code(g_type);
    std::vector<pk_adamw_tensor> table(count);
    for (size_t i = 0; i < count; ++i) {
        const int64_t n = l.p[i]->numel();
        pk_adamw_tensor& t = table[i];
        t = pk_adamw_tensor{};
        if (l.p[i]->device() != first.device()) refuse(ADAMW, "parameters of one call must live on one device");
        dense("a parameter", *l.p[i], first, n, at::kFloat);
        dense("m", *l.m[i], first, n, bits8 ? at::kFloat8_e4m3fn : at::kFloat);
        dense("v", *l.v[i], first, n, bits8 ? at::kFloat8_e5m2 : at::kFloat);
        if (bits8) {
            dense("m_scale", *l.ms[i], first, (n + 255) / 256, at::kFloat);
            dense("v_scale", *l.vs[i], first, (n + 255) / 256, at::kFloat);
        }
        if (!l.copy.empty()) dense("a copy", *l.copy[i], first, n, at::kBFloat16);
        if (!l.g[i]) continue;  // stays as it is; its place in the list is kept
        dense("a gradient", *l.g[i], first, n, g_type);
        t.p = static_cast<float*>(l.p[i]->data_ptr()), t.g = l.g[i]->const_data_ptr(), t.m = l.m[i]->data_ptr(), t.v = l.v[i]->data_ptr(), t.n = n;
        if (bits8) t.m_scale = static_cast<float*>(l.ms[i]->data_ptr()), t.v_scale = static_cast<float*>(l.vs[i]->data_ptr());
        if (!l.copy.empty()) t.copy = l.copy[i]->data_ptr();
    }
    c10::DeviceGuard on(first.device());
    at::AutoDispatchBelowAutograd below;
    Tensor norm, ws;
    if (c.max_norm > 0.0f) {
        norm = new_tensor({}, at::kFloat, first);
        ws = new_tensor({static_cast<int64_t>(pk_adamw_many_workspace_bytes(table.data(), static_cast<int>(count), &c))}, at::kByte, first);
    }
    check(pk_adamw_many(table.data(), static_cast<int>(count), &c, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? static_cast<size_t>(ws.numel()) : 0,
                        norm.defined() ? norm.data_ptr<float>() : nullptr, stream()));
    for (const auto* list : {&l.p, &l.m, &l.v, &l.ms, &l.vs, &l.copy})
        for (size_t i = 0; i < list->size(); ++i)
            if (l.g[i]) changed(*(*list)[i]);
    return norm;
}

// ---- Python side: positional arguments in the order ops.py and blockops.py pass them ----

Refs refs_arg(PyObject* o, const char* what, bool holes) {
    Refs v;
    if (o == Py_None) return v;
    if (!PyList_Check(o) && !PyTuple_Check(o)) throw torch::TypeError(std::string(what) + " must be a list or a tuple of tensors");  // what holds its items
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
    v.reserve(static_cast<size_t>(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* item = PySequence_Fast_GET_ITEM(o, i);
        if (THPVariable_Check(item))
            v.push_back(&THPVariable_Unpack(item));
        else if (holes && item == Py_None)
            v.push_back(nullptr);
        else
            throw torch::TypeError(std::string(what) + " must hold tensors");
    }
    return v;
}
std::vector<Tensor> two_arg(PyObject* o) {
    const Refs r = refs_arg(o, "out", false);
    if (o != Py_None && r.size() != 2) TORCH_CHECK_VALUE(false, "out must be two tensors");
    std::vector<Tensor> v;
    for (const Tensor* t : r) v.push_back(*t);
    return v;
}
QkOptions qk_options(PyObject* const* a) { return QkOptions{float_arg(a[0]), float_arg(a[1]), whole_arg(a[2], "rotary_dim"), bool_arg(a[3])}; }

// (q, k, wq, wk, pos, theta, eps, rotary_dim, halves, out) -> (yq, yk)
PyObject* py_qk_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &wq = tensor_arg(a[2], "wq"), &wk = tensor_arg(a[3], "wk"), &pos = tensor_arg(a[4], "pos");
    const QkOptions o = qk_options(a + 5);
    const std::vector<Tensor> out = two_arg(a[9]);
    std::pair<Tensor, Tensor> y;
    {
        pybind11::gil_scoped_release no_gil;
        y = qk_fwd(q, k, wq, wk, pos, o, out);
    }
    return tuple_of({std::move(y.first), std::move(y.second)});
    END_HANDLE_TH_ERRORS
}
// (dyq, dyk, q, k, wq, wk, pos, theta, eps, rotary_dim, halves, out) -> (dq, dk, dwq, dwk)
PyObject* py_qk_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 12);
    const Tensor &dyq = tensor_arg(a[0], "dyq"), &dyk = tensor_arg(a[1], "dyk"), &q = tensor_arg(a[2], "q"), &k = tensor_arg(a[3], "k"),
                 &wq = tensor_arg(a[4], "wq"), &wk = tensor_arg(a[5], "wk"), &pos = tensor_arg(a[6], "pos");
    const QkOptions o = qk_options(a + 7);
    const std::vector<Tensor> out = two_arg(a[11]);
    std::vector<Tensor> g;
    {
        pybind11::gil_scoped_release no_gil;
        g = qk_bwd(dyq, dyk, q, k, wq, wk, pos, o, out);
    }
    return tuple_of(std::move(g));
    END_HANDLE_TH_ERRORS
}
// (q, k, wq, wk, pos, theta, eps, rotary_dim, halves) -> (yq, yk), on the tape
PyObject* py_qk(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &wq = tensor_arg(a[2], "wq"), &wk = tensor_arg(a[3], "wk"), &pos = tensor_arg(a[4], "pos");
    const QkOptions o = qk_options(a + 5);
    std::pair<Tensor, Tensor> y;
    {
        pybind11::gil_scoped_release no_gil;
        y = qk(q, k, wq, wk, pos, o);
    }
    return tuple_of({std::move(y.first), std::move(y.second)});
    END_HANDLE_TH_ERRORS
}
// (logits, targets, scale) -> (logp, lse)
PyObject* py_logprobs_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3);
    const Tensor &x = tensor_arg(a[0], "logits"), &t = tensor_arg(a[1], "targets");
    const double scale = float_arg(a[2]);
    std::pair<Tensor, Tensor> y;
    {
        pybind11::gil_scoped_release no_gil;
        y = logprobs_fwd(x, t, scale);
    }
    return tuple_of({std::move(y.first), std::move(y.second)});
    END_HANDLE_TH_ERRORS
}
// (logits, targets, lse, dlogp, scale, out or None) -> dlogits
PyObject* py_logprobs_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6);
    const Tensor &x = tensor_arg(a[0], "logits"), &t = tensor_arg(a[1], "targets"), &lse = tensor_arg(a[2], "lse"), &g = tensor_arg(a[3], "dlogp");
    const double scale = float_arg(a[4]);
    const Tensor out = optional_arg(a[5], "out");
    Tensor d;
    {
        pybind11::gil_scoped_release no_gil;
        d = logprobs_bwd(x, t, lse, g, scale, out);
    }
    return THPVariable_Wrap(std::move(d));
    END_HANDLE_TH_ERRORS
}
// (logits, targets, scale) -> logp, on the tape
PyObject* py_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3);
    const Tensor &x = tensor_arg(a[0], "logits"), &t = tensor_arg(a[1], "targets");
    const double scale = float_arg(a[2]);
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        y = logprobs(x, t, scale);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}
// (logits, targets, old_logp, ref_logp or None, advantages, weights, clip_low, clip_high, kl_coef, scale, upstream, out or None) -> (loss, dlogits, logp)
PyObject* py_policy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 12);
    const Tensor &x = tensor_arg(a[0], "logits"), &t = tensor_arg(a[1], "targets"), &old = tensor_arg(a[2], "old_logp"), &adv = tensor_arg(a[4], "advantages"),
                 &w = tensor_arg(a[5], "weights");
    const Tensor ref = optional_arg(a[3], "ref_logp"), out = optional_arg(a[11], "out");
    const pk_policy_config c{number_arg(a[6]), number_arg(a[7]), number_arg(a[8]), number_arg(a[9]), number_arg(a[10])};
    std::vector<Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = policy(x, t, old, ref, adv, w, c, out);
    }
    return tuple_of(std::move(r));
    END_HANDLE_TH_ERRORS
}
// (logits, targets, seq_start, ref_logp, beta, label_smoothing, scale, upstream, out or None) -> (loss, dlogits, margins, logp)
PyObject* py_preference(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    const Tensor &x = tensor_arg(a[0], "logits"), &t = tensor_arg(a[1], "targets"), &starts = tensor_arg(a[2], "seq_start"), &ref = tensor_arg(a[3], "ref_logp");
    const pk_preference_config c{number_arg(a[4]), number_arg(a[5]), number_arg(a[6]), number_arg(a[7])};
    const Tensor out = optional_arg(a[8], "out");
    std::vector<Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = preference(x, t, starts, ref, c, out);
    }
    return tuple_of(std::move(r));
    END_HANDLE_TH_ERRORS
}
// (params, grads, m, v, m_scale or None, v_scale or None, copies or None, lr, b1, b2, eps, wd, t, max_norm, seed) -> norm or None
PyObject* py_adamw_many(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 15);
    Lists l;
    l.p = refs_arg(a[0], "params", false), l.g = refs_arg(a[1], "grads", true), l.m = refs_arg(a[2], "m", false), l.v = refs_arg(a[3], "v", false);
    l.ms = refs_arg(a[4], "m_scale", false), l.vs = refs_arg(a[5], "v_scale", false), l.copy = refs_arg(a[6], "copies", false);
    pk_adamw_config c{};
    c.lr = number_arg(a[7]), c.b1 = number_arg(a[8]), c.b2 = number_arg(a[9]), c.eps = number_arg(a[10]), c.wd = number_arg(a[11]);
    c.t = whole_arg(a[12], "t"), c.max_norm = number_arg(a[13]);
    PyObject* seed = PyNumber_Long(a[14]);
    if (!seed) throw python_error();
    const unsigned long long bits = PyLong_AsUnsignedLongLongMask(seed);  // any whole number; its low 32 bits count
    Py_DECREF(seed);
    if (bits == static_cast<unsigned long long>(-1) && PyErr_Occurred()) throw python_error();
    c.seed = static_cast<uint32_t>(bits);
    Tensor norm = adamw_many(l, c);
    if (!norm.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(norm));
    END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"qk_norm_rope_fwd", reinterpret_cast<PyCFunction>(py_qk_fwd), METH_FASTCALL, "(yq, yk)"},
    {"qk_norm_rope_bwd", reinterpret_cast<PyCFunction>(py_qk_bwd), METH_FASTCALL, "(dq, dk, dwq, dwk)"},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(py_qk), METH_FASTCALL, "(yq, yk), differentiable"},
    {"token_logprobs_fwd", reinterpret_cast<PyCFunction>(py_logprobs_fwd), METH_FASTCALL, "(logp, lse)"},
    {"token_logprobs_bwd", reinterpret_cast<PyCFunction>(py_logprobs_bwd), METH_FASTCALL, "dlogits"},
    {"token_logprobs", reinterpret_cast<PyCFunction>(py_logprobs), METH_FASTCALL, "logp, differentiable"},
    {"policy_loss", reinterpret_cast<PyCFunction>(py_policy), METH_FASTCALL, "(loss, dlogits, logp)"},
    {"preference_loss", reinterpret_cast<PyCFunction>(py_preference), METH_FASTCALL, "(loss, dlogits, margins, logp)"},
    {"adamw_many", reinterpret_cast<PyCFunction>(py_adamw_many), METH_FASTCALL, "one step over a list, in place: the norm before the clip or None"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* post_methods() { return g_methods; }

}  // namespace pk_torch
