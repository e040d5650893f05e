// The operators of a student model of paperkiln_amd.ops and paperkiln_amd.blockops on torch tensors: layer norm with the residual addition, distillation from a
// teacher's top logits. As in post_ops.cpp: argument checks, allocation on the current stream of the tensors' device, the C ABI call, the autograd node.
#include "op_args.h"

namespace pk_torch {
namespace {

// ---- layer norm ----

constexpr const char* LN = "layernorm";
struct Rows {
    int64_t rows, cols, ld;
};
Rows rows_of(const char* what, const Tensor& x) {
    on_gpu(LN, x);
    if (x.dim() != 2 || x.size(1) < 1) refuse(LN, std::string("shape mismatch: ") + what + " is a [rows, cols] matrix");
    if (x.stride(1) != 1 && x.size(1) > 1) refuse(LN, std::string(what) + ": the columns must be contiguous");
    return Rows{x.size(0), x.size(1), x.size(0) > 1 ? x.stride(0) : x.size(1)};
}
Rows rows_like(const char* what, const Tensor& x, const Tensor& like) {
    const Rows r = rows_of(what, x);
    if (x.sizes() != like.sizes()) refuse(LN, std::string("shape mismatch: ") + what);
    if (x.scalar_type() != like.scalar_type()) refuse(LN, std::string("dtype mismatch: ") + what);
    if (x.device() != like.device()) refuse(LN, std::string(what) + " must live on the device of the other tensors");
    return r;
}
struct Normed {
    Tensor y, h, mean, rstd;
};
Normed norm_fwd(const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Tensor& residual) {
    const Rows m = rows_of("x", x);
    const pk_norm_shape s{m.rows, m.cols, dtype_code(x.scalar_type())};
    vector_of(LN, "w", w, at::kFloat, m.cols, x);
    if (b.defined()) vector_of(LN, "b", b, at::kFloat, m.cols, x);
    const Rows r = residual.defined() ? rows_like("residual", residual, x) : Rows{};
    c10::DeviceGuard on(x.device());
    at::AutoDispatchBelowAutograd below;
    Normed o;
    o.y = new_tensor(x.sizes(), x.scalar_type(), x);
    if (residual.defined()) o.h = new_tensor(x.sizes(), x.scalar_type(), x);
    o.mean = new_tensor({m.rows}, at::kFloat, x), o.rstd = new_tensor({m.rows}, at::kFloat, x);
    check(pk_layernorm_fwd(&s, x.const_data_ptr(), m.ld, residual.defined() ? residual.const_data_ptr() : nullptr, r.ld, w.const_data_ptr<float>(),
                           b.defined() ? b.const_data_ptr<float>() : nullptr, static_cast<float>(eps), o.y.data_ptr(), o.h.defined() ? o.h.data_ptr() : nullptr,
                           o.mean.data_ptr<float>(), o.rstd.data_ptr<float>(), stream()));
    return o;
}
std::vector<Tensor> norm_bwd(Tensor dy, const Tensor& h, const Tensor& w, const Tensor& mean, const Tensor& rstd, Tensor dh) {
    const Rows m = rows_of("h", h);
    const pk_norm_shape s{m.rows, m.cols, dtype_code(h.scalar_type())};
    vector_of(LN, "w", w, at::kFloat, m.cols, h);
    vector_of(LN, "mean", mean, at::kFloat, m.rows, h);
    vector_of(LN, "rstd", rstd, at::kFloat, m.rows, h);
    c10::DeviceGuard on(h.device());
    at::AutoDispatchBelowAutograd below;
    if (dy.dim() == 2 && dy.stride(1) != 1) dy = dy.contiguous();
    if (dh.defined() && dh.dim() == 2 && dh.stride(1) != 1) dh = dh.contiguous();
    const Rows g = rows_like("dy", dy, h), a = dh.defined() ? rows_like("dh", dh, h) : Rows{};
    Tensor dx = new_tensor(h.sizes(), h.scalar_type(), h), dw = new_tensor({m.cols}, at::kFloat, h), db = new_tensor({m.cols}, at::kFloat, h);
    const int64_t bytes = static_cast<int64_t>(pk_layernorm_bwd_workspace_bytes(&s));
    Tensor ws = new_tensor({bytes}, at::kByte, h);
    check(pk_layernorm_bwd(&s, dy.const_data_ptr(), g.ld, h.const_data_ptr(), m.ld, dh.defined() ? dh.const_data_ptr() : nullptr, a.ld, w.const_data_ptr<float>(),
                           mean.const_data_ptr<float>(), rstd.const_data_ptr<float>(), dx.data_ptr(), dw.data_ptr<float>(), db.data_ptr<float>(), ws.data_ptr(),
                           static_cast<size_t>(bytes), stream()));
    return {std::move(dx), std::move(dw), std::move(db)};
}
// Keeps what was normalised (its own second output, where there is a residual) and the rows' statistics.
struct LayerNormBackward : public Node {
    SavedVariable h, w, mean, rstd;
    bool has_residual = false;

    explicit LayerNormBackward(torch::autograd::edge_list&& next) : Node(std::move(next)) {}
    std::string name() const override { return "LayerNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        h.reset_data(), w.reset_data(), mean.reset_data(), rstd.reset_data();
    }
    variable_list apply(variable_list&& in) override {
        first_order(LN);
        recordable(LN, *this);
        Tensor th, tw, tm, tr;
        {
            const std::lock_guard<std::mutex> lock(mutex_);
            th = h.unpack(has_residual ? getptr() : nullptr), tw = w.unpack(), tm = mean.unpack(), tr = rstd.unpack();
        }
        auto g = norm_bwd(in[0].defined() ? in[0] : at::zeros_like(th), th, tw, tm, tr, has_residual ? in[1] : Tensor());
        return {g[0], has_residual ? g[0] : Tensor(), g[1], g[2]};  // of x, the residual, w, b
    }
};
Normed norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Tensor& residual) {
    for (const Tensor* t : {&x, &w, &b, &residual})
        if (t->defined()) no_tangent(LN, *t);
    Normed o = norm_fwd(x, w, b, eps, residual);
    const auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(residual))) {
        auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(torch::autograd::collect_next_edges(x, residual, w, b)), torch::autograd::deleteNode);
        node->has_residual = residual.defined();
        torch::autograd::set_history(o.y, node);
        if (o.h.defined()) torch::autograd::set_history(o.h, node);
        node->h = o.h.defined() ? SavedVariable(o.h, true) : SavedVariable(x, false);
        node->w = SavedVariable(w, false), node->mean = SavedVariable(o.mean, false), node->rstd = SavedVariable(o.rstd, false);
    }
    return o;
}

// ---- distillation ----

std::vector<Tensor> distill(const Tensor& logits, const Tensor& indices, const Tensor& teacher, const Tensor& weights, const pk_distill_config& c, const Tensor& lse,
                            bool grad, const Tensor& out) {
    constexpr const char* who = "distill_loss";
    const Logits m = matrix(who, "logits", logits);
    if (indices.dim() != 2 || teacher.dim() != 2 || indices.size(0) != m.rows || teacher.sizes() != indices.sizes())
        refuse(who, "shape mismatch: indices and teacher_logits are [rows, words]");
    const int64_t top = indices.size(1);
    vector_of(who, "indices", indices, at::kInt, m.rows * top, logits);
    vector_of(who, "teacher_logits", teacher, at::kFloat, m.rows * top, logits);
    vector_of(who, "weights", weights, at::kFloat, m.rows, logits);
    if (lse.defined()) vector_of(who, "teacher_lse", lse, at::kFloat, m.rows, logits);
    if (!grad && out.defined()) refuse(who, "out is for the gradient");
    c10::DeviceGuard on(logits.device());
    at::AutoDispatchBelowAutograd below;
    Tensor d = grad ? gradient_of(who, logits, out) : Tensor(), kl = new_tensor({m.rows}, at::kFloat, logits), rows = new_tensor({m.rows}, at::kDouble, logits),
           loss = new_tensor({}, at::kFloat, logits);
    const int64_t dld = grad ? matrix(who, "out", d).ld : 0;
    check(pk_distill_loss(&c, logits.const_data_ptr(), m.ld, indices.const_data_ptr<int>(), teacher.const_data_ptr<float>(),
                          lse.defined() ? lse.const_data_ptr<float>() : nullptr, weights.const_data_ptr<float>(), m.rows, m.vocab, top, grad ? d.data_ptr() : nullptr,
                          dld, kl.data_ptr<float>(), rows.data_ptr<double>(), loss.data_ptr<float>(), m.dtype, stream()));
    if (out.defined()) changed(out);
    return {std::move(loss), std::move(d), std::move(kl)};
}

// ---- gated delta rule ----

constexpr const char* DELTA = "gated_delta_rule";
pk_tensor4 heads_of(const char* what, const Tensor& x) {
    if (x.stride(3) != 1 && x.size(3) > 1 && x.numel() != 0) refuse(DELTA, std::string(what) + ": expected a [B,T,H,d] tensor with contiguous head_dim");
    return pk_tensor4{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}
pk_delta_shape delta_shape(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, double scale, const Tensor& state) {
    on_gpu(DELTA, q);
    if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || k.sizes() != q.sizes() || v.size(0) != q.size(0) || v.size(1) != q.size(1))
        refuse(DELTA, "shape mismatch: q and k are [B,T,Hk,dk], v [B,T,Hv,dv]");
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) refuse(DELTA, "dtype mismatch");
    for (const Tensor* x : {&k, &v})
        if (x->device() != q.device()) refuse(DELTA, "q, k and v must live on one device");
    pk_delta_shape s{};
    s.B = narrow(DELTA, q.size(0)), s.T = narrow(DELTA, q.size(1)), s.Hk = narrow(DELTA, q.size(2)), s.Hv = narrow(DELTA, v.size(2)), s.dk = narrow(DELTA, q.size(3)),
    s.dv = narrow(DELTA, v.size(3)), s.dtype = dtype_code(q.scalar_type()), s.scale = static_cast<float>(scale);
    const auto scalars = [&](const char* what, const Tensor& x) {
        if (x.dim() != 3 || x.size(0) != s.B || x.size(1) != s.T || x.size(2) != s.Hv) refuse(DELTA, std::string("shape mismatch: ") + what + " is [B,T,Hv]");
        vector_of(DELTA, what, x, at::kFloat, x.numel(), q);
    };
    scalars("g", g), scalars("beta", beta);
    if (state.defined()) {
        if (state.dim() != 4 || state.size(0) != s.B || state.size(1) != s.Hv || state.size(2) != s.dk || state.size(3) != s.dv) refuse(DELTA, "shape mismatch: the state is [B,Hv,dk,dv]");
        vector_of(DELTA, "the state", state, at::kFloat, state.numel(), q);
    }
    return s;
}
const float* floats(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
Tensor room(size_t bytes, const Tensor& like) { return bytes ? new_tensor({static_cast<int64_t>(bytes)}, at::kByte, like) : Tensor(); }

// o, and the state behind the last token: a new one, or `into`
std::pair<Tensor, Tensor> delta_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, double scale, const Tensor& state, const Tensor& into) {
    const pk_delta_shape s = delta_shape(q, k, v, g, beta, scale, state);
    c10::DeviceGuard on(q.device());
    at::AutoDispatchBelowAutograd below;
    Tensor o = new_tensor(v.sizes(), v.scalar_type(), q), last = into.defined() ? into : new_tensor({s.B, s.Hv, s.dk, s.dv}, at::kFloat, q);
    const size_t bytes = pk_delta_rule_fwd_workspace_bytes(&s);
    Tensor ws = room(bytes, q);
    const pk_tensor4 q4 = heads_of("q", q), k4 = heads_of("k", k), v4 = heads_of("v", v), o4 = heads_of("o", o);
    check(pk_delta_rule_fwd(&s, &q4, &k4, &v4, floats(g), floats(beta), floats(state), &o4, last.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    if (into.defined()) changed(into);
    return {std::move(o), std::move(last)};
}

std::vector<Tensor> delta_bwd(Tensor d_o, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, double scale, const Tensor& state,
                              const Tensor& dlast) {
    const pk_delta_shape s = delta_shape(q, k, v, g, beta, scale, state);
    if (d_o.sizes() != v.sizes() || d_o.scalar_type() != v.scalar_type() || d_o.device() != q.device()) refuse(DELTA, "shape mismatch: d_o");
    if (dlast.defined()) {
        if (dlast.dim() != 4 || dlast.size(0) != s.B || dlast.size(1) != s.Hv || dlast.size(2) != s.dk || dlast.size(3) != s.dv)
            refuse(DELTA, "shape mismatch: the state's gradient is [B,Hv,dk,dv]");
        vector_of(DELTA, "the state's gradient", dlast, at::kFloat, dlast.numel(), q);
    }
    c10::DeviceGuard on(q.device());
    at::AutoDispatchBelowAutograd below;
    if (d_o.stride(3) != 1) d_o = d_o.contiguous();
    Tensor dq = new_tensor(q.sizes(), q.scalar_type(), q), dk = new_tensor(k.sizes(), k.scalar_type(), q), dv = new_tensor(v.sizes(), v.scalar_type(), q),
           dg = new_tensor(g.sizes(), at::kFloat, q), dbeta = new_tensor(g.sizes(), at::kFloat, q), dfirst;
    if (state.defined()) dfirst = new_tensor(state.sizes(), at::kFloat, q);
    const size_t bytes = pk_delta_rule_bwd_workspace_bytes(&s);
    Tensor ws = room(bytes, q);
    const pk_tensor4 o4 = heads_of("d_o", d_o), q4 = heads_of("q", q), k4 = heads_of("k", k), v4 = heads_of("v", v), dq4 = heads_of("dq", dq), dk4 = heads_of("dk", dk), dv4 = heads_of("dv", dv);
    check(pk_delta_rule_bwd(&s, &o4, floats(dlast), &q4, &k4, &v4, floats(g), floats(beta), floats(state), &dq4, &dk4, &dv4, dg.data_ptr<float>(), dbeta.data_ptr<float>(),
                            dfirst.defined() ? dfirst.data_ptr<float>() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, stream()));
    return {std::move(dq), std::move(dk), std::move(dv), std::move(dg), std::move(dbeta), std::move(dfirst)};
}
// Keeps the inputs only: the backward forms the states again.
struct GatedDeltaRuleBackward : public Node {
    SavedVariable q, k, v, g, beta, state;
    bool has_state = false;
    double scale = 1.0;

    explicit GatedDeltaRuleBackward(torch::autograd::edge_list&& next) : Node(std::move(next)) {}
    std::string name() const override { return "GatedDeltaRuleBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* x : {&q, &k, &v, &g, &beta, &state}) x->reset_data();
    }
    variable_list apply(variable_list&& in) override {
        first_order(DELTA);
        recordable(DELTA, *this);
        Tensor tq, tk, tv, tg, tb, ts;
        {
            const std::lock_guard<std::mutex> lock(mutex_);
            tq = q.unpack(), tk = k.unpack(), tv = v.unpack(), tg = g.unpack(), tb = beta.unpack();
            if (has_state) ts = state.unpack();
        }
        return delta_bwd(in[0].defined() ? in[0] : at::zeros_like(tv), tq, tk, tv, tg, tb, scale, ts, in[1].defined() ? in[1].contiguous() : Tensor());
    }
};
std::pair<Tensor, Tensor> delta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, double scale, const Tensor& state) {
    bool wanted = false;
    for (const Tensor* t : {&q, &k, &v, &g, &beta, &state})
        if (t->defined()) no_tangent(DELTA, *t), wanted = wanted || t->requires_grad();
    auto y = delta_fwd(q, k, v, g, beta, scale, state, Tensor());
    if (at::GradMode::is_enabled() && wanted) {
        auto node = std::shared_ptr<GatedDeltaRuleBackward>(new GatedDeltaRuleBackward(torch::autograd::collect_next_edges(q, k, v, g, beta, state)), torch::autograd::deleteNode);
        torch::autograd::set_history(y.first, node);
        torch::autograd::set_history(y.second, node);
        node->q = SavedVariable(q, false), node->k = SavedVariable(k, false), node->v = SavedVariable(v, false), node->g = SavedVariable(g, false);
        node->beta = SavedVariable(beta, false), node->scale = scale, node->has_state = state.defined();
        if (state.defined()) node->state = SavedVariable(state, false);
    }
    return y;
}

// ---- Python side: positional arguments in the order ops.py and blockops.py pass them ----

PyObject* wrap(const Tensor& t) {  // None for one that there is not
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
PyObject* wrapped(std::initializer_list<Tensor> list) {
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(list.size()));
    if (!t) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor& x : list) PyTuple_SET_ITEM(t, i++, wrap(x));
    return t;
}

// (x, w, b or None, eps, residual or None) -> (y, h or None, mean, rstd)
PyObject* py_norm_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5);
    const Tensor &x = tensor_arg(a[0], "x"), &w = tensor_arg(a[1], "w");
    const Tensor b = optional_arg(a[2], "b"), residual = optional_arg(a[4], "residual");
    const double eps = float_arg(a[3]);
    Normed o;
    {
        pybind11::gil_scoped_release no_gil;
        o = norm_fwd(x, w, b, eps, residual);
    }
    return wrapped({o.y, o.h.defined() ? o.h : x, o.mean, o.rstd});
    END_HANDLE_TH_ERRORS
}
// (dy, h, w, mean, rstd, dh or None) -> (dx, dw, db)
PyObject* py_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6);
    const Tensor &dy = tensor_arg(a[0], "dy"), &h = tensor_arg(a[1], "h"), &w = tensor_arg(a[2], "w"), &mean = tensor_arg(a[3], "mean"), &rstd = tensor_arg(a[4], "rstd");
    const Tensor dh = optional_arg(a[5], "dh");
    std::vector<Tensor> g;
    {
        pybind11::gil_scoped_release no_gil;
        g = norm_bwd(dy, h, w, mean, rstd, dh);
    }
    return tuple_of(std::move(g));
    END_HANDLE_TH_ERRORS
}
// (x, w, b or None, eps, residual or None) -> y, or (y, h) with a residual, on the tape
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5);
    const Tensor &x = tensor_arg(a[0], "x"), &w = tensor_arg(a[1], "w");
    const Tensor b = optional_arg(a[2], "b"), residual = optional_arg(a[4], "residual");
    const double eps = float_arg(a[3]);
    Normed o;
    {
        pybind11::gil_scoped_release no_gil;
        o = norm(x, w, b, eps, residual);
    }
    if (!residual.defined()) return THPVariable_Wrap(std::move(o.y));
    return wrapped({o.y, o.h});
    END_HANDLE_TH_ERRORS
}
// (logits, indices, teacher_logits, weights, temperature, teacher_lse or None, upstream, grad, out or None) -> (loss, dlogits or None, kl)
PyObject* py_distill(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    const Tensor &x = tensor_arg(a[0], "logits"), &i = tensor_arg(a[1], "indices"), &t = tensor_arg(a[2], "teacher_logits"), &w = tensor_arg(a[3], "weights");
    const pk_distill_config c{float_arg(a[4]), number_arg(a[6])};
    const Tensor lse = optional_arg(a[5], "teacher_lse"), out = optional_arg(a[8], "out");
    const bool grad = bool_arg(a[7]);
    std::vector<Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = distill(x, i, t, w, c, lse, grad, out);
    }
    return wrapped({r[0], r[1], r[2]});
    END_HANDLE_TH_ERRORS
}

// (q, k, v, g, beta, scale, state or None) -> (o, state)
PyObject* py_delta_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7);
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &v = tensor_arg(a[2], "v"), &g = tensor_arg(a[3], "g"), &beta = tensor_arg(a[4], "beta");
    const double scale = float_arg(a[5]);
    const Tensor state = optional_arg(a[6], "state");
    std::pair<Tensor, Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = delta_fwd(q, k, v, g, beta, scale, state, Tensor());
    }
    return wrapped({r.first, r.second});
    END_HANDLE_TH_ERRORS
}
// (d_o, q, k, v, g, beta, scale, state or None, dstate or None) -> (dq, dk, dv, dg, dbeta, dstate or None)
PyObject* py_delta_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    const Tensor &d_o = tensor_arg(a[0], "d_o"), &q = tensor_arg(a[1], "q"), &k = tensor_arg(a[2], "k"), &v = tensor_arg(a[3], "v"), &g = tensor_arg(a[4], "g"),
                 &beta = tensor_arg(a[5], "beta");
    const double scale = float_arg(a[6]);
    const Tensor state = optional_arg(a[7], "initial_state"), dstate = optional_arg(a[8], "d_state");
    std::vector<Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = delta_bwd(d_o, q, k, v, g, beta, scale, state, dstate);
    }
    return wrapped({r[0], r[1], r[2], r[3], r[4], r[5]});
    END_HANDLE_TH_ERRORS
}
// (q, k, v, g, beta, scale, state or None) -> (o, state), on the tape
PyObject* py_delta(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7);
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &v = tensor_arg(a[2], "v"), &g = tensor_arg(a[3], "g"), &beta = tensor_arg(a[4], "beta");
    const double scale = float_arg(a[5]);
    const Tensor state = optional_arg(a[6], "initial_state");
    std::pair<Tensor, Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = delta(q, k, v, g, beta, scale, state);
    }
    return wrapped({r.first, r.second});
    END_HANDLE_TH_ERRORS
}
// (q, k, v, g, beta, scale, state) -> o, the state moved on in place
PyObject* py_delta_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7);
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &v = tensor_arg(a[2], "v"), &g = tensor_arg(a[3], "g"), &beta = tensor_arg(a[4], "beta"),
                 &state = tensor_arg(a[6], "state");
    const double scale = float_arg(a[5]);
    Tensor o;
    {
        pybind11::gil_scoped_release no_gil;
        for (const Tensor* t : {&q, &k, &v, &g, &beta, &state}) {
            no_tangent(DELTA, *t);
            if (at::GradMode::is_enabled() && t->requires_grad()) refuse(DELTA, "a step moves its state on in place and is not differentiable: no tensor of it may require a gradient (torch.no_grad)");
        }
        o = delta_fwd(q, k, v, g, beta, scale, state, state).first;
    }
    return THPVariable_Wrap(std::move(o));
    END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"gated_delta_rule_fwd", reinterpret_cast<PyCFunction>(py_delta_fwd), METH_FASTCALL, "(o, state)"},
    {"gated_delta_rule_bwd", reinterpret_cast<PyCFunction>(py_delta_bwd), METH_FASTCALL, "(dq, dk, dv, dg, dbeta, dstate or None)"},
    {"gated_delta_rule", reinterpret_cast<PyCFunction>(py_delta), METH_FASTCALL, "(o, state), differentiable"},
    {"gated_delta_step", reinterpret_cast<PyCFunction>(py_delta_step), METH_FASTCALL, "o, the state moved on in place"},
    {"layernorm_fwd", reinterpret_cast<PyCFunction>(py_norm_fwd), METH_FASTCALL, "(y, h, mean, rstd)"},
    {"layernorm_bwd", reinterpret_cast<PyCFunction>(py_norm_bwd), METH_FASTCALL, "(dx, dw, db)"},
    {"layernorm", reinterpret_cast<PyCFunction>(py_norm), METH_FASTCALL, "y or (y, h), differentiable"},
    {"distill_loss", reinterpret_cast<PyCFunction>(py_distill), METH_FASTCALL, "(loss, dlogits or None, kl)"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* student_methods() { return g_methods; }

}  // namespace pk_torch
