// gast_hip._temporal: the sequence operators as torch functions -- checks of the arguments, autograd nodes and the calls of the C ABI.
//
// A call on one frame is a few microseconds of GPU work, and a training step's nodes run on autograd's own thread: in Python the checks, the
// node and the handing over of the interpreter lock cost several times the kernels.  The C ABI (include/gast_hip.h) stays as it is; its two
// 16-bit flavours are opened here by path and chosen by the tensors' type.  gast_hip/temporal.py documents the functions.
#include <dlfcn.h>
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/gast_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---------------------------------------------------------------- the C ABI
struct Lib {
    decltype(&gast_rotary_multi) rotary;
    decltype(&gast_layer_norm_fwd) norm_fwd;
    decltype(&gast_layer_norm_bwd) norm_bwd;
    decltype(&gast_layer_norm_bwd_ws_floats) norm_ws;
    decltype(&gast_decay_fwd) decay_fwd;
    decltype(&gast_decay_bwd) decay_bwd;
    decltype(&gast_decay_ws_floats) decay_ws;
    decltype(&gast_decay_step) decay_step;
};
std::string paths[2];                  // bfloat16 and binary16 storage

template <typename F> void symbol(void* so, F& f, const char* name) {
    f = (F)dlsym(so, name);
    TORCH_CHECK(f, "gast_hip: no symbol ", name);
}
Lib open_lib(int which) {
    void* so = dlopen(paths[which].c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(so, "gast_hip: ", paths[which], " not found or not loadable -- build it with `python -c \"import __graft_entry__ as g; g.build()\"` "
                "(hipcc --offload-arch=gfx950). There is no CPU/PyTorch fallback. ", dlerror());
    Lib l;
    symbol(so, l.rotary, "gast_rotary_multi");
    symbol(so, l.norm_fwd, "gast_layer_norm_fwd");
    symbol(so, l.norm_bwd, "gast_layer_norm_bwd");
    symbol(so, l.norm_ws, "gast_layer_norm_bwd_ws_floats");
    symbol(so, l.decay_fwd, "gast_decay_fwd");
    symbol(so, l.decay_bwd, "gast_decay_bwd");
    symbol(so, l.decay_ws, "gast_decay_ws_floats");
    symbol(so, l.decay_step, "gast_decay_step");
    return l;
}
const Lib& lib(at::ScalarType t) {
    if (t == at::kHalf) {
        static const Lib l = open_lib(1);
        return l;
    }
    static const Lib l = open_lib(0);
    return l;
}
int code(at::ScalarType t) { return t == at::kFloat ? GAST_F32 : GAST_BF16; }

void done(int rc, const char* what) {
    if (rc == 0) return;
    const std::string name = rc == GAST_EINVAL ? "GAST_EINVAL" : rc == GAST_EALIGN ? "GAST_EALIGN" : rc == GAST_ERANGE ? "GAST_ERANGE" : "hipError " + std::to_string(rc);
    TORCH_CHECK(false, "gast_hip: ", what, " failed with ", name);
}

// kernels go to the current stream of the tensors' device, which is made the current one
struct Here {
    c10::DeviceGuard guard;
    gast_stream_t stream;
    explicit Here(const Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// ---------------------------------------------------------------- checks
void on_device(const char* what, const Tensor& t, std::initializer_list<const Tensor*> others) {
    const auto dt = t.scalar_type();
    TORCH_CHECK_VALUE(dt == at::kFloat || dt == at::kBFloat16 || dt == at::kHalf, what, ": float32, bfloat16 or float16 tensors, got ", dt);
    TORCH_CHECK(t.is_cuda(), what, ": tensors are on ", t.device(), "; the HIP path needs device tensors (no CPU fallback)");
    for (const Tensor* o : others) TORCH_CHECK(!o->defined() || o->device() == t.device(), what, ": tensors on ", t.device(), " and ", o->device());
}
bool records(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// Forward-mode derivatives are not there: a tangent would be left behind, which is a derivative of zero.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, ": there is no forward-mode derivative");
}
Tensor or_none(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }      // (nodes take no undefined inputs)

constexpr int64_t MAX_AXIS = int64_t(1) << 30;         // (the C ABI counts in int)

// (B, T, J, H, D) view of a (B, T, J, H, D) or (B, T, H, D) tensor, its channels contiguous
Tensor heads(const char* what, const char* name, const Tensor& t) {
    const auto n = t.dim();
    TORCH_CHECK_VALUE(n == 4 || n == 5, what, ": ", name, " has to be (B, T, J, H, D) or (B, T, H, D), got ", t.sizes());
    for (int i = 2; i < n; ++i) TORCH_CHECK_VALUE(t.size(i) > 0, what, ": ", name, " has an empty axis: ", t.sizes());
    for (int i = 0; i < n; ++i) TORCH_CHECK_VALUE(t.size(i) <= MAX_AXIS, what, ": ", name, " has an axis longer than ", MAX_AXIS, ": ", t.sizes());
    const Tensor c = t.stride(n - 1) == 1 || t.size(n - 1) == 1 ? t : t.contiguous();
    return n == 4 ? c.unsqueeze(2) : c;
}
gast_seq seq(const Tensor& t) {
    const auto s = t.strides();
    return gast_seq{t.data_ptr(), s[0], s[1], s[2], s[3]};
}
float* f32(const Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor last_contiguous(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

// There is no second derivative: a gradient that is recorded, or that is made from an input of the call that is (of[i], for outs[i]), gets a
// node that says so.
variable_list first_order(const char* what, const variable_list& grads, variable_list outs, std::initializer_list<bool> of = {}) {
    if (!at::GradMode::is_enabled()) return outs;
    bool any = false;
    for (const Tensor& g : grads) any = any || (g.defined() && g.requires_grad());
    for (size_t i = 0; i < outs.size(); ++i) {
        Tensor& o = outs[i];
        if (!o.defined() || !(any || (i < of.size() && of.begin()[i]))) continue;
        Tensor d = o.detach();
        d.set_requires_grad(true);
        o = (*std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": trying to differentiate twice, there is no second derivative", 1))({d})[0];
    }
    return outs;
}

// ---------------------------------------------------------------- rotary positions
using Turn = std::tuple<Tensor, Tensor, bool, double>;      // positions (B or 1, T), frequencies, interleaved, scale

std::vector<Tensor> rotate(const std::vector<Tensor>& xs, const Turn& how, bool backward) {
    const auto& [positions, freqs, interleaved, scale] = how;
    std::vector<Tensor> ys;
    gast_rotary_job jobs[GAST_ROTARY_MAX_BATCH];
    for (const Tensor& x : xs) {
        ys.push_back(fresh(x));
        jobs[ys.size() - 1] = gast_rotary_job{seq(x), seq(ys.back()), (int)x.size(3)};
    }
    const Tensor& x = xs[0];
    if (x.numel() == 0) return ys;
    const Here here(x);
    done(lib(x.scalar_type()).rotary(code(x.scalar_type()), jobs, (int)xs.size(), (int)x.size(0), (int)x.size(1), (int)x.size(2), (int)x.size(4),
                                     2 * (int)freqs.size(0), interleaved, positions.data_ptr(), positions.scalar_type() == at::kLong,
                                     positions.size(0) > 1 ? positions.stride(0) : 0, positions.stride(1), (const double*)freqs.data_ptr(), (float)scale,
                                     backward, here.stream), "gast_rotary_multi");
    return ys;
}

struct RotaryNode : torch::autograd::Function<RotaryNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& a, const optional<Tensor>& b, const optional<Tensor>& c, const optional<Tensor>& d,
                                 const Tensor& positions, const Tensor& freqs, bool interleaved, double scale) {
        ctx->save_for_backward({positions, freqs});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        std::vector<Tensor> xs = {a};
        for (const auto* t : {&b, &c, &d})
            if (t->has_value()) xs.push_back(**t);
        return rotate(xs, {positions, freqs, interleaved, scale}, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        const auto saved = ctx->get_saved_variables();
        std::vector<Tensor> src;
        std::vector<size_t> at;
        for (size_t i = 0; i < dys.size(); ++i)
            if (dys[i].defined() && ctx->needs_input_grad(i)) {
                src.push_back(last_contiguous(dys[i]));
                at.push_back(i);
            }
        variable_list out(8);
        if (!src.empty()) {
            const auto got = rotate(src, {saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble()}, true);
            for (size_t i = 0; i < at.size(); ++i) out[at[i]] = got[i];
        }
        return first_order("rotary", dys, out);
    }
};

std::vector<Tensor> rotary(const std::vector<Tensor>& given, Tensor positions, const Tensor& freqs, bool interleaved, double scale) {
    TORCH_CHECK_VALUE(!given.empty() && given.size() <= GAST_ROTARY_MAX_BATCH, "rotary: 1 to ", GAST_ROTARY_MAX_BATCH, " tensors in a call, got ", given.size());
    std::vector<Tensor> xs;
    for (const Tensor& t : given) {
        no_tangents("rotary", {&t, &freqs});
        xs.push_back(heads("rotary", "x", t));
    }
    const Tensor& x = xs[0];
    const int64_t B = x.size(0), T = x.size(1), D = x.size(4);
    for (const Tensor& t : xs)
        TORCH_CHECK_VALUE(t.size(0) == B && t.size(1) == T && t.size(2) == x.size(2) && t.size(4) == D && t.scalar_type() == x.scalar_type(),
                          "rotary: tensors of one call differ in their heads alone, got ", x.sizes(), " ", x.scalar_type(), " and ", t.sizes(), " ", t.scalar_type());
    TORCH_CHECK_VALUE(freqs.dim() == 1 && freqs.scalar_type() == at::kDouble && freqs.size(0) >= 1 && freqs.size(0) <= D / 2,
                      "rotary: freqs is a float64 vector of 1 to ", D / 2, " frequencies, got ", freqs.scalar_type(), " ", freqs.sizes());
    TORCH_CHECK_VALUE(!records({&freqs}), "rotary: the frequencies are fixed: there is no gradient for freqs (pass freqs.detach())");
    TORCH_CHECK_VALUE(D <= GAST_ROTARY_MAX_D, "rotary: at most ", GAST_ROTARY_MAX_D, " channels a head, got ", D);
    TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "rotary: positions are int32 or int64, got ", positions.scalar_type());
    if (positions.dim() == 1 && positions.size(0) == T) positions = positions.unsqueeze(0);
    TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(1) == T && (positions.size(0) == B || positions.size(0) == 1), "rotary: positions have to be (", T,
                      ",) or (", B, ", ", T, "), got ", positions.sizes());
    on_device("rotary", x, {&positions, &freqs});
    for (const Tensor& t : xs) on_device("rotary", x, {&t});
    const Tensor f = freqs.contiguous();
    bool record = false;
    for (const Tensor& t : xs) record = record || records({&t});
    std::vector<Tensor> ys;
    if (record) {
        Tensor a[GAST_ROTARY_MAX_BATCH];
        for (size_t i = 0; i < xs.size(); ++i) a[i] = xs[i];
        ys = RotaryNode::apply(a[0], maybe(a[1]), maybe(a[2]), maybe(a[3]), positions, f, interleaved, scale);
    } else {
        ys = rotate(xs, {positions, f, interleaved, scale}, false);
    }
    for (size_t i = 0; i < ys.size(); ++i)
        if (given[i].dim() == 4) ys[i] = ys[i].squeeze(2);
    return ys;
}

// ---------------------------------------------------------------- linear attention with a decay
gast_decay_args decay_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const Tensor& lengths, double scale) {
    gast_decay_args a = {};
    a.dtype = code(q.scalar_type());
    a.B = (int)q.size(0); a.T = (int)q.size(1); a.J = (int)q.size(2); a.H = (int)q.size(3); a.Dk = (int)q.size(4); a.Dv = (int)v.size(4);
    a.scale = (float)scale;
    a.log_decay = f32(log_decay);
    a.lengths = (const int32_t*)ptr(lengths);
    a.q = seq(q); a.k = seq(k); a.v = seq(v);
    a.state = f32(state);
    return a;
}
Tensor decay_ws(const Lib& l, gast_decay_args& a, const Tensor& like) {
    const long n = l.decay_ws(a.dtype, a.B, a.T, a.J, a.H, a.Dk, a.Dv);
    Tensor ws;
    if (n) ws = floats(like, {n});
    a.ws = f32(ws);
    return ws;
}

variable_list decay_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const Tensor& lengths,
                            double scale, bool want_state, Tensor* segments = nullptr) {
    const Tensor o = fresh(v);
    Tensor next;
    if (want_state) next = floats(q, {q.size(0), q.size(2), q.size(3), q.size(4), v.size(4)});
    if (q.size(0) * q.size(1) > 0) {
        const Here here(q);
        const Lib& l = lib(q.scalar_type());
        gast_decay_args a = decay_args(q, k, v, log_decay, state, lengths, scale);
        a.o = seq(o);
        a.state_out = f32(next);
        const Tensor ws = decay_ws(l, a, q);
        done(l.decay_fwd(&a, here.stream), "gast_decay_fwd");
        if (segments) *segments = ws;
    } else if (want_state) {
        if (state.defined()) next.copy_(state);
        else next.zero_();
    }
    return want_state ? variable_list{o, next} : variable_list{o};
}

struct DecayNode : torch::autograd::Function<DecayNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                 const optional<Tensor>& state_, const optional<Tensor>& lengths_, double scale, bool want_state) {
        const Tensor state = or_none(state_), lengths = or_none(lengths_);
        Tensor segments;                                   // the states before the segments of a long sequence: the backward pass wants them again
        variable_list out = decay_forward(q, k, v, log_decay, state, lengths, scale, want_state, &segments);
        ctx->save_for_backward({q, k, v, log_decay, state, lengths, segments});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["trained"] = (int64_t)(q.requires_grad() + 2 * k.requires_grad() + 4 * v.requires_grad() + 8 * (state.defined() && state.requires_grad()));
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &state = s[4];
        const bool only_state = !grads[0].defined();
        if (only_state && (grads.size() < 2 || !grads[1].defined())) return variable_list(8);
        const Tensor dq = fresh(q), dk = fresh(k), dv = fresh(v);
        Tensor dstate, dnext = grads.size() > 1 ? grads[1] : Tensor();
        if (state.defined() && ctx->needs_input_grad(4)) dstate = fresh(state);
        if (dnext.defined()) dnext = dnext.contiguous();
        if (q.size(0) * q.size(1) > 0) {
            const Here here(q);
            const Lib& l = lib(q.scalar_type());
            Tensor d_o, queries = q;
            if (only_state) {              // the state does not see the queries, infinities among them neither: one row of zeros stands for all
                const Tensor none = at::zeros({GAST_DECAY_MAX_D}, v.options());
                d_o = none.narrow(0, 0, v.size(4)).expand(v.sizes());
                queries = none.narrow(0, 0, q.size(4)).expand(q.sizes());
            } else {
                d_o = last_contiguous(grads[0]);
            }
            gast_decay_args a = decay_args(queries, k, v, s[3], state, s[5], ctx->saved_data["scale"].toDouble());
            a.d_o = seq(d_o); a.dq = seq(dq); a.dk = seq(dk); a.dv = seq(dv);
            a.dstate_out = f32(dnext);
            a.dstate = f32(dstate);
            const Tensor ws = decay_ws(l, a, q);
            a.ws_fwd = f32(s[6]);
            done(l.decay_bwd(&a, here.stream), "gast_decay_bwd");
        } else if (dstate.defined()) {
            if (dnext.defined()) dstate.copy_(dnext);
            else dstate.zero_();
        }
        // (the outputs are linear in each input: a gradient is made from the others)
        const int64_t t = ctx->saved_data["trained"].toInt();
        const bool tq = t & 1, tk = t & 2, tv = t & 4, ts = t & 8;
        return first_order("decay_attention", grads, {only_state ? Tensor() : dq, dk, dv, Tensor(), dstate, Tensor(), Tensor(), Tensor()},
                           {tk || tv || ts, tq || tv, tq || tk, false, tq});
    }
};

// q, k, v are (B, T, J, H, D) views; brings log_decay and lengths into the kernels' form and returns the scale
double decay_check(const char* what, const Tensor& q, const Tensor& k, const Tensor& v, Tensor& log_decay, const Tensor& state, Tensor& lengths,
                   const optional<double>& scale) {
    const int64_t B = q.size(0), T = q.size(1), J = q.size(2), H = q.size(3), Dk = q.size(4), Dv = v.size(4);
    TORCH_CHECK_VALUE(k.sizes() == q.sizes() && v.sizes().slice(0, 4) == q.sizes().slice(0, 4), what, ": q, k and v differ: ", q.sizes(), ", ", k.sizes(), ", ",
                      v.sizes(), " (shared heads: expand them)");
    TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), what, ": q, k and v have types ", q.scalar_type(), ", ",
                      k.scalar_type(), ", ", v.scalar_type());
    TORCH_CHECK_VALUE(std::max(Dk, Dv) <= GAST_DECAY_MAX_D, what, ": at most ", GAST_DECAY_MAX_D, " channels a head, got ", Dk, " and ", Dv);
    TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == H && log_decay.is_floating_point(), what, ": log_decay holds one number for each of the ", H,
                      " heads, got ", log_decay.scalar_type(), " ", log_decay.sizes());
    TORCH_CHECK_VALUE(!records({&log_decay}), what, ": the decays are fixed: there is no gradient for log_decay (pass log_decay.detach())");
    if (state.defined())
        TORCH_CHECK_VALUE(state.sizes() == at::IntArrayRef({B, J, H, Dk, Dv}) && state.scalar_type() == at::kFloat, what, ": the state has to be float32 (", B, ", ",
                          J, ", ", H, ", ", Dk, ", ", Dv, "), got ", state.scalar_type(), " ", state.sizes());
    if (lengths.defined())
        TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == B && (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong), what,
                          ": lengths holds ", B, " integers, got ", lengths.scalar_type(), " ", lengths.sizes());
    on_device(what, q, {&k, &v, &log_decay, &state, &lengths});
    log_decay = log_decay.to(at::kFloat).contiguous();
    if (lengths.defined()) lengths = (lengths.scalar_type() == at::kInt ? lengths : lengths.clamp(0, T).to(at::kInt)).contiguous();
    return scale.has_value() ? *scale : 1.0 / std::sqrt((double)Dk);
}

variable_list decay_attention(const Tensor& q, const Tensor& k, const Tensor& v, Tensor log_decay, const optional<Tensor>& state_, const optional<Tensor>& lengths_,
                              const optional<double>& scale_, bool return_state) {
    const char* what = "decay_attention";
    const Tensor Q = heads(what, "q", q), K = heads(what, "k", k), V = heads(what, "v", v);
    Tensor state = or_none(state_), lengths = or_none(lengths_);
    no_tangents(what, {&q, &k, &v, &log_decay, &state});
    const double scale = decay_check(what, Q, K, V, log_decay, state, lengths, scale_);
    if (state.defined()) state = state.contiguous();
    variable_list out = records({&q, &k, &v, &state}) ? DecayNode::apply(Q, K, V, log_decay, maybe(state), maybe(lengths), scale, return_state)
                                                      : decay_forward(Q, K, V, log_decay, state, lengths, scale, return_state);
    if (q.dim() == 4) out[0] = out[0].squeeze(2);
    return out;
}

Tensor decay_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, Tensor log_decay, const Tensor& state, const optional<Tensor>& lengths_,
                            const optional<double>& scale_) {
    const char* what = "decay_attention_step";
    TORCH_CHECK_VALUE(q.dim() == k.dim() && q.dim() == v.dim() && (q.dim() == 3 || q.dim() == 4), what, ": q, k and v have to be (B, J, H, D) or (B, H, D), got ",
                      q.sizes(), ", ", k.sizes(), ", ", v.sizes());
    TORCH_CHECK(!records({&q, &k, &v, &state}), what, " updates the state in place and has no gradient: call it under torch.no_grad(), or use decay_attention");
    no_tangents(what, {&q, &k, &v, &log_decay, &state});
    const Tensor Q = heads(what, "q", q.unsqueeze(1)), K = heads(what, "k", k.unsqueeze(1)), V = heads(what, "v", v.unsqueeze(1));
    TORCH_CHECK_VALUE(state.is_contiguous(), what, ": the state has to be contiguous, got strides ", state.strides(), " of ", state.sizes());
    Tensor lengths = or_none(lengths_);
    const double scale = decay_check(what, Q, K, V, log_decay, state, lengths, scale_);
    const Tensor o = fresh(V);
    if (q.size(0)) {
        const Here here(q);
        gast_decay_args a = decay_args(Q, K, V, log_decay, state, lengths, scale);
        a.o = seq(o);
        state.unsafeGetTensorImpl()->bump_version();   // (a graph that has saved this state notices)
        done(lib(q.scalar_type()).decay_step(&a, here.stream), "gast_decay_step");
    }
    return o.view(v.sizes());
}

// ---------------------------------------------------------------- layer norm
// (rows, C) view with contiguous channels and one stride between rows; a copy where there is none
Tensor rows_of(const Tensor& t) {
    const int64_t C = t.size(-1), rows = t.numel() / C;
    if (t.dim() == 2 && (t.stride(1) == 1 || C == 1)) return t;
    if (t.is_contiguous()) return t.view({rows, C});
    if (t.stride(-1) == 1 && t.dim() > 2 && rows) {
        bool even = true;
        for (int64_t i = 0; i + 2 < t.dim(); ++i) even = even && t.stride(i) == t.stride(i + 1) * t.size(i + 1);
        if (even) return t.view({rows, C});
    }
    return t.contiguous().view({rows, C});
}
struct Drop {
    int64_t thresh;
    double inv_keep;
    int64_t salt;
};

struct NormOut { Tensor y, stream, normed, stats; };

NormOut norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, const Tensor& seed, double eps, const Drop& d, bool train) {
    NormOut r;
    const Tensor X = rows_of(x);
    const int64_t rows = X.size(0), C = X.size(1);
    r.y = fresh(x);
    if (train) r.stats = floats(x, {2, rows});
    Tensor R;
    if (residual.defined()) {
        R = rows_of(residual);
        r.stream = fresh(x);
    }
    r.normed = r.stream.defined() ? r.stream.view({rows, C}) : X;
    if (rows) {
        const Here here(x);
        const gast_dropout drop = {(const uint32_t*)ptr(seed), (uint32_t)d.thresh, (float)d.inv_keep};
        float* mean = f32(r.stats);
        done(lib(x.scalar_type()).norm_fwd(code(x.scalar_type()), X.data_ptr(), X.stride(0), ptr(R), R.defined() ? R.stride(0) : 0, rows, (int)C, f32(weight), f32(bias),
                                           (float)eps, seed.defined(), (uint32_t)d.salt, drop, ptr(r.stream), C, r.y.data_ptr(), C, mean,
                                           mean ? mean + rows : nullptr, here.stream), "gast_layer_norm_fwd");
    }
    return r;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual_, const optional<Tensor>& weight_,
                                 const optional<Tensor>& bias_, const optional<Tensor>& seed_, double eps, int64_t thresh, double inv_keep, int64_t salt) {
        const Tensor residual = or_none(residual_), weight = or_none(weight_), bias = or_none(bias_), seed = or_none(seed_);
        ctx->saved_data["given"] = (int64_t)(residual.defined() + 2 * weight.defined() + 4 * bias.defined());
        const bool stream = x.requires_grad() || (residual.defined() && residual.requires_grad());
        ctx->saved_data["trained"] = (int64_t)(stream + 2 * (weight.defined() && weight.requires_grad()));
        const NormOut r = norm_forward(x, residual, weight, bias, seed, eps, {thresh, inv_keep, salt}, true);
        ctx->save_for_backward({r.stream.defined() ? r.stream : r.normed, weight, r.stats, seed});
        ctx->saved_data["thresh"] = thresh;
        ctx->saved_data["inv_keep"] = inv_keep;
        ctx->saved_data["salt"] = salt;
        ctx->set_materialize_grads(false);
        return r.stream.defined() ? variable_list{r.y, r.stream} : variable_list{r.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        // (a node is called with no gradient at all where the one behind it gave none)
        if (!grads[0].defined() && (grads.size() < 2 || !grads[1].defined())) return variable_list(9);
        const auto s = ctx->get_saved_variables();
        const Tensor S = rows_of(s[0]), &weight = s[1], &stats = s[2], &seed = s[3];
        const int64_t rows = S.size(0), C = S.size(1);
        const Tensor dY = grads[0].defined() ? rows_of(grads[0]) : Tensor(), dStream = grads.size() > 1 && grads[1].defined() ? rows_of(grads[1]) : Tensor();
        const auto shape = (grads[0].defined() ? grads[0] : grads[1]).sizes();
        const int64_t given = ctx->saved_data["given"].toInt();
        size_t at = 0;                                 // (inputs are counted without those that were not given)
        const bool want_x = ctx->needs_input_grad(at++), want_r = (given & 1) && ctx->needs_input_grad(at++);
        const bool want_w = (given & 2) && ctx->needs_input_grad(at++), want_b = (given & 4) && ctx->needs_input_grad(at++);
        const bool shared = !seed.defined();           // without dropout the branch and the stream have the same gradient
        Tensor dS, dX, dw, db, ws;
        if (want_r || (want_x && shared)) dS = at::empty(shape, S.options());
        if (want_x && !shared) dX = at::empty(shape, S.options());
        if (want_w) dw = floats(S, {C});
        if (want_b) db = floats(S, {C});
        if (rows) {
            const Here here(S);
            const Lib& l = lib(S.scalar_type());
            if (want_w || want_b) ws = floats(S, {l.norm_ws(rows, (int)C)});
            const gast_dropout drop = {(const uint32_t*)ptr(seed), (uint32_t)ctx->saved_data["thresh"].toInt(), (float)ctx->saved_data["inv_keep"].toDouble()};
            done(l.norm_bwd(code(S.scalar_type()), ptr(dY), dY.defined() ? dY.stride(0) : 0, ptr(dStream), dStream.defined() ? dStream.stride(0) : 0, S.data_ptr(),
                            S.stride(0), rows, (int)C, f32(weight), f32(stats), f32(stats) + rows, !shared, (uint32_t)ctx->saved_data["salt"].toInt(), drop, ptr(dX), C,
                            ptr(dS), C, f32(dw), f32(db), f32(ws), here.stream), "gast_layer_norm_bwd");
        } else {
            if (want_w) dw.zero_();
            if (want_b) db.zero_();
        }
        // (the stream's gradient is made from the stream and the weight, the weight's from the stream, the bias' from neither)
        const int64_t t = ctx->saved_data["trained"].toInt();
        return first_order("layer_norm", grads, {want_x ? (shared ? dS : dX) : Tensor(), want_r ? dS : Tensor(), dw, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()},
                           {t != 0, t != 0, (t & 1) != 0});
    }
};

variable_list norm(const std::string& what, const Tensor& x, const optional<Tensor>& residual_, const optional<Tensor>& weight_, const optional<Tensor>& bias_, double eps,
                   bool dropping, const optional<Tensor>& seed_, int64_t thresh, double inv_keep, int64_t salt) {
    const int64_t C = x.dim() ? x.size(-1) : 0;
    TORCH_CHECK_VALUE(C > 0 && C <= MAX_AXIS, what, ": x needs a last axis of 1 to ", MAX_AXIS, " values to normalise, got ", x.sizes());
    const Tensor residual = or_none(residual_);
    Tensor weight = or_none(weight_), bias = or_none(bias_), seed = or_none(seed_);
    no_tangents(what.c_str(), {&x, &residual, &weight, &bias});
    TORCH_CHECK_VALUE(residual.defined() || what != "add_layer_norm", what, ": a residual is needed (layer_norm goes without)");
    if (residual.defined())
        TORCH_CHECK_VALUE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(), what, ": x and residual differ: ", x.sizes(), " ", x.scalar_type(),
                          " and ", residual.sizes(), " ", residual.scalar_type());
    for (const Tensor* t : {&weight, &bias})
        if (t->defined())
            TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == C && t->is_floating_point(), what, ": ", t == &weight ? "weight" : "bias", " holds ", C, " numbers, got ",
                              t->scalar_type(), " ", t->sizes());
    TORCH_CHECK_VALUE(eps >= 0, what, ": eps has to be at least 0, got ", eps);
    TORCH_CHECK_VALUE(!dropping || (seed.defined() && seed.numel() == 1 && seed.element_size() == 4 && !seed.is_floating_point()), what,
                      ": the dropout seed is a one-element int32 tensor");
    on_device(what.c_str(), x, {&residual, &weight, &bias, &seed});
    if (thresh == 0) seed = Tensor();
    if (weight.defined()) weight = weight.to(at::kFloat).contiguous();
    if (bias.defined()) bias = bias.to(at::kFloat).contiguous();
    if (records({&x, &residual, &weight, &bias})) return NormNode::apply(x, maybe(residual), maybe(weight), maybe(bias), maybe(seed), eps, thresh, inv_keep, salt);
    const NormOut r = norm_forward(x, residual, weight, bias, seed, eps, {thresh, inv_keep, salt}, false);
    return r.stream.defined() ? variable_list{r.y, r.stream} : variable_list{r.y};
}

}  // namespace

PYBIND11_MODULE(_temporal, m) {
    m.def("libraries", [](const std::string& bf16, const std::string& f16) { paths[0] = bf16; paths[1] = f16; });
    m.def("rotary", &rotary);
    m.def("decay_attention", &decay_attention);
    m.def("decay_attention_step", &decay_attention_step);
    m.def("norm", &norm);
}
