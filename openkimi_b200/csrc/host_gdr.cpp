// Native host path of the gated delta rule (chunk_gated_delta_rule and its recurrent forms) and of group_norm: argument checks,
// memory, autograd and launches.  Nothing is kept from one call for the next.
#include "host_util.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

using namespace kda_host;

namespace {

void on_cuda(const Tensor& t, const char* what) {
    if (!t.is_cuda()) throw std::runtime_error(std::string(what) + " runs only on a CUDA device (sm_100a); there is no CPU fallback");
}
void same_device(const Tensor& x, const char* first, const char* name, const Tensor& t) {
    if (t.defined() && t.device() != x.device())
        throw std::runtime_error(std::string("expected ") + name + " on " + x.device().str() + ", the device of " + first +
                                 ", but it is on " + t.device().str());
}
int code(at::ScalarType t) { return t == at::kBFloat16 ? KDA_DTYPE_BF16 : KDA_DTYPE_F32; }
// type in which the kernels read g and beta: theirs where they share one that the kernels have, else FP32
at::ScalarType gate_type(const Tensor& g, const Tensor& beta) {
    return g.scalar_type() == at::kBFloat16 && beta.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
}

// Gradients whose own derivative is asked for (create_graph) raise when it is taken: the backward kernels have none.
variable_list differentiable_once(const char* what, variable_list r) {
    if (!at::GradMode::is_enabled()) return r;
    variable_list have;
    for (const Tensor& t : r)
        if (t.defined()) have.push_back(t.detach().requires_grad_());
    const std::string msg = std::string("the gradient of ") + what + " is not differentiable: its backward has no derivative";
    const variable_list out = (*std::make_shared<torch::autograd::DelayedError>(msg, (int64_t)have.size()))(std::move(have));
    size_t i = 0;
    for (Tensor& t : r)
        if (t.defined()) t = out[i++];
    return r;
}

// ---- gated delta rule ------------------------------------------------------------------------------------------------
struct Inputs {
    Tensor q, k, v, g, beta, A_log, dt_bias, h0;  // contiguous; undefined where absent
    Tensor cu, chunk_seq, seq_off, chunk_tab;     // packed documents only
};
struct Spec {
    double scale = 1.0;
    int flags = 0;
    bool want_state = false;
    bool covered = true;  // every row belongs to a sequence
    int64_t N = 0, NT = 0;
    int64_t longest = 0;  // chunks of the longest packed document
};

// sizes and types of one call; multi: q [B, T, H, K], else [N, H, K].  Returns {B, T, H, HV, K, V}.
std::array<int64_t, 6> check_shapes(const char* what, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                    const Tensor& beta, bool multi) {
    for (const Tensor* t : {&q, &k, &v, &g, &beta}) on_cuda(*t, what);
    const int64_t d = multi ? 4 : 3;
    const std::string lead = multi ? "[B,T," : "[N,";
    if (q.dim() != d || q.sizes() != k.sizes())
        value_error("q and k must have the same shape " + lead + "H,K], got q=" + shape_of(q) + " vs k=" + shape_of(k));
    if (v.dim() != d || v.sizes().slice(0, d - 2) != q.sizes().slice(0, d - 2))
        value_error("v must be " + lead + "HV,V] with the leading sizes of q, got " + shape_of(v));
    const int64_t H = q.size(d - 2), K = q.size(d - 1), HV = v.size(d - 2), V = v.size(d - 1);
    if (H < 1 || HV < 1 || HV % H)
        value_error("the number of value heads must be a multiple of the number of key heads, got HV=" + std::to_string(HV) +
                    " and H=" + std::to_string(H));
    if ((K != 64 && K != 128) || (V != 64 && V != 128))
        value_error("the gated delta rule kernels need K and V in (64, 128), got K=" + std::to_string(K) + ", V=" + std::to_string(V));
    for (const Tensor* t : {&g, &beta})
        if (t->sizes() != v.sizes().slice(0, d - 1))
            value_error(std::string(t == &g ? "g" : "beta") + " must have the shape of v without its last axis, got " + shape_of(*t));
    for (const Tensor* t : {&q, &k, &v, &g, &beta})
        if (!at::isFloatingType(t->scalar_type())) type_error(std::string("expected floating point tensors, got ") + c10::toString(t->scalar_type()));
    dtype_code(q);
    same_device(q, "q", "k", k); same_device(q, "q", "v", v); same_device(q, "q", "g", g); same_device(q, "q", "beta", beta);
    return {q.size(0), multi ? q.size(1) : 1, H, HV, K, V};
}
void check_gate(int64_t flags, const OptTensor& A_log, const OptTensor& dt_bias, int64_t HV) {
    if (!(flags & KDA_FLAG_GATE)) return;
    if (!A_log) value_error("A_log must be provided when use_gate_in_kernel=True.");
    if (A_log->numel() != HV || (dt_bias && dt_bias->numel() != HV)) value_error("A_log and dt_bias must have one entry per value head");
}
std::array<int64_t, 4> state_shape(int64_t N, int64_t HV, int64_t K, int64_t V, int64_t flags) {
    if (flags & KDA_FLAG_STATE_V_FIRST) return {N, HV, V, K};
    return {N, HV, K, V};
}
void check_state(const Tensor& s, const std::array<int64_t, 4>& want, const char* name) {
    if (s.scalar_type() != at::kFloat) type_error(std::string(name) + " must be in float32.");
    if (s.sizes() != at::IntArrayRef(want)) {
        std::string w;
        for (int64_t x : want) w += (w.empty() ? "" : ", ") + std::to_string(x);
        value_error(std::string(name) + " must have shape (" + w + "), got " + shape_of(s));
    }
}

KdaGdrParams params(const Inputs& in, const Spec& sp, int flags) {
    KdaGdrParams p{};
    p.B = (int)in.q.size(0); p.T = (int)in.q.size(1); p.H = (int)in.q.size(2); p.dk = (int)in.q.size(3);
    p.HV = (int)in.v.size(2); p.dv = (int)in.v.size(3);
    p.N = (int)sp.N; p.NT = (int)sp.NT; p.max_chunks = (int)sp.longest;
    p.dtype = code(in.q.scalar_type()); p.g_dtype = code(in.g.scalar_type());
    p.flags = flags;
    p.scale = (float)sp.scale;
    p.q = in.q.data_ptr(); p.k = in.k.data_ptr(); p.v = in.v.data_ptr(); p.g = in.g.data_ptr(); p.beta = in.beta.data_ptr();
    p.A_log = ptr<float>(in.A_log); p.dt_bias = ptr<float>(in.dt_bias); p.h0 = ptr<float>(in.h0);
    if (in.cu.defined()) {
        p.cu_seqlens = ptr<int64_t>(in.cu); p.chunk_seq = ptr<int32_t>(in.chunk_seq);
        p.seq_chunk_off = ptr<int32_t>(in.seq_off); p.chunk_tab = ptr<int32_t>(in.chunk_tab);
    }
    const StatusWord& st = status_word(in.q.device().index());
    p.status = st.dev.load(std::memory_order_relaxed);
    p.status_host = const_cast<int32_t*>(st.host);
    return p;
}
Tensor state_like(const Inputs& in, const Spec& sp) {
    return fresh(state_shape(sp.N, in.v.size(2), in.q.size(3), in.v.size(3), sp.flags), at::kFloat, in.q);
}

struct FwdOut { Tensor o, ht, ws; };

FwdOut run_fwd(const Inputs& in, const Spec& sp, bool keep) {
    FwdOut out;
    out.o = fresh_like(in.v);
    if (!sp.covered) out.o.zero_();
    if (sp.want_state) out.ht = state_like(in, sp);
    if (sp.NT == 0) {
        if (out.ht.defined()) {
            if (in.h0.defined()) out.ht.copy_(in.h0);
            else out.ht.zero_();
        }
        return out;
    }
    KdaGdrParams p = params(in, sp, keep ? sp.flags : sp.flags | KDA_FLAG_NO_SAVE);
    size_t n = 0;
    check_rc(kda_gdr_workspace_bytes(&p, &n, nullptr), "kda_gdr_workspace_bytes");
    out.ws = bytes(n, in.q);
    p.o = out.o.data_ptr(); p.ht = ptr<float>(out.ht);
    p.workspace = out.ws.data_ptr(); p.workspace_bytes = n;
    check_rc(kda_gdr_fwd(&p, stream_of(in.q)), "kda_gdr_fwd");
    return out;
}

struct Grads { Tensor q, k, v, g, beta, A_log, dt_bias, h0; };

Grads run_bwd(const Inputs& in, const Spec& sp, const Tensor& ws, const Tensor& grad_o, const Tensor& grad_ht) {
    Grads r;
    const bool gate = sp.flags & KDA_FLAG_GATE;
    r.q = fresh_like(in.q); r.k = fresh_like(in.k); r.v = fresh_like(in.v); r.g = fresh_like(in.g); r.beta = fresh_like(in.beta);
    if (gate) r.A_log = fresh_like(in.A_log);
    if (gate && in.dt_bias.defined()) r.dt_bias = fresh_like(in.dt_bias);
    if (in.h0.defined()) r.h0 = fresh_like(in.h0);
    const Tensor ght = grad_ht.defined() ? ready(grad_ht, at::kFloat) : Tensor();
    if (!sp.covered || sp.NT == 0)
        for (Tensor* t : {&r.q, &r.k, &r.v, &r.g, &r.beta}) t->zero_();
    if (sp.NT == 0) {
        for (Tensor* t : {&r.A_log, &r.dt_bias})
            if (t->defined()) t->zero_();
        if (r.h0.defined()) {
            if (ght.defined()) r.h0.copy_(ght);
            else r.h0.zero_();
        }
        return r;
    }
    KdaGdrParams p = params(in, sp, sp.flags);
    const Tensor go = grad_o.defined() ? ready(grad_o, in.q.scalar_type()) : at::zeros_like(in.v);
    size_t fwd = 0, bwd = 0;
    check_rc(kda_gdr_workspace_bytes(&p, &fwd, &bwd), "kda_gdr_workspace_bytes");
    const Tensor scratch = bytes(bwd, in.q);
    p.workspace = ws.data_ptr(); p.workspace_bytes = fwd;
    p.grad_o = go.data_ptr(); p.grad_ht = ptr<float>(ght);
    p.grad_q = r.q.data_ptr(); p.grad_k = r.k.data_ptr(); p.grad_v = r.v.data_ptr(); p.grad_g = r.g.data_ptr();
    p.grad_beta = r.beta.data_ptr();
    p.grad_A_log = ptr<float>(r.A_log); p.grad_dt_bias = ptr<float>(r.dt_bias); p.grad_h0 = ptr<float>(r.h0);
    p.bwd_scratch = scratch.data_ptr(); p.bwd_scratch_bytes = bwd;
    check_rc(kda_gdr_bwd(&p, stream_of(in.q)), "kda_gdr_bwd");
    return r;
}

Inputs gather(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Tensor& A_log,
              const Tensor& dt_bias, const Tensor& h0, const Inputs& tables) {
    Inputs in = tables;
    const auto dt = q.scalar_type(), gt = gate_type(g, beta);
    in.q = ready(q, dt); in.k = ready(k, dt); in.v = ready(v, dt); in.g = ready(g, gt); in.beta = ready(beta, gt);
    if (A_log.defined()) in.A_log = ready(A_log, at::kFloat);
    if (dt_bias.defined()) in.dt_bias = ready(dt_bias, at::kFloat);
    if (h0.defined()) in.h0 = ready(h0, at::kFloat);
    return in;
}

struct ChunkGdr : torch::autograd::Function<ChunkGdr> {
    static variable_list forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, OptTensor A_log,
                                 OptTensor dt_bias, OptTensor h0, const Inputs& tables, const Spec& sp) {
        const Inputs in = gather(q, k, v, g, beta, val(A_log), val(dt_bias), val(h0), tables);
        FwdOut f = run_fwd(in, sp, true);
        ctx->save_for_backward({in.q, in.k, in.v, in.g, in.beta, in.A_log, in.dt_bias, in.h0, in.cu, in.chunk_seq, in.seq_off,
                                in.chunk_tab, f.ws});
        ctx->set_materialize_grads(false);  // an unused final state has no gradient, rather than one of zeros
        ctx->saved_data["scale"] = sp.scale;
        ctx->saved_data["flags"] = (int64_t)sp.flags;
        ctx->saved_data["N"] = sp.N;
        ctx->saved_data["NT"] = sp.NT;
        ctx->saved_data["longest"] = sp.longest;
        ctx->saved_data["covered"] = sp.covered;
        if (f.ht.defined()) return {f.o, f.ht};
        return {f.o};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Inputs in = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10], s[11]};
        Spec sp;
        sp.scale = ctx->saved_data["scale"].toDouble();
        sp.flags = (int)ctx->saved_data["flags"].toInt();
        sp.N = ctx->saved_data["N"].toInt();
        sp.NT = ctx->saved_data["NT"].toInt();
        sp.longest = ctx->saved_data["longest"].toInt();
        sp.covered = ctx->saved_data["covered"].toBool();
        c10::cuda::CUDAGuard guard(in.q.device());
        const Grads r = run_bwd(in, sp, s[12], grads[0], grads.size() > 1 ? grads[1] : Tensor());
        // (the engine casts every gradient to its input's dtype)
        return differentiable_once("chunk_gated_delta_rule", {r.q, r.k, r.v, r.g, r.beta, r.A_log, r.dt_bias, r.h0, Tensor(), Tensor()});
    }
};

std::tuple<Tensor, OptTensor> chunk_gdr(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                        OptTensor A_log, OptTensor dt_bias, OptTensor h0, std::optional<double> scale, int64_t flags,
                                        bool want_state, OptTensor cu, OptTensor chunk_seq, OptTensor seq_off, OptTensor chunk_tab,
                                        int64_t NT, int64_t longest, bool covered) {
    const auto [B, T, H, HV, K, V] = check_shapes("chunk_gated_delta_rule", q, k, v, g, beta, true);
    Spec sp;
    Inputs tables;
    sp.N = B;
    sp.NT = B * ((T + CHUNK - 1) / CHUNK);
    if (cu) {
        if (B != 1) value_error("The batch size is expected to be 1 rather than " + std::to_string(B) + " when using `cu_seqlens`.");
        tables.cu = read_here(*cu); tables.chunk_seq = read_here(*chunk_seq); tables.seq_off = read_here(*seq_off); tables.chunk_tab = read_here(*chunk_tab);
        sp.N = cu->numel() - 1;
        sp.NT = NT;
        sp.longest = longest;
        sp.covered = covered;
    }
    check_gate(flags, A_log, dt_bias, HV);
    if (h0) check_state(*h0, state_shape(sp.N, HV, K, V, flags), "initial_state");
    Tensor a, b;
    if (flags & KDA_FLAG_GATE) {
        a = A_log->dim() == 1 ? *A_log : A_log->reshape({HV});
        if (dt_bias) b = dt_bias->dim() == 1 ? *dt_bias : dt_bias->reshape({HV});
    }
    const Tensor& h = val(h0);
    same_device(q, "q", "A_log", a); same_device(q, "q", "dt_bias", b); same_device(q, "q", "initial_state", h);
    sp.scale = scale.value_or(1.0 / std::sqrt((double)K));
    sp.flags = (int)flags;
    sp.want_state = want_state;
    const std::array<const Tensor*, 8> inputs = {&q, &k, &v, &g, &beta, &a, &b, &h};
    refuse_tangents(inputs);
    bool grad = false;
    if (at::GradMode::is_enabled())
        for (const Tensor* t : inputs) grad = grad || (t->defined() && t->requires_grad());
    c10::cuda::CUDAGuard guard(q.device());
    if (!grad) {
        at::NoGradGuard no_grad;
        const FwdOut f = run_fwd(gather(q, k, v, g, beta, a, b, h, tables), sp, false);
        return {f.o, opt(f.ht)};
    }
    const variable_list r = ChunkGdr::apply(q, k, v, g, beta, opt(a), opt(b), opt(h), tables, sp);
    return {r[0], r.size() > 1 ? OptTensor(r[1]) : OptTensor()};
}

std::tuple<Tensor, OptTensor> recurrent_gdr(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                            const OptTensor& state, const OptTensor& A_log, const OptTensor& dt_bias,
                                            std::optional<double> scale, int64_t flags, bool inplace, bool multi, bool want_state) {
    const auto [N, T, H, HV, K, V] = check_shapes(multi ? "fused_recurrent_gated_delta_rule" : "recurrent_gated_delta_rule_step", q, k, v, g, beta, multi);
    check_gate(flags, A_log, dt_bias, HV);
    const auto want = state_shape(N, HV, K, V, flags);
    if (!state && !multi) type_error("recurrent_gated_delta_rule_step needs a state");
    if (state) check_state(*state, want, "state");
    const bool gate = flags & KDA_FLAG_GATE;
    const Tensor &a0 = gate ? val(A_log) : val(std::nullopt), &b0 = gate ? val(dt_bias) : val(std::nullopt), &s0 = val(state);
    same_device(q, "q", "state", s0); same_device(q, "q", "A_log", a0); same_device(q, "q", "dt_bias", b0);
    refuse_tangents(std::array<const Tensor*, 8>{&q, &k, &v, &g, &beta, &s0, &a0, &b0});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(q.device());
    const auto dt = q.scalar_type(), gt = gate_type(g, beta);
    Tensor copies[8];
    const Tensor &qc = ready(q, dt, copies[0]), &kc = ready(k, dt, copies[1]), &vc = ready(v, dt, copies[2]),
                 &gc = ready(g, gt, copies[3]), &bc = ready(beta, gt, copies[4]), &a = ready(a0, at::kFloat, copies[5]),
                 &b = ready(b0, at::kFloat, copies[6]), &s_in = ready(s0, at::kFloat, copies[7]);
    Tensor s_out, s_back;  // s_back: a state to be updated that the kernel cannot write itself
    if (want_state) {
        const Tensor own = inplace ? (state->requires_grad() ? state->detach() : *state) : Tensor();
        if (inplace && at::has_internal_overlap(own) == at::MemOverlap::Yes)
            value_error("a state to be updated in place must not be an expanded tensor");
        if (inplace && s_in.data_ptr() == own.data_ptr()) {
            s_out = own;
        } else {
            s_out = fresh(want, at::kFloat, q);
            if (inplace) s_back = own;
        }
    }
    Tensor o = fresh(v.sizes(), dt, q);
    status_word(q.device().index());  // (a wait that gave up in the call that made the state surfaces here)
    if (N * T == 0) {
        if (s_out.defined() && !(s_in.defined() && s_out.data_ptr() == s_in.data_ptr())) {
            if (s_in.defined()) s_out.copy_(s_in);
            else s_out.zero_();
        }
    } else {
        check_rc(kda_gdr_recurrent_fwd(qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), gc.data_ptr(), bc.data_ptr(), ptr<float>(a), ptr<float>(b),
                                       ptr<float>(s_in), ptr<float>(s_out), o.data_ptr(), (int)N, (int)T, (int)H, (int)HV, (int)K, (int)V,
                                       code(dt), code(gt), (int)flags, (float)scale.value_or(1.0 / std::sqrt((double)K)), stream_of(q)),
                 "kda_gdr_recurrent_fwd");
        if (inplace && !s_back.defined()) written(s_out);
    }
    if (s_back.defined()) s_out = s_back.copy_(s_out);
    return {o, want_state ? OptTensor(s_out) : OptTensor()};
}

// ---- group norm --------------------------------------------------------------------------------------------------------
struct NormSpec {
    int64_t N = 0, S = 0, Ch = 0, G = 0;
    double eps = 1e-5;
    bool silu = false;
};
struct NormOut { Tensor y, mean, rstd; };

NormOut norm_fwd(const Tensor& x, const Tensor& w, const Tensor& b, const NormSpec& sp) {
    NormOut r;
    r.y = fresh_like(x);
    if (x.numel() == 0) return r;
    const int dt = code(x.scalar_type());
    size_t n = 0;
    check_rc(kda_group_norm_scratch_bytes(sp.N, sp.S, (int)sp.Ch, (int)sp.G, dt, &n, nullptr), "kda_group_norm_scratch_bytes");
    Tensor scratch;
    if (n) {
        scratch = bytes(n, x);
        r.mean = fresh({sp.N, sp.G}, at::kFloat, x);
        r.rstd = fresh({sp.N, sp.G}, at::kFloat, x);
    }
    check_rc(kda_group_norm_fwd(x.data_ptr(), ptr<float>(w), ptr<float>(b), r.y.data_ptr(), ptr<float>(r.mean), ptr<float>(r.rstd),
                                ptr<float>(scratch), sp.N, sp.S, (int)sp.Ch, (int)sp.G, (float)sp.eps, sp.silu, dt, stream_of(x)),
             "kda_group_norm_fwd");
    return r;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(AutogradContext* ctx, Tensor x, OptTensor weight, OptTensor bias, const NormSpec& sp) {
        const Tensor xc = ready(x, x.scalar_type());
        const Tensor w = weight ? ready(*weight, at::kFloat) : Tensor(), b = bias ? ready(*bias, at::kFloat) : Tensor();
        const NormOut r = norm_fwd(xc, w, b, sp);
        ctx->save_for_backward({xc, w, b, r.mean, r.rstd});
        ctx->saved_data["sizes"] = std::vector<int64_t>{sp.N, sp.S, sp.Ch, sp.G, sp.silu};
        ctx->saved_data["eps"] = sp.eps;
        return r.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &b = s[2];
        const std::vector<int64_t> z = ctx->saved_data["sizes"].toIntVector();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        c10::cuda::CUDAGuard guard(x.device());
        const Tensor dy = ready(grads[0], x.scalar_type()), dx = fresh_like(x);
        const bool params = w.defined() || b.defined();
        Tensor dw, db;
        if (params) {
            dw = fresh({z[2]}, at::kFloat, x);
            db = fresh({z[2]}, at::kFloat, x);
        }
        if (x.numel() == 0) {
            if (params) dw.zero_(), db.zero_();
        } else {
            const int dt = code(x.scalar_type());
            size_t n = 0;
            check_rc(kda_group_norm_scratch_bytes(z[0], z[1], (int)z[2], (int)z[3], dt, nullptr, &n), "kda_group_norm_scratch_bytes");
            const Tensor scratch = bytes(n, x);
            check_rc(kda_group_norm_bwd(x.data_ptr(), ptr<float>(w), ptr<float>(b), ptr<float>(s[3]), ptr<float>(s[4]), dy.data_ptr(),
                                        dx.data_ptr(), ptr<float>(dw), ptr<float>(db), ptr<float>(scratch), z[0], z[1], (int)z[2], (int)z[3],
                                        (float)ctx->saved_data["eps"].toDouble(), (int)z[4], dt, stream_of(x)),
                     "kda_group_norm_bwd");
        }
        return differentiable_once("group_norm", {dx, w.defined() ? dw : Tensor(), b.defined() ? db : Tensor(), Tensor()});
    }
};

Tensor group_norm(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps, bool silu) {
    on_cuda(x, "group_norm");
    if (x.dim() < 2) value_error("group_norm needs x of shape [N, ..., channels], got " + shape_of(x));
    if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kFloat)
        type_error(std::string("x must be float32 or bfloat16, got ") + c10::toString(x.scalar_type()));
    NormSpec sp;
    sp.N = x.size(0); sp.Ch = x.size(-1); sp.G = groups; sp.eps = eps; sp.silu = silu;
    if (groups < 1 || sp.Ch < 1 || sp.Ch % groups || sp.Ch > 1 << 30)
        value_error("the channels, at most 2^30, must divide into the groups, got " + std::to_string(sp.Ch) + " channels and " + std::to_string(groups) + " groups");
    if (!(eps >= 0.0)) value_error("eps must not be negative");
    int64_t positions = 1;
    for (int64_t i = 1; i + 1 < x.dim(); ++i) positions *= x.size(i);
    if (groups > KDA_GROUP_NORM_MAX_GROUPS && (positions > 1 || sp.Ch / groups > 1024))
        value_error("over several positions, or with more than 1024 channels a group, there may be at most " +
                    std::to_string(KDA_GROUP_NORM_MAX_GROUPS) + " groups, got " + std::to_string(groups));
    for (const OptTensor* t : {&weight, &bias})
        if (*t && ((*t)->dim() != 1 || (*t)->numel() != sp.Ch))
            value_error("weight and bias must have one entry per channel, got " + shape_of(**t));
    same_device(x, "x", "weight", val(weight)); same_device(x, "x", "bias", val(bias));
    sp.S = positions;
    const std::array<const Tensor*, 3> inputs = {&x, &val(weight), &val(bias)};
    refuse_tangents(inputs);
    bool grad = false;
    if (at::GradMode::is_enabled())
        for (const Tensor* t : inputs) grad = grad || (t->defined() && t->requires_grad());
    c10::cuda::CUDAGuard guard(x.device());
    if (grad) return GroupNorm::apply(x, weight, bias, sp);
    at::NoGradGuard no_grad;
    Tensor copies[3];
    return norm_fwd(ready(x, x.scalar_type(), copies[0]), ready(val(weight), at::kFloat, copies[1]), ready(val(bias), at::kFloat, copies[2]), sp).y;
}

}  // namespace

void bind_gdr(py::module_& m) {
    const py::call_guard<py::gil_scoped_release> unlocked;
    m.def("chunk_gdr", &chunk_gdr, unlocked);
    m.def("recurrent_gdr", &recurrent_gdr, unlocked);
    m.def("group_norm", &group_norm, unlocked);
}
