// The host side of a regular `attention()` call in one native call each way: allocations, the problem and tensor
// descriptors, the launches of fa_b200.h and the autograd node. The general code and its node stay in Python (ops.py), and so do all
// messages: a call that is not regular (another layout, device, shape or type than the kernels take as they are) is declined with
// None, and ops.py copies, asks or raises. Bound by per-call overhead: a forward of 8 heads of 200
// queries took 27 us of host time around 8 us of kernel through ctypes; a training step of 4 x 12
// heads x 1000 x 64 in documents 122 us with the node in Python, 92 with the one below, around some 70 of kernels.
#include <ATen/SavedTensorHooks.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>
#include <atomic>
#include <cmath>
#include "../../include/fa_b200.h"

namespace {

using at::Tensor;

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return FA_BF16;
        case at::kHalf: return FA_FP16;
        case at::kFloat: return FA_FP32;
        default: return -1;
    }
}

// what ops.maybe_contiguous leaves as it is
bool taken_as_is(const Tensor& t) {
    if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) return false;
    if (t.is_contiguous() && t.size(3) % 8 == 0) return true;
    if (t.stride(3) != 1) return false;
    for (int i = 0; i < 3; ++i)
        if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8 != 0)) return false;
    return true;
}

fa_tensor view(const Tensor& t) {
    return fa_tensor{t.data_ptr(), {t.stride(0), t.stride(1), t.stride(2), t.stride(3)}};
}

void check(int rc, const char* what) {
    TORCH_CHECK(rc == FA_OK, what, " failed with code ", rc, ": ", fa_error_string(rc));
}

bool plain_cuda(const Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && t.dim() == 4 && !t.is_conj() && !t.is_neg();
}

// Fills `p`, or says that the call is not a regular one on the current device. `prepared`: ops.maybe_contiguous has seen the
// tensors already, and what the library does not take of what it returned the library refuses. There k and v may have more
// batches, and v more keys, than q and k ask for: the first ones are read.
bool regular(const Tensor& q, const Tensor& k, const Tensor& v, bool prepared, bool causal, double sm_scale, int mode, int id_heads,
             fa_problem& p) {
    if (!plain_cuda(q) || !plain_cuda(k) || !plain_cuda(v)) return false;
    const int dt = dtype_of(q);
    if (dt < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
    if (k.device() != q.device() || v.device() != q.device() || q.get_device() != c10::cuda::current_device()) return false;
    const int64_t B = q.size(0), H = q.size(1), M = q.size(2), D = q.size(3), Hk = k.size(1), N = k.size(2);
    if (D != 16 && D != 32 && D != 64 && D != 128) return false;
    if (k.size(3) != D || v.size(1) != Hk || v.size(3) != D) return false;
    if (prepared ? k.size(0) < B || v.size(0) < B || v.size(2) < N : k.size(0) != B || v.size(0) != B || v.size(2) != N) return false;
    if (B < 1 || H < 1 || M < 1 || Hk < 1 || N < 1 || B > 65535 || H > 65535 || M > INT32_MAX || N > INT32_MAX) return false;
    if (H % Hk != 0 || (causal && N < M) || !(sm_scale > 0)) return false;
    if (!prepared && (!taken_as_is(q) || !taken_as_is(k) || !taken_as_is(v))) return false;
    p = fa_problem{int(B), int(H), int(Hk), int(M), int(N), int(D), dt, causal ? 1 : 0, mode, id_heads, float(sm_scale)};
    return true;
}

void* current_stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Would ops.maybe_contiguous return all three as they are? (Where this says no, ops.py goes by that.)
bool as_is(const Tensor& q, const Tensor& k, const Tensor& v) {
    return plain_cuda(q) && plain_cuda(k) && plain_cuda(v) && taken_as_is(q) && taken_as_is(k) && taken_as_is(v);
}

// How many heads the ids of a call have, 1 or H, where they are as the library takes them; 0: ops.py looks, converts or refuses.
int64_t id_heads(const Tensor& eq, const Tensor& ek, int64_t B, int64_t H, int64_t M, int64_t N) {
    for (const Tensor* t : {&eq, &ek})
        if (!t->is_cuda() || t->layout() != at::kStrided || t->dim() != 3 || t->is_neg() || t->size(0) != B || t->size(1) != H ||
            t->size(2) != (t == &eq ? M : N) || (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong))
            return 0;
    return H == 1 || (eq.stride(1) == 0 && ek.stride(1) == 0) ? 1 : H;
}

fa_ids id_view(const Tensor& t) {
    return fa_ids{t.const_data_ptr(), {t.stride(0), t.stride(1), t.stride(2)}, t.scalar_type() == at::kInt ? FA_ID_INT32 : FA_ID_INT64};
}

// The plan of a call: its memory and the launches that fill it. eq and ek, if any, are int32 or int64 tensors [B, H, M] and [B, H, N].
// scores: of attention_scored, else null (here and below).
Tensor build_plan(const fa_problem& p, const Tensor* eq, const Tensor* ek, const Tensor& status, const fa_scores* scores = nullptr, const fa_window* window = nullptr) {
    size_t bytes = 0;
    check(fa_plan_bytes(&p, &bytes), "fa_plan_bytes");
    Tensor plan = at::empty({int64_t(bytes / 4)}, status.options());
    const fa_ids q = eq ? id_view(*eq) : fa_ids{}, k = ek ? id_view(*ek) : fa_ids{};
    if (scores)
        check(fa_plan_build_windowed(&p, scores, window, eq ? &q : nullptr, ek ? &k : nullptr, plan.data_ptr(), bytes, status.data_ptr<int>(), current_stream(status)),
              "fa_plan_build_windowed");
    else
        check(fa_plan_build(&p, eq ? &q : nullptr, ek ? &k : nullptr, plan.data_ptr(), bytes, status.data_ptr<int>(), current_stream(status)),
              "fa_plan_build");
    return plan;
}

// ops.build_plan. `problem` is the address of an fa_problem; ops.py has checked the ids.
Tensor plan(uintptr_t problem, const std::optional<Tensor>& eq, const std::optional<Tensor>& ek, const Tensor& status) {
    py::gil_scoped_release free;
    return build_plan(*reinterpret_cast<const fa_problem*>(problem), eq ? &*eq : nullptr, ek ? &*ek : nullptr, status);
}

// Kernels launched by `attend` and its gradients (ops.LAUNCHES).
std::atomic<int64_t> n_launched{0};

struct Outputs {
    Tensor o, lse;
    int splits;
    Tensor rest;  // of a call of attention_scored that needs a gradient: what the rounding of o has left out
};

// The forward's allocations and launches for a problem that `regular` has filled.
Outputs launch_forward(const fa_problem& p, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& plan, int key_runs,
                       const Tensor& status, const std::optional<Tensor>& out, const fa_scores* scores = nullptr, bool backward = false, const fa_window* window = nullptr) {
    Outputs r;
    r.o = out ? *out : at::empty_like(q);
    if (!taken_as_is(r.o)) r.o = at::empty(q.sizes(), q.options());
    const auto f32 = q.options().dtype(at::kFloat);
    r.lse = at::empty({p.B, p.H, fa_padded_rows(p.M)}, f32);
    // (a number below 1 is the library's to refuse; a prefix may show keys that the window would hide)
    r.splits = key_runs != 0 ? key_runs : fa_fwd_splits_windowed(&p, scores && scores->prefix ? nullptr : window);
    Tensor work;
    size_t bytes = 0;
    if (r.splits > 1) {
        check(fa_fwd_workspace_bytes(&p, r.splits, &bytes), "fa_fwd_workspace_bytes");
        work = at::empty({int64_t(bytes / 4)}, f32);
    }
    const fa_tensor tq = view(q), tk = view(k), tv = view(v), to = view(r.o);
    void* const plan_ptr = plan.defined() ? plan.data_ptr() : nullptr;
    void* const work_ptr = work.defined() ? work.data_ptr() : nullptr;
    if (scores && backward && p.dtype != FA_FP32) r.rest = at::empty({p.B, p.H, p.M, p.D}, q.options());
    if (scores)
        check(fa_fwd_windowed(&p, scores, window, &tq, &tk, &tv, &to, r.rest.defined() && r.splits == 1 ? r.rest.data_ptr() : nullptr, r.lse.data_ptr<float>(), plan_ptr, r.splits, work_ptr, bytes, status.data_ptr<int>(),
                            current_stream(q)),
              "fa_fwd_windowed");
    else
        check(fa_fwd_split(&p, &tq, &tk, &tv, &to, r.lse.data_ptr<float>(), plan_ptr, r.splits, work_ptr, bytes, status.data_ptr<int>(), current_stream(q)),
              "fa_fwd_split");
    if (r.rest.defined() && r.splits > 1)
        check(fa_fwd_rest(&p, r.splits, work_ptr, bytes, r.rest.data_ptr(), status.data_ptr<int>(), current_stream(q)), "fa_fwd_rest");
    return r;
}

// dq, dk, dv. q, k, v, o, lse and the problem are those of a forward, d_o is like q.
std::array<Tensor, 3> launch_backward(const fa_problem& p, const Tensor& d_o, const Tensor& q, const Tensor& k, const Tensor& v,
                                      const Tensor& o, const Tensor& lse, const Tensor& plan, const Tensor& status,
                                      const fa_scores* scores = nullptr, const Tensor& rest = Tensor(), const fa_window* window = nullptr) {
    Tensor delta = at::empty_like(lse);
    Tensor dk = at::empty({p.B, p.Hk, p.N, p.D}, k.options()), dv = at::empty({p.B, p.Hk, p.N, p.D}, v.options());
    Tensor dq = at::empty(q.sizes(), q.options());
    const fa_tensor tq = view(q), tk = view(k), tv = view(v), to = view(o), tdo = view(d_o), tdq = view(dq), tdk = view(dk), tdv = view(dv);
    void* const plan_ptr = plan.defined() ? plan.data_ptr() : nullptr;
    Tensor work;
    size_t bytes = 0;
    if (window && window->keys > 0) check(fa_bwd_workspace_bytes(&p, window, &bytes), "fa_bwd_workspace_bytes");
    if (bytes > 0) {
        work = at::empty({int64_t(bytes / 4)}, q.options().dtype(at::kFloat));
        ++n_launched;
    }
    if (scores)
        check(fa_bwd_windowed(&p, scores, window, &tq, &tk, &tv, &to, rest.defined() ? rest.data_ptr() : nullptr, &tdo, lse.data_ptr<float>(), delta.data_ptr<float>(), &tdq, &tdk, &tdv, plan_ptr, work.defined() ? work.data_ptr() : nullptr, bytes,
                            status.data_ptr<int>(), current_stream(q)),
              "fa_bwd_windowed");
    else
        check(fa_bwd(&p, &tq, &tk, &tv, &to, &tdo, lse.data_ptr<float>(), delta.data_ptr<float>(), &tdq, &tdk, &tdv, plan_ptr, status.data_ptr<int>(),
                     current_stream(q)),
              "fa_bwd");
    return {std::move(dq), std::move(dk), std::move(dv)};
}

bool like_query(const Tensor& d_o, const Tensor& q) {
    return plain_cuda(d_o) && d_o.scalar_type() == q.scalar_type() && d_o.device() == q.device() && d_o.sizes() == q.sizes();
}

// (o, lse, scale, kernels launched), or None. Unprepared calls without a plan are taken only if it would gain nothing. `out`: a
// tensor like q for the result, given where q is of a subclass of torch.Tensor.
py::object forward(const Tensor& q, const Tensor& k, const Tensor& v, bool prepared, bool causal, std::optional<double> scale, int mode,
                   int id_heads, const std::optional<Tensor>& plan, bool backward, int key_runs, const Tensor& status,
                   const std::optional<Tensor>& out) {
    fa_problem p;
    const double sm_scale = scale ? *scale : 1.0 / std::sqrt(double(q.dim() == 4 ? q.size(3) : 1));
    if (!regular(q, k, v, prepared, causal, sm_scale, mode, id_heads, p)) return py::none();
    if (!plan && (mode != FA_MODE0_NOPE || (!prepared && !fa_plan_optional(&p, backward)))) return py::none();
    Outputs r;
    {
        py::gil_scoped_release free;
        r = launch_forward(p, q, k, v, plan ? *plan : Tensor(), key_runs, status, out);
    }
    return py::make_tuple(std::move(r.o), std::move(r.lse), sm_scale, r.splits > 1 ? 2 : 1);
}

// (dq, dk, dv), or None. q, k, v, o, lse and the numbers are those of a forward.
py::object backward(const Tensor& d_o, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
                    bool prepared, bool causal, double sm_scale, int mode, int id_heads, const std::optional<Tensor>& plan,
                    const Tensor& status) {
    fa_problem p;
    if (!regular(q, k, v, true, causal, sm_scale, mode, id_heads, p) || !like_query(d_o, q) || (!prepared && !taken_as_is(d_o)))
        return py::none();
    std::array<Tensor, 3> g;
    {
        py::gil_scoped_release free;
        g = launch_backward(p, d_o, q, k, v, o, lse, plan ? *plan : Tensor(), status);
    }
    return py::make_tuple(std::move(g[0]), std::move(g[1]), std::move(g[2]));
}

// What a regular call is, besides q, k and v.
struct Call {
    fa_problem p;
    double sm_scale;
    const Tensor *eq, *ek;  // null without ids
    const Tensor& status;
    bool needs_grad;
    int plan_kernels;
};

// The autograd node of a regular call: what ops.FlashAttention does, without Python on the way of the gradients, whose thread would
// have to be given the interpreter first. Saves the same tensors; the plan is the node's own.
struct FlashAttention : torch::autograd::Function<FlashAttention> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Call& c) {
        Tensor plan;
        Outputs r = launch(q, k, v, c, plan);
        torch::autograd::variable_list saved{q, k, v, r.o, r.lse};
        if (c.eq) {
            saved.push_back(*c.eq);
            saved.push_back(*c.ek);
        }
        ctx->save_for_backward(std::move(saved));
        ctx->saved_data["plan"] = plan;
        ctx->saved_data["status"] = c.status;
        ctx->saved_data["causal"] = int64_t(c.p.causal);
        ctx->saved_data["mode"] = int64_t(c.p.mode);
        ctx->saved_data["id_heads"] = int64_t(c.p.id_heads);
        ctx->saved_data["scale"] = c.sm_scale;
        return r.o;
    }

    // The plan, where the call needs one, and the forward.
    static Outputs launch(const Tensor& q, const Tensor& k, const Tensor& v, const Call& c, Tensor& plan) {
        py::gil_scoped_release free;
        if (c.eq || !fa_plan_optional(&c.p, c.needs_grad)) plan = build_plan(c.p, c.eq, c.ek, c.status);
        Outputs r = launch_forward(c.p, q, k, v, plan, 0, c.status, std::nullopt);
        n_launched += (plan.defined() ? c.plan_kernels : 0) + (r.splits > 1 ? 2 : 1);
        return r;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
        const c10::cuda::CUDAGuard device(q.device());
        auto& data = ctx->saved_data;
        fa_problem p;
        TORCH_CHECK(regular(q, k, v, true, data["causal"].toInt() != 0, data["scale"].toDouble(), int(data["mode"].toInt()),
                            int(data["id_heads"].toInt()), p),
                    "flash_b200: the saved q, k, v are not plain [bs, H, L, D] CUDA tensors of matching shapes");
        Tensor d_o = grads[0];
        if (d_o.scalar_type() != q.scalar_type()) d_o = d_o.to(q.scalar_type());
        d_o = d_o.resolve_neg();
        TORCH_CHECK(like_query(d_o, q), "flash_b200: the gradient is not a plain [bs, H, M, D] CUDA tensor");
        if (!taken_as_is(d_o)) d_o = d_o.contiguous();  // (ops.maybe_contiguous)
        auto g = launch_backward(p, d_o, q, k, v, saved[3], saved[4], data["plan"].toTensor(), data["status"].toTensor());
        n_launched += 3;
        return {std::move(g[0]), std::move(g[1]), std::move(g[2]), Tensor()};
    }
};

// The whole of a regular call, its gradients included; None: ops.py takes it another way. Saved-tensor hooks count what is saved and by whom, so
// that their calls take ops.FlashAttention.
py::object attend(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, std::optional<double> scale, const std::optional<Tensor>& eq,
                  const std::optional<Tensor>& ek, const py::int_& score_mode, const Tensor& status) {
    fa_problem p;
    int beyond = 0;  // (a number of any size: what no mode has is for ops.py to refuse)
    const long mode = PyLong_AsLongAndOverflow(score_mode.ptr(), &beyond);
    const double sm_scale = scale ? *scale : 1.0 / std::sqrt(double(q.dim() == 4 ? q.size(3) : 1));
    if (beyond != 0 || eq.has_value() != ek.has_value() || mode != (eq ? FA_MODE1_DOC : FA_MODE0_NOPE)) return py::none();
    if (!regular(q, k, v, false, causal, sm_scale, int(mode), 1, p)) return py::none();
    if (eq) {
        if (eq->device() != q.device() || ek->device() != q.device()) return py::none();
        p.id_heads = int(id_heads(*eq, *ek, p.B, p.H, p.M, p.N));
        if (p.id_heads == 0) return py::none();
    }
    const bool needs_grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    if (needs_grad && at::SavedTensorDefaultHooks::get_hooks()) return py::none();
    const int plan_kernels = !eq || (p.M + 127) / 128 + (p.N + 127) / 128 <= FA_PLAN_ONE_KERNEL_BLOCKS ? 1 : 3;
    const Call call{p, sm_scale, eq ? &*eq : nullptr, ek ? &*ek : nullptr, status, needs_grad, plan_kernels};
    if (needs_grad) return py::cast(FlashAttention::apply(q, k, v, call));
    Tensor plan;
    return py::cast(FlashAttention::launch(q, k, v, call, plan).o);
}

// What attention_scored changes: as scored.py has checked it, or None.
bool scores_of(double softcap, const std::optional<Tensor>& slopes, const std::optional<Tensor>& prefix, const Tensor& q, int64_t H, int64_t B, fa_scores& s) {
    if (!(softcap == 0.0 || (softcap >= 1e-6 && softcap <= 1e6))) return false;
    auto vector = [&](const Tensor& t, at::ScalarType type, int64_t n) {
        return t.is_cuda() && t.layout() == at::kStrided && t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.is_contiguous() && !t.is_neg() &&
               t.device() == q.device() && !(at::GradMode::is_enabled() && t.requires_grad());
    };
    if ((slopes && !vector(*slopes, at::kFloat, H)) || (prefix && !vector(*prefix, at::kInt, B))) return false;
    s = fa_scores{float(softcap), slopes ? slopes->const_data_ptr<float>() : nullptr, prefix ? prefix->const_data_ptr<int>() : nullptr};
    return true;
}

// Gradients that a graph is to be made of: an error waits between them and q, k and v, where there would be nothing (scored._once).
void once(std::array<Tensor, 3>& g, const Tensor& q, const Tensor& k, const Tensor& v) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::variable_list in{q, k, v};
    for (int i = 0; i < 3; ++i) in.insert(in.begin() + i, g[i].detach().set_requires_grad(true));
    torch::autograd::DelayedError error("flash_b200: attention_scored has gradients once; these cannot be differentiated", 6);
    auto out = error.apply(std::move(in));
    for (int i = 0; i < 3; ++i) g[i] = std::move(out[i]);
}

// The autograd node of a regular call of attention_scored, as scored.ScoredAttention.
struct ScoredAttention : torch::autograd::Function<ScoredAttention> {
    struct Scores {
        fa_scores s;
        fa_window window;
        const std::optional<Tensor>&slopes, &prefix;
    };

    static Outputs launch(const Tensor& q, const Tensor& k, const Tensor& v, const Call& c, const fa_scores& s, const fa_window& w, Tensor& plan) {
        py::gil_scoped_release free;
        if (c.eq || !fa_plan_optional(&c.p, c.needs_grad)) plan = build_plan(c.p, c.eq, c.ek, c.status, &s, &w);
        Outputs r = launch_forward(c.p, q, k, v, plan, 0, c.status, std::nullopt, &s, c.needs_grad, &w);
        n_launched += (plan.defined() ? c.plan_kernels : 0) + (r.splits > 1 ? 2 + r.rest.defined() : 1);
        return r;
    }

    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Call& c, const Scores& sc) {
        Tensor plan;
        Outputs r = launch(q, k, v, c, sc.s, sc.window, plan);
        torch::autograd::variable_list saved{q, k, v, r.o, r.lse};
        if (sc.slopes) saved.push_back(*sc.slopes);
        if (sc.prefix) saved.push_back(*sc.prefix);
        if (r.rest.defined()) saved.push_back(r.rest);
        ctx->save_for_backward(std::move(saved));
        auto& data = ctx->saved_data;
        data["plan"] = plan;
        data["status"] = c.status;
        data["causal"] = int64_t(c.p.causal);
        data["mode"] = int64_t(c.p.mode);
        data["id_heads"] = int64_t(c.p.id_heads);
        data["scale"] = c.sm_scale;
        data["softcap"] = double(sc.s.softcap);
        data["window"] = int64_t(sc.window.keys);
        data["sinks"] = int64_t(sc.window.sinks);
        data["slopes"] = sc.slopes.has_value();
        data["prefix"] = sc.prefix.has_value();
        return r.o;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
        const c10::cuda::CUDAGuard device(q.device());
        auto& data = ctx->saved_data;
        fa_problem p;
        TORCH_CHECK(regular(q, k, v, true, data["causal"].toInt() != 0, data["scale"].toDouble(), int(data["mode"].toInt()),
                            int(data["id_heads"].toInt()), p),
                    "flash_b200: the saved q, k, v are not plain [bs, H, L, D] CUDA tensors of matching shapes");
        size_t at = 5;
        fa_scores s{float(data["softcap"].toDouble()), nullptr, nullptr};
        const fa_window w{int(data["window"].toInt()), int(data["sinks"].toInt())};
        if (data["slopes"].toBool()) s.slopes = saved[at++].const_data_ptr<float>();
        if (data["prefix"].toBool()) s.prefix = saved[at++].const_data_ptr<int>();
        const Tensor rest = saved.size() > at ? saved[at] : Tensor();
        Tensor d_o = grads[0];
        if (d_o.scalar_type() != q.scalar_type()) d_o = d_o.to(q.scalar_type());
        d_o = d_o.resolve_neg();
        TORCH_CHECK(like_query(d_o, q), "flash_b200: the gradient is not a plain [bs, H, M, D] CUDA tensor");
        if (!taken_as_is(d_o)) d_o = d_o.contiguous();  // (ops.maybe_contiguous)
        auto g = launch_backward(p, d_o, q, k, v, saved[3], saved[4], data["plan"].toTensor(), data["status"].toTensor(), &s, rest, &w);
        n_launched += 3;
        once(g, q, k, v);
        return {std::move(g[0]), std::move(g[1]), std::move(g[2]), Tensor(), Tensor()};
    }
};

// The whole of a regular call of attention_scored, its gradients included; None: scored.py takes it another way.
py::object attend_scored(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, std::optional<double> scale, const std::optional<Tensor>& eq,
                         const std::optional<Tensor>& ek, int64_t mode, double softcap, const std::optional<Tensor>& slopes,
                         const std::optional<Tensor>& prefix, int64_t window, int64_t sinks, const Tensor& status) {
    fa_problem p;
    const double sm_scale = scale ? *scale : 1.0 / std::sqrt(double(q.dim() == 4 ? q.size(3) : 1));
    if (eq.has_value() != ek.has_value() || mode != (eq ? FA_MODE1_DOC : FA_MODE0_NOPE) || ((prefix || window) && !causal)) return py::none();
    if (!regular(q, k, v, false, causal, sm_scale, int(mode), 1, p)) return py::none();
    if (eq) {
        if (eq->device() != q.device() || ek->device() != q.device()) return py::none();
        p.id_heads = int(id_heads(*eq, *ek, p.B, p.H, p.M, p.N));
        if (p.id_heads == 0) return py::none();
    }
    fa_scores s;
    if (!scores_of(softcap, slopes, prefix, q, p.H, p.B, s)) return py::none();
    const fa_window w{int(window), int(sinks)};  // (as scored.py has checked it)
    const bool needs_grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    if (needs_grad && at::SavedTensorDefaultHooks::get_hooks()) return py::none();
    const int plan_kernels = !eq || (p.M + 127) / 128 + (p.N + 127) / 128 <= FA_PLAN_ONE_KERNEL_BLOCKS ? 1 : 3;
    const Call call{p, sm_scale, eq ? &*eq : nullptr, ek ? &*ek : nullptr, status, needs_grad, plan_kernels};
    if (needs_grad) return py::cast(ScoredAttention::apply(q, k, v, call, ScoredAttention::Scores{s, w, slopes, prefix}));
    Tensor plan;
    return py::cast(ScoredAttention::launch(q, k, v, call, s, w, plan).o);
}

// ---- paged cache (paged.py). A call that is not a regular one on the current device is declined, and paged.py copies, raises or does nothing.
bool rows_as_is(const Tensor& t, int dim, int multiple = 8) {
    if (!t.is_cuda() || t.layout() != at::kStrided || t.dim() != dim || t.is_neg() || t.stride(dim - 1) != 1 || t.numel() == 0 ||
        reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0)
        return false;
    for (int i = 0; i < dim - 1; ++i)
        if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % multiple != 0)) return false;
    return !(at::GradMode::is_enabled() && t.requires_grad());
}

bool cache_of(const Tensor& rows, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens, const std::optional<Tensor>& starts,
              const std::optional<Tensor>& k_scales, const std::optional<Tensor>& v_scales, fa_paged_cache& c, fa_paged_more& more) {
    if (k_scales.has_value() != v_scales.has_value()) return false;
    const int multiple = k_scales ? 16 : 8;
    if (!rows_as_is(rows, 3) || !rows_as_is(k_pages, 4, multiple) || !rows_as_is(v_pages, 4, multiple) || rows.get_device() != c10::cuda::current_device()) return false;
    const int dt = dtype_of(rows);
    const auto cached = k_scales ? at::kFloat8_e4m3fn : rows.scalar_type();
    if ((dt != FA_BF16 && dt != FA_FP16) || k_pages.scalar_type() != cached || v_pages.scalar_type() != cached) return false;
    auto ints = [&](const Tensor& t, int dim) {
        return t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == at::kInt && t.dim() == dim && t.device() == rows.device() && !t.is_neg();
    };
    if (k_pages.device() != rows.device() || v_pages.device() != rows.device() || v_pages.sizes() != k_pages.sizes()) return false;
    if (!ints(table, 2) || !ints(lens, 1) || (starts && !ints(*starts, 1))) return false;
    const int64_t B = table.size(0), T = rows.size(0), page = k_pages.size(1), D = rows.size(2);
    if (B < 1 || B > 65535 || table.size(1) < 1 || table.stride(1) != 1 || (B > 1 && table.stride(0) < table.size(1)) || lens.size(0) != B ||
        !lens.is_contiguous() || T > INT32_MAX || k_pages.size(0) > INT32_MAX || page > (1 << 22) || k_pages.size(2) > 1024)
        return false;
    if (starts ? starts->size(0) != B + 1 || !starts->is_contiguous() : T != B) return false;
    if (page < 8 || (page & (page - 1)) != 0 || table.size(1) * page > (1 << 22) || k_pages.size(3) != D || (D != 16 && D != 32 && D != 64 && D != 128)) return false;
    c = fa_paged_cache{int(B), int(k_pages.size(2)), int(D), dt, int(k_pages.size(0)), int(page), int(table.size(1)), table.const_data_ptr<int>(), table.stride(0),
                       lens.const_data_ptr<int>(), k_pages.data_ptr(), v_pages.data_ptr(), {k_pages.stride(0), k_pages.stride(1), k_pages.stride(2)},
                       {v_pages.stride(0), v_pages.stride(1), v_pages.stride(2)}};
    if (k_scales) {
        for (const Tensor* t : {&*k_scales, &*v_scales})
            if (!rows_as_is(*t, 3, 16) || t->scalar_type() != at::kFloat8_e8m0fnu || t->device() != rows.device() || t->size(0) != k_pages.size(0) ||
                t->size(1) != k_pages.size(2) || t->size(2) != page)
                return false;
        if (page < 16) return false;
        more.k_scales = static_cast<uint8_t*>(k_scales->data_ptr());
        more.v_scales = static_cast<uint8_t*>(v_scales->data_ptr());
        for (int i = 0; i < 2; ++i) {
            more.k_scale_stride[i] = k_scales->stride(i);
            more.v_scale_stride[i] = v_scales->stride(i);
        }
    }
    return true;
}

// n contiguous int32 numbers on the device of `like`
bool int_vector(const Tensor& t, const Tensor& like, int64_t n) {
    return t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous() && !t.is_neg() &&
           t.device() == like.device();
}

fa_rows rows_view(const Tensor& t) { return fa_rows{t.data_ptr(), {t.stride(0), t.stride(1)}}; }

void bump(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool paged_append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                  const std::optional<Tensor>& starts, const std::optional<Tensor>& k_scales, const std::optional<Tensor>& v_scales, const Tensor& status) {
    fa_paged_cache c;
    fa_paged_more more{};
    if (!cache_of(k, k_pages, v_pages, table, lens, starts, k_scales, v_scales, c, more) || !rows_as_is(v, 3) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() ||
        v.device() != k.device() || k.size(1) != c.Hk)
        return false;
    {
        py::gil_scoped_release free;
        const fa_rows rk = rows_view(k), rv = rows_view(v);
        check(fa_paged_append_more(&c, &more, int(k.size(0)), starts ? starts->const_data_ptr<int>() : nullptr, &rk, &rv, status.data_ptr<int>(), current_stream(k)),
              "fa_paged_append_more");
        ++n_launched;
    }
    bump(k_pages);
    bump(v_pages);
    if (k_scales) {
        bump(*k_scales);
        bump(*v_scales);
    }
    return true;
}

py::object paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                           const std::optional<Tensor>& starts, std::optional<double> scale, double softcap, const std::optional<Tensor>& slopes,
                           const std::optional<Tensor>& prefix, const std::optional<Tensor>& out, int64_t window, int64_t sinks, const std::optional<Tensor>& parents,
                           const std::optional<Tensor>& k_scales, const std::optional<Tensor>& v_scales, const Tensor& status) {
    fa_paged_cache c;
    fa_scores s;
    fa_paged_more more{};
    if (!cache_of(q, k_pages, v_pages, table, lens, starts, k_scales, v_scales, c, more)) return py::none();
    const int64_t H = q.size(1);
    const double sm_scale = scale ? *scale : 1.0 / std::sqrt(double(c.D));
    if (H % c.Hk != 0 || H / c.Hk > 128 || !(sm_scale > 0) || !std::isfinite(sm_scale) || !scores_of(softcap, slopes, prefix, q, H, c.B, s)) return py::none();
    if (parents && !int_vector(*parents, q, q.size(0))) return py::none();
    more.window = {int(window), int(sinks)};  // (as paged.py has checked them)
    more.parents = parents ? parents->const_data_ptr<int>() : nullptr;
    if (out) {
        if (!rows_as_is(*out, 3) || out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type() || out->device() != q.device() || out->requires_grad())
            return py::none();
        for (const Tensor* t : {&q, &k_pages, &v_pages, k_scales ? &*k_scales : &q, v_scales ? &*v_scales : &q})
            if (t->storage().data() == out->storage().data()) return py::none();  // paged.py looks closer
    }
    Tensor o;
    {
        py::gil_scoped_release free;
        o = out ? *out : at::empty(q.sizes(), q.options().requires_grad(false));
        size_t bytes = 0;
        check(fa_paged_workspace_bytes(&c, &bytes), "fa_paged_workspace_bytes");
        Tensor work = at::empty({int64_t(bytes)}, q.options().dtype(at::kByte));
        const fa_rows rq = rows_view(q), ro = rows_view(o);
        check(fa_paged_fwd_more(&c, &more, int(q.size(0)), int(H), starts ? starts->const_data_ptr<int>() : nullptr, float(sm_scale), &s, &rq, &ro, out ? 0 : 1, work.data_ptr(),
                           bytes, status.data_ptr<int>(), current_stream(q)),
              "fa_paged_fwd_more");
        n_launched += 2;
    }
    if (out) bump(*out);
    return py::cast(o);
}

int64_t launched() { return n_launched; }

// What `grad_fn` of a regular call shows to Python: what it shows of ops.FlashAttention (the reference's contract, flash_triton.py:558-562).
using Node = torch::autograd::CppNode<FlashAttention>;

Node& node_of(PyObject* self) { return static_cast<Node&>(*reinterpret_cast<torch::autograd::THPCppFunction*>(self)->cdata); }

// The engine's thread gives the saved tensors up, behind the node's lock, without the interpreter: so they are asked for.
torch::autograd::variable_list saved_tensors(Node& n) {
    struct Open : torch::autograd::Node {
        static std::mutex& lock_of(torch::autograd::Node& n) { return n.*(&Open::mutex_); }
    };
    py::gil_scoped_release free;
    const std::lock_guard<std::mutex> lock(Open::lock_of(n));
    return n.ctx_.get_saved_variables();
}

using Shown = py::object (*)(Node&);

PyObject* show(PyObject* self, void* get) {
    HANDLE_TH_ERRORS
    return reinterpret_cast<Shown>(get)(node_of(self)).release().ptr();
    END_HANDLE_TH_ERRORS
}

PyGetSetDef property(const char* name, Shown get) { return {name, show, nullptr, nullptr, reinterpret_cast<void*>(get)}; }

PyObject* node_name(PyObject*, PyObject*) { return PyUnicode_FromString("FlashAttentionBackward"); }

void register_node() {
    using namespace torch::autograd;
    static PyGetSetDef properties[] = {
        {"next_functions", THPCppFunction_next_functions, nullptr, nullptr, nullptr},
        {"requires_grad", THPCppFunction_requires_grad, nullptr, nullptr, nullptr},
        {"metadata", THPCppFunction_metadata, nullptr, nullptr, nullptr},
        {"_input_metadata", THPCppFunction_input_metadata, nullptr, nullptr, nullptr},
        property("saved_tensors", [](Node& n) -> py::object { return py::tuple(py::cast(saved_tensors(n))); }),
        property("needs_input_grad", [](Node& n) -> py::object {
            py::tuple t(8);  // of attention()'s arguments
            for (size_t i = 0; i < 8; ++i) t[i] = py::bool_(i < 3 && n.should_compute_output(i));
            return t;
        }),
        property("sm_scale", [](Node& n) -> py::object { return py::cast(n.ctx_.saved_data["scale"].toDouble()); }),
        property("causal", [](Node& n) -> py::object { return py::cast(n.ctx_.saved_data["causal"].toInt() != 0); }),
        property("score_func_info", [](Node& n) -> py::object { return py::make_tuple(n.ctx_.saved_data["mode"].toInt()); }),
        property("id_heads", [](Node& n) -> py::object { return py::cast(n.ctx_.saved_data["id_heads"].toInt()); }),
        property("plan", [](Node& n) -> py::object { return py::cast(n.ctx_.saved_data["plan"].toTensor()); }),  // (None where there is none)
        {nullptr, nullptr, nullptr, nullptr, nullptr},
    };
    static PyMethodDef methods[] = {
        {"name", node_name, METH_NOARGS, nullptr},
        {"register_hook", THPCppFunction_register_hook, METH_O, nullptr},
        {"register_prehook", THPCppFunction_register_prehook, METH_O, nullptr},
        {"_register_hook_dict", THPCppFunction_register_hook_dict, METH_O, nullptr},
        {"_sequence_nr", THPCppFunction_sequence_nr, METH_NOARGS, nullptr},
        {nullptr, nullptr, 0, nullptr},
    };
    static PyTypeObject type{PyVarObject_HEAD_INIT(nullptr, 0)};
    registerCppFunction(typeid(Node), _initFunctionPyTypeObject(type, "flash_b200._host.FlashAttentionNode", properties, methods));
}

}  // namespace

PYBIND11_MODULE(_host, m) {
    m.def("as_is", &as_is);
    m.def("id_heads", &id_heads);
    m.def("plan", &plan);
    m.def("forward", &forward);
    m.def("backward", &backward);
    m.def("attend", &attend);
    m.def("attend_scored", &attend_scored);
    m.def("paged_append", &paged_append);
    m.def("paged_attention", &paged_attention);
    m.def("launched", &launched);
    register_node();
}
