// The operators of sthip_ops.hip for torch: argument checks, memory, streams and autograd nodes around the C ABI of
// include/strassen_hip.h (module _sthip_torch, wrapped by strassen_hip/block.py).  Host code only; all arithmetic is behind the
// C ABI.  In C++ because a small layer's training step is bound by what the host does between launches: the same
// nodes written in Python took 110 to 130 us a step, most of it interpreter time in autograd's own thread.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <unordered_set>

#include "../../include/strassen_hip.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct SthipFailure : std::exception {
    int code;
    std::string message;
    SthipFailure(int c, const char* m) : code(c), message(m) {}
    const char* what() const noexcept override { return message.c_str(); }
};
void check(int rc) {
    if (rc) throw SthipFailure(rc, sthip_last_error());
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return STHIP_F32;
        case at::kHalf: return STHIP_F16;
        case at::kBFloat16: return STHIP_BF16;
        default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t, "; use float32, float16 or bfloat16");
    }
    return -1;
}
void require_gpu(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "strassen_hip runs on MI355X tensors only (got a tensor on ", t.device(), "); there is no CPU implementation in this library");
}
// What torch would follow through its own operations and cannot follow into these: a tangent (forward-mode derivative), a transform's
// wrapped tensor or another one whose operations are dispatched elsewhere (its memory, if any, is not its value), a program that
// is being recorded or run on tensors without memory.  All would get a result as if it were a constant, or none.
template <class Tensors> void refuse_transforms(const Tensors& tensors) {
    auto mode = [](c10::impl::TorchDispatchModeKey k) { return c10::impl::TorchDispatchModeTLS::any_modes_set() && c10::impl::TorchDispatchModeTLS::get_mode(k); };
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !mode(c10::impl::TorchDispatchModeKey::PROXY) && !mode(c10::impl::TorchDispatchModeKey::FAKE),
                "the operators of strassen_hip cannot be traced");
    const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Maybe& t : tensors) {
        if (!t || !t->defined()) continue;
        TORCH_CHECK(!t->key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Python})) &&
                    t->layout() == at::kStrided, "the operators of strassen_hip take plain tensors: no torch.func transforms, no subclass with operations of its own, no sparse ones");
        TORCH_CHECK(!tangents || !t->_fw_grad(0).defined(), "the operators of strassen_hip have no forward-mode derivatives");
    }
}
void same_device(const Tensor& first, const Maybe& t) {
    if (t) TORCH_CHECK(t->device() == first.device(), "tensors on different devices: ", first.device(), " and ", t->device());
}
bool wants_grad(const Maybe& t) { return t && t->requires_grad(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const Maybe& t) { return t ? ptr(*t) : nullptr; }
Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }

// `device` current for the calls made while this lives, on its current stream.
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// A 2-D tensor the kernels can read: unit stride along columns, rows that do not overlap, no pending negation.
Tensor rows_of(const Tensor& t) {
    if (t.is_neg()) return rows_of(t.resolve_neg());
    Tensor r = t.dim() == 2 ? t : t.reshape({t.dim() < 2 ? 1 : c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), t.size(-1)});
    if (r.is_contiguous()) return r;
    if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) return r.contiguous();
    return r;
}
Maybe contiguous(const Maybe& t) { return t && (t->is_neg() || !t->is_contiguous()) ? Maybe(t->resolve_neg().contiguous()) : t; }
Tensor with_last(const Tensor& y, const Tensor& x, int64_t cols) {
    if (x.dim() == 2) return y;
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.back() = cols;
    return y.view(s);
}

// What a node saved, as the backward pass finds it: a hook on saved tensors may give back other strides, or another tensor.
Tensor restored(const Tensor& t, const char* what, at::IntArrayRef sizes, at::ScalarType type, const Tensor& grad) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == grad.device(), "the saved ", what, " came back as ", t.toString(), " of ",
                t.sizes(), " on ", t.device(), ", expected ", type, " of ", sizes, " on ", grad.device());
    refuse_transforms(variable_list{t});
    return t.resolve_neg();
}

// What a backward pass returns, where it was asked for a graph of itself: tensors that refuse to be differentiated again.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list fake;
    for (auto& g : grads) fake.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    auto node = std::make_shared<torch::autograd::DelayedError>("the operators of strassen_hip cannot be differentiated twice", (int64_t)fake.size());
    return (*node)(std::move(fake));
}

// A leaf that a living eager graph uses keeps its accumulation on that graph's stream, and what was computed eagerly goes back on its
// own.  Where that is the default stream, a backward pass under capture would make it wait for the captured one, which ends the
// process: refused before, for leaves and for everything that the operands were computed from.
void refuse_eager_leaves(std::initializer_list<Maybe> tensors) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> kept;   // accumulators that only a weak reference holds
    std::vector<torch::autograd::Node*> open;
    std::unordered_set<torch::autograd::Node*> seen;
    for (const Maybe& t : tensors) {
        if (!t || !t->defined() || !t->requires_grad()) continue;
        kept.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
        open.push_back(kept.back().get());
    }
    while (!open.empty()) {
        torch::autograd::Node* node = open.back();
        open.pop_back();
        if (!node || !seen.insert(node).second) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream || stream->id() != 0, "a graph is being captured while an eager graph of the same leaf is alive on the default stream, or an operand was computed there: "
                    "let go of its results before, or warm up on another stream, or capture under no_grad");
        for (const auto& edge : node->next_edges()) open.push_back(edge.function.get());
    }
}

// ------------------------------------------------------------------------------------------------ linear_act
Tensor linear_forward(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act, Tensor* pre) {
    const On on(x);
    const int64_t rows = x.size(0), in = x.size(1), out = w.size(0);
    const int dt = dtype_code(x.scalar_type());
    Tensor y = at::empty({rows, out}, x.options());
    if (pre) *pre = at::empty({rows, out}, x.options());
    const size_t bytes = sthip_linear_act_workspace_bytes(rows, in, out, dt);
    const Tensor ws = workspace(bytes, x);
    check(sthip_linear_act_forward(x.data_ptr(), w.data_ptr(), ptr(b), ptr(r), y.data_ptr(), pre ? pre->data_ptr() : nullptr, rows, in, out,
                                   x.stride(0), w.stride(0), r ? r->stride(0) : 0, out, dt, (int)act, ptr(ws), bytes, on.stream));
    return y;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act, bool keep) {
        Tensor pre;
        Tensor y = linear_forward(x, w, b, r, act, keep ? &pre : nullptr);
        ctx->save_for_backward({x, w, pre});
        ctx->saved_data["act"] = act;
        ctx->saved_data["in"] = x.size(1);
        ctx->saved_data["given"] = (int64_t)((b ? 1 : 0) | (r ? 2 : 0));
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_transforms(grads);
        const variable_list saved = ctx->get_saved_variables();
        const int64_t act = ctx->saved_data["act"].toInt(), rows = grads[0].size(0), in = ctx->saved_data["in"].toInt(), out = grads[0].size(1);
        // needs_input_grad counts the tensors that were given
        const int64_t given = ctx->saved_data["given"].toInt();
        const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
        const bool nb = (given & 1) && ctx->needs_input_grad(2), nr = (given & 2) && ctx->needs_input_grad(given & 1 ? 3 : 2);
        Tensor dx, dw, db;
        if (nx || nw || nb) {
            const at::NoGradGuard no_grad;
            const On on(grads[0]);
            const auto type = grads[0].scalar_type();
            const Tensor x = rows_of(restored(saved[0], "input", {rows, in}, type, grads[0])), w = rows_of(restored(saved[1], "weight", {out, in}, type, grads[0]));
            const Tensor pre = act ? restored(saved[2], "pre-activation", {rows, out}, type, grads[0]).contiguous() : Tensor();
            const Tensor dy = rows_of(grads[0]);
            const int dt = dtype_code(type);
            if (nx) dx = at::empty({rows, in}, x.options());
            if (nw) dw = at::empty({out, in}, x.options());
            if (nb) db = at::empty({out}, x.options());
            const size_t bytes = sthip_linear_act_backward_workspace_bytes(rows, in, out, dt, (int)act);
            const Tensor ws = workspace(bytes, x);
            check(sthip_linear_act_backward(dy.data_ptr(), x.data_ptr(), w.data_ptr(), ptr(pre), ptr(dx), ptr(dw), ptr(db), rows, in, out,
                                            dy.stride(0), x.stride(0), w.stride(0), dt, (int)act, ptr(ws), bytes, on.stream));
        }
        return once({dx, dw, db, nr ? grads[0] : Tensor(), Tensor(), Tensor()});
    }
};

Tensor linear_act(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act) {
    refuse_transforms(std::initializer_list<Maybe>{x, w, b, r});
    require_gpu(x);
    same_device(x, w), same_device(x, b), same_device(x, r);
    TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), "shape mismatch: ", x.sizes(), " @ ", w.sizes(), "^T");
    dtype_code(x.scalar_type());
    const int64_t out = w.size(0);
    auto typed = [&](const char* what, const Maybe& t) { if (t) TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type(), what, " has dtype ", t->scalar_type(), ", the input ", x.scalar_type()); };
    typed("weight", w), typed("bias", b), typed("residual", r);
    if (b) TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == out, "bias has shape ", b->sizes(), ", expected [", out, "]");
    if (r) TORCH_CHECK_VALUE(r->dim() == x.dim() && r->size(-1) == out && r->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                             "residual has shape ", r->sizes(), ", expected that of the input with ", out, " columns");
    const Tensor x2 = rows_of(x), w2 = rows_of(w);
    const Maybe b2 = contiguous(b), r2 = r ? Maybe(rows_of(*r)) : r;
    const bool inner = x2.requires_grad() || w2.requires_grad() || wants_grad(b2);
    Tensor y;
    if (at::GradMode::is_enabled() && (inner || wants_grad(r2))) {
        refuse_eager_leaves({x, w, b, r});
        y = LinearAct::apply(x2, w2, b2, r2, act, inner && act != STHIP_ACT_NONE);
    }
    else y = linear_forward(x2, w2, b2, r2, act, nullptr);
    return with_last(y, x, out);
}

// ------------------------------------------------------------------------------------------------ layer_norm
int param_code(const Tensor& x, const Maybe& w, const Maybe& b) { return dtype_code(w ? w->scalar_type() : b ? b->scalar_type() : x.scalar_type()); }

Tensor norm_forward(const Tensor& x, const Maybe& w, const Maybe& b, double eps, Tensor* stats) {
    const On on(x);
    const int64_t rows = x.size(0), cols = x.size(1);
    Tensor y = at::empty({rows, cols}, x.options());
    if (stats) *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    float* mean = stats && rows > 0 ? stats->data_ptr<float>() : nullptr;
    check(sthip_layer_norm_forward(x.data_ptr(), ptr(w), ptr(b), y.data_ptr(), mean, mean ? mean + rows : nullptr, rows, cols, x.stride(0), cols,
                                   dtype_code(x.scalar_type()), param_code(x, w, b), eps, on.stream));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, double eps) {
        Tensor stats;
        Tensor y = norm_forward(x, w, b, eps, &stats);
        ctx->save_for_backward({x, w ? *w : Tensor(), stats});
        ctx->saved_data["given"] = (int64_t)((w ? 1 : 0) | (b ? 2 : 0));
        ctx->saved_data["params"] = (int64_t)(w ? w->scalar_type() : b ? b->scalar_type() : x.scalar_type());
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_transforms(grads);
        const variable_list saved = ctx->get_saved_variables();
        const auto params = (at::ScalarType)ctx->saved_data["params"].toInt();
        const int64_t rows = grads[0].size(0), cols = grads[0].size(1);
        const int64_t given = ctx->saved_data["given"].toInt();
        const bool nx = ctx->needs_input_grad(0), nw = (given & 1) && ctx->needs_input_grad(1);
        const bool nb = (given & 2) && ctx->needs_input_grad(given & 1 ? 2 : 1);
        Tensor dx, dw, db;
        {
            const at::NoGradGuard no_grad;
            const On on(grads[0]);
            const Tensor x = rows_of(restored(saved[0], "input", {rows, cols}, grads[0].scalar_type(), grads[0]));
            const Tensor w = given & 1 ? restored(saved[1], "weight", {cols}, params, grads[0]).contiguous() : Tensor();
            const Tensor stats = restored(saved[2], "statistics", {2, rows}, at::kFloat, grads[0]).contiguous();
            const Tensor dy = rows_of(grads[0]);
            if (nx) dx = at::empty({rows, cols}, x.options());
            if (nw) dw = at::empty({cols}, x.options().dtype(params));
            if (nb) db = at::empty({cols}, x.options().dtype(params));
            const size_t bytes = nw || nb ? sthip_layer_norm_backward_workspace_bytes(rows, cols) : 0;
            const Tensor ws = workspace(bytes, x);
            const float* mean = rows > 0 ? stats.data_ptr<float>() : nullptr;
            check(sthip_layer_norm_backward(dy.data_ptr(), x.data_ptr(), ptr(w), mean, mean ? mean + rows : nullptr, ptr(dx), ptr(dw), ptr(db), rows, cols,
                                            dy.stride(0), x.stride(0), cols, dtype_code(x.scalar_type()), dtype_code(params), ptr(ws), bytes, on.stream));
        }
        return once({dx, dw, db, Tensor()});
    }
};

Tensor layer_norm(const Tensor& x, const Maybe& w, const Maybe& b, double eps) {
    refuse_transforms(std::initializer_list<Maybe>{x, w, b});
    require_gpu(x);
    same_device(x, w), same_device(x, b);
    TORCH_CHECK_VALUE(x.dim() >= 1, "layer_norm needs at least one dimension");
    dtype_code(x.scalar_type());
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
    const int64_t cols = x.size(-1);
    auto fits = [&](const char* what, const Maybe& t) {
        if (!t) return;
        TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == cols, what, " has shape ", t->sizes(), ", expected [", cols, "]");
        TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, what, " has dtype ", t->scalar_type(), "; it must be ", x.scalar_type(), " or Float");
    };
    fits("weight", w), fits("bias", b);
    if (w && b) TORCH_CHECK_TYPE(w->scalar_type() == b->scalar_type(), "weight and bias have different dtypes: ", w->scalar_type(), " and ", b->scalar_type());
    const Tensor x2 = rows_of(x);
    const Maybe w2 = contiguous(w), b2 = contiguous(b);
    Tensor y;
    if (at::GradMode::is_enabled() && (x2.requires_grad() || wants_grad(w2) || wants_grad(b2))) {
        refuse_eager_leaves({x, w, b});
        y = LayerNorm::apply(x2, w2, b2, eps);
    }
    else y = norm_forward(x2, w2, b2, eps, nullptr);
    return x.dim() == 2 ? y : y.view(x.sizes());
}

// ---------------------------------------------------------------------------------------------------- rotary
struct RotaryHow { int64_t first; double gain; int64_t interleaved; };

// pos: (tokens,) or (batch, tokens), or not given.
void rotary_into(const Tensor& q, const Tensor& k, const Tensor& qo, const Tensor& ko, const Tensor& freq, const Maybe& pos, const RotaryHow& h, int inverse) {
    const On on(q);
    const bool two = k.defined(), given = pos && pos->defined();
    const int64_t pos_batch = given && pos->dim() == 2 ? pos->stride(0) : 0, pos_token = given ? pos->stride(-1) : 0;
    check(sthip_rotary(q.data_ptr(), ptr(k), qo.data_ptr(), ptr(ko), q.size(0), q.size(1), q.size(2), two ? k.size(2) : 0, q.size(3), 2 * freq.size(0),
                       q.strides().data(), two ? k.strides().data() : nullptr, qo.strides().data(), two ? ko.strides().data() : nullptr,
                       freq.data_ptr<double>(), ptr(pos), given ? (int)pos->element_size() * 8 : 0, pos_batch, pos_token, h.first,
                       h.gain, (int)h.interleaved, inverse, dtype_code(q.scalar_type()), on.stream));
}
Tensor unit_heads(const Tensor& t) {
    if (t.defined() && t.is_neg()) return unit_heads(t.resolve_neg());
    return !t.defined() || t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous();
}
Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : t; }

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k, const Tensor& freq, const Maybe& pos, RotaryHow h) {
        const Tensor kt = k ? *k : Tensor();
        Tensor qo = like(q), ko = like(kt);
        rotary_into(q, kt, qo, ko, freq, pos, h, 0);
        ctx->save_for_backward({freq, pos ? *pos : Tensor()});
        ctx->saved_data["how"] = std::vector<int64_t>{h.first, h.interleaved, freq.size(0), pos ? (int64_t)pos->scalar_type() : -1, pos ? pos->dim() : 0};
        ctx->saved_data["gain"] = h.gain;
        ctx->set_materialize_grads(false);
        if (k) return {qo, ko};
        return {qo};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_transforms(grads);
        const variable_list saved = ctx->get_saved_variables();
        const auto v = ctx->saved_data["how"].toIntVector();
        const RotaryHow h = {v[0], ctx->saved_data["gain"].toDouble(), v[1]};
        variable_list out(5), in, turned;
        int at[2], n = 0;
        {
            const at::NoGradGuard no_grad;
            for (int i = 0; i < (int)grads.size(); ++i)
                if (grads[i].defined() && ctx->needs_input_grad(i)) { in.push_back(unit_heads(grads[i])); at[n++] = i; }
            if (n) {
                const c10::DeviceGuard guard(in[0].device());
                for (auto& t : in) turned.push_back(like(t));
                in.resize(2), turned.resize(2);
                const Tensor freq = restored(saved[0], "frequencies", {v[2]}, at::kDouble, in[0]).contiguous();
                Maybe pos;
                if (v[4]) pos = restored(saved[1], "positions", in[0].sizes().slice(2 - v[4], v[4]), (at::ScalarType)v[3], in[0]);
                rotary_into(in[0], in[1], turned[0], turned[1], freq, pos, h, 1);
            }
        }
        for (int i = 0; i < n; ++i) out[at[i]] = turned[i];
        return once(std::move(out));
    }
};

// Whether integers within their bounds give sum(step * number) = target.  Terms in descending order of their steps (all positive): of
// each only those numbers are tried whose rest the terms behind it can reach, one or two where strides nest.  Yes where `tries` run out.
struct Term { int64_t step, lo, hi; };
int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
bool reaches(const Term* t, const Term* end, int64_t target, int& tries) {
    if (t == end) return target == 0;
    if (--tries < 0) return true;
    int64_t lo = 0, hi = 0;   // of the terms behind
    for (const Term* r = t + 1; r != end; ++r) lo += r->step * r->lo, hi += r->step * r->hi;
    const int64_t last = std::min(t->hi, floor_div(target - lo, t->step));
    for (int64_t n = std::max(t->lo, -floor_div(hi - target, t->step)); n <= last; ++n)
        if (reaches(t + 1, end, target - n * t->step, tries)) return true;
    return false;
}
constexpr int kTries = 100000;   // a millisecond
bool descending(const Term& a, const Term& b) { return a.step > b.step; }

// Whether two elements share memory: their indices differ, first in some dimension and there by a positive number.
bool overlaps_itself(const Tensor& t) {
    std::vector<Term> d;
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) == 0) return false;
        if (t.size(i) > 1) d.push_back({t.stride(i), 1 - t.size(i), t.size(i) - 1});
    }
    std::sort(d.begin(), d.end(), descending);
    if (!d.empty() && d.back().step == 0) return true;
    int tries = kTries;
    for (size_t i = 0; i < d.size(); ++i) {
        const int64_t lo = std::exchange(d[i].lo, 1);
        if (reaches(d.data() + i, d.data() + d.size(), 0, tries)) return true;
        d[i].lo = lo;
    }
    return false;
}

// Whether an element of q and one of k share memory: byte q + sum(index * stride) + byte of the element = the same of k.
bool share(const Tensor& q, const Tensor& k) {
    if (!q.numel() || !k.numel()) return false;
    const int64_t es = q.element_size();
    std::vector<Term> d = {{1, 1 - es, es - 1}};
    auto add = [&](const Tensor& t, int sign) {
        for (int64_t i = 0; i < t.dim(); ++i) {
            const int64_t step = t.stride(i) * es, most = sign * (t.size(i) - 1);
            if (most == 0 || step == 0) continue;
            auto same = std::find_if(d.begin(), d.end(), [&](const Term& u) { return u.step == step; });
            if (same == d.end()) same = d.insert(d.end(), {step, 0, 0});
            (most < 0 ? same->lo : same->hi) += most;
        }
    };
    add(q, 1), add(k, -1);
    std::sort(d.begin(), d.end(), descending);
    int tries = kTries;
    return reaches(d.data(), d.data() + d.size(), (const char*)k.data_ptr() - (const char*)q.data_ptr(), tries);
}

std::tuple<Tensor, Maybe> rotary(const Tensor& q, const Maybe& k, const Tensor& freq, const Maybe& pos, bool interleaved, double gain, int64_t first, bool inplace) {
    refuse_transforms(std::initializer_list<Maybe>{q, k, freq, pos});
    require_gpu(q);
    same_device(q, k), same_device(q, freq), same_device(q, pos);
    const int64_t d = q.dim();
    TORCH_CHECK_VALUE((d == 3 || d == 4) && (!k || (k->dim() == d && k->sizes().slice(0, d - 2) == q.sizes().slice(0, d - 2) && k->size(-1) == q.size(-1))),
                      "expected q and k of (batch, tokens, heads, dim), got ", q.sizes(), " and ", k ? k->sizes() : at::IntArrayRef());
    dtype_code(q.scalar_type());
    if (k) TORCH_CHECK_TYPE(k->scalar_type() == q.scalar_type(), "q and k have different dtypes: ", q.scalar_type(), " and ", k->scalar_type());
    TORCH_CHECK_TYPE(freq.dim() == 1 && freq.scalar_type() == at::kDouble, "frequencies must be a 1-D float64 tensor (rotary_frequencies)");
    TORCH_CHECK_VALUE(2 <= 2 * freq.size(0) && 2 * freq.size(0) <= q.size(-1), freq.size(0), " frequencies do not fit a head of ", q.size(-1), " elements");
    const bool flat = d == 3;
    Tensor q4 = flat ? q.unsqueeze(0) : q, k4 = !k ? Tensor() : flat ? k->unsqueeze(0) : *k;
    const int64_t batch = q4.size(0), tokens = q4.size(1);
    const RotaryHow h = {first, gain, interleaved};
    if (pos) {
        TORCH_CHECK_TYPE(pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong, "positions must be int32 or int64, got ", pos->scalar_type());
        TORCH_CHECK_VALUE((pos->dim() == 1 && pos->size(0) == tokens) || (!flat && pos->dim() == 2 && pos->size(0) == batch && pos->size(1) == tokens),
                          "positions have shape ", pos->sizes(), ", expected [", tokens, "] or [", batch, ", ", tokens, "]");
    }
    TORCH_CHECK(!freq.requires_grad(), "rotary has no gradient for its frequencies");
    const Tensor f = freq.resolve_neg().contiguous();
    const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k));
    if (inplace) {
        TORCH_CHECK(!grad, "rotary(inplace=True) has no gradient");
        for (const Tensor& t : {q4, k4}) {
            if (!t.defined()) continue;
            TORCH_CHECK_VALUE(!t.is_neg(), "rotary(inplace=True) on a tensor with a pending negation");
            TORCH_CHECK_VALUE(t.size(3) <= 1 || t.stride(3) == 1, "rotary(inplace=True) needs unit stride within a head");
            TORCH_CHECK_VALUE(!overlaps_itself(t), "rotary(inplace=True) on a tensor whose elements share memory");
        }
        TORCH_CHECK_VALUE(!k || !share(q4, k4), "rotary(inplace=True) on q and k that share memory");
        rotary_into(q4, k4, q4, k4, f, pos, h, 0);
        if (!q.is_inference()) q.unsafeGetTensorImpl()->bump_version();
        if (k && !k->is_inference()) k->unsafeGetTensorImpl()->bump_version();
        return {q, k};
    }
    q4 = unit_heads(q4), k4 = unit_heads(k4);
    Tensor qo, ko;
    if (grad) {
        refuse_eager_leaves({q, k});
        variable_list out = Rotary::apply(q4, k ? Maybe(k4) : Maybe(), f, pos, h);
        qo = out[0];
        if (k) ko = out[1];
    } else {
        const c10::DeviceGuard guard(q.device());
        qo = like(q4), ko = like(k4);
        rotary_into(q4, k4, qo, ko, f, pos, h, 0);
    }
    if (flat) { qo = qo.squeeze(0); if (k) ko = ko.squeeze(0); }
    return {qo, k ? Maybe(ko) : Maybe()};
}

}  // namespace

PYBIND11_MODULE(_sthip_torch, m) {
    pybind11::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const SthipFailure& e) {
            const pybind11::object kind = pybind11::module_::import("strassen_hip._capi").attr("SthipError");
            PyErr_SetObject(kind.ptr(), kind(e.code, e.message).ptr());
        }
    });
    namespace py = pybind11;
    m.def("linear_act", &linear_act, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("residual"), py::arg("activation"));
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
    m.def("rotary", &rotary, py::arg("q"), py::arg("k"), py::arg("frequencies"), py::arg("positions"), py::arg("interleaved"), py::arg("gain"), py::arg("first"), py::arg("inplace"));
    m.def("overlaps_itself", &overlaps_itself);
    m.def("share", &share);
}
