// The ends of a training step, one native call each: rows of a table for token ids, the loss of hidden rows against a vocabulary, both
// with their gradients, and the norm and clipping of all gradients.
#include "host.h"

#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace cdssm_host {
namespace {

// One buffer of a call, 256-byte aligned, from the framework's allocator: of this call alone, whatever streams or graphs run beside it.
Tensor scratch(size_t bytes, const Tensor& on) { return empty_cuda({(int64_t)std::max<size_t>(bytes, 1)}, at::kByte, on); }

void need_same_device(const Tensor& t, const Tensor& as, const char* name) {
    if (t.device() != as.device()) throw Error(std::string(name) + " is on " + t.device().str() + ", not on " + as.device().str());
}

// Values as they lie in memory: of the imaginary part of a conjugate, say, the sign is pending.
Tensor signed_values(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// (rows, d) of a matrix whose rows are dense, wherever they lie; else a copy.
Tensor row_matrix(const Tensor& t, int64_t d) {
    const Tensor m = signed_values(t).reshape({-1, d});
    return d == 1 || m.stride(1) == 1 ? m : m.contiguous();
}
int64_t row_stride(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

// (vocab, d), rows dense and apart: as it lies, or a copy
Tensor table(const Tensor& t) {
    const Tensor w = signed_values(t);
    return (w.size(1) == 1 || w.stride(1) == 1) && (w.size(0) == 1 || w.stride(0) >= w.size(1)) ? w : w.contiguous();
}
void need_table(const Tensor& w, const char* name) {
    need_cuda(w, name);
    need_dims(w, 2, name);
    if (w.size(0) < 1 || w.size(1) < 1) throw Error(std::string(name) + " is empty");
    if (w.size(0) > INT32_MAX || w.size(1) > INT32_MAX) check(CDSSM_ERR_UNSUPPORTED, name);
    dtype_code(w);
}
bool wants_grad(const Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }
// A tangent (torch.autograd.forward_ad) has no formula here: kernels that read the values alone would drop it without a word.
// (Whether there may be any is asked first: 32 gradients one by one took 1.6 us of a call's 12.)
void need_no_tangents(const char* what, at::ArrayRef<Tensor> a, at::ArrayRef<Tensor> b = {}) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !torch::autograd::ForwardADLevel::try_get_by_idx(0)) return;
    for (const auto& list : {a, b})
        for (const Tensor& t : list)
            if (t._fw_grad(/*level=*/0).defined()) throw Error(std::string(what) + " has no forward-mode gradient");
}
// A tracer (torch.jit.trace, make_fx) records what the dispatcher sees: the outputs' allocation, and a graph that returns memory nobody has written.
void need_no_trace(const char* what) {
    using c10::impl::TorchDispatchModeTLS;
    if (at::tracer::impl::is_dispatch_enabled() || TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY)) throw Error(std::string(what) + " cannot be traced");
}
// The gradients come from kernels that autograd does not see into: a graph of them would leave out what they depend on.
void once_only(const char* what) {
    if (c10::GradMode::is_enabled()) throw Error(std::string(what) + " is differentiable once: no create_graph=True");
}

// What a forward pass saved passes through the program's hooks on its way to the backward, and kernels go by what it was then.
void need_as_saved(const char* what, const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
    if (t.device() != device || t.scalar_type() != type || t.sizes() != sizes)
        throw Error(std::string(what) + ": a saved tensor came back on another device, in another shape or of another type");
}

// ---- loss ------------------------------------------------------------------------------------------
struct CeOut {
    Tensor loss, saved;
};
CeOut ce_forward(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore, int64_t reduction, int64_t flags) {
    const c10::cuda::CUDAGuard guard(hidden.device());
    const int64_t d = weight.size(1), vocab = weight.size(0), rows = targets.numel();
    const int dt = dtype_code(hidden);
    const Tensor loss = reduction == CDSSM_CE_NONE ? empty_f32(targets.sizes(), hidden) : empty_f32({}, hidden);
    if (rows == 0) {   // mean of nothing: NaN, as everywhere
        if (reduction != CDSSM_CE_NONE) loss.fill_(reduction == CDSSM_CE_MEAN ? NAN : 0.0);
        return {loss, scratch(0, hidden)};
    }
    const Tensor w = table(weight);
    const size_t sb = cdssm_b200_linear_ce_saved_bytes(rows, (int)d, (int)vocab, cptr(w), row_stride(w), dt);
    if (sb == 0) check(CDSSM_ERR_UNSUPPORTED, "linear_cross_entropy");
    const size_t wb = cdssm_b200_linear_ce_workspace_bytes(rows, (int)d, (int)vocab, dt, 0);
    const Tensor x = row_matrix(hidden, d), y = targets.contiguous(), ws = scratch(wb, hidden), saved = scratch(sb, hidden);
    check(cdssm_b200_linear_ce_fwd(cptr(x), row_stride(x), cptr(w), row_stride(w), y.const_data_ptr<int64_t>(), fmut(loss), mptr(saved), sb, mptr(ws),
                                   wb, rows, (int)d, (int)vocab, ignore, (int)reduction, dt, (int)flags, stream_of(x)),
          "linear_cross_entropy");
    return {loss, saved};
}
struct CeGrads {
    Tensor x, w;
};
CeGrads ce_backward(const Tensor& grad, const Tensor& weight, const Tensor& targets, const Tensor& saved, int64_t ignore, int64_t reduction,
                    bool want_x, bool want_w, at::IntArrayRef hidden_sizes, int64_t flags) {
    const c10::cuda::CUDAGuard guard(weight.device());
    const int64_t d = weight.size(1), vocab = weight.size(0), rows = targets.numel();
    const int dt = dtype_code(weight);
    CeGrads r;
    if (want_x) r.x = empty_like_dims(hidden_sizes, weight);
    if (want_w) r.w = rows ? empty_like_dims({vocab, d}, weight) : at::zeros({vocab, d}, weight.options());
    if (rows == 0 || (!want_x && !want_w)) return r;
    const size_t wb = cdssm_b200_linear_ce_workspace_bytes(rows, (int)d, (int)vocab, dt, 1);
    Tensor w = table(weight);
    // (a weight that the forward read in place, moved since to where it cannot be, as a hook of saved tensors may: rows apart again)
    if ((size_t)saved.numel() < cdssm_b200_linear_ce_saved_bytes(rows, (int)d, (int)vocab, cptr(w), row_stride(w), dt)) {
        w = empty_like_dims({vocab, (d + 7) / 8 * 8}, weight).narrow(1, 0, d);
        w.copy_(weight);
    }
    const Tensor g = signed_values(grad.scalar_type() == at::kFloat ? grad : grad.to(at::kFloat)).contiguous(), y = targets.contiguous(), ws = scratch(wb, weight);
    check(cdssm_b200_linear_ce_bwd(fptr(g), cptr(w), row_stride(w), y.const_data_ptr<int64_t>(), cptr(saved), (size_t)saved.numel(), mptr(r.x), mptr(r.w),
                                   mptr(ws), wb, rows, (int)d, (int)vocab, ignore, (int)reduction, dt, (int)flags, stream_of(w)),
          "linear_cross_entropy backward");
    return r;
}
struct CeNode : torch::autograd::Function<CeNode> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore,
                          int64_t reduction, int64_t flags) {
        CeOut o = ce_forward(hidden, weight, targets, ignore, reduction, flags);
        ctx->save_for_backward({weight, targets, o.saved});
        ctx->saved_data["args"] = std::vector<int64_t>{ignore, reduction, flags, weight.size(0), (int64_t)weight.scalar_type(), o.saved.numel()};
        ctx->saved_data["sizes"] = hidden.sizes().vec();
        return o.loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once_only("linear_cross_entropy");
        const auto saved = ctx->get_saved_variables();
        const auto args = ctx->saved_data["args"].toIntVector(), sizes = ctx->saved_data["sizes"].toIntVector();
        const at::IntArrayRef all(sizes);
        const at::Device device = grads[0].device();
        need_as_saved("linear_cross_entropy", saved[0], {args[3], all.back()}, (at::ScalarType)args[4], device);
        need_as_saved("linear_cross_entropy", saved[1], all.slice(0, all.size() - 1), at::kLong, device);
        need_as_saved("linear_cross_entropy", saved[2], {args[5]}, at::kByte, device);
        CeGrads g = ce_backward(grads[0], saved[0], saved[1], saved[2].contiguous(), args[0], args[1], ctx->needs_input_grad(0), ctx->needs_input_grad(1), sizes, args[2]);
        return {g.x, g.w, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// linear_cross_entropy(hidden (.., d), weight (vocab, d), targets (..) int64, ignore_index, reduction, flags) -> loss
PyObject* py_linear_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        const Tensor hidden = in.tensor("hidden"), weight = in.tensor("weight"), targets = in.tensor("targets");
        const int64_t ignore = in.integer(), reduction = in.integer(), flags = in.integer();
        need_no_trace("linear_cross_entropy");
        need_no_tangents("linear_cross_entropy", hidden, weight);
        need_cuda(hidden, "hidden");
        need_table(weight, "weight");
        need_cuda(targets, "targets");
        need_same_device(weight, hidden, "weight");
        need_same_device(targets, hidden, "targets");
        dtype_code(hidden);
        if (weight.scalar_type() != hidden.scalar_type())
            throw Error(std::string("weight has dtype ") + c10::toString(weight.scalar_type()) + ", hidden " + c10::toString(hidden.scalar_type()));
        if (targets.scalar_type() != at::kLong) throw Error("targets must be int64");
        if (hidden.dim() < 1 || hidden.size(-1) != weight.size(1)) throw Error("hidden and weight must agree in their last dimension");
        if (targets.sizes() != hidden.sizes().slice(0, hidden.dim() - 1)) throw Error("targets must have hidden's shape without its last dimension");
        return wrap(without_gil([&] {
            return wants_grad(hidden) || wants_grad(weight) ? CeNode::apply(hidden, weight, targets, ignore, reduction, flags)
                                                            : ce_forward(hidden, weight, targets, ignore, reduction, flags).loss;
        }));
    });
}

// ---- embedding -----------------------------------------------------------------------------------------
Tensor embed_forward(const Tensor& ids_, const Tensor& weight, double scale) {
    const c10::cuda::CUDAGuard guard(weight.device());
    const int64_t d = weight.size(1), count = ids_.numel();
    auto sizes = ids_.sizes().vec();
    sizes.push_back(d);
    const Tensor out = empty_like_dims(sizes, weight);
    if (count == 0) return out;
    const Tensor ids = ids_.contiguous(), w = table(weight);
    check(cdssm_b200_embedding_fwd(ids.const_data_ptr<int64_t>(), cptr(w), row_stride(w), mptr(out), count, (int)weight.size(0), (int)d, (float)scale,
                                   dtype_code(weight), stream_of(w)),
          "embedding");
    return out;
}
Tensor embed_backward(const Tensor& grad_, const Tensor& ids_, int64_t vocab, int64_t d, int64_t padding, double scale) {
    const c10::cuda::CUDAGuard guard(grad_.device());
    const int64_t count = ids_.numel();
    if (count == 0) return at::zeros({vocab, d}, grad_.options());
    const Tensor out = empty_like_dims({vocab, d}, grad_);
    const int dt = dtype_code(grad_);
    const size_t bytes = cdssm_b200_embedding_bwd_workspace_bytes(count, (int)vocab, (int)d, dt);
    if (bytes == 0) check(CDSSM_ERR_UNSUPPORTED, "embedding backward");
    Tensor grad = signed_values(grad_).contiguous();
    if (reinterpret_cast<uintptr_t>(grad.const_data_ptr()) & 15) grad = grad.clone();
    const Tensor ids = ids_.contiguous(), ws = scratch(bytes, grad_);
    check(cdssm_b200_embedding_bwd(ids.const_data_ptr<int64_t>(), cptr(grad), mptr(out), mptr(ws), bytes, count, (int)vocab, (int)d, padding,
                                   (float)scale, dt, stream_of(grad)),
          "embedding backward");
    return out;
}
struct EmbedNode : torch::autograd::Function<EmbedNode> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t padding) {
        ctx->save_for_backward({ids});
        ctx->saved_data["args"] = std::vector<int64_t>{weight.size(0), weight.size(1), padding};
        ctx->saved_data["scale"] = scale;
        return embed_forward(ids, weight, scale);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once_only("embedding");
        const auto args = ctx->saved_data["args"].toIntVector();
        const Tensor ids = ctx->get_saved_variables()[0], &g = grads[0];
        need_as_saved("embedding", ids, g.sizes().slice(0, g.dim() - 1), at::kLong, g.device());
        return {embed_backward(g, ids, args[0], args[1], args[2], ctx->saved_data["scale"].toDouble()), Tensor(),
                Tensor(), Tensor()};
    }
};

// embedding(ids (..) int64, weight (vocab, d), scale, padding_idx (-1: none)) -> (.., d)
PyObject* py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        const Tensor ids = in.tensor("ids"), weight = in.tensor("weight");
        const double scale = in.number();
        const int64_t padding = in.integer();
        need_no_trace("embedding");
        need_no_tangents("embedding", weight);
        need_cuda(ids, "ids");
        need_table(weight, "weight");
        need_same_device(ids, weight, "ids");
        if (ids.scalar_type() != at::kLong) throw Error("ids must be int64");
        if (padding < -1 || padding >= weight.size(0)) throw Error("padding_idx " + std::to_string(padding) + " is no row of the table");
        return wrap(without_gil([&] { return wants_grad(weight) ? EmbedNode::apply(weight, ids, scale, padding) : embed_forward(ids, weight, scale); }));
    });
}

// ---- gradient norm ---------------------------------------------------------------------------------------
// Tensors as the kernels walk them: every value once, in the order of memory.
void need_dense(const Tensor& t, const char* name) {
    need_cuda(t, name);
    if (t.layout() != at::kStrided) throw Error(std::string(name) + ": a sparse tensor");
    dtype_code(t);
    if (t.is_neg()) throw Error(std::string(name) + ": a tensor whose sign is pending (resolve_neg() it)");
    if (!t.is_non_overlapping_and_dense()) throw Error(std::string(name) + ": a tensor with holes or overlaps in memory");
}

// No output may lie over another tensor of the call (its own input apart): blocks would read what others have written.
void need_apart(const std::vector<Tensor>& ins, const std::vector<Tensor>& outs) {
    struct Range {
        uintptr_t at, end;
        size_t i;
        bool out;
    };
    std::vector<Range> r;
    r.reserve(ins.size() + outs.size());
    auto add = [&](const Tensor& t, size_t i, bool out) {
        const uintptr_t p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        if (t.numel()) r.push_back({p, p + t.numel() * t.element_size(), i, out});
    };
    for (size_t i = 0; i < outs.size(); i++) {
        add(outs[i], i, true);
        if (outs[i].const_data_ptr() != ins[i].const_data_ptr() || outs[i].scalar_type() != ins[i].scalar_type()) add(ins[i], i, false);
    }
    const auto before = [](const Range& x, const Range& y) { return x.at < y.at; };
    if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
    uintptr_t end = 0, end_out = 0;   // of all before, of the outputs before
    for (const Range& x : r) {
        if (x.at < (x.out ? end : end_out)) throw Error("clip_grads_: an output overlaps another tensor of the call");
        end = std::max(end, x.end);
        if (x.out) end_out = std::max(end_out, x.end);
    }
}

// grad_clip(list of tensors, list of outputs or None, max_norm) -> norm; outputs may be the tensors themselves; None: the norm alone
PyObject* py_grad_clip(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        auto list = [&](PyObject* o, const char* name) {
            std::vector<Tensor> v;
            if (!PyList_Check(o)) throw Error(std::string(name) + " must be a list");
            Args items{PySequence_Fast_ITEMS(o), PyList_GET_SIZE(o)};
            v.reserve(items.n);
            for (Py_ssize_t i = 0; i < items.n; i++) v.push_back(items.tensor(name));
            return v;
        };
        const std::vector<Tensor> ins = list(in.next(), "gradients");
        PyObject* o = in.next();
        const bool scale = o != Py_None;
        const std::vector<Tensor> outs = scale ? (o == a[0] ? ins : list(o, "out")) : std::vector<Tensor>();
        const float max_norm = (float)in.number();
        if (ins.empty()) throw Error("no gradients");
        if (scale && outs.size() != ins.size()) throw Error("out must have as many tensors as the gradients");
        std::vector<const void*> pi;
        std::vector<void*> po;
        std::vector<int64_t> sizes;
        std::vector<int> di, dout;
        pi.reserve(ins.size()); po.reserve(ins.size()); sizes.reserve(ins.size()); di.reserve(ins.size()); dout.reserve(ins.size());
        const char* const what = scale ? "clip_grads_" : "grad_norm";
        need_no_trace(what);
        need_no_tangents(what, ins, outs);
        for (size_t i = 0; i < ins.size(); i++) {
            need_dense(ins[i], "gradients");
            need_same_device(ins[i], ins[0], "gradients");
            pi.push_back(cptr(ins[i]));
            sizes.push_back(ins[i].numel());
            di.push_back(dtype_code(ins[i]));
            if (!scale) continue;
            if (outs[i].is_same(ins[i])) {
                po.push_back(const_cast<void*>(pi.back()));
                dout.push_back(di.back());
                continue;
            }
            need_dense(outs[i], "out");
            need_same_device(outs[i], ins[0], "out");
            if (outs[i].sizes() != ins[i].sizes() || outs[i].strides() != ins[i].strides()) throw Error("out must have the gradients' shapes and strides");
            if (outs[i].scalar_type() != ins[i].scalar_type() && outs[i].scalar_type() != at::kFloat) throw Error("out must have the gradients' types or float32");
            po.push_back(mptr(outs[i]));
            dout.push_back(dtype_code(outs[i]));
        }
        if (scale) need_apart(ins, outs);
        return wrap(without_gil([&] {
            const c10::cuda::CUDAGuard guard(ins[0].device());
            const Tensor norm = empty_f32({}, ins[0]);
            const size_t bytes = cdssm_b200_grad_clip_workspace_bytes(sizes.data(), (int)sizes.size());
            const Tensor ws = scratch(bytes, ins[0]);
            check(cdssm_b200_grad_clip(pi.data(), scale ? po.data() : nullptr, sizes.data(), di.data(), dout.data(), (int)sizes.size(), max_norm,
                                       fmut(norm), mptr(ws), bytes, stream_of(ins[0])),
                  "grad_clip");
            for (const Tensor& t : outs)
                if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();   // written in place, as autograd counts it
            return norm;
        }));
    });
}

#define FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn)), METH_FASTCALL, nullptr
PyMethodDef g_ends_methods[] = {
    {"linear_cross_entropy", FAST(py_linear_cross_entropy)},
    {"embedding", FAST(py_embedding)},
    {"grad_clip", FAST(py_grad_clip)},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef* ends_methods() { return g_ends_methods; }

}  // namespace cdssm_host
