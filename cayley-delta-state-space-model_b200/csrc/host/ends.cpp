// The ends of a training step, one native call each: rows of a table for token ids, the loss of hidden rows against a vocabulary, both
// with their gradients, and the norm and clipping of all gradients.
#include "host.h"

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

// (rows, d) of a matrix whose rows are dense, wherever they lie; else a copy.
Tensor row_matrix(const Tensor& t, int64_t d) {
    const Tensor m = t.reshape({-1, d});
    return d == 1 || m.stride(1) == 1 ? m : m.contiguous();
}
int64_t row_stride(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

struct CeArgs {
    Tensor weight;   // (vocab, d), rows dense
    int64_t rows, d, vocab, ignore;
    int reduction, dtype;
};
Tensor ce_weight(const Tensor& weight) {
    return (weight.size(1) == 1 || weight.stride(1) == 1) && (weight.size(0) == 1 || weight.stride(0) >= weight.size(1)) ? weight : weight.contiguous();
}

// linear_ce_fwd(hidden (.., d), weight (vocab, d), targets (..) int64, ignore_index, reduction, flags) -> (loss, saved bytes)
PyObject* py_linear_ce_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        const Tensor hidden = in.tensor("hidden"), weight_ = in.tensor("weight"), targets = in.tensor("targets");
        const int64_t ignore = in.integer(), reduction = in.integer(), flags = in.integer();
        need_cuda(hidden, "hidden");
        need_cuda(weight_, "weight");
        need_cuda(targets, "targets");
        need_same_device(weight_, hidden, "weight");
        need_same_device(targets, hidden, "targets");
        const int dt = dtype_code(hidden);
        if (weight_.scalar_type() != hidden.scalar_type())
            throw Error(std::string("weight has dtype ") + c10::toString(weight_.scalar_type()) + ", hidden " + c10::toString(hidden.scalar_type()));
        if (targets.scalar_type() != at::kLong) throw Error("targets must be int64");
        need_dims(weight_, 2, "weight");
        if (hidden.dim() < 1 || hidden.size(-1) != weight_.size(1)) throw Error("hidden and weight must agree in their last dimension");
        const int64_t d = weight_.size(1), vocab = weight_.size(0);
        if (d < 1 || vocab < 1) throw Error("weight is empty");
        if (targets.sizes() != hidden.sizes().slice(0, hidden.dim() - 1)) throw Error("targets must have hidden's shape without its last dimension");
        const int64_t rows = targets.numel();
        Tensor loss, saved;
        without_gil([&] {
            const c10::cuda::CUDAGuard guard(hidden.device());
            loss = reduction == CDSSM_CE_NONE ? empty_f32(targets.sizes(), hidden) : empty_f32({}, hidden);
            if (rows == 0) {   // mean of nothing: NaN, as everywhere
                if (reduction != CDSSM_CE_NONE) loss.fill_(reduction == CDSSM_CE_MEAN ? NAN : 0.0);
                saved = scratch(0, hidden);
                return;
            }
            const size_t sb = cdssm_b200_linear_ce_saved_bytes(rows, (int)std::min<int64_t>(d, INT32_MAX), (int)std::min<int64_t>(vocab, INT32_MAX), dt);
            const size_t wb = cdssm_b200_linear_ce_workspace_bytes(rows, (int)std::min<int64_t>(d, INT32_MAX), (int)std::min<int64_t>(vocab, INT32_MAX), dt, 0);
            if (sb == 0) check(CDSSM_ERR_UNSUPPORTED, "linear_ce_fwd");
            const Tensor x = row_matrix(hidden, d), w = ce_weight(weight_), y = targets.contiguous(), ws = scratch(wb, hidden);
            saved = scratch(sb, hidden);
            check(cdssm_b200_linear_ce_fwd(cptr(x), row_stride(x), cptr(w), row_stride(w), y.const_data_ptr<int64_t>(), fmut(loss), mptr(saved), sb,
                                           mptr(ws), wb, rows, (int)d, (int)vocab, ignore, (int)reduction, dt, (int)flags, stream_of(x)),
                  "linear_ce_fwd");
        });
        return Py_BuildValue("(NN)", wrap(std::move(loss)), wrap(std::move(saved)));
    });
}

// linear_ce_bwd(grad_loss, weight, targets, saved, ignore_index, reduction, want_x, want_w, flags) -> (grad_x (rows, d) or None, grad_w or None)
PyObject* py_linear_ce_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        const Tensor grad_ = in.tensor("grad_loss"), weight_ = in.tensor("weight"), targets = in.tensor("targets"), saved = in.tensor("saved");
        const int64_t ignore = in.integer(), reduction = in.integer();
        const bool want_x = in.flag(), want_w = in.flag();
        const int64_t flags = in.integer();
        const int64_t rows = targets.numel(), d = weight_.size(1), vocab = weight_.size(0);
        const int dt = dtype_code(weight_);
        Tensor gx, gw;
        without_gil([&] {
            const c10::cuda::CUDAGuard guard(weight_.device());
            if (want_x) gx = empty_like_dims({rows, d}, weight_);
            if (want_w) gw = rows ? empty_like_dims({vocab, d}, weight_) : at::zeros({vocab, d}, weight_.options());
            if (rows == 0 || (!want_x && !want_w)) return;
            const size_t wb = cdssm_b200_linear_ce_workspace_bytes(rows, (int)d, (int)vocab, dt, 1);
            const Tensor g = grad_.to(at::kFloat).contiguous(), w = ce_weight(weight_), y = targets.contiguous(), ws = scratch(wb, weight_);
            check(cdssm_b200_linear_ce_bwd(fptr(g), cptr(w), row_stride(w), y.const_data_ptr<int64_t>(), mptr(saved), (size_t)saved.numel(), mptr(gx),
                                           mptr(gw), mptr(ws), wb, rows, (int)d, (int)vocab, ignore, (int)reduction, dt, (int)flags, stream_of(w)),
                  "linear_ce_bwd");
        });
        auto give = [](Tensor& t) { return t.defined() ? wrap(std::move(t)) : (Py_INCREF(Py_None), Py_None); };
        PyObject* x = give(gx);
        return Py_BuildValue("(NN)", x, give(gw));
    });
}

// embedding_fwd(ids (..) int64, weight (vocab, d), scale) -> out (.., d)
PyObject* py_embedding_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        const Tensor ids_ = in.tensor("ids"), weight = in.tensor("weight");
        const float scale = (float)in.number();
        need_cuda(ids_, "ids");
        need_cuda(weight, "weight");
        need_same_device(ids_, weight, "ids");
        if (ids_.scalar_type() != at::kLong) throw Error("ids must be int64");
        need_dims(weight, 2, "weight");
        const int64_t d = weight.size(1), vocab = weight.size(0), count = ids_.numel();
        if (d < 1 || vocab < 1) throw Error("weight is empty");
        const int dt = dtype_code(weight);
        return wrap(without_gil([&] {
            const c10::cuda::CUDAGuard guard(weight.device());
            auto sizes = ids_.sizes().vec();
            sizes.push_back(d);
            const Tensor out = empty_like_dims(sizes, weight);
            if (count == 0) return out;
            if (d > INT32_MAX || vocab > INT32_MAX) check(CDSSM_ERR_UNSUPPORTED, "embedding_fwd");
            const Tensor ids = ids_.contiguous(), w = ce_weight(weight);
            check(cdssm_b200_embedding_fwd(ids.const_data_ptr<int64_t>(), cptr(w), row_stride(w), mptr(out), count, (int)vocab, (int)d, scale, dt,
                                           stream_of(w)),
                  "embedding_fwd");
            return out;
        }));
    });
}

// embedding_bwd(grad (.., d), ids, vocab, padding_idx (-1: none), scale) -> grad_weight (vocab, d)
PyObject* py_embedding_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&] {
        Args in{a, n};
        const Tensor grad_ = in.tensor("grad"), ids_ = in.tensor("ids");
        const int64_t vocab = in.integer(), padding = in.integer();
        const float scale = (float)in.number();
        const int64_t d = grad_.size(-1), count = ids_.numel();
        return wrap(without_gil([&] {
            const c10::cuda::CUDAGuard guard(grad_.device());
            if (count == 0) return at::zeros({vocab, d}, grad_.options());
            const Tensor out = empty_like_dims({vocab, d}, grad_);
            const int dt = dtype_code(grad_);
            const size_t bytes = cdssm_b200_embedding_bwd_workspace_bytes(count, (int)vocab, (int)d, dt);
            if (bytes == 0) check(CDSSM_ERR_UNSUPPORTED, "embedding_bwd");
            Tensor grad = grad_.contiguous();
            if (reinterpret_cast<uintptr_t>(grad.const_data_ptr()) & 15) grad = grad.clone();
            const Tensor ids = ids_.contiguous(), ws = scratch(bytes, grad_);
            check(cdssm_b200_embedding_bwd(ids.const_data_ptr<int64_t>(), cptr(grad), mptr(out), mptr(ws), bytes, count, (int)vocab, (int)d, padding,
                                           scale, dt, stream_of(grad)),
                  "embedding_bwd");
            return out;
        }));
    });
}

// Tensors as the kernels walk them: every value once, in the order of memory.
void need_dense(const Tensor& t, const char* name) {
    need_cuda(t, name);
    if (t.layout() != at::kStrided) throw Error(std::string(name) + ": a sparse tensor");
    dtype_code(t);
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
    std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.at < y.at; });
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
        for (size_t i = 0; i < ins.size(); i++) {
            need_dense(ins[i], "gradients");
            need_same_device(ins[i], ins[0], "gradients");
            pi.push_back(cptr(ins[i]));
            sizes.push_back(ins[i].numel());
            di.push_back(dtype_code(ins[i]));
            if (!scale) continue;
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
    {"linear_ce_fwd", FAST(py_linear_ce_fwd)},
    {"linear_ce_bwd", FAST(py_linear_ce_bwd)},
    {"embedding_fwd", FAST(py_embedding_fwd)},
    {"embedding_bwd", FAST(py_embedding_bwd)},
    {"grad_clip", FAST(py_grad_clip)},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef* ends_methods() { return g_ends_methods; }

}  // namespace cdssm_host
