// The ends of a training step: the loss of hidden rows against a vocabulary, forward and backward, one native call each.
#include "host.h"

#include <cmath>

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

#define FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn)), METH_FASTCALL, nullptr
PyMethodDef g_ends_methods[] = {
    {"linear_ce_fwd", FAST(py_linear_ce_fwd)},
    {"linear_ce_bwd", FAST(py_linear_ce_bwd)},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef* ends_methods() { return g_ends_methods; }

}  // namespace cdssm_host
