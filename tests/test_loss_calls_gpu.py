"""Calls of ops.linear_cross_entropy and of its C entry points that go beyond one forward and one backward pass."""
import pytest
import torch

from test_loss_gpu import _grads, _inputs

pytestmark = pytest.mark.gpu


class Entry:
    """The C entry points on tensors: one forward, then any number of backward passes over what it saved."""

    def __init__(self, ops, x, w, y):
        self.h, self.ops, self.x, self.w, self.y = ops._lib.lib(), ops, x, w, y
        self.dt = ops._lib.BF16 if x.dtype == torch.bfloat16 else ops._lib.F32
        (self.T, self.d), self.V = x.shape, w.shape[0]
        self.saved = self._bytes(self.h.cdssm_b200_linear_ce_saved_bytes(self.T, self.d, self.V, w.data_ptr(), w.stride(0), self.dt))
        self.loss = torch.empty((), device="cuda")
        ws = self._bytes(self.h.cdssm_b200_linear_ce_workspace_bytes(self.T, self.d, self.V, self.dt, 0))
        assert self.h.cdssm_b200_linear_ce_fwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), y.data_ptr(), self.loss.data_ptr(),
                                               self.saved.data_ptr(), self.saved.numel(), ws.data_ptr(), ws.numel(), self.T, self.d, self.V, -100,
                                               1, self.dt, 0, torch.cuda.current_stream().cuda_stream) == 0

    @staticmethod
    def _bytes(n):                                                   # (what lay in the memory before is no part of a call)
        return torch.full((n,), 255, dtype=torch.uint8, device="cuda")

    def backward(self, flags=0, wait=True):
        ws = self.ws = self._bytes(self.h.cdssm_b200_linear_ce_workspace_bytes(self.T, self.d, self.V, self.dt, 1))
        gx, gw, one = torch.empty_like(self.x), torch.empty_like(self.w), torch.ones((), device="cuda")
        assert self.h.cdssm_b200_linear_ce_bwd(one.data_ptr(), self.w.data_ptr(), self.w.stride(0), self.y.data_ptr(), self.saved.data_ptr(),
                                               self.saved.numel(), gx.data_ptr(), gw.data_ptr(), ws.data_ptr(), ws.numel(), self.T, self.d, self.V,
                                               -100, 1, self.dt, flags, torch.cuda.current_stream().cuda_stream) == 0
        if wait:
            torch.cuda.synchronize()
        return gx, gw


@pytest.mark.parametrize("T,V,d,dtype", [(300, 700, 96, torch.bfloat16), (20, 700, 96, torch.bfloat16), (20, 700, 1000, torch.bfloat16),
                                         (300, 700, 96, torch.float32), (20, 700, 96, torch.float32), (65600, 8191, 8, torch.bfloat16)])
def test_a_backward_that_gave_up_leaves_nothing_to_the_next(ops, T, V, d, dtype):
    """One forward, a backward pass whose loads are withheld, then a whole one: its gradients are those of a forward of its own, and what the
    forward saved is as it was.  (The last size forms the logits' gradient in three pieces.)"""
    x, w, y = _inputs(T, V, d, dtype, seed=40)
    want = _grads(ops, x, w, y, torch.ones((), device="cuda"))
    e = Entry(ops, x, w, y)
    kept = e.saved.clone()
    assert torch.equal(e.loss, want[0])
    assert all(torch.equal(a, b) for a, b in zip(e.backward(), want[1:]))
    old = ops.set_wait_limit_ns(2_000_000)
    try:
        assert all(g.isnan().all() for g in e.backward(ops.TEST_WITHHOLD))
    finally:
        ops.set_wait_limit_ns(old)
    assert torch.equal(e.saved, kept)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(e.backward(), want[1:]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [20, 300])
def test_saved_tensors_that_move(ops, T, dtype):
    """Hooks that keep what was saved elsewhere: the weight comes back dense, though its rows lay apart or at an odd address when the forward read it,
    and what was dense comes back with rows apart."""
    V, d = 200, 100
    x, w, y = _inputs(T, V, d, dtype, seed=41)
    apart = lambda t, pitch: torch.zeros(V, pitch, device="cuda", dtype=dtype)[:, :d].copy_(t)  # noqa: E731
    odd = torch.zeros(V * d + 1, device="cuda", dtype=dtype)[1:].view(V, d).copy_(w)
    g = torch.randn(T, device="cuda")
    want = _grads(ops, x, w, y, g, reduction="none")

    def through(hooks, wt):
        a, b = x.detach().requires_grad_(), wt.detach().requires_grad_()
        with hooks:
            loss = ops.linear_cross_entropy(a, b, y, reduction="none")
        return (loss.detach(), *torch.autograd.grad(loss, [a, b], [g]))

    for wt in (w, apart(w, 104), apart(w, 101), odd):
        assert all(torch.equal(p, q) for p, q in zip(through(torch.autograd.graph.save_on_cpu(), wt), want))
        for move in (lambda t: apart(t, 104), lambda t: apart(t, 103)):
            hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t, move=move: move(t) if t.dim() == 2 else t)
            assert all(torch.equal(p, q) for p, q in zip(through(hooks, wt), want))


def test_transforms_are_refused(ops):
    """vmap, func.grad and func.jvp hand over tensors without memory of their own: an error, not a value."""
    x, w, y = _inputs(6, 10, 16, torch.bfloat16, seed=42)
    loss = lambda t: ops.linear_cross_entropy(t, w, y)  # noqa: E731
    for call in (lambda: torch.vmap(loss)(torch.stack([x, x])), lambda: torch.func.grad(loss)(x), lambda: torch.func.jvp(loss, (x,), (x,)),
                 lambda: torch.vmap(lambda t: ops.embedding(y.clamp(min=0), t))(torch.stack([w, w])),
                 lambda: torch.vmap(lambda t: ops.grad_norm([t]))(torch.stack([w, w]))):
        with pytest.raises(RuntimeError):
            call()


def test_saved_tensors_that_come_back_as_something_else(ops):
    """On the host, of another type, of another shape: an error before anything is launched."""
    x, w, y = _inputs(20, 30, 16, torch.float32, seed=43, ignored=0.0)
    calls = [lambda: ops.linear_cross_entropy(x.detach().requires_grad_(), w.detach().requires_grad_(), y),
             lambda: ops.embedding(y, w.detach().requires_grad_()).sum()]
    kinds = {"weight": lambda t: t.dim() == 2, "ids": lambda t: t.dtype == torch.int64, "rows": lambda t: t.dtype == torch.uint8}
    other = {torch.float32: torch.bfloat16, torch.int64: torch.int32, torch.uint8: torch.int32}
    for change in (lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.to(other[t.dtype])):
        for kind, mine in kinds.items():
            for call in calls[:2 if kind == "ids" else 1]:
                with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if mine(t) else t):
                    loss = call()
                with pytest.raises(RuntimeError, match="a saved tensor came back"):
                    loss.backward()


@pytest.mark.parametrize("T,V,d", [(40, 50, 24), (40, 50, 1), (1, 1, 1)])
def test_signs_that_are_pending(ops, T, V, d):
    """Views whose values are the negatives of what lies in memory, as operands and as upstream gradients."""
    x, w, y = _inputs(T, V, d, torch.float32, seed=44, ignored=0.0)
    neg = lambda t: torch._neg_view((-t).contiguous())  # noqa: E731
    g, ge = torch.randn(T, device="cuda"), torch.randn(T, d, device="cuda")
    assert neg(w).is_neg() and torch.equal(neg(w), w)
    want = _grads(ops, x, w, y, g, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(_grads(ops, neg(x), neg(w), y, neg(g), reduction="none"), want))
    leaf = w.clone().requires_grad_()
    rows = ops.embedding(y, leaf)
    assert torch.equal(rows, ops.embedding(y, neg(w)))
    assert torch.equal(torch.autograd.grad(rows, [leaf], [neg(ge)], retain_graph=True)[0], torch.autograd.grad(rows, [leaf], [ge])[0])
    # as they come about: the loss is an imaginary part, and what is read is its conjugate's
    leaf = w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(x, leaf, y)
    got, = torch.autograd.grad(torch.complex(loss, loss).conj().imag, [leaf], retain_graph=True)
    assert torch.equal(got, -torch.autograd.grad(loss, [leaf])[0])
    assert torch.equal(ops.grad_norm([w]), ops.grad_norm([-w]))
    for call in (lambda: ops.grad_norm([neg(w)]), lambda: ops.clip_grads_([w.clone()], 1.0, out=[neg(w)])):
        with pytest.raises(ops.CdssmError, match="sign is pending"):
            call()


def test_two_passes_at_once_over_one_forward(ops):
    """On two streams, each with a workspace of its own."""
    x, w, y = _inputs(900, 2000, 64, torch.bfloat16, seed=45)
    want = _grads(ops, x, w, y, torch.ones((), device="cuda"))[1:]
    e = Entry(ops, x, w, y)
    streams, kept, got = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(e.backward(wait=False))
            kept.append(e.ws)                                        # (its memory is nobody else's while a stream may read it)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
