"""Rows of a table for token ids and the table's gradient (ops.embedding) against the formula in 64 bits.

Tolerances, u = 2^-24 and h the half step of the type (bf16 2^-8, float32 2^-24): out is one product in float32 and one rounding (u + h of
itself); a gradient entry is a sum of n float32 values in any order (n u of the absolute sum), a product and a rounding (u + h)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _ids(kind, T, V, g):
    if kind == "same":
        return torch.full((T,), V // 2, device="cuda")
    if kind == "few":
        return torch.randint(0, min(V, 3), (T,), generator=g, device="cuda")
    if kind == "runs":                                   # whole tiles of one id, ending at tile borders and inside them
        return (torch.arange(T, device="cuda") // 32 * 7 + (torch.arange(T, device="cuda") % 3 == 0)) % V
    rank = torch.rand(T, generator=g, device="cuda", dtype=torch.float64).mul_(torch.tensor(float(V)).log().item()).exp_().long() - 1
    return rank.clamp_(0, V - 1) if kind == "zipf" else torch.randint(0, V, (T,), generator=g, device="cuda")


def _check(ops, ids, w, grad, scale, padding=None):
    w = w.detach().requires_grad_()
    out = ops.embedding(ids, w, scale=scale, padding_idx=padding)
    dw, = torch.autograd.grad(out, [w], [grad])
    V, d, h = *w.shape, HALF[w.dtype]
    want = w.detach().double()[ids] * scale
    assert out.shape == want.shape and out.dtype == w.dtype
    assert ((out.double() - want).abs() <= (U + h) * want.abs()).all()
    flat, g = ids.reshape(-1), grad.double().reshape(-1, d)
    if padding is not None:
        g = torch.where((flat == padding)[:, None], 0.0, g)
    total, size = (torch.zeros(V, d, device="cuda", dtype=torch.float64).index_add_(0, flat, x) for x in (g, g.abs()))
    n = torch.bincount(flat, minlength=V)[:, None]
    assert dw.shape == w.shape and dw.dtype == w.dtype
    off = (dw.double() - scale * total).abs()
    assert (off <= abs(scale) * ((n + 1) * U * size) + (U + h) * (abs(scale) * total.abs() + n * U * size)).all(), off.max()
    assert (dw[n[:, 0] == 0] == 0).all()
    assert torch.equal(dw, torch.autograd.grad(ops.embedding(ids, w, scale=scale, padding_idx=padding), [w], [grad])[0])   # run to run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "same", "few", "runs"])
@pytest.mark.parametrize("T,V,d", [(1, 1, 1), (31, 5, 8), (32, 600, 100), (33, 3, 257), (523, 32000, 768), (4096, 511, 64), (4097, 512, 65), (20000, 50257, 96)])
def test_rows_and_gradient(ops, T, V, d, kind, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + V + d)
    w, grad = (torch.randn(n, d, generator=g, device="cuda").to(dtype) for n in (V, T))
    _check(ops, _ids(kind, T, V, g), w, grad, 1.0)
    _check(ops, _ids(kind, T, V, g), w, grad, -(d ** 0.5))


@pytest.mark.parametrize("T,V", [(70000, 300000), (300000, 7)])      # three passes of the sort; many pairs a block
def test_large(ops, T, V):
    g = torch.Generator(device="cuda").manual_seed(T)
    w, grad = (torch.randn(n, 16, generator=g, device="cuda").bfloat16() for n in (V, T))
    _check(ops, torch.randint(0, V, (T,), generator=g, device="cuda"), w, grad, 0.5)


def test_tables_and_ids_anywhere(ops):
    g = torch.Generator(device="cuda").manual_seed(1)
    V, d = 40, 24
    for dtype in (torch.bfloat16, torch.float32):
        base = torch.randn(V, d + 11, generator=g, device="cuda").to(dtype)
        ids = torch.randint(0, V, (5, 14), generator=g, device="cuda")
        for w in (base[:, :d], base[:, 8:8 + d], base[:, 3:3 + d], base[:, :d].t().contiguous().t(), base[::2, :d]):
            part = ids % w.shape[0]
            for i in (part, part.t(), part[:, ::3], part[2, 4], part[:, :0]):
                grad = torch.randn(*i.shape, d + 1, generator=g, device="cuda").to(dtype)[..., 1:]      # an odd stride and address
                _check(ops, i, w, grad, 1.0)


def test_padding_and_ids_that_are_no_row(ops):
    g = torch.Generator(device="cuda").manual_seed(2)
    V, d, T = 60, 33, 500
    w, grad = (torch.randn(n, d, generator=g, device="cuda") for n in (V, T))
    ids = torch.randint(0, 9, (T,), generator=g, device="cuda")
    _check(ops, ids, w, grad, 2.0, padding=4)
    wrong = ids.clone()
    wrong[[1, 7, 100]] = torch.tensor([-1, V, 2 ** 40], device="cuda")
    ok = torch.ones(T, dtype=torch.bool, device="cuda")
    ok[[1, 7, 100]] = False
    w.requires_grad_()
    out = ops.embedding(wrong, w)
    assert out[~ok].isnan().all() and torch.equal(out[ok], w[ids[ok]])
    spoilt = torch.where(ok[:, None], grad, float("nan"))
    assert torch.equal(torch.autograd.grad(out, [w], [spoilt])[0], torch.autograd.grad(ops.embedding(wrong[ok], w), [w], [grad[ok]])[0])


def test_another_stream_and_captured(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    V, d, T = 1000, 64, 9000
    w, grad = torch.randn(V, d, generator=g, device="cuda").bfloat16().requires_grad_(), torch.randn(T, d, generator=g, device="cuda").bfloat16()
    ids = _ids("zipf", T, V, g)
    run = lambda: [(o := ops.embedding(ids, w)).detach(), *torch.autograd.grad(o, [w], [grad])]  # noqa: E731
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = run()
    for kind in ("same", "uniform", "runs"):
        ids.copy_(_ids(kind, T, V, g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


def test_refusals(ops):
    w, ids = torch.randn(10, 8, device="cuda"), torch.arange(4, device="cuda")
    for i, t, kw in ((ids.cpu(), w, {}), (ids, w.cpu(), {}), (ids.int(), w, {}), (ids, w.half(), {}), (ids, w[0], {}), (ids, w[:0], {}),
                     (ids, w, dict(padding_idx=10)), (ids, w, dict(padding_idx=-2))):
        with pytest.raises(ops.CdssmError):
            ops.embedding(i, t, **kw)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ops.embedding(ids, w.requires_grad_()).sum(), [w], create_graph=True)
