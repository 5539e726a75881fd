"""The norm of many tensors together and the clipped tensors (ops.grad_norm, clip_grads_, clip_grad_norm_) against 64 bits.

Tolerances, u = 2^-24: squares are exact products summed eight at a time in float32 (8 u) and then in float64, the norm is half of that and one
rounding (5 u); the factor is off by three roundings more, an output by one more and its type's (bf16 2^-8, float32 u)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _tensors(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def _exact(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


SIZES = {"one": [(1,)], "odd": [(3,), (16384,), (16385,), (0,), (7, 5), (100, 331), (2, 3, 4, 5)], "many": [(i % 77 + 1, 13) for i in range(1000)],
         "large": [(4_000_037,), (8,), (512, 4096)], "limit": [(24,)] * 48, "above": [(24,)] * 49}


@pytest.mark.parametrize("dtypes", [(torch.bfloat16,), (torch.float32,), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("kind", SIZES)
def test_norm_and_clip(ops, kind, dtypes):
    ts = _tensors(SIZES[kind], dtypes)
    n = _exact(ts)
    assert abs(float(ops.grad_norm(ts)) - n) <= 6 * U * n
    for bound in (0.37 * n, 2 * n, 0.0):
        c = min(1.0, bound / (n + 1e-6))
        wide = [torch.full_like(t, math.nan, dtype=torch.float32) for t in ts]
        same = [torch.full_like(t, math.nan) for t in ts]
        inplace = [t.clone() for t in ts]
        norms = [ops.clip_grads_(ts, bound, out=wide), ops.clip_grads_(ts, bound, out=same), ops.clip_grads_(inplace, bound)]
        assert all(abs(float(x) - n) <= 6 * U * n for x in norms) and norms[0].shape == () and norms[0].dtype == torch.float32
        for t, a, b, d in zip(ts, wide, same, inplace):
            want = t.double() * c
            assert ((a.double() - want).abs() <= 12 * U * want.abs()).all()
            assert ((b.double() - want).abs() <= (12 * U + HALF[t.dtype]) * want.abs()).all()
            assert torch.equal(b, d)
            if c == 1.0:
                assert torch.equal(b, t)


def test_views_of_a_bucket(ops):
    """Tensors that lie behind one another at every offset."""
    flat = _tensors([(50_000,)], (torch.bfloat16,))[0]
    sizes = [1, 2, 3, 5, 7, 11, 1000, 17, 16001, 31, 9999]
    sizes.append(flat.numel() - sum(sizes))
    n = _exact([flat])
    out = torch.empty(50_000 + 3, device="cuda")[3:]
    norm = ops.clip_grads_(list(flat.split(sizes)), 1.0, out=list(out.split(sizes)))
    assert abs(float(norm) - n) <= 6 * U * n
    want = flat.double() / (n + 1e-6)
    assert ((out.double() - want).abs() <= 12 * U * want.abs()).all()
    ops.clip_grads_(list(flat.split(sizes)), 1.0)
    assert ((flat.double() - want).abs() <= (12 * U + 2.0 ** -8) * want.abs()).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e19, 1e30])
def test_range(ops, scale):
    """Squares outside of float32's range."""
    ts = _tensors([(10_001,), (77,)], (torch.float32,), scale=scale) + _tensors([(5000,)], (torch.bfloat16,), scale=scale)
    n = _exact(ts)
    assert abs(float(ops.grad_norm(ts)) - n) <= 6 * U * n


def test_parameters(ops):
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((33, 5), (7,), (100,))]
    ps[0].grad, ps[2].grad = torch.randn(33, 5, device="cuda"), torch.randn(100, device="cuda")
    grads = [ps[0].grad.clone(), ps[2].grad.clone()]
    norm = ops.clip_grad_norm_(ps, 0.5)
    n = _exact(grads)
    assert abs(float(norm) - n) <= 6 * U * n and ps[1].grad is None
    for g, p in zip(grads, (ps[0], ps[2])):
        want = g.double() * 0.5 / (n + 1e-6)
        assert ((p.grad.double() - want).abs() <= 13 * U * want.abs()).all()
    assert float(ops.clip_grad_norm_([ps[1]], 1.0)) == 0.0


def test_values_that_are_no_numbers(ops):
    for bad in (math.nan, math.inf, -math.inf):
        ts = _tensors([(100,), (33,)], (torch.float32, torch.bfloat16))
        ts[0][5] = bad
        norm = ops.grad_norm(ts)
        assert norm.isnan() if math.isnan(bad) else norm.isposinf()
        out = [torch.empty_like(t) for t in ts]
        ops.clip_grads_(ts, 1.0, out=out)
        if math.isnan(bad):
            assert all(t.isnan().all() for t in out)
        else:
            assert out[0][5].isnan() and (out[0][:5] == 0).all() and (out[1] == 0).all()


def test_orders_streams_and_graphs(ops):
    ts = [torch.randn(30, 40, device="cuda").t(), torch.randn(4, 5, 6, device="cuda").permute(2, 0, 1)]      # dense, in another order
    want = [t * (0.5 / (_exact(ts) + 1e-6)) for t in ts]
    a = [t.clone(memory_format=torch.preserve_format) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.clip_grads_(a, 0.5)
    side.synchronize()
    for x, y in zip(a, want):
        assert ((x - y).abs() <= 13 * U * y.abs()).all()
    src = [torch.randn(5000, device="cuda") for _ in range(60)]
    out = [torch.empty_like(t) for t in src]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = ops.clip_grads_(src, 1.0, out=out)
    for s in (1.0, 1e-4):
        for t in src:
            t.normal_().mul_(s)
        graph.replay()
        torch.cuda.synchronize()
        n = _exact(src)
        assert abs(float(norm) - n) <= 6 * U * n
        c = min(1.0, 1.0 / (n + 1e-6))
        assert all(((o.double() - t.double() * c).abs() <= 12 * U * t.double().abs()).all() for o, t in zip(out, src))


def test_autograd_sees_the_write(ops):
    t = torch.randn(10, device="cuda")
    before = t._version
    ops.clip_grads_([t], 0.1)
    assert t._version > before


def test_refusals(ops):
    t = torch.randn(100, device="cuda")
    e = torch.empty(100, device="cuda")
    for grads, kw in (([], {}), ([t.cpu()], {}), ([t.half()], {}), ([t[::2]], {}), ([t[:1].expand(5)], {}), ([t, t], {}), ([t, t[50:]], {}),
                      ([t], dict(out=[e[:50]])), ([t], dict(out=[])), ([t], dict(out=[e.bfloat16()])), ([t[:99]], dict(out=[t[1:]])),
                      ([t, e], dict(out=[e, t])), ([t, e], dict(out=[torch.empty_like(t)] * 2)), ([t.to_sparse()], {}), ([t], dict(out=[e.cpu()]))):
        with pytest.raises(ops.CdssmError):
            ops.clip_grads_(grads, 1.0, **kw)
    for bound in (-1.0, math.nan):
        with pytest.raises(ops.CdssmError):
            ops.clip_grads_([t], bound)
    assert float(ops.grad_norm([t, t])) == pytest.approx(math.sqrt(2) * _exact([t]), rel=6 * U)      # reading twice is no conflict
