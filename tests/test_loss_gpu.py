"""The loss of hidden rows against a vocabulary (ops.linear_cross_entropy), forward and backward, against its formula in 64 bits.

Tolerances.  Operands are exact in the products; sums are float32.  With u = 2^-24:
  loss rows, bf16 and float32: a logit is a sum of K products in float32 in any order, cut off instead of rounded (2 u a step): off by at most
      2 K u sum |x w|, and by four times that for the six part products of float32 operands; the loss is off by at most two of those and the
      roundings of exp, sum and log (16 u of 1 + |loss| + |z|).
  gradients: dz is off by the logits' error times itself and one rounding to bf16 (2^-8 of itself; none to speak of for float32, whose
      three parts keep 24 bits), the sums by their length times u, the result by its own rounding.  All of them are bounded
      entry by entry from the absolute values of what is summed, and doubled: with an upstream gradient a row, x is rounded with it to its two parts' 16 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _inputs(T, V, d, dtype, seed=0, ignored=0.2, sure=8.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, d, generator=g, device="cuda") / d ** 0.5
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    x = torch.randn(T, d, generator=g, device="cuda") + sure * torch.rand(T, 1, generator=g, device="cuda") * w[y]
    y = torch.where(torch.rand(T, generator=g, device="cuda") < ignored, -100, y)
    return x.to(dtype), w.to(dtype), y


def _exact(x, w, y, g):
    """loss rows, dx, dw and, entry by entry, how far off each may be (in 64 bits); g: upstream gradient a row."""
    f32 = x.dtype == torch.float32
    x, w, g = x.double(), w.double(), g.double()
    K = x.shape[1]
    on = y != -100
    x = torch.where(on[:, None], x, 0.0)
    z = x @ w.T
    dz_off = K * 8 * U * (x.abs() @ w.abs().T) + 8 * U            # six part products of a float32 one: as many sums again
    logp = torch.log_softmax(z, -1)
    pick = y.clamp(min=0)[:, None]
    rows = torch.where(on, -logp.gather(1, pick)[:, 0], 0.0)
    rows_off = 2 * dz_off.amax(-1) + 16 * U * (1 + rows.abs() + z.abs().amax(-1))
    p = logp.exp()
    hot = torch.zeros_like(p).scatter_(1, pick, 1.0)
    g = torch.where(on, g, 0.0)[:, None]
    dz = g * (p - hot)
    off = g.abs() * (p * (2 * dz_off + 16 * U) + hot * 4 * U + p * 2 * dz_off.amax(-1, keepdim=True)) + dz.abs() * (2.0 ** -23 if f32 else 2.0 ** -8)
    out = 2.0 ** -24 if f32 else 2.0 ** -8
    T, V = z.shape
    dx, dw = dz @ w, dz.T @ x
    dx_off = off @ w.abs() + 8 * V * U * (dz.abs() @ w.abs()) + out * dx.abs()
    dw_off = off.T @ x.abs() + 8 * T * U * (dz.abs().T @ x.abs()) + out * dw.abs()
    return (rows, dx, dw), (rows_off, 2 * dx_off + 1e-30, 2 * dw_off + 1e-30)


def _check(got, want, off, what):
    bad = (got.double() - want).abs() > off
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(got.double() - want).abs().max():.3e}"
    assert torch.isfinite(got).all()


SHAPES = [(1, 1, 1), (1, 50257, 768), (3, 7, 5), (61, 503, 100), (128, 256, 64), (129, 257, 65), (300, 1000, 256), (523, 8191, 768), (777, 2049, 520),
          (2048, 1024, 128), (5, 9000, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,d", SHAPES)
def test_loss_and_gradients(ops, T, V, d, dtype):
    x, w, y = _inputs(T, V, d, dtype, seed=T + V + d)
    y[0] = V - 1                                                     # at least one row, and the last word
    g = torch.randn(T, device="cuda")
    want, off = _exact(x, w, y, g)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y, reduction="none")
    assert loss.dtype == torch.float32 and loss.shape == y.shape
    _check(loss.detach(), want[0], off[0], "loss")
    gx, gw = torch.autograd.grad(loss, [x, w], [g])
    assert gx.dtype == dtype and gw.dtype == dtype and gx.shape == x.shape and gw.shape == w.shape
    _check(gx, want[1], off[1], "grad of hidden")
    _check(gw, want[2], off[2], "grad of weight")
    assert (gx[y == -100] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reductions(ops, dtype, reduction):
    T, V, d = 700, 1100, 96
    x, w, y = _inputs(T, V, d, dtype, seed=3)
    n = (y != -100).sum()
    g = torch.full((T,), 1.7, device="cuda", dtype=torch.float64) / (n if reduction == "mean" else 1)
    want, off = _exact(x, w, y, g)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x.view(7, 100, d), w, y.view(7, 100), reduction=reduction)
    total = want[0].sum() / (n if reduction == "mean" else 1)
    assert loss.shape == () and abs(loss.double() - total) <= off[0].sum() / (n if reduction == "mean" else 1) + U * total
    gx, gw = torch.autograd.grad(loss * 1.7, [x, w])
    _check(gx, want[1], off[1] + 4 * U * want[1].abs(), "grad of hidden")
    _check(gw, want[2], off[2] + 4 * U * want[2].abs(), "grad of weight")


def _grads(ops, x, w, y, g, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, [x, w], [g]))


def test_pieces_of_the_vocabulary(ops):
    """So many rows that the logits' gradient is formed in two pieces."""
    T, V, d = 65600, 8191, 40
    x, w, y = _inputs(T, V, d, torch.bfloat16, seed=9)
    g = torch.randn(T, device="cuda")
    want, off = _exact(x, w, y, g)
    got = _grads(ops, x, w, y, g, reduction="none")
    for name, a, b, c in zip(("loss", "grad of hidden", "grad of weight"), got, want, off):
        _check(a, b, c, name)
    assert all(torch.equal(a, b) for a, b in zip(got, _grads(ops, x, w, y, g, reduction="none")))   # run to run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 72, 77])
def test_operands_anywhere(ops, dtype, d):
    """Column slices, rows of other strides, transposes, odd addresses, one row for all."""
    T, V = 150, 300
    g = torch.randn(T, device="cuda")
    x, w, y = _inputs(T, V, d, dtype, seed=d)
    want = _grads(ops, x, w, y, g, reduction="none")
    wide = lambda t, o: torch.cat([torch.full_like(t, float("nan"))[:, :o], t, torch.full_like(t, float("nan"))[:, :5]], 1)[:, o:o + d]  # noqa: E731
    column = lambda t: t.t().contiguous().t()  # noqa: E731
    for xs in (x, wide(x, 8), wide(x, 3), column(x)):
        for ws in (w, wide(w, 8), wide(w, 1), column(w)):
            assert all(torch.equal(a, b) for a, b in zip(_grads(ops, xs, ws, y, g, reduction="none"), want))
    strided = torch.stack([y, torch.zeros_like(y)], 1)[:, 0]
    assert torch.equal(_grads(ops, x, w, strided, g, reduction="none")[2], want[2])
    one = _grads(ops, x[:1].expand(T, d), w, y, g, reduction="none")[0]
    assert torch.equal(one, ops.linear_cross_entropy(x[:1].repeat(T, 1), w, y, reduction="none"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_target(ops, dtype):
    T, V, d = 600, 777, 128
    x, w, y = _inputs(T, V, d, dtype, seed=5, ignored=0.4)
    g = torch.randn(T, device="cuda")
    want = _grads(ops, x, w, y, g, reduction="none")
    gone = y == -100
    bad = torch.where(gone[:, None], torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").repeat(d // 4), x.float()).to(dtype)
    got = _grads(ops, bad, w, y, torch.where(gone, float("nan"), g), reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got[0][gone] == 0).all() and (got[1][gone] == 0).all()
    # the other kind of ignored rows: a word
    y0 = torch.where(gone, 7, y)
    assert not (y == 7).any() or torch.equal(y0 == 7, gone | (y == 7))
    y0 = torch.where((y == 7) & ~gone, 8, y0)
    a = _grads(ops, bad, w, y0, g, reduction="none", ignore_index=7)
    b = _grads(ops, bad, w, torch.where(gone, -100, y0), g, reduction="none")
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # none left
    none = torch.full_like(y, -100)
    one = torch.ones((), device="cuda")
    for reduction, value in (("mean", float("nan")), ("sum", 0.0)):
        loss, gx, gw = _grads(ops, bad, w, none, one, reduction=reduction)
        assert torch.equal(loss.nan_to_num(-1.0), torch.tensor(value, device="cuda").nan_to_num(-1.0))
        assert (gx == 0).all() and (gw == 0).all()
    assert (ops.linear_cross_entropy(bad, w, none, reduction="none") == 0).all()


def test_no_rows(ops):
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    x, y = torch.randn(3, 0, 16, device="cuda", requires_grad=True), torch.zeros(3, 0, dtype=torch.int64, device="cuda")
    assert ops.linear_cross_entropy(x, w, y, reduction="none").shape == (3, 0)
    assert float(ops.linear_cross_entropy(x, w, y, reduction="sum").detach()) == 0.0 and ops.linear_cross_entropy(x, w, y).isnan()
    gx, gw = torch.autograd.grad(ops.linear_cross_entropy(x, w, y, reduction="sum"), [x, w])
    assert gx.shape == x.shape and (gw == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_that_are_no_numbers(ops, dtype):
    """A target that is no word, and rows with infinities or NaN, spoil their own loss."""
    T, V, d = 40, 300, 64
    x, w, y = _inputs(T, V, d, dtype, seed=6, ignored=0.0)
    want = ops.linear_cross_entropy(x, w, y, reduction="none")
    y2, x2 = y.clone(), x.clone()
    y2[3], y2[4], y2[5] = V, -1, 2 ** 40
    x2[7, 0], x2[8, 1] = float("nan"), float("inf")
    got = ops.linear_cross_entropy(x2, w, y2, reduction="none")
    spoilt = torch.zeros(T, dtype=torch.bool, device="cuda")
    spoilt[[3, 4, 5, 7, 8]] = True
    assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], want[~spoilt])
    loss, gx, gw = _grads(ops, x, w, y2, torch.ones((), device="cuda"), reduction="sum")
    assert loss.isnan() and gx[3:6].isnan().all() and gx[6:].isfinite().all() and gw.isnan().all()


def test_large_logits(ops):
    """Logits of thousands: the maximum is taken off before anything is an exponent."""
    T, V, d = 64, 512, 64
    x, w, y = _inputs(T, V, d, torch.float32, seed=7)
    x, w = 300 * x, 10 * w
    want, off = _exact(x, w, y, torch.ones(T, device="cuda"))
    got = _grads(ops, x, w, y, torch.ones(T, device="cuda"), reduction="none")
    for name, a, b, c in zip(("loss", "grad of hidden", "grad of weight"), got, want, off):
        _check(a, b, c, name)


def test_one_operand_trained(ops):
    """The other operand's gradient is not formed.  Which tiles a launch has decides where long sums are cut, so the bits are not those of
    both together, but either sum is one of the same terms in float32 in some order: the bound of _exact() holds for any."""
    T, V, d = 333, 1500, 256
    x, w, y = _inputs(T, V, d, torch.bfloat16, seed=8)
    want, off = _exact(x, w, y, torch.full((T,), 1.0, device="cuda", dtype=torch.float64) / (y != -100).sum())
    gx, = torch.autograd.grad(ops.linear_cross_entropy(x.requires_grad_(), w, y), [x])
    gw, = torch.autograd.grad(ops.linear_cross_entropy(x.detach(), w.requires_grad_(), y), [w])
    _check(gx, want[1], off[1] + 4 * U * want[1].abs(), "grad of hidden")
    _check(gw, want[2], off[2] + 4 * U * want[2].abs(), "grad of weight")


def test_gradient_against_differences(ops):
    """Along a direction a of the logits the third derivative of a row's loss is a third cumulant of a: at most R^3 / (6 sqrt 3) for the
    range R of a, so a central difference of step h is off by h^2 / 6 of that, and by the losses' own errors over h."""
    T, V, d, h = 90, 400, 48, 0.02
    x, w, y = _inputs(T, V, d, torch.float32, seed=10)
    gen = torch.Generator(device="cuda").manual_seed(1)
    dx, dw = torch.randn(T, d, generator=gen, device="cuda") / d ** 0.5, torch.randn(V, d, generator=gen, device="cuda") / d ** 0.5
    g = torch.randn(T, generator=gen, device="cuda")
    _, gx, gw = _grads(ops, x, w, y, g, reduction="none")
    for a, b, grad in ((dx, 0 * dw, gx), (0 * dx, dw, gw)):
        up, down = (ops.linear_cross_entropy(x + s * a, w + s * b, y, reduction="none").double() for s in (h, -h))
        rows = (up - down) / (2 * h) * g
        along = x.double() @ b.double().T + a.double() @ w.double().T
        R = along.amax(-1) - along.amin(-1)
        off = max(_exact(x + s * a, w + s * b, y, g)[1][0].max() for s in (h, -h))
        step = 2 * U * ((x.abs() + h * a.abs()) @ w.abs().T + x.abs() @ (w.abs() + h * b.abs()).T).max() / h    # the shifted operands' own rounding
        tol = (g.abs() * (h * h / 6 * R ** 3 / (6 * 3 ** 0.5) + off / h + step)).sum()
        assert abs(float(rows.sum() - (grad.double() * (a + 0).double()).sum() if b.abs().max() == 0 else rows.sum() - (grad.double() * b.double()).sum())) <= tol


def test_another_stream_and_captured(ops):
    T, V, d = 500, 3000, 128
    x, w, y = _inputs(T, V, d, torch.bfloat16, seed=11)
    one = torch.ones((), device="cuda")
    want = _grads(ops, x, w, y, one)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _grads(ops, x, w, y, one)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two captured steps of one pool, replayed in turn with new inputs in place
    xs, ys = [torch.zeros_like(x) for _ in range(2)], [torch.zeros_like(y) for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        with torch.cuda.stream(side):
            _grads(ops, xs[i], w, ys[i], one)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, pool=graphs[0].pool() if graphs else None):
            outs.append(_grads(ops, xs[i], w, ys[i], one))
        graphs.append(graph)
    for seed in (12, 13):
        for i in range(2):
            x2, _, y2 = _inputs(T, V, d, torch.bfloat16, seed=seed + 7 * i, ignored=0.1 * seed - 1)
            xs[i].copy_(x2), ys[i].copy_(y2)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], _grads(ops, x2, w, y2, one)))


def test_two_calls_at_once(ops):
    """Two streams, each with buffers of its own."""
    sets = [_inputs(900, 2000, 64, torch.bfloat16, seed=s) for s in (20, 21)]
    one = torch.ones((), device="cuda")
    want = [_grads(ops, *s, one) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_grads(ops, *sets[i], one))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for r in got[i] for a, b in zip(r, want[i]))


@pytest.mark.parametrize("T,d,dtype", [(300, 96, torch.bfloat16), (20, 96, torch.bfloat16), (20, 1000, torch.bfloat16), (300, 1000, torch.bfloat16),
                                       (300, 96, torch.float32), (20, 96, torch.float32)])
def test_waits_run_out_and_the_next_call_is_right(ops, T, d, dtype):
    """The products' loads are withheld, in pairs of blocks and blocks by themselves, with sums in one piece and folded: every wait ends, the loss
    says so, and nothing stays behind."""
    V = 700
    x, w, y = _inputs(T, V, d, dtype, seed=14)
    one = torch.ones((), device="cuda")
    want = _grads(ops, x, w, y, one)
    old = ops.set_wait_limit_ns(2_000_000)
    try:
        assert ops.linear_cross_entropy(x, w, y, flags=ops.TEST_WITHHOLD).isnan()
        loss, gx, gw = _grads(ops, x, w, y, one, flags=ops.TEST_WITHHOLD)
        assert loss.isnan() and gx.isnan().all() and gw.isnan().all()
        torch.cuda.synchronize()
    finally:
        ops.set_wait_limit_ns(old)
    assert all(torch.equal(a, b) for a, b in zip(_grads(ops, x, w, y, one), want))


def test_refusals(ops):
    x, w, y = _inputs(20, 30, 16, torch.bfloat16)
    bad = [(x.cpu(), w, y, {}), (x, w.cpu(), y, {}), (x, w, y.cpu(), {}), (x.float(), w, y, {}), (x.half(), w.half(), y, {}), (x, w, y.int(), {}),
           (x, w[:, :8], y, {}), (x, w, y[:10], {}), (x, w[0], y, {}), (x, w[:0], y, {}), (x, w, y, dict(reduction="batch")), (x.view(2, 10, 16), w, y, {})]
    for a, b, c, kw in bad:
        with pytest.raises(ops.CdssmError):
            ops.linear_cross_entropy(a, b, c, **kw)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ops.linear_cross_entropy(x, w, y), [x], create_graph=True)
    loss = ops.linear_cross_entropy(x, w.requires_grad_(), y)
    with torch.no_grad():
        w += 1.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, [x])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_model_loss(ops, dtype):
    """The LM's loss against the cross entropy of its logits: these are rounded to the type, so off by its half step of themselves."""
    from cdssm_b200.model import CdssmConfig, CdssmLM
    lm = CdssmLM(CdssmConfig(d_model=256, n_layers=2, context_length=1024, vocab_size=503, state_dim=4), dtype=dtype, seed=5)
    ids = torch.randint(0, 503, (3, 70), generator=torch.Generator().manual_seed(2)).cuda()
    z = lm.forward(ids).double()
    rows = torch.nn.functional.cross_entropy(z[:, :-1].reshape(-1, 503), ids[:, 1:].reshape(-1), reduction="none").view(3, 69)
    tol = 2 * (2.0 ** -8 if dtype == torch.bfloat16 else 1e-5) * float(z.abs().max())
    got = lm.loss(ids, reduction="none")
    assert got.shape == (3, 70) and (got[:, -1] == 0).all() and (got[:, :-1].double() - rows).abs().max() <= tol
    assert abs(float(lm.loss(ids)) - float(rows.mean())) <= tol
    assert torch.equal(lm.loss(ids, torch.roll(ids, -1, 1), reduction="none")[:, :-1], got[:, :-1])
    assert torch.equal(lm.loss(ids.cpu(), reduction="none"), got) and torch.equal(lm.loss(ids.tolist(), reduction="none"), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("seed", range(24))
def test_sizes_at_random(ops, dtype, seed):
    """Sizes whose tiles go round the blocks evenly, with one left over, or with fewer tiles than blocks; rows all, some or hardly any."""
    r = __import__("random").Random(1000 + seed)
    size = lambda most: max(1, int(most ** r.random() + r.randint(-1, 1)))  # noqa: E731
    T, V, d = size(1500), size(30000), size(900)
    x, w, y = _inputs(T, V, d, dtype, seed=seed, ignored=r.choice([0.0, 0.3, 0.9]), sure=r.choice([0.0, 8.0, 30.0]))
    y[T // 2] = 0
    reduction = r.choice(["none", "mean", "sum"])
    g = torch.randn(T, device="cuda") if reduction == "none" else torch.randn((), device="cuda")
    rows = g.double() if reduction == "none" else (g.double() / ((y != -100).sum() if reduction == "mean" else 1)).expand(T)
    want, off = _exact(x, w, y, rows)
    got = _grads(ops, x, w, y, g, reduction=reduction)
    if reduction == "none":
        _check(got[0], want[0], off[0], "loss")
    else:
        n = (y != -100).sum() if reduction == "mean" else 1
        assert abs(got[0].double() - want[0].sum() / n) <= (off[0].sum() + U * want[0].sum()) / n
    _check(got[1], want[1], off[1] + 4 * U * want[1].abs(), f"grad of hidden {T} {V} {d}")
    _check(got[2], want[2], off[2] + 4 * U * want[2].abs(), f"grad of weight {T} {V} {d}")


def test_one_row_without_a_batch_and_a_graph_kept(ops):
    """hidden (d,) with a target (); backward twice from one forward; memory filled beforehand as deterministic runs have it."""
    x, w, y = _inputs(1, 90, 33, torch.float32, seed=30, ignored=0.0)
    want = _grads(ops, x, w, y, torch.ones(1, device="cuda"), reduction="none")
    xs, ws = x[0].clone().requires_grad_(), w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(xs, ws, y[0], reduction="none")
    assert loss.shape == () and torch.equal(loss.detach(), want[0][0])
    for _ in range(2):
        gx, gw = torch.autograd.grad(loss, [xs, ws], retain_graph=True)
        assert gx.shape == xs.shape and torch.equal(gx, want[1][0]) and torch.equal(gw, want[2])
    torch.use_deterministic_algorithms(True)
    try:
        x, w, y = _inputs(700, 900, 200, torch.bfloat16, seed=31)
        a = _grads(ops, x, w, y, torch.ones((), device="cuda"))
    finally:
        torch.use_deterministic_algorithms(False)
    assert all(torch.equal(p, q) for p, q in zip(a, _grads(ops, x, w, y, torch.ones((), device="cuda"))))
