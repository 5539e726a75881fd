"""The loss of hidden rows against a vocabulary (ops.linear_cross_entropy), forward and backward, against its formula in 64 bits.

Tolerances.  Operands are exact in the products; sums are float32.  With u = 2^-24:
  loss rows, bf16 and float32: a logit is a sum of K products in float32 in any order, off by at most K u sum |x w|; the loss is
      off by at most two of those and the roundings of exp, sum and log (8 u of 1 + |loss|).
  gradients: dz is off by the logits' error times itself and one rounding to bf16 (2^-8 of itself; none to speak of for float32, whose
      three parts keep 24 bits), the sums by their length times u, the result by its own rounding.  All of them are bounded
      entry by entry from the absolute values of what is summed."""
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
