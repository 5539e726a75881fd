"""How many bits the loss keeps and where: sums that are cut off, logits' gradients in one, two and three parts, upstream gradients.

The cases are made so that all but one source of error is nothing: with x or W zero every logit is 0 and the probabilities of 2^k words are
2^-k, exact in any of the types, as are the targets' 2^-k - 1 for k <= 8.  What is left is summed here in 64 bits."""
import pytest
import torch

from test_loss_gpu import _grads

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _half_step(t):
    """Half the distance of t's neighbours in bfloat16: of m 2^E with m in [1/2, 1) it is 2^(E - 9)."""
    return torch.ldexp(torch.ones_like(t), torch.frexp(t)[1] - 9)


def _positive(n, d, gen):
    """Values over three decades, bfloat16: their sums have more digits than float32 holds."""
    return torch.rand(n, d, generator=gen, device="cuda").mul_(-8).exp_().bfloat16()


# Long sums of one sign.  A cut-off costs at most 2^-23 of the running sum every 16 terms; folds of 1024 terms (two parts of x g: of twice as many
# products) are off by 128 of these, 1.6e-5; up to 1024 folds and parts of tiles are added up and rounded, 2^-24 of the sum each at most and in
# either direction: 6.1e-5 in the worst case; the two parts of x g hold 16 bits, 1.6e-5.  Their sum is 9.3e-5.  Unfolded, the sums
# here lose 1.4e-4 (the rows of dx) to 7e-4 (dW, in shares of 262 144 rows).
LONG = 128 * 2.0 ** -23 + 1024 * U + 2.0 ** -16


@pytest.mark.parametrize("T", [16385, 262144])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_long_sums_over_rows(ops, reduction, T):
    V, d = 1024, 4096
    gen = torch.Generator(device="cuda").manual_seed(50)
    x, w, y = _positive(T, d, gen), torch.zeros(V, d, device="cuda", dtype=torch.bfloat16), torch.zeros(T, dtype=torch.int64, device="cuda")
    g = torch.rand(T, generator=gen, device="cuda") + 0.5 if reduction == "none" else torch.ones((), device="cuda")
    gw = _grads(ops, x, w, y, g, reduction=reduction)[2]
    total = sum((a.double() * b.double()).sum(0) for a, b in zip(x.split(8192), (g if reduction == "none" else g / T).expand(T)[:, None].split(8192))) / V
    off = (gw[1:].double() - total).abs()                                # (word 0 is every row's target; its 2^-10 - 1 is no bfloat16)
    assert (off <= _half_step(total) + (LONG + 4 * U) * total).all(), float((off / total).max())


@pytest.mark.parametrize("T", [20, 200])
def test_long_sums_over_words(ops, T):
    V, d = 262144, 4096
    gen = torch.Generator(device="cuda").manual_seed(51)
    w = _positive(V, d, gen)
    w[0] = 0                                                             # the target of every row
    x, y = torch.zeros(T, d, device="cuda", dtype=torch.bfloat16), torch.zeros(T, dtype=torch.int64, device="cuda")
    gx = _grads(ops, x, w, y, torch.ones((), device="cuda"), reduction="sum")[1]
    total = sum(a.double().sum(0) for a in w.split(8192)) / V
    off = (gx.double() - total).abs()
    assert (off <= _half_step(total) + (LONG + 4 * U) * total).all(), float((off / total).max())


def _exact_logits(kind, T, V, d, gen):
    """Operands whose logits are all 0: x = 0 shows dx, W = 0 shows dW."""
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()  # noqa: E731
    x, w = (rn(T, d), torch.zeros(V, d, device="cuda", dtype=torch.bfloat16)) if kind == "dw" else (torch.zeros(T, d, device="cuda", dtype=torch.bfloat16), rn(V, d))
    y = torch.randint(0, V, (T,), generator=gen, device="cuda")
    y[::7] = -100
    return x, w, y


@pytest.mark.parametrize("T", [100, 300])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("kind", ["dx", "dw"])
def test_upstream_gradients_keep_their_bits(ops, kind, reduction, T):
    """Of 256 words p - [v = y] is 2^-8 or 2^-8 - 1, exact.  A common upstream gradient is then a float32 factor of the sums; one a row keeps 16 bits
    (2^-16), as a factor of dz (up to 128 rows) or of x.  Sums of n values: 2 U each of what is summed."""
    V, d = 256, 96
    gen = torch.Generator(device="cuda").manual_seed(52)
    x, w, y = _exact_logits(kind, T, V, d, gen)
    g = torch.randn(T if reduction == "none" else (), generator=gen, device="cuda")
    got = _grads(ops, x, w, y, g, reduction=reduction)[1 if kind == "dx" else 2]
    on = (y != -100).double()
    dz = torch.full((T, V), 1.0 / V, device="cuda", dtype=torch.float64)
    dz.scatter_add_(1, y.clamp(min=0)[:, None], -on[:, None])
    dz *= (g.double() / (on.sum() if reduction == "mean" else 1) * on).expand(T)[:, None]
    a, b = (dz, w.double()) if kind == "dx" else (dz.t(), x.double())
    want, size = a @ b, a.abs() @ b.abs()
    off = _half_step(want) + ((2.0 ** -16 if reduction == "none" else 0.0) + (2 * a.shape[1] + 8) * U) * size
    assert ((got.double() - want).abs() <= off).all(), float(((got.double() - want).abs() / off).max())


@pytest.mark.parametrize("T", [1, 100, 128])
def test_few_rows_keep_sixteen_bits_of_the_logits_gradient(ops, T):
    """Where the target's entry is nearly all of a row its rounding to 8 bits would be the gradient's: 2^-9 of it beside the result's own rounding.
    Width 16 is one step of the tensor cores: a logit is off by 16 terms' cut-offs, 2 U each, and dz by twice that and the exponential's 16 U."""
    V, d = 512, 16
    gen = torch.Generator(device="cuda").manual_seed(53)
    w = torch.randn(V, d, generator=gen, device="cuda").bfloat16()
    y = torch.randint(0, V, (T,), generator=gen, device="cuda")
    x = (torch.randn(T, d, generator=gen, device="cuda") * 0.1 + torch.rand(T, 1, generator=gen, device="cuda") * w[y] * (12 / d)).bfloat16()
    _, gx, gw = _grads(ops, x, w, y, torch.ones((), device="cuda"), reduction="sum")
    x, w = x.double(), w.double()
    p = torch.softmax(x @ w.t(), -1)
    dz = p.scatter_add(1, y[:, None], torch.full((T, 1), -1.0, device="cuda", dtype=torch.float64))
    z_off = (2 * d * U * (x.abs() @ w.abs().t())).amax(-1, keepdim=True)
    dz_off = p * (2 * z_off + 16 * U) + dz.abs() * 2.0 ** -16 + 4 * U * (dz < 0)
    for got, a, a_off, b in ((gx, dz, dz_off, w), (gw, dz.t(), dz_off.t(), x)):
        want = a @ b
        off = _half_step(want) + a_off @ b.abs() + 2 * a.shape[1] * U * (a.abs() @ b.abs())
        assert ((got.double() - want).abs() <= off).all(), float(((got.double() - want).abs() / off).max())


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("dtype,fold", [(torch.bfloat16, 768), (torch.float32, 256)])
def test_long_logits_are_folded(ops, dtype, fold, T):
    """One word's logit is a sum of 32 768 positive terms, the others' are 0, and so is the target's: the loss is that sum.  A fold is off by 2^-23 of
    itself every 16 terms, their sum by 2^-24 a fold; in one piece it would be 6e-5."""
    V, d = 3, 32768
    gen = torch.Generator(device="cuda").manual_seed(54)
    x, w = _positive(T, d, gen).to(dtype), torch.zeros(V, d, device="cuda", dtype=dtype)
    if dtype == torch.float32:
        x = x * (1 + torch.rand(T, d, generator=gen, device="cuda") * 2.0 ** -8)
    w[0] = _positive(1, d, gen)[0].to(dtype)
    loss = ops.linear_cross_entropy(x, w, torch.ones(T, dtype=torch.int64, device="cuda"), reduction="none")
    want = x.double() @ w[0].double()                                   # (above 100: log(1 + 2 exp(-z)) is nothing)
    assert want.min() > 100
    assert ((loss.double() - want).abs() <= (fold // 16 * 2.0 ** -23 + d // fold * U + 4 * U) * want).all(), float(((loss.double() - want) / want).abs().max())


def test_float32_gradients_over_a_vocabulary(ops):
    """Against float32's own 6e-8: logits of a size of 1 and folds of 256 terms are off by 16 cut-offs, 1.9e-6 at most and half of that on
    average, the gradient's sums over 50 257 words by as much: 3e-6 of the whole.  (Unfolded, 1e-5 to 5e-5.)"""
    T, V, d = 1024, 50257, 768
    gen = torch.Generator(device="cuda").manual_seed(55)
    x, w = torch.randn(T, d, generator=gen, device="cuda"), torch.randn(V, d, generator=gen, device="cuda") / d ** 0.5
    y = torch.randint(0, V, (T,), generator=gen, device="cuda")
    _, gx, gw = _grads(ops, x, w, y, torch.ones((), device="cuda"), reduction="sum")
    dz = torch.softmax(x.double() @ w.double().t(), -1)
    dz.scatter_add_(1, y[:, None], torch.full((T, 1), -1.0, device="cuda", dtype=torch.float64))
    for got, want in ((gx, dz @ w.double()), (gw, dz.t() @ x.double())):
        assert (got.double() - want).norm() <= 3e-6 * want.norm(), float((got.double() - want).norm() / want.norm())
