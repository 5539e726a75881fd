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
