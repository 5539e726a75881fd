"""The loss's gradients where the logits' gradient is formed a piece of the vocabulary at a time: dx is summed over the pieces in float32 and rounded by
the last, dW's rows begin at a piece's offset.  16 384 float32 rows leave room for 5376 words at a time: 8191 words are pieces of 4096 and 4095;
65 600 bfloat16 rows for 3840: pieces of 2816, 2816 and 2559."""
import pytest
import torch

from test_loss_gpu import U, _check, _exact, _grads, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("T,d,dtype", [(16384, 40, torch.float32), (16384, 272, torch.float32), (65600, 40, torch.bfloat16), (65600, 272, torch.bfloat16)])
def test_pieces(ops, T, d, dtype, reduction):
    V = 8191
    x, w, y = _inputs(T, V, d, dtype, seed=60 + d)
    g = torch.randn(T if reduction == "none" else (), device="cuda")
    n = (y != -100).sum() if reduction == "mean" else 1
    want, off = _exact(x, w, y, (g.double() / n).expand(T))
    got = _grads(ops, x, w, y, g, reduction=reduction)
    if reduction == "none":
        _check(got[0], want[0], off[0], "loss")
    else:
        assert abs(got[0].double() - want[0].sum() / n) <= (off[0].sum() + U * want[0].sum()) / n
    for name, a, b, c in zip(("grad of hidden", "grad of weight"), got[1:], want[1:], off[1:]):
        _check(a, b, c + 4 * U * b.abs(), name)
    assert (got[1][y == -100] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip(got, _grads(ops, x, w, y, g, reduction=reduction)))
