"""The ends of a training step together with the operators between them: embedding, short convolution, loss against the embedding's own table,
gradients, clipping, in the order in which cdssm/training/trainer.py:219-262 runs them; against the same step in 64 bits."""
import pytest
import torch
import torch.nn.functional as F

from util import BF16_TOL, FP32_TOL, rel_err, to_np

pytestmark = pytest.mark.gpu


class Step(torch.nn.Module):
    def __init__(self, V, d, dtype):
        super().__init__()
        g = torch.Generator(device="cuda").manual_seed(3)
        rn = lambda *s: torch.nn.Parameter((torch.randn(*s, generator=g, device="cuda") / s[-1] ** 0.5).to(dtype))  # noqa: E731
        self.table, self.conv_w, self.conv_b = rn(V, d), rn(d, 1, 4), rn(d)
        self.scale = d ** 0.5

    def forward(self, ops, ids, targets):
        x = ops.embedding(ids, self.table, scale=self.scale, padding_idx=0)
        h = ops.CUDAConv1dSiLUOp.apply(x, self.conv_w, self.conv_b)
        return ops.linear_cross_entropy(h, self.table, targets)

    def exact(self, ids, targets):
        p = {n: q.detach().double().requires_grad_() for n, q in self.named_parameters()}
        x = F.embedding(ids, p["table"], padding_idx=0) * self.scale
        h = F.silu(F.conv1d(F.pad(x.transpose(1, 2), (3, 0)), p["conv_w"], p["conv_b"], groups=x.shape[-1])).transpose(1, 2)
        z = h @ p["table"].t()
        loss = F.cross_entropy(z.reshape(-1, z.shape[-1]), targets.reshape(-1))
        return loss, dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def _batch(V, seed, B=3, L=41):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, V, (B, L), generator=g, device="cuda")
    ids[:, L - 5:] = 0                                      # padding: no gradient of its row's embedding, no targets
    targets = torch.roll(ids, -1, 1)
    targets[:, L - 6:] = -100
    return ids, targets


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_step(ops, dtype):
    V, d = 611, 96
    tol = BF16_TOL if dtype == torch.bfloat16 else FP32_TOL
    m = Step(V, d, dtype)
    for seed in range(2):
        ids, targets = _batch(V, seed)
        want, grads = m.exact(ids, targets)
        m.zero_grad()
        loss = m(ops, ids, targets)
        loss.backward()
        assert rel_err(loss.item(), want.item()) <= tol
        norm = torch.cat([g.reshape(-1) for g in grads.values()]).norm()
        for bound in (10 * norm, 0.1 * norm):              # within it, then beyond
            got = ops.clip_grad_norm_(m.parameters(), float(bound))
            assert rel_err(got.item(), norm.item()) <= tol
            c = min(1.0, float(bound / norm))
            for n, p in m.named_parameters():
                assert rel_err(to_np(p.grad), (grads[n] * c).cpu().numpy()) <= tol, n


def test_captured_step(ops):
    """Forward, backward and clipping as one graph, replayed on new batches."""
    V, d = 611, 96
    m = Step(V, d, torch.float32)
    params = list(m.parameters())
    ids, targets = _batch(V, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        loss = m(ops, ids, targets)
        grads = torch.autograd.grad(loss, params)
        return loss.detach(), ops.clip_grads_(grads, 0.05), grads

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss, norm, grads = step()
    for seed in (1, 2):
        new = _batch(V, seed)
        ids.copy_(new[0]), targets.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        w_loss, w = m.exact(*new)
        w_norm = torch.cat([g.reshape(-1) for g in w.values()]).norm()
        assert rel_err(loss.item(), w_loss.item()) <= FP32_TOL and rel_err(norm.item(), w_norm.item()) <= FP32_TOL
        c = min(1.0, 0.05 / float(w_norm))
        for g, n in zip(grads, w):
            assert rel_err(to_np(g), (w[n] * c).cpu().numpy()) <= FP32_TOL
