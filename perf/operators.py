"""The operators at the ends of a training step, as they are timed: plain forms and the framework's calls.

``listed()`` names the fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes what a
user's program holds before the call, ``run(state)`` is one pass, ``work(case)`` the bytes and operations that no
implementation can do without, ``exact(case, seed)`` the results from the definitions in 64 bits.

Kinds:
  loss   softmax cross entropy of hidden rows against a vocabulary: the loss, and in training its two gradients
  embed  rows of a table for token ids, scaled; in training the table's gradient too
  clip   the norm of all gradients together, and the gradients scaled down to a bound
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
IGNORE = -100


def listed():
    return [
        # log-likelihoods of one short completion, token by token: the weight's bytes and the call's latency
        dict(name="loss_score", kind="loss", T=61, V=50257, d=768, dtype="bf16", train=False, reduction="none", ignored=0.0),
        # perplexity of an evaluation batch by document, 8 x 2048 tokens of the 32 000-word model
        dict(name="loss_eval", kind="loss", T=16384, V=32000, d=768, dtype="bf16", train=False, reduction="none", ignored=0.0),
        # a training step's loss on a padded batch with the default vocabulary
        dict(name="loss_train", kind="loss", T=16384, V=50257, d=768, dtype="bf16", train=True, reduction="mean", ignored=0.125),
        # the same end of the 2048-wide model
        dict(name="loss_train_wide", kind="loss", T=4096, V=32000, d=2048, dtype="bf16", train=True, reduction="mean", ignored=0.0),
        # full precision, an odd number of tokens
        dict(name="loss_train_f32", kind="loss", T=1531, V=50257, d=768, dtype="f32", train=True, reduction="mean", ignored=0.1),
        # the next token of a handful of streams: latency
        dict(name="embed_step", kind="embed", T=16, V=50257, d=768, dtype="bf16", train=False, scaled=False),
        # one ragged document of a fine-tuning run
        dict(name="embed_document", kind="embed", T=523, V=32000, d=768, dtype="bf16", train=True, scaled=False),
        # a training batch of 8 x 2048 tokens
        dict(name="embed_train", kind="embed", T=16384, V=50257, d=768, dtype="bf16", train=True, scaled=False),
        # a large batch of the 2048-wide model in full precision, rows scaled by sqrt(d)
        dict(name="embed_train_f32", kind="embed", T=32768, V=32000, d=2048, dtype="f32", train=True, scaled=True),
        # a two-layer model's gradients, below the bound: they stay as they are
        dict(name="clip_small", kind="clip", layers=2, d=256, N=4, V=503, dtype="f32", wide_out=False, over=False),
        # the 12-layer model's bf16 gradients into the optimizer's float32 buffers
        dict(name="clip_lm", kind="clip", layers=12, d=768, N=16, V=50257, dtype="bf16", wide_out=True, over=True),
        # a 24-layer model's float32 gradients, below the bound
        dict(name="clip_deep", kind="clip", layers=24, d=1024, N=16, V=50257, dtype="f32", wide_out=False, over=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


LOSS_MOST = 16384 * 50257 * 768        # tokens x vocabulary x width of loss_train
EMBED_MOST = (32768 + 32000) * 2048    # values read and written by embed_train_f32


def draw(rng):
    kind = rng.choice(["loss", "loss", "loss", "embed", "embed", "clip"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if kind == "loss":
        V, d = rng.choice([503, 1000, 8191, 32000, 50257]), rng.choice([100, 256, 512, 768, 768, 1024, 2048])
        most = LOSS_MOST // (V * d) // (8 if dtype == "f32" else 1)
        train = rng.random() < 0.6
        return dict(kind=kind, T=_log_int(rng, 1, max(1, min(16384, most))), V=V, d=d, dtype=dtype, train=train,
                    reduction=rng.choice(["mean", "mean", "sum", "none"]) if train else "none", ignored=rng.choice([0.0, 0.1, 0.5]))
    if kind == "embed":
        V, d = rng.choice([503, 1000, 8191, 32000, 50257]), rng.choice([100, 256, 512, 768, 1024, 2048])
        most = EMBED_MOST // d - V
        return dict(kind=kind, T=_log_int(rng, 1, max(1, min(65536, most))), V=V, d=d, dtype=dtype, train=rng.random() < 0.7,
                    scaled=rng.random() < 0.5)
    over = rng.random() < 0.5
    return dict(kind=kind, layers=rng.randint(1, 12), d=rng.choice([100, 128, 256, 512, 768]), N=rng.choice([2, 4, 16]),
                V=rng.choice([503, 1000, 8191, 32000]), dtype=dtype, wide_out=over and (dtype == "f32" or rng.random() < 0.5),
                over=over)


def _layer_shapes(d, N):
    """Weights of one block of the language model."""
    di = 2 * d
    H = max(1, di // 64)
    G = (N + 5) * H
    return [(d,), (3 * di + H * N, d), (3 * di + H * N,), (di, 1, 4), (di,), (G, di), (G,), (H,), (di, di), (di, H * N),
            (d, di), (di,), (di,), (di,), (H,)]


def _clip_groups(case):
    """Shapes by bucket: a layer's gradients lie in one buffer, as a data-parallel trainer keeps them; the table has its own."""
    return [_layer_shapes(case["d"], case["N"])] * case["layers"] + [[(case["V"], case["d"])], [(case["d"],)]]


def _views(flat, shapes):
    sizes = [math.prod(s) for s in shapes]
    return [v.view(s) for v, s in zip(flat.split(sizes), shapes)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if case["kind"] == "clip":
        s["grads"], s["flat"], s["out"], s["flat_out"] = [], [], [], []
        for i, shapes in enumerate(_clip_groups(case)):
            n = sum(math.prod(x) for x in shapes)
            flat = (randn(n) * (0.02 / (1 + i))).to(dtype)
            out = torch.empty(n, device="cuda", dtype=torch.float32 if case["wide_out"] else dtype) if case["over"] else flat
            s["flat"].append(flat)
            s["flat_out"].append(out)
            s["grads"] += _views(flat, shapes)
            s["out"] += _views(out, shapes)
        s["max_norm"] = 1.0 if case["over"] else 1e4
        return s
    T, V, d = case["T"], case["V"], case["d"]
    weight = randn(V, d) * (1.0 / math.sqrt(d))
    # words by Zipf's law: a few make up most of a text
    rank = torch.rand(T, generator=g, device="cuda", dtype=torch.float64).mul_(math.log(V)).exp_().long().sub_(1).clamp_(0, V - 1)
    words = torch.randperm(V, generator=g, device="cuda")[rank]
    if case["kind"] == "embed":
        s.update(weight=weight.to(dtype).requires_grad_(case["train"]), ids=words, scale=math.sqrt(d) if case["scaled"] else 1.0,
                 grad=randn(T, d).mul_(1e-2).to(dtype))
        return s
    # rows of a final norm that point to their word more or less: its probability goes from next to nothing to next to one
    sure = torch.rand(T, 1, generator=g, device="cuda")
    hidden = randn(T, d) + 16.0 * sure * weight[words]
    hidden = hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + 1e-6)
    targets = torch.where(torch.rand(T, generator=g, device="cuda") < case["ignored"], torch.full_like(words, IGNORE), words)
    s.update(hidden=hidden.to(dtype).requires_grad_(case["train"]), weight=weight.to(dtype).requires_grad_(case["train"]),
             targets=targets, grad=randn(T) if case["reduction"] == "none" else torch.ones((), device="cuda"))
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"loss": _plain_loss, "embed": _plain_embed, "clip": _plain_clip}[s["kind"]](s)


def _own(s):
    from cdssm_b200 import ops
    if s["kind"] == "clip":
        norm = ops.clip_grads_(s["grads"], s["max_norm"], out=s["out"] if s["over"] else None)
        return [norm] + s["flat_out"]
    if s["kind"] == "embed":
        out = ops.embedding(s["ids"], s["weight"], scale=s["scale"])
        if not s["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, [s["weight"]], [s["grad"]])]
    loss = ops.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], ignore_index=IGNORE, reduction=s["reduction"])
    if not s["train"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, [s["hidden"], s["weight"]], [s["grad"]])]


def _plain_loss(s):
    x, w, y = s["hidden"].float(), s["weight"].float(), s["targets"]
    valid = y != IGNORE
    z = x @ w.T
    top = z.amax(-1, keepdim=True)
    hit = z.gather(1, y.clamp(min=0)[:, None])[:, 0]
    p = torch.exp(z.sub_(top), out=z)
    total = p.sum(-1)
    rows = torch.where(valid, top[:, 0] + total.log() - hit, 0.0)
    count = valid.sum()
    loss = rows if s["reduction"] == "none" else rows.sum() if s["reduction"] == "sum" else rows.sum() / count
    if not s["train"]:
        return [loss]
    g = torch.where(valid, s["grad"] / count if s["reduction"] == "mean" else s["grad"], 0.0)
    p.mul_((g / total)[:, None])
    p[torch.arange(len(y), device=y.device), y.clamp(min=0)] -= g
    return [loss, (p @ w).to(s["hidden"].dtype), (p.T @ x).to(s["weight"].dtype)]


def _plain_embed(s):
    w = s["weight"]
    out = (w[s["ids"]].float() * s["scale"]).to(w.dtype)
    if not s["train"]:
        return [out]
    grad = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
    grad.index_add_(0, s["ids"], s["grad"].float() * s["scale"])
    return [out, grad.to(w.dtype)]


def _plain_clip(s):
    # bucket by bucket: the same sums and products as tensor by tensor, in a fraction of the launches
    norm = torch.stack([f.float().square().sum() for f in s["flat"]]).sum().sqrt()
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(f.float() * c) for f, o in zip(s["flat"], s["flat_out"])]
    return [norm] + s["flat_out"]


def work(case):
    es = SIZE[case["dtype"]]
    if case["kind"] == "clip":
        n = sum(math.prod(x) for shapes in _clip_groups(case) for x in shapes)
        return {"bytes": n * es + (n * (4 if case["wide_out"] else es) if case["over"] else 0), "flops": 2 * n + (n if case["over"] else 0)}
    T, V, d = case["T"], case["V"], case["d"]
    if case["kind"] == "embed":
        rows = min(T, V) * d * es
        return {"bytes": rows + T * (8 + d * es) + (T * d * es + V * d * es if case["train"] else 0), "flops": T * d * (2 if case["train"] else 1)}
    kept = max(1, round(T * (1 - case["ignored"])))     # rows without a target need no products
    loss = (T if case["reduction"] == "none" else 1) * 4
    if not case["train"]:
        return {"bytes": (kept + V) * d * es + 8 * T + loss, "flops": 2 * kept * V * d}
    return {"bytes": (kept + T + 2 * V) * d * es + 8 * T + loss, "flops": 6 * kept * V * d}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "clip":
            total = sum(float(f.double().pow(2).sum()) for f in s["flat"])
            c = min(1.0, s["max_norm"] / (math.sqrt(total) + 1e-6))
            return [torch.tensor(math.sqrt(total), dtype=torch.float64)] + [f.double() * c for f in s["flat"]]
        w = s["weight"].double()
        if case["kind"] == "embed":
            out = torch.index_select(w, 0, s["ids"]) * s["scale"]
            if not case["train"]:
                return [out]
            order = torch.argsort(s["ids"], stable=True)
            sums = torch.cat([torch.zeros(1, case["d"], device="cuda", dtype=torch.float64),
                              s["grad"].double()[order].cumsum(0)])
            ends = torch.searchsorted(s["ids"][order], torch.arange(case["V"], device="cuda"), right=True)
            starts = torch.cat([ends.new_zeros(1), ends[:-1]])
            return [out, (sums[ends] - sums[starts]) * s["scale"]]
        x, y = s["hidden"].double(), s["targets"]
        keep = (y != IGNORE).nonzero()[:, 0]
        rows, dx, dw = torch.zeros(case["T"], device="cuda", dtype=torch.float64), torch.zeros_like(x), torch.zeros_like(w)
        g = s["grad"].double().expand(case["T"])
        if case["reduction"] == "mean":
            g = g / max(1, len(keep))
        for part in keep.split(2048):
            logp = torch.log_softmax(x[part] @ w.T, -1)
            rows[part] = -logp[torch.arange(len(part), device="cuda"), y[part]]
            if case["train"]:
                dz = logp.exp_()
                dz[torch.arange(len(part), device="cuda"), y[part]] -= 1.0
                dz *= g[part, None]
                dx[part] = dz @ w
                dw += dz.T @ x[part]
        loss = rows if case["reduction"] == "none" else rows.sum() if case["reduction"] == "sum" else rows.sum() / len(keep)
        return [loss, dx, dw] if case["train"] else [loss]
