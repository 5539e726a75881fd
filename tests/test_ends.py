"""The operators at the ends of a training step refuse what they do not take before anything touches a GPU (these run without one)."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import cdssm_b200
    from cdssm_b200 import build
    build.build()
    return cdssm_b200._lib


def test_tensors_that_are_not_on_a_gpu(lib):
    from cdssm_b200 import ops
    w, ids = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.embedding(ids, w), lambda: ops.linear_cross_entropy(torch.zeros(3, 8), w, ids), lambda: ops.grad_norm([w]),
                 lambda: ops.clip_grads_([w], 1.0), lambda: ops.clip_grads_([], 1.0),
                 lambda: ops.linear_cross_entropy(torch.zeros(3, 8), w, ids, reduction="most"), lambda: ops.clip_grads_([w], float("nan"))):
        with pytest.raises(lib.CdssmError):
            call()
    p = torch.nn.Parameter(w)
    assert float(ops.clip_grad_norm_([p], 1.0)) == 0.0       # no gradients: nothing to do


def test_arguments_of_the_abi(lib):
    h = lib.lib()
    null, one = ctypes.c_void_p(0), ctypes.c_void_p(256)
    ce = lambda rows, d, vocab, reduction=1, x=one: h.cdssm_b200_linear_ce_fwd(x, d, one, d, one, one, one, 1 << 40, one, 1 << 40, rows, d,  # noqa: E731
                                                                               vocab, -100, reduction, 0, 0, null)
    assert ce(4, 8, 10, x=null) == -1 and ce(4, 8, 10, reduction=3) == -1 and ce(0, 8, 10) == -1 and ce(4, 0, 10) == -1 and ce(4, 8, 0) == -1
    assert ce((1 << 24) + 1, 8, 10) == -2 and ce(4, (1 << 16) + 1, 10) == -2 and ce(4, 8, (1 << 24) + 1) == -2
    back = lambda gx, gw, stride=8: h.cdssm_b200_linear_ce_bwd(one, one, stride, one, one, 1 << 40, gx, gw, one, 1 << 40, 4, 8, 10, -100, 1, 0,  # noqa: E731
                                                               0, null)
    assert back(null, null) == -1 and back(ctypes.c_void_p(264), one) == -1 and back(one, one, stride=7) == -1
    # host arithmetic: pairs twice, partial sums of 8 or 32 pairs, the list of what goes on over tiles
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    for n, tile in ((1, 8), (8192, 8), (8193, 32), (100000, 32)):
        tiles = -(-n // tile)
        assert h.cdssm_b200_embedding_bwd_workspace_bytes(n, 1000, 96, 0) == 2 * up(8 * n) + 2 * up(4 * tiles * 96) + up(4 * (tiles + 1))
    assert h.cdssm_b200_embedding_bwd_workspace_bytes(0, 1000, 96, 0) == 0 and h.cdssm_b200_embedding_bwd_workspace_bytes(5, 1000, 96, 2) == 0
    assert h.cdssm_b200_embedding_fwd(null, one, 8, one, 4, 10, 8, 1.0, 0, null) == -1
    assert h.cdssm_b200_embedding_fwd(one, one, 8, one, (1 << 28) + 1, 10, 8, 1.0, 0, null) == -2
    assert h.cdssm_b200_embedding_bwd(one, one, one, one, 8, 4, 10, 8, -1, 1.0, 0, null) == -3
    assert h.cdssm_b200_embedding_bwd(one, ctypes.c_void_p(257), one, one, 1 << 30, 4, 10, 8, -1, 1.0, 0, null) == -1
    sizes = (ctypes.c_int64 * 3)(16384, 0, 16385)
    assert h.cdssm_b200_grad_clip_workspace_bytes(sizes, 3) == 256 + 8 * 3
    assert h.cdssm_b200_grad_clip_workspace_bytes((ctypes.c_int64 * 1)(-1), 1) == 0
    ptrs, types = (ctypes.c_void_p * 3)(256, 0, 512), (ctypes.c_int * 3)(0, 0, 0)
    assert h.cdssm_b200_grad_clip(ptrs, null, sizes, types, null, 3, 1.0, one, one, 8, null) == -3
    assert h.cdssm_b200_grad_clip(ptrs, null, sizes, types, null, 3, 1.0, null, one, 1 << 20, null) == -1
    assert h.cdssm_b200_grad_clip(ptrs, null, sizes, (ctypes.c_int * 3)(0, 0, 7), null, 3, 1.0, one, one, 1 << 20, null) == -1
    assert h.cdssm_b200_grad_clip(ptrs, ptrs, sizes, (ctypes.c_int * 3)(1, 1, 1), types, 3, 1.0, one, one, 1 << 20, null) == -1   # float32 into bf16


@pytest.mark.parametrize("padding_idx", [-1, -2, -5])
def test_padding_row_does_not_count_from_the_end(lib, padding_idx):
    """Not taken for "none" either: the row that was meant would be trained."""
    from cdssm_b200 import ops
    with pytest.raises(lib.CdssmError, match="padding_idx"):
        ops.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8), padding_idx=padding_idx)


def _calls():
    from cdssm_b200 import ops
    ids = torch.zeros(3, dtype=torch.int64)
    return {"hidden": lambda t: ops.linear_cross_entropy(t, torch.zeros(5, 8), ids), "weight": lambda t: ops.linear_cross_entropy(torch.zeros(3, 8), t, ids),
            "embedding": lambda t: ops.embedding(ids, t), "norm": lambda t: ops.grad_norm([torch.zeros(2), t]),
            "clip": lambda t: ops.clip_grads_([t], 1.0), "out": lambda t: ops.clip_grads_([torch.zeros(3, 8)], 1.0, out=[t])}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("call", ["hidden", "weight", "embedding", "norm", "clip", "out"])
def test_tangents_are_refused(lib, call, requires_grad):
    """Not lost: the kernels know values alone."""
    import torch.autograd.forward_ad as forward_ad
    t = torch.zeros(3, 8, requires_grad=requires_grad)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones(3, 8))
        for mode in (torch.no_grad, torch.enable_grad):
            with mode(), pytest.raises(lib.CdssmError, match="no forward-mode gradient"):
                _calls()[call](dual)
        with pytest.raises(lib.CdssmError, match="CUDA tensor"):     # (a plain one is read)
            _calls()[call](t.detach())


@pytest.mark.parametrize("call", ["hidden", "weight", "embedding", "norm", "clip", "out"])
def test_tracing_is_refused(lib, call):
    """A traced graph would return memory that nobody has written."""
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(lib.CdssmError, match="cannot be traced"):
        torch.jit.trace(_calls()[call], (torch.zeros(3, 8),), check_trace=False)
    with pytest.raises(lib.CdssmError, match="cannot be traced"):
        make_fx(_calls()[call])(torch.zeros(3, 8))
