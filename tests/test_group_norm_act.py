"""Group norm with an activation on the CPU: the float64 reference of the GPU tests, and every refusal."""

import pytest
import torch
import torch.nn.functional as F

import _norm_act_reference as R


@pytest.mark.parametrize("per_position", [False, True])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_reference_against_autograd(act, per_position, monkeypatch):
    monkeypatch.setattr(R, "half_step", lambda dtype: R.H)
    g = torch.Generator().manual_seed(1)
    n, S, C, G = 3, 5, 6, 2
    x = torch.randn(n, S, C, generator=g, dtype=torch.float64, requires_grad=True)
    w = (1 + 0.3 * torch.randn(C, generator=g, dtype=torch.float64)).expand(n, C).clone().requires_grad_(True)
    w.data[:] = w.data[0]
    b = (0.3 * torch.randn(C, generator=g, dtype=torch.float64)).expand(n, C).clone().requires_grad_(True)
    dy = torch.randn(n, S, C, generator=g, dtype=torch.float64)
    if per_position:
        norm = F.group_norm(x.reshape(n * S, C), G, eps=1e-5).reshape(n, S, C)
    else:
        norm = F.group_norm(x.transpose(1, 2), G, eps=1e-5).transpose(1, 2)
    z = norm * w[:, None] + b[:, None]
    y = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[act](z)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    val, _ = R.norm_act_reference(x, G, w[0], b[0], 1e-5, act, per_position, dy)
    for k, want in (("y", y.detach()), ("grad_x", dx), ("grad_weight", dw), ("grad_bias", db)):
        torch.testing.assert_close(val[k], want, rtol=1e-9, atol=1e-11)


def test_c_entry_points_refuse_before_any_launch():
    from opacus_amd import _lib

    L = _lib.lib()
    one = 4096  # an aligned address that nothing dereferences: every call below is refused first
    ARGS = dict(x=one, dy=one, dtype=0, w=one, b=one, pdt=0, y=one, stats=one, n=2, S=8, C=8, G=2, eps=1e-5, act=0, pp=0,
                ws=one, wsb=1 << 30)

    def fwd(**k):
        a = {**ARGS, **k}
        return L.dpk_group_norm_act(a["x"], a["dtype"], a["w"], a["b"], a["pdt"], a["y"], a["stats"], a["n"], a["S"], a["C"],
                                    a["G"], a["eps"], a["act"], a["pp"], a["ws"], a["wsb"], None)

    def bwd(**k):
        a = {**ARGS, **k}
        return L.dpk_group_norm_act_backward(a["x"], a["dy"], a["dtype"], a["w"], a["b"], a["pdt"], a["stats"], a["y"], None,
                                             None, a["n"], a["S"], a["C"], a["G"], a["eps"], a["act"], a["pp"], a["ws"],
                                             a["wsb"], None)

    SHAPE, DTYPE, ALIGN, WS, ARG = -1, -2, -3, -5, -6
    for call in (fwd, bwd):
        assert call(n=-1) == SHAPE and call(S=-1) == SHAPE and call(C=0) == SHAPE and call(G=0) == SHAPE
        assert call(C=9) == SHAPE and call(C=1 << 30, G=1) == SHAPE
        assert call(dtype=2) == DTYPE and call(pdt=9) == DTYPE
        assert call(act=4) == ARG and call(act=-1) == ARG and call(pp=2) == ARG and call(eps=-1.0) == ARG
        assert call(eps=float("nan")) == ARG and call(x=None) == ARG and call(y=None) == ARG and call(stats=None) == ARG
        assert call(x=one + 2) == ALIGN and call(w=one + 1) == ALIGN and call(stats=one + 4) == ALIGN
        for k in (dict(S=10**6), dict(S=10**6, pp=1)):
            assert call(ws=None, **k) == WS and call(wsb=0, **k) == WS
        assert call(ws=one + 8) == ALIGN
        assert call(n=0) == 0 and call(S=0) == 0
        assert b"group_norm_act" in L.dpk_last_error()
    assert bwd(dy=None) == ARG
    need = L.dpk_group_norm_act_workspace_bytes
    assert need(0, 4, 8, 2, 0) == 0 and need(1, 4, 8, 2**32, 0) == 0 and need(1, 4, 2**40, 2, 0) == 0
    # none where a block holds a sample's groups, or a wave a position's and a sample is one chunk
    assert need(33, 49, 210, 14, 0) == 0 and need(64, 64, 2048, 16, 1) == 0
    assert need(3, 40000, 128, 32, 0) > 0 and need(16, 1024, 2048, 16, 1) > 0 and need(2, 4, 600, 1, 1) > 0


@pytest.mark.parametrize(
    "n, S, C, groups, per_position",
    [
        (2**23, 1, 8, 2, 0),  # a block of 512 threads per sample
        (2**24, 2**20, 8, 2, 0),  # at least one block of 256 per chunk of a sample
        (2**24, 1, 8, 2, 1),  # and backward, per position (forward cuts all positions of the tensor together)
        (2**24, 16, 2**20, 1, 1),  # a wave per position
    ],
)
def test_more_threads_than_a_launch_may_have_are_refused(n, S, C, groups, per_position):
    from opacus_amd import _lib

    L = _lib.lib()
    one, big, SHAPE = 4096, 1 << 62, -1
    if (C, per_position) != (8, 1):
        assert L.dpk_group_norm_act(
            one, 0, one, one, 0, one, one, n, S, C, groups, 1e-5, 0, per_position, one, big, None
        ) == SHAPE
    assert L.dpk_group_norm_act_backward(
        one, one, 0, one, one, 0, one, one, one, one, n, S, C, groups, 1e-5, 0, per_position, one, big, None
    ) == SHAPE


def test_wrappers_refuse():
    from opacus_amd import kernels

    x = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.group_norm_act(x, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.group_norm_act_backward(x, x, None, 2, per_position=True)
