"""The gated scan on the CPU: the float64 reference the GPU tests use, and every refusal."""

import pytest
import torch

from _scan_reference import scan_reference, softplus


def test_reference_gradients_against_autograd():
    g = torch.Generator().manual_seed(0)
    n, T, D = 3, 9, 4
    gates = torch.randn(n, T, 3 * D, generator=g, dtype=torch.float64, requires_grad=True)
    decay = torch.randn(D, generator=g, dtype=torch.float64)
    rows = decay.expand(n, D).clone().requires_grad_(True)
    state = torch.randn(n, D, generator=g, dtype=torch.float64, requires_grad=True)
    lengths = torch.tensor([9, 4, 0])
    dy, dl = torch.randn(n, T, D, generator=g, dtype=torch.float64), torch.randn(n, D, generator=g, dtype=torch.float64)
    for reverse in (False, True):
        x, r, i = gates.split(D, 2)
        a = torch.exp(-softplus(rows)[:, None] * torch.sigmoid(r))
        u = torch.sqrt(1 - a * a) * torch.sigmoid(i) * x
        h, outs = state, [None] * T
        for t in range(T - 1, -1, -1) if reverse else range(T):
            on = (lengths > t)[:, None]
            h = torch.where(on, a[:, t] * h + u[:, t], h)
            outs[t] = h * on
        want = torch.autograd.grad(
            (torch.stack(outs, 1) * dy).sum() + (h * dl).sum(), (gates, rows, state)
        )
        # the dtype of the gates only sets the rounding allowance: float32 here
        val, _ = scan_reference(gates.detach().float().double().to(torch.float32), decay, state, lengths, reverse, dy, dl)
        val64, _ = _in_float64(gates, decay, state, lengths, reverse, dy, dl)
        for k, w in zip(("grad_gates", "grad_decay", "grad_state"), want):
            torch.testing.assert_close(val64[k], w, rtol=1e-9, atol=1e-12)
            torch.testing.assert_close(val[k], w, rtol=1e-3, atol=1e-4)
        torch.testing.assert_close(val64["out"], torch.stack(outs, 1).detach())
        torch.testing.assert_close(val64["last"], h.detach())


def _in_float64(gates, *args):
    import _scan_reference as R

    keep = R.half_step
    R.half_step = lambda dtype: R.H
    try:
        return scan_reference(gates, *args)
    finally:
        R.half_step = keep


def test_c_entry_points_refuse_before_any_launch():
    from opacus_amd import _lib

    L = _lib.lib()
    one = 4096  # an aligned address that nothing dereferences: every call below is refused first
    fwd = lambda **k: L.dpk_gated_scan(  # noqa: E731
        k.get("gates", one), k.get("dtype", 0), k.get("decay", one), k.get("ddt", 0), k.get("state"), k.get("lengths"),
        k.get("out", one), k.get("last", one), k.get("kept"), k.get("n", 2), k.get("T", 8), k.get("D", 8),
        k.get("sn", 192), k.get("st", 24), k.get("reverse", 0), k.get("ws"), k.get("wsb", 0), None,
    )
    bwd = lambda **k: L.dpk_gated_scan_backward(  # noqa: E731
        k.get("gates", one), k.get("dtype", 0), k.get("decay", one), k.get("ddt", 0), k.get("kept", one), k.get("lengths"),
        k.get("dy", one), k.get("dl"), k.get("dg", one), None, None, k.get("n", 2), k.get("T", 8), k.get("D", 8),
        k.get("sn", 192), k.get("st", 24), k.get("reverse", 0), k.get("ws"), k.get("wsb", 0), None,
    )
    SHAPE, DTYPE, ALIGN, WS, ARG = -1, -2, -3, -5, -6
    for call in (fwd, bwd):
        assert call(n=-1) == SHAPE and call(T=-1) == SHAPE and call(D=-1) == SHAPE
        assert call(dtype=2) == DTYPE and call(ddt=5) == DTYPE
        assert call(gates=None) == ARG and call(decay=None) == ARG and call(reverse=2) == ARG and call(sn=-1) == ARG
        assert call(gates=one + 2) == ALIGN and call(lengths=one + 4) == ALIGN
        assert call(n=2**40, D=2**20) == SHAPE
        assert call(n=0) == 0 and call(D=0) == 0
        # one row of a long sequence is cut into segments and needs the workspace
        assert call(n=1, T=4096) == WS
        assert b"gated_scan" in L.dpk_last_error()
    assert fwd(out=None) == ARG and fwd(last=None) == ARG and fwd(last=one + 2) == ALIGN
    assert bwd(kept=None) == ARG and bwd(dy=None) == ARG and bwd(dg=None) == ARG
    assert L.dpk_gated_scan_workspace_bytes(1, 4096, 8) > 0
    assert L.dpk_gated_scan_workspace_bytes(0, 4096, 8) == 0 and L.dpk_gated_scan_workspace_bytes(4, 1, 8) == 0
    step = L.dpk_gated_scan_step
    assert step(one, 0, one, 0, None, one, 2, 8, 24, None) == ARG
    assert step(one, 3, one, 0, one, one, 2, 8, 24, None) == DTYPE
    assert step(one, 0, one, 0, one + 1, one, 2, 8, 24, None) == ALIGN
    assert step(None, 0, None, 0, None, None, 0, 8, 24, None) == 0


def test_more_threads_than_a_launch_may_have_are_refused():
    from opacus_amd import _lib

    L = _lib.lib()
    one, SHAPE = 4096, -1
    # a block of 256 threads takes a tile of a sample: 2^24 samples are 2^32 threads
    n = 2**24
    assert L.dpk_gated_scan(one, 0, one, 0, None, None, one, one, None, n, 1, 1, 3, 3, 0, None, 0, None) == SHAPE
    assert L.dpk_gated_scan_backward(
        one, 0, one, 0, one, None, one, None, one, None, None, n, 1, 1, 3, 3, 0, None, 0, None
    ) == SHAPE
    assert L.dpk_gated_scan_step(one, 0, one, 0, one, one, 2**30, 31, 93, None) == SHAPE


def test_wrappers_take_gpu_tensors_only():
    from opacus_amd import kernels

    gates, decay = torch.zeros(1, 2, 6), torch.zeros(2)
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.gated_scan(gates, decay)
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.gated_scan_backward(gates, decay, torch.zeros(1, 1, 2), torch.zeros(1, 2, 2))
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.gated_scan_step(gates[:, 0], decay, torch.zeros(1, 2))


def test_positions_too_far_apart_for_the_kernels_are_copied():
    """A [T, n, 3 D] storage seen as [n, T, 3 D] has n * 3 D elements between positions, which may be more than
    the kernels' 32-bit offsets inside a tile reach."""
    from opacus_amd import _lib, kernels

    most, D = _lib.DPK_SCAN_MAX_STRIDE, 4
    for stride, kept in ((most, True), (most + 1, False), (2 * most, False)):
        gates = torch.empty_strided((2, 3, 3 * D), (3 * D, stride, 1), device="meta")
        view, sn, st = kernels._gates_layout(gates, D)
        assert (view is gates) == kept and (sn, st) == ((3 * D, stride) if kept else (9 * D, 3 * D))
    one = torch.empty_strided((2, 1, 3 * D), (3 * D, 2 * most, 1), device="meta")  # no second position
    assert kernels._gates_layout(one, D)[0] is one
    # the C entry points say so
    L, at, SHAPE, WS = _lib.lib(), 4096, -1, -5
    for st, code in ((most, WS), (most + 1, SHAPE)):
        assert L.dpk_gated_scan(at, 0, at, 0, None, None, at, at, None, 1, 4096, D, 12, st, 0, None, 0, None) == code
        assert L.dpk_gated_scan_backward(
            at, 0, at, 0, at, None, at, None, at, None, None, 1, 4096, D, 12, st, 0, None, 0, None
        ) == code
