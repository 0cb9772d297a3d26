"""The gated scan kernels against the definition in float64 (tests/_scan_reference.py)."""

import pytest
import torch

from _scan_reference import assert_within, scan_reference

pytestmark = pytest.mark.gpu


def make(n, T, D, dtype, seed=0, ragged=False, with_state=False, wide=False):
    g = torch.Generator().manual_seed(seed * 7919 + n * 131 + T * 17 + D)
    gates = torch.randn(n, T, 3 * D, generator=g)
    if wide:  # gates that close and open all the way, decays beyond the series' range
        gates = gates * 2.5
        decay = torch.randn(D, generator=g) * 3.0
    else:
        decay = torch.log(torch.expm1(-2.0 * torch.log(0.9 + 0.099 * torch.rand(D, generator=g))))
    gates = gates.clamp(-8, 8).to(dtype).cuda()
    state = torch.randn(n, D, generator=g).cuda() if with_state else None
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (n,), generator=g)
        lengths[0] = 0
        if n > 1:
            lengths[1] = min(1, T)
        if n > 2:
            lengths[2] = T
        lengths = lengths.cuda()
    dy = (torch.randn(n, T, D, generator=g) * 0.05).to(dtype).cuda()
    dl = torch.randn(n, D, generator=g).cuda() if with_state else None
    return gates, decay.cuda(), state, lengths, dy, dl


def check(gates, decay, state, lengths, dy, dl, reverse=False):
    from opacus_amd import kernels

    out, last, kept = kernels.gated_scan(gates, decay, state, lengths, reverse, keep_states=True)
    out2, last2, none = kernels.gated_scan(gates, decay, state, lengths, reverse)
    assert none is None and torch.equal(out, out2) and torch.equal(last, last2)
    dg, dd, ds = kernels.gated_scan_backward(gates, decay, kept, dy, dl, lengths, reverse)
    again = kernels.gated_scan_backward(gates, decay, kept, dy, dl, lengths, reverse)
    assert all(torch.equal(p, q) for p, q in zip((dg, dd, ds), again))  # fixed order: the same bits
    val, tol = scan_reference(gates, decay, state, lengths, reverse, dy, dl)
    for name, got in (("out", out), ("last", last), ("grad_gates", dg), ("grad_decay", dd), ("grad_state", ds)):
        assert_within(got, val[name], tol[name], name)


SHAPES = [
    (1, 1, 1), (1, 1, 64), (3, 2, 5), (2, 7, 4), (2, 8, 66), (2, 9, 64), (1, 63, 3), (1, 64, 16), (2, 65, 65), (1, 127, 34),
    (2, 128, 64), (1, 129, 130), (5, 200, 20), (1, 1025, 8), (2, 700, 72), (1, 2500, 6),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,T,D", SHAPES)
def test_shapes(n, T, D, dtype):
    check(*make(n, T, D, dtype))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,T,D", [(4, 5, 6), (6, 150, 68), (3, 1500, 10), (5, 64, 33)])
def test_padded_batches_states_and_directions(n, T, D, dtype, reverse):
    check(*make(n, T, D, dtype, ragged=True, with_state=True), reverse=reverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_and_decays_over_their_whole_range(dtype):
    check(*make(3, 300, 48, dtype, with_state=True, wide=True))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,T,D", [(3, 130, 66), (2, 192, 5), (4, 193, 64), (3, 256, 6), (2, 257, 64)])
def test_lengths_around_the_longest_that_one_block_takes(n, T, D, dtype, reverse):
    check(*make(n, T, D, dtype, ragged=True, with_state=True), reverse=reverse)


# 512 blocks fill the GPU backward: every row by one block, whatever its length; 400 do not
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("n,T,D,dtype", [
    (512, 300, 4, torch.float32), (500, 260, 3, torch.bfloat16), (64, 330, 512, torch.bfloat16), (400, 300, 4, torch.float32),
    (171, 65, 130, torch.float32),
])
def test_rows_that_fill_the_gpu(n, T, D, dtype, ragged):
    from opacus_amd import _lib

    fills = n * -(-D // 64) >= 436
    # (forward, 256 positions are the most that need no workspace)
    assert (_lib.lib().dpk_gated_scan_workspace_bytes(n, min(T, 256), D) == 0) == (fills or T <= 192)
    check(*make(n, T, D, dtype, ragged=ragged, with_state=ragged), reverse=ragged)


def test_many_rows_leave_the_time_axis_whole():
    check(*make(40, 140, 1024, torch.bfloat16))


def test_slices_and_unaligned_views_are_read_in_place():
    gates, decay, state, lengths, dy, dl = make(4, 90, 24, torch.bfloat16, ragged=True, with_state=True)
    big = torch.full((9, 95, 80), float("nan"), dtype=torch.bfloat16, device="cuda")
    view = big[1::2, 3:93, 5:77]  # odd offset, strides that are no multiple of the vector width
    view.copy_(gates)
    check(view, decay, state, lengths, dy, dl)
    by_time = gates.transpose(0, 1).contiguous().transpose(0, 1)  # [T, n, 3D] storage
    check(by_time, decay, state, lengths, dy, dl)
    check(gates[..., ::1].flip(2).flip(2), decay, state, lengths, dy.transpose(0, 1).contiguous().transpose(0, 1), dl)


@pytest.mark.parametrize("reverse", [False, True])
def test_padding_is_never_read_and_comes_out_as_zero(reverse):
    from opacus_amd import kernels

    gates, decay, state, lengths, dy, dl = make(5, 130, 20, torch.float32, ragged=True, with_state=True)
    dead = torch.arange(130, device="cuda")[None, :] >= lengths[:, None]
    want = kernels.gated_scan(gates, decay, state, lengths, reverse, keep_states=True)
    want_b = kernels.gated_scan_backward(gates, decay, want[2], dy, dl, lengths, reverse)
    for bad in (float("nan"), float("inf"), torch.finfo(torch.float32).min):
        gb, yb = gates.clone(), dy.clone()
        gb[dead], yb[dead] = bad, bad
        got = kernels.gated_scan(gb, decay, state, lengths, reverse, keep_states=True)
        got_b = kernels.gated_scan_backward(gb, decay, got[2], yb, dl, lengths, reverse)
        for p, q in zip(got + got_b, want + want_b):
            assert torch.equal(p, q)
        assert (got[0][dead] == 0).all() and (got_b[0][dead] == 0).all()
    # a sequence of length zero: the state as it came, its gradient as it came
    assert torch.equal(want[1][0], state[0]) and torch.equal(want_b[2][0], dl[0]) and (want_b[1][0] == 0).all()


def test_lengths_outside_the_range_are_clamped():
    from opacus_amd import kernels

    gates, decay, *_ = make(3, 20, 8, torch.float32)
    bad = torch.tensor([-5, 21, 2**40], device="cuda")
    good = torch.tensor([0, 20, 20], device="cuda")
    for p, q in zip(kernels.gated_scan(gates, decay, None, bad)[:2], kernels.gated_scan(gates, decay, None, good)[:2]):
        assert torch.equal(p, q)


def test_closed_gates_have_finite_gradients():
    from opacus_amd import kernels

    gates, decay, *_ = make(2, 40, 8, torch.float32)
    gates[..., 8:16] = torch.tensor([-200.0, -90.0, float("-inf"), -30.0, 200.0, float("inf"), 90.0, 0.0], device="cuda")
    decay = torch.tensor([0.5, -120.0, 3.0, -60.0, 40.0, -20.0, 100.0, -200.0], device="cuda")
    out, last, kept = kernels.gated_scan(gates, decay, keep_states=True)
    dg, dd, ds = kernels.gated_scan_backward(gates, decay, kept, torch.ones_like(out))
    for t in (out, last, dg, dd, ds):
        assert torch.isfinite(t).all()


def test_not_a_number_goes_forward_only():
    from opacus_amd import kernels

    gates, decay, *_ = make(1, 200, 4, torch.float32)
    clean = kernels.gated_scan(gates, decay)[0]
    gates[0, 100, 1] = float("nan")
    out = kernels.gated_scan(gates, decay)[0]
    assert torch.equal(out[:, :100], clean[:, :100]) and torch.equal(out[..., [0, 2, 3]], clean[..., [0, 2, 3]])
    assert out[0, 100:, 1].isnan().all()


def test_empty_sizes():
    from opacus_amd import kernels

    for dtype in (torch.float32, torch.bfloat16):
        for n, T, D in ((0, 5, 4), (3, 0, 4), (3, 5, 0), (0, 0, 4)):
            gates, decay = torch.zeros(n, T, 3 * D, dtype=dtype, device="cuda"), torch.zeros(D, device="cuda")
            state = torch.randn(n, D, device="cuda")
            out, last, kept = kernels.gated_scan(gates, decay, state, keep_states=True)
            dg, dd, ds = kernels.gated_scan_backward(gates, decay, kept, out, state)
            assert out.shape == (n, T, D) and dg.shape == gates.shape and dd.shape == (n, D)
            if T == 0:
                assert torch.equal(last, state) and torch.equal(ds, state) and (dd == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,D", [(1, 1), (1, 2048), (7, 130), (250, 33), (64, 1000)])
def test_step_is_one_position_of_the_scan(n, D, dtype):
    from opacus_amd import kernels

    gates, decay, state, _, _, _ = make(n, 1, D, dtype, with_state=True)
    val, tol = scan_reference(gates, decay, state)
    run = state.clone()
    version = run._version
    out = kernels.gated_scan_step(gates[:, 0], decay, run)
    assert run._version > version
    assert_within(out, val["out"][:, 0], tol["out"][:, 0], "out")
    assert_within(run, val["last"], tol["last"], "state")


def test_steps_after_a_prefix_continue_the_scan():
    from opacus_amd import kernels

    gates, decay, state, _, _, _ = make(3, 70, 40, torch.float32, with_state=True)
    whole = kernels.gated_scan(gates, decay, state)[0]
    _, run, _ = kernels.gated_scan(gates[:, :50], decay, state)
    val, tol = scan_reference(gates, decay, state)
    for t in range(50, 70):
        out = kernels.gated_scan_step(gates[:, t], decay, run)  # rows of a longer tensor, read with its stride
        assert_within(out, val["out"][:, t], tol["out"][:, t], f"step {t}")
    assert_within(whole, val["out"], tol["out"], "whole")


def test_bfloat16_decay_and_gradients_by_differences():
    """The float32 kernels' gradient against central differences of the float64 definition."""
    from opacus_amd import kernels

    gates, decay, state, lengths, dy, dl = make(2, 12, 3, torch.float32, ragged=True, with_state=True)
    decay = decay.to(torch.bfloat16)
    check(gates, decay, state, lengths, dy, dl)
    _, _, kept = kernels.gated_scan(gates, decay, state, lengths, keep_states=True)
    dg, dd, ds = kernels.gated_scan_backward(gates, decay, kept, dy, dl, lengths)

    import _scan_reference as R

    def loss(g, lam, s):
        keep, R.half_step = R.half_step, lambda dtype: R.H
        try:
            val, _ = scan_reference(g, lam, s, lengths)
        finally:
            R.half_step = keep
        return (val["out"] * dy.double().cpu()).sum((1, 2)) + (val["last"] * dl.double().cpu()).sum(1)

    base = [gates.double().cpu(), decay.double().cpu(), state.double().cpu()]
    step = 1e-5  # central differences: truncation about step^2 = 1e-10, rounding 1e-16 / step = 1e-11 of values near 1
    for which, grad in enumerate((dg, dd, ds)):
        grad = grad.double().cpu()
        shape = base[which].shape if which != 1 else (2, 3)
        for idx in range(grad.numel()):
            lo, hi = [t.clone() for t in base], [t.clone() for t in base]
            at = idx if which != 1 else idx % 3
            lo[which].view(-1)[at] -= step
            hi[which].view(-1)[at] += step
            d = (loss(*hi) - loss(*lo)) / (2 * step)
            want = d[idx // (grad.numel() // shape[0])] if which != 1 else d[idx // 3]
            assert abs(grad.reshape(-1)[idx] - want) <= 2e-5 * (1 + abs(want)), (which, idx)


def test_refusals_on_the_gpu():
    from opacus_amd import kernels

    gates, decay, state, lengths, dy, _ = make(2, 6, 4, torch.float32, ragged=True, with_state=True)
    _, _, kept = kernels.gated_scan(gates, decay, keep_states=True)
    with pytest.raises(ValueError, match="dimensions"):
        kernels.gated_scan(gates[0], decay)
    with pytest.raises(ValueError, match="3 \\* D"):
        kernels.gated_scan(gates, decay[:3])
    with pytest.raises(ValueError, match="state"):
        kernels.gated_scan(gates, decay, state.bfloat16())
    with pytest.raises(ValueError, match="state"):
        kernels.gated_scan(gates, decay, state[:1])
    with pytest.raises(ValueError, match="lengths"):
        kernels.gated_scan(gates, decay, None, lengths.int())
    with pytest.raises(ValueError, match="lengths"):
        kernels.gated_scan(gates, decay, None, lengths[:1])
    with pytest.raises(TypeError):
        kernels.gated_scan(gates.half(), decay)
    with pytest.raises(TypeError):
        kernels.gated_scan(gates, decay.double())
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.gated_scan(gates, decay.cpu())
    with pytest.raises(ValueError, match="kept"):
        kernels.gated_scan_backward(gates, decay, kept[:, :0], dy)
    with pytest.raises(ValueError, match="keep_states"):
        kernels.gated_scan_backward(gates, decay, kernels.gated_scan(gates, decay)[2], dy)
    with pytest.raises(ValueError, match="grad_out"):
        kernels.gated_scan_backward(gates, decay, kept, dy[:, :3])
    with pytest.raises(ValueError, match="grad_last"):
        kernels.gated_scan_backward(gates, decay, kept, dy, state[:, :2])
    with pytest.raises(ValueError, match="dense"):
        kernels.gated_scan_step(gates[:, 0], decay, state.t().contiguous().t())
    with pytest.raises(ValueError, match="not differentiable"):
        kernels.gated_scan_step(gates[:, 0], decay, state.clone().requires_grad_(True))


def test_captured_calls_replay_on_new_inputs():
    from opacus_amd import kernels

    # one shape that cuts T into segments (workspace inside the graph's pool), two graphs alive at once
    sets = [make(1, 1500, 64, torch.bfloat16, seed=s, with_state=True) for s in range(4)]
    gates, decay, state, _, dy, dl = (t.clone() if t is not None else None for t in sets[0])

    def call():
        out, last, kept = kernels.gated_scan(gates, decay, state, keep_states=True)
        return (out, last) + kernels.gated_scan_backward(gates, decay, kept, dy, dl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = call()
        graphs.append((g, res))
    for k in (1, 2, 3, 1):
        for dst, src in zip((gates, decay, state, dy, dl), (sets[k][0], sets[k][1], sets[k][2], sets[k][4], sets[k][5])):
            dst.copy_(src)
        want = [t.clone() for t in call()]
        for g, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            for p, q in zip(res, want):
                assert torch.equal(p, q)


def test_another_stream():
    from opacus_amd import kernels

    gates, decay, state, lengths, dy, dl = make(2, 300, 64, torch.bfloat16, ragged=True, with_state=True)
    want = kernels.gated_scan(gates, decay, state, lengths)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kernels.gated_scan(gates, decay, state, lengths)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got[:2], want[:2]))


def test_graphs_that_share_a_memory_pool_replay_in_turn():
    """The second graph's workspaces lie where the first one's were."""
    from opacus_amd import kernels

    a, b = make(1, 1500, 64, torch.bfloat16, seed=21, with_state=True), make(2, 900, 40, torch.float32, seed=22, with_state=True)

    def call(t):
        gates, decay, state, _, dy, dl = t
        out, last, kept = kernels.gated_scan(gates, decay, state, keep_states=True)
        return (out, last) + kernels.gated_scan_backward(gates, decay, kept, dy, dl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(a), call(b)
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        ra = call(a)
    with torch.cuda.graph(second, pool=first.pool()):
        rb = call(b)
    want_a, want_b = call(a), call(b)
    for _ in range(3):
        first.replay()
        second.replay()
        call(b)
        torch.cuda.synchronize()
        for p, q in zip(ra + rb, want_a + want_b):
            assert torch.equal(p, q)


def test_two_calls_on_two_streams_at_once():
    from opacus_amd import kernels

    sets = [make(4, 3000, 128, torch.bfloat16, seed=30 + k) for k in range(2)]
    want = [kernels.gated_scan(g, d, keep_states=True) for g, d, *_ in sets]
    want_b = [kernels.gated_scan_backward(s[0], s[1], w[2], s[4]) for s, w in zip(sets, want)]
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                out = kernels.gated_scan(sets[k][0], sets[k][1], keep_states=True)
                got[k].append(out + kernels.gated_scan_backward(sets[k][0], sets[k][1], out[2], sets[k][4]))
    torch.cuda.synchronize()
    for k in range(2):
        for res in got[k]:
            for p, q in zip(res, want[k] + want_b[k]):
                assert torch.equal(p, q)


def test_offsets_past_32_bits():
    """3.2 billion gate elements: the second sample's results against the same sample alone, whose
    offsets are small. What is folded, and how, depends on T and D alone: the same bits."""
    from opacus_amd import kernels

    n, T, D = 2, 65536, 8192
    g = torch.Generator(device="cuda").manual_seed(5)
    gates = torch.empty(n, T, 3 * D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert gates.numel() > 2**31
    dy = torch.empty(n, T, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    decay = torch.randn(D, device="cuda", generator=g)
    out, last, kept = kernels.gated_scan(gates, decay, keep_states=True)
    dg, dd, ds = kernels.gated_scan_backward(gates, decay, kept, dy)
    one, one_dy = gates[1:].clone(), dy[1:].clone()
    out1, last1, kept1 = kernels.gated_scan(one, decay, keep_states=True)
    dg1, dd1, ds1 = kernels.gated_scan_backward(one, decay, kept1, one_dy)
    for p, q in ((out, out1), (last, last1), (kept, kept1), (dg, dg1), (dd, dd1), (ds, ds1)):
        assert torch.equal(p[1:], q)
    # and a slice of it against the definition: the first 40 positions of the last 8 channels
    from _scan_reference import assert_within, scan_reference

    cols = torch.cat([torch.arange(k * D + D - 8, k * D + D, device="cuda") for k in range(3)])
    sub = gates[1:, :40].index_select(2, cols)
    val, tol = scan_reference(sub.clamp(-8, 8), decay[-8:])
    assert_within(out[1:, :40, -8:], val["out"], tol["out"], "out")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beyond", [-1, 0, 1])
def test_positions_far_apart(beyond, dtype, reverse):
    """At the largest position stride that the kernels take, in pairs of elements and (an odd stride) one by one, and
    just beyond it, where the gates are copied."""
    from opacus_amd import _lib

    gates, decay, state, lengths, dy, dl = make(2, 131, 64, dtype, ragged=True, with_state=True)
    stride = _lib.DPK_SCAN_MAX_STRIDE + beyond
    storage = torch.empty(130 * stride + 2 * 192, dtype=dtype, device="cuda")
    view = storage.as_strided((2, 131, 192), (192, stride, 1))
    view.copy_(gates)
    check(view, decay, state, lengths, dy, dl, reverse)


def test_a_sample_alone_and_in_a_batch_that_fills_the_gpu():
    """Backward, 512 rows are walked by a block each, where one row of the same length is a chain of tiles. The states are
    the same bits (forward depends on T alone); the gradients are sums in another order, most of all that of the decay,
    which the walk adds up over all of a thread's positions and the chain tile by tile: each within its bound,
    not the same bits."""
    from opacus_amd import _lib, kernels

    n, T, D, k = 512, 300, 4, 317
    L = _lib.lib()  # (256 positions: the longest that one block takes forward, so only backward may need a workspace)
    assert L.dpk_gated_scan_workspace_bytes(n, 256, D) == 0 and L.dpk_gated_scan_workspace_bytes(1, 256, D) > 0
    gates, decay, state, lengths, dy, dl = make(n, T, D, torch.float32, ragged=True, with_state=True)
    lengths[k] = T - 7
    batch = (gates, decay, state, lengths, dy, dl)
    one = (gates[k : k + 1], decay, state[k : k + 1], lengths[k : k + 1], dy[k : k + 1], dl[k : k + 1])
    val, tol = scan_reference(one[0], decay, one[2], one[3], False, one[4], one[5])
    runs = []
    for (g, d, s, l, y, z), at in ((batch, k), (one, 0)):
        out, last, kept = kernels.gated_scan(g, d, s, l, keep_states=True)
        runs.append([t[at : at + 1] for t in (out, last, kept) + kernels.gated_scan_backward(g, d, kept, y, z, l)])
    for p, q in zip(runs[0][:3], runs[1][:3]):
        assert torch.equal(p, q)
    for run in runs:
        for name, got in zip(("grad_gates", "grad_decay", "grad_state"), run[3:]):
            assert_within(got, val[name], tol[name], name)


@pytest.mark.parametrize("reverse", [False, True])
def test_a_long_row_walked_by_one_block(reverse):
    """47 tiles in turn: a thread adds up 375 positions of the decay's gradient in a row (the bound allows T)."""
    check(*make(512, 3000, 2, torch.float32, ragged=True, with_state=True), reverse=reverse)
