"""The group norm + activation kernels against float64 (tests/_norm_act_reference.py)."""

import pytest
import torch

from _norm_act_reference import norm_act_reference
from _scan_reference import assert_within

pytestmark = pytest.mark.gpu


def make(n, S, C, dtype, seed=0, offset=1.0):
    g = torch.Generator().manual_seed(seed * 1009 + n * 31 + S * 7 + C)
    x = torch.randn(n, S, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset * torch.randn(n, 1, C, generator=g)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    dy = 0.1 * torch.randn(n, S, C, generator=g)
    return x.to(dtype).cuda(), w.cuda(), b.cuda(), dy.to(dtype).cuda()


def check(x, w, b, dy, groups, act, per_position, eps=1e-5):
    from opacus_amd import kernels

    args = (groups, w, b, eps, act)
    y, stats = kernels.group_norm_act(x, *args, per_position=per_position)
    got = kernels.group_norm_act_backward(x, dy, stats, *args, per_position=per_position)
    again = kernels.group_norm_act_backward(x, dy, stats, *args, per_position=per_position)
    assert all(torch.equal(p, q) for p, q in zip(got, again))  # fixed order: the same bits
    assert torch.equal(y, kernels.group_norm_act(x, *args, per_position=per_position)[0])
    val, tol = norm_act_reference(x, groups, w, b, eps, act, per_position, dy)
    for name, t in (("y", y), ("grad_x", got[0]), ("grad_weight", got[1]), ("grad_bias", got[2])):
        assert_within(t, val[name], tol[name], name)


SAMPLE_SHAPES = [  # n, S, C, groups
    (1, 1, 2, 1), (2, 1, 4, 4), (3, 4, 6, 2), (2, 5, 7, 7), (2, 9, 30, 5), (4, 49, 64, 32), (1, 64, 8, 1), (3, 65, 24, 4),
    (2, 256, 64, 16), (1, 1024, 64, 32), (2, 1000, 33, 3), (1, 3000, 16, 2), (5, 16, 512, 32), (1, 70, 1030, 10),
    (2, 33, 2056, 1), (1, 5000, 128, 32),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,S,C,groups", SAMPLE_SHAPES)
def test_statistics_per_sample(n, S, C, groups, dtype):
    check(*make(n, S, C, dtype), groups, "silu", False)


POSITION_SHAPES = [
    (1, 1, 2, 1), (3, 1, 64, 4), (2, 5, 6, 2), (2, 7, 30, 3), (1, 130, 128, 2), (4, 33, 256, 4), (2, 65, 512, 8),
    (1, 9, 1024, 16), (2, 6, 2048, 16), (2, 3, 4096, 1), (1, 4, 2048, 1), (3, 10, 100, 5), (1, 300, 40, 8), (2, 40, 96, 12),
    (1, 2, 10000, 2), (1, 70, 8, 8), (2, 50, 24, 24), (2, 1111, 64, 2), (1, 67, 12, 3), (3, 129, 5, 5), (2, 999, 4, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,S,C,groups", POSITION_SHAPES)
def test_statistics_per_position(n, S, C, groups, dtype):
    check(*make(n, S, C, dtype), groups, "silu", True)


@pytest.mark.parametrize("per_position", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_activations(act, dtype, per_position):
    check(*make(3, 40, 64, dtype), 4, act, per_position)
    check(*make(2, 21, 18, dtype), 3, act, per_position)


@pytest.mark.parametrize("per_position", [False, True])
def test_parameters_absent_or_in_bfloat16(per_position):
    x, w, b, dy = make(2, 30, 32, torch.float32)
    for ww, bb in ((None, None), (w, None), (None, b), (w.bfloat16(), b.bfloat16())):
        check(x, ww, bb, dy, 4, "silu", per_position)


@pytest.mark.parametrize("per_position", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unaligned_strided_and_nd_inputs(dtype, per_position):
    from opacus_amd import kernels

    x, w, b, dy = make(2, 24, 16, dtype)
    flat = torch.zeros(2 * 24 * 16 + 1, dtype=dtype, device="cuda")
    off = flat[1:].view(2, 24, 16)  # one element off every vector alignment
    off.copy_(x)
    check(off, w, b, dy, 2, "silu", per_position)
    check(x.transpose(0, 1).contiguous().transpose(0, 1), w, b, dy.transpose(1, 2).contiguous().transpose(1, 2), 2, "gelu", per_position)
    y4, _ = kernels.group_norm_act(x.view(2, 4, 6, 16), 2, w, b, per_position=per_position)
    y3, _ = kernels.group_norm_act(x, 2, w, b, per_position=per_position)
    assert y4.shape == (2, 4, 6, 16) and torch.equal(y4.view_as(y3), y3)
    y2, _ = kernels.group_norm_act(x[:, 0], 2, w, b, per_position=per_position)  # [n, C]: one position
    assert y2.shape == (2, 16)


@pytest.mark.parametrize("S,C,groups,per_position", [(1024, 64, 8, False), (9000, 32, 4, False), (20, 128, 2, True), (20, 50, 2, True)])
def test_a_large_mean_and_a_lone_outlier_cost_no_digits(S, C, groups, per_position):
    x, w, b, dy = make(2, S, C, torch.float32)
    check(x + 300.0, w, b, dy, groups, "none", per_position)
    x[0, 0, 0] = 3.0e4
    x[1, -1, -1] = -3.0e4
    check(x, w, b, dy, groups, "none", per_position)


@pytest.mark.parametrize("S,C,groups,per_position", [(60, 16, 4, False), (6000, 64, 4, False), (60, 64, 4, True), (60, 20, 4, True)])
def test_not_a_number_stays_in_its_statistics(S, C, groups, per_position):
    from opacus_amd import kernels

    x, w, b, dy = make(2, S, C, torch.float32)
    clean, _ = kernels.group_norm_act(x, groups, w, b, activation="silu", per_position=per_position)
    x[1, 3, 0] = float("nan")
    y, _ = kernels.group_norm_act(x, groups, w, b, activation="silu", per_position=per_position)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, 3 if per_position else slice(None), : C // groups] = True
    assert y[hit].isnan().all() and torch.equal(y[~hit], clean[~hit])


def test_constant_inputs_normalise_to_the_bias():
    from opacus_amd import kernels

    for per_position in (False, True):
        x, w, b, dy = make(2, 12, 16, torch.float32)
        y, st = kernels.group_norm_act(torch.full_like(x, 3.0), 2, w, b, per_position=per_position)
        # the mean is off by at most 266 half-steps of 3, times rstd = eps ** -0.5 and a weight below 2
        assert (y - b).abs().max() <= 266 * 2.0**-24 * 3 * 317 * 2
        for t in kernels.group_norm_act_backward(torch.full_like(x, 3.0), dy, st, 2, w, b, per_position=per_position):
            assert torch.isfinite(t).all()


def test_empty_sizes():
    from opacus_amd import kernels

    for per_position in (False, True):
        for n, S in ((0, 4), (3, 0)):
            x = torch.zeros(n, S, 8, device="cuda")
            y, st = kernels.group_norm_act(x, 2, per_position=per_position)
            dx, dw, db = kernels.group_norm_act_backward(x, x, st, 2, per_position=per_position)
            assert y.shape == x.shape and dx.shape == x.shape and dw.shape == (n, 8)
            assert (dw == 0).all() and (db == 0).all()


def test_refusals_on_the_gpu():
    from opacus_amd import kernels

    x, w, b, dy = make(2, 6, 8, torch.float32)
    _, st = kernels.group_norm_act(x, 2, w, b)
    for kw, what in (
        (dict(num_groups=3), "divide"), (dict(num_groups=0), "divide"), (dict(num_groups=2, activation="tanh"), "activation"),
        (dict(num_groups=2, eps=-1.0), "eps"), (dict(num_groups=2, weight=w[:4]), "shape"),
        (dict(num_groups=2, weight=w, bias=b.bfloat16()), "dtype"),
    ):
        with pytest.raises(ValueError, match=what):
            kernels.group_norm_act(x, **kw)
    with pytest.raises(TypeError):
        kernels.group_norm_act(x.half(), 2)
    with pytest.raises(TypeError):
        kernels.group_norm_act(x, 2, w.double(), b.double())
    with pytest.raises(RuntimeError, match="GPU only"):
        kernels.group_norm_act(x, 2, w.cpu())
    with pytest.raises(ValueError, match="grad_out"):
        kernels.group_norm_act_backward(x, dy[:1], st, 2, w, b)
    with pytest.raises(ValueError, match="stats"):
        kernels.group_norm_act_backward(x, dy, None, 2, w, b)
    with pytest.raises(ValueError, match="stats"):
        kernels.group_norm_act_backward(x, dy, st[:, :1], 2, w, b)
    with pytest.raises(ValueError, match="n, \\*, C"):
        kernels.group_norm_act(x[0, 0], 2)


@pytest.mark.parametrize("S,C,groups,per_position", [(4000, 64, 8, False), (100, 64, 8, False), (200, 256, 4, True), (40, 30, 3, True)])
def test_captured_calls_replay_on_new_inputs(S, C, groups, per_position):
    from opacus_amd import kernels

    sets = [make(2, S, C, torch.bfloat16, seed=s) for s in range(4)]
    x, w, b, dy = (t.clone() for t in sets[0])

    def call():
        y, st = kernels.group_norm_act(x, groups, w, b, activation="silu", per_position=per_position)
        return (y,) + kernels.group_norm_act_backward(x, dy, st, groups, w, b, activation="silu", per_position=per_position)

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
        for dst, src in zip((x, w, b, dy), sets[k]):
            dst.copy_(src)
        want = [t.clone() for t in call()]
        for g, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            for p, q in zip(res, want):
                assert torch.equal(p, q)


def test_offsets_past_32_bits():
    """2.2 billion elements: the last rows against the same rows in a small tensor."""
    from opacus_amd import kernels

    S, C, G = 17_000_000, 64, 4
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty(2, S, C, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    dy = torch.empty(2, S, C, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert x.numel() > 2**31
    w, b = torch.rand(C, device="cuda", generator=g) + 0.5, torch.randn(C, device="cuda", generator=g)
    args = (G, w, b, 1e-5, "silu")
    y, _ = kernels.group_norm_act(x, *args, per_position=True)
    dx, dw, db = kernels.group_norm_act_backward(x, dy, None, *args, per_position=True)
    xs, dys = x[1:, -50:].clone(), dy[1:, -50:].clone()
    ys, _ = kernels.group_norm_act(xs, *args, per_position=True)
    dxs, _, _ = kernels.group_norm_act_backward(xs, dys, None, *args, per_position=True)
    assert torch.equal(y[1:, -50:], ys) and torch.equal(dx[1:, -50:], dxs)
    # per sample: the second sample alone is cut into other chunks, so sums agree to their rounding
    y, st = kernels.group_norm_act(x, *args)
    dx, dw, db = kernels.group_norm_act_backward(x, dy, st, *args)
    one, one_dy = x[1:].clone(), dy[1:].clone()
    y1, st1 = kernels.group_norm_act(one, *args)
    dx1, dw1, db1 = kernels.group_norm_act_backward(one, one_dy, st1, *args)
    # 264 half-steps of the sums' terms: mean |x| is 0.8, the variance 1, mean |dz| below 1, and sums of S terms
    bar = 264 * 2.0**-24
    assert (st[1] - st1[0]).abs().max() <= 2 * bar
    assert (dw[1] - dw1[0]).abs().max() <= 2 * bar * S and (db[1] - db1[0]).abs().max() <= 2 * bar * S
    # outputs: at most a rounding apart (2**-8 of values below 16 and of gradients below 16)
    assert (y[1] - y1[0]).abs().max() <= 2.0**-4 and (dx[1] - dx1[0]).abs().max() <= 2.0**-4


# 64 channels in 32 groups: one block holds a slab of up to 512 positions in bfloat16, 1024 in float32; beyond it the
# statistics, their merge and the application are launches of their own
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("S,dtype", [
    (512, torch.bfloat16), (513, torch.bfloat16), (1024, torch.float32), (1025, torch.float32),
])
def test_both_sides_of_the_longest_slab(S, dtype, act):
    check(*make(2, S, 64, dtype), 32, act, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,S,C,groups", [(3, 16, 2048, 1), (2, 8, 2040, 1), (2, 3, 2046, 2), (3, 16, 1000, 1), (2, 64, 512, 2)])
def test_wide_groups_within_one_block(n, S, C, groups, dtype, monkeypatch):
    """One thread adds up a group's channels, so the longest path is the group's width, after 16 positions and up to 512
    row groups."""
    import _norm_act_reference

    monkeypatch.setattr(_norm_act_reference, "P", C // groups + 16 + 512)
    check(*make(n, S, C, dtype), groups, "silu", False)
