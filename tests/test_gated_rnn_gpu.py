"""DPGatedRNN, GatedScan, GroupNormAct and HeadNormAct in the engines: per-sample gradients, norms and
clipped sums against batch-of-one automatic differentiation of the same formulas in float64 on the CPU.

Bars for float32: one scan over T <= 40 positions adds at most 12 half-steps of relative error a
position (40 * 12 * 2**-24 = 2.9e-5), a second layer the same, the products of the projections (24
terms) and the norms less than that: 1e-4 at every scale of tests/_compare.py."""

import copy
from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from _compare import assert_rel

pytestmark = pytest.mark.gpu
REL = 1e-4


# ---- the formulas in plain torch ---------------------------------------------------------------
def ref_norm(mod, x):
    C, G = mod.num_channels, mod.num_groups
    if mod.per_position:
        z = F.group_norm(x.reshape(-1, C), G, mod.weight, mod.bias, mod.eps).reshape(x.shape)
    else:
        z = F.group_norm(x, G, mod.weight, mod.bias, mod.eps)
    return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[mod.activation](z)


def ref_scan(mod, gates, state=None, length=None):
    """One sample ``[1, T, 3D]``."""
    D, T = mod.hidden_size, gates.shape[1]
    x, r, i = gates.split(D, 2)
    L = -F.softplus(mod.decay) * torch.sigmoid(r)
    a, u = L.exp(), (-torch.expm1(2 * L)).sqrt() * torch.sigmoid(i) * x
    h = gates.new_zeros(1, D) if state is None else state
    outs = [gates.new_zeros(1, D) for _ in range(T)]
    length = T if length is None else length
    for t in reversed(range(length)) if mod.reverse else range(length):
        h = a[:, t] * h + u[:, t]
        outs[t] = h
    return (torch.stack(outs, 1) if T else gates.new_zeros(1, 0, D)), h


def ref_rnn(mod, x, state=None, length=None):
    """One sample ``[1, T, D]`` through a DPGatedRNN without dropout."""
    last = []
    for layer in range(mod.num_layers):
        outs = []
        for d in range(mod.num_directions):
            k = layer * mod.num_directions + d
            cell = mod.cells[k]
            out, h = ref_scan(cell.scan, F.linear(x, cell.ih.weight, cell.ih.bias), None if state is None else state[k], length)
            outs.append(out if cell.norm is None else ref_norm(cell.norm, out))
            last.append(h)
        x = torch.cat(outs, 2)
    return x, torch.stack(last)


class Net(nn.Module):
    """Embedding, recurrent layers, projection; the loss reads outputs and last states."""

    def __init__(self, layers=2, bidirectional=False, heads=4, batch_first=True):
        super().__init__()
        self.emb = nn.Embedding(11, 6)
        self.rnn = DPGatedRNN_(6, 24, layers, bidirectional, heads, batch_first)
        self.out = nn.Linear(24 * (2 if bidirectional else 1), 5)

    def forward(self, ids, lengths=None):  # ids [B, T]
        x = self.emb(ids)
        y, h = self.rnn(x, lengths=lengths)
        return self.out(y).mean(1) + h.mean((0, 2))[:, None].to(y.dtype)

    def reference(self, ids, length=None):  # one sample
        y, h = ref_rnn(self.rnn, F.embedding(ids, self.emb.weight), None, length)
        return F.linear(y, self.out.weight, self.out.bias).mean(1) + h.mean((0, 2))[:, None]


def DPGatedRNN_(i, h, layers, bi, heads, batch_first):
    from opacus_amd.layers import DPGatedRNN

    m = DPGatedRNN(i, h, layers, batch_first=batch_first, bidirectional=bi, num_heads=heads)
    with torch.no_grad():  # parameters that are not at their starting values
        for p in m.parameters():
            p.add_(0.1 * torch.randn(p.shape))
    return m


def per_sample_reference(net, ids, target, lengths=None):
    ref = copy.deepcopy(net).cpu().double()
    out = []
    for k in range(len(ids)):
        for p in ref.parameters():
            p.grad = None
        logits = ref.reference(ids[k : k + 1], None if lengths is None else int(lengths[k]))
        F.cross_entropy(logits, target[k : k + 1]).backward()
        # (a sequence of length zero leaves some parameters unused)
        out.append({n: torch.zeros_like(p) if p.grad is None else p.grad.clone() for n, p in ref.named_parameters()})
    return {n: torch.stack([o[n] for o in out]) for n in out[0]}


def data(n=5, T=33):
    g = torch.Generator().manual_seed(7)
    return torch.randint(0, 11, (n, T), generator=g), torch.randint(0, 5, (n,), generator=g)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("layers,bidirectional,heads", [(1, False, None), (2, False, 4), (2, True, 3)])
def test_hooks_per_sample_gradients(layers, bidirectional, heads, reduction, ragged):
    from opacus_amd import GradSampleModule

    torch.manual_seed(0)
    net = Net(layers, bidirectional, heads)
    ids, y = data()
    lengths = torch.tensor([33, 1, 0, 17, 32]) if ragged else None
    want = per_sample_reference(net, ids, y, lengths)
    wrapped = GradSampleModule(net.cuda(), loss_reduction=reduction)
    logits = wrapped(ids.cuda(), None if lengths is None else lengths.cuda())
    F.cross_entropy(logits, y.cuda(), reduction=reduction).backward()
    for name, p in net.named_parameters():
        assert_rel(p.grad_sample, want[name], REL, name)
        total = want[name].sum(0) / (len(ids) if reduction == "mean" else 1)
        assert_rel(p.grad.reshape(1, -1), total.reshape(1, -1), REL, f"{name} (aggregate)")


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("layers,bidirectional,heads", [(1, False, None), (2, True, 3)])
def test_ghost_norms_and_clipped_sum(layers, bidirectional, heads, single):
    from opacus_amd import GradSampleModuleFastGradientClipping
    from opacus_amd.optimizers import DPOptimizerFastGradientClipping
    from opacus_amd.utils.fast_gradient_clipping_utils import DPLossFastGradientClipping

    torch.manual_seed(1)
    net = Net(layers, bidirectional, heads)
    ids, y = data()
    want = per_sample_reference(net, ids, y)
    norms = torch.stack([g.flatten(1).norm(dim=1) for g in want.values()]).norm(dim=0)
    C = float(norms.median())
    coef = (C / (norms + 1e-6)).clamp(max=1.0)
    model = GradSampleModuleFastGradientClipping(net.cuda(), loss_reduction="mean", max_grad_norm=C, single_backward=single)
    opt = DPOptimizerFastGradientClipping(
        torch.optim.SGD(net.parameters(), lr=0.1), noise_multiplier=0.0, max_grad_norm=C, expected_batch_size=len(ids)
    )
    crit = DPLossFastGradientClipping(model, opt, nn.CrossEntropyLoss(), loss_reduction="mean")
    for _ in range(2):  # the second step starts from what the first one left
        opt.zero_grad()
        crit(model(ids.cuda()), y.cuda()).backward()
        assert_rel(model.per_sample_gradient_norms, norms, REL, "norms")
        for name, p in net.named_parameters():
            total = torch.einsum("n,n...->...", coef, want[name])
            assert_rel(p.grad.reshape(1, -1), total.reshape(1, -1), REL, name)


def test_make_private_trains_with_poisson_batches_and_an_empty_one():
    from opacus_amd import PrivacyEngine

    torch.manual_seed(2)
    for mode in ("hooks", "ghost"):
        net = Net(1, False, 4).cuda()
        ids, y = data(16, 9)
        loader = torch.utils.data.DataLoader(torch.utils.data.TensorDataset(ids, y), batch_size=8)
        opt = torch.optim.SGD(net.parameters(), lr=0.05)
        if mode == "hooks":
            model, opt, loader = PrivacyEngine().make_private(
                module=net, optimizer=opt, data_loader=loader, noise_multiplier=1.0, max_grad_norm=1.0
            )
            crit = nn.CrossEntropyLoss()
        else:
            model, opt, crit, loader = PrivacyEngine().make_private(
                module=net, optimizer=opt, data_loader=loader, noise_multiplier=1.0, max_grad_norm=1.0,
                criterion=nn.CrossEntropyLoss(), grad_sample_mode="ghost",
            )
        before = [p.detach().clone() for p in net.parameters()]
        for bi, by in loader:
            opt.zero_grad()
            crit(model(bi.cuda()), by.cuda()).backward()
            opt.step()
        assert all(torch.isfinite(p).all() for p in net.parameters())
        assert all(not torch.equal(p, q) for p, q in zip(net.parameters(), before))
        opt.zero_grad()
        empty = model(ids[:0].cuda())
        if mode == "hooks":
            empty.sum().backward()
            for p in net.parameters():
                assert p.grad_sample.shape[0] == 0


def test_packed_sequences_follow_the_callers_order_and_layout():
    from opacus_amd import GradSampleModule

    torch.manual_seed(3)
    rnn = DPGatedRNN_(6, 24, 2, True, 4, False)
    lens = [4, 9, 1, 9]
    seqs = [torch.randn(k, 6) for k in lens]
    ref = copy.deepcopy(rnn).double()
    want_out, want_h, want_g = [], [], []
    for s in seqs:
        for p in ref.parameters():
            p.grad = None
        o, h = ref_rnn(ref, s[None].double())
        (o.pow(2).sum() + h.sum()).backward()
        want_out.append(o[0].detach())
        want_h.append(h.detach())
        want_g.append({n: p.grad.clone() for n, p in ref.named_parameters()})
    model = GradSampleModule(rnn.cuda(), batch_first=False, loss_reduction="sum")
    packed = nn.utils.rnn.pack_sequence([s.cuda() for s in seqs], enforce_sorted=False)
    out, h = model(packed)
    (out.data.pow(2).sum() + h.sum()).backward()
    padded, got_lens = nn.utils.rnn.pad_packed_sequence(out, batch_first=True)
    assert got_lens.tolist() == lens and h.dtype == torch.float32
    for k, n in enumerate(lens):
        assert_rel(padded[k, :n], want_out[k], REL, f"output {k}")
        assert_rel(h[:, k : k + 1], want_h[k], REL, f"state {k}")
    for name, p in rnn.named_parameters():
        assert_rel(p.grad_sample, torch.stack([g[name] for g in want_g]), REL, name)
    # a padded tensor with lengths gives the same, time first and batch first
    x = nn.utils.rnn.pad_sequence([s.cuda() for s in seqs])
    out2, h2 = rnn(x, lengths=torch.tensor(lens).cuda())
    for k, n in enumerate(lens):
        assert_rel(out2[:n, k], want_out[k], REL, f"padded output {k}")
    assert_rel(h2, h, 1e-6, "states")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_continue_a_forward_pass(dtype):
    torch.manual_seed(4)
    rnn = DPGatedRNN_(6, 24, 2, False, 4, True).cuda().to(dtype)
    x = torch.randn(3, 20, 6, device="cuda").to(dtype)
    whole, last = rnn(x)
    _, state = rnn(x[:, :12])
    state = state.detach().clone()
    for t in range(12, 20):
        y = rnn.step(x[:, t], state)
    # the projections' products may be summed in another order for one token: a few half-steps of each
    bar = {torch.float32: 1e-4, torch.bfloat16: 6e-2, torch.float16: 8e-3}[dtype]
    assert y.dtype == dtype and state.dtype == torch.float32
    assert_rel(y, whole[:, -1], bar, "output")
    assert_rel(state, last, bar, "state")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_group_norm_act_is_group_norm_and_activation(act):
    from opacus_amd import GradSampleModule
    from opacus_amd.layers import GroupNormAct

    torch.manual_seed(5)

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.conv = nn.Conv2d(3, 16, 3, padding=1)
            self.norm = GroupNormAct(4, 16, activation=act)
            self.fc = nn.Linear(16, 5)

        def forward(self, x):
            return self.fc(self.norm(self.conv(x)).mean((2, 3)))

        def reference(self, x, _length):
            y = ref_norm(self.norm, F.conv2d(x, self.conv.weight, self.conv.bias, padding=1))
            return self.fc(y.mean((2, 3)))

    net = Block()
    with torch.no_grad():
        net.norm.weight.add_(0.2 * torch.randn(16))
        net.norm.bias.add_(0.2 * torch.randn(16))
    x, y = torch.randn(4, 3, 7, 9), torch.randint(0, 5, (4,))
    want = per_sample_reference(net, x.double(), y)
    wrapped = GradSampleModule(net.cuda(), loss_reduction="mean")
    for xin in (x.cuda(), x.cuda().contiguous(memory_format=torch.channels_last)):
        for p in net.parameters():
            p.grad_sample = None
        F.cross_entropy(wrapped(xin), y.cuda()).backward()
        for name, p in net.named_parameters():
            assert_rel(p.grad_sample, want[name], REL, name)
    img = torch.randn(2, 16, 5, 6, device="cuda").contiguous(memory_format=torch.channels_last)
    out = net.norm(img)
    assert out.shape == img.shape and out.is_contiguous(memory_format=torch.channels_last)


def test_frozen_parameters_and_layers_used_twice():
    from opacus_amd import GradSampleModule
    from opacus_amd.layers import HeadNormAct

    torch.manual_seed(6)
    norm = HeadNormAct(2, 8).cuda()
    x = torch.randn(3, 4, 8, device="cuda")
    model = GradSampleModule(norm, loss_reduction="sum")
    model(x).sum().backward()
    gw, gb = norm.weight.grad_sample.clone(), norm.bias.grad_sample.clone()
    norm.weight.grad_sample = norm.bias.grad_sample = None
    norm.bias.requires_grad_(False)
    model(x).sum().backward()
    assert torch.equal(norm.weight.grad_sample, gw)
    norm.bias.requires_grad_(True)
    norm.weight.grad_sample = norm.bias.grad_sample = None
    (model(x).sum() + model(x).sum()).backward()
    assert_rel(norm.weight.grad_sample, 2 * gw, 1e-6, "weight")
    assert_rel(norm.bias.grad_sample, 2 * gb, 1e-6, "bias")


def test_plain_training_and_no_grad_need_no_hooks():
    from opacus_amd.layers import DPGatedRNN

    torch.manual_seed(8)
    rnn = DPGatedRNN(4, 8, num_heads=2, batch_first=True).cuda()
    x = torch.randn(2, 5, 4, device="cuda", requires_grad=True)
    out, h = rnn(x)
    h.sum().backward()  # only the state is used: the outputs have no gradient
    assert all(torch.isfinite(p.grad).all() for p in rnn.cells[0].scan.parameters()) and x.grad is not None
    assert "_dpk_param_rows" not in rnn.cells[0].scan.__dict__
    with torch.no_grad():
        assert torch.equal(rnn(x)[0], out)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(rnn(x)[0].sum(), x, create_graph=True)


def test_autocast_gives_bfloat16_gates_and_float32_parameters():
    from opacus_amd import GradSampleModule

    torch.manual_seed(9)
    net = Net(1, False, 4)
    ids, y = data(4, 20)
    want = per_sample_reference(net, ids, y)
    wrapped = GradSampleModule(net.cuda(), loss_reduction="sum")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = F.cross_entropy(wrapped(ids.cuda()).float(), y.cuda(), reduction="sum")
    loss.backward()
    for name in ("rnn.cells.0.scan.decay", "rnn.cells.0.norm.weight"):
        p = dict(net.named_parameters())[name]
        err = (p.grad_sample.double().cpu() - want[name]).norm() / want[name].norm()
        # bfloat16 gates, outputs and logits: a few of their half-steps (2**-8), most of which average out
        assert p.grad_sample.dtype == torch.float32 and err < 8 * 2**-8, (name, err)


def test_a_captured_training_pass_replays():
    """Forward and gradients inside one graph, on leaves that no other graph refers to."""
    from opacus_amd.layers import DPGatedRNN

    torch.manual_seed(10)
    rnn = DPGatedRNN(8, 16, num_heads=2, batch_first=True).cuda()
    x = torch.randn(2, 200, 8, device="cuda", requires_grad=True)
    leaves = [x] + list(rnn.parameters())

    def call():
        out, h = rnn(x)
        return torch.autograd.grad(out.float().pow(2).mean() + h.mean(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(2, 200, 8))
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert_rel(p.reshape(1, -1), q.reshape(1, -1), 1e-5, f"replay {k}")


def test_inference_mode_and_kernel_times():
    from opacus_amd import kernels
    from opacus_amd.layers import DPGatedRNN

    torch.manual_seed(11)
    rnn = DPGatedRNN(6, 24, 2, batch_first=True, num_heads=4).cuda()
    x = torch.randn(3, 9, 6, device="cuda")
    want, last = rnn(x)
    with torch.inference_mode(), kernels.record_kernel_times() as times:
        out, h = rnn(x[:, :8])
        y = rnn.step(x[:, 8], h)
        state = rnn.initial_state(3)
        for t in range(9):
            z = rnn.step(x[:, t], state)
    torch.cuda.synchronize()
    assert set(times) == {"gated_scan", "gated_scan_step", "group_norm_act"}
    assert all(s.elapsed_time(e) >= 0 for pairs in times.values() for s, e in pairs)
    for got in (y, z):
        assert_rel(got, want[:, -1], 1e-4, "output")
    assert_rel(state, last, 1e-4, "state")


def test_large_rows_take_the_clipped_sum_from_the_rows_again():
    """Per-sample gradients too large to be kept (KEEP_GRAD_SAMPLES_BELOW) are taken from the rows a second time."""
    from opacus_amd import GradSampleModuleFastGradientClipping
    from opacus_amd.layers import HeadNormAct
    from opacus_amd.optimizers import DPOptimizerFastGradientClipping
    from opacus_amd.utils.fast_gradient_clipping_utils import DPLossFastGradientClipping

    class Loss(nn.Module):
        reduction = "sum"

        def forward(self, out, tgt):
            l = (out - tgt).pow(2).flatten(1).sum(1)
            return l if self.reduction == "none" else l.sum()

    torch.manual_seed(12)
    grads = []
    for keep in (1 << 22, 0):
        torch.manual_seed(13)
        norm = HeadNormAct(4, 32).cuda()
        model = GradSampleModuleFastGradientClipping(norm, loss_reduction="sum", max_grad_norm=0.5)
        model.KEEP_GRAD_SAMPLES_BELOW = keep
        opt = DPOptimizerFastGradientClipping(
            torch.optim.SGD(norm.parameters(), lr=0.1), noise_multiplier=0.0, max_grad_norm=0.5, expected_batch_size=5,
            loss_reduction="sum",
        )
        x, t = torch.randn(5, 7, 32, device="cuda"), torch.randn(5, 7, 32, device="cuda")
        DPLossFastGradientClipping(model, opt, Loss(), loss_reduction="sum")(model(x), t).backward()
        grads.append([p.grad.clone() for p in norm.parameters()])
    for p, q in zip(*grads):
        assert torch.equal(p, q) and p.abs().max() > 0


class TimeFirst(nn.Module):
    """``[T, B, 6]`` inputs; a layer of each kind that keeps the samples along the second dimension."""

    def __init__(self):
        super().__init__()
        from opacus_amd.layers import HeadNormAct

        self.inp, self.norm = nn.Linear(6, 24), HeadNormAct(4, 24, activation="gelu")
        self.rnn = DPGatedRNN_(24, 24, 1, False, 3, False)
        self.out = nn.Linear(24, 5)

    def forward(self, x):
        return self.out(self.rnn(self.norm(self.inp(x)))[0])  # [T, B, 5]

    def reference(self, x):  # one sample [1, T, 6]
        z = ref_norm(self.norm, F.linear(x, self.inp.weight, self.inp.bias))
        return F.linear(ref_rnn(self.rnn, z)[0], self.out.weight, self.out.bias)


@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("T", [7, 5])  # as many positions as samples, too
def test_samples_along_the_second_dimension(T, reduction):
    from opacus_amd import GradSampleModule, GradSampleModuleFastGradientClipping

    torch.manual_seed(3)
    net = TimeFirst()
    with torch.no_grad():
        for p in net.norm.parameters():
            p.add_(0.3 * torch.randn(p.shape))
    x, mask = torch.randn(T, 5, 6), torch.randn(T, 5, 5)
    ref = copy.deepcopy(net).double()
    rows = []
    for k in range(5):
        ref.zero_grad(set_to_none=True)
        (ref.reference(x[:, k].double()[None])[0] * mask[:, k].double()).sum().backward()
        rows.append({n: p.grad.clone() for n, p in ref.named_parameters()})
    want = {n: torch.stack([r[n] for r in rows]) for n in rows[0]}
    plain = copy.deepcopy(net).cuda()(x.cuda())
    wrapped = GradSampleModule(copy.deepcopy(net).cuda(), batch_first=False, loss_reduction=reduction)
    out = wrapped(x.cuda())
    assert torch.equal(out, plain)
    loss = (out * mask.cuda()).sum()
    (loss / 5 if reduction == "mean" else loss).backward()
    for name, p in wrapped._module.named_parameters():
        assert_rel(p.grad_sample, want[name], REL, name)
    ghost = GradSampleModuleFastGradientClipping(
        copy.deepcopy(net).cuda(), batch_first=False, loss_reduction=reduction, max_grad_norm=1.0, use_ghost_clipping=True
    )
    loss = (ghost(x.cuda()) * mask.cuda()).sum()
    (loss / 5 if reduction == "mean" else loss).backward()
    norms = sum(w.flatten(1).square().sum(1) for w in want.values()).sqrt()
    assert_rel(ghost.get_norm_sample()[None], norms[None], REL, "norms")
    with pytest.raises(ValueError, match="batch_first=False"):
        wrapped._module.norm(torch.zeros(5, 24, device="cuda"))


# ---- what an optimizer step leaves, with no noise in it -------------------------------------------
def clipped_sum(want, C):
    norms = torch.stack([g.flatten(1).norm(dim=1) for g in want.values()]).norm(dim=0)
    coef = (C / (norms + 1e-6)).clamp(max=1.0)
    return norms, {k: torch.einsum("n,n...->...", coef, g) for k, g in want.items()}


@pytest.mark.parametrize("mode", ["hooks", "ghost"])
def test_make_private_without_noise_applies_the_clipped_sum(mode):
    """Poisson batches, the update against the formula's; then an empty batch, which changes nothing."""
    from opacus_amd import PrivacyEngine

    torch.manual_seed(14)
    net = Net(1, False, 4)
    ref = copy.deepcopy(net)
    net = net.cuda()
    ids, y = data(16, 9)
    loader = torch.utils.data.DataLoader(torch.utils.data.TensorDataset(ids, y), batch_size=8)
    settings = dict(
        module=net, optimizer=torch.optim.SGD(net.parameters(), lr=0.05), data_loader=loader, noise_multiplier=0.0,
        max_grad_norm=0.5, grad_sample_mode=mode,
    )
    if mode == "hooks":
        model, opt, loader = PrivacyEngine().make_private(**settings)
        crit = nn.CrossEntropyLoss()
    else:
        model, opt, crit, loader = PrivacyEngine().make_private(criterion=nn.CrossEntropyLoss(), **settings)
    batches = [(bi, by) for bi, by in loader if len(bi)][:3] + [(ids[:0], y[:0])]
    assert len(batches) > 1
    for bi, by in batches:
        before = {k: p.detach().clone() for k, p in net.named_parameters()}
        opt.zero_grad()
        crit(model(bi.cuda()), by.cuda()).backward()
        if len(bi) == 0:
            if mode == "hooks":
                assert all(p.grad_sample.shape[0] == 0 for p in net.parameters())
            else:
                assert model.per_sample_gradient_norms.shape == (0,)
            opt.step()
            assert all(torch.equal(p, before[k]) for k, p in net.named_parameters())
            continue
        ref.load_state_dict({k: v.cpu() for k, v in before.items()})
        norms, want = clipped_sum(per_sample_reference(ref, bi, by), 0.5)
        assert (norms > 0.5).any()
        opt.step()
        for k, p in net.named_parameters():
            assert_rel(p.grad.reshape(1, -1), want[k].reshape(1, -1) / 8, REL, k)
            # the product and the difference, each rounded once
            step = 0.05 * p.grad.double()
            assert ((p.double() - (before[k].double() - step)).abs() <= 2**-23 * (before[k].double().abs() + step.abs())).all()


@pytest.mark.parametrize("channels_last", [False, True])
@pytest.mark.parametrize("single", [True, False])
def test_group_norm_act_under_ghost_clipping(single, channels_last):
    from opacus_amd import GradSampleModuleFastGradientClipping
    from opacus_amd.layers import GroupNormAct
    from opacus_amd.optimizers import DPOptimizerFastGradientClipping
    from opacus_amd.utils.fast_gradient_clipping_utils import DPLossFastGradientClipping

    torch.manual_seed(15)

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.conv, self.norm, self.fc = nn.Conv2d(3, 16, 3, padding=1), GroupNormAct(4, 16, activation="gelu"), nn.Linear(16, 5)

        def forward(self, x):
            return self.fc(self.norm(self.conv(x)).mean((2, 3)))

        def reference(self, x, _length):
            return self.fc(ref_norm(self.norm, F.conv2d(x, self.conv.weight, self.conv.bias, padding=1)).mean((2, 3)))

    net = Block()
    with torch.no_grad():
        net.norm.weight.add_(0.2 * torch.randn(16))
        net.norm.bias.add_(0.2 * torch.randn(16))
    x, y = torch.randn(5, 3, 7, 9), torch.randint(0, 5, (5,))
    want = per_sample_reference(net, x.double(), y)
    C = float(torch.stack([g.flatten(1).norm(dim=1) for g in want.values()]).norm(dim=0).median())
    norms, total = clipped_sum(want, C)
    model = GradSampleModuleFastGradientClipping(net.cuda(), loss_reduction="mean", max_grad_norm=C, single_backward=single)
    opt = DPOptimizerFastGradientClipping(
        torch.optim.SGD(net.parameters(), lr=0.1), noise_multiplier=0.0, max_grad_norm=C, expected_batch_size=5
    )
    crit = DPLossFastGradientClipping(model, opt, nn.CrossEntropyLoss(), loss_reduction="mean")
    xin = x.cuda().contiguous(memory_format=torch.channels_last) if channels_last else x.cuda()
    for _ in range(2):
        opt.zero_grad()
        crit(model(xin), y.cuda()).backward()
        assert_rel(model.per_sample_gradient_norms, norms, REL, "norms")
        for name, p in net.named_parameters():
            assert_rel(p.grad.reshape(1, -1), total[name].reshape(1, -1), REL, name)


# ---- initial states, dropout ----------------------------------------------------------------------
def rnn_rows(ref, seqs, state, middle=None):
    """Per sample: outputs, last states, gradients of the state and of every parameter, for the loss
    ``sum out^2 + sum h * (1, 2, ..)``. ``middle[k]``: what dropout multiplies sample k's second layer's input by."""
    res = []
    weight = torch.arange(1.0, 1 + len(ref.cells), dtype=torch.float64)[:, None, None]
    for k, s in enumerate(seqs):
        ref.zero_grad(set_to_none=True)
        init = state[:, k : k + 1].detach().clone().double().requires_grad_(True)
        if middle is None:
            o, h = ref_rnn(ref, s[None].double(), init)
        else:
            half = ref.num_directions
            first, last = (SimpleNamespace(num_layers=1, num_directions=half, cells=c) for c in (ref.cells[:half], ref.cells[half:]))
            o, h0 = ref_rnn(first, s[None].double(), init[:half])
            o, h1 = ref_rnn(last, o * middle[k : k + 1], init[half:])
            h = torch.cat([h0, h1])
        (o.pow(2).sum() + (h * weight).sum()).backward()
        res.append((o[0].detach(), h.detach(), init.grad, {n: p.grad.clone() for n, p in ref.named_parameters()}))
    return res


def check_rnn(rnn, out_rows, h, state, res):
    for k, (o, hk, gk, _) in enumerate(res):
        assert_rel(out_rows[k], o, REL, f"output {k}")
        assert_rel(h[:, k : k + 1], hk, REL, f"last state {k}")
        assert_rel(state.grad[:, k : k + 1], gk, REL, f"gradient of state {k}")
    for name, p in rnn.named_parameters():
        assert_rel(p.grad_sample, torch.stack([r[3][name] for r in res]), REL, name)


def rnn_loss(data_, h):
    return data_.pow(2).sum() + (h * torch.arange(1.0, 1 + len(h), device=h.device)[:, None, None]).sum()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("batch_first", [False, True])
def test_initial_states_of_every_layer_and_direction(batch_first, packed):
    from opacus_amd import GradSampleModule

    torch.manual_seed(16)
    rnn = DPGatedRNN_(6, 24, 2, True, 4, batch_first)
    lens = [4, 9, 1, 8] if packed else [7] * 4  # (packed order: samples 1, 3, 0, 2)
    seqs, start = [torch.randn(k, 6) for k in lens], torch.randn(4, 4, 24)
    res = rnn_rows(copy.deepcopy(rnn).double(), seqs, start)
    model = GradSampleModule(rnn.cuda(), batch_first=batch_first, loss_reduction="sum")
    state = start.cuda().requires_grad_(True)
    if packed:
        out, h = model(nn.utils.rnn.pack_sequence([s.cuda() for s in seqs], enforce_sorted=False), state)
        rnn_loss(out.data, h).backward()
        padded = nn.utils.rnn.pad_packed_sequence(out, batch_first=True)[0]
        rows = [padded[k, :n] for k, n in enumerate(lens)]
    else:
        x = torch.stack(seqs, 0 if batch_first else 1).cuda()
        out, h = model(x, state)
        rnn_loss(out, h).backward()
        rows = out if batch_first else out.transpose(0, 1)
    check_rnn(rnn, rows, h, state, res)


def test_dropout_acts_between_the_layers_only():
    from opacus_amd import GradSampleModule
    from opacus_amd.layers import DPGatedRNN

    torch.manual_seed(17)
    rnn = DPGatedRNN(6, 24, 2, batch_first=True, dropout=0.5, num_heads=4)
    seqs, start = [torch.randn(7, 6) for _ in range(3)], torch.randn(2, 3, 24)
    ref = copy.deepcopy(rnn).double()
    model = GradSampleModule(rnn.cuda(), loss_reduction="sum")
    kept = []
    rnn.dropout_layer.register_forward_hook(lambda _m, _i, o: kept.append((o != 0).double().cpu() * 2))
    state = start.cuda().requires_grad_(True)
    out, h = model(torch.stack(seqs).cuda(), state)
    rnn_loss(out, h).backward()
    assert len(kept) == 1 and 0.2 < float(kept[0].mean()) / 2 < 0.8
    check_rnn(rnn, out, h, state, rnn_rows(ref, seqs, start, kept[0]))
    model.eval()
    with torch.no_grad():
        out, _ = model(torch.stack(seqs).cuda(), state)
    for k, (o, *_rest) in enumerate(rnn_rows(ref, seqs, start)):
        assert_rel(out[k], o, REL, f"output {k} in evaluation")
