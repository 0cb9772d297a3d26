"""What is measured of the recurrent layer's operators: the gated scan (forward, forward + backward,
one token) and the group norm with an activation on channels-last tensors (statistics per sample
and per position, forward and forward + backward, with per-sample parameter gradients).

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the calls of
``opacus_amd.kernels``.
"""

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---- the cases ----------------------------------------------------------------------------------
def listed():
    return [
        # one sequence answered token by token: what one layer costs per token
        dict(name="step_b1", op="step", n=1, d=2048, dtype="bf16"),
        # a full batch of sequences decoded together, an odd batch and width
        dict(name="step_b250", op="step", n=250, d=1000, dtype="fp32"),
        # one long prompt: few rows, the time axis is all the parallelism there is
        dict(name="scan_prompt_16k", op="scan", n=1, t=16384, d=2048, dtype="bf16", ragged=False, reverse=False, state=False),
        # a padded batch of prompts of odd lengths (none at all and one token among them), with states to go on from
        dict(name="scan_padded", op="scan", n=12, t=1027, d=1000, dtype="fp32", ragged=True, reverse=False, state=True),
        # training at the decoder's shape: batch 16, sequence 1024, width 2048
        dict(name="scan_train", op="scan_train", n=16, t=1024, d=2048, dtype="bf16", ragged=False, reverse=False, state=False),
        # training on long documents, two at a time
        dict(name="scan_train_8k", op="scan_train", n=2, t=8192, d=2048, dtype="bf16", ragged=False, reverse=False, state=False),
        # a small padded batch of a bidirectional layer: the reverse direction, odd sizes, a state
        dict(name="scan_train_padded", op="scan_train", n=7, t=333, d=130, dtype="fp32", ragged=True, reverse=True, state=True),
        # heads of one token a sequence, decoded together
        dict(name="norm_token", op="norm", n=64, s=1, c=2048, groups=16, dtype="bf16", act="silu", per_position=True),
        # heads of a training batch of tokens: batch 16, sequence 1024, width 2048
        dict(name="norm_token_train", op="norm_train", n=16, s=1024, c=2048, groups=16, dtype="bf16", act="silu", per_position=True),
        # the ResNet block's norm: batch 256, 64 channels, 32 x 32, 32 groups
        dict(name="norm_block_train", op="norm_train", n=256, s=1024, c=64, groups=32, dtype="fp32", act="silu", per_position=False),
        # large feature maps, few of them
        dict(name="norm_map_train", op="norm_train", n=3, s=40000, c=128, groups=32, dtype="bf16", act="gelu", per_position=False),
        # small feature maps with an odd channel count, forward only
        dict(name="norm_odd", op="norm", n=33, s=49, c=210, groups=14, dtype="fp32", act="gelu", per_position=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


_SCAN_MOST = 16 * 1024 * 2048  # elements of the largest listed scans
_NORM_MOST = 16 * 1024 * 2048


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "norm", "norm_train", "norm_train"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "step":
        return dict(op=op, n=_log_int(rng, 1, 256), d=_log_int(rng, 64, 2048), dtype=dtype)
    if op in ("scan", "scan_train"):
        d = _log_int(rng, 64, 2048)
        if rng.random() < 0.5:
            d = -(-d // 64) * 64
        t = _log_int(rng, 1, 16384 if op == "scan" else 8192)
        n = _log_int(rng, 1, max(1, min(64, _SCAN_MOST // (t * d))))
        return dict(op=op, n=n, t=t, d=d, dtype=dtype, ragged=rng.random() < 0.5, reverse=rng.random() < 0.3,
                    state=rng.random() < 0.5)
    act = rng.choice(["silu", "gelu", "none"])
    if rng.random() < 0.5:
        groups = rng.choice([1, 2, 3, 5, 8, 16, 32])
        c = groups * (rng.choice([32, 64, 128]) if rng.random() < 0.6 else _log_int(rng, 4, 130))
        s = _log_int(rng, 1, 4096)
        n = _log_int(rng, 1, max(1, min(64, _NORM_MOST // (s * c))))
        return dict(op=op, n=n, s=s, c=c, groups=groups, dtype=dtype, act=act, per_position=True)
    groups = rng.choice([1, 4, 7, 16, 32])
    c = groups * rng.choice([2, 3, 4, 5, 8, 16])
    s = _log_int(rng, 4, 65536)
    n = _log_int(rng, 1, max(1, min(256, _NORM_MOST // (s * c))))
    return dict(op=op, n=n, s=s, c=c, groups=groups, dtype=dtype, act=act, per_position=False)


# ---- what a program has in hand -----------------------------------------------------------------
def _inputs(case, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    st = dict(case)
    n = case["n"]
    if case["op"] in ("step", "scan", "scan_train"):
        d = case["d"]
        t = case.get("t", 1)
        gates = normal(n, t, 3 * d).to(dt)
        # a half-open gate decays by 0.9 to 0.999 a token, as the layer starts out
        a0 = 0.9 + 0.099 * torch.rand(d, generator=g, device=device)
        st["decay"] = torch.log(torch.expm1(-2.0 * torch.log(a0)))
        if case["op"] == "step":
            st["gates"] = gates[:, 0].contiguous()
            st["state"] = normal(n, d)
            return st
        st["gates"] = gates
        st["state"] = normal(n, d) if case["state"] else None
        st["lengths"] = None
        if case["ragged"]:
            lengths = torch.randint(0, t + 1, (n,), generator=g, device=device)
            lengths[0] = t
            if n > 1:
                lengths[1] = 0
            if n > 2:
                lengths[2] = 1
            st["lengths"] = lengths
        if case["op"] == "scan_train":
            st["grad"] = (0.02 * normal(n, t, d)).to(dt)
        return st
    s, c = case["s"], case["c"]
    # activations with a mean of their own per channel and sample
    st["x"] = (normal(n, s, c) * (0.5 + torch.rand(c, generator=g, device=device)) + normal(n, 1, c)).to(dt)
    st["weight"] = 1.0 + 0.1 * normal(c)
    st["bias"] = 0.1 * normal(c)
    if case["op"] == "norm_train":
        st["grad"] = (0.02 * normal(n, s, c)).to(dt)
    return st


_EPS = 1e-5


def prepare(case, seed):
    return _inputs(case, seed, torch.device("cuda"))


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "step":
        return _plain_step(state)
    if state["op"] in ("scan", "scan_train"):
        return _plain_scan(state)
    return _plain_norm(state)


def _run_own(st):
    from opacus_amd import kernels

    op = st["op"]
    if op == "step":
        # the state is advanced in place, as a decoding loop keeps it
        out = kernels.gated_scan_step(st["gates"], st["decay"], st["state"])
        return {"out": out, "state": st["state"]}
    if op in ("scan", "scan_train"):
        train = op == "scan_train"
        kw = dict(lengths=st["lengths"], reverse=st["reverse"])
        out, last, kept = kernels.gated_scan(st["gates"], st["decay"], st["state"], keep_states=train, **kw)
        res = {"out": out, "last": last}
        if train:
            d_gates, d_decay, d_state = kernels.gated_scan_backward(st["gates"], st["decay"], kept, st["grad"], **kw)
            res.update(d_gates=d_gates, d_decay=d_decay)
            if st["state"] is not None:
                res["d_state"] = d_state
        return res
    args = (st["groups"], st["weight"], st["bias"], _EPS, st["act"])
    y, stats = kernels.group_norm_act(st["x"], *args, per_position=st["per_position"])
    if op == "norm":
        return {"y": y}
    dx, dw, db = kernels.group_norm_act_backward(st["x"], st["grad"], stats, *args, per_position=st["per_position"])
    return {"y": y, "dx": dx, "d_weight": dw, "d_bias": db}


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _plain_gates(gates, decay):
    """x, sigma(r), sigma(i), log a, 1 - a, sqrt(1 - a^2) of packed gates, in 32 bits."""
    d = decay.shape[0]
    x, r, i = gates.float().split(d, dim=-1)
    sp = torch.clamp(decay, min=0.0) + torch.log1p(torch.exp(-decay.abs()))
    rho, s = _sigmoid(r), _sigmoid(i)
    log_a = -sp * rho
    q = -torch.expm1(log_a)
    return x, rho, s, log_a, q, torch.sqrt(q * (2.0 - q)), sp


def _plain_step(st):
    x, _rho, s, _log_a, q, m, _sp = _plain_gates(st["gates"], st["decay"])
    h = st["state"]
    h.copy_(h - q * h + m * s * x)
    return {"out": h.to(st["gates"].dtype), "state": h}


def _plain_scan(st):
    gates, decay = st["gates"], st["decay"]
    n, t, d = st["n"], st["t"], st["d"]
    x, rho, s, log_a, q, m, sp = _plain_gates(gates, decay)
    live = None
    if st["lengths"] is not None:
        live = (torch.arange(t, device=gates.device) < st["lengths"][:, None])[:, :, None]
        zero = torch.zeros((), device=gates.device)
        x, log_a, q, m = (torch.where(live, v, zero) for v in (x, log_a, q, m))
    a = torch.where(q < 0.5, 1.0 - q, torch.exp(log_a))
    u = m * s * x
    order = range(t - 1, -1, -1) if st["reverse"] else range(t)
    h = st["state"] if st["state"] is not None else torch.zeros(n, d, device=gates.device)
    prev = torch.empty(n, t, d, device=gates.device)
    hs = torch.empty(n, t, d, device=gates.device)
    for k in order:
        prev[:, k] = h
        h = a[:, k] * h + u[:, k]
        hs[:, k] = h
    out = hs if live is None else torch.where(live, hs, torch.zeros_like(hs))
    res = {"out": out.to(gates.dtype), "last": h}
    if st["op"] == "scan":
        return res
    gy = st["grad"].float()
    if live is not None:
        gy = torch.where(live, gy, torch.zeros_like(gy))
    g = torch.zeros(n, d, device=gates.device)
    gs = torch.empty(n, t, d, device=gates.device)
    for k in reversed(order):
        g = gy[:, k] + g
        gs[:, k] = g
        g = a[:, k] * g
    kappa = torch.where(m > 0, -log_a / m, torch.zeros_like(m))
    dx = gs * m * s
    di = dx * x * (1.0 - s)
    w = gs * (log_a * a * prev + s * x * a * a * kappa)
    dr = w * (1.0 - rho)
    res["d_gates"] = torch.cat([dx, dr, di], dim=2).to(gates.dtype)
    res["d_decay"] = w.sum(dim=1) * (_sigmoid(decay) / sp)
    if st["state"] is not None:
        res["d_state"] = g
    return res


def _act(z, act):
    """act(z) and its derivative."""
    if act == "silu":
        s = _sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return z, torch.ones_like(z)


def _plain_norm(st):
    x = st["x"]
    n, s, c = x.shape
    groups = st["groups"]
    xf = x.float().reshape(n, s, groups, c // groups)
    dims = (3,) if st["per_position"] else (1, 3)
    centred = xf - xf.mean(dim=dims, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=dims, keepdim=True) + _EPS)
    xh = centred * rstd
    w, b = st["weight"].reshape(groups, -1), st["bias"].reshape(groups, -1)
    y, slope = _act(xh * w + b, st["act"])
    res = {"y": y.reshape(n, s, c).to(x.dtype)}
    if st["op"] == "norm":
        return res
    dz = st["grad"].float().reshape(n, s, groups, c // groups) * slope
    dxh = dz * w
    dx = rstd * (dxh - dxh.mean(dim=dims, keepdim=True) - xh * (dxh * xh).mean(dim=dims, keepdim=True))
    res["dx"] = dx.reshape(n, s, c).to(x.dtype)
    res["d_weight"] = (dz * xh).sum(dim=1).reshape(n, c)
    res["d_bias"] = dz.sum(dim=1).reshape(n, c)
    return res


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    n, op = case["n"], case["op"]
    if op == "step":
        d = case["d"]
        return {"bytes": n * d * (4 * e + 8) + 4 * d, "flops": 40 * n * d}
    if op in ("scan", "scan_train"):
        t, d = case["t"], case["d"]
        # half the positions of a padded batch are inputs (its outputs are written whole)
        live = 0.5 if case["ragged"] else 1.0
        el = n * t * d
        b = el * e * (3 * live + 1) + 4 * n * d * (2 if case["state"] else 1) + 4 * d
        f = 40 * el * live
        if op == "scan_train":
            b += el * e * (live + 3) + 4 * n * d * (2 if case["state"] else 1)
            f += 60 * el * live
        return {"bytes": int(b), "flops": int(f)}
    s, c = case["s"], case["c"]
    el = n * s * c
    if op == "norm":
        return {"bytes": 2 * el * e + 8 * c, "flops": 25 * el}
    return {"bytes": 4 * el * e + 8 * c + 8 * n * c, "flops": 70 * el}


# ---- the definition in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    """The definition evaluated in float64, gradients by automatic differentiation of it."""
    st = prepare(case, seed)
    if case["op"] in ("step", "scan", "scan_train"):
        return _exact_scan(case, st)
    return _exact_norm(case, st)


def _exact_scan(case, st):
    train = case["op"] == "scan_train"
    d = case["d"]
    gates = st["gates"].double()
    if case["op"] == "step":
        gates = gates[:, None]
    n, t = gates.shape[:2]
    rows = st["decay"].double().expand(n, d).clone()
    h0 = st["state"].double() if st["state"] is not None else torch.zeros(n, d, dtype=torch.float64, device=gates.device)
    if train:
        for v in (gates, rows, h0):
            v.requires_grad_(True)
    decay_rate = torch.logaddexp(rows, torch.zeros_like(rows))[:, None]
    log_a = -decay_rate * torch.sigmoid(gates[..., d : 2 * d])
    a = log_a.exp()
    u = (-torch.expm1(2.0 * log_a)).sqrt() * torch.sigmoid(gates[..., 2 * d :]) * gates[..., :d]
    lengths = st.get("lengths")
    ends = torch.full((n,), t, device=gates.device) if lengths is None else lengths
    h, hs = h0, [None] * t
    a_t, u_t = a.unbind(1), u.unbind(1)
    blank = torch.zeros_like(h0)
    for k in reversed(range(t)) if case.get("reverse") else range(t):
        new = torch.addcmul(u_t[k], a_t[k], h)
        if lengths is None:
            h = hs[k] = new
        else:
            on = (ends > k)[:, None]
            h = torch.where(on, new, h)
            hs[k] = torch.where(on, new, blank)
    if case["op"] == "step":
        return {"out": h, "state": h}
    out = torch.stack(hs, dim=1)
    res = {"out": out.detach(), "last": h.detach()}
    if train:
        wanted = [gates, rows] + ([h0] if case["state"] else [])
        grads = torch.autograd.grad(out, wanted, st["grad"].double())
        res.update(zip(("d_gates", "d_decay", "d_state"), grads))
    return res


def _exact_norm(case, st):
    train = case["op"] == "norm_train"
    x = st["x"].double()
    n, s, c = x.shape
    w, b = (v.double().expand(n, 1, c).clone() for v in (st["weight"], st["bias"]))
    if train:
        for v in (x, w, b):
            v.requires_grad_(True)
    grouped = x.unflatten(2, (case["groups"], -1))
    dims = [3] if case["per_position"] else [1, 3]
    var, mean = torch.var_mean(grouped, dim=dims, correction=0, keepdim=True)
    z = ((grouped - mean) * (var + _EPS).rsqrt()).flatten(2) * w + b
    if case["act"] == "silu":
        y = z * torch.sigmoid(z)
    elif case["act"] == "gelu":
        y = 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    else:
        y = z
    res = {"y": y.detach()}
    if train:
        dx, dw, db = torch.autograd.grad(y, (x, w, b), st["grad"].double())
        res.update(dx=dx, d_weight=dw.reshape(n, c), d_bias=db.reshape(n, c))
    return res
