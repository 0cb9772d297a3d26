"""Group norm + activation on channels-last tensors in float64, with a bound for what float32 adds.

Tolerances, in half-steps ``H = 2**-24``. A sum of N terms is taken as a tree whose longest path has
P = 264 roundings (up to 256 row groups in a row plus the terms of one thread), so it is off by at
most P H times the sum of its terms' magnitudes. With sum|x| / N = M and var the variance:
  mean: (P + 2) H M;  rstd: (P / 2 + 6) H of itself (the variance's relative error halves), plus the
  mean's error squared over the variance;  xh: mean error * rstd + (P / 2 + 8) H |xh|;  z: |w| times that + 2 H (|w xh| + |b|)
  act(z): its slope is at most 1.13, its own evaluation 24 H (|z| + |act|) (sigmoid 17, erf 4)
  act'(z): |act''| is at most 1, its own evaluation 60 H (1 + |z|); relu's slope is undecided within the error of z
Every output in bfloat16 adds half a step (2**-8 of the value) for its one rounding.
"""

import math

import torch

H = 2.0**-24
P = 264


def half_step(dtype):
    return {torch.float32: H, torch.bfloat16: 2.0**-8}[dtype]


def act_and_slope(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    return z, torch.ones_like(z)


def norm_act_reference(x, groups, weight, bias, eps, act, per_position, grad_out=None):
    """Dicts (values, tolerances) of float64 CPU tensors: y and, with ``grad_out``, grad_x,
    grad_weight and grad_bias (per sample)."""
    hs = half_step(x.dtype)
    n, C = x.shape[0], x.shape[-1]
    v = x.detach().double().cpu().reshape(n, -1, groups, C // groups)
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    w, b = w.reshape(groups, -1), b.reshape(groups, -1)
    dims = (3,) if per_position else (1, 3)
    mean = v.mean(dims, keepdim=True)
    var = (v - mean).pow(2).mean(dims, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (v - mean) * rstd
    z = xh * w + b
    y, sl = act_and_slope(z, act)
    mean_t = (P + 2) * H * v.abs().mean(dims, keepdim=True)
    rstd_r = (P / 2 + 6) * H + (mean_t * rstd).pow(2)
    xh_t = mean_t * rstd + (rstd_r + 2 * H) * xh.abs()
    z_t = w.abs() * xh_t + 2 * H * ((w * xh).abs() + b.abs())
    y_t = 1.13 * z_t + 24 * H * (z.abs() + y.abs())
    val = {"y": y.reshape(x.shape)}
    tol = {"y": (y_t + hs * (y.abs() + y_t)).reshape(x.shape)}
    if grad_out is None:
        return val, tol
    dy = grad_out.detach().double().cpu().reshape(v.shape)
    dz = dy * sl
    sl_t = z_t + 60 * H * (1 + z.abs())
    if act == "relu":
        sl_t = (z.abs() <= z_t).double()
    elif act == "none":
        sl_t = torch.zeros_like(z)
    dz_t = dy.abs() * sl_t + 2 * H * dz.abs()
    gb, gw = dz.sum(1), (dz * xh).sum(1)
    val["grad_bias"], val["grad_weight"] = gb.reshape(n, C), gw.reshape(n, C)
    tol["grad_bias"] = (dz_t.sum(1) + P * H * dz.abs().sum(1)).reshape(n, C)
    dxh_abs = (dz * xh).abs()
    tol["grad_weight"] = ((dz_t * xh.abs() + dz.abs() * xh_t).sum(1) + P * H * dxh_abs.sum(1)).reshape(n, C)
    d, d_t = dz * w, dz_t * w.abs()
    s1, s2 = d.mean(dims, keepdim=True), (d * xh).mean(dims, keepdim=True)
    s1_t = d_t.mean(dims, keepdim=True) + 2 * P * H * d.abs().mean(dims, keepdim=True)
    s2_t = (d_t * xh.abs() + d.abs() * xh_t).mean(dims, keepdim=True) + 2 * P * H * (d * xh).abs().mean(dims, keepdim=True)
    dx = rstd * (d - s1 - xh * s2)
    dx_t = rstd * (d_t + s1_t + xh.abs() * s2_t + xh_t * s2.abs() + (rstd_r + 4 * H) * (d.abs() + s1.abs() + (xh * s2).abs()))
    val["grad_x"], tol["grad_x"] = dx.reshape(x.shape), (dx_t + hs * (dx.abs() + dx_t)).reshape(x.shape)
    return val, tol
