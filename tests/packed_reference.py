"""Packed attention in 64 bits from its definition, with bounds of what rounding may change."""

import math

import torch


def attention64(q, k, v, lens, scale=None, do=None):
    """Outputs (o[, dq, dk, dv]) in fp64 and, of the same shapes, bounds of the error of kernels that
    round their softmax weights and score gradients once to the operands' type and results once more.

    With u = finfo.eps / 2 of the type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and r the relative error of a softmax
    weight before that rounding:
      o:  (u + r) sum_j P |v| + u |o|
      delta = o . do is formed from the rounded o: its error is at most e = (2 u + r) sum_d |o| |do|, so
      dS: (u + r) |dS| + P (e + r' sum |do| |v|);  dq, dk: the sums of that against |k|, |q|, times scale; dv like o.
    fp16 has a smallest step of 2^-24, so rounding is off by up to 2^-25 however small the value is. The kernels
    round P times 2^10: 2^-35 of P. They round dS times a power of two f that brings the largest |do| of its rows to
    [1/2, 1): with f >= 1 / (2 max |do|) that is 2^-25 / f <= 2^-24 max |do| of dS.
    r: the scores are fp32 sums of D products (D 2^-24 of the absolute sum), a sum over n keys adds n 2^-24,
    and the exponential and the final division a few more.
    """
    rows, hq, d = q.shape
    hk = k.shape[1]
    group = hq // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    f = torch.finfo(torch.float32).eps / 2
    step_p = step_ds = 0.0
    if q.dtype == torch.float16 and do is not None:
        step_p, step_ds = 2.0**-35, 2.0**-24 * do.abs().nan_to_num(0, 0, 0).max().item()
    names = ["o"] + (["dq", "dk", "dv"] if do is not None else [])
    shapes = {"o": q.shape, "dq": q.shape, "dk": k.shape, "dv": k.shape}
    out = {n: torch.zeros(shapes[n], dtype=torch.float64, device=q.device) for n in names}
    tol = {n: torch.zeros(shapes[n], dtype=torch.float64, device=q.device) for n in names}
    at = 0
    for n in lens:
        r_ = slice(at, at + n)
        at += n
        if n == 0:
            continue
        Q = q[r_].double().transpose(0, 1)
        K = k[r_].double().transpose(0, 1).repeat_interleave(group, 0)
        V = v[r_].double().transpose(0, 1).repeat_interleave(group, 0)
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        S = (Q @ K.mT * scale).masked_fill(hidden, -math.inf)
        P = torch.softmax(S, -1)
        absS = (Q.abs() @ K.abs().mT * scale).masked_fill(hidden, 0.0)
        r = 2 * ((d + 8) * f * absS.amax() + (n + 16) * f) + 16 * f
        O = P @ V
        A = P @ V.abs()
        out["o"][r_] = O.transpose(0, 1)
        tol["o"][r_] = ((u + r) * A + u * O.abs()).transpose(0, 1)
        if do is None:
            continue
        G = do[r_].double().transpose(0, 1)
        dP = G @ V.mT
        delta = (O * G).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        e = (2 * u + r) * (A * G.abs()).sum(-1, keepdim=True) + (d + 8) * f * (G.abs() @ V.abs().mT)
        eS = (u + r) * dS.abs() + P * e + (step_ds * ~hidden)
        dQ, eQ = scale * dS @ K, scale * eS @ K.abs()
        dK, eK = scale * dS.mT @ Q, scale * eS.mT @ Q.abs()
        dV, eV = P.mT @ G, ((u + r) * P + step_p * ~hidden).mT @ G.abs()
        s = (n * group + 16) * f  # the sum over the rows and the heads of a group
        aQ, aK, aV = scale * dS.abs() @ K.abs(), scale * dS.abs().mT @ Q.abs(), P.mT @ G.abs()
        out["dq"][r_] = dQ.transpose(0, 1)
        tol["dq"][r_] = (eQ + s * aQ + u * dQ.abs()).transpose(0, 1)
        for name, x, ex, ax in (("dk", dK, eK, aK), ("dv", dV, eV, aV)):
            x = x.reshape(hk, group, n, d).sum(1)
            ex = (ex + s * ax).reshape(hk, group, n, d).sum(1) + u * x.abs()
            out[name][r_] = x.transpose(0, 1)
            tol[name][r_] = ex.transpose(0, 1)
    return out, tol


def assert_within(got, want, tol, what="", factor=1.0, floor=1e-30):
    """|got - want| <= factor * tol + floor everywhere (NaN fails)."""
    diff = (got.double() - want).abs()
    bad = ~(diff <= factor * tol + floor)
    if bad.any():
        i = (diff / (factor * tol + floor)).nan_to_num(nan=1e300).reshape(-1).argmax().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst at {i}: got "
                             f"{got.reshape(-1)[i].item()}, want {want.reshape(-1)[i].item()}, "
                             f"bound {tol.reshape(-1)[i].item()}")
