"""Bounds of the packed attention's errors that hold document by document."""

import math

import torch


def attention_bounds64(q, k, v, lens, do, scale=None, exact_weights=False):
    """Outputs (o, dq, dk, dv) in fp64 and bounds of the kernels' errors, with u = finfo.eps / 2 of the type, f that
    of fp32, r the relative error of a softmax weight before it is rounded (scores are fp32 sums of D products, a
    sum over n keys adds n f, the exponential and the division a few more), A = P |v|:

      o:      (u + r) A + u |o|
      delta:  |do| . w + (D + 8) f |do| . |o|.  16 bits: w = (u + r) A + u^2 |o|, as what rounding took from o is kept and
              rounded in its turn (fp16: off by up to 2^-25 however small it is).  fp32: w = (2 u + r) A.
      dS:     (u + r) |dS| + P (delta's error + (D + 8) f |do| . |v|)
      dq, dk: the sums of that against |k|, |q|, times scale; dv: (u + r) P against |do|; then one rounding.

    fp16 has a smallest step of 2^-24.  P is rounded times 2^10: off by up to 2^-35.  dS is rounded times a power of two
    that brings B, a bound of |do . v - delta| over the rows and keys concerned, to [2^14, 2^15): off by up to
    2^-25 B / 2^14.  B is at most max sum|do| max|v| + max|delta| of the document's own rows and heads.

    `exact_weights`: all scores are zero, so that the forward pass rounds weights of 1, which is exact.
    """
    rows, hq, d = q.shape
    hk = k.shape[1]
    group = hq // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u, f = torch.finfo(q.dtype).eps / 2, torch.finfo(torch.float32).eps / 2
    wide, half = q.dtype == torch.float32, q.dtype == torch.float16
    shapes = {"o": q.shape, "dq": q.shape, "dk": k.shape, "dv": k.shape}
    out, tol = ({n: torch.zeros(s, dtype=torch.float64, device=q.device) for n, s in shapes.items()} for _ in range(2))
    at = 0
    for n in lens:
        own = slice(at, at + n)
        at += n
        if n == 0:
            continue
        Q, G = q[own].double().transpose(0, 1), do[own].double().transpose(0, 1)
        K, V = (x[own].double().transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        P = torch.softmax((Q @ K.mT * scale).masked_fill(~seen, -math.inf), -1)
        r = 2 * ((d + 8) * f * (Q.abs() @ K.abs().mT * scale * seen).amax() + (n + 16) * f) + 16 * f
        O, A = P @ V, P @ V.abs()
        uw = 0.0 if exact_weights else u
        out["o"][own] = O.transpose(0, 1)
        tol["o"][own] = ((uw + r) * A + u * O.abs()).transpose(0, 1)
        delta = (O * G).sum(-1, keepdim=True)
        dS = P * (G @ V.mT - delta)
        w = (2 * u + r) * A if wide else (uw + r) * A + u * u * O.abs() + (2.0**-25 if half else 0.0)
        e = (G.abs() * (w + (d + 8) * f * O.abs())).sum(-1, keepdim=True) + (d + 8) * f * (G.abs() @ V.abs().mT)
        eS, step_p = (u + r) * dS.abs() + P * e, 0.0
        if half:
            most = lambda x: x.reshape(hk, -1).amax(1).repeat_interleave(group)[:, None, None]  # noqa: E731
            B = most(G.abs().sum(-1)) * most(V.abs()[::group]) + most(delta.abs())
            eS, step_p = eS + 2.0**-39 * B * seen, 2.0**-35
        s = (n * group + 16) * f  # the sums over the rows and the heads of a group
        out["dq"][own] = (scale * dS @ K).transpose(0, 1)
        tol["dq"][own] = (scale * eS @ K.abs() + s * scale * dS.abs() @ K.abs()).transpose(0, 1)
        tol["dq"][own] += u * out["dq"][own].abs()
        for name, x, ex in (("dk", scale * dS.mT @ Q, scale * (eS + s * dS.abs()).mT @ Q.abs()),
                            ("dv", P.mT @ G, ((u + r + s) * P + step_p * seen).mT @ G.abs())):
            x, ex = (y.reshape(hk, group, n, d).sum(1).transpose(0, 1) for y in (x, ex))
            out[name][own] = x
            tol[name][own] = ex + u * x.abs()
    return out, tol


def far_values(dtype):
    """Documents of few rows, scores of zero, values of some 100: o is far larger than the differences that make dS."""
    g = torch.Generator().manual_seed(790)
    lens = [2, 3, 5, 4, 6, 2, 7]
    k, v, do = (torch.randn(sum(lens), 2, 64, generator=g) for _ in range(3))
    return torch.zeros_like(k).to(dtype), k.to(dtype), (v + 100).to(dtype), do.to(dtype), lens
