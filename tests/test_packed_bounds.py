"""The packed attention's error bounds see what they are there to see."""

import pytest
import torch

from .packed_bounds import attention_bounds64, far_values
from .packed_reference import assert_within


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_see_a_delta_from_the_rounded_output(dtype):
    """dq with delta from o as it is rounded is far outside; with o's rounding rest, rounded in its turn, inside."""
    q, k, v, do, lens = far_values(dtype)
    want, tol = attention_bounds64(q, k, v, lens, do, exact_weights=True)
    dq = {True: [], False: []}
    at = 0
    for n in lens:
        K, V, G, O = (x[at:at + n].double().transpose(0, 1) for x in (k, v, do, want["o"]))
        P = torch.ones(n, n, dtype=torch.float64).tril() / torch.arange(1, n + 1)[:, None]
        at += n
        kept = O.to(dtype).double()
        for rest in dq:
            delta = ((kept + (O - kept).to(dtype).double() * rest) * G).sum(-1, keepdim=True)
            dq[rest].append((P * (G @ V.mT - delta) @ K / 8).transpose(0, 1))
    assert_within(torch.cat(dq[True]), want["dq"], tol["dq"], floor=6e-8)
    off = (torch.cat(dq[False]) - want["dq"]).abs()
    assert (off > tol["dq"] + 6e-8).float().mean() > 0.1


def test_bounds_see_a_gradient_scaled_by_another_document():
    """fp16: dS rounded with the factor of a neighbour's gradients, 2^18 times as large."""
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(120, 1, 64, generator=g).half() for _ in range(4))
    do[:80] = (do[:80].float() * 2.0**-10).half()
    do[80:] = (do[80:].float() * 2.0**8).half()
    want, tol = attention_bounds64(q, k, v, [80, 40], do)
    Q, K, V, G = (x[:80, 0].double() for x in (q, k, v, do))
    P = torch.softmax((Q @ K.T / 8).masked_fill(torch.ones(80, 80, dtype=torch.bool).triu(1), -torch.inf), 1)
    dP = G @ V.T
    dS = P * (dP - (P * dP).sum(1, keepdim=True))
    for factor, fine in ((2.0**10, True), (2.0**-9, False)):  # of this document, of the neighbour
        dq = ((dS * factor).half().double() / factor @ K / 8)[:, None]
        bad = (dq - want["dq"][:80]).abs() > tol["dq"][:80] + 6e-8
        assert not bad.any() if fine else bad.float().mean() > 0.1
