"""Packed documents and distillation on torch operations, where values and calls are out of the ordinary."""

import math

import pytest
import torch

from bergson_b200 import ops


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_distillation_of_teacher_logits_that_are_not_finite(value):
    """Such an entry has no distribution: NaN, unless the entry is not one."""
    z = torch.randn(4, 9, requires_grad=True)
    ids, t = torch.tensor([[1, 2], [3, 4], [5, -1], [0, 6]]), torch.randn(4, 2)
    t[1, 0] = value
    t[2, 1] = value
    loss = ops.token_distillation(z, ids, t, 1.5)
    (g,) = torch.autograd.grad(loss.sum(), z)
    assert torch.isnan(loss[1]) and torch.isnan(g[1, [3, 4]]).all()
    assert torch.isfinite(loss[[0, 2, 3]]).all() and torch.isfinite(g[[0, 2, 3]]).all()


def test_documents_of_many_lengths_leave_no_masks_behind():
    from bergson_b200.ops import functional

    before = dict(functional._CAUSAL_BIAS)
    lens = list(range(1, 40))
    q = torch.randn(sum(lens), 1, 8)
    ops.packed_causal_attention(q, q, q, ops.PackedSequences(lens))
    assert functional._CAUSAL_BIAS.keys() == before.keys()


def check_empty_batches(device, dtype):
    """No rows, or rows of no document: every operand has a gradient, of zeros."""
    for rows in (0, 5):
        for lens in ([], [0, 0]):
            q, k, v = (torch.randn(rows, h, 64, device=device, dtype=dtype, requires_grad=True) for h in (4, 2, 2))
            with torch.no_grad():
                for x in (q, k, v):
                    x[1:] = math.nan
            p = ops.PackedSequences(lens, device=device, total=rows)
            for only in (q, k, v):
                xs = [x if x is only else x.detach() for x in (q, k, v)]
                o = ops.packed_causal_attention(*xs, p)
                assert o.shape == q.shape and o.dtype == dtype and (o == 0).all() and o.requires_grad
            grads = torch.autograd.grad(ops.packed_causal_attention(q, k, v, p).sum(), (q, k, v))
            assert all(g.shape == x.shape and (g == 0).all() for g, x in zip(grads, (q, k, v)))


def test_empty_batches():
    check_empty_batches("cpu", torch.float64)


def test_a_plan_made_in_inference_mode_serves_training():
    with torch.inference_mode():
        p = ops.PackedSequences([3, 2])
    x = torch.randn(5, 2, 8, requires_grad=True)
    cos, sin = ops.rotary_tables(3, 8, 1e4, "cpu")
    q, k = ops.packed_rotary(x, x, cos, sin, 8, p)
    (g,) = torch.autograd.grad(ops.packed_causal_attention(q, k, x, p).sum(), x)
    assert torch.isfinite(g).all()
    emb = torch.nn.Embedding(3, 4)
    emb(p.position).sum().backward()
