"""Packed documents on the CPU: the plan, the refusals, and the torch paths against 64-bit definitions."""

import math

import numpy as np
import pytest
import torch

from bergson_b200 import ops

from .packed_reference import assert_within, attention64


@pytest.mark.parametrize("lens,total", [([], 0), ([], 5), ([1], None), ([3, 0, 2], 7), ([130, 1, 255], 400), ([0, 0], 3)])
def test_plan_describes_every_row(lens, total):
    p = ops.PackedSequences(lens, total=total)
    rows = sum(lens) if total is None else total
    assert (p.rows, p.num_tokens, p.lengths) == (rows, sum(lens), tuple(lens))
    assert p.cu_seqlens.tolist() == [0, *np.cumsum(lens).tolist()]
    t = 0
    for n in lens:
        for i in range(n):
            assert p.first_key[t + i] == t and p.end_query[t + i] == t + n and p.position[t + i] == i
        t += n
    for r in range(t, rows):
        assert p.first_key[r] == r + 1 and p.end_query[r] == r and p.position[r] == 0
    valid = sum(lens)
    queries, keys = {}, {}
    for row0 in range(0, rows, 128):
        own = range(row0, min(row0 + 128, valid))
        some = len(own) > 0
        queries[row0] = [row0] + ([int(p.first_key[own[0]]), int(p.first_key[own[-1]]), own[-1] + 1] if some else [0, 0, 0])
        keys[row0] = [row0] + ([int(p.end_query[own[-1]]), int(p.end_query[own[0]]), 0] if some else [row0, 0, 0])
    assert {e[0]: e for e in p.query_tiles.view(-1, 4).tolist()} == queries
    assert {e[0]: e for e in p.key_tiles.view(-1, 4).tolist()} == keys
    pairs = p.query_pairs.view(-1, 8).tolist()
    assert sorted(e[0] for e in pairs) == list(range(0, rows, 256))
    for e in pairs:
        assert e[:4] == queries[e[0]]
        assert e[4:] == queries[e[0] + 128] if e[0] + 128 in queries else e[4] >= rows and e[5:] == [0, 0, 0]
    assert all(x.dtype == torch.int32 for x in (p.first_key, p.end_query, p.position, p.query_tiles))


def test_plan_orders_tiles_by_work():
    p = ops.PackedSequences([1000, 24])  # one long document, then a short one in the last tile
    assert p.query_tiles.view(-1, 4)[:, 0].tolist() == list(range(896, -1, -128))
    assert p.query_pairs.view(-1, 8)[:, 0].tolist() == [768, 512, 256, 0]
    assert p.key_tiles.view(-1, 4)[:, 0].tolist() == list(range(0, 1024, 128))


def test_plan_accepts_arrays_and_tensors():
    for lens in (np.array([2, 3]), torch.tensor([2, 3], dtype=torch.int32), (2, 3)):
        assert ops.PackedSequences(lens).lengths == (2, 3)


@pytest.mark.parametrize("lens,total", [([-1], None), ([2.5], None), ([[1, 2]], None), ([4], 3), ([1 << 30], None)])
def test_plan_refuses(lens, total):
    with pytest.raises(ValueError):
        ops.PackedSequences(lens, total=total)


def test_mask_labels():
    p = ops.PackedSequences([2, 0, 3], total=6)
    labels = torch.arange(10, 16)[None]
    assert p.mask_labels(labels).tolist() == [[-100, 11, -100, 13, 14, -100]]
    with pytest.raises(ValueError):
        p.mask_labels(labels[:, :5])


def _qkv(rows, hq, hk, d, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(rows, h, d, generator=g, dtype=torch.float64).to(dtype) for h in (hq, hk, hk)]


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2), (6, 2)])
@pytest.mark.parametrize("lens,pad", [([5], 0), ([1, 0, 7, 3], 0), ([2, 9], 4), ([], 3)])
def test_reference_attention_matches_definition(lens, pad, hq, hk):
    q, k, v = (x.requires_grad_() for x in _qkv(sum(lens) + pad, hq, hk, 6))
    p = ops.PackedSequences(lens, total=sum(lens) + pad)
    o = ops.packed_causal_attention(q, k, v, p, scale=0.7)
    do = torch.randn_like(o)
    grads = torch.autograd.grad(o, (q, k, v), do, allow_unused=True)
    want, _ = attention64(q.detach(), k.detach(), v.detach(), lens, 0.7, do)
    torch.testing.assert_close(o, want["o"], rtol=1e-12, atol=1e-12)
    for g, name in zip(grads, ("dq", "dk", "dv")):
        torch.testing.assert_close(torch.zeros_like(want[name]) if g is None else g, want[name], rtol=1e-11, atol=1e-12)


def test_reference_attention_against_differences():
    p = ops.PackedSequences([3, 4], total=8)
    q, k, v = (x.requires_grad_() for x in _qkv(8, 2, 1, 4))
    assert torch.autograd.gradcheck(lambda *x: ops.packed_causal_attention(*x, p), (q, k, v))
    assert torch.autograd.gradgradcheck(lambda *x: ops.packed_causal_attention(*x, p), (q, k, v))


def test_reference_attention_keeps_documents_apart():
    p = ops.PackedSequences([4, 3, 5], total=14)
    q, k, v = _qkv(14, 2, 2, 8)
    clean = ops.packed_causal_attention(q, k, v, p)
    for x in (q, k, v):
        x[4:7] = float("nan")
        x[12:] = float("inf")
    o = ops.packed_causal_attention(q, k, v, p)
    assert torch.equal(o[:4], clean[:4]) and torch.equal(o[7:12], clean[7:12]) and o[12:].abs().max() == 0


def test_attention_refusals():
    p = ops.PackedSequences([3, 2])
    q, k, v = _qkv(5, 4, 2, 8, torch.float32)
    call = ops.packed_causal_attention
    bad = [
        (q[:4], k, v, p), (q, k[:4], v, p), (q, k, v[:, :1], p), (q[..., :4], k, v, p), (q.half(), k, v, p),
        (q[0], k, v, p), (q[:, :3], k, v, p), (q.long(), k.long(), v.long(), p), (q, k[:, :0], v[:, :0], p),
        (q[..., :0], k[..., :0], v[..., :0], p),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            call(*args)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            call(q, k, v, p, scale=scale)
    with pytest.raises(TypeError):
        call(q, k, v, [3, 2])


@pytest.mark.parametrize("rot", [2, 6, 8])
def test_reference_rotary(rot):
    p = ops.PackedSequences([3, 0, 4], total=9)
    q, k, _ = _qkv(9, 2, 1, 8)
    cos, sin = ops.rotary_tables(5, rot, 100.0, "cpu", torch.float64)
    a, b = ops.packed_rotary(q, k, cos, sin, rot, p)
    for x, y in ((q, a), (k, b)):
        for begin, n in ((0, 3), (3, 4)):
            want = ops.rotary(x[None, begin:begin + n], cos, sin, rot)[0]
            torch.testing.assert_close(y[begin:begin + n], want, rtol=0, atol=0)
        assert torch.equal(y[7:], x[7:])
    q.requires_grad_(), k.requires_grad_()
    assert torch.autograd.gradcheck(lambda x, y: ops.packed_rotary(x, y, cos, sin, rot, p), (q, k))


def test_rotary_refusals():
    p = ops.PackedSequences([3, 2])
    q, k, _ = _qkv(5, 2, 1, 8, torch.float32)
    cos, sin = ops.rotary_tables(3, 4, 1e4, "cpu")
    for args in [(q, k, cos, sin, 3, p), (q, k, cos, sin, 6, p), (q, k, cos, sin, 0, p), (q, k, cos[:2], sin[:2], 4, p),
                 (q, k, cos, sin[:2], 4, p), (q, k[:4], cos, sin, 4, p), (q, k, cos.clone().requires_grad_(), sin, 4, p)]:
        with pytest.raises(ValueError):
            ops.packed_rotary(*args)


def _kl(z, ids, t, tau):
    """One row at a time, in python numbers."""
    out = []
    for r in range(z.shape[0]):
        lse = torch.logsumexp(z[r] / tau, 0).item()
        use = [(i, x) for i, x in zip(ids[r].tolist(), t[r].tolist()) if 0 <= i < z.shape[1] and x != -math.inf]
        if not use:
            out.append(0.0)
            continue
        m = max(x for _, x in use)
        w = [math.exp((x - m) / tau) for _, x in use]
        p = [x / sum(w) for x in w]
        out.append(tau**2 * sum(a * (math.log(a) - (z[r, i].item() / tau - lse)) for a, (i, _) in zip(p, use) if a > 0))
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_reference_distillation(tau):
    torch.manual_seed(0)
    z = torch.randn(6, 11, dtype=torch.float64) * 3
    ids = torch.randint(0, 11, (6, 4))
    t = torch.randn(6, 4, dtype=torch.float64) * 3
    ids[1, 2] = -1
    ids[2] = -1  # no entry at all
    ids[3] = 5   # one id four times
    t[4, 1] = -math.inf
    ids[5, 0] = 11  # past the vocabulary
    torch.testing.assert_close(ops.token_distillation(z, ids, t, tau).double(), _kl(z, ids, t, tau), rtol=1e-12, atol=1e-12)
    z.requires_grad_()
    assert torch.autograd.gradcheck(lambda x: ops.token_distillation(x, ids, t, tau), (z,))
    (g,) = torch.autograd.grad(ops.token_distillation(z, ids, t, tau).sum(), z)
    assert g[2].abs().max() == 0 and g.sum(1).abs().max() < 1e-12


def test_reference_distillation_masked_student():
    """Vocabulary entries at -inf that the teacher does not use take no part."""
    z = torch.tensor([[1.0, -math.inf, 0.5, 2.0]], dtype=torch.float64, requires_grad=True)
    ids, t = torch.tensor([[0, 3]]), torch.tensor([[0.3, 0.1]], dtype=torch.float64)
    loss = ops.token_distillation(z, ids, t)
    (g,) = torch.autograd.grad(loss.sum(), z)
    assert torch.isfinite(loss).all() and torch.isfinite(g).all() and g[0, 1] == 0


@pytest.mark.parametrize("value", [math.nan, -math.inf, math.inf])
def test_reference_distillation_rows_without_entries(value):
    """Such a row gives 0 and a zero gradient, whatever its logits are."""
    z = torch.randn(3, 7)
    z[1] = value
    z.requires_grad_()
    ids, t = torch.tensor([[1, 2], [-1, 7], [0, 6]]), torch.randn(3, 2)
    loss = ops.token_distillation(z, ids, t)
    (g,) = torch.autograd.grad(loss.sum(), z)
    assert loss[1] == 0 and (g[1] == 0).all() and torch.isfinite(loss).all() and torch.isfinite(g).all()


def test_distillation_refusals():
    z, ids, t = torch.randn(4, 9), torch.zeros(4, 2, dtype=torch.int64), torch.randn(4, 2)
    call = ops.token_distillation
    for args in [(z[0], ids, t), (z, ids[:3], t[:3]), (z, ids, t[:, :1]), (z, ids.float(), t), (z, ids, t.long()),
                 (z, ids[:, :0], t[:, :0]), (z[:, :0], ids, t), (z.long(), ids, t), (z, ids, t.clone().requires_grad_()),
                 (z, ids.repeat(1, 600), t.repeat(1, 600))]:
        with pytest.raises(ValueError):
            call(*args)
    for tau in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            call(z, ids, t, temperature=tau)


def test_bounds_helper_sees_a_planted_error():
    q, k, v = _qkv(9, 2, 1, 8, torch.float32)
    want, tol = attention64(q, k, v, [4, 5])
    assert_within(want["o"].float(), want["o"], tol["o"])
    wrong = want["o"].clone()
    wrong[5, 1, 3] += 1e-3
    with pytest.raises(AssertionError):
        assert_within(wrong, want["o"], tol["o"])
