"""Packed attention, rotary and distillation where values, gradients and calls are out of the ordinary."""

import math

import pytest
import torch

from bergson_b200 import ops
from bergson_b200.ops.functional import token_distillation_ref

from .packed_bounds import attention_bounds64, far_values
from .packed_reference import assert_within, attention64
from .test_packed_edges import check_empty_batches
from .test_packed_gpu import DTYPES, _attend, _rand, native  # noqa: F401

pytestmark = pytest.mark.gpu


def _check_documents(got, q, k, v, lens, do, scale=None, which=None):
    """Each document against the bounds that its own values give."""
    at = 0
    for i, n in enumerate(lens):
        own = slice(at, at + n)
        at += n
        if which is not None and i not in which:
            continue
        want, tol = attention64(q[own], k[own], v[own], [n], scale, do[own])
        for name in got:
            assert_within(got[name][own], want[name], tol[name], f"{name} of document {i}", floor=6e-8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (4, 1, 128)])
def test_gradients_of_other_documents_do_not_set_the_precision(native, hq, hk, d, dtype):
    """Documents that share tiles, with output gradients 2^18 apart, as losses of very different weights give."""
    lens = [300, 200, 260, 7, 9, 40]
    rows = sum(lens)
    q, k, v, do = (_rand((rows, h, d), dtype, 700 + i) for i, h in enumerate((hq, hk, hk, hq)))
    sizes = torch.repeat_interleave(torch.tensor([2.0**-10, 2.0**8, 2.0**-10, 2.0**6, 2.0**-9, 2.0**3]), torch.tensor(lens))
    do = (do.float() * sizes.cuda()[:, None, None]).to(dtype)
    _check_documents(_attend(native, q, k, v, lens, do=do), q, k, v, lens, do)


@pytest.mark.parametrize("small", ["q", "k"])
@pytest.mark.parametrize("poison", [float("inf"), float("nan"), 60000.0])
def test_a_poisoned_document_leaves_small_fp16_gradients(native, poison, small):
    """An infinity, a NaN or a huge value in a neighbour's output gradient, beside gradients of some 2^-16."""
    lens, dtype = [300, 90, 260], torch.float16
    q, k, v, do = (_rand((sum(lens), 2, 64), dtype, 710 + i) for i in range(4))
    # large k make dq large against fp16's smallest step, large q make dk so; the scores stay as they are
    q, k = ((q / 32).half(), (k * 32).half()) if small == "q" else ((q * 32).half(), (k / 32).half())
    do = (do.float() * 2.0**-16).half()
    do[300:390] = poison
    _check_documents(_attend(native, q, k, v, lens, do=do), q, k, v, lens, do, which=(0, 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[500], [130, 600, 11]])
def test_large_values_along_the_gradient_do_not_overflow(native, lens, dtype):
    """v of 3000 along do: score gradients above fp16's largest value, results far below it."""
    d, scale = 128, 1.0 / 512
    rows = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(720)
    q, k = (_rand((rows, 2, d), dtype, 721 + i, std=24.0) for i in range(2))
    along = torch.randint(0, 2, (d,), generator=g, device="cuda") * 2.0 - 1
    sign = torch.randint(0, 2, (rows, 2, 1), generator=g, device="cuda") * 2.0 - 1
    v = (sign * along * 3000).to(dtype)
    do = (along * 0.99).expand(rows, 2, d).to(dtype)
    want, tol = attention_bounds64(q, k, v, lens, do, scale)  # the step of dS as it is for values of this size
    P = torch.softmax((q[:lens[0], 0].double() @ k[:lens[0], 0].double().T * scale)
                      .masked_fill(torch.ones(lens[0], lens[0], dtype=torch.bool, device="cuda").triu(1), -math.inf), 1)
    dP = do[:lens[0], 0].double() @ v[:lens[0], 0].double().T
    assert (P * (dP - (P * dP).sum(1, keepdim=True))).abs().max() > 65504
    assert max(want[n].abs().max() for n in want) < 65504  # the largest fp16
    got = _attend(native, q, k, v, lens, 0, scale, do)
    for name in got:
        assert_within(got[name], want[name], tol[name], name, floor=6e-8)


def test_fp16_outliers_in_a_neighbours_values(native):
    """Values of 60000, an infinity or a NaN in another document's v: this one's gradients keep their precision."""
    lens = [200, 100, 230]
    q, k, v, do = (_rand((530, 2, 64), torch.float16, 730 + i) for i in range(4))
    do = (do.float() * 2.0**-10).half()
    for x in (60000.0, float("inf"), float("nan")):
        v[200:300] = x
        _check_documents(_attend(native, q, k, v, lens, do=do), q, k, v, lens, do, which=(0, 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,hq,hk,d", [([2, 3, 1, 5, 4, 2], 4, 2, 64), ([130, 3, 200], 2, 2, 128), ([33, 95, 31, 1, 64, 300], 6, 2, 40),
                                          ([1100], 4, 1, 64)])
def test_attention_within_the_documents_own_bounds(native, lens, hq, hk, d, dtype):
    """With what rounding took from o kept for delta, and scales of dS from a document's own rows."""
    q, k, v, do = (_rand((sum(lens), h, d), dtype, 740 + i) for i, h in enumerate((hq, hk, hk, hq)))
    sizes = 2.0 ** torch.randint(-8, 5, (len(lens),), generator=torch.Generator().manual_seed(1))
    do = (do.float() * sizes.repeat_interleave(torch.tensor(lens)).cuda()[:, None, None]).to(dtype)
    got = _attend(native, q, k, v, lens, do=do)
    want, tol = attention_bounds64(q, k, v, lens, do)
    for name in got:
        assert_within(got[name], want[name], tol[name], name, floor=6e-8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_delta_is_taken_from_more_than_the_rounded_output(native, dtype):
    """Scores of zero and values far from zero: rounding o alone would be off by many times the bound."""
    q, k, v, do, lens = far_values(dtype)
    q, k, v, do = (x.cuda() for x in (q, k, v, do))
    got = _attend(native, q, k, v, lens, do=do)
    want, tol = attention_bounds64(q, k, v, lens, do, exact_weights=True)
    for name in got:
        assert_within(got[name], want[name], tol[name], name, floor=6e-8)


def _sharp(dtype, n=300, at=150, d=64, begin=0):
    """Scores that rise by far from key to key: the weight of key `at` is zero in every later row but the next few."""
    q, k, v, do = (_rand((n, 2, d), dtype, 750 + i) for i in range(4))
    q[..., 0] = 16.0
    k[..., 0] = torch.linspace(0, 3000, n, device="cuda")[:, None].to(dtype)
    return q, k, v, do


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_attention_zero_weights_hide_nothing(native, value, dtype):
    """An attended key's weight may underflow to zero; what is not finite reaches the row all the same, as in the
    definition, where zero times it is NaN."""
    n, at, lens = 300, 150, [300]
    q, k, v, do = _sharp(dtype, n, at)
    P = torch.softmax((q[..., 0, :].double() @ k[..., 0, :].double().T / 8).masked_fill(
        torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf), 1)
    assert P[at + 20:, at].max() < 1e-60  # zero in 32 bits
    bad = v.clone()
    bad[at, 1, 5] = value
    got = _attend(native, q, k, bad, lens)["o"]
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at:, 1, 5] = True
    assert torch.equal(~torch.isfinite(got), hit) and torch.isnan(got[at + 20:, 1, 5]).all()
    bad = do.clone()
    bad[at, 1, 5] = value
    got = _attend(native, q, k, v, lens, do=bad)
    hit = torch.zeros_like(got["dv"], dtype=torch.bool)
    hit[:at + 1, 1, 5] = True
    assert torch.equal(~torch.isfinite(got["dv"]), hit) and torch.isnan(got["dv"][:at - 20, 1, 5]).all()
    hit[:at + 1, 1] = True
    assert torch.equal(~torch.isfinite(got["dk"]), hit) and torch.isfinite(got["dq"][:at]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_keys_at_minus_infinity(native, dtype):
    """A key of -inf along a positive query has no weight: o is finite, dq = 0 * -inf is NaN in that feature."""
    n, at = 300, 150
    q, k, v, do = (_rand((n, 2, 64), dtype, 760 + i) for i in range(4))
    q[..., 3] = 1.0
    k[at, 1, 3] = float("-inf")
    got = _attend(native, q, k, v, [n], do=do)
    assert torch.isfinite(got["o"][at + 1:]).all()
    hit = torch.zeros_like(got["dq"], dtype=torch.bool)
    hit[at + 1:, 1, 3] = True
    assert torch.equal(torch.isnan(got["dq"][at + 1:]), hit[at + 1:])
    assert torch.isfinite(got["dq"][:at]).all() and torch.isfinite(got["dv"]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", [(3, 777), (700, 1003), (2, 50257)])
def test_distillation_nan_among_masked_logits(native, T, V, dtype):
    """A NaN whose neighbours are all -inf, in every place of a packet: the row's loss and gradient are NaN."""
    ids, t = torch.randint(400, 600, (T, 4), device="cuda"), _rand((T, 4), torch.float32, 771)
    for at in (*range(96, 112), V - 1, 0):
        z = _rand((T, V), dtype, 770)
        z[1, :300] = -math.inf
        z[1, 700:] = -math.inf
        z[1, at] = float("nan")
        leaf = z.requires_grad_()
        loss = ops.token_distillation(leaf, ids, t)
        (g,) = torch.autograd.grad(loss.sum(), leaf)
        others = [0] + list(range(2, T))
        assert torch.isnan(loss[1]) and torch.isnan(g[1]).all(), at
        assert torch.isfinite(loss[others]).all() and torch.isfinite(g[others]).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("T", [4, 700])
def test_distillation_of_teacher_logits_that_are_not_finite(native, T, value):
    """NaN as on torch operations, unless the entry is not one; other rows are as they were."""
    z, t = _rand((T, 1003), torch.bfloat16, 772), _rand((T, 5), torch.float32, 773)
    ids = torch.randint(0, 1003, (T, 5), device="cuda")
    ids[2, 1] = -1
    t[1, 0] = t[2, 1] = value
    leaf = z.requires_grad_()
    loss = ops.token_distillation(leaf, ids, t, 1.5)
    (g,) = torch.autograd.grad(loss.sum(), leaf)
    want = token_distillation_ref(z.detach().double(), ids, t.double(), 1.5)
    assert torch.equal(torch.isnan(loss), torch.isnan(want)) and torch.isnan(loss[1])
    assert torch.isnan(g[1, ids[1]]).all()
    others = [i for i in range(T) if i != 1]
    torch.testing.assert_close(loss[others].double(), want[others], rtol=1e-5, atol=1e-5)
    assert torch.isfinite(g[others]).all()


@pytest.mark.parametrize("place", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(native, place):
    """The kernels have no tangents: a dual tensor is refused and not computed without its tangent."""
    import torch.autograd.forward_ad as fw

    p = ops.PackedSequences([20], device="cuda")
    q, k, v = (_rand((20, 2, 64), torch.float32, 780 + i) for i in range(3))
    cos, sin = ops.rotary_tables(20, 64, 1e4, "cuda")
    z, ids, t = _rand((20, 90), torch.float32, 783), torch.randint(0, 90, (20, 3), device="cuda"), _rand((20, 3), torch.float32, 784)
    with fw.dual_level():
        def dual(*xs):
            return [fw.make_dual(x, torch.ones_like(x)) if i == place else x for i, x in enumerate(xs)]

        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.packed_causal_attention(*dual(q, k, v), p)
        with pytest.raises((RuntimeError, NotImplementedError)), torch.no_grad():
            ops.packed_causal_attention(*dual(q, k, v), p)
        x = [*dual(q, k), cos, sin] if place < 2 else [q, k, fw.make_dual(cos, torch.ones_like(cos)), sin]
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.packed_rotary(*x, 64, p)
        if place < 2:
            a, b = dual(z, t)
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.token_distillation(a, ids, b)
            with ops.composable():
                assert fw.unpack_dual(ops.token_distillation(a, ids, t)).tangent is not None or place == 1


def test_a_wait_that_ran_out_is_raised_by_the_next_call(native):
    """The words that a kernel which gives up sets, set here by the host: calls raise until the status is cleared."""
    p = ops.PackedSequences([20], device="cuda")
    q, k, v = (_rand((20, 2, 64), torch.bfloat16, 790 + i).requires_grad_() for i in range(3))
    o = ops.packed_causal_attention(q, k, v, p)
    want, word = o.detach().clone(), native.packed_gave_up(0)
    assert word.item() == 0
    try:
        native.kernel_status(0).fill_(2)
        word.fill_(1)
        for _ in range(2):
            with pytest.raises(RuntimeError, match="gave up"):
                ops.packed_causal_attention(q, k, v, p)
        with pytest.raises(RuntimeError, match="gave up"):
            torch.autograd.grad(o.sum(), q, retain_graph=True)
    finally:
        native.kernel_status(0).zero_()
    assert torch.equal(ops.packed_causal_attention(q, k, v, p), want) and word.item() == 0
    assert torch.isfinite(torch.autograd.grad(o.sum(), q)[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches_have_gradients_for_all_operands(native, dtype):
    check_empty_batches("cuda", dtype)


def test_a_dropped_plan_stays_until_other_streams_have_read_it(native):
    """A plan made on one stream, used on another and dropped at once: its memory is not given away before."""
    side, lens = torch.cuda.Stream(), [100] * 300
    q, k, v = (_rand((30000, 1, 64), torch.bfloat16, 800 + i) for i in range(3))
    cos, sin = ops.rotary_tables(100, 64, 1e4, "cuda")
    torch.cuda.synchronize()
    for call in (lambda p: ops.packed_causal_attention(q, k, v, p), lambda p: ops.packed_rotary(q, k, cos, sin, 64, p)):
        with torch.no_grad():
            call(ops.PackedSequences(lens, device="cuda"))  # the kernels' code is loaded
        torch.cuda.synchronize()
        p = ops.PackedSequences(lens, device="cuda")
        storage = p.first_key.untyped_storage()
        at, size = storage.data_ptr(), storage.nbytes()
        with torch.cuda.stream(side), torch.no_grad():
            torch.cuda._sleep(100_000_000)  # some 50 ms
            out = call(p)
        del p, storage
        assert not side.query()
        others = [torch.empty(size, device="cuda", dtype=torch.uint8) for _ in range(8)]
        assert all(not at <= x.data_ptr() < at + size for x in others)
        torch.cuda.synchronize()
        del out, others
