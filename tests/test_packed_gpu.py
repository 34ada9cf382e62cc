"""The kernels on packed documents and of the distillation loss against 64-bit definitions."""

import math

import pytest
import torch

from bergson_b200 import ops
from bergson_b200.ops.functional import token_distillation_ref

from .packed_reference import assert_within, attention64

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def native():
    from bergson_b200.ops import native as n

    assert n.available()
    return n


def _status_ok(native):
    torch.cuda.synchronize()
    assert int(native.kernel_status(0).item()) == 0


def _rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _attend(native, q, k, v, lens, pad=0, scale=None, do=None, packing=None):
    p = packing or ops.PackedSequences(lens, device="cuda", total=sum(lens) + pad)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = ops.packed_causal_attention(*leaves, p, scale=scale)
    got = {"o": o.detach()}
    if do is not None:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))
    _status_ok(native)
    return got


def _check_attention(native, lens, pad, hq, hk, d, dtype, seed=0, scale=None, train=True):
    rows = sum(lens) + pad
    q, k, v = (_rand((rows, h, d), dtype, seed + i) for i, h in enumerate((hq, hk, hk)))
    do = _rand((rows, hq, d), dtype, seed + 3) if train else None
    got = _attend(native, q, k, v, lens, pad, scale, do)
    want, tol = attention64(q, k, v, lens, scale, do)
    for name, x in got.items():
        assert x.dtype == dtype and x.shape == want[name].shape and x.is_contiguous()
        # 6e-8: half of fp16's smallest step
        assert_within(x, want[name], tol[name], f"{name} {lens} {hq}/{hk}x{d} {dtype}", floor=6e-8)


LENGTHS = [([1], 0), ([37], 0), ([128], 0), ([129, 1, 127], 3), ([0, 1, 0, 64, 0], 0), ([63, 65, 64, 64], 0),
           ([300, 0, 5, 211], 70), ([1] * 140, 9), ([700], 0), ([250, 262], 129)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,pad", LENGTHS)
def test_attention_lengths(native, lens, pad, dtype):
    _check_attention(native, lens, pad, 4, 2, 64, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 8), (3, 3, 16), (6, 2, 32), (5, 1, 40), (8, 1, 128), (4, 4, 128), (3, 1, 80),
                                     (12, 4, 96), (2, 2, 120)])
def test_attention_heads(native, hq, hk, d, dtype):
    _check_attention(native, [200, 3, 150], 5, hq, hk, d, dtype, seed=10)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_long_documents(native, d, dtype):
    _check_attention(native, [2111, 1, 1500], 77, 4, 2, d, dtype, seed=20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_attention_scale(native, scale, dtype):
    # scale 1 with 64 features: scores of some +-8 (sharp softmax); 0.01: nearly uniform
    _check_attention(native, [333, 90], 0, 2, 1, 64, dtype, seed=30, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rising_scores(native, dtype):
    """The running maximum rises by far from key tile to key tile, and falls."""
    n, d = 900, 64
    q, k, v, do = (_rand((n, 2, d), dtype, 40 + i, std=0.3) for i in range(4))
    ramp = torch.linspace(0, 40, n, device="cuda")[:, None]
    q[..., 0] = 8.0
    k[..., 0] = ramp.to(dtype)
    for order in (torch.arange(n), torch.arange(n - 1, -1, -1)):
        kk = k[order.cuda()].contiguous()
        got = _attend(native, q, kk, v, [n], 0, None, do)
        want, tol = attention64(q, kk, v, [n], None, do)
        for name in got:
            assert_within(got[name], want[name], tol[name], name, floor=6e-8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_reads_views_in_place(native, dtype):
    """Slices of a fused projection, head-major storage, an expanded key head, an unaligned base."""
    rows, h, d, lens = 300, 3, 32, [170, 130]
    do = _rand((rows, h, d), dtype, 54)
    fused = _rand((rows, h, 3 * d), dtype, 50).split(d, dim=-1)
    head_major = [_rand((h, rows, d), dtype, 51 + i).transpose(0, 1) for i in range(3)]
    expanded = [_rand((rows, h, d), dtype, 55), *(_rand((rows, 1, d), dtype, 56 + i).expand(rows, h, d) for i in range(2))]
    odd = [_rand((rows * h * d + 1,), dtype, 58 + i)[1:].view(rows, h, d) for i in range(3)]
    wide = [_rand((rows, h + 2, d + 8), dtype, 61 + i)[:, 1:-1, :d] for i in range(3)]
    strided = [_rand((rows, h, 2 * d), dtype, 64 + i)[..., ::2] for i in range(3)]
    for q, k, v in (fused, head_major, expanded, odd, wide, strided):
        got = _attend(native, q, k, v, lens, do=do)
        want, tol = attention64(q, k, v, lens, do=do)
        for name in got:
            assert_within(got[name], want[name], tol[name], name, floor=6e-8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_gradient_of_views_and_broadcasts(native, dtype):
    """The output's gradient as a broadcast and as a transposed view; a key head shared by expansion."""
    rows, h, d, lens = 140, 2, 64, [90, 50]
    q, k, v = (_rand((rows, h, d), dtype, 70 + i) for i in range(3))
    g = _rand((h, rows, d), dtype, 73)
    for do in (g.transpose(0, 1), g[0, 0].expand(rows, h, d), g[:, :1].transpose(0, 1).expand(rows, h, d)):
        got = _attend(native, q, k, v, lens, do=do)
        want, tol = attention64(q, k, v, lens, do=do)
        for name in got:
            assert_within(got[name], want[name], tol[name], name, floor=6e-8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_keeps_documents_apart(native, d, poison, dtype):
    """Whatever stands in one document or behind the last one changes no other document's values."""
    lens, pad, bad = [100, 30, 200, 500], 60, 2
    rows = sum(lens) + pad
    q, k, v, do = (_rand((rows, h, d), dtype, 80 + i) for i, h in enumerate((4, 2, 2, 4)))
    clean = _attend(native, q, k, v, lens, pad, do=do)
    begin = sum(lens[:bad])
    for x in (q, k, v, do):
        x[begin:begin + lens[bad]] = poison
        x[sum(lens):] = poison
    got = _attend(native, q, k, v, lens, pad, do=do)
    want, tol = attention64(*(x.nan_to_num(0, 0, 0) for x in (q, k, v)), lens, do=do.nan_to_num(0, 0, 0))
    for name in got:
        for part in (slice(0, begin), slice(begin + lens[bad], sum(lens))):
            assert torch.isfinite(got[name][part]).all(), name
            assert_within(got[name][part], want[name][part], tol[name][part], name, floor=6e-8)
        assert got[name][sum(lens):].abs().max() == 0, name
        assert torch.equal(clean[name][sum(lens):], got[name][sum(lens):])
        assert not torch.isfinite(got[name][begin:begin + lens[bad]]).all()


def test_offsets_beyond_32_bits(native):
    """More than 2^31 elements in q, o and the logits: the last rows are as they are alone."""
    n, docs, hq, d = 128, 1100, 120, 128
    rows = n * docs
    assert rows * hq * d > 2**31
    p, alone = ops.PackedSequences([n] * docs, device="cuda"), ops.PackedSequences([n], device="cuda")
    q = torch.empty(rows, hq, d, device="cuda", dtype=torch.bfloat16).normal_()
    k, v = (_rand((rows, 1, d), torch.bfloat16, 190 + i) for i in range(2))
    cos, sin = ops.rotary_tables(n, d, 1e4, "cuda")

    def run(packing, q, k, v):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        turned = ops.packed_rotary(*leaves[:2], cos, sin, d, packing)
        o = ops.packed_causal_attention(*turned, leaves[2], packing)
        return (o.detach(), *torch.autograd.grad(o, leaves, o.detach()))

    got, want = run(p, q, k, v), run(alone, q[-n:], k[-n:], v[-n:])
    for x, y in zip(got, want):
        assert torch.equal(x[-n:], y)
    _status_ok(native)
    del got, q
    T, V = 17000, 128256
    assert T * V > 2**31
    z = torch.empty(T, V, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_()
    ids, t = torch.randint(0, V, (T, 8), device="cuda"), _rand((T, 8), torch.float32, 195)
    loss = ops.token_distillation(z, ids, t)
    (g,) = torch.autograd.grad(loss.sum(), z)
    end = slice(T - 600, T)
    last = z.detach()[end].clone().requires_grad_()
    one = ops.token_distillation(last, ids[end], t[end])
    (g1,) = torch.autograd.grad(one.sum(), last)
    assert torch.equal(loss[end], one) and torch.equal(g[end], g1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_some_operands_only(native, dtype):
    lens = [150, 3, 70]
    p = ops.PackedSequences(lens, device="cuda")
    rows, d = sum(lens), 64
    q, k, v, do = (_rand((rows, h, d), dtype, 200 + i) for i, h in enumerate((4, 2, 2, 4)))
    want, tol = attention64(q, k, v, lens, do=do)
    for i, name in enumerate(("dq", "dk", "dv")):
        xs = [q, k, v]
        leaf = xs[i] = xs[i].detach().requires_grad_()
        (g,) = torch.autograd.grad(ops.packed_causal_attention(*xs, p), leaf, do)
        assert_within(g, want[name], tol[name], name, floor=6e-8)
    # one tensor in all three places gets the sum
    x = _rand((rows, 2, d), dtype, 210)
    apart, _ = attention64(x, x, x, lens, do=do[:, :2])
    leaf = x.requires_grad_()
    (g,) = torch.autograd.grad(ops.packed_causal_attention(leaf, leaf, leaf, p), leaf, do[:, :2])
    _, tol = attention64(x.detach(), x.detach(), x.detach(), lens, do=do[:, :2])
    u = torch.finfo(dtype).eps / 2  # the two additions of the three gradients round twice
    parts = [apart[n] for n in ("dq", "dk", "dv")]
    assert_within(g, sum(parts), sum(tol[n] for n in ("dq", "dk", "dv")) + 3 * u * sum(y.abs() for y in parts), floor=6e-8)
    # only one of the rotated tensors is used
    cos, sin = ops.rotary_tables(150, d, 1e4, "cuda")
    a, b = q.detach().requires_grad_(), k.detach().requires_grad_()
    turned, other = ops.packed_rotary(a, b, cos, sin, d, p)
    ga, gb = torch.autograd.grad(turned, (a, b), do, retain_graph=True)
    back, _ = ops.packed_rotary(do, k, cos, -sin, d, p)
    assert torch.equal(ga, back) and gb.abs().max() == 0
    with torch.inference_mode():
        assert torch.equal(ops.packed_causal_attention(q, k, v, p), ops.packed_causal_attention(q, k, v, p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(4, 2), (3, 3)])
def test_attention_a_nan_reaches_what_depends_on_it(native, hq, hk, d, dtype):
    """One NaN in v, then one in the output's gradient, in the middle of a long document."""
    lens = [700, 40, 1500]
    begin, at, rows = 740, 740 + 900, sum(lens)
    q, k, v, do = (_rand((rows, h, d), dtype, 170 + i) for i, h in enumerate((hq, hk, hk, hq)))
    want, tol = attention64(q, k, v, lens, do=do)
    group, kv = hq // hk, hk - 1

    def check(got, name, hit):
        assert torch.equal(torch.isnan(got[name]), hit), name
        assert_within(got[name][~hit], want[name][~hit], tol[name][~hit], name, floor=6e-8)

    bad = v.clone()
    bad[at, kv, 5] = float("nan")
    hit = torch.zeros((rows, hq, d), dtype=torch.bool, device="cuda")
    hit[at:, kv * group:, 5] = True
    check(_attend(native, q, k, bad, lens), "o", hit)

    bad = do.clone()
    bad[at, hq - 1, 5] = float("nan")
    got = _attend(native, q, k, v, lens, do=bad)
    hit_v, hit_k = (torch.zeros((rows, hk, d), dtype=torch.bool, device="cuda") for _ in range(2))
    hit_v[begin:at + 1, kv, 5] = True
    hit_k[begin:at + 1, kv] = True
    hit_q = torch.zeros_like(hit)
    hit_q[at, hq - 1] = True
    for name, h in (("dv", hit_v), ("dk", hit_k), ("dq", hit_q)):
        check(got, name, h)


def test_attention_nan_in_a_very_long_document(native):
    """Putting rows right takes time where they are long; nobody waits for it with a limit."""
    from bergson_b200.ops import attribution

    n = 30000
    q, k, v, do = (_rand((n, h, 64), torch.bfloat16, 180 + i) for i, h in enumerate((4, 1, 1, 4)))
    do[-1] = float("nan")
    got = _attend(native, q, k, v, [n], do=do)
    assert torch.isnan(got["dv"]).all() and torch.isnan(got["dk"]).all()
    assert torch.isfinite(got["dq"][:-1]).all() and torch.isnan(got["dq"][-1]).all()
    do[-1] = do[0]
    do[100] = float("nan")
    got = _attend(native, q, k, v, [n], do=do)
    assert torch.isnan(got["dv"][:101]).all() and torch.isfinite(got["dv"][101:]).all()
    assert torch.isnan(got["dk"][:101]).all() and torch.isfinite(got["dk"][101:]).all()
    v[-1] = float("nan")
    got = _attend(native, q, k, v, [n])
    assert torch.isfinite(got["o"][:-1]).all() and torch.isnan(got["o"][-1]).all()
    q[0] = float("nan")
    got = _attend(native, q, k, v, [n], do=do)
    assert torch.isnan(got["o"][0]).all() and torch.isfinite(got["o"][1:-1]).all()
    assert attribution.kernel_status(0) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_later_rows_do_not_reach_earlier_ones(native, dtype):
    n, at = 400, 207
    q, k, v = (_rand((n, 2, 64), dtype, 90 + i) for i in range(3))
    clean = _attend(native, q, k, v, [n])["o"]
    for x in (q, k, v):
        x[at:] = float("nan")
    got = _attend(native, q, k, v, [n])["o"]
    want, tol = attention64(q[:at], k[:at], v[:at], [at])
    assert_within(got[:at], want["o"], tol["o"], floor=6e-8)
    assert torch.isfinite(clean).all() and torch.isnan(got[at:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_single_tokens_have_no_score_gradient(native, dtype):
    n = 130
    q, k, v, do = (_rand((n, 2, 64), dtype, 95 + i) for i in range(4))
    got = _attend(native, q, k, v, [1] * n, do=do)
    assert torch.equal(got["o"], v) and torch.equal(got["dv"], do)
    assert got["dq"].abs().max() == 0 and got["dk"].abs().max() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (3, 3, 64)])
def test_attention_is_reproducible(native, hq, hk, d, dtype):
    lens = [513, 40, 300]
    q, k, v, do = (_rand((sum(lens), h, d), dtype, 100 + i) for i, h in enumerate((hq, hk, hk, hq)))
    a, b = (_attend(native, q, k, v, lens, do=do) for _ in range(2))
    for name in a:
        assert torch.equal(a[name], b[name])


def test_attention_small_fp16_gradients_keep_their_precision(native):
    """fp16: the output's gradient far below 1, as an unscaled mean loss gives it; the results, scaled
    back, match as those of a gradient near 1 do."""
    lens = [300, 211]
    q, k, v = (_rand((511, 2, 64), torch.float16, 110 + i) for i in range(3))
    do = _rand((511, 2, 64), torch.float16, 113)
    tiny = (do.float() * 2.0**-8).half()
    got = _attend(native, q, k, v, lens, do=tiny)
    want, tol = attention64(q, k, v, lens, do=tiny)
    for name in got:
        assert_within(got[name], want[name], tol[name], name, floor=6e-8)


def test_attention_backward_accepts_saved_graph_twice(native):
    lens = [77, 100]
    q, k, v, do = (_rand((177, 2, 64), torch.bfloat16, 120 + i) for i in range(4))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    p = ops.PackedSequences(lens, device="cuda")
    o = ops.packed_causal_attention(*leaves, p)
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    second = torch.autograd.grad(o, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(ops.packed_causal_attention(*leaves, p).sum(), leaves, create_graph=True)
        g[0].sum().backward()


def test_attention_composable_is_twice_differentiable(native):
    q, k, v = (_rand((20, 2, 8), torch.float32, 125 + i).requires_grad_() for i in range(3))
    p = ops.PackedSequences([12, 8], device="cuda")
    with ops.composable():
        (g,) = torch.autograd.grad(ops.packed_causal_attention(q, k, v, p).square().sum(), q, create_graph=True)
        (h,) = torch.autograd.grad(g.square().sum(), k)
    assert torch.isfinite(h).all() and h.abs().max() > 0


def test_attention_other_head_sizes_and_types_take_the_torch_path(native):
    for d, dtype in ((136, torch.float32), (12, torch.float32), (64, torch.float64)):
        q, k, v = (_rand((50, 2, d), dtype, 130 + i) for i in range(3))
        o = ops.packed_causal_attention(q, k, v, ops.PackedSequences([30, 20], device="cuda"))
        want, _ = attention64(q, k, v, [30, 20])
        torch.testing.assert_close(o.double(), want["o"], rtol=1e-4, atol=1e-5)


def test_attention_empty_batches(native):
    for rows in (0, 5):
        q = torch.randn(rows, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        o = ops.packed_causal_attention(q, q, q, ops.PackedSequences([], device="cuda", total=rows))
        assert o.shape == q.shape and (rows == 0 or o.abs().max() == 0)
        (g,) = torch.autograd.grad(o.sum(), q)
        assert g.shape == q.shape and (rows == 0 or g.abs().max() == 0)


def test_packing_on_another_device_is_refused(native):
    q = torch.randn(5, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        ops.packed_causal_attention(q, q, q, ops.PackedSequences([5]))
    with pytest.raises(ValueError):
        ops.PackedSequences(torch.tensor([5], device="cuda"))


# --------------------------------------------------------------------------- #
# rotary
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,d,rot", [(1, 1, 8, 8), (4, 2, 16, 16), (12, 12, 64, 16), (32, 8, 128, 128), (3, 1, 20, 6),
                                         (5, 5, 256, 2)])
def test_rotary(native, hq, hk, d, rot, dtype):
    lens, pad = [70, 0, 1, 130], 3
    rows = sum(lens) + pad
    p = ops.PackedSequences(lens, device="cuda", total=rows)
    q, k = _rand((rows, hq, d), dtype, 0), _rand((rows, hk, d), dtype, 1)
    if hq == hk:  # views of one projection
        q, k, _ = _rand((rows, hq, 3 * d), dtype, 2).split(d, dim=-1)
    cos, sin = ops.rotary_tables(130, rot, 5e5, "cuda")
    leaves = [q.detach().requires_grad_(), k.detach().requires_grad_()]
    out = ops.packed_rotary(*leaves, cos, sin, rot, p)
    up = [_rand((rows, h, d), dtype, 5) for h in (hq, hk)]
    grads = torch.autograd.grad(out, leaves, up)
    at = p.position.long()
    c, s = cos[at].double()[:, None], sin[at].double()[:, None]
    u, f, half = torch.finfo(dtype).eps / 2, torch.finfo(torch.float32).eps / 2, rot // 2

    def check(got, x, sign):
        x = x.double()
        a, b = x[..., :half], x[..., half:rot]
        want = torch.cat([a * c - sign * b * s, b * c + sign * a * s, x[..., rot:]], -1)
        mag = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), 0 * x[..., rot:]], -1)
        # two products and a sum in fp32, one rounding to the type; fp16's smallest step
        assert_within(got, want, u * want.abs() * (1 + 2 * f) + 2 * f * mag, floor=3e-8)

    for x, y, g, w in zip((q, k), out, grads, up):
        check(y.detach(), x, 1.0)
        check(g, w, -1.0)
        assert torch.equal(y[sum(lens):], x[sum(lens):])


# --------------------------------------------------------------------------- #
# distillation
# --------------------------------------------------------------------------- #


def _distill64(z, ids, t, tau, dloss):
    zd = z.double().detach().requires_grad_()
    loss = token_distillation_ref(zd, ids, t.double(), tau)
    (g,) = torch.autograd.grad(loss, zd, dloss.double())
    return loss.detach(), g


def _check_distill(native, z, ids, t, tau, seed=0):
    dloss = _rand((z.shape[0],), torch.float32, seed + 9) + 2
    leaf = z.detach().requires_grad_()
    loss = ops.token_distillation(leaf, ids, t, tau)
    (g,) = torch.autograd.grad(loss, leaf, dloss)
    torch.cuda.synchronize()
    want, dz = _distill64(z, ids, t, tau, dloss)
    f = torch.finfo(torch.float32).eps / 2
    # The exponents of the sums are differences of logits, rounded once after the factor (log2 e / tau):
    # an error of some 4 f times the row's range r of them, relative in each summand; the sums over V / 512
    # values of a thread and the join add to it.  The loss is a mean of such exponents.
    finite = z.double().masked_fill(torch.isinf(z.double()), 0)
    used = t.double().masked_fill(torch.isinf(t.double()), 0)
    r = 3 * (finite.amax(1) - finite.amin(1) + used.amax(1) - used.amin(1)) / tau + 4
    rel = f * (4 * r + z.shape[1] / 128 + ids.shape[1] + 32)
    tol = tau**2 * rel * (r + math.log(z.shape[1]))
    assert loss.dtype == torch.float32
    assert_within(loss, want, tol, "loss")
    u = torch.finfo(z.dtype).eps / 2
    # g (q - p): both carry the relative error rel, and one rounding to the type at the end
    scale = (dloss.abs().double() * tau)[:, None]
    q = torch.softmax(z.double() / tau, 1)
    assert_within(g, dz, u * dz.abs() + scale * rel[:, None] * (2 * q + dz.abs() / scale), "gradient", floor=3e-8)
    assert g.dtype == z.dtype and g.shape == z.shape
    return loss.detach(), g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,K", [(1, 2, 1), (3, 7, 5), (5, 1000, 20), (300, 513, 64), (7, 50257, 33), (2, 128256, 256),
                                   (40, 32000, 1024)])
def test_distillation(native, T, V, K, dtype):
    torch.manual_seed(T)
    z = _rand((T, V), dtype, 1, std=2.5)
    ids = torch.stack([torch.randperm(V, device="cuda")[: min(K, V)] for _ in range(T)])
    ids = ids.repeat(1, -(-K // V))[:, :K].contiguous()
    t = _rand((T, K), torch.float32, 2, std=2.0)
    _check_distill(native, z, ids, t, 1.0)
    _check_distill(native, z, ids.int(), t.to(dtype), 2.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_entries(native, dtype):
    """Unused entries, rows without any, repeated ids, ids past the vocabulary, -inf teacher logits."""
    V = 4099
    z = _rand((8, V), dtype, 3, std=2.0)
    ids = torch.randint(0, V, (8, 12), device="cuda")
    t = _rand((8, 12), torch.float32, 4)
    ids[1] = -1
    ids[2, 3:] = -1
    ids[3] = 4098
    ids[4, ::2] = 17
    ids[5, 0], ids[5, 1], ids[5, 2] = V, -7, 2**40
    t[6, :11] = -math.inf
    t[7] = -math.inf
    loss, g = _check_distill(native, z, ids, t, 1.7)
    for r in (1, 7):
        assert loss[r] == 0 and g[r].abs().max() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_masked_student_entries(native, dtype):
    """Student logits of -inf and of the type's lowest value outside the teacher's entries."""
    V = 2050
    z = _rand((6, V), dtype, 5)
    ids = torch.randint(0, 1000, (6, 9), device="cuda")
    t = _rand((6, 9), torch.float32, 6)
    z[0, 1000:] = -math.inf
    z[1, 1000:] = torch.finfo(dtype).min
    z[2, 1000:] = -math.inf
    z[2, :8] = -math.inf
    ids[2] = ids[2].clamp(min=8)
    z[3] = torch.finfo(dtype).min  # every entry alike: a uniform student
    leaf = z.detach().requires_grad_()
    loss = ops.token_distillation(leaf, ids, t, 0.5)
    (g,) = torch.autograd.grad(loss.sum(), leaf)
    want, dz = _distill64(z, ids, t, 0.5, torch.ones(6, device="cuda"))
    assert torch.isfinite(loss).all() and torch.isfinite(g).all()
    torch.testing.assert_close(loss.double(), want, rtol=1e-5, atol=1e-5)
    u = torch.finfo(dtype).eps / 2
    assert_within(g, dz, 1.1 * u * dz.abs(), floor=1e-5)


def test_distillation_far_logits(native):
    """Large offsets cancel before anything is rounded."""
    z = _rand((4, 5000), torch.float32, 7)
    ids = torch.randint(0, 5000, (4, 30), device="cuda")
    t = _rand((4, 30), torch.float32, 8)
    base = ops.token_distillation(z, ids, t)
    moved = ops.token_distillation((z * 64).round() / 64 + 4096.0, ids, t + 1000.0)
    want = token_distillation_ref(((z * 64).round() / 64).double(), ids, ((t + 1000.0) - 1000.0).double(), 1.0)
    torch.testing.assert_close(moved.double(), want.double(), rtol=2e-6, atol=2e-6)
    assert torch.isfinite(base).all()


def test_distillation_nan_stays_in_its_row(native):
    z = _rand((3, 777), torch.bfloat16, 9)
    z[1, 5] = float("nan")
    leaf = z.requires_grad_()
    ids, t = torch.randint(0, 777, (3, 4), device="cuda"), _rand((3, 4), torch.float32, 10)
    loss = ops.token_distillation(leaf, ids, t)
    (g,) = torch.autograd.grad(loss.sum(), leaf)
    assert torch.isnan(loss[1]) and torch.isfinite(loss[[0, 2]]).all() and torch.isfinite(g[[0, 2]]).all()
    assert torch.isnan(g[1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_views(native, dtype):
    """Rows of a wider buffer, an unaligned base, transposed storage; sliced teachers."""
    V = 1001
    ids = torch.randint(0, V, (10, 12), device="cuda")[:, ::2]
    t = _rand((10, 12), torch.float32, 11)[:, 1::2]
    wide = _rand((10, 1008), dtype, 12)[:, :V]
    odd = _rand((10 * V + 3,), dtype, 13)[3:].view(10, V)
    cols = _rand((V, 10), dtype, 14).t()
    every_other = _rand((20, V), dtype, 15)[::2]
    for z in (wide, odd, cols, every_other, wide[:1].expand(10, V)):
        _check_distill(native, z, ids, t, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_rows_without_a_loss(native, dtype):
    """Rows whose entries are all unused and rows whose loss gets no gradient: zeros, whatever stands there."""
    T, V = 700, 1003  # more rows than share out to several blocks each
    z = _rand((T, V), dtype, 30)
    ids = torch.randint(0, V, (T, 5), device="cuda")
    t = _rand((T, 5), torch.float32, 31)
    ids[::3] = -1
    z[::3] = float("nan")
    up = torch.ones(T, device="cuda")
    up[1::3] = 0.0
    leaf = z.detach().requires_grad_()
    loss = ops.token_distillation(leaf, ids, t)
    (g,) = torch.autograd.grad(loss, leaf, up)
    assert (loss[::3] == 0).all() and torch.isfinite(loss).all()
    assert (g[::3] == 0).all() and (g[1::3] == 0).all()
    kept = slice(2, None, 3)
    _check_distill(native, z[kept], ids[kept], t[kept], 1.0)
    alone = z[kept].contiguous().requires_grad_()
    one = ops.token_distillation(alone, ids[kept], t[kept])
    want = torch.autograd.grad(one, alone, up[kept])[0]
    torch.testing.assert_close(loss[kept], one, rtol=2e-6, atol=2e-6)  # sums of other parts
    assert_within(g[kept], want.double(), (torch.finfo(dtype).eps + 4e-6) * want.double().abs(), floor=1e-6)


def test_distillation_gradient_of_far_apart_rows(native):
    """One position of each sequence: the gradient takes no more memory than its own rows."""
    z = _rand((4, 64, 1000), torch.bfloat16, 32)
    ids, t = torch.randint(0, 1000, (4, 6), device="cuda"), _rand((4, 6), torch.float32, 33)
    for rows in (z[:, -1], z[:, 5, 3:900], z[:, 5, 8:901]):
        ids_in = ids % rows.shape[1]
        _check_distill(native, rows, ids_in, t, 1.0)
        leaf = rows.detach().requires_grad_()
        (g,) = torch.autograd.grad(ops.token_distillation(leaf, ids_in, t).sum(), leaf)
        assert g.untyped_storage().nbytes() <= rows.numel() * 2 + 256


def test_distillation_is_reproducible(native):
    z = _rand((5, 50257), torch.float32, 16).requires_grad_()
    ids, t = torch.randint(0, 9, (5, 100), device="cuda"), _rand((5, 100), torch.float32, 17)
    runs = []
    for _ in range(2):
        loss = ops.token_distillation(z, ids, t)
        runs.append((loss.detach(), torch.autograd.grad(loss.sum(), z)[0]))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


# --------------------------------------------------------------------------- #
# streams and graphs
# --------------------------------------------------------------------------- #


def _step(q, k, v, cos, sin, p, w, ids, t):
    q2, k2 = ops.packed_rotary(q, k, cos, sin, 64, p)
    o = ops.packed_causal_attention(q2, k2, v, p)
    logits = o.flatten(1) @ w
    loss = ops.token_distillation(logits, ids, t, 2.0)
    return loss, torch.autograd.grad(loss.sum(), (q, k, v))


def _step_inputs(seed):
    lens = [100, 60, 97]
    p = ops.PackedSequences(lens, device="cuda")
    q, k, v = (_rand((257, h, 64), torch.bfloat16, seed + i).requires_grad_() for i, h in enumerate((4, 2, 2)))
    cos, sin = ops.rotary_tables(100, 64, 1e4, "cuda")
    w = _rand((256, 1000), torch.bfloat16, seed + 3, std=0.1)
    ids = torch.randint(0, 1000, (257, 8), device="cuda")
    return [q, k, v, cos, sin, p, w, ids, _rand((257, 8), torch.float32, seed + 4)]


def test_two_streams_at_once(native):
    a, b = _step_inputs(200), _step_inputs(300)
    want = [_step(*x) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append([_step(*x) for _ in range(5)])
    torch.cuda.synchronize()
    for (loss, grads), runs in zip(want, got):
        for l2, g2 in runs:
            assert torch.equal(loss, l2) and all(torch.equal(x, y) for x, y in zip(grads, g2))


def test_captured_and_replayed(native):
    """Two captured steps replayed in turn, with new values in the captured inputs."""
    steps = [_step_inputs(400), _step_inputs(500)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for x in steps:
            _step(*x)
    torch.cuda.synchronize()
    for x in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, grads = _step(*x)
            loss = loss.detach()
        graphs.append(g)
        outs.append((loss, grads))
    for turn in range(3):
        for x in steps:
            with torch.no_grad():
                x[0].copy_(_rand(x[0].shape, torch.bfloat16, 600 + turn))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, (loss, grads) in zip(steps, outs):
            l2, g2 = _step(*x)
            assert torch.equal(loss, l2.detach()) and all(torch.equal(a, b) for a, b in zip(grads, g2))


def test_capture_over_a_leaf_of_a_living_eager_graph_is_refused(native):
    x = _step_inputs(600)
    q, k, v, cos, sin, p, w, ids, t = x
    alive = ops.packed_causal_attention(q, k, v, p)
    turned = ops.packed_rotary(q, k, cos, sin, 64, p)
    z = _rand((257, 1000), torch.bfloat16, 601).requires_grad_()
    loss = ops.token_distillation(z, ids, t)
    torch.cuda.synchronize()
    calls = (lambda: ops.packed_causal_attention(q, k, v, p), lambda: ops.packed_rotary(q, k, cos, sin, 64, p),
             lambda: ops.token_distillation(z, ids, t))
    for call in calls:
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    torch.cuda.synchronize()
    del alive, turned, loss
    want = _step(*x)
    want = (want[0].detach(), want[1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, grads = _step(*x)
        loss = loss.detach()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))
