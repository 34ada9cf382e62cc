"""Measured calls of the packed-sequence operators: attention over packed documents, rotary embedding
at each document's own positions, and distillation from a teacher's top logits.

``own`` selects what ``run`` does: the plain forms written with elementary torch operations (fp32), or
the framework's public entry points.  ``prepare`` makes the inputs and the plan that a program keeps.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------


def _attention(train, dtype, heads, kv_heads, head_dim, docs, tokens, spread, pad=0, fused=False, lens_seed=1):
    """``docs`` documents that hold ``tokens`` tokens together, lengths log-normally spread by
    ``spread`` (0: all alike); ``pad`` rows behind the last one; ``fused``: q, k, v are views of one
    projection's output, ``[tokens, heads, 3 * head_dim]``."""
    return {"op": "attention", "train": train, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "docs": docs, "tokens": tokens, "spread": spread, "pad": pad, "fused": fused,
            "lens_seed": lens_seed}


def _rotary(train, dtype, heads, kv_heads, head_dim, rot_dim, docs, tokens, spread, pad=0, fused=False, lens_seed=1):
    return {"op": "rotary", "train": train, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rot_dim": rot_dim, "docs": docs, "tokens": tokens, "spread": spread, "pad": pad,
            "fused": fused, "lens_seed": lens_seed}


def _distill(train, dtype, tokens, vocab, top, temperature, holes=0.0, pitch=0):
    """``top`` teacher entries a token, a share ``holes`` of them unused (id -1); ``pitch``: row pitch
    of the logits where they are a view of a wider buffer (0: contiguous)."""
    return {"op": "distill", "train": train, "dtype": dtype, "tokens": tokens, "vocab": vocab, "top": top,
            "temperature": temperature, "holes": holes, "pitch": pitch}


def listed():
    cases = [
        # One short question through a tiny grouped-head model: launch latency is all there is.
        ("attn_fwd_short_query", _attention(False, "bf16", 4, 2, 16, 1, 37, 0.0)),
        # Forward pass (scoring without gradients) of a ragged batch of web documents, 8-billion-parameter heads.
        ("attn_fwd_ragged_8k", _attention(False, "bf16", 32, 8, 128, 19, 8192, 0.9, pad=0)),
        # Gradient collection on a packed 16k-token batch, the same heads: the ordinary build step.
        ("attn_train_ragged_16k", _attention(True, "bf16", 32, 8, 128, 24, 16321, 1.0, pad=63)),
        # Many short facts packed into one batch (recall-style data), 12 heads of 64, fused projection, fp16.
        ("attn_train_facts_fp16", _attention(True, "fp16", 12, 12, 64, 211, 8187, 0.5, pad=5, fused=True)),
        # One long document: the quadratic part at full size.
        ("attn_train_long_16k", _attention(True, "bf16", 32, 8, 128, 1, 16384, 0.0)),
        # Full-precision run of a small model (numerics checks, twice-differentiated baselines).
        ("attn_train_fp32_small", _attention(True, "fp32", 4, 4, 32, 7, 2000, 0.7, fused=True)),
        # Rotation of a tiny batch: latency.
        ("rotary_short_query", _rotary(False, "bf16", 4, 2, 16, 16, 1, 37, 0.0)),
        # Rotation and its gradient at the packed 16k batch.
        ("rotary_train_ragged_16k", _rotary(True, "bf16", 32, 8, 128, 128, 24, 16321, 1.0, pad=63)),
        # A handful of supervised tokens of one query, odd vocabulary, fp32 logits: few rows, long rows.
        ("distill_train_query_fp32", _distill(True, "fp32", 5, 50257, 20, 2.0)),
        # Validation pass of a student at a 128k vocabulary, loss only.
        ("distill_fwd_128k", _distill(False, "bf16", 4096, 128256, 64, 1.0)),
        # Training step of the student at the same vocabulary, some entries unused.
        ("distill_train_128k", _distill(True, "bf16", 4096, 128256, 128, 2.0, holes=0.1)),
        # Logits as the view of a padded head's output, odd vocabulary.
        ("distill_train_padded_50k", _distill(True, "fp16", 2047, 50257, 32, 1.5, holes=0.3, pitch=50264)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "distill", "distill"])
    train = rng.random() < 0.6
    if op == "distill":
        vocab = _log_int(rng, 512, 131072)
        # fp32 logits at most 1 GB, 16-bit ones 1.05 GB
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = max(1, min(8192, (4096 * 128256 if dtype != "fp32" else 2048 * 128256) // vocab))
        tokens = _log_int(rng, 1, most)
        pitch = -(-vocab // 8) * 8 if rng.random() < 0.4 else 0
        return _distill(train, dtype, tokens, vocab, _log_int(rng, 1, min(256, vocab)),
                        rng.choice([1.0, 1.5, 2.0, 4.0]), rng.choice([0.0, 0.0, 0.2]), pitch)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    head_dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12])
    heads = kv_heads * rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * kv_heads <= 32])
    tokens = _log_int(rng, 1, 16384)
    docs = _log_int(rng, 1, max(1, min(300, tokens // 2)))
    if dtype == "fp32":
        # full precision is for small models: at most 2048 tokens to a document on average
        head_dim, tokens = min(head_dim, 64), min(tokens, 4096)
        docs = min(docs, tokens)
    fused = heads == kv_heads and rng.random() < 0.5
    pad = rng.choice([0, 0, 1, 7, 100])
    spread = rng.choice([0.0, 0.5, 1.0])
    seed = rng.randrange(1 << 20)
    if op == "attention":
        return _attention(train, dtype, heads, kv_heads, head_dim, docs, tokens, spread, pad, fused, seed)
    rot = head_dim if rng.random() < 0.6 else max(2, head_dim // 4 // 2 * 2)
    return _rotary(train, dtype, heads, kv_heads, head_dim, rot, docs, tokens, spread, pad, fused, seed)


def _lengths(case):
    """Lengths of the documents: positive, ``tokens`` together."""
    n, total = case["docs"], case["tokens"]
    rng = np.random.default_rng(case["lens_seed"])
    w = np.exp(case["spread"] * rng.standard_normal(n))
    lens = np.maximum(1, np.floor(w / w.sum() * (total - n)).astype(np.int64) + 1)
    lens[np.argmax(lens)] += total - lens.sum()
    return [int(x) for x in lens]


def _rows(case):
    return case["tokens"] + case["pad"]


# --------------------------------------------------------------------------------------------------
# work
# --------------------------------------------------------------------------------------------------


def work(case):
    item = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        pairs = sum(n * (n + 1) // 2 for n in _lengths(case))
        d, hq, hk, t = case["head_dim"], case["heads"], case["kv_heads"], _rows(case)
        byt = item * d * t * (2 * hq + 2 * hk)  # q, o; k, v
        flops = 4 * d * hq * pairs
        if case["train"]:
            byt += item * d * t * (2 * hq + 2 * hk)  # do, dq; dk, dv
            flops += 10 * d * hq * pairs
        return {"bytes": byt, "flops": flops}
    if case["op"] == "rotary":
        n = _rows(case) * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        times = 2 if case["train"] else 1
        table = 4 * case["rot_dim"] * max(_lengths(case))
        return {"bytes": times * 2 * item * n + table, "flops": times * 3 * n}
    n = case["tokens"] * case["vocab"]
    small = case["tokens"] * case["top"] * 12 + case["tokens"] * 8
    return {"bytes": (2 if case["train"] else 1) * n * item + small, "flops": (6 if case["train"] else 3) * n}


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(to)

    state = {"case": case}
    if case["op"] == "distill":
        t, v, k = case["tokens"], case["vocab"], case["top"]
        pitch = case["pitch"] or v
        logits = torch.empty(t, pitch, device="cuda", dtype=dtype)
        ids = torch.empty(t, k, device="cuda", dtype=torch.int64)
        top = torch.empty(t, k, device="cuda", dtype=torch.float32)
        for r in range(0, t, 512):  # slices: the teacher's full rows are not kept
            n = min(512, t - r)
            z = torch.randn(n, pitch, generator=g, device="cuda") * 2.5
            teacher = z[:, :v] + torch.randn(n, v, generator=g, device="cuda")
            top[r:r + n], ids[r:r + n] = teacher.topk(k, dim=1)
            logits[r:r + n] = z
        if case["holes"]:
            hole = torch.rand(t, k, generator=g, device="cuda") < case["holes"]
            ids.masked_fill_(hole, -1)
        state.update(logits=logits[:, :v], ids=ids, top=top)
        if case["train"]:
            # The mean over the tokens; fp16 gradients come scaled, as a program must scale them to keep them
            # above the type's smallest values.
            scale = 64.0 if dtype == torch.float16 else 1.0 / t
            state["dloss"] = torch.rand(t, generator=g, device="cuda") * scale
    else:
        hq, hk, d, rows, lens = case["heads"], case["kv_heads"], case["head_dim"], _rows(case), _lengths(case)
        if case["fused"]:
            q, k, v = normal(rows, hq, 3 * d).split(d, dim=-1)
        else:
            q, k, v = normal(rows, hq, d), normal(rows, hk, d), normal(rows, hk, d)
        state["lens"] = lens
        if own:
            from bergson_b200 import ops

            state["packing"] = ops.PackedSequences(lens, device="cuda", total=rows)
        elif case["op"] == "rotary":
            pos = np.concatenate([np.arange(n) for n in lens] + [np.zeros(case["pad"], np.int64)])
            state["pos"] = torch.from_numpy(pos).cuda()
        if case["op"] == "attention":
            state.update(q=q, k=k, v=v)
            if case["train"]:
                state["do"] = normal(rows, hq, d, std=0.05)
        else:
            rot = case["rot_dim"]
            inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
            ang = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * inv
            state.update(q=q, k=k, cos=ang.cos().float(), sin=ang.sin().float())
            if case["train"]:
                state.update(dq=normal(rows, hq, d, std=0.05), dk=normal(rows, hk, d, std=0.05))
    if case["train"] and own:
        # Leaves of the step; the graph is built anew in every pass.
        for name in ("logits",) if case["op"] == "distill" else ("q", "k", "v"):
            if name in state:
                state[name] = state[name].detach().requires_grad_()
    return state


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rotary": _own_rotary, "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"attention": _plain_attention, "rotary": _plain_rotary, "distill": _plain_distill}[op](state)


def _own_attention(s):
    from bergson_b200 import ops

    if not s["case"]["train"]:
        with torch.no_grad():
            return ops.packed_causal_attention(s["q"], s["k"], s["v"], s["packing"])
    o = ops.packed_causal_attention(s["q"], s["k"], s["v"], s["packing"])
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_rotary(s):
    from bergson_b200 import ops

    rot = s["case"]["rot_dim"]
    if not s["case"]["train"]:
        with torch.no_grad():
            q, k = ops.packed_rotary(s["q"], s["k"], s["cos"], s["sin"], rot, s["packing"])
        return {"q": q, "k": k}
    q, k = ops.packed_rotary(s["q"], s["k"], s["cos"], s["sin"], rot, s["packing"])
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _own_distill(s):
    from bergson_b200 import ops

    tau = s["case"]["temperature"]
    if not s["case"]["train"]:
        with torch.no_grad():
            return ops.token_distillation(s["logits"], s["ids"], s["top"], temperature=tau)
    loss = ops.token_distillation(s["logits"], s["ids"], s["top"], temperature=tau)
    (dz,) = torch.autograd.grad(loss, s["logits"], s["dloss"])
    return {"loss": loss.detach(), "dlogits": dz}


def _plain_attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    dtype, hq, hk, d = q.dtype, case["heads"], case["kv_heads"], case["head_dim"]
    group, scale, train = hq // hk, 1.0 / math.sqrt(case["head_dim"]), case["train"]
    o = torch.zeros(q.shape, dtype=dtype, device=q.device)
    if train:
        dq, dk = torch.zeros_like(o), torch.zeros(k.shape, dtype=dtype, device=q.device)
        dv = torch.zeros_like(dk)
    at = 0
    for n in s["lens"]:
        rows = slice(at, at + n)
        at += n
        mask = torch.arange(n, device=q.device)[:, None] < torch.arange(n, device=q.device)[None, :]
        step = max(1, min(hk, (1 << 30) // (group * n * n)))  # kv heads at a time: 4 GB of scores
        for h in range(0, hk, step):
            m = min(step, hk - h)
            qf = q[rows, h * group:(h + m) * group].float().permute(1, 0, 2).reshape(m, group, n, d)
            kf = k[rows, h:h + m].float().permute(1, 0, 2)[:, None]
            vf = v[rows, h:h + m].float().permute(1, 0, 2)[:, None]
            p = torch.matmul(qf * scale, kf.transpose(-1, -2)).masked_fill_(mask, float("-inf"))
            p -= p.amax(-1, keepdim=True)
            p = p.exp_()
            p /= p.sum(-1, keepdim=True)
            of = torch.matmul(p, vf)
            o[rows, h * group:(h + m) * group] = of.reshape(m * group, n, d).permute(1, 0, 2).to(dtype)
            if train:
                gf = s["do"][rows, h * group:(h + m) * group].float().permute(1, 0, 2).reshape(m, group, n, d)
                dvf = torch.matmul(p.transpose(-1, -2), gf).sum(1)
                ds = torch.matmul(gf, vf.transpose(-1, -2))
                ds -= (of * gf).sum(-1, keepdim=True)
                ds *= p
                del p
                dqf = torch.matmul(ds, kf) * scale
                dkf = torch.matmul(ds.transpose(-1, -2), qf).sum(1) * scale
                dq[rows, h * group:(h + m) * group] = dqf.reshape(m * group, n, d).permute(1, 0, 2).to(dtype)
                dk[rows, h:h + m] = dkf.permute(1, 0, 2).to(dtype)
                dv[rows, h:h + m] = dvf.permute(1, 0, 2).to(dtype)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if train else o


def _plain_rotary(s):
    rot, half = s["case"]["rot_dim"], s["case"]["rot_dim"] // 2
    c, sn = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]

    def turn(x, sin):
        f = x.float()
        a, b = f[..., :half], f[..., half:rot]
        return torch.cat([a * c - b * sin, b * c + a * sin, f[..., rot:]], dim=-1).to(x.dtype)

    out = {"q": turn(s["q"], sn), "k": turn(s["k"], sn)}
    if s["case"]["train"]:
        out.update(dq=turn(s["dq"], -sn), dk=turn(s["dk"], -sn))
    return out


def _plain_distill(s):
    case, tau, v = s["case"], s["case"]["temperature"], s["case"]["vocab"]
    z = s["logits"].float() / tau
    z -= z.amax(1, keepdim=True)
    lse = z.exp().sum(1, keepdim=True).log()
    valid = s["ids"] >= 0
    t = (s["top"] / tau).masked_fill(~valid, float("-inf"))
    some = valid.any(1, keepdim=True)
    t = torch.where(some, t, torch.zeros_like(t))
    t = t - t.amax(1, keepdim=True)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    p = log_p.exp() * valid
    at = s["ids"].clamp(min=0)
    loss = torch.where(valid, p * (log_p - (z.gather(1, at) - lse)), torch.zeros_like(p)).sum(1) * (tau * tau)
    if not case["train"]:
        return loss
    z -= lse
    dz = z.exp_()
    dz.scatter_add_(1, at, -p)
    dz *= torch.where(some, s["dloss"][:, None] * tau, torch.zeros_like(s["dloss"][:, None]))
    return {"loss": loss, "dlogits": dz.to(s["logits"].dtype)}


# --------------------------------------------------------------------------------------------------
# 64-bit values, from the definitions
# --------------------------------------------------------------------------------------------------


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_distill(case, s)


def _exact_attention(case, s):
    pairs = sum(n * n for n in s["lens"])
    if pairs * case["heads"] * case["head_dim"] > 1.3e12:  # over some 20 s in 64 bits
        return None
    group, rows, hq = case["heads"] // case["kv_heads"], _rows(case), case["heads"]
    o, dq = (torch.zeros(rows, hq, case["head_dim"], dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.zeros(rows, case["kv_heads"], case["head_dim"], dtype=torch.float64, device="cuda") for _ in range(2))
    begin = 0
    for n in s["lens"]:
        at = slice(begin, begin + n)
        begin += n
        i = torch.arange(n, device="cuda")
        hidden = i[None, :] > i[:, None]
        step = max(1, int(2e8) // (n * n))  # heads at a time
        for h in range(0, hq, step):
            to = min(h + step, hq)
            of = torch.arange(h, to, device="cuda") // group  # the key head of each
            leaf = [x.double().transpose(0, 1).contiguous().requires_grad_(case["train"])
                    for x in (s["q"][at, h:to], s["k"][at][:, of], s["v"][at][:, of])]
            logit = (leaf[0] @ leaf[1].mT / math.sqrt(case["head_dim"])).masked_fill(hidden, -math.inf)
            out = torch.softmax(logit, dim=-1) @ leaf[2]
            o[at, h:to] = out.detach().transpose(0, 1)
            if case["train"]:
                grads = torch.autograd.grad(out, leaf, s["do"][at, h:to].double().transpose(0, 1))
                dq[at, h:to] = grads[0].transpose(0, 1)
                dk[at] = dk[at].index_add(1, of, grads[1].transpose(0, 1))
                dv[at] = dv[at].index_add(1, of, grads[2].transpose(0, 1))
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if case["train"] else o


def _exact_rotary(case, s):
    """As a product of complex numbers: (a + ib) e^{i angle}, the tables as given."""
    rot = case["rot_dim"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"]][:, None]

    def apply(x, w):
        x = x.double()
        y = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * w
        return torch.cat([y.real, y.imag, x[..., rot:]], dim=-1)

    out = {"q": apply(s["q"], turn), "k": apply(s["k"], turn)}
    if case["train"]:
        out.update(dq=apply(s["dq"], turn.conj()), dk=apply(s["dk"], turn.conj()))
    return out


def _exact_distill(case, s):
    """Teacher's distribution written into the whole vocabulary, differentiated by autograd, 64 rows at a time."""
    tau, loss, grad = case["temperature"], [], []
    for r in range(0, case["tokens"], 64):
        z = s["logits"][r:r + 64].double().requires_grad_(case["train"])
        ids, top = s["ids"][r:r + 64], s["top"][r:r + 64].double() / tau
        with torch.no_grad():
            used = (ids >= 0) & (ids < case["vocab"])
            e = torch.where(used, (top - top.max(dim=1, keepdim=True).values).exp(), 0.0)
            total = e.sum(1, keepdim=True)
            p = torch.where(total > 0, e / total.clamp(min=1e-300), 0.0)
        log_q = torch.log_softmax(z / tau, dim=1).gather(1, ids.clamp(0, case["vocab"] - 1))
        one = (torch.xlogy(p, p) - torch.where(p > 0, p * log_q, 0.0)).sum(1) * tau ** 2
        loss.append(one.detach())
        if case["train"]:
            grad.append(torch.autograd.grad(one, z, s["dloss"][r:r + 64].double())[0])
            if sum(g.numel() for g in grad) > 7e8:
                return None
    loss = torch.cat(loss)
    return {"loss": loss, "dlogits": torch.cat(grad)} if case["train"] else loss
