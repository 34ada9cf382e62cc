"""Models on packed documents: the same as document by document, in the forward pass, the loss and the gradients."""

import pytest
import torch

from bergson_b200 import ops
from bergson_b200.models import load_model

FAMILIES = {
    "llama": "native:llama-tiny?seed=3",
    "gpt_neox": "native:gpt_neox?vocab_size=512&hidden_size=64&intermediate_size=128&num_hidden_layers=2"
                "&num_attention_heads=4&rotary_pct=0.5&max_position_embeddings=512&seed=4",
    "gpt2": "native:gpt2-tiny?seed=5",
}


def batch(lens, pad, device="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 512, (1, sum(lens) + pad), generator=g).to(device)
    return ids, ops.PackedSequences(lens, device=device, total=sum(lens) + pad)


def spans(lens):
    at = 0
    for n in lens:
        if n:
            yield slice(at, at + n)
        at += n


@pytest.mark.parametrize("family", FAMILIES)
@pytest.mark.parametrize("lens,pad", [([9, 1, 0, 14], 0), ([20], 3), ([5, 6], 1)])
def test_packed_equals_document_by_document(family, lens, pad):
    model = load_model(FAMILIES[family], dtype=torch.float64)
    ids, packing = batch(lens, pad)
    out = model(ids, labels=ids, packing=packing)
    out.loss.backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    total, count = 0.0, 0
    for s in spans(lens):
        one = model(ids[:, s])
        torch.testing.assert_close(out.logits[:, s], one.logits, rtol=1e-9, atol=1e-10)
        if s.stop - s.start > 1:
            lp = torch.log_softmax(one.logits[0, :-1], -1)
            total = total - lp.gather(1, ids[0, s][1:, None]).sum()
            count += s.stop - s.start - 1
    (total / count).backward()
    torch.testing.assert_close(out.loss, (total / count).detach(), rtol=1e-9, atol=1e-10)
    for n, p in model.named_parameters():
        torch.testing.assert_close(grads[n], p.grad, rtol=1e-7, atol=1e-10, msg=n)


@pytest.mark.parametrize("family", FAMILIES)
def test_packed_with_checkpointing_and_traced_ops(family):
    model = load_model(FAMILIES[family], dtype=torch.float64)
    ids, packing = batch([7, 5], 0)
    plain = model(ids, labels=ids, packing=packing).loss
    model.gradient_checkpointing_enable()
    torch.testing.assert_close(model(ids, labels=ids, packing=packing).loss, plain)
    with ops.composable():
        torch.testing.assert_close(model(ids, labels=ids, packing=packing).loss, plain)


def test_packed_refusals():
    model = load_model(FAMILIES["gpt2"], dtype=torch.float32)
    ids, packing = batch([7, 5], 0)
    for bad in (ids[:, :11], ids[0], ids.expand(2, -1)):
        with pytest.raises(ValueError):
            model(bad, packing=packing)
    long, plan = batch([300], 0)  # gpt2-tiny has 256 learned positions
    with pytest.raises(ValueError):
        model(long, packing=plan)


# --------------------------------------------------------------------------- #
# on the kernels: a distillation step on packed documents
# --------------------------------------------------------------------------- #

LENS, PAD = [40, 1, 130, 0, 77], 8


def _step(model, ids, packing, teacher_ids, teacher_logits, weight):
    """Attention, rotary embedding and distillation together, as a training step of a student uses them."""
    logits = model(ids, packing=packing).logits[0]
    loss = ops.token_distillation(logits, teacher_ids, teacher_logits, temperature=2.0)
    (loss * weight).sum().backward()
    grads = {n: p.grad.detach().clone() for n, p in model.named_parameters()}
    model.zero_grad()
    return loss.detach(), grads


def _by_document(model, ids, teacher_ids, teacher_logits, weight):
    for s in spans(LENS):
        logits = model(ids[:, s]).logits[0]
        loss = ops.token_distillation(logits, teacher_ids[s], teacher_logits[s], temperature=2.0)
        (loss * weight[s]).sum().backward()
    grads = {n: p.grad.detach().clone() for n, p in model.named_parameters()}
    model.zero_grad()
    return grads


def _off(a, b):
    """2-norm of the difference over the 2-norm, of all parameters' gradients together."""
    d = sum((a[n].double().cpu() - b[n].double().cpu()).square().sum() for n in b)
    return (d / sum(b[n].double().square().sum().cpu() for n in b)).sqrt().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("family", FAMILIES)
def test_distillation_step_on_packed_documents(family, dtype):
    from bergson_b200.ops import native

    exact = load_model(FAMILIES[family], dtype=torch.float64)
    model = load_model(FAMILIES[family], dtype=dtype, device="cuda")
    exact.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})
    ids, _ = batch(LENS, PAD)
    g = torch.Generator().manual_seed(1)
    rows = sum(LENS) + PAD
    teacher_ids = torch.randint(0, 512, (rows, 16), generator=g)
    teacher_ids[sum(LENS):] = -1  # nothing to learn behind the last document
    teacher_logits = torch.randn(rows, 16, generator=g) * 2
    weight = torch.rand(rows, generator=g)
    want = _by_document(exact, ids, teacher_ids, teacher_logits, weight)
    there = [x.cuda() for x in (ids, teacher_ids, teacher_logits, weight)]
    native.reset_launch_count()
    loss, got = _step(model, there[0], ops.PackedSequences(LENS, device="cuda", total=rows), *there[1:])
    assert native.launch_count() > 0 and int(native.kernel_status(0).item()) == 0
    assert loss[sum(LENS):].abs().max() == 0
    separate = _by_document(model, *there)
    # The packed step rounds where the documents' own steps do: it may be as far from 64 bits as they are, by
    # a factor for the few roundings that differ (the kernels' P and dS), and never by more than a thousandth
    # in fp32 (some hundred roundings of 6e-8 in a row, amplified by the softmaxes).
    assert _off(got, want) <= max(2 * _off(separate, want), 1e-5)
    if dtype == torch.float32:
        assert _off(got, want) <= 1e-3
