"""Packed attention, rotary and distillation where values, gradients and calls are out of the ordinary."""

import math

import pytest
import torch

from bergson_b200 import ops

from .packed_reference import assert_within, attention64
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
