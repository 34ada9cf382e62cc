"""Documents of different lengths in one token axis, without padding between them.

``PackedSequences`` is the plan of such a batch: made once from the documents' lengths, used by every
layer and in both directions.  ``packed_causal_attention`` attends inside each document,
``packed_rotary`` turns q and k by the positions inside each document; both stand beside
``causal_attention`` and ``rotary`` of the rectangular batches and pick their path the same way: the
sm_100a kernels on CUDA (their graph nodes are in the extension), differentiable torch expressions on the
CPU and inside ``ops.composable()``.  The kernels' backward passes cannot be differentiated again.
"""

from __future__ import annotations

import math
from typing import Sequence

import numpy as np
import torch
from torch import Tensor

from . import native
from .functional import causal_attention_ref, new_causal_bias, rotary_pairs, use_fused

_TILE = 128  # rows of the kernels' tiles
_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class PackedSequences:
    """Plan of a packed batch.

    ``lengths``: the documents' lengths in their order (0 allowed), on the host.  ``total``: rows of the
    batch's tensors (default: the sum of the lengths); the rows behind the last document belong to
    nobody: attention gives zeros there.  The plan's tensors are on ``device`` when the constructor
    returns, so any stream may use them, and the plan may be dropped while it does.  A plan is made before a
    capture begins; the captured graph replays its lengths, so it is kept as long as the graph is.
    """

    def __init__(self, lengths: Sequence[int] | np.ndarray | Tensor, device="cpu", total: int | None = None):
        if isinstance(lengths, Tensor):
            if lengths.is_cuda:
                raise ValueError("lengths are read on the host: pass a list, an array or a CPU tensor")
            lengths = lengths.numpy()
        lens = np.asarray(lengths)
        if lens.ndim != 1 or (lens.size and lens.dtype.kind not in "iu"):
            raise ValueError("lengths must be a flat sequence of whole numbers")
        lens = lens.astype(np.int64)
        if lens.size and lens.min() < 0:
            raise ValueError(f"negative length {int(lens.min())}")
        self.lengths = tuple(int(n) for n in lens)
        self.num_tokens = int(lens.sum())
        self.rows = self.num_tokens if total is None else int(total)
        if self.rows < self.num_tokens:
            raise ValueError(f"total {self.rows} is less than the {self.num_tokens} tokens of the documents")
        if self.rows >= 1 << 30:
            raise ValueError(f"{self.rows} rows: at most {(1 << 30) - 1}")
        self.max_length = int(lens.max()) if lens.size else 0

        rows, valid = self.rows, self.num_tokens
        ends = np.cumsum(lens)
        begins = ends - lens
        at = np.arange(rows, dtype=np.int64)
        first_key, end_query, position = at + 1, at.copy(), np.zeros(rows, np.int64)
        first_key[:valid] = np.repeat(begins, lens)
        end_query[:valid] = np.repeat(ends, lens)
        position[:valid] = at[:valid] - first_key[:valid]
        # Tiles of 128 rows with what their blocks need to know, by their work, most first: blocks are dealt
        # in this order, and a long tile that starts last would be waited for.
        row0 = np.arange(0, rows, _TILE)
        end = np.minimum(row0 + _TILE, valid)
        some = end > row0
        first = np.minimum(row0, max(valid - 1, 0))
        last = np.maximum(end - 1, 0)
        query = np.zeros((len(row0), 4), np.int64)  # first row, first key of it, first key of the last row, last key + 1
        query[:, 0] = row0
        key = np.zeros((len(row0), 4), np.int64)  # first key, last query + 1, the same of the first key alone
        key[:, 0] = key[:, 1] = row0
        if valid:
            query[some, 1:] = np.stack([first_key[first], first_key[last], end], 1)[some]
            key[some, 1:3] = np.stack([end_query[last], end_query[first]], 1)[some]
        work = query[:, 3] - query[:, 1]
        if len(row0) % 2:  # pairs of neighbouring tiles: the last one alone has an empty second
            query = np.concatenate([query, [[rows + _TILE, 0, 0, 0]]])
            pair_work = np.append(work, 0)
        else:
            pair_work = work
        pairs = query.reshape(-1, 8)[np.argsort(-pair_work.reshape(-1, 2).max(1), kind="stable")]
        query = query[np.argsort(-work, kind="stable")]
        key = key[np.argsort(-(key[:, 1] - key[:, 0]), kind="stable")]
        parts = [query, pairs, key, first_key, end_query, position, np.concatenate([[0], ends])]
        flat = np.concatenate([x.reshape(-1) for x in parts]).astype(np.int32)
        with torch.inference_mode(False):  # a graph may save the tables, wherever the plan was made
            table = torch.from_numpy(flat).to(device)
            (self.query_tiles, self.query_pairs, self.key_tiles, self.first_key, self.end_query, self.position,
             self.cu_seqlens) = table.split([x.size for x in parts])
        self.device = table.device
        self._tables = (self.first_key, self.end_query, self.query_tiles, self.query_pairs, self.key_tiles)

    def __repr__(self) -> str:
        return f"PackedSequences({len(self.lengths)} documents, {self.num_tokens} tokens, {self.rows} rows)"

    def tables(self):
        """What the attention kernels read of the plan."""
        return self._tables

    def spans(self):
        """(begin, end) of each document that has tokens."""
        at = 0
        for n in self.lengths:
            if n:
                yield at, at + n
            at += n

    def mask_labels(self, labels: Tensor, ignore_index: int = -100) -> Tensor:
        """``labels`` ``[..., rows]`` without each document's first token, which no token of its own
        document predicts, and without the rows behind the last document."""
        if labels.shape[-1] != self.rows:
            raise ValueError(f"labels of {labels.shape[-1]} rows for a packing of {self.rows}")
        own = self.position > 0  # rows behind the last document have position 0
        return labels.masked_fill(~own.to(labels.device), ignore_index)


def _check(name: str, packing: PackedSequences, q: Tensor, *others: Tensor) -> None:
    if type(packing) is not PackedSequences and not isinstance(packing, PackedSequences):
        raise TypeError(f"{name}: packing must be a PackedSequences, got {type(packing).__name__}")
    dtype, device, rows = q.dtype, q.device, packing.rows
    for t in (q, *others):
        if t.ndim != 3:
            raise ValueError(f"{name}: [tokens, heads, features] expected, got shape {tuple(t.shape)}")
        if t.dtype != dtype or t.device != device or not dtype.is_floating_point:
            raise ValueError(f"{name}: operands of one floating-point dtype and one device expected")
        if t.shape[0] != rows:
            raise ValueError(f"{name}: {t.shape[0]} rows for a packing of {rows}")
        if t.shape[2] != q.shape[2] or t.shape[2] == 0:
            raise ValueError(f"{name}: head sizes {q.shape[2]} and {t.shape[2]}")
    if q.is_cuda and packing.device != q.device:
        raise ValueError(f"{name}: packing on {packing.device}, operands on {q.device}")


# --------------------------------------------------------------------------- #
# attention
# --------------------------------------------------------------------------- #


def packed_causal_attention_ref(q: Tensor, k: Tensor, v: Tensor, packing: PackedSequences, scale: float) -> Tensor:
    """Document by document with differentiable torch operations."""
    parts = []
    bias = new_causal_bias(packing.max_length, q.dtype, q.device)  # the longest document's; every other one is a corner of it
    for begin, end in packing.spans():
        one = [x[begin:end].transpose(0, 1)[None] for x in (q, k, v)]
        parts.append(causal_attention_ref(*one, scale, bias[: end - begin, : end - begin])[0].transpose(0, 1))
    if packing.rows > packing.num_tokens or not parts:
        # zeros that stay in the graph, whatever stands there
        behind = q[packing.num_tokens :] if parts else q + (k.sum() + v.sum())
        parts.append(behind.masked_fill(torch.ones((), dtype=torch.bool, device=q.device), 0.0))
    return torch.cat(parts)


def packed_causal_attention(q: Tensor, k: Tensor, v: Tensor, packing: PackedSequences,
                            scale: float | None = None) -> Tensor:
    """Causal attention inside each document of a packed batch.

    q: ``[rows, Hq, D]``; k, v: ``[rows, Hkv, D]`` (Hq a multiple of Hkv); returns ``[rows, Hq, D]``.
    Row t attends the rows of its own document up to t; nothing that stands in other documents or behind
    the last one, not even an infinity or NaN, reaches it.  Rows behind the last document give zeros and
    get zero gradients.  ``scale`` (default ``1 / sqrt(D)``) must be positive.  The kernels take bf16, fp16 and fp32 with D a
    multiple of 8 up to 128; views of a fused projection are read in place.  Other dtypes and head sizes
    run document by document on torch operations.

    A kernel that gives up on one of its bounded waits leaves its results incomplete; the next call on that device
    raises (``ops.attribution.kernel_status`` tells at once, by waiting for the device).
    """
    _check("packed_causal_attention", packing, q, k, v)
    if k.shape != v.shape:
        raise ValueError(f"packed_causal_attention: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"packed_causal_attention: {q.shape[1]} query heads over {k.shape[1]} key heads")
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"packed_causal_attention: scale must be positive, got {scale}")
    if q.dtype in _KERNEL_DTYPES and q.shape[2] % 8 == 0 and q.shape[2] <= 128 and use_fused(q):
        if q.numel() == 0:
            return q + (k.sum() + v.sum())  # no rows or no heads: nothing to launch, and a place in the graph
        return native.packed_attention(q, k, v, *packing.tables(), packing.num_tokens, scale)
    return packed_causal_attention_ref(q, k, v, packing, scale)


# --------------------------------------------------------------------------- #
# rotary embedding
# --------------------------------------------------------------------------- #


def packed_rotary(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, rot_dim: int,
                  packing: PackedSequences) -> tuple[Tensor, Tensor]:
    """Rotary embedding of q ``[rows, Hq, D]`` and k ``[rows, Hkv, D]`` at each document's own positions.

    ``cos``, ``sin``: ``[positions, rot_dim / 2]`` as ``rotary_tables`` gives them, at least as many
    positions as the longest document has tokens.  The first ``rot_dim`` features of a head turn in pairs
    ``(i, i + rot_dim / 2)``; the rest are copied.  Rows behind the last document count as position 0.  The
    tables get no gradient.
    """
    _check("packed_rotary", packing, q, k)
    if rot_dim % 2 or not 0 < rot_dim <= q.shape[2]:
        raise ValueError(f"packed_rotary: rot_dim {rot_dim} for heads of {q.shape[2]} features")
    if cos.shape != sin.shape or cos.ndim != 2 or cos.shape[1] != rot_dim // 2:
        raise ValueError(f"packed_rotary: tables [positions, {rot_dim // 2}] expected, got {tuple(cos.shape)}")
    if cos.shape[0] < max(1, packing.max_length) and packing.rows:
        raise ValueError(f"packed_rotary: tables of {cos.shape[0]} positions for documents of {packing.max_length}")
    if cos.device != q.device or sin.device != q.device:
        raise ValueError(f"packed_rotary: tables on {cos.device}, operands on {q.device}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("packed_rotary: the tables get no gradient")
    if q.dtype in _KERNEL_DTYPES and q.shape[2] <= 256 and use_fused(q) and q.numel() and k.numel():
        cos, sin = cos.float().contiguous(), sin.float().contiguous()
        return native.packed_rotary(q, k, cos, sin, packing.position, rot_dim)
    at = packing.position.to(q.device, torch.int64)
    c, s = cos[at][:, None].to(q.dtype), sin[at][:, None].to(q.dtype)
    return rotary_pairs(q, c, s, rot_dim), rotary_pairs(k, c, s, rot_dim)
