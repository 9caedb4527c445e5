"""Attention over documents of different lengths packed one behind the other into one token axis.

A training batch that is filled with documents has no padding and no attention across documents;
`flash_attention` knows batches of equal-length sequences only. The documents of a batch are
described once by a `PackedLayout`, which every layer's forward and backward then use.
"""
from __future__ import annotations

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import native, raw

_TILE = 128     # rows of a query or key tile of the kernels (csrc/attention_packed_sm100.cu)


class PackedLayout:
    """Documents of `lengths` tokens, one behind the other from row 0, on an axis of `total` rows (their
    sum by default; more rows belong to no document: outputs and gradients there are 0).

    `lengths` are whole numbers >= 0 known on the host: a sequence, an array or a CPU tensor (a CUDA
    tensor is copied back, which waits for its stream). On a CUDA `device` the kernels' work lists are
    built and copied there once (about 0.1 ms of host time for tens of documents), so a layout is made per
    batch, outside CUDA graph capture, and kept."""

    def __init__(self, lengths, device="cpu", total=None):
        if isinstance(lengths, torch.Tensor):
            lengths = lengths.detach().cpu().numpy()
        lengths = np.asarray(lengths)
        if lengths.size == 0:
            lengths = lengths.astype(np.int64)
        if lengths.ndim != 1 or lengths.dtype.kind not in "iu":
            raise ValueError("PackedLayout: lengths must be a 1-D sequence of whole numbers")
        if lengths.size and int(lengths.min()) < 0:
            raise ValueError("PackedLayout: a document cannot have fewer than 0 tokens")
        if lengths.size and int(lengths.max()) >= 2 ** 31:      # also keeps the 64-bit sum below from wrapping
            raise ValueError(f"PackedLayout: a document of {int(lengths.max())} tokens is too long")
        lengths = lengths.astype(np.int64)
        self.used = int(lengths.sum())
        self.total = self.used if total is None else int(total)
        if total is not None and self.total != total:
            raise ValueError(f"PackedLayout: total must be a whole number, got {total}")
        if not self.used <= self.total < 2 ** 31 - 256:
            raise ValueError(f"PackedLayout: documents of {self.used} tokens do not fit {self.total} rows")
        self.lengths = tuple(int(n) for n in lengths)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._lists = None
        if self.device.type == "cuda":
            native.status(self.device)      # a call inside a graph capture must not be the one that makes it
            parts = list(self._work_lists(lengths))
            host = torch.from_numpy(np.concatenate([x for _, x in parts]))
            flat = host.to(self.device)
            tables, at = {}, 0
            for name, x in parts:
                tables[name] = flat[at:at + len(x)]
                at += len(x)
            self._lists = {True: (tables["causal128"], tables["causal256"], tables["keys128"]),
                           False: (tables["full128"], tables["full256"], tables["full128"])}

    def documents(self):
        """(first row, rows) of every document that has tokens."""
        at = 0
        for n in self.lengths:
            if n:
                yield at, n
            at += n

    @staticmethod
    def _work_lists(lengths):
        """(name, int32 [n, 4] rows (start, len, tile, 0)): one row per tile, heaviest first. Under the
        causal mask query tile i meets i + 1 key tiles and key tile j meets tiles - j query tiles;
        without it every tile meets all tiles of its document."""
        starts = np.cumsum(lengths) - lengths
        for rows in (_TILE, 2 * _TILE):
            count = -(-lengths // rows)
            doc = np.repeat(np.arange(len(lengths)), count)
            tile = np.arange(len(doc)) - np.repeat(np.cumsum(count) - count, count)
            table = np.stack([starts[doc], lengths[doc], tile, np.zeros_like(tile)], 1).astype(np.int32)
            orders = {"causal": -(tile + 1), "full": -count[doc]}
            if rows == _TILE:
                orders["keys"] = tile - count[doc]
            for name, weight in orders.items():
                yield f"{name}{rows}", table[np.argsort(weight, kind="stable")]

    def work_lists(self, causal):
        """The kernels' device tables for one mask: 128-row tiles, 256-row blocks, key tiles."""
        if self._lists is None:
            raise ValueError(f"PackedLayout on {self.device} has no work lists for CUDA tensors")
        return self._lists[bool(causal)]


class _PackedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, layout, scale, causal):
        out, lse = raw.attention_packed_fwd(q, k, v, layout, scale, causal)
        ctx.layout, ctx.scale, ctx.causal = layout, scale, causal
        ctx.save_for_backward(q, k, v, out, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = raw.attention_packed_bwd(d_out, q, k, v, out, lse, ctx.layout, ctx.scale, ctx.causal)
        return dq, dk, dv, None, None, None


def flash_attention_packed(q, k, v, layout, scale=None, causal=True):
    """Flash attention inside each document of `layout`: q [total, heads, head_dim], k / v [total,
    kv_heads, head_dim] with heads a multiple of kv_heads (head h reads key/value head
    h // (heads / kv_heads)); returns [total, heads, head_dim].

    On CUDA: fp16 / bf16, head_dim 64 or 128; views such as the q, k and v slices of one projection are
    read in place, what a tensor map cannot address is copied. A document attends to itself only: what
    stands in other documents or behind the last one, infinities and NaN included, does not reach it.
    P and dS are rounded to the input type for the tensor cores, sums are fp32. Where a gradient is needed,
    the forward also keeps what rounding took off its result (one more tensor like it) for the backward.
    Waits inside the kernels are bounded: one that gave up leaves results unwritten and a mark that
    `native.check_status` raises on, which a training loop calls once per step.
    `scale` (1e-30 to 1e3) defaults to 1 / sqrt(head_dim). Scores and their log-sum-exp are fp32: a scaled
    score of magnitude x is off by about x 2^-22, its probability by that part of itself (from x = 10^8 on,
    results would not be finite)."""
    if native.use_native(q):     # the autograd node is native too
        return native.lib().flash_attention_packed(q, k, v, *layout.work_lists(causal), layout.used, layout.total,
                                                   scale, bool(causal),
                                                   native.status(q.device))
    return _PackedAttnFn.apply(q, k, v, layout, scale, bool(causal))
