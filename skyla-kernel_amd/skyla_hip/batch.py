"""Decoding a batch of sequences: rows of many sequences over a paged KV cache.

The reference's engine serves one sequence over a contiguous cache (kv.rs); this module has
what a server of many needs beside it, over the same weights, arena rows and C-ABI:

  Paged           a pool of pages in the contiguous cache's row layout, and its page table
  BatchKernels    kv_append (QK-norm, rotation, keys and values into their pages) and
                  attention_paged (attention of rows over their pages, a leading run of positions
                  that many rows share read once for all of them)
  LogitsKernels   logits_adjust (penalties for repeated tokens, biases, grammar masks)

The operators read the batch's rows from four words each, {sequence, length, share, 0}: the
row's token is at position length - 1, a row of length 0 has none.  Their push words are in
kernels/batch.hip.
"""
from __future__ import annotations

import dataclasses
from typing import Sequence

import numpy as np

from . import engine as E
from .abi import Buffer, Context, Recorder

MAX_PARTS = 1024        # partials of a row and head (runtime/batch.h)
PAGE_SIZES = tuple(16 << i for i in range(9))  # 16 to 4096 positions
CTL_ROWS, CTL_SHARED, CTL_LEADER = 2, 3, 4     # control words: live rows, shared positions, their sequence


class Paged:
    """A pool of `n_pages` pages of `page` positions for one layer's keys and values (the
    contiguous cache's layout with slots for positions, kv.rs), and a table of up to
    `seq_pages` pages for each of `n_seq` sequences."""

    def __init__(self, precision: E.KvPrecision, page: int, n_pages: int, n_seq: int, seq_pages: int, kv_dim: int):
        if page not in PAGE_SIZES:
            raise ValueError(f"pages of {page} positions: one of {', '.join(map(str, PAGE_SIZES))}")
        if min(n_pages, n_seq, seq_pages, kv_dim) < 1 or kv_dim % 128:
            raise ValueError(f"{n_pages} pages, {n_seq} sequences of {seq_pages} pages, rows of {kv_dim} values")
        self.precision, self.page, self.n_pages = E.KvPrecision(precision), page, n_pages
        self.n_seq, self.seq_pages = n_seq, seq_pages
        self.layout = E.KvLayout(self.precision, [True], n_pages * page, kv_dim)

    @property
    def page_log2(self) -> int:
        return self.page.bit_length() - 1

    def bytes(self) -> int:
        return self.layout.bytes()


@dataclasses.dataclass
class BatchRegions:
    """Arena offsets of a batch: the rows' words, the page table, the attention's partials."""
    rows: int
    table: int
    part: int = 0


@dataclasses.dataclass
class LogitsRegions:
    """Arena offsets and row strides (in words) of what acts on logits: eight words a row, token
    histories, (id, bias) pairs, one-bit masks.  A stride of 0: the batch has none."""
    controls: int
    history: int = 0
    history_stride: int = 0
    bias: int = 0
    bias_stride: int = 0
    mask: int = 0
    mask_stride: int = 0


def splits(rows: int, n_kv: int, rep: int, shared: int, own: int) -> tuple[int, int]:
    """Parts that a batch's attention cuts the shared run and each row's own run into, for
    `shared` shared positions and at most `own` of a row's own: enough workgroups to fill the
    GPU, each with some tiles of 64 positions."""
    def parts(positions: int, groups: int, most: int) -> int:
        tiles = -(-positions // 64)
        return max(1, min(tiles, -(-2048 // max(1, groups)), most))
    n_shared = parts(shared, n_kv * -(-rows * rep // 16), 128) if shared > 0 else 0
    return n_shared, parts(own, n_kv * rows, 512)


def part_size(rows: int, n_head: int, parts: tuple[int, int]) -> int:
    """Words of the partials' region."""
    return rows * n_head * sum(parts) * 130


class BatchKernels:
    """kv_append and attention_paged over one pool buffer for each layer."""

    def __init__(self, ctx: Context, tables: Buffer, a: Buffer, pools: Sequence[Buffer], c: E.Config, paged: Paged):
        if c.head_dim != 128 or c.n_head % c.n_head_kv or c.n_head // c.n_head_kv not in (1, 2, 4, 8):
            raise ValueError(f"no batch attention kernels for head_dim {c.head_dim}, {c.n_head}/{c.n_head_kv} heads")
        if paged.layout.per_layer != paged.n_pages * paged.page * c.n_head_kv * c.head_dim:
            raise ValueError("the pool's rows are not the model's")
        if any(b.size < paged.bytes() for b in pools):
            raise ValueError(f"a pool of {paged.n_pages} pages takes {paged.bytes()} bytes")
        self.c, self.paged = c, paged
        k8, v8 = int(paged.precision.keys_q8), int(paged.precision.values_q8)

        def build(name, bufs, push, spec):
            p = ctx.create_pipeline_sets(name, len(bufs) + 2 if name == "kv_append" else 5, 4 * push, spec, len(pools))
            for i, kv in enumerate(pools):
                p.bind_set_buffers(i, bufs + [kv, kv] + ([] if name == "kv_append" else [kv]))
            return p

        self._append = build("kv_append", [tables, a, a], 24, [k8, v8, 128])
        self._attend = build("attention_paged", [a, a], 19, [c.n_head // c.n_head_kv, k8, v8, 128])
        self._merge = ctx.create_pipeline("attention_paged_merge", 2, 40, [128])
        self._merge.bind_buffers([a, a])

    def _pages(self) -> list[int]:
        p = self.paged
        return [p.seq_pages, p.n_seq, p.n_pages, p.page_log2]

    def append(self, r: Recorder, layer: int, at: BatchRegions, q, k, v: int, out, q_norm: int, k_norm: int,
               rope: int, rows: int, mscale: float = 1.0) -> None:
        """Rows of raw q, k, v ((offset, stride); v has k's stride): q and k normed and rotated, q
        into out, k and v into layer's pool at each row's position."""
        c, kv = self.c, self.paged.layout
        push = [q[0], k[0], v, out[0], q_norm, k_norm, rope, E.f32_bits(c.eps), E.f32_bits(mscale), c.n_head,
                c.n_head_kv, q[1], k[1], out[1], kv.keys(0), kv.values(0), kv.key_scales(0), kv.value_scales(0),
                at.rows, at.table, *self._pages()]
        r.dispatch_set(self._append, layer, [1, rows, 1], push)

    def attend(self, r: Recorder, layer: int, at: BatchRegions, q, out, rows: int, parts: tuple[int, int]) -> None:
        """Attention of rows of rotated q ((offset, stride)) over layer's pool into out.  `parts`:
        how many pieces the shared positions (0: none are shared, whatever the rows say) and a
        row's own are cut into (splits); at.part holds part_size words."""
        c, kv = self.c, self.paged.layout
        scale = np.float32(1.0) / np.sqrt(np.float32(c.head_dim))
        push = [q[0], q[1], out[0], out[1], at.part, kv.keys(0), kv.values(0), kv.key_scales(0), kv.value_scales(0),
                c.n_head_kv, E.f32_bits(scale), *parts, at.rows, at.table, *self._pages()]
        r.dispatch_set(self._attend, layer, [1, rows, 1], push)
        r.barrier()
        push = [at.part, out[0], out[1], c.n_head, *parts, at.rows, self.paged.seq_pages, self.paged.n_seq,
                self.paged.page_log2]
        r.dispatch(self._merge, [1, rows, 1], push)

    def free(self) -> None:
        for p in (self._append, self._attend, self._merge):
            p.free()


class LogitsKernels:
    """logits_adjust over an arena's rows of logits."""

    def __init__(self, ctx: Context, a: Buffer):
        self._adjust = ctx.create_pipeline("logits_adjust", 2, 48, [])
        self._adjust.bind_buffers([a, a])

    def adjust(self, r: Recorder, at: LogitsRegions, x, y, n_vocab: int, rows: int) -> None:
        """Rows of logits x ((offset, stride)) into y, which may be x."""
        push = [x[0], y[0], x[1], y[1], n_vocab, at.controls, at.history, at.history_stride, at.bias, at.bias_stride,
                at.mask, at.mask_stride]
        r.dispatch(self._adjust, [1, rows, 1], push)

    def free(self) -> None:
        self._adjust.free()
