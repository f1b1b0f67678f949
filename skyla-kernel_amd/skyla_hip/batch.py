"""Decoding a batch of sequences: rows of many sequences over a paged KV cache.

The reference's engine serves one sequence over a contiguous cache (kv.rs); this module has
what a server of many needs beside it, over the same weights, arena rows and C-ABI:

  Paged           a pool of pages in the contiguous cache's row layout, and its page table
  BatchKernels    kv_append (QK-norm, rotation, keys and values into their pages), kv_append_axes
                  (the rotation by positions of several axes), attention_paged (attention of rows
                  over their pages, a leading run of positions that many rows share read once for
                  all of them) and attention_paged_shaped (scores capped by a tanh or biased by
                  distance, windows, rows that see from a document's start or to a prefix's end)
  LogitsKernels   logits_adjust (penalties for repeated tokens, biases, grammar masks) and
                  logits_sample (a token of each row by temperature, top-k, min-p and top-p)
  BatchEngine     sequences of one model: open, fork, prefill, step, close

The operators read the batch's rows from four words each, {sequence, length, share, 0}: the
row's token is at position length - 1, a row of length 0 has none.  Their push words are in
kernels/batch.hip.
"""
from __future__ import annotations

import dataclasses
from typing import NamedTuple, Sequence

import numpy as np

from . import engine as E
from .abi import Buffer, Context, Recorder

MAX_PARTS = 1024        # partials of a row and head (runtime/batch.h)
PAGE_SIZES = tuple(16 << i for i in range(9))  # 16 to 4096 positions
# control words: live rows, shared positions, their sequence, and for attention_paged_shaped the first of them and the
# longest row's length
CTL_ROWS, CTL_SHARED, CTL_LEADER, CTL_FIRST, CTL_LONGEST = 2, 3, 4, 5, 6
MIN_CAP, MAX_CAP = 2.0**-10, 2.0**14           # of scores (runtime/batch.h)


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
    """Arena offsets of a batch: the rows' words, the page table, the attention's partials; of
    kv_append_axes four positions a row, of attention_paged_shaped two words a row, the first position
    that it attends to and the end of a prefix that it sees past its own (0: none)."""
    rows: int
    table: int
    part: int = 0
    axes: int = 0
    spans: int = 0


@dataclasses.dataclass
class Shape:
    """What attention_paged_shaped does to scores: a cap (cap tanh(s / cap); 0: none), a window (a row
    attends to so many positions, its own the last; 0: all) and the arena offset of the heads' slopes (a
    score at a distance d loses slope d, slopes of 2^16 at most; None: none do)."""
    cap: float = 0.0
    window: int = 0
    slopes: int | None = None


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


@dataclasses.dataclass
class SampleRegions:
    """Arena offsets of what a row's token is drawn by (eight words a row: temperature, top_p, min_p,
    top_k, a random number of 32 bits), of what is drawn (four words a row: token, tokens kept, log
    probability) and of sample_size words between the two."""
    controls: int
    out: int
    part: int


class Parts(NamedTuple):
    """The pieces that a batch's attention cuts the shared run (0: none is shared, whatever the rows
    say) and each row's own run into, and whether the shared run takes 128 query rows a workgroup
    (else 16)."""
    shared: int
    own: int
    wide: bool = False


def splits(rows: int, n_kv: int, rep: int, shared: int, own: int) -> Parts:
    """Parts for `shared` shared positions and at most `own` of a row's own: enough workgroups to
    fill the GPU's 256 compute units, each with some tiles of 64 positions.

    128 query rows a workgroup stage keys and values once for all of them and pay for it at the
    start, so they are taken where a key head has 64 query rows or more, and query rows, key heads and
    positions make 1.5 Mi.  Attention and merge, us with 16 rows / 128 rows a workgroup, f16 and 8-bit
    caches (f16 keys with 8-bit values between them); of 600 cases over 2, 4 and 8 key heads the line
    is within 8% of the better form in 585:

      8 key heads, 64 query rows of each, 2000 positions (1.0 Mi)  17.6 / 20.0  20.2 / 25.3
      8, 64, 4000 (2.0 Mi)                                         24.8 / 23.0  28.3 / 28.0
      8, 128, 1000 (1.0 Mi)                                        18.7 / 19.8  22.2 / 25.0
      4, 256, 1000 (1.0 Mi)                                        17.4 / 19.7  20.1 / 24.8
      2, 512, 2000 (2.0 Mi)                                        24.4 / 22.9  27.8 / 27.7
      8, 32, 32768 (8.0 Mi, few rows)                              49.3 / 44.3  47.5 / 71.3
      8, 512, 256 (1.0 Mi, the furthest off)                       24.1 / 20.3  28.5 / 25.0"""
    q, tiles, own_tiles = rows * rep, -(-shared // 64), -(-own // 64)
    # (a workgroup without a run costs as much as a short one: 128 rows of 8 key heads in 1 / 2 / 4 parts
    # 27 / 31 / 47 us; one row of 16384 positions in 16 / 32 / 64 20.2 / 15.3 / 16.1)
    n_own = max(1, min(-(-512 // (n_kv * rows)), -(-own_tiles // 4), 128))
    if shared == 0:
        return Parts(0, n_own)
    if q >= 64 and q * n_kv * shared >= 3 << 19:
        # one workgroup a compute unit, two where a part stays long: 512 query rows of 8 key heads over
        # 32768 positions 157 / 144 us with the merge, of 4 over 8192 56 / 71, of 8 over 4000 51 / 58
        groups = n_kv * -(-q // 128)
        n = -(-(512 if shared * groups >= 1024 * 512 else 256) // groups)
        return Parts(min(n, -(-tiles // 2), 128), n_own, True)
    return Parts(min(-(-512 // (n_kv * -(-q // 16))), -(-tiles // 4), 128), n_own)


def part_size(rows: int, n_head: int, parts) -> int:
    """Words of the partials' region."""
    return rows * n_head * (parts[0] + parts[1]) * 130


class ShapedParts(NamedTuple):
    """Parts, and the pieces of a row's positions before the shared run (its lead; 0: none has any)."""
    shared: int
    own: int
    wide: bool = False
    lead: int = 0


def shaped_splits(rows: int, n_kv: int, rep: int, shared: int, own: int, lead: int = 0) -> ShapedParts:
    """Parts for a shared run of `shared` positions, at most `own` of a row's own and `lead` of those
    before the run.

    Where nothing is shared one part saves the merge.  It is taken from 256 rows x key heads on, and below for up
    to 8 positions for each of these.  A pass of 8 key heads, f16, us in one part / the best of two and more: 8
    rows of 512 / 1024 / 2048 positions 22.0 / 23.5, 27.7 / 25.8, 36.8 / 30.1; 16 rows 23.7 / 26.1, 28.0 / 31.3,
    39.3 / 39.0; 24 rows 24.1 / 31.4, 30.7 / 37.7, 51.2 / 52.7; 32 rows 25.9 / 32.1, 34.0 / 40.4, 60.6 / 67.3, of
    4096 99.9 / 113; 48 rows of 4096 168 / 157.  Rows are taken to be about as long: one of 16000 among 31 of 200 takes
    168 in its one part, 49 in 16, and 37 alone."""
    parts = splits(rows, n_kv, rep, shared, own)
    if shared == 0 and (n_kv * rows >= 256 or own <= 8 * n_kv * rows):
        parts = Parts(0, 1)
    n_lead = max(1, min(-(-512 // (n_kv * rows)), -(-lead // 256), 128)) if lead and shared else 0
    return ShapedParts(*parts, n_lead)


def shaped_part_size(rows: int, n_head: int, parts) -> int:
    """Words of attention_paged_shaped's partials."""
    return rows * n_head * (parts[0] + parts[1] + parts[3]) * 130


SAMPLE_CHUNK, SAMPLE_PART, SAMPLE_VOCAB = 8192, 5128, 1 << 20  # (runtime/batch.h)


def sample_size(rows: int, n_vocab: int) -> int:
    """Words of logits_sample's partials."""
    return rows * -(-n_vocab // SAMPLE_CHUNK) * SAMPLE_PART


class BatchKernels:
    """kv_append and attention_paged over one pool buffer for each layer."""

    def __init__(self, ctx: Context, tables: Buffer, a: Buffer, pools: Sequence[Buffer], c: E.Config, paged: Paged):
        self.check(c)
        if paged.layout.per_layer != paged.n_pages * paged.page * c.n_head_kv * c.head_dim:
            raise ValueError("the pool's rows are not the model's")
        if any(b.size < paged.bytes() for b in pools):
            raise ValueError(f"a pool of {paged.n_pages} pages takes {paged.bytes()} bytes")
        self.c, self.paged = c, paged
        k8, v8 = int(paged.precision.keys_q8), int(paged.precision.values_q8)

        def build(name, bufs, push, spec):
            p = ctx.create_pipeline_sets(name, 5, 4 * push, spec, len(pools))
            for i, kv in enumerate(pools):
                p.bind_set_buffers(i, (bufs + [kv, kv, kv])[:5])
            return p

        self._append = build("kv_append", [tables, a, a], 24, [k8, v8, 128])
        self._attend = build("attention_paged", [a, a], 20, [c.n_head // c.n_head_kv, k8, v8, 128])
        self._append_axes = build("kv_append_axes", [tables, a, a], 26, [k8, v8, 128])
        self._shaped = build("attention_paged_shaped", [a, a], 25, [c.n_head // c.n_head_kv, k8, v8, 128])
        self._merge = ctx.create_pipeline("attention_paged_merge", 2, 40, [128])
        self._merge.bind_buffers([a, a])
        self._shaped_merge = ctx.create_pipeline("attention_paged_shaped_merge", 2, 56, [128])
        self._shaped_merge.bind_buffers([a, a])

    @staticmethod
    def check(c: E.Config) -> None:
        if c.head_dim != 128 or c.n_head % c.n_head_kv or c.n_head // c.n_head_kv not in (1, 2, 4, 8):
            raise ValueError(f"no batch attention kernels for head_dim {c.head_dim}, {c.n_head}/{c.n_head_kv} heads")

    def _pages(self) -> list[int]:
        p = self.paged
        return [p.seq_pages, p.n_seq, p.n_pages, p.page_log2]

    def append(self, r: Recorder, layer: int, at: BatchRegions, q, k, v: int, out, q_norm: int, k_norm: int,
               rope: int, rows: int, mscale: float = 1.0) -> None:
        """Rows of raw q, k, v ((offset, stride); v has k's stride): q and k normed and rotated, q
        into out, k and v into layer's pool at each row's position."""
        r.dispatch_set(self._append, layer, [1, rows, 1], self._append_push(at, q, k, v, out, q_norm, k_norm, rope, mscale))

    def append_axes(self, r: Recorder, layer: int, at: BatchRegions, q, k, v: int, out, q_norm: int, k_norm: int,
                    rope: int, n_axes: int, rows: int, mscale: float = 1.0) -> None:
        """append, with each row turned by its `n_axes` (1 to 4) positions at at.axes: rope holds 64
        frequencies for each axis (those of a pair's other axes 0)."""
        push = self._append_push(at, q, k, v, out, q_norm, k_norm, rope, mscale)
        r.dispatch_set(self._append_axes, layer, [1, rows, 1], push + [at.axes, n_axes])

    def _append_push(self, at, q, k, v, out, q_norm, k_norm, rope, mscale) -> list[int]:
        c, kv = self.c, self.paged.layout
        return [q[0], k[0], v, out[0], q_norm, k_norm, rope, E.f32_bits(c.eps), E.f32_bits(mscale), c.n_head,
                c.n_head_kv, q[1], k[1], out[1], kv.keys(0), kv.values(0), kv.key_scales(0), kv.value_scales(0),
                at.rows, at.table, *self._pages()]

    def attend(self, r: Recorder, layer: int, at: BatchRegions, q, out, rows: int, parts) -> None:
        """Attention of rows of rotated q ((offset, stride)) over layer's pool into out, in `parts`
        (splits); at.part holds part_size words."""
        parts = Parts(*parts)
        r.dispatch_set(self._attend, layer, [1, rows, 1], self._attend_push(at, q, out, parts))
        if parts.shared + parts.own == 1:  # nothing to merge: the rows are the result
            return
        r.barrier()
        r.dispatch(self._merge, [1, rows, 1], self._merge_push(at, out, parts))

    def attend_shaped(self, r: Recorder, layer: int, at: BatchRegions, q, out, rows: int, parts, shape: Shape) -> None:
        """attend, each row over the positions that at.spans and the window leave it, with scores as
        `shape` has them, in `parts` (shaped_splits); at.part holds shaped_part_size words."""
        parts = ShapedParts(*parts)
        push = self._attend_push(at, q, out, parts)
        push += [at.spans, 0xFFFFFFFF if shape.slopes is None else shape.slopes, shape.window, parts.lead, E.f32_bits(shape.cap)]
        r.dispatch_set(self._shaped, layer, [1, rows, 1], push)
        if parts.shared + parts.own + parts.lead == 1:
            return
        r.barrier()
        push = self._merge_push(at, out, parts) + [at.spans, shape.window, parts.lead, self.c.n_head // self.c.n_head_kv]
        r.dispatch(self._shaped_merge, [1, rows, 1], push)

    def _attend_push(self, at, q, out, parts) -> list[int]:
        c, kv = self.c, self.paged.layout
        scale = np.float32(1.0) / np.sqrt(np.float32(c.head_dim))
        return [q[0], q[1], out[0], out[1], at.part, kv.keys(0), kv.values(0), kv.key_scales(0), kv.value_scales(0),
                c.n_head_kv, E.f32_bits(scale), parts.shared, parts.own, at.rows, at.table, *self._pages(), parts.wide]

    def _merge_push(self, at, out, parts) -> list[int]:
        return [at.part, out[0], out[1], self.c.n_head, parts.shared, parts.own, at.rows, self.paged.seq_pages,
                self.paged.n_seq, self.paged.page_log2]

    def free(self) -> None:
        for p in (self._append, self._append_axes, self._attend, self._shaped, self._merge, self._shaped_merge):
            p.free()


class LogitsKernels:
    """logits_adjust and logits_sample over an arena's rows of logits."""

    def __init__(self, ctx: Context, a: Buffer):
        build = lambda name, words: ctx.create_pipeline(name, 2, 4 * words, [])  # noqa: E731
        self._adjust, self._sample, self._draw = (build("logits_adjust", 12), build("logits_sample", 5),
                                                  build("logits_sample_draw", 6))
        for p in (self._adjust, self._sample, self._draw):
            p.bind_buffers([a, a])

    def adjust(self, r: Recorder, at: LogitsRegions, x, y, n_vocab: int, rows: int) -> None:
        """Rows of logits x ((offset, stride)) into y, which may be x."""
        push = [x[0], y[0], x[1], y[1], n_vocab, at.controls, at.history, at.history_stride, at.bias, at.bias_stride,
                at.mask, at.mask_stride]
        r.dispatch(self._adjust, [1, rows, 1], push)

    def sample(self, r: Recorder, at: SampleRegions, x, n_vocab: int, rows: int) -> None:
        """A token of each row of logits x ((offset, stride)) into at.out; at.part holds sample_size words."""
        push = [x[0], x[1], n_vocab, at.controls, at.part]
        r.dispatch(self._sample, [1, rows, 1], push)
        r.barrier()
        r.dispatch(self._draw, [1, rows, 1], push + [at.out])

    def free(self) -> None:
        for p in (self._adjust, self._sample, self._draw):
            p.free()


# ---- sequences of one model ----------------------------------------------------------------
@dataclasses.dataclass
class Controls:
    """What acts on a sequence's logits (logits_adjust): a repetition penalty over all its tokens
    (1: none), frequency and presence penalties over its generated ones, biases by token id, and
    the tokens allowed (a truth value each; None: all)."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict = dataclasses.field(default_factory=dict)
    allowed: np.ndarray | None = None

    @property
    def counts(self) -> bool:
        return self.repetition != 1.0 or self.frequency != 0.0 or self.presence != 0.0


@dataclasses.dataclass
class Sampling:
    """How a sequence's tokens are drawn (logits_sample): at a temperature (0: the likeliest token), among the
    top_k likeliest (0: any number of them), those at least min_p as likely as the likeliest, and the likeliest
    that make up top_p of these."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


class Drawn(NamedTuple):
    """A step's tokens, a row each (-1: its controls leave none), the log probabilities that they were drawn
    with, and among how many tokens."""
    token: np.ndarray
    logprob: np.ndarray
    kept: np.ndarray


class _Sequence:
    """A sequence's pages, the tokens of its prompts and those that it generated (a conversation's
    follow in turns; what acts on the logits asks only which), its controls, the row of the batch
    that these lie in (None: they do not), how many words of its history, the prompts' tokens before
    the others, lie there, whether its controls do not yet, how its tokens are drawn, and how far the
    rotation's positions of further text are past the cache's (behind images, mostly below 0)."""

    def __init__(self, pages=(), prompt=(), made=(), controls=None, sampling=None, shift=0):
        self.pages, self.prompt, self.made = list(pages), list(prompt), list(made)
        self.controls, self.row, self.placed, self.stale = controls or Controls(), None, 0, True
        self.sampling, self.shift = sampling or Sampling(), shift

    def __len__(self):
        return len(self.prompt) + len(self.made)

    def add(self, tokens, prompt):
        if prompt:
            self.placed = min(self.placed, len(self.prompt))
            self.prompt += tokens
        else:
            self.made += tokens

    def drop(self, n, prompt):
        """Takes the last n tokens of add back."""
        keep = self.prompt if prompt else self.made
        del keep[len(keep) - n:]
        self.placed = min(self.placed, len(self.prompt) if prompt else len(self))


class _BatchGraph(E.Graph):
    """A layer's dispatches with the batch's cache in place of the contiguous one; `parts` by the layers'
    windows where scores are shaped."""

    def __init__(self, r: Recorder, eng: "BatchEngine", batched: bool, rows: int, parts):
        super().__init__(r, eng.kernels, eng.arena, eng.c, batched)
        self.eng, self.rows, self.parts = eng, rows, parts

    def qk_rope(self, l: int, q_norm: int, k_norm: int, rope: int) -> None:
        a, e = self.a, self.eng
        q = (a.q, a.s_q)
        if e.n_axes:
            e.batch.append_axes(self.r, l, e.at, q, (a.k, a.s_kv), a.v, q, q_norm, k_norm, e.weights.rope_axes, e.n_axes,
                                self.rows, self.c.rope_mscale)
        else:
            e.batch.append(self.r, l, e.at, q, (a.k, a.s_kv), a.v, q, q_norm, k_norm, rope, self.rows, self.c.rope_mscale)
        self.stage("kv append")

    def attend(self, l: int) -> None:
        a, e = self.a, self.eng
        q, out = (a.q, a.s_q), (a.attn, a.s_attn)
        if isinstance(self.parts, Parts):
            e.batch.attend(self.r, l, e.at, q, out, self.rows, self.parts)
        else:
            window = e.window(l)
            shape = Shape(self.c.score_cap, window, e.slopes)
            e.batch.attend_shaped(self.r, l, e.at, q, out, self.rows, dict(self.parts)[window], shape)
        self.stage("attention")


class BatchEngine:
    """Up to BATCH sequences of one model, decoded together.  A sequence is a number from open() or
    fork(); extend() puts tokens into its cache, step() takes a token of each of several sequences
    and returns the logits after them, with their controls applied, sample() the tokens drawn from
    these; close() gives its pages back.

    A forked sequence shares the whole pages of the one it came from (the rest of the last page is
    copied), and a step reads the pages that its sequences share once for all of them.  A step has a
    row for each of its sequences and no others, so that it takes what it would if they were the only
    ones open; a sequence keeps its row from step to step while it can, since what acts on logits
    lies by rows."""

    MAX_BIASES = 512

    def __init__(self, ctx: Context, model: dict, c: E.Config, max_ctx: int, n_pages: int, page: int = 64,
                 precision: E.KvPrecision = E.KvPrecision.F16_KEYS_Q8_VALUES, max_seq: int = E.BATCH):
        if not 1 <= max_seq <= E.BATCH:
            raise ValueError(f"{max_seq} sequences: a batch holds 1 to {E.BATCH}")
        if max_ctx < 1:
            raise ValueError(f"max_ctx {max_ctx}")
        BatchKernels.check(c)
        self._check_shape(c)
        self.ctx, self.c, self.max_ctx, self.max_seq = ctx, c, max_ctx, max_seq
        self.paged = Paged(precision, page, n_pages, max_seq, min(-(-max_ctx // page), n_pages),
                           c.n_head_kv * c.head_dim)
        if self.paged.bytes() > ctx.max_buffer():
            raise ValueError(f"a layer's pool of {n_pages} pages needs {self.paged.bytes() >> 20} MiB, above the "
                             "allocation cap")
        self.rep = c.n_head // c.n_head_kv
        self.s_vocab, self.s_mask = E._next64(c.n_vocab), -(-c.n_vocab // 32)
        self.s_hist = -(-max_ctx // 4) * 4
        self.n_axes = max(c.axes) + 1 if c.axes is not None else 0
        self.windows = sorted(set(c.windows or [0]))
        part = max(max(part_size(r, c.n_head, self._parts(r, shared, own)),
                       *(shaped_part_size(r, c.n_head, p) for lead in (False, True)
                         for _, p in self._shaped_parts(r, shared, own, lead)))
                   for r in self._buckets(E.BATCH) for shared in [0, *self._buckets(max_ctx)]
                   for own in self._buckets(max_ctx))
        part = max(part, sample_size(max_seq, c.n_vocab) if self._draws() else 0)
        self.weights = self.arena = self.batch = self.logits = None
        self.pools, self.recordings = [], {}
        try:
            self._allocate(model, precision, part)
        except BaseException:  # as where the card has no room for so many pages
            self.free()
            raise
        self.free_pages = list(range(n_pages - 1, -1, -1))
        self.uses = np.zeros(n_pages, np.int64)  # sequences that hold a page
        self.sequences: dict[int, _Sequence] = {}
        self.rows: list[int | None] = [None] * max_seq  # the sequence whose controls lie in a row

    def _allocate(self, model: dict, precision: E.KvPrecision, part: int) -> None:
        ctx, c, max_seq = self.ctx, self.c, self.max_seq
        self.weights = E.load_weights(ctx, model, c)
        a = self.arena = E.Arena(ctx, c, extra={
            "rows": 4 * E.BATCH, "table": max_seq * self.paged.seq_pages, "part": part,
            "logits": self.s_vocab * max_seq, "controls": 8 * max_seq, "history": self.s_hist * max_seq,
            "bias": 2 * self.MAX_BIASES * max_seq, "mask": self.s_mask * max_seq,
            "axes": 4 * E.BATCH, "spans": 2 * E.BATCH, "slopes": c.n_head, "sampling": 8 * max_seq,
            "drawn": 4 * max_seq})
        x = a.extra
        for _ in range(c.n_layer):
            self.pools.append(ctx.alloc_host(self.paged.bytes()))
        self.at = BatchRegions(rows=x["rows"], table=x["table"], part=x["part"], axes=x["axes"], spans=x["spans"])
        # (a step's draws come when its attention's partials have been merged, and lie in their place)
        self.sample_at = SampleRegions(controls=x["sampling"], out=x["drawn"], part=x["part"])
        self.slopes = None
        if c.slopes is not None:
            self.slopes = x["slopes"]
            a.f32()[self.slopes: self.slopes + c.n_head] = c.slopes
            a.buffer.upload(self.slopes * 4, c.n_head * 4)
        self.logits_at = LogitsRegions(x["controls"], x["history"], self.s_hist, x["bias"], 2 * self.MAX_BIASES,
                                       x["mask"], self.s_mask)
        self.kernels = E.Kernels(ctx, self.weights.buffers, a.buffer, kv=self.pools[0], c=c, precision=precision,
                                 embd_dtype=self.weights.embd.dtype)
        self.batch = BatchKernels(ctx, self.weights.buffers[0], a.buffer, self.pools, c, self.paged)
        self.logits = LogitsKernels(ctx, a.buffer)

    @staticmethod
    def _check_shape(c: E.Config) -> None:
        if c.axes is not None and (len(c.axes) != c.head_dim // 2 or any(a not in (0, 1, 2, 3) for a in c.axes)):
            raise ValueError(f"axes: one of 0 to 3 for each of {c.head_dim // 2} pairs")
        if c.score_cap != 0 and not MIN_CAP <= c.score_cap <= MAX_CAP:
            raise ValueError(f"scores capped at {c.score_cap}: {MIN_CAP} to {MAX_CAP}, or 0")
        if c.windows is not None and (len(c.windows) != c.n_layer or any(not 0 <= w < 2**32 for w in c.windows)):
            raise ValueError(f"windows: a number of positions for each of {c.n_layer} layers (0: all)")
        if c.slopes is not None and (len(c.slopes) != c.n_head or not (np.abs(c.slopes) <= 2**16).all()):
            raise ValueError(f"slopes: a number of 2^16 at most for each of {c.n_head} heads")

    def _draws(self) -> bool:
        return self.c.n_vocab <= SAMPLE_VOCAB

    def window(self, layer: int) -> int:
        return self.c.windows[layer] if self.c.windows is not None else 0

    # ---- sequences ----
    def open(self) -> int:
        return self._add(_Sequence())

    def _add(self, s: _Sequence) -> int:
        n = next((i for i in range(self.max_seq) if i not in self.sequences), None)
        if n is None:
            raise ValueError(f"all {self.max_seq} sequences are open")
        self.sequences[n] = s
        return n

    def _get(self, seq: int) -> _Sequence:
        if seq not in self.sequences:
            raise ValueError(f"no open sequence {seq}")
        return self.sequences[seq]

    def length(self, seq: int) -> int:
        """Positions in a sequence's cache."""
        return len(self._get(seq))

    def fork(self, seq: int) -> int:
        """A new sequence that goes on from where `seq` is, with its controls."""
        s, page = self._get(seq), self.paged.page
        whole, rest = divmod(len(s), page)
        if len(self.sequences) == self.max_seq:
            raise ValueError(f"all {self.max_seq} sequences are open")
        own = self._take(1 if rest else 0)
        try:
            if rest:
                self._copy_page(s.pages[whole], own[0], rest)
        except BaseException:
            self._give(own)
            raise
        self.uses[s.pages[:whole]] += 1
        n = self._add(_Sequence(s.pages[:whole] + own, s.prompt, s.made, s.controls, s.sampling, s.shift))
        self._upload_table(n)
        return n

    def close(self, seq: int) -> None:
        s = self._get(seq)
        self._give(s.pages)
        if s.row is not None:
            self.rows[s.row] = None
        del self.sequences[seq]

    def control(self, seq: int, controls: Controls) -> None:
        """Sets what acts on a sequence's logits from its next step on: `controls` as they are now (what
        the caller changes in them later acts on nothing)."""
        s = self._get(seq)
        with np.errstate(over="ignore", under="ignore"):  # as the kernel has them
            penalties = np.float32([controls.repetition, controls.frequency, controls.presence])
        if not penalties[0] > 0 or not np.isfinite(penalties).all():
            raise ValueError("a repetition penalty above 0 and finite penalties, in 32 bits")
        bias = {int(t): float(v) for t, v in controls.bias.items()}
        if any(np.isnan(v) for v in bias.values()):
            raise ValueError("biases that are numbers")
        if len(bias) > self.MAX_BIASES or any(not 0 <= t < self.c.n_vocab for t in bias):
            raise ValueError(f"at most {self.MAX_BIASES} biases, of tokens of the vocabulary")
        allowed = controls.allowed
        if allowed is not None:
            if np.shape(allowed) != (self.c.n_vocab,):
                raise ValueError(f"allowed: a truth value for each of {self.c.n_vocab} tokens")
            allowed = np.array(allowed, bool)
        s.controls = Controls(*(float(v) for v in penalties), bias, allowed)
        s.stale = True

    def sampling(self, seq: int, sampling: Sampling) -> None:
        """Sets how a sequence's tokens are drawn from its next sample() on: `sampling` as it is now."""
        s = self._get(seq)
        with np.errstate(over="ignore", under="ignore"):
            t, p, m = (float(np.float32(v)) for v in (sampling.temperature, sampling.top_p, sampling.min_p))
        if not 0 <= t < np.inf or not 0 < p <= 1 or not 0 <= m <= 1:
            raise ValueError("a temperature of 0 or more, top_p in (0, 1] and min_p in [0, 1], in 32 bits")
        if not 0 <= sampling.top_k < 2**32:
            raise ValueError("top_k: a number of tokens (0: any)")
        s.sampling = Sampling(t, int(sampling.top_k), p, m)

    # ---- pages ----
    def _take(self, n: int) -> list[int]:
        if n > len(self.free_pages):
            raise ValueError(f"{n} pages needed, {len(self.free_pages)} free")
        got = [self.free_pages.pop() for _ in range(n)]
        self.uses[got] += 1
        return got

    def _give(self, pages: Sequence[int]) -> None:
        for p in pages:
            self.uses[p] -= 1
            if self.uses[p] == 0:
                self.free_pages.append(p)

    def _trim(self, seq: int) -> None:
        """Gives back the pages past a sequence's last."""
        s = self._get(seq)
        keep = -(-len(s) // self.paged.page)
        self._give(s.pages[keep:])
        del s.pages[keep:]

    def _copy_page(self, src: int, dst: int, n: int) -> None:
        lay, page, dim = self.paged.layout, self.paged.page, self.c.n_head_kv * self.c.head_dim
        pr = lay.precision
        for kv in self.pools:
            for off, scales, q8 in ((lay.keys(0), lay.key_scales(0), pr.keys_q8),
                                    (lay.values(0), lay.value_scales(0), pr.values_q8)):
                size = 1 if q8 else 2
                at = lambda p: (off + p * page * dim) * size  # noqa: E731
                kv.copy_from(at(dst), kv, at(src), n * dim * size)
                if q8:
                    at = lambda p: (scales + p * page * (dim // 32)) * 2  # noqa: E731
                    kv.copy_from(at(dst), kv, at(src), n * (dim // 32) * 2)

    def _room(self, need: dict[int, int]) -> None:
        """Pages for sequences to grow by need[seq] positions: all of them or none."""
        page, new = self.paged.page, {}
        for seq, n in need.items():
            s = self._get(seq)
            if len(s) + n > self.max_ctx:
                raise ValueError(f"sequence {seq}: context full ({self.max_ctx} tokens)")
            new[seq] = -(-(len(s) + n) // page) - len(s.pages)
        if sum(new.values()) > len(self.free_pages):
            raise ValueError(f"{sum(new.values())} pages needed, {len(self.free_pages)} free")
        for seq, n in new.items():
            if n > 0:
                self._get(seq).pages += self._take(n)
                try:
                    self._upload_table(seq)
                except BaseException:
                    self._trim(seq)
                    raise

    # ---- words ----
    def _place(self, seqs: list[int]) -> None:
        """Gives the sequences rows 0 to len(seqs) - 1, each the one it has where that is among them."""
        free = [r for r in range(len(seqs)) if self.rows[r] not in seqs]
        for q in seqs:
            s = self._get(q)
            if s.row is None or s.row >= len(seqs):
                if s.row is not None:
                    self.rows[s.row] = None
                s.row, s.placed, s.stale = free.pop(0), 0, True
                if self.rows[s.row] is not None:
                    self._get(self.rows[s.row]).row = None
                self.rows[s.row] = q
            if s.stale:
                self._upload_controls(q)
                s.stale = False

    def _upload_table(self, seq: int) -> None:
        a, pages = self.arena, self._get(seq).pages
        off = self.at.table + seq * self.paged.seq_pages
        a.u32()[off: off + len(pages)] = pages
        if pages:
            a.buffer.upload(off * 4, len(pages) * 4)

    def _upload_history(self, seq: int) -> None:
        a, s = self.arena, self._get(seq)
        n = s.placed - len(s.prompt)
        new = s.made[n:] if n >= 0 else s.prompt[n:] + s.made
        off = self.logits_at.history + s.row * self.s_hist + s.placed
        if new:
            a.u32()[off: off + len(new)] = new
            a.buffer.upload(off * 4, len(new) * 4)
        s.placed = len(s)

    def _upload_controls(self, seq: int) -> None:
        a, s = self.arena, self._get(seq)
        k, u, f = s.controls, a.u32(), a.f32()
        bias = self.logits_at.bias + 2 * self.MAX_BIASES * s.row
        n = len(k.bias)
        if n:
            u[bias: bias + 2 * n: 2] = list(k.bias)
            with np.errstate(over="ignore", under="ignore"):
                f[bias + 1: bias + 2 * n: 2] = list(k.bias.values())
            a.buffer.upload(bias * 4, n * 8)
        if k.allowed is not None:
            mask = self.logits_at.mask + self.s_mask * s.row
            bits = np.zeros(32 * self.s_mask, bool)
            bits[: self.c.n_vocab] = k.allowed
            u[mask: mask + self.s_mask] = np.packbits(bits, bitorder="little").view("<u4")
            a.buffer.upload(mask * 4, self.s_mask * 4)

    def _words(self, live: int, rows: np.ndarray, tokens: Sequence[int], shared: int, leader: int, axes=None,
               spans=None, first: int = 0) -> None:
        a = self.arena
        u, n = a.u32(), len(rows)
        u[a.tokens: a.tokens + n] = tokens
        u[self.at.rows: self.at.rows + 4 * n] = rows.ravel()
        u[0], u[1], u[2], u[3], u[4], u[5], u[6] = int(tokens[0]), 0, live, shared, leader, first, rows[:, 1].max()
        a.buffer.upload(0, 64 * 4)
        a.buffer.upload(a.tokens * 4, n * 4)
        a.buffer.upload(self.at.rows * 4, n * 16)
        if spans is not None or self.c.shapes_scores:
            u[self.at.spans: self.at.spans + 2 * n] = np.broadcast_to(spans or (0, 0), (n, 2)).ravel()
            a.buffer.upload(self.at.spans * 4, n * 8)
        if self.n_axes:
            u[self.at.axes: self.at.axes + 4 * n] = np.broadcast_to(axes, (n, 4)).ravel()
            a.buffer.upload(self.at.axes * 4, n * 16)

    def _check(self, tokens) -> list[int]:
        tokens = [int(t) for t in tokens]
        if any(not 0 <= t < self.c.n_vocab for t in tokens):
            raise ValueError("token outside the vocabulary")
        return tokens

    # ---- recordings ----
    @staticmethod
    def _buckets(most: int) -> list[int]:
        out = [1]
        while out[-1] < most:
            out.append(min(2 * out[-1], most))
        return out

    def _parts(self, rows: int, shared: int, own: int) -> Parts:
        return splits(rows, self.c.n_head_kv, self.rep, shared, own)

    def _shaped_parts(self, rows: int, shared: int, own: int, lead: bool) -> tuple:
        """((window, its layers' parts), ...): a window leaves that much of the shared run at most, and of a row that
        does not take the run; rows' leads are as long as the rows' lengths differ, or end a tile."""
        def parts(w):
            run, alone = (min(shared, w), min(shared + own, w)) if w else (shared, own)
            return shaped_splits(rows, self.c.n_head_kv, self.rep, run, max(alone, 1), max(own, 64) if w or lead else 0)
        return tuple((w, parts(w)) for w in self.windows)

    def _recording(self, rows: int, shared: int, own: int, head: bool, shaped: bool = False, lead: bool = False,
                   sample: bool = False, vectors: bool = False):
        """The recording for up to `rows` rows over `shared` shared and `own` positions of their own,
        with the output head and the logits' controls or without (extend); with shaped scores or spans, some of
        which start inside a tile (lead); with tokens drawn; of rows given as vectors."""
        up = lambda n, most: next(b for b in self._buckets(most) if b >= n)  # noqa: E731
        rows = up(rows, E.BATCH)
        shared, own = up(shared, self.max_ctx) if shared else 0, up(own, self.max_ctx)
        if shaped or self.c.shapes_scores:
            parts = self._shaped_parts(rows, shared, own, lead)
        else:
            parts = self._parts(rows, shared, own)
        key = rows, parts, head, sample, vectors
        if key not in self.recordings:
            self.recordings[key] = self.ctx.record(False, lambda r: self._record(r, rows, parts, head, sample, vectors))
        return self.recordings[key]

    def _record(self, r: Recorder, rows: int, parts, head: bool, sample: bool = False, vectors: bool = False) -> None:
        a, w, c, batched = self.arena, self.weights, self.c, rows > 1
        g = _BatchGraph(r, self, batched, rows, parts)
        if not vectors:
            g.embed(w.embd)
        for l, lw in enumerate(w.layers):
            g.layer(l, lw, w.rope)
        if head:
            g.rmsnorm(a.x, w.out_norm, a.n, rows)
            g.stage("rmsnorm")
            y = (a.extra["logits"], self.s_vocab)
            g.matvec(w.output, (a.n, a.s_embd), y, False, batched)
            g.stage("matvec output")
            self.logits.adjust(r, self.logits_at, y, y, c.n_vocab, min(rows, self.max_seq))
            if sample:
                r.barrier()
                self.logits.sample(r, self.sample_at, y, c.n_vocab, min(rows, self.max_seq))
        r.host_barrier()

    # ---- decoding ----
    def extend(self, seq: int, tokens, axes=None, vectors=None, since: int = 0, together: bool = False) -> None:
        """Puts tokens into a sequence's cache, as its prompt or a further turn's, BATCH of them at a
        time.  What it generated before counts as generated still.

        axes: the tokens' positions for the rotation, a row each and a column for each of the model's axes, as an
        image's patches or a video's have them; without, they follow one another as text, which goes on behind the
        largest so far.  vectors: rows of n_embd numbers in place of the tokens' own (an image's; the tokens then
        are what the history says of them).  since: the first position that the tokens attend to, as where a document
        of its own begins (these tokens alone: what is generated behind them attends to all).  together: the tokens, BATCH at most, attend to one another, later ones too."""
        s, tokens = self._get(seq), self._check(tokens)
        n_all = len(tokens)
        if axes is not None:
            axes = np.asarray(axes)
            if not self.n_axes:
                raise ValueError("axes: the model's rotation has one position")
            if axes.shape != (n_all, self.n_axes) or (n_all and (axes.dtype.kind not in "iu" or axes.min() < 0 or
                                                                 axes.max() >= 2**31)):
                raise ValueError(f"axes: {n_all} rows of {self.n_axes} positions")
            axes = np.concatenate([axes.astype(np.int64), np.zeros((n_all, 4 - self.n_axes), np.int64)], 1)
        if vectors is not None:
            vectors = np.asarray(vectors, np.float32)
            if vectors.shape != (n_all, self.c.n_embd):
                raise ValueError(f"vectors: {n_all} rows of {self.c.n_embd} numbers")
        if not 0 <= since <= len(s):
            raise ValueError(f"since: a position of the sequence or its end (0 to {len(s)})")
        if together and n_all > E.BATCH:
            raise ValueError(f"together: at most {E.BATCH} tokens see one another")
        self._room({seq: n_all})
        shaped = since > 0 or together
        try:
            for i in range(0, n_all, E.BATCH):
                chunk, pos = tokens[i: i + E.BATCH], len(s)
                n = len(chunk)
                rows = np.zeros((n, 4), np.uint32)
                rows[:, 0], rows[:, 1], rows[:, 2] = seq, pos + 1 + np.arange(n), pos
                turn = axes[i: i + n] if axes is not None else (pos + s.shift + np.arange(n))[:, None]
                if vectors is not None:
                    self._upload_vectors(vectors[i: i + n])
                spans = (since, pos + n if together else 0) if shaped else None
                self._words(n, rows, chunk, pos, seq, turn, spans, since)
                self.ctx.replay(self._recording(n, pos, n, False, shaped, since > 0, vectors=vectors is not None))
                s.add(chunk, True)
                if axes is not None:
                    s.shift = max(int(turn.max()) + 1, pos + s.shift) - len(s)
        except BaseException:  # what was decoded stays
            self._trim(seq)
            raise

    def _upload_vectors(self, vectors: np.ndarray) -> None:
        a, (n, width) = self.arena, vectors.shape
        a.f32()[a.x: a.x + n * a.s_embd].reshape(n, a.s_embd)[:, :width] = vectors
        a.buffer.upload(a.x * 4, n * a.s_embd * 4)

    def shared_run(self, seqs) -> tuple[int, list[int]]:
        """The positions that sequences of a step read once for all: (how many, whose).  Of the
        sequences that begin with the same page the largest group's common whole pages."""
        groups = {}
        for q in seqs:
            pages = self._get(q).pages
            if pages:
                groups.setdefault(pages[0], []).append(q)
        members = max(groups.values(), key=len, default=[])
        if len(members) < 2:
            return 0, []
        lists = [self._get(q).pages for q in members]
        n = 0
        while all(len(p) > n and p[n] == lists[0][n] for p in lists):
            n += 1
        return n * self.paged.page, members

    def step(self, tokens: dict, prompt=()) -> np.ndarray:
        """One token of each of several sequences ({sequence: token}): the logits after them, a row
        each in the order given.  `prompt`: sequences whose token is a prompt's (the others' count as
        generated)."""
        seqs = self._step(tokens, prompt)
        a, v = self.arena, self.c.n_vocab
        out = np.empty((len(seqs), v), np.float32)
        for i, q in enumerate(seqs):
            off = a.extra["logits"] + self._get(q).row * self.s_vocab
            a.buffer.download(off * 4, v * 4)
            out[i] = a.f32()[off: off + v]
        return out

    def sample(self, tokens: dict, draws: dict, prompt=()) -> Drawn:
        """step(), but the tokens that come next, each drawn as its sequence's sampling has it from the logits after
        its controls, by its random number draws[sequence], an integer of 32 bits: from the same logits the same
        number draws the same token, whatever else is in the batch."""
        if not self._draws():
            raise ValueError(f"tokens are drawn from a vocabulary of {SAMPLE_VOCAB} at most, not of {self.c.n_vocab}")
        if set(draws) != set(tokens):
            raise ValueError("draws: a random number for each sequence of this step")
        draws = {q: int(d) for q, d in draws.items()}
        if any(not 0 <= d < 2**32 for d in draws.values()):
            raise ValueError("draws: integers of 32 bits")
        seqs = self._step(tokens, prompt, draws)
        a, off, live = self.arena, self.sample_at.out, len(seqs)
        a.buffer.download(off * 4, live * 16)
        order = [self._get(q).row for q in seqs]
        out = a.u32()[off: off + 4 * live].reshape(live, 4)[order].copy()
        return Drawn(out[:, 0].astype(np.int32).astype(np.int64), out[:, 2].copy().view(np.float32), out[:, 1].astype(np.int64))

    def _step(self, tokens: dict, prompt, draws: dict | None = None) -> list[int]:
        """Decodes one token of each sequence; the sequences."""
        if not tokens:
            raise ValueError("step needs a token of at least one sequence")
        values, seqs, prompt = self._check(tokens.values()), list(tokens), set(prompt)
        if any(q not in tokens for q in prompt):
            raise ValueError("prompt: sequences of this step")
        self._room({q: 1 for q in seqs})
        for q, t in zip(seqs, values):
            self._get(q).add([t], q in prompt)
        try:
            self._replay_step(seqs, values, draws)
        except BaseException:  # nothing was decoded: the sequences are as they were
            for q in seqs:
                self._get(q).drop(1, q in prompt)
                self._trim(q)
            raise
        return seqs

    def _replay_step(self, seqs: list[int], values: list[int], draws: dict | None) -> None:
        """One row for each of the sequences' last tokens, through the model and its head."""
        self._place(seqs)
        live = len(seqs)
        shared, members = self.shared_run(seqs)
        rows, ids, own = np.zeros((live, 4), np.uint32), np.zeros(live, np.uint32), 1
        turn = np.zeros((live, 1), np.int64)
        for q, t in zip(seqs, values):
            s = self._get(q)
            n, take = len(s), shared if q in members and len(s) >= shared else 0
            rows[s.row], ids[s.row], own = (q, n, take, 0), t, max(own, n - take)
            turn[s.row] = n - 1 + s.shift
            if s.controls.counts:
                self._upload_history(q)
        self._words(live, rows, ids, shared, members[0] if members else 0, turn)
        self._control_words(live)
        if draws is not None:
            self._sampling_words(live, draws)
        self.ctx.replay(self._recording(live, shared, own, True, sample=draws is not None))

    def _control_words(self, live: int) -> None:
        a, off = self.arena, self.logits_at.controls
        u, f = a.u32(), a.f32()
        for r in range(live):
            s, o = self._get(self.rows[r]), off + 8 * r
            k = s.controls
            u[o: o + 4] = len(s), len(s.prompt), len(k.bias), k.allowed is not None
            f[o + 4: o + 7] = k.repetition, k.frequency, k.presence
        a.buffer.upload(off * 4, live * 32)

    def _sampling_words(self, live: int, draws: dict) -> None:
        a, off = self.arena, self.sample_at.controls
        u, f = a.u32(), a.f32()
        for r in range(live):
            k, o = self._get(self.rows[r]).sampling, off + 8 * r
            f[o: o + 3] = k.temperature, k.top_p, k.min_p
            u[o + 3: o + 8] = k.top_k, draws[self.rows[r]], 0, 0, 0
        a.buffer.upload(off * 4, live * 32)

    def free(self) -> None:
        for rec in self.recordings.values():
            rec.free()
        self.recordings = {}
        for k in (self.batch, self.logits):
            if k:
                k.free()
        for b in [*(self.weights.buffers if self.weights else ()), *self.pools, *([self.arena.buffer] if self.arena else ())]:
            b.free()
