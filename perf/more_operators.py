"""What three more operators of a served batch are measured on: those that a step needs for prompts
with images, for models that shape their scores, and for the token itself.

  axes    rows of q, k, v into the cache's pages, the rotation by positions of several axes
  shaped  attention over pages with scores capped by a tanh or biased by distance, a window, rows that
          see from a document's start on, or to a prefix's end
  sample  a token of each row of logits by temperature, top-k, min-p and top-p, from given numbers

Sizes are those of the benchmark's and tests' models (Qwen3-0.6B: 16 heads over 8, Qwen3-8B: 32
over 8, Qwen3-30B-A3B: 32 over 4, a vocabulary of 151936), and batches up to the engine's 128 rows.

In the framework the operands live in its own buffers (an arena of rows, a pool of pages), so
where its calls are made the same inputs are written into such buffers and the call is recorded,
as its engine does once at load.
"""
import hashlib
import math
import os
import sys

import numpy as np
import torch

own = False

HEAD = 128
EPS = 1e-6
THETA = 1e6
PAGES = (16, 32, 64, 128, 256)
STORES = ("f16", "q8", "f16_keys_q8_values")
SETTINGS = ("free", "top_k", "nucleus", "min_p", "mixed")


def listed():
    b06 = {"n_kv": 8, "rep": 2}
    b8 = {"n_kv": 8, "rep": 4}
    a3 = {"n_kv": 4, "rep": 8}
    plain = {"window": 0, "cap": 0.0, "slopes": False, "docs": False, "prefix": False, "chunk": False, "mix": False}
    return [
        # one user's next token behind an image, in a small model: latency alone
        {"name": "axes-1", "op": "axes", "rows": 1, "axes": 3, "far": 900, "page": 64, "slots": 4096, "kv": "f16", **b06},
        # a ragged batch, some rows idle, 8-bit cache, small pages
        {"name": "axes-37-q8", "op": "axes", "rows": 37, "axes": 3, "far": 5000, "page": 16, "slots": 8192, "kv": "q8",
         **a3},
        # a video's patches, far into a context
        {"name": "axes-2048-video", "op": "axes", "rows": 2048, "axes": 3, "far": 120000, "page": 128, "slots": 32768,
         "kv": "f16_keys_q8_values", **b8},
        # a few short chats of a model with capped scores: latency
        {"name": "shaped-8-cap", "op": "shaped", "rows": 8, "shared": 0, "own": 100, "page": 16, "kv": "f16", **b06,
         **plain, "cap": 50.0},
        # long chats in a layer that sees a window of them; one idle row, one that sees nothing
        {"name": "shaped-32-window", "op": "shaped", "rows": 32, "shared": 0, "own": 16000, "page": 64,
         "kv": "f16_keys_q8_values", **b8, **plain, "window": 1024, "mix": True},
        # a full batch of answers over a long shared context, scores capped: the matrix cores' case
        {"name": "shaped-128-cap", "op": "shaped", "rows": 128, "shared": 16384, "own": 300, "page": 128, "kv": "f16",
         **b8, **plain, "cap": 30.0},
        # a prompt's chunk in a layer with a window, 8-bit values
        {"name": "shaped-chunk-window", "op": "shaped", "rows": 128, "shared": 12000, "own": 128, "page": 64,
         "kv": "f16_keys_q8_values", **b8, **plain, "chunk": True, "window": 4096},
        # a chunk of packed documents whose rows see one another, distances biased, 8-bit cache
        {"name": "shaped-chunk-documents", "op": "shaped", "rows": 100, "shared": 4000, "own": 100, "page": 32,
         "kv": "q8", **a3, **plain, "chunk": True, "slopes": True, "docs": True, "prefix": True},
        # one user's token: top-k and top-p as most set them
        {"name": "sample-1", "op": "sample", "rows": 1, "vocab": 151936, "settings": "mixed", "flat": False,
         "masked": False},
        # creative writing: the whole vocabulary at its temperature
        {"name": "sample-16-free", "op": "sample", "rows": 16, "vocab": 151936, "settings": "free", "flat": True,
         "masked": False},
        # a batch behind grammars
        {"name": "sample-48-masked", "op": "sample", "rows": 48, "vocab": 151936, "settings": "top_k", "flat": False,
         "masked": True},
        # a full batch of wide nuclei
        {"name": "sample-128-nucleus", "op": "sample", "rows": 128, "vocab": 151936, "settings": "nucleus", "flat": True,
         "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("axes", "shaped", "shaped", "sample"))
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 128), "vocab": _log(rng, 1000, 151936), "settings": rng.choice(SETTINGS),
                "flat": rng.random() < 0.4, "masked": rng.random() < 0.3}
    n_kv = rng.choice((1, 2, 4, 8))
    rep = rng.choice((1, 2, 4, 8) if n_kv < 8 else (1, 2, 4))
    case = {"op": op, "n_kv": n_kv, "rep": rep, "page": rng.choice(PAGES), "kv": rng.choice(STORES)}
    rows = _log(rng, 1, 2048 if op == "axes" else 128)
    if op == "axes":
        return {**case, "rows": rows, "axes": rng.choice((1, 2, 3, 4)), "far": _log(rng, 1, 120000),
                "slots": rng.choice((4096, 8192, 32768))}
    chunk = rows > 1 and rng.random() < 0.4
    shared = rng.choice((0, _log(rng, 1, 16384)))
    window = 0 if shared and not chunk else rng.choice((0, _log(rng, 1, 8192)))
    return {**case, "rows": rows, "shared": shared, "chunk": chunk, "window": window,
            "own": rows if chunk else _log(rng, 1, max(1, min(16384, 65536 // rows))),
            "cap": rng.choice((0.0, rng.uniform(5.0, 60.0))), "slopes": rng.random() < 0.4,
            "docs": (chunk or not shared) and rng.random() < 0.4, "prefix": chunk and rng.random() < 0.5,
            "mix": not chunk and rows >= 4 and rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------
class Source:
    """Seeded inputs on the GPU, each tensor from its own name."""

    def __init__(self, seed):
        self.seed = seed

    def _gen(self, name):
        key = hashlib.sha256(f"{self.seed}/{name}".encode()).digest()[:8]
        return torch.Generator("cuda").manual_seed(int.from_bytes(key, "little") >> 1)

    def normal(self, name, *shape):
        return torch.randn(*shape, generator=self._gen(name), device="cuda")

    def uniform(self, name, lo, hi, *shape):
        return torch.rand(*shape, generator=self._gen(name), device="cuda") * (hi - lo) + lo

    def integers(self, name, lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self._gen(name), device="cuda", dtype=dtype)

    def order(self, name, n):
        return torch.randperm(n, generator=self._gen(name), device="cuda").to(torch.int32)


class State:
    pass


def _bits(case):
    """(keys in 8 bits, values in 8 bits)"""
    return case["kv"] == "q8", case["kv"] != "f16"


def _store(rows, q8):
    """Cache rows of random values as they are held: f16, or 8 bits and an f16 scale for each 32."""
    if not q8:
        return rows.half(), None
    y = rows.view(*rows.shape[:-1], -1, 32)
    s = y.abs().amax(-1) / 127.0
    return torch.round(y / s[..., None]).to(torch.int8).view(rows.shape), s.half()


def _frequencies(axes):
    """[axes][64]: each pair's frequency at the axis that turns it, 0 at the others; the axes take the
    pairs in turn, the first also those of the last quarter."""
    f = torch.tensor(THETA ** (-2.0 * np.arange(HEAD // 2) / HEAD), dtype=torch.float32)
    pair = torch.arange(HEAD // 2)
    axis = torch.where(pair < 48, pair % axes, 0)
    return torch.where(axis[None, :] == torch.arange(axes)[:, None], f[None, :], torch.zeros(())).cuda()


def _prepare_axes(case, src, st):
    rows, page, dim = case["rows"], case["page"], case["n_kv"] * HEAD
    st.q = src.normal("q", rows, case["n_kv"] * case["rep"] * HEAD)
    st.k, st.v = src.normal("k", rows, dim), src.normal("v", rows, dim)
    st.q_norm, st.k_norm = src.uniform("q_norm", 0.5, 1.5, HEAD), src.uniform("k_norm", 0.5, 1.5, HEAD)
    st.freq = _frequencies(case["axes"])
    # every row its own slot of the pool: a prompt's rows follow one another, a batch's lie in pages of their own
    st.n_pages = max(case["slots"] // page, rows + 1 if rows <= 256 else rows // page + 2)
    first = int(src.integers("far", 0, case["far"], 1))
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    if rows > 256:  # one sequence's consecutive patches: frames of 16 rows of 24
        st.n_seq, st.len = 1, first + 1 + r
        st.seq = torch.zeros(rows, dtype=torch.int32, device="cuda")
        st.pos = first + torch.stack([r // 384, r // 24 % 16, r % 24, r % 7], 1)
    else:  # text and patches, behind earlier images (positions below the slot's)
        st.n_seq, st.len = rows, 1 + src.integers("len", 0, case["far"], rows)
        st.seq = src.order("seq", rows)
        back = (st.len.float() * src.uniform("back", 0, 1, rows)).int()
        st.pos = back[:, None] + src.integers("patch", 0, 40, rows, 4) * (r % 2)[:, None]
    if rows >= 8:
        st.len[5] = 0  # an idle row
    at = ((st.len - 1).clamp(min=0) // page).long()
    width = int(at.max()) + 1
    st.table = torch.full((st.n_seq, width), st.n_pages - 1, dtype=torch.int32, device="cuda")
    pages = src.order("pages", st.n_pages)
    key, _ = torch.unique(st.seq.long() * width + at, return_inverse=True)
    st.table.view(-1)[key] = pages[: key.numel()]


def _spans(case):
    """A case's rows: what each one's own words say, but for the lengths, which a batch draws.
    (from, until) by row, or how a batch's follow from its length."""
    rows, shared = case["rows"], case["shared"]
    begin, until = [0] * rows, [0] * rows
    if case["chunk"]:
        half = rows // 2 if case["docs"] and rows >= 16 else rows  # the chunk's second document starts here
        for r in range(rows):
            if case["docs"]:
                begin[r] = shared // 3 if r < half else shared + half
            if case["prefix"]:
                until[r] = shared + (half if r < half else rows)
    return begin, until


def _prepare_shaped(case, src, st):
    rows, page, P, window = case["rows"], case["page"], case["shared"], case["window"]
    heads = case["n_kv"] * case["rep"]
    st.q = src.normal("q", rows, heads * HEAD) * 2
    st.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32,
                             device="cuda") if case["slopes"] else None
    begin, until = _spans(case)
    if case["chunk"]:
        st.n_seq, st.seq = 1, torch.zeros(rows, dtype=torch.int32, device="cuda")
        lens = [P + 1 + r for r in range(rows)]
    else:
        st.n_seq, st.seq = rows, src.order("seq", rows)
        lens = [P + (int(n) if rows > 1 else case["own"]) for n in 1 + src.integers("len", 0, case["own"], rows)]
        if case["docs"]:
            begin = [n // 2 if r % 2 else 0 for r, n in enumerate(lens)]
        if case["mix"]:
            lens[1] = 0              # an idle row
            begin[2] = lens[2] + 5   # a row whose mask leaves nothing
    seqs = [int(v) for v in st.seq.cpu()]
    # what a row sees: [lo, hi)
    lo = [max(b, n - window if window and n > window else 0) for b, n in zip(begin, lens)]
    hi = [max(n, u) if n else 0 for n, u in zip(lens, until)]
    lo = [min(a, b) for a, b in zip(lo, hi)]
    take = [P > 0 and n >= P and a < P and a < b for n, a, b in zip(lens, lo, hi)]
    st.first = max((a for a, t in zip(lo, take) if t), default=P)  # the shared run: [first, P)
    st.lead = max((st.first + 63) // 64 * 64 - min((a for a, t in zip(lo, take) if t), default=st.first), 0)
    st.own_max = max([1] + [b - (P if t else a) for a, b, t in zip(lo, hi, take)])
    width = max(1, -(-max(hi) // page))
    whole = P // page  # pages shared; one that the shared run ends in is each sequence's own
    table, n = np.zeros((st.n_seq, width), np.int64), whole
    for r, s in enumerate(seqs):
        if case["chunk"] and r != rows - 1:
            continue
        need = -(-hi[r] // page)
        from_ = min(whole, need) if P else 0
        table[s, :from_] = np.arange(from_)
        table[s, from_:need] = n + np.arange(need - from_)
        n += need - from_
    st.n_pages = n + 1
    pages = src.order("pages", st.n_pages)
    st.table = pages[torch.from_numpy(table).cuda()].contiguous()
    st.leader = seqs[next((r for r in range(rows) if take[r]), 0)]
    word = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    st.len, st.share, st.begin, st.until = word(lens), word([int(P > 0)] * rows), word(begin), word(until)
    st.lo, st.hi, st.take = word(lo), word(hi), torch.tensor(take, device="cuda")
    k8, v8 = _bits(case)
    st.keys, st.key_scales = _store(src.normal("keys", st.n_pages * page, case["n_kv"] * HEAD), k8)
    st.values, st.value_scales = _store(src.normal("values", st.n_pages * page, case["n_kv"] * HEAD), v8)
    if P % page and not case["chunk"]:
        # the shared run's tail lies in a page of every sequence: the same rows in each
        tail = torch.arange(whole * page, P, device="cuda")
        of = _slots(st, torch.tensor([st.leader], device="cuda"), tail)[0]
        members = st.seq[st.take].long()
        to = _slots(st, members, tail)
        for pool in (st.keys, st.key_scales, st.values, st.value_scales):
            if pool is not None:
                pool[to.view(-1)] = pool[of].repeat(len(members), *([1] * (pool.dim() - 1)))


def _prepare_sample(case, src, st):
    rows, v, kind = case["rows"], case["vocab"], case["settings"]
    # a few hundred tokens stand out of the rest, in flat rows barely
    st.logits = src.normal("logits", rows, v) * (2.5 if case["flat"] else 1.5)
    n = min(v, 300)
    at = (src.integers("at", 0, v, rows, 1, dtype=torch.int64) + torch.arange(n, device="cuda") * (v // n)) % v
    st.logits.scatter_add_(1, at, src.uniform("peaks", 0, 1, rows, n) ** 3 * (4.0 if case["flat"] else 16.0))
    if case["masked"]:
        st.logits[::2] = st.logits[::2].masked_fill(src.uniform("mask", 0, 1, (rows + 1) // 2, v) < 0.9, -math.inf)
    if rows >= 8:
        st.logits[5] = -math.inf  # a grammar that allows nothing
    st.temperature = src.uniform("temperature", 0.5, 1.5, rows)
    st.top_k = torch.zeros(rows, dtype=torch.int32, device="cuda")
    st.top_p, st.min_p = torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda")
    r = torch.arange(rows, device="cuda")
    if kind in ("top_k", "mixed"):
        k = src.integers("top_k", 1, 100, rows)
        st.top_k = torch.where(r % 3 != 1, k, st.top_k) if kind == "mixed" else k
    if kind in ("nucleus", "mixed"):
        p = src.uniform("top_p", 0.8, 0.99, rows)
        st.top_p = torch.where(r % 3 != 2, p, st.top_p) if kind == "mixed" else p
    if kind in ("min_p", "mixed"):
        m = src.uniform("min_p", 0.01, 0.2, rows)
        st.min_p = torch.where(r % 4 == 2, m, st.min_p) if kind == "mixed" else m
    if kind == "mixed":
        st.temperature[3::8] = 0.0  # greedy
    st.draws = src.integers("draws", 0, 2**32, rows, dtype=torch.int64)


PREPARE = {"axes": _prepare_axes, "shaped": _prepare_shaped, "sample": _prepare_sample}


def prepare(case, seed):
    st, src = State(), Source(seed)
    st.case = case
    PREPARE[case["op"]](case, src, st)
    if case["op"] == "axes":
        k8, v8 = _bits(case)
        n, dim = st.n_pages * case["page"], case["n_kv"] * HEAD
        st.keys = torch.zeros(n, dim, dtype=torch.int8 if k8 else torch.float16, device="cuda")
        st.values = torch.zeros(n, dim, dtype=torch.int8 if v8 else torch.float16, device="cuda")
        st.key_scales = torch.zeros(n, dim // 32, dtype=torch.float16, device="cuda") if k8 else None
        st.value_scales = torch.zeros(n, dim // 32, dtype=torch.float16, device="cuda") if v8 else None
        st.out = torch.zeros_like(st.q)
    if own:
        _place(case, st)
    return st


# ---- the plain forms --------------------------------------------------------------------------
def _slots(st, seq, pos):
    page = st.case["page"]
    return st.table[seq.long()[:, None], (pos // page)[None, :].long()].long() * page + pos % page


def _wide(rows, scales):
    """Cache rows in f32, whatever they are held in."""
    if scales is None:
        return rows.float()
    return (rows.view(*scales.shape, 32).float() * scales.float()[..., None]).view(rows.shape)


def _plain_norm_rope(x, w, pos, freq):
    x = x.view(x.shape[0], -1, HEAD)
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    angle = (pos[:, : freq.shape[0], None].double() * freq.double()).sum(1)  # far positions: 64 bits
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = n[..., : HEAD // 2], n[..., HEAD // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1).view(x.shape[0], -1)


def _held(rows, q8):
    if not q8:
        return rows.clamp(-65504, 65504).half(), None
    y = rows.view(rows.shape[0], -1, 32)
    s = y.abs().amax(-1) / 127.0
    q = torch.where(s[..., None] > 0, torch.round(y / s[..., None]), torch.zeros_like(y))
    return q.to(torch.int8).view(rows.shape), s.clamp(max=65504).half()


def _plain_axes(st):
    page, (k8, v8) = st.case["page"], _bits(st.case)
    live = st.len > 0
    q = _plain_norm_rope(st.q, st.q_norm, st.pos, st.freq)
    k, ks = _held(_plain_norm_rope(st.k, st.k_norm, st.pos, st.freq), k8)
    v, vs = _held(st.v, v8)
    st.out = torch.where(live[:, None], q, st.out)
    at = (st.len - 1).clamp(min=0)
    slot = st.table[st.seq.long(), (at // page).long()].long() * page + at % page
    # an idle row's slot is given its own old contents back
    first = live.to(torch.int32).argmax()
    slot = torch.where(live, slot, slot[first])
    for pool, new in ((st.keys, k), (st.key_scales, ks), (st.values, v), (st.value_scales, vs)):
        if pool is not None:
            pool[slot] = torch.where(live[:, None], new, new[first])


def _shape_scores(st, s, pos, head_dims):
    """Scores of each row's heads at positions `pos` (which broadcast to them): capped, then biased."""
    cap = st.case["cap"]
    if cap:
        s = cap * torch.tanh(s / cap)
    if st.slopes is not None:
        n_kv, rep = st.case["n_kv"], st.case["rep"]
        s = s - st.slopes.view(n_kv, rep).view(head_dims) * (pos - (st.len - 1).view(-1, 1, 1, 1)).abs().float()
    return s


def _plain_shaped(st):
    case, P = st.case, st.case["shared"]
    rows, n_kv, rep, page = case["rows"], case["n_kv"], case["rep"], case["page"]
    q = st.q.view(rows, n_kv, rep, HEAD) / math.sqrt(HEAD)
    pick = lambda pool, i: None if pool is None else pool[i]  # noqa: E731
    lo, hi = st.lo.view(-1, 1, 1, 1), st.hi.view(-1, 1, 1, 1)
    pieces = []  # scores [rows, n_kv, rep, n] and the values they weigh
    begin = torch.where(st.take, torch.full_like(st.lo, P), st.lo)
    if case["chunk"]:  # one sequence: every position once
        begin, first, last = st.hi, int(st.lo.min()), int(st.hi.max())
    else:  # the shared run once
        first, last = (0, P) if bool(st.take.any()) else (0, 0)
    if last > first:
        pos = torch.arange(first, last, device="cuda")
        slot = _slots(st, torch.full((1,), st.leader, device="cuda"), pos)[0]
        K = _wide(st.keys[slot], pick(st.key_scales, slot)).view(-1, n_kv, HEAD).permute(1, 2, 0).contiguous()
        V = _wide(st.values[slot], pick(st.value_scales, slot)).view(-1, n_kv, HEAD).permute(1, 0, 2).contiguous()
        s = torch.matmul(q.permute(1, 0, 2, 3).reshape(n_kv, rows * rep, HEAD), K)
        s = _shape_scores(st, s.view(n_kv, rows, rep, -1).permute(1, 0, 2, 3), pos, (1, n_kv, rep, 1))
        sees = (pos >= lo) & (pos < hi)
        if not case["chunk"]:
            sees = sees & st.take.view(-1, 1, 1, 1)
        pieces.append((s.masked_fill(~sees, -math.inf), V, True))
    if not case["chunk"]:  # each row's own positions, padded to the longest
        pos = begin[:, None] + torch.arange(st.own_max, device="cuda")
        at = (pos // page).clamp(max=st.table.shape[1] - 1).long()
        slot = st.table[st.seq.long()[:, None], at].long() * page + pos % page
        K = _wide(st.keys[slot], pick(st.key_scales, slot)).view(rows, -1, n_kv, HEAD).permute(0, 2, 3, 1).contiguous()
        V = _wide(st.values[slot], pick(st.value_scales, slot)).view(rows, -1, n_kv, HEAD).permute(0, 2, 1, 3).contiguous()
        pos = pos[:, None, None, :]
        s = _shape_scores(st, torch.matmul(q, K), pos, (1, n_kv, rep, 1))
        pieces.append((s.masked_fill((pos < lo) | (pos >= hi), -math.inf), V, False))
    m = torch.stack([s.amax(-1) for s, _, _ in pieces]).amax(0)
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    total, o = 0.0, 0.0
    for s, V, common in pieces:
        e = torch.exp(s - m[..., None])
        total = total + e.sum(-1)
        if common:
            o = o + torch.matmul(e.permute(1, 0, 2, 3).reshape(n_kv, rows * rep, -1), V) \
                .view(n_kv, rows, rep, HEAD).permute(1, 0, 2, 3)
        else:
            o = o + torch.matmul(e, V)
    o = torch.where(total[..., None] > 0, o / total[..., None], torch.zeros_like(o))
    return o.reshape(rows, -1)


def _plain_sample(st):
    """In 64 bits, as a sum's border decides which token it is."""
    rows, v = st.logits.shape
    x, ids = torch.sort(st.logits, dim=-1, descending=True, stable=True)
    some = x[:, 0] > -math.inf
    greedy = st.temperature <= 0
    T = torch.where(greedy, torch.ones_like(st.temperature), st.temperature).double()
    top = torch.where(some, x[:, 0], torch.zeros_like(x[:, 0])).double()
    y = (x.double() - top[:, None]) / T[:, None]
    w = torch.exp(y)
    n = torch.where(st.top_k > 0, st.top_k.long(), torch.full_like(ids[:, 0], v))
    n = torch.minimum(n, (x > -math.inf).sum(-1))
    n = torch.minimum(n, (w >= st.min_p.double()[:, None]).sum(-1))
    n = torch.where(greedy, torch.ones_like(n), n).clamp(min=1)
    C = torch.cumsum(w, -1)
    S = C.gather(1, n[:, None] - 1)
    p = st.top_p.double()[:, None]
    n = torch.where(p[:, 0] < 1, (C < p * S).sum(-1) + 1, n)
    S = C.gather(1, n[:, None] - 1)
    u = (st.draws.double() + 0.5) * 2.0**-32
    at = torch.minimum((C <= u[:, None] * S).sum(-1), n - 1)
    y, token = y.gather(1, at[:, None])[:, 0], ids.gather(1, at[:, None])[:, 0]
    none = torch.full_like(token, -1)
    return {"token": torch.where(some, token, none).int(), "kept": torch.where(some, n, torch.zeros_like(n)).int(),
            "logprob": torch.where(some, y - torch.log(S[:, 0]), torch.full_like(y, -math.inf)).float()}


def _values(rows, scales):
    """A pool as the values it holds; 8-bit entries as their products with the scales, to f16's 2^-11."""
    return rows if scales is None else rows.view(*scales.shape, 32) * scales[..., None]


def run(state):
    op = state.case["op"]
    if own:
        state.call()
        if op != "axes":
            return state.out
    elif op == "axes":
        _plain_axes(state)
    elif op == "shaped":
        return _plain_shaped(state)
    else:
        return _plain_sample(state)
    return {"q": state.out, "keys": _values(state.keys, state.key_scales),
            "values": _values(state.values, state.value_scales)}


# ---- the framework's buffers and calls --------------------------------------------------------
_framework = None


def _skyla():
    global _framework
    if _framework is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "skyla-kernel_amd"))
        from skyla_hip import batch, engine
        from skyla_hip.abi import Context
        _framework = (batch, engine, Context.new(0))
    return _framework


class _Memory:
    def __init__(self, keep, ptr, n, kind):
        self.keep = keep
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": kind, "data": (ptr, False), "version": 3,
                                         "strides": None}


class _Held:
    """Frees what a state holds once nothing refers to it (its outputs do)."""

    def __init__(self):
        self.recording, self.buffers = None, []

    def __del__(self):
        if self.recording is not None:
            self.recording.free()
        for b in self.buffers:
            b.free()


class _Arena:
    """Rows placed one after another in an arena buffer, as the engine's are: 64 control words first."""

    def __init__(self):
        self.size, self.items = 64, []

    def put(self, rows):
        """Rows of f32 or 32-bit words; their (offset, row stride)."""
        rows = rows.view(rows.shape[0], -1) if rows.dim() > 1 else rows.view(1, -1)
        off, stride = self.size, -(-rows.shape[1] // 64) * 64
        self.size += stride * rows.shape[0]
        self.items.append((off, stride, rows))
        return off, stride

    def room(self, n):
        off = self.size
        self.size += -(-n // 64) * 64
        return off

    def place(self, ctx, held):
        buf = ctx.alloc_host(self.size * 4)
        held.buffers.append(buf)
        flat = _view(held, buf, "<f4")
        for off, stride, rows in self.items:
            to = flat[off: off + stride * rows.shape[0]].view(rows.shape[0], stride)[:, : rows.shape[1]]
            to.copy_(rows.contiguous().view(torch.float32))
        return buf, flat


def _view(held, buf, kind, first=0, count=None):
    size = np.dtype(kind).itemsize
    count = buf.size // size - first if count is None else count
    return torch.as_tensor(_Memory(held, buf.device_ptr() + first * size, count, kind), device="cuda")


def _words(*columns):
    """Columns of 32-bit words (those of 64 bits by their low halves) as rows of them."""
    low = lambda c: ((c & 0xFFFFFFFF) - ((c & 0x80000000) << 1)).int() if c.dtype == torch.int64 else c  # noqa: E731
    return torch.stack([low(c).contiguous().view(torch.int32) for c in columns], 1)


def _control(flat, rows, shared=0, leader=0, first=0):
    flat[:8].view(torch.int32)[2:6] = torch.tensor([rows, shared, leader, first], dtype=torch.int32, device="cuda")


def _pool(ctx, held, st, paged):
    """The state's cache rows in a pool buffer; the state's tensors become views of it."""
    buf = ctx.alloc_host(max(16, paged.bytes()))
    held.buffers.append(buf)
    at = paged.layout
    for name, off in (("keys", at.keys(0)), ("key_scales", at.key_scales(0)), ("values", at.values(0)),
                      ("value_scales", at.value_scales(0))):
        rows = getattr(st, name)
        if rows is not None:
            to = _view(held, buf, "|i1" if rows.dtype == torch.int8 else "<f2", off, rows.numel()).view(rows.shape)
            to.copy_(rows)
            setattr(st, name, to)
    return buf


def _place(case, st):
    batch, E, ctx = _skyla()
    held, a, rows = _Held(), _Arena(), case["rows"]
    if case["op"] == "sample":
        zero = torch.zeros_like(st.top_k)
        words = a.put(_words(st.temperature, st.top_p, st.min_p, st.top_k, st.draws, zero, zero, zero).view(-1))
        x = a.put(st.logits)
        at = batch.SampleRegions(controls=words[0], out=a.room(4 * rows),
                                 part=a.room(batch.sample_size(rows, case["vocab"])))
        arena, flat = a.place(ctx, held)
        _control(flat, rows)
        out = flat[at.out: at.out + 4 * rows].view(rows, 4)
        st.out = {"token": out.view(torch.int32)[:, 0], "kept": out.view(torch.int32)[:, 1], "logprob": out[:, 2]}
        kernels = batch.LogitsKernels(ctx, arena)
        body = lambda r: kernels.sample(r, at, x, case["vocab"], rows)  # noqa: E731
    else:
        n_head = case["n_kv"] * case["rep"]
        c = E.Config(n_embd=256, n_head=n_head, n_head_kv=case["n_kv"], head_dim=HEAD, eps=EPS, rope_theta=THETA)
        paged = batch.Paged(E.KvPrecision[case["kv"].upper()], case["page"], st.n_pages, st.n_seq, st.table.shape[1],
                            case["n_kv"] * HEAD)
        pool = _pool(ctx, held, st, paged)
        zero = torch.zeros_like(st.seq)
        words = a.put(_words(st.seq, st.len, zero if case["op"] == "axes" else st.share, zero).view(-1))
        table = a.room(st.table.numel())
        q = a.put(st.q)
        at = batch.BatchRegions(rows=words[0], table=table)
        if case["op"] == "axes":
            k, v = a.put(st.k), a.put(st.v)
            norms = [a.put(t.view(-1))[0] for t in (st.q_norm, st.k_norm, st.freq)]
            at.axes = a.put(st.pos.int().view(-1))[0]
        else:
            shape = batch.Shape(cap=case["cap"], window=case["window"],
                                slopes=None if st.slopes is None else a.put(st.slopes)[0])
            at.spans = a.put(_words(st.begin, st.until).view(-1))[0]
            run_ = case["shared"] - st.first
            parts = batch.shaped_splits(rows, case["n_kv"], case["rep"], run_, st.own_max, st.lead if run_ else 0)
            at.part = a.room(batch.shaped_part_size(rows, n_head, parts))
        out = a.room(q[1] * rows), q[1]
        arena, flat = a.place(ctx, held)
        flat[table: table + st.table.numel()].view(torch.int32).copy_(st.table.view(-1))
        if case["op"] == "axes":
            _control(flat, rows)
        else:
            _control(flat, rows, case["shared"], st.leader, st.first)
        st.out = flat[out[0]: out[0] + out[1] * rows].view(rows, out[1])[:, : n_head * HEAD]
        st.out.zero_()
        kernels = batch.BatchKernels(ctx, arena, arena, [pool], c, paged)
        if case["op"] == "axes":
            body = lambda r: kernels.append_axes(r, 0, at, q, k, v[0], out, *norms, case["axes"], rows)  # noqa: E731
        else:
            body = lambda r: kernels.attend_shaped(r, 0, at, q, out, rows, parts, shape)  # noqa: E731
    torch.cuda.synchronize()
    held.recording = ctx.record(False, body)
    # the arena's copies are the inputs now
    for name in ("logits", "q", "k", "v", "table", "pos"):
        st.__dict__.pop(name, None)
    st.held = held
    st.call = lambda: ctx.replay(held.recording)


# ---- what a pass cannot do without ------------------------------------------------------------
def _entry_bytes(case):
    """Bytes of one position's keys and values."""
    dim = case["n_kv"] * HEAD
    return sum(dim + dim // 16 if q8 else 2 * dim for q8 in _bits(case))


def _seen(case):
    """(distinct positions, (row, position) pairs) that a case's rows attend to, on average over its lengths."""
    rows, P, window = case["rows"], case["shared"], case["window"] or 1 << 40
    if case["chunk"]:
        begin, until = _spans(case)
        spans = [(max(b, P + 1 + r - window, 0), max(P + 1 + r, u)) for r, (b, u) in enumerate(zip(begin, until))]
        return max(b for _, b in spans) - min(a for a, _ in spans), sum(b - a for a, b in spans)
    n = case["own"]

    def mean(share):  # of min(share length, window), the length up to n
        edge = min(n, window / share)
        return (share * edge * (edge + 1) / 2 + min(window, share * n) * (n - edge)) / n
    each = (mean(1.0) + mean(0.5)) / 2 if case["docs"] else mean(1.0)
    if rows == 1:
        each = min(n, window)
    return P + rows * each, rows * (each + P)


def work(case):
    rows = case["rows"]
    if case["op"] == "sample":
        return {"bytes": rows * (4 * case["vocab"] + 32 + 12), "flops": 0}
    heads = case["n_kv"] * case["rep"]
    if case["op"] == "axes":
        return {"bytes": rows * (4 * HEAD * (2 * heads + 2 * case["n_kv"]) + _entry_bytes(case) + 36),
                "flops": rows * HEAD * (heads + case["n_kv"]) * 8.0}
    distinct, pairs = _seen(case)
    return {"bytes": distinct * _entry_bytes(case) + rows * heads * HEAD * 8, "flops": 4.0 * HEAD * heads * pairs}


# ---- the same in 64 bits ----------------------------------------------------------------------
def _exact_axes(case, st):
    k8, v8 = _bits(case)
    angle = torch.zeros(case["rows"], HEAD // 2, dtype=torch.float64, device="cuda")
    for a in range(case["axes"]):
        angle += st.pos[:, a].double()[:, None] * st.freq[a].double()[None, :]
    turn = torch.polar(torch.ones_like(angle), angle)

    def rotated(x, w):
        x = x.double().view(case["rows"], -1, 2, HEAD // 2)
        x = x * torch.rsqrt(x.pow(2).sum((2, 3), keepdim=True) / HEAD + EPS) * w.double().view(2, HEAD // 2)
        z = torch.complex(x[:, :, 0], x[:, :, 1]) * turn[:, None]
        return torch.stack([z.real, z.imag], 2).reshape(case["rows"], -1)

    live = (st.len > 0).nonzero().view(-1)
    q = torch.zeros(st.q.shape, dtype=torch.float64, device="cuda")
    q[live] = rotated(st.q, st.q_norm)[live]
    out = {"q": q}
    page, n = case["page"], st.n_pages * case["page"]
    p = (st.len - 1).clamp(min=0).long()
    slot = st.table[st.seq.long(), p // page].long() * page + p % page
    for name, rows, q8 in (("keys", rotated(st.k, st.k_norm), k8), ("values", st.v.double(), v8)):
        pool = torch.zeros(n, case["n_kv"] * HEAD, dtype=torch.float64, device="cuda")
        pool[slot[live]] = rows[live]
        out[name] = None if q8 else pool  # what 8 bits hold is their rounding's choice
    return out


def _exact_shaped(case, st):
    n_kv, rep, page = case["n_kv"], case["rep"], case["page"]
    out = torch.zeros(case["rows"], n_kv * rep, HEAD, dtype=torch.float64, device="cuda")

    def read(pool, scales, slot):
        x = pool[slot].double()
        if scales is not None:
            x = x * scales[slot].double().repeat_interleave(32, 1)
        return x.view(-1, n_kv, HEAD).transpose(0, 1)

    def entries(seq, lo, hi):
        pos = torch.arange(lo, hi, device="cuda")
        slot = st.table[seq, pos // page].long() * page + pos % page
        return read(st.keys, st.key_scales, slot), read(st.values, st.value_scales, slot)

    if case["chunk"]:
        every = entries(0, 0, int(st.hi.max()))
    for r in range(case["rows"]):
        length, begin, until = int(st.len[r]), int(st.begin[r]), int(st.until[r])
        if length == 0:
            continue
        at, end = length - 1, max(length, until)
        start = max(begin, length - case["window"]) if case["window"] else begin
        if start >= end:
            continue
        K, V = (x[:, start:end] for x in every) if case["chunk"] else entries(int(st.seq[r]), start, end)
        q = st.q[r].double().view(n_kv, rep, HEAD)
        s = torch.matmul(q, K.transpose(1, 2).contiguous()) / math.sqrt(HEAD)
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        if case["slopes"]:
            away = torch.abs(torch.arange(start, end, device="cuda") - at).double()
            s = s - st.slopes.double().view(n_kv, rep, 1) * away
        out[r] = torch.matmul(torch.softmax(s, -1), V.contiguous()).reshape(n_kv * rep, HEAD)
    return out.view(case["rows"], -1)


def _exact_sample(case, st):
    token, kept, logprob = [], [], []
    for r in range(case["rows"]):
        x = st.logits[r].cpu().numpy().astype(np.float64)
        ids = np.argsort(-x, kind="stable")
        ids = ids[: int((x > -np.inf).sum())]
        if len(ids) == 0:
            token.append(-1), kept.append(0), logprob.append(-np.inf)
            continue
        T = float(st.temperature[r])
        y = (x[ids] - x[ids[0]]) / (T if T > 0 else 1.0)
        if int(st.top_k[r]):
            y = y[: int(st.top_k[r])]
        y = y[: max(1, int((np.exp(y) >= float(st.min_p[r])).sum()))]
        if T <= 0:
            y = y[:1]
        total = np.cumsum(np.exp(y))
        p = float(st.top_p[r])
        if p < 1:
            total = total[: int(np.searchsorted(total, p * total[-1], side="left")) + 1]
        u = (int(st.draws[r]) + 0.5) / 2**32
        i = min(int(np.searchsorted(total, u * total[-1], side="right")), len(total) - 1)
        token.append(int(ids[i])), kept.append(len(total)), logprob.append(y[i] - math.log(total[-1]))
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"token": whole(token), "kept": whole(kept),
            "logprob": torch.tensor(logprob, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    st, src = State(), Source(seed)
    st.case = case
    PREPARE[case["op"]](case, src, st)
    return {"axes": _exact_axes, "shaped": _exact_shaped, "sample": _exact_sample}[case["op"]](case, st)
