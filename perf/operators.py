"""What the operators of a served batch are measured on: decode rows of many sequences over a
paged KV cache.

Three kinds of case:

  append  rows of q, k, v: QK-norm, rotary positions, keys and values into the cache's pages
  attend  attention of a batch's rows over their pages, a leading run of positions shared by all
  logits  penalties for repeated tokens, biases and a grammar's mask on rows of logits

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


def listed():
    b06 = {"n_kv": 8, "rep": 2}
    b8 = {"n_kv": 8, "rep": 4}
    a3 = {"n_kv": 4, "rep": 8}
    return [
        # one user's next token in a small model: latency alone
        {"name": "append-1", "op": "append", "rows": 1, "far": 900, "page": 64, "slots": 4096, "kv": "f16", **b06},
        # a ragged batch, some rows idle, 8-bit cache, small pages
        {"name": "append-37-q8", "op": "append", "rows": 37, "far": 5000, "page": 16, "slots": 8192, "kv": "q8", **a3},
        # a long prompt's rows, far into a context
        {"name": "append-2048", "op": "append", "rows": 2048, "far": 120000, "page": 128, "slots": 32768,
         "kv": "f16_keys_q8_values", **b8},
        # a few short chats, nothing shared: latency
        {"name": "attend-8-short", "op": "attend", "rows": 8, "shared": 0, "own": 100, "page": 16, "kv": "f16",
         "mix": False, "chunk": False, **b06},
        # chats behind one system prompt that ends inside a page; one idle row, one that shares nothing
        {"name": "attend-32-system", "op": "attend", "rows": 32, "shared": 1000, "own": 200, "page": 64,
         "kv": "f16_keys_q8_values", "mix": True, "chunk": False, **b8},
        # questions about one document, eight query heads a key head, 8-bit cache
        {"name": "attend-64-document", "op": "attend", "rows": 64, "shared": 8192, "own": 777, "page": 32, "kv": "q8",
         "mix": False, "chunk": False, **a3},
        # a full batch of answers over a long shared context: the matrix cores' case
        {"name": "attend-128-long", "op": "attend", "rows": 128, "shared": 32768, "own": 512, "page": 128, "kv": "f16",
         "mix": False, "chunk": False, **b8},
        # one sequence's next token after a long document: the length has to be split
        {"name": "attend-1-16k", "op": "attend", "rows": 1, "shared": 0, "own": 16384, "page": 64,
         "kv": "f16_keys_q8_values", "mix": False, "chunk": False, **b8},
        # a prompt's chunk of 128 rows after 4000 positions of the same sequence
        {"name": "attend-chunk-128", "op": "attend", "rows": 128, "shared": 4000, "own": 128, "page": 64,
         "kv": "f16_keys_q8_values", "mix": False, "chunk": True, **b8},
        # one user's logits with a repetition penalty
        {"name": "logits-1", "op": "logits", "rows": 1, "vocab": 151936, "history": 1000, "biases": 8, "masked": False},
        # a batch with penalties, biases and grammars
        {"name": "logits-48", "op": "logits", "rows": 48, "vocab": 151936, "history": 4096, "biases": 300, "masked": True},
        # a full batch late in long contexts
        {"name": "logits-128-long", "op": "logits", "rows": 128, "vocab": 151936, "history": 32768, "biases": 16,
         "masked": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "logits"))
    if op == "logits":
        return {"op": op, "rows": _log(rng, 1, 128), "vocab": _log(rng, 1000, 151936), "history": _log(rng, 1, 32768),
                "biases": rng.choice((0, _log(rng, 1, 300))), "masked": rng.random() < 0.6}
    n_kv = rng.choice((1, 2, 4, 8))
    rep = rng.choice((1, 2, 4, 8) if n_kv < 8 else (1, 2, 4))
    case = {"op": op, "n_kv": n_kv, "rep": rep, "page": rng.choice(PAGES), "kv": rng.choice(STORES)}
    if op == "append":
        rows = _log(rng, 1, 2048)
        return {**case, "rows": rows, "far": _log(rng, 1, 120000), "slots": rng.choice((4096, 8192, 32768))}
    rows = _log(rng, 1, 128)
    shared = rng.choice((0, _log(rng, 1, 32768), _log(rng, 1, 32768)))
    chunk = rows > 1 and rng.random() < 0.25
    if chunk:
        return {**case, "rows": rows, "shared": shared, "own": rows, "mix": False, "chunk": True}
    own_max = max(1, min(16384, 65536 // rows))
    return {**case, "rows": rows, "shared": shared, "own": _log(rng, 1, own_max),
            "mix": rows >= 4 and rows * shared <= 65536 and rng.random() < 0.5, "chunk": False}


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

    def integers(self, name, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self._gen(name), device="cuda", dtype=torch.int32)

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


def _frequencies():
    return torch.tensor(THETA ** (-2.0 * np.arange(HEAD // 2) / HEAD), dtype=torch.float32, device="cuda")


def _prepare_append(case, src, st):
    rows, page, dim = case["rows"], case["page"], case["n_kv"] * HEAD
    st.q = src.normal("q", rows, case["n_kv"] * case["rep"] * HEAD)
    st.k, st.v = src.normal("k", rows, dim), src.normal("v", rows, dim)
    st.q_norm, st.k_norm = src.uniform("q_norm", 0.5, 1.5, HEAD), src.uniform("k_norm", 0.5, 1.5, HEAD)
    st.freq = _frequencies()
    # every row its own slot of the pool: a prompt's rows follow one another, a batch's lie in pages of their own
    st.n_pages = max(case["slots"] // page, rows + 1 if rows <= 256 else rows // page + 2)
    first = int(src.integers("far", 0, case["far"], 1))
    if rows > 256:  # one sequence's consecutive positions
        st.n_seq, st.len = 1, first + 1 + torch.arange(rows, device="cuda", dtype=torch.int32)
        st.seq = torch.zeros(rows, dtype=torch.int32, device="cuda")
    else:
        st.n_seq, st.len = rows, 1 + src.integers("len", 0, case["far"], rows)
        st.seq = src.order("seq", rows)
    if rows >= 8:
        st.len[5] = 0  # an idle row
    at = ((st.len - 1).clamp(min=0) // page).long()
    width = int(at.max()) + 1
    st.table = torch.full((st.n_seq, width), st.n_pages - 1, dtype=torch.int32, device="cuda")
    pages = src.order("pages", st.n_pages)
    key, back = torch.unique(st.seq.long() * width + at, return_inverse=True)
    st.table.view(-1)[key] = pages[: key.numel()]
    st.share = torch.zeros_like(st.len)
    st.shared, st.leader = 0, 0


def _prepare_attend(case, src, st):
    rows, page, shared = case["rows"], case["page"], case["shared"]
    st.q = src.normal("q", rows, case["n_kv"] * case["rep"] * HEAD) * 2
    if case["chunk"]:
        st.n_seq, st.seq = 1, torch.zeros(rows, dtype=torch.int32, device="cuda")
        st.len = shared + 1 + torch.arange(rows, device="cuda", dtype=torch.int32)
    else:
        st.n_seq, st.seq = rows, src.order("seq", rows)
        st.len = shared + (1 + src.integers("len", 0, case["own"], rows) if rows > 1 else
                           torch.full((1,), case["own"], dtype=torch.int32, device="cuda"))
    st.share = torch.full_like(st.len, shared)
    if case["mix"]:
        st.len[1] = 0   # an idle row
        st.share[2] = 0  # a row whose pages are all its own
    lens = [int(v) for v in st.len.cpu()]
    seqs = [int(v) for v in st.seq.cpu()]
    takes = [int(v) for v in st.share.cpu()]
    width = max(1, -(-max(lens) // page))
    whole = shared // page  # pages shared; one that the shared run ends in is each sequence's own
    table, n = np.zeros((st.n_seq, width), np.int64), whole
    for r, s in enumerate(seqs):
        need = -(-lens[r] // page)
        from_ = whole if takes[r] else 0
        if case["chunk"] and r != rows - 1:
            continue
        table[s, :from_] = np.arange(from_)
        if need > from_:
            table[s, from_:need] = n + np.arange(need - from_)
            n += need - from_
    st.n_pages = n + 1
    pages = src.order("pages", st.n_pages)
    st.table = pages[torch.from_numpy(table).cuda()].contiguous()
    st.leader = seqs[next((r for r in range(rows) if takes[r] and lens[r]), 0)]
    st.shared = shared
    st.own_max = max(n - (shared if take else 0) for n, take in zip(lens, takes))  # the longest of the rows' own runs
    k8, v8 = _bits(case)
    st.keys, st.key_scales = _store(src.normal("keys", st.n_pages * page, case["n_kv"] * HEAD), k8)
    st.values, st.value_scales = _store(src.normal("values", st.n_pages * page, case["n_kv"] * HEAD), v8)
    if shared % page and not case["chunk"]:
        # the shared run's tail lies in a page of every sequence: the same rows in each
        tail = torch.arange(whole * page, shared, device="cuda")
        of = _slots(st, torch.tensor([st.leader], device="cuda"), tail)[0]
        members = st.seq[(st.share > 0) & (st.len > 0)].long()
        to = _slots(st, members, tail)
        for pool in (st.keys, st.key_scales, st.values, st.value_scales):
            if pool is not None:
                pool[to.view(-1)] = pool[of].repeat(len(members), *([1] * (pool.dim() - 1)))


def _prepare_logits(case, src, st):
    rows, v, h, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    st.logits = src.normal("logits", rows, v) * 3
    # tokens repeat as text does: a small share of the vocabulary makes most of a history
    st.history = (src.uniform("history", 0, 1, rows, h) ** 4 * v).int().clamp(max=v - 1)
    st.history_len = src.integers("history_len", max(1, h // 2), h + 1, rows)
    st.prompt_len = (st.history_len * src.uniform("prompt", 0, 1, rows)).int()
    st.repetition = src.uniform("repetition", 1.0, 1.5, rows)
    st.frequency, st.presence = src.uniform("frequency", 0, 0.5, rows), src.uniform("presence", 0, 1, rows)
    st.bias_id = torch.stack([src.order(f"bias.{r}", v)[: max(1, nb)] for r in range(rows)])
    st.bias = src.normal("bias", rows, max(1, nb)) * 5
    st.bias_len = src.integers("bias_len", nb // 2, nb + 1, rows)
    st.masked = torch.zeros(rows, dtype=torch.int32, device="cuda")
    if case["masked"]:
        st.masked[::2] = 1
    st.mask = src.integers("mask", -2**31, 2**31 - 1, rows, -(-v // 32))


def prepare(case, seed):
    st, src = State(), Source(seed)
    st.case = case
    {"append": _prepare_append, "attend": _prepare_attend, "logits": _prepare_logits}[case["op"]](case, src, st)
    if case["op"] == "append":
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
    angle = pos.double()[:, None] * freq.double()  # far positions: 64 bits
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


def _plain_append(st):
    page, (k8, v8) = st.case["page"], _bits(st.case)
    live = st.len > 0
    pos = (st.len - 1).clamp(min=0)
    q = _plain_norm_rope(st.q, st.q_norm, pos, st.freq)
    k, ks = _held(_plain_norm_rope(st.k, st.k_norm, pos, st.freq), k8)
    v, vs = _held(st.v, v8)
    st.out = torch.where(live[:, None], q, st.out)
    slot = st.table[st.seq.long(), (pos // page).long()].long() * page + pos % page
    # an idle row's slot is given its own old contents back
    slot = torch.where(live, slot, slot[live.to(torch.int32).argmax()])
    first = live.to(torch.int32).argmax()
    for pool, new in ((st.keys, k), (st.key_scales, ks), (st.values, v), (st.value_scales, vs)):
        if pool is not None:
            pool[slot] = torch.where(live[:, None], new, new[first])


def _plain_attend(st):
    case, P = st.case, st.shared
    rows, n_kv, rep, page = case["rows"], case["n_kv"], case["rep"], case["page"]
    q = st.q.view(rows, n_kv, rep, HEAD) / math.sqrt(HEAD)
    member = (st.share > 0) & (st.len >= P)
    start = torch.where(member, P, 0)
    n = st.len - start
    # each row's own positions, padded to the longest
    pos = start[:, None] + torch.arange(st.own_max, device="cuda")
    at = torch.minimum(pos // page, torch.tensor(st.table.shape[1] - 1, device="cuda")).long()
    slot = st.table[st.seq.long()[:, None], at].long() * page + pos % page
    scales = lambda pool, i: None if pool is None else pool[i]  # noqa: E731
    K = _wide(st.keys[slot], scales(st.key_scales, slot)).view(rows, -1, n_kv, HEAD).permute(0, 2, 3, 1)
    V = _wide(st.values[slot], scales(st.value_scales, slot)).view(rows, -1, n_kv, HEAD).permute(0, 2, 1, 3)
    s = torch.matmul(q, K).masked_fill((pos >= st.len[:, None])[:, None, None, :], -math.inf)
    m = s.amax(-1)
    if P > 0:
        slot = _slots(st, torch.full((1,), st.leader, device="cuda"), torch.arange(P, device="cuda"))[0]
        PK = _wide(st.keys[slot], scales(st.key_scales, slot)).view(P, n_kv, HEAD).permute(1, 2, 0)
        PV = _wide(st.values[slot], scales(st.value_scales, slot)).view(P, n_kv, HEAD).permute(1, 0, 2)
        ps = torch.matmul(q.permute(1, 0, 2, 3).reshape(n_kv, rows * rep, HEAD), PK).view(n_kv, rows, rep, P)
        ps = ps.masked_fill(~member[None, :, None, None], -math.inf)
        m = torch.maximum(m, ps.amax(-1).permute(1, 0, 2))
    m = torch.where(st.len[:, None, None] > 0, m, torch.zeros_like(m))
    e = torch.exp(s - m[..., None])
    total, o = e.sum(-1), torch.matmul(e, V)
    if P > 0:
        e = torch.exp(ps - m.permute(1, 0, 2)[..., None])
        total = total + e.sum(-1).permute(1, 0, 2)
        o = o + torch.matmul(e.view(n_kv, rows * rep, P), PV).view(n_kv, rows, rep, HEAD).permute(1, 0, 2, 3)
    o = torch.where(st.len[:, None, None, None] > 0, o / total[..., None], torch.zeros_like(o))
    return o.reshape(rows, -1)


def _plain_logits(st):
    rows, v = st.logits.shape
    at = torch.arange(st.history.shape[1], device="cuda")[None, :]
    live = at < st.history_len[:, None]
    ids = st.history.long()
    seen = torch.zeros(rows, v, device="cuda").scatter_add_(1, ids, live.float())
    made = torch.zeros(rows, v, device="cuda").scatter_add_(1, ids, (live & (at >= st.prompt_len[:, None])).float())
    rho = st.repetition[:, None]
    y = torch.where(seen > 0, torch.where(st.logits > 0, st.logits / rho, st.logits * rho), st.logits)
    y = torch.where(made > 0, y - (st.frequency[:, None] * made + st.presence[:, None]), y)
    counts = torch.arange(st.bias.shape[1], device="cuda")[None, :] < st.bias_len[:, None]
    y = y.scatter_add(1, st.bias_id.long(), torch.where(counts, st.bias, torch.zeros_like(st.bias)))
    bit = torch.arange(v, device="cuda")
    allowed = (st.mask[:, bit // 32] >> (bit % 32)) & 1
    return torch.where((allowed == 0) & (st.masked > 0)[:, None], torch.full_like(y, -math.inf), y)


def _values(rows, scales):
    """A pool as the values it holds; 8-bit entries as their products with the scales, to f16's 2^-11."""
    return rows if scales is None else rows.view(*scales.shape, 32) * scales[..., None]


def run(state):
    op = state.case["op"]
    if own:
        state.call()
        if op != "append":
            return state.out
    elif op == "append":
        _plain_append(state)
    elif op == "attend":
        return _plain_attend(state)
    else:
        return _plain_logits(state)
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
    return torch.stack([c.contiguous().view(torch.int32) for c in columns], 1)


def _control(flat, rows, shared=0, leader=0):
    flat[:8].view(torch.int32)[2:5] = torch.tensor([rows, shared, leader], dtype=torch.int32, device="cuda")


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
    if case["op"] == "logits":
        words = _words(st.history_len, st.prompt_len, st.bias_len, st.masked, st.repetition, st.frequency, st.presence,
                       torch.zeros_like(st.masked))
        entries = torch.stack([st.bias_id, st.bias.view(torch.int32)], 2).view(rows, -1)
        x, history, bias, mask = a.put(st.logits), a.put(st.history), a.put(entries), a.put(st.mask)
        controls = a.put(words.view(-1))
        y = a.room(x[1] * rows), x[1]
        arena, flat = a.place(ctx, held)
        _control(flat, rows)
        st.out = flat[y[0]: y[0] + y[1] * rows].view(rows, y[1])[:, : case["vocab"]]
        at = batch.LogitsRegions(controls=controls[0], history=history[0], history_stride=history[1], bias=bias[0],
                                 bias_stride=bias[1], mask=mask[0], mask_stride=mask[1])
        kernels = batch.LogitsKernels(ctx, arena)
        body = lambda r: kernels.adjust(r, at, x, y, case["vocab"], rows)  # noqa: E731
    else:
        n_head = case["n_kv"] * case["rep"]
        c = E.Config(n_embd=256, n_head=n_head, n_head_kv=case["n_kv"], head_dim=HEAD, eps=EPS, rope_theta=THETA)
        paged = batch.Paged(E.KvPrecision[case["kv"].upper()], case["page"], st.n_pages, st.n_seq, st.table.shape[1],
                            case["n_kv"] * HEAD)
        pool = _pool(ctx, held, st, paged)
        words = a.put(_words(st.seq, st.len, st.share, torch.zeros_like(st.seq)).view(-1))
        table = a.room(st.table.numel())
        q = a.put(st.q)
        if case["op"] == "append":
            k, v = a.put(st.k), a.put(st.v)
            norms = [a.put(t)[0] for t in (st.q_norm, st.k_norm, st.freq)]
            parts, splits = 0, (0, 0)
        else:
            splits = batch.splits(rows, case["n_kv"], case["rep"], st.shared, st.own_max)
            parts = a.room(batch.part_size(rows, n_head, splits))
        out = a.room(q[1] * rows), q[1]
        arena, flat = a.place(ctx, held)
        flat[table: table + st.table.numel()].view(torch.int32).copy_(st.table.view(-1))
        _control(flat, rows, st.shared, st.leader)
        st.out = flat[out[0]: out[0] + out[1] * rows].view(rows, out[1])[:, : n_head * HEAD]
        st.out.zero_()
        at = batch.BatchRegions(rows=words[0], table=table, part=parts)
        kernels = batch.BatchKernels(ctx, arena, arena, [pool], c, paged)
        if case["op"] == "append":
            body = lambda r: kernels.append(r, 0, at, q, k, v[0], out, *norms, rows)  # noqa: E731
        else:
            body = lambda r: kernels.attend(r, 0, at, q, out, rows, splits)  # noqa: E731
    torch.cuda.synchronize()
    held.recording = ctx.record(False, body)
    # the arena's copies are the inputs now
    for name in ("logits", "history", "mask", "bias", "bias_id", "q", "k", "v", "table"):
        st.__dict__.pop(name, None)
    st.held = held
    st.call = lambda: ctx.replay(held.recording)


# ---- what a pass cannot do without ------------------------------------------------------------
def _entry_bytes(case):
    """Bytes of one position's keys and values."""
    dim = case["n_kv"] * HEAD
    return sum(dim + dim // 16 if q8 else 2 * dim for q8 in _bits(case))


def work(case):
    rows = case["rows"]
    if case["op"] == "logits":
        v = case["vocab"]
        masks = rows * v / 16 if case["masked"] else 0
        return {"bytes": rows * (8 * v + 3 * case["history"] + 6 * case["biases"] + 32) + masks, "flops": 0}
    heads = case["n_kv"] * case["rep"]
    if case["op"] == "append":
        return {"bytes": rows * (4 * HEAD * (2 * heads + 2 * case["n_kv"]) + _entry_bytes(case) + 20),
                "flops": rows * HEAD * (heads + case["n_kv"]) * 8.0}
    if case["chunk"]:
        distinct, pairs = case["shared"] + rows, rows * (rows + 1) / 2
    else:
        each = (case["own"] + 1) / 2 if rows > 1 else case["own"]
        distinct = case["shared"] * (2 if case["mix"] else 1) + rows * each
        pairs = rows * each
    pairs += rows * case["shared"]
    return {"bytes": distinct * _entry_bytes(case) + rows * heads * HEAD * 8, "flops": 4.0 * HEAD * heads * pairs}


# ---- the same in 64 bits ----------------------------------------------------------------------
def _exact_append(case, st):
    k8, v8 = _bits(case)
    pos = (st.len.double() - 1).clamp(min=0)
    angle = pos[:, None] * st.freq.double()[None, :]
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
    p = pos.long()
    slot = st.table[st.seq.long(), p // page].long() * page + p % page
    for name, rows, q8 in (("keys", rotated(st.k, st.k_norm), k8), ("values", st.v.double(), v8)):
        pool = torch.zeros(n, case["n_kv"] * HEAD, dtype=torch.float64, device="cuda")
        pool[slot[live]] = rows[live]
        out[name] = None if q8 else pool  # what 8 bits hold is their rounding's choice
    return out


def _exact_attend(case, st):
    n_kv, rep, page = case["n_kv"], case["rep"], case["page"]
    out = torch.zeros(case["rows"], n_kv * rep, HEAD, dtype=torch.float64, device="cuda")

    def read(pool, scales, slot):
        x = pool[slot].double()
        if scales is not None:
            x = x * scales[slot].double().repeat_interleave(32, 1)
        return x.view(-1, n_kv, HEAD).transpose(0, 1)

    for r in range(case["rows"]):
        n = int(st.len[r])
        if n == 0:
            continue
        pos = torch.arange(n, device="cuda")
        slot = st.table[int(st.seq[r]), pos // page].long() * page + pos % page
        if case["chunk"] and r:
            K, V = last
            K, V = K[:, :n], V[:, :n]
        elif case["chunk"]:
            pos = torch.arange(int(st.len[-1]), device="cuda")
            slot = st.table[0, pos // page].long() * page + pos % page
            last = read(st.keys, st.key_scales, slot), read(st.values, st.value_scales, slot)
            K, V = last[0][:, :n], last[1][:, :n]
        else:
            K, V = read(st.keys, st.key_scales, slot), read(st.values, st.value_scales, slot)
        q = st.q[r].double().view(n_kv, rep, HEAD)
        w = torch.softmax(torch.matmul(q, K.transpose(1, 2).contiguous()) / math.sqrt(HEAD), -1)
        out[r] = torch.matmul(w, V).reshape(n_kv * rep, HEAD)
    return out.view(case["rows"], -1)


def _exact_logits(case, st):
    out = st.logits.double()
    for r in range(case["rows"]):
        n, p = int(st.history_len[r]), int(st.prompt_len[r])
        ids = st.history[r].long()
        seen = torch.bincount(ids[:n], minlength=case["vocab"]) > 0
        made = torch.bincount(ids[p:n], minlength=case["vocab"])
        rho, f, g = float(st.repetition[r]), float(st.frequency[r]), float(st.presence[r])
        row = out[r]
        row[seen & (row > 0)] /= rho
        row[seen & (st.logits[r] <= 0)] *= rho
        row -= f * made + g * (made > 0)
        k = int(st.bias_len[r])
        row[st.bias_id[r, :k].long()] += st.bias[r, :k].double()
        if int(st.masked[r]):
            bits = np.unpackbits(st.mask[r].cpu().numpy().view(np.uint8), bitorder="little")[: case["vocab"]]
            row[torch.from_numpy(bits == 0).cuda()] = -math.inf
    return out


def exact(case, seed):
    st, src = State(), Source(seed)
    st.case = case
    if case["op"] == "append":
        _prepare_append(case, src, st)
        return _exact_append(case, st)
    if case["op"] == "attend":
        _prepare_attend(case, src, st)
        return _exact_attend(case, st)
    _prepare_logits(case, src, st)
    return _exact_logits(case, st)
