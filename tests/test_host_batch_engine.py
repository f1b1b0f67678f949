"""CPU tests of BatchEngine's host side: what lies in the device's buffers when a step is replayed,
with a context that keeps them in memory and computes nothing."""
import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip import engine as E


class _Buffer:
    """A buffer whose device side is an array of its own, reached by upload and download alone."""

    def __init__(self, size):
        self.freed = 0
        self.size, self.mirror, self.device = size, np.zeros(size, np.uint8), np.zeros(size, np.uint8)

    def host(self):
        return self.mirror

    def as_f32(self):
        return self.mirror.view("<f4")

    def as_u32(self):
        return self.mirror.view("<u4")

    def upload(self, off=0, length=None):
        end = self.size if length is None else off + length
        self.device[off:end] = self.mirror[off:end]

    def download(self, off=0, length=None):
        end = self.size if length is None else off + length
        self.mirror[off:end] = self.device[off:end]

    def copy_from(self, dst, src, at, length):
        self.device[dst: dst + length] = src.device[at: at + length]

    def free(self):
        self.freed += 1


class _Context:
    def __init__(self):
        self.fails, self.steps, self.buffers, self.room = None, [], [], 100

    def alloc_host(self, size):
        if len(self.buffers) == self.room:
            raise MemoryError("alloc_host")
        self.buffers.append(_Buffer(size))
        return self.buffers[-1]

    def max_buffer(self):
        return 4 << 30

    def record(self, profile, body):
        if self.fails == "record":
            raise MemoryError("record")
        return object()

    def replay(self, rec):
        if self.fails == "replay":
            raise RuntimeError("replay")
        self.steps.append(self.eng.seen())


class _Weights:
    buffers, embd, layers, output, out_norm, rope = [_Buffer(64)], type("T", (), {"dtype": E.DType.Q8_0})(), [], None, 0, 0


class _Kernels:
    check = staticmethod(B.BatchKernels.check)

    def __init__(self, *a, **k):
        pass

    def free(self):
        pass


@pytest.fixture
def make(monkeypatch):
    """engine(...): a BatchEngine over such a context; its device's rows at each replay are in ctx.steps."""
    monkeypatch.setattr(E, "load_weights", lambda *a: _Weights())
    for where, name in ((E, "Kernels"), (B, "BatchKernels"), (B, "LogitsKernels")):
        monkeypatch.setattr(where, name, _Kernels)

    class Engine(B.BatchEngine):
        def seen(self):
            """The live rows as the device has them: words, token, controls, history, biases, mask."""
            u = self.arena.buffer.device.view("<u4").copy()
            f, at, rows = u.view("<f4"), self.logits_at, []
            for r in range(u[2]):
                k = at.controls + 8 * r
                h, b, m = (o + r * n for o, n in ((at.history, at.history_stride), (at.bias, at.bias_stride),
                                                  (at.mask, at.mask_stride)))
                bits = np.unpackbits(u[m: m + at.mask_stride].view(np.uint8), bitorder="little")[: self.c.n_vocab]
                seq, n = (int(x) for x in u[self.at.rows + 4 * r:][:2])
                table = u[self.at.table + seq * self.paged.seq_pages:][: -(-n // self.paged.page)]
                rows.append(dict(
                    seq=seq, len=n, share=int(u[self.at.rows + 4 * r + 2]), token=int(u[self.arena.tokens + r]),
                    prompt=int(u[k + 1]), history=u[h: h + u[k]].tolist(), pages=table.tolist(),
                    bias=dict(zip(u[b: b + 2 * u[k + 2]: 2].tolist(), f[b + 1: b + 1 + 2 * u[k + 2]: 2].tolist())),
                    allowed=bits.astype(bool) if u[k + 3] else None, penalties=f[k + 4: k + 7].tolist()))
                if r < self.max_seq:  # the device's answer: the row's token in every logit
                    self.arena.buffer.device.view("<f4")[self.arena.extra["logits"] + r * self.s_vocab:][: self.c.n_vocab] = (
                        rows[-1]["token"])
            return rows

    def engine(ctx=None, **over):
        ctx = ctx or _Context()
        c = E.Config(n_embd=256, n_ff=256, n_head=2, n_head_kv=1, head_dim=128, n_vocab=1000, n_layer=2)
        eng = ctx.eng = Engine(ctx, {}, c, **(dict(max_ctx=300, n_pages=40, page=16, max_seq=6) | over))
        return eng, ctx
    return engine


def _row(ctx, seq):
    rows = [r for r in ctx.steps[-1] if r["len"] and r["seq"] == seq]
    assert len(rows) == 1
    return rows[0]


def test_generated_tokens_stay_generated(make):
    """A conversation: prompts and answers in turns.  The frequency and presence penalties count every
    answer's tokens, none of the prompts'."""
    eng, ctx = make()
    a = eng.open()
    eng.control(a, B.Controls(frequency=0.5))
    eng.extend(a, [1, 2, 3])
    eng.step({a: 4}, prompt=[a])
    for t in (10, 11, 10):
        eng.step({a: t})
    eng.extend(a, [])
    eng.step({a: 12})
    r = _row(ctx, a)
    assert (r["len"], r["prompt"], r["history"]) == (8, 4, [1, 2, 3, 4, 10, 11, 10, 12])
    eng.extend(a, range(20, 29))
    eng.step({a: 30}, prompt=[a])
    eng.step({a: 13})
    r = _row(ctx, a)
    assert r["len"] == eng.length(a) == 19 and r["prompt"] == 14
    assert r["history"] == [1, 2, 3, 4, *range(20, 29), 30, 10, 11, 10, 12, 13]
    # a fork goes on from there, and penalties set later find the whole history
    b = eng.fork(a)
    eng.control(a, B.Controls())
    eng.step({a: 14, b: 15})
    eng.step({a: 16})
    eng.control(a, B.Controls(presence=1.0))
    eng.step({a: 17, b: 18}, prompt=[b])
    assert _row(ctx, a)["history"] == [1, 2, 3, 4, *range(20, 29), 30, 10, 11, 10, 12, 13, 14, 16, 17]
    assert _row(ctx, b)["history"] == [1, 2, 3, 4, *range(20, 29), 30, 18, 10, 11, 10, 12, 13, 15]
    assert (_row(ctx, a)["prompt"], _row(ctx, b)["prompt"]) == (14, 15)


def test_controls_are_taken_as_they_are(make):
    """What the caller does to its Controls, or to what they hold, after control() acts on nothing; a
    fork's are its own."""
    eng, ctx = make()
    a = eng.open()
    allowed, bias = np.arange(1000) % 3 == 0, {5: 1.5, 7: -np.inf}
    k = B.Controls(repetition=1.25, bias=bias, allowed=allowed)
    eng.control(a, k)
    b = eng.fork(a)
    k.repetition, k.frequency, bias[9], allowed[:] = 3.0, 1.0, 2.0, False
    del bias[5]
    k.allowed = None
    eng.control(b, B.Controls(presence=0.5, bias={1: 1.0}))
    eng.step({a: 20, b: 21})
    for want, seq in ((([1.25, 0, 0], {5: 1.5, 7: -np.inf}, np.arange(1000) % 3 == 0, [20]), a),
                      (([1.0, 0, 0.5], {1: 1.0}, None, [21]), b)):
        r = _row(ctx, seq)
        assert (r["penalties"], r["bias"], r["history"]) == (want[0], want[1], want[3])
        assert np.array_equal(r["allowed"], want[2]) if want[2] is not None else r["allowed"] is None
    k = B.Controls()
    eng.control(a, k)
    k.repetition, k.bias[3] = 2.0, 1.0
    eng.step({a: 22})
    assert (_row(ctx, a)["penalties"], _row(ctx, a)["bias"]) == ([1, 0, 0], {})


@pytest.mark.parametrize("bad", [dict(repetition=1e-50), dict(repetition=1e39), dict(frequency=-1e39), dict(presence=1e300),
                                 dict(repetition=np.nan), dict(bias={-1: 0.0}), dict(allowed=True)])
def test_controls_beyond_32_bits_are_refused(make, bad):
    eng, ctx = make()
    a = eng.open()
    eng.control(a, B.Controls(repetition=1.5))
    with pytest.raises(ValueError):
        eng.control(a, B.Controls(**bad))
    eng.step({a: 1})
    assert _row(ctx, a)["penalties"] == [1.5, 0, 0]


@pytest.mark.parametrize("where", ["record", "replay"])
def test_a_step_that_fails_leaves_the_sequences_as_they_were(make, where):
    eng, ctx = make()
    a, b = eng.open(), eng.open()
    eng.control(a, B.Controls(frequency=1.0))
    eng.control(b, B.Controls(repetition=1.5))
    eng.extend(a, range(16))   # a page is full: the next token needs another
    eng.extend(b, [1, 2])
    eng.step({b: 3})
    kept = eng.recordings
    for prompt in ((), [b]):
        free, ctx.fails, eng.recordings = len(eng.free_pages), where, {}
        with pytest.raises((MemoryError, RuntimeError)):
            eng.step({a: 50, b: 51}, prompt=prompt)
        assert (eng.length(a), eng.length(b), len(eng.free_pages)) == (16, 3, free)
    with pytest.raises((MemoryError, RuntimeError)):
        eng.extend(a, range(100, 200))
    assert (eng.length(a), len(eng.free_pages)) == (16, free)
    ctx.fails, eng.recordings = None, kept
    eng.step({a: 60, b: 61})
    r, s = _row(ctx, a), _row(ctx, b)
    assert (r["len"], r["prompt"], r["history"]) == (17, 16, [*range(16), 60])
    assert (s["len"], s["prompt"], s["history"]) == (4, 2, [1, 2, 3, 61])
    eng.close(a)
    eng.close(b)
    assert len(eng.free_pages) == 40 and not eng.uses.any()


def test_prompt_may_be_any_iterable(make):
    eng, ctx = make()
    a = eng.open()
    eng.control(a, B.Controls(presence=1.0))
    eng.step({a: 1}, prompt=(q for q in [a]))
    eng.step({a: 2}, prompt=iter([a]))
    eng.step({a: 3})
    assert (_row(ctx, a)["prompt"], _row(ctx, a)["history"]) == (2, [1, 2, 3])
    with pytest.raises(ValueError):
        eng.step({a: 4}, prompt=(q for q in [a, 5]))
    assert eng.length(a) == 3


def test_a_step_has_a_row_for_each_of_its_sequences(make):
    """Whichever numbers the sequences have, a step's rows are theirs and no idle ones, with their own
    controls, histories and pages."""
    eng, ctx = make()
    g, told = np.random.default_rng(1), {}
    for q in range(6):
        assert eng.open() == q
        k = B.Controls(repetition=1 + q / 8, presence=q / 4, bias={q: 1.0 + q} if q % 2 else {},
                       allowed=np.arange(1000) % (q + 2) == 0 if q > 2 else None)
        eng.control(q, k)
        eng.extend(q, [100 + q] * (10 + q))
        told[q] = k, [100 + q] * (10 + q)
    eng.step({4: 9})
    assert len(ctx.steps[-1]) == 1 and _row(ctx, 4)["token"] == 9
    told[4][1].append(9)
    for step in range(40):
        seqs = [int(q) for q in g.permutation(6)[: g.integers(1, 7)]]
        if step == 20:  # a sequence goes, another comes in its place
            eng.close(3)
            assert eng.open() == 3
            told[3] = B.Controls(), []
        out = eng.step({q: 10 * step + q for q in seqs})
        assert out[:, 0].tolist() == [10 * step + q for q in seqs]  # each its own row's answer
        assert len(ctx.steps[-1]) == len(seqs)
        for q in seqs:
            k, history = told[q]
            history.append(10 * step + q)
            r = _row(ctx, q)
            assert (r["len"], r["token"], r["bias"], r["penalties"]) == (
                len(history), history[-1], k.bias, [k.repetition, k.frequency, k.presence])
            if k.counts:
                assert r["history"] == history
            assert r["pages"] == eng.sequences[q].pages
            assert np.array_equal(r["allowed"], k.allowed) if k.allowed is not None else r["allowed"] is None


@pytest.mark.parametrize("room", [0, 1, 2])
def test_an_engine_that_finds_no_room_gives_back_what_it_took(make, room):
    ctx = _Context()
    ctx.room = room
    with pytest.raises(MemoryError):
        make(ctx)
    assert len(ctx.buffers) == room and all(b.freed == 1 for b in ctx.buffers)
    ctx.room = 100
    eng, _ = make(ctx)
    eng.free()
    assert all(b.freed == 1 for b in ctx.buffers)


def test_a_fork_that_fails_gives_its_page_back(make, monkeypatch):
    eng, ctx = make()
    a = eng.open()
    eng.extend(a, range(20))
    with monkeypatch.context() as m:
        m.setattr(_Buffer, "copy_from", lambda *k: 1 / 0)
        with pytest.raises(ZeroDivisionError):
            eng.fork(a)
    assert len(eng.free_pages) == 38 and list(eng.sequences) == [a] and eng.uses.max() == 1
    eng.close(a)
    assert len(eng.free_pages) == 40


@pytest.mark.parametrize("n", range(9))
@pytest.mark.parametrize("what", ["step", "control"])
def test_uploads_that_fail_are_made_again(make, monkeypatch, n, what):
    """The n-th upload of a step fails (a table's, controls', a history's, the words'): the next step
    brings what did not reach the device."""
    eng, ctx = make()
    a, b = eng.open(), eng.open()
    allowed = np.arange(1000) % 2 == 0
    eng.extend(a, range(16))  # a page: the next token needs another
    if what == "control":
        eng.step({a: 30, b: 31})
        eng.extend(a, range(15))
    eng.control(a, B.Controls(bias={3: 1.0}, presence=1.0, allowed=allowed))
    up, calls, failed = _Buffer.upload, iter(range(100)), False
    with monkeypatch.context() as m:
        m.setattr(_Buffer, "upload", lambda s, *k: 1 / (next(calls) != n) and up(s, *k))
        try:
            eng.step({a: 40})
        except ZeroDivisionError:
            failed = True
    assert failed == (n < 8)
    eng.step({b: 51, a: 50})
    r = _row(ctx, a)
    assert r["pages"] == eng.sequences[a].pages and len(r["pages"]) == -(-r["len"] // 16)
    assert r["bias"] == {3: 1.0} and np.array_equal(r["allowed"], allowed)
    assert r["len"] == len(r["history"]) == eng.length(a) and r["history"][-1] == 50
    assert _row(ctx, b)["bias"] == {} and _row(ctx, b)["pages"] == eng.sequences[b].pages


def test_controls_of_every_step_leave_the_history_where_it_is(make):
    """A grammar's mask at each token: the mask and the token go to the device, not the history again."""
    eng, ctx = make()
    a = eng.open()
    eng.extend(a, range(200))
    for t in range(5):
        eng.control(a, B.Controls(repetition=1.5, allowed=np.arange(1000) % 7 == t))
        placed = eng.sequences[a].placed
        eng.step({a: 300 + t})
        r = _row(ctx, a)
        assert r["history"] == [*range(200), *range(300, 301 + t)] and np.flatnonzero(r["allowed"])[0] == t
        assert placed == (200 + t if t else 0)
