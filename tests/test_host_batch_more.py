"""CPU tests of the host side of kv_append_axes, attention_paged_shaped and logits_sample: what the
runtime refuses, the launches it makes, and what BatchEngine puts into the device's buffers for them."""
import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip import engine as E
from test_host_batch import A, KV_DIM, POOL, SLOTS, W, _append, _attend, _refuse, host  # noqa: F401
from test_host_batch_engine import _Context, make  # noqa: F401
from test_host_batch_launch import shape  # noqa: F401


def _axes(axes=21000, n_axes=3, **over):
    return _append(**over) + [axes, n_axes]


def _bits(v):
    return int(np.float32(v).view(np.uint32))


def _shaped(spans=21000, slopes=0xFFFFFFFF, window=0, lead=1, cap=0.0, **over):
    return _attend(**over) + [spans, slopes, window, lead, _bits(cap)]


def _merge(spans=21000, window=0, lead=1, rep=2, **over):
    w = dict(part=8192, o=4096, os=512, n_head=4, n_shared=1, n_own=2, rows=20000, ts=4, n_seq=3, log2=5)
    return list((w | over).values()) + [spans, window, lead, rep]


def test_axes_words(host):  # noqa: F811
    ok = lambda rows=4, **k: _refuse(host, "kv_append_axes", [0, 1, 128], _axes(**k), rows, [W, A, A, POOL, POOL])  # noqa: E731
    assert ok() == "" and ok(rows=0) == "" and ok(n_axes=1) == "" and ok(n_axes=4) == ""
    for bad in (dict(n_axes=0), dict(n_axes=5), dict(n_axes=2**31), dict(axes=21001), dict(axes=A // 4 - 12), dict(axes=2**32 - 4),
                dict(axes=8192), dict(rope=W // 4 - 191), dict(q_off=A // 4 - 100), dict(n_pages=9), dict(o_off=512)):
        assert ok(**bad), bad
    # (one axis needs 64 frequencies, kv_append's)
    assert ok(n_axes=1, rope=W // 4 - 64) == "" and ok(n_axes=3, rope=W // 4 - 192) == ""


def test_shaped_words(host):  # noqa: F811
    def ok(rows=4, **k):
        return _refuse(host, "attention_paged_shaped", [2, 0, 1, 128], _shaped(**k), rows, [A, A, POOL, POOL, POOL])
    assert ok() == "" and ok(lead=0) == "" and ok(slopes=21100) == "" and ok(cap=30.0) == "" and ok(window=2**32 - 1) == ""
    assert ok(cap=2.0**-10) == "" and ok(cap=2.0**14) == "" and ok(cap=-0.0) == ""
    for bad in (dict(spans=21001), dict(spans=A // 4 - 6), dict(spans=4096), dict(spans=8192), dict(slopes=A // 4 - 3),
                dict(slopes=8192), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(cap=2.0**-11),
                dict(cap=2.0**15), dict(lead=1022), dict(lead=2**32 - 1), dict(n_own=0), dict(wide=2), dict(part=A // 4 - 100),
                dict(lead=200)):
        assert ok(**bad), bad
    # a lead's parts count among the partials
    assert ok(lead=1, part=A // 4 - 4 * 4 * 4 * 130) == "" and ok(lead=2, part=A // 4 - 4 * 4 * 4 * 130)


def test_shaped_merge_words(host):  # noqa: F811
    ok = lambda rows=4, **k: _refuse(host, "attention_paged_shaped_merge", [128], _merge(**k), rows, [A, A])  # noqa: E731
    assert ok() == "" and ok(lead=0) == "" and ok(rep=4) == ""
    for bad in (dict(rep=0), dict(rep=3), dict(rep=16), dict(rep=8), dict(spans=21001), dict(spans=A // 4 - 6), dict(spans=4096),
                dict(lead=2**32 - 3), dict(lead=1022), dict(n_shared=0, n_own=1, lead=0), dict(part=A // 4 - 100)):
        assert ok(**bad), bad


def test_sample_words(host):  # noqa: F811
    n = 8 << 20

    def ok(name="logits_sample_draw", rows=4, **k):
        w = dict(x=64, xs=20000, v=20000, ctrl=90000, part=100000, out=95000) | k
        w = list(w.values())
        return _refuse(host, name, [0], w if name.endswith("draw") else w[:5], rows, [n, n])
    for name in ("logits_sample", "logits_sample_draw"):
        assert ok(name) == "" and ok(name, rows=0) == "" and ok(name, v=1) == ""
        for bad in (dict(v=0), dict(v=(1 << 20) + 1), dict(x=66), dict(xs=19996), dict(x=n // 4 - 100), dict(ctrl=90002),
                    dict(ctrl=n // 4 - 4), dict(part=100002), dict(part=n // 4 - 12 * 5128 + 4)):
            assert ok(name, **bad), (name, bad)
        assert ok(name, part=n // 4 - 12 * 5128) == ""
    for bad in (dict(out=64), dict(out=90000), dict(out=100000), dict(out=n // 4 - 12), dict(out=95001)):
        assert ok(**bad), bad
    assert ok("logits_sample", part=64) and ok("logits_sample", part=90000 - 100)


@pytest.mark.parametrize("n_kv,rep", [(1, 1), (8, 4), (4, 8), (3, 2), (8, 1)])
@pytest.mark.parametrize("n_shared,n_own,lead", [(0, 1, 0), (1, 1, 2), (5, 3, 1), (8, 2, 0)])
def test_shaped_launch(shape, n_kv, rep, n_shared, n_own, lead):  # noqa: F811
    """attention_paged's workgroups, and of the rows' own parts whole tiles of the rows that may go together."""
    for rows in (1, 2, 15, 16, 17, 128, 129):
        for wide in (0, 1):
            for cap in (0.0, 30.0):
                words = _shaped(n_kv=n_kv, n_shared=n_shared, n_own=n_own, wide=wide, lead=lead, cap=cap)
                g, threads, form, extra = shape("attention_paged_shaped", [rep, 0, 1, 128], words, rows)
                plain = shape("attention_paged", [rep, 0, 1, 128], words[:20], rows)[0][0] - rows * n_kv * n_own
                T = 16 // rep
                padded = -(-rows // T) * T
                assert g == [plain + padded * n_kv * (n_own + lead), 1, 1] and threads == 256 and extra == [rows]
                assert form == (cap > 0)
                # the kernel's map of these: every row once, the first of each T before the others
                tiles = padded // T
                at = np.arange(padded) % tiles * T + np.arange(padded) // tiles
                assert sorted(at) == list(range(padded)) and (at[:tiles] % T == 0).all()


def test_the_other_launches(shape):  # noqa: F811
    for rows in (1, 128, 1365, 1366):
        assert (shape("kv_append_axes", [0, 1, 128], _axes(n_head=32, n_kv=8), rows)
                == shape("kv_append", [0, 1, 128], _append(n_head=32, n_kv=8), rows))
    for lead in (0, 1, 15):
        g, threads, form, extra = shape("attention_paged_shaped_merge", [128], _merge(n_head=32, lead=lead), 4)
        assert form == (3 + lead > 16) and g == [32 if form else 8, 4, 1] and threads == (512 if form else 256)
    for v in (1, 8192, 8193, 151936):
        g, threads, form, extra = shape("logits_sample", [0], [64, 200000, v, 0, 0], 7)
        assert (g, threads, form, extra) == ([-(-v // 8192), 7, 1], 512, 0, [])
        assert shape("logits_sample_draw", [0], [64, 200000, v, 0, 0, 0], 7)[:2] == ([1, 7, 1], 1024)


def test_shaped_parts():
    for rows in (1, 7, 128):
        for shared, own, lead in ((0, 1, 0), (4000, 128, 0), (4000, 128, 300), (0, 20000, 500), (100000, 1, 100000)):
            p = B.shaped_splits(rows, 8, 4, shared, own, lead)
            assert p[:3] == B.splits(rows, 8, 4, shared, own) and (p.lead > 0) == bool(lead and shared) and p.lead <= 128
            assert sum(p[:2]) + p.lead <= B.MAX_PARTS
    assert B.shaped_part_size(3, 8, (2, 5, False, 4)) == 3 * 8 * 11 * 130 and B.sample_size(3, 8193) == 6 * 5128


# ---- BatchEngine ----
def _seen(ctx):
    """The device's words at the last replay."""
    return ctx.eng.arena.buffer.device.view("<u4")


def test_spans_and_first_positions(make):  # noqa: F811
    eng, ctx = make()
    s = eng.open()
    eng.extend(s, range(100))
    eng.extend(s, range(50), since=70)
    u, at = _seen(ctx), eng.at
    assert list(u[2:7]) == [50, 100, s, 70, 150]
    assert u[at.spans: at.spans + 100].reshape(50, 2).tolist() == [[70, 0]] * 50
    eng.extend(s, range(30), since=150, together=True)
    assert list(u[2:7]) == [30, 150, s, 150, 180]
    assert u[at.spans: at.spans + 60].reshape(30, 2).tolist() == [[150, 180]] * 30
    for bad in (dict(since=-1), dict(since=181), dict(axes=np.zeros((1, 1), int)), dict(vectors=np.zeros((1, 3)))):
        with pytest.raises(ValueError):
            eng.extend(s, [1], **bad)
    with pytest.raises(ValueError):
        eng.extend(s, range(129), together=True)
    assert eng.length(s) == 180


def test_positions_of_axes(make, monkeypatch):  # noqa: F811
    eng, ctx = make()
    eng.n_axes = 3  # as a model with axes has them
    s = eng.open()
    turn = lambda n: _seen(ctx)[eng.at.axes: eng.at.axes + 4 * n].reshape(n, 4).tolist()  # noqa: E731
    eng.extend(s, range(5))
    assert turn(5) == [[i] * 4 for i in range(5)]
    eng.extend(s, [9] * 4, axes=[[5, 5, 5], [5, 5, 6], [5, 6, 5], [5, 6, 6]])
    assert turn(4) == [[5, 5, 5, 0], [5, 5, 6, 0], [5, 6, 5, 0], [5, 6, 6, 0]]
    eng.step({s: 1})
    assert turn(1) == [[7] * 4]  # text goes on behind the largest
    t = eng.fork(s)
    eng.extend(t, [1, 2])
    assert turn(2) == [[8] * 4, [9] * 4]
    eng.step({t: 1, s: 2})
    assert turn(2)[eng.sequences[t].row] == [10] * 4 and turn(2)[eng.sequences[s].row] == [8] * 4
    for bad in ([[1, 2]], [[-1, 0, 0]], [[0.5, 0, 0]], [[2**31, 0, 0]], [[0, 0, 0]] * 2):
        with pytest.raises(ValueError):
            eng.extend(s, [1], axes=bad)


def test_vectors(make):  # noqa: F811
    eng, ctx = make()
    s = eng.open()
    v = np.arange(3 * 256, dtype=np.float32).reshape(3, 256)
    eng.extend(s, [0] * 3, vectors=v)
    a = eng.arena
    f = ctx.eng.arena.buffer.device.view("<f4")
    assert (f[a.x: a.x + 3 * a.s_embd].reshape(3, a.s_embd)[:, :256] == v).all()
    assert eng.length(s) == 3 and {k[-1] for k in eng.recordings} == {True}
    eng.extend(s, [1])
    assert {k[-1] for k in eng.recordings} == {True, False}


def test_samplings_and_draws(make):  # noqa: F811
    eng, ctx = make()
    a, b = eng.open(), eng.open()
    eng.sampling(a, B.Sampling(0.5, 7, 0.9, 0.125))
    c = eng.fork(a)
    eng.sample({b: 1, a: 2, c: 3}, {a: 11, c: 2**32 - 1, b: 0})
    u = _seen(ctx)
    f, off = u.view("<f4"), eng.sample_at.controls
    for q, draw in ((a, 11), (b, 0), (c, 2**32 - 1)):
        o = off + 8 * eng.sequences[q].row
        k = B.Sampling() if q == b else B.Sampling(0.5, 7, np.float32(0.9), 0.125)
        assert (f[o], f[o + 1], f[o + 2], u[o + 3], u[o + 4]) == (k.temperature, np.float32(k.top_p), k.min_p, k.top_k, draw)
    before = eng.length(a)
    for bad in ({a: 1}, {a: 1, b: -1}, {a: 1, b: 2**32}, {a: 1, b: 2, c: 3}):
        with pytest.raises(ValueError):
            eng.sample({a: 1, b: 2}, bad)
    for bad in (B.Sampling(-1.0), B.Sampling(float("nan")), B.Sampling(float("inf")), B.Sampling(1.0, -1), B.Sampling(1.0, 2**32),
                B.Sampling(1.0, 0, 0.0), B.Sampling(1.0, 0, 1.5), B.Sampling(1.0, 0, 1.0, -0.1), B.Sampling(1.0, 0, 1.0, 2.0)):
        with pytest.raises(ValueError):
            eng.sampling(a, bad)
    assert eng.length(a) == before
    ctx.fails = "replay"
    with pytest.raises(RuntimeError):
        eng.sample({a: 1}, {a: 2})
    assert eng.length(a) == before


def test_drawn_rows_in_the_order_asked_for(make, monkeypatch):  # noqa: F811
    eng, ctx = make()
    seqs = [eng.open() for _ in range(4)]

    def answer(rec):
        u = eng.arena.buffer.device.view("<u4")
        for r in range(u[2]):  # each row's token, as drawn
            o = eng.sample_at.out + 4 * r
            u[o: o + 2] = u[eng.arena.tokens + r], r
            u.view("<f4")[o + 2] = -0.5 * r
    monkeypatch.setattr(ctx, "replay", answer)
    got = eng.sample({3: 30, 1: 10, 2: 20}, {1: 0, 2: 0, 3: 0})
    assert got.token.tolist() == [30, 10, 20] and seqs == [0, 1, 2, 3]
    rows = [eng.sequences[q].row for q in (3, 1, 2)]
    assert got.kept.tolist() == rows and got.logprob.tolist() == [-0.5 * r for r in rows]


def test_configs_that_no_kernel_serves():
    base = dict(n_embd=256, n_head=2, n_head_kv=1, n_vocab=1000, n_layer=2)
    for bad in (dict(axes=(0,) * 63), dict(axes=(4,) * 64), dict(axes=(-1,) * 64), dict(score_cap=-1.0), dict(score_cap=1e6),
                dict(score_cap=float("nan")), dict(windows=(1,)), dict(windows=(1, -1)), dict(slopes=(1.0,)),
                dict(slopes=(1.0, float("nan")))):
        with pytest.raises(ValueError):
            B.BatchEngine(_Context(), {}, E.Config(**(base | bad)), 64, 8)


def test_vocabularies_that_no_draw_takes(make, monkeypatch):  # noqa: F811
    """They are decoded as any other; only drawing is refused."""
    monkeypatch.setattr(B, "SAMPLE_VOCAB", 999)
    eng, _ = make()
    a = eng.open()
    eng.step({a: 900})
    with pytest.raises(ValueError):
        eng.sample({a: 1}, {a: 2})
    assert eng.length(a) == 1


def test_rope_axes_table():
    c = E.Config(n_embd=256, axes=tuple(i % 3 if i < 60 else 0 for i in range(64)))
    t = E.rope_axes_table(c)
    assert t.shape == (3, 64) and (t.sum(0) == E.rope_frequencies(c)).all() and ((t != 0).sum(0) == 1).all()
    assert (t[1, 1], t[2, 1]) == (E.rope_frequencies(c)[1], 0)


@pytest.mark.parametrize("rows,n_kv,own,more", [(8, 8, 512, 2), (8, 8, 513, 3), (5, 8, 320, 2), (5, 8, 321, 2), (31, 8, 1984, 3),
                                                (31, 8, 1985, 3), (32, 8, 1985, 2), (32, 8, 100000, 2), (255, 1, 2041, 3),
                                                (256, 1, 2041, 2)])
def test_one_part_of_rows_that_share_nothing(rows, n_kv, own, more):
    """Where splits has `more`, one from 256 rows x key heads on, and below for 8 positions for each of these; with a
    shared run always splits'."""
    assert B.splits(rows, n_kv, 4, 0, own) == (0, more, False)
    one = rows * n_kv >= 256 or own <= 8 * rows * n_kv
    assert B.shaped_splits(rows, n_kv, 4, 0, own) == (0, 1 if one else more, False, 0)
    assert B.shaped_splits(rows, n_kv, 4, 1000, own)[:3] == B.splits(rows, n_kv, 4, 1000, own)


def test_draws_take_the_attentions_partials(make, monkeypatch):  # noqa: F811
    """An engine's arena holds what is larger of the two, not both."""
    eng, _ = make()
    x, sample = eng.arena.extra, B.sample_size(eng.max_seq, eng.c.n_vocab)
    part = max(B.shaped_part_size(r, eng.c.n_head, p) for r in eng._buckets(E.BATCH)
               for shared in [0, *eng._buckets(eng.max_ctx)] for own in eng._buckets(eng.max_ctx)
               for lead in (False, True) for _, p in eng._shaped_parts(r, shared, own, lead))
    assert eng.sample_at.part == eng.at.part == x["part"]
    assert x["logits"] - x["part"] == -(-max(part, sample) // 64) * 64
    monkeypatch.setattr(B, "SAMPLE_VOCAB", eng.c.n_vocab - 1)
    plain, _ = make()
    assert plain.arena.extra["logits"] - plain.arena.extra["part"] == -(-part // 64) * 64
    assert eng.arena.size - plain.arena.size == max(0, -(-sample // 64) * 64 - -(-part // 64) * 64)
