"""The served batch's newer operators (kernels/batch.hip, kernels/sample.hip) by every way there is to run
them: as a recording's launches, as its graph while what it reads changes, and one dispatch at a time."""
import threading

import numpy as np
import pytest

from skyla_hip.abi import Context, SkylaHipError
from test_gpu_batch import P, _Direct
from test_gpu_batch_axes import Axes
from test_gpu_batch_shaped import Shaped
from test_gpu_sample import Rows, _some

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reps", [0, 3])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_shaped_dispatches(ctx, reps, cap):
    lens = [400, 333, 256, 257]
    b = Shaped(ctx, P["f16k_q8v"], 2, 4, 32, lens, cap=cap, window=300, shares=[256] * 4, shared=256, parts=(2, 1, True, 1))
    try:
        b.prepare()
        b.check()
        want = b.rows_of(b.out, b.sq, b.sq, b.grid).copy()
        b.rows_of(b.out, b.sq, b.sq, b.grid)[:] = 7.5
        b.arena.upload()
        step = lambda at: b.kernels.attend_shaped(_Direct(ctx, reps), 0, at, (b.q, b.sq), (b.out, b.sq), b.grid,  # noqa: E731
                                                  b.shaped_parts, b.shape)
        step(b.at)
        b.arena.download()
        assert np.array_equal(b.rows_of(b.out, b.sq, b.sq, b.grid), want)
        b.at.spans = b.arena.size // 4
        with pytest.raises(SkylaHipError) as e:
            step(b.at)
        assert e.value.code == -1
    finally:
        b.free()


@pytest.mark.parametrize("reps", [0, 3])
def test_axes_dispatches(ctx, reps):
    b = Axes(ctx, P["q8"], 2, 4, 16, [40, 33, 1, 70])
    try:
        f = b.arena.as_f32()
        start, pool = f.copy(), b.pool.host().copy()
        b.check()
        want, stored = b.rows_of(b.out, b.sq, b.sq, b.grid).copy(), b.pool.host().copy()
        f[:], b.pool.host()[:] = start, pool
        b.arena.upload()
        b.pool.upload()
        qn, kn, rope = b.norms
        step = lambda n: b.kernels.append_axes(_Direct(ctx, reps), 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v,  # noqa: E731
                                               (b.out, b.sq), qn, kn, rope, n, b.grid)
        step(b.n_axes)
        b.arena.download()
        b.pool.download()
        assert np.array_equal(b.rows_of(b.out, b.sq, b.sq, b.grid), want) and np.array_equal(b.pool.host(), stored)
        with pytest.raises(SkylaHipError) as e:
            step(5)
        assert e.value.code == -1
    finally:
        b.free()


@pytest.mark.parametrize("reps", [0, 3])
def test_sample_dispatches(ctx, reps):
    g = np.random.default_rng(3)
    rows = Rows(ctx, (g.standard_normal((8, 20000)) * 2).astype(np.float32), _some(g, 8), grid=9)
    try:
        rows.check()
        want = rows.arena.as_u32()[rows.at.out: rows.at.out + 36].copy()
        rows.arena.as_f32()[rows.at.out: rows.at.out + 36] = 7.5
        rows.arena.upload()
        rows.kernels.sample(_Direct(ctx, reps), rows.at, (rows.xo, rows.stride), rows.v, rows.grid)
        rows.arena.download(rows.at.out * 4, 36 * 4)
        assert np.array_equal(rows.arena.as_u32()[rows.at.out: rows.at.out + 36], want)
    finally:
        rows.free()


def test_sample_as_a_graph(ctx):
    """Rows, logits, settings and draws change from replay to replay, with other work between; a recording of more
    than one draw, its partials one region."""
    g = np.random.default_rng(4)
    rows = Rows(ctx, (g.standard_normal((6, 30000)) * 2).astype(np.float32), _some(g, 6))
    try:
        def record(times):
            def body(r):
                for i in range(times):
                    if i:
                        r.barrier()
                    rows.kernels.sample(r, rows.at, (rows.xo, rows.stride), rows.v, rows.grid)
            return ctx.record(False, body)
        one, many = record(1), record(5)
        try:
            f, u = rows.arena.as_f32(), rows.arena.as_u32()
            direct, kept = rows.rec, []
            for step in range(6):
                rows.x = (g.standard_normal((6, 30000)) * (0.5 + step)).astype(np.float32)
                rows.settings = _some(g, 6 + step)[step:]
                for r, (T, p, m, k, d) in enumerate(rows.settings):
                    o = rows.at.controls + 8 * r
                    f[o: o + 3] = T, p, m
                    u[o + 3: o + 5] = k, d
                    f[rows.xo + r * rows.stride:][: rows.v] = rows.x[r]
                f[rows.at.out: rows.at.out + 24] = 7.5
                rows.arena.upload()
                ctx.replay_timed(one) if step % 2 else ctx.replay(many)
                rows.arena.download(rows.at.out * 4, 24 * 4)
                kept.append(u[rows.at.out: rows.at.out + 24].copy())
                rows.rec = direct
                rows.check()  # against the oracle, by launches
                assert np.array_equal(u[rows.at.out: rows.at.out + 24], kept[-1]), step
        finally:
            one.free()
            many.free()
    finally:
        rows.free()


def test_two_contexts_at_once(ctx):
    """A draw and an attention on streams of their own, from two threads: each as alone."""
    g = np.random.default_rng(6)
    other = Context.new(0)
    rows = Rows(ctx, (g.standard_normal((40, 50000)) * 2).astype(np.float32), _some(g, 40))
    b = Shaped(other, P["f16"], 2, 4, 32, [400, 333, 256, 257], cap=30.0, window=300, shares=[256] * 4, shared=256)
    try:
        b.prepare()
        b.check()
        alone, failed = b.rows_of(b.out, b.sq, b.sq, b.grid).copy(), []

        def attend():
            try:
                for _ in range(20):
                    b.attend()
                    assert np.array_equal(b.rows_of(b.out, b.sq, b.sq, b.grid), alone)
            except BaseException as e:  # (a thread's own goes nowhere)
                failed.append(e)
        t = threading.Thread(target=attend)
        t.start()
        try:
            rows.check(times=10)
        finally:
            t.join()
        assert not failed, failed
    finally:
        b.free()
        rows.free()
        other.free()
