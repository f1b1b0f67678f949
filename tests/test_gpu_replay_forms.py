"""Recordings of a few launches replay as those launches or as one HIP graph (tactic nograph): the
same bits whichever, replay after replay, with other work on the buffers between."""
import numpy as np
import pytest

from helpers import Setup, tactics
from skyla_hip import engine as E
from skyla_hip import synth
from test_gpu_moe import CFG, N_EMBD, MoeSetup

pytestmark = pytest.mark.gpu

FORMS = (None, "0", "1")  # the default (at most six launches: directly), a graph, directly


def _same(ctx, body, load, read, launches):
    """What `read` gives after each replay of body's recording in every form, and after timed ones."""
    outs = []
    for form in FORMS:
        with tactics(nograph=form):
            rec = ctx.record(False, body)
        try:
            assert rec.launches() == launches
            for timed in (False, False, True, True, False):
                load()
                if timed:
                    assert ctx.replay_timed(rec) > 0
                else:
                    ctx.replay(rec)
                outs.append(read())
        finally:
            rec.free()
    assert np.isfinite(outs[0]).all() and outs[0].any()
    assert all(np.array_equal(o.view(np.uint32), outs[0].view(np.uint32)) for o in outs[1:])


@pytest.mark.parametrize("dtype", [E.DType.Q4K, E.DType.Q6K, E.DType.Q8_0])
@pytest.mark.parametrize("accum", [False, True])
def test_matvecs(ctx, dtype, accum):
    """Three matrices in one fused launch, then one that reads its rows (two launches)."""
    n_in, outs = 1024, [512, 256, 256]
    mats = [(dtype, n_in, n, synth.matrix("replay-forms", f"{dtype.name}-{i}", dtype, n_in, n)) for i, n in enumerate(outs)]
    mats.append((dtype, 512, 96, synth.matrix("replay-forms", f"{dtype.name}-o", dtype, 512, 96)))
    s = Setup(ctx, mats, n_in, 512, rows=4)
    x = synth.activations("replay-forms", "x", n_in)
    y0 = synth.activations("replay-forms", "y", (4, 512))

    def body(r):
        g = E.Graph(r, s.k, None, None, False)
        for i in range(3):
            g.matvec(s.q[i], (s.x_off, 0), (s.y_off + i * s.s_out, 0), accum, False)
        r.barrier()
        g.matvec(s.q[3], (s.y_off, 0), (s.y_off + 3 * s.s_out, 0), accum, False)

    def load():
        s.set_x(x)
        s.set_y(y0)
    try:
        _same(ctx, body, load, lambda: s.y(4, 512), 2)
    finally:
        s.free()


@pytest.mark.parametrize("dtype,n_in", [(E.DType.Q4K, 4096), (E.DType.Q6K, 2048), (E.DType.Q8_0, 2048)])
def test_matmul_of_few_tiles(ctx, dtype, n_in):
    """A batched product that is split along K: its counters are left at zero by every launch."""
    n_out, n_tok = 384, 100
    s = Setup(ctx, [(dtype, n_in, n_out, synth.matrix("replay-forms", f"mm-{dtype.name}", dtype, n_in, n_out))], n_in, n_out,
              rows=n_tok)
    x = synth.activations("replay-forms", f"mm-x-{n_in}", (n_tok, n_in))

    def body(r):
        g = E.Graph(r, s.k, None, None, True)
        g.matvec(s.q[0], (s.x_off, s.s_in), (s.y_off, s.s_out), False, True, groups_z=-(-n_tok // E.MATMUL_TILE_COLS))

    def load():
        s.set_x(x)
        s.set_y(np.zeros((n_tok, n_out), np.float32))
    try:
        rec = ctx.record(False, body)
        launches = rec.launches()
        rec.free()
        assert launches <= 6
        _same(ctx, body, load, lambda: s.y(n_tok, n_out), launches)
    finally:
        s.free()


@pytest.mark.parametrize("forms,launches", [("0", 6), ("26", 3)])
def test_experts(ctx, forms, launches):
    """A MoE decode layer in six launches and in three."""
    m = MoeSetup(ctx)
    n, x0 = synth.activations(CFG, "replay-n", (1, N_EMBD)), synth.activations(CFG, "replay-x", (1, N_EMBD))

    def body(r):
        E.Graph(r, m.k, m.a, m.c, False).moe(m.qg, m.qu, m.qd, m.router_off)

    def read():
        m.a.buffer.download()
        return m.rows(m.a.x, m.a.s_embd, 1, N_EMBD)[0].copy()
    try:
        with tactics(moe_fuse=forms):
            _same(ctx, body, lambda: m.load(n, x0), read, launches)
    finally:
        m.free()
