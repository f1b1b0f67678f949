"""kv_append_axes (kernels/batch.hip) against the same in 64 bits: rows turned by positions of several
axes, as an image's patches and a video's frames have them."""
import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip.abi import SkylaHipError
from test_gpu_batch import EPS, P, THETA, Batch

pytestmark = pytest.mark.gpu

# What is kept of a value: f32's rounding of a norm's sum of 128 squares and of eight products (16 2^-24 of the head's
# norm, 1e-6), of the sines 2^-23; an f16 entry half a step, 2^-11 of itself; an 8-bit one half a step of its block.
F32 = 1.5e-6
F16 = 2.0**-11


class Axes(Batch):
    def __init__(self, ctx, *args, n_axes=3, far=1000, **more):
        super().__init__(ctx, *args, **more)
        self.n_axes = n_axes
        old, size = self.arena, self.arena.size // 4
        self.arena = ctx.alloc_host((size + 4 * self.grid + 256) * 4)
        f, u = self.arena.as_f32(), self.arena.as_u32()
        u[:size] = old.as_u32()
        self.kernels.free()
        old.free()
        self.kernels = B.BatchKernels(ctx, self.arena, self.arena, [self.pool], self.c, self.paged)
        self.at.axes, rope = size, size + 4 * self.grid
        self.norms = (*self.norms[:2], rope)
        freq = np.float32(THETA ** (-2.0 * np.arange(64) / 128))
        axis = np.arange(64) % n_axes
        self.freq = np.where(axis == np.arange(n_axes)[:, None], freq, np.float32(0))
        f[rope: rope + 256] = np.nan
        f[rope: rope + 64 * n_axes] = self.freq.ravel()
        self.pos = self.g.integers(0, far, (self.rows, 4))
        u[self.at.axes: self.at.axes + 4 * self.grid] = 0xFFFFFFFF
        u[self.at.axes: self.at.axes + 4 * self.rows] = self.pos.ravel()
        for off in self.norms[:2]:
            f[off: off + 128] = self.g.uniform(0.5, 1.5, 128)
        for off, s, w in ((self.q, self.sq, self.n_head * 128), (self.k, self.skv, self.dim), (self.v, self.skv, self.dim)):
            self.rows_of(off, s, w)[:] = self.g.standard_normal((self.rows, w))

    def append(self):
        qn, kn, rope = self.norms
        self.run(lambda r: self.kernels.append_axes(r, 0, self.at, (self.q, self.sq), (self.k, self.skv), self.v,
                                                    (self.out, self.sq), qn, kn, rope, self.n_axes, self.grid))

    def turned(self, x, norm):
        w = self.arena.as_f32()[norm: norm + 128].astype(np.float64)
        x = x.astype(np.float64).reshape(self.rows, -1, 128)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
        angle = (self.pos[:, : self.n_axes, None] * self.freq.astype(np.float64)).sum(1)[:, None]
        c, s, a, b = np.cos(angle), np.sin(angle), x[..., :64], x[..., 64:]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)

    def check(self):
        q = self.turned(self.rows_of(self.q, self.sq, self.n_head * 128), self.norms[0])
        k = self.turned(self.rows_of(self.k, self.skv, self.dim), self.norms[1])
        v = self.rows_of(self.v, self.skv, self.dim).astype(np.float64).reshape(self.rows, -1, 128)
        before = [(e.copy(), None if s is None else s.copy()) for e, s in self.halves()]
        self.append()
        out = self.rows_of(self.out, self.sq, self.n_head * 128).reshape(self.rows, -1, 128)
        touched = set()
        for r in range(self.rows):
            if self.lens[r] == 0:
                assert (out[r] == 7.5).all()
                continue
            assert (np.linalg.norm(out[r] - q[r], axis=-1) < F32 * np.linalg.norm(q[r], axis=-1)).all(), r
            slot = int(self.slots(self.seqs[r], self.lens[r])[-1])
            touched.add(slot)
            for (e, s), want in zip(self.halves(), (k[r], v[r])):
                if s is None:
                    got = e[slot].astype(np.float64).reshape(-1, 128)
                    assert (np.abs(got - want) <= F16 * np.abs(want) + F32 * np.linalg.norm(want, axis=-1, keepdims=True)).all(), r
                else:
                    got = (e[slot].reshape(-1, 32).astype(np.float64) * s[slot].astype(np.float64)[:, None])
                    want = want.reshape(-1, 32)
                    step = np.abs(want).max(-1, keepdims=True) / 127
                    # half a step, 2^-11 of the scale on at most 127 steps, and f32's
                    assert (np.abs(got - want) <= step * (0.5 + 127 * F16 + 127 * 12 * F32)).all(), r
        rest = np.array(sorted(set(range(self.n_pages * self.page)) - touched))
        for (e, s), (e0, s0) in zip(self.halves(), before):
            assert (e[rest] == e0[rest]).all() and (s is None or (s[rest] == s0[rest]).all())
        assert (self.rows_of(self.out, self.sq, self.sq, self.grid)[self.rows:] == 7.5).all()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("n_axes", [1, 2, 3, 4])
@pytest.mark.parametrize("heads,lens,page", [((1, 1), [1], 16), ((8, 2), [900], 64), ((2, 4), [5, 0, 64, 65, 1, 130], 16),
                                             ((1, 8), [300, 17, 2, 0], 32), ((3, 1), [40] * 5, 128)])
def test_rows(ctx, precision, n_axes, heads, lens, page):
    b = Axes(ctx, P[precision], *heads, page, lens, n_axes=n_axes, far=100000, grid=len(lens) + 2)
    try:
        b.check()
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
def test_many_rows(ctx, precision):
    """Enough rows for the form of 64 heads a workgroup: 1400 of one sequence, 48 heads each."""
    n = 1400
    b = Axes(ctx, P[precision], 8, 4, 64, 3 + 1 + np.arange(n), seqs=np.zeros(n, int), n_axes=3, far=2**20)
    try:
        b.check()
    finally:
        b.free()


def test_positions_past_31_bits(ctx):
    b = Axes(ctx, P["f16"], 2, 2, 16, [4, 9], far=2**32)
    try:
        b.check()
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
def test_as_kv_append_on_one_axis(ctx, precision):
    """One axis whose positions are the rows' own: kv_append's bits."""
    lens = [5, 1000, 64, 0, 1]
    b = Axes(ctx, P[precision], 2, 4, 32, lens, n_axes=1)
    try:
        u = b.arena.as_u32()
        u[b.at.axes: b.at.axes + 4 * b.rows: 4] = np.maximum(np.asarray(lens), 1) - 1
        b.append()
        got = [b.arena.host()[b.out * 4: (b.out + b.sq * b.rows) * 4].copy()] + [b.pool.host().copy()]
        b.pool.host()[:] = 0
        Batch.append(b)
        assert (got[0] == b.arena.host()[b.out * 4: (b.out + b.sq * b.rows) * 4]).all()
        assert (got[1] == b.pool.host()).all()
    finally:
        b.free()


def test_refusals(ctx):
    b = Axes(ctx, P["f16"], 2, 2, 16, [4, 9])
    try:
        end = b.arena.size // 4

        def record(axes=b.at.axes, n=3, rope=b.norms[2]):
            keep, b.at.axes = b.at.axes, axes
            try:
                ctx.record(False, lambda r: b.kernels.append_axes(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.out, b.sq),
                                                                  *b.norms[:2], rope, n, b.grid)).free()
            finally:
                b.at.axes = keep
        record()
        for bad in (dict(n=0), dict(n=5), dict(axes=end - 4), dict(axes=b.at.axes + 2), dict(axes=b.out),
                    dict(rope=end - 128), dict(rope=b.out)):
            with pytest.raises(SkylaHipError):
                record(**bad)
    finally:
        b.free()
