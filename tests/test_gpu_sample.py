"""logits_sample (kernels/sample.hip) against the same in 64 bits: which token, how many it was drawn
from, and its log probability."""
import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip.abi import SkylaHipError

pytestmark = pytest.mark.gpu

# A weight is held to 2^-37 of its bin's upper edge (7.3e-12, and 1.1 times that of itself), a series is off by
# 6e-14 and t by 3 2^-53 |t| (|t| < 1e6 here: 3.4e-10 of ln 2 / 8 = 3e-11): a sum, and so a log probability, is off by
# 4e-11 at most.  It is rounded to f32.
LOGPROB = 1e-10
F32 = 2.0**-24


def _pad(n):
    return -(-n // 64) * 64


def want(x, temperature, top_p, min_p, top_k, draw):
    """(token, kept, logprob) of one row by the definition."""
    x = np.float32(x).astype(np.float64)
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, float(np.finfo(np.float32).max))
    ids = np.argsort(-x, kind="stable")[: int((x > -np.inf).sum())]
    if len(ids) == 0:
        return 0xFFFFFFFF, 0, -np.inf
    T = float(np.float32(temperature))
    hot = T > 0
    with np.errstate(divide="ignore", over="ignore", under="ignore"):
        y = (x[ids] - x[ids[0]]) / (T if hot else 1.0)
        n = min(top_k or len(ids), len(ids))
        if min_p > 0:
            n = min(n, max(1, int((np.exp(y) >= float(np.float32(min_p))).sum())))
        c = np.cumsum(np.exp(y))
    n = n if hot else 1
    if np.float32(top_p) < 1:
        n = min(n, int(np.searchsorted(c[:n], max(0.0, float(np.float32(top_p))) * c[n - 1], side="left")) + 1)
    at = int(np.searchsorted(c[:n], (draw + 0.5) / 2**32 * c[n - 1], side="right"))
    return int(ids[at]), n, y[at] - np.log(c[n - 1])


class Rows:
    def __init__(self, ctx, x, settings, grid=None, pad=0):
        self.ctx, self.rows, self.v, self.x, self.settings = ctx, len(x), len(x[0]), x, settings
        self.grid = grid or self.rows
        self.stride = -(-self.v // 4) * 4 + pad
        size = 64
        off = []
        for n in (8 * self.grid, self.stride * self.grid, 4 * self.grid, B.sample_size(self.grid, self.v)):
            off.append(size)
            size += _pad(n)
        self.at = B.SampleRegions(controls=off[0], out=off[2], part=off[3])
        self.xo = off[1]
        self.arena = ctx.alloc_host(size * 4)
        f, u = self.arena.as_f32(), self.arena.as_u32()
        f[:] = np.float32(7.5)
        u[:64] = 0
        u[2] = self.rows
        for r, (T, p, m, k, d) in enumerate(settings):
            o = off[0] + 8 * r
            f[o: o + 3] = T, p, m
            u[o + 3: o + 8] = k, d, 0, 0, 0
            f[self.xo + r * self.stride: self.xo + r * self.stride + self.v] = x[r]
        self.arena.upload()
        self.kernels = B.LogitsKernels(ctx, self.arena)
        self.rec = ctx.record(False, lambda r: self.kernels.sample(r, self.at, (self.xo, self.stride), self.v, self.grid))

    def run(self):
        self.ctx.replay(self.rec)
        self.arena.download(self.at.out * 4, 16 * self.grid)
        f, u, o = self.arena.as_f32(), self.arena.as_u32(), self.at.out
        return [(int(u[o + 4 * r]), int(u[o + 4 * r + 1]), float(f[o + 4 * r + 2])) for r in range(self.rows)]

    def check(self, times=1):
        for _ in range(times):
            got = self.run()
            for r, (token, kept, logprob) in enumerate(got):
                w = want(self.x[r], *self.settings[r])
                assert (token, kept) == w[:2], (r, self.settings[r], got[r], w)
                assert logprob == w[2] or abs(logprob - w[2]) < LOGPROB + F32 * abs(w[2]), (r, self.settings[r], got[r], w)
        rest = self.arena.as_f32()[self.at.out + 4 * self.rows: self.at.out + 4 * self.grid]
        assert (rest == 7.5).all()

    def free(self):
        self.rec.free()
        self.kernels.free()
        self.arena.free()


def _check(ctx, x, settings, times=1, **more):
    rows = Rows(ctx, x, settings, **more)
    try:
        rows.check(times)
    finally:
        rows.free()


def _some(g, n):
    """Settings of every kind, the draws from end to end."""
    kinds = [(1.0, 1.0, 0.0, 0), (0.7, 1.0, 0.0, 50), (1.3, 0.9, 0.0, 0), (0.8, 1.0, 0.05, 0), (0.9, 0.95, 0.02, 40),
             (0.0, 0.9, 0.0, 0), (1.0, 0.5, 0.3, 3), (2.0, 0.999, 0.0, 1000)]
    return [(*kinds[r % len(kinds)], int(g.integers(0, 2**32))) for r in range(n)]


@pytest.mark.parametrize("v", [1, 2, 3, 63, 1000, 8191, 8192, 8193, 16384, 50001, 151936])
@pytest.mark.parametrize("spread", [0.3, 3.0, 30.0])
def test_rows_of_every_kind(ctx, v, spread):
    g = np.random.default_rng(v)
    x = (g.standard_normal((16, v)) * spread).astype(np.float32)
    _check(ctx, x, _some(g, 16), grid=19, pad=64)


@pytest.mark.parametrize("draw", [0, 1, 2**31, 2**32 - 2, 2**32 - 1])
def test_the_ends_of_a_draw(ctx, draw):
    g = np.random.default_rng(draw)
    x = (g.standard_normal((8, 20000)) * 2).astype(np.float32)
    _check(ctx, x, [(*s[:4], draw) for s in _some(g, 8)])


def test_equal_logits(ctx):
    """Ties go by id: rows of one value, of few values, of values rounded as a 16-bit head leaves them."""
    g = np.random.default_rng(5)
    v = 30000
    x = np.zeros((12, v), np.float32)
    x[3:6] = g.integers(0, 3, (3, v))
    x[6:9] = np.round(g.standard_normal((3, v)) * 16) / 16
    x[9:] = np.where(g.random((3, v)) < 0.5, np.float32(-0.0), np.float32(0.0))  # equal as numbers
    for p, k, m in ((1.0, 0, 0.0), (0.5, 0, 0.0), (1.0, 777, 0.0), (0.25, 4000, 0.0), (1.0, 0, 0.9)):
        _check(ctx, x, [(1.0, p, m, k, int(d)) for d in g.integers(0, 2**32, 12)])


@pytest.mark.parametrize("v", [70, 600, 5000, 8192, 20000])
@pytest.mark.parametrize("step", [2.0**-7, 2.0**-4, 0.5, 8.0])
def test_logits_on_a_grid(ctx, v, step):
    """From a few tokens of each value to thousands: those of one value are in order by their ids alone."""
    g = np.random.default_rng(v)
    x = (np.round(g.standard_normal((16, v)) / step) * step).astype(np.float32)
    _check(ctx, x, [(*s[:4], int(d)) for s, d in zip(_some(g, 16), g.integers(0, 2**32, 16))])
    _check(ctx, x, [(1.0, 0.37, 0.6, v // 3, int(d)) for d in g.integers(0, 2**32, 16)])


@pytest.mark.parametrize("v", [5, 9000, 40000])
def test_logits_without_a_place(ctx, v):
    """-inf and NaN are never drawn, +inf always, rows of nothing give no token; whole chunks of nothing."""
    g = np.random.default_rng(v)
    x = (g.standard_normal((9, v)) * 2).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, : v - 2] = -np.inf
    x[3, 1:] = -np.inf
    x[4, g.random(v) < 0.5] = np.nan
    x[5, v // 2] = np.inf
    x[6, [1, v - 1]] = np.inf
    x[7, g.random(v) < 0.9] = -np.inf
    x[7, v - 1] = 0
    x[8] = np.where(np.arange(v) % 2, np.nan, -np.inf)
    for s in ((1.0, 1.0, 0.0, 0), (0.7, 0.9, 0.05, 20), (0.0, 1.0, 0.0, 0)):
        _check(ctx, x, [(*s, int(d)) for d in g.integers(0, 2**32, 9)])


@pytest.mark.parametrize("shift", [-1e4, 0.0, 3e5])
@pytest.mark.parametrize("T", [0.01, 0.05, 1.0, 5.0, 100.0, float("inf")])
def test_temperatures_and_sizes(ctx, shift, T):
    """Hot rows are flat (bins of more tokens than are put in order), cold ones leave one or two; logits far from 0."""
    g = np.random.default_rng(7)
    x = (g.standard_normal((6, 60000)) * 2 + shift).astype(np.float32)
    kinds = ((1.0, 0.0, 0), (0.9, 0.0, 0), (1.0, 0.0, 30000), (0.3, 0.0, 59999), (1.0, 0.999, 0), (0.7, 0.5, 20000))
    _check(ctx, x, [(T, *s, int(d)) for s, d in zip(kinds, g.integers(0, 2**32, 6))])


def test_borders_below_every_bin(ctx):
    """Borders among tokens far below the largest: a few at the top, the rest 70 to 90 below them."""
    g = np.random.default_rng(11)
    x = (g.uniform(-90, -70, (5, 30000))).astype(np.float32)
    x[:, 100:103] = [0.0, -1.0, -50.0]
    s = [(1.0, 1.0, 0.0, 20000), (1.0, 1.0, 1e-36, 0), (1.0, 1.0, 0.0, 0), (1.0, 0.9, 1e-36, 25000), (0.5, 1.0, 0.0, 4)]
    _check(ctx, x, [(*k, int(d)) for k, d in zip(s, g.integers(0, 2**32, 5))])


@pytest.mark.parametrize("settings", [(-1.0, 0.9, 0.0, 0), (float("nan"), 1.0, 0.0, 0), (1.0, -3.0, 0.0, 0), (1.0, 0.0, 0.0, 0),
                                      (1.0, float("nan"), 0.0, 0), (1.0, 7.0, float("nan"), 0), (1.0, 1.0, 1.0, 0),
                                      (1.0, 1.0, 3.0, 0), (1.0, 1.0, -1.0, 0), (1.0, 1.0, 0.0, 2**32 - 1), (1e-40, 1.0, 0.0, 0)])
def test_settings_outside_the_usual(ctx, settings):
    g = np.random.default_rng(3)
    x = g.standard_normal((2, 10000)).astype(np.float32)
    x[1, [7, 70]] = 9.0  # two largest
    s = list(settings)
    if not s[2] == s[2]:
        s[2] = 0.0  # min_p that is no number: none
    got, ref = [(*settings, d) for d in (123456789, 4 * 10**9)], [(*s, d) for d in (123456789, 4 * 10**9)]
    rows = Rows(ctx, x, got)
    try:
        rows.settings = ref
        rows.check()
    finally:
        rows.free()


@pytest.mark.parametrize("v", [30000, 151936, 1 << 20])
@pytest.mark.parametrize("T", [2.0, 5.0, 40.0])
def test_borders_among_thousands(ctx, v, T):
    """So even that a bin has more tokens than are taken at once, of values all their own and of few."""
    g = np.random.default_rng(v + int(T))
    x = (g.standard_normal((6, v)) * 2.5).astype(np.float32)
    x[4:] = np.round(x[4:] * 4) / 4
    for p, m, k in ((1.0, 0.0, 0), (0.95, 0.0, 0), (0.9, 0.0, v // 3), (0.8, 0.02, 0), (0.5, 0.1, v // 2)):
        _check(ctx, x, [(T, p, m, k, int(d)) for d in g.integers(0, 2**32, 6)])


def test_many_rows_again_and_again(ctx):
    """A full batch of the benchmark's vocabulary, replayed: the same tokens each time."""
    g = np.random.default_rng(1)
    x = (g.standard_normal((128, 151936)) * 2.5).astype(np.float32)
    x[5] = -np.inf
    _check(ctx, x, _some(g, 128), times=3)


def test_refusals(ctx):
    arena = ctx.alloc_host(1 << 20)
    kernels = B.LogitsKernels(ctx, arena)
    try:
        ok = dict(controls=64, out=512, part=1024)
        for at, x, v in ((dict(ok, out=1 << 18), (4096, 1024), 1000), (dict(ok, part=(1 << 18) - 64), (4096, 1024), 1000),
                         (ok, (4098, 1024), 1000), (ok, (4096, 1000 - 4), 1000), (ok, (4096, 1024), 0),
                         (ok, (4096, 1024), (1 << 20) + 1), (dict(ok, out=4096), (4096, 1024), 1000),
                         (dict(ok, part=4096), (4096, 1024), 1000), (dict(ok, controls=66), (4096, 1024), 1000)):
            with pytest.raises(SkylaHipError):
                ctx.record(False, lambda r: kernels.sample(r, B.SampleRegions(**at), x, v, 2)).free()
    finally:
        kernels.free()
        arena.free()


@pytest.mark.parametrize("v", [5, 9000, 40000])
@pytest.mark.parametrize("T", [0.0, 0.7, 30.0])
def test_nan_beside_infinity(ctx, v, T):
    """NaN has no place where a chunk's largest is +inf either: before it and behind it, in its chunk and in others,
    most of a row, and beside more +inf than are put in order."""
    g = np.random.default_rng(v)
    x = (g.standard_normal((7, v)) * 2).astype(np.float32)
    x[0, 0], x[0, 1] = np.nan, np.inf
    x[1, 0], x[1, v - 1] = np.nan, np.inf
    x[2, 0], x[2, v - 1] = np.inf, np.nan
    x[3], x[3, v // 2] = np.nan, np.inf
    x[4, g.random(v) < 0.5], x[4, [1, v - 2]] = np.nan, np.inf
    x[5] = np.where(np.arange(v) % 3 == 0, np.nan, np.inf)
    x[6] = np.where(np.arange(v) % 3 == 0, np.nan, np.where(np.arange(v) % 3 == 1, -np.inf, x[6]))
    x[6, v // 2] = np.inf
    for s in ((1.0, 0.0, 0), (0.9, 0.05, 20), (1.0, 0.0, 3)):
        _check(ctx, x, [(T, *s, int(d)) for d in g.integers(0, 2**32, 7)])
