"""attention_paged_shaped (kernels/batch.hip) against the same in 64 bits: scores capped and biased by
distance, windows, rows that see from a document's start or to a prefix's end, with and without
positions that many rows share."""
import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip.abi import SkylaHipError
from test_gpu_batch import P, Batch

pytestmark = pytest.mark.gpu

# attention_paged's 4e-6 of a row, and of e what shaping a score of at most 8 costs: a capped score is off by 5e-7 of
# it (the polynomial 1.3e-8 and five roundings of 2^-24, the other form 4e-7), 4e-6; a bias that leaves an e that counts
# is at most 20, rounded three times, 3.6e-6.
BAR = 1.2e-5


class Shaped(Batch):
    """A Batch whose rows have spans; lens are the rows' own, `until` past them where given."""

    def __init__(self, ctx, precision, n_kv, rep, page, lens, cap=0.0, window=0, slopes=None, begin=None, until=None,
                 first=0, parts=None, lead=None, wide=None, **more):
        n = len(lens)
        self.begin, self.until = (np.zeros(n, int) if v is None else np.asarray(v) for v in (begin, until))
        lens = np.asarray(lens)
        self.cap, self.window, self.first = cap, window, first
        ends = np.where(lens > 0, np.maximum(lens, self.until), 0)
        super().__init__(ctx, precision, n_kv, rep, page, ends, **more)
        self.lens, self.ends = lens, ends
        self.lo = np.maximum(self.begin, np.where((window > 0) & (lens > window), lens - window, 0))
        some = B.shaped_splits(self.grid, n_kv, rep, max(self.shared - first, 0), max(1, int(ends.max(initial=1))),
                               self.shared if lead is None else lead)
        self.shaped_parts = B.ShapedParts(*(parts or some))
        if wide is not None:
            self.shaped_parts = self.shaped_parts._replace(wide=wide)
        old, size = self.arena, self.arena.size // 4
        extra = B.shaped_part_size(self.grid, self.n_head, self.shaped_parts)
        self.arena = ctx.alloc_host((size + 2 * self.grid + 128 + self.n_head + extra) * 4)
        f, u = self.arena.as_f32(), self.arena.as_u32()
        u[:size] = old.as_u32()
        f[size:] = np.float32(7.5)
        self.kernels.free()
        old.free()
        self.kernels = B.BatchKernels(ctx, self.arena, self.arena, [self.pool], self.c, self.paged)
        at = self.at
        at.spans, slopes_at = size, size + (2 * self.grid + 3) // 4 * 4
        at.part = slopes_at + (self.n_head + 63) // 64 * 64
        self.slopes = None if slopes is None else np.float32(slopes)
        if slopes is not None:
            f[slopes_at: slopes_at + self.n_head] = self.slopes
        self.shape = B.Shape(cap, window, None if slopes is None else slopes_at)
        u[5] = first
        u[at.rows: at.rows + 4 * self.rows] = np.stack([self.seqs, self.lens, self.shares, np.zeros(n)], 1).ravel()
        u[at.spans: at.spans + 2 * self.grid] = 0xFFFFFFFF
        u[at.spans: at.spans + 2 * n] = np.stack([self.begin, self.until], 1).ravel()

    def prepare(self, spread=1.0):
        self.fill()
        if self.shared:
            keep, self.lens = self.lens, self.ends
            self.copy_shared()
            self.lens = keep
        self.rows_of(self.q, self.sq, self.n_head * 128)[:] = self.g.standard_normal((self.rows, self.n_head * 128)) * spread
        return self

    def want(self):
        o = np.zeros((self.rows, self.n_head, 128))
        q = self.rows_of(self.q, self.sq, self.n_head * 128).astype(np.float64).reshape(self.rows, self.n_head, 128)
        for r in range(self.rows):
            lo, hi = int(self.lo[r]), int(self.ends[r])
            if lo >= hi or self.lens[r] == 0:
                continue
            K, V = self.read64(self.slots(self.seqs[r], hi)[lo:])
            away = np.abs(np.arange(lo, hi) - (self.lens[r] - 1))
            for h in range(self.n_head):
                s = K[:, h // self.rep] @ q[r, h] / np.sqrt(128.0)
                if self.cap:
                    s = self.cap * np.tanh(s / self.cap)
                if self.slopes is not None:
                    s = s - float(self.slopes[h]) * away
                e = np.exp(s - s.max())
                o[r, h] = e @ V[:, h // self.rep] / e.sum()
        return o

    def attend(self):
        self.run(lambda r: self.kernels.attend_shaped(r, 0, self.at, (self.q, self.sq), (self.out, self.sq), self.grid,
                                                      self.shaped_parts, self.shape))
        return self.rows_of(self.out, self.sq, self.n_head * 128).astype(np.float64).reshape(self.rows, self.n_head, 128)

    def check(self, bar=BAR):
        got, want = self.attend(), self.want()
        for r in range(self.rows):
            if not want[r].any():
                assert not got[r].any(), r
            else:
                d = np.linalg.norm(got[r] - want[r])
                assert d < bar * np.linalg.norm(want[r]), (r, d / np.linalg.norm(want[r]))
        rest = self.rows_of(self.out, self.sq, self.sq, self.grid)
        assert (rest[self.rows:] == 7.5).all() and (rest[:, self.n_head * 128:] == 7.5).all()  # nothing else written


def _alibi(heads):
    return 2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)


def _check(ctx, *args, spread=1.0, bar=BAR, **more):
    b = Shaped(ctx, *args, **more)
    try:
        b.prepare(spread).check(bar)
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (2, 4), (1, 8)])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (5.0, False), (50.0, True), (0.0, True)])
def test_scores_of_rows_of_their_own(ctx, precision, heads, cap, slopes):
    lens = [65, 1, 0, 16, 17, 130, 300, 64]
    _check(ctx, P[precision], *heads, 32, lens, cap=cap, slopes=_alibi(heads[0] * heads[1]) if slopes else None,
           grid=len(lens) + 3, spread=3.0 if cap else 1.0)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 299, 300, 10000, 2**32 - 1])
def test_windows(ctx, precision, window):
    _check(ctx, P[precision], 2, 2, 16, [300, 1, 0, 16, 17, 100, 299, 64], window=window, cap=30.0)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
def test_spans(ctx, precision, wide):
    """Rows from a document's start and to a prefix's end; ones that see themselves alone, later positions
    alone, or nothing."""
    lens = [100, 100, 100, 100, 50, 50, 50, 50, 0, 1]
    begin = [0, 37, 99, 100, 0, 20, 60, 200, 0, 0]
    until = [0, 50, 100, 101, 90, 70, 77, 190, 30, 65]
    _check(ctx, P[precision], 2, 2, 16, lens, begin=begin, until=until, cap=20.0, slopes=_alibi(4), wide=wide)
    _check(ctx, P[precision], 1, 4, 64, lens, begin=begin, until=until, window=33, wide=wide)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("heads", [(2, 1), (2, 2), (1, 4), (2, 8)])
@pytest.mark.parametrize("shared,page,n", [(1, 16, 2), (37, 16, 5), (64, 64, 17), (1000, 64, 9), (129, 32, 33)])
def test_shared_positions(ctx, precision, wide, heads, shared, page, n):
    """Rows behind a shared run, all of it seen: one idle, one that shares nothing, one shorter than the run, one
    that is the run and no more, one that starts inside it, one that sees nothing."""
    g = np.random.default_rng(shared + n)
    lens = shared + g.integers(1, 150, n)
    shares, begin = np.full(n, shared), np.zeros(n, int)
    if n > 4:
        lens[0], lens[3], lens[4] = 0, max(1, shared // 2), shared
        shares[2] = 0
    if n > 8:
        begin[5], begin[6] = shared // 2, lens[6] + 1
    _check(ctx, P[precision], *heads, page, lens, shares=shares, shared=shared, leader=1 if n > 4 else 0, seed=shared,
           wide=wide, begin=begin, cap=25.0, slopes=_alibi(heads[0] * heads[1]), lead=0)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("shared,n,window", [(0, 19, 7), (100, 40, 60), (640, 128, 300), (640, 128, 129), (1500, 128, 1000),
                                             (1000, 50, 20)])
def test_chunks_with_a_window(ctx, precision, wide, shared, n, window):
    """Rows of one sequence at consecutive positions: what all of them see before the chunk shared, each row's lead
    before that and its own end behind it."""
    lens = shared + 1 + np.arange(n)
    lo = np.maximum(lens - window, 0)
    first = int(lo[lo < shared].max(initial=0)) if shared else 0
    _check(ctx, P[precision], 2, 4, 64, lens, seqs=np.zeros(n, int), shares=np.full(n, shared), shared=shared,
           wide=wide, window=window, first=first)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("first", [0, 1, 63, 64, 65, 500, 639, 640, 2000])
@pytest.mark.parametrize("lead", [0, 200])
def test_where_the_shared_run_starts(ctx, precision, first, lead):
    """Whatever the control word says: rows that do not see all of the run, or have no parts for a lead, read
    their own pages."""
    lens = 640 + 1 + np.arange(24)
    begin = np.where(np.arange(24) % 3 == 0, 64, np.where(np.arange(24) % 3 == 1, 0, 500))
    _check(ctx, P[precision], 2, 2, 32, lens, seqs=np.zeros(24, int), shares=np.full(24, 640), shared=640, begin=begin,
           first=first, lead=lead)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
def test_a_chunk_of_documents(ctx, precision, wide):
    """A chunk that ends one document and begins another, the rows of each seeing one another."""
    shared, n, half = 700, 100, 40
    r = np.arange(n)
    begin = np.where(r < half, 233, shared + half)
    until = np.where(r < half, shared + half, shared + n)
    _check(ctx, P[precision], 1, 8, 32, shared + 1 + r, seqs=np.zeros(n, int), shares=np.full(n, shared), shared=shared,
           begin=begin, until=until, first=233, wide=wide, slopes=_alibi(8))


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("parts", [(1, 1, False, 0), (1, 1, False, 1), (3, 2, False, 2), (64, 40, False, 7), (0, 5, False, 0),
                                   (1, 1, True, 1), (3, 2, True, 3), (21, 1, True, 1), (0, 1, False, 0), (0, 1, False, 3)])
def test_parts(ctx, precision, parts):
    lens = [2900, 1290, 1287, 1300]
    _check(ctx, P[precision], 2, 2, 32, lens, shares=[1287] * 4, shared=1287, parts=parts, begin=[100, 0, 128, 900],
           first=128, cap=40.0)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("wide", [False, True])
def test_what_a_mask_leaves_out_reaches_nothing(ctx, precision, bad, wide):
    """NaN and infinities in every slot that no row sees, among them ones next to what they see, in the shared run's
    pages before it and inside a tile."""
    shared, n, window = 300, 40, 150
    lens = shared + 1 + np.arange(n)
    lo = lens - window
    b = Shaped(ctx, P[precision], 2, 2, 32, lens, seqs=np.zeros(n, int), shares=np.full(n, shared), shared=shared,
               wide=wide, window=window, first=int(lo.max()), cap=30.0)
    try:
        b.prepare()
        want = b.want()
        live = set(b.slots(0, int(lens.max()))[int(lo.min()):].tolist())
        dead = np.array(sorted(set(range(b.n_pages * b.page)) - live))
        for e, s in b.halves():
            (e if s is None else s)[dead] = bad
        got = b.attend()
        for r in range(n):
            assert np.linalg.norm(got[r] - want[r]) < BAR * np.linalg.norm(want[r]), r
        # a position that the first rows see and the last do not: not in the shared run, so these stay whole
        for e, s in b.halves():
            (e if s is None else s)[b.slots(0, int(lo[3]) + 1)[-1]] = bad
        got = b.attend()
        for r in range(n):
            if r > 3:
                assert np.linalg.norm(got[r] - want[r]) < BAR * np.linalg.norm(want[r]), r
            else:
                assert not np.isfinite(got[r]).all(), r
    finally:
        b.free()


@pytest.mark.parametrize("cap", [2.0**-10, 0.01, 1.0, 2.0**14])
@pytest.mark.parametrize("spread", [1e-6, 1.0, 300.0])
def test_caps_and_scores_of_any_size(ctx, cap, spread):
    """Scores far below and far above the cap, on one wave and in the shared run's wide form."""
    # (uncapped, scores of 300 standard deviations are off by 2^-22 of 1000: 2.5e-4)
    bar = 5e-4 if spread > 1 and cap > 100 else BAR
    _check(ctx, P["f16"], 2, 2, 16, [500, 90], cap=cap, spread=spread, bar=bar)
    _check(ctx, P["f16k_q8v"], 2, 4, 16, [500] * 20, shares=[400] * 20, shared=400,
           cap=cap, spread=spread, bar=bar, wide=True)


def test_words_that_name_nothing(ctx):
    b = Shaped(ctx, P["f16"], 2, 2, 16, [50, 40, 30, 20, 45], n_seq=6, window=30, until=[0, 0, 0, 0, 48])
    try:
        b.prepare()
        want = b.want()
        u = b.arena.as_u32()
        u[b.at.rows + 4] = 6                    # row 1: no such sequence
        u[b.at.rows + 9] = 0xFFFFFFFF           # row 2: longer than its table
        u[b.at.table + 3 * b.table.shape[1]] = 0xFFFFFFF0  # row 3's first page: no such page
        u[3], u[4], u[5] = 1 << 30, 77, 0xFFFFFFFF  # shared positions of no sequence
        got = b.attend()
        for r in (0, 4):
            assert np.linalg.norm(got[r] - want[r]) < BAR * np.linalg.norm(want[r])
        assert not got[1].any() and np.isfinite(got).all()
        u[b.at.spans + 8: b.at.spans + 10] = 0, 0xFFFFFFFF  # row 4's prefix: past its table, whose end it is
        assert np.isfinite(b.attend()).all()
    finally:
        b.free()


def test_as_attention_paged_where_nothing_is_shaped(ctx):
    """Without cap, slopes, window and spans: attention_paged's definition, its parts and its result to rounding."""
    lens, shared = [70, 45, 41, 1000], 40
    b = Shaped(ctx, P["f16k_q8v"], 2, 2, 32, lens, shares=[40] * 4, shared=shared, leader=2)
    try:
        b.prepare()
        got = b.attend().copy()
        plain = Batch.attend
        b.at.part, keep = b.at.part, b.parts
        b.parts = B.Parts(*b.shaped_parts[:3])
        same = plain(b)
        b.parts = keep
        for r in range(4):
            assert np.linalg.norm(got[r] - same[r]) < 4e-6 * np.linalg.norm(same[r]), r
    finally:
        b.free()


def test_recorded_steps(ctx):
    """A recording replayed while its rows, spans and control words change, as launches and as a graph."""
    b = Shaped(ctx, P["f16k_q8v"], 2, 4, 32, [400, 300, 200], window=100, shares=[128] * 3, shared=128, cap=30.0, grid=5)
    try:
        b.prepare()
        b.arena.upload()
        b.pool.upload()
        rec = ctx.record(False, lambda r: b.kernels.attend_shaped(r, 0, b.at, (b.q, b.sq), (b.out, b.sq), b.grid,
                                                                  b.shaped_parts, b.shape))
        try:
            for step in range(6):
                b.lens = b.ends = np.array([400 - step, 300 - 50 * step, 130 + step])
                b.begin = np.array([0, 10 * step, 3])
                b.lo = np.maximum(b.begin, np.maximum(b.lens - 100, 0))
                u = b.arena.as_u32()
                u[b.at.rows: b.at.rows + 12] = np.stack([b.seqs, b.lens, b.shares, np.zeros(3)], 1).ravel()
                u[b.at.spans: b.at.spans + 6] = np.stack([b.begin, b.until], 1).ravel()
                b.arena.upload()
                (ctx.replay if step % 2 else ctx.replay_timed)(rec)
                b.arena.download()
                got = b.rows_of(b.out, b.sq, b.n_head * 128).astype(np.float64).reshape(3, b.n_head, 128)
                want = b.want()
                for r in range(3):
                    assert np.linalg.norm(got[r] - want[r]) <= BAR * np.linalg.norm(want[r]), (step, r)  # (zeros: the same)
        finally:
            rec.free()
    finally:
        b.free()


def test_more_live_rows_than_the_grid(ctx):
    """The control word says more rows than the recording has: those of the recording are right, the words behind
    them (another sequence's, at their place) no part of them."""
    lens = 200 + np.arange(6)
    b = Shaped(ctx, P["f16"], 2, 2, 32, lens, seqs=np.zeros(6, int), shares=[100] * 6, shared=100, window=150, first=56,
               parts=(2, 2, False, 1))
    try:
        b.prepare()
        b.arena.as_u32()[2] = 5000
        b.check()
    finally:
        b.free()


@pytest.mark.parametrize("rows", [3, 16, 17])
def test_rows_that_go_together_or_not(ctx, rows):
    """Rows of one sequence among idle ones, rows in any order, two sequences in one tile, rows far apart."""
    g = np.random.default_rng(rows)
    for seqs, lens in ((np.zeros(rows, int), 300 + g.permutation(rows)),
                       (np.zeros(rows, int), np.where(g.random(rows) < 0.4, 0, 200 + np.arange(rows))),
                       (np.arange(rows) // 5 % 2, 100 + np.arange(rows)),
                       (np.zeros(rows, int), 1 + 257 * (np.arange(rows) % 4) + np.arange(rows))):
        for parts in (None, (0, 1, False, 0), (0, 7, False, 0)):
            _check(ctx, P["f16k_q8v"], 2, 2, 16, lens, seqs=seqs, window=90, cap=20.0, parts=parts,
                   until=np.where(np.arange(rows) % 3 == 1, lens.max(), 0))


@pytest.mark.parametrize("heads", [(2, 1), (2, 2), (1, 4), (1, 8)])
@pytest.mark.parametrize("parts", [(0, 1, False, 0), (0, 3, False, 0)])
@pytest.mark.parametrize("lens", ["all", "one", "first idle"])
def test_rows_that_go_together_and_see_nothing(ctx, heads, parts, lens):
    """Tiles of one sequence's rows, and what is left of one, whose masks leave nothing, one live row among idle
    ones, rows that name no sequence: zeros in all of them, whatever the output held."""
    T = 16 // heads[1]
    n = 2 * T + T // 2
    ends = 40 + np.arange(n)
    if lens == "one":
        ends[np.arange(n) % T != T // 2] = 0
    elif lens == "first idle":
        ends[::T] = 0
    for begin in (ends + 3, np.where(np.arange(n) // T == 1, 5, ends + 3)):  # all, all but the second tile
        _check(ctx, P["f16k_q8v"], *heads, 16, ends, seqs=np.zeros(n, int), parts=parts, begin=begin, grid=n + 3)
    b = Shaped(ctx, P["f16"], *heads, 16, ends, seqs=np.zeros(n, int), parts=parts, grid=n + 3)
    try:
        b.prepare()
        b.arena.as_u32()[b.at.rows: b.at.rows + 4 * n: 4] = 3  # no such sequence
        b.lens = b.ends = np.zeros(n, int)
        b.check()
    finally:
        b.free()


@pytest.mark.parametrize("heads", [(2, 1), (2, 2), (1, 4), (1, 8)])
@pytest.mark.parametrize("word", [0xFFFFFFFF, 0xFFFFFFFE, 1])
@pytest.mark.parametrize("at", ["first", "last", "first of all"])
def test_rows_of_no_sequence_among_ones_that_go_together(ctx, heads, word, at):
    """The attention and its merge cut the others' positions the same, whichever rows of a tile name no sequence."""
    T = 16 // heads[1]
    n = 2 * T + T // 2
    b = Shaped(ctx, P["f16k_q8v"], *heads, 16, 300 + 9 * np.arange(n) % 100, seqs=np.zeros(n, int), window=90,
               parts=(0, 5, False, 0), until=np.where(np.arange(n) % 3 == 1, 400, 0))
    try:
        b.prepare()
        bad = {"first": slice(0, n, T), "last": slice(T - 1, n, T), "first of all": slice(0, 1)}[at]
        b.arena.as_u32()[b.at.rows: b.at.rows + 4 * n].reshape(n, 4)[bad, 0] = word
        b.lens[bad] = 0  # (as the result has them; the words keep their lengths)
        b.check()
    finally:
        b.free()


def test_refusals(ctx):
    b = Shaped(ctx, P["f16"], 2, 2, 16, [50, 40])
    try:
        def record(parts=b.shaped_parts, shape=b.shape, **at):
            old = {k: getattr(b.at, k) for k in at}
            for k, v in at.items():
                setattr(b.at, k, v)
            try:
                ctx.record(False, lambda r: b.kernels.attend_shaped(r, 0, b.at, (b.q, b.sq), (b.out, b.sq), b.grid, parts,
                                                                    shape)).free()
            finally:
                for k, v in old.items():
                    setattr(b.at, k, v)
        record()
        end = b.arena.size // 4
        for bad in (dict(spans=end - 2), dict(spans=b.at.spans + 1), dict(spans=b.out), dict(shape=B.Shape(slopes=end - 3)),
                    dict(shape=B.Shape(slopes=b.out)), dict(shape=B.Shape(cap=-1.0)), dict(shape=B.Shape(cap=float("nan"))),
                    dict(shape=B.Shape(cap=1e-4)), dict(shape=B.Shape(cap=1e5)), dict(parts=B.ShapedParts(0, 0)),
                    dict(parts=B.ShapedParts(1000, 20, False, 10)), dict(parts=B.ShapedParts(0, 400, False, 400)),
                    dict(part=end - 100)):
            with pytest.raises(SkylaHipError):
                record(**bad)
    finally:
        b.free()
