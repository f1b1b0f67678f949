"""The batch operators (kernels/batch.hip) against the same in 64 bits: rows of several
sequences over a paged cache with pages in any order, idle rows, runs of shared positions that
end inside a page and a tile, and rows that do not share them."""
import numpy as np
import pytest

from helpers import tactics
from skyla_hip import batch as B
from skyla_hip import engine as E
from skyla_hip.abi import SkylaHipError

pytestmark = pytest.mark.gpu

P = {"f16": E.KvPrecision.F16, "q8": E.KvPrecision.Q8, "f16k_q8v": E.KvPrecision.F16_KEYS_Q8_VALUES}
EPS, THETA = 1e-6, 1e6


def _pad(n):
    return -(-n // 64) * 64


class Batch:
    """A pool and an arena for `rows` rows, with what the tests write and read in numpy."""

    def __init__(self, ctx, precision, n_kv, rep, page, lens, seqs=None, shares=None, shared=0, leader=0, n_seq=None,
                 n_pages=None, parts=None, grid=None, seed=0, wide=None):
        g = self.g = np.random.default_rng(seed)
        self.ctx, self.lens, self.rows = ctx, np.asarray(lens), len(lens)
        self.n_kv, self.rep, self.n_head, self.dim = n_kv, rep, n_kv * rep, n_kv * 128
        self.seqs = np.arange(self.rows) if seqs is None else np.asarray(seqs)
        self.shares = np.zeros(self.rows, int) if shares is None else np.asarray(shares)
        self.shared, self.leader, self.page = shared, leader, page
        n_seq = n_seq or int(self.seqs.max()) + 1
        width = max(1, -(-int(self.lens.max(initial=1)) // page))
        # every sequence's pages, the whole shared ones the same for those that share
        whole = shared // page
        table = np.zeros((n_seq, width), int)
        n = whole
        for s in range(n_seq):
            own = [r for r in range(self.rows) if self.seqs[r] == s]
            first = whole if own and all(self.shares[r] and self.lens[r] >= shared for r in own) else 0
            table[s, :first] = np.arange(first)
            table[s, first:] = n + np.arange(width - first)
            n += width - first
        self.n_pages = n_pages or n + 2
        order = g.permutation(self.n_pages)
        self.table = order[np.minimum(table, self.n_pages - 1)]
        self.paged = B.Paged(precision, page, self.n_pages, n_seq, width, self.dim)
        self.pool = ctx.alloc_host(max(16, self.paged.bytes()))
        c = self.c = E.Config(n_embd=256, n_head=self.n_head, n_head_kv=n_kv, eps=EPS, rope_theta=THETA)
        self.grid = grid or self.rows
        own = int((self.lens - np.where((self.shares > 0) & (self.lens >= shared), shared, 0)).max(initial=1))
        self.parts = B.Parts(*(parts or B.splits(self.grid, n_kv, rep, shared, max(1, own))))
        if wide is not None:
            self.parts = self.parts._replace(wide=wide)
        size = 64

        def room(n):
            nonlocal size
            off, size = size, size + _pad(n)
            return off
        self.sq, self.skv = _pad(self.n_head * 128) + 64, _pad(self.dim)
        at = B.BatchRegions(rows=room(4 * self.grid), table=room(self.table.size))
        self.q, self.out = room(self.sq * self.grid), room(self.sq * self.grid)
        self.k, self.v = room(self.skv * self.grid), room(self.skv * self.grid)
        self.norms = room(128), room(128), room(64)
        at.part = room(B.part_size(self.grid, self.n_head, self.parts))
        self.at = at
        self.arena = ctx.alloc_host(size * 4)
        f, u = self.arena.as_f32(), self.arena.as_u32()
        f[:] = np.float32(7.5)
        u[:64] = 0
        u[2:5] = self.rows, shared, leader
        u[at.rows: at.rows + 4 * self.grid] = 0xFFFFFFFF  # rows past the live ones: nothing valid
        u[at.rows: at.rows + 4 * self.rows] = np.stack([self.seqs, self.lens, self.shares, np.zeros(self.rows)], 1).ravel()
        u[at.table: at.table + self.table.size] = self.table.ravel()
        self.kernels = B.BatchKernels(ctx, self.arena, self.arena, [self.pool], c, self.paged)

    def rows_of(self, off, stride, width, n=None):
        n = self.rows if n is None else n
        f = self.arena.as_f32()
        return f[off: off + stride * n].reshape(n, stride)[:, :width]

    def halves(self):
        """(entries, scales or None) of keys and values in the pool's host mirror, a row a slot."""
        lay, n, out = self.paged.layout, self.n_pages * self.page, []
        h = self.pool.host()
        for off, sc, q8 in ((lay.keys(0), lay.key_scales(0), self.paged.precision.keys_q8),
                            (lay.values(0), lay.value_scales(0), self.paged.precision.values_q8)):
            e = (h.view(np.int8) if q8 else h.view("<f2"))[off: off + n * self.dim].reshape(n, self.dim)
            out.append((e, h.view("<f2")[sc: sc + n * self.dim // 32].reshape(n, -1) if q8 else None))
        return out

    def fill(self, spread=1.0):
        for e, s in self.halves():
            if s is None:
                e[:] = (self.g.standard_normal(e.shape) * spread).astype(np.float16)
            else:
                e[:] = self.g.integers(-127, 128, e.shape)
                s[:] = (np.exp(self.g.uniform(-5, -3.5, s.shape)) * spread).astype(np.float16)

    def slots(self, seq, n):
        p = np.arange(n)
        return self.table[seq, p // self.page] * self.page + p % self.page

    def copy_shared(self):
        """The shared rows that lie in a page of each sequence's own."""
        members = [r for r in range(self.rows) if self.shares[r] and self.lens[r] >= self.shared]
        src = self.slots(self.leader, self.shared)
        for r in members:
            for e, s in self.halves():
                to = self.slots(self.seqs[r], self.shared)
                e[to] = e[src].copy()
                if s is not None:
                    s[to] = s[src].copy()

    def read64(self, slots):
        out = []
        for e, s in self.halves():
            x = e[slots].astype(np.float64)
            out.append((x if s is None else x * np.repeat(s[slots].astype(np.float64), 32, 1)).reshape(-1, self.n_kv, 128))
        return out

    def want(self):
        o = np.zeros((self.rows, self.n_head, 128))
        q = self.rows_of(self.q, self.sq, self.n_head * 128).astype(np.float64).reshape(self.rows, self.n_head, 128)
        for r in range(self.rows):
            n = int(self.lens[r])
            if n == 0:
                continue
            K, V = self.read64(self.slots(self.seqs[r], n))
            for h in range(self.n_head):
                s = K[:, h // self.rep] @ q[r, h] / np.sqrt(128.0)
                e = np.exp(s - s.max())
                o[r, h] = e @ V[:, h // self.rep] / e.sum()
        return o

    def run(self, body):
        self.arena.upload()
        self.pool.upload()
        rec = self.ctx.record(False, body)
        try:
            self.ctx.replay(rec)
        finally:
            rec.free()
        self.arena.download()
        self.pool.download()

    def attend(self):
        self.run(lambda r: self.kernels.attend(r, 0, self.at, (self.q, self.sq), (self.out, self.sq), self.grid, self.parts))
        return self.rows_of(self.out, self.sq, self.n_head * 128).astype(np.float64).reshape(self.rows, self.n_head, 128)

    def append(self):
        qn, kn, rope = self.norms
        self.run(lambda r: self.kernels.append(r, 0, self.at, (self.q, self.sq), (self.k, self.skv), self.v,
                                               (self.out, self.sq), qn, kn, rope, self.grid))

    def free(self):
        self.kernels.free()
        self.pool.free()
        self.arena.free()


# Query parts of 22 bits put a score off by 2^-22 of |q| |k| / sqrt(128) <= 8 powers of two here:
# 2e-6 of e at worst, a tenth of that on average; e in two parts and 22-bit values add 2^-22 each,
# f32 sums of n terms sqrt(n) 2^-24 (n <= 3000: 3e-6).  Of the row's norm, 4e-6.
BAR = 4e-6


def _check_attend(b):
    got, want = b.attend(), b.want()
    for r in range(b.rows):
        if b.lens[r] == 0:
            assert not got[r].any(), r
        else:
            assert np.linalg.norm(got[r] - want[r]) < BAR * np.linalg.norm(want[r]), r
    rest = b.rows_of(b.out, b.sq, b.sq, b.grid)
    assert (rest[b.rows:] == 7.5).all() and (rest[:, b.n_head * 128:] == 7.5).all()  # nothing else written


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (2, 4), (1, 8)])
@pytest.mark.parametrize("lens,page", [([1], 16), ([0], 16), ([64], 64), ([65, 1, 0, 16, 17, 130], 16),
                                       ([300, 5, 64, 63, 127, 128, 129], 32), ([700], 256)])
def test_attention_of_rows_of_their_own(ctx, precision, heads, lens, page):
    b = Batch(ctx, P[precision], *heads, page, lens, seed=len(lens) + page, grid=len(lens) + 3)
    try:
        b.fill()
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        _check_attend(b)
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("heads", [(2, 1), (2, 2), (1, 4), (2, 8)])
@pytest.mark.parametrize("shared,page,n", [(1, 16, 2), (37, 16, 5), (64, 64, 17), (1000, 64, 9), (129, 32, 33)])
def test_attention_with_shared_positions(ctx, precision, wide, heads, shared, page, n):
    """Rows behind a shared run: one idle, one that shares nothing though it is longer, one shorter
    than the run, one that is the run and no more."""
    g = np.random.default_rng(shared + n)
    lens = shared + g.integers(1, 150, n)
    shares = np.full(n, shared)
    if n > 4:
        lens[0], lens[3], lens[4] = 0, max(1, shared // 2), shared
        shares[2] = 0
    leader = 1 if n > 4 else 0
    b = Batch(ctx, P[precision], *heads, page, lens, shares=shares, shared=shared, leader=leader, seed=shared,
              wide=wide)
    try:
        b.fill()
        b.copy_shared()
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        _check_attend(b)
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("shared,n", [(0, 19), (100, 40), (640, 128)])
def test_attention_of_a_prompt_chunk(ctx, precision, wide, shared, n):
    """Rows of one sequence at consecutive positions: the run before them shared, each row its own end."""
    lens = shared + 1 + np.arange(n)
    b = Batch(ctx, P[precision], 2, 4, 64, lens, seqs=np.zeros(n, int), shares=np.full(n, shared), shared=shared,
              wide=wide)
    try:
        b.fill()
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        _check_attend(b)
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("parts", [(1, 1), (3, 2), (64, 40), (0, 5), (1, 1, True), (3, 2, True), (21, 1, True), (0, 1)])
def test_attention_parts(ctx, precision, parts):
    """Any number of parts gives the same attention, and none for the shared run leaves it to the rows."""
    lens = [2900, 1290, 1287, 1300]
    b = Batch(ctx, P[precision], 2, 2, 32, lens, shares=[1287] * 4, shared=1287, parts=parts)
    try:
        b.fill()
        b.copy_shared()
        if parts[0] == 0:  # every sequence's own pages hold the whole run
            assert (b.table[:, :1287 // 32] == b.table[0, :1287 // 32]).all()
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        _check_attend(b)
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_keeps_out_what_lies_outside_a_row(ctx, precision, bad, wide):
    """Everything but the rows' live positions is NaN or infinite: unused slots, the rest of a last
    page, the slots of a sequence's own page under the shared run."""
    lens, shared = [70, 45, 41, 100], 40
    b = Batch(ctx, P[precision], 2, 2, 32, lens, shares=[40] * 4, shared=shared, leader=2, wide=wide)
    try:
        b.fill()
        live = set(b.slots(2, shared).tolist())
        for r in range(4):
            live |= set(b.slots(r, lens[r])[shared:].tolist())
        dead = np.array(sorted(set(range(b.n_pages * b.page)) - live))
        want_src = b.slots(2, shared)
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        saved = b.halves()
        for r in range(4):  # the definition's rows: the shared run from the leader
            for e, s in saved:
                to = b.slots(r, shared)
                e[to] = e[want_src].copy()
                if s is not None:
                    s[to] = s[want_src].copy()
        want = b.want()
        for e, s in saved:
            (e if s is None else s)[dead] = bad
        got = b.attend()
        for r in range(4):
            assert np.linalg.norm(got[r] - want[r]) < BAR * np.linalg.norm(want[r]), r
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
def test_attention_scales_of_any_size(ctx, precision):
    """Caches of values near 1e-4 and 1e4, and queries whose scores span a thousand."""
    for spread in (1e-4, 1e3):
        b = Batch(ctx, P[precision], 1, 4, 16, [500, 90], seed=3)
        try:
            b.fill(spread)
            q = b.rows_of(b.q, b.sq, b.n_head * 128)
            q[:] = b.g.standard_normal(q.shape) * (8 / max(spread, 1e-2) if spread > 1 else 8 / spread * 1e-2)
            got, want = b.attend(), b.want()
            for r in range(b.rows):
                # scores up to 2^6: 2^-22 of them
                assert np.linalg.norm(got[r] - want[r]) < 2e-5 * np.linalg.norm(want[r]), (spread, r)
        finally:
            b.free()


def test_attention_words_that_name_nothing(ctx):
    """Sequences and pages past the table's reach nothing outside the pool; a length past the table
    ends there; the other rows are right."""
    b = Batch(ctx, P["f16"], 2, 2, 16, [50, 40, 30, 20], n_seq=6)
    try:
        b.fill()
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        want = b.want()
        u = b.arena.as_u32()
        u[b.at.rows + 4] = 6                    # row 1: no such sequence
        u[b.at.rows + 9] = 0xFFFFFFFF           # row 2: longer than its table
        u[b.at.table + 3 * b.table.shape[1]] = 0xFFFFFFF0  # row 3's first page: no such page
        u[3], u[4] = 1 << 30, 77                # shared positions of no sequence
        got = b.attend()
        assert np.linalg.norm(got[0] - want[0]) < BAR * np.linalg.norm(want[0])
        assert not got[1].any() and np.isfinite(got).all()
    finally:
        b.free()


# ---- kv_append ---------------------------------------------------------------------------------
def _rope64(x, w, pos, freq):
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
    c, s = np.cos(pos * freq), np.sin(pos * freq)
    a, b = n[..., :64], n[..., 64:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("heads", [(1, 1), (2, 4), (8, 4), (4, 8)])
@pytest.mark.parametrize("lens,page", [([1], 16), ([0], 16), ([5, 0, 17, 1000, 64], 32), ([120001, 3, 65536], 4096)])
def test_append(ctx, precision, heads, lens, page):
    b = Batch(ctx, P[precision], *heads, page, lens, seed=7, grid=len(lens) + 2, parts=(0, 1),
              n_pages=None if max(lens) < 5000 else 100)
    try:
        f, g = b.arena.as_f32(), b.g
        for off, stride, width in ((b.q, b.sq, b.n_head * 128), (b.k, b.skv, b.dim), (b.v, b.skv, b.dim)):
            b.rows_of(off, stride, width)[:] = g.standard_normal((b.rows, width))
        x = [b.rows_of(o, s, w).astype(np.float64).reshape(b.rows, -1, 128)
             for o, s, w in ((b.q, b.sq, b.n_head * 128), (b.k, b.skv, b.dim), (b.v, b.skv, b.dim))]
        qn, kn, rope = b.norms
        for n in (qn, kn):
            f[n: n + 128] = g.uniform(0.5, 1.5, 128)
        f[rope: rope + 64] = THETA ** (-2.0 * np.arange(64) / 128)
        freq = f[rope: rope + 64].astype(np.float64)
        wq, wk = f[qn: qn + 128].astype(np.float64), f[kn: kn + 128].astype(np.float64)
        b.fill()
        before = [(e.copy(), None if s is None else s.copy()) for e, s in b.halves()]
        b.append()
        got = b.rows_of(b.out, b.sq, b.n_head * 128).astype(np.float64).reshape(b.rows, -1, 128)
        touched = []
        for r in range(b.rows):
            if lens[r] == 0:
                assert (got[r] == 7.5).all()
                continue
            # norm, product with the weight, two products and a sum of the rotation: 8 half steps of
            # 2^-24 of a pair's length, and the angle's 2e-7
            want = _rope64(x[0][r], wq, lens[r] - 1, freq)
            assert np.abs(got[r] - want).max() < 1e-6 * np.abs(want).max() * 4
            slot = b.table[b.seqs[r], (lens[r] - 1) // page] * page + (lens[r] - 1) % page
            touched.append(slot)
            for (e, s), y in zip(b.halves(), (_rope64(x[1][r], wk, lens[r] - 1, freq), x[2][r])):
                y = y.ravel()
                if s is None:
                    assert (np.abs(e[slot].astype(np.float64) - y) <= 2.0 ** -11 * np.abs(y) + 2e-6).all()
                else:  # half a step, the scale's rounding (2^-11 of 127 steps) and what k is off by
                    scale = np.repeat(s[slot].astype(np.float64), 32)
                    assert (np.abs(e[slot] * scale - y) <= (0.5 + 127 * 2.0 ** -11 + 1e-3) * scale).all()
                    assert np.allclose(s[slot], np.abs(y).reshape(-1, 32).max(1) / 127, rtol=2.0 ** -10)
        rest = np.setdiff1d(np.arange(b.n_pages * page), touched)
        for (e, s), (e0, s0) in zip(b.halves(), before):
            assert np.array_equal(e[rest], e0[rest]) and (s is None or np.array_equal(s[rest], s0[rest]))
        out = b.rows_of(b.out, b.sq, b.sq, b.grid)
        assert (out[b.rows:] == 7.5).all() and (out[:, b.n_head * 128:] == 7.5).all()
    finally:
        b.free()


def test_append_in_place_and_past_f16(ctx):
    """q rewritten where it lies; values past f16's largest stay finite, NaN stays NaN; a page that
    does not exist takes nothing."""
    b = Batch(ctx, P["f16"], 1, 2, 16, [3, 20, 9], parts=(0, 1))
    try:
        f = b.arena.as_f32()
        for off, stride, width in ((b.q, b.sq, b.n_head * 128), (b.k, b.skv, b.dim), (b.v, b.skv, b.dim)):
            b.rows_of(off, stride, width)[:] = b.g.standard_normal((b.rows, width))
        v = b.rows_of(b.v, b.skv, b.dim)
        v[0, :4] = 1e6, -np.inf, 65504, np.nan
        qn, kn, rope = b.norms
        f[qn: qn + 128] = f[kn: kn + 128] = 1
        f[rope: rope + 64] = 1
        b.arena.as_u32()[b.at.table + 2 * b.table.shape[1]] = b.n_pages  # row 2's page
        want = _rope64(b.rows_of(b.q, b.sq, 256).astype(np.float64).reshape(3, 2, 128), np.ones(128),
                       np.array([2, 19, 8])[:, None, None], np.ones(64))
        b.run(lambda r: b.kernels.append(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.q, b.sq), qn, kn, rope, 3))
        got = b.rows_of(b.q, b.sq, 256).reshape(3, 2, 128)
        assert np.abs(got - want).max() < 4e-6 * np.abs(want).max()
        (k, _), (vals, _) = b.halves()
        slot = b.table[0, 0] * 16 + 2
        assert np.array_equal(vals[slot, :4], np.array([65504, -65504, 65504, np.nan], np.float16), equal_nan=True)
        assert np.count_nonzero(np.abs(k).sum(1)) == 2  # rows 0 and 1 alone
    finally:
        b.free()


# ---- logits_adjust -----------------------------------------------------------------------------
def _adjust64(x, hist, n, prompt, bias, mask, rho, f, g):
    y, v = x.astype(np.float64), len(x)
    ids = hist[:n]
    seen = np.bincount(ids[ids < v], minlength=v) > 0
    late = ids[prompt:]
    made = np.bincount(late[late < v], minlength=v)
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(seen, np.where(y > 0, y / np.float64(rho), y * np.float64(rho)), y)
        y = np.where(made > 0, y - (np.float64(f) * made + np.float64(g)), y)
        for i, b in dict(bias).items():
            if i < v:
                y[i] += np.float64(b)
    if mask is not None:
        y[~mask] = -np.inf
    return y


@pytest.mark.parametrize("v", [1, 31, 4096, 4097, 32003])
@pytest.mark.parametrize("in_place", [False, True])
def test_logits_adjust(ctx, v, in_place):
    g = np.random.default_rng(v)
    rows, grid, h, nb = 7, 9, 300, 12
    sx, sm = _pad(v) + 4, -(-v // 32) + 1
    size, off = 64, {}
    for name, n in (("ctrl", 8 * grid), ("x", sx * grid), ("y", sx * grid), ("hist", h * grid), ("bias", 2 * nb * grid),
                    ("mask", sm * grid)):
        off[name], size = size, size + _pad(n)
    a = ctx.alloc_host(size * 4)
    k = B.LogitsKernels(ctx, a)
    try:
        f, u = a.as_f32(), a.as_u32()
        f[:] = 7.5
        u[:64] = 0
        u[2] = rows
        x = (g.standard_normal((rows, v)) * 4).astype(np.float32)
        x[1, v // 2] = -np.inf
        hist = g.integers(0, max(2, v // 3), (rows, h)).astype(np.uint32)
        hist[:, ::7] = v - 1
        hist[:, 3] = v + 5            # past the vocabulary
        n = np.array([0, 1, h, h, 250, h, 17])
        prompt = np.array([0, 0, 100, h, 300, 0, 5])
        par = np.array([[1.3, .2, .5], [1.3, .2, .5], [1.1, .3, 0], [2, 1, 1], [1, .25, .75], [1, 0, 0], [0.7, -.5, -.1]], np.float32)
        bias = [[(int(i), np.float32(b)) for i, b in zip(g.integers(0, v + 3, nb), g.standard_normal(nb) * 9)] for _ in range(rows)]
        bias[4] = [(v - 1, np.float32(1)), (v - 1, np.float32(-np.inf)), (v - 1, np.float32(3))]  # the last entry counts
        bias[0] = []
        bits = g.random((rows, v)) < 0.5
        bits[2] = False               # a grammar with no way on
        masked = np.array([1, 0, 1, 1, 0, 1, 0])
        for r in range(rows):
            f[off["x"] + r * sx: off["x"] + r * sx + v] = x[r]
            u[off["hist"] + r * h: off["hist"] + (r + 1) * h] = hist[r]
            for i, (t, b) in enumerate(bias[r]):
                u[off["bias"] + 2 * nb * r + 2 * i] = t
                f[off["bias"] + 2 * nb * r + 2 * i + 1] = b
            packed = np.packbits(np.concatenate([bits[r], np.zeros(-v % 32, bool)]), bitorder="little").view("<u4")
            u[off["mask"] + r * sm: off["mask"] + r * sm + len(packed)] = packed
            c = off["ctrl"] + 8 * r
            u[c: c + 4] = n[r], prompt[r], len(bias[r]), masked[r]
            f[c + 4: c + 7] = par[r]
        u[off["ctrl"] + 8 * 3] = 1 << 31  # a history longer than its row: cut there
        a.upload()
        y = off["x"] if in_place else off["y"]
        at = B.LogitsRegions(off["ctrl"], off["hist"], h, off["bias"], 2 * nb, off["mask"], sm)
        rec = ctx.record(False, lambda r: k.adjust(r, at, (off["x"], sx), (y, sx), v, grid))
        ctx.replay(rec)
        rec.free()
        a.download()
        out = a.as_f32()[y: y + sx * grid].reshape(grid, sx)
        for r in range(rows):
            want = _adjust64(x[r], hist[r], n[r], prompt[r], bias[r], bits[r] if masked[r] else None, *par[r])
            got = out[r, :v]
            fin = np.isfinite(want)
            assert np.array_equal(np.isneginf(got), np.isneginf(want)), r
            # one rounding for each of the four steps, of numbers up to the largest on the way
            top = np.abs(x[r][np.isfinite(x[r])]).max(initial=0) * 2 + 300 + 40
            assert np.abs(got[fin] - want[fin]).max(initial=0) <= 4 * 2.0 ** -24 * top, r
            assert (out[r, v:] == 7.5).all()
        assert (out[rows:] == 7.5).all()
    finally:
        k.free()
        a.free()


def test_refused_words(ctx):
    """Words that would leave the buffers are refused before anything is launched."""
    b = Batch(ctx, P["f16"], 2, 2, 16, [5, 6])
    try:
        for bad in (dict(q=(b.arena.size // 4, 512)), dict(q=(b.q + 1, b.sq)), dict(out=(b.at.part, b.sq)),
                    dict(rows=70000), dict(parts=(0, 0)), dict(parts=(1000, 1000)), dict(out=(b.out, 100))):
            args = dict(q=(b.q, b.sq), out=(b.out, b.sq), rows=2, parts=b.parts) | bad
            with pytest.raises(SkylaHipError) as e:
                ctx.record(False, lambda r: b.kernels.attend(r, 0, b.at, **args))
            assert e.value.code == -1 and "attention_paged" in e.value.message
    finally:
        b.free()


# ---- together, as a decode step runs them ------------------------------------------------------
@pytest.mark.parametrize("precision", list(P))
def test_a_recorded_step_replayed(ctx, precision):
    """Append and attend of four layers (here the same pool) as one HIP graph, replayed as the
    sequences grow, pages are handed out and rows fall idle, against direct launches: the same
    bits; and against 64 bits."""
    b = Batch(ctx, P[precision], 2, 4, 16, [40, 33, 90, 70, 1], shares=[32] * 5, shared=32, parts=(2, 3, True), n_pages=60)
    try:
        g, f, u = b.g, b.arena.as_f32(), b.arena.as_u32()
        b.fill()
        b.copy_shared()
        qn, kn, rope = b.norms
        for n in (qn, kn):
            f[n: n + 128] = g.uniform(0.5, 1.5, 128)
        f[rope: rope + 64] = THETA ** (-2.0 * np.arange(64) / 128)
        b.arena.upload()
        b.pool.upload()

        def body(r):
            for _ in range(4):
                b.kernels.append(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.q, b.sq), qn, kn, rope, b.grid)
                r.barrier()
                b.kernels.attend(r, 0, b.at, (b.q, b.sq), (b.out, b.sq), b.grid, b.parts)
                r.barrier()
        with tactics(nograph="0"):
            graph = ctx.record(False, body)
        with tactics(nograph="1"):
            direct = ctx.record(False, body)
        assert graph.launches() == 12
        for step in range(5):
            lens = b.lens + step
            lens[step % 4] = 0 if step else lens[0]
            u[b.at.rows + 1: b.at.rows + 4 * b.rows: 4] = lens
            x = [g.standard_normal((b.rows, w)).astype(np.float32) for w in (b.n_head * 128, b.dim, b.dim)]
            outs = []
            for rec in (direct, graph):
                for (off, stride), rows in zip(((b.q, b.sq), (b.k, b.skv), (b.v, b.skv)), x):
                    b.rows_of(off, stride, rows.shape[1])[:] = rows
                b.arena.upload()
                ctx.replay(rec)
                b.arena.download()
                outs.append((b.rows_of(b.out, b.sq, b.n_head * 128).copy(), b.rows_of(b.q, b.sq, b.n_head * 128).copy()))
            assert np.array_equal(*[o[0] for o in outs]) and np.array_equal(*[o[1] for o in outs])
            b.pool.download()
            keep, b.lens = b.lens, lens
            want = b.want().reshape(b.rows, -1)
            b.lens = keep
            for r in range(b.rows):
                assert np.linalg.norm(outs[0][0][r] - want[r]) <= BAR * np.linalg.norm(want[r]), (step, r)
        graph.free()
        direct.free()
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("wide", [False, True])
def test_pages_at_the_end_of_a_large_pool(ctx, precision, wide):
    """A pool of nearly 4 GiB, the sequences in its last pages: the bits of the same rows in a small
    pool (offsets past 2^31 entries and bytes)."""
    n_kv, page = 8, 4096
    bits = P[precision]
    per = sum((n_kv * 128 + n_kv * 8) if q8 else 2 * n_kv * 128 for q8 in (bits.keys_q8, bits.values_q8))
    far = (4 << 30) // (per * page)
    lens, shares = [130, 4200, 200], [100] * 3
    small = Batch(ctx, bits, n_kv, 2, page, lens, shares=shares, shared=100, parts=(1, 1, wide), n_pages=6, seed=4)
    big = Batch(ctx, bits, n_kv, 2, page, lens, shares=shares, shared=100, parts=(1, 1, wide), n_pages=far, seed=4)
    try:
        assert small.table.max() < 6
        small.fill()
        small.copy_shared()
        q = small.g.standard_normal((3, small.n_head * 128)).astype(np.float32)
        k, v = (small.g.standard_normal((3, small.dim)).astype(np.float32) for _ in range(2))
        small.pool.upload()
        # page i of the small pool lies in page far - 6 + i of the large one
        for off, sc, q8 in (("keys", "key_scales", bits.keys_q8), ("values", "value_scales", bits.values_q8)):
            for name, size, width in ((off, 1 if q8 else 2, small.dim), (sc, 2, small.dim // 32)) if q8 else ((off, 2, small.dim),):
                a, z = (getattr(x.paged.layout, name)(0) * size for x in (small, big))
                n = page * width * size
                big.pool.copy_from(z + (far - 6) * n, small.pool, a, 6 * n)
        outs = []
        for b, first in ((small, 0), (big, far - 6)):
            f, u = b.arena.as_f32(), b.arena.as_u32()
            u[b.at.table: b.at.table + b.table.size] = small.table.ravel() + first
            qn, kn, rope = b.norms
            f[qn: qn + 128] = f[kn: kn + 128] = 1.25
            f[rope: rope + 64] = 0.01
            b.rows_of(b.q, b.sq, q.shape[1])[:] = q
            b.rows_of(b.k, b.skv, b.dim)[:] = k
            b.rows_of(b.v, b.skv, b.dim)[:] = v
            b.arena.upload()

            def body(r, b=b):
                b.kernels.append(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.q, b.sq), qn, kn, rope, 3)
                r.barrier()
                b.kernels.attend(r, 0, b.at, (b.q, b.sq), (b.out, b.sq), 3, b.parts)
            rec = ctx.record(False, body)
            ctx.replay(rec)
            rec.free()
            b.arena.download()
            outs.append(b.rows_of(b.out, b.sq, b.n_head * 128).copy())
        assert np.isfinite(outs[0]).all() and np.array_equal(*outs)
    finally:
        small.free()
        big.free()


def test_attention_in_place(ctx):
    """The output over the queries, with one part (written by the attention) and with several."""
    for parts in ((0, 1), (1, 1, True), (1, 2)):
        b = Batch(ctx, P["f16k_q8v"], 2, 4, 32, [60, 45, 0, 130], shares=[40] * 4, shared=40, parts=parts)
        try:
            b.fill()
            b.copy_shared()
            b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
            want = b.want()
            b.run(lambda r: b.kernels.attend(r, 0, b.at, (b.q, b.sq), (b.q, b.sq), b.grid, b.parts))
            got = b.rows_of(b.q, b.sq, b.n_head * 128).astype(np.float64).reshape(want.shape)
            for r in range(b.rows):
                assert np.linalg.norm(got[r] - want[r]) <= BAR * np.linalg.norm(want[r]), (parts, r)
        finally:
            b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("heads,grid", [((2, 1), 4100), ((16, 4), 690)])
def test_append_of_many_rows(ctx, precision, heads, grid):
    """A launch of many rows, most of them idle, against one of the live rows alone: the same bits in
    the output and in the pool, nothing written for the rest."""
    b = Batch(ctx, P[precision], *heads, 16, [5, 0, 17, 100, 64], seed=3, grid=grid, parts=(0, 1))
    try:
        f = b.arena.as_f32()
        for off, stride, width in ((b.q, b.sq, b.n_head * 128), (b.k, b.skv, b.dim), (b.v, b.skv, b.dim)):
            b.rows_of(off, stride, width, grid)[:] = b.g.standard_normal((grid, width))
        qn, kn, rope = b.norms
        f[qn: qn + 128] = f[kn: kn + 128] = b.g.uniform(0.5, 1.5, 128)
        f[rope: rope + 64] = THETA ** (-2.0 * np.arange(64) / 128)
        b.fill()
        pool, out = b.pool.host().copy(), b.rows_of(b.out, b.sq, b.sq, grid).copy()
        got = []
        for rows in (b.rows, grid):
            b.pool.host()[:] = pool
            b.rows_of(b.out, b.sq, b.sq, grid)[:] = out
            b.run(lambda r: b.kernels.append(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.out, b.sq), qn, kn, rope, rows))
            got.append((b.rows_of(b.out, b.sq, b.sq, grid).copy(), b.pool.host().copy()))
        (o, p), (o_many, p_many) = got
        assert np.array_equal(o, o_many) and np.array_equal(p, p_many)
        assert not np.array_equal(o[0], out[0]) and (o[b.rows:] == 7.5).all() and not np.array_equal(p, pool)
    finally:
        b.free()


@pytest.mark.parametrize("v", [1, 16384, 16385, 40001])
def test_logits_adjust_of_long_histories(ctx, v):
    """Histories of none, one and thousands of tokens, the same ones thousands of times."""
    g = np.random.default_rng(v)
    rows, grid, h, nb = 6, 7, 9004, 3
    sx, sm = _pad(v), -(-v // 32)
    size, off = 64, {}
    for name, n in (("ctrl", 8 * grid), ("x", sx * grid), ("hist", h * grid), ("bias", 2 * nb * grid), ("mask", sm * grid)):
        off[name], size = size, size + _pad(n)
    a = ctx.alloc_host(size * 4)
    k = B.LogitsKernels(ctx, a)
    try:
        f, u = a.as_f32(), a.as_u32()
        f[:] = 7.5
        u[:64] = 0
        u[2] = rows
        x = (g.standard_normal((rows, v)) * 4).astype(np.float32)
        hist = np.minimum(g.integers(0, v + 5, (rows, h)), g.integers(0, v + 5, (rows, h))).astype(np.uint32)
        hist[3] = v - 1
        n, prompt = np.array([0, 1, h, h, 8999, 4097]), np.array([0, 0, 1000, 0, 9004, 4096])
        par = np.array([[1.25, .01, .5]] * rows, np.float32)
        bits = g.random((rows, v)) < 0.5
        bias = [[(v - 1, np.float32(2.5)), (v, np.float32(1))]] * rows
        for r in range(rows):
            f[off["x"] + r * sx: off["x"] + r * sx + v] = x[r]
            u[off["hist"] + r * h: off["hist"] + (r + 1) * h] = hist[r]
            for i, (t, w) in enumerate(bias[r]):
                u[off["bias"] + 2 * nb * r + 2 * i] = t
                f[off["bias"] + 2 * nb * r + 2 * i + 1] = w
            packed = np.packbits(np.concatenate([bits[r], np.zeros(-v % 32, bool)]), bitorder="little").view("<u4")
            u[off["mask"] + r * sm: off["mask"] + r * sm + len(packed)] = packed
            c = off["ctrl"] + 8 * r
            u[c: c + 4] = n[r], prompt[r], len(bias[r]), r & 1
            f[c + 4: c + 7] = par[r]
        a.upload()
        at = B.LogitsRegions(off["ctrl"], off["hist"], h, off["bias"], 2 * nb, off["mask"], sm)
        rec = ctx.record(False, lambda r: k.adjust(r, at, (off["x"], sx), (off["x"], sx), v, grid))
        ctx.replay(rec)
        rec.free()
        a.download()
        out = a.as_f32()[off["x"]: off["x"] + sx * grid].reshape(grid, sx)
        for r in range(rows):
            want, got = _adjust64(x[r], hist[r], n[r], prompt[r], bias[r], bits[r] if r & 1 else None, *par[r]), out[r, :v]
            fin = np.isfinite(want)
            assert np.array_equal(np.isneginf(got), np.isneginf(want)), r
            # one rounding for each of the four steps (a product, f made and its sum with g, two sums)
            # of numbers up to the largest on the way: 30 and 9004 times 0.01 here
            assert np.abs(got[fin] - want[fin]).max(initial=0) <= 5 * 2.0 ** -24 * 130, r
            assert (out[r, v:] == 7.5).all()
        assert (out[rows:] == 7.5).all()
    finally:
        k.free()
        a.free()


class _Direct:
    """A recorder's calls as single dispatches, or as timed ones of the same words."""

    def __init__(self, ctx, reps):
        self.ctx, self.reps = ctx, reps

    def dispatch(self, p, groups, push):
        if self.reps:
            ns = self.ctx.time_dispatch(p, groups, push, self.reps)
            assert len(ns) == self.reps and min(ns) > 0
        else:
            self.ctx.dispatch_noalloc(p, groups, push)

    def dispatch_set(self, p, i, groups, push):
        assert i == 0
        self.dispatch(p, groups, push)

    def barrier(self):
        pass


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("reps", [0, 3])
@pytest.mark.parametrize("parts", [(1, 2, True), (2, 1), (3, 30)])
def test_single_dispatches(ctx, precision, reps, parts):
    """dispatch_noalloc and time_dispatch of the operators: the bits of a recording, the same refusals."""
    b = Batch(ctx, P[precision], 2, 4, 16, [140, 33, 0, 70, 45], shares=[32] * 5, shared=32, parts=parts, grid=7)
    try:
        f = b.arena.as_f32()
        for off, stride, width in ((b.q, b.sq, b.n_head * 128), (b.k, b.skv, b.dim), (b.v, b.skv, b.dim)):
            b.rows_of(off, stride, width)[:] = b.g.standard_normal((b.rows, width))
        qn, kn, rope = b.norms
        f[qn: qn + 128] = f[kn: kn + 128] = 1
        f[rope: rope + 64] = THETA ** (-2.0 * np.arange(64) / 128)
        b.fill()
        b.copy_shared()

        def step(r):  # the queries stay raw, so that it can run any number of times
            b.kernels.append(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.out, b.sq), qn, kn, rope, b.grid)
            r.barrier()
            b.kernels.attend(r, 0, b.at, (b.q, b.sq), (b.out, b.sq), b.grid, parts)
        start, pool = f.copy(), b.pool.host().copy()
        b.run(step)
        want, stored = b.rows_of(b.out, b.sq, b.sq, b.grid).copy(), b.pool.host().copy()
        f[:], b.pool.host()[:] = start, pool
        b.arena.upload()
        b.pool.upload()
        step(_Direct(ctx, reps))
        b.arena.download()
        b.pool.download()
        assert np.array_equal(b.rows_of(b.out, b.sq, b.sq, b.grid), want) and np.array_equal(b.pool.host(), stored)
        assert not np.array_equal(stored, pool) and np.isfinite(want[: b.rows, : b.n_head * 128]).all()
        with pytest.raises(SkylaHipError) as e:
            b.kernels.attend(_Direct(ctx, reps), 0, b.at, (b.arena.size // 4, 1024), (b.out, b.sq), b.grid, parts)
        assert e.value.code == -1
    finally:
        b.free()
