"""The batch operators where their number formats end: scales of a cache far apart, weights' rounding,
what an 8-bit cache makes of NaN, infinities and values past its largest."""
import numpy as np
import pytest

from test_gpu_batch import Batch, P

pytestmark = pytest.mark.gpu


def _reference(b):
    """The rows' attention in 64 bits, and that of the values' sizes: (o, sum p |v|)."""
    q = b.rows_of(b.q, b.sq, b.n_head * 128).astype(np.float64).reshape(b.rows, b.n_head, 128)
    o, size = np.zeros((2, b.rows, b.n_head, 128))
    for r in range(b.rows):
        K, V = b.read64(b.slots(b.seqs[r], int(b.lens[r])))
        for h in range(b.n_head):
            s = K[:, h // b.rep] @ q[r, h] / np.sqrt(128.0)
            p = np.exp(s - s.max())
            p /= p.sum()
            o[r, h], size[r, h] = p @ V[:, h // b.rep], p @ np.abs(V[:, h // b.rep])
    return o, size


def _two_kinds(b, small, gap):
    """Keys and queries along one direction: positions of `small` score `gap` nats above the others."""
    u = np.where(b.g.random(128) < 0.5, -1.0, 1.0)
    # q . k / sqrt(128) = +- gap / 2 for q = gap / (4 * 128) sqrt(128) u, k = +- 2 u
    b.rows_of(b.q, b.sq, b.n_head * 128)[:] = np.tile(u * gap / (4 * np.sqrt(128.0)), (b.rows, b.n_head))
    (k, ks), _ = b.halves()
    sign = np.where(small, 1, -1)[:, None]
    if ks is None:
        k[:] = sign * np.tile(2 * u, b.n_kv)
    else:
        k[:] = sign * np.tile(64 * u, b.n_kv).astype(int)
        ks[:] = 2.0 ** -5


@pytest.mark.parametrize("precision", ["q8", "f16k_q8v"])
@pytest.mark.parametrize("form", ["own", "narrow", "wide"])
@pytest.mark.parametrize("order", ["first", "last", "mixed"])
def test_scales_far_apart(ctx, precision, form, order):
    """Values with scales from 2^-20 to 2^12 in one run, the rows attending to the small ones: what a row
    leaves out does not cost what it takes its bits."""
    shared = 0 if form == "own" else 400
    lens = [400 + n for n in (1, 77, 33)]
    b = Batch(ctx, P[precision], 2, 4, 16, lens, shares=[shared] * 3, shared=shared, wide=form == "wide",
              parts=None if form == "own" else (2, 1))
    try:
        b.fill()
        small = np.zeros(b.n_pages * b.page, bool)
        for r in range(3):
            at = b.slots(r, lens[r])
            place = {"first": np.arange(lens[r]) < 130, "last": np.arange(lens[r]) >= 330,
                     "mixed": b.g.random(lens[r]) < 0.3}[order]
            if r and shared:
                place[:shared] = small[b.slots(0, shared)]
            small[at] = place
        _two_kinds(b, small, 100.0)
        _, (v, vs) = b.halves()
        vs[:] = np.where(small[:, None], 2.0 ** b.g.uniform(-20, -16, vs.shape), 2.0 ** b.g.uniform(8, 12, vs.shape))
        vs[::5, ::3] = 0    # and blocks of nothing
        if shared:
            b.copy_shared()
        want, size = _reference(b)
        assert 0 < np.linalg.norm(want) < 1e-2  # the others' weight is 1e-43
        got = b.attend()
        # queries and keys are exact, so a score is off by f32's sum: 2^-24 of 72 powers of two a product,
        # common to the positions of a kind.  Weights are within 2^-23, values exact, f32 sums of n <= 477
        # terms within sqrt(n) 2^-24 of sum p |v|: 2e-6 in all
        for r in range(3):
            for h in range(b.n_head):
                for k in range(0, 128, 32):
                    d = slice(k, k + 32)
                    assert np.linalg.norm(got[r, h, d] - want[r, h, d]) <= 2e-6 * np.linalg.norm(size[r, h, d]), (r, h, k)
    finally:
        b.free()


@pytest.mark.parametrize("precision", ["f16", "f16k_q8v"])
@pytest.mark.parametrize("form", ["own", "narrow", "wide"])
def test_weights_far_below_the_largest(ctx, precision, form):
    """Values 2^16 times the others' where the weights are 2^-20: a weight is held to 2^-32 of the row's
    largest, so their share, a sixteenth of the sum, to 2^-12."""
    shared = 0 if form == "own" else 256
    b = Batch(ctx, P[precision], 1, 4, 16, [300, 290], shares=[shared] * 2, shared=shared, wide=form == "wide",
              parts=None if form == "own" else (1, 1))
    try:
        b.fill()
        small = b.g.random(b.n_pages * b.page) < 0.5
        gap = 20.37 * np.log(2.0)
        _two_kinds(b, small, gap)
        _, (v, vs) = b.halves()
        if vs is None:
            v[:] = np.where(small[:, None], 0.25, 2.0 ** 14) * b.g.uniform(0.5, 1, v.shape)
        else:
            v[:] = b.g.integers(64, 128, v.shape)
            vs[:] = np.where(small[:, None], 2.0 ** -9, 2.0 ** 7)
        if shared:
            b.copy_shared()
        want, size = _reference(b)
        got = b.attend()
        # the big values' weights 2^-20.4 +- 2^-32 each (alike, so off alike): 2^-11.6 of a share of 2^16
        # 2^-20.4 of the sum are 1.6e-5 of it; weights 2^-23, f32 sums sqrt(300) 2^-24, scores (20 powers of
        # two) 20 2^-24 ln 2: 3e-6
        assert (np.abs(got - want) <= 2e-5 * size).all()
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("form", ["own", "narrow", "wide"])
def test_one_position_is_its_value(ctx, precision, form):
    """A weight's two parts hold all of it (of one position the largest), so the quotient is the value
    to a rounding of the product and one of the quotient."""
    shared = 0 if form == "own" else 1
    rows = 64
    b = Batch(ctx, P[precision], 2, 2, 16, [1] * rows, shares=[shared] * rows, shared=shared, wide=form == "wide",
              parts=(0, 1) if form == "own" else (1, 1))
    try:
        b.fill()
        b.copy_shared()
        q = b.rows_of(b.q, b.sq, b.n_head * 128)
        q[:] = b.g.standard_normal(q.shape) * 3
        want, _ = _reference(b)
        got = b.attend()
        assert (np.abs(got - want) <= 2.0 ** -23 * np.abs(want)).all()
    finally:
        b.free()


def test_an_8_bit_cache_of_no_numbers_and_large_ones(ctx):
    """A block of 32 that holds a NaN is NaN; an infinity or a value past 127 of the largest scale is
    held as that, and the block's other values to half a step of it."""
    b = Batch(ctx, P["q8"], 1, 2, 16, [3, 20], parts=(0, 1))
    try:
        f = b.arena.as_f32()
        for off, stride, width in ((b.q, b.sq, b.n_head * 128), (b.k, b.skv, b.dim), (b.v, b.skv, b.dim)):
            b.rows_of(off, stride, width)[:] = b.g.standard_normal((b.rows, width))
        v, k = b.rows_of(b.v, b.skv, b.dim), b.rows_of(b.k, b.skv, b.dim)
        v[0, 5] = np.nan
        v[0, 32:36] = 1e9, 8e6, -2e5, 40000
        v[0, 64:67] = np.inf, -np.inf, -7e6
        v[1, 96:98] = np.nan, np.inf
        k[1, 7] = np.nan
        qn, kn, rope = b.norms
        f[qn: qn + 128] = f[kn: kn + 128] = 1
        f[rope: rope + 64] = 1
        b.run(lambda r: b.kernels.append(r, 0, b.at, (b.q, b.sq), (b.k, b.skv), b.v, (b.out, b.sq), qn, kn, rope, 2))
        (_, ks), (e, s) = b.halves()
        top = 127 * 65504.0
        for r, nan in ((0, [0]), (1, [3])):
            slot = b.table[r, (b.lens[r] - 1) // 16] * 16 + (b.lens[r] - 1) % 16
            for blk in range(4):
                d = slice(32 * blk, 32 * blk + 32)
                if blk in nan:
                    assert np.isnan(s[slot, blk])
                    continue
                step = float(s[slot, blk])
                y = np.clip(v[r, d].astype(np.float64), -top, top)
                assert 0 < step <= 65504
                # half a step, and the scale's own rounding of at most 127 steps
                assert (np.abs(e[slot, d] * step - y) <= (0.5 + 127 * 2.0 ** -11 + 1e-6) * step).all(), (r, blk)
            if r == 1:  # a NaN in a key makes its norm one: the whole head
                assert np.isnan(ks[slot]).all()
    finally:
        b.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("half", ["keys", "values"])
def test_a_row_that_attends_to_no_number(ctx, precision, half):
    """NaN at a position of one row's own run: what it reaches of that row is NaN, nothing else."""
    shared = 40
    b = Batch(ctx, P[precision], 2, 2, 16, [90, 70, 140], shares=[shared] * 3, shared=shared)
    try:
        b.fill()
        b.copy_shared()
        b.rows_of(b.q, b.sq, b.n_head * 128)[:] = b.g.standard_normal((b.rows, b.n_head * 128))
        want = b.want()
        e, s = b.halves()[half == "values"]
        at = b.slots(1, 70)[55]
        (e if s is None else s)[at, (128 + 35) // (1 if s is None else 32)] = np.nan  # dim 35 of key head 1
        got = b.attend()
        bad = np.zeros(want.shape, bool)
        if half == "keys":
            bad[1, 2:] = True
        else:
            bad[1, 2:, 35 if s is None else slice(32, 64)] = True
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
        assert np.abs(got - want)[~bad].max() <= 4e-6 * np.abs(want).max()
    finally:
        b.free()
