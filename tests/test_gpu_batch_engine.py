"""Sequences decoded together (batch.BatchEngine) against the oracle's Model, one by one: prompts
of several chunks, forks that share pages, idle rows, controls on the logits, and what the engine
refuses."""
import numpy as np
import pytest

from helpers import rel_l2
from oracle.model import Model
from skyla_hip import batch as B
from skyla_hip import engine as E
from skyla_hip import synth

pytestmark = pytest.mark.gpu

P = E.KvPrecision
KV = {P.F16: (False, False), P.Q8: (True, True), P.F16_KEYS_Q8_VALUES: (False, True)}
# Rows of a batch go through the matrix cores with f16 activations (6e-4 a product); through three
# layers the logits stay within the bar that the smoke run holds a model of this size to.
BAR = 2e-2


def _oracle(c, tensors, precision, tokens):
    m = Model(c, tensors, KV[precision])
    return np.stack([m.forward(t) for t in tokens])


def _tokens(g, c, n):
    return [int(t) for t in g.integers(0, c.n_vocab, n)]


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("quant,page", [("q8_0", 16), ("q4_k_m", 64)])
def test_sequences_of_different_lengths(ctx, precision, quant, page):
    c, g = synth.qwen3_config("tiny"), np.random.default_rng(5)
    tensors = synth.qwen3("test-batch", c, quant, "random")
    prompts = [_tokens(g, c, n) for n in (3, 140, 1, 17)]
    more = [_tokens(g, c, 3) for _ in prompts]
    eng = B.BatchEngine(ctx, tensors, c, 256, 64, page, precision, max_seq=6)
    try:
        seqs = [eng.open() for _ in prompts]
        assert seqs == [0, 1, 2, 3]
        for q, p in zip(seqs, prompts):
            eng.extend(q, p[:-1])
        got = [eng.step({q: p[-1] for q, p in zip(seqs, prompts)}, prompt=seqs)]
        for i in range(3):  # the second step leaves two sequences out
            live = seqs if i != 1 else [3, 1]
            got.append(eng.step({q: more[q][i] for q in live}))
        want = [_oracle(c, tensors, precision, p + (m if q in (1, 3) else [m[0], m[2]]))[len(p) - 1:]
                for q, (p, m) in enumerate(zip(prompts, more))]
        for i, out in enumerate(got):
            for row, q in zip(out, seqs if i != 2 else [3, 1]):
                k = i if q in (1, 3) else [0, 1, None, 2][i]
                assert rel_l2(row, want[q][k]) < BAR, (i, q)
        assert [eng.length(q) for q in seqs] == [5, 143, 3, 20]
    finally:
        eng.free()


def test_one_sequence_as_the_engine_decodes_it(ctx):
    """Alone, a sequence's rows go through the decode matvecs: the engine's logits to the order of sums."""
    c = synth.qwen3_config("tiny")
    tensors = synth.qwen3("test-batch", c, "q4_k_m", "random")
    tokens = _tokens(np.random.default_rng(6), c, 70)
    one, eng = E.Engine(ctx, tensors, c, 128), B.BatchEngine(ctx, tensors, c, 128, 8, 16)
    try:
        q = eng.open()
        for t in tokens:
            assert rel_l2(eng.step({q: t})[0], one.step(t)) < 1e-4
    finally:
        one.free()
        eng.free()


@pytest.mark.parametrize("precision", list(P))
def test_forks_share_their_pages(ctx, precision):
    c, g = synth.qwen3_config("tiny"), np.random.default_rng(7)
    tensors = synth.qwen3("test-batch", c, "q8_0", "random")
    prompt = _tokens(g, c, 75)
    eng = B.BatchEngine(ctx, tensors, c, 200, 40, 16, precision, max_seq=8)
    try:
        first = eng.open()
        alone = eng.open()          # shares nothing
        eng.extend(first, prompt)
        eng.extend(alone, prompt[:9])
        free = len(eng.free_pages)
        forks = [first] + [eng.fork(first) for _ in range(3)]
        assert free - len(eng.free_pages) == 3  # four whole pages shared, the last one's own
        assert eng.shared_run(forks + [alone]) == (64, forks)
        history = {q: list(prompt) for q in forks} | {alone: prompt[:9]}
        for _ in range(3):
            step = {q: t for q, t in zip([alone] + forks, _tokens(g, c, 5))}
            out = eng.step(step)
            for row, (q, t) in zip(out, step.items()):
                history[q].append(t)
                assert rel_l2(row, _oracle(c, tensors, precision, history[q])[-1]) < BAR, q
        # the first goes; what its forks share stays theirs
        eng.close(first)
        out = eng.step({forks[1]: 5, forks[3]: 6})
        for row, (q, t) in zip(out, ((forks[1], 5), (forks[3], 6))):
            history[q].append(t)
            assert rel_l2(row, _oracle(c, tensors, precision, history[q])[-1]) < BAR
        for q in list(eng.sequences):
            eng.close(q)
        assert len(eng.free_pages) == 40 and not eng.uses.any()
    finally:
        eng.free()


def test_experts(ctx):
    c, g = synth.qwen3_config("tiny-moe"), np.random.default_rng(8)
    tensors = synth.qwen3moe("test-batch-moe", c)
    eng = B.BatchEngine(ctx, tensors, c, 64, 16, 16, max_seq=4)
    try:
        a, b = eng.open(), eng.open()
        ta, tb = _tokens(g, c, 20), _tokens(g, c, 6)
        eng.extend(a, ta[:-1])
        eng.extend(b, tb[:-1])
        out = eng.step({a: ta[-1], b: tb[-1]})
        for row, t in zip(out, (ta, tb)):
            assert rel_l2(row, _oracle(c, tensors, P.F16_KEYS_Q8_VALUES, t)[-1]) < BAR
    finally:
        eng.free()


def test_controls(ctx):
    """Each sequence's controls act on its own logits, over its own tokens."""
    c, g = synth.qwen3_config("tiny"), np.random.default_rng(9)
    tensors = synth.qwen3("test-batch", c, "q8_0", "random")
    plain, eng = (B.BatchEngine(ctx, tensors, c, 64, 16, 16, max_seq=4) for _ in range(2))
    allowed = g.random(c.n_vocab) < 0.3
    controls = [B.Controls(repetition=1.5), B.Controls(frequency=0.5, presence=1.0, bias={7: 3.0, 9: -np.inf}),
                B.Controls(allowed=allowed), B.Controls(repetition=0.8, frequency=-0.25, bias={3: 1.0}, allowed=~allowed)]
    try:
        prompts = [_tokens(g, c, n) for n in (5, 12, 1, 30)]
        for e in (plain, eng):
            for p in prompts:
                e.extend(e.open(), p)
        for q, k in enumerate(controls):
            eng.control(q, k)
        made = {q: [] for q in range(4)}
        for i in range(3):
            step = {q: (made[q][-1] if i == 2 else _tokens(g, c, 1)[0]) for q in range(4)}  # repeated once
            for q, t in step.items():
                made[q].append(t)
            raw, got = plain.step(step), eng.step(step)
            for q, k in enumerate(controls):
                y = raw[q].astype(np.float64)
                seen = np.zeros(c.n_vocab, bool)
                seen[prompts[q] + made[q]] = True
                count = np.bincount(made[q], minlength=c.n_vocab)
                y = np.where(seen, np.where(y > 0, y / k.repetition, y * k.repetition), y)
                y -= k.frequency * count + k.presence * (count > 0)
                for t, b in k.bias.items():
                    y[t] += b
                if k.allowed is not None:
                    y[~k.allowed] = -np.inf
                assert np.array_equal(np.isneginf(got[q]), np.isneginf(y))
                fin = np.isfinite(y)
                assert np.abs(got[q][fin] - y[fin]).max() <= 4 * 2.0 ** -24 * (np.abs(y[fin]).max() + 8)
        eng.control(2, B.Controls())
        assert np.isfinite(eng.step({2: 1})).all()
    finally:
        plain.free()
        eng.free()


def test_refusals_leave_the_sequences_as_they_were(ctx):
    c = synth.qwen3_config("tiny")
    tensors = synth.qwen3("test-batch", c, "q8_0", "random")
    for bad in (dict(max_ctx=0), dict(n_pages=0), dict(page=24), dict(max_seq=0), dict(max_seq=129)):
        with pytest.raises(ValueError):
            B.BatchEngine(ctx, tensors, c, **(dict(max_ctx=64, n_pages=4, page=16) | bad))
    eng = B.BatchEngine(ctx, tensors, c, 40, 4, 16, max_seq=2)
    try:
        a, b = eng.open(), eng.open()
        with pytest.raises(ValueError):
            eng.open()
        eng.extend(a, range(30))
        eng.extend(b, range(16))
        for call in (lambda: eng.fork(a), lambda: eng.step({}), lambda: eng.step({2: 1}), lambda: eng.step({a: c.n_vocab}),
                     lambda: eng.step({a: -1}), lambda: eng.extend(a, range(11)), lambda: eng.step({a: 1}, prompt=[b]),
                     lambda: eng.extend(b, range(17)), lambda: eng.close(7), lambda: eng.control(a, B.Controls(repetition=0)),
                     lambda: eng.control(a, B.Controls(bias={c.n_vocab: 1.0})), lambda: eng.control(a, B.Controls(bias={1: np.nan})),
                     lambda: eng.control(a, B.Controls(allowed=np.ones(3, bool))),
                     lambda: eng.control(a, B.Controls(frequency=np.inf))):
            with pytest.raises(ValueError):
                call()
            assert (eng.length(a), eng.length(b), len(eng.free_pages)) == (30, 16, 1)
        eng.extend(a, [])
        want = eng.step({a: 5, b: 6})
        eng.close(b)
        assert eng.open() == b
        eng.extend(b, range(16))
        assert rel_l2(eng.step({b: 6})[0], want[1]) < BAR
        with pytest.raises(ValueError):
            eng.step({a: 1, 5: 1})
        assert eng.length(a) == 31
    finally:
        eng.free()
