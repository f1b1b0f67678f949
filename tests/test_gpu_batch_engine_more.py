"""What BatchEngine serves beyond the reference's models, against the same in 64 bits: shaped scores,
documents and prefixes, rotary positions of several axes with rows given as vectors, drawn tokens."""
import dataclasses

import numpy as np
import pytest

from helpers import rel_l2
from model64 import Model64, _rms
from oracle import skyla_oracle as so
from skyla_hip import batch as B
from skyla_hip import engine as E
from skyla_hip import synth
from test_gpu_batch_engine import BAR, KV
from test_gpu_sample import want

pytestmark = pytest.mark.gpu

P = E.KvPrecision


class Model(Model64):
    """Model64 over chunks of rows, which attend as BatchEngine.extend says, with the cache held as the engine
    holds it (f16, or 8 bits and a scale for each 32)."""

    kv = (False, False)

    def stored(self, rows, q8):
        return [so.kv_stored(np.ascontiguousarray(r, np.float32).reshape(-1), q8).astype(np.float64).reshape(r.shape) for r in rows]

    def extend(self, tokens, axes=None, vectors=None, since=0, together=False):
        """The logits after each row."""
        c, w, hd = self.c, self.w, self.c.head_dim
        n, pos = len(tokens), self.pos
        x = w["token_embd.weight"][list(tokens)].copy() if vectors is None else np.asarray(vectors, np.float64)
        shift = getattr(self, "shift", 0)
        turn = np.repeat(pos + shift + np.arange(n)[:, None], 4, 1) if axes is None else np.asarray(axes)
        axis = np.asarray(c.axes if c.axes is not None else [0] * (hd // 2))
        angle = turn[:, axis] * self.freqs
        cs, sn = self.mscale * np.cos(angle)[:, None], self.mscale * np.sin(angle)[:, None]

        def rope(h):
            a, b = h[..., : hd // 2], h[..., hd // 2:]
            return np.concatenate([a * cs - b * sn, a * sn + b * cs], -1)
        for l in range(c.n_layer):
            p = lambda s: w[f"blk.{l}.{s}.weight"]  # noqa: E731
            h = np.stack([_rms(r, p("attn_norm"), c.eps) for r in x])
            head = lambda m, k: (h @ p(m).T).reshape(n, k, hd)  # noqa: E731
            norm = lambda v, g: v / np.sqrt((v * v).mean(-1, keepdims=True) + c.eps) * p(g)  # noqa: E731
            q = rope(norm(head("attn_q", c.n_head), "attn_q_norm"))
            self.k_cache[l] += self.stored(rope(norm(head("attn_k", c.n_head_kv), "attn_k_norm")), self.kv[0])
            self.v_cache[l] += self.stored(head("attn_v", c.n_head_kv), self.kv[1])
            K, V = np.stack(self.k_cache[l]), np.stack(self.v_cache[l])
            window = c.windows[l] if c.windows else 0
            out = np.zeros((n, c.n_head, hd))
            for r in range(n):
                at, end = pos + r, pos + n if together else pos + r + 1
                lo = max(since, at + 1 - window if window else 0)
                for i in range(c.n_head):
                    s = K[lo:end, i * c.n_head_kv // c.n_head] @ q[r, i] / np.sqrt(hd)
                    if c.score_cap:
                        s = c.score_cap * np.tanh(s / c.score_cap)
                    if c.slopes is not None:
                        s = s - c.slopes[i] * np.abs(np.arange(lo, end) - at)
                    e = np.exp(s - s.max())
                    out[r, i] = e @ V[lo:end, i * c.n_head_kv // c.n_head] / e.sum()
            x = x + out.reshape(n, -1) @ p("attn_output").T
            x = x + np.stack([self._ffn(l, _rms(r, p("ffn_norm"), c.eps)) for r in x])
        self.pos += n
        if axes is not None:
            self.shift = max(int(np.max(turn[:, : axis.max() + 1])) + 1, pos + shift) - self.pos
        return np.stack([self.head @ _rms(r, w["output_norm.weight"], c.eps) for r in x])


def _tokens(g, c, n):
    return [int(t) for t in g.integers(0, c.n_vocab, n)]


def _config(**more):
    return dataclasses.replace(synth.qwen3_config("tiny"), **more)


def _model(c, tensors, precision):
    m = Model(c, tensors)
    m.kv = KV[precision]
    return m


def _both(ctx, c, tensors, precision):
    return B.BatchEngine(ctx, tensors, c, 512, 96, 16, precision, max_seq=6), _model(c, tensors, precision)


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("shape", ["cap", "windows", "slopes", "all"])
def test_models_with_shaped_scores(ctx, precision, shape):
    """Prompts of several chunks, a fork that shares pages, and steps, windows shorter and longer than either."""
    c = _config()
    heads, layers = c.n_head, c.n_layer
    more = {}
    if shape in ("cap", "all"):
        more["score_cap"] = 4.0
    if shape in ("windows", "all"):
        more["windows"] = tuple((20, 0, 150)[l % 3] for l in range(layers))
    if shape in ("slopes", "all"):
        more["slopes"] = tuple(2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads))
    c, g = _config(**more), np.random.default_rng(3)
    tensors = synth.qwen3("test-shaped", c, "q8_0", "random")
    eng, a = _both(ctx, c, tensors, precision)
    try:
        prompt, rest = _tokens(g, c, 300), _tokens(g, c, 6)
        s = eng.open()
        eng.extend(s, prompt)
        a.extend(prompt)
        t = eng.fork(s)
        b = _model(c, tensors, precision)
        b.k_cache, b.v_cache, b.pos = [list(k) for k in a.k_cache], [list(v) for v in a.v_cache], a.pos
        for i in range(0, 6, 2):
            got = eng.step({s: rest[i], t: rest[i + 1]})
            assert rel_l2(got[0], a.extend([rest[i]])[0]) < BAR, i
            assert rel_l2(got[1], b.extend([rest[i + 1]])[0]) < BAR, i
        eng.extend(t, prompt[:40])  # one goes on alone, further than the other
        b.extend(prompt[:40])
        got = eng.step({t: 5, s: 7})
        assert rel_l2(got[0], b.extend([5])[0]) < BAR and rel_l2(got[1], a.extend([7])[0]) < BAR
    finally:
        eng.free()


@pytest.mark.parametrize("precision", list(P))
@pytest.mark.parametrize("since", [0, 1, 64, 100, 150])
def test_documents_and_prefixes(ctx, precision, since):
    c, g = _config(), np.random.default_rng(since)
    tensors = synth.qwen3("test-spans", c, "q8_0", "random")
    eng, m = _both(ctx, c, tensors, precision)
    try:
        s = eng.open()
        for n, kw in ((150, {}), (200, dict(since=since)), (90, dict(together=True)), (30, dict(since=since, together=True)),
                      (1, dict(since=since))):
            tokens = _tokens(g, c, n)
            eng.extend(s, tokens, **kw)
            m.extend(tokens[:128], **kw)
            if n > 128:
                m.extend(tokens[128:], **kw)
        for _ in range(3):
            t = _tokens(g, c, 1)
            assert rel_l2(eng.step({s: t[0]})[0], m.extend(t)[0]) < BAR
    finally:
        eng.free()


@pytest.mark.parametrize("precision", list(P))
def test_images_in_a_prompt(ctx, precision):
    """Text, an image's patches as vectors at positions of three axes that see one another, text behind them; a text
    sequence beside it."""
    c = _config(axes=tuple(i % 3 if i < 60 else 0 for i in range(64)))
    g = np.random.default_rng(8)
    tensors = synth.qwen3("test-axes", c, "q8_0", "random")
    eng, m = _both(ctx, c, tensors, precision)
    other = _model(c, tensors, precision)
    try:
        s, t = eng.open(), eng.open()
        text, more = _tokens(g, c, 20), _tokens(g, c, 140)
        patches = (m.w["token_embd.weight"][_tokens(g, c, 48)] * g.uniform(0.5, 2, (48, 1))).astype(np.float32)
        at = np.stack([np.full(48, 20), 20 + np.arange(48) // 8, 20 + np.arange(48) % 8], 1)
        for eng_seq, model in ((s, m),):
            eng.extend(eng_seq, text)
            model.extend(text)
            eng.extend(eng_seq, [0] * 48, axes=at, vectors=patches, together=True)
            model.extend([0] * 48, axes=np.concatenate([at, at[:, :1]], 1), vectors=patches, together=True)
            assert eng.sequences[eng_seq].shift == model.shift == 28 - 68
        eng.extend(t, more)
        other.extend(more[:128])
        other.extend(more[128:])
        for i in range(3):
            k = _tokens(g, c, 2)
            got = eng.step({s: k[0], t: k[1]})
            assert rel_l2(got[0], m.extend(k[:1])[0]) < BAR and rel_l2(got[1], other.extend(k[1:])[0]) < BAR, i
        eng.extend(s, more)  # and a further turn's text
        m.extend(more[:128])
        m.extend(more[128:])
        u = eng.fork(s)
        assert rel_l2(eng.step({u: 3})[0], m.extend([3])[0]) < BAR
    finally:
        eng.free()


@pytest.mark.parametrize("n", [1, 2, 130])
def test_frames_behind_a_document(ctx, n):
    """Vectors at positions of axes, of any number, that see from a document's start on, in a model with a window."""
    c = _config(axes=tuple(i % 3 if i < 60 else 0 for i in range(64)), windows=(40, 0, 100))
    g = np.random.default_rng(n)
    tensors = synth.qwen3("test-frames", c, "q8_0", "random")
    eng, m = _both(ctx, c, tensors, P.F16_KEYS_Q8_VALUES)
    try:
        s, text = eng.open(), _tokens(g, c, 70)
        rows = (m.w["token_embd.weight"][_tokens(g, c, n)] * g.uniform(0.5, 2, (n, 1))).astype(np.float32)
        at = np.stack([70 + np.arange(n) // 64, 70 + np.arange(n) % 64 // 8, 70 + np.arange(n) % 8], 1)
        eng.extend(s, text)
        m.extend(text)
        eng.extend(s, [1] * n, axes=at, vectors=rows, since=66)
        for i in range(0, n, 128):
            k = slice(i, i + 128)
            m.extend([1] * len(at[k]), axes=np.concatenate([at, at[:, :1]], 1)[k], vectors=rows[k], since=66)
        for t in _tokens(g, c, 3):
            assert rel_l2(eng.step({s: t})[0], m.extend([t])[0]) < BAR
    finally:
        eng.free()


def test_one_axis_as_none(ctx):
    """A model whose axes are all the first, served as text: the logits of the model without them, to the bit."""
    g = np.random.default_rng(2)
    c = _config()
    tensors = synth.qwen3("test-one", c, "q8_0", "random")
    tokens, out = _tokens(g, c, 40), []
    for axes in (None, (0,) * 64):
        eng = B.BatchEngine(ctx, tensors, dataclasses.replace(c, axes=axes), 128, 32, 16, max_seq=2)
        try:
            s = eng.open()
            eng.extend(s, tokens)
            out.append(eng.step({s: 5}))
        finally:
            eng.free()
    assert (out[0] == out[1]).all()


def test_drawn_tokens(ctx):
    """sample() draws by the definition from the logits that step() gives, controls applied, alone and in a batch."""
    c, g = _config(), np.random.default_rng(4)
    tensors = synth.qwen3("test-drawn", c, "q8_0", "random")
    eng = B.BatchEngine(ctx, tensors, c, 256, 128, 16, max_seq=12)
    try:
        first = eng.open()
        eng.extend(first, _tokens(g, c, 50))
        kinds = [B.Sampling(), B.Sampling(0.0), B.Sampling(0.7, 5), B.Sampling(1.5, 0, 0.8), B.Sampling(1.0, 0, 1.0, 0.3)]
        seqs = [first] + [eng.fork(first) for _ in kinds[1:]]
        for q, k in zip(seqs, kinds):
            eng.sampling(q, k)
            eng.control(q, B.Controls(repetition=1.1, bias={3: 2.0}, allowed=np.arange(c.n_vocab) % 3 != 1))
        twins = [eng.fork(q) for q in seqs]
        for i in range(4):
            tokens = _tokens(g, c, len(seqs))
            draws = [int(d) for d in g.integers(0, 2**32, len(seqs))]
            order = [seqs, twins][i % 2], [twins, seqs][i % 2]
            logits = eng.step(dict(zip(order[0], tokens)))
            got = eng.sample(dict(zip(order[1], tokens)), dict(zip(order[1], draws)))
            for r, k in enumerate(kinds):
                w = want(logits[r], k.temperature, k.top_p, k.min_p, k.top_k, draws[r])
                assert (got.token[r], got.kept[r]) == w[:2], (i, r)
                assert abs(got.logprob[r] - w[2]) < 1e-10 + 2.0**-24 * abs(w[2])
        eng.control(seqs[0], B.Controls(allowed=np.zeros(c.n_vocab, bool)))
        got = eng.sample({seqs[0]: 1, seqs[1]: 2}, {seqs[1]: 5, seqs[0]: 6})
        assert got.token[0] == -1 and got.kept[0] == 0 and got.logprob[0] == -np.inf and got.token[1] >= 0
    finally:
        eng.free()


def test_shaped_models_need_the_batch_engine(ctx):
    c = _config(score_cap=30.0)
    with pytest.raises(ValueError):
        E.Engine(ctx, {}, c, 64)
