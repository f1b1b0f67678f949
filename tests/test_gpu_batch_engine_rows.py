"""What a step computes does not depend on the numbers that its sequences happen to have."""
import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", ["tiny", "tiny-moe"])
def test_any_number_gives_the_same_logits(ctx, model):
    """One sequence, and then two, decoded under the first numbers and under the last, with their
    controls: the same bits."""
    c, g = synth.qwen3_config(model), np.random.default_rng(3)
    tensors = synth.qwen3("test-rows", c, "q4_k_m", "random") if model == "tiny" else synth.qwen3moe("test-rows", c)
    prompt = [int(t) for t in g.integers(0, c.n_vocab, 21)]
    outs = []
    for idle in (0, 2):
        eng = B.BatchEngine(ctx, tensors, c, 64, 24, 16, max_seq=4)
        try:
            for _ in range(idle):
                eng.extend(eng.open(), [5, 6, 7])
            a, b = eng.open(), eng.open()
            assert (a, b) == (idle, idle + 1)
            for q, n in ((a, 20), (b, 7)):
                eng.extend(q, prompt[:n])
                eng.control(q, B.Controls(repetition=1.1 + q - a, bias={n: 2.0}))
            out = [eng.step({b: 8}), eng.step({a: 9}), eng.step({a: 10, b: 11}), eng.step({b: 12})]
            if idle:  # the others' own steps between change nothing
                eng.step({0: 1, 1: 2})
            outs.append(np.concatenate([*out, eng.step({b: 13, a: 14})[::-1]]))
        finally:
            eng.free()
    assert np.array_equal(*outs)
