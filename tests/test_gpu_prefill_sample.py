"""Sampling right after a prompt: row 0 of the last step holds the prompt's logits for short prompts
(token steps) and for those of 16 tokens and more (tensor-core chunks, whose last row is another)."""
import numpy as np
import pytest

from tinferno_b200 import synth
from tinferno_b200.model import Model, RunConfig

pytestmark = pytest.mark.gpu

CFG = synth.mini(synth.CFG0, 2, 4096)


@pytest.mark.parametrize("n", [1, 7, 15, 16, 40, 128, 200])
def test_sample_after_prefill_is_the_prompts(n, model_cache):
    m = Model(synth.model_path(CFG, model_cache), RunConfig(max_seq=256))
    prompt = [int(t) for t in synth.prompt_tokens(CFG, n, stream=4)]
    first = int(np.argmax(m.prefill(prompt)))
    assert m.sample(0.0, 1.0, 0.0) == first
    want = m.generate_greedy(first, 10)
    m.reset()
    assert m.generate(prompt, 10, 0.0, 1.0) == want
    m.close()
