"""Speculative steps of the engine: models of every mix of weight types, the order of calls between a
tree step and its acceptance, and what a failed acceptance leaves behind."""
from dataclasses import replace

import numpy as np
import pytest

from tinferno_b200 import native, synth
from tinferno_b200.gguf import GGML_F16, GGML_Q4_1, GGML_Q6_K, GGML_Q8_0
from tinferno_b200.model import Model, RunConfig

pytestmark = pytest.mark.gpu

CFG = synth.mini(synth.CFG1, 2, 4096)
LOGIT_TOL = 2e-3  # the bound of batched against single steps (tests/test_gpu_batch.py)

# layers of types that the tensor-core GEMM does not take; the output matrix, or one layer's, is Q8_0
MIXED = [synth.mini(replace(synth.CFG0, name="tree-q4_1-head-q8_0", wtype=GGML_Q4_1, etype=GGML_Q8_0), 2, 4096),
         synth.mini(replace(synth.CFG0, name="tree-f16-down-q8_0", wtype=GGML_F16, etype=GGML_Q6_K,
                            down_override=((0, GGML_Q8_0),)), 2, 4096)]


def branch(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


@pytest.mark.parametrize("n", [2, 16, 40])
@pytest.mark.parametrize("cfg", MIXED, ids=lambda c: c.name)
def test_tree_step_of_a_model_without_gemm_buffers(cfg, n, model_cache):
    """Its few matrices of the GEMM's types take the multi-row GEMV like the others."""
    rng = np.random.default_rng(n)
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 12, stream=5)]
    tokens = rng.integers(0, cfg.n_vocab, n).tolist()
    parents = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
    m = Model(synth.model_path(cfg, model_cache), RunConfig(max_seq=80))
    m.prefill(prompt)
    _, lg = m.tree_step(tokens, parents, want_logits=True)
    for leaf in sorted(set(range(n)) - set(parents))[:4]:
        m.rewind(len(prompt))
        for i in branch(parents, leaf):
            want = m.decode(tokens[i])
            assert np.abs(lg[i] - want).max() < LOGIT_TOL, (leaf, i, np.abs(lg[i] - want).max())
    m.close()
