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


@pytest.fixture(scope="module")
def path(model_cache):
    return synth.model_path(CFG, model_cache)


def prompts(n=2):
    return [[int(t) for t in synth.prompt_tokens(CFG, 18 + i, stream=3 + i)] for i in range(n)]


def started(path, **kw):
    """Two sequences behind their prompts; the greedy tokens after them."""
    m = Model(path, RunConfig(max_seq=96, max_batch=2, **kw))
    return m, [int(np.argmax(m.prefill(p, seq=i))) for i, p in enumerate(prompts())]


STEPS = {
    "decode another": lambda m, t: m.decode(t[1], seq=1),
    "decode the same": lambda m, t: m.decode(t[0], seq=0),
    "decode both": lambda m, t: m.decode_batch([1, 0], [t[1], t[0]]),
    "short prompt of another": lambda m, t: m.prefill([5, 6, 7], seq=1),
    "long prompt of another": lambda m, t: m.prefill(list(range(20, 60)), seq=1),
    "prompts of both": lambda m, t: m.prefill_batch([0, 1], [[3, 4], [5, 6]]),
    "generation of another": lambda m, t: m.generate_greedy(t[1], 3, seq=1),
    "sharded step of another": lambda m, t: (m.set_vocab_shard(0, 1), m.decode_shard(t[1], seq=1)),
    "reset": lambda m, t: m.reset(0),
    "reset of all": lambda m, t: m.reset(),
}


@pytest.mark.parametrize("step", list(STEPS))
def test_a_step_in_between_ends_the_tree(step, path):
    """The logits and the context that a tree was scored with are gone after another step: accepting it
    is refused, and every sequence goes on as if the tree had never been drafted."""
    m, t = started(path)
    m.tree_step([t[0], 11, 12, 13], [-1, 0, 1, 0], seq=0)
    STEPS[step](m, t)
    with pytest.raises(native.TFError, match="no tree step"):
        m.tree_accept(seq=0)
    plain, _ = started(path)
    STEPS[step](plain, t)
    for s in (0, 1):
        assert m.n_pos(seq=s) == plain.n_pos(seq=s)
        assert np.array_equal(m.decode(9, seq=s), plain.decode(9, seq=s))
    m.close()
    plain.close()


@pytest.mark.parametrize("what", ["reset", "rewind"])
def test_another_sequences_position_does_not_end_the_tree(what, path):
    m, t = started(path)
    am = m.tree_step([t[0], 11], [-1, 0], seq=0)
    if what == "reset":
        m.reset(1)
    else:
        m.rewind(4, seq=1)
    kept, nxt = m.tree_accept(seq=0)
    assert nxt == am[len(kept)] and m.n_pos(seq=0) == len(prompts()[0]) + 1 + len(kept)
    m.close()


def test_an_operator_calls_error_is_not_the_engines(path):
    """The operator level's error word belongs to its callers: a code that waits there fails no
    acceptance and stays to be read."""
    torch = pytest.importorskip("torch")
    L = native.lib()
    m, t = started(path)
    want = m.generate_greedy(t[0], 12)
    m.rewind(len(prompts()[0]))
    k = torch.zeros((1, 1, 1, 8, 8), device="cuda")
    one = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")
    n_ctx, p, n = one(0), one(5), one(1)
    slot = one(7)  # outside the cache
    native.check(L.tf_op_kv_commit(k.data_ptr(), k.data_ptr(), native.TF_KV_F32, 1, 64, 64, 8, 1, slot.data_ptr(), n_ctx.data_ptr(),
                                   p.data_ptr(), 1, n.data_ptr(), None, 1, 1, 8, None))
    torch.cuda.synchronize()
    m.tree_step(want[:3], [-1, 0, 1])
    kept, nxt = m.tree_accept()
    assert kept == want[1:3] and nxt == want[3] and m.n_pos() == len(prompts()[0]) + 3
    assert m.generate_greedy(nxt, 8) == want[3:11]  # device and host positions agree
    code = native.C.c_int(0)
    native.check(L.tf_op_device_error(None, native.C.byref(code)))
    assert code.value == 4  # TF_DEV_ERR_POS of the operator call
    m.close()


def test_a_refused_acceptance_leaves_the_tree(path):
    m, t = started(path)
    am = m.tree_step([t[0], 11], [-1, 0], seq=0)
    for temperature, text in ((float("nan"), "NaN"), (1e-45, "range"), (float("inf"), "range")):
        with pytest.raises(native.TFError, match=text):
            m.tree_accept(temperature, [0.5, 0.5], seq=0)
    with pytest.raises(native.TFError, match="no tree step"):
        m.tree_accept(seq=1)
    kept, nxt = m.tree_accept(seq=0)
    assert nxt == am[len(kept)] and m.n_pos(seq=0) == len(prompts()[0]) + 1 + len(kept)
    m.close()


def test_accept_without_a_step(path):
    m, _ = started(path)
    with pytest.raises(native.TFError, match="no tree step"):
        m.tree_accept()
    m.close()


def test_accept_without_random_numbers(path):
    """Numbers of zero in their place would keep every draft."""
    m, t = started(path)
    m.tree_step([t[0], 11], [-1, 0])
    with pytest.raises(native.TFError, match="u must not be null"):
        m.tree_accept(0.8)
    with pytest.raises(ValueError):
        m.tree_accept(0.8, [0.5])
    m.tree_accept(0.8, [0.5, 0.5])
    m.close()


def test_accepted_tokens_are_the_stepped_ones(path):
    """The caller may reuse its array between the step and the acceptance."""
    m, t = started(path)
    want = m.generate_greedy(t[0], 4)
    m.rewind(len(prompts()[0]))
    tokens = np.array(want[:3], np.int32)
    m.tree_step(tokens, [-1, 0, 1])
    tokens[:] = 0
    assert m.tree_accept() == (want[1:3], want[3])
    m.close()
