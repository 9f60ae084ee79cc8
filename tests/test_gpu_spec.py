"""Speculative decoding through the engine: a tree step's logits against decode() along every branch,
acceptance against the greedy stream, positions and refusals."""
import numpy as np
import pytest

from tinferno_b200 import native, synth
from tinferno_b200.model import Model, RunConfig, lookup_tree

pytestmark = pytest.mark.gpu

# GEMM models (Q8_0), a mixed one whose lm_head and some layers run the multi-row GEMV
CFGS = [synth.mini(synth.CFG0, 2, 4096), synth.mini(synth.CFG1, 2, 4096), synth.mini(synth.CFG2, 2, 4096),
        synth.mini(synth.CFG4, 2, 4096)]
LOGIT_TOL = 2e-3  # the bound of batched against single steps (tests/test_gpu_batch.py)


@pytest.fixture(scope="module")
def paths(model_cache):
    return {c.name: synth.model_path(c, model_cache) for c in CFGS}


def branch(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


@pytest.mark.parametrize("kv", [native.TF_KV_F32, native.TF_KV_F16, native.TF_KV_BF16])
@pytest.mark.parametrize("n", [1, 3, 9, 21])
@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
def test_tree_step_matches_decode_along_every_branch(cfg, n, kv, paths):
    rng = np.random.default_rng(n)
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 37, stream=5)]
    tokens = rng.integers(0, cfg.n_vocab, n).tolist()
    parents = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
    m = Model(paths[cfg.name], RunConfig(max_seq=96, max_batch=2, kv_type=kv))
    m.prefill(prompt, seq=1)
    am, lg = m.tree_step(tokens, parents, seq=1, want_logits=True)
    assert m.n_pos(seq=1) == len(prompt)
    again, lg2 = m.tree_step(tokens, parents, seq=1, want_logits=True)  # a step leaves the state as it was
    assert np.array_equal(lg, lg2) and np.array_equal(am, again)
    leaves = set(range(n)) - set(parents)
    for leaf in leaves:
        m.rewind(len(prompt), seq=1)
        for i in branch(parents, leaf):
            want = m.decode(tokens[i], seq=1)
            assert np.abs(lg[i] - want).max() < LOGIT_TOL, (leaf, i, np.abs(lg[i] - want).max())
            assert am[i] == int(np.argmax(lg[i]))
    m.close()


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
def test_accepting_keeps_the_greedy_stream(cfg, graph, paths):
    """Trees with right, wrong and half-right branches: what is kept is the greedy stream, and decoding
    goes on from the compacted cache as if every token had been decoded by itself."""
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 20, stream=9)]
    m = Model(paths[cfg.name], RunConfig(max_seq=128, use_graph=graph))
    first = int(np.argmax(m.prefill(prompt)))
    want = m.generate_greedy(first, 40)
    m.reset()
    m.prefill(prompt)
    wrong = lambda t: (t + 1) % cfg.n_vocab
    out, root = [], want[0]
    steps = 0
    while len(out) < 30:
        w = want[len(out):]
        assert root == w[0]
        # root -> wrong; root -> right, right -> wrong; right -> right -> right (a node in between)
        tokens = [root, wrong(w[1]), w[1], wrong(w[2]), w[2], wrong(w[1]), w[3]]
        parents = [-1, 0, 0, 2, 2, 1, 4]
        m.tree_step(tokens, parents)
        kept, nxt = m.tree_accept()
        assert kept == w[1:4] and nxt == w[4]
        out += [root] + kept
        root = nxt
        assert m.n_pos() == len(prompt) + len(out)
        steps += 1
    logits = m.decode(root)
    assert int(np.argmax(logits)) == want[len(out) + 1]
    m.close()


def test_wrong_drafts_cost_nothing_but_the_step(paths):
    cfg = CFGS[0]
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 12, stream=2)]
    m = Model(paths[cfg.name], RunConfig(max_seq=64))
    root = int(np.argmax(m.prefill(prompt)))
    want = int(np.argmax(m.decode(root)))
    m.rewind(len(prompt))
    m.tree_step([root, (want + 1) % cfg.n_vocab, (want + 2) % cfg.n_vocab], [-1, 0, 1])
    assert m.tree_accept() == ([], want)
    assert m.n_pos() == len(prompt) + 1
    m.close()


@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
def test_generate_lookup_is_greedy_at_temperature_zero(cfg, paths):
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 16, stream=4)] * 2  # repeats itself, so that there is something to look up
    m = Model(paths[cfg.name], RunConfig(max_seq=160))
    first = int(np.argmax(m.prefill(prompt)))
    want = m.generate_greedy(first, 60)
    m.reset()
    assert m.generate_lookup(prompt, 60) == want
    m.reset()
    got = m.generate_lookup(prompt, 25, temperature=0.8, seed=3)
    assert len(got) == 25 and all(0 <= t < cfg.n_vocab for t in got)
    m.close()


def test_draft_model_distribution(paths):
    """A draft with its distribution: the model drafting for itself keeps every token."""
    cfg = CFGS[1]
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 10, stream=6)]
    m = Model(paths[cfg.name], RunConfig(max_seq=64))
    torch = pytest.importorskip("torch")
    root = int(np.argmax(m.prefill(prompt)))
    tokens, parents = [root, 5, 900], [-1, 0, 1]
    _, lg = m.tree_step(tokens, parents, want_logits=True)
    draft = torch.from_numpy(lg).cuda()
    u = [0.5, 1 - 2 ** -20, 1 - 2 ** -20]
    kept, _ = m.tree_accept(1.0, u, draft_ptr=draft.data_ptr())
    assert kept == tokens[1:] and m.n_pos() == len(prompt) + 3
    m.close()


def test_refusals(paths):
    cfg = CFGS[0]
    m = Model(paths[cfg.name], RunConfig(max_seq=70))
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 4, stream=1)]
    m.prefill(prompt)
    with pytest.raises(native.TFError, match="no tree step"):
        m._tree = np.zeros(1, np.int32)
        m.tree_accept()
    cap = m.tree_capacity
    assert cap >= 64
    for tokens, parents, text in (([], [], "size"), ([1] * (cap + 1), [-1] + [0] * cap, "size"), ([1, cfg.n_vocab], [-1, 0], "token"),
                                  ([1, 2], [-1, 1], "parent"), ([1, 2], [0, 0], "parent")):
        with pytest.raises(native.TFError, match=text):
            m.tree_step(tokens, parents)
    with pytest.raises(native.TFError, match="rewound"):
        m.rewind(5)
    m.rewind(2)
    assert m.n_pos() == 2
    m.prefill(prompt * 16 + prompt[:2])  # position 68
    with pytest.raises(native.TFError, match="max_seq"):
        m.tree_step([1, 2, 3], [-1, 0, 1])
    m.tree_step([1, 2], [-1, 0])
    kept, nxt = m.tree_accept()
    assert m.n_pos() == 69 + len(kept)
    m.close()
