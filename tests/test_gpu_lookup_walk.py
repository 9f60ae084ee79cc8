"""generate_lookup at a positive temperature, replayed: every step's kept tokens and next token are those of the
definition's walk (tests/test_gpu_tree.py, 64 bits) over the step's own logits, tree and random
numbers, whose outcome follows the model's distribution; and the first token follows its softmax."""
import numpy as np
import pytest

from tinferno_b200 import synth
from tinferno_b200.model import Model, RunConfig
from test_gpu_tree import walk, weights

pytestmark = pytest.mark.gpu

CFG = synth.mini(synth.CFG1, 2, 4096)
TEMPERATURE = 0.1  # low enough that drafts are kept and refused


class Watched(Model):
    """Records every step and checks every acceptance against the walk."""
    steps, kept, offered = 0, 0, 0

    def tree_step(self, tokens, parents, seq=0, want_logits=False):
        am, self.lg = super().tree_step(tokens, parents, seq=seq, want_logits=True)
        self.tree = list(tokens), list(parents)
        return am

    def tree_accept(self, temperature=0.0, u=None, draft_ptr=0, seq=0):
        kept, nxt = super().tree_accept(temperature, u, draft_ptr, seq)
        tokens, parents = self.tree
        path, want = walk(self.lg, None, tokens, parents, len(tokens), np.float32(u), temperature)
        assert kept == [tokens[i] for i in path[1:]] and nxt == want
        assert len(set(u)) == len(u)  # numbers of its own for every node
        self.steps, self.kept, self.offered = self.steps + 1, self.kept + len(kept), self.offered + len(tokens) - 1
        return kept, nxt


def test_every_step_is_the_definitions_walk(model_cache):
    m = Watched(synth.model_path(CFG, model_cache), RunConfig(max_seq=256))
    prompt = [int(t) for t in synth.prompt_tokens(CFG, 16, stream=4)] * 3
    outs = []
    for seed in range(6):
        m.reset()
        outs.append(m.generate_lookup(prompt, 40, temperature=TEMPERATURE, seed=seed))
        assert len(outs[-1]) == 40
    assert m.steps > 40 and m.offered > 0
    assert len({tuple(o) for o in outs}) > 1
    m.close()


def test_first_tokens_follow_the_softmax(model_cache):
    """The likeliest tokens' frequencies over 400 seeds, within 5 standard deviations."""
    m = Model(synth.model_path(CFG, model_cache), RunConfig(max_seq=64))
    prompt = [int(t) for t in synth.prompt_tokens(CFG, 6, stream=7)]
    p = weights(m.prefill(prompt), 1.0 / TEMPERATURE)
    p /= p.sum()
    n, seen = 400, np.zeros(CFG.n_vocab)
    for seed in range(n):
        m.reset()
        seen[m.generate_lookup(prompt, 1, temperature=TEMPERATURE, seed=seed)[0]] += 1
    top = np.argsort(p)[-8:]
    assert (np.abs(seen[top] - n * p[top]) <= 5 * np.sqrt(n * p[top] * (1 - p[top])) + 1).all()
    m.close()
