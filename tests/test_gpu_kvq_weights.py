"""Attention over a quantised cache where the products of probability and V scale are spread wide: small weights are
not rounded away against large ones."""
import numpy as np
import pytest

from test_gpu_kvq import Case, TYPES, device_error

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

# (H, HK, T): up to 4, 8 and 16 rows a kv head
ROWS = [(4, 1, 1), (8, 1, 1), (8, 2, 3)]


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("H,HK,T", ROWS)
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("big,small", [(6, -8), (14, 0), (14, -4)])
def test_groups_of_dims_of_different_sizes(kv, H, HK, T, hd, big, small):
    """Within one head, groups of 32 dims whose values are 2^14 and 2^18 apart: each is right relative to itself (the 2-norm bound
    of the operator's other tests, 5e-6, for every group)."""
    c = Case(kv, hd, H, HK, [300], [T], T, 7)
    rng = np.random.default_rng(hd)
    size = np.repeat(2.0 ** np.where(np.arange(hd // 32) % 2, small, big), 32)
    c.fill("v", 0, 0, (rng.standard_normal((HK, 300 + T, hd)) * 0.7 * size).astype(np.float32))
    got = c.run().got()
    assert device_error() == 0
    want, _ = c.want(0)
    for g in range(hd // 32):
        a, b = (v[..., 32 * g:32 * g + 32] for v in (got[0], want))
        assert np.linalg.norm(a - b) <= 5e-6 * np.linalg.norm(b), (g, np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("H,HK,T", ROWS)
@pytest.mark.parametrize("gap", [6, 12, 18])
def test_one_position_far_above_the_others(kv, H, HK, T, gap):
    """Position 0 takes a score `gap` above all others' and its values are zero, so that the output is what 20000 small
    weights of one sign make of values of one sign.  Bound: 5e-6, as elsewhere, and the score's own error: in the
    exponent a score S has four roundings of 2^-24 S (the query's halves, the sum over dims, the factor to powers of
    two, the difference to the reference)."""
    hd, n = 64, 20000
    c = Case(kv, hd, H, HK, [n - T], [T], T, 3)
    rng = np.random.default_rng(gap)
    base = rng.standard_normal((HK, hd))
    noise = rng.standard_normal((T, HK, H // HK, hd)) * 0.2
    c.q[0, :, :H * hd] = (base[None, :, None] + noise).reshape(T, H * hd)
    k = rng.standard_normal((HK, n, hd))
    k[:, 0] = base * gap * hd ** 0.5 / (base ** 2).sum(-1, keepdims=True)
    v = np.abs(rng.standard_normal((HK, n, hd))) + 0.1
    v[:, 0] = 0
    c.fill("k", 0, 0, k.astype(np.float32))
    c.fill("v", 0, 0, v.astype(np.float32))
    got = c.run().got()
    assert device_error() == 0
    want, _ = c.want(0)
    stored = c.c.values("k", c.slots[0], n)
    q = c.q[0, :, :H * hd].reshape(T, HK, H // HK, hd).astype(np.float64)
    top = np.abs(np.einsum("tgrd,gnd->tgrn", q, stored)).max() / hd ** 0.5
    off = np.linalg.norm(got[0] - want) / np.linalg.norm(want)
    assert off <= 5e-6 + 4 * 2.0 ** -24 * top, off
