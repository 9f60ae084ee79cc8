"""Tree attention over the range of the values: rows of one tile that lie many powers of two apart, queries
and keys near zero, and rows far apart in memory.

A tile of an fp32 or bf16 cache shares one power-of-two scale, so the bounds of tests/test_gpu_tree.py
(fixed there before their first run) are held here to each group of rows by itself: 22 significant
bits of what a row sees, whatever lies beside it."""
import pytest

from tinferno_b200 import native
from test_gpu_tree import TYPES, Case, device_error, torch

pytestmark = pytest.mark.gpu

SCALED = [native.TF_KV_F32, native.TF_KV_BF16]  # cache types whose tiles are scaled
HEADS = [(8, 2, 64), (12, 2, 128), (6, 2, 80)]


@pytest.mark.parametrize("T", [6, 64])
@pytest.mark.parametrize("scale", [1e-4, 3e-5, 1e-9, 1e-30])
@pytest.mark.parametrize("kv", TYPES)
def test_zero_queries_over_small_keys(kv, scale, T):
    """A query of zeros weighs everything that it sees alike, however small the keys are."""
    if kv == native.TF_KV_F16 and scale < 1e-7:
        scale = 6e-8
    for heads in HEADS:
        c = Case([70, 0], [T, T - 1], T, *heads, kv, seed=T)
        c.k *= scale
        c.q[:, ::3] = 0.0
        c.check(c.call())
        c.q.zero_()
        c.check(c.call())
    assert device_error() == 0


@pytest.mark.parametrize("T", [6, 64])
@pytest.mark.parametrize("kv", SCALED)
def test_small_queries_over_small_keys(kv, T):
    """Scores whose scale is below the smallest 32-bit number."""
    c = Case([70, 0], [T, T - 1], T, 8, 2, 64, kv, seed=T)
    c.k *= 1e-20
    c.q *= 1e-25
    c.check(c.call())


def test_query_offsets_beyond_32_bits():
    """Query rows so far apart that the last one starts beyond 2^31 elements."""
    T, H, HK, hd = 256, 8, 8, 64
    c = Case([40], [T], T, H, HK, hd, native.TF_KV_F32, seed=7)
    ld = (1 << 23) + (1 << 16)
    assert (T - 1) * ld > 2 ** 31
    q = torch.empty((1, T, ld), device="cuda")
    q[..., :H * hd] = c.q[..., :H * hd]
    c.q, c.ld_q = q, ld
    c.check(c.call())
