"""Tree attention over the range of the values: rows of one tile that lie many powers of two apart, queries
and keys near zero, and rows far apart in memory.

A tile of an fp32 or bf16 cache shares one power-of-two scale, so the bounds of tests/test_gpu_tree.py
(fixed there before their first run) are held here to each group of rows by itself: 22 significant
bits of what a row sees, whatever lies beside it."""
import numpy as np
import pytest

from tinferno_b200 import native
from test_gpu_tree import TYPES, Case, device_error, mask_bits, torch

pytestmark = pytest.mark.gpu

SCALED = [native.TF_KV_F32, native.TF_KV_BF16]  # cache types whose tiles are scaled
HEADS = [(8, 2, 64), (12, 2, 128), (6, 2, 80)]


def held(c, got, b, rows):
    """The bound of every element and the 2-norm of `rows`, a selection of nodes of sequence b."""
    want, tol = c.want(b)
    err = (got[b][rows] - want[rows]).abs()
    assert (err <= tol[rows]).all(), float((err - tol[rows]).max())
    norm = want[rows].norm()
    assert (got[b][rows] - want[rows]).norm() <= 5e-6 * norm, float((got[b][rows] - want[rows]).norm() / norm)


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


@pytest.mark.parametrize("big", [1e5, 1e6, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("T", [10, 64])
@pytest.mark.parametrize("kv", TYPES)
def test_large_unseen_rows_do_not_reach_the_output(kv, T, big):
    """A drafted node's keys and values, however large, change the rows that do not see it by no bit of
    what those are good for, and the rows that see it are right too."""
    if kv == native.TF_KV_F16:
        big = min(big, 6e4 / 5)
    for ctx, heads in ((70, HEADS[0]), (0, HEADS[0]), (70, HEADS[1]), (3, HEADS[2])):
        c = Case([ctx], [T], T, *heads, kv, seed=9)
        j = 4
        for which in (c.k, c.v):
            which[c.slots[0], :, ctx + j] *= big
        got = c.call()
        sees = torch.from_numpy(c.bits[0][:, j]).cuda()
        assert sees.any() and not sees.all()
        held(c, got, 0, ~sees)
        want, tol = c.want(0)
        assert ((got[0] - want).abs() <= tol)[sees].all()
    assert device_error() == 0


@pytest.mark.parametrize("lens,T", [([70, 5000], 6), ([300, 2500, 129], 40), ([20000], 64)])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("kv", SCALED)
def test_large_committed_keys(kv, heads, lens, T):
    """Keys of committed positions 10^6 times the others': a head's score with one is either far above
    the rest or far below, and below it the rest keeps its bits.  Contexts within one CTA's range and
    split over several."""
    c = Case(lens, [T] * len(lens), T, *heads, kv, seed=3)
    rng = np.random.default_rng(5)
    for b, n in enumerate(lens):
        # one position, so that no two large scores compete (their own rounding would decide)
        c.k[c.slots[b], :, int(rng.integers(0, n))] *= 1e6
    got = c.call()
    for b in range(len(lens)):
        held(c, got, b, slice(None))
    assert device_error() == 0


@pytest.mark.parametrize("T", [6, 64])
@pytest.mark.parametrize("kv", SCALED)
def test_values_of_every_size_in_one_tile(kv, T):
    """Values that fall from 1 to 2^-60 over a tile: a row that sees small ones alone keeps their bits."""
    c = Case([0], [T], T, 8, 2, 64, kv, seed=12)
    fall = 2.0 ** -(torch.arange(T, device="cuda") * (60.0 / T)).floor()
    c.v[c.slots[0], :, :T] = (c.v[c.slots[0], :, :T].float() * fall[None, :, None]).to(c.v.dtype)
    m = np.zeros((1, T, 1), np.uint64)
    m[0, :, 0] = np.uint64(1) << np.arange(T, dtype=np.uint64)  # every node sees itself
    c.set_mask(m)
    c.bits = [mask_bits(m[0], T)]
    got = c.call()
    for t in range(T):
        held(c, got, 0, slice(t, t + 1))


@pytest.mark.parametrize("T", [6, 64])
@pytest.mark.parametrize("kv", SCALED)
def test_zero_rows_and_zero_columns(kv, T):
    """Rows and channels of exact zeros beside ordinary ones are exact at any scale."""
    c = Case([200, 64], [T, T], T, 8, 2, 64, kv, seed=15)
    c.k[:, :, ::3] = 0.0
    c.v[:, :, 1::4] = 0.0
    c.k[..., 8:24] = 0.0
    c.v[..., 40:48] = 0.0
    c.check(c.call())


@pytest.mark.parametrize("T", [6, 64])
def test_large_rows_in_a_batch_leave_the_others(T):
    """One sequence's large rows, among others' ordinary ones, and non-finite drafted values beside them."""
    c = Case([900, 33, 2000, 64], [T] * 4, T, 8, 2, 64, native.TF_KV_F32, seed=13)
    c.k[c.slots[1], :, 33 + 3] *= 1e9
    c.v[c.slots[2], :, 2000 + 2] *= 1e12
    c.v[c.slots[2], :, 2000 + 3] = float("inf")
    got = c.call()
    for b, j in ((0, None), (1, [3]), (2, [2, 3]), (3, None)):
        sees = torch.zeros(T, dtype=torch.bool) if j is None else torch.from_numpy(c.bits[b][:, j].any(1))
        held(c, got, b, ~sees.cuda())
    sees_inf = torch.from_numpy(c.bits[2][:, 3]).cuda()
    assert not got[2][sees_inf].isfinite().any()
    assert torch.equal(got, c.call())


@pytest.mark.parametrize("T", [4, 64])
@pytest.mark.parametrize("kv", TYPES)
def test_a_row_does_not_depend_on_its_batch_beyond_rounding(kv, T):
    """A sequence alone, with others, and with others in another order: the split over CTAs differs, the
    values by the rounding of either (twice the bound of one)."""
    lens = [900, 33, 2000, 1]
    c = Case(lens, [T] * 4, T, 8, 2, 64, kv, seed=13)
    full = c.call().clone()
    q, mask, slots, bits = c.q, c.mask, c.slots, c.bits
    for order in ([0], [1], [2], [3], [2, 0], [3, 2, 1, 0]):
        c.B, c.lens, c.nodes, c.slots = len(order), [lens[b] for b in order], [T] * len(order), [slots[b] for b in order]
        c.q, c.mask, c.out = q[order].contiguous(), mask[order].contiguous(), torch.full((len(order), T, c.ld_out), 7.0, device="cuda")
        c.bits = [bits[b] for b in order]
        got = c.call()
        for i, b in enumerate(order):
            assert (got[i] - full[b]).norm() <= 1e-5 * full[b].norm()
            assert ((got[i] - full[b]).abs() <= 2 * c.want(i)[1]).all()
