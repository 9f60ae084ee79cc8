"""The quantised KV cache's operators (tf_op_qk_norm_rope, tf_op_kv_quant, tf_op_kv_dequant, tf_op_qkv_store,
tf_op_attn_quant) against plain implementations in 64 bits.

Writing and reading are compared byte by byte and value by value.  Tolerances, fixed before their first run:

Norm and rotation.  The mean's rounding, eps, root and reciprocal put inv off by at most 3 x 2^-24, two products add
2 x 2^-24; cosine and sine (fp32) each 2^-24, the sum of the two products 2^-24 of the result.  With |y| the normed
pair's length, an element is off by at most (5 + sqrt(2) + 1) 2^-24 |y| < 8 x 2^-24 |y|.

Attention.  The cache's values are exact (f16 scale times an integer), q carries 22 bits or more, sums are fp32: a
score of hd products is off by at most about d = hd 2^-23 max_j(scale sum |q k_j|), every probability by a factor
1 +- d, and the output by (2 d + 2^-18) max |v|.  That bound is for the worst case; errors that do not conspire
leave a 2-norm error of a few 2^-22, so the norm is held to 5e-6, which a rounding of q or p to 11 bits (2e-4) does not
meet."""
import ctypes as C

import numpy as np
import pytest

import kvq_layout as lay
from tinferno_b200 import native

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = [native.TF_KV_Q4_0, native.TF_KV_Q8_0]


def ptr(t):
    return None if t is None else t.data_ptr()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def device_error():
    code = C.c_int(-1)
    native.check(native.lib().tf_op_device_error(None, C.byref(code)))
    return code.value


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Cache:
    """K and V, every byte random (scales among them: NaN and infinities too), on the host and on the GPU."""

    def __init__(self, kv, hd, HK, cap, n_slots, seed, gap=0):
        rng = np.random.default_rng(seed)
        self.kv, self.hd, self.HK, self.cap, self.n_slots = kv, hd, HK, cap, n_slots
        shape = (n_slots, HK + gap, cap // 16, lay.block_bytes(kv, hd))  # `gap` heads' room between the slots
        self.k, self.v = (rng.integers(0, 256, shape, np.uint8) for _ in range(2))
        self.stride = (HK + gap) * cap * hd

    def upload(self):
        self.dk, self.dv = cuda(self.k), cuda(self.v)
        return self

    def args(self):
        return (ptr(self.dk), ptr(self.dv), self.kv, self.stride, self.cap, self.n_slots)

    def put(self, slot, pos, k, v):
        """Rows [HK][hd] of position pos, on the host."""
        for kind, x in (("k", k), ("v", v)):
            codes, scales = lay.quantise(self.kv, x)
            for h in range(self.HK):
                lay.write(getattr(self, kind), kind, self.kv, self.hd, slot, h, pos, codes[h], scales[h])

    def same(self):
        return np.array_equal(self.dk.cpu().numpy(), self.k) and np.array_equal(self.dv.cpu().numpy(), self.v)

    def values(self, kind, slot, n):
        """[HK][n][hd] in 64 bits."""
        c = getattr(self, kind)[slot, :self.HK, :(n + 15) // 16]
        return lay.values(c.reshape(-1, c.shape[-1]), kind, self.kv, self.hd).reshape(self.HK, -1, self.hd)[:, :n]


def awkward_rows(rng, rows, HK, hd):
    """Rows whose groups try the corners of the definition."""
    x = (rng.standard_normal((rows, HK, hd)) * 2).astype(np.float32)
    g = x.reshape(-1, 32)
    corners = [np.zeros(32), np.full(32, 3.0), np.full(32, -3.0),
               np.r_[1.5, -1.5, np.linspace(-1.5, 1.5, 30)], np.r_[-1.5, 1.5, np.linspace(-1.5, 1.5, 30)],
               np.linspace(-8, 7.5, 32), np.linspace(-8, 7.5, 32) * 2.0 ** -24, rng.standard_normal(32) * 1e-40,
               rng.standard_normal(32) * 1e6, np.r_[3e38, -3e38, np.zeros(30)],
               np.r_[np.zeros(31), np.nan], np.r_[np.zeros(16), np.inf, np.ones(15)], np.r_[-np.inf, np.ones(31)],
               np.r_[127.0, np.arange(31) + 0.5], np.r_[-8.0, np.arange(31) % 8 - 0.5], np.r_[65504 * 8.0, np.arange(31)]]
    for i, c in enumerate(corners):
        if i < len(g):
            g[(i * 7) % len(g)] = c
    return x


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd,HK,rows,cap", [(32, 1, 1, 16), (32, 3, 45, 64), (64, 2, 33, 48), (64, 8, 5, 16), (96, 2, 21, 32),
                                            (128, 2, 40, 32), (128, 5, 7, 96)])
def test_write_and_read(kv, hd, HK, rows, cap):
    rng = np.random.default_rng(rows)
    c = Cache(kv, hd, HK, cap, 4, rows, gap=1).upload()
    x = awkward_rows(rng, rows, 2 * HK, hd)
    places = rng.permutation(4 * cap)[:rows]
    slots, pos = (places // cap).tolist(), (places % cap).tolist()
    slots[::7] = [-1] * len(slots[::7])                      # rows of a padded batch
    for r in range(rows):
        if slots[r] >= 0:
            c.put(slots[r], pos[r], x[r, :HK], x[r, HK:])
    ld = (2 * HK) * hd + 8                                   # fused rows with a tail
    kvrows = cuda(np.concatenate([x.reshape(rows, -1), np.full((rows, 8), np.nan, np.float32)], 1))
    s, p = i32(slots), i32(pos)
    L = native.lib()
    native.check(L.tf_op_kv_quant(*c.args(), ptr(s), ptr(p), ptr(kvrows), ld, ptr(kvrows) + 4 * HK * hd, ld, rows, HK, hd, None))
    assert device_error() == 0
    assert c.same()
    out = torch.full((rows, 2, HK * hd + 4), 7.0, device="cuda")
    native.check(L.tf_op_kv_dequant(ptr(out), 2 * HK * hd + 8, ptr(out) + 4 * (HK * hd + 4), 2 * HK * hd + 8, *c.args(), ptr(s), ptr(p),
                                    rows, HK, hd, None))
    assert device_error() == 0
    got = out.cpu().numpy()
    assert (got[..., HK * hd:] == 7).all()
    for r in range(rows):
        if slots[r] < 0:
            assert (got[r] == 7).all()
            continue
        for i, kind in enumerate("kv"):
            want = c.values(kind, slots[r], cap)[:, pos[r]].astype(np.float32)
            np.testing.assert_array_equal(got[r, i, :HK * hd].reshape(HK, hd), want)
    # one side alone
    only = torch.zeros((rows, HK * hd), device="cuda")
    native.check(L.tf_op_kv_dequant(None, 0, ptr(only), HK * hd, *c.args(), ptr(s), ptr(p), rows, HK, hd, None))
    keep = np.array(slots) >= 0
    np.testing.assert_array_equal(only.cpu().numpy()[keep], got[keep, 1, :HK * hd])


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd,HK,first,rows", [(32, 7, 0, 64), (64, 9, 3, 61), (96, 5, 16, 48), (128, 8, 1, 30), (128, 1, 0, 16)])
def test_every_group_its_own_corner(kv, hd, HK, first, rows):
    """Rows of neighbouring positions: groups that the kernel reduces together are of different kinds."""
    rng = np.random.default_rng(hd + rows)
    c = Cache(kv, hd, HK, 64, 1, 5).upload()
    corners = awkward_rows(rng, 40, 1, 32).reshape(40, 32)
    x = corners[rng.integers(0, 40, rows * 2 * HK * hd // 32)].reshape(rows, 2 * HK, hd)
    for r in range(rows):
        c.put(0, first + r, x[r, :HK], x[r, HK:])
    s, p, d = i32([0] * rows), i32(range(first, first + rows)), cuda(x.reshape(rows, -1))
    ld = 2 * HK * hd
    native.check(native.lib().tf_op_kv_quant(*c.args(), ptr(s), ptr(p), ptr(d), ld, ptr(d) + 4 * HK * hd, ld, rows, HK, hd, None))
    assert device_error() == 0
    assert c.same()


@pytest.mark.parametrize("kv", TYPES)
def test_values_next_to_the_border_of_two_codes(kv):
    """Every half between two codes, and its neighbours in fp32 on both sides, at scales of all mantissas: the code is the
    nearest, ties to even."""
    top = 8 if kv == native.TF_KV_Q4_0 else 127
    rng = np.random.default_rng(11)
    scale = rng.uniform(2.0 ** -12, 2.0 ** 6, 8192).astype(np.float16).astype(np.float32)
    x = np.zeros((len(scale), 32), np.float32)
    half = rng.integers(-top, top, (len(scale), 31)) + 0.5
    half[:, 0], half[:, 1] = top - 1.5, -top + 1.5
    mid = (scale[:, None] * half).astype(np.float32)          # exact: 11 + 8 bits
    x[:, 1:] = np.where(np.arange(31) % 3 == 0, mid, np.nextafter(mid, np.float32(np.inf) * np.where(np.arange(31) % 3 == 1, 1, -1), dtype=np.float32))
    x[:, 0] = -top * scale
    rows, HK, hd = 64, 32, 128
    x = x.reshape(rows, HK, hd)
    c = Cache(kv, hd, HK, 64, 1, 5)
    codes, scales = lay.quantise(kv, x)
    assert (scales.astype(np.float32).reshape(-1) == scale).all()
    k, v = np.zeros_like(c.k), np.zeros_like(c.v)
    c.k, c.v = k, v
    c.upload()
    for r in range(rows):
        for h in range(HK):
            lay.write(c.k, "k", kv, hd, 0, h, r, codes[r, h], scales[r, h])
            lay.write(c.v, "v", kv, hd, 0, h, r, codes[r, h], scales[r, h])
    d, s, p = cuda(x), i32([0] * rows), i32(range(rows))
    native.check(native.lib().tf_op_kv_quant(*c.args(), ptr(s), ptr(p), ptr(d), HK * hd, ptr(d), HK * hd, rows, HK, hd, None))
    assert device_error() == 0
    assert c.same()


@pytest.mark.parametrize("kv", TYPES)
def test_rows_outside_the_cache(kv):
    c = Cache(kv, 64, 2, 32, 3, 1).upload()
    x = torch.randn((5, 2, 128), device="cuda")
    L = native.lib()
    for slots, pos, code in [([0, 3, 0, 0, 1], [1, 2, 3, 4, 5], native.TF_DEV_ERR_BAD_INDEX),
                             ([0, 1, 0, 0, 1], [1, 2, 32, 4, 5], native.TF_DEV_ERR_POS),
                             ([0, 1, 0, 0, 1], [1, 2, 3, -1, 5], native.TF_DEV_ERR_POS)]:
        s, p = i32(slots), i32(pos)
        native.check(L.tf_op_kv_quant(*c.args(), ptr(s), ptr(p), ptr(x), 256, ptr(x) + 512, 256, 5, 2, 64, None))
        assert device_error() == code
        h = x.cpu().numpy()
        for r in range(5):
            if 0 <= slots[r] < 3 and 0 <= pos[r] < 32:
                c.put(slots[r], pos[r], h[r, 0].reshape(2, 64), h[r, 1].reshape(2, 64))
        assert c.same()
        out = torch.full((5, 2, 128), 7.0, device="cuda")
        native.check(L.tf_op_kv_dequant(ptr(out), 256, ptr(out) + 512, 256, *c.args(), ptr(s), ptr(p), 5, 2, 64, None))
        assert device_error() == code
        for r in range(5):
            bad = not (0 <= slots[r] < 3 and 0 <= pos[r] < 32)
            assert bool((out[r] == 7.0).all()) == bad


def test_rows_without_slots():
    """slots nullptr: row r in slot r; a row beyond the slots is an error."""
    kv = native.TF_KV_Q4_0
    c = Cache(kv, 32, 1, 16, 3, 2).upload()
    x = np.random.default_rng(0).standard_normal((4, 2, 32)).astype(np.float32)
    d, p = cuda(x), i32([5, 0, 15, 3])
    native.check(native.lib().tf_op_kv_quant(*c.args(), None, ptr(p), ptr(d), 64, ptr(d) + 128, 64, 4, 1, 32, None))
    assert device_error() == native.TF_DEV_ERR_BAD_INDEX
    for r, at in enumerate([5, 0, 15]):
        c.put(r, at, x[r, :1], x[r, 1:])
    assert c.same()


# ---- norm and rotation ---------------------------------------------------------------------------------

def norm_rope_64(x, w, eps, freq, pos):
    """x [rows][heads][hd] -> the result in 64 bits, and the bound of the module's docstring."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float32(eps)) * w.astype(np.float64)
    size = np.abs(y)
    out = y.copy()
    if freq is not None:
        n = len(freq)
        a = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)
        c, s = np.cos(a), np.sin(a)
        x0, x1 = y[..., :n], y[..., n:2 * n]
        out[..., :n], out[..., n:2 * n] = x0 * c - x1 * s, x0 * s + x1 * c
        length = np.hypot(x0, x1)
        size[..., :n], size[..., n:2 * n] = length, length
    return out, 8 * 2.0 ** -24 * size


@pytest.mark.parametrize("hd,rot,H,HK", [(8, 8, 3, 1), (40, 24, 5, 2), (64, 64, 14, 2), (64, 32, 32, 8), (96, 96, 6, 2), (128, 128, 12, 2),
                                         (128, 64, 7, 1), (128, 8, 2, 2)])
@pytest.mark.parametrize("normed", [0, 1, 2])
@pytest.mark.parametrize("rows", [1, 77, 3000])
def test_norm_rope(hd, rot, H, HK, normed, rows):
    rng = np.random.default_rng(hd + rot + rows)
    ld = (H + HK) * hd + 12
    x = rng.standard_normal((rows, ld)).astype(np.float32) * 3
    x[0, :hd] = 0
    x[-1, hd:2 * hd] *= 1e-18
    wq = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) if normed else None
    wk = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) if normed == 2 else None
    freq = (500000.0 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)
    pos = rng.integers(0, 2 ** 31 - 1, rows) if rows == 77 else rng.integers(0, 131072, rows)
    skip = np.zeros(rows, bool)
    skip[1::13] = True                                       # rows that are left as they are
    dx, df, dp = cuda(x), cuda(freq), i32(np.where(skip, -1, pos).tolist())
    dwq, dwk = cuda(wq) if wq is not None else None, cuda(wk) if wk is not None else None
    q, k = torch.full((rows, H * hd + 4), 7.0, device="cuda"), torch.full((rows, HK * hd), 7.0, device="cuda")
    call = native.lib().tf_op_qk_norm_rope
    native.check(call(ptr(q), H * hd + 4, ptr(k), HK * hd, ptr(dx), ld, ptr(dx) + 4 * H * hd, ld, ptr(dwq), ptr(dwk), 1e-6, ptr(df), rot,
                      ptr(dp), rows, H, HK, hd, None))
    torch.cuda.synchronize()
    gq, gk = q.cpu().numpy(), k.cpu().numpy()
    assert (gq[:, H * hd:] == 7).all() and (gq[skip] == 7).all() and (gk[skip] == 7).all()
    for got, a, b, w in ((gq[:, :H * hd], 0, H, wq), (gk, H, H + HK, wk)):
        want, tol = norm_rope_64(x[:, a * hd:b * hd].reshape(rows, -1, hd), w, 1e-6, freq, pos)
        err = np.abs(got.reshape(rows, -1, hd) - want) - tol
        assert (err[~skip] <= 1e-44).all(), err[~skip].max()
    # in place, and queries or keys alone
    dy = cuda(x)
    native.check(call(ptr(dy), ld, ptr(dy) + 4 * H * hd, ld, ptr(dy), ld, ptr(dy) + 4 * H * hd, ld, ptr(dwq), ptr(dwk), 1e-6, ptr(df), rot,
                      ptr(dp), rows, H, HK, hd, None))
    gy = dy.cpu().numpy()
    np.testing.assert_array_equal(gy[~skip, :H * hd], gq[~skip, :H * hd])
    np.testing.assert_array_equal(gy[~skip, H * hd:(H + HK) * hd], gk[~skip])
    np.testing.assert_array_equal(gy[skip], x[skip])
    np.testing.assert_array_equal(gy[:, (H + HK) * hd:], x[:, (H + HK) * hd:])
    q2, k2 = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    native.check(call(ptr(q2), H * hd + 4, None, 0, ptr(dx), ld, None, 0, ptr(dwq), None, 1e-6, ptr(df), rot, ptr(dp), rows, H, 0, hd, None))
    native.check(call(None, 0, ptr(k2), HK * hd, None, 0, ptr(dx) + 4 * H * hd, ld, None, ptr(dwk), 1e-6, ptr(df), rot, ptr(dp), rows, 0, HK,
                      hd, None))
    assert torch.equal(q2, q) and torch.equal(k2, k)


def test_rotation_of_values_that_are_not_finite():
    """An infinity or NaN reaches its own pair alone, as the formula has it, in queries and in keys."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 4, 64)).astype(np.float32)
    x[0, 0, 3], x[1, 1, 40], x[2, 2, 5], x[3, 3, 63], x[4, 3, 0] = np.inf, -np.inf, np.inf, np.nan, -np.inf
    pos, freq = np.array([5, 0, 9, 1, 0, 77]), (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    d, df, dp, out = cuda(x), cuda(freq), i32(pos.tolist()), torch.zeros((6, 4, 64), device="cuda")
    native.check(native.lib().tf_op_qk_norm_rope(ptr(out), 256, ptr(out) + 512, 256, ptr(d), 256, ptr(d) + 512, 256, None, None, 0.0, ptr(df), 64,
                                                 ptr(dp), 6, 2, 2, 64, None))
    with np.errstate(invalid="ignore"):
        want, tol = norm_rope_64(x, None, 0.0, freq, pos)
        got = out.cpu().numpy()
        fin = np.isfinite(want)
        assert (np.isfinite(got) == fin).all() and (np.isnan(got) == np.isnan(want)).all()
        assert (got[np.isinf(want)] == want[np.isinf(want)]).all()
        assert (np.abs(got - want) <= tol)[fin].all()


def test_norm_alone_and_copy():
    """Without a rotation no positions are needed; without weights either, rows are copied."""
    x = torch.randn((9, 6, 64), device="cuda")
    w = 1 + torch.rand(64, device="cuda")
    q, k = torch.zeros((9, 4, 64), device="cuda"), torch.zeros((9, 2, 64), device="cuda")
    native.check(native.lib().tf_op_qk_norm_rope(ptr(q), 256, ptr(k), 128, ptr(x), 384, ptr(x) + 1024, 384, ptr(w), None, 1e-5, None, 0, None, 9,
                                                 4, 2, 64, None))
    torch.cuda.synchronize()
    assert torch.equal(k, x[:, 4:])
    row = torch.zeros((36, 64), device="cuda")
    native.check(native.lib().tf_op_rmsnorm(ptr(row), ptr(x[:, :4].contiguous()), ptr(w), 64, 36, 1e-5, None))
    assert torch.equal(q.reshape(36, 64), row)               # the row norm's own rounding


# ---- the step's form -----------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("H,HK,hd,rot,rows", [(14, 2, 64, 64, 1), (12, 2, 128, 64, 50), (4, 4, 32, 32, 9), (6, 1, 96, 48, 130), (32, 8, 64, 64, 700)])
@pytest.mark.parametrize("normed", [0, 1])
def test_store_is_norm_rope_then_quant(kv, H, HK, hd, rot, rows, normed):
    rng = np.random.default_rng(rows)
    cap = 256
    a, b = (Cache(kv, hd, HK, cap, 4, 3).upload() for _ in range(2))
    ld = (H + 2 * HK) * hd
    x = cuda(rng.standard_normal((rows, ld)).astype(np.float32) * 2)
    w = cuda((1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32))
    wq, wk = (ptr(w), ptr(w) + 4 * hd) if normed else (None, None)
    freq = cuda((10000.0 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32))
    places = rng.permutation(4 * cap)[:rows]
    slots = places // cap
    slots[::5] = -1
    s, p = i32(slots.tolist()), i32((places % cap).tolist())
    at = lambda h: ptr(x) + 4 * h * hd
    L = native.lib()
    q1, q2, k2 = (torch.full((rows, n * hd), 7.0, device="cuda") for n in (H, H, HK))
    native.check(L.tf_op_qkv_store(ptr(q1), H * hd, *a.args(), ptr(s), ptr(p), at(0), ld, at(H), ld, at(H + HK), ld, wq, wk, 1e-6, ptr(freq), rot,
                                   rows, H, HK, hd, None))
    native.check(L.tf_op_qk_norm_rope(ptr(q2), H * hd, ptr(k2), HK * hd, at(0), ld, at(H), ld, wq, wk, 1e-6, ptr(freq), rot, ptr(p), rows, H, HK,
                                      hd, None))
    native.check(L.tf_op_kv_quant(*b.args(), ptr(s), ptr(p), ptr(k2), HK * hd, at(H + HK), ld, rows, HK, hd, None))
    assert device_error() == 0
    assert torch.equal(a.dk, b.dk) and torch.equal(a.dv, b.dv)
    keep = torch.from_numpy(slots >= 0).cuda()
    assert torch.equal(q1[keep], q2[keep]) and (q1[~keep] == 7.0).all()
    # queries in place, in a fused row
    y = x.clone()
    native.check(L.tf_op_qkv_store(ptr(y), ld, *b.args(), ptr(s), ptr(p), ptr(y), ld, ptr(y) + 4 * H * hd, ld, ptr(y) + 4 * (H + HK) * hd, ld, wq, wk,
                                   1e-6, ptr(freq), rot, rows, H, HK, hd, None))
    assert torch.equal(y[keep, :H * hd], q1[keep]) and torch.equal(y[~keep], x[~keep]) and torch.equal(y[:, H * hd:], x[:, H * hd:])
    assert torch.equal(a.dk, b.dk) and torch.equal(a.dv, b.dv)
    assert not torch.equal(a.dk.cpu(), torch.from_numpy(a.k)) or not keep.any()


# ---- attention -----------------------------------------------------------------------------------------

class Case:
    """One attention problem; cache rows that nobody may read hold random bytes (NaN scales among them)."""

    def __init__(self, kv, hd, H, HK, lens, news, T, seed, cap=None, q_size=1.0, gap=0):
        rng = np.random.default_rng(seed)
        self.hd, self.H, self.HK, self.lens, self.news, self.T, self.B = hd, H, HK, lens, news, T, len(lens)
        top = max(n + m for n, m in zip(lens, news))
        cap = cap or (top + 5 + 15) // 16 * 16
        self.c = c = Cache(kv, hd, HK, cap, self.B + 1, seed, gap)
        self.slots = rng.permutation(self.B + 1)[:self.B].tolist()
        for b in range(self.B):
            n = lens[b] + news[b]
            for kind in "kv":
                x = rng.standard_normal((HK, n, hd)).astype(np.float32) * (1.5 if kind == "k" else 0.7)
                self.fill(kind, b, 0, x)
        self.ld_q = (H + 2 * HK) * hd
        self.q = (rng.standard_normal((self.B, T, self.ld_q)) * q_size).astype(np.float32)

    def fill(self, kind, b, first, x):
        """Rows x [HK][n][hd] at positions first .. of sequence b, on the host, a block at a time."""
        c = self.c
        at, shift, sat = lay.tables(kind, c.kv, c.hd)
        codes, scales = lay.quantise(c.kv, x)
        blocks = getattr(c, kind)[self.slots[b]]
        bits = lay.BITS[c.kv]
        pos = np.arange(first, first + x.shape[1])
        for p in range(16):
            rows = np.nonzero(pos % 16 == p)[0]
            if not len(rows):
                continue
            blk = pos[rows] // 16
            for h in range(c.HK):
                cur = blocks[h][blk]
                for s in range(0, 8, bits):
                    e = np.nonzero(shift[p] == s)[0]
                    if len(e):
                        keep = 255 ^ ((2 ** bits - 1) << s)
                        cur[:, at[p, e]] = (cur[:, at[p, e]] & keep) | (codes[h][rows][:, e] << s)
                raw = scales[h][rows].astype(np.float16).view(np.uint16)
                cur[:, sat[p]] = raw & 255
                cur[:, sat[p] + 1] = raw >> 8
                blocks[h][blk] = cur

    def run(self, stream=None, ws=None, upload=True, **kw):
        L, c = native.lib(), self.c
        if upload:
            c.upload()
            self.dq = cuda(self.q)
            self.ld_out = self.H * self.hd + 4
            self.out = torch.full((self.B, self.T, self.ld_out), 7.0, device="cuda")
            self.meta = dict(slots=i32(self.slots), n_ctx=i32(self.lens), n_new=i32(self.news))
        m = dict(self.meta, **kw)
        if ws is None:
            ws = self.workspace()
        self.ws = ws
        native.check(L.tf_op_attn_quant(ptr(self.out), self.ld_out, ptr(self.dq), self.ld_q, *c.args(), ptr(m["slots"]), ptr(m["n_ctx"]),
                                        ptr(m["n_new"]), self.B, self.T, self.H, self.HK, self.hd, ptr(ws), ws.numel(), stream))
        return self

    def workspace(self):
        n = C.c_size_t(0)
        native.check(native.lib().tf_op_attn_quant_workspace(self.B, self.T, self.H, self.HK, self.hd, C.byref(n)))
        return torch.full((n.value,), 255, dtype=torch.uint8, device="cuda")

    def got(self):
        torch.cuda.synchronize()
        assert (self.out[..., self.H * self.hd:] == 7.0).all()
        return self.out[..., :self.H * self.hd].reshape(self.B, self.T, self.H, self.hd).double().cpu().numpy()

    def want(self, b):
        H, HK, hd, n, m = self.H, self.HK, self.hd, self.lens[b], self.news[b]
        out, tol = np.zeros((self.T, H, hd)), np.zeros((self.T, H, 1))
        k, v = self.c.values("k", self.slots[b], n + m), self.c.values("v", self.slots[b], n + m)
        rep = H // HK
        for t in range(m):
            e = n + t + 1
            q = self.q[b, t, :H * hd].reshape(HK, rep, hd).astype(np.float64)
            s = np.einsum("grd,gnd->grn", q, k[:, :e]) / hd ** 0.5
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[t] = np.einsum("grn,gnd->grd", p, v[:, :e]).reshape(H, hd)
            d = hd * 2.0 ** -23 * np.einsum("grd,gnd->grn", np.abs(q), np.abs(k[:, :e])).max(-1) / hd ** 0.5
            tol[t, :, 0] = ((2 * d + 2.0 ** -18) * np.abs(v[:, :e]).max((1, 2))[:, None]).reshape(-1)
        return out, tol

    def check(self, got=None):
        got = self.got() if got is None else got
        assert device_error() == 0
        for b in range(self.B):
            want, tol = self.want(b)
            err = np.abs(got[b] - want) - tol
            assert (err <= 0).all(), (b, err.max())
            assert np.linalg.norm(got[b] - want) <= 5e-6 * np.linalg.norm(want), b
        return self


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd,H,HK", [(32, 4, 4), (64, 14, 2), (64, 32, 8), (96, 6, 2), (128, 12, 2), (128, 32, 8), (64, 24, 1), (128, 5, 5)])
@pytest.mark.parametrize("T", [1, 2, 5])
def test_attention(kv, hd, H, HK, T):
    lens = [0, 1, 14, 15, 16, 17, 130, 700]
    Case(kv, hd, H, HK, lens, [T] * len(lens), T, hd + T).run().check()


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd,H,HK,T,lens", [(64, 8, 2, 1, [9000]), (128, 4, 1, 1, [20011]), (64, 14, 2, 3, [6001, 5, 4090]), (128, 16, 2, 16, [1000]),
                                            (32, 8, 8, 64, [333, 0]), (96, 12, 3, 7, [2047, 2048])])
def test_attention_split_over_ctas(kv, hd, H, HK, T, lens):
    Case(kv, hd, H, HK, lens, [T] * len(lens), T, T).run().check()


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd,H,HK,T", [(64, 8, 2, 1), (128, 6, 1, 1), (32, 10, 2, 3), (96, 6, 3, 20)])
def test_short_contexts_in_a_long_cache(kv, hd, H, HK, T):
    """The split is chosen by the capacity: short and empty contexts where long ones could be."""
    lens = [0, 1, 95, 96, 97, 370, 13, 0, 1800]
    news = [T, T, T, T, T, T, 0, 1, max(1, T - 1)]
    Case(kv, hd, H, HK, lens, news, T, 3 * T, cap=8192).run().check()


@pytest.mark.parametrize("n", [385, 480, 481, 800, 1137])
def test_every_cut(n):
    """Ranges that end next to a unit's first and last blocks."""
    Case(native.TF_KV_Q4_0, 32, 4, 4, [n, n + 30, 5, n - 16], [1, 1, 1, 1], 1, n, cap=8192).run().check()


@pytest.mark.parametrize("cap", [0, 8192])
def test_two_streams_at_once(cap):
    """Calls in flight together, each with its workspace; then both through one workspace, one after the other."""
    a = Case(native.TF_KV_Q4_0, 64, 8, 2, [900, 40], [1, 1], 1, 1, cap=cap or None).run()
    b = Case(native.TF_KV_Q8_0, 64, 14, 2, [700, 1111], [2, 2], 2, 2, cap=cap or None).run()
    one, two = a.got(), b.got()
    a.check(one), b.check(two)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    a.out.zero_(), b.out.zero_()
    a.out[..., a.H * a.hd:] = b.out[..., b.H * b.hd:] = 7.0
    torch.cuda.synchronize()
    for _ in range(20):
        a.run(stream=s.cuda_stream, ws=a.ws, upload=False)
        b.run(stream=t.cuda_stream, ws=b.ws, upload=False)
    assert (a.got() == one).all() and (b.got() == two).all()
    big = a.ws if a.ws.numel() > b.ws.numel() else b.ws
    graphs = []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.run(stream=s.cuda_stream, ws=big, upload=False)
        graphs.append(g)
    for c in (a, b):
        c.out[..., :c.H * c.hd] = 0
    with torch.cuda.stream(s):
        for _ in range(5):
            for g in graphs:
                g.replay()
    torch.cuda.synchronize()
    assert (a.got() == one).all() and (b.got() == two).all()


def test_many_sequences():
    """More sequences than lanes and CTAs, most of them short."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 60, 700).tolist()
    news = rng.integers(0, 3, 700).tolist()
    Case(native.TF_KV_Q4_0, 32, 2, 1, lens, news, 2, 4).run().check()


@pytest.mark.parametrize("kv", TYPES)
def test_rows_behind_the_new_ones_are_zero(kv):
    Case(kv, 64, 8, 2, [40, 0, 33, 7], [3, 0, 0, 5], 5, 1, gap=1).run().check()


@pytest.mark.parametrize("kv", TYPES)
def test_without_slots_and_counts(kv):
    c = Case(kv, 64, 4, 2, [20, 50, 3], [2, 2, 2], 2, 6)
    c.slots = [0, 1, 2]
    rng = np.random.default_rng(9)
    for b in range(3):
        for kind in "kv":
            c.fill(kind, b, 0, rng.standard_normal((2, c.lens[b] + 2, 64)).astype(np.float32))
    c.run(slots=None, n_new=None).check()


@pytest.mark.parametrize("cap", [96, 8192])
def test_sequences_that_do_not_fit(cap):
    """Refused on the device: their rows are zero, the others' are right."""
    c = Case(native.TF_KV_Q4_0, 64, 8, 2, [40, 90, 33, 20], [2, 2, 2, 2], 2, 1, cap=cap).run()
    good = c.got()
    for bad, code in [(dict(slots=[9, 1, 2, 3]), 0), (dict(slots=[-1, 1, 2, 3]), 0), (dict(n_ctx=[40, cap - 1, 33, 20]), 1), (dict(n_ctx=[-1, 90, 33, 20]), 0),
                      (dict(n_new=[2, 2, -1, 2]), 2)]:
        kw = {k: i32(v if k != "slots" else [s if not 0 <= s < 4 or i == code else c.slots[i] for i, s in enumerate(v)]) for k, v in bad.items()}
        c.out.fill_(7.0)
        c.run(upload=False, **kw)
        got = c.got()
        assert device_error() == native.TF_DEV_ERR_POS
        for b in range(4):
            assert (got[b] == (0 if b == code else good[b])).all(), (bad, b)


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("T", [1, 3, 9])
def test_what_a_row_does_not_see(kv, T):
    """A later row's key and value, however large or not finite, leave an earlier row's bits alone."""
    c = Case(kv, 64, 4, 2, [75, 16], [T, T], T, 2)
    first = c.run().check().got()
    rng = np.random.default_rng(0)
    for value in (5e5, np.nan, np.inf):
        x = (rng.standard_normal((2, 1, 64)) * value).astype(np.float32)
        for b in range(2):
            for kind in "kv":
                c.fill(kind, b, c.lens[b] + T - 1, x)
        got = c.run().got()
        assert (got[:, :T - 1] == first[:, :T - 1]).all()
        if value != value or value == np.inf:
            assert np.isnan(got[:, T - 1]).all()


@pytest.mark.parametrize("kv", TYPES)
def test_sizes_far_apart(kv):
    """Values of very different sizes, in every group: errors are relative to the largest that a row sees."""
    c = Case(kv, 64, 8, 2, [300], [1], 1, 3)
    rng = np.random.default_rng(1)
    for exps in ((-14, 0), (0, 14), (-18, -16)):
        x = rng.standard_normal((2, 301, 64)) * 2.0 ** rng.integers(*exps, (2, 301, 1))
        c.fill("v", 0, 0, x.astype(np.float32))
        c.run().check()
    for size in (2.0 ** -60, 2.0 ** -20, 2.0 ** 40):         # queries too; keys the other way round
        c.q = (rng.standard_normal(c.q.shape) * size).astype(np.float32)
        k = rng.standard_normal((2, 301, 64)) * min(1.0 / size, 2.0 ** 12)
        if size > 2.0 ** 12:
            k *= 2.0 ** -12
            c.q *= np.float32(2.0 ** -24)
        c.fill("k", 0, 0, k.astype(np.float32))
        c.run().check()


@pytest.mark.parametrize("kv", TYPES)
def test_equal_scores_and_sharp_ones(kv):
    c = Case(kv, 128, 4, 1, [513], [1], 1, 3, q_size=0.0).run().check()
    for size in (20.0, 200.0):                               # one position takes (almost) all
        c.q = (np.random.default_rng(2).standard_normal(c.q.shape) * size).astype(np.float32)
        got = c.run().got()
        want, tol = c.want(0)
        assert (np.abs(got[0] - want) <= tol).all()


@pytest.mark.parametrize("kv", TYPES)
def test_maximum_that_keeps_growing(kv):
    """Scores that rise from position to position, and V scales with them: the running references move."""
    c = Case(kv, 64, 4, 1, [800], [2], 2, 3)
    ramp = np.linspace(-3, 3, 802)[None, :, None]
    c.q[:] = np.abs(c.q)
    c.fill("k", 0, 0, np.broadcast_to(ramp, (1, 802, 64)).astype(np.float32))
    rng = np.random.default_rng(4)
    c.fill("v", 0, 0, (rng.standard_normal((1, 802, 64)) * 2.0 ** (3 * ramp)).astype(np.float32))
    c.run().check()
    c.fill("v", 0, 0, (rng.standard_normal((1, 802, 64)) * 2.0 ** (-3 * ramp)).astype(np.float32))
    c.run().check()


@pytest.mark.parametrize("kv", TYPES)
def test_zero_and_not_finite(kv):
    c = Case(kv, 64, 4, 2, [40], [1], 1, 3)
    z = np.zeros((2, 41, 64), np.float32)
    c.fill("v", 0, 0, z)
    assert (c.run().got() == 0).all()
    c.fill("k", 0, 0, z)
    c.run().check()
    v = np.random.default_rng(0).standard_normal((2, 41, 64)).astype(np.float32)
    c.fill("v", 0, 0, v)
    v[1, 7, 40] = np.nan                                     # one group of one kv head
    c.fill("v", 0, 0, v)
    got = c.run().got()
    assert np.isnan(got[0, 0, 2:, 32:]).all() and np.isfinite(got[0, 0, 2:, :32]).all() and np.isfinite(got[0, 0, :2]).all()
    c.fill("v", 0, 0, z)
    c.q[0, 0, 0] = np.inf                                    # head 0 alone
    got = c.run().got()
    assert np.isnan(got[0, 0, 0]).all() and np.isfinite(got[0, 0, 1:]).all()


@pytest.mark.parametrize("kv", TYPES)
def test_rows_do_not_hang_on_the_batch(kv):
    """Bits repeat from call to call, and a whole sequence's do not change with its neighbours' values."""
    c = Case(kv, 64, 8, 2, [300, 200], [3, 3], 3, 8).run()
    a = c.got()
    assert (c.run(ws=c.ws).got() == a).all()
    c.fill("v", 1, 0, np.full((2, 203, 64), 1e5, np.float32))
    b = c.run().got()
    assert (a[0] == b[0]).all() and not (a[1] == b[1]).all()


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB per side: the last slot's last positions."""
    kv, hd, HK, cap, n_slots = native.TF_KV_Q8_0, 128, 8, 65536, 70
    L = native.lib()
    shape = (n_slots, HK, cap // 16, lay.block_bytes(kv, hd))
    dk, dv = torch.zeros(shape, dtype=torch.uint8, device="cuda"), torch.zeros(shape, dtype=torch.uint8, device="cuda")
    assert dk.numel() > 1 << 32
    args = (ptr(dk), ptr(dv), kv, HK * cap * hd, cap, n_slots)
    n = 50
    x = torch.randn((n, 2, HK * hd), device="cuda")
    s, p = i32([n_slots - 1] * n), i32(range(cap - n, cap))
    native.check(L.tf_op_kv_quant(*args, ptr(s), ptr(p), ptr(x), 2 * HK * hd, ptr(x) + 4 * HK * hd, 2 * HK * hd, n, HK, hd, None))
    back = torch.zeros_like(x)
    native.check(L.tf_op_kv_dequant(ptr(back), 2 * HK * hd, ptr(back) + 4 * HK * hd, 2 * HK * hd, *args, ptr(s), ptr(p), n, HK, hd, None))
    assert device_error() == 0
    group = x.reshape(n, 2, HK, 4, 32).abs().amax(-1, keepdim=True)
    # half a step, the step's own rounding on 127 of them, and what clipping adds
    assert ((back - x).reshape(n, 2, HK, 4, 32).abs() <= group / 127 * (0.5 + 127 * 2.0 ** -11)).all()
    assert not dk[:-1].any() and not dk[-1, :, :-4].any()
    q = torch.randn((1, 1, HK * hd), device="cuda") * 8
    out = torch.zeros_like(q)
    nb = C.c_size_t(0)
    native.check(L.tf_op_attn_quant_workspace(1, 1, HK, HK, hd, C.byref(nb)))
    ws = torch.empty(nb.value, dtype=torch.uint8, device="cuda")
    slots, ctx = i32([n_slots - 1]), i32([cap - 1])
    native.check(L.tf_op_attn_quant(ptr(out), HK * hd, ptr(q), HK * hd, *args, ptr(slots), ptr(ctx), None, 1, 1, HK, HK, hd, ptr(ws), nb.value,
                                    None))
    kk, vv = (torch.zeros((HK, cap, hd), dtype=torch.float64, device="cuda") for _ in range(2))
    kk[:, -n:] = back[:, 0].double().reshape(n, HK, hd).transpose(0, 1)
    vv[:, -n:] = back[:, 1].double().reshape(n, HK, hd).transpose(0, 1)
    w = torch.softmax(torch.einsum("hd,hnd->hn", q.double().reshape(HK, hd), kk) / hd ** 0.5, -1)
    want = torch.einsum("hn,hnd->hd", w, vv)
    assert (out.double().reshape(HK, hd) - want).norm() <= 5e-6 * want.norm()


@pytest.mark.parametrize("kv", TYPES)
def test_long_sums_do_not_drift(kv):
    """Values of one sign over a cache that a warp walks for hundreds of blocks: an accumulator that truncates loses
    2^-24 of the sum at every step (2.5e-5 in all), which the norm's bound does not allow."""
    B, HK, rep, hd, n = 80, 8, 6, 32, 16384
    L = native.lib()
    nb = lay.block_bytes(kv, hd)
    codes = 16 * hd * lay.BITS[kv] // 8
    g = torch.Generator(device="cuda").manual_seed(1)
    c = torch.randint(0, 256, (2, B, HK, n // 16, nb), generator=g, device="cuda", dtype=torch.uint8)
    c[1, ..., :codes] |= 0x88 if kv == native.TF_KV_Q4_0 else 0x80     # values are not negative
    scale = (0.02 + 0.1 * torch.rand((2, B, HK, n // 16, hd // 2), generator=g, device="cuda")).half()
    c[..., codes:] = scale.view(torch.uint8)
    q = torch.randn((B, HK * rep * hd), generator=g, device="cuda")
    out = torch.zeros_like(q)
    ctx = i32([n - 1] * B)
    size = C.c_size_t(0)
    native.check(L.tf_op_attn_quant_workspace(B, 1, HK * rep, HK, hd, C.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    native.check(L.tf_op_attn_quant(ptr(out), HK * rep * hd, ptr(q), HK * rep * hd, ptr(c[0]), ptr(c[1]), kv, HK * n * hd, n, B, None, ptr(ctx), None,
                                    B, 1, HK * rep, HK, hd, ptr(ws), size.value, None))
    assert device_error() == 0
    for b, h in ((0, 0), (37, 5), (79, 7)):
        k, v = (torch.from_numpy(lay.values(c[i, b, h].cpu().numpy(), kind, kv, hd).reshape(n, hd)).cuda() for i, kind in ((0, "k"), (1, "v")))
        w = torch.softmax(q[b].double().reshape(HK, rep, hd)[h] @ k.T / hd ** 0.5, -1) @ v
        got = out[b].double().reshape(HK, rep, hd)[h]
        assert (got - w).norm() <= 5e-6 * w.norm(), float((got - w).norm() / w.norm())


# ---- together --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("captured", [False, True])
def test_a_few_steps_together(kv, captured):
    """A packed prompt into the cache, then decode steps of a batch (store, then attention) on a stream of their own,
    eager or as one graph replayed with the lengths on the device; each step against 64 bits over what the
    cache holds."""
    H, HK, hd, cap, B, steps = 14, 2, 64, 128, 3, 4
    L = native.lib()
    rng = np.random.default_rng(5)
    c = Cache(kv, hd, HK, cap, B + 1, 7).upload()
    slots = [2, 0, 3]
    lens = [33, 1, 60]
    freq = cuda((10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32))
    w = cuda((1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32))
    ld = (H + 2 * HK) * hd
    at = lambda x, h: ptr(x) + 4 * h * hd
    prompt = cuda(rng.standard_normal((sum(lens), ld)).astype(np.float32))
    ps, pp = i32([s for s, n in zip(slots, lens) for _ in range(n)]), i32([i for n in lens for i in range(n)])
    pq = torch.empty((sum(lens), H * hd), device="cuda")
    native.check(L.tf_op_qkv_store(ptr(pq), H * hd, *c.args(), ptr(ps), ptr(pp), at(prompt, 0), ld, at(prompt, H), ld, at(prompt, H + HK), ld,
                                   ptr(w), ptr(w) + 4 * hd, 1e-6, ptr(freq), hd, sum(lens), H, HK, hd, None))
    torch.cuda.synchronize()
    x = torch.empty((B, ld), device="cuda")
    q, out = torch.empty((B, H * hd), device="cuda"), torch.empty((B, H * hd), device="cuda")
    ds, n_ctx = i32(slots), i32(lens)
    nb = C.c_size_t(0)
    native.check(L.tf_op_attn_quant_workspace(B, 1, H, HK, hd, C.byref(nb)))
    ws = torch.empty(nb.value, dtype=torch.uint8, device="cuda")

    def step(stream):
        native.check(L.tf_op_qkv_store(ptr(q), H * hd, *c.args(), ptr(ds), ptr(n_ctx), at(x, 0), ld, at(x, H), ld, at(x, H + HK), ld, ptr(w),
                                       ptr(w) + 4 * hd, 1e-6, ptr(freq), hd, B, H, HK, hd, stream))
        native.check(L.tf_op_attn_quant(ptr(out), H * hd, ptr(q), H * hd, *c.args(), ptr(ds), ptr(n_ctx), None, B, 1, H, HK, hd, ptr(ws),
                                        nb.value, stream))
        n_ctx.add_(1)

    side, graph = torch.cuda.Stream(), None
    if captured:
        x.zero_()
        with torch.cuda.stream(side):
            step(side.cuda_stream)                           # the kernels' attributes are set before the capture
            n_ctx.sub_(1)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(side.cuda_stream)
    for i in range(steps):
        new = cuda(rng.standard_normal((B, ld)).astype(np.float32))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            x.copy_(new)
            graph.replay() if captured else step(side.cuda_stream)
        side.synchronize()
        assert device_error() == 0
        c.k, c.v = c.dk.cpu().numpy(), c.dv.cpu().numpy()
        hx, hw = new.cpu().numpy().reshape(B, -1, hd), w.cpu().numpy()
        pos = np.array([n + i for n in lens])
        assert n_ctx.tolist() == (pos + 1).tolist()
        q64, tol = norm_rope_64(hx[:, :H], hw[0], 1e-6, freq.cpu().numpy(), pos)
        assert (np.abs(q.cpu().numpy().reshape(B, H, hd) - q64) <= tol).all()
        for b in range(B):
            n = lens[b] + i + 1
            k, v = c.values("k", slots[b], n), c.values("v", slots[b], n)
            scale = np.abs(hx[b, H + HK:].reshape(HK, 2, 32)).max(-1, keepdims=True)
            off = np.abs(v[:, n - 1].reshape(HK, 2, 32) - hx[b, H + HK:].reshape(HK, 2, 32))
            assert (off <= scale * (1.01 / 8 if kv == native.TF_KV_Q4_0 else 0.6 / 127)).all()
            s = np.einsum("grd,gnd->grn", q[b].double().cpu().numpy().reshape(HK, H // HK, hd), k) / hd ** 0.5
            p = np.exp(s - s.max(-1, keepdims=True))
            want = np.einsum("grn,gnd->grd", p / p.sum(-1, keepdims=True), v).reshape(-1)
            got = out[b].double().cpu().numpy()
            assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)
