"""The quantised cache's row operators where a warp has several vectors of keys and values: from some hundred rows
on, a row's heads are no longer shared out among warps.  Everything here is compared byte by byte, bit by bit, or
with a 64-bit result rounded once."""
import numpy as np
import pytest

import kvq_layout as lay
from test_gpu_kvq import Cache, TYPES, awkward_rows, cuda, device_error, i32, ptr
from tinferno_b200 import native

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def put_rows(c, kind, slots, pos, x):
    """Rows x [n][HK][hd] into the host's cache at (slots, pos), by place in the block."""
    at, shift, sat = lay.tables(kind, c.kv, c.hd)
    codes, scales = lay.quantise(c.kv, x)
    raw, mem, bits = scales.astype(np.float16).view(np.uint16), getattr(c, kind), lay.BITS[c.kv]
    for p in range(16):
        r = np.nonzero((pos % 16 == p) & (slots >= 0))[0]
        if not len(r):
            continue
        where = (slots[r][:, None], np.arange(c.HK)[None], (pos[r] // 16)[:, None])
        cur = mem[where]
        for s in range(0, 8, bits):
            e = np.nonzero(shift[p] == s)[0]
            if len(e):
                cur[..., at[p, e]] = (cur[..., at[p, e]] & (255 ^ ((2 ** bits - 1) << s))) | (codes[r][..., e] << s)
        cur[..., sat[p]] = raw[r] & 255
        cur[..., sat[p] + 1] = raw[r] >> 8
        mem[where] = cur


def host_rows(c, kind, slots, pos):
    """[n][HK][hd] in fp32, as the definition reads them."""
    blocks = getattr(c, kind)[slots, :c.HK, pos // 16]
    v = lay.values(blocks.reshape(-1, blocks.shape[-1]), kind, c.kv, c.hd).reshape(len(slots), c.HK, 16, c.hd)
    return v[np.arange(len(slots)), :, pos % 16].astype(np.float32)


def places(rng, rows, n_slots, cap):
    """Rows of packed prompts (one position after another), then rows anywhere, all at distinct places; every 17th is left
    out."""
    free = rng.permutation(n_slots * cap)
    slots, pos, taken = [], [], set()
    for s in range(n_slots):
        n, first = min(cap // 2, rows // (2 * n_slots)), int(rng.integers(0, cap // 2))
        slots += [s] * n
        pos += range(first, first + n)
    taken = {s * cap + p for s, p in zip(slots, pos)}
    for f in free:
        if len(slots) == rows:
            break
        if f not in taken:
            slots.append(int(f) // cap)
            pos.append(int(f) % cap)
    slots, pos = np.array(slots), np.array(pos)
    slots[5::17] = -1
    return slots, pos


# (hd, kv heads, rows): one vector a warp for each of four heads' places and more, and more than four
MANY = [(64, 8, 3000), (128, 8, 3001), (128, 24, 1200), (96, 5, 2999), (32, 40, 1500)]


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd,HK,rows", MANY)
def test_write_and_read(kv, hd, HK, rows):
    rng = np.random.default_rng(rows + hd)
    n_slots, cap = 3, (rows + 47) // 48 * 32
    c = Cache(kv, hd, HK, cap, n_slots, rows, gap=1).upload()
    corners = awkward_rows(rng, 40, 1, 32).reshape(40, 32)
    x = (rng.standard_normal((rows, 2 * HK, hd)) * 2).astype(np.float32)
    groups = x.reshape(-1, 32)
    some = rng.random(len(groups)) < 0.3                      # groups of all kinds beside one another
    groups[some] = corners[rng.integers(0, 40, int(some.sum()))]
    slots, pos = places(rng, rows, n_slots, cap)
    put_rows(c, "k", slots, pos, x[:, :HK])
    put_rows(c, "v", slots, pos, x[:, HK:])
    d, s, p = cuda(x.reshape(rows, -1)), i32(slots.tolist()), i32(pos.tolist())
    ld, L = 2 * HK * hd, native.lib()
    native.check(L.tf_op_kv_quant(*c.args(), ptr(s), ptr(p), ptr(d), ld, ptr(d) + 4 * HK * hd, ld, rows, HK, hd, None))
    assert device_error() == 0
    assert c.same()
    back = torch.full((rows, ld + 4), 7.0, device="cuda")
    native.check(L.tf_op_kv_dequant(ptr(back), ld + 4, ptr(back) + 4 * HK * hd, ld + 4, *c.args(), ptr(s), ptr(p), rows, HK, hd, None))
    assert device_error() == 0
    got, keep = back.cpu().numpy(), slots >= 0
    assert (got[:, ld:] == 7).all() and (got[~keep] == 7).all()
    for i, kind in enumerate("kv"):
        want = host_rows(c, kind, slots[keep], pos[keep])
        np.testing.assert_array_equal(got[keep, i * HK * hd:(i + 1) * HK * hd].reshape(want.shape), want)


@pytest.mark.parametrize("kv", TYPES)
def test_the_same_place_read_twice(kv):
    """Reading has no distinct places: a row per request, the same one several times, in any order."""
    HK, hd, cap = 3, 64, 64
    c = Cache(kv, hd, HK, cap, 2, 3)
    x = np.random.default_rng(0).standard_normal((cap, 2 * HK, hd)).astype(np.float32)
    for slot in range(2):
        for i, kind in enumerate("kv"):
            put_rows(c, kind, np.full(cap, slot), np.arange(cap), x[:, i * HK:(i + 1) * HK] * (slot + 1))
    c.upload()
    slots = np.array([0, 0, 0, 1, 1, 0, 0, 1, 1, 1, 0, 0, 0, 0])
    pos = np.array([5, 5, 6, 6, 7, 7, 6, 63, 0, 0, 1, 9, 9, 2])
    s, p, out = i32(slots.tolist()), i32(pos.tolist()), torch.zeros((len(pos), 2, HK * hd), device="cuda")
    native.check(native.lib().tf_op_kv_dequant(ptr(out), 2 * HK * hd, ptr(out) + 4 * HK * hd, 2 * HK * hd, *c.args(), ptr(s), ptr(p), len(pos),
                                               HK, hd, None))
    assert device_error() == 0
    for i, kind in enumerate("kv"):
        want = host_rows(c, kind, slots, pos)
        np.testing.assert_array_equal(out[:, i].cpu().numpy().reshape(want.shape), want)


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("H,HK,hd,rot,rows", [(32, 8, 64, 64, 3000), (32, 8, 128, 64, 2500), (8, 24, 128, 128, 3000), (6, 1, 96, 48, 13),
                                              (4, 40, 32, 32, 1500), (12, 2, 128, 0, 50), (32, 8, 64, 0, 3000), (8, 24, 128, 0, 1200),
                                              (6, 3, 96, 0, 2000), (3, 7, 32, 0, 7)])
@pytest.mark.parametrize("normed", ["", "q", "k", "qk"])
def test_store_is_norm_rope_then_quant(kv, H, HK, hd, rot, rows, normed):
    """With a rotation and without (rot 0), norms of either kind alone: the step's form against its two parts, whose
    results at these sizes are compared with 64 bits and byte by byte."""
    rng = np.random.default_rng(rows + HK)
    n_slots, cap = 3, (rows + 47) // 48 * 32
    a, b = (Cache(kv, hd, HK, cap, n_slots, 3).upload() for _ in range(2))
    ld = (H + 2 * HK) * hd
    x = cuda(rng.standard_normal((rows, ld)).astype(np.float32) * 2)
    w = cuda((1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32))
    wq, wk = ptr(w) if "q" in normed else None, ptr(w) + 4 * hd if "k" in normed else None
    freq = cuda((10000.0 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)) if rot else None
    slots, pos = places(rng, rows, n_slots, cap)
    s, p = i32(slots.tolist()), i32(pos.tolist())
    at = lambda h: ptr(x) + 4 * h * hd
    L = native.lib()
    q1, q2, k2 = (torch.full((rows, n * hd), 7.0, device="cuda") for n in (H, H, HK))
    native.check(L.tf_op_qkv_store(ptr(q1), H * hd, *a.args(), ptr(s), ptr(p), at(0), ld, at(H), ld, at(H + HK), ld, wq, wk, 1e-6, ptr(freq), rot,
                                   rows, H, HK, hd, None))
    native.check(L.tf_op_qk_norm_rope(ptr(q2), H * hd, ptr(k2), HK * hd, at(0), ld, at(H), ld, wq, wk, 1e-6, ptr(freq), rot, ptr(p), rows, H, HK,
                                      hd, None))
    assert device_error() == 0
    keep = torch.from_numpy(slots >= 0).cuda()
    assert torch.equal(q1[keep], q2[keep]) and (q1[~keep] == 7.0).all()
    for i, rowsof in enumerate((k2.cpu().numpy(), x[:, (H + HK) * hd:].cpu().numpy())):
        put_rows(b, "kv"[i], slots, pos, rowsof.reshape(rows, HK, hd))
    assert np.array_equal(a.dk.cpu().numpy(), b.k) and np.array_equal(a.dv.cpu().numpy(), b.v)
    if not rot and not normed:
        assert torch.equal(q1[keep], x[keep, :H * hd]) and torch.equal(k2, x[:, H * hd:(H + HK) * hd])


@pytest.mark.parametrize("rot", [0, 64])
def test_stored_rows_outside_the_cache(rot):
    """The step's form leaves such rows out, in the caches and in q_out, and reports them."""
    H, HK, hd, cap = 4, 2, 64, 32
    rng = np.random.default_rng(2)
    freq = cuda((10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)) if rot else None
    x = cuda(rng.standard_normal((5, (H + 2 * HK) * hd)).astype(np.float32))
    ld, L = (H + 2 * HK) * hd, native.lib()
    for slots, pos, code in [([0, 3, 0, 0, 1], [1, 2, 3, 4, 5], native.TF_DEV_ERR_BAD_INDEX),
                             ([0, 1, 0, 0, 1], [1, 2, 32, 4, 5], native.TF_DEV_ERR_POS),
                             ([0, 1, 0, 0, 1], [1, 2, 3, -1, 5], native.TF_DEV_ERR_POS)]:
        c = Cache(native.TF_KV_Q8_0, hd, HK, cap, 3, 1).upload()
        s, p = i32(slots), i32(pos)
        q, q2, k2 = (torch.full((5, n * hd), 7.0, device="cuda") for n in (H, H, HK))
        native.check(L.tf_op_qkv_store(ptr(q), H * hd, *c.args(), ptr(s), ptr(p), ptr(x), ld, ptr(x) + 4 * H * hd, ld,
                                       ptr(x) + 4 * (H + HK) * hd, ld, None, None, 0.0, ptr(freq), rot, 5, H, HK, hd, None))
        assert device_error() == code
        native.check(L.tf_op_qk_norm_rope(ptr(q2), H * hd, ptr(k2), HK * hd, ptr(x), ld, ptr(x) + 4 * H * hd, ld, None, None, 0.0, ptr(freq), rot,
                                          ptr(p), 5, H, HK, hd, None))
        torch.cuda.synchronize()
        ok = np.array([0 <= u < 3 and 0 <= v < cap for u, v in zip(slots, pos)])
        put_rows(c, "k", np.where(ok, slots, -1), np.array(pos), k2.cpu().numpy().reshape(5, HK, hd))
        put_rows(c, "v", np.where(ok, slots, -1), np.array(pos), x[:, (H + HK) * hd:].cpu().numpy().reshape(5, HK, hd))
        assert c.same()
        for r in range(5):
            assert torch.equal(q[r], q2[r]) if ok[r] else bool((q[r] == 7.0).all())


@pytest.mark.parametrize("rows", [400, 3000])
def test_norm_without_a_rotation(rows):
    """The norm alone, at many rows, is the row norm of each head."""
    H, HK, hd = 12, 4, 64
    x = torch.randn((rows, H + HK, hd), device="cuda")
    w = 1 + torch.rand((2, hd), device="cuda")
    q, k, one = torch.zeros((rows, H, hd), device="cuda"), torch.zeros((rows, HK, hd), device="cuda"), torch.zeros((rows * (H + HK), hd), device="cuda")
    L, ld = native.lib(), (H + HK) * hd
    native.check(L.tf_op_qk_norm_rope(ptr(q), H * hd, ptr(k), HK * hd, ptr(x), ld, ptr(x) + 4 * H * hd, ld, ptr(w), ptr(w) + 4 * hd, 1e-5, None, 0,
                                      None, rows, H, HK, hd, None))
    for got, part, i in ((q, x[:, :H], 0), (k, x[:, H:], 1)):
        flat = part.reshape(-1, hd).contiguous()
        out = one[:len(flat)]
        native.check(L.tf_op_rmsnorm(ptr(out), ptr(flat), ptr(w) + 4 * hd * i, hd, len(flat), 1e-5, None))
        assert torch.equal(got.reshape(-1, hd), out)
