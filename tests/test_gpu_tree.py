"""Speculative decoding operators (tf_op_attn_tree, tf_op_verify_tree, tf_op_kv_commit) against plain
implementations in 64 bits, at the sizes, masks and values where they can go wrong.

Tolerance of the attention, fixed before its first run.  Operands and probabilities carry at
least 22 significant bits and sums are fp32, so a score of hd products is off by at most about
d = hd 2^-23 max_j(scale sum |q k_j|), every probability by a factor 1 +- d, and the output by
(2 d + 2^-18) max |v|.  That bound is for the worst case; errors of 2^-22 that do not conspire
leave a 2-norm error of a few 2^-22 relative to the output, so the norm is held to 5e-6, which a
rounding of any operand to 11 bits (2e-4) or 16 bits (4e-6 for each of four operands) does not
meet."""
import ctypes as C

import numpy as np
import pytest

from tinferno_b200 import native

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

KV = {native.TF_KV_F32: torch.float32, native.TF_KV_F16: torch.float16, native.TF_KV_BF16: torch.bfloat16}


def ptr(t):
    return None if t is None else t.data_ptr()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def workspace(fn, *shape):
    n = C.c_size_t(0)
    native.check(fn(*shape, C.byref(n)))
    return torch.zeros(max(1, n.value), dtype=torch.uint8, device="cuda")


def device_error():
    code = C.c_int(-1)
    native.check(native.lib().tf_op_device_error(None, C.byref(code)))
    return code.value


def random_parents(t, rng):
    return [-1] + [int(rng.integers(0, i)) for i in range(1, t)]


def tree_mask(parents, t_max):
    p = np.ascontiguousarray(parents, np.int32)
    w = (t_max + 63) // 64
    m = np.zeros((t_max, w), np.uint64)
    depth = np.zeros(t_max, np.int32)
    native.check(native.lib().tf_tree_mask(p.ctypes.data_as(native.i32p), len(p), t_max, m.ctypes.data_as(native.u64p),
                                           depth.ctypes.data_as(native.i32p)))
    return m, depth


def mask_bits(m, t_max):
    return (((m[:, np.arange(t_max) // 64] >> (np.arange(t_max, dtype=np.uint64) % np.uint64(64))) & np.uint64(1)) != 0)


class Case:
    """One attention problem with its cache; rows that nobody may read hold NaN."""

    def __init__(self, lens, nodes, T, H, HK, hd, kv, seed, cap=None, extra_slots=1, fused=True):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.nodes, self.T, self.H, self.HK, self.hd, self.kv = lens, nodes, T, H, HK, hd, kv
        self.B = B = len(lens)
        self.cap = cap or max(n + m for n, m in zip(lens, nodes)) + 3
        self.n_slots = B + extra_slots
        self.slots = rng.permutation(self.n_slots)[:B].tolist()
        self.k = torch.full((self.n_slots, HK, self.cap, hd), float("nan"), device="cuda", dtype=KV[kv])
        self.v = self.k.clone()
        for b in range(B):
            n = lens[b] + nodes[b]
            for c in (self.k, self.v):
                c[self.slots[b], :, :n] = torch.randn((HK, n, hd), generator=g, device="cuda").to(KV[kv])
        self.ld_q = (H + 2 * HK) * hd if fused else H * hd
        self.q = torch.randn((B, T, self.ld_q), generator=g, device="cuda")
        self.trees = [random_parents(max(1, m), rng)[:m] for m in nodes]
        masks = [tree_mask(p, T)[0] for p in self.trees]
        self.bits = [mask_bits(m, T) for m in masks]
        self.set_mask(np.stack(masks))
        self.ld_out = H * hd + 4
        self.out = torch.full((B, T, self.ld_out), 7.0, device="cuda")

    def set_mask(self, m):
        self.mask = torch.from_numpy(np.ascontiguousarray(m).view(np.int64)).cuda()

    def call(self, stream=None, ws=None, **kw):
        L = native.lib()
        a = dict(mask=self.mask, slots=i32(self.slots), n_ctx=i32(self.lens), n_node=i32(self.nodes))
        a.update(kw)
        if ws is None:
            ws = workspace(L.tf_op_attn_tree_workspace, self.B, self.T, self.H, self.HK, self.hd)
        self.keep = (a, ws)
        native.check(L.tf_op_attn_tree(ptr(self.out), self.ld_out, ptr(self.q), self.ld_q, ptr(self.k), ptr(self.v), self.kv,
                                       self.k.stride(0), self.cap, self.n_slots, ptr(a["slots"]), ptr(a["n_ctx"]),
                                       ptr(a["n_node"]), ptr(a["mask"]), self.B, self.T, self.H, self.HK, self.hd, ptr(ws),
                                       ws.numel(), stream))
        torch.cuda.synchronize()
        assert (self.out[..., self.H * self.hd:] == 7.0).all()  # nothing outside the rows is written
        return self.out[..., :self.H * self.hd].reshape(self.B, self.T, self.H, self.hd).double()

    def want(self, b):
        """[T][H][hd] in 64 bits, and the error bound of the module's docstring [T][H][1]."""
        H, HK, hd, n, m = self.H, self.HK, self.hd, self.lens[b], self.nodes[b]
        out = torch.zeros((self.T, H, hd), dtype=torch.float64, device="cuda")
        tol = torch.zeros((self.T, H, 1), dtype=torch.float64, device="cuda")
        vis = torch.cat([torch.ones((m, n), dtype=torch.bool), torch.from_numpy(self.bits[b][:m, :m])], 1).cuda()
        for h in range(H):
            k = self.k[self.slots[b], h // (H // HK), :n + m].double()
            v = self.v[self.slots[b], h // (H // HK), :n + m].double()
            q = self.q[b, :m, h * hd:(h + 1) * hd].double()
            s = (q @ k.T) / hd ** 0.5
            for t in range(m):
                e = vis[t]
                if not e.any():
                    continue
                p = torch.softmax(s[t, e], 0)
                out[t, h] = p @ v[e]
                d = hd * 2.0 ** -23 * (q[t].abs() @ k[e].abs().T).max() / hd ** 0.5
                tol[t, h] = (2 * d + 2.0 ** -18) * v[e].abs().max()
        return out, tol

    def check(self, got, rows=None):
        for b in (rows if rows is not None else range(self.B)):
            want, tol = self.want(b)
            err = (got[b] - want).abs()
            assert (err <= tol).all(), (b, float((err - tol).max()))
            norm = want.norm()
            assert (got[b] - want).norm() <= 5e-6 * norm, (b, float((got[b] - want).norm() / norm))


TYPES = list(KV)


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("heads", [(32, 8, 64), (14, 2, 64), (12, 2, 128), (8, 8, 128), (8, 1, 64)])
@pytest.mark.parametrize("T,ctx", [(1, 1), (1, 96), (3, 63), (5, 1000), (16, 129), (21, 514)])
def test_attention_shapes(heads, T, ctx, kv):
    c = Case([ctx], [T], T, *heads, kv, seed=ctx + T)
    c.check(c.call())
    assert device_error() == 0


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd", [8, 24, 32, 80, 96, 104])
def test_attention_head_sizes(hd, kv):
    c = Case([70, 3], [9, 4], 9, 6, 2, hd, kv, seed=hd)
    c.check(c.call())


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("T,ctx", [(64, 0), (64, 777), (65, 128), (130, 64), (256, 300)])
def test_attention_wide_trees(T, ctx, kv):
    c = Case([ctx, ctx + 31], [T, T - 1], T, 8, 2, 64, kv, seed=T)
    c.check(c.call())


@pytest.mark.parametrize("kv", TYPES)
def test_attention_wide_trees_of_wide_heads(kv):
    c = Case([200, 1025], [64, 40], 64, 12, 2, 128, kv, seed=3)
    c.check(c.call())


@pytest.mark.parametrize("kv", TYPES)
def test_attention_ragged_batch(kv):
    """Lengths of zero and one, a sequence without nodes, tile edges, one long sequence among short ones."""
    lens = [0, 1, 0, 63, 64, 65, 127, 128, 129, 2500, 5, 31]
    nodes = [1, 1, 6, 0, 6, 5, 4, 6, 2, 6, 3, 1]
    c = Case(lens, nodes, 6, 14, 2, 64, kv, seed=11)
    got = c.call()
    c.check(got, [b for b in range(len(lens)) if nodes[b]])
    for b in range(len(lens)):
        assert (got[b, nodes[b]:] == 0).all()
    assert device_error() == 0


@pytest.mark.parametrize("kv", TYPES)
def test_attention_long_context(kv):
    c = Case([16300], [3], 3, 8, 2, 64, kv, seed=5)
    c.check(c.call())


def test_attention_free_masks_and_empty_rows():
    """Any subset may be visible: rows without a bit see the context alone, or nothing at all."""
    for lens in ([0, 0], [40, 0]):
        c = Case(lens, [12, 12], 12, 8, 2, 64, native.TF_KV_F32, seed=8)
        rng = np.random.default_rng(1)
        m = rng.integers(0, 1 << 12, (2, 12, 1)).astype(np.uint64)
        m[:, 3] = 0
        m[1, 7] = 0
        m[:, 5] |= np.uint64(0xFFFFFFFF00000000)  # bits behind the last node mean nothing
        c.set_mask(m)
        c.bits = [mask_bits(m[b], 12) for b in range(2)]
        got = c.call()
        c.check(got)
        for b in range(2):
            if lens[b] == 0:
                assert (got[b, 3] == 0).all()


def test_attention_chain_default_equals_chain_mask():
    c = Case([37, 900], [7, 5], 7, 8, 2, 64, native.TF_KV_F32, seed=4)
    m = np.stack([tree_mask(list(range(-1, 6)), 7)[0]] * 2)
    c.set_mask(m)
    c.bits = [mask_bits(m[0], 7)] * 2
    a = c.call()
    b = c.call(mask=None)
    assert torch.equal(a, b)
    c.check(a)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("T", [10, 64])
@pytest.mark.parametrize("kv", TYPES)
def test_attention_unseen_rows_do_not_reach_the_output(kv, T, bad):
    """Non-finite keys and values of a drafted node reach its descendants and itself alone."""
    c = Case([70], [T], T, 8, 2, 64, kv, seed=9)
    clean = c.call().clone()
    j = 4
    c.k[c.slots[0], :, 70 + j] = bad
    c.v[c.slots[0], :, 70 + j] = bad
    got = c.call()
    sees = c.bits[0][:, j]
    assert sees.any() and not sees.all()
    assert torch.equal(got[0, ~sees], clean[0, ~sees])
    if bad != bad:
        assert got[0, sees].isnan().all()
    c.k[c.slots[0], :, 70 + j] = 0.5  # a value alone: its weight is positive, so it dominates
    got = c.call()
    assert torch.equal(got[0, ~sees], clean[0, ~sees])
    assert not got[0, sees].isfinite().any()


def test_attention_extreme_values():
    """Scores far apart and values beyond the range of 16-bit floats, in a 32-bit cache."""
    c = Case([300, 17], [6, 6], 6, 8, 2, 64, native.TF_KV_F32, seed=2)
    c.q *= 30
    c.k[:, :, 5] *= 1e4
    c.v[:, :, 6:60] *= 1e6
    c.v[:, :, 100:] *= 1e-6
    got = c.call()
    for b in range(2):
        want, tol = c.want(b)
        assert ((got[b] - want).abs() <= tol).all()
    c = Case([300], [6], 6, 8, 2, 64, native.TF_KV_BF16, seed=2)
    c.k *= 1e-9
    c.v[:, :, :200] *= 1e20
    got = c.call()
    want, tol = c.want(0)
    assert ((got[0] - want).abs() <= tol).all()


def test_attention_equal_scores_and_tiny_values():
    c = Case([515], [4], 4, 8, 2, 64, native.TF_KV_F32, seed=6)
    c.q.zero_()
    c.v *= 1e-30
    c.check(c.call())


@pytest.mark.parametrize("T", [4, 64])
def test_attention_batch_does_not_change_a_row_beyond_rounding(T):
    """The split over CTAs depends on the batch; the values follow it only by rounding, and the
    same call twice gives the same bits."""
    lens = [900, 33, 2000]
    c = Case(lens, [T] * 3, T, 8, 2, 64, native.TF_KV_F32, seed=13)
    a = c.call().clone()
    assert torch.equal(a, c.call())
    c.check(a)


def test_attention_own_stream_and_graph():
    c = Case([777, 20], [6, 6], 6, 8, 2, 64, native.TF_KV_F32, seed=14)
    a = c.call().clone()
    L = native.lib()
    ws = workspace(L.tf_op_attn_tree_workspace, c.B, c.T, c.H, c.HK, c.hd)
    st = torch.cuda.Stream()
    assert torch.equal(a, c.call(stream=st.cuda_stream, ws=ws))
    # captured once, replayed at other lengths: the lengths are read on the device
    n_ctx, n_node, slots = i32(c.lens), i32(c.nodes), i32(c.slots)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        native.check(L.tf_op_attn_tree(ptr(c.out), c.ld_out, ptr(c.q), c.ld_q, ptr(c.k), ptr(c.v), c.kv, c.k.stride(0),
                                       c.cap, c.n_slots, ptr(slots), ptr(n_ctx), ptr(n_node), ptr(c.mask), c.B, c.T, c.H,
                                       c.HK, c.hd, ptr(ws), ws.numel(), torch.cuda.current_stream().cuda_stream))
    for lens in ([777, 20], [300, 20], [1, 0]):
        c.lens = lens
        n_ctx.copy_(i32(lens))
        g.replay()
        torch.cuda.synchronize()
        c.check(c.out[..., :c.H * c.hd].reshape(c.B, c.T, c.H, c.hd).double())


def test_attention_offsets_beyond_32_bits():
    """A slot whose elements start beyond 2^31, in caches of more than 2^32 bytes each."""
    H, HK, hd, cap, n_slots = 8, 2, 128, 65536, 134
    k = torch.empty((n_slots, HK, cap, hd), device="cuda", dtype=torch.float16)
    v = torch.empty_like(k)
    assert k.stride(0) * (n_slots - 1) > 2 ** 31
    c = Case([300], [5], 5, H, HK, hd, native.TF_KV_F16, seed=7)
    for big, small in ((k, c.k), (v, c.v)):
        big[n_slots - 1, :, :305] = small[c.slots[0], :, :305]
    c.k, c.v, c.cap, c.n_slots, c.slots = k, v, cap, n_slots, [n_slots - 1]
    c.check(c.call())


def test_attention_device_checks():
    """A slot, a length or a count outside the cache: zeros and an error word; the others are served."""
    c = Case([50, 60, 70], [4, 4, 4], 4, 8, 2, 64, native.TF_KV_F32, seed=1)
    for kw in (dict(slots=[99] + c.slots[1:]), dict(slots=[-1] + c.slots[1:]), dict(n_ctx=[-1, 60, 70]),
               dict(n_ctx=[c.cap - 3, 60, 70])):
        got = c.call(**{k: i32(v) for k, v in kw.items()})
        assert (got[0] == 0).all()
        c.check(got, [1, 2])
        assert device_error() == 4  # TF_DEV_ERR_POS
    assert device_error() == 0


def test_attention_refusals():
    c = Case([10], [3], 3, 8, 2, 64, native.TF_KV_F32, seed=1)
    L = native.lib()
    ws = workspace(L.tf_op_attn_tree_workspace, 1, 3, 8, 2, 64)
    n_ctx = i32([10])
    good = dict(out=ptr(c.out), ld_out=c.ld_out, q=ptr(c.q), ld_q=c.ld_q, k=ptr(c.k), v=ptr(c.v), kv=c.kv,
                stride=c.k.stride(0), cap=c.cap, n_slots=c.n_slots, slots=None, n_ctx=ptr(n_ctx), n_node=None,
                mask=ptr(c.mask), B=1, T=3, H=8, HK=2, hd=64, ws=ptr(ws), n=ws.numel(), st=None)
    for bad, text in ((dict(T=0), "T must"), (dict(T=257), "T must"), (dict(B=-1), "B must"), (dict(H=7), "multiple"),
                      (dict(HK=0), "multiple"), (dict(hd=12), "head_dim"), (dict(hd=136), "head_dim"),
                      (dict(H=18, HK=2), "8 query heads"), (dict(out=None), "null"), (dict(n_ctx=None), "null"),
                      (dict(ws=None), "null"), (dict(kv=3), "kv_type"), (dict(ld_q=511), "ld_"), (dict(ld_out=513), "ld_"),
                      (dict(cap=0), "cache shape"), (dict(stride=8), "cache shape"), (dict(q=ptr(c.q) + 4), "aligned"),
                      (dict(k=ptr(c.k) + 8), "aligned"), (dict(ws=ptr(ws) + 16), "aligned"), (dict(n=0), "workspace")):
        with pytest.raises(native.TFError, match=text):
            native.check(L.tf_op_attn_tree(*{**good, **bad}.values()))
    native.check(L.tf_op_attn_tree(*{**good, "B": 0}.values()))
    native.check(L.tf_op_attn_tree(*good.values()))
    torch.cuda.synchronize()


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("heads,T", [((12, 2, 128), 8), ((14, 2, 64), 9), ((6, 1, 80), 6), ((32, 8, 64), 16)])
@pytest.mark.parametrize("cap", [80, 16384])
def test_attention_kernel_choice_by_capacity(cap, heads, T, kv):
    """33 to 64 rows per kv head: a small and a large cache are read by different kernels, from the
    same workspace, whatever it holds."""
    c = Case([60, 0, 33], [T, T - 1, 1], T, *heads, kv, seed=cap + T, cap=cap)
    ws = workspace(native.lib().tf_op_attn_tree_workspace, 3, T, *heads).fill_(255)
    c.check(c.call(ws=ws))
    assert device_error() == 0


def test_attention_refuses_too_many_tiles():
    """Tiles are counted in 32 bits: 65535 x 8 units of 2^30 positions are not."""
    c = Case([10], [3], 3, 8, 2, 64, native.TF_KV_F32, seed=1)
    ws = workspace(native.lib().tf_op_attn_tree_workspace, 1, 3, 8, 2, 64)
    with pytest.raises(native.TFError, match=r"2\^31"):
        native.check(native.lib().tf_op_attn_tree(
            ptr(c.out), c.ld_out, ptr(c.q), c.ld_q, ptr(c.k), ptr(c.v), c.kv, 8 * 64 << 30, 1 << 30, 1, None, ptr(i32([10])),
            None, None, 65535, 3, 8, 8, 64, ptr(ws), ws.numel(), None))


# ---- verification ---------------------------------------------------------------------------------

def weights(l, inv):
    l = l.astype(np.float32)
    l = np.where(np.isnan(l), -np.inf, l)
    m = l.max()
    with np.errstate(invalid="ignore"):
        x = (l - m) * np.float32(inv)
    return np.where(l == m, 1.0, np.exp(np.where(l == m, 0, x).astype(np.float64)))


def walk(logits, draft, tokens, parents, n, u, temperature):
    """The walk of one sequence, in 64 bits and from the definition (normalised residuals)."""
    if n == 0:
        return [], -1
    inv = 0.0 if temperature <= 0 else 1.0 / float(np.float32(temperature))
    cur, path = 0, [0]
    while True:
        if inv == 0.0:
            r = np.zeros(logits.shape[1])
            r[int(np.argmax(logits[cur]))] = 1.0
        else:
            p = weights(logits[cur], inv)
            p /= p.sum()
            r = p.copy()
            if draft is not None:
                q = weights(draft[cur], inv)
                q /= q.sum()
        for t in range(cur + 1, n):
            if parents[t] != cur:
                continue
            x = tokens[t]
            if inv == 0.0:
                ok = r[x] > 0
            elif draft is not None:
                ok = float(u[t]) * q[x] < r[x]
            else:
                ok = float(u[t]) < r[x]
            if ok:
                path.append(t)
                cur = t
                break
            if inv > 0.0:
                if draft is not None:
                    r = np.maximum(r - q, 0.0)
                else:
                    r[x] = 0.0
                r = r / r.sum() if r.sum() > 1e-12 else p.copy()
        else:
            if inv == 0.0:
                return path, int(np.argmax(logits[cur]))
            c = np.cumsum(r)
            return path, int(np.argmax(c > float(u[0]) * c[-1]))


def verify(logits, draft, tokens, parents, n_node, u, temperature, ld=None, stream=None):
    B, T, V = logits.shape
    L = native.lib()
    ld = ld or V

    def rows(x):
        if x is None:
            return None
        t = torch.full((B, T, ld), float("nan"), device="cuda")
        t[..., :V] = torch.from_numpy(x)
        return t
    lt, dt = rows(logits), rows(draft)
    path, n_path, nxt = i32([[9] * T] * B), i32([9] * B), i32([9] * B)
    ut = torch.from_numpy(np.ascontiguousarray(u, np.float32)).cuda()
    tk, pr, nn = i32(tokens.tolist()), i32(parents.tolist()), i32(list(n_node))
    ws = workspace(L.tf_op_verify_tree_workspace, B, T, V)
    torch.cuda.synchronize()
    for _ in range(2):  # a workspace serves call after call
        native.check(L.tf_op_verify_tree(ptr(path), ptr(n_path), ptr(nxt), ptr(lt), ld, ptr(dt), ld, ptr(tk), ptr(pr), ptr(nn),
                                         ptr(ut), temperature, B, T, V, ptr(ws), ws.numel(), stream))
    torch.cuda.synchronize()
    return path.cpu().numpy(), n_path.cpu().numpy(), nxt.cpu().numpy()


def problem(B, T, V, seed, chain=False, spread=2.0, noise=0.7, with_draft=True, temperature=1.0):
    rng = np.random.default_rng(seed)
    logits = (rng.standard_normal((B, T, V)) * spread).astype(np.float32)
    parents = np.stack([np.arange(-1, T - 1) if chain else np.array(random_parents(T, rng)) for _ in range(B)]).astype(np.int32)
    draft = (logits + rng.standard_normal((B, T, V)) * noise).astype(np.float32) if with_draft else None
    src = draft if with_draft else logits
    tokens = np.zeros((B, T), np.int32)
    for b in range(B):
        for t in range(1, T):
            w = weights(src[b, parents[b, t]], 1.0 / max(temperature, 0.3))
            tokens[b, t] = rng.choice(V, p=w / w.sum())
    u = rng.random((B, T)).astype(np.float32)
    return logits, draft, tokens, parents, u


def check_verify(prob, n_node, temperature, **kw):
    logits, draft, tokens, parents, u = prob
    path, n_path, nxt = verify(logits, draft, tokens, parents, n_node, u, temperature, **kw)
    for b in range(len(logits)):
        want, tok = walk(logits[b], None if draft is None else draft[b], tokens[b], parents[b], n_node[b], u[b], temperature)
        assert path[b].tolist() == want + [-1] * (logits.shape[1] - len(want)), b
        assert n_path[b] == len(want) and nxt[b] == tok, b
    return n_path


@pytest.mark.parametrize("mode", ["draft", "nodist", "greedy"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4099, 32768, 50257])
@pytest.mark.parametrize("T,chain", [(1, True), (6, True), (17, False)])
def test_verify_walk(T, chain, V, mode):
    temp = 0.0 if mode == "greedy" else 0.75
    B = 9 if V < 5000 else 4
    prob = problem(B, T, V, seed=V + T, chain=chain, with_draft=mode != "nodist", temperature=temp)
    check_verify(prob, [T] * B, temp)
    assert device_error() == 0


@pytest.mark.parametrize("V", [128256, 151936])
@pytest.mark.parametrize("mode", ["draft", "nodist", "greedy"])
def test_verify_model_vocabularies(V, mode):
    temp = 0.0 if mode == "greedy" else 1.0
    prob = problem(3, 7, V, seed=V, spread=3.0, with_draft=mode != "nodist", temperature=temp)
    check_verify(prob, [7, 3, 1], temp)


@pytest.mark.parametrize("mode", ["draft", "nodist"])
def test_verify_many_rejections(mode):
    """Wide trees of one level whose children are mostly refused: residual after residual."""
    rng = np.random.default_rng(0)
    B, T, V = 24, 200, 97
    logits, draft, tokens, parents, u = problem(B, T, V, seed=5, noise=3.0, with_draft=mode == "draft")
    parents[:, 1:] = 0
    for b in range(B):
        w = weights((draft if draft is not None else logits)[b, 0], 1.0)
        tokens[b, 1:] = rng.choice(V, T - 1, p=w / w.sum())
    u[:, 1:] = 1 - 1e-3 * rng.random((B, T - 1))
    n = check_verify((logits, draft, tokens, parents, u.astype(np.float32)), rng.integers(0, T + 1, B).tolist(), 1.0)
    assert (n <= 2).all()


def test_verify_ragged_and_strided():
    B, T, V = 7, 12, 777
    prob = problem(B, T, V, seed=21)
    check_verify(prob, [0, 1, 2, 12, 7, 0, 11], 0.6, ld=V + 5)
    check_verify(prob, [0, 1, 2, 12, 7, 0, 11], 0.0, ld=V + 5)


def test_verify_on_another_stream():
    st = torch.cuda.Stream()
    check_verify(problem(3, 9, 2000, seed=3), [9] * 3, 0.8, stream=st.cuda_stream)


def test_verify_equal_distributions_accept_everything():
    """p = q bit for bit: every drafted token stays, whatever the random numbers."""
    logits, _, tokens, parents, u = problem(5, 8, 3001, seed=2, chain=True)
    u[:] = np.float32(1 - 2 ** -24)
    path, n_path, _ = verify(logits, logits, tokens, parents, [8] * 5, u, 1.0)
    assert (n_path == 8).all() and (path == np.arange(8)).all()


def test_verify_masked_logits():
    """Tokens of logit -inf (and NaN) have no weight; one finite logit takes all; a row of -inf alone
    is uniform; +inf takes all."""
    V, T, B = 40, 3, 5
    logits, draft, tokens, parents, u = problem(B, T, V, seed=6, chain=True)
    logits[:, :, 1::2] = -np.inf
    logits[0, 0, 2] = np.nan
    logits[1, 0] = -np.inf
    logits[1, 0, 17] = -3.0
    logits[2, 0] = -np.inf
    logits[3, 0, 8] = np.inf
    draft[4] = -np.inf
    draft[4, :, 6] = 1.0
    tokens[1, 1], tokens[3, 1], tokens[4, 1] = 17, 8, 6
    for ui in (0.0, 0.3, 1 - 2 ** -24):
        u[:, 0] = ui
        check_verify((logits, draft, tokens, parents, u), [T] * B, 1.0)
        check_verify((logits, None, tokens, parents, u), [T] * B, 1.0)
    _, n_path, nxt = verify(logits, draft, tokens, parents, [1] * B, u, 1.0)
    assert nxt[1] == 17 and nxt[3] == 8 and all(nxt[b] % 2 == 0 for b in (0, 4))


def test_verify_greedy_ties_and_duplicates():
    V, T = 300, 5
    logits = np.zeros((1, T, V), np.float32)
    logits[0, 0, [7, 250]] = 2.0
    logits[0, 1, 3] = logits[0, 1, 299] = 1.0
    parents = np.array([[-1, 0, 0, 1, 1]], np.int32)
    tokens = np.array([[0, 7, 7, 299, 3]], np.int32)
    path, n_path, nxt = verify(logits, None, tokens, parents, [T], np.zeros((1, T)), 0.0)
    assert path[0].tolist() == [0, 1, 4, -1, -1] and n_path[0] == 3 and nxt[0] == 0


@pytest.mark.parametrize("mode", ["draft", "nodist"])
def test_verify_follows_the_target_distribution(mode):
    """The first token after the root follows p, whatever was drafted: frequencies of 40000 walks
    within 5 standard deviations, for a draft far from the target."""
    B, T, V, rounds = 4000, 4, 11, 10
    rng = np.random.default_rng(77)
    lp, lq = rng.standard_normal(V).astype(np.float32), (2 * rng.standard_normal(V)).astype(np.float32)
    p, q = weights(lp, 1.0), weights(lq, 1.0)
    p, q = p / p.sum(), q / q.sum()
    logits = np.broadcast_to(lp, (B, T, V)).copy()
    draft = np.broadcast_to(lq, (B, T, V)).copy() if mode == "draft" else None
    parents = np.broadcast_to(np.array([-1, 0, 0, 0], np.int32), (B, T)).copy()
    seen = np.zeros(V)
    for _ in range(rounds):
        tokens = rng.choice(V, (B, T), p=q).astype(np.int32)
        u = rng.random((B, T)).astype(np.float32)
        path, n_path, nxt = verify(logits, draft, tokens, parents, [T] * B, u, 1.0)
        first = np.where(n_path > 1, tokens[np.arange(B), path[:, 1]], nxt)
        seen += np.bincount(first, minlength=V)
    n = B * rounds
    assert (np.abs(seen - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all(), (seen / n, p)


def test_verify_device_checks():
    """A drafted token outside the vocabulary is refused and recorded, a parent that does not precede
    its node is nobody's child."""
    logits, draft, tokens, parents, u = problem(2, 5, 64, seed=4, chain=True)
    u[:, 1:] = 0.0
    tokens[0, 2] = 64
    tokens[1, 3] = -5
    path, n_path, _ = verify(logits, draft, tokens, parents, [5, 5], u, 1.0)
    assert n_path.tolist() == [2, 3] and device_error() == 3
    logits, draft, tokens, parents, u = problem(1, 4, 64, seed=4, chain=True)
    u[:, 1:] = 0.0
    parents[0] = [-1, 0, 2, 99]
    path, n_path, _ = verify(logits, draft, tokens, parents, [4], u, 1.0)
    assert path[0].tolist() == [0, 1, -1, -1]


def test_verify_refusals():
    L = native.lib()
    t = torch.zeros(4096, device="cuda")
    good = dict(path=ptr(t), n_path=ptr(t), nxt=ptr(t), logits=ptr(t), ld=8, draft=None, ldd=8, tokens=ptr(t), parents=ptr(t),
                n_node=None, u=ptr(t), temp=1.0, B=1, T=2, V=8, ws=ptr(t), n=1 << 30, st=None)
    for bad, text in ((dict(T=0), "T must"), (dict(T=300), "T must"), (dict(B=-1), "B must"), (dict(V=0), "V must"),
                      (dict(path=None), "null"), (dict(logits=None), "null"), (dict(u=None), "u must"),
                      (dict(temp=float("nan")), "NaN"), (dict(temp=1e-45), "range"), (dict(temp=float("inf")), "range"),
                      (dict(ld=7), "ld must"), (dict(draft=ptr(t), ldd=7), "ld must"), (dict(ws=None), "null"),
                      (dict(ws=ptr(t) + 4), "aligned"), (dict(n=1), "workspace")):
        with pytest.raises(native.TFError, match=text):
            native.check(L.tf_op_verify_tree(*{**good, **bad}.values()))
    native.check(L.tf_op_verify_tree(*{**good, "B": 0}.values()))


@pytest.mark.parametrize("V,with_draft,text", [(409601, True, "409600"), (819201, False, "819200")])
def test_verify_refuses_a_vocabulary_that_does_not_fit(V, with_draft, text):
    t = torch.zeros(4096, device="cuda")
    with pytest.raises(native.TFError, match=text):
        native.check(native.lib().tf_op_verify_tree(ptr(t), ptr(t), ptr(t), ptr(t), V, ptr(t) if with_draft else None, V, ptr(t),
                                                    ptr(t), None, ptr(t), 1.0, 1, 2, V, ptr(t), 1 << 30, None))


@pytest.mark.parametrize("V,with_draft", [(409600, True), (819200, False)])
def test_verify_largest_vocabulary(V, with_draft):
    logits, draft, tokens, parents, u = problem(1, 3, V, seed=6, with_draft=with_draft, chain=True)
    check_verify((logits, draft, tokens, parents, u), [3], 0.9)


# ---- commit ---------------------------------------------------------------------------------------

def commit(k, v, kv, slots, n_ctx, path, n_path, n_new, stream=None):
    L = native.lib()
    n_layer, n_slots, HK, cap, hd = k.shape
    native.check(L.tf_op_kv_commit(ptr(k), ptr(v), kv, n_layer, k.stride(0), k.stride(1), cap, n_slots, ptr(slots), ptr(n_ctx),
                                   ptr(path), path.shape[1], ptr(n_path), ptr(n_new), len(n_path), HK, hd, stream))
    torch.cuda.synchronize()


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("hd", [8, 64, 80, 128])
@pytest.mark.parametrize("T", [1, 6, 70, 256])
def test_commit(T, hd, kv):
    rng = np.random.default_rng(T + hd)
    n_layer, n_slots, HK, cap, B = 3, 7, 2, 300, 5
    k = torch.randn((n_layer, n_slots, HK, cap, hd), device="cuda").to(KV[kv])
    v = torch.randn((n_layer, n_slots, HK, cap, hd), device="cuda").to(KV[kv])
    slots = rng.permutation(n_slots)[:B].tolist()
    n_ctx = [0, cap - T, 11, 3, 29]
    n_path = [0, T, 1, min(T, 4), max(1, T // 2)]
    path = np.full((B, T), -1)
    for b in range(B):
        path[b, :n_path[b]] = np.sort(rng.permutation(T)[:n_path[b]])
    path[2, 0] = 0
    want = [k.clone(), v.clone()]
    for w in want:
        for b in range(B):
            idx = torch.from_numpy(path[b, :n_path[b]]).cuda() + n_ctx[b]
            w[:, slots[b], :, n_ctx[b]:n_ctx[b] + n_path[b]] = w[:, slots[b], :, idx].clone()
    n_new = i32([-7] * B)
    commit(k, v, kv, i32(slots), i32(n_ctx), i32(path.tolist()), i32(n_path), n_new)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert n_new.tolist() == [a + b for a, b in zip(n_ctx, n_path)]
    assert device_error() == 0


def test_commit_refuses_wrong_paths():
    k = torch.randn((2, 3, 2, 40, 64), device="cuda")
    v, k0 = k + 1, k.clone()
    bad = [[0, 2, 2], [1, 0, 2], [0, 3, 40], [-1, 1, 2]]
    for p in bad:
        n_new = i32([0])
        commit(k, v, native.TF_KV_F32, i32([1]), i32([10]), i32([p]), i32([3]), n_new)
        assert torch.equal(k, k0) and torch.equal(v, k0 + 1)
        assert n_new.tolist() == [10] and device_error() == 4
    commit(k, v, native.TF_KV_F32, i32([3]), i32([10]), i32([[0, 1, 2]]), i32([3]), None)
    assert device_error() == 4
    L = native.lib()
    a = i32([0])
    good = dict(k=ptr(k), v=ptr(v), kv=0, nl=2, ls=k.stride(0), ss=k.stride(1), cap=40, ns=3, slots=None, n_ctx=ptr(a),
                path=ptr(a), ld=1, n_path=ptr(a), n_new=None, B=1, HK=2, hd=64, st=None)
    for b, text in ((dict(k=None), "null"), (dict(path=None), "null"), (dict(kv=7), "kv_type"), (dict(nl=0), "shape"),
                    (dict(hd=4), "head_dim"), (dict(ss=64), "strides"), (dict(ls=64), "strides"), (dict(B=-1), "B must"),
                    (dict(k=ptr(k) + 8), "aligned"), (dict(n_new=ptr(a)), "n_new")):
        with pytest.raises(native.TFError, match=text):
            native.check(L.tf_op_kv_commit(*{**good, **b}.values()))
