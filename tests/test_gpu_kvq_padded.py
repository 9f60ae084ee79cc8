"""Padded batches through tf_op_qkv_store and tf_op_attn_quant: a sequence without new rows is empty, whatever its
slot and length say."""
import numpy as np
import pytest

from test_gpu_kvq import Case, TYPES, cuda, device_error, i32, ptr
from tinferno_b200 import native

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def others_hold(c, got, sequences):
    for b in sequences:
        want, tol = c.want(b)
        assert (np.abs(got[b] - want) <= tol).all()
        assert np.linalg.norm(got[b] - want) <= 5e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("cap", [96, 8192])
@pytest.mark.parametrize("T", [1, 3])
def test_empty_sequences(kv, cap, T):
    c = Case(kv, 64, 8, 2, [40, 90, 33, 20, 0], [T] * 5, T, 1, cap=cap).run().check()
    for slots, ctx in (([-1, -1], [33, 20]), ([-7, 99], [-5, 10 ** 9]), ([0, 1], [cap, cap + 1]), ([-2 ** 31, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31])):
        kw = dict(slots=i32([c.slots[0], slots[0], c.slots[2], slots[1], c.slots[4]]), n_ctx=i32([40, ctx[0], 33, ctx[1], 0]), n_new=i32([T, 0, T, 0, T]))
        c.out.fill_(7.0)
        c.run(upload=False, **kw)
        got = c.got()
        assert device_error() == 0
        assert (got[[1, 3]] == 0).all()
        others_hold(c, got, (0, 2, 4))


@pytest.mark.parametrize("cap", [96, 8192])
def test_nothing_but_padding(cap):
    c = Case(native.TF_KV_Q4_0, 64, 4, 2, [40, 90], [2, 2], 2, 1, cap=cap).run()
    c.out.fill_(7.0)
    c.run(upload=False, slots=i32([-1, -1]), n_new=i32([0, 0]))
    assert (c.got() == 0).all() and device_error() == 0


@pytest.mark.parametrize("cap", [96, 8192])
def test_more_new_rows_than_the_call_holds(cap):
    """n_new above T is refused like a length that does not fit, not cut."""
    c = Case(native.TF_KV_Q8_0, 64, 8, 2, [40, 70, 33], [2, 2, 2], 2, 1, cap=cap).run()
    for n in (3, 2 ** 31 - 1):
        c.out.fill_(7.0)
        c.run(upload=False, n_new=i32([2, n, 2]))
        got = c.got()
        assert device_error() == native.TF_DEV_ERR_POS
        assert (got[1] == 0).all()
        others_hold(c, got, (0, 2))


@pytest.mark.parametrize("kv", TYPES)
@pytest.mark.parametrize("captured", [False, True])
def test_padded_step(kv, captured):
    """A step of a batch that is padded: store, then attention, with one slots array for both; the cache's other slots and
    the padded rows' places stay as they were, and nothing is reported."""
    H, HK, hd, cap, B = 4, 2, 64, 64, 5
    L = native.lib()
    rng = np.random.default_rng(8)
    c = Case(kv, hd, H, HK, [20, 7, 33, 0, 50], [1] * B, 1, 5, cap=cap)
    slots, n_new = [c.slots[0], -1, c.slots[2], c.slots[3], -1], [1, 0, 1, 1, 0]
    ctx = [20, 7, 33, 0, -1]
    c.c.upload()
    before = c.c.dk.clone(), c.c.dv.clone()
    x = cuda(rng.standard_normal((B, (H + 2 * HK) * hd)).astype(np.float32))
    freq = cuda((10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32))
    ds, dc, dn, ld = i32(slots), i32(ctx), i32(n_new), (H + 2 * HK) * hd
    q, out, ws = torch.full((B, H * hd), 7.0, device="cuda"), torch.full((B, H * hd), 7.0, device="cuda"), c.workspace()

    def step(stream):
        native.check(L.tf_op_qkv_store(ptr(q), H * hd, *c.c.args(), ptr(ds), ptr(dc), ptr(x), ld, ptr(x) + 4 * H * hd, ld,
                                       ptr(x) + 4 * (H + HK) * hd, ld, None, None, 0.0, ptr(freq), hd, B, H, HK, hd, stream))
        native.check(L.tf_op_attn_quant(ptr(out), H * hd, ptr(q), H * hd, *c.c.args(), ptr(ds), ptr(dc), ptr(dn), B, 1, H, HK, hd, ptr(ws),
                                        ws.numel(), stream))

    if captured:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        step(side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(side.cuda_stream)
        out.fill_(7.0)
        graph.replay()
    else:
        step(None)
    torch.cuda.synchronize()
    assert device_error() == 0
    assert (out[[1, 4]] == 0).all() and (q[[1, 4]] == 7.0).all()
    c.c.k, c.c.v = c.c.dk.cpu().numpy(), c.c.dv.cpu().numpy()
    for s in range(B + 1):
        if s not in slots:
            assert torch.equal(c.c.dk[s], before[0][s]) and torch.equal(c.c.dv[s], before[1][s])
    for b in (0, 2, 3):
        n = ctx[b] + 1
        k, v = c.c.values("k", slots[b], n), c.c.values("v", slots[b], n)
        s = np.einsum("grd,gnd->grn", q[b].double().cpu().numpy().reshape(HK, H // HK, hd), k) / hd ** 0.5
        p = np.exp(s - s.max(-1, keepdims=True))
        want = np.einsum("grn,gnd->grd", p / p.sum(-1, keepdims=True), v).reshape(-1)
        assert np.linalg.norm(out[b].double().cpu().numpy() - want) <= 5e-6 * np.linalg.norm(want)
