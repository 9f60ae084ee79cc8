"""Refusals of the quantised cache's operators without a GPU: they come before any device work."""
import ctypes as C

import pytest

from tinferno_b200 import native

AT = 1 << 20  # addresses that are compared only

CACHE = dict(kc=AT, vc=2 * AT, kv=native.TF_KV_Q4_0, stride=2 * 64 * 64, cap=64, n_slots=3)
WHERE = dict(slots=3 * AT, pos=4 * AT)


def call(name, base, kw):
    a = dict(base)
    assert set(kw) <= set(a)
    a.update(kw)
    native.check(getattr(native.lib(), name)(*a.values()))


def quant(**kw):
    call("tf_op_kv_quant", dict(CACHE, **WHERE, k=5 * AT, ld_k=128, v=6 * AT, ld_v=128, rows=4, n_kv=2, hd=64, stream=None), kw)


def dequant(**kw):
    call("tf_op_kv_dequant", dict(k=5 * AT, ld_k=128, v=6 * AT, ld_v=128, **CACHE, **WHERE, rows=4, n_kv=2, hd=64, stream=None), kw)


def store(**kw):
    call("tf_op_qkv_store", dict(q_out=7 * AT, ld_qo=256, **CACHE, **WHERE, q=8 * AT, ld_q=256, k=5 * AT, ld_k=128, v=6 * AT,
                                 ld_v=128, wq=9 * AT, wk=9 * AT, eps=1e-6, freq=10 * AT, rot=64, rows=4, H=4, n_kv=2, hd=64,
                                 stream=None), kw)


def rope(**kw):
    call("tf_op_qk_norm_rope", dict(q_out=7 * AT, ld_qo=256, k_out=5 * AT, ld_ko=128, q=8 * AT, ld_q=256, k=6 * AT, ld_k=128,
                                    wq=9 * AT, wk=9 * AT, eps=1e-6, freq=10 * AT, rot=64, pos=4 * AT, rows=4, H=4, n_kv=2, hd=64,
                                    stream=None), kw)


def attn(**kw):
    call("tf_op_attn_quant", dict(out=7 * AT, ld_out=256, q=8 * AT, ld_q=256, **CACHE, slots=3 * AT, n_ctx=4 * AT, n_new=11 * AT,
                                  B=2, T=3, H=4, n_kv=2, hd=64, ws=12 * AT, ws_bytes=1 << 30, stream=None), kw)


CACHES = [dict(kv=native.TF_KV_F16), dict(kv=5), dict(kv=-1), dict(kc=None), dict(vc=None), dict(kc=AT + 8), dict(vc=AT + 2),
          dict(cap=0), dict(cap=40), dict(cap=-16), dict(n_slots=0), dict(stride=2 * 64 * 64 - 1024), dict(stride=2 * 64 * 64 + 64),
          dict(n_kv=0), dict(hd=48), dict(hd=160), dict(hd=0), dict(hd=-64)]


@pytest.mark.parametrize("kw", CACHES + [dict(pos=None), dict(k=None), dict(v=None), dict(ld_k=127), dict(ld_v=130), dict(k=AT + 4),
                                         dict(rows=-1)], ids=str)
def test_quant(kw):
    with pytest.raises(native.TFError):
        quant(**kw)


@pytest.mark.parametrize("kw", CACHES + [dict(pos=None), dict(k=None, v=None), dict(ld_k=127), dict(v=AT + 8), dict(rows=-1)], ids=str)
def test_dequant(kw):
    with pytest.raises(native.TFError):
        dequant(**kw)


@pytest.mark.parametrize("kw", CACHES + [dict(pos=None), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(H=0), dict(rot=0),
                                         dict(rot=12), dict(rot=72), dict(eps=-1.0), dict(eps=float("nan")), dict(wq=AT + 4),
                                         dict(ld_qo=252), dict(ld_q=258), dict(rows=-1)], ids=str)
def test_store(kw):
    with pytest.raises(native.TFError):
        store(**kw)


@pytest.mark.parametrize("kw", [dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(q=None, q_out=None, k=None, k_out=None),
                                dict(hd=0), dict(hd=60), dict(hd=136), dict(H=0), dict(n_kv=0), dict(H=2000), dict(pos=None), dict(rot=4),
                                dict(rot=72), dict(rot=-8), dict(eps=-1e-9), dict(eps=float("nan")), dict(ld_q=255), dict(ld_ko=124),
                                dict(q_out=AT + 4), dict(wk=AT + 8), dict(rows=-1)], ids=str)
def test_norm_rope(kw):
    with pytest.raises(native.TFError):
        rope(**kw)


@pytest.mark.parametrize("kw", CACHES + [dict(out=None), dict(q=None), dict(n_ctx=None), dict(ws=None), dict(ws=12 * AT + 16), dict(ws_bytes=0),
                                         dict(B=-1), dict(B=65536), dict(T=0), dict(T=65), dict(H=0), dict(H=5), dict(H=2048),
                                         dict(ld_out=252), dict(ld_q=250), dict(out=AT + 4),
                                         dict(B=65535, cap=1 << 20, stride=2 * 64 << 20)], ids=str)
def test_attn(kw):
    with pytest.raises(native.TFError):
        attn(**kw)


@pytest.mark.parametrize("kw", [dict(B=1, T=65), dict(T=0), dict(B=-1), dict(hd=48), dict(H=3)], ids=str)
def test_workspace(kw):
    a = dict(B=1, T=1, H=4, n_kv=2, hd=64)
    a.update(kw)
    n = C.c_size_t(7)
    with pytest.raises(native.TFError):
        native.check(native.lib().tf_op_attn_quant_workspace(*a.values(), C.byref(n)))
    assert n.value == 0
    with pytest.raises(native.TFError):
        native.check(native.lib().tf_op_attn_quant_workspace(1, 1, 4, 2, 64, None))


def test_no_rows_is_no_work():
    """Nothing to do is no error, and needs no device."""
    quant(rows=0)
    dequant(rows=0)
    store(rows=0)
    rope(rows=0)
    attn(B=0)
