"""What takes F32, F16 and BF16 caches refuses the quantised types, whose rows it would read as 16-bit ones."""
import ctypes as C

import pytest

from tinferno_b200 import native

AT = 1 << 20  # addresses that are compared only


@pytest.mark.parametrize("kv", [native.TF_KV_Q4_0, native.TF_KV_Q8_0, -1, 7])
def test_other_operators_and_the_engine(kv):
    L = native.lib()
    for decode in (L.tf_op_attn_decode, L.tf_op_attn_decode_noalloc):
        with pytest.raises(native.TFError, match="kv_type"):
            native.check(decode(AT, 2 * AT, 3 * AT, 4 * AT, kv, 64, 10, 4, 2, 64, None))
    with pytest.raises(native.TFError, match="kv_type"):
        native.check(L.tf_op_attn_tree(AT, 256, 2 * AT, 256, 3 * AT, 4 * AT, kv, 2 * 64 * 64, 64, 1, None, 5 * AT, None, None, 1, 1, 4, 2, 64,
                                       6 * AT, 1 << 30, None))
    with pytest.raises(native.TFError, match="kv_type"):
        native.check(L.tf_op_kv_commit(AT, 2 * AT, kv, 1, 8 * 64, 8 * 64, 8, 1, None, 3 * AT, 4 * AT, 4, 5 * AT, None, 1, 1, 64, None))
    desc = (native.TensorDesc * 1)()
    hp, opt, out = native.HParams(), native.Options(64, 1, 0, kv, 1, 0), C.c_void_p()
    with pytest.raises(native.TFError, match="kv_type"):
        native.check(L.tf_cuda_create(desc, 0, C.byref(hp), C.byref(opt), C.byref(out)))
