"""tf_op_kv_commit's refusals without a GPU: they come before any device work."""
import pytest

from tinferno_b200 import native

AT = 1 << 20  # addresses that are compared only


def call(B=3, ld_path=4, **kw):
    a = dict(k=AT, v=2 * AT, kv=native.TF_KV_F32, layers=1, layer_stride=8 * 8, slot_stride=8 * 8, cap=8, n_slots=1, slots=3 * AT,
             n_ctx=4 * AT, path=5 * AT, ld_path=ld_path, n_path=6 * AT, n_new=7 * AT, B=B, n_kv=1, hd=8, stream=None)
    a.update(kw)
    native.check(native.lib().tf_op_kv_commit(*a.values()))


@pytest.mark.parametrize("array,first,last", [("n_ctx", -2, 2), ("n_path", -2, 2), ("slots", -2, 2), ("path", -2, 11)])
def test_n_new_has_memory_of_its_own(array, first, last):
    """Every block of the launch reads the lengths, slots and paths while one writes n_new."""
    at = dict(n_ctx=4, n_path=6, slots=3, path=5)[array] * AT
    for off in (first, 0, 1, last):
        with pytest.raises(native.TFError, match="n_new"):
            call(n_new=at + 4 * off)
