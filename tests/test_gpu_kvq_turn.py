"""tf_op_qk_norm_rope rounds the rotation's two products and their sum once, in queries and in keys."""
import numpy as np
import pytest

from test_gpu_kvq import cuda, i32, ptr
from tinferno_b200 import native

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def far_from_a_tie(a):
    """Where a 64-bit value rounds to the same fp32 value though it is off by 2^-40 of itself."""
    return (np.float32(a * (1 + 2.0 ** -40)) == np.float32(a)) & (np.float32(a * (1 - 2.0 ** -40)) == np.float32(a))


@pytest.mark.parametrize("rows,H", [(3, 2), (2000, 4)])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 64), (128, 128), (40, 24)])
def test_rounded_once(rows, H, hd, rot):
    """Against y c + m s in 64 bits, c and s being the fp32 cosine and sine: half a step of the result, 2^-24 of it, and
    what the carried errors' own roundings leave, 2^-46 of the products.  In half of the pairs the products cancel."""
    rng = np.random.default_rng(rows + rot)
    half = rot // 2
    freq = (500000.0 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)
    pos = rng.integers(0, 131072, rows)
    a = pos[:, None].astype(np.float64) * freq.astype(np.float64)
    c64, s64 = np.cos(a), np.sin(a)
    c, s = (v.astype(np.float32).astype(np.float64)[:, None] for v in (c64, s64))
    x = rng.standard_normal((rows, H, hd)).astype(np.float32)
    size = rng.standard_normal((rows, H, half))
    cancel = rng.random((rows, H, half)) < 0.5               # (a, b) = (s, c) t: a c - b s is what their roundings leave
    x[..., :half] = np.where(cancel, s * size, x[..., :half])
    x[..., half:rot] = np.where(cancel, c * size, x[..., half:rot])
    d, df, dp = cuda(x), cuda(freq), i32(pos.tolist())
    q, k = torch.zeros((rows, H, hd), device="cuda"), torch.zeros((rows, H, hd), device="cuda")
    native.check(native.lib().tf_op_qk_norm_rope(ptr(q), H * hd, ptr(k), H * hd, ptr(d), H * hd, ptr(d), H * hd, None, None, 0.0, ptr(df), rot, ptr(dp),
                                                 rows, H, H, hd, None))
    torch.cuda.synchronize()
    sure = np.broadcast_to((far_from_a_tie(c64) & far_from_a_tie(s64))[:, None], cancel.shape)
    assert sure.mean() > 0.99
    x0, x1 = x[..., :half].astype(np.float64), x[..., half:rot].astype(np.float64)
    for got in (k.cpu().numpy(), q.cpu().numpy()):
        for out, u, v in ((got[..., :half], x0 * c, -x1 * s), (got[..., half:rot], x0 * s, x1 * c)):
            want = u + v
            off = np.abs(out - want) - (2.0 ** -24 * np.abs(want) + 2.0 ** -46 * (np.abs(u) + np.abs(v)) + 2.0 ** -149)
            assert (off[sure] <= 0).all(), off[sure].max()
        np.testing.assert_array_equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("rows", [1, 3000])
def test_queries_and_keys_alike(rows):
    """The same rows with the same weights are the same bits as queries and as keys."""
    H, hd = 3, 64
    x, w = torch.randn((rows, H, hd), device="cuda") * 3, 1 + 0.3 * torch.randn(hd, device="cuda")
    freq = cuda((10000.0 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32))
    pos = torch.randint(0, 100000, (rows,), device="cuda", dtype=torch.int32)
    q, k = torch.zeros_like(x), torch.zeros_like(x)
    native.check(native.lib().tf_op_qk_norm_rope(ptr(q), H * hd, ptr(k), H * hd, ptr(x), H * hd, ptr(x), H * hd, ptr(w), ptr(w), 1e-6, ptr(freq), hd,
                                                 ptr(pos), rows, H, H, hd, None))
    torch.cuda.synchronize()
    assert torch.equal(q, k)
