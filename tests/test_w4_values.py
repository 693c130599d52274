"""4-bit products of activations at the ends of their types' ranges.

Bounds as in test_w4: activations enter exactly, sums are fp32."""
import numpy as np
import pytest

from conftest import load_pkg
from test_w4 import BITS, dense, on_gpu, product_bound, silu, stream, torch_dtype, weights


def product(pkg, w, x, dt, group, gated=False, **kw):
    import torch
    N = w[0].shape[1] // 2 if gated else w[0].shape[1]
    y = torch.full((len(x), N), -7, dtype=torch_dtype(dt), device="cuda")
    with pkg.W4Matrix(*w, group=group, gated=gated) as m:
        m.matvec(x.data_ptr(), y.data_ptr(), len(x), dt, stream(), **kw)
    return y.double().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,K", [(1, 128), (8, 256), (3, 4096), (17, 192)])
@pytest.mark.parametrize("dt,size", [(0, 2.0 ** 122), (1, 2.0 ** 116), (1, 2.0 ** 122), (1, 2.0 ** -118), (2, 2.0 ** 12)])
def test_rows_near_the_ends_of_a_type(dt, size, rows, K, group):
    """Finite results come out finite, and a matrix row of zeros gives zeros."""
    pkg = load_pkg()
    N = 40
    codes, scales, zeros = weights(K, 1, N, K, group, False)
    scales[:, 5] = 0
    x = on_gpu(size * np.random.default_rng(rows).standard_normal((rows, K)), dt)
    got = product(pkg, (codes, scales, zeros), x, dt, group)
    d, xd = dense(codes, scales, zeros, group)[0], x.double().cpu().numpy()
    want = xd @ d.T
    assert (got[:, 5] == 0).all()
    tol = product_bound(d, xd, dt, want) + (2.0 ** -126 if size < 1 else 0)   # subnormal results may be flushed
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,K,N", [(2, 128, 40), (17, 192, 40), (9, 4096, 1100)])
def test_one_row_of_x_for_all_products(rows, K, N, dt):
    """x_share up to the largest integer."""
    pkg = load_pkg()
    w = weights(7, 1, N, K, 64, True)
    x = on_gpu(np.random.default_rng(0).standard_normal((1, K)), dt)
    d, xd = dense(*w, 64)[0], x.double().cpu().numpy()
    want = (xd @ d.T).repeat(rows, 0)
    for share in (rows, 2 ** 31 - 1):
        got = product(pkg, w, x.expand(rows, K), dt, 64, x_share=share)
        assert (np.abs(got - want) <= product_bound(d, xd, dt, want)).all()
