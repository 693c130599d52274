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
