"""4-bit products of activations at the ends of their types' ranges.

Bounds as in test_w4: activations enter exactly, sums are fp32."""
import numpy as np
import pytest

from conftest import load_pkg
from test_w4 import BITS, dense, gated_bound, on_gpu, product_bound, silu, stream, torch_dtype, weights


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


def as_defined(w, x, group):
    """x [m][K] and one matrix, term by term in float64: 0 * inf is a NaN there too."""
    d = dense(*w, group)[0]
    with np.errstate(invalid="ignore"):
        return np.stack([(row[None] * d).sum(1) for row in x])


def same_or_near(got, want, tol):
    """NaN where want is, the same infinity where it is one, else within tol."""
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all()


def put_infinities(x):
    """Rows 0.. of x [m][K]: one of each sign, two that agree or not, the largest
    finite number beside one, a NaN beside one; the last rows stay as they were."""
    m, K = x.shape
    inf = np.inf
    at = [{3: inf}, {K - 1: -inf}, {0: inf, K // 2: inf}, {1: inf, 33 % K: -inf}, {7: inf, 9: np.nan}]
    for r, cells in enumerate(at[:max(1, m - 1)]):
        for k, v in cells.items():
            x[r, k] = v
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,K,N", [(1, 64, 40), (3, 160, 33), (4, 448, 16), (7, 4096, 100), (17, 192, 260), (6, 4224, 7200)])
def test_infinite_activations(rows, K, N, group, dt):
    """What the definition gives, one tile of rows a block and several, operands
    made in the block and apart."""
    pkg = load_pkg()
    w = weights(K, 1, N, K, group, True)
    w[0][0, :, 1] = 0x55     # columns 2 and 3: some weights of exactly zero
    w[2][0, ::2] = 5
    x = put_infinities(np.random.default_rng(rows).standard_normal((rows, K)))
    x = on_gpu(x, dt)
    xd = x.double().cpu().numpy()
    want = as_defined(w, xd, group)
    got = product(pkg, w, x, dt, group)
    with np.errstate(invalid="ignore"):
        tol = product_bound(dense(*w, group)[0], np.where(np.isfinite(xd), xd, 0), dt, np.where(np.isfinite(want), want, 0))
    same_or_near(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1], ids=["f32", "bf16"])
def test_infinite_activations_gated(dt):
    pkg = load_pkg()
    ff, K, group, rows = 48, 192, 64, 6
    w = weights(2, 1, 2 * ff, K, group, True)
    x = on_gpu(put_infinities(np.random.default_rng(1).standard_normal((rows, K))), dt)
    xd = x.double().cpu().numpy()
    a = as_defined(w, xd, group)
    with np.errstate(invalid="ignore", over="ignore"):
        want = silu(a[:, :ff]) * a[:, ff:]
    got = product(pkg, w, x, dt, group, gated=True)
    tol = np.zeros(want.shape)      # only the last row is finite
    tol[-1:] = gated_bound(dense(*w, group)[0], xd[-1:], a[-1:, :ff], a[-1:, ff:]) + 2.0 ** -BITS[dt] * np.abs(want[-1:])
    assert np.isfinite(want[-1]).all() and not np.isfinite(want[:-1]).any()
    same_or_near(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("ff", [96, 4608])
def test_infinite_activations_experts(ff):
    """Through both products, the down product's columns in one part and in two:
    a token's infinity stays that token's."""
    import torch
    pkg = load_pkg()
    T, k, E, d, group = 4, 2, 4, 256, 128
    gu, dn = weights(1, E, 2 * ff, d, group, True), weights(2, E, d, ff, group, True)
    g = np.random.default_rng(5)
    x = g.standard_normal((T, d)).astype(np.float32)
    clean = x.copy()
    x[1, 7] = np.inf
    idx = torch.from_numpy(np.stack([g.permutation(E)[:k] for _ in range(T)]).astype(np.int32)).cuda()
    wt = torch.from_numpy(g.random((T, k)).astype(np.float32) + 0.1).cuda()
    with pkg.W4Matrix(*gu, group=group, gated=True) as a, pkg.W4Matrix(*dn, group=group) as b:
        out = []
        for v in (clean, x):
            t, y = torch.from_numpy(v).cuda(), torch.zeros(T, d, device="cuda")
            pkg.w4_experts(a, b, t.data_ptr(), idx.data_ptr(), wt.data_ptr(), y.data_ptr(), T, k, 0, stream())
            out.append(y)
    assert torch.equal(out[0][[0, 2, 3]], out[1][[0, 2, 3]])
    # gate and up are infinities of either sign or NaN: silu gives inf, NaN at -inf;
    # some hidden values are NaN, so that every output is.
    assert torch.isnan(out[1][1]).all()


@pytest.mark.gpu
def test_handles_that_come_and_go():
    """Handles of many sizes made and destroyed in turn: each keeps its weights and
    its workspace to itself."""
    import torch
    pkg = load_pkg()
    g = np.random.default_rng(11)
    live = []
    for step in range(60):
        if len(live) > 12 or (live and g.random() < 0.35):
            live.pop(int(g.integers(len(live))))[0].close()
        N, K, group = int(g.integers(1, 900)), 32 * int(g.integers(1, 40)), int(g.choice([32, 64, 128]))
        w = weights(step, 1, N, K, group, True)
        live.append((pkg.W4Matrix(*w, group=group, max_rows=int(g.integers(0, 40))), w, group))
        if step % 6:
            continue
        outs = []
        for m, w, group in live:       # all at once: none waits for another's result
            x = on_gpu(g.standard_normal((20, w[0].shape[2] * 2)), 0)
            y = torch.full((20, w[0].shape[1]), -7, dtype=torch.float32, device="cuda")
            m.matvec(x.data_ptr(), y.data_ptr(), 20, 0, stream())
            outs.append((x, y))
        for (m, w, group), (x, y) in zip(live, outs):
            d, xd = dense(*w, group)[0], x.double().cpu().numpy()
            want = xd @ d.T
            assert (np.abs(y.double().cpu().numpy() - want) <= product_bound(d, xd, 0, want)).all()
    for m, *_ in live:
        m.close()
