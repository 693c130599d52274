"""Matrix-vector products with 4-bit group-scaled weights and the routed
experts on them, against plain products in 64 bits.

Bounds: activations enter the products exactly and the sums are fp32.  A sum
runs over products within a group, then over groups; in whatever order, its
error is at most (128 + K / 32 + 16) 2^-23 sum |w||x| (the doubled unit roundoff
covers adders that truncate), plus half a unit in the last place of a 16-bit
result.  Over a whole result the errors' 2-norm stays below (K / 16 + 16) 2^-24
of the result's.  The experts' hidden values carry the gate/up product's error
into the down product; silu has slope at most 1.1.
"""
import numpy as np
import pytest

from conftest import load_pkg

BITS = {0: 24, 1: 8, 2: 11}


def torch_dtype(dt):
    import torch
    return (torch.float32, torch.bfloat16, torch.float16)[dt]


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def weights(seed, E, N, K, group, zeros):
    g = np.random.default_rng(seed)
    G = -(-K // group)
    codes = g.integers(0, 256, (E, N, K // 2), dtype=np.uint8)
    scales = (0.01 * (0.5 + g.random((E, N, G)))).astype(np.float16)
    z = g.integers(0, 16, (E, N, G), dtype=np.uint8) if zeros else None
    return codes, scales, z


def dense(codes, scales, zeros, group):
    """float64 weights [E][N][K]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(np.float64)
    at = np.arange(c.shape[-1]) // group
    z = 8.0 if zeros is None else zeros.astype(np.float64)[..., at]
    return (c - z) * scales.astype(np.float64)[..., at]


def product_bound(w, x, dt, y):
    K = w.shape[1]
    tol = (128 + K / 32 + 16) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    return tol + 2.0 ** -BITS[dt] * np.abs(y)


def on_gpu(x, dt):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(torch_dtype(dt))


DTYPES = pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("N,K,group,zeros", [
    (1, 32, 32, True), (16, 64, 64, False), (33, 96, 64, True), (100, 448, 128, True),
    (257, 1408, 32, False), (48, 4096, 128, False), (31, 14336, 64, True), (2000, 160, 128, True),
])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8, 17])
def test_matvec(N, K, group, zeros, rows, dt):
    import torch
    pkg = load_pkg()
    w = weights(N + K, 1, N, K, group, zeros)
    x = on_gpu(np.random.default_rng(rows).standard_normal((rows, K)), dt)
    y = torch.full((rows, N), float("nan"), dtype=x.dtype, device="cuda")
    with pkg.W4Matrix(*w, group=group) as m:
        m.matvec(x.data_ptr(), y.data_ptr(), rows, dt, stream())
        got = y.double().cpu().numpy()
        again = torch.empty_like(y)
        m.matvec(x.data_ptr(), again.data_ptr(), rows, dt, stream())
        assert torch.equal(again, y)
    d, xd = dense(*w, group)[0], x.double().cpu().numpy()
    want = xd @ d.T
    assert (np.abs(got - want) <= product_bound(d, xd, dt, want)).all()
    if dt == 0:
        assert np.linalg.norm(got - want) <= (K / 16 + 16) * 2.0 ** -24 * np.linalg.norm(want) \
            + 2.0 ** -24 * np.linalg.norm(np.abs(xd) @ np.abs(d).T) * 4


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [16, 24, 33, 64, 200, 512])
def test_matvec_many_rows(rows):
    """Row counts past one pass of the kernel, fp32 (the widest operand)."""
    import torch
    pkg = load_pkg()
    N, K = 70, 480
    w = weights(3, 1, N, K, 32, True)
    x = on_gpu(np.random.default_rng(rows).standard_normal((rows, K)), 0)
    y = torch.full((rows, N), float("nan"), device="cuda")
    with pkg.W4Matrix(*w, group=32, max_rows=0) as m:
        m.matvec(x.data_ptr(), y.data_ptr(), rows, 0, stream())
    d, xd = dense(*w, 32)[0], x.double().cpu().numpy()
    want = xd @ d.T
    assert (np.abs(y.double().cpu().numpy() - want) <= product_bound(d, xd, 0, want)).all()


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("E,rows,share", [(3, 7, 1), (5, 24, 2), (64, 64, 8), (256, 5, 1)])
def test_matvec_by_matrix(E, rows, share, dt):
    """Each product with a matrix of its own; entries outside the range give
    zeros; products that share a matrix; strided activations."""
    import torch
    pkg = load_pkg()
    N, K, group = 50, 224, 64
    w = weights(E, E, N, K, group, True)
    g = np.random.default_rng(rows)
    pick = g.integers(0, E, rows).astype(np.int32)
    pick[1] = pick[0]
    pick[2], pick[-1] = -1, E
    wide = on_gpu(g.standard_normal((-(-rows // share), K + 3)), dt)
    x = wide[:, 3:]
    y = torch.full((rows, N), float("nan"), dtype=x.dtype, device="cuda")
    t = torch.from_numpy(pick).cuda()
    with pkg.W4Matrix(*w, group=group) as m:
        m.matvec(x.data_ptr(), y.data_ptr(), rows, dt, stream(), matrix_ptr=t.data_ptr(),
                 x_row_stride=x.stride(0), x_share=share)
    d, xd, got = dense(*w, group), x.double().cpu().numpy(), y.double().cpu().numpy()
    for i in range(rows):
        if not 0 <= pick[i] < E:
            assert (got[i] == 0).all()
            continue
        xi = xd[i // share][None]
        want = xi @ d[pick[i]].T
        assert (np.abs(got[i] - want[0]) <= product_bound(d[pick[i]], xi, dt, want)[0]).all(), i


def silu(v):
    return v / (1 + np.exp(-v))


def gated_bound(d, x, want_gate, want_up):
    half = d.shape[0] // 2
    b = product_bound(d, x, 0, x @ d.T)
    eg, eu = b[:, :half], b[:, half:]
    h = silu(want_gate) * want_up
    return 1.1 * eg * np.abs(want_up) + np.abs(silu(want_gate)) * eu + eg * eu + 2.0 ** -20 * np.abs(h)


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("ff,K", [(1, 32), (40, 128), (448, 256), (131, 96)])
def test_gated(ff, K, dt):
    import torch
    pkg = load_pkg()
    rows, group = 4, 32
    w = weights(ff, 1, 2 * ff, K, group, True)
    x = on_gpu(3 * np.random.default_rng(ff).standard_normal((rows, K)), dt)
    y = torch.full((rows, ff), float("nan"), dtype=x.dtype, device="cuda")
    with pkg.W4Matrix(*w, group=group, gated=True) as m:
        assert m.outputs == ff
        m.matvec(x.data_ptr(), y.data_ptr(), rows, dt, stream())
    d, xd = dense(*w, group)[0], x.double().cpu().numpy()
    a = xd @ d.T
    gate, up = a[:, :ff], a[:, ff:]
    want = silu(gate) * up
    tol = gated_bound(d, xd, gate, up) + 2.0 ** -BITS[dt] * np.abs(want)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("T,k,E,d,ff,group", [
    (1, 1, 1, 64, 32, 32), (1, 2, 16, 256, 448, 128), (3, 2, 4, 128, 96, 64),
    (8, 2, 8, 512, 1408, 128), (17, 8, 64, 96, 64, 32), (64, 8, 8, 64, 96, 32),
])
def test_experts(T, k, E, d, ff, group, dt):
    import torch
    pkg = load_pkg()
    gu, dn = weights(1, E, 2 * ff, d, group, True), weights(2, E, d, ff, group, False)
    g = np.random.default_rng(T)
    x = on_gpu(g.standard_normal((T, d)), dt)
    idx = np.stack([g.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    wt = g.random((T, k)).astype(np.float32)
    if T > 2:
        idx[1, 0], idx[2, k - 1] = -1, E      # skipped
        wt[1, 0] = np.nan                     # and its weight not looked at
    y = torch.full((T, d), float("nan"), dtype=x.dtype, device="cuda")
    ti, tw = torch.from_numpy(idx).cuda(), torch.from_numpy(wt).cuda()
    with pkg.W4Matrix(*gu, group=group, gated=True) as a, pkg.W4Matrix(*dn, group=group) as b:
        pkg.w4_experts(a, b, x.data_ptr(), ti.data_ptr(), tw.data_ptr(), y.data_ptr(), T, k, dt,
                       stream())
        got = y.double().cpu().numpy()
    dg, dd, xd = dense(*gu, group), dense(*dn, group), x.double().cpu().numpy()
    for t in range(T):
        want, tol = np.zeros(d), np.zeros(d)
        for s in range(k):
            e = idx[t, s]
            if not 0 <= e < E:
                continue
            a = xd[t:t + 1] @ dg[e].T
            h = silu(a[:, :ff]) * a[:, ff:]
            eh = gated_bound(dg[e], xd[t:t + 1], a[:, :ff], a[:, ff:])
            v = (h @ dd[e].T)[0]
            ev = product_bound(dd[e], h, 0, v[None])[0] + (eh @ np.abs(dd[e]).T)[0]
            want += wt[t, s] * v
            tol += wt[t, s] * (ev + 2.0 ** -22 * np.abs(v))
        tol += 2.0 ** -BITS[dt] * np.abs(want)
        assert (np.abs(got[t] - want) <= tol).all(), t


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K", [3968, 4096, 8064, 8192, 8320])
@pytest.mark.parametrize("rows,share", [(1, 1), (2, 2), (4, 4), (8, 8), (2, 1)])
def test_matvec_at_the_inline_limits(rows, share, K, group, dt):
    """Sizes on both sides of where a product makes its operands itself: one
    row of x that several products share, by one matrix and by several."""
    import torch
    pkg = load_pkg()
    N, E = 48, 3
    w = weights(K + group, E, N, K, group, True)
    x = on_gpu(np.random.default_rng(K).standard_normal((-(-rows // share), K)), dt)
    d, xd = dense(*w, group), x.double().cpu().numpy()
    with pkg.W4Matrix(*w, group=group) as m:
        for pick in (None, np.zeros(rows, np.int32), (np.arange(rows) % E).astype(np.int32)):
            t = None if pick is None else torch.from_numpy(pick).cuda()
            y = torch.full((rows, N), float("nan"), dtype=x.dtype, device="cuda")
            m.matvec(x.data_ptr(), y.data_ptr(), rows, dt, stream(),
                     matrix_ptr=0 if t is None else t.data_ptr(), x_share=share)
            got = y.double().cpu().numpy()
            for i in range(rows):
                e = 0 if pick is None else pick[i]
                xi = xd[i // share][None]
                want = xi @ d[e].T
                assert (np.abs(got[i] - want[0]) <= product_bound(d[e], xi, dt, want)[0]).all(), i


@pytest.mark.gpu
def test_wide_range_and_non_finite_activations():
    """fp32 activations over the whole exponent range enter exactly; an
    infinity or a NaN stays in its own row."""
    import torch
    pkg = load_pkg()
    N, K = 40, 128
    w = weights(5, 1, N, K, 32, False)
    g = np.random.default_rng(1)
    x = g.standard_normal((4, K)) * 10.0 ** g.integers(-30, 30, (4, K))
    x[1] = 1e-41 * g.standard_normal(K)       # subnormals
    x = x.astype(np.float32)
    x[2, 3], x[3, 5] = np.inf, np.nan
    xt = torch.from_numpy(x).cuda()
    y = torch.zeros(4, N, device="cuda")
    with pkg.W4Matrix(*w, group=32) as m:
        m.matvec(xt.data_ptr(), y.data_ptr(), 4, 0, stream())
    got = y.double().cpu().numpy()
    d = dense(*w, 32)[0]
    want = x[0:1].astype(np.float64) @ d.T
    assert (np.abs(got[0] - want[0]) <= product_bound(d, x[0:1].astype(np.float64), 0, want)[0]).all()
    # Subnormal activations may be flushed: the result is below the smallest normal number's.
    assert (np.abs(got[1]) <= 1.2e-38 * np.abs(d).sum(1)).all()
    assert not np.isfinite(got[2][np.abs(d[:, 3]) > 0]).any()
    assert np.isnan(got[3]).all()


@pytest.mark.gpu
def test_from_device_another_stream_and_growth():
    import torch
    pkg = load_pkg()
    N, K, E = 64, 256, 2
    c, s, z = weights(6, E, N, K, 64, True)
    dev = [torch.from_numpy(a).cuda() for a in (c, s, z)]
    with pkg.W4Matrix(c, s, z, group=64) as host, pkg.W4Matrix.from_device_pointers(
            *(a.data_ptr() for a in dev), matrices=E, rows=N, cols=K, group=64) as m:
        for a in dev:
            a.zero_()          # copied: the caller's arrays may go
        x = torch.randn(100, K, device="cuda")
        pick = torch.randint(0, E, (100,), dtype=torch.int32, device="cuda")
        want, y = torch.empty(100, N, device="cuda"), torch.zeros(100, N, device="cuda")
        host.matvec(x.data_ptr(), want.data_ptr(), 100, 0, stream(), matrix_ptr=pick.data_ptr())
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        late = torch.zeros_like(x)
        with torch.cuda.stream(st):
            torch.cuda._sleep(20_000_000)
            late.copy_(x)
            m.matvec(late.data_ptr(), y.data_ptr(), 100, 0, st.cuda_stream,
                     matrix_ptr=pick.data_ptr())
        st.synchronize()
        assert torch.equal(y, want)
        assert m.device_bytes() > 0


# ------------------------------------------------------------ host helpers
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("K,group", [(128, 32), (448, 128), (96, 64)])
def test_quantize_w4(K, group, zeros):
    """Off by at most half a step, plus what float16 rounds off the scale."""
    pkg = load_pkg()
    g = np.random.default_rng(K)
    w = (0.02 * g.standard_normal((2, 20, K))).astype(np.float32)
    w[0, 0] = 0
    c, s, z = pkg.quantize_w4(w, group, zeros)
    assert c.shape == (2, 20, K // 2) and s.shape == (2, 20, -(-K // group))
    assert (z is None) == (not zeros)
    at = np.arange(K) // group
    step = s.astype(np.float64)[..., at]
    # Without zeros the range is -8..7 steps of max / 7.5: its upper end is cut by half a step.
    assert (np.abs(dense(c, s, z, group) - w) <= 0.5 * step * 1.01 + 16 * step * 2.0 ** -11).all()


# --------------------------------------------------------------- refusals
@pytest.mark.parametrize("kw", [
    dict(num_matrices=0), dict(num_matrices=257), dict(rows=0), dict(rows=3, gated=1),
    dict(rows=(1 << 24) + 1), dict(cols=48), dict(cols=0), dict(cols=65568), dict(group=16),
    dict(max_rows=513), dict(max_rows=-1), dict(device=-1),
])
def test_create_refuses(kw):
    import ctypes
    pkg = load_pkg()
    L = pkg.load_library()
    cfg = pkg.MoeW4Config()
    L.moe_w4_config_init(ctypes.byref(cfg))
    for k, v in kw.items():
        setattr(cfg, k, v)
    h = ctypes.c_void_p()
    buf = ctypes.create_string_buffer(16)
    for fn in (L.moe_w4_create, L.moe_w4_create_from_device):
        assert fn(ctypes.byref(cfg), buf, buf, None, ctypes.byref(h)) == -1
        assert not h


def test_null_arguments():
    pkg = load_pkg()
    L = pkg.load_library()
    assert L.moe_w4_create(None, None, None, None, None) == -1
    assert L.moe_w4_device_bytes(None) == 0
    L.moe_w4_destroy(None)
    L.moe_w4_config_init(None)
    assert L.moe_w4_matvec_device(None, None, 0, 1, 0, 1, None, None, None) == -1
    assert L.moe_w4_experts_device(None, None, None, 0, 1, 1, None, None, None, None) == -1
    with pytest.raises(ValueError):
        pkg.W4Matrix(np.zeros((2, 4, 32), np.uint8), np.zeros((2, 4, 1), np.float16), group=32)
    with pytest.raises(ValueError):
        pkg.quantize_w4(np.zeros((2, 40), np.float32))


@pytest.mark.gpu
def test_calls_refuse():
    pkg = load_pkg()
    a = pkg.W4Matrix(*weights(1, 2, 64, 64, 32, False), group=32, gated=True)
    b = pkg.W4Matrix(*weights(1, 2, 64, 32, 32, False), group=32)
    p = 4096   # an address that is never touched: every call is refused on the host

    def bad(f, *args, **kw):
        with pytest.raises(pkg.MoeError) as e:
            f(*args, **kw)
        return e.value.code
    assert bad(b.matvec, p, p, 513, 0) == bad(b.matvec, p, p, -1, 0) == bad(b.matvec, 0, p, 1, 0) == -1
    assert bad(b.matvec, p, 0, 1, 0) == bad(b.matvec, p, p, 1, 3) == bad(b.matvec, p + 2, p, 1, 0) == -1
    assert bad(b.matvec, p, p + 1, 1, 1) == bad(b.matvec, p, p, 1, 0, x_share=0) == -1
    ex = lambda g=a, d=b, x=p, i=p, w=p, y=p, T=1, k=1, dt=0: pkg.w4_experts(  # noqa: E731
        g, d, x, i, w, y, T, k, dt)
    other = pkg.W4Matrix(*weights(1, 3, 64, 32, 32, False), group=32)
    for kw in (dict(g=b), dict(d=a), dict(d=other), dict(x=0), dict(i=0), dict(w=0), dict(y=0),
               dict(x=p + 2), dict(T=-1), dict(k=0), dict(T=257, k=2), dict(dt=7)):
        assert bad(ex, **kw) == -1, kw
    b.matvec(0, 0, 0, 0)
    ex(T=0, x=0)
