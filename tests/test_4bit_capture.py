"""The 4-bit operators in CUDA graphs: a first call may be a captured one, a
replay takes the inputs of its time, later larger calls leave a captured graph's
workspace alone, and a call that would have to allocate is refused before it
spoils the capture.  Replays are compared bit for bit with direct calls."""
import numpy as np
import pytest

from conftest import load_pkg
from test_kv4 import cache_of, granule, stream, torch_dtype
from test_w4 import on_gpu, weights


def captured(call):
    """A graph of what call() enqueues on the capturing stream."""
    import torch
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    return g


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K", [(1, 256), (4, 4096), (16, 256)])
@pytest.mark.parametrize("dt", [0, 1], ids=["f32", "bf16"])
def test_first_matvec_captured(rows, K, dt):
    import torch
    pkg = load_pkg()
    N, group = 96, 64
    w = weights(1, 1, N, K, group, True)
    x = on_gpu(np.random.default_rng(0).standard_normal((rows, K)), dt)
    y, want = torch.zeros(rows, N, dtype=x.dtype, device="cuda"), torch.zeros(rows, N, dtype=x.dtype, device="cuda")
    with pkg.W4Matrix(*w, group=group) as m, pkg.W4Matrix(*w, group=group) as direct:
        g = captured(lambda: m.matvec(x.data_ptr(), y.data_ptr(), rows, dt, stream()))
        for _ in range(2):
            x.mul_(-1.5)
            direct.matvec(x.data_ptr(), want.data_ptr(), rows, dt, stream())
            g.replay()
            assert torch.equal(y, want) and want.abs().max() > 0
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,d,ff", [(1, 2, 16, 256, 448), (8, 2, 8, 512, 1408), (4, 2, 4, 4096, 4608)])
@pytest.mark.parametrize("dt", [0, 2], ids=["f32", "f16"])
def test_first_experts_captured(T, k, E, d, ff, dt):
    import torch
    pkg = load_pkg()
    group = 128
    gu, dn = weights(1, E, 2 * ff, d, group, True), weights(2, E, d, ff, group, False)
    g = np.random.default_rng(T)
    x = on_gpu(g.standard_normal((T, d)), dt)
    idx = torch.from_numpy(np.stack([g.permutation(E)[:k] for _ in range(T)]).astype(np.int32)).cuda()
    wt = torch.from_numpy(g.random((T, k)).astype(np.float32)).cuda()
    y, want = torch.zeros_like(x), torch.zeros_like(x)

    def pair():
        return pkg.W4Matrix(*gu, group=group, gated=True), pkg.W4Matrix(*dn, group=group)
    a, b = pair()
    a2, b2 = pair()
    graph = captured(lambda: pkg.w4_experts(a, b, x.data_ptr(), idx.data_ptr(), wt.data_ptr(),
                                            y.data_ptr(), T, k, dt, stream()))
    for _ in range(2):
        x.mul_(-0.75)
        idx.copy_((idx + 1) % E)
        pkg.w4_experts(a2, b2, x.data_ptr(), idx.data_ptr(), wt.data_ptr(), want.data_ptr(), T, k,
                       dt, stream())
        graph.replay()
        assert torch.equal(y, want) and want.abs().max() > 0
    torch.cuda.synchronize()
    for m in (a, b, a2, b2):
        m.close()


@pytest.mark.gpu
def test_a_captured_call_survives_growth():
    """The graph's workspace stays the handle's when larger calls need more."""
    import torch
    pkg = load_pkg()
    E, d, ff, group, dt = 4, 256, 192, 64, 0
    gu, dn = weights(1, E, 2 * ff, d, group, True), weights(2, E, d, ff, group, True)
    a = pkg.W4Matrix(*gu, group=group, gated=True, max_rows=16)
    b = pkg.W4Matrix(*dn, group=group, max_rows=16)
    g = np.random.default_rng(3)

    def inputs(T, k=2):
        return (on_gpu(g.standard_normal((T, d)), dt),
                torch.from_numpy(g.integers(0, E, (T, k)).astype(np.int32)).cuda(),
                torch.from_numpy(g.random((T, k)).astype(np.float32)).cuda(),
                torch.zeros(T, d, device="cuda"))

    def run(x, idx, wt, y):
        pkg.w4_experts(a, b, x.data_ptr(), idx.data_ptr(), wt.data_ptr(), y.data_ptr(), len(x), 2,
                       dt, stream())
    small, large = inputs(8), inputs(200)
    run(*small)
    want = small[3].clone()
    graph = captured(lambda: run(*small))
    before = a.device_bytes(), b.device_bytes()
    run(*large)
    first = large[3].clone()
    assert a.device_bytes() > before[0] and b.device_bytes() > before[1]
    others = [torch.full((1 << 20,), -3, dtype=torch.int32, device="cuda") for _ in range(8)]
    for _ in range(3):
        small[3].zero_()
        graph.replay()
        assert torch.equal(small[3], want)
        run(*large)
        assert torch.equal(large[3], first)
    assert all((o == -3).all() for o in others)
    torch.cuda.synchronize()
    a.close(), b.close()


@pytest.mark.gpu
def test_growth_inside_a_capture_is_refused():
    """Refused on the host; the capture goes on and its graph holds the rest."""
    import torch
    pkg = load_pkg()
    N, K, group, rows = 64, 256, 64, 20
    x = torch.randn(rows, K, device="cuda")
    y, want = torch.zeros(rows, N, device="cuda"), torch.zeros(rows, N, device="cuda")
    with pkg.W4Matrix(*weights(1, 1, N, K, group, True), group=group, max_rows=rows - 1) as m:
        m.matvec(x.data_ptr(), want.data_ptr(), rows - 1, 0, stream())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(pkg.MoeError, match="max_rows") as e:
                m.matvec(x.data_ptr(), y.data_ptr(), rows, 0, stream())
            assert e.value.code == -2
            m.matvec(x.data_ptr(), y.data_ptr(), rows - 1, 0, stream())
        graph.replay()
        assert torch.equal(y, want)
        m.matvec(x.data_ptr(), y.data_ptr(), rows, 0, stream())      # outside it grows
        assert torch.equal(y[:-1], want[:-1]) and y[-1].abs().max() > 0
    # The results of a single matrix's experts are not pre-sized: a call outside first.
    d, ff = 64, 32
    a = pkg.W4Matrix(*weights(2, 1, 2 * ff, d, 32, True), group=32, gated=True)
    b = pkg.W4Matrix(*weights(3, 1, d, ff, 32, True), group=32)
    x, out = torch.randn(2, d, device="cuda"), torch.zeros(2, 2, d, device="cuda")
    idx, wt = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda")

    def experts(i):
        pkg.w4_experts(a, b, x.data_ptr(), idx.data_ptr(), wt.data_ptr(), out[i].data_ptr(), 2, 1,
                       0, stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(pkg.MoeError, match="capture"):
            experts(0)
        out[0].fill_(5.0)
    experts(1)
    captured(lambda: experts(0)).replay()
    assert torch.equal(out[0], out[1]) and out[1].abs().max() > 0
    torch.cuda.synchronize()
    a.close(), b.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1], ids=["f32", "bf16"])
def test_first_plan_append_and_attention_captured(dt):
    """One step of a request that grows, as a graph."""
    import torch
    pkg = load_pkg()
    D, H, bs, nb, W = 64, 2, 16, 4, 4
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731

    def world():
        return dict(cached=i32(0), new=i32(1), ring=torch.arange(nb, dtype=torch.int32, device="cuda"),
                    state=[i32(0, nb), i32(0, 0)], table=torch.full((1, W), -1, dtype=torch.int32, device="cuda"),
                    kv=i32(0), qo=i32(0, 0), pos=i32(0), slot=torch.zeros(1, dtype=torch.int64, device="cuda"),
                    cache=torch.zeros(nb * H * granule(D), dtype=torch.uint8, device="cuda"),
                    out=torch.zeros(1, H, D, dtype=t, device="cuda"))
    t = torch_dtype(dt)
    x = torch.randn(3, 1, H, D, device="cuda").to(t)

    def step(h, w):
        p = lambda k: w[k].data_ptr()  # noqa: E731
        h.plan(p("cached"), p("new"), 1, p("ring"), w["state"][0].data_ptr(), p("table"), p("kv"),
               p("qo"), p("pos"), p("slot"), 1, w["state"][1].data_ptr(), stream())
        h.append(p("cache"), x[0].data_ptr(), x[1].data_ptr(), dt, 1, p("slot"), stream())
        h.attention(p("cache"), x[2].data_ptr(), p("out"), dt, 1, H, p("table"), p("kv"), p("qo"),
                    1, stream())
        w["state"][0].copy_(w["state"][1])
        w["cached"].copy_(w["kv"])
    a, b = world(), world()
    with cache_of(pkg, H=H, D=D, bs=bs, nb=nb, W=W, R=1) as h, \
            cache_of(pkg, H=H, D=D, bs=bs, nb=nb, W=W, R=1) as h2:
        graph = captured(lambda: step(h, a))
        for i in range(40):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(t))
            graph.replay()
            step(h2, b)
            assert torch.equal(a["out"], b["out"]) and torch.equal(a["cache"], b["cache"]), i
            assert int(a["kv"]) == i + 1 and a["out"].abs().max() > 0
        torch.cuda.synchronize()
