"""Several cache handles alive at a time, and the far end of a call's sizes."""
import numpy as np
import pytest

from conftest import load_pkg
from test_kv4 import plan_reference, stream


def plan_once(kv, cached, new, bs, W, nb, cap):
    import torch
    R = len(cached)
    used = -(-cached // bs)
    ids = np.random.default_rng(1).permutation(nb).astype(np.int32)
    table = np.full((R, W), -1, np.int32)
    own = np.arange(W)[None] < used[:, None]
    table[own] = ids[:own.sum()]
    free = nb - int(own.sum())
    ring = np.full(nb, -1, np.int32)
    ring[:free] = ids[own.sum():]
    state = np.array([0, free], np.int32)
    want = plan_reference(cached, new, ring, state, table, cap, bs, nb)
    d = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
    tc, tn, tr, ts, tt = d(cached), d(new), d(ring), d(state), d(table)
    out = [torch.full((n,), -7, dtype=t, device="cuda")
           for n, t in ((R, torch.int32), (R + 1, torch.int32), (cap, torch.int32),
                        (cap, torch.int64), (2, torch.int32))]
    kv.plan(tc.data_ptr(), tn.data_ptr(), R, tr.data_ptr(), ts.data_ptr(), tt.data_ptr(),
            out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), cap,
            out[4].data_ptr(), stream())
    for a, b in zip((tt, tr, *out), want):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [8192, 512])
def test_a_small_handle_beside_a_large_one(R):
    """What one handle can plan does not depend on which others were made."""
    pkg = load_pkg()
    bs, W = 16, 4
    g = np.random.default_rng(R)
    cached = g.integers(0, 2 * bs, R).astype(np.int32)
    new = np.ones(R, np.int32)
    kw = dict(num_kv_heads=1, head_dim=64, block_tokens=bs, table_width=W)
    with pkg.Kv4Cache(num_blocks=R * W, max_requests=R, **kw) as large:
        plan_once(large, cached, new, bs, W, R * W, R)
        with pkg.Kv4Cache(num_blocks=4, max_requests=1, **kw) as small:
            plan_once(large, cached, new, bs, W, R * W, R)
            plan_once(small, cached[:1], new[:1], bs, W, 4, 1)
        plan_once(large, cached, new, bs, W, R * W, R)


@pytest.mark.gpu
def test_many_handles_alive():
    """More handles than share a page of pinned memory, each with a workspace and
    an error word of its own; what is destroyed serves the next ones."""
    import torch
    from test_kv4 import Batch
    pkg = load_pkg()
    b = Batch(pkg, [100, 7], [1, 1], H=2, Hkv=1, D=64, bs=16, dt=0)
    want, lse = b.run()
    first = b.kv
    kw = dict(num_kv_heads=1, head_dim=64, block_tokens=16, num_blocks=b.nb, table_width=b.W,
              max_requests=2)
    for _ in range(2):
        many = [pkg.Kv4Cache(**kw) for _ in range(1030)]
        for h in (many[0], many[512], many[-1]):
            b.kv = h
            out, ls = b.run()
            assert torch.equal(out, want) and torch.equal(ls, lse)
        for h in many:
            h.close()
    b.kv = first
    assert torch.equal(b.run()[0], want)
