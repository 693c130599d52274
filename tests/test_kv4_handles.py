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


@pytest.mark.gpu
def test_plan_with_the_largest_token_count():
    """A step of 2^31 - 1 places, of which three requests use a few (26 GB of
    outputs): every place is written once, none beyond."""
    import torch
    pkg = load_pkg()
    cap, bs, W, nb = 2 ** 31 - 1, 16, 8, 16
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cached, new = i32(3, 16, 0), i32(20, 1, 5)
    ring, state = torch.arange(nb, dtype=torch.int32, device="cuda"), i32(0, nb)
    table = torch.full((3, W), -1, dtype=torch.int32, device="cuda")
    table[0, 0], table[1, 0] = 14, 15
    kv_len, q_offset, out = i32(0, 0, 0), i32(0, 0, 0, 0), i32(0, 0)
    pad = 1024
    pos = torch.full((cap + pad,), -7, dtype=torch.int32, device="cuda")
    slot = torch.full((cap + pad,), -7, dtype=torch.int64, device="cuda")
    with pkg.Kv4Cache(num_kv_heads=1, head_dim=64, block_tokens=bs, num_blocks=nb, table_width=W,
                      max_requests=3) as kv:
        kv.plan(cached.data_ptr(), new.data_ptr(), 3, ring.data_ptr(), state.data_ptr(),
                table.data_ptr(), kv_len.data_ptr(), q_offset.data_ptr(), pos.data_ptr(),
                slot.data_ptr(), cap, out.data_ptr(), stream())
        torch.cuda.synchronize()
    assert q_offset.tolist() == [0, 20, 21, 26] and kv_len.tolist() == [23, 17, 5]
    assert pos[:26].tolist() == [*range(3, 23), 16, *range(5)]
    # One new page each: 0, 1 and 2 of the ring.
    assert slot[:26].tolist() == [*range(14 * 16 + 3, 15 * 16), *range(7), 16, *range(32, 37)]
    for x in (pos, slot):
        assert all((x[a:min(a + (1 << 28), cap)] == -1).all() for a in range(26, cap, 1 << 28))
        assert (x[cap:] == -7).all()
