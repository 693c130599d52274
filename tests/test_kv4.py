"""The paged 4-bit key/value cache: plan (block tables and slot maps), append
and attention, against plain implementations in 64 bits.

The cache's layout is rebuilt here from its description, byte by byte; the
quantiser's result is compared bit for bit, since every step of it is defined.

Attention's bound: a score is a sum of D products whose factors carry 22 (fp32)
or 11 (16-bit types) significant bits or are exact, summed in fp32 in an
unknown order, so it is off by at most e = (D + 16) 2^-23 S, S the largest
scale * sum |q||k| of the row (the doubled unit roundoff covers adders that
truncate).  Each probability is then off by 2 e relative, the output by that
times the largest |v|; rounding the probabilities to 11 bits adds 2^-11 max|v|
for the 16-bit types, summing L of them in fp32 (L + 16) 2^-23 max|v|, and the
output's own rounding half a unit in the last place.
"""
import math

import numpy as np
import pytest

from conftest import load_pkg

BITS = {0: 24, 1: 8, 2: 11}   # significant bits of f32, bf16, f16


def torch_dtype(dt):
    import torch
    return (torch.float32, torch.bfloat16, torch.float16)[dt]


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def cache_of(pkg, H=2, D=128, bs=16, nb=32, W=8, R=8):
    return pkg.Kv4Cache(num_kv_heads=H, head_dim=D, block_tokens=bs, num_blocks=nb, table_width=W,
                        max_requests=R)


# ------------------------------------------------------------------ layout
def places(D):
    """Byte and nibble of (token, dim) in a granule, K and V: [16][D] each."""
    G = D // 64
    k, v = np.zeros((16, D), int), np.zeros((16, D), int)
    at = 0
    for t in range(16):
        for j in range(4):
            for g in range(G):
                for h in range(2):
                    for b in range(4):
                        d = 64 * g + 16 * j + 8 * h + 2 * b
                        k[t, d], k[t, d + 1] = 2 * at, 2 * at + 1
                        at += 1
    for p in range(G):
        for n in range(8):
            for j in range(4):
                for w in range(4 // G):
                    u = p * (4 // G) + w
                    t = 8 * (u // 2) + 2 * j + u % 2
                    for g in range(G):
                        for b in range(4):
                            d = 64 * g + 8 * n + 2 * b
                            v[t, d], v[t, d + 1] = 2 * at, 2 * at + 1
                            at += 1
    assert at == 16 * D
    return k, v


def read_cache(cache, page, head, off, D):
    """(k, v) values of one token, float64; cache [nb][H][bs/16][granule]."""
    G = D // 64
    gran = cache[page, head, off // 16]
    nib = np.stack([gran[:16 * D] & 15, gran[:16 * D] >> 4], -1).reshape(-1).astype(np.float64)
    par = gran[16 * D:].copy().view(np.float16).astype(np.float64).reshape(2, 16, G, 2)
    at, t = np.arange(D) // 64, off % 16
    with np.errstate(invalid="ignore"):
        return tuple(nib[p[t]] * par[i, t, at, 0] + par[i, t, at, 1]
                     for i, p in enumerate(places(D)))


def quantise(x):
    """x [D] float32 -> codes [D], (scale, minimum) [G][2] float16."""
    x = x.astype(np.float32).reshape(-1, 64)
    nan = np.isnan(x).any(1)
    x = np.clip(np.where(np.isnan(x), 0, x), np.float32(-65504), np.float32(65504))
    lo, hi = x.min(1), x.max(1)
    s = ((hi - lo) * np.float32(1 / 15)).astype(np.float16)
    m = lo.astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((x - m.astype(np.float32)[:, None]) / s.astype(np.float32)[:, None])
    c = np.where(s[:, None] > 0, np.clip(q, 0, 15), 0)
    c[nan], s[nan], m[nan] = 0, np.nan, np.nan
    return c.reshape(-1).astype(np.uint8), np.stack([s, m], -1)


def write_cache(cache, page, head, off, k, v, D):
    G = D // 64
    gran = cache[page, head, off // 16]
    t = off % 16
    par = gran[16 * D:].view(np.float16).reshape(2, 16, G, 2)
    for i, (x, p) in enumerate(zip((k, v), places(D))):
        c, par[i, t] = quantise(x)
        for d in range(D):
            byte, shift = p[t, d] // 2, 4 * (p[t, d] % 2)
            gran[byte] = (gran[byte] & (0xF0 if shift == 0 else 0x0F)) | (c[d] << shift)


def granule(D):
    return 16 * D + 128 * (D // 64)


# ------------------------------------------------------------------- plan
def plan_reference(cached, new, ring, state, table, cap, bs, nb):
    """One request after the other."""
    R, W = table.shape
    ring, table = ring.copy(), table.copy()
    head, count = state
    if not (0 <= head < nb and 0 <= count <= nb):
        head = count = 0
    kv, qo = np.zeros(R, np.int32), np.zeros(R + 1, np.int32)
    pos, slot = np.full(cap, -1, np.int32), np.full(cap, -1, np.int64)
    start = asked = taken = given = 0
    for r in range(R):
        c, n = int(cached[r]), int(new[r])
        qo[r] = min(start, cap)
        stop = start + max(n, 0)
        inside = 0 <= c <= W * bs
        ok = inside and n >= 0 and c + n <= W * bs and (n == 0 or stop <= cap)
        if ok:
            need = -(-(c + n) // bs) - -(-c // bs)
            asked += need
            ok = need == 0 or asked <= count
            if ok:
                for i in range(need):
                    table[r, -(-c // bs) + i] = ring[(head + taken + i) % nb]
                taken += need
                kv[r] = c + n
        if inside and n < 0:
            for i in range(-(-c // bs)):
                if given < nb - count:
                    ring[(head + count + given) % nb] = table[r, i]
                    given += 1
        for t in range(start, min(stop, cap)):
            p = c + t - start
            pos[t] = np.array(p).astype(np.int32)
            if ok and 0 <= table[r, p // bs] < nb:
                slot[t] = int(table[r, p // bs]) * bs + p % bs
        start = stop
    qo[R] = min(start, cap)
    return (table, ring, kv, qo, pos, slot,
            np.array([(head + taken) % nb, count - taken + given], np.int32))


PLAN_CASES = {
    # cached, new, block, width, pool, head, free, cap
    "one": dict(cached=[0], new=[1], bs=16, W=1, nb=1, head=0, free=1, cap=1),
    "page_boundaries": dict(cached=[15, 16, 17, 0, 31, 32], new=[1, 1, 1, 16, 2, 17], bs=16, W=4,
                            nb=24, head=20, free=8, cap=38),
    "ends_and_padding": dict(cached=[33, 5, 64, 0], new=[-1, 3, -7, -1], bs=16, W=4, nb=16, head=3,
                             free=2, cap=9),
    "pool_runs_dry": dict(cached=[16, 3, 16, 4, 16], new=[1, 2, 20, 1, 1], bs=16, W=4, nb=12,
                          head=11, free=2, cap=25),
    "out_of_range": dict(cached=[-1, 60, 64, 2 ** 31 - 1, 5], new=[2, 5, 1, 3, 4], bs=16, W=4,
                         nb=12, head=0, free=12, cap=15),
    "cap_cuts": dict(cached=[1, 2, 3, 4], new=[5, 6, 0, 3], bs=16, W=4, nb=12, head=0, free=5,
                     cap=8),
    "no_tokens": dict(cached=[4, 20], new=[0, 0], bs=48, W=2, nb=4, head=0, free=1, cap=0),
    "bad_state": dict(cached=[4, 16], new=[1, 1], bs=16, W=2, nb=4, head=9, free=1, cap=2),
    "page_outside_pool": dict(cached=[4, 16], new=[1, 1], bs=16, W=2, nb=4, head=0, free=2, cap=2,
                              spoil=True),
}


def plan_case(name):
    if name.startswith("random"):
        g = np.random.default_rng(int(name[6:]))
        R, bs, W = int(g.integers(1, 1500)), int(g.choice([16, 48, 64])), 20
        cached = g.integers(0, W * bs // 2, R)
        new = np.where(g.random(R) < 0.7, 1, g.integers(-1, W * bs // 2, R))
        nb = R * W
        free = int(g.integers(0, nb // 2))
        return dict(cached=cached, new=new, bs=bs, W=W, nb=nb, head=int(g.integers(nb)),
                    free=free, cap=int(np.maximum(new, 0).sum() * g.uniform(0.8, 1.2)) + 1)
    return PLAN_CASES[name]


@pytest.mark.gpu
@pytest.mark.parametrize("name", [*PLAN_CASES, "random1", "random2", "random3"])
def test_plan(name):
    import torch
    pkg = load_pkg()
    c = plan_case(name)
    bs, W, nb, cap = c["bs"], c["W"], c["nb"], c["cap"]
    cached, new = np.array(c["cached"], np.int32), np.array(c["new"], np.int32)
    R = len(cached)
    perm = np.random.default_rng(5).permutation(nb).astype(np.int32)
    used = np.array([min(W, -(-int(x) // bs)) if x > 0 else 0 for x in cached])
    free = min(c["free"], nb)
    table = np.full((R, W), -1, np.int32)
    own = np.arange(W)[None] < used[:, None]
    table[own] = perm[(np.arange(own.sum()) + free) % nb]
    if c.get("spoil"):
        table[0, 0] = nb
    ring = np.full(nb, -1, np.int32)
    ring[(c["head"] + np.arange(free)) % nb] = perm[:free]
    state = np.array([c["head"], c["free"]], np.int32)
    want = plan_reference(cached, new, ring, state, table, cap, bs, nb)
    with cache_of(pkg, bs=bs, nb=nb, W=W, R=R) as kv:
        d = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        tc, tn, tr, ts, tt = d(cached), d(new), d(ring), d(state), d(table)
        out = [torch.full((n,), -7, dtype=t, device="cuda")
               for n, t in ((R, torch.int32), (R + 1, torch.int32), (cap, torch.int32),
                            (cap, torch.int64), (2, torch.int32))]
        for again in range(2):   # the inputs are left as they were: a step can be planned again
            kv.plan(tc.data_ptr(), tn.data_ptr(), R, tr.data_ptr(), ts.data_ptr(), tt.data_ptr(),
                    out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
                    cap, out[4].data_ptr(), stream())
            got = [x.cpu().numpy() for x in (tt, tr, *out)]
            for what, a, b in zip(("table", "ring", "kv_len", "q_offset", "position", "slot",
                                   "state"), got, want):
                assert np.array_equal(a, b), (what, again)


# ----------------------------------------------------------------- append
def edge_rows(g, N, H, D):
    """Rows with the values a quantiser can stumble on in their first heads."""
    x = g.standard_normal((N, H, D)).astype(np.float32)
    if N >= 6:
        x[0, 0, :64] = 0.0
        x[1, 0, :64] = 3.25                 # a constant group
        x[2, 0, 5] = np.nan
        x[3, 0, 7], x[3, 0, 8] = np.inf, -np.inf
        x[4, 0] *= 1e-6                     # a scale that float16 holds with few bits
        x[5, 0, :64] *= 2.0e4
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,H,D,bs,layout", [
    (1, 1, 64, 16, "dense"), (7, 3, 64, 48, "dense"), (33, 2, 128, 16, "fused"),
    (16, 4, 128, 32, "odd"), (130, 1, 64, 64, "fused"),
])
def test_append(N, H, D, bs, layout, dt):
    import torch
    pkg = load_pkg()
    g = np.random.default_rng(N * 31 + D)
    nb = -(-N // bs) + 2
    t = torch_dtype(dt)
    if layout == "fused":      # slices of one projection's rows
        both = torch.zeros(N, 3, H, D, dtype=t, device="cuda")
        k, v = both[:, 1], both[:, 2]
    elif layout == "odd":      # rows that start off 16 bytes
        both = torch.zeros(2, N, H, D + 1, dtype=t, device="cuda")
        k, v = both[0, :, :, 1:], both[1, :, :, 1:]
    else:
        k, v = (torch.zeros(N, H, D, dtype=t, device="cuda") for _ in range(2))
    for x in (k, v):
        x.copy_(torch.from_numpy(edge_rows(g, N, H, D)))
    slot = g.permutation(nb * bs)[:N].astype(np.int64)
    if N >= 16:
        slot[9], slot[10] = -1, nb * bs   # not stored
    start = g.integers(0, 256, (nb, H, bs // 16, granule(D)), dtype=np.uint8)
    want = start.copy()
    kf, vf = k.float().cpu().numpy(), v.float().cpu().numpy()
    vals = np.zeros((2, N, H, D))
    for i in range(N):
        for h in range(H):
            for a, x in enumerate((kf, vf)):
                c, p = quantise(x[i, h])
                p = p.astype(np.float64).repeat(64, 0)
                vals[a, i, h] = c * p[:, 0] + p[:, 1]
            if 0 <= slot[i] < nb * bs:
                write_cache(want, slot[i] // bs, h, slot[i] % bs, kf[i, h], vf[i, h], D)
    with cache_of(pkg, H=H, D=D, bs=bs, nb=nb) as kv:
        assert kv.cache_bytes() == start.size
        cache, ts = torch.from_numpy(start).cuda(), torch.from_numpy(slot).cuda()
        ko, vo = (torch.zeros(N, H, D, dtype=t, device="cuda") for _ in range(2))
        kv.append(cache.data_ptr(), k.data_ptr(), v.data_ptr(), dt, N, ts.data_ptr(), stream(),
                  k_strides=k.stride()[:2], v_strides=v.stride()[:2], k_out_ptr=ko.data_ptr(),
                  v_out_ptr=vo.data_ptr())
        got = cache.cpu().numpy()
        # A float16 NaN has many encodings: compared as the header's one.
        assert np.array_equal(got[..., :16 * D], want[..., :16 * D])
        a, b = (x[..., 16 * D:].copy().view(np.float16) for x in (got, want))
        assert np.array_equal(a, b, equal_nan=True)
        for o, w in ((ko, vals[0]), (vo, vals[1])):
            exact = torch.from_numpy(w).to(torch.float32).to(t).float().cpu().numpy()
            assert np.array_equal(o.float().cpu().numpy(), exact, equal_nan=True)
        # Without the optional outputs the cache is the same.
        again = torch.from_numpy(start).cuda()
        kv.append(again.data_ptr(), k.data_ptr(), v.data_ptr(), dt, N, ts.data_ptr(), stream(),
                  k_strides=k.stride()[:2], v_strides=v.stride()[:2])
        assert torch.equal(again, cache)


# -------------------------------------------------------------- attention
class Batch:
    """Ragged requests over a cache of normal keys and values; bytes of tokens
    that were never stored are 0xff, which are NaN scales."""

    def __init__(self, pkg, lens, nqs, *, H, Hkv, D, bs, dt, seed=0, spare=2, pad_tokens=0):
        import torch
        g = np.random.default_rng(seed)
        self.R, self.H, self.Hkv, self.D, self.bs, self.dt = len(lens), H, Hkv, D, bs, dt
        self.lens, self.nqs = np.array(lens, np.int32), np.array(nqs, np.int32)
        pages = -(-self.lens // bs)
        self.nb, self.W = int(pages.sum()) + spare, max(1, int(pages.max())) + 1
        self.kv = cache_of(pkg, H=Hkv, D=D, bs=bs, nb=self.nb, W=self.W, R=self.R)
        ids = g.permutation(self.nb).astype(np.int32)
        self.table = np.full((self.R, self.W), -1, np.int32)
        self.table[np.arange(self.W)[None] < pages[:, None]] = ids[:pages.sum()]
        slot = np.concatenate([[int(self.table[r, t // bs]) * bs + t % bs for t in range(n)]
                               for r, n in enumerate(self.lens)] or [[]]).astype(np.int64)
        n = len(slot)
        self.cache = torch.full((self.nb, Hkv, bs // 16, granule(D)), 255, dtype=torch.uint8,
                                device="cuda")
        k, v, self.k, self.v = (torch.from_numpy(a).cuda() for a in (
            g.standard_normal((max(n, 1), Hkv, D)).astype(np.float32),
            (2 * g.standard_normal((max(n, 1), Hkv, D)) + 1).astype(np.float32),
            np.zeros((max(n, 1), Hkv, D), np.float32), np.zeros((max(n, 1), Hkv, D), np.float32)))
        if n:
            ts = torch.from_numpy(slot).cuda()
            self.kv.append(self.cache.data_ptr(), k.data_ptr(), v.data_ptr(), 0, n, ts.data_ptr(),
                           stream(), k_out_ptr=self.k.data_ptr(), v_out_ptr=self.v.data_ptr())
        self.first = np.concatenate([[0], np.cumsum(self.lens)])
        self.qo = np.concatenate([[0], np.cumsum(self.nqs)]).astype(np.int32)
        self.N = int(self.qo[-1]) + pad_tokens
        self.q = torch.from_numpy(g.standard_normal((self.N, H, D)).astype(np.float32)).cuda()
        self.q = self.q.to(torch_dtype(dt))

    def run(self, window=0, scale=None, q=None, lse=True, kv_len=None, table=None):
        import torch
        q = self.q if q is None else q
        out = torch.full((self.N, self.H, self.D), -7, dtype=q.dtype, device="cuda")
        ls = torch.full((self.N, self.H), -7, dtype=torch.float32, device="cuda")
        d = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        t, n, o = d(self.table if table is None else table), d(
            self.lens if kv_len is None else kv_len), d(self.qo)
        self.kv.attention(self.cache.data_ptr(), q.data_ptr(), out.data_ptr(), self.dt, self.N,
                          self.H, t.data_ptr(), n.data_ptr(), o.data_ptr(), self.R, stream(),
                          window=window, scale=scale, q_strides=q.stride()[:2],
                          lse_ptr=ls.data_ptr() if lse else 0)
        torch.cuda.synchronize()
        return out, ls

    def check(self, out, ls, window=0, scale=None, hidden=()):
        """`hidden`: (request, page index) pairs that lie outside the pool."""
        scale = self.D ** -0.5 if scale is None else scale
        o = out.double().cpu().numpy()
        ls = ls.double().cpu().numpy()
        q = self.q.double().cpu().numpy()
        kd, vd = self.k.double().cpu().numpy(), self.v.double().cpu().numpy()
        G = self.H // self.Hkv
        for r in range(self.R):
            n = int(self.lens[r])
            rows = slice(self.first[r], self.first[r + 1])
            for i in range(self.nqs[r]):
                pos = n - int(self.nqs[r]) + i
                t = np.arange(n)
                see = (t <= pos) & ((t > pos - window) if window else True)
                for rr, b in hidden:
                    if rr == r:
                        see &= t // self.bs != b
                row = self.qo[r] + i
                if not see.any():
                    assert (o[row] == 0).all() and np.isneginf(ls[row]).all(), (r, i)
                    continue
                k, v = kd[rows][see], vd[rows][see]
                for h in range(self.H):
                    kk, vv, qq = k[:, h // G], v[:, h // G], q[row, h]
                    x = scale * kk @ qq
                    p = np.exp(x - x.max())
                    want = p @ vv / p.sum()
                    S = (abs(scale) * np.abs(kk) @ np.abs(qq)).max()
                    e = (self.D + 16) * 2.0 ** -23 * S
                    vmax = np.abs(vv).max()
                    tol = vmax * (2 * e + (len(kk) + 16) * 2.0 ** -23)
                    if self.dt:
                        tol += 2.0 ** -11 * vmax
                    tol = tol + 2.0 ** -BITS[self.dt] * np.abs(want)
                    err = np.abs(o[row, h] - want)
                    assert (err <= tol).all(), (r, i, h, (err / tol).max())
                    le = abs(ls[row, h] - (x.max() + math.log(p.sum())))
                    assert le <= e + (len(kk) + 16) * 2.0 ** -23 + 2.0 ** -22 * abs(ls[row, h]), (r, i, h)
        assert (o[self.qo[-1]:] == -7).all() and (ls[self.qo[-1]:] == -7).all()


DTYPES = pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (6, 2), (8, 1), (12, 1), (40, 2)])
def test_attention_heads_and_lengths(H, Hkv, D, dt):
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 64, 100, 257]
    b = Batch(load_pkg(), lens, [1] * len(lens), H=H, Hkv=Hkv, D=D, bs=16, dt=dt, pad_tokens=2)
    b.check(*b.run())


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("bs", [16, 48, 128])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 100])
def test_attention_many_queries_and_windows(window, bs, dt):
    # Queries of one request: none, one, as many as keys, more than keys (the
    # first ones then see nothing).
    lens, nqs = [40, 0, 3, 65, 130, 7, 200], [3, 2, 1, 65, 0, 9, 17]
    b = Batch(load_pkg(), lens, nqs, H=4, Hkv=2, D=64, bs=bs, dt=dt, seed=bs)
    b.check(*b.run(window=window), window=window)


@pytest.mark.gpu
@DTYPES
def test_attention_one_long_and_many_short(dt):
    lens = [5000] + [3, 40, 1] * 6
    b = Batch(load_pkg(), lens, [1] * len(lens), H=8, Hkv=2, D=128, bs=32, dt=dt, seed=9)
    out, ls = b.run()
    b.check(out, ls)
    again, ls2 = b.run()       # the same bits every time
    assert (out == again).all() and (ls == ls2).all()


@pytest.mark.gpu
@DTYPES
def test_attention_strided_and_scaled_queries(dt):
    import torch
    b = Batch(load_pkg(), [20, 70], [2, 1], H=4, Hkv=2, D=64, bs=16, dt=dt)
    wide = torch.zeros(b.N, b.H + 3, b.D + 1, dtype=b.q.dtype, device="cuda")
    wide[:, 2:2 + b.H, 1:] = b.q
    out, ls = b.run(scale=0.3, q=wide[:, 2:2 + b.H, 1:])
    b.check(out, ls, scale=0.3)
    plain, _ = b.run(scale=0.3, lse=False)
    assert torch.equal(plain, out)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-4, 3e4])
def test_attention_large_and_small_queries(size):
    """Queries far from unit size, with scores of ordinary size (fp32)."""
    b = Batch(load_pkg(), [90], [1], H=2, Hkv=1, D=128, bs=16, dt=0)
    b.q.mul_(size)
    b.check(*b.run(scale=0.1 / size), scale=0.1 / size)


@pytest.mark.gpu
def test_attention_large_scores():
    """Scores of several hundred: the softmax is nearly one key, and its
    exponentials must not overflow."""
    b = Batch(load_pkg(), [300], [2], H=2, Hkv=2, D=64, bs=16, dt=0)
    b.check(*b.run(scale=20.0), scale=20.0)
    b.check(*b.run(scale=-3.0), scale=-3.0)


@pytest.mark.gpu
@DTYPES
def test_attention_pages_outside_the_pool_and_short_lengths(dt):
    b = Batch(load_pkg(), [64, 64, 40], [1, 1, 1], H=2, Hkv=1, D=64, bs=16, dt=dt)
    table = b.table.copy()
    table[0, 1], table[1, :], table[2, 0] = b.nb, -1, -2 ** 31
    out, ls = b.run(table=table)
    b.check(out, ls, hidden=[(0, 1), (2, 0)] + [(1, i) for i in range(4)])
    # A length beyond the table is cut to it; a negative one sees nothing.
    W = b.W
    lens = np.array([2 ** 31 - 1, -5, 40], np.int32)
    out, ls = b.run(kv_len=lens)
    assert (out[1] == 0).all() and (ls[1] == -math.inf).all()
    full = Batch(load_pkg(), [64, 64, 40], [1, 1, 1], H=2, Hkv=1, D=64, bs=16, dt=dt)
    assert W == full.W and (out[2] == full.run()[0][2]).all()


@pytest.mark.gpu
def test_attention_nan_stays_in_its_row():
    """A NaN that a visible key holds makes its head's rows NaN; others do not change."""
    import torch
    b = Batch(load_pkg(), [50, 50], [1, 1], H=4, Hkv=2, D=64, bs=16, dt=0)
    clean, _ = b.run()
    k = torch.full((1, 2, 64), float("nan"), device="cuda")
    slot = torch.tensor([int(b.table[1, 2]) * 16 + 3], device="cuda")
    v = torch.zeros_like(k)
    b.kv.append(b.cache.data_ptr(), k.data_ptr(), v.data_ptr(), 0, 1, slot.data_ptr(), stream())
    out, _ = b.run()
    assert torch.equal(out[0], clean[0]) and torch.isnan(out[1]).all()
    masked, _ = b.run(kv_len=np.array([50, 35], np.int32))   # the NaN's token is not visible now
    assert not torch.isnan(masked).any()


@pytest.mark.gpu
def test_attention_and_append_past_4_gib():
    """Pages beyond 2^32 bytes of the cache."""
    import torch
    pkg = load_pkg()
    D, H, bs = 128, 8, 64
    nb = (5 << 30) // (H * bs // 16 * granule(D))
    with cache_of(pkg, H=H, D=D, bs=bs, nb=nb, W=2, R=1) as kv:
        assert kv.cache_bytes() > 2 ** 32
        cache = torch.empty(kv.cache_bytes(), dtype=torch.uint8, device="cuda")
        small = Batch(pkg, [100], [1], H=16, Hkv=H, D=D, bs=bs, dt=0)
        want, _ = small.run()
        pages = np.array([[nb - 1, nb - 3]], np.int32)
        gran = small.cache.view(small.nb, -1)
        dst = cache.view(nb, -1)
        for i in range(2):
            dst[int(pages[0, i])] = gran[int(small.table[0, i])]
        out = torch.zeros_like(want)
        t, n, o = (torch.from_numpy(a).cuda() for a in (pages, small.lens, small.qo))
        kv.attention(cache.data_ptr(), small.q.data_ptr(), out.data_ptr(), 0, 1, 16, t.data_ptr(),
                     n.data_ptr(), o.data_ptr(), 1, stream())
        assert torch.equal(out, want)
        one = torch.randn(1, H, D, device="cuda")
        slot = torch.tensor([(nb - 1) * bs + 40], device="cuda")
        kv.append(cache.data_ptr(), one.data_ptr(), one.data_ptr(), 0, 1, slot.data_ptr(),
                  stream())
        got = read_cache(dst[nb - 1].cpu().numpy().reshape(1, H, bs // 16, -1), 0, 3, 40, D)
        assert np.abs(got[0] - one[0, 3].double().cpu().numpy()).max() < 0.3


@pytest.mark.gpu
def test_another_stream():
    """Work is enqueued on the stream it is given, after what runs there."""
    import torch
    b = Batch(load_pkg(), [200], [1], H=4, Hkv=2, D=64, bs=16, dt=0)
    want, _ = b.run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    q = torch.zeros_like(b.q)
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        q.copy_(b.q)
        out, _ = b.run(q=q)
    s.synchronize()
    assert torch.equal(out, want)


# --------------------------------------------------------------- refusals
@pytest.mark.parametrize("field,value,code", [
    ("num_kv_heads", 0, -1), ("num_kv_heads", 257, -1), ("head_dim", 96, -2),
    ("block_tokens", 8, -1), ("block_tokens", 24, -1), ("block_tokens", 1040, -1),
    ("num_blocks", 0, -1), ("table_width", 0, -1), ("table_width", 2 ** 28, -1),
    ("max_requests", 0, -1), ("max_requests", 8193, -1), ("device", -1, -1),
])
def test_create_refuses(field, value, code):
    pkg = load_pkg()
    kw = dict(num_kv_heads=2, head_dim=64, block_tokens=16, num_blocks=4, table_width=2,
              max_requests=2, device=0)
    kw[field] = value
    with pytest.raises(pkg.MoeError) as e:
        pkg.Kv4Cache(**kw)
    assert e.value.code == code


def test_null_handles():
    pkg = load_pkg()
    L = pkg.load_library()
    z = [None] * 3
    assert L.moe_kv4_create(None, None) == -1
    assert L.moe_kv4_cache_bytes(None) == 0 and L.moe_kv4_device_bytes(None) == 0
    L.moe_kv4_destroy(None)
    L.moe_kv4_config_init(None)
    assert L.moe_kv4_plan_device(None, *z[:2], 1, *z, *z, None, 1, *z[:2]) == -1
    assert L.moe_kv4_append_device(None, *z, 0, 1, 0, 0, 0, 0, *z, None) == -1
    assert L.moe_kv4_attention_device(None, *z[:2], 0, 1, 1, 0, 0, *z, 1, 1.0, 0, *z) == -1
    assert b"null handle" in L.moe_last_error()


@pytest.mark.gpu
def test_calls_refuse():
    pkg = load_pkg()
    with cache_of(pkg, R=2) as kv:
        def bad(f, *a, **k):
            with pytest.raises(pkg.MoeError) as e:
                f(*a, **k)
            return e.value.code
        p = 4096   # an address that is never touched: every call is refused on the host
        plan = lambda R=1, cap=1, out=p + 64, tab=p: kv.plan(  # noqa: E731
            p, p, R, p, p, tab, p, p, p, p, cap, out)
        assert bad(plan, R=0) == bad(plan, R=3) == bad(plan, cap=-1) == -1
        assert bad(plan, out=p) == bad(plan, tab=0) == -1
        with pytest.raises(pkg.MoeError, match="kv_len"):
            kv.plan(p, p + 64, 1, p, p, p, p, p, p, p, 1, p + 64)
        app = lambda c=p, k=p, dt=0, n=1, slot=p, out=0: kv.append(  # noqa: E731
            c, k, p, dt, n, slot, k_out_ptr=out)
        for kw in (dict(c=0), dict(c=p + 8), dict(k=0), dict(k=p + 2), dict(dt=3), dict(n=-1),
                   dict(slot=0), dict(slot=p + 4), dict(out=p + 4)):
            assert bad(app, **kw) == -1, kw
        att = lambda c=p, q=p, o=p, dt=0, n=1, H=2, R=1, **k: kv.attention(  # noqa: E731
            c, q, o, dt, n, H, p, p, p, R, **k)
        for kw in (dict(c=0), dict(c=p + 4), dict(q=p + 1), dict(o=p + 8), dict(dt=-1),
                   dict(n=-1), dict(H=3), dict(H=0), dict(H=2 * 65), dict(R=0), dict(R=3),
                   dict(window=-1), dict(scale=math.nan), dict(scale=math.inf)):
            assert bad(att, **kw) == -1, kw
        assert bad(att, n=2 ** 31 - 1) == -2
        # Nothing to do is not an error.
        app(n=0, c=0)
        att(n=0, q=0)
