"""Attention over the 4-bit cache where the values' size, or how they share the
probability, is far from ordinary: small and large values, a first key that
takes nearly all of it and holds next to nothing, a large value that nobody
looks at, groups of 64 dims of very different size.

Bound, on the 2-norm of a call's error.  With R_t,d = v_t,d - min of the value's
group (scale times code) the kernel's rounded operands are p_t R_t,d, so errors
of relative size u in them, whatever their signs, leave at most about
  u n,  n = || (sum_t (p_t R_t,d)^2)^(1/2) ||  over all outputs
where they are independent.  u = 2^-11 for the probabilities of 16-bit types (11
significant bits).  A score x carries the 22 bits of its operands, its sum's
fp32 roundings and its exponential's: at most about (|x| + 8) 2^-22, below 2^-17
for the scores here (|x| <= 24), on p (R + |v|); fp32 has that alone.  The
output's own rounding adds 2^-bits of it, and 2^-25 an element where float16
runs into its smallest step.
"""
import numpy as np
import pytest

from conftest import load_pkg
from test_kv4 import BITS, Batch, stream

DTYPES = pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])


def refill(b, k, v):
    """The batch's cache with these keys and values [tokens][Hkv][D] instead."""
    import torch
    slot = np.concatenate([[int(b.table[r, t // b.bs]) * b.bs + t % b.bs for t in range(n)]
                           for r, n in enumerate(b.lens)]).astype(np.int64)
    ts = torch.from_numpy(slot).cuda()
    k, v = (torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda() for a in (k, v))
    b.kv.append(b.cache.data_ptr(), k.data_ptr(), v.data_ptr(), 0, len(slot), ts.data_ptr(),
                stream(), k_out_ptr=b.k.data_ptr(), v_out_ptr=b.v.data_ptr())


def exact(b, window=0):
    """(out, lse, n, n with |v| too) in 64 bits, rows of no request left out."""
    import torch
    G = b.H // b.Hkv
    outs, lses, noise, all_noise = [], [], [], []
    for r in range(b.R):
        rows = slice(int(b.first[r]), int(b.first[r + 1]))
        k, v = b.k[rows].double(), b.v[rows].double()
        lo = v.unflatten(-1, (-1, 64)).amin(-1, keepdim=True)
        R = (v.unflatten(-1, (-1, 64)) - lo).flatten(-2)
        k, v, R = (a.repeat_interleave(G, 1) for a in (k, v, R))
        q = b.q[int(b.qo[r]):int(b.qo[r + 1])].double()
        x = torch.einsum("qhd,thd->qht", q, k) * b.D ** -0.5
        n, nq = int(b.lens[r]), int(b.nqs[r])
        pos = n - nq + torch.arange(nq, device="cuda")[:, None, None]
        t = torch.arange(n, device="cuda")
        hide = (t > pos) | ((t <= pos - window) if window else torch.zeros_like(t, dtype=torch.bool))
        x = x.masked_fill(hide, -np.inf)
        p = torch.softmax(x, -1)
        outs.append(torch.einsum("qht,thd->qhd", p, v))
        lses.append(torch.logsumexp(x, -1))
        noise.append(torch.einsum("qht,thd->qhd", p ** 2, R ** 2))
        all_noise.append(torch.einsum("qht,thd->qhd", p ** 2, (R + v.abs()) ** 2))
    out, lse, n, na = (torch.cat(a) for a in (outs, lses, noise, all_noise))
    return out, lse, n.sum().sqrt().item(), na.sum().sqrt().item()


def check(b, window=0):
    out, ls = b.run(window=window)
    want, lse, n, na = exact(b, window)
    err = (out.double()[:len(want)] - want).norm().item()
    tol = 2.0 ** -17 * na + 2.0 ** -BITS[b.dt] * want.norm().item()
    if b.dt:
        tol += 2.0 ** -11 * n
    if b.dt == 2:
        tol += 2.0 ** -25 * want.numel() ** 0.5
    assert err <= tol, (err / want.norm().item(), tol / want.norm().item())
    assert (ls.double()[:len(lse)] - lse).abs().max().item() <= 24 * 2.0 ** -17
    again, _ = b.run(window=window)
    assert (again == out).all()


def keys_and_values(b, seed=3):
    g = np.random.default_rng(seed)
    n = int(b.lens.sum())
    return (g.standard_normal((n, b.Hkv, b.D)), g.standard_normal((n, b.Hkv, b.D)))


def batch(dt, D, H=4, Hkv=1, lens=(2048, 300, 17), nqs=(1, 1, 1), bs=16):
    return Batch(load_pkg(), list(lens), list(nqs), H=H, Hkv=Hkv, D=D, bs=bs, dt=dt, seed=D + H)


def sink(b, k, gap, token=0):
    """Makes every query of every request see one of its keys `gap` above the others."""
    import torch
    g = np.random.default_rng(9)
    u = g.standard_normal(b.D)
    u *= b.D ** 0.5 / np.linalg.norm(u)
    k -= (k @ u)[..., None] * u / (u @ u) * 0.9      # the others' scores near 0
    b.q.copy_(torch.from_numpy(u + 0.05 * g.standard_normal((b.N, b.H, b.D))).to(b.q.dtype))
    for r in range(b.R):
        k[b.first[r] + token] = u * gap / b.D ** 0.5


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spread", [1.0, 2.5])
@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-2, 1.0, 1e4])
def test_values_of_any_size(size, spread, D, dt):
    b = batch(dt, D)
    k, v = keys_and_values(b)
    refill(b, k * spread, v * size)
    check(b)


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("H,Hkv,nqs,window", [(16, 1, (3, 2, 5), 0), (2, 2, (9, 1, 2), 100)])
def test_small_values_many_rows(H, Hkv, nqs, window, dt):
    b = batch(dt, 128, H=H, Hkv=Hkv, nqs=nqs, bs=48)
    k, v = keys_and_values(b)
    refill(b, k, v * 1e-4)
    check(b, window)


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("token", [0, 13])
@pytest.mark.parametrize("size", [0.02, 1.0])
def test_a_key_that_takes_all_and_holds_nothing(size, token, D, dt):
    b = batch(dt, D)
    k, v = keys_and_values(b)
    sink(b, k, 12.0, token)
    for r in range(b.R):
        v[b.first[r] + token] *= 1e-4
    refill(b, k, v * size)
    check(b)


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("token", [0, 13])
def test_a_large_value_that_nobody_looks_at(token, dt):
    b = batch(dt, 128)
    k, v = keys_and_values(b)
    sink(b, k, -23.0, token)
    v *= 0.01
    for r in range(b.R):
        v[b.first[r] + token] *= 1e6
    refill(b, k, v)
    check(b)


@pytest.mark.gpu
@DTYPES
def test_groups_of_different_size(dt):
    b = batch(dt, 128)
    k, v = keys_and_values(b)
    v[..., 64:] *= 1e-4
    refill(b, k, v)
    check(b)
    out, _ = b.run()
    want, *_ = exact(b)
    e = (out.double() - want)[..., 64:].norm() / want[..., 64:].norm()
    # The small group by itself: n is at most 3.5 times its result here (as a
    # normal distribution over 16 steps gives), fp32's sum half of that again.
    small = 2.0 ** -17 * 6 + 2.0 ** -BITS[dt] + (2.0 ** -11 * 3.5 if dt else 0)
    if dt == 2:
        small += 2.0 ** -25 * (want[..., 64:].numel() ** 0.5 / want[..., 64:].norm().item())
    assert e.item() <= small


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,nq", [(1, 1), (2, 3)])
def test_fp32_sums_of_evenly_shared_values(H, nq, D):
    """Short queries give thousands of keys nearly the same probability, so that
    an fp32 result is a mean of their values, far smaller than each, and its
    sum's roundings are most of what is left.  Terms counted from the middle of
    the codes, p s (c - 8), have both signs: a warp's sum of 16 j of them is
    about 12 sqrt(j) s p, and its steps' losses, 2^-24 of that each and of either
    sign, are together 2^-24 * 12 s p L / 64 / sqrt(2); four warps, p = 1 / L:
    0.27 * 2^-24 s.  Eight times that, and 2^-21 on each p v for the scores (below
    2) and their exponentials."""
    import torch
    # So many that a block has a whole item or more: runs of 64 steps a warp.
    b = batch(0, D, H=H * 8, Hkv=8, lens=(4096,) * 24, nqs=(nq,) * 24, bs=64)
    k, v = keys_and_values(b)
    refill(b, k, v)
    b.q.mul_(0.3)
    out, _ = b.run()
    want, *_ = exact(b)
    scale = []
    for r in range(b.R):
        x = b.v[int(b.first[r]):int(b.first[r + 1])].double().unflatten(-1, (-1, 64))
        s = (x.amax(-1) - x.amin(-1)).square().mean((0, 1)).sqrt() / 15      # a group's rms step
        scale.append(s.repeat_interleave(64).expand(nq, b.H, D))
    # || (sum (p v)^2)^(1/2) || is the result's own norm, its values being independent.
    tol = 2.0 ** -23 * torch.cat(scale).norm().item() + 2.0 ** -21 * want.norm().item()
    err = (out.double() - want).norm().item()
    assert err <= tol, (err / want.norm().item(), tol / want.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,nq", [(4, 1, 1), (2, 2, 3), (6, 1, 1), (8, 1, 1), (4, 1, 2), (16, 1, 1), (8, 2, 4)])
@pytest.mark.parametrize("dt", [1, 2], ids=["bf16", "f16"])
def test_16_bit_results_are_as_good_as_their_type(H, Hkv, nq, dt):
    """A result rounded once from an exact one is off by a relative error that is
    spread evenly, 2^-bits at most.  What the probabilities' rounding adds is
    nothing to speak of with two float16 numbers each (up to four rows a
    key/value head); with one, an error spread alike on each p s (c - 7.5), which
    is the value but for the middle of its group's range: as much as a float16
    result's own, 1.5 times that with room for the middle.  So the total stays
    below 1.5 times the own rounding's norm, and below sqrt(1 + 1.5^2) times for
    float16 results with one number."""
    b = batch(dt, 128, H=H, Hkv=Hkv, lens=(2048, 700, 1500), nqs=(nq,) * 3, bs=32)
    k, v = keys_and_values(b)
    refill(b, k, v)
    out, _ = b.run()
    want, *_ = exact(b)
    once = (want.to(b.q.dtype).double() - want).norm().item()
    most = 1.5 if dt == 1 or H // Hkv * nq <= 4 else (1 + 1.5 ** 2) ** 0.5
    err = (out.double() - want).norm().item()
    assert err <= most * once, (err / once, most)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H", [4, 8, 24])
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["f32", "bf16", "f16"])
def test_lse_of_one_key(dt, H, D):
    """The log of the sum is fp32 whatever the type, and of one key it is the
    score.  A score of unit size is a sum of D / 16 steps whose partial sums are of
    that size too, each off by an error spread over 2^-23 of it: together sqrt(8 /
    3) 2^-23 at D = 128.  Twice that and more, with the exponential's and the
    logarithm's: 2^-21 of the norm."""
    lens = (1,) * 96
    b = batch(dt, D, H=H, Hkv=4, lens=lens, nqs=lens)
    k, v = keys_and_values(b)
    refill(b, k, v)
    _, ls = b.run()
    _, want, *_ = exact(b)
    err = (ls.double() - want).norm().item()
    assert err <= 2.0 ** -21 * want.norm().item(), err / want.norm().item()
