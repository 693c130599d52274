"""The operators of a 4-bit decode step, as measured cases.

Serving a Mixture-of-Experts decoder in 4 bits takes, per step: block tables
and slot maps for the requests' new tokens (``plan``), the new keys and values
quantised into a paged 4-bit cache (``append``), attention over that cache
(``attention``), matrix-vector products with 4-bit group-scaled weights
(``matvec``) and the routed experts on such weights (``experts``).

``run`` computes each in plain torch where ``own`` is false, and through the
package's public calls where it is true.

Cache layout (one uint8 buffer, pages of ``block`` tokens, a multiple of 16):
[num_blocks][kv heads][block / 16][granule], a granule holding 16 tokens of
one head as
  K codes   [16 tokens][4 j][D/64 groups][2 h][4 bytes], the byte pair b of
            (j, g, h) holding dims 64 g + 16 j + 8 h + 2 b (low nibble), + 1
  V codes   [D/64 p][8 n][4 j][256/D v][D/64 groups][4 bytes], token
            8 (u // 2) + 2 j + u % 2 for u = p * (256 / D) + v, byte b of
            group g holding dims 64 g + 8 n + 2 b (low nibble), + 1
  K params  [16 tokens][D/64 groups] of (scale, minimum), float16
  V params  the same
and a code c of a group standing for scale * c + minimum.
"""
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _pkg():
    name = "moe_b200"
    if name not in sys.modules:
        init = (Path(__file__).resolve().parents[1] / "accelerating-moe-inference_b200"
                / "__init__.py")
        spec = importlib.util.spec_from_file_location(name, init)
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One decode step of the repository's toy decoder: 16 requests, one
        # new token each, 640 positions (prompt 512 + 128 tokens).
        dict(name="plan_decode", op="plan", R=16, block=16, W=40, longest=512, new=1,
             release=0.0, pool=1.0),
        # A mixed step of a busy server: 512 requests in pages of 32 tokens,
        # prompts of up to 1024 tokens among decodes, some requests ending.
        dict(name="plan_mixed", op="plan", R=512, block=32, W=1024, longest=16384, new=1024,
             release=0.05, pool=1.0),
        # The toy decoder's decode step: 16 requests, 16 heads of 128, fp32
        # (the framework's activations).
        dict(name="append_decode", op="append", N=16, Hkv=16, D=128, block=16, dtype="f32",
             fused=False),
        # A prefill of 16384 tokens, keys and values taken as slices of the
        # fused projection's output.
        dict(name="append_prefill", op="append", N=16384, Hkv=8, D=128, block=32, dtype="bf16",
             fused=True),
        # One sequence of the toy decoder near its end: latency.
        dict(name="attend_one", op="attention", R=1, H=16, Hkv=16, D=128, block=16, longest=640,
             shortest=640, nq=1, window=0, dtype="f32"),
        # 64 ragged requests, grouped heads: an ordinary decode batch.
        dict(name="attend_batch", op="attention", R=64, H=32, Hkv=8, D=128, block=32,
             longest=8192, shortest=100, nq=1, window=0, dtype="bf16"),
        # Eight long documents: the cache read is everything.
        dict(name="attend_long", op="attention", R=8, H=32, Hkv=8, D=128, block=64,
             longest=131072, shortest=16384, nq=1, window=0, dtype="f16"),
        # A projection of the toy decoder (d 2048), one token, fp32: latency.
        dict(name="matvec_proj", op="matvec", rows=1, N=2048, K=2048, group=128, zeros=False,
             dtype="f32"),
        # Its output head (vocab 32000) for a batch of 16.
        dict(name="matvec_head", op="matvec", rows=16, N=32000, K=2048, group=64, zeros=True,
             dtype="bf16"),
        # A down projection of the Mixtral-shaped layer, four tokens.
        dict(name="matvec_down", op="matvec", rows=4, N=4096, K=14336, group=128, zeros=True,
             dtype="f16"),
        # The reference's layer (d 4096, d_ff 448, 16 experts, top-2), one token.
        dict(name="experts_one", op="experts", T=1, d=4096, ff=448, E=16, k=2, group=128,
             zeros=True, dtype="f32"),
        # The Mixtral-shaped layer, a decode batch of 8.
        dict(name="experts_batch", op="experts", T=8, d=4096, ff=14336, E=8, k=2, group=128,
             zeros=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "matvec", "matvec", "experts"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "plan":
        block = rng.choice([16, 32, 64])
        longest = _log(rng, 64, 16384)
        new = min(longest, _log(rng, 1, 1024))
        return dict(op=op, R=_log(rng, 1, 512), block=block, W=-(-(longest + new) // block) + 1,
                    longest=longest, new=new, release=rng.choice([0.0, 0.05, 0.3]),
                    pool=rng.choice([1.0, 1.0, 0.7]))
    if op == "append":
        D = rng.choice([64, 128])
        Hkv = rng.randint(1, 16)
        return dict(op=op, N=_log(rng, 1, 16384 * 8 * 128 // (16 * D)), Hkv=Hkv, D=D,
                    block=rng.choice([16, 32, 64]), dtype=dtype, fused=rng.random() < 0.5)
    if op == "attention":
        D = rng.choice([64, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        nq = rng.choice([1, 1, 1, 2, 4])
        R = _log(rng, 1, 64)
        longest = max(nq, _log(rng, 1, min(65536, 524288 // R)))
        return dict(op=op, R=R, H=Hkv * rng.choice([1, 2, 4, 6, 8]), Hkv=Hkv, D=D,
                    block=rng.choice([16, 32, 64]), longest=longest,
                    shortest=max(nq, longest // 16), nq=nq,
                    window=rng.choice([0, 0, 0, max(1, longest // 3)]), dtype=dtype)
    if op == "matvec":
        return dict(op=op, rows=rng.choice([1, 1, 2, 3, 4, 5, 8, 11, 16]),
                    N=_log(rng, 500, 32000), K=32 * _log(rng, 16, 128),
                    group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, dtype=dtype)
    k = rng.choice([1, 2, 2, 4])
    return dict(op=op, T=rng.choice([1, 2, 3, 5, 8]), d=128 * _log(rng, 4, 32),
                ff=32 * _log(rng, 6, 448), E=rng.choice([4, 8]), k=k,
                group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _codes(shape, g):
    """Packed 4-bit codes of the bell shape that quantised weights, keys and
    values have (standard deviation 2.9 of 16 levels)."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for a in range(0, flat.numel(), step):
        part = flat[a:a + step]
        v = torch.randn(2, part.numel(), generator=g, device="cuda")
        v = v.mul_(2.9).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
        part.copy_(v[0] | (v[1] << 4))
    return out


def _granule(D):
    return 16 * D + 2 * 16 * (D // 64) * 4


def _new_tokens(c):
    """Expected new tokens of a step: one in four live requests brings a prompt."""
    live = c["R"] * (1 - c["release"])
    return live * (1 if c["new"] == 1 else 0.75 + 0.25 * (c["new"] + 1) / 2)


def _prepare_plan(c, seed):
    g = _gen(seed)
    R, bs, W = c["R"], c["block"], c["W"]
    rand = lambda lo, hi: torch.randint(lo, hi, (R,), generator=g, device="cuda")  # noqa: E731
    if c["new"] == 1:
        cached = torch.full((R,), c["longest"], device="cuda") + rand(0, bs)
        new = torch.ones(R, dtype=torch.int64, device="cuda")
    else:
        # Three in four requests decode one token, the others bring a prompt.
        cached = rand(0, c["longest"] + 1)
        new = torch.where(rand(0, 4) > 0, torch.ones_like(cached), rand(1, c["new"] + 1))
    gone = torch.rand(R, generator=g, device="cuda") < c["release"]
    cached = cached.clamp_(max=W * bs)
    new = torch.minimum(new, W * bs - cached)
    new = torch.where(gone, -torch.ones_like(new), new)
    used = (cached + bs - 1) // bs
    need = torch.where(new > 0, (cached + new.clamp(min=0) + bs - 1) // bs - used, 0)
    # A pool that could hold every request at its longest; less than the step
    # needs is left free where the case says that it runs dry.
    nb = R * W
    free = nb - int(used.sum())
    free = free if c["pool"] >= 1 else min(free, int(int(need.sum()) * c["pool"]))
    perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    # The requests' blocks, then the free ones in a ring that starts anywhere.
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(W, device="cuda")
    owned = col[None, :] < used[:, None]
    table[owned] = perm[:int(used.sum())]
    head = int(torch.randint(0, nb, (1,), generator=g, device="cuda"))
    ring = torch.full((nb,), -1, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(free, device="cuda")) % nb] = perm[int(used.sum()):][:free]
    # A step of a fixed shape, a little larger than what the mix brings.
    cap = R if c["new"] == 1 else min(R * c["new"], int(1.1 * _new_tokens(c)) + 2 * c["new"])
    e = lambda n, t: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    return dict(cached=cached.to(torch.int32), new=new.to(torch.int32), table=table, ring=ring,
                state=torch.tensor([head, free], dtype=torch.int32, device="cuda"), cap=cap,
                nb=nb, kv_len=e(R, torch.int32), q_offset=e(R + 1, torch.int32),
                position=e(cap, torch.int32), slot=e(cap, torch.int64),
                state_out=e(2, torch.int32))


def _prepare_append(c, seed):
    g = _gen(seed)
    N, Hkv, D, bs = c["N"], c["Hkv"], c["D"], c["block"]
    nb = -(-N // bs) + 2
    if c["fused"]:
        # q, k and v side by side in one projection's output; as many query
        # heads as key heads.
        qkv = torch.randn(N, 3, Hkv, D, generator=g, device="cuda").to(DT[c["dtype"]])
        k, v = qkv[:, 1], qkv[:, 2]
    else:
        k = torch.randn(N, Hkv, D, generator=g, device="cuda").to(DT[c["dtype"]])
        v = torch.randn(N, Hkv, D, generator=g, device="cuda").to(DT[c["dtype"]])
    if N <= 64:  # decode: one token each at any place of its own page
        slot = (torch.randperm(nb * bs, generator=g, device="cuda")[:N]).to(torch.int64)
    else:        # a prompt's pages in any order, filled from the front
        page = torch.randperm(nb, generator=g, device="cuda")
        t = torch.arange(N, device="cuda")
        slot = page[t // bs] * bs + t % bs
    cache = torch.zeros(nb, Hkv, bs // 16, _granule(D), dtype=torch.uint8, device="cuda")
    return dict(k=k, v=v, slot=slot, cache=cache, nb=nb,
                k_out=torch.empty(N, Hkv, D, dtype=DT[c["dtype"]], device="cuda"),
                v_out=torch.empty(N, Hkv, D, dtype=DT[c["dtype"]], device="cuda"))


def _lengths(c, g):
    """Ragged lengths between shortest and longest, spread over their logarithm."""
    if c["R"] == 1:
        return torch.full((1,), c["longest"], dtype=torch.int32, device="cuda")
    lo, hi = math.log(c["shortest"]), math.log(c["longest"])
    u = torch.rand(c["R"], generator=g, device="cuda")
    # Evenly spaced and jittered, so that every draw of a case costs alike.
    u = (torch.arange(c["R"], device="cuda") + u) / c["R"]
    n = torch.exp(lo + (hi - lo) * u).round()
    n = n.clamp_(c["shortest"], c["longest"]).to(torch.int32)
    return n[torch.randperm(c["R"], generator=g, device="cuda")]


def _prepare_attention(c, seed):
    g = _gen(seed)
    R, H, Hkv, D, bs, nq = c["R"], c["H"], c["Hkv"], c["D"], c["block"], c["nq"]
    kv_len = _lengths(c, g)
    used = (kv_len.long() + bs - 1) // bs
    total = int(used.sum())
    nb, W = total + 3, int(used.max())
    G = D // 64
    cache = torch.empty(nb, Hkv, bs // 16, _granule(D), dtype=torch.uint8, device="cuda")
    cache[..., :16 * D] = _codes((nb, Hkv, bs // 16, 16 * D), g)
    # Keys and values of unit scale: 16 levels over about +-2.5.
    s = torch.rand(nb, Hkv, bs // 16, 32 * G, 2, generator=g, device="cuda")
    s = torch.stack([0.27 + 0.1 * s[..., 0], -2.7 + 0.8 * s[..., 1]], -1).to(torch.float16)
    cache[..., 16 * D:] = s.view(torch.uint8).flatten(-2)
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    owned = torch.arange(W, device="cuda")[None, :] < used[:, None]
    table[owned] = torch.randperm(nb, generator=g, device="cuda")[:total].to(torch.int32)
    q = torch.randn(R * nq, H, D, generator=g, device="cuda").to(DT[c["dtype"]])
    st = dict(cache=cache, table=table, kv_len=kv_len, q=q, nb=nb, W=W,
              q_offset=torch.arange(0, R * nq + 1, nq, dtype=torch.int32, device="cuda"),
              out=torch.empty_like(q), lse=torch.empty(R * nq, H, device="cuda"))
    return st


def _weights(E, N, K, group, zeros, g):
    gr = -(-K // group)
    s = (0.0069 * (0.8 + 0.4 * torch.rand(E, N, gr, generator=g, device="cuda")))
    z = None
    if zeros:
        z = torch.randint(6, 10, (E, N, gr), generator=g, device="cuda", dtype=torch.uint8)
    return dict(codes=_codes((E, N, K // 2), g), scales=s.to(torch.float16), zeros=z, E=E, N=N,
                K=K, group=group)


def _handle(w, gated):
    """The package's weight handle, which keeps its own layout of them."""
    return _pkg().W4Matrix.from_device_pointers(
        w["codes"].data_ptr(), w["scales"].data_ptr(),
        0 if w["zeros"] is None else w["zeros"].data_ptr(), matrices=w["E"], rows=w["N"],
        cols=w["K"], group=w["group"], gated=gated)


def _kv(c, nb, W=1):
    return _pkg().Kv4Cache(num_kv_heads=c.get("Hkv", 1), head_dim=c.get("D", 128),
                           block_tokens=c["block"], num_blocks=nb, table_width=W,
                           max_requests=c.get("R", 1))


def prepare(case, seed):
    c, op = case, case["op"]
    if op == "plan":
        st = _prepare_plan(c, seed)
    elif op == "append":
        st = _prepare_append(c, seed)
    elif op == "attention":
        st = _prepare_attention(c, seed)
    elif op == "matvec":
        g = _gen(seed)
        st = dict(w=_weights(1, c["N"], c["K"], c["group"], c["zeros"], g),
                  x=torch.randn(c["rows"], c["K"], generator=g, device="cuda").to(DT[c["dtype"]]),
                  y=torch.empty(c["rows"], c["N"], dtype=DT[c["dtype"]], device="cuda"))
    else:
        g = _gen(seed)
        T, d, ff, E, k = c["T"], c["d"], c["ff"], c["E"], c["k"]
        logits = torch.randn(T, E, generator=g, device="cuda")
        top = torch.topk(logits, k, dim=1)
        st = dict(gu=_weights(E, 2 * ff, d, c["group"], c["zeros"], g),
                  dn=_weights(E, d, ff, c["group"], c["zeros"], g),
                  x=torch.randn(T, d, generator=g, device="cuda").to(DT[c["dtype"]]),
                  idx=top.indices.to(torch.int32).contiguous(),
                  wt=torch.softmax(top.values, 1).contiguous(),
                  y=torch.empty(T, d, dtype=DT[c["dtype"]], device="cuda"))
    if own:
        if op in ("plan", "attention", "append"):
            st["kv"] = _kv(c, st["nb"], c.get("W") or st.get("W", 1))
        elif op == "matvec":
            st["h"] = _handle(st["w"], False)
        else:
            st["hgu"], st["hdn"] = _handle(st["gu"], True), _handle(st["dn"], False)
    st["case"] = c
    return st


# -------------------------------------------------------------- plain forms
def _plain_plan(s):
    c = s["case"]
    bs, W, nb, cap = c["block"], c["W"], s["nb"], s["cap"]
    cached, new = s["cached"].long(), s["new"].long()
    head, count = s["state"][0].long(), s["state"][1].long()
    grow = new.clamp(min=0)
    end = torch.cumsum(grow, 0)
    used = (cached + bs - 1) // bs
    fits = (new >= 0) & (cached >= 0) & (cached + grow <= W * bs) & ((new == 0) | (end <= cap))
    need = torch.where(fits, (cached + grow + bs - 1) // bs - used, 0)
    cum = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (cum <= count))
    first = cum - need
    need = torch.where(ok, need, 0)
    col = torch.arange(W, device="cuda")[None, :] - used[:, None]
    fresh = s["ring"][((head + first)[:, None] + col.clamp(min=0)) % nb]
    table = torch.where((col >= 0) & (col < need[:, None]), fresh, s["table"])
    s["table"].copy_(table)
    back = torch.where((new < 0) & (cached >= 0) & (cached <= W * bs), used, 0)
    bcum = torch.cumsum(back, 0)
    at = ((head + count) + (bcum - back)[:, None] + torch.arange(W, device="cuda")) % nb
    give = torch.arange(W, device="cuda")[None, :] < back[:, None]
    s["ring"][at[give]] = s["table"][give]
    q_offset = torch.cat([torch.zeros_like(end[:1]), end]).clamp(max=cap)
    t = torch.arange(cap, device="cuda")
    r = torch.searchsorted(q_offset[1:].contiguous(), t, right=True)
    inside = r < new.numel()
    r = r.clamp(max=new.numel() - 1)
    pos = cached[r] + t - q_offset[r]
    page = table[r, (pos // bs).clamp(0, W - 1)].long()
    good = inside & ok[r] & (page >= 0) & (page < nb)
    taken, given = need.sum(), back.sum()
    return dict(table=s["table"], ring=s["ring"],
                kv_len=torch.where(ok, cached + grow, 0).to(torch.int32),
                q_offset=q_offset.to(torch.int32),
                position=torch.where(inside, pos, -1).to(torch.int32),
                slot=torch.where(good, page * bs + pos % bs, -1),
                state=torch.stack([(head + taken) % nb, count - taken + given]).to(torch.int32))


def _plain_quantise(x):
    """[..., D] -> codes [..., D] (int32), (scale, minimum) [..., D/64, 2]
    float16 and the values these stand for, each step rounded to fp32."""
    x = x.float().clamp(-65504, 65504).unflatten(-1, (-1, 64))
    lo, hi = x.amin(-1), x.amax(-1)
    sc = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).half()
    mn = lo.half()
    s32, m32 = sc.float()[..., None], mn.float()[..., None]
    code = torch.where(s32 > 0, torch.round((x - m32) / s32).clamp(0, 15), 0)
    return code.flatten(-2).int(), torch.stack([sc, mn], -1), (s32 * code + m32).flatten(-2)


def _plain_append(s):
    c = s["case"]
    N, Hkv, D, bs = c["N"], c["Hkv"], c["D"], c["block"]
    G = D // 64
    kc, kp, kd = _plain_quantise(s["k"])
    vc, vp, vd = _plain_quantise(s["v"])
    pack = lambda x: (x[..., 0::2] | (x[..., 1::2] << 4)).to(torch.uint8)  # noqa: E731
    # [N][Hkv][G][4 j][2 h][4 b] -> [4 j][G][2 h][4 b]
    kb = pack(kc).view(N, Hkv, G, 4, 2, 4).permute(0, 1, 3, 2, 4, 5).reshape(N, Hkv, -1)
    # [N][Hkv][G][8 n][4 b] -> [8 n][G][4 b]
    vb = pack(vc).view(N, Hkv, G, 8, 4).permute(0, 1, 3, 2, 4).reshape(N, Hkv, 8, -1)
    page, off = s["slot"] // bs, s["slot"] % bs
    gr, t = off // 16, off % 16
    gran = s["cache"]
    kv = gran[..., :8 * D].unflatten(-1, (16, D // 2))
    kv[page, :, gr, t] = kb
    vv = gran[..., 8 * D:16 * D].unflatten(-1, (G, 8, 4, 4 // G, 4 * G))
    u = (t // 8) * 2 + t % 2
    vv[page, :, gr, u // (4 // G), :, (t % 8) // 2, u % (4 // G)] = vb
    pp = gran[..., 16 * D:].unflatten(-1, (2, 16, G * 4))
    pp[page, :, gr, 0, t] = kp.flatten(-2).contiguous().view(torch.uint8)
    pp[page, :, gr, 1, t] = vp.flatten(-2).contiguous().view(torch.uint8)
    return dict(k=kd.to(s["k"].dtype), v=vd.to(s["v"].dtype), cache=s["cache"])


def _unpack(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _plain_dequant(gran, D):
    """Granules [..., granule bytes] -> K and V [..., 16, D] in fp32."""
    G = D // 64
    kc = _unpack(gran[..., :8 * D].unflatten(-1, (16, 4, G, 2, 4)))          # ... 16 j g h 8
    kc = kc.transpose(-4, -3).flatten(-4).float()
    vc = _unpack(gran[..., 8 * D:16 * D].unflatten(-1, (G, 8, 4, 4 // G, G, 4)))
    n = vc.dim()
    lead = list(range(n - 6))
    p, nn, j, u, g, e = range(n - 6, n)
    # (p, u) = (half, s) -> token (half, j, s); dims (g, n, e)
    vc = vc.permute(*lead, p, u, j, g, nn, e).flatten(n - 6, n - 5).unflatten(n - 6, (2, 2))
    vc = vc.transpose(n - 5, n - 4).flatten(n - 6, n - 4).flatten(-3).float()
    par = gran[..., 16 * D:].contiguous().view(torch.float16).unflatten(-1, (2, 16, G, 2)).float()
    up = lambda x: x.repeat_interleave(64, -1)  # noqa: E731
    k = kc * up(par[..., 0, :, :, 0]) + up(par[..., 0, :, :, 1])
    v = vc * up(par[..., 1, :, :, 0]) + up(par[..., 1, :, :, 1])
    return k, v


def _plain_attention(s):
    c = s["case"]
    R, H, Hkv, D, bs, nq = c["R"], c["H"], c["Hkv"], c["D"], c["block"], c["nq"]
    W = s["W"]
    pages = s["cache"][s["table"].clamp(min=0).long()]               # R W Hkv gr B
    k, v = _plain_dequant(pages, D)                                  # R W Hkv gr 16 D
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(R, Hkv, W * bs, D)
    v = v.permute(0, 2, 1, 3, 4, 5).reshape(R, Hkv, W * bs, D)
    G = H // Hkv
    q = s["q"].float().view(R, nq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(R, Hkv, nq * G, D)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    pos = s["kv_len"].long()[:, None] - nq + torch.arange(nq, device="cuda")    # R nq
    t = torch.arange(W * bs, device="cuda")
    see = t <= pos[..., None]
    if c["window"]:
        see = see & (t > pos[..., None] - c["window"])
    see = see.repeat_interleave(G, 1)[:, None]                       # R 1 nq*G L
    x = torch.where(see, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    p = torch.where(see, torch.exp(x - m), 0.0)
    l = p.sum(-1, keepdim=True)
    o = torch.where(l > 0, torch.matmul(p, v) / l.clamp(min=1e-30), 0.0)
    lse = (m + torch.log(l)).squeeze(-1)
    back = lambda a: a.view(R, Hkv, nq, G, -1).transpose(1, 2).reshape(R * nq, H, -1)  # noqa: E731
    return dict(out=back(o).to(s["q"].dtype), lse=back(lse).squeeze(-1))


def _plain_w(w):
    v = _unpack(w["codes"]).to(torch.float32)
    z = 8.0 if w["zeros"] is None else w["zeros"].float().repeat_interleave(w["group"], -1)
    z = z if w["zeros"] is None else z[..., :w["K"]]
    return v.sub_(z).mul_(w["scales"].float().repeat_interleave(w["group"], -1)[..., :w["K"]])


def _plain_matvec(s):
    return torch.matmul(s["x"].float(), _plain_w(s["w"])[0].t()).to(s["x"].dtype)


def _plain_experts(s):
    c = s["case"]
    ff = c["ff"]
    gu = torch.matmul(s["x"].float(), _plain_w(s["gu"]).transpose(1, 2))     # E T 2ff
    gate, up = gu[..., :ff], gu[..., ff:]
    h = gate / (1 + torch.exp(-gate)) * up
    y = torch.matmul(h, _plain_w(s["dn"]).transpose(1, 2))                   # E T d
    t = torch.arange(c["T"], device="cuda")[:, None]
    return (y[s["idx"].long(), t] * s["wt"][..., None]).sum(1).to(s["x"].dtype)


# --------------------------------------------------------------------- run
def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        return dict(plan=_plain_plan, append=_plain_append, attention=_plain_attention,
                    matvec=_plain_matvec, experts=_plain_experts)[op](s)
    stream = torch.cuda.current_stream().cuda_stream
    if op == "plan":
        s["kv"].plan(s["cached"].data_ptr(), s["new"].data_ptr(), c["R"], s["ring"].data_ptr(),
                     s["state"].data_ptr(), s["table"].data_ptr(), s["kv_len"].data_ptr(),
                     s["q_offset"].data_ptr(), s["position"].data_ptr(), s["slot"].data_ptr(),
                     s["cap"], s["state_out"].data_ptr(), stream)
        return dict(table=s["table"], ring=s["ring"], kv_len=s["kv_len"], q_offset=s["q_offset"],
                    position=s["position"], slot=s["slot"], state=s["state_out"])
    dt = {"f32": 0, "bf16": 1, "f16": 2}[c["dtype"]]
    if op == "append":
        k, v = s["k"], s["v"]
        s["kv"].append(s["cache"].data_ptr(), k.data_ptr(), v.data_ptr(), dt, c["N"],
                       s["slot"].data_ptr(), stream, k_strides=k.stride()[:2],
                       v_strides=v.stride()[:2], k_out_ptr=s["k_out"].data_ptr(),
                       v_out_ptr=s["v_out"].data_ptr())
        return dict(k=s["k_out"], v=s["v_out"], cache=s["cache"])
    if op == "attention":
        s["kv"].attention(s["cache"].data_ptr(), s["q"].data_ptr(), s["out"].data_ptr(), dt,
                          c["R"] * c["nq"], c["H"], s["table"].data_ptr(),
                          s["kv_len"].data_ptr(), s["q_offset"].data_ptr(), c["R"], stream,
                          window=c["window"], lse_ptr=s["lse"].data_ptr())
        return dict(out=s["out"], lse=s["lse"])
    if op == "matvec":
        s["h"].matvec(s["x"].data_ptr(), s["y"].data_ptr(), c["rows"], dt, stream)
        return s["y"]
    _pkg().w4_experts(s["hgu"], s["hdn"], s["x"].data_ptr(), s["idx"].data_ptr(),
                      s["wt"].data_ptr(), s["y"].data_ptr(), c["T"], c["k"], dt, stream)
    return s["y"]


# -------------------------------------------------------------------- work
def work(case):
    c, op = case, case["op"]
    if op == "plan":
        n = _new_tokens(c)
        blocks = n / c["block"]
        return {"bytes": 16 * c["R"] + 12 * n + 8 * blocks, "flops": 0}
    if op == "append":
        el = c["N"] * c["Hkv"] * c["D"] * 2
        return {"bytes": 2 * el * SIZE[c["dtype"]] + el / 2 + el / 64 * 4 + 8 * c["N"],
                "flops": 6 * el}
    if op == "attention":
        R, lo, hi = c["R"], c["shortest"], c["longest"]
        mean = hi if R == 1 or hi == lo else (hi - lo) / math.log(hi / lo)
        mean = min(mean, c["window"] + c["nq"] - 1) if c["window"] else mean
        el = R * mean * c["Hkv"] * c["D"] * 2
        io = R * c["nq"] * c["H"] * (2 * c["D"] * SIZE[c["dtype"]] + 4)
        return {"bytes": el / 2 + el / 64 * 4 + io, "flops": 2 * el * c["nq"] * c["H"] / c["Hkv"]}
    wb = lambda N, K: N * K / 2 + N * -(-K // c["group"]) * (3 if c["zeros"] else 2)  # noqa: E731
    if op == "matvec":
        return {"bytes": wb(c["N"], c["K"]) + c["rows"] * (c["N"] + c["K"]) * SIZE[c["dtype"]],
                "flops": 2 * c["rows"] * c["N"] * c["K"]}
    # Distinct experts that T tokens with k of E each are expected to reach.
    active = c["E"] * (1 - (1 - c["k"] / c["E"]) ** c["T"])
    return {"bytes": active * (wb(2 * c["ff"], c["d"]) + wb(c["d"], c["ff"]))
            + 2 * c["T"] * c["d"] * SIZE[c["dtype"]] + 8 * c["T"] * c["k"],
            "flops": 6 * c["T"] * c["k"] * c["d"] * c["ff"]}


# ------------------------------------------------------- exact, in 64 bits
def _nibbles(b):
    """uint8 array [..., n] -> float64 codes [..., 2n], low nibble first."""
    out = torch.empty(*b.shape[:-1], b.shape[-1] * 2, dtype=torch.float64, device=b.device)
    out[..., 0::2] = (b % 16).double()
    out[..., 1::2] = (b // 16).double()
    return out


def _exact_rows(w, e, rows):
    """Rows of matrix e of a 4-bit weight, dequantised in float64."""
    c = _nibbles(w["codes"][e, rows])
    at = torch.arange(w["K"], device="cuda") // w["group"]
    z = 8.0 if w["zeros"] is None else w["zeros"][e, rows].double()[:, at]
    return (c - z) * w["scales"][e, rows].double()[:, at]


def _exact_product(w, e, x, step=4096):
    """x [m][K] float64 times matrix e transposed, in blocks of rows."""
    return torch.cat([x @ _exact_rows(w, e, slice(a, a + step)).T
                      for a in range(0, w["N"], step)], 1)


def _exact_dims(D):
    """Where dimension d of token t of a granule lies: byte offsets of its K
    and V codes [16][D], and the nibble's shift [D]."""
    t, d = np.meshgrid(np.arange(16), np.arange(D), indexing="ij")
    G = D // 64
    g, r = d // 64, d % 64
    kb = t * (D // 2) + (r // 16) * (D // 8) + g * 8 + (r % 16) // 8 * 4 + (r % 8) // 2
    u = t // 8 * 2 + t % 2
    per = 4 // G
    vb = ((((u // per) * 8 + r // 8) * 4 + (t % 8) // 2) * per + u % per) * 4 * G
    vb = 8 * D + vb + g * 4 + (r % 8) // 2
    return kb, vb, (d % 2) * 4


def _exact_attention(c, s):
    D, Hkv, H, nq, bs = c["D"], c["Hkv"], c["H"], c["nq"], c["block"]
    kb, vb, sh = (torch.from_numpy(a).cuda() for a in _exact_dims(D))
    G = D // 64
    at = torch.arange(D, device="cuda") // 64
    out = torch.zeros(c["R"] * nq, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((c["R"] * nq, H), -math.inf, dtype=torch.float64, device="cuda")
    for r in range(c["R"]):
        n = int(s["kv_len"][r])
        rows = slice(r * nq, (r + 1) * nq)
        pages = s["table"][r, :-(-n // bs)].long()
        for h in range(Hkv):
            gran = s["cache"][pages, h].flatten(0, 1)                # granules of 16 tokens
            par = gran[:, 16 * D:].contiguous().view(torch.float16).double()
            par = par.view(-1, 2, 16, G, 2)[..., at, :]
            k, v = (((gran[:, b.flatten()].view(-1, 16, D) >> sh) & 15).double()
                    * par[:, i, :, :, 0] + par[:, i, :, :, 1] for i, b in ((0, kb), (1, vb)))
            k, v = k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]
            hs = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            x = s["q"][rows, hs].double() @ k.T / math.sqrt(D)      # nq G n
            pos = n - nq + torch.arange(nq, device="cuda")[:, None, None]
            t = torch.arange(n, device="cuda")
            hide = (t > pos) | ((t <= pos - c["window"]) if c["window"] else False)
            x = x.masked_fill(hide, -math.inf)
            lse[rows, hs] = torch.logsumexp(x, -1)
            out[rows, hs] = torch.softmax(x, -1).nan_to_num(0.0) @ v
    return dict(out=out, lse=lse)


def _exact_append(c, s):
    """Scale, minimum and code are defined with their roundings (fp32 steps,
    float16 scale and minimum), so the 64-bit arithmetic rounds there too."""
    def one(x):
        x = x.double().clamp(-65504, 65504).unflatten(-1, (-1, 64))
        lo, hi = x.min(-1).values, x.max(-1).values
        rng = (hi - lo).float().double() * float(np.float32(1 / 15))
        sc, mn = rng.float().half().double()[..., None], lo.half().double()[..., None]
        q = ((x - mn).float().double() / sc).float().double()
        code = torch.where(sc > 0, torch.round(q).clamp(0, 15), 0.0)
        return (sc * code + mn).flatten(-2)
    return dict(k=one(s["k"]), v=one(s["v"]), cache=None)


def exact(case, seed):
    c, op = case, case["op"]
    if op == "plan":
        return None
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if op == "append":
        return _exact_append(c, s)
    if op == "attention":
        return _exact_attention(c, s)
    if op == "matvec":
        return _exact_product(s["w"], 0, s["x"].double())
    x, y = s["x"].double(), torch.zeros(c["T"], c["d"], dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        t, slot = torch.nonzero(s["idx"] == e, as_tuple=True)
        if not t.numel():
            continue
        gu = _exact_product(s["gu"], e, x[t])
        h = torch.sigmoid(gu[:, :c["ff"]]) * gu[:, :c["ff"]] * gu[:, c["ff"]:]
        y.index_add_(0, t, _exact_product(s["dn"], e, h) * s["wt"][t, slot].double()[:, None])
    return y
