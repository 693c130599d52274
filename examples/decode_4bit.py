#!/usr/bin/env python
"""Greedy decoding of a small Mixture-of-Experts decoder in 4 bits.

    python examples/decode_4bit.py [--requests 5] [--new-tokens 12] [--check]

Ragged requests share one pool of pages of a 4-bit key/value cache.  Every step
takes the requests' new tokens (their whole prompts first, one token each
afterwards) through

    Kv4Cache.plan         block tables and slot map of the step
    per layer:
      W4Matrix.matvec     q, k and v projections in one product
      Kv4Cache.append     keys and values into the cache
      Kv4Cache.attention  over everything cached so far
      W4Matrix.matvec     output projection
      MoeLayer.route_device, w4_experts   router and routed experts
    W4Matrix.matvec       output head

and ends requests as they reach their length, which returns their pages.
Norms, rotary embedding and the embedding lookup are plain torch.  The weights
are random; --check runs the same model in torch on the dequantised weights and
the values that the cache's codes stand for, and compares logits and tokens.
"""
import argparse
import importlib.util
import sys
from pathlib import Path

import numpy as np
import torch


def load_pkg():
    name = "moe_b200"
    if name not in sys.modules:
        init = Path(__file__).resolve().parents[1] / "accelerating-moe-inference_b200" / "__init__.py"
        spec = importlib.util.spec_from_file_location(name, init)
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


LAYERS, D, HEADS, KV_HEADS, HEAD_DIM, VOCAB = 2, 512, 8, 2, 64, 1000
EXPERTS, TOP_K, FF, GROUP, PAGE = 8, 2, 448, 64, 16


def dequant(codes, scales, zeros):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(np.float32)
    at = np.arange(c.shape[-1]) // GROUP
    z = zeros[..., at].astype(np.float32) if zeros is not None else 8
    return torch.from_numpy((c - z) * scales[..., at].astype(np.float32)).cuda()


class Model:
    """Random weights, their 4-bit handles and (for the check) their values."""

    def __init__(self, pkg, seed=0):
        g = np.random.default_rng(seed)
        w = lambda *s: (g.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)  # noqa: E731

        def pack(a, gated=False):
            q = pkg.quantize_w4(a, GROUP)
            return pkg.W4Matrix(*q, group=GROUP, gated=gated, max_rows=512), dequant(*q)
        self.embed = torch.from_numpy(g.standard_normal((VOCAB, D)).astype(np.float32)).cuda()
        self.head, self.head_w = pack(w(VOCAB, D))
        self.layers = []
        for i in range(LAYERS):
            moe = pkg.synthetic_layer(seed + i, D, FF, EXPERTS, std=D ** -0.5)
            qkv, qkv_w = pack(w((HEADS + 2 * KV_HEADS) * HEAD_DIM, D))
            out, out_w = pack(w(D, HEADS * HEAD_DIM))
            gu, gu_w = pack(np.stack([np.concatenate([a, b]) for a, b in zip(moe.w1, moe.w3)]), True)
            dn, dn_w = pack(np.stack(moe.w2))
            self.layers.append(dict(
                router=pkg.MoeLayer(moe, top_k=TOP_K, precision=pkg.PREC_BF16), qkv=qkv, out=out,
                gu=gu, dn=dn, qkv_w=qkv_w, out_w=out_w, gu_w=gu_w, dn_w=dn_w))


def rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)


def rope(x, pos):
    half = HEAD_DIM // 2
    f = 10000.0 ** (-torch.arange(half, device=x.device) / half)
    a = pos[:, None, None] * f
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat([x0 * a.cos() - x1 * a.sin(), x1 * a.cos() + x0 * a.sin()], -1).contiguous()


def product(w, x, y, stream):
    """y = w x for the rows of x, as many at a time as a call takes."""
    for t in range(0, x.shape[0], 512):
        w.matvec(x[t:].data_ptr(), y[t:].data_ptr(), min(512, x.shape[0] - t), 0, stream)


class Server:
    """The pool of pages, the block tables and one cache per layer."""

    def __init__(self, pkg, model, requests, longest):
        self.pkg, self.model, self.R = pkg, model, requests
        width = -(-longest // PAGE)
        self.kv = pkg.Kv4Cache(num_kv_heads=KV_HEADS, head_dim=HEAD_DIM, block_tokens=PAGE,
                               num_blocks=requests * width, table_width=width,
                               max_requests=requests)
        nb = requests * width
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.cached = i32(requests, width), i32(requests)
        self.kv_len, self.q_offset = i32(requests), i32(requests + 1)
        self.ring = torch.arange(nb, dtype=torch.int32, device="cuda")
        self.state = [torch.tensor([0, nb], dtype=torch.int32, device="cuda"), i32(2)]
        self.cache = [torch.empty(self.kv.cache_bytes(), dtype=torch.uint8, device="cuda")
                      for _ in model.layers]
        self.seen = [[[] for _ in range(requests)] for _ in model.layers]   # for the check only

    def plan(self, new, tokens):
        """Slots and positions of a step that adds new[r] tokens to request r."""
        s = torch.cuda.current_stream().cuda_stream
        pos = torch.empty(tokens, dtype=torch.int32, device="cuda")
        slot = torch.empty(tokens, dtype=torch.int64, device="cuda")
        self.kv.plan(self.cached.data_ptr(), new.data_ptr(), self.R, self.ring.data_ptr(),
                     self.state[0].data_ptr(), self.table.data_ptr(), self.kv_len.data_ptr(),
                     self.q_offset.data_ptr(), pos.data_ptr(), slot.data_ptr(), tokens,
                     self.state[1].data_ptr(), s)
        self.state.reverse()
        self.cached.copy_(self.kv_len)
        return pos, slot

    def step(self, ids, new, check):
        """Logits [R][vocab] of each request's last new token (and torch's)."""
        pkg, f32 = self.pkg, self.pkg.DTYPE_F32
        s = torch.cuda.current_stream().cuda_stream
        N = ids.numel()
        pos, slot = self.plan(new, N)
        x = self.model.embed[ids]
        plain = x.clone() if check else None
        owner = torch.repeat_interleave(torch.arange(self.R, device="cuda"), new.clamp(min=0),
                                        output_size=N)
        for i, (L, cache) in enumerate(zip(self.model.layers, self.cache)):
            h = rms(x)
            qkv = torch.empty(N, HEADS + 2 * KV_HEADS, HEAD_DIM, device="cuda")
            product(L["qkv"], h, qkv, s)
            q = rope(qkv[:, :HEADS], pos)
            k, v = rope(qkv[:, HEADS:HEADS + KV_HEADS], pos), qkv[:, HEADS + KV_HEADS:]
            ko, vo = torch.empty_like(k), torch.empty(v.shape, device="cuda")
            self.kv.append(cache.data_ptr(), k.data_ptr(), v.data_ptr(), f32, N, slot.data_ptr(),
                           s, v_strides=v.stride()[:2], k_out_ptr=ko.data_ptr(),
                           v_out_ptr=vo.data_ptr())
            a = torch.empty(N, HEADS * HEAD_DIM, device="cuda")
            self.kv.attention(cache.data_ptr(), q.data_ptr(), a.data_ptr(), f32, N, HEADS,
                              self.table.data_ptr(), self.kv_len.data_ptr(),
                              self.q_offset.data_ptr(), self.R, s)
            o = torch.empty(N, D, device="cuda")
            product(L["out"], a, o, s)
            x = x + o
            h = rms(x)
            logits = torch.empty(N, EXPERTS, device="cuda")
            idx = torch.empty(N, TOP_K, dtype=torch.int32, device="cuda")
            wt, y = torch.empty(N, TOP_K, device="cuda"), torch.empty_like(x)
            L["router"].route_device(h.data_ptr(), N, logits.data_ptr(), idx.data_ptr(),
                                     wt.data_ptr(), s)
            for t in range(0, N, 512 // TOP_K):
                n = min(N - t, 512 // TOP_K)
                pkg.w4_experts(L["gu"], L["dn"], h[t:].data_ptr(), idx[t:].data_ptr(),
                               wt[t:].data_ptr(), y[t:].data_ptr(), n, TOP_K, f32, s)
            x = x + y
            if check:
                plain = self.plain_layer(i, L, plain, pos, owner, ko, vo, idx, wt)
        last = self.q_offset[1:].long() - 1
        h = rms(x[last.clamp(min=0)])
        logits = torch.empty(self.R, VOCAB, device="cuda")
        product(self.model.head, h, logits, s)
        want = rms(plain[last.clamp(min=0)]) @ self.model.head_w.T if check else None
        return logits, want

    def plain_layer(self, i, L, x, pos, owner, k, v, idx, wt):
        h = rms(x)
        qkv = (h @ L["qkv_w"].T).view(-1, HEADS + 2 * KV_HEADS, HEAD_DIM)
        q = rope(qkv[:, :HEADS], pos)
        out = torch.empty(x.shape[0], HEADS, HEAD_DIM, device="cuda")
        group = HEADS // KV_HEADS
        for r in range(self.R):
            t = torch.nonzero(owner == r).flatten()
            if not t.numel():
                continue
            self.seen[i][r].append((k[t], v[t]))
            kk, vv = (torch.cat([e[j] for e in self.seen[i][r]]).repeat_interleave(group, 1)
                      for j in (0, 1))
            sc = torch.einsum("thd,shd->hts", q[t], kk) * HEAD_DIM ** -0.5
            later = torch.arange(kk.shape[0], device="cuda") > pos[t][:, None]
            out[t] = torch.einsum("hts,shd->thd", sc.masked_fill(later, -torch.inf).softmax(-1), vv)
        x = x + out.flatten(1) @ L["out_w"].T
        h = rms(x)
        gu = torch.einsum("td,efd->tef", h, L["gu_w"])
        act = torch.nn.functional.silu(gu[..., :FF]) * gu[..., FF:]
        y = torch.einsum("tef,edf->ted", act, L["dn_w"])
        pick = torch.take_along_dim(y, idx.long()[..., None], 1)
        return x + (pick * wt[..., None]).sum(1)


def decode(requests=5, new_tokens=12, check=False, seed=0):
    """Generated ids per request; with check the largest relative 2-norm error
    of a step's logits and how many of the tokens torch's logits choose too."""
    pkg = load_pkg()
    g = np.random.default_rng(seed)
    lens = g.integers(1, 40, requests)
    ends = g.integers(1, new_tokens + 1, requests)   # tokens each request generates
    server = Server(pkg, Model(pkg, seed), requests, int(lens.max()) + new_tokens + 1)
    ids = torch.from_numpy(np.concatenate([g.integers(0, VOCAB, n) for n in lens])).cuda()
    new = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, worst, same, total = [[] for _ in range(requests)], 0.0, 0, 0
    for step in range(new_tokens):
        logits, want = server.step(ids, new, check)
        pick = logits.argmax(-1)
        live = [r for r in range(requests) if step < ends[r]]
        for r in live:
            out[r].append(int(pick[r]))
        if check:
            a, b = logits[live].double(), want[live].double()
            worst = max(worst, float((a - b).norm() / b.norm()))
            same += int((pick[live] == want[live].argmax(-1)).sum())
            total += len(live)
        # Requests that have their tokens end (once), the others go on.
        state = [1 if step + 1 < ends[r] else -1 if step + 1 == ends[r] else 0
                 for r in range(requests)]
        new = torch.tensor(state, dtype=torch.int32, device="cuda")
        if max(state) < 1:
            server.plan(new, 0)
            break
        ids = pick[new > 0]
    free = int(server.state[0][1])
    return out, worst, same, total, free == server.kv.cfg.num_blocks


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=5)
    ap.add_argument("--new-tokens", type=int, default=12)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    out, worst, same, total, whole = decode(a.requests, a.new_tokens, a.check)
    for r, ids in enumerate(out):
        print(f"request {r}: {ids}")
    print("all pages back in the pool:", whole)
    if a.check:
        print(f"logits against torch: rel-L2 {worst:.2e}; same token {same} of {total}")


if __name__ == "__main__":
    main()
