"""Inputs and 64-bit definitions shared by the tests of the 8-bit KV cache and of windowed attention."""

import math

import torch

D = 128


def pages(gen, lens, nkv, bs, bits, spare=2):
    """Random paged caches of sequences of these lengths: (k, v, k_scale, v_scale, table, dense k, dense v), the
    dense ones in 64 bits per sequence.  Everything no sequence owns is hostile: NaN codes or values, exponent
    255, page ids far outside the cache."""
    from psrl_b200.ops.kv_quant import dequantise_ref, quantise_ref

    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=gen).tolist()
    table = torch.full((len(lens), max(need + [1]) + 1), 2 ** 30, dtype=torch.int32)
    table[::2, -1] = -7
    if bits == 8:
        cache = [torch.full((blocks, nkv, bs, D), 0x7F, dtype=torch.uint8) for _ in range(2)]
        scale = [torch.full((blocks, nkv, bs), 255, dtype=torch.uint8) for _ in range(2)]
    else:
        cache = [torch.full((blocks, nkv, bs, D), math.nan, dtype=torch.bfloat16) for _ in range(2)]
        scale = [None, None]
    dense = [[], []]
    for i, n in enumerate(lens):
        ids = order[:need[i]]
        order = order[need[i]:]
        table[i, :need[i]] = torch.tensor(ids, dtype=torch.int32)
        for c in range(2):
            size = torch.rand(D, generator=gen) * 1.5 + 0.25
            x = (torch.randn(n, nkv, D, generator=gen) * size).to(torch.bfloat16)
            p = torch.arange(n)
            blk, off = torch.tensor(ids, dtype=torch.long)[p // bs], p % bs
            if bits == 8:
                codes, byte = quantise_ref(x)
                cache[c][blk, :, off] = codes.view(torch.uint8)
                scale[c][blk, :, off] = byte
                dense[c].append(dequantise_ref(codes, byte, torch.float64))
            else:
                cache[c][blk, :, off] = x
                dense[c].append(x.double())
    if bits == 8:
        cache = [x.view(torch.float8_e4m3fn) for x in cache]
    return cache[0], cache[1], scale[0], scale[1], table, dense[0], dense[1]


def attention64(q, k, v, window=None, sinks=0, scale=None):
    """q [n, nq, D] are the last n positions of k, v [L, nkv, D]: (o, sum of p |v|) in 64 bits."""
    n, nq, _ = q.shape
    L, nkv, _ = k.shape
    g = nq // nkv
    o = torch.zeros(n, nq, D, dtype=torch.float64)
    a = torch.zeros_like(o)
    if L == 0:
        return o, a
    i = torch.arange(L - n, L)[:, None]
    j = torch.arange(L)[None, :]
    ok = j <= i
    if window:
        ok = ok & ((i - j < window) | (j < sinks))
    for h in range(nq):
        s = q[:, h].double() @ k[:, h // g].t() * (scale or 1 / math.sqrt(D))
        top = s.masked_fill(~ok, -math.inf).amax(-1, keepdim=True)
        p = torch.where(ok, torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros(()).double())
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        o[:, h] = p @ v[:, h // g]
        a[:, h] = p @ v[:, h // g].abs()
    return o, a


def train64(q, k, v, do, window=None, sinks=0):
    """Gradients of one sequence's attention in 64 bits with the bounds of a kernel that keeps sums in fp32 and
    rounds the output, P and dS to bf16 (half a step: 2^-8 of the value): {name: (value, bound)}.  q, do [n, nq, D]
    are the last n positions of k, v [L, nkv, D]."""
    u = 2.0 ** -8
    tiny = 2.0 ** -14                                # fp32 scores and exponentials of |score| < 2^7
    n, nq, _ = q.shape
    L, nkv, _ = k.shape
    g, scale = nq // nkv, 1 / math.sqrt(D)
    q, k, v, do = (x.double() for x in (q, k, v, do))
    i = torch.arange(L - n, L, device=q.device)[:, None]
    j = torch.arange(L, device=q.device)[None, :]
    ok = j <= i
    if window:
        ok = ok & ((i - j < window) | (j < sinks))
    out = {m: (torch.zeros_like(x), torch.zeros_like(x)) for m, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    for h in range(nq):
        hk = h // g
        p = (q[:, h] @ k[:, hk].t() * scale).masked_fill(~ok, -math.inf).softmax(-1)
        o = p @ v[:, hk]
        eo = u * o.abs() + (u + tiny) * (p @ v[:, hk].abs())
        dp = do[:, h] @ v[:, hk].t()
        dd = (o * do[:, h]).sum(-1, keepdim=True)
        ed = (eo * do[:, h].abs()).sum(-1, keepdim=True)
        ds = p * (dp - dd)
        es = u * ds.abs() + p * (ed + tiny * (dp.abs() + dd.abs()))
        out["o"][0][:, h], out["o"][1][:, h] = o, eo
        out["dq"][0][:, h] = ds @ k[:, hk] * scale
        out["dq"][1][:, h] = es @ k[:, hk].abs() * scale
        out["dk"][0][:, hk] += ds.t() @ q[:, h] * scale
        out["dk"][1][:, hk] += es.t() @ q[:, h].abs() * scale
        out["dv"][0][:, hk] += p.t() @ do[:, h]
        out["dv"][1][:, hk] += (u + tiny) * (p.t() @ do[:, h].abs())
    for m in ("dq", "dk", "dv"):
        out[m][1].add_(u * out[m][0].abs())          # the gradient's own rounding
    return out
