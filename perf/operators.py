"""Workloads of the 8-bit KV cache and of sliding-window attention.

Four operators around the paged KV cache of the rollout engine and the packed
batches of the trainer:

* ``write`` / ``read`` — rotary embedding fused with the write of keys and
  values into an 8-bit paged cache, and pages read back as bf16;
* ``decode`` — one new token per sequence attends to its paged context;
* ``chunk``  — a chunk of new tokens per sequence attends to its paged context;
* ``train``  — packed causal attention with a sliding window and visible first
  tokens (sinks), forward and backward.

An 8-bit cache holds every (token, kv head) vector of keys or of values as
float8 e4m3 codes and one byte with a power-of-two exponent: value = code *
2^(byte - 127).  The exponent is the smallest with max|x| <= 448 * 2^e, kept in
[-63, 120] (a zero vector has -63); a vector with a NaN or an infinity has byte
255 and reads as NaN.  A query at position p sees the keys j <= p with
p - j < window or j < sinks; a row that sees nothing gives zeros.
"""

import math

import torch

own = False

D = 128
THETA = 1_000_000.0


# -------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of a small batch: one rotated row per sequence
        dict(name="write_step", op="write", tokens=24, nq=16, nkv=2, block=64, far=9216),
        # a full prefill step of the engine (its default token budget)
        dict(name="write_chunk", op="write", tokens=10240, nq=32, nkv=8, block=64, far=32768),
        # one short request moved to an engine that keeps bf16 keys and values
        dict(name="read_request", op="read", blocks=11, nkv=2, block=64),
        # a batch of long requests moved
        dict(name="read_batch", op="read", blocks=3001, nkv=8, block=64),
        # the last request of a rollout batch: latency
        dict(name="decode_one", op="decode", batch=1, longest=517, nq=16, nkv=2, block=64, bits=8, window=0, sinks=0),
        # an ordinary rollout batch, ragged lengths
        dict(name="decode_batch", op="decode", batch=64, longest=9216, nq=16, nkv=2, block=64, bits=8, window=0, sinks=0),
        # long contexts, wide cache
        dict(name="decode_long", op="decode", batch=48, longest=32768, nq=32, nkv=8, block=64, bits=8, window=0, sinks=0),
        # a windowed model on the bf16 cache
        dict(name="decode_window", op="decode", batch=96, longest=16384, nq=32, nkv=8, block=64, bits=16, window=4096, sinks=4),
        # next turns of conversations: a few new tokens each over long contexts
        dict(name="chunk_turns", op="chunk", seqs=9, new=61, longest=8191, nq=16, nkv=2, block=64, bits=8, window=0, sinks=0),
        # a long prompt's last prefill chunk
        dict(name="chunk_prompt", op="chunk", seqs=1, new=8192, longest=24576, nq=32, nkv=8, block=64, bits=8, window=0, sinks=0),
        # a micro-batch of a windowed model, forward and backward
        dict(name="train_micro", op="train", seqs=6, longest=1700, nq=16, nkv=2, window=512, sinks=4),
        # one long document
        dict(name="train_long", op="train", seqs=1, longest=16384, nq=32, nkv=8, window=4096, sinks=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk", "train"])
    nq, nkv = rng.choice([(16, 2), (28, 4), (32, 8), (32, 4), (8, 2), (8, 8)])
    block = rng.choice([16, 32, 64, 64, 128])
    if op == "write":
        return dict(op=op, tokens=_log(rng, 1, 10240), nq=nq, nkv=nkv, block=block, far=_log(rng, 4096, 65536))
    if op == "read":
        return dict(op=op, blocks=_log(rng, 1, 3001), nkv=nkv, block=min(block, 64))
    window = rng.choice([0, 0, _log(rng, 16, 8192)])
    sinks = rng.choice([0, 1, 4, 70]) if window else 0
    if op == "train":
        return dict(op=op, seqs=_log(rng, 1, 8), longest=_log(rng, 1, 2048), nq=nq, nkv=nkv,
                    window=window or _log(rng, 16, 2048), sinks=sinks)
    bits = rng.choice([8, 8, 16]) if window else 8
    if op == "decode":
        batch = _log(rng, 1, 256)
        longest = _log(rng, 1, max(2, min(32768, 48 * 32768 * 8 // (batch * nkv))))
        return dict(op=op, batch=batch, longest=longest, nq=nq, nkv=nkv, block=block, bits=bits, window=window,
                    sinks=sinks)
    seqs = _log(rng, 1, 16)
    longest = _log(rng, 1, 16384)
    new = min(longest, _log(rng, 1, max(2, 4096 // seqs)))
    return dict(op=op, seqs=seqs, new=new, longest=longest, nq=nq, nkv=nkv, block=block, bits=bits, window=window,
                sinks=sinks)


def _lengths(n, longest):
    """Ragged lengths: the longest first, then spread down to a third of it; the
    last of four or more is a single token (a padded row of a decode batch)."""
    lens = [max(1, longest - (longest * 2 // 3) * ((i * 37) % n) // n) for i in range(n)]
    if n >= 4:
        lens[-1] = 1
    return lens


def _chunk_lengths(case):
    lens = _lengths(case["seqs"], case["longest"])
    return [min(n, max(1, case["new"] - 3 * i)) for i, n in enumerate(lens)], lens


def _pairs(new, length, window, sinks):
    """(query, key) pairs that the last `new` of `length` positions see."""
    if not window:
        return sum(range(length - new + 1, length + 1))
    return sum(min(p + 1, window + min(sinks, max(0, p + 1 - window))) for p in range(length - new, length))


def work(case):
    op = case["op"]
    if op == "write":
        t, nq, nkv = case["tokens"], case["nq"], case["nkv"]
        return {"bytes": t * ((nq + 2 * nkv) * 2 * D + nq * 2 * D + 2 * nkv * (D + 1) + 8 + 8 * (D // 2)),
                "flops": t * (nq + nkv) * 3 * D}
    if op == "read":
        n = case["blocks"] * case["nkv"] * case["block"]
        return {"bytes": n * (D + 1 + 2 * D), "flops": n * D}
    nq, nkv, window, sinks = case["nq"], case["nkv"], case["window"], case["sinks"]
    if op == "train":
        lens = _lengths(case["seqs"], case["longest"])
        pairs = sum(_pairs(n, n, window, sinks) for n in lens)
        row = 2 * D * (nq + 2 * nkv)
        # forward: qkv in, o out; backward: qkv, o, dout in, dqkv out; seven products in all
        return {"bytes": sum(lens) * (3 * row + 3 * 2 * D * nq), "flops": 7 * 2 * D * nq * pairs}
    per_key = 2 * nkv * (D + 1 if case["bits"] == 8 else 2 * D)
    if op == "decode":
        lens = _lengths(case["batch"], case["longest"])
        new = [1] * len(lens)
    else:
        new, lens = _chunk_lengths(case)
    seen = sum(n if not window else min(n, window + q - 1 + min(sinks, max(0, n - window - q + 1)))
               for q, n in zip(new, lens))
    pairs = sum(_pairs(q, n, window, sinks) for q, n in zip(new, lens))
    return {"bytes": seen * per_key + sum(new) * 2 * 2 * D * nq, "flops": 4 * D * nq * pairs}


# -------------------------------------------------------------------- inputs
def _quantise(x):
    """fp32 [..., D] -> (e4m3 codes as float8, exponent bytes); see the head of this file."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)
    k = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-63, 120)      # 448 = 0.875 * 2^9
    k = torch.where(amax == 0, torch.full_like(k, -63), k)
    bad = ~torch.isfinite(amax)
    k = torch.where(bad, torch.zeros_like(k), k)
    codes = torch.where(bad[..., None], torch.zeros_like(x), torch.ldexp(x, -k[..., None]))
    return codes.to(torch.float8_e4m3fn), torch.where(bad, torch.full_like(k, 255), k + 127).to(torch.uint8)


def _vectors(gen, *shape):
    """Keys or values as a model has them: channels of unequal size, a few large."""
    size = torch.rand(shape[-1], generator=gen, device="cuda") * 1.5 + 0.25
    size[:: shape[-1] // 4] *= 4.0
    return (torch.randn(*shape, generator=gen, device="cuda") * size).to(torch.bfloat16)


def _pages(gen, blocks, nkv, block, bits):
    """(cache, exponent bytes or None) of random pages, filled in pieces."""
    if bits == 16:
        cache = torch.empty(blocks, nkv, block, D, dtype=torch.bfloat16, device="cuda")
        scale = None
    else:
        cache = torch.empty(blocks, nkv, block, D, dtype=torch.float8_e4m3fn, device="cuda")
        scale = torch.empty(blocks, nkv, block, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (nkv * block * D))
    for s in range(0, blocks, step):
        x = _vectors(gen, min(step, blocks - s), nkv, block, D)
        if bits == 16:
            cache[s:s + step] = x
        else:
            c, e = _quantise(x.float())
            cache[s:s + step].view(torch.uint8).copy_(c.view(torch.uint8))
            scale[s:s + step] = e
    return cache, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op = case["op"]
    if op == "write":
        t, nq, nkv, bs = case["tokens"], case["nq"], case["nkv"], case["block"]
        blocks = -(-t // bs) + 3
        slots = torch.randperm(blocks * bs, generator=host)[:t].to(torch.int32)
        if t >= 16:
            slots[-3:] = -1                                    # padded rows of a decode bucket
        cache = [torch.zeros(blocks, nkv, bs, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
                 for _ in range(2)]
        scale = [torch.zeros(blocks, nkv, bs, dtype=torch.uint8, device="cuda") for _ in range(2)]
        return dict(case=case, qkv=_vectors(gen, t, (nq + 2 * nkv), D).view(t, -1),
                    pos=torch.randint(0, case["far"], (t,), generator=host, dtype=torch.int32).cuda(),
                    slots=slots.cuda(), k=cache[0], v=cache[1], ks=scale[0], vs=scale[1])
    if op == "read":
        n = case["blocks"]
        cache, scale = _pages(gen, n + 5, case["nkv"], case["block"], 8)
        return dict(case=case, cache=cache, scale=scale,
                    blocks=torch.randperm(n + 5, generator=host)[:n].to(torch.int32).cuda())
    nq, nkv, window = case["nq"], case["nkv"], case["window"]
    if op == "train":
        lens = _lengths(case["seqs"], case["longest"])
        cu = torch.tensor([0] + lens).cumsum(0)
        t = int(cu[-1])
        qkv = _vectors(gen, t, nq + 2 * nkv, D)
        qkv[:, :nq] *= 0.7
        return dict(case=case, qkv=qkv.view(t, -1).requires_grad_(True), cu=cu.to(torch.int32).cuda(), lens=lens,
                    dout=torch.randn(t, nq * D, generator=gen, device="cuda").to(torch.bfloat16))
    bs = case["block"]
    if op == "decode":
        lens = _lengths(case["batch"], case["longest"])
        new = [1] * len(lens)
    else:
        new, lens = _chunk_lengths(case)
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + 1
    order = torch.randperm(blocks, generator=host).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at: at + n]
        at += n
    k, ks = _pages(gen, blocks, nkv, bs, case["bits"])
    v, vs = _pages(gen, blocks, nkv, bs, case["bits"])
    q = (_vectors(gen, sum(new), nq, D).float() * 0.7).to(torch.bfloat16)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return dict(case=case, q=q, k=k, v=v, ks=ks, vs=vs, table=table.cuda(), cu=cu.cuda(), new=new, lens=lens,
                kv_lens=torch.tensor(lens, dtype=torch.int32).cuda())


# ---------------------------------------------------------------- plain forms
def _values(codes, scale):
    """fp32 values of cache rows (codes [..., D], exponent bytes [...] or None)."""
    if scale is None:
        return codes.float()
    x = torch.ldexp(codes.float(), scale.to(torch.int32)[..., None] - 127)
    return torch.where((scale == 255)[..., None], torch.full_like(x, math.nan), x)


def _rows(cache, scale, table, pos):
    """Cache rows at positions pos [B, M] of each sequence: fp32 [B, M, nkv, D]."""
    bs = cache.shape[2]
    blk = torch.gather(table.long(), 1, pos // bs)
    codes = cache.view(torch.uint8 if scale is not None else cache.dtype)[blk, :, pos % bs]
    if scale is None:
        return codes.float()
    return _values(codes.view(torch.float8_e4m3fn), scale[blk, :, pos % bs])


def _weights(s, mask):
    """Softmax over the last axis of the scores that the mask keeps; zeros where it keeps none."""
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total)), top, total


def _seen(qpos, kpos, window, sinks):
    ok = kpos <= qpos
    if window:
        ok = ok & ((qpos - kpos < window) | (kpos < sinks))
    return ok


def _plain_write(s):
    c = s["case"]
    t, nq, nkv = c["tokens"], c["nq"], c["nkv"]
    inv = 1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    ang = s["pos"].double()[:, None] * inv
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    x = s["qkv"].view(t, nq + 2 * nkv, D).float()
    a, b = x[:, : nq + nkv, : D // 2], x[:, : nq + nkv, D // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    blk, off = at // c["block"], at % c["block"]
    for cache, scale, y in ((s["k"], s["ks"], qk[:, nq:].float()), (s["v"], s["vs"], x[:, nq + nkv:])):
        codes, e = _quantise(y)
        cache.view(torch.uint8)[blk, :, off] = codes.view(torch.uint8)[keep]
        scale[blk, :, off] = e[keep]
    return qk[:, :nq].reshape(t, nq * D)


def _plain_decode(s):
    c = s["case"]
    n, window, sinks = s["kv_lens"].long()[:, None], c["window"], c["sinks"]
    longest = s["table"].shape[1] * c["block"]
    if window and window + sinks < longest:
        recent = n - window + torch.arange(window, device="cuda")
        first = torch.arange(sinks, device="cuda").expand(n.shape[0], -1)
        pos = torch.cat([first, recent], 1)
        ok = torch.cat([first < n - window, recent >= 0], 1)
    else:
        pos = torch.arange(longest, device="cuda").expand(n.shape[0], -1)
        ok = (pos < n) & _seen(n - 1, pos, window, sinks)
    pos = pos.clamp(0, longest - 1)
    k = _rows(s["k"], s["ks"], s["table"], pos)
    q = s["q"].float().view(n.shape[0], c["nkv"], -1, D)
    p, _, _ = _weights(torch.einsum("bhgd,bmhd->bhgm", q, k) / math.sqrt(D), ok[:, None, None])
    del k
    v = _rows(s["v"], s["vs"], s["table"], pos)
    v = torch.where(ok[:, :, None, None], v, torch.zeros_like(v))
    return torch.einsum("bhgm,bmhd->bhgd", p, v).reshape(n.shape[0], c["nq"], D).to(torch.bfloat16)


def _query_blocks(new, length, heads, window):
    """Ranges of the new positions whose scores against the keys fit comfortably."""
    span = length if not window else min(length, window + 1024)
    step = max(16, min(new, 1024 if window else (1 << 30) // (heads * span)))
    return [(a, min(a + step, new)) for a in range(0, new, step)]


def _key_range(lo, hi, window, sinks):
    """Key positions that queries lo..hi-1 can see, as an index."""
    if not window or lo - window + 1 <= sinks:
        return torch.arange(hi, device="cuda")
    return torch.cat([torch.arange(sinks, device="cuda"), torch.arange(lo - window + 1, hi, device="cuda")])


def _plain_chunk(s):
    c = s["case"]
    out = torch.empty_like(s["q"])
    at = 0
    for i, (new, length) in enumerate(zip(s["new"], s["lens"])):
        table = s["table"][i: i + 1]
        pos = torch.arange(length, device="cuda")[None]
        k = _rows(s["k"], s["ks"], table, pos)[0]
        v = _rows(s["v"], s["vs"], table, pos)[0]
        for a, b in _query_blocks(new, length, c["nq"], c["window"]):
            q = s["q"][at + a: at + b].float().view(b - a, c["nkv"], -1, D)
            qpos = torch.arange(length - new + a, length - new + b, device="cuda")
            kpos = _key_range(length - new + a, length - new + b, c["window"], c["sinks"])
            ok = _seen(qpos[:, None], kpos[None], c["window"], c["sinks"])
            p, _, _ = _weights(torch.einsum("qhgd,khd->hgqk", q, k[kpos]) / math.sqrt(D), ok)
            o = torch.einsum("hgqk,khd->qhgd", p, v[kpos])
            out[at + a: at + b] = o.reshape(b - a, c["nq"], D).to(torch.bfloat16)
        at += new
    return out


def _plain_train(s):
    c = s["case"]
    nq, nkv, scale = c["nq"], c["nkv"], 1.0 / math.sqrt(D)
    x = s["qkv"].detach().view(-1, nq + 2 * nkv, D)
    out = torch.empty(x.shape[0], nq, D, dtype=torch.bfloat16, device="cuda")
    grad = torch.zeros(x.shape, dtype=torch.float32, device="cuda")
    dout = s["dout"].view(-1, nq, D)
    at = 0
    for length in s["lens"]:
        rows = slice(at, at + length)
        k, v = x[rows, nq: nq + nkv].float(), x[rows, nq + nkv:].float()
        dk, dv = grad[rows, nq: nq + nkv], grad[rows, nq + nkv:]
        for a, b in _query_blocks(length, length, nq, c["window"]):
            q = x[at + a: at + b, :nq].float().view(b - a, nkv, -1, D)
            do = dout[at + a: at + b].float().view(b - a, nkv, -1, D)
            kpos = _key_range(a, b, c["window"], c["sinks"])
            ok = _seen(torch.arange(a, b, device="cuda")[:, None], kpos[None], c["window"], c["sinks"])
            kk, vv = k[kpos], v[kpos]
            p, _, _ = _weights(torch.einsum("qhgd,khd->hgqk", q, kk) * scale, ok)
            o = torch.einsum("hgqk,khd->qhgd", p, vv)
            dp = torch.einsum("qhgd,khd->hgqk", do, vv)
            ds = p * (dp - (o * do).sum(-1).permute(1, 2, 0)[..., None])
            grad[at + a: at + b, :nq] = (torch.einsum("hgqk,khd->qhgd", ds, kk) * scale).reshape(b - a, nq, D)
            dk.index_add_(0, kpos, torch.einsum("hgqk,qhgd->khd", ds, q) * scale)
            dv.index_add_(0, kpos, torch.einsum("hgqk,qhgd->khd", p, do))
            out[at + a: at + b] = o.reshape(b - a, nq, D).to(torch.bfloat16)
        at += length
    return {"o": out.view(-1, nq * D), "dqkv": grad.to(torch.bfloat16).view(x.shape[0], -1)}


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        return _own(s, c, op)
    if op == "write":
        return {"q": _plain_write(s), "k": s["k"], "v": s["v"], "k_exp": s["ks"], "v_exp": s["vs"]}
    if op == "read":
        at = s["blocks"].long()
        codes = s["cache"].view(torch.uint8)[at].view(torch.float8_e4m3fn)
        return _values(codes, s["scale"][at]).to(torch.bfloat16)
    return {"decode": _plain_decode, "chunk": _plain_chunk, "train": _plain_train}[op](s)


def _own(s, c, op):
    from psrl_b200 import ops

    if op == "write":
        q = ops.rope_quant_kv(s["qkv"], s["pos"], c["nq"], c["nkv"], D, THETA, s["k"], s["v"], s["ks"], s["vs"],
                              s["slots"])
        return {"q": q, "k": s["k"], "v": s["v"], "k_exp": s["ks"], "v_exp": s["vs"]}
    if op == "read":
        return ops.read_kv_cache(s["cache"], s["scale"], s["blocks"])
    how = dict(window=c["window"] or None, sinks=c["sinks"])
    if op == "train":
        o = ops.varlen_attention(s["qkv"], s["cu"], max(s["lens"]), c["nq"], c["nkv"], D, **how)
        (g,) = torch.autograd.grad(o, s["qkv"], s["dout"])
        return {"o": o.detach(), "dqkv": g}
    how.update(k_scale=s["ks"], v_scale=s["vs"])
    if op == "decode":
        return ops.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["kv_lens"], **how)
    return ops.paged_prefill_attention(s["q"], s["k"], s["v"], s["cu"], s["kv_lens"], s["table"], max(s["new"]), **how)


# --------------------------------------------------------- 64-bit definitions
def _exact_attention(q, k, v, window, sinks):
    """One head in 64 bits: q [n, D] are the last n positions of k, v [L, D]."""
    n, length = q.shape[0], k.shape[0]
    i = torch.arange(length - n, length, device=q.device).view(n, 1)
    j = torch.arange(length, device=q.device).view(1, length)
    hide = j > i
    if window:
        hide = hide | ((i - j >= window) & (j >= sinks))
    s = (q @ k.t() / math.sqrt(D)).masked_fill(hide, -math.inf)
    return torch.softmax(s, dim=1) @ v


def _exact_cache(cache, scale, table, i, length):
    """[L, nkv, D] in 64 bits of sequence i."""
    n = -(-length // cache.shape[2])
    ids = table[i, :n].long()
    if scale is None:
        x = cache[ids].double()
    else:
        x = cache.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        x = x * torch.pow(2.0, scale[ids].double() - 127.0)[..., None]
    return x.transpose(1, 2).reshape(-1, cache.shape[1], D)[:length]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "write":
        t, nq = case["tokens"], case["nq"]
        x = s["qkv"].view(t, -1, D)[:, :nq].double()
        half = torch.complex(x[..., : D // 2], x[..., D // 2:])
        power = torch.arange(D // 2, dtype=torch.float64, device="cuda") * (-2.0 / D)
        turn = s["pos"].double()[:, None] * torch.exp(power * math.log(THETA))
        z = half * torch.polar(torch.ones_like(turn), turn)[:, None]
        q = torch.cat([z.real, z.imag], -1).reshape(t, nq * D)
        return {"q": q, "k": None, "v": None, "k_exp": None, "v_exp": None}
    if op == "read":
        ids = s["blocks"].long()
        x = s["cache"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        return x * torch.pow(2.0, s["scale"][ids].double() - 127.0)[..., None]
    nq, nkv = case["nq"], case["nkv"]
    if op == "train":
        x = s["qkv"].detach().view(-1, nq + 2 * nkv, D).double()
        dout = s["dout"].view(-1, nq, D).double()
        o, g = torch.empty_like(dout), torch.zeros_like(x)
        at = 0
        for length in s["lens"]:
            rows = slice(at, at + length)
            for h in range(nq):
                hk = nq + h // (nq // nkv)
                leaf = [x[rows, c].clone().requires_grad_(True) for c in (h, hk, hk + nkv)]
                y = _exact_attention(*leaf, case["window"], case["sinks"])
                o[rows, h] = y.detach()
                for c, gx in zip((h, hk, hk + nkv), torch.autograd.grad(y, leaf, dout[rows, h])):
                    g[rows, c] += gx
                del y
            at += length
        return {"o": o.view(-1, nq * D), "dqkv": g.view(x.shape[0], -1)}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (new, length) in enumerate(zip(s["new"], s["lens"])):
        k = _exact_cache(s["k"], s["ks"], s["table"], i, length)
        v = _exact_cache(s["v"], s["vs"], s["table"], i, length)
        for h in range(nq):
            hk = h // (nq // nkv)
            out[at: at + new, h] = _exact_attention(s["q"][at: at + new, h].double(), k[:, hk], v[:, hk],
                                                    case["window"], case["sinks"])
        at += new
    return out
