"""8-bit KV cache on the GPU: quantised write, read back, decode and chunk attention."""

import math

import pytest
import torch

from kv8_cases import D, attention64, pages
from psrl_b200 import ops
from psrl_b200.ops.kv_quant import FP8, dequantise_ref, quantise_ref

pytestmark = pytest.mark.gpu
dev = torch.device("cuda", 0)


def _cuda(*xs):
    return [x.to(dev) if x is not None else None for x in xs]


def _fp8(x):
    return x.view(torch.uint8).cpu()


# -------------------------------------------------------------- write, read
@pytest.mark.parametrize("T,nq,nkv,d,bs", [(1, 16, 2, 128, 64), (7, 28, 4, 128, 16), (24, 4, 2, 64, 32),
                                           (333, 8, 8, 128, 48), (4099, 32, 8, 128, 64), (600, 5, 1, 64, 16)])
def test_write_equals_reference(T, nq, nkv, d, bs):
    gen = torch.Generator().manual_seed(T)
    blocks = -(-T // bs) + 2
    wide = torch.randn(T, (nq + 2 * nkv) * d + 8, generator=gen)
    wide[:, 3::41] *= 2.0 ** torch.randint(-60, 60, (T, 1), generator=gen)
    wide[T // 2, :d] = 0
    wide[T // 3, -d - 8:] = 0                        # a zero vector
    wide[T // 4, nq * d + 5] = math.nan
    wide[T // 5, (nq + nkv) * d + 1] = -math.inf
    qkv = wide.to(torch.bfloat16)[:, : (nq + 2 * nkv) * d]          # strided rows
    pos = torch.randint(0, 65536, (T,), generator=gen, dtype=torch.int32)
    slots = torch.randperm(blocks * bs, generator=gen)[:T].to(torch.int32)
    slots[::9] = -1
    if T > 5:
        slots[4] = blocks * bs + 3                   # outside the cache: skipped
    mk = lambda: ([torch.full((blocks, nkv, bs, d), 7, dtype=torch.uint8).view(FP8) for _ in range(2)]  # noqa: E731
                  + [torch.full((blocks, nkv, bs), 9, dtype=torch.uint8) for _ in range(2)])
    ref, got = mk(), _cuda(*mk())
    want = ops.rope_quant_kv(qkv, pos, nq, nkv, d, 1e6, *ref, slots)
    q = ops.rope_quant_kv(qkv.to(dev), pos.to(dev), nq, nkv, d, 1e6, *got, slots.to(dev))
    assert torch.equal(q.cpu().view(torch.int16), want.view(torch.int16)) or torch.equal(
        torch.nan_to_num(q.cpu().float()), torch.nan_to_num(want.float()))
    for a, b in zip(got[2:], ref[2:]):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(got[:2], ref[:2]):
        assert torch.equal(_fp8(a), b.view(torch.uint8))


def test_write_position_outside_table_is_nan():
    nq, nkv, d, bs = 4, 2, 128, 16
    got = _cuda(*([torch.zeros(1, nkv, bs, d, dtype=torch.uint8).view(FP8) for _ in range(2)]
                  + [torch.zeros(1, nkv, bs, dtype=torch.uint8) for _ in range(2)]))
    qkv = torch.randn(2, (nq + 2 * nkv) * d, device=dev).to(torch.bfloat16)
    pos = torch.tensor([1 << 20, -1], dtype=torch.int32, device=dev)
    q = ops.rope_quant_kv(qkv, pos, nq, nkv, d, 1e6, *got, torch.tensor([0, 1], dtype=torch.int32, device=dev))
    assert torch.isnan(q).all() and (got[2][0, :, :2] == 255).all() and (got[3][0, :, :2] < 255).all()


@pytest.mark.parametrize("n,nkv,bs,d", [(1, 1, 16, 64), (5, 2, 64, 128), (37, 8, 48, 128)])
def test_read_equals_reference(n, nkv, bs, d):
    gen = torch.Generator().manual_seed(n)
    codes = torch.randint(0, 256, (n + 3, nkv, bs, d), generator=gen, dtype=torch.uint8).view(FP8)
    scale = torch.randint(0, 256, (n + 3, nkv, bs), generator=gen, dtype=torch.uint8)
    ids = torch.randperm(n + 3, generator=gen)[:n].to(torch.int32)
    want = dequantise_ref(codes.view(torch.uint8)[ids.long()].view(FP8), scale[ids.long()], torch.bfloat16)
    got = ops.read_kv_cache(codes.to(dev), scale.to(dev), ids.to(dev)).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float(), nan=5.0), torch.nan_to_num(want.float(), nan=5.0))
    out = torch.full((n + 9, nkv, bs, d), 3.0, dtype=torch.bfloat16, device=dev)
    to = torch.randperm(n + 9, generator=gen)[:n].to(torch.int32)
    to[0] = n + 9                                    # outside: skipped
    ops.read_kv_cache(codes.to(dev), scale.to(dev), ids.to(dev), out, to.to(dev))
    keep = torch.ones(n + 9, dtype=torch.bool)
    keep[to[1:].long()] = False
    assert (out[keep.to(dev)] == 3).all()
    assert torch.equal(torch.nan_to_num(out[to[1:].long().to(dev)].cpu().float(), nan=5.0),
                       torch.nan_to_num(want[1:].float(), nan=5.0))


# ------------------------------------------------------------------- decode
def _decode_bound(ref, mag, bits):
    """bf16 output: half a step, 2^-8 of the value.  Weights: rounded to f16 (8-bit cache, 2^-11) or bf16 (2^-8);
    scores and exponentials in fp32 (|score| < 2^7 here: 2^7 * 2^-24 * few < 2^-15)."""
    return ref.abs() * 2 ** -8 + mag * ((2 ** -11 if bits == 8 else 2 ** -8) + 2 ** -14)


def _check_decode(lens, nq, nkv, bs, bits, window, sinks, seed=0, q_pad=0, **how):
    gen = torch.Generator().manual_seed(seed)
    k, v, ks, vs, table, kd, vd = pages(gen, lens, nkv, bs, bits)
    q = torch.randn(len(lens), nq * D + q_pad, generator=gen).to(torch.bfloat16)
    dk, dv, dks, dvs, dt, dq = _cuda(k, v, ks, vs, table, q)
    o = ops.paged_decode_attention(dq[:, : nq * D].view(len(lens), nq, D) if not q_pad else
                                   dq[:, : nq * D].unflatten(1, (nq, D)), dk, dv, dt,
                                   torch.tensor(lens, dtype=torch.int32, device=dev), k_scale=dks, v_scale=dvs,
                                   window=window, sinks=sinks, **how).cpu().double()
    for i in range(len(lens)):
        ref, mag = attention64(q[i, : nq * D].view(1, nq, D), kd[i], vd[i], window, sinks)
        assert ((o[i] - ref[0]).abs() <= _decode_bound(ref[0], mag[0], bits)).all(), (i, lens[i])


LENS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000, 0, 777, 1]


@pytest.mark.parametrize("nq,nkv", [(16, 2), (28, 4), (8, 8), (32, 2), (3, 1)])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_decode_fp8(nq, nkv, bs):
    _check_decode(LENS, nq, nkv, bs, 8, None, 0, seed=nq + bs, q_pad=8 if bs == 32 else 0)


@pytest.mark.parametrize("lens", [[1], [517], [5000], [3] * 300, [4000, 1, 1, 1], [0, 0], [0, 70, 0]])
def test_decode_fp8_shares(lens):
    _check_decode(lens, 16, 2, 64, 8, None, 0, seed=len(lens))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (100, 4), (100, 70), (128, 200), (777, 3), (5000, 9)])
def test_decode_window(bits, window, sinks):
    for bs in (16, 64):
        _check_decode(LENS, 16, 2, bs, bits, window, sinks, seed=window + sinks)


@pytest.mark.parametrize("splits", [1, 2, 7, 32])
def test_decode_window_bf16_splits(splits):
    _check_decode(LENS, 8, 2, 64, 16, 300, 70, seed=splits, splits=splits)


def test_decode_fp8_extreme_vectors():
    """Exponents far apart, zero vectors, tiny and huge queries; NaN vectors reach exactly the rows that see them."""
    gen = torch.Generator().manual_seed(5)
    nq, nkv, bs, L = 8, 2, 64, 200
    k, v, ks, vs, table, kd, vd = pages(gen, [L, L, L], nkv, bs, 8)
    size = torch.exp2(torch.randint(-30, 30, (L, nkv, 1), generator=gen).double())
    size[::7] = 0
    for c, (cache, scale, dense) in enumerate(((k, ks, kd), (v, vs, vd))):
        if c == 0:
            continue
        x = (torch.randn(L, nkv, D, generator=gen).double() * size).to(torch.bfloat16)
        codes, byte = quantise_ref(x)
        p = torch.arange(L)
        cache.view(torch.uint8)[table[1, : 4].long()[p // bs], :, p % bs] = codes.view(torch.uint8)
        scale[table[1, : 4].long()[p // bs], :, p % bs] = byte
        dense[1] = dequantise_ref(codes, byte, torch.float64)
    vs[table[2, 1].long(), 1, 3] = 255              # position 67, kv head 1 of sequence 2
    q = torch.randn(3, nq, D, generator=gen)
    q[0, 0] *= 1e-30
    q[0, 1] = 0
    q[0, 2, 1:] *= 1e-6
    q = q.to(torch.bfloat16)
    dk, dv, dks, dvs, dt, dq = _cuda(k, v, ks, vs, table, q)
    run = lambda w: ops.paged_decode_attention(dq, dk, dv, dt, torch.full((3,), L, dtype=torch.int32, device=dev),  # noqa: E731
                                               k_scale=dks, v_scale=dvs, window=w).cpu().double()
    o = run(None)
    for i in (0, 1):
        ref, mag = attention64(q[i:i + 1], kd[i], vd[i])
        assert ((o[i] - ref[0]).abs() <= _decode_bound(ref[0], mag[0], 8)).all(), i
    assert torch.isnan(o[2, 4:]).all() and torch.isfinite(o[2, :4]).all()
    assert torch.isfinite(run(L - 68)).all() and torch.isnan(run(L - 67)[2, 4:]).all()


def test_decode_fp8_graph_stream_and_workspace():
    """Captured on a side stream, replayed with other lengths; two graphs do not share a workspace."""
    gen = torch.Generator().manual_seed(9)
    lens, nq, nkv, bs = [900, 130, 64, 2000], 16, 2, 64
    k, v, ks, vs, table, kd, vd = pages(gen, lens, nkv, bs, 8)
    q = torch.randn(4, nq, D, generator=gen).to(torch.bfloat16)
    dk, dv, dks, dvs, dt, dq = _cuda(k, v, ks, vs, table, q)
    dl = torch.tensor(lens, dtype=torch.int32, device=dev)
    run = lambda: ops.paged_decode_attention(dq, dk, dv, dt, dl, k_scale=dks, v_scale=dvs)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for new in ([900, 130, 64, 2000], [1, 0, 33, 1999], [64, 65, 1, 700]):
        dl.copy_(torch.tensor(new, dtype=torch.int32))
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        torch.cuda.synchronize()
        for o in outs:
            for i, n in enumerate(new):
                ref, mag = attention64(q[i:i + 1], kd[i][:n], vd[i][:n])
                assert ((o[i].cpu().double() - ref[0]).abs() <= _decode_bound(ref[0], mag[0], 8)).all()


def test_decode_is_repeatable():
    gen = torch.Generator().manual_seed(4)
    k, v, ks, vs, table, _, _ = pages(gen, [3000, 5, 800], 2, 64, 8)
    dk, dv, dks, dvs, dt = _cuda(k, v, ks, vs, table)
    q = torch.randn(3, 16, D, device=dev).to(torch.bfloat16)
    lens = torch.tensor([3000, 5, 800], dtype=torch.int32, device=dev)
    outs = [ops.paged_decode_attention(q, dk, dv, dt, lens, k_scale=dks, v_scale=dvs) for _ in range(5)]
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_refusals():
    gen = torch.Generator().manual_seed(3)
    k, v, ks, vs, table = _cuda(*pages(gen, [9], 2, 16, 8)[:5])
    q = torch.randn(1, 4, D, device=dev).to(torch.bfloat16)
    lens = torch.tensor([9], dtype=torch.int32, device=dev)
    call = ops.paged_decode_attention
    with pytest.raises(ValueError, match="8-bit cache"):
        call(q, k, v, table, lens)
    with pytest.raises(ValueError, match="8-bit cache"):
        call(q, k.float().to(torch.bfloat16), v, table, lens, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="exponents"):
        call(q, k, v, table, lens, k_scale=ks[:1], v_scale=vs)
    with pytest.raises(RuntimeError, match="exponents"):
        call(q, k, v, table, lens, k_scale=ks.cpu(), v_scale=vs)
    with pytest.raises(RuntimeError, match="kv_lens"):
        call(q, k, v, table, lens.long(), k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="block_table"):
        call(q, k, v, table.long(), lens, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="GQA"):
        call(q[:, :3], k, v, table, lens, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="wrong dtype"):
        call(q.float(), k, v, table, lens, k_scale=ks, v_scale=vs)
    odd = torch.zeros(3, 2, 24, D, dtype=torch.uint8, device=dev).view(FP8)
    with pytest.raises(RuntimeError, match="power of two"):
        call(q, odd, odd, table, lens, k_scale=torch.zeros(3, 2, 24, dtype=torch.uint8, device=dev),
             v_scale=torch.zeros(3, 2, 24, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError, match="head_dim"):
        small = torch.zeros(1, 1, 16, 32, dtype=torch.uint8, device=dev).view(FP8)
        ops.read_kv_cache(small, torch.zeros(1, 1, 16, dtype=torch.uint8, device=dev),
                          torch.zeros(1, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="slots"):
        ops.rope_quant_kv(torch.zeros(2, 8 * D, device=dev, dtype=torch.bfloat16),
                          torch.zeros(2, dtype=torch.int32, device=dev), 4, 2, D, 1e6, k, v, ks, vs,
                          torch.zeros(3, dtype=torch.int32, device=dev))
    assert call(q[:0], k, v, table[:0], lens[:0], k_scale=ks, v_scale=vs).shape == (0, 4, D)


# -------------------------------------------------------------------- chunk
def _check_chunk(new, lens, nq, nkv, bs, bits, window=None, sinks=0, seed=0, pad=0, tail=0, max_q=None):
    from psrl_b200.ops.gemm import check_errors
    gen = torch.Generator().manual_seed(seed)
    k, v, ks, vs, table, kd, vd = pages(gen, lens, nkv, bs, bits)
    T = sum(new) + tail
    q = torch.randn(T, nq * (D + pad), generator=gen).to(torch.bfloat16).view(T, nq, D + pad)[:, :, :D]
    if tail:
        q = q.clone()
        q[-tail:] = math.nan
    dk, dv, dks, dvs, dt = _cuda(k, v, ks, vs, table)
    dq = torch.empty(T, nq, D + pad, dtype=torch.bfloat16, device=dev)[:, :, :D]
    dq.copy_(q)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)
    o = ops.paged_prefill_attention(dq, dk, dv, cu, torch.tensor(lens, dtype=torch.int32, device=dev), dt,
                                    max_q or max(new), k_scale=dks, v_scale=dvs, window=window, sinks=sinks).cpu().double()
    check_errors()
    at = 0
    for i, n in enumerate(new):
        m = min(n, lens[i])                          # queries before position 0 see nothing: zeros
        ref, mag = attention64(q[at + n - m: at + n], kd[i], vd[i], window, sinks)
        # P is bf16 whatever the cache's type
        worst = ((o[at + n - m: at + n] - ref).abs() / (_decode_bound(ref, mag, 16) + 1e-30)).max() if m else 0
        assert worst <= 1, (i, n, lens[i], float(worst))
        assert (o[at: at + n - m] == 0).all()
        at += n
    assert (o[at:] == 0).all()


NEW = [1, 5, 16, 17, 64, 130, 300, 3, 0, 2, 1]
CTX = [1, 200, 16, 129, 1000, 130, 511, 3, 40, 1, 0]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("nq,nkv", [(16, 2), (28, 4), (8, 8), (32, 2), (3, 1), (64, 1)])
def test_chunk_heads(nq, nkv, bits):
    win = dict() if bits == 8 else dict(window=150, sinks=5)
    _check_chunk(NEW, CTX, nq, nkv, 64, bits, seed=nq, pad=8 if nq == 28 else 0, tail=9, **win)


@pytest.mark.parametrize("bs", [16, 32, 128, 512])
def test_chunk_pages(bs):
    _check_chunk(NEW, CTX, 8, 2, bs, 8, seed=bs)
    _check_chunk(NEW, CTX, 8, 2, bs, 16, 100, 4, seed=bs)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (128, 130), (200, 4), (5000, 0)])
def test_chunk_window(bits, window, sinks):
    _check_chunk(NEW, CTX, 8, 2, 64, bits, window, sinks, seed=window)


def test_chunk_split_and_whole():
    _check_chunk([5], [3000], 16, 2, 64, 8, seed=1)                      # few tokens, long context: keys are split
    _check_chunk([5, 1, 33], [3000, 2, 900], 8, 8, 64, 8, seed=2)
    _check_chunk([5], [3000], 16, 2, 64, 8, 300, 70, seed=3)
    _check_chunk([1500], [1500], 32, 8, 64, 8, seed=4, max_q=4000)       # many blocks: whole; max_q may be an upper bound


def test_chunk_extreme_exponents_and_nan():
    gen = torch.Generator().manual_seed(5)
    nq, nkv, bs, L, n = 8, 2, 64, 300, 40
    k, v, ks, vs, table, kd, vd = pages(gen, [L], nkv, bs, 8)
    p = torch.arange(L)
    at = table[0, :5].long()[p // bs]
    size = torch.exp2(torch.randint(-60, 110, (L, nkv, 1), generator=gen).double())
    size[::7] = 0
    codes, byte = quantise_ref((torch.randn(L, nkv, D, generator=gen).double() * size).to(torch.bfloat16))
    v.view(torch.uint8)[at, :, p % bs] = codes.view(torch.uint8)
    vs[at, :, p % bs] = byte
    vd = dequantise_ref(codes, byte, torch.float64)
    q = torch.randn(n, nq, D, generator=gen).to(torch.bfloat16)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    call = lambda **w: ops.paged_prefill_attention(  # noqa: E731
        *_cuda(q, k, v), cu, torch.tensor([L], dtype=torch.int32, device=dev), table.to(dev), n,
        k_scale=ks.to(dev), v_scale=vs.to(dev), **w).cpu().double()
    ref, mag = attention64(q, kd[0], vd)
    assert ((call() - ref).abs() <= _decode_bound(ref, mag, 16)).all()
    # a NaN value vector at position 280 (kv head 1): only the rows that see it
    vs[at[280], 1, 280 % bs] = 255
    o = call()
    assert torch.isnan(o[280 - (L - n):, 4:]).all()
    assert torch.isfinite(o[: 280 - (L - n)]).all() and torch.isfinite(o[:, :4]).all()
    o = call(window=10)
    first = 280 - (L - n)
    assert torch.isnan(o[first: first + 10, 4:]).all() and torch.isfinite(o[first + 10:]).all()


def test_chunk_graph():
    gen = torch.Generator().manual_seed(6)
    nq, nkv, lens, new = 16, 2, [700, 90], [30, 64]
    k, v, ks, vs, table, kd, vd = pages(gen, lens, nkv, 64, 8)
    q = torch.randn(sum(new), nq, D, generator=gen).to(torch.bfloat16)
    dk, dv, dks, dvs, dt, dq = _cuda(k, v, ks, vs, table, q)
    cu = torch.tensor([0, 30, 94], dtype=torch.int32, device=dev)
    dl = torch.tensor(lens, dtype=torch.int32, device=dev)
    run = lambda: ops.paged_prefill_attention(dq, dk, dv, cu, dl, dt, 64, k_scale=dks, v_scale=dvs)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = run()
    for new_lens in ([700, 90], [31, 64], [256, 65]):
        dl.copy_(torch.tensor(new_lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, run())
        for i, (a, b) in enumerate(((0, 30), (30, 94))):
            ref, mag = attention64(q[a:b], kd[i][:new_lens[i]], vd[i][:new_lens[i]])
            assert ((o[a:b].cpu().double() - ref).abs() <= _decode_bound(ref, mag, 16)).all()


def test_chunk_refusals():
    gen = torch.Generator().manual_seed(3)
    k, v, ks, vs, table = _cuda(*pages(gen, [9], 2, 16, 8)[:5])
    q = torch.randn(4, 4, D, device=dev).to(torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    lens = torch.tensor([9], dtype=torch.int32, device=dev)
    call = ops.paged_prefill_attention
    with pytest.raises(ValueError, match="both k_scale"):
        call(q, k, v, cu, lens, table, 4, k_scale=ks)
    with pytest.raises(RuntimeError, match="cu_q"):
        call(q, k, v, cu.long(), lens, table, 4, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="block_table"):
        call(q, k, v, cu, lens, table[:, 0], 4, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="kv_lens"):
        call(q, k, v, cu, lens.cpu(), table, 4, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="multiple"):
        call(q[:, :3], k, v, cu, lens, table, 4, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="window"):
        call(q, k, v, cu, lens, table, 4, k_scale=ks, v_scale=vs, window=0)
    assert call(q[:0], k, v, cu[:1] * 0, lens[:0], table[:0], 0, k_scale=ks, v_scale=vs).shape == (0, 4, D)
