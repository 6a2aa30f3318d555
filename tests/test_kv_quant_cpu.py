"""8-bit KV cache: format, references and refusals on the CPU."""

import math

import pytest
import torch

from psrl_b200 import ops
from psrl_b200.ops.kv_quant import FP8, dequantise_ref, quantise_ref


def test_format():
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(257, 128, generator=gen) * torch.exp2(torch.randint(-40, 40, (257, 1), generator=gen).float()))
    x = x.to(torch.bfloat16)
    codes, byte = quantise_ref(x)
    amax = x.float().abs().amax(-1).double()
    unit = torch.exp2(byte.double() - 127)
    assert (amax <= 448 * unit).all() and (amax > 224 * unit).all()      # smallest exponent that holds the vector
    y = dequantise_ref(codes, byte, torch.float64)
    assert torch.equal(y, y.to(torch.bfloat16).double())                 # exact in bf16
    # a code is off by at most half a step: 2^-4 of the value, or half of 2^-9 (the subnormals' step)
    assert ((y - x.double()).abs() <= torch.maximum(x.double().abs() * 2 ** -4, unit[:, None] * 2 ** -10)).all()


@pytest.mark.parametrize("top,byte", [(448.0, 127), (450.0, 128), (0.875, 118), (0.87890625, 119), (0.0, 64),
                                      (1e-30, 64), (3.0e38, 247), (math.inf, 255), (math.nan, 255)])
def test_exponents(top, byte):
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    x[0, 5] = top
    codes, b = quantise_ref(x)
    assert int(b) == byte
    y = dequantise_ref(codes, b)
    if byte == 255:
        assert torch.isnan(y).all()
    else:
        assert torch.isfinite(y).all() and abs(float(y[0, 5]) - float(x[0, 5])) <= max(float(x[0, 5]) * 2 ** -4, 2 ** -73)


def _cache(blocks=5, nkv=2, bs=16, d=64):
    return ([torch.zeros(blocks, nkv, bs, d, dtype=torch.uint8).view(FP8) for _ in range(2)]
            + [torch.zeros(blocks, nkv, bs, dtype=torch.uint8) for _ in range(2)])


def test_write_read_cpu():
    gen = torch.Generator().manual_seed(1)
    T, nq, nkv, d, bs = 21, 4, 2, 64, 16
    qkv = torch.randn(T, (nq + 2 * nkv) * d, generator=gen).to(torch.bfloat16)
    before = qkv.clone()
    pos = torch.randint(0, 5000, (T,), generator=gen, dtype=torch.int32)
    slots = torch.randperm(5 * bs, generator=gen)[:T].to(torch.int32)
    slots[3] = -1
    k, v, ks, vs = _cache()
    q = ops.rope_quant_kv(qkv, pos, nq, nkv, d, 1e6, k, v, ks, vs, slots)
    assert torch.equal(qkv, before)
    kb, vb = torch.zeros(5, nkv, bs, d, dtype=torch.bfloat16), torch.zeros(5, nkv, bs, d, dtype=torch.bfloat16)
    want = ops.rope_qkv_(qkv.clone(), pos, nq, nkv, d, 1e6, k_cache=kb, v_cache=vb, slots=slots)
    assert torch.equal(q, want[:, : nq * d])
    for cache, scale, dense in ((k, ks, kb), (v, vs, vb)):
        got = ops.read_kv_cache(cache, scale, torch.arange(5))
        hit = dense.abs().amax(-1) > 0
        assert torch.equal(scale > 0, hit)
        codes, byte = quantise_ref(dense[hit])
        assert torch.equal(scale[hit], byte) and torch.equal(got[hit], dequantise_ref(codes, byte, torch.bfloat16))
    out = torch.full((7, nkv, bs, d), 3.0, dtype=torch.bfloat16)
    ops.read_kv_cache(k, ks, torch.tensor([4, 0]), out, torch.tensor([1, 6]))
    assert torch.equal(out[1], ops.read_kv_cache(k, ks, torch.tensor([4]))[0]) and (out[[0, 2, 3, 4, 5]] == 3).all()


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (5, 0), (5, 2), (40, 3), (3, 90)])
def test_paged_references_against_64_bits(window, sinks):
    from kv8_cases import D, attention64, pages
    gen = torch.Generator().manual_seed(2)
    lens, new, nq, nkv, bs = [37, 1, 64, 19], [5, 1, 64, 2], 4, 2, 16
    for bits in (8, 16):
        k, v, ks, vs, table, kd, vd = pages(gen, lens, nkv, bs, bits)
        q = torch.randn(sum(new), nq, D, generator=gen).to(torch.bfloat16)
        cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        o = ops.paged_prefill_attention(q, k, v, cu, torch.tensor(lens, dtype=torch.int32), table, max(new),
                                        k_scale=ks, v_scale=vs, window=window, sinks=sinks)
        at = 0
        for i, n in enumerate(new):
            ref, mag = attention64(q[at: at + n], kd[i], vd[i], window, sinks)
            # the output's bf16 rounding, and fp32 sums
            assert ((o[at: at + n].double() - ref).abs() <= ref.abs() * 2 ** -8 + mag * 2 ** -16).all()
            at += n


def test_refusals_cpu():
    from kv8_cases import pages
    gen = torch.Generator().manual_seed(3)
    k, v, ks, vs, table, _, _ = pages(gen, [9], 2, 16, 8)
    q = torch.randn(1, 4, 128).to(torch.bfloat16)
    lens = torch.tensor([9], dtype=torch.int32)
    with pytest.raises(ValueError, match="both k_scale and v_scale"):
        ops.paged_decode_attention(q, k, v, table, lens, k_scale=ks)
    with pytest.raises(ValueError, match="window must be"):
        ops.paged_decode_attention(q, k, v, table, lens, k_scale=ks, v_scale=vs, window=0)
    with pytest.raises(ValueError, match="sinks"):
        ops.paged_decode_attention(q, k, v, table, lens, k_scale=ks, v_scale=vs, window=4, sinks=-1)
    with pytest.raises(ValueError, match="sinks need a window"):
        ops.paged_decode_attention(q, k, v, table, lens, k_scale=ks, v_scale=vs, sinks=4)
    with pytest.raises(ValueError, match="out_blocks"):
        ops.read_kv_cache(k, ks, torch.tensor([0]), out_blocks=torch.tensor([0]))
