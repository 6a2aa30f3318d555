"""Sliding-window attention: CPU references against 64 bits and differences, and refusals."""

import pytest
import torch

from kv8_cases import attention64
from psrl_b200 import ops
from psrl_b200.ops.attention import attention_kv, varlen_attention_ref, window_mask


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 2), (4, 0), (7, 3), (40, 2), (5, 100)])
def test_references(window, sinks):
    gen = torch.Generator().manual_seed(0)
    lens, nq, nkv, d = [11, 1, 30], 4, 2, 128
    T = sum(lens)
    qkv = torch.randn(T, (nq + 2 * nkv) * d, generator=gen)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    o = ops.varlen_attention(qkv, cu, max(lens), nq, nkv, d, window=window, sinks=sinks).view(T, nq, d)
    q, k, v = (x.reshape(T, -1, d) for x in qkv.split([nq * d, nkv * d, nkv * d], -1))
    r = varlen_attention_ref(q, k, v, cu, d ** -0.5, window, sinks)
    kv = attention_kv(qkv[:, : nq * d], qkv[:, nq * d:], cu, cu, max(lens), max(lens), nq, nkv, d, window=window,
                      sinks=sinks).view(T, nq, d)
    at = 0
    for n in lens:
        ref, mag = attention64(q[at: at + n], k[at: at + n].double(), v[at: at + n].double(), window, sinks)
        for got in (o, r, kv):
            assert ((got[at: at + n].double() - ref).abs() <= mag * 2 ** -17).all()
        at += n


def test_window_of_the_context_is_full_attention():
    pos = torch.arange(9)
    full = window_mask(pos[:, None], pos[None])
    assert torch.equal(window_mask(pos[:, None], pos[None], 9, 0), full)
    assert torch.equal(window_mask(pos[:, None], pos[None], 2, 9), full)
    assert int(window_mask(pos[:, None], pos[None], 2, 0).sum()) == 17


def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(1)
    lens, nq, nkv, d = [6, 3], 2, 1, 128
    cu = torch.tensor([0, 6, 9], dtype=torch.int32)
    qkv = torch.randn(11, (nq + 2 * nkv) * d, generator=gen, dtype=torch.float64, requires_grad=True)
    out = ops.varlen_attention(qkv, cu, 6, nq, nkv, d, window=2, sinks=1)
    w = torch.randn(out.shape, generator=gen, dtype=torch.float64)
    (out * w).sum().backward()
    assert (out[9:] == 0).all() and (qkv.grad[9:] == 0).all()
    step = torch.randn(qkv.shape, generator=gen, dtype=torch.float64)
    f = lambda e: float((ops.varlen_attention((qkv + e * step).detach(), cu, 6, nq, nkv, d, window=2, sinks=1) * w).sum())  # noqa: E731
    assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - float((qkv.grad * step).sum())) < 1e-6


@pytest.mark.parametrize("how", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(sinks=2)])
def test_refusals(how):
    qkv = torch.zeros(4, 4 * 128)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="window|sinks"):
        ops.varlen_attention(qkv, cu, 4, 2, 1, 128, **how)
    with pytest.raises(ValueError, match="window|sinks"):
        attention_kv(qkv[:, :256], qkv[:, 256:], cu, cu, 4, 4, 2, 1, 128, **how)
