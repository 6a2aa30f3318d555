"""Sliding-window attention with sinks on the tcgen05 kernels: forward and gradients against 64 bits."""

import pytest
import torch

from kv8_cases import D, train64
from psrl_b200 import ops
from psrl_b200.ops.attention import attention_kv
from psrl_b200.ops.gemm import check_errors

pytestmark = pytest.mark.gpu
dev = torch.device("cuda", 0)


def _check(got, want):
    for m, (value, bound) in want.items():
        err = (got[m].double() - value).abs()
        worst = float((err / (bound + 1e-30)).max())
        assert worst <= 1, (m, worst)


def _run(lens, nq, nkv, window, sinks, seed=0, tail=0, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens) + tail
    wide = torch.randn(T, (nq + 2 * nkv) * D + pad, generator=gen, device=dev).to(torch.bfloat16)
    if tail:
        wide[-tail:] = float("nan")
    qkv = wide[:, : (nq + 2 * nkv) * D].detach().requires_grad_(True)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    do = torch.randn(T, nq * D, generator=gen, device=dev).to(torch.bfloat16)
    o = ops.varlen_attention(qkv, cu, max(lens), nq, nkv, D, window=window, sinks=sinks)
    (g,) = torch.autograd.grad(o, qkv, do)
    with torch.no_grad():
        assert torch.equal(ops.varlen_attention(qkv, cu, max(lens), nq, nkv, D, window=window, sinks=sinks), o)
    check_errors()
    x, gx = qkv.detach().view(T, -1, D) if not pad else qkv.detach().unflatten(1, (-1, D)), g.view(T, -1, D)
    at = 0
    for n in lens:
        r = slice(at, at + n)
        want = train64(x[r, :nq], x[r, nq:nq + nkv], x[r, nq + nkv:], do.view(T, nq, D)[r], window, sinks)
        _check(dict(o=o.detach().view(T, nq, D)[r], dq=gx[r, :nq], dk=gx[r, nq:nq + nkv], dv=gx[r, nq + nkv:]), want)
        at += n
    if tail:
        assert (o[at:] == 0).all() and (g[at:] == 0).all()


LENS = [1, 17, 128, 129, 255, 256, 257, 300, 700]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 130), (64, 0), (100, 4), (127, 0), (128, 0), (129, 65),
                                          (200, 300), (256, 4), (513, 1), (5000, 0)])
def test_window_fwd_bwd(window, sinks):
    _run(LENS, 4, 2, window, sinks, seed=window)


@pytest.mark.parametrize("nq,nkv", [(16, 2), (28, 4), (8, 8), (3, 1)])
def test_heads(nq, nkv):
    _run([513, 40], nq, nkv, 90, 3, seed=nq, pad=8)


def test_long_window_and_tail():
    _run([2500], 4, 1, 700, 4, seed=1, tail=131)
    _run([40, 1, 5], 4, 1, 9, 0, seed=2, tail=3)


def test_window_over_everything_equals_full():
    lens, nq, nkv = [300, 513], 8, 2
    T = sum(lens)
    qkv = torch.randn(T, (nq + 2 * nkv) * D, device=dev).to(torch.bfloat16).requires_grad_(True)
    cu = torch.tensor([0, 300, 813], dtype=torch.int32, device=dev)
    do = torch.randn(T, nq * D, device=dev).to(torch.bfloat16)
    res = []
    for how in (dict(), dict(window=513), dict(window=3, sinks=600)):
        o = ops.varlen_attention(qkv, cu, 513, nq, nkv, D, **how)
        res.append((o.detach(), torch.autograd.grad(o, qkv, do)[0]))
    # the windowed forward divides by the sum of the rounded weights, the full one by the unrounded sum, so the
    # two differ by at most the sum of their bounds
    x = qkv.detach().view(T, -1, D)
    at = 0
    for n in lens:
        r = slice(at, at + n)
        want = train64(x[r, :nq], x[r, nq:nq + nkv], x[r, nq + nkv:], do.view(T, nq, D)[r])
        heads = {"o": (0, nq), "dq": (0, nq), "dk": (nq, nq + nkv), "dv": (nq + nkv, None)}
        for m, (a, b) in heads.items():
            pick = [(o if m == "o" else g).view(T, -1, D)[r, a:b].double() for o, g in res]
            for y in pick[1:]:
                assert ((y - pick[0]).abs() <= 2 * want[m][1] + 1e-30).all(), m
        assert torch.equal(res[1][0], res[2][0]) and torch.equal(res[1][1], res[2][1])
        at += n


@pytest.mark.parametrize("window,sinks", [(1, 0), (70, 3), (128, 0), (300, 200)])
def test_suffix_queries(window, sinks):
    """Context-parallel form: queries are the last Lq of Lk positions; keys no query sees get zero gradients."""
    pairs, nq, nkv = [(128, 128), (100, 700), (257, 300), (1, 77)], 8, 2
    gen = torch.Generator(device="cuda").manual_seed(window)
    Tq, Tk = sum(p[0] for p in pairs), sum(p[1] for p in pairs)
    q = torch.randn(Tq, nq * D, generator=gen, device=dev).to(torch.bfloat16).requires_grad_(True)
    kv = torch.randn(Tk, 2 * nkv * D, generator=gen, device=dev).to(torch.bfloat16).requires_grad_(True)
    cq, ck = (torch.tensor([0] + [p[c] for p in pairs]).cumsum(0).to(torch.int32).to(dev) for c in (0, 1))
    o = attention_kv(q, kv, cq, ck, 257, 700, nq, nkv, D, window=window, sinks=sinks)
    do = torch.randn(Tq, nq * D, generator=gen, device=dev).to(torch.bfloat16)
    gq, gkv = torch.autograd.grad(o, (q, kv), do)
    check_errors()
    a = b = 0
    for lq, lk in pairs:
        r, s = slice(a, a + lq), slice(b, b + lk)
        kvh = kv.detach().view(Tk, 2 * nkv, D)[s]
        want = train64(q.detach().view(Tq, nq, D)[r], kvh[:, :nkv], kvh[:, nkv:], do.view(Tq, nq, D)[r], window, sinks)
        gk = gkv.view(Tk, 2 * nkv, D)[s]
        _check(dict(o=o.detach().view(Tq, nq, D)[r], dq=gq.view(Tq, nq, D)[r], dk=gk[:, :nkv], dv=gk[:, nkv:]), want)
        a, b = a + lq, b + lk


def test_captured_backward():
    lens, nq, nkv = [300, 129], 4, 2
    T = sum(lens)
    qkv = torch.randn(T, (nq + 2 * nkv) * D, device=dev).to(torch.bfloat16).requires_grad_(True)
    cu = torch.tensor([0, 300, 429], dtype=torch.int32, device=dev)
    do = torch.randn(T, nq * D, device=dev).to(torch.bfloat16)

    def step():
        o = ops.varlen_attention(qkv, cu, 300, nq, nkv, D, window=100, sinks=2)
        return o.detach(), torch.autograd.grad(o, qkv, do)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    with torch.no_grad():
        qkv.copy_(torch.randn_like(qkv))
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)
