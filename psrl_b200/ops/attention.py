"""Attention ops (K1, K2, K3).

* :func:`varlen_attention` — causal attention over a packed batch (training,
  remove-padding), autograd-enabled.  CUDA: forward on the tcgen05 / TMEM
  kernels ``attn_fwd_sm100`` / ``attn_bwd_sm100`` (``csrc/attn_sm100.cu``).
* :func:`paged_prefill_attention` — chunked prefill against the paged KV cache.
* :func:`paged_decode_attention` — one query token per sequence, split-KV.

The PyTorch implementations below are the numerical oracles and the CPU path.
"""

from __future__ import annotations

import math

import torch

from ._ext import ext
from .gemm import _err


# --------------------------------------------------------------- references
def varlen_attention_ref(q, k, v, cu_seqlens, scale, window=None, sinks=0):
    """q [T, nq, d], k/v [T, nkv, d]; causal per sequence; fp32 math."""
    T, nq, d = q.shape
    nkv = k.shape[1]
    g = nq // nkv
    out = torch.zeros(T, nq, d, dtype=q.dtype, device=q.device)
    cu = cu_seqlens.tolist()
    for i in range(len(cu) - 1):
        s, e = cu[i], cu[i + 1]
        if e <= s:
            continue
        qs = q[s:e].float().transpose(0, 1)                     # [nq, L, d]
        ks = k[s:e].float().transpose(0, 1).repeat_interleave(g, 0)
        vs = v[s:e].float().transpose(0, 1).repeat_interleave(g, 0)
        att = (qs @ ks.transpose(1, 2)) * scale
        L = e - s
        pos = torch.arange(L, device=q.device)
        att = att.masked_fill(~window_mask(pos[:, None], pos[None], window, sinks), float("-inf")).softmax(-1)
        out[s:e] = (att @ vs).transpose(0, 1).to(q.dtype)
    return out


def gather_paged_kv(k_cache, v_cache, block_table_row, length):
    bs = k_cache.shape[2]
    nblk = (length + bs - 1) // bs
    blocks = block_table_row[:nblk].long()
    k = k_cache[blocks].permute(0, 2, 1, 3).reshape(-1, k_cache.shape[1], k_cache.shape[3])[:length]
    v = v_cache[blocks].permute(0, 2, 1, 3).reshape(-1, v_cache.shape[1], v_cache.shape[3])[:length]
    return k, v


def window_mask(qpos, kpos, window=None, sinks=0):
    """True where the query at ``qpos`` sees the key at ``kpos``: causal, and with
    a ``window`` only the last ``window`` positions and the first ``sinks``."""
    ok = kpos <= qpos
    if window:
        ok = ok & ((qpos - kpos < window) | (kpos < sinks))
    return ok


def _masked_softmax(att, ok):
    """Softmax over the kept scores; a row that keeps none gives zeros."""
    return torch.where(ok, att.masked_fill(~ok, float("-inf")).softmax(-1), torch.zeros((), dtype=att.dtype,
                                                                                         device=att.device))


def _window_args(window, sinks):
    """(window or 0, sinks) checked: a window is a positive number of positions."""
    if window is None:
        if sinks:
            raise ValueError("sinks need a window (without one every earlier position is visible)")
        return 0, 0
    if int(window) < 1 or int(sinks) < 0:
        raise ValueError(f"window must be >= 1 and sinks >= 0, not {window} and {sinks}")
    return int(window), int(sinks)


def _paged_args(q, k_cache, v_cache, k_scale, v_scale):
    if (k_scale is None) != (v_scale is None):
        raise ValueError("an 8-bit cache needs both k_scale and v_scale")
    want = torch.bfloat16 if k_scale is None else torch.float8_e4m3fn
    if q.is_cuda and (k_cache.dtype != want or v_cache.dtype != want):
        raise ValueError(f"caches of {k_cache.dtype} and {v_cache.dtype} {'with' if k_scale is not None else 'without'} "
                         "exponent bytes: an 8-bit cache is float8_e4m3fn with k_scale and v_scale")


def paged_attention_ref(q, k_cache, v_cache, cu_q, kv_lens, block_table, scale, k_scale=None, v_scale=None,
                        window=None, sinks=0):
    """Queries are the last q_len positions of each context (causal)."""
    T, nq, d = q.shape
    nkv = k_cache.shape[1]
    g = nq // nkv
    out = torch.zeros_like(q)
    cu = cu_q.tolist()
    lens = kv_lens.tolist()
    for i in range(len(cu) - 1):
        s, e = cu[i], cu[i + 1]
        if e <= s:
            continue
        L = lens[i]
        if k_scale is None:
            k, v = gather_paged_kv(k_cache, v_cache, block_table[i], L)
        else:
            from .kv_quant import read_kv_cache
            ids = block_table[i, : -(-L // k_cache.shape[2])].long()
            k, v = (read_kv_cache(c, e, ids).transpose(1, 2).reshape(-1, nkv, d)[:L]
                    for c, e in ((k_cache, k_scale), (v_cache, v_scale)))
        qs = q[s:e].float().transpose(0, 1)
        ks = k.float().transpose(0, 1).repeat_interleave(g, 0)
        vs = v.float().transpose(0, 1).repeat_interleave(g, 0)
        att = (qs @ ks.transpose(1, 2)) * scale            # [nq, ql, L]
        ql = e - s
        qpos = torch.arange(L - ql, L, device=q.device)[:, None]
        kpos = torch.arange(L, device=q.device)[None, :]
        ok = window_mask(qpos, kpos, window, sinks)
        vs = vs.masked_fill(~ok.any(0)[None, :, None], 0.0)
        out[s:e] = (_masked_softmax(att, ok) @ vs).transpose(0, 1).to(q.dtype)
    return out


# ----------------------------------------------------------------- autograd
class _VarlenAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, cu_seqlens, max_seqlen, nq, nkv, d, scale, window, sinks):
        T = qkv.shape[0]
        # a windowed forward also returns what o's rounding left out (o_lo), for D = rowsum(do * o)
        o, lse, o_lo = _varlen_fwd(qkv, cu_seqlens, max_seqlen, nq, nkv, scale, True, window, sinks)
        o = o.view(T, nq, d)
        ctx.save_for_backward(qkv, o, lse, cu_seqlens, o_lo)
        ctx.cfg = (max_seqlen, nq, nkv, d, scale, window, sinks)
        return o.view(T, nq * d)

    @staticmethod
    def backward(ctx, do):
        qkv, o, lse, cu, o_lo = ctx.saved_tensors
        max_seqlen, nq, nkv, d, scale, window, sinks = ctx.cfg
        if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
            qkv = qkv.contiguous()
        # tcgen05 backward (csrc/attn_sm100.cu): dK/dV per key tile and dQ per
        # query tile, written straight into one [T, (nq + 2 nkv) * d] gradient
        dqkv = ext().attn_bwd_sm100(qkv, o.reshape(qkv.shape[0], nq * d), do.contiguous(), lse, cu, max_seqlen,
                                    nq, nkv, scale, _err(qkv.device), window, sinks, o_lo)
        return dqkv, None, None, None, None, None, None, None, None


def varlen_attention_fwd(qkv: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, nq: int, nkv: int,
                         scale: float, want_lse: bool = True, window: int = 0, sinks: int = 0):
    """Forward of causal varlen attention on the tcgen05 kernel
    (``csrc/attn_sm100.cu``): ``qkv`` [T, (nq + 2 nkv) * 128] bf16 ->
    (o [T, nq * 128] bf16, lse [nq, T] fp32 natural log).  ``window`` 0: none."""
    return tuple(_varlen_fwd(qkv, cu_seqlens, max_seqlen, nq, nkv, scale, want_lse, window, sinks)[:2])


def _varlen_fwd(qkv, cu_seqlens, max_seqlen, nq, nkv, scale, want_lse, window, sinks):
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
        qkv = qkv.contiguous()
    return ext().attn_fwd_sm100(qkv, cu_seqlens, int(max_seqlen), int(nq), int(nkv), float(scale), bool(want_lse),
                                _err(qkv.device), int(window), int(sinks))


def varlen_attention(qkv: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, nq: int, nkv: int, d: int,
                     scale: float | None = None, window: int | None = None, sinks: int = 0) -> torch.Tensor:
    """Causal attention over a packed batch; ``qkv`` [T, (nq+2nkv)*d] -> [T, nq*d].

    ``window``: position p of a sequence sees only its last ``window`` positions,
    p included, and the sequence's first ``sinks``; rows of ``qkv`` behind the
    last sequence then give zeros, and zero gradients."""
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    win, sinks = _window_args(window, sinks)
    if qkv.is_cuda and qkv.dtype == torch.bfloat16 and d == 128:
        if not torch.is_grad_enabled() or not qkv.requires_grad:
            return varlen_attention_fwd(qkv, cu_seqlens, max_seqlen, nq, nkv, scale, False, win, sinks)[0]
        return _VarlenAttnFn.apply(qkv, cu_seqlens, int(max_seqlen), nq, nkv, d, scale, win, sinks)
    T = qkv.shape[0]
    q = qkv[:, : nq * d].view(T, nq, d)
    k = qkv[:, nq * d: (nq + nkv) * d].view(T, nkv, d)
    v = qkv[:, (nq + nkv) * d:].view(T, nkv, d)
    return _ref_autograd(q, k, v, cu_seqlens, scale, win, sinks).reshape(T, nq * d)


def _ref_autograd(q, k, v, cu_seqlens, scale, window=0, sinks=0):
    # differentiable reference (CPU training path)
    T, nq, d = q.shape
    nkv = k.shape[1]
    g = nq // nkv
    outs = []
    cu = cu_seqlens.tolist()
    for i in range(len(cu) - 1):
        s, e = cu[i], cu[i + 1]
        if e <= s:
            continue
        qs = q[s:e].transpose(0, 1)
        ks = k[s:e].transpose(0, 1).repeat_interleave(g, 0)
        vs = v[s:e].transpose(0, 1).repeat_interleave(g, 0)
        L = e - s
        pos = torch.arange(L, device=q.device)
        mask = ~window_mask(pos[:, None], pos[None], window, sinks)
        att = ((qs @ ks.transpose(1, 2)) * scale).masked_fill(mask, float("-inf")).softmax(-1)
        outs.append((att @ vs).transpose(0, 1))
    if window and cu[-1] < T:
        outs.append(q.new_zeros(T - cu[-1], nq, d))
    return torch.cat(outs, 0) if outs else q.new_zeros(0, nq, d)


def paged_prefill_attention(q, k_cache, v_cache, cu_q, kv_lens, block_table, max_q_len, scale=None, k_scale=None,
                            v_scale=None, window=None, sinks=0):
    """A chunk of new tokens per sequence against its paged context, which holds
    the chunk's own keys already: q [T, nq, d] (view ok), sequence b's queries
    [cu_q[b], cu_q[b+1]) being its last positions; returns [T, nq, d].

    ``k_scale`` / ``v_scale``: exponent bytes of an 8-bit cache (:mod:`.kv_quant`).
    ``window`` / ``sinks``: see :func:`window_mask`."""
    d = q.shape[-1]
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    win, sinks = _window_args(window, sinks)
    _paged_args(q, k_cache, v_cache, k_scale, v_scale)
    if q.is_cuda and d == 128:
        if k_scale is None and not win:
            return ext().attn_paged_prefill(q, k_cache, v_cache, cu_q, kv_lens, block_table, int(max_q_len), scale)
        if not (q.stride(2) == 1 and q.stride(1) % 8 == 0 and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0):
            q = q.contiguous()
        return ext().attn_paged_chunk(q, k_cache, v_cache, k_scale, v_scale, cu_q, kv_lens, block_table,
                                      int(max_q_len), scale, win, sinks, _err(q.device))
    return paged_attention_ref(q, k_cache, v_cache, cu_q, kv_lens, block_table, scale, k_scale, v_scale, window, sinks)


def decode_splits(batch: int, nkv: int, max_ctx: int) -> int:
    return int(ext().decode_num_splits(batch, nkv, max_ctx))


def paged_decode_attention(q, k_cache, v_cache, block_table, kv_lens, scale=None, splits: int | None = None,
                           scratch: torch.Tensor | None = None, stages: int = 0, k_scale=None, v_scale=None,
                           window: int | None = None, sinks: int = 0):
    """One new token per sequence against its paged context: q [B, nq, d] ->
    [B, nq, d]; kv_lens include the current token.

    ``k_scale`` / ``v_scale``: exponent bytes of an 8-bit cache (:mod:`.kv_quant`),
    whose kernel shares the work out by itself (``splits``, ``scratch`` and
    ``stages`` do not apply).  ``window`` / ``sinks``: see :func:`window_mask`."""
    d = q.shape[-1]
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    win, sinks = _window_args(window, sinks)
    _paged_args(q, k_cache, v_cache, k_scale, v_scale)
    if q.is_cuda and d == 128:
        if not (q.stride(2) == 1 and q.stride(1) == d and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0):
            q = q.contiguous()
        if k_scale is not None:
                return ext().attn_decode_fp8(q, k_cache, v_cache, k_scale, v_scale, block_table, kv_lens, scale, win,
                                         sinks, _err(q.device))
        if splits is None:
            ctx = int(block_table.shape[1] * k_cache.shape[2])
            splits = decode_splits(q.shape[0], k_cache.shape[1], min(ctx, win + sinks) if win else ctx)
        return ext().attn_decode(q, k_cache, v_cache, block_table, kv_lens, scale, int(splits), scratch, int(stages),
                                 win, sinks)
    B = q.shape[0]
    cu = torch.arange(B + 1, dtype=torch.int32, device=q.device)
    return paged_attention_ref(q, k_cache, v_cache, cu, kv_lens, block_table, scale, k_scale, v_scale, window, sinks)


# ------------------------------------------- queries against separate keys
def attention_kv_ref(q, k, v, cu_q, cu_k, scale, window=None, sinks=0):
    """q [Tq, nq, d]; k / v [Tk, nkv, d]; sequence b's queries
    [cu_q[b], cu_q[b+1]) are the last of its key positions [cu_k[b], cu_k[b+1]),
    so query row p sees keys 0 .. p + Lk - Lq.  Differentiable, fp32 math."""
    Tq, nq, d = q.shape
    g = nq // k.shape[1]
    outs = []
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cq) - 1):
        qs, qe, ks, ke = cq[b], cq[b + 1], ck[b], ck[b + 1]
        Lq, Lk = qe - qs, ke - ks
        if Lq <= 0:
            continue
        qq = q[qs:qe].float().transpose(0, 1)
        kk = k[ks:ke].float().transpose(0, 1).repeat_interleave(g, 0)
        vv = v[ks:ke].float().transpose(0, 1).repeat_interleave(g, 0)
        rows = torch.arange(Lq, device=q.device)[:, None] + (Lk - Lq)
        mask = ~window_mask(rows, torch.arange(Lk, device=q.device)[None, :], window, sinks)
        att = ((qq @ kk.transpose(1, 2)) * scale).masked_fill(mask, float("-inf")).softmax(-1)
        outs.append((att @ vv).transpose(0, 1).to(q.dtype))
    return torch.cat(outs, 0) if outs else q.new_zeros(0, nq, d)


class _AttnKVFn(torch.autograd.Function):
    """tcgen05 forward / backward of queries against separately stored keys
    (``attn_fwd_sm100_kv`` / ``attn_bwd_sm100_kv``)."""

    @staticmethod
    def forward(ctx, q, kv, cu_q, cu_k, max_q, max_k, nq, nkv, scale, window, sinks):
        o, lse, o_lo = ext().attn_fwd_sm100_kv(q, kv, cu_q, cu_k, int(max_q), int(nq), int(nkv), float(scale), True,
                                         _err(q.device), window, sinks)
        ctx.save_for_backward(q, kv, o, lse, cu_q, cu_k, o_lo)
        ctx.cfg = (max_q, max_k, nq, nkv, scale, window, sinks)
        return o

    @staticmethod
    def backward(ctx, do):
        q, kv, o, lse, cu_q, cu_k, o_lo = ctx.saved_tensors
        max_q, max_k, nq, nkv, scale, window, sinks = ctx.cfg
        dq, dkv = ext().attn_bwd_sm100_kv(q, kv, o, do.contiguous(), lse, cu_q, cu_k, int(max_q), int(max_k),
                                          int(nq), int(nkv), float(scale), _err(q.device), window, sinks, o_lo)
        return dq, dkv, None, None, None, None, None, None, None, None, None


def attention_kv(q: torch.Tensor, kv: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor, max_q: int, max_k: int,
                 nq: int, nkv: int, d: int, scale: float | None = None, window: int | None = None,
                 sinks: int = 0) -> torch.Tensor:
    """Causal attention of queries ``q`` [Tq, nq * d] against keys / values
    ``kv`` [Tk, 2 nkv * d] (k heads, then v heads) where each sequence's queries
    are the last ``Lq`` of its ``Lk >= Lq`` key positions; returns [Tq, nq * d].
    Context-parallel attention runs a rank's query chunks through this against
    the gathered key prefix.  ``window`` / ``sinks`` as in :func:`varlen_attention`."""
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    win, sinks = _window_args(window, sinks)
    if q.is_cuda and q.dtype == torch.bfloat16 and d == 128:
        if q.stride(1) != 1 or q.stride(0) % 8 or q.data_ptr() % 16:
            q = q.contiguous()
        return _AttnKVFn.apply(q, kv.contiguous(), cu_q, cu_k, int(max_q), int(max_k), nq, nkv, scale, win,
                              sinks)
    Tq, Tk = q.shape[0], kv.shape[0]
    o = attention_kv_ref(q.reshape(Tq, -1)[:, : nq * d].reshape(Tq, nq, d), kv[:, : nkv * d].reshape(Tk, nkv, d),
                         kv[:, nkv * d:].reshape(Tk, nkv, d), cu_q, cu_k, scale, win, sinks)
    return o.reshape(Tq, nq * d)
