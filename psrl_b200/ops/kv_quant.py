"""8-bit paged KV cache: the quantised write of new keys and values, fused with
their rotary embedding, and pages read back as bf16 (``csrc/kv_fp8.cu``).

A cache is a pair of tensors per layer for the keys and one for the values:

* codes ``[blocks, nkv, block_size, d]`` float8_e4m3fn;
* exponents ``[blocks, nkv, block_size]`` uint8, one per (token, kv head) vector.

``value = code * 2^(byte - 127)``, with the smallest exponent in [-63, 120]
whose 448 * 2^e reaches the vector's largest magnitude (-63 for zeros).  The
power-of-two scale loses a float code nothing and makes the value exact in
bf16.  A vector with a NaN or an infinity gets byte 255 and reads as NaN.

:func:`psrl_b200.ops.paged_decode_attention` and
:func:`psrl_b200.ops.paged_prefill_attention` read such a cache when given its
exponents.  The PyTorch functions below are the numerical oracles and the CPU
path.
"""

from __future__ import annotations

import torch

from ._ext import ext
from .rope import apply_rope_ref, rope_tables

FP8 = torch.float8_e4m3fn
_ROPE: dict = {}          # (theta, d, device) -> rotary tables, as rope_tables keeps them


def _i32(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype == torch.int32 else x.int()


# --------------------------------------------------------------- references
def quantise_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., d] -> (codes float8_e4m3fn [..., d], exponent bytes uint8 [...])."""
    x = x.float()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    m, e = torch.frexp(torch.where(bad, torch.zeros_like(amax), amax))   # amax = m 2^e, m in [1/2, 1)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-63, 120)               # 448 = 0.875 * 2^9
    e = torch.where(m == 0, torch.full_like(e, -63), e)
    codes = torch.ldexp(x.masked_fill(bad[..., None], 0.0), -e[..., None]).to(FP8)
    return codes, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def dequantise_ref(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """Values of cache rows: codes [..., d], exponent bytes [...]."""
    x = torch.ldexp(codes.float(), scale.to(torch.int32)[..., None] - 127)
    return x.masked_fill((scale == 255)[..., None], float("nan")).to(dtype)


def write_kv_cache_fp8_ref(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    """k / v [T, nkv, d]; slots outside the cache are skipped."""
    bs = k_cache.shape[2]
    sl = slots.long()
    ok = (sl >= 0) & (sl < k_cache.shape[0] * bs)
    blk, off = sl[ok] // bs, sl[ok] % bs
    for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        codes, byte = quantise_ref(x[ok])
        cache.view(torch.uint8)[blk, :, off] = codes.view(torch.uint8)
        scale[blk, :, off] = byte


# ---------------------------------------------------------------------- ops
def rope_quant_kv(qkv: torch.Tensor, positions: torch.Tensor, nq: int, nkv: int, d: int, theta, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  slots: torch.Tensor) -> torch.Tensor:
    """Rotate the queries and keys of ``qkv`` [T, (nq + 2 nkv) * d] (left as it
    is) and write the rotated keys, rounded to bf16 as a bf16 cache would hold
    them, and the values into the 8-bit paged caches at ``slots`` [T] (distinct;
    a slot outside the cache, -1 by custom, is skipped).  Returns the rotated
    queries [T, nq * d].

    ``positions`` [T] lie below the 65536 rows of the rotary table; a position
    outside it turns the token's queries and keys into NaN."""
    if qkv.is_cuda:
        tabs = _ROPE.get((theta, d, qkv.device))
        if tabs is None:
            tabs = _ROPE[(theta, d, qkv.device)] = rope_tables(theta, d, 65536, qkv.device)
        cos, sin = tabs
        if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
            qkv = qkv.contiguous()
        return ext().rope_quant_kv(qkv, _i32(positions), cos, sin, int(nq), int(nkv), int(d), k_cache, v_cache,
                                   k_scale, v_scale, _i32(slots))
    T = qkv.shape[0]
    if T == 0:
        return qkv.new_empty(0, nq * d)
    cos, sin = rope_tables(theta, d, int(positions.max().item()) + 1, qkv.device)
    q, k, v = qkv.split([nq * d, nkv * d, nkv * d], dim=-1)
    k = apply_rope_ref(k.reshape(T, nkv, d), positions, cos, sin)
    write_kv_cache_fp8_ref(k, v.reshape(T, nkv, d), k_cache, v_cache, k_scale, v_scale, slots)
    return apply_rope_ref(q.reshape(T, nq, d), positions, cos, sin).reshape(T, nq * d)


def read_kv_cache(cache: torch.Tensor, scale: torch.Tensor, blocks: torch.Tensor, out: torch.Tensor | None = None,
                  out_blocks: torch.Tensor | None = None) -> torch.Tensor:
    """Pages ``blocks`` [n] of an 8-bit cache as bf16 pages, exactly: into a new
    [n, nkv, block_size, d] tensor, or into ``out`` (a bf16 cache), at its pages
    ``out_blocks`` if given.  Ids outside their tensor are skipped on the GPU."""
    if out is None:
        if out_blocks is not None:
            raise ValueError("out_blocks name pages of out")
        out = torch.empty((blocks.numel(),) + tuple(cache.shape[1:]), dtype=torch.bfloat16, device=cache.device)
    if cache.is_cuda:
        ext().read_kv_cache(cache, scale, _i32(blocks), out, _i32(out_blocks) if out_blocks is not None else None)
        return out
    at = blocks.long()
    x = dequantise_ref(cache.view(torch.uint8)[at].view(FP8), scale[at], out.dtype)
    if out_blocks is None:
        out[: at.numel()] = x
    else:
        out[out_blocks.long()] = x
    return out
