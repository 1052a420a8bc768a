"""Query and key heads made ready for attention, K and V written to the cache.

One pass over the projection's output: RMS norm of each query and key head
(optional), the position rotation, and the write of K and V into the paged cache
at the step's slots (``locks.backend.tables.BlockTables`` makes positions and
slots).
"""
from __future__ import annotations

import torch

from .. import _lib
from .decode import _kv_args


def _rows(name: str, t, n: int, heads, d: int, device) -> None:
    if t.dtype != torch.bfloat16 or t.dim() != 3 or t.stride(-1) != 1:
        raise TypeError(f"{name} must be bf16 (tokens, heads, d) with a contiguous last dim, got {t.dtype} "
                        f"{tuple(t.shape)} strides {t.stride()}")
    if t.shape[0] < n or t.shape[1] != heads or t.shape[2] != d:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, the call needs ({n}, {heads}, {d})")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")


def qk_norm_rope_write(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, *, n_tokens: int = None,
                       q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                       k_out=None) -> None:
    """``q`` (T, H, d), ``k``, ``v`` (T, n_kv, d) bf16 (views of a packed
    projection are fine); the first ``n_tokens`` rows (default: all) are read.

    ``y = x * rsqrt(mean(x^2) + eps) * weight`` per head (``q_weight``,
    ``k_weight``: (d,) bf16 or fp32, both of one type, or None for no norm), then
    each pair of the first ``rot`` entries is turned by its angle at
    ``positions`` (T,) int32: entries (i, i + rot / 2), or with ``interleaved``
    (2 i, 2 i + 1).  ``cos_sin`` (max_pos, rot) fp32 holds rot / 2 cosines, then
    rot / 2 sines of each position (None: no rotation).  Queries go to ``q_out``
    (T, H, d), which may be ``q``; keys and values to ``kv_cache`` at
    ``slot_mapping`` (T,) int64 (block * page + offset), and the keys also to
    ``k_out`` (T, n_kv, d) if given.

    A slot outside the cache (padding: -1) writes no cache row.  A position
    outside the table writes none either, and NaN to the token's ``q_out`` and
    ``k_out`` rows.  Slots of one call are distinct."""
    kp, vp, ks, (NB, page, n_kv, d) = _kv_args(kv_cache)
    if vp is None:
        raise ValueError("qk_norm_rope_write needs a cache with a V half")
    if kv_cache.dtype != torch.bfloat16 or kv_cache.stride(-1) != 1:
        raise TypeError("kv_cache must be bf16 with a contiguous last dim")
    n = int(q.shape[0] if n_tokens is None else n_tokens)
    dev = kv_cache.device
    if n < 0:
        raise ValueError(f"n_tokens {n} < 0")
    if q.dim() != 3:
        raise TypeError(f"q must be (tokens, heads, d), got shape {tuple(q.shape)}")
    H = int(q.shape[1])
    _rows("q", q, n, H, d, dev)
    _rows("k", k, n, n_kv, d, dev)
    _rows("v", v, n, n_kv, d, dev)
    _rows("q_out", q_out, n, H, d, dev)
    if k_out is not None:
        _rows("k_out", k_out, n, n_kv, d, dev)
    for name, t, dt in (("positions", positions, torch.int32), ("slot_mapping", slot_mapping, torch.int64)):
        if t.dtype != dt or t.dim() != 1 or (t.numel() > 1 and t.stride(0) != 1):
            raise TypeError(f"{name} must be a contiguous {dt} vector, got {t.dtype} {tuple(t.shape)}")
        if t.shape[0] < n or t.device != dev:
            raise ValueError(f"{name} must hold {n} entries on {dev}, got {t.shape[0]} on {t.device}")
    rot, max_pos = 0, 0x7FFFFFFF
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
            raise TypeError("cos_sin must be contiguous fp32 (max_pos, rot)")
        if cos_sin.device != dev:
            raise ValueError(f"cos_sin is on {cos_sin.device}, the cache on {dev}")
        max_pos, rot = (int(x) for x in cos_sin.shape)
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.dtype not in (torch.bfloat16, torch.float32) or tuple(w.shape) != (d,) or not w.is_contiguous():
            raise TypeError(f"a norm weight must be contiguous bf16 or fp32 ({d},), got {w.dtype} {tuple(w.shape)}")
        if w.dtype != weights[0].dtype:
            raise TypeError("q_weight and k_weight must have one type")
        if w.device != dev:
            raise ValueError(f"a norm weight is on {w.device}, the cache on {dev}")
    if dev.type != "cuda":
        raise ValueError(f"qk_norm_rope_write runs on the GPU, the cache is on {dev}")
    if n == 0:
        return
    ko = k_out.stride()[:2] if k_out is not None else (0, 0)
    with _lib.on_device(dev):
        _lib.check(_lib.load().locks_qkv_write(
            q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2],
            positions.data_ptr(), slot_mapping.data_ptr(), kp, *ks, vp, *ks, NB, _lib.ptr(cos_sin), max_pos, rot,
            1 if interleaved else 0, _lib.ptr(q_weight), _lib.ptr(k_weight),
            1 if weights and weights[0].dtype == torch.float32 else 0, float(eps), q_out.data_ptr(),
            *q_out.stride()[:2], _lib.ptr(k_out), *ko, n, H, n_kv, d, page, _lib.stream_ptr(dev)), "qkv_write")
