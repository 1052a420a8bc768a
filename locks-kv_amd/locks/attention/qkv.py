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


_BF16, _F32 = torch.bfloat16, torch.float32


def _rows(name: str, t, n: int, heads, d: int, device) -> None:
    if t.dtype is not _BF16 or t.dim() != 3 or t.stride(-1) != 1:
        raise TypeError(f"{name} must be bf16 (tokens, heads, d) with a contiguous last dim, got {t.dtype} "
                        f"{tuple(t.shape)} strides {t.stride()}")
    if t.shape[0] < n or t.shape[1] != heads or t.shape[2] != d:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, the call needs ({n}, {heads}, {d})")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")


def _refuse(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, n: int, q_weight, k_weight, k_out) -> None:
    """The error of a call that qk_norm_rope_write does not take."""
    if kv_cache.dtype is not _BF16 or kv_cache.dim() != 5 or kv_cache.stride(-1) != 1:
        raise TypeError(f"kv_cache must be a 5-d bf16 cache with a contiguous last dim, got {kv_cache.dtype} "
                        f"{tuple(kv_cache.shape)}")
    _, vp, _, (_, _, n_kv, d) = _kv_args(kv_cache)
    if vp is None:
        raise ValueError("qk_norm_rope_write needs a cache with a V half")
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
        if t.dtype is not dt or t.dim() != 1 or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous {dt} vector, got {t.dtype} {tuple(t.shape)}")
        if t.shape[0] < n or t.device != dev:
            raise ValueError(f"{name} must hold {n} entries on {dev}, got {t.shape[0]} on {t.device}")
    if cos_sin is not None:
        if cos_sin.dtype is not _F32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
            raise TypeError("cos_sin must be contiguous fp32 (max_pos, rot)")
        if cos_sin.device != dev:
            raise ValueError(f"cos_sin is on {cos_sin.device}, the cache on {dev}")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.dtype not in (_BF16, _F32) or tuple(w.shape) != (d,) or not w.is_contiguous():
            raise TypeError(f"a norm weight must be contiguous bf16 or fp32 ({d},), got {w.dtype} {tuple(w.shape)}")
        if w.dtype != weights[0].dtype:
            raise TypeError("q_weight and k_weight must have one type")
        if w.device != dev:
            raise ValueError(f"a norm weight is on {w.device}, the cache on {dev}")
    raise ValueError(f"qk_norm_rope_write runs on the GPU, the cache is on {dev}")


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
    n = q.shape[0] if n_tokens is None else n_tokens
    index = kv_cache.get_device()
    # one pass over the tensors' attributes; _refuse has the messages
    cs, qs, ks_, vs_, os = kv_cache.shape, q.shape, k.shape, v.shape, q_out.shape
    qt, kt, vt, ot = q.stride(), k.stride(), v.stride(), q_out.stride()
    ok = (index >= 0 and len(cs) == 5 and kv_cache.dtype is _BF16 and q.dtype is _BF16 and k.dtype is _BF16
          and v.dtype is _BF16 and q_out.dtype is _BF16 and positions.dtype is torch.int32
          and slot_mapping.dtype is torch.int64 and len(qs) == 3 and len(ks_) == 3 and vs_[1:] == ks_[1:]
          and os[1:] == qs[1:] and n >= 0 and qs[0] >= n and ks_[0] >= n and vs_[0] >= n and os[0] >= n
          and ks_[1:] == cs[3:] and qs[2] == cs[4] and qt[2] == 1 and kt[2] == 1 and vt[2] == 1 and ot[2] == 1
          and positions.dim() == 1 and positions.is_contiguous() and slot_mapping.dim() == 1
          and slot_mapping.is_contiguous() and positions.shape[0] >= n and slot_mapping.shape[0] >= n
          and q.get_device() == index and k.get_device() == index and v.get_device() == index
          and q_out.get_device() == index and positions.get_device() == index and slot_mapping.get_device() == index)
    rot, max_pos, cp, f32, ko = 0, 0x7FFFFFFF, 0, None, (0, 0, 0)
    if ok and cos_sin is not None:
        ok = (cos_sin.dtype is _F32 and cos_sin.dim() == 2 and cos_sin.is_contiguous() and cos_sin.get_device() == index)
        cp = cos_sin.data_ptr()
        if ok:
            max_pos, rot = cos_sin.shape
    for w in (q_weight, k_weight):
        if ok and w is not None:
            t = w.dtype
            ok = ((t is _BF16 or t is _F32) and (f32 is None or t is f32) and w.dim() == 1 and w.shape[0] == cs[4]
                  and w.is_contiguous() and w.get_device() == index)
            f32 = t
    if ok and k_out is not None:
        kos, kot = k_out.shape, k_out.stride()
        ok = (k_out.dtype is _BF16 and len(kos) == 3 and kos[0] >= n and kos[1:] == ks_[1:] and kot[2] == 1
              and k_out.get_device() == index)
        ko = (k_out.data_ptr(), *kot[:2])
    if ok:
        kp, vp, ks, (NB, page, n_kv, d) = _kv_args(kv_cache)
        ok = vp is not None and kv_cache.stride(4) == 1
    if not ok:
        _refuse(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, n, q_weight, k_weight, k_out)
    if n == 0:
        return
    _lib.launch(_lib.load().locks_qkv_write, "qkv_write", index, (
        q.data_ptr(), qt[0], qt[1], k.data_ptr(), kt[0], kt[1], v.data_ptr(), vt[0], vt[1], positions.data_ptr(),
        slot_mapping.data_ptr(), kp, *ks, vp, *ks, NB, cp, max_pos, rot, 1 if interleaved else 0, _lib.ptr(q_weight),
        _lib.ptr(k_weight), 1 if f32 is _F32 else 0, eps, q_out.data_ptr(), ot[0], ot[1], *ko, n, qs[1], n_kv, d, page))
