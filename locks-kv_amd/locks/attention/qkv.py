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


_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


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
    # one pass over the tensors' attributes, unpacked at once (slices of shapes and a
    # message at each check took longer than the launch); _refuse has the messages
    index = kv_cache.get_device()
    try:
        n0, n1, page, n_kv, d = kv_cache.shape
        tq, H, dq = q.shape
        tk, hk, dk = k.shape
        tv, hv, dv = v.shape
        to, ho, do = q_out.shape
        (tp,), (ts,) = positions.shape, slot_mapping.shape
        c0, c1, cst, csh, c4 = kv_cache.stride()
        (q0, q1, q2), (k0, k1, k2), (v0, v1, v2), (o0, o1, o2) = q.stride(), k.stride(), v.stride(), q_out.stride()
        (ps,), (ss,) = positions.stride(), slot_mapping.stride()
        rot, max_pos, cp, f32, qw, kw, ko, ko0, ko1 = 0, 0x7FFFFFFF, 0, None, 0, 0, 0, 0, 0
        n = tq if n_tokens is None else n_tokens
        # either cache layout: K and V halves by the first or the second dim
        first = n0 == 2 and n1 != 2
        NB = n1 if first else n0
        ok = (index >= 0 and kv_cache.dtype is _BF16 and q.dtype is _BF16 and k.dtype is _BF16 and v.dtype is _BF16
              and q_out.dtype is _BF16 and positions.dtype is _I32 and slot_mapping.dtype is _I64 and 0 <= n <= tq
              and n <= tk and n <= tv and n <= to and n <= tp and n <= ts and hk == n_kv and hv == n_kv and ho == H
              and dq == d and dk == d and dv == d and do == d and c4 == 1 and q2 == 1 and k2 == 1 and v2 == 1 and o2 == 1
              and (ps == 1 or tp < 2) and (ss == 1 or ts < 2) and (first or n1 != 1) and q.get_device() == index
              and k.get_device() == index and v.get_device() == index and q_out.get_device() == index
              and positions.get_device() == index and slot_mapping.get_device() == index)
        if ok and cos_sin is not None:
            max_pos, rot = cos_sin.shape
            ok = cos_sin.dtype is _F32 and cos_sin.is_contiguous() and cos_sin.get_device() == index
            cp = cos_sin.data_ptr()
        for w in (q_weight, k_weight):
            if ok and w is not None:
                (wd,), t = w.shape, w.dtype
                ok = (wd == d and (t is _BF16 or t is _F32) and (f32 is None or t is f32) and w.is_contiguous()
                      and w.get_device() == index)
                f32 = t
        if ok and k_out is not None:
            (t0, t1, t2), (ko0, ko1, ko2) = k_out.shape, k_out.stride()
            ok = (k_out.dtype is _BF16 and t0 >= n and t1 == n_kv and t2 == d and ko2 == 1
                  and k_out.get_device() == index)
            ko = k_out.data_ptr()
    except ValueError:                                       # another number of dims
        ok, n = False, q.shape[0] if n_tokens is None else n_tokens
    if not ok:
        _refuse(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, n, q_weight, k_weight, k_out)
    if n == 0:
        return
    kp = kv_cache.data_ptr()
    cb = c1 if first else c0
    if q_weight is not None:
        qw = q_weight.data_ptr()
    if k_weight is not None:
        kw = k_weight.data_ptr()
    _lib.launch("locks_qkv_write", index, (
        q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, positions.data_ptr(), slot_mapping.data_ptr(),
        kp, cb, cst, csh, kp + 2 * (c0 if first else c1), cb, cst, csh, NB, cp, max_pos, rot, 1 if interleaved else 0,
        qw, kw, 1 if f32 is _F32 else 0, eps, q_out.data_ptr(), o0, o1, ko, ko0, ko1, n, H, n_kv, d, page))
