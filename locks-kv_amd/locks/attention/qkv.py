"""Query and key heads made ready for attention, K and V written to the cache.

One pass over the projection's output: RMS norm of each query and key head
(optional), the position rotation, and the write of K and V into the paged cache
at the step's slots (``locks.backend.tables.BlockTables`` makes positions and
slots).  Pairs turn by one position, or by that along one of several axes
(``RopeAxes``); the cache is one in bf16 or in 4 bits (``locks.attention.kv4``).
"""
from __future__ import annotations

import torch

from .. import _lib
from .decode import _kv_args
from .kv4 import kv4_geometry


_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


class RopeAxes:
    """Which axis (time, height, width, ...) each rotated pair's angle follows:
    ``pairs[j]`` in [0, ``n_axes``) for pair j of the first rot = 2 * len(pairs)
    entries.  Made once per model."""

    __slots__ = ("pairs", "n_axes", "words")

    def __init__(self, pairs, n_axes: int = None):
        self.pairs = tuple(int(a) for a in pairs)
        self.n_axes = max(self.pairs, default=0) + 1 if n_axes is None else int(n_axes)
        if not 1 <= self.n_axes <= 4 or any(not 0 <= a < self.n_axes for a in self.pairs):
            raise ValueError(f"RopeAxes: 1 to 4 axes, each pair's in [0, n_axes), got n_axes {self.n_axes} and "
                             f"{self.pairs}")
        if not self.pairs or len(self.pairs) % 8 or len(self.pairs) > 128:
            raise ValueError(f"RopeAxes: {len(self.pairs)} pairs: need a multiple of 8 in [8, 128]")
        words = [0, 0, 0, 0]
        for j, a in enumerate(self.pairs):
            words[j >> 5] |= a << (2 * (j & 31))
        self.words = tuple(w - (1 << 64) if w >> 63 else w for w in words)      # as signed 64 bits

    @classmethod
    def sections(cls, counts) -> "RopeAxes":
        """The first ``counts[0]`` pairs follow axis 0, the next ``counts[1]`` axis 1, ..."""
        counts = cls._counts(counts)
        return cls([a for a, n in enumerate(counts) for _ in range(n)], len(counts))

    @classmethod
    def cycled(cls, counts) -> "RopeAxes":
        """The axes in turn, pair by pair; one that has its ``counts[a]`` pairs is passed
        over."""
        left, pairs = cls._counts(counts), []
        while any(left):
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    pairs.append(a)
        return cls(pairs, len(left))

    @staticmethod
    def _counts(counts) -> list:
        counts = [int(n) for n in counts]
        if any(n < 0 for n in counts):
            raise ValueError(f"RopeAxes: pairs per axis {counts} must not be negative")
        return counts


def _rows(name: str, t, n: int, heads, d: int, device) -> None:
    if t.dtype is not _BF16 or t.dim() != 3 or t.stride(-1) != 1:
        raise TypeError(f"{name} must be bf16 (tokens, heads, d) with a contiguous last dim, got {t.dtype} "
                        f"{tuple(t.shape)} strides {t.stride()}")
    if t.shape[0] < n or t.shape[1] != heads or t.shape[2] != d:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, the call needs ({n}, {heads}, {d})")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")


def _refuse(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, n: int, q_weight, k_weight, k_out,
            axes) -> None:
    """The error of a call that qk_norm_rope_write does not take."""
    if kv_cache.dtype is _U8:
        _, _, n_kv, d = kv4_geometry("qk_norm_rope_write", kv_cache)
    else:
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
    vectors = [("slot_mapping", slot_mapping, torch.int64)]
    if axes is None:
        vectors.insert(0, ("positions", positions, torch.int32))
    else:
        if not isinstance(axes, RopeAxes):
            raise TypeError(f"axes must be a RopeAxes, got {type(axes).__name__}")
        if positions.dtype is not _I32 or positions.dim() != 2 or (positions.shape[1] > 1 and positions.stride(1) != 1):
            raise TypeError(f"positions must be int32 ({axes.n_axes}, tokens) with contiguous rows, got {positions.dtype} "
                            f"{tuple(positions.shape)}")
        if positions.shape[0] != axes.n_axes or positions.shape[1] < n or positions.device != dev:
            raise ValueError(f"positions must be ({axes.n_axes}, {n}) on {dev}, got {tuple(positions.shape)} on "
                             f"{positions.device}")
        if cos_sin is None or cos_sin.dim() != 2 or cos_sin.shape[1] != 2 * len(axes.pairs):
            raise ValueError(f"axes has {len(axes.pairs)} pairs, cos_sin "
                             + ("is None" if cos_sin is None else f"has shape {tuple(cos_sin.shape)}"))
    for name, t, dt in vectors:
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
                       k_out=None, axes: RopeAxes = None) -> None:
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

    With ``axes`` each pair turns by the position along its own axis: ``positions``
    is (axes, T), pair j's angle that of ``cos_sin[positions[axes.pairs[j]], j]``.

    ``kv_cache`` is the paged cache in bf16, or one in 4 bits (``kv4_cache``), whose
    keys are rounded from norm and rotation in 64 bits; ``k_out`` has them in bf16.

    A slot outside the cache (padding: -1) writes no cache row.  A position
    outside the table (along any axis) writes none either, and NaN to the token's
    ``q_out`` and ``k_out`` rows.  Slots of one call are distinct."""
    # one pass over the tensors' attributes, unpacked at once (slices of shapes and a
    # message at each check took longer than the launch); _refuse has the messages
    index = kv_cache.get_device()
    four = kv_cache.dtype is _U8
    try:
        if four:
            NB, n_kv, tiles, rec = kv_cache.shape
            cb, csh, cst, c4 = kv_cache.stride()
            page, d = 16 * tiles, rec // 17
            held = rec % 17 == 0 and cst == rec
        else:
            n0, n1, page, n_kv, d = kv_cache.shape
            c0, c1, cst, csh, c4 = kv_cache.stride()
            # either cache layout: K and V halves by the first or the second dim
            first = n0 == 2 and n1 != 2
            NB = n1 if first else n0
            held = kv_cache.dtype is _BF16 and (first or n1 != 1)
        tq, H, dq = q.shape
        tk, hk, dk = k.shape
        tv, hv, dv = v.shape
        to, ho, do = q_out.shape
        pa = 0
        if axes is None:
            (tp,), (ps,) = positions.shape, positions.stride()
        else:
            (na, tp), (pa, ps) = positions.shape, positions.stride()
            held = held and na == axes.n_axes and cos_sin is not None and cos_sin.shape[1] == 2 * len(axes.pairs)
        (ts,) = slot_mapping.shape
        (q0, q1, q2), (k0, k1, k2), (v0, v1, v2), (o0, o1, o2) = q.stride(), k.stride(), v.stride(), q_out.stride()
        (ss,) = slot_mapping.stride()
        rot, max_pos, cp, f32, qw, kw, ko, ko0, ko1 = 0, 0x7FFFFFFF, 0, None, 0, 0, 0, 0, 0
        n = tq if n_tokens is None else n_tokens
        ok = (index >= 0 and held and q.dtype is _BF16 and k.dtype is _BF16 and v.dtype is _BF16
              and q_out.dtype is _BF16 and positions.dtype is _I32 and slot_mapping.dtype is _I64 and 0 <= n <= tq
              and n <= tk and n <= tv and n <= to and n <= tp and n <= ts and hk == n_kv and hv == n_kv and ho == H
              and dq == d and dk == d and dv == d and do == d and c4 == 1 and q2 == 1 and k2 == 1 and v2 == 1 and o2 == 1
              and (ps == 1 or tp < 2) and (ss == 1 or ts < 2) and q.get_device() == index
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
    except (ValueError, AttributeError, IndexError):         # another number of dims, no RopeAxes
        ok, n = False, q.shape[0] if n_tokens is None else n_tokens
    if not ok:
        _refuse(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, n, q_weight, k_weight, k_out, axes)
    if n == 0:
        return
    if q_weight is not None:
        qw = q_weight.data_ptr()
    if k_weight is not None:
        kw = k_weight.data_ptr()
    kp = kv_cache.data_ptr()
    turn = ((pa, 0, 0, 0, 0, 0) if axes is None else (pa, axes.n_axes, *axes.words)) if four or axes is not None else ()
    if four:
        entry, cache = "locks_kv4_write", (kp, cb, csh)
    else:
        cb = c1 if first else c0
        entry = "locks_qkv_write" if axes is None else "locks_qkv_write_axes"
        cache = (kp, cb, cst, csh, kp + 2 * (c0 if first else c1), cb, cst, csh)
    _lib.launch(entry, index, (
        q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, positions.data_ptr(), *turn,
        slot_mapping.data_ptr(), *cache, NB, cp, max_pos, rot, 1 if interleaved else 0, qw, kw,
        1 if f32 is _F32 else 0, eps, q_out.data_ptr(), o0, o1, ko, ko0, ko1, n, H, n_kv, d, page))
