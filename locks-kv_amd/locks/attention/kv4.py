"""The paged cache in 4 bits: 17 / 64 of the bf16 cache's bytes.

32 consecutive entries of one head of one token share a power of two 2^e, and
each is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} 2^e: e is the smallest whole number of
[-125, 125] with ``max |x| <= 7 * 2^e``, and the nearest of them is taken, ties to
the even one.  A block with an infinite or NaN entry reads as NaN.

``kv4_cache`` makes one; ``qk_norm_rope_write``, ``window_decode``, ``window_prefill``
and ``LocksEngine.forward_dense`` take it where they take a bf16 cache, at the same
block tables and slots; ``kv4_read`` gives rows of it back.
"""
from __future__ import annotations

import torch

from .. import _lib

_BF16, _I64, _U8 = torch.bfloat16, torch.int64, torch.uint8


def kv4_cache(num_blocks: int, *, n_kv: int, head_dim: int, page: int, device) -> torch.Tensor:
    """A cache of ``num_blocks`` pages, all zeros: uint8 (num_blocks, n_kv, page / 16,
    17 * head_dim), 16 tokens of K and V of one head in each last dim."""
    if num_blocks < 1 or n_kv < 1 or head_dim not in (64, 128, 256) or page not in (16, 32, 64):
        raise ValueError(f"num_blocks {num_blocks}, n_kv {n_kv}, head_dim {head_dim}, page {page}: need positive counts, "
                         "head_dim 64, 128 or 256, page 16, 32 or 64")
    return torch.zeros(int(num_blocks), int(n_kv), page // 16, 17 * head_dim, dtype=_U8, device=device)


def kv4_geometry(what: str, kv_cache) -> tuple:
    """(num_blocks, page, n_kv, head_dim) of a cache in 4 bits; raises where it is none."""
    if kv_cache.dtype is not _U8 or kv_cache.dim() != 4 or kv_cache.shape[3] % 17:
        raise TypeError(f"{what}: a cache in 4 bits is uint8 (num_blocks, n_kv, page / 16, 17 * head_dim) (kv4_cache), "
                        f"got {kv_cache.dtype} {tuple(kv_cache.shape)}")
    NB, n_kv, tiles, rec = kv_cache.shape
    if kv_cache.stride(3) != 1 or kv_cache.stride(2) != rec:
        raise TypeError(f"{what}: the tiles of a (block, head) of a cache in 4 bits must be contiguous, got strides "
                        f"{kv_cache.stride()}")
    return NB, 16 * tiles, n_kv, rec // 17


def kv4_read(kv_cache, slots, k_out, v_out) -> None:
    """Rows ``slots`` (T,) int64 (block * page + offset) of a cache in 4 bits as bf16
    (T, n_kv, d): the values that the codes stand for, exactly.  A slot outside the
    cache (padding: -1) leaves its rows as they were."""
    # one pass over the tensors' attributes (as qk_norm_rope_write); _refuse_read has the messages
    index = kv_cache.get_device()
    try:
        (NB, n_kv, tiles, rec), (cb, ch, ct, c1) = kv_cache.shape, kv_cache.stride()
        (n,), (ss,) = slots.shape, slots.stride()
        (tk, hk, dk), (tv, hv, dv) = k_out.shape, v_out.shape
        (k0, k1, k2), (v0, v1, v2) = k_out.stride(), v_out.stride()
        d = rec // 17
        ok = (index >= 0 and kv_cache.dtype is _U8 and rec % 17 == 0 and ct == rec and c1 == 1 and slots.dtype is _I64
              and (ss == 1 or n < 2) and k_out.dtype is _BF16 and v_out.dtype is _BF16 and k2 == 1 and v2 == 1
              and tk >= n and tv >= n and hk == n_kv and hv == n_kv and dk == d and dv == d
              and slots.get_device() == index and k_out.get_device() == index and v_out.get_device() == index)
    except ValueError:                                       # another number of dims
        ok = False
    if not ok:
        _refuse_read(kv_cache, slots, k_out, v_out)
    if n == 0:
        return
    _lib.launch("locks_kv4_read", index, (
        kv_cache.data_ptr(), cb, ch, NB, slots.data_ptr(), k_out.data_ptr(), k0, k1, v_out.data_ptr(), v0, v1, n, n_kv, d,
        16 * tiles))


def _refuse_read(kv_cache, slots, k_out, v_out) -> None:
    """The error of a call that kv4_read does not take."""
    _, _, n_kv, d = kv4_geometry("kv4_read", kv_cache)
    if slots.dtype is not _I64 or slots.dim() != 1 or not slots.is_contiguous():
        raise TypeError(f"kv4_read: slots must be a contiguous int64 vector, got {slots.dtype} {tuple(slots.shape)}")
    n = slots.shape[0]
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t.dtype is not _BF16 or t.dim() != 3 or t.stride(2) != 1:
            raise TypeError(f"kv4_read: {name} must be bf16 (tokens, heads, d) with a contiguous last dim, got {t.dtype} "
                            f"{tuple(t.shape)} strides {t.stride()}")
        if t.shape[0] < n or t.shape[1] != n_kv or t.shape[2] != d:
            raise ValueError(f"kv4_read: {name} has shape {tuple(t.shape)}, the call needs ({n}, {n_kv}, {d})")
    raise ValueError(f"kv4_read runs on one GPU: the cache is on {kv_cache.device}, slots on {slots.device}, outputs on "
                     f"{k_out.device} and {v_out.device}")
