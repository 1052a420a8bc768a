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
    _, page, n_kv, d = kv4_geometry("kv4_read", kv_cache)
    index = kv_cache.get_device()
    if slots.dtype is not _I64 or slots.dim() != 1 or not slots.is_contiguous():
        raise TypeError(f"kv4_read: slots must be a contiguous int64 vector, got {slots.dtype} {tuple(slots.shape)}")
    n = slots.shape[0]
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t.dtype is not _BF16 or t.dim() != 3 or t.stride(2) != 1:
            raise TypeError(f"kv4_read: {name} must be bf16 (tokens, heads, d) with a contiguous last dim, got {t.dtype} "
                            f"{tuple(t.shape)} strides {t.stride()}")
        if t.shape[0] < n or t.shape[1] != n_kv or t.shape[2] != d:
            raise ValueError(f"kv4_read: {name} has shape {tuple(t.shape)}, the call needs ({n}, {n_kv}, {d})")
    if index < 0 or any(t.get_device() != index for t in (slots, k_out, v_out)):
        raise ValueError(f"kv4_read runs on one GPU: the cache is on {kv_cache.device}, slots on {slots.device}, outputs on "
                         f"{k_out.device} and {v_out.device}")
    if n == 0:
        return
    _lib.launch("locks_kv4_read", index, (
        kv_cache.data_ptr(), kv_cache.stride(0), kv_cache.stride(1), kv_cache.shape[0], slots.data_ptr(),
        k_out.data_ptr(), k_out.stride(0), k_out.stride(1), v_out.data_ptr(), v_out.stride(0), v_out.stride(1), n, n_kv,
        d, page))
