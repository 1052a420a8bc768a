"""Attention over the whole paged cache or a sliding window of it.

The dense layers that stand between the selected ones: ``window_decode`` (one
new token per request) and ``window_prefill`` (prompt chunks, mixed batches)
attend to the last ``window`` tokens and to the first ``sinks`` ones, or to
everything; ``prefix_decode`` reads the pages that a group of requests shares
once for the whole group.
"""
from __future__ import annotations

import torch

from .. import _lib
from .decode import _kv_args


def attn_workspace(device, *, max_tokens: int, n_kv: int, G: int, head_dim: int, max_reqs: int = None) -> torch.Tensor:
    """Workspace of the calls in this module, allocated once: single-token calls
    of up to ``max_reqs`` requests (default: ``max_tokens``) and prefill calls of up
    to ``max_tokens`` tokens.  Calls that share it follow each other."""
    max_reqs = max_tokens if max_reqs is None else max_reqs
    if max_tokens < 1 or max_reqs < 0 or n_kv < 1 or not 1 <= G <= 16 or head_dim not in (64, 128, 256):
        raise ValueError(f"max_tokens {max_tokens}, max_reqs {max_reqs}, n_kv {n_kv}, G {G}, head_dim {head_dim}: need "
                         "positive counts, G in [1, 16], head_dim 64, 128 or 256")
    n = _lib.load().locks_attn_workspace_bytes(int(max_reqs), int(max_tokens), int(n_kv), int(G), int(head_dim))
    return torch.empty(n, dtype=torch.uint8, device=device)


_BF16, _I32, _F32 = torch.bfloat16, torch.int32, torch.float32


def _i32(name: str, t, n: int, index: int) -> None:
    if t.dtype is not _I32 or t.dim() != 1 or (t.numel() > 1 and t.stride(0) != 1):
        raise TypeError(f"{name} must be a contiguous int32 vector, got {t.dtype} {tuple(t.shape)}")
    if t.shape[0] < n or t.get_device() != index:
        raise ValueError(f"{name} must hold {n} entries on the cache's device, got {t.shape[0]} on {t.device}")


def _refuse(what: str, q, kv_cache, block_table, seq_lens, out, ws, lse, rows: int, n_req: int) -> None:
    """The error of a call that _args does not take."""
    if kv_cache.dim() != 5 or kv_cache.dtype is not _BF16 or kv_cache.stride(-1) != 1:
        raise TypeError(f"{what}: kv_cache must be a 5-d bf16 cache with a contiguous last dim, got "
                        f"{kv_cache.dtype} {tuple(kv_cache.shape)}")
    _, vp, _, (_, _, n_kv, d) = _kv_args(kv_cache)
    if vp is None:
        raise ValueError(f"{what} needs a cache with a V half")
    dev = kv_cache.device
    for name, t in (("q", q), ("out", out)):
        if t.dtype is not _BF16 or t.dim() != 3 or t.stride(-1) != 1:
            raise TypeError(f"{what}: {name} must be bf16 (rows, heads, d) with a contiguous last dim, got {t.dtype} "
                            f"{tuple(t.shape)} strides {t.stride()}")
        if t.shape[0] < rows or t.shape[2] != d or t.shape[1] % n_kv or t.shape[1] != q.shape[1]:
            raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}; the call has {rows} rows, head_dim {d} and a "
                             f"multiple of {n_kv} heads")
        if t.device != dev:
            raise ValueError(f"{what}: {name} is on {t.device}, the cache on {dev}")
    if block_table.dtype is not _I32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise TypeError(f"{what}: block_table must be int32 (requests, pages) with contiguous rows")
    if block_table.shape[0] < n_req or block_table.device != dev:
        raise ValueError(f"{what}: block_table must hold {n_req} rows on {dev}, got {block_table.shape[0]} on "
                         f"{block_table.device}")
    _i32(f"{what}: seq_lens", seq_lens, n_req, kv_cache.get_device())
    if lse is not None:
        if lse.dtype is not _F32 or lse.dim() != 2 or lse.stride(1) != 1:
            raise TypeError(f"{what}: lse must be fp32 (rows, heads) with contiguous rows")
        raise ValueError(f"{what}: lse must be ({rows}, {q.shape[1]}) on {dev}, got {tuple(lse.shape)} on {lse.device}")
    if ws is not None and (ws.device != dev or not ws.is_contiguous()):
        raise ValueError(f"{what}: the workspace must be contiguous, on {dev}")
    raise ValueError(f"{what} runs on the GPU, the cache is on {dev}, and n_req {n_req} and the rows {rows} must not "
                     "be negative")


def _args(what: str, q, kv_cache, block_table, seq_lens, out, ws, lse, rows: int, n_req: int):
    """The checks that the calls share (one pass over the tensors' attributes:
    with a message at each check they took 7 us of a small call), and their common
    arguments: of q up to seq_lens; from out to the workspace; n_kv, G, d, page; the
    device's index."""
    index = kv_cache.get_device()
    try:
        n0, n1, page, n_kv, d = kv_cache.shape
        c0, c1, cst, csh, c4 = kv_cache.stride()
        (tq, H, dq), (to, ho, do), (rb, cols), (ts,) = q.shape, out.shape, block_table.shape, seq_lens.shape
        (q0, q1, q2), (o0, o1, o2), (b0, b1), (ss,) = q.stride(), out.stride(), block_table.stride(), seq_lens.stride()
        # either cache layout: K and V halves by the first or the second dim
        first = n0 == 2 and n1 != 2
        ok = (index >= 0 and kv_cache.dtype is _BF16 and q.dtype is _BF16 and out.dtype is _BF16
              and block_table.dtype is _I32 and seq_lens.dtype is _I32 and 0 <= rows <= tq and rows <= to
              and 0 <= n_req <= rb and n_req <= ts and H % n_kv == 0 and ho == H and dq == d and do == d and c4 == 1
              and q2 == 1 and o2 == 1 and b1 == 1 and (ss == 1 or ts < 2) and (first or n1 != 1)
              and q.get_device() == index and out.get_device() == index and block_table.get_device() == index
              and seq_lens.get_device() == index)
        lp = ls = wp = wb = 0
        if ok and ws is not None:
            ok = ws.get_device() == index and ws.is_contiguous()
            wp, wb = ws.data_ptr(), ws.nbytes
        if ok and lse is not None:
            (tl, hl), (ls, l1) = lse.shape, lse.stride()
            ok = lse.dtype is _F32 and l1 == 1 and tl >= rows and hl == H and lse.get_device() == index
            lp = lse.data_ptr()
    except ValueError:                                       # another number of dims
        ok = False
    if not ok:
        _refuse(what, q, kv_cache, block_table, seq_lens, out, ws, lse, rows, n_req)
    kp = kv_cache.data_ptr()
    cb = c1 if first else c0
    head = (q.data_ptr(), q0, q1, kp, cb, cst, csh, kp + 2 * (c0 if first else c1), cb, cst, csh, n1 if first else n0,
            block_table.data_ptr(), b0, cols, seq_lens.data_ptr())
    return head, (out.data_ptr(), o0, o1, lp, ls, wp, wb), (n_kv, H // n_kv, d, page), index


def window_decode(q, kv_cache, block_table, seq_lens, out, ws, *, n_req: int, scale: float, window: int = 0,
                  sinks: int = 0, lse=None, max_seq_len: int = 0) -> None:
    """One new token per request, at position ``seq_lens - 1``: ``out[:n_req]``
    (T, H, d) bf16 = softmax attention of ``q`` over the keys of the last
    ``window`` positions, its own included, and of the first ``sinks`` (window 0:
    all), and ``lse[:n_req]`` (T, H) fp32 the log-sum-exp of the scores.  Request r
    reads and writes row r: padding takes a row here, though no token in
    ``BlockTables.step``, and so stands behind the requests.  A request of length 0
    (padding) gives zeros and -inf.  ``max_seq_len``: an upper bound of
    the lengths, where one is known, sizes the launch.  ``ws``: attn_workspace."""
    head, tail, geo, index = _args("window_decode", q, kv_cache, block_table, seq_lens, out, ws, lse, n_req, n_req)
    if n_req == 0:
        return
    _lib.launch("locks_window_decode", index,
                (*head, window, sinks, *tail, n_req, *geo, max_seq_len, scale))


def window_prefill(q, kv_cache, block_table, seq_lens, query_start_loc, out, ws, *, n_req: int, scale: float,
                   window: int = 0, sinks: int = 0, lse=None, n_tokens: int = None, max_seq_len: int = 0) -> None:
    """Rows ``query_start_loc[r] .. query_start_loc[r + 1]`` of ``q`` (T, H, d)
    are the last tokens of request r, whose K and V are in the cache; each sees
    the keys up to its own position, in the window or among the first ``sinks`` as
    for ``window_decode``.  Rows from ``query_start_loc[n_req]`` on stay as they
    were.  ``n_tokens`` (default: the rows of q) bounds the rows read."""
    n_tokens = q.shape[0] if n_tokens is None else n_tokens
    head, tail, geo, index = _args("window_prefill", q, kv_cache, block_table, seq_lens, out, ws, lse, n_tokens, n_req)
    _i32("window_prefill: query_start_loc", query_start_loc, n_req + 1, index)
    if n_req == 0 or n_tokens == 0:
        return
    _lib.launch("locks_window_prefill", index,
                (*head, query_start_loc.data_ptr(), window, sinks, *tail, n_tokens, n_req, *geo, max_seq_len, scale))


def prefix_decode(q, kv_cache, block_table, seq_lens, group_start, prefix_pages, out, ws, *, n_req: int,
                  n_groups: int, scale: float, lse=None, max_prefix_pages: int = 0, max_seq_len: int = 0) -> None:
    """``window_decode`` without a window for requests that share pages: requests
    ``group_start[g] .. group_start[g + 1]`` (ascending) hold the same ids in their
    first ``prefix_pages[g]`` columns, which are read once for the group, through
    the row of a member that is as long (of the longest where none is).  Both are
    int32 on the GPU, so that a captured call follows them.  Requests outside all
    groups, members shorter than the prefix and padding (length 0) are attended
    like any other; their rows need hold no more pages than their lengths.
    ``n_groups`` is at least 1; a group may hold no request."""
    head, tail, geo, index = _args("prefix_decode", q, kv_cache, block_table, seq_lens, out, ws, lse, n_req, n_req)
    _i32("prefix_decode: group_start", group_start, n_groups + 1, index)
    _i32("prefix_decode: prefix_pages", prefix_pages, n_groups, index)
    if n_req == 0:
        return
    _lib.launch("locks_prefix_decode", index,
                (*head, group_start.data_ptr(), prefix_pages.data_ptr(), n_groups, *tail, n_req, *geo, max_prefix_pages,
                 max_seq_len, scale))
