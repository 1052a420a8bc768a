"""Block tables of a paged KV cache, kept and extended on the GPU.

``BlockTables`` holds one row of page ids per running request and the list of
free blocks.  ``step`` makes everything a step's kernels read from the requests'
lengths alone -- the batch's block table, ``seq_lens``, ``query_start_loc``, the
tokens' positions and cache slots -- and takes the blocks that the new tokens
need; ``trim`` gives blocks back (a finished request, rejected draft tokens).
Neither reads anything back to the host, so both can be captured in a HIP graph;
the outputs are the same buffers on every call.  Calls on one object follow each
other on one stream (or are ordered by events).
"""
from __future__ import annotations

import torch

from .. import _lib

MAX_REQS = 2048                # LOCKS_TABLES_MAX_REQS
MAX_BLOCKS = 1 << 22


def _padded(rows: int, cols: int, device) -> torch.Tensor:
    """(rows, cols) int32 zeros whose rows start at 16-byte boundaries."""
    return torch.zeros(rows, -(-cols // 4) * 4, dtype=torch.int32, device=device)[:, :cols]


class BlockTables:
    """Requests live in rows [0, max_reqs) that the caller hands out; a row that
    holds no request has length 0.

    State: ``table`` (max_reqs, max_pages) page ids and ``lens`` (max_reqs,)
    tokens of every row; ``free`` (num_blocks,) whose entries [head, num_blocks)
    are the free blocks, the next one first; ``state`` (4,): head, the last
    step's unserved requests, and a count that every call leaves at zero.
    ``reserved`` blocks, the lowest ids, are never handed out.

    Outputs of ``step``: ``block_table`` (max_reqs, max_pages), ``seq_lens``
    (max_reqs,), ``query_start_loc`` (max_reqs + 1,), ``positions`` (max_tokens,)
    int32 and ``slot_mapping`` (max_tokens,) int64.  All of these are written in
    place and never replaced.
    """

    def __init__(self, device, *, num_blocks: int, page: int, max_reqs: int, max_pages: int, max_tokens: int,
                 reserved: int = 0):
        if page not in (16, 32, 64):
            raise ValueError(f"page must be 16, 32 or 64, got {page}")
        if not 1 <= max_reqs <= MAX_REQS:
            raise ValueError(f"max_reqs must be in [1, {MAX_REQS}], got {max_reqs}")
        if not 1 <= num_blocks <= MAX_BLOCKS:
            raise ValueError(f"num_blocks must be in [1, {MAX_BLOCKS}], got {num_blocks}")
        if max_pages < 1 or max_tokens < 1:
            raise ValueError(f"max_pages {max_pages} and max_tokens {max_tokens} must be positive")
        if not 0 <= reserved <= num_blocks:
            raise ValueError(f"reserved {reserved} outside [0, num_blocks {num_blocks}]")
        if max_pages * page > 0x7FFFFFFF - page:
            raise ValueError(f"max_pages {max_pages} x page {page} passes 32-bit lengths")
        z = dict(dtype=torch.int32, device=device)
        self.num_blocks, self.page, self.max_reqs = int(num_blocks), int(page), int(max_reqs)
        self.max_pages, self.max_tokens = int(max_pages), int(max_tokens)
        self.table = _padded(max_reqs, max_pages, device)
        self.lens = torch.zeros(max_reqs, **z)
        self.free = torch.cat([torch.zeros(reserved, **z), torch.arange(reserved, num_blocks, **z)])
        self.state = torch.zeros(4, **z)
        self.set_free(reserved)
        self.block_table = _padded(max_reqs, max_pages, device)
        self.seq_lens = torch.zeros(max_reqs, **z)
        self.query_start_loc = torch.zeros(max_reqs + 1, **z)
        self.positions = torch.zeros(max_tokens, **z)
        self.slot_mapping = torch.full((max_tokens,), -1, dtype=torch.int64, device=device)
        self.device, self._index = self.table.device, self.table.get_device()
        # what the two entries take of the object's own buffers, which stay where they are
        pool = (self.lens.data_ptr(), self.table.data_ptr(), self.table.stride(0), self.max_reqs, self.max_pages,
                self.free.data_ptr(), self.num_blocks, self.state.data_ptr())
        self._step_args = (*pool, self.block_table.data_ptr(), self.block_table.stride(0), self.seq_lens.data_ptr(),
                           self.query_start_loc.data_ptr(), self.positions.data_ptr(), self.slot_mapping.data_ptr(),
                           self.page)
        self._trim_args = (*pool, self.page)

    def set_free(self, head: int) -> None:
        """The free blocks are ``free[head:]`` (for a caller that fills ``free``,
        ``table`` and ``lens`` itself)."""
        if not 0 <= head <= self.num_blocks:
            raise ValueError(f"head {head} outside [0, num_blocks {self.num_blocks}]")
        self.state[0] = int(head)

    def _check(self, name: str, t, n_req: int) -> int:
        """The address of a vector of n_req entries on the tables' device."""
        if (t.dtype is torch.int32 and t.dim() == 1 and t.is_contiguous() and t.shape[0] >= n_req
                and t.get_device() == self._index and self._index >= 0):
            return t.data_ptr()
        if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous int32 vector, got {t.dtype} {tuple(t.shape)}")
        if t.shape[0] < n_req:
            raise ValueError(f"{name} has {t.shape[0]} entries for n_req {n_req}")
        raise ValueError(f"{name} is on {t.device}, the tables on {self.device}: both must be on one GPU")

    def step(self, rows, new_lens, n_req: int, n_tokens: int) -> None:
        """The step of requests ``rows[:n_req]`` (distinct rows; -1 pads the
        batch) with ``new_lens`` new tokens each, laid out one request after the
        other; ``n_tokens`` counts them, padding included.

        A request is served when the blocks that it and those before it need are
        there, its pages fit the table and its row exists and is named for the
        first time: its row and length grow.  Any other changes nothing: its
        ``seq_lens`` entry is 0 and its tokens' slots are -1 (``state[1]`` counts
        such requests).  Padding requests have ``seq_lens`` 0, tokens past the
        last request position 0 and slot -1.  Entries of ``block_table`` past a
        request's pages, and of all outputs past ``n_req`` and ``n_tokens``, stay
        as they were.

        Padding (whatever its ``new_lens``) and requests without a new token take
        no row of the step's tokens, an unserved request keeps its own.  Calls
        that read row r for request r (``window_decode``, ``prefix_decode``, the
        selected decode) therefore need padding and such requests behind all
        others; calls that take ``query_start_loc`` find every request's rows."""
        n_req, n_tokens = int(n_req), int(n_tokens)
        if not 0 <= n_req <= self.max_reqs:
            raise ValueError(f"n_req {n_req} outside [0, max_reqs {self.max_reqs}]")
        if not 0 <= n_tokens <= self.max_tokens:
            raise ValueError(f"n_tokens {n_tokens} outside [0, max_tokens {self.max_tokens}]")
        _lib.launch("locks_tables_step", self._index, (
            self._check("rows", rows, n_req), self._check("new_lens", new_lens, n_req), n_req, n_tokens, *self._step_args))

    def trim(self, rows, keep_lens, n_req: int) -> None:
        """Shorten requests ``rows[:n_req]`` to ``keep_lens`` tokens (0: the
        request is done); the blocks past them are free again, in front of the
        list and in the order in which ``step`` takes blocks, so that the roll-back
        of a step restores the list.  A length that is not shorter changes nothing,
        a row named twice takes the first length.

        A row whose first pages belong to others (a shared prefix that the caller
        wrote into ``table``) is trimmed to the prefix's length, and its ``lens``
        entry set to 0 afterwards."""
        n_req = int(n_req)
        if not 0 <= n_req <= self.max_reqs:
            raise ValueError(f"n_req {n_req} outside [0, max_reqs {self.max_reqs}]")
        _lib.launch("locks_tables_trim", self._index, (
            self._check("rows", rows, n_req), self._check("keep_lens", keep_lens, n_req), n_req, *self._trim_args))
