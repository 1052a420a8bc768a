"""Engine-neutral host side of the LOCKS decode path.

One object per model replaces the three places the reference's vLLM
integration spreads this over:

* state allocation, as the metadata builder does once the KV cache exists
  (src/locks/backend/builder.py:658-787): the rki4 state sized by the
  model geometry and the scheduler limits, budget ``cfg.budget`` or 0.1
  when only ``budget_pages`` / a coverage is given, the split-K buffers,
  and the kv-cache pointer -> layer map the select adapter keys on;
* the per-step prologue (builder.py:1100-1136 with the refresh gate
  :1138-1282): summaries refreshed for pages that finalized, then the
  per-request page parameters derived when they can have changed;
* the pure single-token decode forward of the attention impl
  (backend/attn.py:338-378): select the pages of every kv head, then the
  split-K sparse decode with the LSE merge.  Other steps (prefill, mixed
  batches) are the engine's dense attention, as in the reference;
* for the DRAM-tier variants (``mem-v`` / ``mem-kv``) the tier of
  ``locks.tier`` (tier/tier.py:38-302, its decode source :704-784): the
  prologue runs its per-step lifecycle (tier.py:239-301), ``write_kv``
  copies each layer's new V (K) into the staging pool (tier.py:386-392),
  and ``forward`` runs the layer's residency step between selection and the
  decode, which then reads V (K) through ``TierVSource``;
* around the selected layers, for an engine without kernels of its own:
  ``block_tables`` (the step's tables and slots from the requests' lengths),
  ``write_qkv`` (norm, rotation and cache write of a layer's projection),
  ``forward_dense`` (prompt chunks and mixed batches, and layers that keep a
  window) and ``forward_prefix`` (decode of requests on a shared prefix).  Layers
  that only ever attend densely may hold their cache in 4 bits (``kv4_cache``).

A vLLM-ROCm attention backend calls ``prologue`` from its metadata builder
and ``forward`` from its impl; any other engine can drive it directly.
"""
from __future__ import annotations

import torch

from ..attention import attn_workspace, kv4_cache, prefix_decode, qk_norm_rope_write, window_decode, window_prefill
from ..attention.decode import _split_kv, ensure_stage_b_buffers
from ..selection import Rki4State, derive_page_params
from ..tier import Tier
from . import _runtime
from .refresh import RefreshGate
from .tables import BlockTables


class LocksEngine:
    def __init__(self, cfg, kv_caches, *, num_heads_q: int, num_heads_kv: int, head_dim: int,
                 block_size: int, max_num_seqs: int, max_model_len: int, split: int = 128,
                 max_num_batched_tokens: int = 8192):
        if cfg.mem_summary_cache:
            raise ValueError("locks: mem_summary_cache (summary records in the engine page, K only "
                             "in the tier) is not built; use mem-kv with the K half resident")
        if num_heads_q % num_heads_kv:
            raise ValueError("num_heads_q must be a multiple of num_heads_kv")
        if not kv_caches:
            raise ValueError("kv_caches is empty")
        self.cfg = cfg
        self.kv_caches = list(kv_caches)
        dev = self.kv_caches[0].device
        K0 = _split_kv(self.kv_caches[0])[0]
        page = int(block_size)
        self.st = Rki4State(
            dev, num_layers=len(self.kv_caches), num_blocks=int(K0.shape[0]),
            n_kv=int(num_heads_kv), G=int(num_heads_q // num_heads_kv), head_dim=int(head_dim),
            page=page, max_reqs=int(max_num_seqs), max_pages=-(-int(max_model_len) // page),
            budget=cfg.budget if cfg.budget is not None else 0.1,
            budget_pages=cfg.budget_pages, sink_pages=cfg.sink_pages,
            window_pages=cfg.window_pages, combine=cfg.quad_combine, zsplit=cfg.rki4_zsplit)
        ensure_stage_b_buffers(self.st, dev, split)
        self.st._layer_of = {kv.data_ptr(): i for i, kv in enumerate(self.kv_caches)}
        self.k_layers = [_split_kv(kv)[0] for kv in self.kv_caches]
        self.gate = RefreshGate(page)
        self.max_tokens = int(max_num_batched_tokens)
        self._dense_ws = None
        self._k_out = None
        self.tier = None
        if cfg.is_mem:
            self.tier = Tier.from_config(
                cfg, num_layers=len(self.kv_caches), num_blocks=int(K0.shape[0]),
                n_kv=int(num_heads_kv), page=page, d=int(head_dim), max_reqs=int(max_num_seqs),
                max_pages=self.st.max_pages, max_tokens=int(max_num_batched_tokens), device=dev)
            if self.tier.offload_k:                  # the keys as cached, for the tier
                self._k_out = torch.empty(self.max_tokens, int(num_heads_kv), int(head_dim), dtype=torch.bfloat16,
                                          device=dev)

    @torch.no_grad()
    def prologue(self, block_table, seq_lens, query_start_loc, n_req: int,
                 seq_lens_cpu=None, query_start_loc_cpu=None):
        """Refresh the summaries and derive the page parameters of this step.

        ``seq_lens`` counts this step's in-flight tokens; the keys of earlier
        steps are in the cache.  Returns the state the layers read."""
        if n_req > self.st.max_reqs:
            raise ValueError(f"n_req {n_req} > max_num_seqs {self.st.max_reqs}")
        if self.tier is not None:
            qsl = query_start_loc
            n_tok = (int(query_start_loc_cpu[n_req]) if query_start_loc_cpu is not None
                     else int(qsl[n_req].item()))
            self.tier.begin_step(block_table, seq_lens, qsl[: n_req + 1], n_req, n_tok)
        need_derive = self.gate.refresh(self.st, self.k_layers, block_table, seq_lens,
                                        query_start_loc, n_req, seq_lens_cpu,
                                        query_start_loc_cpu)
        if need_derive:
            derive_page_params(self.st, seq_lens, n_req)
        return self.st

    @torch.no_grad()
    def forward(self, q, kv_cache, block_table, seq_lens, n_req: int, scale: float, out) -> None:
        """One layer of a pure single-token decode step: ``q`` (n_req, H, d)
        bf16, the layer's kv_cache (its new token already written), ``out``
        (n_req, H, d) written in place."""
        _state, _derive, select_pages, _graph_safe = _runtime.resolve_selection()
        select_pages(q, kv_cache, block_table, seq_lens, self.st, n_req, scale, self.cfg)
        vsource = None
        if self.tier is not None:
            layer = _runtime._layer_index(self.st, kv_cache)
            self.tier.step(layer, self.st.page_table, self.st.page_cnt, block_table, seq_lens, n_req)
            vsource = self.tier.vsource(layer)
        _runtime.decode_dispatch(q, kv_cache, block_table, seq_lens, self.st, out, vsource, scale,
                                 self.cfg)

    @torch.no_grad()
    def write_kv(self, layer: int, key, value) -> None:
        """After the engine wrote this step's K / V (n_tokens, n_kv, d) of one
        layer into its cache: the DRAM tier's copy of them (tier.py:386-392).
        A no-op for the resident variant."""
        if self.tier is not None:
            self.tier.write_kv(layer, value, key)

    # ---- around the selected layers ------------------------------------------
    def block_tables(self, reserved: int = 0) -> BlockTables:
        """Block tables for this engine's cache and limits: ``step`` gives
        ``prologue`` and the layers their block table, lengths and slots."""
        return BlockTables(self.kv_caches[0].device, num_blocks=self.st.NB, page=self.st.page,
                           max_reqs=self.st.max_reqs, max_pages=self.st.max_pages, max_tokens=self.max_tokens,
                           reserved=reserved)

    def kv4_cache(self) -> torch.Tensor:
        """A cache in 4 bits of this engine's geometry, for a layer outside
        ``kv_caches`` that ``write_qkv`` and ``forward_dense`` get it for: the same block
        ids and slots hold for it."""
        st = self.st
        return kv4_cache(st.NB, n_kv=st.n_kv, head_dim=st.D, page=st.page, device=self.kv_caches[0].device)

    @torch.no_grad()
    def write_qkv(self, layer: int, q, k, v, positions, slot_mapping, cos_sin, q_out, *, n_tokens: int = None,
                  q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False, axes=None,
                  kv_cache=None) -> None:
        """A layer's projection made ready (``qk_norm_rope_write``): queries to
        ``q_out``, keys and values to the layer's cache and, for the mem variants,
        V (mem-kv: and the keys) to the tier's staging pool (``write_kv``).  This
        and the dense calls need a cache with both halves: a K-only one, which the
        mem variants' ``forward`` takes too, is refused.  ``axes``: the axis of each
        pair, where positions have several (``RopeAxes``).  ``kv_cache``: the cache of a
        layer outside ``kv_caches`` (bf16, or ``kv4_cache``), which has no part in
        selection and tier; ``layer`` does not matter then."""
        n = int(q.shape[0] if n_tokens is None else n_tokens)
        if kv_cache is not None:
            qk_norm_rope_write(q, k, v, positions, slot_mapping, kv_cache, cos_sin, q_out, n_tokens=n, q_weight=q_weight,
                               k_weight=k_weight, eps=eps, interleaved=interleaved, axes=axes)
            return
        if self.tier is not None and n > self.max_tokens:
            raise ValueError(f"write_qkv: {n} tokens > max_num_batched_tokens {self.max_tokens}")
        qk_norm_rope_write(q, k, v, positions, slot_mapping, self.kv_caches[layer], cos_sin, q_out, n_tokens=n,
                           q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved, k_out=self._k_out,
                           axes=axes)
        if self.tier is not None and n:
            self.write_kv(layer, None if self._k_out is None else self._k_out[:n], v[:n])

    def _ws(self):
        """Workspace of the dense calls, made by the first of them (a captured
        step is run once before its capture)."""
        if self._dense_ws is None:
            st = self.st
            self._dense_ws = attn_workspace(self.kv_caches[0].device, max_tokens=self.max_tokens,
                                            max_reqs=st.max_reqs, n_kv=st.n_kv, G=st.G, head_dim=st.D)
        return self._dense_ws

    @torch.no_grad()
    def forward_dense(self, q, kv_cache, block_table, seq_lens, n_req: int, scale: float, out, *,
                      query_start_loc=None, n_decode: int = None, n_tokens: int = None, window: int = 0, sinks: int = 0,
                      lse=None, max_seq_len: int = 0) -> None:
        """One layer of any step with attention over the whole row, or over the
        last ``window`` tokens and the first ``sinks``, read from the paged cache (in
        bf16 or in 4 bits).
        The first ``n_decode`` requests have one new token each, in rows 0 to
        ``n_decode`` - 1 (default: all, without ``query_start_loc``; none with it),
        the others the rows that ``query_start_loc`` gives.  Padding takes no
        token: it stands behind the requests with one, or after ``n_decode``.
        ``max_seq_len``: an upper bound of the lengths, where the caller's host knows
        one; else the calls size themselves for the table, ``max_model_len`` tokens,
        and short requests take longer (a length past the bound is attended to all
        the same)."""
        if n_decode is None:
            n_decode = n_req if query_start_loc is None else 0
        if not 0 <= n_decode <= n_req or (n_decode < n_req and query_start_loc is None):
            raise ValueError(f"n_decode {n_decode} of {n_req} requests"
                             + ("" if query_start_loc is not None else " and no query_start_loc"))
        kw = dict(scale=scale, window=window, sinks=sinks, lse=lse, max_seq_len=max_seq_len)
        if n_decode:
            window_decode(q, kv_cache, block_table, seq_lens, out, self._ws(), n_req=n_decode, **kw)
        if n_decode < n_req:
            window_prefill(q, kv_cache, block_table[n_decode:], seq_lens[n_decode:], query_start_loc[n_decode:], out,
                           self._ws(), n_req=n_req - n_decode, n_tokens=n_tokens, **kw)

    @torch.no_grad()
    def forward_prefix(self, q, kv_cache, block_table, seq_lens, group_start, prefix_pages, n_req: int, n_groups: int,
                       scale: float, out, *, max_prefix_pages: int = 0, lse=None) -> None:
        """One layer of a single-token step over the whole rows of requests that
        share their first pages (``prefix_decode``); request r is row r of ``q``,
        padding behind the requests."""
        prefix_decode(q, kv_cache, block_table, seq_lens, group_start, prefix_pages, out, self._ws(), n_req=n_req,
                      n_groups=n_groups, scale=scale, max_prefix_pages=max_prefix_pages, lse=lse)
