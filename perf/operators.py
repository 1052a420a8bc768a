"""The step of a paged-cache serving loop around the page selector, as timed cases.

Five operators, each through the entry points a serving program calls:

* ``tables``: a step's block tables, lengths, positions and cache slots from
  the requests' lengths, with blocks taken from the free list on the GPU, and
  the roll-back of that step (``BlockTables.step`` / ``.trim``);
* ``qkv``: RMS norm of each query and key head, the position rotation, and the
  write of K and V into the paged cache (``qk_norm_rope_write``);
* ``window``: single-token attention over the last ``window`` tokens and the
  first ``sinks`` ones (``window_decode``);
* ``prefill``: the same for many new tokens of each request, causal, also with
  no window (``window_prefill``);
* ``prefix``: single-token attention of requests that share a long prefix, the
  prefix read once for all of a group (``prefix_decode``).

``own`` false: the plain forms, elementary torch operations in 32 bits on
padded batches.  Lengths, groups and page counts are plain values of the case.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False


# ---- cases -------------------------------------------------------------------
def _attn(name, kind, lens, n_kv, group, *, d=128, page=16, window=0, sinks=0, **more):
    return dict(name=name, kind=kind, lens=lens, n_kv=n_kv, group=group, d=d, page=page, window=window, sinks=sinks,
                **more)


def listed():
    return [
        # a decode step of a small batch: one new token each
        dict(name="tables-decode-32", kind="tables", n=32, chunks=0, chunk=1, ctx_lo=2000, ctx_hi=32768, page=16,
             slots=64, pick=1),
        # a full batch, most requests decoding and some in a chunk of their prompt
        dict(name="tables-mixed-256", kind="tables", n=256, chunks=48, chunk=512, ctx_lo=500, ctx_hi=65536, page=16,
             slots=256, pick=2),
        # the new token of one user
        dict(name="qkv-1", kind="qkv", tokens=1, heads=32, n_kv=8, d=128, rot=128, page=16, norm=True,
             interleaved=False, far=131000),
        # a prompt chunk of the engine's largest step
        dict(name="qkv-8192", kind="qkv", tokens=8192, heads=32, n_kv=8, d=128, rot=128, page=16, norm=True,
             interleaved=False, far=0),
        # half of each head rotated in adjacent pairs, no norm, an odd number of tokens far into a 1M context
        dict(name="qkv-half-2049", kind="qkv", tokens=2049, heads=32, n_kv=2, d=128, rot=64, page=16, norm=False,
             interleaved=True, far=1040000),
        # one user, deep into a long chat, in a layer that keeps a window
        _attn("window-128k-1", "window", "131072", 8, 4, window=4096, sinks=4),
        # a ragged serving batch in such a layer, some requests shorter than the window
        _attn("window-batch-32", "window", "32768,31007,28123,24576,21333,19001,16384,15001,12288,11117,9999,8192,"
              "7001,5555,4097,3001,2500,2049,1777,1500,1025,1024,1000,800,513,400,257,100,33,17,2,1", 8, 4,
              window=8192, sinks=64),
        # a whole prompt in a layer that attends to everything before
        _attn("prefill-8192", "prefill", "8192", 8, 4, new="8192"),
        # a whole prompt in a layer that keeps a window, wide query groups
        _attn("prefill-window-8192", "prefill", "8192", 2, 16, new="8192", window=1024, sinks=4),
        # chunks of several prompts and a decoding request together, a model of another head size and cache page
        _attn("prefill-ragged-d64", "prefill", "5003,2049,4096,700,129", 4, 8, d=64, page=32, new="1301,2049,1024,1,129"),
        # a batch that answers about one long document
        dict(name="prefix-32k-64", kind="prefix", groups="64", pages="2048", own_lo=20, own_hi=1500, n_kv=8, group=4,
             d=128, page=16, pick=3),
        # two system prompts, few users each, wide query groups
        dict(name="prefix-2-groups", kind="prefix", groups="5,3", pages="300,64", own_lo=1, own_hi=3000, n_kv=2,
             group=16, d=128, page=16, pick=4),
    ]


def draw(rng):
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))  # noqa: E731
    kind = rng.choice(["tables", "qkv", "window", "window", "prefill", "prefill", "prefix", "prefix"])
    d, page = rng.choice([(128, 16)] * 4 + [(64, 16), (256, 16), (128, 32), (128, 64), (64, 32), (256, 64)])
    n_kv, group = rng.choice([(8, 4), (8, 4), (8, 8), (4, 8), (4, 7), (2, 16), (16, 1), (1, 16), (3, 5)])
    if kind == "tables":
        n = log(1, 256)
        return dict(kind=kind, n=n, chunks=rng.randint(0, min(n, 32)), chunk=log(2, 512), ctx_lo=1,
                    ctx_hi=log(100, 60000), page=page, slots=n + rng.choice([0, 3, 40]), pick=rng.randint(0, 1 << 30))
    if kind == "qkv":
        rot = rng.choice([d, d, d // 2, d // 4])
        return dict(kind=kind, tokens=max(1, min(log(1, 8192), (8192 * 48 * 128) // ((group + 2) * n_kv * d))),
                    heads=n_kv * group, n_kv=n_kv, d=d, rot=rot, page=page, norm=rng.random() < 0.6,
                    interleaved=rng.random() < 0.4, far=rng.choice([0, 0, log(1, 131000)]))
    if kind == "window":
        window = rng.choice([0, log(16, 8192), log(16, 8192)])
        lens = _spread(log(1, 48), 1, log(100, 100000), rng.randint(0, 1 << 30))
        most = (110000 * 8 * 128) // (n_kv * d)                    # key rows that all of a pass may reach
        while len(lens) * min(window or max(lens), max(lens)) > most or sum(lens) > 400000:
            lens = lens[1:] if len(lens) > 1 else [lens[0] // 2]
        return {k: v for k, v in _attn("", kind, ",".join(map(str, lens)), n_kv, group, d=d, page=page, window=window,
                                       sinks=rng.choice([0, 4, rng.randint(1, 300)]) if window else 0).items()
                if k != "name"}
    if kind == "prefill":
        window = rng.choice([0, log(16, 4096)])
        new = _spread(rng.choice([1, 1, 2, 4, 6]), 1, log(16, 4096), rng.randint(0, 1 << 30))
        lens = [n + rng.choice([0, log(1, 4000)]) for n in new]
        while len(new) * max(new) * max(lens) * n_kv * group * d > 8192 * 8192 * 32 * 128 // 2:
            new, lens = [-(-n // 2) for n in new], [-(-n // 2) for n in lens]
        return {k: v for k, v in _attn("", kind, ",".join(map(str, lens)), n_kv, group, d=d, page=page, window=window,
                                       sinks=rng.choice([0, rng.randint(1, 100)]) if window else 0,
                                       new=",".join(map(str, new))).items() if k != "name"}
    groups = [log(1, 48) for _ in range(rng.choice([1, 1, 2, 3]))]
    pages = [log(1, 32768 // page) for _ in groups]
    own_hi = log(1, 1500)
    while (sum(groups) * (max(pages) * page + own_hi) * n_kv * d > 64 * 33000 * 8 * 128
           or (sum(pages) * page + sum(groups) * own_hi) * n_kv * d > 100000 * 8 * 128):
        groups, pages = [-(-m // 2) for m in groups], [-(-p * 2 // 3) for p in pages]
    return dict(kind=kind, groups=",".join(map(str, groups)), pages=",".join(map(str, pages)), own_lo=1, own_hi=own_hi,
                n_kv=n_kv, group=group, d=d, page=page, pick=rng.randint(0, 1 << 30))


def _spread(n, lo, hi, pick):
    """n whole numbers of [lo, hi], spread over their logarithm."""
    r = random.Random(pick)
    return [min(hi, max(lo, int(math.exp(r.uniform(math.log(lo), math.log(hi + 1)))))) for _ in range(n)]


def _ints(text):
    return [int(x) for x in text.split(",")]


def _table_lens(case):
    """(tokens already in the cache, new tokens) of each request."""
    had = _spread(case["n"], case["ctx_lo"], case["ctx_hi"], case["pick"])
    new = _spread(case["chunks"], 2, max(2, case["chunk"]), case["pick"] + 1) + [1] * (case["n"] - case["chunks"])
    random.Random(case["pick"] + 2).shuffle(new)
    return had, new


def _prefix_lens(case):
    """(members, prefix pages) of each group, and the whole length of each request."""
    groups, pages = _ints(case["groups"]), _ints(case["pages"])
    tail = _spread(sum(groups), case["own_lo"], case["own_hi"], case["pick"])
    lens, at = [], 0
    for g, p in zip(groups, pages):
        lens += [p * case["page"] + t for t in tail[at:at + g]]
        at += g
    return groups, pages, lens


def _visible(case, position):
    """How many keys a query at `position` sees."""
    w, s = case["window"], case["sinks"]
    return position + 1 if not w else min(position + 1, w) + min(s, max(0, position + 1 - w))


def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "tables":
        had, new = _table_lens(case)
        pages = sum(-(-(h + n) // page) for h, n in zip(had, new))
        fresh = pages - sum(-(-h // page) for h in had)
        # every page id read once (from the request's row or the free list) and written to the batch's row, the
        # fresh ones to the request's row too and back to the list; positions, slots; lengths and rows
        return dict(bytes=4 * (2 * pages + 3 * fresh) + 12 * sum(new) + 4 * 6 * len(new), flops=0)
    if kind == "qkv":
        t, h, n_kv, d = case["tokens"], case["heads"], case["n_kv"], case["d"]
        rows = t * (h + 2 * n_kv) * d
        return dict(bytes=2 * 2 * rows + t * (4 + 8 + 4 * case["rot"]), flops=t * (h + n_kv) * d * 10)
    n_kv, group, d = case["n_kv"], case["group"], case["d"]
    row = 2 * 2 * n_kv * d                                         # K and V of one token
    qo = 4 * n_kv * group * d                                      # q and the output of one token
    dot = 4 * n_kv * group * d
    if kind == "window":
        keys = sum(_visible(case, n - 1) for n in _ints(case["lens"]))
        n = len(_ints(case["lens"]))
        return dict(bytes=keys * row + n * qo, flops=keys * dot)
    if kind == "prefill":
        lens, new = _ints(case["lens"]), _ints(case["new"])
        pairs = sum(sum(_visible(case, p) for p in range(n - m, n)) for n, m in zip(lens, new))
        keys = sum(min(n, (case["window"] or n) + m - 1 + case["sinks"]) for n, m in zip(lens, new))
        return dict(bytes=keys * row + sum(new) * qo, flops=pairs * dot)
    groups, pages, lens = _prefix_lens(case)
    keys = sum(p * page for p in pages)
    tails = sum(lens) - sum(g * p * page for g, p in zip(groups, pages))
    return dict(bytes=(keys + tails) * row + len(lens) * qo, flops=sum(lens) * dot)


# ---- inputs ------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _cache(g, blocks, page, n_kv, d):
    """(blocks, 2, page, n_kv, d) bf16: N(0, 1), four channels of each key head x8."""
    scale = torch.ones(2, 1, n_kv, d, device="cuda")
    for h in range(n_kv):
        scale[0, 0, h, torch.randperm(d, generator=g, device="cuda")[:4]] = 8.0
    out = torch.empty(blocks, 2, page, n_kv, d, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 27) // (2 * page * n_kv * d))
    for lo in range(0, blocks, step):
        n = min(step, blocks - lo)
        out[lo:lo + n] = (torch.randn(n, 2, page, n_kv, d, generator=g, device="cuda") * scale).to(torch.bfloat16)
    return out


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "locks-kv_amd")
    if root not in sys.path:
        sys.path.insert(0, root)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["kind"] == "tables":
        _prepare_tables(case, g, st)
    elif case["kind"] == "qkv":
        _prepare_qkv(case, g, st)
    else:
        _prepare_attention(case, g, st)
    if own:
        _framework()
        if case["kind"] == "tables":
            from locks.backend.tables import BlockTables
            t = BlockTables("cuda", num_blocks=st["blocks"], page=case["page"], max_reqs=case["slots"],
                            max_pages=st["max_pages"], max_tokens=st["n_tokens"])
            t.lens.copy_(st["lens"])
            t.table.copy_(st["table"])
            t.free.copy_(st["free"])
            t.set_free(st["head"])
            st["tables"] = t
        elif case["kind"] != "qkv":
            from locks.attention import attn_workspace
            st["ws"] = attn_workspace("cuda", max_tokens=st["q"].shape[0], n_kv=case["n_kv"], G=case["group"],
                                      head_dim=case["d"])
    return st


def _prepare_tables(case, g, st):
    had, new = _table_lens(case)
    page, slots = case["page"], case["slots"]
    pages = [-(-n // page) for n in had]
    fresh = sum(-(-(h + n) // page) for h, n in zip(had, new)) - sum(pages)
    blocks = sum(pages) + fresh + 7
    width = max(-(-(h + n) // page) for h, n in zip(had, new)) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    rows = torch.randperm(slots, generator=g, device="cuda")[:case["n"]].to(torch.int32)
    table = torch.zeros(slots, width, dtype=torch.int32, device="cuda")
    lens = torch.zeros(slots, dtype=torch.int32, device="cuda")
    lens[rows.long()] = _i32(had)
    # the free list holds its blocks at [head, blocks); the entries before it are what earlier steps have taken
    head = sum(pages)
    at = 0
    for r, n in zip(rows.tolist(), pages):
        table[r, :n] = order[at:at + n]
        at += n
    st |= dict(blocks=blocks, max_pages=width, n_tokens=sum(new), lens=lens, table=table, free=order.clone(), head=head,
               rows=rows, new=_i32(new), had=_i32(had), n=case["n"])


def _prepare_qkv(case, g, st):
    t, h, n_kv, d, rot, page = (case[k] for k in ("tokens", "heads", "n_kv", "d", "rot", "page"))
    blocks = -(-t // page) + 5
    # the projection's output, q, k and v of a token side by side; a few channels of the keys large
    packed = torch.randn(t, (h + 2 * n_kv) * d, generator=g, device="cuda")
    packed[:, h * d:(h + n_kv) * d].view(t, n_kv, d)[:, :, torch.randperm(d, generator=g, device="cuda")[:4]] *= 8
    packed = packed.to(torch.bfloat16)
    q, k, v = (x.view(t, -1, d) for x in packed.split([h * d, n_kv * d, n_kv * d], dim=1))
    pages = torch.randperm(blocks, generator=g, device="cuda")
    pos = torch.arange(t, device="cuda")
    slots = pages[pos // page] * page + pos % page
    positions = pos + case["far"]
    freq = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(case["far"] + t, dtype=torch.float64, device="cuda")[:, None] * freq
    st |= dict(q=q, k=k, v=v, positions=positions.to(torch.int32), slots=slots, eps=1e-6,
               cos_sin=torch.cat([angle.cos(), angle.sin()], dim=1).float(),
               cache=torch.zeros(blocks, 2, page, n_kv, d, dtype=torch.bfloat16, device="cuda"),
               q_weight=(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16) if case["norm"] else None,
               k_weight=(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16) if case["norm"] else None,
               q_out=torch.zeros(t, h, d, dtype=torch.bfloat16, device="cuda"))


def _prepare_attention(case, g, st):
    page, n_kv, d = case["page"], case["n_kv"], case["d"]
    H = n_kv * case["group"]
    groups, pages = None, None
    if case["kind"] == "prefix":
        groups, pages, lens = _prefix_lens(case)
        shared = [p for m, p in zip(groups, pages) for _ in range(m)]
    else:
        lens = _ints(case["lens"])
        shared = [0] * len(lens)
    new = _ints(case["new"]) if "new" in case else [1] * len(lens)
    width = max(-(-n // page) for n in lens)
    need = [-(-n // page) - s for n, s in zip(lens, shared)]
    blocks = sum(need) + sum(pages or [0]) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at, r = 0, 0
    for m, p in zip(groups or [], pages or []):
        table[r:r + m, :p] = order[at:at + p]
        at, r = at + p, r + m
    for i, (n, s) in enumerate(zip(need, shared)):
        table[i, s:s + n] = order[at:at + n]
        at += n
    total = sum(new)
    st |= dict(lens=lens, new=new, kv=_cache(g, blocks, page, n_kv, d), q=_normal(g, total, H, d), table=table,
               seq_lens=_i32(lens), starts=_i32(_starts(new)), scale=1.0 / math.sqrt(d),
               out=torch.zeros(total, H, d, dtype=torch.bfloat16, device="cuda"),
               lse=torch.zeros(total, H, device="cuda"), groups=groups, pages=pages)
    if groups:
        st |= dict(group_start=_i32(_starts(groups)), prefix_pages=_i32(pages))


# ---- one pass ----------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return {"tables": _own_tables, "qkv": _own_qkv, "window": _own_window, "prefill": _own_prefill,
                "prefix": _own_prefix}[case["kind"]](case, st)
    return {"tables": _plain_tables, "qkv": _plain_qkv, "window": _plain_window, "prefill": _plain_prefill,
            "prefix": _plain_prefix}[case["kind"]](case, st)


def _own_tables(case, st):
    t = st["tables"]
    t.step(st["rows"], st["new"], n_req=st["n"], n_tokens=st["n_tokens"])
    t.trim(st["rows"], st["had"], n_req=st["n"])
    return dict(block_table=t.block_table[:st["n"], :st["max_pages"]], seq_lens=t.seq_lens[:st["n"]],
                query_start_loc=t.query_start_loc[:st["n"] + 1], positions=t.positions, slot_mapping=t.slot_mapping,
                free=t.free, lens=t.lens)


def _own_qkv(case, st):
    from locks.attention import qk_norm_rope_write
    qk_norm_rope_write(st["q"], st["k"], st["v"], st["positions"], st["slots"], st["cache"], st["cos_sin"],
                       st["q_out"], q_weight=st["q_weight"], k_weight=st["k_weight"], eps=st["eps"],
                       interleaved=case["interleaved"])
    return dict(q=st["q_out"], cache=st["cache"])


def _own_window(case, st):
    from locks.attention import window_decode
    window_decode(st["q"], st["kv"], st["table"], st["seq_lens"], st["out"], st["ws"], n_req=len(st["lens"]),
                  window=case["window"], sinks=case["sinks"], scale=st["scale"], lse=st["lse"])
    return dict(out=st["out"], lse=st["lse"])


def _own_prefill(case, st):
    from locks.attention import window_prefill
    window_prefill(st["q"], st["kv"], st["table"], st["seq_lens"], st["starts"], st["out"], st["ws"],
                   n_req=len(st["lens"]), window=case["window"], sinks=case["sinks"], scale=st["scale"], lse=st["lse"])
    return dict(out=st["out"], lse=st["lse"])


def _own_prefix(case, st):
    from locks.attention import prefix_decode
    prefix_decode(st["q"], st["kv"], st["table"], st["seq_lens"], st["group_start"], st["prefix_pages"], st["out"],
                  st["ws"], n_req=len(st["lens"]), n_groups=len(st["groups"]), scale=st["scale"], lse=st["lse"])
    return dict(out=st["out"], lse=st["lse"])


def _plain_tables(case, st):
    page, n, head, free = case["page"], st["n"], st["head"], st["free"]
    rows, new = st["rows"].long(), st["new"].long()
    had = st["lens"][rows].long()
    have, all_ = (had + page - 1) // page, (had + new + page - 1) // page
    need = all_ - have
    first = need.cumsum(0) - need
    served = (need == 0) | (first + need <= free.shape[0] - head)
    cols = torch.arange(st["max_pages"], device="cuda")
    # a column is an owned page, a fresh one (the free list's in order), or none
    fresh = (cols >= have[:, None]) & (cols < all_[:, None]) & served[:, None]
    at = (head + first[:, None] + cols - have[:, None]).clamp(0, free.shape[0] - 1)
    owned = (cols < have[:, None]) & served[:, None]
    table = torch.where(owned, st["table"][rows], torch.where(fresh, free[at], torch.zeros_like(free[at])))
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    tok = torch.arange(st["n_tokens"], device="cuda")
    r = torch.searchsorted(starts, tok, right=True) - 1
    pos = had[r] + tok - starts[r]
    slots = torch.where(served[r], table[r, pos // page].long() * page + pos % page, torch.full_like(pos, -1))
    # the roll-back puts the fresh blocks back where they were taken from
    back = free.clone()
    back[at[fresh]] = table[fresh]
    lens = st["lens"].clone()
    lens[rows] = torch.minimum(had + new, st["had"].long()).to(torch.int32)
    return dict(block_table=table, seq_lens=torch.where(served, had + new, torch.zeros_like(had)).to(torch.int32),
                query_start_loc=starts.to(torch.int32), positions=pos.to(torch.int32), slot_mapping=slots, free=back,
                lens=lens)


def _plain_rotate(x, cos, sin, rot, interleaved):
    """x (t, heads, d) rotated in pairs of its first `rot` entries by the angle of (token, pair)."""
    a, rest = x[..., :rot], x[..., rot:]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        u, w = a[..., 0::2], a[..., 1::2]
        a = torch.stack([u * cos - w * sin, w * cos + u * sin], dim=-1).flatten(-2)
    else:
        u, w = a[..., :rot // 2], a[..., rot // 2:]
        a = torch.cat([u * cos - w * sin, w * cos + u * sin], dim=-1)
    return torch.cat([a, rest], dim=-1)


def _plain_qkv(case, st):
    rot, page = case["rot"], case["page"]
    q, k = st["q"].float(), st["k"].float()
    if case["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + st["eps"]) * st["q_weight"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + st["eps"]) * st["k_weight"].float()
    cs = st["cos_sin"][st["positions"].long()]
    cos, sin = cs[:, :rot // 2], cs[:, rot // 2:]
    q = _plain_rotate(q, cos, sin, rot, case["interleaved"]).to(torch.bfloat16)
    k = _plain_rotate(k, cos, sin, rot, case["interleaved"]).to(torch.bfloat16)
    block, at = st["slots"] // page, st["slots"] % page
    st["cache"][block, 0, at] = k
    st["cache"][block, 1, at] = st["v"]
    return dict(q=q, cache=st["cache"])


def _plain_softmax(q, k, v, seen):
    """q (b, kv, rows, d) scaled, k, v (b, kv, keys, d), seen (b, 1, rows, keys): outputs and log-sum-exp."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total, (top + total.log())[..., 0]


def _plain_keys(st, token):
    """K and V (b, kv, keys, d) in 32 bits of the token numbers (b, keys) of each request's row."""
    page = st["kv"].shape[2]
    block = st["table"].long().gather(1, token // page)
    kv = st["kv"][block, :, token % page].float()                  # (b, keys, 2, kv, d)
    return kv[:, :, 0].transpose(1, 2).contiguous(), kv[:, :, 1].transpose(1, 2).contiguous()


def _plain_window(case, st):
    n_kv, group, w, s = case["n_kv"], case["group"], case["window"], case["sinks"]
    lens = st["seq_lens"].long()
    longest = max(st["lens"])
    # the first `sinks` tokens and the last `window` ones, side by side (all of them with no window)
    tail = torch.arange(min(w or longest, longest), device="cuda")
    low = (lens - w).clamp(min=0) if w else torch.zeros_like(lens)
    token = torch.cat([torch.arange(s, device="cuda").expand(len(lens), s), low[:, None] + tail], dim=1)
    seen = torch.cat([token[:, :s] < low[:, None], token[:, s:] < lens[:, None]], dim=1)
    k, v = _plain_keys(st, token.clamp(max=longest - 1))
    q = st["q"].float().view(len(lens), n_kv, group, -1) * st["scale"]
    o, lse = _plain_softmax(q, k, v, seen[:, None, None])
    return dict(out=o.flatten(1, 2).to(torch.bfloat16), lse=lse.flatten(1, 2))


def _plain_prefill(case, st):
    n_kv, group, w = case["n_kv"], case["group"], case["window"]
    b, most, longest = len(st["lens"]), max(st["new"]), max(st["lens"])
    lens, starts = st["seq_lens"].long(), st["starts"].long()
    new = starts[1:] - starts[:-1]
    at = torch.arange(most, device="cuda")
    real = at < new[:, None]
    row = (starts[:-1, None] + at).clamp(max=st["q"].shape[0] - 1)
    pos = (lens - new)[:, None] + at
    token = torch.arange(longest, device="cuda")
    seen = token <= pos[..., None]
    if w:
        seen &= (token > pos[..., None] - w) | (token < case["sinks"])
    k, v = _plain_keys(st, token.expand(b, longest))
    q = st["q"][row].float() * st["scale"]                         # (b, most, H, d)
    q = q.view(b, most, n_kv, group, -1).permute(0, 2, 3, 1, 4).reshape(b, n_kv, group * most, -1)
    seen = seen[:, None, None].expand(b, 1, group, most, longest).reshape(b, 1, group * most, longest)
    o, lse = _plain_softmax(q, k, v, seen)
    o = o.view(b, n_kv, group, most, -1).permute(0, 3, 1, 2, 4).flatten(2, 3)
    lse = lse.view(b, n_kv, group, most).permute(0, 3, 1, 2).flatten(2, 3)
    return dict(out=o[real].to(torch.bfloat16), lse=lse[real])


def _plain_prefix(case, st):
    n_kv, group = case["n_kv"], case["group"]
    lens, longest = st["seq_lens"].long(), max(st["lens"])
    b = len(st["lens"])
    token = torch.arange(longest, device="cuda").expand(b, longest)
    k, v = _plain_keys(st, token)
    q = st["q"].float().view(b, n_kv, group, -1) * st["scale"]
    o, lse = _plain_softmax(q, k, v, (token < lens[:, None])[:, None, None])
    return dict(out=o.flatten(1, 2).to(torch.bfloat16), lse=lse.flatten(1, 2))


# ---- the definition in 64 bits -----------------------------------------------
def exact(case, seed):
    st = {"case": case}
    {"tables": _prepare_tables, "qkv": _prepare_qkv}.get(case["kind"], _prepare_attention)(case, _gen(seed), st)
    return {"tables": _exact_tables, "qkv": _exact_qkv}.get(case["kind"], _exact_attention)(case, st)


def _exact_tables(case, st):
    """One request after the other."""
    page, head = case["page"], st["head"]
    free, table, lens = st["free"].tolist(), st["table"].tolist(), st["lens"].tolist()
    rows, new = st["rows"].tolist(), st["new"].tolist()
    batch = [[0] * st["max_pages"] for _ in rows]
    starts, positions, slots, total = [0], [], [], []
    for i, (r, n) in enumerate(zip(rows, new)):
        row = table[r][:-(-lens[r] // page)]
        while len(row) * page < lens[r] + n:
            row.append(free[head])
            head += 1
        batch[i][:len(row)] = row
        total.append(lens[r] + n)
        starts.append(starts[-1] + n)
        for p in range(lens[r], lens[r] + n):
            positions.append(p)
            slots.append(row[p // page] * page + p % page)
    return dict(block_table=_i32(batch), seq_lens=_i32(total), query_start_loc=_i32(starts), positions=_i32(positions),
                slot_mapping=torch.tensor(slots, device="cuda"), free=st["free"], lens=st["lens"])


def _exact_qkv(case, st):
    """Each pair of entries as a complex number, turned by its token's unit number."""
    rot, page, t = case["rot"], case["page"], case["tokens"]
    cs = st["cos_sin"].double().index_select(0, st["positions"].long())
    turn = torch.complex(cs[:, :rot // 2], cs[:, rot // 2:])[:, None]

    def made(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + st["eps"]).sqrt() * weight.double()
        pairs = (torch.arange(rot, device="cuda").view(-1, 2).T if case["interleaved"]
                 else torch.arange(rot, device="cuda").view(2, -1))
        z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * turn
        x = x.clone()
        x[..., pairs[0]], x[..., pairs[1]] = z.real, z.imag
        return x

    cache = st["cache"].double().view(-1, 2, page * case["n_kv"] * case["d"])
    k, v = made(st["k"], st["k_weight"]), st["v"].double()
    width = case["n_kv"] * case["d"]
    flat = cache.view(cache.shape[0], 2, page, width)
    flat[st["slots"] // page, 0, st["slots"] % page] = k.reshape(t, width)
    flat[st["slots"] // page, 1, st["slots"] % page] = v.reshape(t, width)
    return dict(q=made(st["q"], st["q_weight"]), cache=flat.view(st["cache"].shape))


def _exact_attention(case, st):
    """Request by request and head by head, over every token of the request."""
    page, group, w = case["page"], case["group"], case.get("window", 0)
    if sum(n * m for n, m in zip(st["lens"], st["new"])) * case["n_kv"] * group * case["d"] > 1 << 43:
        return None
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["lse"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (n, m) in enumerate(zip(st["lens"], st["new"])):
        blocks = st["table"][r, :-(-n // page)].long()
        kv = st["kv"].index_select(0, blocks).transpose(1, 2).flatten(0, 1)[:n].double()     # (n, 2, kv, d)
        i = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = (j > i) | ((i - j >= w) & (j >= case["sinks"]) if w else torch.zeros_like(j > i))
        for h in range(case["n_kv"] * group):
            k, v = kv[:, 0, h // group].contiguous(), kv[:, 1, h // group].contiguous()
            logit = st["q"][at:at + m, h].double() @ k.T.contiguous() * st["scale"]
            logit[hidden] = -math.inf
            z = torch.logsumexp(logit, dim=1)
            lse[at:at + m, h] = z
            out[at:at + m, h] = torch.exp(logit - z[:, None]) @ v
        at += m
    return dict(out=out, lse=lse)
