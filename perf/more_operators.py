"""Positions of several axes and a paged cache held in 4 bits, as timed cases.

Four operators, each through the entry points a serving program calls:

* ``axes``: norm, rotation and cache write of query and key heads whose pairs
  turn by the position along one of several axes (time, height, width), with a
  ``RopeAxes`` (``qk_norm_rope_write(..., axes=...)``);
* ``write4``: the same into a cache held in 4 bits, and the cache's rows read
  back as the values they stand for (``qk_norm_rope_write``, ``kv4_read``);
* ``decode4``: single-token attention over such a cache, over a whole row or
  a window with sinks (``window_decode``);
* ``prefill4``: the same for many new tokens of each request, causal
  (``window_prefill``).

A cache in 4 bits: 32 consecutive entries of one head of one token share a
scale 2^e, e the smallest whole number of [-125, 125] with max |x| <= 7 * 2^e,
and each is the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} 2^e, ties to the even
one of the eight.  Keys are rounded as they leave norm and rotation.

``own`` false: the plain forms, elementary torch operations in 32 bits (the
entries of ``write4``'s keys in 64: they are next to the borders of their codes)
on padded batches.  Lengths are plain values of the case.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases -------------------------------------------------------------------
def _heads(name, kind, tokens, n_kv, group, *, d=128, page=16, rot=None, sections="", cycled=False, norm=True,
           interleaved=False, far=0):
    return dict(name=name, kind=kind, tokens=tokens, n_kv=n_kv, group=group, d=d, page=page, rot=d if rot is None else rot,
                sections=sections, cycled=cycled, norm=norm, interleaved=interleaved, far=far)


def _attn(name, kind, lens, n_kv, group, *, d=128, page=16, window=0, sinks=0, **more):
    return dict(name=name, kind=kind, lens=lens, n_kv=n_kv, group=group, d=d, page=page, window=window, sinks=sinks,
                **more)


def listed():
    return [
        # the new token of one user in a conversation about a long video
        _heads("axes-1", "axes", 1, 8, 4, sections="16,24,24", far=90000),
        # a prompt chunk of text and images, the engine's largest step, axes in turn over the pairs
        _heads("axes-8192", "axes", 8192, 8, 4, sections="24,20,20", cycled=True),
        # the patches of a few images and a summary token in an image encoder: two axes, as many key heads as query heads
        _heads("axes-image-4097", "axes", 4097, 16, 1, d=64, sections="16,16", norm=False),
        # a decode step of a small batch into the 4-bit cache
        _heads("write4-32", "write4", 32, 8, 4, far=30000),
        # a prompt chunk with images into it
        _heads("write4-8192", "write4", 8192, 8, 4, sections="16,24,24"),
        # one user, a short chat
        _attn("decode4-500-1", "decode4", "500", 8, 4),
        # one user, deep into a long one
        _attn("decode4-128k-1", "decode4", "131072", 8, 4),
        # a ragged serving batch
        _attn("decode4-batch-32", "decode4", "32768,31007,28123,24576,21333,19001,16384,15001,12288,11117,9999,8192,"
              "7001,5555,4097,3001,2500,2049,1777,1500,1025,1024,1000,800,513,400,257,100,33,17,2,1", 8, 4),
        # many users in a layer that keeps a window, another head size and cache page
        _attn("decode4-window-d64", "decode4", ",".join(str(301 * i + 5) for i in range(1, 97)), 4, 8, d=64, page=32,
              window=4096, sinks=4),
        # a whole prompt
        _attn("prefill4-8192", "prefill4", "8192", 8, 4, new="8192"),
        # a chunk at the end of a long document, wide query groups
        _attn("prefill4-64k-512", "prefill4", "65536", 2, 16, new="512"),
        # chunks of several prompts and a decoding request together, in a layer that keeps a window, wide heads
        _attn("prefill4-ragged-d256", "prefill4", "5003,2049,4096,700,129", 4, 4, d=256, page=32,
              new="1301,2049,1024,1,129", window=1024, sinks=4),
    ]


def draw(rng):
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))  # noqa: E731
    kind = rng.choice(["axes", "axes", "write4", "write4", "decode4", "decode4", "decode4", "prefill4", "prefill4"])
    d, page = rng.choice([(128, 16)] * 4 + [(64, 16), (256, 16), (128, 32), (128, 64), (64, 32), (256, 64)])
    n_kv, group = rng.choice([(8, 4), (8, 4), (8, 8), (4, 8), (4, 7), (2, 16), (16, 1), (1, 16), (3, 5)])
    if kind in ("axes", "write4"):
        rot = rng.choice([d, d, d // 2, d // 4])
        axes = rng.choice([2, 3, 3, 4]) if kind == "axes" or rng.random() < 0.4 else 0
        cut = sorted(rng.randint(1, rot // 2) for _ in range(axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0] + cut, cut + [rot // 2])) if axes else ""
        return {k: v for k, v in _heads("", kind, max(1, min(log(1, 8192), (8192 * 48 * 128) // ((group + 2) * n_kv * d))),
                                        n_kv, group, d=d, page=page, rot=rot, sections=sections,
                                        cycled=rng.random() < 0.5, norm=rng.random() < 0.6,
                                        interleaved=rng.random() < 0.4, far=rng.choice([0, 0, log(1, 131000)])).items()
                if k != "name"}
    window = rng.choice([0, 0, log(16, 8192)])
    sinks = rng.choice([0, 4, rng.randint(1, 300)]) if window else 0
    if kind == "decode4":
        lens = _spread(log(1, 64), 1, log(100, 131072), rng.randint(0, 1 << 30))
        while sum(lens) * n_kv * d > 250000 * 8 * 128 or len(lens) * min(window or max(lens), max(lens)) * n_kv * d > 1 << 30:
            lens = lens[1:] if len(lens) > 1 else [lens[0] // 2]
        return {k: v for k, v in _attn("", kind, ",".join(map(str, lens)), n_kv, group, d=d, page=page, window=window,
                                       sinks=sinks).items() if k != "name"}
    new = _spread(rng.choice([1, 1, 2, 4, 6]), 1, log(16, 4096), rng.randint(0, 1 << 30))
    lens = [n + rng.choice([0, log(1, 4000), log(1, 40000)]) for n in new]
    while len(new) * max(new) * max(lens) * n_kv * group * d > 8192 * 8192 * 32 * 128 // 2:
        new, lens = [-(-n // 2) for n in new], [-(-n // 2) for n in lens]
    return {k: v for k, v in _attn("", kind, ",".join(map(str, lens)), n_kv, group, d=d, page=page, window=window,
                                   sinks=sinks, new=",".join(map(str, new))).items() if k != "name"}


def _spread(n, lo, hi, pick):
    """n whole numbers of [lo, hi], spread over their logarithm."""
    r = random.Random(pick)
    return [min(hi, max(lo, int(math.exp(r.uniform(math.log(lo), math.log(hi + 1)))))) for _ in range(n)]


def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _blocks(case):
    return -(-case["tokens"] // case["page"]) + 5


def _visible(case, position):
    """How many keys a query at `position` sees."""
    w, s = case["window"], case["sinks"]
    return position + 1 if not w else min(position + 1, w) + min(s, max(0, position + 1 - w))


def work(case):
    kind, n_kv, group, d = case["kind"], case["n_kv"], case["group"], case["d"]
    row4 = 2 * n_kv * (d // 2 + d // 32)                           # K and V of one token in 4 bits
    if kind in ("axes", "write4"):
        t, H, axes = case["tokens"], n_kv * group, len(_ints(case["sections"])) or 1
        heads_in, q_out = t * (H + 2 * n_kv) * d * 2, t * H * d * 2
        small = t * (4 * axes + 8 + 4 * case["rot"])               # positions, slots, angles
        if kind == "axes":
            return dict(bytes=heads_in + q_out + t * 2 * n_kv * d * 2 + small, flops=t * (H + n_kv) * d * 10)
        rows = _blocks(case) * case["page"]                        # all of the cache, read back
        return dict(bytes=heads_in + q_out + t * row4 + small + rows * (row4 + 4 * n_kv * d),
                    flops=t * (H + n_kv) * d * 10)
    qo = 4 * n_kv * group * d                                      # q and the output of one token
    dot = 4 * n_kv * group * d
    lens = _ints(case["lens"])
    if kind == "decode4":
        keys = sum(_visible(case, n - 1) for n in lens)
        return dict(bytes=keys * row4 + len(lens) * qo, flops=keys * dot)
    new = _ints(case["new"])
    pairs = sum(sum(_visible(case, p) for p in range(n - m, n)) for n, m in zip(lens, new))
    keys = sum(min(n, (case["window"] or n) + m - 1 + case["sinks"]) for n, m in zip(lens, new))
    return dict(bytes=keys * row4 + sum(new) * qo, flops=pairs * dot)


# ---- inputs ------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _codes(x):
    """x (..., d) in 32 or 64 bits as 4-bit codes, one a byte, and the scales' biased exponents (..., d / 32)."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    frac, exp = torch.frexp(top)                                   # frac in [1/2, 1): top <= 7/8 * 2^exp or not
    e = torch.where(frac <= 0.875, exp - 3, exp - 2).clamp(-125, 125)
    e = torch.where(top == 0, torch.full_like(e, -125), e)
    y = torch.ldexp(b, -e[..., None].to(b.dtype)) if b.dtype == torch.float64 else b * torch.exp2(-e[..., None].float())
    y, a = y.flatten(-2), y.flatten(-2).abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, (lo, hi) in enumerate(zip(LEVELS, LEVELS[1:])):
        border = (lo + hi) / 2
        code += (a >= border) if i % 2 else (a > border)           # ties go to the even code
    code += 8 * (y < 0).to(torch.uint8)
    return code, torch.where(top.isfinite(), e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _pack(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def _values(packed, scale):
    """The values (..., d) in 32 bits that packed codes (..., d / 2) and exponents (..., d / 32) stand for."""
    table = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=packed.device)
    x = torch.stack([table[(packed & 15).long()], table[(packed >> 4).long()]], dim=-1).flatten(-2)
    s = torch.where(scale == 255, torch.full((), math.nan, device=packed.device), torch.exp2(scale.float() - 127))
    return (x.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _random_cache(g, blocks, page, n_kv, d):
    """Codes (blocks, 2, page, n_kv, d / 2) and exponents (blocks, 2, page, n_kv, d / 32) of K and V from N(0, 1), four
    channels of each key head x8; and, for the framework's side, its cache of the same rows."""
    scale = torch.ones(2, 1, n_kv, d, device="cuda")
    for h in range(n_kv):
        scale[0, 0, h, torch.randperm(d, generator=g, device="cuda")[:4]] = 8.0
    packed = torch.empty(blocks, 2, page, n_kv, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(blocks, 2, page, n_kv, d // 32, dtype=torch.uint8, device="cuda")
    cache = _own_cache(blocks, page, n_kv, d) if own else None
    step = max(1, (1 << 25) // (2 * page * n_kv * d))
    for lo in range(0, blocks, step):
        n = min(step, blocks - lo)
        x = (torch.randn(n, 2, page, n_kv, d, generator=g, device="cuda") * scale).to(torch.bfloat16).float()
        code, scales[lo:lo + n] = _codes(x)
        packed[lo:lo + n] = _pack(code)
        if own:
            _own_fill(cache, lo * page, _values(packed[lo:lo + n], scales[lo:lo + n]).to(torch.bfloat16))
    return (cache,) if own else (packed, scales)


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "locks-kv_amd")
    if root not in sys.path:
        sys.path.insert(0, root)


def _own_cache(blocks, page, n_kv, d):
    _framework()
    from locks.attention import kv4_cache
    return kv4_cache(blocks, n_kv=n_kv, head_dim=d, page=page, device="cuda")


def _own_fill(cache, slot, kv):
    """Rows of values kv (n, 2, page, n_kv, d) into the framework's cache from `slot` on: values that 4 bits hold are
    written as they are."""
    from locks.attention import qk_norm_rope_write
    k, v = (kv[:, i].flatten(0, 1) for i in range(2))
    at = torch.arange(k.shape[0], device="cuda")
    qk_norm_rope_write(k, k, v, at.to(torch.int32), slot + at, cache, None, torch.empty_like(k))


def prepare(case, seed):
    if own:
        _framework()
    st = {"case": case}
    (_prepare_heads if case["kind"] in ("axes", "write4") else _prepare_attention)(case, _gen(seed), st)
    if own and case["kind"] in ("decode4", "prefill4"):
        from locks.attention import attn_workspace
        st["ws"] = attn_workspace("cuda", max_tokens=st["q"].shape[0], n_kv=case["n_kv"], G=case["group"],
                                  head_dim=case["d"])
    return st


def _axis_of_pair(case):
    """The axis of each pair: sections one after the other, or in turn until an axis has its count."""
    left = _ints(case["sections"])
    if not case["cycled"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    out, a = [], 0
    while any(left):
        if left[a]:
            out.append(a)
            left[a] -= 1
        a = (a + 1) % len(left)
    return out


def _grid_positions(case, g):
    """Positions (axes, tokens) of text and images in turn: along all axes the same for text, and a grid's for an image,
    which text goes on behind of; from `far` on."""
    n, axes = case["tokens"], len(_ints(case["sections"])) or 1
    parts, have, at, image = [], 0, case["far"], False
    sides = torch.randint(3, 48, (64, 4), generator=g, device="cuda").tolist()
    while have < n:
        t, h, w, text = sides[len(parts) % 64]
        if image and axes > 1:
            shape = ([h, w] if axes == 2 else [t % 4 + 1, h, w] + [2] * (axes - 3))
            grid = torch.stack(torch.meshgrid(*(torch.arange(s, device="cuda") for s in shape), indexing="ij")).flatten(1)
            parts.append(at + grid)
            at += max(shape)
        else:
            parts.append((at + torch.arange(text, device="cuda")).expand(axes, text))
            at += text
        have += parts[-1].shape[1]
        image = not image
    return torch.cat(parts, dim=1)[:, :n].to(torch.int32).contiguous()


def _prepare_heads(case, g, st):
    t, n_kv, d, rot, page = (case[k] for k in ("tokens", "n_kv", "d", "rot", "page"))
    H, blocks = n_kv * case["group"], _blocks(case)
    # the projection's output, q, k and v of a token side by side; a few channels of the keys large
    packed = torch.randn(t, (H + 2 * n_kv) * d, generator=g, device="cuda")
    packed[:, H * d:(H + n_kv) * d].view(t, n_kv, d)[:, :, torch.randperm(d, generator=g, device="cuda")[:4]] *= 8
    packed = packed.to(torch.bfloat16)
    q, k, v = (x.view(t, -1, d) for x in packed.split([H * d, n_kv * d, n_kv * d], dim=1))
    pages = torch.randperm(blocks, generator=g, device="cuda")
    at = torch.arange(t, device="cuda")
    positions = _grid_positions(case, g)
    freq = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(case["far"] + t + 64, dtype=torch.float64, device="cuda")[:, None] * freq
    weight = lambda: (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)  # noqa: E731
    st |= dict(q=q, k=k, v=v, positions=positions if case["sections"] else positions[0],
               slots=pages[at // page] * page + at % page, eps=1e-6,
               cos_sin=torch.cat([angle.cos(), angle.sin()], dim=1).float(),
               q_weight=weight() if case["norm"] else None, k_weight=weight() if case["norm"] else None,
               q_out=torch.zeros(t, H, d, dtype=torch.bfloat16, device="cuda"))
    if case["kind"] == "axes":
        st["cache"] = torch.zeros(blocks, 2, page, n_kv, d, dtype=torch.bfloat16, device="cuda")
    else:
        st["kv4"] = _random_cache(g, blocks, page, n_kv, d)
        st |= dict(all_slots=torch.arange(blocks * page, device="cuda"),
                   k_rows=torch.zeros(blocks * page, n_kv, d, dtype=torch.bfloat16, device="cuda"),
                   v_rows=torch.zeros(blocks * page, n_kv, d, dtype=torch.bfloat16, device="cuda"))
    if own:
        from locks.attention import RopeAxes
        made = RopeAxes.cycled if case["cycled"] else RopeAxes.sections
        st["axes"] = made(_ints(case["sections"])) if case["sections"] else None


def _prepare_attention(case, g, st):
    page, n_kv, d = case["page"], case["n_kv"], case["d"]
    lens = _ints(case["lens"])
    new = _ints(case["new"]) if "new" in case else [1] * len(lens)
    need = [-(-n // page) for n in lens]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at, starts = 0, [0]
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
        starts.append(starts[-1] + new[i])
    st |= dict(lens=lens, new=new, kv4=_random_cache(g, blocks, page, n_kv, d), table=table, seq_lens=_i32(lens),
               starts=_i32(starts), scale=1.0 / math.sqrt(d))
    H, total = n_kv * case["group"], sum(new)
    st |= dict(q=torch.randn(total, H, d, generator=g, device="cuda").to(torch.bfloat16),
               out=torch.zeros(total, H, d, dtype=torch.bfloat16, device="cuda"),
               lse=torch.zeros(total, H, device="cuda"))


# ---- one pass ----------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return {"axes": _own_axes, "write4": _own_write4, "decode4": _own_decode4, "prefill4": _own_prefill4}[
            case["kind"]](case, st)
    return {"axes": _plain_axes, "write4": _plain_write4, "decode4": _plain_decode4, "prefill4": _plain_prefill4}[
        case["kind"]](case, st)


def _own_write(case, st, cache):
    from locks.attention import qk_norm_rope_write
    qk_norm_rope_write(st["q"], st["k"], st["v"], st["positions"], st["slots"], cache, st["cos_sin"], st["q_out"],
                       q_weight=st["q_weight"], k_weight=st["k_weight"], eps=st["eps"],
                       interleaved=case["interleaved"], axes=st["axes"])


def _own_axes(case, st):
    _own_write(case, st, st["cache"])
    return dict(q=st["q_out"], cache=st["cache"])


def _own_write4(case, st):
    from locks.attention import kv4_read
    _own_write(case, st, st["kv4"][0])
    kv4_read(st["kv4"][0], st["all_slots"], st["k_rows"], st["v_rows"])
    return dict(q=st["q_out"], k=st["k_rows"], v=st["v_rows"])


def _own_decode4(case, st):
    from locks.attention import window_decode
    window_decode(st["q"], st["kv4"][0], st["table"], st["seq_lens"], st["out"], st["ws"], n_req=len(st["lens"]),
                  window=case["window"], sinks=case["sinks"], scale=st["scale"], lse=st["lse"])
    return dict(out=st["out"], lse=st["lse"])


def _own_prefill4(case, st):
    from locks.attention import window_prefill
    window_prefill(st["q"], st["kv4"][0], st["table"], st["seq_lens"], st["starts"], st["out"], st["ws"],
                   n_req=len(st["lens"]), window=case["window"], sinks=case["sinks"], scale=st["scale"], lse=st["lse"])
    return dict(out=st["out"], lse=st["lse"])


def _plain_angles(case, st):
    """Cosines and sines (tokens, rot / 2) of each token and pair."""
    half = case["rot"] // 2
    if not case["sections"]:
        return st["cos_sin"][st["positions"].long()].split(half, dim=1)
    row = st["positions"].long()[torch.tensor(_axis_of_pair(case), device="cuda")].T     # (tokens, rot / 2)
    return st["cos_sin"][:, :half].gather(0, row), st["cos_sin"][:, half:].gather(0, row)


def _plain_heads(x, weight, cos, sin, case, eps):
    rot = case["rot"]
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype)
    a, rest = x[..., :rot], x[..., rot:]
    cos, sin = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    if case["interleaved"]:
        u, w = a[..., 0::2], a[..., 1::2]
        a = torch.stack([u * cos - w * sin, w * cos + u * sin], dim=-1).flatten(-2)
    else:
        u, w = a[..., :rot // 2], a[..., rot // 2:]
        a = torch.cat([u * cos - w * sin, w * cos + u * sin], dim=-1)
    return torch.cat([a, rest], dim=-1)


def _plain_axes(case, st):
    page = case["page"]
    cos, sin = _plain_angles(case, st)
    block, at = st["slots"] // page, st["slots"] % page
    st["cache"][block, 0, at] = _plain_heads(st["k"].float(), st["k_weight"], cos, sin, case, st["eps"]).to(torch.bfloat16)
    st["cache"][block, 1, at] = st["v"]
    return dict(q=_plain_heads(st["q"].float(), st["q_weight"], cos, sin, case, st["eps"]).to(torch.bfloat16),
                cache=st["cache"])


def _plain_write4(case, st):
    page, n_kv, d = case["page"], case["n_kv"], case["d"]
    packed, scales = st["kv4"]
    cos, sin = _plain_angles(case, st)
    block, at = st["slots"] // page, st["slots"] % page
    for i, x in enumerate((_plain_heads(st["k"].double(), st["k_weight"], cos, sin, case, st["eps"]), st["v"].float())):
        code, scale = _codes(x)
        packed[block, i, at] = _pack(code)
        scales[block, i, at] = scale
    k, v = (_values(packed[:, i], scales[:, i]).to(torch.bfloat16).view(-1, n_kv, d) for i in range(2))
    return dict(q=_plain_heads(st["q"].float(), st["q_weight"], cos, sin, case, st["eps"]).to(torch.bfloat16), k=k, v=v)


def _plain_softmax(q, k, v, seen):
    """q (b, kv, rows, d) scaled, k, v (b, kv, keys, d), seen (b, 1, rows, keys): outputs and log-sum-exp."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total, (top + total.log())[..., 0]


def _plain_keys(case, st, token):
    """K and V (b, kv, keys, d) in 32 bits of the token numbers (b, keys) of each request's row."""
    page = case["page"]
    packed, scales = st["kv4"]
    block = st["table"].long().gather(1, token // page)
    return [_values(packed[block, i, token % page], scales[block, i, token % page]).transpose(1, 2).contiguous()
            for i in range(2)]


def _plain_decode4(case, st):
    n_kv, group, w, s = case["n_kv"], case["group"], case["window"], case["sinks"]
    lens = st["seq_lens"].long()
    longest = max(st["lens"])
    # the first `sinks` tokens and the last `window` ones, side by side (all of them with no window)
    tail = torch.arange(min(w or longest, longest), device="cuda")
    low = (lens - w).clamp(min=0) if w else torch.zeros_like(lens)
    token = torch.cat([torch.arange(s, device="cuda").expand(len(lens), s), low[:, None] + tail], dim=1)
    seen = torch.cat([token[:, :s] < low[:, None], token[:, s:] < lens[:, None]], dim=1)
    k, v = _plain_keys(case, st, token.clamp(max=longest - 1))
    q = st["q"].float().view(len(lens), n_kv, group, -1) * st["scale"]
    o, lse = _plain_softmax(q, k, v, seen[:, None, None])
    return dict(out=o.flatten(1, 2).to(torch.bfloat16), lse=lse.flatten(1, 2))


def _plain_prefill4(case, st):
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
    k, v = _plain_keys(case, st, token.expand(b, longest))
    q = st["q"][row].float() * st["scale"]                         # (b, most, H, d)
    q = q.view(b, most, n_kv, group, -1).permute(0, 2, 3, 1, 4).reshape(b, n_kv, group * most, -1)
    seen = seen[:, None, None].expand(b, 1, group, most, longest).reshape(b, 1, group * most, longest)
    o, lse = _plain_softmax(q, k, v, seen)
    o = o.view(b, n_kv, group, most, -1).permute(0, 3, 1, 2, 4).flatten(2, 3)
    lse = lse.view(b, n_kv, group, most).permute(0, 3, 1, 2).flatten(2, 3)
    return dict(out=o[real].to(torch.bfloat16), lse=lse[real])


# ---- the definition in 64 bits -----------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False                                          # the inputs in their plain layout
    try:
        st = {"case": case}
        (_prepare_heads if case["kind"] in ("axes", "write4") else _prepare_attention)(case, _gen(seed), st)
    finally:
        own = was
    return (_exact_heads if case["kind"] in ("axes", "write4") else _exact_attention)(case, st)


def _exact_values(packed, scale):
    """The values of 4-bit entries in 64 bits, from the bits: sign, two of exponent, one of mantissa."""
    c = torch.stack([packed % 16, packed // 16], dim=-1).flatten(-2).long()
    sign, ex, man = 1 - 2 * (c // 8), c // 2 % 4, (c % 2).double()
    mag = torch.where(ex == 0, man / 2, (1 + man / 2) * 2.0 ** (ex - 1).double())
    s = 2.0 ** (scale.double() - 127)
    s[scale == 255] = math.nan
    return sign * mag * s.repeat_interleave(32, dim=-1)


def _exact_round(x):
    """x (..., d) rounded to 4 bits: a step that follows the magnitude, round half to even."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -140)
    e = torch.ceil(torch.log2(top / 7))
    e = torch.where(7 * 2.0 ** (e - 1) >= top, e - 1, e)           # where the logarithm was off
    e = torch.where(7 * 2.0 ** e < top, e + 1, e).clamp(-125, 125)
    y = b / 2.0 ** e
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return ((y / step).round() * step).clamp(-6, 6).mul(2.0 ** e).flatten(-2)


def _exact_heads(case, st):
    """Each pair of entries as a complex number, turned by its token's unit number."""
    rot, page, t, n_kv, d = (case[k] for k in ("rot", "page", "tokens", "n_kv", "d"))
    half = rot // 2
    turn = torch.empty(t, half, dtype=torch.complex128, device="cuda")
    axis = _axis_of_pair(case) if case["sections"] else [0] * half
    for j, a in enumerate(axis):
        rows = (st["positions"][a] if case["sections"] else st["positions"]).long()
        turn[:, j] = torch.complex(st["cos_sin"][rows, j].double(), st["cos_sin"][rows, half + j].double())

    def made(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / d + st["eps"]).sqrt() * weight.double()
        pairs = (torch.arange(rot, device="cuda").view(-1, 2).T if case["interleaved"]
                 else torch.arange(rot, device="cuda").view(2, -1))
        z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * turn[:, None]
        x = x.clone()
        x[..., pairs[0]], x[..., pairs[1]] = z.real, z.imag
        return x

    q, k, v = made(st["q"], st["q_weight"]), made(st["k"], st["k_weight"]), st["v"].double()
    if case["kind"] == "axes":
        flat = st["cache"].double()
        flat[st["slots"] // page, 0, st["slots"] % page] = k
        flat[st["slots"] // page, 1, st["slots"] % page] = v
        return dict(q=q, cache=flat)
    packed, scales = st["kv4"]
    rows = [_exact_values(packed[:, i], scales[:, i]).reshape(-1, n_kv, d) for i in range(2)]
    for r, x in zip(rows, (k, v)):
        r[st["slots"]] = _exact_round(x)
    return dict(q=q, k=rows[0], v=rows[1])


def _exact_attention(case, st):
    """Request by request and head by head, over every token of the request."""
    page, group, w = case["page"], case["group"], case["window"]
    if sum(n * m for n, m in zip(st["lens"], st["new"])) * case["n_kv"] * group * case["d"] > 1 << 43:
        return None
    packed, scales = st["kv4"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["lse"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (n, m) in enumerate(zip(st["lens"], st["new"])):
        blocks = st["table"][r, :-(-n // page)].long()
        i = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = (j > i) | ((i - j >= w) & (j >= case["sinks"]) if w else torch.zeros_like(j > i))
        for kh in range(case["n_kv"]):
            k, v = (_exact_values(packed[blocks, x, :, kh], scales[blocks, x, :, kh]).flatten(0, 1)[:n].contiguous()
                    for x in range(2))
            kt = k.T.contiguous()
            for h in range(kh * group, (kh + 1) * group):
                logit = st["q"][at:at + m, h].double() @ kt * st["scale"]
                logit[hidden] = -math.inf
                z = torch.logsumexp(logit, dim=1)
                lse[at:at + m, h] = z
                out[at:at + m, h] = torch.exp(logit - z[:, None]) @ v
        at += m
    return dict(out=out, lse=lse)
