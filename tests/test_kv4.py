"""The paged cache in 4 bits: what is written, read back and attended to, against the
definition in 64 bits, and the calls that are refused.

Tolerance of attention: that of tests/test_window.py, whose arithmetic it is (the
values of the codes are exact in bf16).  What is written has none: a code is decided
in 64 bits, and so are the oracle's; only an entry that the two put on opposite sides
of a border by their own rounding (2^-40 of the border, a few hundred roundings of
2^-53) may differ."""
import pytest
import torch

from locks import _lib
from locks.attention import (RopeAxes, attn_workspace, kv4_cache, kv4_read, prefix_decode, qk_norm_rope_write,
                             window_decode, window_prefill)
from tests.test_rope_axes import formula, inputs
from tests.test_window import GEOMETRY, LENS, _agree, _empty_row, _exact, _no_rows, _outs

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantised(x):
    """x (..., d) float64: (codes (..., d), exponents (..., d / 32), values (..., d), next to a border)."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.full_like(top, -125)
    for k in range(-125, 125):                                   # the smallest e with top <= 7 * 2^e
        e = torch.where(top > 7 * 2.0 ** k, torch.full_like(e, k + 1.0), e)
    y = (b * torch.exp2(-e)[..., None]).flatten(-2)
    a, code, near = y.abs(), torch.zeros_like(y, dtype=torch.long), torch.zeros_like(y, dtype=torch.bool)
    for i in range(7):
        border = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += (a >= border) if i % 2 else (a > border)
        near |= ((a - border).abs() < 2.0 ** -40) & (a != border)
    near |= ((a - 7).abs() < 2.0 ** -38)                         # the border of the scale
    value = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[code] * y.sign()
    value = (value.unflatten(-1, (-1, 32)) * torch.exp2(e)[..., None])
    value = torch.where(top.isfinite()[..., None], value, torch.nan).flatten(-2)
    return code + 8 * (y < 0), torch.where(top.isfinite(), e, 128), value, near


def _blank(blocks, n_kv, d, page, gap=0):
    """A cache full of 255: codes of -6 and NaN scales wherever nothing is written.
    ``gap``: bytes between its blocks' and heads' records."""
    if gap:
        wide = torch.full((blocks, n_kv + 1, page // 16 * 17 * d + gap), 255, dtype=torch.uint8, device="cuda")
        return wide[:, 1:, gap:].unflatten(2, (page // 16, 17 * d))
    return kv4_cache(blocks, n_kv=n_kv, head_dim=d, page=page, device="cuda").fill_(255)


def _read(cache, slots):
    n_kv, d = cache.shape[1], cache.shape[3] // 17
    k = torch.full((slots.shape[0], n_kv, d), 7.0, dtype=torch.bfloat16, device="cuda")
    v = torch.full((slots.shape[0], n_kv, d), 7.0, dtype=torch.bfloat16, device="cuda")
    kv4_read(cache, slots, k, v)
    return k, v


def _written(x, axes, cache, *, interleaved=False, eps=1e-6):
    before = cache.clone()
    T = x["q"].shape[0]
    q, k_out = torch.zeros_like(x["q"]), torch.zeros_like(x["k"])
    pos = x["pos"] if axes is not None else x["pos"][0].contiguous()
    qk_norm_rope_write(x["q"], x["k"], x["v"], pos, x["slots"], cache, x["cs"], q, q_weight=x["qw"], k_weight=x["kw"],
                       eps=eps, interleaved=interleaved, k_out=k_out, axes=axes)
    one = axes or RopeAxes([0] * (x["cs"].shape[1] // 2))
    # the entry's eps is fp32
    k64 = formula(x["k"], x["kw"], x["pos"], x["cs"], one, float(torch.tensor(eps)), interleaved)
    k, v = _read(cache, x["slots"])
    _, _, want, near = quantised(k64[0])
    assert torch.equal(torch.where(near, 0, k.double()), torch.where(near, 0, want)) and int(near.sum()) < 3
    assert torch.equal(v.double(), quantised(x["v"].double())[2])
    tol = 2.0 ** -16 * 1.01
    for got, (y, mag) in ((q, formula(x["q"], x["qw"], x["pos"], x["cs"], one, eps, interleaved)), (k_out, k64)):
        assert bool(((got.double() - y).abs() <= 2.0 ** -8 * y.abs() + tol * mag).all())
    # nothing else has changed
    others = torch.ones(cache.shape[0] * cache.shape[2] * 16, dtype=torch.bool, device="cuda")
    others[x["slots"]] = False
    rest = others.nonzero()[:, 0]
    old, new = _read(before, rest), _read(cache, rest)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(old, new))
    assert T + rest.shape[0] == others.shape[0]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d, rot, page", [(64, 64, 16), (64, 16, 32), (128, 128, 16), (128, 48, 64), (256, 256, 32),
                                          (256, 64, 16)])
@pytest.mark.parametrize("T, H, n_kv", [(1, 32, 8), (7, 5, 1), (130, 14, 2)])
def test_write(T, H, n_kv, d, rot, page, interleaved):
    x = inputs(T, H, n_kv, d, rot, 1, page=page, seed=T + d + rot)
    _written(x, None, _blank(x["blocks"], n_kv, d, page), interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("w", [None, torch.float32])
@pytest.mark.parametrize("d, axes", [(128, RopeAxes.sections((16, 24, 24))), (64, RopeAxes.cycled((11, 11, 10))),
                                     (256, RopeAxes.sections((30, 34, 64)))])
def test_write_axes_and_gaps(d, axes, w):
    x = inputs(91, 8, 4, d, d, 3, w=w, far=5000)
    _written(x, axes, _blank(x["blocks"], 4, d, 16, gap=48))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [9, 700])
def test_write_where_fp32_would_not_do(T, interleaved):
    """Weights past 2^60, sums of squares that overflow fp32 or underflow, rows whose entries
    cancel: the codes are those of 64 bits all the same."""
    x = inputs(T, 8, 4, 128, 128, 1, w=torch.float32, seed=T)
    x["kw"][5], x["kw"][70] = 1e30, -1e19
    x["k"][0], x["k"][1] = x["k"][0] * 1e30, x["k"][1] * 1e-30
    x["k"][2, :, :64] = x["k"][2, :, 64:]
    x["q"][0] = 0
    x["pos"][0, 0:2] = 3
    cache = _blank(x["blocks"], 4, 128, 16)
    q = torch.zeros_like(x["q"])
    for kw in (x["kw"], torch.ones_like(x["kw"])):
        qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"][0], x["slots"], cache, x["cs"], q, q_weight=x["qw"],
                           k_weight=kw, interleaved=interleaved)
        k64 = formula(x["k"], kw, x["pos"], x["cs"], RopeAxes([0] * 64), float(torch.tensor(1e-6)), interleaved)[0]
        _, _, want, near = quantised(k64)
        k, _ = _read(cache, x["slots"])
        assert torch.equal(torch.where(near, 0, k.double()), torch.where(near, 0, want)) and int(near.sum()) < 3


@pytest.mark.gpu
def test_write_many_tokens():
    x = inputs(5000, 3, 1, 128, 128, 1, page=16)
    _written(x, None, _blank(x["blocks"], 1, 128, 16))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_layout(d):
    """The bytes of a tile, as its documentation has them."""
    page, n_kv = 32, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    k, v = (torch.randn(2 * page, n_kv, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    cache = _blank(2, n_kv, d, page)
    at = torch.arange(2 * page, device="cuda")
    qk_norm_rope_write(k, k, v, at.int(), at, cache, None, torch.empty_like(k))
    raw = cache.cpu()
    for half, x in enumerate((k, v)):
        code, e, _, _ = (y.cpu() for y in quantised(x.double()))
        for t, h in ((0, 0), (5, 1), (15, 0), (16, 1), (43, 1), (63, 0)):
            tile, key = raw[t // page, h, t % page // 16], t % 16
            for i in range(d):
                if half == 0:
                    lane, n = 16 * (i // (d // 4)) + key, i % (d // 4)
                else:
                    lane, n = 16 * (key // 4) + i // (d // 16), (key % 4) * (d // 16) + i % (d // 16)
                byte = n // 2                                    # of the lane's d / 8 bytes
                place = half * 8 * d + (byte // 16 * 1024 + lane * 16 + byte % 16 if d == 256 else lane * (d // 8) + byte)
                assert int(tile[place]) >> 4 * (n % 2) & 15 == int(code[t, h, i])
                blk = i // 32
                if half:
                    place = 16 * d + d // 2 + (key // 4 * (d // 32) + blk) * 4 + key % 4
                else:
                    place = 16 * d + ((blk // 2 * 16 + key) * 2 + blk % 2 if d == 256 else blk * 16 + key)
                assert int(tile[place]) - 127 == int(e[t, h, blk])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_extreme_values(d):
    """Zeros, ties, the smallest and largest numbers, infinities and NaN; no weight and
    no rotation, so that K holds the same as V."""
    x = torch.zeros(40, 1, d, device="cuda")
    tie = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5., 7., -.25, -.75, -5., 6.5, 1e-30, .2509765625], device="cuda")
    for i, s in enumerate((1.0, 2.0 ** -120, 2.0 ** 124, 2.0 ** 20)):
        x[i, 0, :14] = tie * s
    x[4, 0, :2] = torch.tensor([3.3895e38, -3e38], device="cuda")        # past 7 * 2^125: the largest value
    x[5, 0, :3] = torch.tensor([1e-40, 2.0 ** -126, -2.0 ** -133], device="cuda")
    x[6, 0, 31], x[7, 0, 32], x[8, 0, d - 1] = torch.inf, -torch.inf, torch.nan
    x[6:9, 0, 0] = 1.0
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x[9:] = torch.randn(31, 1, d, generator=g, device="cuda") * torch.exp(20 * torch.randn(31, 1, 1, generator=g, device="cuda"))
    x = x.to(torch.bfloat16)
    cache, at = _blank(3, 1, d, 16), torch.arange(40, device="cuda")
    qk_norm_rope_write(x, x, x, at.int(), at, cache, None, torch.empty_like(x))
    _, _, want, _ = quantised(x.double())
    for got in _read(cache, at):
        assert torch.equal(got.double().nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))


@pytest.mark.gpu
def test_read_slots():
    """Slots twice, outside the cache, outputs with gaps; values that 4 bits hold come
    back as they went in."""
    n_kv, d = 3, 128
    x = inputs(50, 3, n_kv, d, d, 1)
    cache = _blank(x["blocks"], n_kv, d, 16)
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"][0], x["slots"], cache, x["cs"], torch.empty_like(x["q"]))
    k, v = _read(cache, x["slots"])
    slots = torch.stack([x["slots"], x["slots"].flip(0), torch.full_like(x["slots"], -1)], 1).flatten().contiguous()
    slots[0] = x["blocks"] * 16
    wide = torch.full((151, n_kv, 2, d), 7.0, dtype=torch.bfloat16, device="cuda")
    kv4_read(cache, slots, wide[:, :, 1], wide[:, :, 0])
    want = torch.full_like(wide, 7.0)
    want[:150:3, :, 1], want[:150:3, :, 0] = k, v
    want[1:150:3, :, 1], want[1:150:3, :, 0] = k.flip(0), v.flip(0)
    want[0] = 7.0
    assert torch.equal(wide, want)
    again = _blank(x["blocks"], n_kv, d, 16)
    qk_norm_rope_write(k, k, v, x["pos"][0], x["slots"], again, None, torch.empty_like(k))
    assert torch.equal(again, cache)
    kv4_read(cache, slots[:0], k[:0], v[:0])


def case(lens, new, n_kv, G, d, page, *, seed=0, gap=0, width=None):
    """As tests/test_window.py's: a cache of NaN wherever no token lies, ids out of range
    past each request's pages; k, v the values that were written."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    width = width or max(max(pages), 1) + 1
    order = torch.randperm(sum(pages) + 5, generator=g, device="cuda").to(torch.int32)
    bt = torch.randint(-5, 1 << 20, (len(lens), width), generator=g, device="cuda", dtype=torch.int32)
    cache, at, k64, v64 = _blank(sum(pages) + 5, n_kv, d, page, gap), 0, [], []
    for r, n in enumerate(pages):
        bt[r, :n] = order[at:at + n][:width]
        t = torch.arange(lens[r], device="cuda")
        slots = order[at:at + n].long()[t // page] * page + t % page
        at += n
        k = (torch.randn(lens[r], n_kv, d, generator=g, device="cuda") * 1.5).to(torch.bfloat16)
        v = torch.randn(lens[r], n_kv, d, generator=g, device="cuda").to(torch.bfloat16)
        if lens[r]:
            qk_norm_rope_write(k, k, v, t.int(), slots, cache, None, torch.empty_like(k))
        k, v = _read(cache, slots)
        k64.append(k)
        v64.append(v)
    T, starts = sum(new), [0]
    for n in new:
        starts.append(starts[-1] + n)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(q=torch.randn(T, n_kv * G, d, generator=g, device="cuda").to(torch.bfloat16), kv=cache, bt=bt, sl=i(lens),
                qsl=i(starts), k=k64, v=v64, lens=lens, new=new, n_kv=n_kv, G=G, d=d, page=page, scale=1.0 / d ** 0.5)


def _ws(c, tokens=None):
    return attn_workspace("cuda", max_tokens=tokens or max(c["q"].shape[0], 1), n_kv=c["n_kv"], G=c["G"],
                          head_dim=c["d"]).fill_(255)


def _decode(c, window=0, sinks=0, **kw):
    out, lse = _outs(c)
    window_decode(c["q"], c["kv"], c["bt"], c["sl"], out, _ws(c), n_req=len(c["lens"]), window=window, sinks=sinks,
                  scale=c["scale"], lse=lse, **kw)
    return out, lse


def _prefill(c, window=0, sinks=0, **kw):
    out, lse = _outs(c, 3)
    T = c["q"].shape[0]
    window_prefill(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out, _ws(c), n_req=len(c["lens"]), window=window,
                   sinks=sinks, scale=c["scale"], lse=lse, **kw)
    assert bool((out[T:] == 7).all()) and bool((lse[T:] == 7).all())
    return out[:T], lse[:T]


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (1, 1), (16, 4), (17, 16), (64, 17), (100, 300), (512, 5),
                                           (5000, 64)])
@pytest.mark.parametrize("d, page, n_kv, G", GEOMETRY)
def test_decode(d, page, n_kv, G, window, sinks):
    lens = LENS + [0, 3000]
    c = case(lens, [1] * len(lens), n_kv, G, d, page, seed=window + sinks)
    _agree(*_decode(c, window, sinks), _empty_row(c, _exact(_no_rows(c), window, sinks)))


@pytest.mark.gpu
def test_decode_long():
    """Long rows among short ones, bounds of the lengths that are exact, and too low;
    a cache, q and out with gaps; no log-sum-exp asked for."""
    c = case([70001, 5, 33000], [1, 1, 1], 2, 4, 128, 16, gap=16)
    for window, sinks in ((0, 0), (4096, 4), (30000, 100)):
        want = _exact(c, window, sinks)
        _agree(*_decode(c, window, sinks), want)
        _agree(*_decode(c, window, sinks, max_seq_len=70001), want)
        _agree(*_decode(c, window, sinks, max_seq_len=600), want)
    wide = torch.zeros(3, 3, 8, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = c["q"]
    out = torch.zeros(3, 8, 2, 128, dtype=torch.bfloat16, device="cuda")
    window_decode(wide[:, 1], c["kv"], c["bt"], c["sl"], out[:, :, 1], _ws(c), n_req=3, scale=c["scale"])
    assert torch.equal(out[:, :, 1], _decode(c)[0]) and not bool(out[:, :, 0].any())


@pytest.mark.gpu
def test_decode_one_split_many_requests():
    """As many rows as workgroups: the split kernel writes the output itself."""
    lens = [(37 * i) % 300 + 1 for i in range(150)] + [0] * 3
    c = case(lens, [1] * 153, 8, 2, 64, 16)
    _agree(*_decode(c), _empty_row(c, _exact(_no_rows(c), 0, 0)))


@pytest.mark.gpu
def test_lengths_past_the_table():
    """A length past the table sees the table's tokens; a window still ends at the length."""
    c = case([200, 900], [1, 1], 2, 4, 128, 16, width=30)           # 480 tokens of the table
    seen = {**c, "k": [x[:480] for x in c["k"]], "v": [x[:480] for x in c["v"]], "lens": [200, 480]}
    _agree(*_decode(c), _exact(seen, 0, 0))
    # request 1 sees 400 .. 479 and 0 .. 2
    first, second = _exact(seen, 500, 3), _exact(seen, 80, 3)
    _agree(*_decode(c, 500, 3), [torch.stack([x[0], y[1]]) for x, y in zip(first, second)])


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (33, 4), (64, 64), (200, 17), (300, 1000)])
@pytest.mark.parametrize("d, page, n_kv, G", GEOMETRY)
def test_prefill(d, page, n_kv, G, window, sinks):
    lens = [1, 16, 17, 40, 128, 129, 700, 333, 90, 513]
    new = [1, 16, 5, 40, 127, 1, 650, 0, 65, 64]
    c = case(lens, new, n_kv, G, d, page, seed=window)
    _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefill_long(d):
    """A few tokens against a long cache (keys split over workgroups and joined), and
    enough tokens for one split; more than 64 tiles of keys."""
    c = case([12001], [40], 1, 4, d, 16, gap=32)
    _agree(*_prefill(c), _exact(c, 0, 0))
    c = case([9000, 4100], [2100, 4100], 4, 8, d, 64)
    _agree(*_prefill(c), _exact(c, 0, 0))


@pytest.mark.gpu
def test_values_that_are_not_finite():
    """NaN blocks of V reach the rows that see them and no others; a NaN block of K makes
    the rows that see it NaN."""
    for bad_key, n_kv, G, d in ((100, 2, 4, 128), (0, 1, 8, 64), (299, 2, 2, 256)):
        c = case([300, 300], [1, 1], n_kv, G, d, 16)
        slot = c["bt"][0, bad_key // 16].long() * 16 + bad_key % 16
        v = c["v"][0][bad_key:bad_key + 1].clone()
        v[0, 0, 5] = torch.nan
        k = c["k"][0][bad_key:bad_key + 1]
        qk_norm_rope_write(k, k, v, slot[None].int() * 0, slot[None], c["kv"], None, torch.empty_like(k))
        c["v"][0][bad_key, 0, :32] = torch.nan
        for window, sinks in ((0, 0), (50, 0), (250, 1), (100, 120)):
            _agree(*_decode(c, window, sinks), _exact(c, window, sinks))
        p = {**c, "new": [250, 3], "qsl": torch.tensor([0, 250, 253], dtype=torch.int32, device="cuda"),
             "q": torch.randn(253, n_kv * G, d, device="cuda").to(torch.bfloat16)}
        for window, sinks in ((0, 0), (50, 2)):
            _agree(*_prefill(p, window, sinks), _exact(p, window, sinks))
        k = k.clone()
        k[0, 0, 3] = torch.inf
        qk_norm_rope_write(k, k, c["k"][0][bad_key:bad_key + 1], slot[None].int() * 0, slot[None], c["kv"], None,
                           torch.empty_like(k))
        out, lse = _decode(c)
        assert bool(out[0, :G].isnan().all()) and bool(lse[0, :G].isnan().all())
        assert not bool(out[0, G:].isnan().any()) and not bool(out[1].isnan().any())
        if bad_key < 250:
            out, lse = _decode(c, 50)
            assert not bool(out.isnan().any()) and not bool(lse.isnan().any())


@pytest.mark.gpu
def test_large_scores():
    """Scores up to thousands: the running maximum grows again and again.

    Outputs reach below fp32's and bf16's normal numbers here, which the common
    tolerance leaves out: a weight below 2^-126 may count as zero, at most 2^-126 |v| of
    each key over a sum l >= 1 (the largest weight is at least 1), and a bf16 number
    below 2^-126 is off by half of 2^-133."""
    c = case([3000, 1111], [1, 1], 2, 4, 128, 16)
    c["q"] = (c["q"].float() * torch.tensor([300.0, 0.0], device="cuda")[:, None, None]).to(torch.bfloat16)
    o, z, to, tz = _exact(c, 0, 0)
    to += 3000 * 2.0 ** -126 * max(float(v.abs().max()) for v in c["v"]) + 2.0 ** -134
    _agree(*_decode(c), (o, z, to, tz))


@pytest.mark.gpu
def test_replay_follows_lengths():
    """A captured step of write, decode and prefill, replayed with new tokens, lengths and
    tables, with eager work between."""
    n_kv, G, d, page, blocks = 2, 4, 128, 16, 200
    cache = _blank(blocks, n_kv, d, page)
    x = inputs(6, n_kv * G, n_kv, d, d, 1)
    bt = torch.randperm(blocks, device="cuda", dtype=torch.int32)[:180].view(6, 30).contiguous()
    sl = torch.ones(6, dtype=torch.int32, device="cuda")
    qsl = torch.arange(7, dtype=torch.int32, device="cuda")
    slots, pos = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    q, out, out2 = (torch.zeros_like(x["q"]) for _ in range(3))
    ws = attn_workspace("cuda", max_tokens=6, n_kv=n_kv, G=G, head_dim=d)

    def step():
        qk_norm_rope_write(x["q"], x["k"], x["v"], pos, slots, cache, x["cs"], q, q_weight=x["qw"], k_weight=x["kw"])
        window_decode(q, cache, bt, sl, out, ws, n_req=6, scale=0.1)
        window_prefill(q, cache, bt, sl, qsl, out2, ws, n_req=6, scale=0.1)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for n in range(150):
        y = inputs(6, n_kv * G, n_kv, d, d, 1, seed=n)
        for name in ("q", "k", "v"):
            x[name].copy_(y[name])
        at = torch.full((6,), n, device="cuda")
        slots.copy_(bt[:, n // page].long() * page + n % page)
        pos.copy_(at.int())
        sl.copy_(at.int() + 1)
        g.replay()
        if n in (0, 1, 17, 149):
            one, two = out.clone(), out2.clone()
            rows = (bt.long()[:, torch.arange(n + 1, device="cuda") // page] * page + torch.arange(n + 1, device="cuda") % page)
            kv = [_read(cache, r.contiguous()) for r in rows]
            c = dict(q=q, k=[a for a, _ in kv], v=[b for _, b in kv], lens=[n + 1] * 6, new=[1] * 6, n_kv=n_kv, G=G, d=d,
                     scale=0.1)
            want = _exact(c, 0, 0)
            for got in (one, two):
                assert bool(((got.double() - want[0]).abs() <= want[2]).all())
            step()                                               # the same values again
            torch.cuda.synchronize()
            assert torch.equal(out, one) and torch.equal(out2, two)


@pytest.mark.gpu
def test_other_stream():
    c = case([700, 20], [1, 1], 2, 4, 128, 16)
    want = _decode(c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _decode(c)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_engine_step():
    """A serving engine whose dense layer holds its cache in 4 bits: prompt chunk, mixed
    step and decode steps, positions of three axes, through LocksEngine."""
    from locks import LocksConfig
    from locks.backend.engine import LocksEngine
    n_kv, G, d, page, blocks = 2, 4, 128, 16, 64
    selected = torch.zeros(blocks, 2, page, n_kv, d, dtype=torch.bfloat16, device="cuda")
    eng = LocksEngine(LocksConfig(budget_pages=8), [selected], num_heads_q=n_kv * G, num_heads_kv=n_kv, head_dim=d,
                      block_size=page, max_num_seqs=4, max_model_len=512, max_num_batched_tokens=256)
    cache, axes, t = eng.kv4_cache(), RopeAxes.sections((16, 24, 24)), eng.block_tables()
    assert cache.shape == (blocks, n_kv, 1, 17 * d)
    have, ks, vs = [0, 0, 0], [[], [], []], [[], [], []]
    for seed, (new, n_decode) in enumerate((([100, 37, 0], 0), ([1, 1, 150], 2), ([1, 1, 1], 3), ([1, 1, 1], 3))):
        T = sum(new)
        x = inputs(T, n_kv * G, n_kv, d, d, 3, seed=seed)
        rows = torch.arange(3, dtype=torch.int32, device="cuda")
        t.step(rows, torch.tensor(new, dtype=torch.int32, device="cuda"), n_req=3, n_tokens=T)
        q, out = torch.zeros_like(x["q"]), torch.zeros_like(x["q"])
        eng.write_qkv(None, x["q"], x["k"], x["v"], x["pos"], t.slot_mapping[:T], x["cs"], q, q_weight=x["qw"],
                      k_weight=x["kw"], axes=axes, kv_cache=cache)
        eng.forward_dense(q, cache, t.block_table, t.seq_lens, 3, 0.09, out, query_start_loc=t.query_start_loc,
                          n_decode=n_decode, window=120, sinks=4)
        k = quantised(formula(x["k"], x["kw"], x["pos"], x["cs"], axes, float(torch.tensor(1e-6)), False)[0])[2]
        v = quantised(x["v"].double())[2]
        at = 0
        for r, n in enumerate(new):
            have[r] += n
            ks[r].append(k[at:at + n])
            vs[r].append(v[at:at + n])
            at += n
        c = dict(q=q, k=[torch.cat(y) for y in ks], v=[torch.cat(y) for y in vs], lens=have, new=new, n_kv=n_kv, G=G, d=d,
                 scale=0.09)
        want = _exact(c, 120, 4)
        assert bool(((out.double() - want[0]).abs() <= want[2]).all())
    assert not bool(selected.any())


# ---- what is refused -------------------------------------------------------------
def test_refusals():
    for kw in (dict(num_blocks=0), dict(n_kv=0), dict(head_dim=96), dict(page=8)):
        with pytest.raises(ValueError):
            kv4_cache(**{**dict(num_blocks=4, n_kv=2, head_dim=128, page=16, device="cpu"), **kw})
    x = inputs(4, 4, 2, 128, 64, 1, dev="cpu")
    cache = kv4_cache(x["blocks"], n_kv=2, head_dim=128, page=16, device="cpu")
    assert cache.shape == (4, 2, 1, 2176) and not cache.any()
    slots = torch.arange(4)
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    ok = dict(kv_cache=cache, slots=slots, k_out=k, v_out=k)
    for bad in (dict(kv_cache=cache.short()), dict(kv_cache=cache[0]), dict(kv_cache=cache[..., :100]),
                dict(kv_cache=cache.transpose(2, 3)), dict(kv_cache=torch.zeros(4, 2, 2, 2200, dtype=torch.uint8)[..., :2176]),
                dict(slots=slots.int()), dict(slots=slots[None]), dict(k_out=k.float()), dict(v_out=k[..., ::2])):
        with pytest.raises(TypeError):
            kv4_read(**{**ok, **bad})
    for bad in (dict(k_out=k[:3]), dict(v_out=k[:, :1]), dict(k_out=k[..., :64]), dict()):   # the last: on the CPU
        with pytest.raises(ValueError):
            kv4_read(**{**ok, **bad})
    write = dict(q=x["q"], k=x["k"], v=x["v"], positions=x["pos"][0], slot_mapping=x["slots"], kv_cache=cache,
                 cos_sin=x["cs"], q_out=torch.zeros_like(x["q"]))
    for bad in (dict(kv_cache=cache[0]), dict(kv_cache=cache[..., :100]), dict(q=x["q"].float())):
        with pytest.raises(TypeError):
            qk_norm_rope_write(**{**write, **bad})
    for bad in (dict(k=x["q"]), dict(kv_cache=cache[:, :1]), dict()):
        with pytest.raises(ValueError):
            qk_norm_rope_write(**{**write, **bad})
    i = torch.zeros(5, dtype=torch.int32)
    call = dict(q=x["q"], kv_cache=cache, block_table=i[:4, None], seq_lens=i[:4], out=torch.zeros_like(x["q"]), ws=None,
                n_req=4, scale=1.0)
    for f, more in ((window_decode, {}), (window_prefill, dict(query_start_loc=i))):
        for bad in (dict(kv_cache=cache[0]), dict(kv_cache=cache[..., :100]), dict(q=x["q"].float())):
            with pytest.raises(TypeError):
                f(**{**call, **more, **bad})
        for bad in (dict(q=x["q"][..., :64], out=x["q"][..., :64]), dict()):
            with pytest.raises(ValueError):
                f(**{**call, **more, **bad})
    with pytest.raises(TypeError):                               # a prefix is read in bf16
        prefix_decode(group_start=i, prefix_pages=i, n_groups=1, **call)


def test_c_entry_refusals():
    lib = _lib.load()
    attn = "q qs qh c cb ch nb bt bs bc sl".split()
    tail = "win sink out os oh lse ls ws wb".split()
    geo = dict(nb=4, bc=4, win=0, sink=0, wb=0, n=1, r=1, kv=2, G=4, d=128, page=16, ms=0, scale=0.1, stream=0, ws=0)
    for entry, names in ((lib.locks_kv4_decode, attn + tail + "r kv G d page ms scale stream".split()),
                         (lib.locks_kv4_prefill, attn + ["qsl"] + tail + "n r kv G d page ms scale stream".split())):
        ok = {**dict.fromkeys(names, 16), **{k: v for k, v in geo.items() if k in names}}
        for bad in (dict(d=96), dict(page=8), dict(G=17), dict(kv=0), dict(r=-1), dict(nb=0), dict(bc=0), dict(win=-1),
                    dict(sink=-1), dict(scale=0.0), dict(scale=float("nan")), dict(q=0), dict(c=0), dict(sl=0), dict(out=0),
                    dict(c=8), dict(cb=24), dict(ch=-16), dict(qs=4), dict(q=8), dict(os=2), dict(bc=1 << 28),
                    dict(bc=4096, r=1, kv=1)):                   # the last: no workspace
            assert entry(*{**ok, **bad}.values()) == -1, bad
            assert lib.locks_last_error().startswith(b"locks_kv4_")
    names = "c cb ch nb slots k ks kh v vs vh n kv d page stream".split()
    ok = {**dict.fromkeys(names, 16), **{k: v for k, v in geo.items() if k in names}}
    for bad in (dict(d=32), dict(page=128), dict(n=-1), dict(c=0), dict(slots=0), dict(k=0), dict(v=8), dict(ks=4),
                dict(vh=2), dict(cb=8), dict(nb=0)):
        assert lib.locks_kv4_read(*{**ok, **bad}.values()) == -1, bad
    names = ("q qst qsh k kst ksh v vst vsh pos pax na a0 a1 a2 a3 slot c cb ch nb cs mp rot inter qw kw f32 eps qo qost "
             "qosh ko kost kosh n H kv d page stream").split()
    ok = dict.fromkeys(names, 16)
    ok |= dict(na=0, a0=0, a1=0, a2=0, a3=0, nb=4, mp=8, rot=64, inter=0, f32=0, eps=1e-6, n=1, H=4, kv=2, d=128, page=16,
               stream=0)
    for bad in (dict(na=5), dict(na=-1), dict(na=2, a0=2), dict(d=96), dict(page=8), dict(rot=8), dict(c=0), dict(c=8),
                dict(cb=40), dict(q=0), dict(qst=4), dict(H=5000), dict(eps=-1.0), dict(n=-1), dict(slot=0)):
        assert lib.locks_kv4_write(*{**ok, **bad}.values()) == -1, bad
        assert lib.locks_last_error().startswith(b"locks_kv4_write")


# ---- calls at the edges of what is allowed ------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n", [65, 300, 700])
@pytest.mark.parametrize("window, sinks", [(0, 0), (2500, 7)])
def test_decode_more_requests_than_lanes(n, window, sinks):
    """Shares over more requests than a wave has lanes, and than a workgroup has threads; many
    of them without a token."""
    g = torch.Generator()
    g.manual_seed(n)
    lens = [int(x) if i % 7 else 0 for i, x in enumerate(torch.randint(1, 200, (n,), generator=g))]
    lens[3], lens[n // 2], lens[-1] = 2900, 1333, 2100
    c = case(lens, [1] * n, 2, 2, 64, 16, width=190)
    _agree(*_decode(c, window, sinks), _empty_row(c, _exact(_no_rows(c), window, sinks)))


@pytest.mark.gpu
@pytest.mark.parametrize("d, G", [(64, 7), (128, 1), (128, 16), (256, 3)])
def test_decode_short_rows_of_a_wide_table(d, G):
    """A table for far more tokens than there are: few shares, rows in one of them or cut
    anywhere; no tokens at all."""
    for lens in ([1], [33], [900], [17, 0, 1], [0, 0], [500, 1, 700, 64, 16], [2000] * 9):
        c = case(lens, [1] * len(lens), 3, G, d, 16, width=4000, seed=len(lens))
        want = _empty_row(c, _exact(_no_rows(c), 0, 0)) if any(lens) else None
        out, lse = _decode(c)
        if want is None:
            assert not bool(out.any()) and bool((lse == -torch.inf).all())
        else:
            _agree(out, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("d, G", [(64, 8), (64, 9), (64, 16), (128, 8), (256, 16)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (9000, 33)])
def test_decode_full_grids_of_shares(d, G, window, sinks):
    """Without a window every share of the grid has work, at each count of shares."""
    c = case([20011, 3, 9007, 0, 12500], [1] * 5, 8, G, d, 32)
    _agree(*_decode(c, window, sinks), _empty_row(c, _exact(_no_rows(c), window, sinks)))


@pytest.mark.gpu
def test_prefill_many_requests_and_table_ends():
    """More requests than lanes, some without a token; rows past the table's end see what
    the table holds, or nothing where a window lies behind it."""
    lens = [(37 * i) % 90 + 1 for i in range(150)]
    new = [min(n, (11 * i) % 9) for i, n in enumerate(lens)]
    c = case(lens, new, 2, 4, 128, 16)
    _agree(*_prefill(c, 40, 3), _exact(c, 40, 3))
    c = case([900], [900], 2, 4, 64, 16, width=30)                  # 480 tokens of the table
    out, lse = _prefill(c, 100)
    k, v = c["k"][0][:480], c["v"][0][:480]
    head = {**c, "lens": [480], "new": [480], "q": c["q"][:480], "k": [k], "v": [v]}
    _agree(out[:480], lse[:480], _exact(head, 100, 0))
    assert not bool(out[579:].any()) and bool((lse[579:] == -torch.inf).all())


@pytest.mark.gpu
def test_in_place():
    """q_out is q and k_out is k, views of one packed projection; fewer tokens than rows."""
    x = inputs(70, 8, 2, 128, 128, 3)
    axes = RopeAxes.sections((16, 24, 24))
    one, two = (_blank(x["blocks"], 2, 128, 16) for _ in range(2))
    q, k = torch.zeros_like(x["q"]), torch.zeros_like(x["k"])
    kw = dict(q_weight=x["qw"], k_weight=x["kw"], axes=axes, n_tokens=64)
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], one, x["cs"], q, k_out=k, **kw)
    packed = torch.cat([x["q"], x["k"], x["v"]], 1)
    qp, kp, vp = packed.split([8, 2, 2], dim=1)
    qk_norm_rope_write(qp, kp, vp, x["pos"], x["slots"], two, x["cs"], qp, k_out=kp, **kw)
    assert torch.equal(one, two) and torch.equal(q[:64], qp[:64]) and torch.equal(k[:64], kp[:64])
    assert torch.equal(qp[64:], x["q"][64:]) and not bool(q[64:].any())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache of more than 4 GiB, its last pages in use."""
    n_kv, d, page, blocks = 8, 128, 16, 250001
    cache = kv4_cache(blocks, n_kv=n_kv, head_dim=d, page=page, device="cuda")
    assert cache.nbytes > 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    pages = torch.tensor([blocks - 1, 3, blocks - 77, 130000, 249000], device="cuda")
    t = torch.arange(75, device="cuda")
    slots = pages[t // page] * page + t % page
    k, v = (torch.randn(75, n_kv, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    qk_norm_rope_write(k, k, v, t.int(), slots, cache, None, torch.empty_like(k))
    kr, vr = _read(cache, slots)
    assert torch.equal(kr.double(), quantised(k.double())[2]) and torch.equal(vr.double(), quantised(v.double())[2])
    c = dict(q=torch.randn(75, 16, d, generator=g, device="cuda").to(torch.bfloat16), kv=cache, bt=pages[None].int().contiguous(),
             sl=torch.tensor([75], dtype=torch.int32, device="cuda"), qsl=torch.tensor([0, 75], dtype=torch.int32, device="cuda"),
             k=[kr], v=[vr], lens=[75], new=[75], n_kv=n_kv, G=2, d=d, page=page, scale=0.1)
    _agree(*_prefill(c), _exact(c, 0, 0))
    one = {**c, "q": c["q"][:1].contiguous(), "new": [1]}
    _agree(*_decode(one), _exact(one, 0, 0))


@pytest.mark.gpu
def test_replay_in_shares():
    """A captured decode over a wide table follows the lengths: rows whole, cut and empty."""
    n_kv, G, d = 2, 4, 128
    c = case([2900, 1500, 40, 700], [1] * 4, n_kv, G, d, 16, width=200)
    out, lse = _outs(c)
    ws = _ws(c)
    sl = c["sl"].clone()
    call = lambda: window_decode(c["q"], c["kv"], c["bt"], sl, out, ws, n_req=4, scale=c["scale"], lse=lse)  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ([2900, 1500, 40, 700], [1, 2, 3, 4], [0, 1500, 0, 0], [2900, 0, 40, 699], [2048, 1499, 1, 16]):
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        part = {**c, "lens": lens, "k": [k[:n] for k, n in zip(c["k"], lens)], "v": [v[:n] for v, n in zip(c["v"], lens)]}
        _agree(out, lse, _empty_row(part, _exact(_no_rows(part), 0, 0)))
        torch.cuda.synchronize()
