"""Window, prefill and shared-prefix attention against softmax attention in 64
bits, and the calls that are refused.

Tolerance, with A = sum_j p_j |v_j| / l of the exact weights.  The output is one
rounding to bf16 (2^-8 of it); every weight is rounded once to bf16 (2^-8 of it:
2^-8 A); a score is an fp32 sum of exact products, off by at most d 2^-24 of
S = scale sum |q| |k| (with the products of the softmax argument, (d + 8) 2^-24 S),
which moves a weight by as much of itself, and the sum l too: 2 delta A.  The
exponentials and the fp32 sums over at most 2^14 keys per lane are covered by 2^-10
of A.  lse: delta, and 2^-10 for the sum, 2^-22 of it for its rounding."""
import pytest
import torch

from locks import _lib
from locks.attention import attn_workspace, prefix_decode, window_decode, window_prefill


def _cache(g, blocks, page, n_kv, d, layout):
    shape = (blocks, 2, page, n_kv, d) if layout == "nb2" else (2, blocks, page, n_kv, d)
    return torch.full(shape, float("nan"), dtype=torch.bfloat16, device=g.device)


def _case(lens, new, n_kv, G, d, page, *, seed=0, layout="nb2", shared=(), width=None, dev="cuda"):
    """Caches that are NaN wherever no token of a request lies; block tables with
    ids out of range past each request's pages.  ``shared``: (first request, last,
    pages) whose leading pages are the first one's."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    width = width or max(max(pages), 1) + 1
    blocks = sum(pages) + 5
    order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    bt = torch.randint(-5, 1 << 20, (len(lens), width), generator=g, device=dev, dtype=torch.int32)
    at = 0
    for r, n in enumerate(pages):
        bt[r, :n] = order[at:at + n]
        at += n
    for a, b, p in shared:
        for r in range(a + 1, b):
            n = min(p, pages[r])
            bt[r, :n] = bt[a, :n]
    kv = _cache(g, blocks, page, n_kv, d, layout)
    K, V = (kv[:, 0], kv[:, 1]) if layout == "nb2" else (kv[0], kv[1])
    k64, v64 = [], []
    for r, n in enumerate(lens):
        t = torch.arange(n, device=dev)
        b, o = bt[r].long()[t // page] if n else t, t % page
        fresh = K[b, o, 0, 0].isnan() if n else t.bool()
        k = (torch.randn(n, n_kv, d, generator=g, device=dev) * 1.5).to(torch.bfloat16)
        v = torch.randn(n, n_kv, d, generator=g, device=dev).to(torch.bfloat16)
        if n:
            K[b[fresh], o[fresh]], V[b[fresh], o[fresh]] = k[fresh], v[fresh]
            k, v = K[b, o], V[b, o]
        k64.append(k)
        v64.append(v)
    T, H = sum(new), n_kv * G
    q = torch.randn(T, H, d, generator=g, device=dev).to(torch.bfloat16)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    return dict(q=q, kv=kv, bt=bt, sl=i(lens), qsl=i(starts), k=k64, v=v64, lens=lens, new=new, n_kv=n_kv, G=G, d=d,
                page=page, scale=1.0 / d ** 0.5, K=K, V=V)


def _exact(c, window, sinks):
    """(out, lse, tolerance of out, tolerance of lse) row by row of q."""
    d, G = c["d"], c["G"]
    o, z, to, tz = [], [], [], []
    at = 0
    for r, (n, m) in enumerate(zip(c["lens"], c["new"])):
        pos = torch.arange(n - m, n, device=c["q"].device)[:, None]
        key = torch.arange(n, device=c["q"].device)[None]
        seen = key <= pos
        if window:
            seen &= (key > pos - window) | (key < sinks)
        q = c["q"][at:at + m].double().unflatten(1, (c["n_kv"], G)).permute(1, 2, 0, 3)     # (kv, G, m, d)
        k = c["k"][r].double().permute(1, 0, 2)[:, None]                                   # (kv, 1, n, d)
        v = c["v"][r].double().permute(1, 0, 2)[:, None]
        s = torch.where(seen, c["scale"] * (q @ k.mT.contiguous()), -torch.inf)
        big = torch.where(seen, c["scale"] * (q.abs() @ k.abs().mT.contiguous()), 0).amax(-1) if n else s.sum(-1)
        lse = torch.logsumexp(s, -1) if n else s.sum(-1) - torch.inf
        empty = (~seen.any(-1)) if n else torch.ones(m, dtype=torch.bool, device=q.device)
        p = torch.where(empty[:, None], 0, torch.exp(s - lse[..., None]))
        p = torch.where(seen, p, 0)
        v0 = torch.where(v.isfinite(), v, 0)
        out, A = p @ v0, p @ v0.abs()
        if not bool(v.isfinite().all()):                     # a value that is not finite reaches the rows that see it
            for j in (~v.isfinite()).flatten(0, 1).any(-1).any(0).nonzero()[:, 0].tolist():
                x = torch.where(v[:, :, j].isfinite(), 0, v[:, :, j])[:, :, None]           # (kv, 1, 1, d)
                out = torch.where((seen[:, j])[:, None], out + x, out)
        delta = (d + 8) * 2.0 ** -24 * big
        o.append(out.permute(2, 0, 1, 3).flatten(1, 2))
        z.append(torch.where(empty, -torch.inf, lse).permute(2, 0, 1).flatten(1, 2))
        to.append((2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -10 + 2 * delta[..., None]) * A).permute(2, 0, 1, 3).flatten(1, 2))
        tz.append((delta + 2.0 ** -10 + 2.0 ** -22 * lse.abs()).permute(2, 0, 1).flatten(1, 2))
        at += m
    return [torch.cat(x) for x in (o, z, to, tz)]


def _agree(got, lse, want, rows=None):
    o, z, to, tz = want if rows is None else [x[:rows] for x in want]
    fin = o.isfinite()
    assert torch.equal(got.isnan(), o.isnan())
    assert torch.equal(got.double()[~fin & ~o.isnan()], o[~fin & ~o.isnan()])
    off = torch.where(fin, (got.double() - o).abs() - to, 0.0)
    assert bool((off <= 0).all()), f"out {off.max().item()} over, at {(off > 0).nonzero()[:4].tolist()}"
    inf = z == -torch.inf
    assert torch.equal(lse == -torch.inf, inf)
    off = torch.where(inf, 0.0, (lse.double() - z).abs() - tz)
    assert bool((off <= 0).all()), f"lse {off.max().item()} over"


def _ws(c, tokens=None):
    ws = attn_workspace("cuda", max_tokens=tokens or max(c["q"].shape[0], 1), n_kv=c["n_kv"], G=c["G"], head_dim=c["d"])
    return ws.fill_(255)                                     # NaN, as fp32: nothing may rely on its content


def _outs(c, extra=0):
    T, H = c["q"].shape[:2]
    return (torch.full((T + extra, H, c["d"]), 7.0, dtype=torch.bfloat16, device="cuda"),
            torch.full((T + extra, H), 7.0, device="cuda"))


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


GEOMETRY = [(128, 16, 8, 4), (128, 32, 2, 16), (128, 64, 1, 1), (64, 16, 4, 7), (64, 32, 1, 16), (64, 64, 3, 5),
            (256, 16, 2, 8), (256, 32, 1, 3), (256, 64, 4, 1)]
LENS = [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 129, 500, 1025]


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (1, 1), (16, 4), (17, 16), (64, 17), (100, 300), (512, 5),
                                           (5000, 64)])
@pytest.mark.parametrize("d, page, n_kv, G", GEOMETRY)
def test_decode(d, page, n_kv, G, window, sinks):
    lens = LENS + [0, 3000]
    c = _case(lens, [1] * len(lens), n_kv, G, d, page, seed=window + sinks)
    _agree(*_decode(c, window, sinks), _empty_row(c, _exact(_no_rows(c), window, sinks)))


def _no_rows(c):
    """The case with the requests of length 0 out of the oracle's way."""
    return {**c, "new": [min(1, n) for n in c["lens"]], "q": c["q"][torch.tensor(c["lens"]).bool().to(c["q"].device)]}


def _empty_row(c, want):
    """Rows of requests of length 0 put back: zero, -inf."""
    live = torch.tensor(c["lens"]).bool().to(c["q"].device)
    out = []
    for x, fill in zip(want, (0.0, -torch.inf, 0.0, 0.0)):
        y = torch.full((len(c["lens"]), *x.shape[1:]), fill, dtype=torch.float64, device=x.device)
        y[live] = x
        out.append(y)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["nb2", "2nb"])
def test_decode_long_and_layouts(layout):
    """A long row among short ones, an exact bound of the lengths, strided q and out."""
    c = _case([70001, 5, 33000], [1, 1, 1], 2, 4, 128, 16, layout=layout)
    for window, sinks in ((0, 0), (4096, 4), (30000, 100)):
        want = _exact(c, window, sinks)
        _agree(*_decode(c, window, sinks), want)
        _agree(*_decode(c, window, sinks, max_seq_len=70001), want)
    wide = torch.zeros(3, 3, 8, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = c["q"]
    out = torch.zeros(3, 8, 2, 128, dtype=torch.bfloat16, device="cuda")
    window_decode(wide[:, 1], c["kv"], c["bt"], c["sl"], out[:, :, 1], _ws(c), n_req=3, scale=c["scale"])
    assert torch.equal(out[:, :, 1], _decode(c)[0]) and not bool(out[:, :, 0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (33, 4), (64, 64), (200, 17), (300, 1000)])
@pytest.mark.parametrize("d, page, n_kv, G", GEOMETRY)
def test_prefill(d, page, n_kv, G, window, sinks):
    """Whole prompts and chunks, from one token to several tiles, and requests
    without a new token."""
    lens = [1, 16, 17, 40, 128, 129, 700, 333, 90, 513]
    new = [1, 16, 5, 40, 127, 1, 650, 0, 65, 64]
    c = _case(lens, new, n_kv, G, d, page, seed=window)
    _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("lens, new, window, sinks", [
    ([6000], [1], 0, 0), ([9001], [7], 0, 0), ([20000, 3], [2, 1], 0, 0),           # few rows, long keys: split
    ([9001], [7], 4000, 100), ([5000], [300], 1000, 4), ([4096], [4096], 0, 0), ([4099], [4099], 555, 70),
])
@pytest.mark.parametrize("d, n_kv, G", [(128, 2, 4), (64, 1, 16), (256, 1, 2)])
def test_prefill_long(d, n_kv, G, lens, new, window, sinks):
    c = _case(lens, new, n_kv, G, d, 16)
    want = _exact(c, window, sinks)
    _agree(*_prefill(c, window, sinks), want)
    _agree(*_prefill(c, window, sinks, max_seq_len=max(lens)), want)


@pytest.mark.gpu
def test_prefill_equals_decode_of_each_token():
    """A prompt's rows against single-token calls at each length."""
    c = _case([150], [150], 2, 4, 128, 16)
    out, lse = _prefill(c, 40, 3)
    for n in (1, 2, 17, 64, 65, 150):
        c1 = {**c, "q": c["q"][n - 1:n], "sl": c["sl"] * 0 + n, "lens": [n]}
        o, z = _decode(c1, 40, 3)
        assert (o.float() - out[n - 1].float()).abs().max() < 2.0 ** -6 and (z - lse[n - 1]).abs().max() < 2.0 ** -9


@pytest.mark.gpu
def test_masked_places_do_not_matter():
    """NaN and infinities in V and K of tokens that a row does not see (later ones,
    ones behind the window), and in V of ones that it does."""
    for d in (64, 128, 256):
        c = _case([200, 90], [200, 50], 2, 4, d, 16, seed=d)
        for r, t, x in ((0, 150, float("nan")), (0, 160, float("inf")), (0, 30, -float("inf")), (1, 70, float("inf")),
                        (0, 199, float("nan"))):
            b, o = int(c["bt"][r, t // 16]), t % 16
            c["V"][b, o, 1, 3:d:7] = x
            c["v"][r][t, 1, 3:d:7] = x
        for window, sinks in ((0, 0), (48, 10), (20, 35)):
            got = _prefill(c, window, sinks)
            _agree(*got, _exact(c, window, sinks))
            assert bool(got[0].isnan().any()) and bool(got[0].isinf().any())
        b, o = int(c["bt"][0, 6]), 5                         # a key in the middle: rows before and past the window
        c["K"][b, o] = float("nan")
        out, lse = _prefill(c, 48, 10)
        sees = torch.zeros(250, dtype=torch.bool, device="cuda")
        sees[101:101 + 48] = True
        assert bool(lse[sees].isnan().all()) and not bool(lse[~sees].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("d, page, n_kv, G", GEOMETRY)
def test_prefix(d, page, n_kv, G):
    """Two groups, one of them of a single request, requests in no group before and
    after, members shorter than the prefix, of its length, padding."""
    P = 320 // page
    lens = [40, 320 + 77, 320, 321, 300, 1, 0, 320 + 1500, 5 * page + 3, 9, 700]
    shared = [(1, 8, P), (8, 9, 5)]
    c = _case(lens, [1] * len(lens), n_kv, G, d, page, shared=shared)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    want = _empty_row(c, _exact(_no_rows(c), 0, 0))
    for kw in ({}, dict(max_prefix_pages=P, max_seq_len=2000)):
        out, lse = _outs(c)
        prefix_decode(c["q"], c["kv"], c["bt"], c["sl"], i(1, 8, 9), i(P, 5), out, _ws(c), n_req=len(lens), n_groups=2,
                      scale=c["scale"], lse=lse, **kw)
        _agree(out, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n, prefix, d, n_kv, G", [(1, 16, 128, 8, 4), (50, 2048, 128, 2, 4), (140, 1024, 64, 1, 16),
                                                   (3, 30000, 128, 2, 16), (33, 512, 256, 1, 5), (70, 4096, 128, 1, 1)])
def test_prefix_sizes(n, prefix, d, n_kv, G):
    lens = [prefix + 1 + (37 * r) % 300 for r in range(n)]
    c = _case(lens, [1] * n, n_kv, G, d, 16, shared=[(0, n, prefix // 16)])
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = _outs(c)
    prefix_decode(c["q"], c["kv"], c["bt"], c["sl"], i(0, n), i(prefix // 16), out, _ws(c), n_req=n, n_groups=1,
                  scale=c["scale"], lse=lse)
    _agree(out, lse, _exact(c, 0, 0))


@pytest.mark.gpu
def test_many_groups():
    """More groups than lanes, with and without pages, of changing sizes."""
    sizes = [(g * 7) % 4 for g in range(130)]
    pages = [(g * 5) % 9 for g in range(130)]
    lens, shared, starts = [], [], [0]
    for s, p in zip(sizes, pages):
        if s:
            shared.append((len(lens), len(lens) + s, p))
        lens += [p * 16 + 1 + (k * 13) % 40 for k in range(s)]
        starts.append(len(lens))
    c = _case(lens, [1] * len(lens), 2, 2, 64, 16, shared=shared)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = _outs(c)
    prefix_decode(c["q"], c["kv"], c["bt"], c["sl"], i(starts), i(pages), out, _ws(c), n_req=len(lens), n_groups=130,
                  scale=c["scale"], lse=lse)
    _agree(out, lse, _exact(c, 0, 0))


@pytest.mark.gpu
def test_replayed_with_other_lengths():
    """The three calls captured on one workspace and replayed with other lengths,
    starts and prefixes, with eager calls between the replays."""
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    c = _case([400, 300, 500], [1, 1, 1], 2, 4, 128, 16, shared=[(0, 3, 10)])
    p = _case([400, 300, 500], [60, 30, 20], 2, 4, 128, 16)
    ws = _ws(p)
    sl, psl, qsl, gs, gp = i(1, 1, 1), i(60, 30, 20), p["qsl"].clone(), i(0, 3), i(0)
    (o1, z1), (o2, z2), (o3, z3) = _outs(c), _outs(p), _outs(c)

    def calls():
        window_decode(c["q"], c["kv"], c["bt"], sl, o1, ws, n_req=3, window=100, sinks=8, scale=c["scale"], lse=z1)
        window_prefill(p["q"], p["kv"], p["bt"], psl, qsl, o2, ws, n_req=3, scale=c["scale"], lse=z2)
        prefix_decode(c["q"], c["kv"], c["bt"], sl, gs, gp, o3, ws, n_req=3, n_groups=1, scale=c["scale"], lse=z3)

    calls()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls()
    for lens, new, pre in (([400, 300, 500], [60, 30, 20], 10), ([17, 222, 160], [10, 70, 30], 1),
                           ([160, 160, 170], [1, 100, 9], 10), ([1, 300, 2], [1, 1, 1], 0)):
        sl.copy_(i(*lens)), psl.copy_(i(*lens)), gp.copy_(i(pre))
        qsl.copy_(i(0, new[0], new[0] + new[1], sum(new)))
        o2.fill_(7)
        g.replay()
        cut = lambda x, n: [t[:k] for t, k in zip(x, n)]  # noqa: E731
        cc = {**c, "lens": lens, "k": cut(c["k"], lens), "v": cut(c["v"], lens)}
        pp = {**p, "lens": lens, "new": new, "k": cut(p["k"], lens), "v": cut(p["v"], lens)}
        _agree(o1, z1, _exact(cc, 100, 8))
        _agree(o3, z3, _exact(cc, 0, 0))
        _agree(o2[:sum(new)], z2[:sum(new)], _exact(pp, 0, 0))
        assert bool((o2[sum(new):] == 7).all())
        _decode(c)                                           # eager work between


@pytest.mark.gpu
def test_other_stream_and_short_batches():
    """Work on a stream of its own; n_req and n_tokens smaller than the buffers;
    calls of nothing."""
    c = _case([100, 50, 7], [1, 1, 1], 2, 4, 128, 16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out, lse = _outs(c)
    ws = _ws(c)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        window_decode(c["q"], c["kv"], c["bt"], c["sl"], out, ws, n_req=2, scale=c["scale"], lse=lse)
    s.synchronize()
    _agree(out[:2], lse[:2], _exact(c, 0, 0), rows=2)
    assert bool((out[2] == 7).all()) and bool((lse[2] == 7).all())
    window_decode(c["q"], c["kv"], c["bt"], c["sl"], out, ws, n_req=0, scale=1.0)
    window_prefill(c["q"][:0], c["kv"], c["bt"], c["sl"], c["qsl"], out, ws, n_req=3, scale=1.0)
    assert bool((out[2] == 7).all())


@pytest.mark.gpu
def test_many_requests():
    """More requests than lanes, from none to a few tiles of new tokens each."""
    new = [(r * 37) % 90 if r % 5 else 0 for r in range(150)]
    lens = [n + (r * 53) % 200 for r, n in enumerate(new)]
    c = _case(lens, new, 2, 4, 64, 16)
    for window, sinks in ((0, 0), (60, 9)):
        _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("lens, new", [([90, 70], [40, 30]), ([6000, 5000], [3, 2])])
def test_fewer_rows_than_the_starts_say(lens, new):
    """n_tokens inside the second request: its first rows keep their positions, the
    others stay as they were."""
    c = _case(lens, new, 2, 4, 128, 16)
    n = new[0] + 1
    out, lse = _outs(c)
    window_prefill(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out, _ws(c), n_req=2, n_tokens=n, window=33, sinks=2,
                   scale=c["scale"], lse=lse)
    _agree(out[:n], lse[:n], _exact(c, 33, 2), rows=n)
    assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all())


@pytest.mark.gpu
def test_large_scores_and_wide_values():
    """Scores of hundreds (one key takes all) and V past fp16's range."""
    c = _case([300], [1], 1, 4, 128, 16)
    c["q"] *= 60
    c["V"][int(c["bt"][0, 3])] *= 1e30
    c["v"][0] = torch.where((torch.arange(300, device="cuda") // 16 == 3)[:, None, None], c["v"][0] * 1e30, c["v"][0])
    _agree(*_decode(c), _exact(c, 0, 0))
    _agree(*_prefill(c), _exact(c, 0, 0))


@pytest.mark.gpu
def test_workspace_too_small():
    c = _case([9000], [1], 2, 4, 128, 16)
    out, _ = _outs(c)
    with pytest.raises(RuntimeError, match="workspace"):
        window_decode(c["q"], c["kv"], c["bt"], c["sl"], out, _ws(c)[:1024], n_req=1, scale=1.0)
    with pytest.raises(RuntimeError, match="workspace"):
        window_prefill(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out, None, n_req=1, scale=1.0)


def test_refusals():
    c = _case([20, 5], [1, 1], 2, 4, 128, 16, dev="cpu")
    out = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    ws = attn_workspace("cpu", max_tokens=2, n_kv=2, G=4, head_dim=128)
    ok = dict(q=c["q"], kv_cache=c["kv"], block_table=c["bt"], seq_lens=c["sl"], out=out, ws=ws, n_req=2, scale=1.0)
    typed = (dict(q=c["q"].float()), dict(out=out.float()), dict(out=out[..., ::2]), dict(kv_cache=c["kv"].float()),
             dict(kv_cache=c["kv"][0]), dict(block_table=c["bt"].long()), dict(block_table=c["bt"].T),
             dict(seq_lens=c["sl"].long()), dict(lse=torch.zeros(2, 8).double()))
    valued = (dict(n_req=3), dict(out=out[:1]), dict(out=out[:, :4]), dict(q=c["q"][:, :7], out=out[:, :7]),
              dict(kv_cache=c["kv"][:, :1]), dict(lse=torch.zeros(1, 8)), dict(lse=torch.zeros(2, 4)), dict())
    more = {window_decode: {}, window_prefill: dict(query_start_loc=c["qsl"]),
            prefix_decode: dict(group_start=c["sl"], prefix_pages=c["sl"], n_groups=1)}
    for fn, extra in more.items():
        for bad in typed:
            with pytest.raises(TypeError):
                fn(**{**ok, **extra, **bad})
        for bad in valued:                                   # the last: on the CPU
            with pytest.raises(ValueError):
                fn(**{**ok, **extra, **bad})
    for bad in (dict(max_tokens=0), dict(max_reqs=-1), dict(n_kv=0), dict(G=17), dict(head_dim=96)):
        with pytest.raises(ValueError):
            attn_workspace("cpu", **{**dict(max_tokens=2, n_kv=2, G=4, head_dim=128), **bad})


COMMON = "q qst qsh k kb kt kh v vb vt vh nb bt bst cols sl".split()
OUT = "out ost osh lse lst ws wsb".split()


def test_c_entry_refusals():
    """The C entries turn bad arguments into errors before they touch a GPU."""
    lib = _lib.load()
    ok = dict(nb=4, cols=4096, window=0, sinks=0, n=2, T=4, nkv=2, G=4, d=128, page=16, maxs=0, maxp=0, ng=1, scale=1.0,
              wsb=1 << 30, stream=0)
    calls = [
        (lib.locks_window_decode, COMMON + ["window", "sinks"] + OUT + "n nkv G d page maxs scale stream".split()),
        (lib.locks_window_prefill, COMMON + ["qsl", "window", "sinks"] + OUT + "T n nkv G d page maxs scale stream".split()),
        (lib.locks_prefix_decode, COMMON + ["gs", "gp", "ng"] + OUT + "n nkv G d page maxp maxs scale stream".split()),
    ]
    for fn, names in calls:
        base = {n: ok.get(n, 16) for n in names}
        bads = [dict(d=96), dict(page=8), dict(G=0), dict(G=17), dict(nkv=0), dict(n=-1), dict(n=70000), dict(nb=0),
                dict(cols=0), dict(cols=1 << 28), dict(maxs=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                dict(scale=float("nan")), dict(q=0), dict(sl=0), dict(out=0), dict(qst=4), dict(vh=12), dict(osh=2),
                dict(q=8), dict(k=24), dict(out=4), dict(ws=0), dict(ws=8), dict(wsb=100)]
        if "window" in base:
            bads += [dict(window=-1), dict(sinks=-1)]
        if "gs" in base:
            bads += [dict(gs=0), dict(gp=0), dict(ng=0), dict(ng=70000), dict(maxp=-1)]
        if "qsl" in base:
            bads += [dict(qsl=0), dict(T=-1)]
        for bad in bads:
            assert fn(*{**base, **bad}.values()) == -1, (fn, bad)
            assert lib.locks_last_error()


def test_workspace_covers_every_call():
    """The bytes grow with the tokens, so a workspace of more covers fewer."""
    lib = _lib.load()
    for n_kv, G, d in ((8, 4, 128), (1, 16, 64), (2, 3, 256)):
        b = [lib.locks_attn_workspace_bytes(n, n, n_kv, G, d) for n in (1, 2, 7, 64, 65, 300, 5000)]
        assert b == sorted(b) and b[0] > 0
    # about 4096 workgroups' partials at most, past that one per row
    assert lib.locks_attn_workspace_bytes(256, 8192, 8, 4, 128) < 1 << 28
    assert lib.locks_attn_workspace_bytes(8192, 8192, 8, 4, 128) < 1 << 29
