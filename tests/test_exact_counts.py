"""Which keys an attention call sees, to the key: with q = 0 every visible key has
weight one, so

* lse = ln(visible keys).  The score is an exact 0, each weight an exact 1, the
  sums whole numbers below 2^24 and so exact; what is left are logf (at most 2 ulp)
  and its addition to 0.  4 ulp are allowed: below ln 2^17 < 16 that is 4 x 2^-20 =
  3.9e-6, and one key more or less of 90000 moves ln by 1.1e-5.
* out = (sum of the visible V) / (visible keys).  V is zero but for one column per
  chosen key (a power of two, so that the quotient is near 1): seen once it gives
  that quotient to one rounding to bf16 (2^-8 of it; the fp32 division and product
  before it 2^-22), seen twice the double, unseen an exact 0."""
import math

import pytest
import torch

from locks.attention import prefix_decode, window_decode, window_prefill
from tests.test_window import _case, _outs, _ws


def _seen(n, window, sinks):
    """Counts of keys that the query at position n - 1 sees: [0, s) and [lo, n)."""
    lo = max(n - window, 0) if window else 0
    return min(sinks, lo), lo


def _chosen(n, lo, s, d, g):
    """d keys: the edges of what is seen, ends of steps and tiles, any others."""
    edge = {x + e for x in (0, s, lo, n) for e in (-17, -16, -1, 0, 1, 15, 16, 63, 64)}
    keys = [x for x in sorted(edge) if 0 <= x < n][:d]
    more = torch.randint(0, n, (d - len(keys),), generator=g, device="cuda").tolist()
    return keys + more                                       # a key may come twice: it has two columns


def _mark(c, r, keys, unit):
    """V of request r: zero but for column i of key keys[i]."""
    at = torch.tensor(keys, device="cuda")
    b, o = c["bt"][r].long()[at // c["page"]], at % c["page"]
    for i, (bi, oi) in enumerate(zip(b.tolist(), o.tolist())):
        c["V"][bi, oi, :, i] = unit


def _cleared(c):
    c["V"].copy_(torch.where(c["V"].isnan(), c["V"], 0.0))   # places of no token stay NaN
    c["q"].zero_()


def _check(out, lse, count, keys, seen, unit):
    """Rows of one query (H, d) and (H,)."""
    z = math.log(count)
    assert (lse.double() - z).abs().max() <= 4 * 2.0 ** -20, f"lse says {lse.double().exp().tolist()} keys, not {count}"
    want = torch.tensor([unit / count if seen(k) else 0.0 for k in keys], dtype=torch.float64, device="cuda")
    off = (out.double() - want).abs() - (2.0 ** -8 + 2.0 ** -20) * want
    bad = (off > 0).any(0).nonzero()[:, 0].tolist()
    assert not bad, f"keys {[keys[i] for i in bad][:8]}: {out[:, bad[:8]].double().mul(count / unit).tolist()[0]} times"


WINDOWS = [(0, 0), (1, 0), (1, 1), (2000, 0), (2048, 5), (4095, 17), (30000, 100), (65536, 64), (88000, 1999)]


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", WINDOWS)
@pytest.mark.parametrize("d, page, n_kv, G", [(128, 16, 2, 4), (64, 64, 1, 16), (256, 32, 1, 2)])
def test_decode(d, page, n_kv, G, window, sinks):
    lens = [70001, 33000, 90000, 2049]
    c = _case(lens, [1] * 4, n_kv, G, d, page)
    _cleared(c)
    g = torch.Generator(device="cuda")
    g.manual_seed(window)
    marks = []
    for r, n in enumerate(lens):
        s, lo = _seen(n, window, sinks)
        unit = 2.0 ** round(math.log2(n - lo + s))
        keys = _chosen(n, lo, s, d, g)
        _mark(c, r, keys, unit)
        marks.append((n - lo + s, keys, lambda k, s=s, lo=lo: k >= lo or k < s, unit))
    for kw in ({}, dict(max_seq_len=90000)):
        for rows in (range(4), range(1)):                    # one row alone has more splits
            out, lse = _outs(c)
            window_decode(c["q"], c["kv"], c["bt"], c["sl"], out, _ws(c), n_req=len(rows), scale=c["scale"],
                          window=window, sinks=sinks, lse=lse, **kw)
            for r in rows:
                _check(out[r], lse[r], *marks[r])


@pytest.mark.gpu
@pytest.mark.parametrize("lens, new", [([20000], [2]), ([9001, 30000], [3, 1]), ([5000], [300])])
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 3), (1500, 4), (4097, 70), (8192, 0)])
@pytest.mark.parametrize("d, page, n_kv, G", [(128, 16, 2, 4), (64, 64, 1, 16), (256, 32, 1, 2)])
def test_prefill(d, page, n_kv, G, lens, new, window, sinks):
    c = _case(lens, new, n_kv, G, d, page)
    _cleared(c)
    g = torch.Generator(device="cuda")
    g.manual_seed(window)
    marks = []
    for r, (n, m) in enumerate(zip(lens, new)):
        s, lo = _seen(n, window, sinks)                      # the edges of the last row; the others' lie beside them
        unit = 2.0 ** round(math.log2(n - lo + s))
        keys = _chosen(n, lo, s, d, g)
        _mark(c, r, keys, unit)
        marks += [(p + 1, keys, unit) for p in range(n - m, n)]
    out, lse = _outs(c)
    window_prefill(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out, _ws(c), n_req=len(lens), scale=c["scale"],
                   window=window, sinks=sinks, lse=lse)
    for row, (n, keys, unit) in enumerate(marks):
        if len(marks) > 50 and row % 37 and row < len(marks) - 2:
            continue
        s, lo = _seen(n, window, sinks)
        _check(out[row], lse[row], n - lo + s, keys, lambda k: k < n and (k >= lo or k < s), unit)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, pages", [([30000 + 77], 1875), ([30000 + 16, 30001, 31000], 1875), ([17, 64, 65], 1),
                                         ([4096 + r for r in range(70)], 256)])
@pytest.mark.parametrize("d, n_kv, G", [(128, 2, 4), (64, 1, 16), (256, 1, 2)])
def test_prefix(d, n_kv, G, lens, pages):
    page, pre = 16, pages * 16
    c = _case(lens, [1] * len(lens), n_kv, G, d, page, shared=[(0, len(lens), pages)])
    _cleared(c)
    g = torch.Generator(device="cuda")
    g.manual_seed(pages)
    unit = 2.0 ** round(math.log2(pre + 1))
    keys = _chosen(pre, 0, 0, d // 2, g)
    _mark(c, 0, keys, unit)                                  # the prefix, once for all
    marks = []
    for r, n in enumerate(lens):
        tail = [min(pre + x, n - 1) for x in (0, 1, 14, 15, 16, 17, 62, 63, 64, 65, 900)] if n > pre else []
        tail = sorted(set(tail))[:d - d // 2]
        at = torch.tensor(tail, device="cuda", dtype=torch.long)
        for i, (b, o) in enumerate(zip(c["bt"][r].long()[at // page].tolist(), (at % page).tolist())):
            c["V"][b, o, :, d // 2 + i] = unit
        rest = d - d // 2 - len(tail)
        marks.append((n, keys + tail + [-1] * rest, unit))
    out, lse = _outs(c)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    prefix_decode(c["q"], c["kv"], c["bt"], c["sl"], i(0, len(lens)), i(pages), out, _ws(c), n_req=len(lens), n_groups=1,
                  scale=c["scale"], lse=lse)
    for r, (n, ks, u) in enumerate(marks):
        _check(out[r], lse[r], n, ks, lambda k: 0 <= k < n, u)
