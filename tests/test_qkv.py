"""Norm, rotation and cache write (qk_norm_rope_write) against the formulas in 64
bits, and the calls that are refused.

Tolerance.  The result is one rounding to bf16 of an fp32 value: half a step is
2^-8 of it.  The fp32 value itself: the sum of d <= 256 squares is off by at most
256 * 2^-24 = 2^-16 of it, its inverse root by half of that, and the eight or so
products and sums after it by 2^-24 each of the pair's magnitude |a cos| + |b sin|;
2^-16 of that magnitude covers all."""
import pytest
import torch

from locks import _lib
from locks.attention import qk_norm_rope_write


def _inputs(T, H, n_kv, d, rot, page, *, layout="nb2", far=0, w=torch.bfloat16, seed=0, dev="cuda"):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    blocks = -(-T // page) + 3
    packed = (r(T, (H + 2 * n_kv) * d) * 3).to(torch.bfloat16)
    q, k, v = (x.view(T, -1, d) for x in packed.split([H * d, n_kv * d, n_kv * d], dim=1))
    shape = (blocks, 2, page, n_kv, d) if layout == "nb2" else (2, blocks, page, n_kv, d)
    cache = r(*shape).to(torch.bfloat16)
    slots = torch.randperm(blocks * page, generator=g, device=dev)[:T]
    pos = far + torch.randperm(max(T, 1), generator=g, device=dev)[:T].to(torch.int32)
    ang = torch.arange(far + T + 1, dtype=torch.float64, device=dev)[:, None] * (
        10000.0 ** (-torch.arange(0, max(rot, 1), 2, dtype=torch.float64, device=dev) / max(rot, 1)))
    cs = torch.cat([ang.cos(), ang.sin()], 1).float() if rot else None
    weights = [(1 + 0.3 * r(d)).to(w) for _ in range(2)] if w is not None else [None, None]
    return dict(q=q, k=k, v=v, cache=cache, slots=slots, pos=pos, cs=cs, qw=weights[0], kw=weights[1], page=page)


def _formula(x, weight, pos, cs, eps, interleaved):
    """(value, magnitude of its pair) in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    y, mag = x.clone(), x.abs()
    if cs is not None:
        rot = cs.shape[1]
        c, s = cs.double()[pos.long()].split(rot // 2, dim=1)
        i = torch.arange(rot // 2, device=x.device)
        i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        a, b, c, s = x[..., i], x[..., j], c[:, None], s[:, None]
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return y, mag


def _halves(cache, layout):
    return (cache[:, 0], cache[:, 1]) if layout == "nb2" else (cache[0], cache[1])


def _close(got, want, what):
    y, mag = want
    off = (got.double() - y).abs()
    tol = 2.0 ** -8 * y.abs() + 2.0 ** -16 * mag * 1.01
    assert bool((off <= tol).all()), f"{what}: {(off - tol).max().item()} over"


def _run_and_check(x, *, eps=1e-6, interleaved=False, layout="nb2", q_out=None, k_out=None, n=None):
    T = x["q"].shape[0] if n is None else n
    before = x["cache"].clone()
    want_q = _formula(x["q"], x["qw"], x["pos"], x["cs"], eps, interleaved)
    want_k = _formula(x["k"], x["kw"], x["pos"], x["cs"], eps, interleaved)
    v = x["v"].clone()
    q_out = torch.full(x["q"].shape, 7.0, dtype=torch.bfloat16, device="cuda") if q_out is None else q_out
    rest = q_out[T:].clone()
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], x["cache"], x["cs"], q_out, n_tokens=n,
                       q_weight=x["qw"], k_weight=x["kw"], eps=eps, interleaved=interleaved, k_out=k_out)
    _close(q_out[:T], [y[:T] for y in want_q], "q")
    assert torch.equal(q_out[T:], rest)
    K, V = _halves(x["cache"], layout)
    at = (x["slots"][:T] // x["page"], x["slots"][:T] % x["page"])
    _close(K[at], [y[:T] for y in want_k], "k")
    assert torch.equal(V[at], v[:T])
    if k_out is not None:
        assert torch.equal(k_out[:T], K[at])
    bk, bv = _halves(before, layout)                         # every other row as it was
    bk[at], bv[at] = K[at], V[at]
    assert torch.equal(before, x["cache"])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d, rot", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 48), (256, 256), (256, 64), (128, 0)])
@pytest.mark.parametrize("T, H, n_kv", [(1, 32, 8), (7, 5, 1), (130, 14, 2)])
def test_formula(T, H, n_kv, d, rot, interleaved):
    _run_and_check(_inputs(T, H, n_kv, d, rot, 16, seed=T + d + rot), interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("layout", ["nb2", "2nb"])
def test_cache_layouts(page, layout):
    x = _inputs(75, 8, 2, 128, 128, page, layout=layout)
    _run_and_check(x, layout=layout, k_out=torch.zeros(75, 2, 128, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("w", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("only", ["", "q", "k"])
def test_weights(w, only):
    x = _inputs(19, 8, 4, 128, 128, 16, w=w)
    if only == "q":
        x["kw"] = None
    if only == "k":
        x["qw"] = None
    _run_and_check(x, eps=1e-5)


@pytest.mark.gpu
def test_in_place_and_strided():
    """q_out is q, a view of the packed projection; then a q_out with gaps between
    its rows; far positions; fewer tokens than rows."""
    x = _inputs(33, 8, 2, 128, 128, 16, far=1000000)
    _run_and_check(x, q_out=x["q"])
    x = _inputs(33, 8, 2, 64, 32, 16)
    _run_and_check(x, q_out=torch.zeros(33, 8, 3, 64, dtype=torch.bfloat16, device="cuda")[:, :, 1], n=20)


@pytest.mark.gpu
def test_zero_rows_and_large_values():
    """A head of zeros stays zero under the norm; values near bf16's largest do
    not overflow without one."""
    x = _inputs(4, 4, 2, 128, 128, 16)
    x["q"][1, 2] = 0
    x["k"][0, 1] = 0
    _run_and_check(x)
    x = _inputs(4, 4, 2, 128, 128, 16, w=None)
    x["q"][:] = 1e38 * x["q"].sign()
    _run_and_check(x)


@pytest.mark.gpu
def test_padding_and_bad_positions():
    """Slots of -1 or past the cache write no row; a position outside the table
    writes none either and NaN to the outputs; the other tokens are untouched."""
    x = _inputs(40, 4, 2, 128, 128, 16)
    x["slots"][3], x["slots"][9], x["slots"][39] = -1, x["cache"].shape[0] * 16, -5
    x["pos"][5], x["pos"][20] = -1, x["cs"].shape[0]
    before = x["cache"].clone()
    q = torch.zeros(40, 4, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(40, 2, 128, dtype=torch.bfloat16, device="cuda")
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], x["cache"], x["cs"], q, q_weight=x["qw"],
                       k_weight=x["kw"], k_out=k)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[5, 20]] = True
    assert bool(q[bad].isnan().all()) and bool(k[bad].isnan().all())
    assert bool(q[~bad].isfinite().all()) and bool(k[~bad].isfinite().all())
    y, mag = _formula(x["q"], x["qw"], x["pos"].clamp(0, 39), x["cs"], 1e-6, False)
    _close(q[~bad], (y[~bad], mag[~bad]), "q")
    ok = ~bad
    ok[[3, 9, 39]] = False
    at = x["slots"][ok] // 16, x["slots"][ok] % 16
    before[at[0], 0, at[1]] = k[ok]
    before[at[0], 1, at[1]] = x["v"][ok]
    assert torch.equal(before, x["cache"])


@pytest.mark.gpu
def test_many_tokens_and_no_tokens():
    """More tokens than a grid dimension holds; a call of none."""
    x = _inputs(70001, 1, 1, 64, 64, 64)
    _run_and_check(x)
    x = _inputs(3, 2, 1, 64, 64, 16)
    before = x["cache"].clone()
    qk_norm_rope_write(x["q"][:0], x["k"][:0], x["v"][:0], x["pos"][:0], x["slots"][:0], x["cache"], x["cs"],
                       x["q"][:0], q_weight=x["qw"], k_weight=x["kw"])
    assert torch.equal(before, x["cache"])


@pytest.mark.gpu
def test_other_stream_and_replay():
    x = _inputs(17, 8, 2, 128, 128, 16)
    q = torch.zeros_like(x["q"])
    call = lambda: qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], x["cache"], x["cs"], q,  # noqa: E731
                                      q_weight=x["qw"], k_weight=x["kw"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in range(3):
        y = _inputs(17, 8, 2, 128, 128, 16, seed=seed + 5)
        for n in ("q", "k", "v", "pos", "slots"):
            x[n].copy_(y[n])
        g.replay()
        _close(q, _formula(x["q"], x["qw"], x["pos"], x["cs"], 1e-6, False), "replayed")


def test_refusals():
    x = _inputs(4, 4, 2, 128, 64, 16, dev="cpu")
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    ok = dict(q=x["q"], k=x["k"], v=x["v"], positions=x["pos"], slot_mapping=x["slots"], kv_cache=x["cache"],
              cos_sin=x["cs"], q_out=q, q_weight=x["qw"], k_weight=x["kw"])
    for bad in (dict(q=x["q"].float()), dict(q=x["q"][..., ::2]), dict(q_out=q.float()), dict(q=x["q"][0]),
                dict(positions=x["pos"].long()), dict(slot_mapping=x["slots"].int()), dict(cos_sin=x["cs"].double()),
                dict(cos_sin=x["cs"].T), dict(q_weight=x["qw"].half()), dict(q_weight=x["qw"].float()),
                dict(k_weight=x["kw"][:64]), dict(kv_cache=x["cache"].float())):
        with pytest.raises(TypeError):
            qk_norm_rope_write(**{**ok, **bad})
    for bad in (dict(k=x["q"]), dict(v=x["v"][:3]), dict(q_out=q[:3]), dict(positions=x["pos"][:2]), dict(n_tokens=5),
                dict(n_tokens=-1), dict(kv_cache=x["cache"][:, :1]), dict(k_out=q), dict()):     # the last: on the CPU
        with pytest.raises(ValueError):
            qk_norm_rope_write(**{**ok, **bad})


def test_c_entry_refusals():
    lib = _lib.load()
    names = ("q qst qsh k kst ksh v vst vsh pos slot kc kb kt kh vc vb vt vh nb cs mp rot inter qw kw f32 eps qo qost "
             "qosh ko kost kosh n H nkv d page stream").split()
    ok = dict.fromkeys(names, 16)
    ok |= dict(nb=4, mp=8, rot=64, inter=0, f32=0, eps=1e-6, n=1, H=4, nkv=2, d=128, page=16, stream=0)
    for bad in (dict(d=96), dict(page=8), dict(rot=8), dict(rot=144), dict(rot=-16), dict(n=-1), dict(H=0), dict(nb=0),
                dict(mp=0), dict(eps=-1.0), dict(eps=float("nan")), dict(q=0), dict(cs=0), dict(slot=0), dict(qst=4),
                dict(vh=12), dict(kost=2), dict(q=8), dict(kc=24), dict(cs=4), dict(qw=2), dict(H=5000)):
        assert lib.locks_qkv_write(*{**ok, **bad}.values()) == -1, bad
        assert lib.locks_last_error()
