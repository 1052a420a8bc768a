"""Rotation by positions of several axes (qk_norm_rope_write with RopeAxes), against
the formulas in 64 bits, and the calls that are refused.

Tolerance: as for one position (tests/test_qkv.py): one rounding to bf16, 2^-8 of the
value, and 2^-16 of the pair's magnitude |a| + |b| for the fp32 norm, products and sums."""
import pytest
import torch

from locks import _lib
from locks.attention import RopeAxes, kv4_cache, qk_norm_rope_write


def test_axes_of_pairs():
    assert RopeAxes.sections((2, 3, 3)).pairs == (0, 0, 1, 1, 1, 2, 2, 2)
    assert RopeAxes.cycled((3, 2, 3)).pairs == (0, 1, 2, 0, 1, 2, 0, 2)
    assert RopeAxes.sections((0, 8)).n_axes == 2 and RopeAxes([0] * 8).n_axes == 1
    a = RopeAxes(([0] * 15 + [3]) * 8)
    assert a.n_axes == 4 and len(a.pairs) == 128 and a.words[0] == -(1 << 62) | 3 << 30
    for bad in ([], [0] * 7, [0] * 136, [4] * 8, [-1] * 8):
        with pytest.raises(ValueError):
            RopeAxes(bad)
    with pytest.raises(ValueError):
        RopeAxes([0, 1] * 4, 1)
    with pytest.raises(ValueError):
        RopeAxes.cycled((9, -1))


def inputs(T, H, n_kv, d, rot, n_axes, *, page=16, far=0, w=torch.bfloat16, seed=0, dev="cuda"):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    blocks = -(-T // page) + 3
    q, k, v = ((r(T, h, d) * 3).to(torch.bfloat16) for h in (H, n_kv, n_kv))
    slots = torch.randperm(blocks * page, generator=g, device=dev)[:T]
    ang = torch.arange(far + 200, dtype=torch.float64, device=dev)[:, None] * (
        10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot))
    pos = far + torch.randint(0, 200, (n_axes, T), generator=g, device=dev, dtype=torch.int32)
    weights = [(1 + 0.3 * r(d)).to(w) for _ in range(2)] if w is not None else [None, None]
    return dict(q=q, k=k, v=v, slots=slots, pos=pos, cs=torch.cat([ang.cos(), ang.sin()], 1).float(), qw=weights[0],
                kw=weights[1], page=page, blocks=blocks)


def formula(x, weight, pos, cs, axes, eps, interleaved):
    """(value, magnitude of its pair) in 64 bits, pair by pair."""
    x = x.double()
    if weight is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    y, mag = x.clone(), x.abs()
    half = cs.shape[1] // 2
    for p, a in enumerate(axes.pairs):
        c, s = cs[pos[a].long(), p].double()[:, None], cs[pos[a].long(), half + p].double()[:, None]
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        mag[..., i] = mag[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, mag


def _close(got, want):
    y, mag = want
    assert bool(((got.double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -16 * mag * 1.01).all())


def _check(x, axes, *, interleaved=False, eps=1e-6):
    n_kv, d = x["k"].shape[1:]
    cache = torch.randn(x["blocks"], 2, x["page"], n_kv, d, device="cuda").to(torch.bfloat16)
    before, q, k = cache.clone(), torch.zeros_like(x["q"]), torch.zeros_like(x["k"])
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], cache, x["cs"], q, q_weight=x["qw"],
                       k_weight=x["kw"], eps=eps, interleaved=interleaved, k_out=k, axes=axes)
    _close(q, formula(x["q"], x["qw"], x["pos"], x["cs"], axes, eps, interleaved))
    _close(k, formula(x["k"], x["kw"], x["pos"], x["cs"], axes, eps, interleaved))
    at = x["slots"] // x["page"], x["slots"] % x["page"]
    before[at[0], 0, at[1]], before[at[0], 1, at[1]] = k, x["v"]
    assert torch.equal(before, cache)
    return q, k


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d, rot, axes", [
    (128, 128, RopeAxes.sections((16, 24, 24))), (128, 128, RopeAxes.cycled((24, 20, 20))),
    (64, 64, RopeAxes.sections((16, 16))), (256, 256, RopeAxes.cycled((1, 63, 40, 24))),
    (128, 32, RopeAxes.sections((3, 0, 13))), (64, 16, RopeAxes([2, 0, 1, 0, 0, 2, 1, 1]))])
@pytest.mark.parametrize("T, H, n_kv", [(1, 32, 8), (77, 5, 3)])
def test_formula(T, H, n_kv, d, rot, axes, interleaved):
    _check(inputs(T, H, n_kv, d, rot, axes.n_axes, seed=T + d), axes, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("w", [None, torch.float32])
def test_weights_far_and_padded_rows(w):
    """Far positions; positions whose rows have gaps between them."""
    axes = RopeAxes.sections((16, 24, 24))
    x = inputs(40, 8, 2, 128, 128, 3, far=1000000, w=w)
    wide = torch.full((3, 64), -7, dtype=torch.int32, device="cuda")
    wide[:, :40] = x["pos"]
    x["pos"] = wide[:, :40]
    _check(x, axes)


@pytest.mark.gpu
def test_equal_axes_are_one_position():
    """The same position along every axis: the same bits as without axes."""
    x = inputs(50, 8, 2, 128, 128, 3)
    x["pos"][1:] = x["pos"][0]
    q, k = _check(x, RopeAxes.cycled((24, 20, 20)))
    one, cache = torch.zeros_like(q), torch.zeros(x["blocks"], 2, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"][0].contiguous(), x["slots"], cache, x["cs"], one,
                       q_weight=x["qw"], k_weight=x["kw"])
    assert torch.equal(one, q)


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
def test_bad_positions_and_slots(four):
    """A position outside the table along any axis: NaN, and no row written."""
    axes = RopeAxes.sections((16, 24, 24))
    x = inputs(30, 4, 2, 128, 128, 3)
    x["pos"][0, 3], x["pos"][1, 8], x["pos"][2, 29] = -1, 200, 1 << 30
    x["slots"][5], x["slots"][6] = -1, x["blocks"] * 16
    cache = (kv4_cache(x["blocks"], n_kv=2, head_dim=128, page=16, device="cuda") if four
             else torch.zeros(x["blocks"], 2, 16, 2, 128, dtype=torch.bfloat16, device="cuda"))
    before, q, k = cache.clone(), torch.zeros_like(x["q"]), torch.zeros_like(x["k"])
    bad = torch.tensor([3, 8, 29], device="cuda")
    keep = x["slots"].clone()
    x["slots"][:] = -1
    x["slots"][bad] = keep[bad]
    for s in (5, 6):
        x["slots"][s] = keep[s]
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], cache, x["cs"], q, q_weight=x["qw"],
                       k_weight=x["kw"], k_out=k, axes=axes)
    assert torch.equal(cache, before)
    for y in (q, k):
        assert bool(y[bad].isnan().all())
        y[bad] = 0
        assert bool(y.isfinite().all())


@pytest.mark.gpu
def test_replay_on_another_stream():
    axes = RopeAxes.cycled((24, 20, 20))
    x = inputs(21, 8, 2, 128, 128, 3)
    cache = torch.zeros(x["blocks"], 2, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros_like(x["q"])
    call = lambda: qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"], x["slots"], cache, x["cs"], q,  # noqa: E731
                                      q_weight=x["qw"], k_weight=x["kw"], axes=axes)
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in range(3):
        y = inputs(21, 8, 2, 128, 128, 3, seed=seed + 5)
        for n in ("q", "k", "v", "pos", "slots"):
            x[n].copy_(y[n])
        g.replay()
        _close(q, formula(x["q"], x["qw"], x["pos"], x["cs"], axes, 1e-6, False))


def test_refusals():
    axes = RopeAxes.sections((16, 24, 24))
    x = inputs(4, 4, 2, 128, 128, 3, dev="cpu")
    cache = torch.zeros(x["blocks"], 2, 16, 2, 128, dtype=torch.bfloat16)
    ok = dict(q=x["q"], k=x["k"], v=x["v"], positions=x["pos"], slot_mapping=x["slots"], kv_cache=cache,
              cos_sin=x["cs"], q_out=torch.zeros_like(x["q"]), q_weight=x["qw"], k_weight=x["kw"], axes=axes)
    for bad in (dict(axes=(16, 24, 24)), dict(positions=x["pos"][0]), dict(positions=x["pos"].long()),
                dict(positions=x["pos"].T.contiguous().T), dict(axes=None)):
        with pytest.raises(TypeError):
            qk_norm_rope_write(**{**ok, **bad})
    for bad in (dict(positions=x["pos"][:2]), dict(positions=x["pos"][:, :3]), dict(cos_sin=None),
                dict(cos_sin=x["cs"][:, :64].contiguous()), dict(axes=RopeAxes.sections((8, 8, 8))),
                dict(axes=RopeAxes.sections((32, 32))), dict()):                        # the last: on the CPU
        with pytest.raises(ValueError):
            qk_norm_rope_write(**{**ok, **bad})


def test_c_entry_refusals():
    lib = _lib.load()
    names = ("q qst qsh k kst ksh v vst vsh pos pax na a0 a1 a2 a3 slot kc kb kt kh vc vb vt vh nb cs mp rot inter qw kw "
             "f32 eps qo qost qosh ko kost kosh n H nkv d page stream").split()
    ok = dict.fromkeys(names, 16)
    ok |= dict(na=2, a0=1, a1=0, a2=0, a3=0, nb=4, mp=8, rot=64, inter=0, f32=0, eps=1e-6, n=1, H=4, nkv=2, d=128,
               page=16, stream=0)
    for bad in (dict(na=0), dict(na=5), dict(na=-1), dict(a0=2), dict(a0=-1), dict(na=1), dict(rot=128, a1=-1), dict(d=96),
                dict(page=8), dict(rot=8), dict(q=0), dict(cs=0), dict(pos=0), dict(qst=4), dict(kc=24), dict(H=5000)):
        assert lib.locks_qkv_write_axes(*{**ok, **bad}.values()) == -1, bad
        assert lib.locks_last_error().startswith(b"locks_qkv_write_axes")
