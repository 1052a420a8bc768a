"""The paged cache in 4 bits at the edges of its documentation: memory that nobody wrote,
and weights and angles of any size.  Tolerances: those of tests/test_kv4.py."""
import pytest
import torch

from locks.attention import RopeAxes, qk_norm_rope_write
from tests.test_kv4 import _blank, _decode, _prefill, _read, case, quantised
from tests.test_rope_axes import formula, inputs
from tests.test_window import _agree, _exact


def _unwritten(c, fill):
    """The case with `fill` in every byte where no token lies (not what a cache's rows hold)."""
    page, cache = c["page"], c["kv"]
    whole = cache.clone()
    cache.fill_(fill)
    for r, n in enumerate(c["lens"]):
        t = torch.arange(n, device="cuda")
        slots = c["bt"][r].long()[t // page] * page + t % page
        k, v = _read(whole, slots)
        qk_norm_rope_write(k, k, v, t.int(), slots, cache, None, torch.empty_like(k))
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0, 127, 252, 253, 254, 255])
@pytest.mark.parametrize("d, page, n_kv, G", [(64, 32, 1, 8), (128, 16, 2, 4), (256, 64, 1, 4)])
def test_bytes_that_nobody_wrote(d, page, n_kv, G, fill):
    """Scales that no write makes (253 and 254: entries past bf16's range) lie in masked
    places only, and reach no row there."""
    c = _unwritten(case([130, 300, 65], [40, 7, 65], n_kv, G, d, page), fill)
    for window, sinks in ((0, 0), (50, 3)):
        _agree(*_prefill(c, window, sinks), _exact(c, window, sinks))
    c = _unwritten(case([130, 300, 65], [1, 1, 1], n_kv, G, d, page), fill)
    for window, sinks in ((0, 0), (50, 3)):
        _agree(*_decode(c, window, sinks), _exact(c, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [150, 6000])
@pytest.mark.parametrize("weight, table", [(2.0 ** 59, 1.0), (2.0 ** 30, 1.0), (1.0, 2.0 ** 59), (2.0 ** 15, 2.0 ** 5)])
def test_large_weights_over_small_entries(weight, table, T, interleaved):
    """Blocks whose normed entries lie below fp32's normal numbers, where weights or angles
    bring them back: the codes are those of 64 bits."""
    d, n_kv = 128, 1
    x = inputs(T, 2, n_kv, d, d, 1, w=torch.float32)
    x["kw"], x["cs"] = torch.full_like(x["kw"], weight), x["cs"] * table
    # one block in two of a pair's halves (or of adjacent pairs) tiny, the norm that of the others
    tiny = torch.arange(d, device="cuda") // 32 % 2 == 0
    x["k"] = torch.where(tiny, x["k"].float() * 2.0 ** -110, x["k"].float() * 2.0 ** 35).to(torch.bfloat16)
    cache = _blank(x["blocks"], n_kv, d, 16)
    qk_norm_rope_write(x["q"], x["k"], x["v"], x["pos"][0], x["slots"], cache, x["cs"], torch.zeros_like(x["q"]),
                       k_weight=x["kw"], interleaved=interleaved)
    k64 = formula(x["k"], x["kw"], x["pos"], x["cs"], RopeAxes([0] * (d // 2)), float(torch.tensor(1e-6)), interleaved)[0]
    _, _, want, near = quantised(k64)
    k, _ = _read(cache, x["slots"])
    assert torch.equal(torch.where(near, 0, k.double()), torch.where(near, 0, want)) and int(near.sum()) < 3
