"""The paged cache in 4 bits at the edges of its documentation: memory that nobody wrote.
Tolerances: those of tests/test_kv4.py."""
import pytest
import torch

from locks.attention import qk_norm_rope_write
from tests.test_kv4 import _blank, _decode, _prefill, _read, case
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
