"""LocksEngine.forward_dense refuses a split of the batch that it cannot serve
(before anything touches a GPU)."""
import pytest

from locks.backend.engine import LocksEngine


@pytest.mark.parametrize("n_decode, starts", [(-1, None), (4, None), (2, None), (0, None), (4, [0, 1, 2, 3])])
def test_refusals(n_decode, starts):
    eng = LocksEngine.__new__(LocksEngine)
    with pytest.raises(ValueError, match="n_decode"):
        eng.forward_dense(None, None, None, None, 3, 1.0, None, query_start_loc=starts, n_decode=n_decode)
