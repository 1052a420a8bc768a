"""What LocksEngine.write_qkv hands to the DRAM tier: the keys only where the tier takes
them, and no more tokens than it has slots for."""
import types

import pytest
import torch

from locks.backend.engine import LocksEngine


def test_more_tokens_than_the_tier_has_slots():
    eng = LocksEngine.__new__(LocksEngine)
    eng.tier, eng.max_tokens, eng._k_out, eng.kv_caches = types.SimpleNamespace(offload_k=False), 4, None, [None]
    with pytest.raises(ValueError, match="max_num_batched_tokens 4"):
        eng.write_qkv(0, torch.zeros(5, 8, 128), None, None, None, None, None, None)
    with pytest.raises(ValueError, match="max_num_batched_tokens 4"):
        eng.write_qkv(0, torch.zeros(9, 8, 128), None, None, None, None, None, None, n_tokens=5)


@pytest.mark.gpu
def test_keys_only_where_the_tier_takes_them():
    from tests.test_gpu_serving_step import Model
    for variant, rows in (("fast", None), ("mem-v", None), ("mem-kv", 400)):
        eng = Model(variant).eng
        assert (None if eng._k_out is None else eng._k_out.shape[0]) == rows, variant


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["fast", "mem-v", "mem-kv"])
def test_no_tokens(variant):
    """A step without tokens is no error, with a tier or without."""
    from tests.test_gpu_serving_step import D, G, N_KV, Model
    m = Model(variant)
    z = lambda h: torch.zeros(3, h, D, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    qo = torch.full_like(z(N_KV * G), 7.0)
    m.eng.write_qkv(0, z(N_KV * G), z(N_KV), z(N_KV), m.t.positions, m.t.slot_mapping, m.cs, qo, n_tokens=0)
    assert bool((qo == 7).all())
