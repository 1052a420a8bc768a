"""LocksEngine.write_qkv beside the DRAM tier."""
import pytest
import torch


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
