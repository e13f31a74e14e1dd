"""``ops.cache_load`` without slots: empty tensors, as the writers take none."""
import numpy as np
import pytest
import torch

import span_plain as plain
from tq4_decode import codebook, ops

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("preset", ["4bit", "k8v4"])
def test_no_slots(dev, preset, dtype):
    kb, vb = plain.PRESETS[preset]
    cache, _, _ = plain.make_cache(np.random.default_rng(1), 3, 16, 2, preset, "soa")
    cents = None if kb == 8 else torch.from_numpy(codebook.centroids(D, kb).astype(np.float32)).to(dev)
    rot = None if kb == 8 else torch.eye(D, device=dev)
    slots = torch.empty(0, dtype=torch.int32, device=dev)
    key, value = ops.cache_load(cache.to(dev), slots, rot, cents, key_bits=kb, value_bits=vb, dtype=dtype)
    assert key.shape == value.shape == (0, 2, D) and key.dtype == value.dtype == dtype
    with pytest.raises(RuntimeError, match="slot_mapping"):
        ops.cache_load(cache.to(dev), slots[None], rot, cents, key_bits=kb, value_bits=vb, dtype=dtype)
