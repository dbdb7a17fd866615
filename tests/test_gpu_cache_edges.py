"""Cache-maintenance operators on a B200 at the edges of their ranges: uneven head counts with long tile
tables, numbers that are not numbers where a query sees them, scales at the end of FP32, scratch sizes,
and DeviceKVCache's failures and captures."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from kvssd_b200 import ops
from kvssd_b200.quant import quantize_tensor

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def key_pool(nb, bt, kvh, d, bits, group, seed):
    q = quantize_tensor(torch.randn(nb, bt, kvh, d, generator=gen(seed)) * 1.5, bits, group)
    return q.packed.to(DEV), q.scales.to(DEV)


# ------------------------------------------------------------------------------- attention weights


@pytest.mark.parametrize("kvh, places, d, bits, group, dtype", [
    (60, 9_000, 64, 4, 32, torch.float16), (60, 9_000, 64, 2, 16, torch.float32),
    (20, 23_000, 96, 4, 32, torch.bfloat16), (20, 23_000, 64, 4, 32, torch.float32),
    (9, 30_000, 64, 2, 32, torch.float16), (14, 45_000, 64, 4, 16, torch.float16),
    (12, 44_400, 128, 4, 32, torch.float16), (7, 90_000, 64, 2, 32, torch.bfloat16)])
def test_weights_step_many_short_blocks_of_uneven_heads(kvh, places, d, bits, group, dtype):
    """Head counts that leave warps of a CTA over, with more than 256 tiles a CTA: every place gets what
    its pool block gets in a short call over the pool, bit for bit."""
    pool = 97
    kp, ks = key_pool(pool, 1, kvh, d, bits, group, kvh)
    valid = torch.ones(pool, dtype=torch.int32, device=DEV)
    valid[5] = 0
    query = torch.randn(kvh, d, generator=gen(1)).to(dtype).to(DEV)
    lse = torch.linspace(-1.0, 2.0, kvh, device=DEV)
    scale = 1 / math.sqrt(d)
    table = torch.randint(0, pool, (places,), generator=gen(places)).int().to(DEV)
    once, _ = ops.attention_weights(query, kp, ks, valid, bits, group, scale, lse=lse)
    assert (once[:, 5] == 0).all() and (once[:, 6:] > 0).all()
    many, _ = ops.attention_weights(query, kp, ks, valid, bits, group, scale, lse=lse, block_table=table)
    assert torch.equal(many, once[:, table.long()])
    assert ops.read_device_status(DEV) == 0
