"""A pool that is used first on one stream and then on another, with nothing of the caller's between them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("kind", ["interleaved", "split", "int8"])
def test_first_use_on_a_busy_stream(kind):
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    args = dict(num_blocks=6, block_size_tokens=16, num_layers=1, num_kv_heads=2, head_dim=64, dtype=torch.float16,
                device=DEV)
    pool = Int8KVBlockPool(**args) if kind == "int8" else GpuKVBlockPool(**args, kv_layout=kind)
    # Small integers with a 64 in every page: the 8-bit pool holds them exactly.
    g = torch.Generator().manual_seed(1)
    kv = torch.randint(-60, 61, (2, 1, 2, 40, 64), generator=g).half()
    kv[..., ::16, 0] = 64.0
    kv = kv.to(DEV)
    table, start = torch.tensor([[4, 0, 3]], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(40_000_000)  # tens of milliseconds
        pool._ensure_pools()
    with torch.cuda.stream(other):
        pool.write_tokens_batch(0, table, start, kv[0], kv[1])
    torch.cuda.synchronize()
    k, v = pool.gather_layer(0, [4, 0, 3], 40)
    assert torch.equal(k, kv[0]) and torch.equal(v, kv[1])
    assert pool.allocated_block_count() == 3
