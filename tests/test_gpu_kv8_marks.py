"""Which blocks of an 8-bit pool count as written: exactly those that a token went to."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _pool(nb, hkv, bs, d, layers=1):
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool

    return Int8KVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=layers, num_kv_heads=hkv, head_dim=d,
                           dtype=torch.float16, device=DEV)


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _marked(used):
    return used.nonzero().flatten().tolist()


@pytest.mark.parametrize("bs,d", [(4, 64), (16, 128), (32, 64)])
def test_writes_mark_their_blocks(bs, d):
    pool = _pool(12, 2, bs, d)
    tables = _int([[7, 3, 0], [5, 12, 9], [1, -1, 11]])  # two blocks outside the pool
    for starts, t, want in (([0, 0, 0], 1, [1, 5, 7]),
                            ([bs - 1, 2 * bs, 0], 2, [1, 3, 5, 7, 9]),
                            ([bs, bs, bs], bs, [1, 3, 5, 7, 9]),              # rows 1 and 2 miss the pool
                            ([2 * bs, 0, 2 * bs], bs, [0, 1, 3, 5, 7, 9, 11]),
                            ([3 * bs, -bs, 7], 0, [0, 1, 3, 5, 7, 9, 11])):
        x = torch.randn(3, 2, t, d, device=DEV).half()
        pool.write_tokens_batch(0, tables, _int(starts), x, x)
        assert _marked(pool._used_map) == want


@pytest.mark.parametrize("partials", [False, True])
@pytest.mark.parametrize("bs,d", [(16, 128), (4, 64)])
def test_rotary_writes_mark_their_blocks(bs, d, partials):
    from runtime_amd.phase2.kv8 import kv8_rope_append

    hq, hkv, b = 4, 2, 5
    pool = _pool(12, hkv, bs, d)
    layer = pool.layer_store(0)
    tables = _int([[7, 3], [5, 12], [1, 11], [4, 2], [8, 6]])
    rope = torch.ones(2 * bs + 1, d // 2, 2, device=DEV)
    used, q = torch.zeros(12, dtype=torch.uint8, device=DEV), torch.empty(b, hq * d, dtype=torch.float16, device=DEV)
    part = torch.randn(2, b, (hq + 2 * hkv) * d, device=DEV)
    for pos, want in (([0, bs, 1, -1, 2 * bs], [1, 7]),       # outside the pool, the rope table and the block table
                      ([bs, 1, bs, bs - 1, 2 * bs + 1], [1, 3, 4, 5, 7, 11])):
        kv8_rope_append(None if partials else part[0].half(), rope, _int(pos), q, layer, tables, hq,
                        partials=part if partials else None, splits=2 if partials else 0, used_blocks=used)
        assert _marked(used) == want


@pytest.mark.parametrize("batch", [2, 16, 40])
def test_a_native_step_marks_the_blocks_of_its_tokens(batch):
    from runtime_amd.phase2.decode_step import DecoderShape, Int8DecodeModel

    shape = DecoderShape(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, intermediate=512, vocab=1024, qkv_bias=True)
    model = Int8DecodeModel(shape, device=DEV, seed=batch, max_positions=256)
    g = torch.Generator().manual_seed(batch)
    tables = torch.randperm(batch * 4, generator=g).view(batch, 4).int()
    lens = torch.randint(0, 64, (batch,), generator=g).int()
    pool = _pool(batch * 4, 2, 16, 64, layers=2)
    x = torch.randn(batch, 2, 64, 64, generator=g).half().to(DEV)
    for li in range(2):
        pool.write_tokens_batch(li, tables.to(DEV), torch.zeros(batch, dtype=torch.int32, device=DEV), x, x)
    pool._used_map.zero_()
    model.step(torch.zeros(batch, dtype=torch.int64, device=DEV), pool, tables.to(DEV), lens.to(DEV))
    assert _marked(pool._used_map) == sorted(int(tables[i, n // 16]) for i, n in enumerate(lens.tolist()))
    assert model.error_flag() == 0
