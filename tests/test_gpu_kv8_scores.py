"""Scores of the 8-bit cache's decode attention where they are hard: queries whose mean is far from zero,
negative scales, scores of any size.

Bars: every score here is a sum whose products and partial sums, in any order, are multiples of one unit and
below 2**24 of it, so fp32 holds it exactly. What is left is the attention's own bar, 6 u of the largest
|value| that a head averages, u half a step of the 16-bit type: weights rounded to it in numerator and
denominator (4 u), the output (u), scale, exponentials and sums in fp32 (u).
"""

from __future__ import annotations

import pytest
import torch

from oracle.kv8 import Kv8Cache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
LENS = [200, 700]


def _int(x):
    return torch.tensor(x, dtype=torch.int32)


def _filled(keys, g, bs, d, dtype):
    """A pool and its definition with one head's ``keys`` [n, d] of each row, and values of a normal spread."""
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool

    nb = sum(-(-len(k) // bs) for k in keys)
    pool = Int8KVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=1, num_kv_heads=1, head_dim=d, dtype=dtype,
                           device=DEV)
    cache = Kv8Cache(nb, 1, bs, d, dtype)
    tables, at = torch.full((len(keys), max(-(-len(k) // bs) for k in keys)), -1, dtype=torch.int32), 0
    for i, k in enumerate(keys):
        n = -(-len(k) // bs)
        tables[i, :n] = torch.arange(at, at + n).flip(0)
        at += n
        k, v = k.to(dtype)[None, None], torch.randn(1, 1, len(k), d, generator=g).to(dtype)
        pool.write_tokens_batch(0, tables[i:i + 1].to(DEV), _int([0]).to(DEV), k.to(DEV), v.to(DEV))
        cache.write(tables[i:i + 1], [0], k, v)
    return pool, cache, tables


def _check(pool, cache, tables, q, scale, dtype):
    want, most = cache.attend(q, tables, LENS, scale)
    wide = torch.cat([tables, torch.full((len(tables), 140_000 // cache.bs), -7, dtype=torch.int32)], dim=1)
    for table in (tables, wide):  # a workgroup per row; rows shared out between waves
        out = pool.attend(0, q[:, :, None].to(DEV), table.to(DEV), _int(LENS).to(DEV), scale, q.shape[1])
        got = out.cpu().double().view(want.shape)
        assert torch.isfinite(got).all()
        worst = ((got - want).abs() - 6 * torch.finfo(dtype).eps / 2 * most[..., None]).max()
        assert worst <= 0, f"{float(worst)} over the bound"
    return want


@pytest.mark.parametrize("scale", [0.5, -0.5])
@pytest.mark.parametrize("bs,d,dt", [(16, 128, "fp16"), (16, 128, "bf16"), (32, 64, "fp16"), (4, 128, "bf16"),
                                     (8, 64, "bf16"), (4, 64, "fp16")])
def test_queries_with_a_mean(bs, d, dt, scale):
    """Query elements of 256 to 511 against keys that are pairs (a, -a), but for one channel: what the large
    elements add is exactly zero, whatever their sum."""
    dtype, g = DTYPES[dt], torch.Generator().manual_seed(bs + d)
    step = 0.25 if dtype == torch.float16 else 2.0  # of the type's numbers there
    q = 256 + step * torch.randint(0, int(256 / step), (2, 4, d // 2), generator=g).repeat_interleave(2, dim=-1)
    q[..., 0], q[..., 1] = 0.0, torch.tensor([0.125, -0.125, 0.0, 0.25])
    keys = []
    for n in LENS:
        k = torch.randint(-3, 4, (n, d // 2), generator=g).repeat_interleave(2, dim=-1).float()
        k[:, 1::2] *= -1
        k[:, 1] = torch.randint(-100, 101, (n,), generator=g).float()
        k[:, 0] = 127.0                               # the page's scale is 1 ...
        k *= 1 + (torch.arange(n) // bs % 3 == 1).float()[:, None]  # ... or 2
        keys.append(k)
    pool, cache, tables = _filled(keys, g, bs, d, dtype)
    want = _check(pool, cache, tables, q.to(dtype), scale, dtype)
    assert (want[:, 0] - want[:, 1]).abs().max() > 0.1


@pytest.mark.parametrize("scale", [1.0, -1.0])
@pytest.mark.parametrize("bs,d,dt", [(16, 64, "fp16"), (16, 128, "bf16"), (4, 128, "fp16"), (32, 64, "bf16")])
def test_large_scores(bs, d, dt, scale):
    """Integer scores up to 10**5 that rise and fall along a row, so that the running maximum moves, with one
    token ahead by more than 100: it takes the output alone."""
    dtype, g = DTYPES[dt], torch.Generator().manual_seed(d)
    q = torch.zeros(2, 3, d)
    q[:, 0, 0], q[:, 1, 0], q[:, 2, 0] = 30.0, -30.0, 800.0
    q[..., 1] = 1.0
    keys = []
    for n in LENS:
        k = torch.zeros(n, d)
        k[:, 0] = torch.randint(-120, 121, (n,), generator=g).float()
        k[n // 3, 0], k[n // 2, 0] = 126.0, -126.0
        k[:, 2:] = torch.randint(-127, 128, (n, d - 2), generator=g).float()  # the query has zeros there
        k[:, 1] = 127.0
        keys.append(k)
    pool, cache, tables = _filled(keys, g, bs, d, dtype)
    want = _check(pool, cache, tables, q.to(dtype), scale, dtype)
    for b, n in enumerate(LENS):
        v, _ = cache.row(tables[b], n, 0, 1)
        for h, sign in ((0, 1), (1, -1), (2, 1)):
            winner = v[n // 3 if sign * scale > 0 else n // 2]
            assert (want[b, h] - winner).abs().max() <= 1e-10 * v.abs().max()
