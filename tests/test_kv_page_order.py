"""Copies of pages that depend on each other, in lists that one launch each can take: the same pages as all at once."""

from __future__ import annotations

import ctypes
import random
from types import SimpleNamespace

import pytest
import torch

from runtime_amd.phase2 import _hip
from runtime_amd.phase2.paged_kv_kernel import MAX_DEPENDENT, GpuKVBlockPool, dependent_batches


def _entries(src, dst):
    """Entries of an ordered launch: the pairs whose pages depend on each other, one more per cycle."""
    of = dict(zip(dst, src))
    assert len(of) == len(dst)
    tied = [d for d, s in of.items() if s in of or d in set(of.values())]
    seen, cycles = set(), 0
    for d in tied:
        path = []
        while d in of and d not in seen:
            seen.add(d)
            path.append(d)
            d = of[d]
        cycles += d in path
    return len(tied) + cycles


def _check(src, dst, pages):
    batches = dependent_batches(src, dst)
    now = list(range(pages))
    for s, d in batches:
        assert 0 < len(s) == len(d) and _entries(s, d) <= MAX_DEPENDENT
        was = list(now)
        for a, b in zip(s, d):
            now[b] = was[a]
    of = {b: a for a, b in zip(src, dst)}
    assert now == [of.get(i, i) for i in range(pages)]
    return batches


@pytest.mark.parametrize("n", [2, 446, 447, 448, 449, 893, 894, 895, 1000, 2500])
def test_chains_and_cycles(n):
    ids = random.Random(n).sample(range(n + 1), n + 1)
    assert len(_check(ids[:-1], ids[1:], n + 1)) == -(-n // MAX_DEPENDENT)
    _check(ids[:-1], [*ids[1:-1], ids[0]], n + 1)


def test_many_small_cycles_share_lists():
    src = list(range(1200))
    assert len(_check(src, [i ^ 1 for i in src], 1200)) == 5  # 600 pairs of pages, 149 in a list


@pytest.mark.parametrize("seed", range(30))
def test_any_lists(seed):
    rng = random.Random(seed)
    pages = rng.choice([3, 40, 600, 3000])
    if seed % 3 == 0:  # permutations: cycles of any length
        dst = list(range(pages))
        src = rng.sample(dst, pages)
    else:              # trees, cycles with branches, destinations that occur again
        dst = [rng.randrange(pages) for _ in range(pages)]
        src = [rng.randrange(pages // 3 + 1) if seed % 3 == 1 else rng.randrange(pages) for _ in dst]
    _check(src, dst, pages)


def test_a_device_pool_copies_long_chains_with_its_own_launches(monkeypatch):
    """The pool's calls over a library that refuses what one launch does not hold, on host memory."""
    pool = GpuKVBlockPool(num_blocks=1201, block_size_tokens=4, num_layers=2, num_kv_heads=1, head_dim=8,
                          dtype=torch.float32, device="cuda")
    data = torch.randn(2, 1201, 1, 2, 4, 8)
    pool._regions, pool._k_pool, pool._used_map = [data], data[:, :, :, 0], torch.zeros(1201, dtype=torch.uint8)
    calls = []

    def copy(base, page, stride, base2, page2, stride2, layers, pages, src, dst, n, used, move, stream):
        of, to = ([*(ctypes.c_int32 * n).from_address(p)] for p in (src, dst))
        assert base == data.data_ptr() and used == pool._used_map.data_ptr() and not move
        if _entries(of, to) > MAX_DEPENDENT:
            return _hip.MX_ERR_UNSUPPORTED
        calls.append(n)
        data[:, to] = data[:, of]
        return _hip.MX_OK

    monkeypatch.setattr(_hip, "load", lambda: SimpleNamespace(mx_kv_copy_pages=copy))
    monkeypatch.setattr(_hip, "stream_handle", lambda device: None)
    was = data.clone()
    pool.copy_blocks(range(1200), range(1, 1201))
    assert torch.equal(data[:, 1:], was[:, :-1]) and calls == [448, 448, 304]
