"""CPU: ``PrefixBatch.fork`` and ``compact`` keep the block bookkeeping whole (reference counts, free list,
tables), and the pairs they return carry a CPU pool's tokens along."""

from __future__ import annotations

import math
import random

import pytest
import torch

from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool
from runtime_amd.phase2.prefix_batch import BlockAllocator, PrefixBatch


def _whole(pb: PrefixBatch, num_blocks: int) -> None:
    """Every block's references are the rows and groups that hold it; the others are free, once each."""
    refs = [0] * num_blocks
    for ids in [r.blocks for r in pb.rows] + pb.prefix_blocks:
        assert len(set(ids)) == len(ids)
        for i in ids:
            refs[i] += 1
    assert [pb.alloc.refcount(i) for i in range(num_blocks)] == refs
    assert sorted(pb.alloc._free) == [i for i in range(num_blocks) if refs[i] == 0]
    for r in pb.rows:
        assert len(r.blocks) >= math.ceil(r.length / pb.block_size)


def test_allocator_compacts_with_the_fewest_moves():
    a = BlockAllocator(10, seed=3)
    ids = a.alloc(8)
    a.incref(ids[:2])
    gone = [i for i in (0, 3, 9) if i in ids]
    for i in gone:
        while a.refcount(i):
            a.decref([i])
    live = {i: a.refcount(i) for i in range(10) if a.refcount(i)}
    moves = a.compact()
    n = len(live)
    assert set(moves) == {i for i in live if i >= n} and all(new < n for new in moves.values())
    assert {moves.get(i, i): c for i, c in live.items()} == {i: a.refcount(i) for i in range(n)}
    assert a.free_blocks == 10 - n and a.alloc(10 - n) == list(range(n, 10)) and a.compact() == {}
    with pytest.raises(RuntimeError):
        a.alloc(1)


@pytest.mark.parametrize("prefix", [0, 16])
def test_forks_and_compaction_carry_every_rows_tokens(prefix):
    bs, blocks = 4, 200
    rng = random.Random(prefix)
    pb = PrefixBatch(batch=8, groups=2, prefix_tokens=prefix, lo=3, hi=40, block_size=bs, num_blocks=blocks, headroom=6,
                     seed=1)
    pool = GpuKVBlockPool(num_blocks=blocks, block_size_tokens=bs, num_layers=2, num_kv_heads=1, head_dim=2,
                          dtype=torch.float32, device="cpu")
    tokens: dict[int, torch.Tensor] = {}

    def fill(b):
        r = pb.rows[b]
        for li in range(2):  # the prefix's tokens are written by every row that holds it, alike
            x = torch.randn(1, 1, r.length, 2)
            if r.shared:
                x[:, :, :prefix] = r.group + 1
            pool.write_tokens(li, r.blocks, 0, x, -x)
            tokens[b, li] = x[0, 0].clone()

    def check():
        _whole(pb, blocks)
        for b, r in enumerate(pb.rows):
            for li in range(2):
                k, v = pool.gather_layer(li, r.blocks, r.length)
                assert torch.equal(k[0, 0], tokens[b, li]) and torch.equal(v, -k)

    for b in range(8):
        fill(b)
    check()
    for turn in range(12):
        group = rng.randrange(2)
        row = 4 * group + rng.randrange(4)
        slots = [s for s in range(4 * group, 4 * group + 4) if s != row and rng.random() < 0.7]
        pool.copy_blocks(*pb.fork(row, slots))
        for s in slots:
            for li in range(2):
                tokens[s, li] = tokens[row, li].clone()
        check()
        for b in range(8):  # a step: every row appends a token of its own
            r = pb.rows[b]
            for li in range(2):
                x = torch.randn(1, 1, 1, 2)
                pool.write_tokens(li, r.blocks, r.length, x, -x)
                tokens[b, li] = torch.cat([tokens[b, li], x[0, 0]])
        pb.advance()
        check()
        tables = pb.tables
        src, dst = pb.compact()
        if src:
            got = pool.move_blocks(src, dst, tables)
            for b, r in enumerate(pb.rows):
                assert got[b, :len(r.blocks)].tolist() == r.blocks
        assert pb.compact() == ([], [])
        check()
        # A row has room for `headroom` steps: the ones that are out of it finish, and some others.
        again = [b for b in range(8) if pb.rows[b].length == len(pb.rows[b].blocks) * bs or rng.random() < 0.2]
        pb.rotate(again)
        for b in again:
            fill(b)


def test_fork_refusals_and_byte_accounting():
    pb = PrefixBatch(batch=4, groups=2, prefix_tokens=8, lo=10, hi=10, block_size=4, num_blocks=40, headroom=4,
                     lengths=[18, 10, 11, 12])
    for row, slots in ((0, [0]), (0, [1, 1]), (0, [2]), (3, [1])):
        with pytest.raises(ValueError):
            pb.fork(row, slots)
    assert pb.fork(0, []) == ([], [])
    src, dst = pb.fork(0, [1])
    assert len(src) == 1 and src[0] == pb.rows[0].blocks[4] and dst[0] == pb.rows[1].blocks[4]
    assert pb.rows[0].blocks[:4] == pb.rows[1].blocks[:4] and pb.rows[0].shared == pb.rows[1].shared == 4
    # 16 tokens of rows 0 and 1 are stored once and 2 twice; rows 2 and 3 share 8, and hold 3 and 4 more.
    assert pb.unique_tokens() == 16 + 2 + 2 + 8 + 3 + 4 and pb.logical_tokens() == 18 + 18 + 11 + 12
    src, dst = pb.fork(3, [2])  # length 12: no partial block, nothing to copy
    assert (src, dst) == ([], []) and pb.rows[2].blocks[:3] == pb.rows[3].blocks[:3]


def test_fork_names_rows_from_zero():
    pb = PrefixBatch(batch=4, groups=1, prefix_tokens=0, lo=9, hi=9, block_size=4, num_blocks=40, headroom=4)
    before = [list(r.blocks) for r in pb.rows]
    for row, slots in ((-1, [3]), (3, [-1]), (0, [4]), (4, [0])):  # row -1 would be row 3 itself
        with pytest.raises(ValueError):
            pb.fork(row, slots)
    assert [r.blocks for r in pb.rows] == before
    _whole(pb, 40)


def test_fork_of_a_row_that_used_its_headroom_fits_the_tables():
    pb = PrefixBatch(batch=2, groups=1, prefix_tokens=0, lo=10, hi=10, block_size=4, num_blocks=16, headroom=6)
    pb.advance(5)  # 15 of the 16 tokens that a table row has room for
    pb.fork(0, [1])
    assert pb.tables.shape == (2, 4) and [len(r.blocks) for r in pb.rows] == [4, 4]
    _whole(pb, 16)
    pb.advance()
    assert pb.fork(1, [0]) == ([], []) and pb.rows[0].blocks == pb.rows[1].blocks  # full: nothing of its own
    with pytest.raises(RuntimeError):
        pb.advance()


def test_fork_without_room_changes_nothing():
    pb = PrefixBatch(batch=3, groups=1, prefix_tokens=0, lo=9, hi=9, block_size=4, num_blocks=10, headroom=4,
                     lengths=[9, 1, 1])
    assert [len(r.blocks) for r in pb.rows] == [4, 2, 2] and pb.alloc.free_blocks == 2
    pb.fork(0, [1, 2])  # 2 of their own each, out of 2 free and 4 given back
    assert pb.alloc.free_blocks == 2
    _whole(pb, 10)
    tight = PrefixBatch(batch=3, groups=1, prefix_tokens=0, lo=1, hi=9, block_size=4, num_blocks=6, headroom=4,
                        lengths=[9, 0, 0])
    state = [list(r.blocks) for r in tight.rows], list(tight.alloc._free)
    with pytest.raises(RuntimeError):
        tight.fork(0, [1, 2])
    assert ([list(r.blocks) for r in tight.rows], list(tight.alloc._free)) == state
    _whole(tight, 6)
