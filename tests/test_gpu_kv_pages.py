"""Pages of a pool on the GPU: copies (with chains, cycles and fan-out), compaction, renamed tables, freed
pages, for the 16-bit pool's two layouts and the 8-bit pool. Bar: bit-identical (nothing is computed)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
POOLS = ["interleaved", "split", "int8"]


def _pool(kind, nb, layers=3, hkv=2, bs=16, d=64, seed=0):
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    args = dict(num_blocks=nb, block_size_tokens=bs, num_layers=layers, num_kv_heads=hkv, head_dim=d,
                dtype=torch.float16, device=DEV)
    pool = Int8KVBlockPool(**args) if kind == "int8" else GpuKVBlockPool(**args, kv_layout=kind)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for t in pool._page_regions():
        t.copy_(torch.randint(1, 250, t.shape, generator=g, device=DEV).to(t.dtype))
    return pool


def _pages(pool):
    return [t.clone() for t in pool._page_regions()]


def _check(pool, was, of):
    """Page i holds what page of.get(i, i) held."""
    index = torch.tensor([of.get(i, i) for i in range(pool.shape.num_blocks)], device=DEV)
    for now, old in zip(pool._page_regions(), was):
        assert torch.equal(now, old[:, index])


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("hkv,bs,d", [(2, 16, 64), (1, 4, 64), (8, 32, 128), (3, 8, 128)])
def test_copies_of_independent_pages(kind, hkv, bs, d):
    pool = _pool(kind, 40, hkv=hkv, bs=bs, d=d)
    was = _pages(pool)
    src, dst = [0, 0, 5, 39, 7, 9], [1, 2, 38, 3, 7, 4]
    pool.copy_blocks(src, dst)
    _check(pool, was, {d: s for s, d in zip(src, dst)})
    assert pool.allocated_block_count() == 9  # 7 -> 7 is no copy


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("src,dst", [
    ([1, 2, 3], [2, 3, 4]), ([4, 3, 2], [5, 4, 3]), ([1, 2], [2, 1]), ([1, 2, 3, 6, 5], [2, 3, 1, 5, 6]),
    ([1, 1, 2, 2], [2, 3, 4, 5]), ([1, 2, 1], [2, 1, 3]), ([0, 1, 2, 8], [1, 2, 0, 9]), ([4, 5, 6], [7, 7, 5])])
def test_copies_that_depend_on_each_other(kind, src, dst):
    pool = _pool(kind, 12)
    was = _pages(pool)
    pool.copy_blocks(src, dst)
    _check(pool, was, {d: s for s, d in zip(src, dst)})


@pytest.mark.parametrize("n", [448, 449, 1000])
def test_more_pages_than_a_launch_holds(n):
    pool = _pool("int8", 2 * n + 5, layers=2, hkv=1, bs=4)
    was = _pages(pool)
    g = torch.Generator().manual_seed(n)
    ids = torch.randperm(2 * n + 5, generator=g).tolist()
    pool.copy_blocks(ids[:n], ids[n:2 * n])
    _check(pool, was, dict(zip(ids[n:2 * n], ids[:n])))


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("n", [400, 500])
def test_a_long_chain_and_a_long_cycle(kind, n):  # within a launch, and beyond one
    pool = _pool(kind, n + 1, layers=1, hkv=1, bs=4)
    was = _pages(pool)
    pool.copy_blocks(list(range(n)), list(range(1, n + 1)))
    _check(pool, was, {i + 1: i for i in range(n)})
    was = _pages(pool)
    pool.copy_blocks(list(range(n)), [*range(1, n), 0])
    _check(pool, was, {(i + 1) % n: i for i in range(n)})


@pytest.mark.parametrize("kind", POOLS)
@pytest.mark.parametrize("n", [1, 37, 500])
def test_move_blocks_renames_tables_and_frees_the_sources(kind, n):
    nb = 3 * n + 4
    pool = _pool(kind, nb, layers=2, hkv=1, bs=4)
    was = _pages(pool)
    g = torch.Generator().manual_seed(n)
    ids = torch.randperm(nb, generator=g).tolist()
    src, dst, rest = ids[:n], ids[n:2 * n], ids[2 * n:]
    pool._touch_ids(src + rest)
    pool._used_map[torch.tensor(src, device=DEV)] = 1
    tables = torch.tensor(src + rest + src, dtype=torch.int32)[None].repeat(3, 1)
    tables[1], tables[2, 0], tables[2, -1] = tables[1].flip(0), -1, nb + 7  # ids that name no page stay
    name = dict(zip(src, dst))
    want = [[name.get(i, i) for i in row] for row in tables.tolist()]
    wide = torch.zeros(3, tables.shape[1] + 5, dtype=torch.int32, device=DEV)
    wide[:, :tables.shape[1]] = tables.to(DEV)
    view = wide[:, :tables.shape[1]]
    got = pool.move_blocks(src, dst, view)
    assert got.tolist() == want and torch.equal(view.cpu(), tables)
    _check(pool, was, {d: s for s, d in name.items()})
    assert pool.allocated_block_count() == n + len(rest) == pool.peak_allocated_block_count()
    pool.move_blocks(dst, src, got, out=got)  # back again, in place
    assert torch.equal(got.cpu()[:2], tables[:2])


@pytest.mark.parametrize("kind", POOLS)
def test_freed_blocks(kind):
    pool = _pool(kind, 1100, layers=2, hkv=1, bs=4)
    was = _pages(pool)
    pool._used_map.fill_(1)
    assert pool.allocated_block_count() == 1100
    gone = list(range(0, 1000)) + [5]
    pool.free_blocks(gone)
    assert pool.allocated_block_count() == 100 and pool.peak_allocated_block_count() == 1100
    if kind == "int8":
        assert (pool._codes[:, :1000] == 0).all() and torch.equal(pool._codes[:, 1000:], was[1][:, 1000:])
        k, _ = pool.gather_layer(0, [3], 4)
        assert (k == 0).all()
    assert torch.equal(pool._page_regions()[0], was[0])


def test_copies_in_a_captured_graph_and_on_a_side_stream():
    pool = _pool("interleaved", 20)
    tables = torch.arange(20, dtype=torch.int32, device=DEV).view(2, 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        out = pool.move_blocks([11], [1], tables)
        with torch.cuda.graph(graph, stream=side):
            pool.copy_blocks([3, 4, 5], [4, 3, 6])
            pool.move_blocks([12], [2], tables, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        was = _pages(pool)
        out.zero_()
        graph.replay()
        _check(pool, was, {4: 3, 3: 4, 6: 5, 2: 12})
        assert out.tolist()[1][2] == 2 and out.tolist()[1][1] == 11
        pool.copy_blocks([i], [13 + i])
        torch.cuda.synchronize()


@pytest.mark.parametrize("kind", POOLS)
def test_refusals_leave_the_pool_as_it_was(kind):
    pool = _pool(kind, 8)
    was = _pages(pool)
    for src, dst in (([1], [1]), ([1, 1], [2, 3]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([1], [])):
        with pytest.raises(ValueError):
            pool.move_blocks(src, dst)
    for call in (lambda: pool.move_blocks([1], [8]), lambda: pool.move_blocks([-1], [2]), lambda: pool.copy_blocks([1], [8]),
                 lambda: pool.free_blocks([8]), lambda: pool.move_blocks([2**31], [1])):
        with pytest.raises(IndexError):
            call()
    tables = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    for bad in (tables.cpu(), tables.long(), tables.t(), tables[0]):
        with pytest.raises(ValueError):
            pool.move_blocks([1], [2], bad)
    with pytest.raises(ValueError):
        pool.move_blocks([1], [2], tables, out=tables[:1])
    _check(pool, was, {})
    pool.copy_blocks([], []), pool.free_blocks([])
    assert torch.equal(pool.move_blocks([], [], tables), tables)


@pytest.mark.parametrize("kind", POOLS)
def test_forked_and_compacted_rows_decode_as_before(kind):
    """``PrefixBatch`` rows that share a prefix, fork and are compacted, with the pool's copies and moves and
    attention over it: a fork decodes as its parent, and not a bit changes when blocks move."""
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool
    from runtime_amd.phase2.paged_attention_hip import PagedDecodeBatchMetadata, paged_attention_decode_batched
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool
    from runtime_amd.phase2.prefix_batch import PrefixBatch

    bs, hkv, d, layers = 16, 2, 64, 2
    pb = PrefixBatch(batch=6, groups=2, prefix_tokens=32, lo=33, hi=200, block_size=bs, num_blocks=160, headroom=20, seed=2)
    args = dict(num_blocks=160, block_size_tokens=bs, num_layers=layers, num_kv_heads=hkv, head_dim=d,
                dtype=torch.float16, device=DEV)
    pool = Int8KVBlockPool(**args) if kind == "int8" else GpuKVBlockPool(**args, kv_layout=kind)
    g = torch.Generator().manual_seed(4)
    shared = torch.randn(2, layers, 2, 1, hkv, 32, d, generator=g).half()
    for r in pb.rows:
        for li in range(layers):
            kv = torch.randn(2, 1, hkv, r.length, d, generator=g).half()
            kv[:, :, :, :32] = shared[r.group, li]
            pool.write_tokens(li, r.blocks, 0, kv[0].to(DEV), kv[1].to(DEV))
    tables, lens = torch.zeros(6, pb.max_blocks, dtype=torch.int32, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
    q = torch.randn(6, 3 * hkv, 1, d, generator=g).half().to(DEV)

    def attend(query=q):
        return [paged_attention_decode_batched(query, PagedDecodeBatchMetadata(
            pool=pool, layer_idx=li, block_tables=tables, seq_lens=lens, shared_blocks=True), 3, d ** -0.5)
            for li in range(layers)]

    pool.copy_blocks(*pb.fork(1, [0, 2]))
    pb.upload(tables, lens)
    # Forks hold the parent's tokens bit for bit. Their outputs for one query differ only by where a row is
    # cut into pieces: each is within 6 half steps of 2**-11 of the largest |v| of the exact one.
    same = q[1:2].expand(6, -1, -1, -1).contiguous()
    for li, out in enumerate(attend(same)):
        rows = [pool.gather_layer(li, r.blocks, r.length) for r in pb.rows[:3]]
        for k, v in rows:
            assert torch.equal(k, rows[1][0]) and torch.equal(v, rows[1][1])
        assert (out[[0, 2]] - out[1]).abs().max() <= 12 * 2.0 ** -11 * rows[1][1].abs().max()
        assert (out[3] - out[1]).abs().max() > 0.1
    before = attend()
    for li in range(layers):  # a step: each row's own token, beside the shared blocks
        kv = torch.randn(2, 6, hkv, 1, d, generator=g).half().to(DEV)
        pool.write_tokens_batch(li, tables, lens, kv[0], kv[1])
    for a, b in zip(before, attend()):
        assert torch.equal(a, b)  # what the rows held is untouched
    pb.advance()
    lens.add_(1)
    before = attend()
    assert not torch.equal(before[0][0], before[0][1])
    pool.free_blocks([i for i in range(160) if pb.alloc.refcount(i) == 0])
    held = pool.allocated_block_count()
    src, dst = pb.compact()
    assert len(src) > 4
    pool.move_blocks(src, dst, tables, out=tables)
    assert torch.equal(tables.cpu()[:, :2], pb.tables[:, :2])
    for a, b in zip(before, attend()):
        assert torch.equal(a, b)
    assert pool.allocated_block_count() == held
    live = {i for i in range(160) if pb.alloc.refcount(i)}
    assert live == set(range(len(live))) and pool._used_blocks <= live
    pool.check_write_errors()


@pytest.mark.parametrize("kind", POOLS)
def test_long_chains_and_cycles_in_a_captured_graph(kind):
    """More copies that depend on each other than a launch takes, a chain of 900 pages and a cycle of 1000 with
    a branch, captured and replayed: nothing is copied to the device or allocated."""
    pool = _pool(kind, 2000, layers=1, hkv=1, bs=4)
    g = torch.Generator().manual_seed(7)
    ids = torch.randperm(2000, generator=g).tolist()
    chain, ring = ids[:901], ids[901:1901]
    src = [*chain[:-1], *ring, ring[500]]
    dst = [*chain[1:], *ring[1:], ring[0], ids[1950]]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        pool.copy_blocks(src, dst)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        was = _pages(pool)
        pool._used_map.zero_()
        graph.replay()
        _check(pool, was, dict(zip(dst, src)))
        assert torch.equal(pool._used_map.nonzero().flatten().cpu(), torch.tensor(sorted(dst)))
        pool.copy_blocks([3], [ids[1999]])
        torch.cuda.synchronize()
