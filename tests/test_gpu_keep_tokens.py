"""``GpuKVBlockPool.keep_tokens``: a path of drafted tokens moved behind the context in every layer, exactly."""

from __future__ import annotations

import pytest
import torch

from oracle import speculative as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _pool(layers, hkv, d, bs, nb, dtype=torch.float16, layout="interleaved", seed=0):
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    pool = GpuKVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=layers, num_kv_heads=hkv, head_dim=d, dtype=dtype,
                          device=DEV, kv_layout=layout)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(layers, nb, hkv, bs, d, generator=g).to(dtype) for _ in range(2))
    for i in range(layers):
        pool.k_layer_view(i).copy_(k[i])
        pool.v_layer_view(i).copy_(v[i])
    return pool, k, v


def _state(pool):
    n = pool.shape.num_layers
    return (torch.stack([pool.k_layer_view(i) for i in range(n)]).cpu(),
            torch.stack([pool.v_layer_view(i) for i in range(n)]).cpu())


def _tables(rows, width, nb, seed=1):
    return torch.randperm(nb, generator=torch.Generator().manual_seed(seed))[:rows * width].to(torch.int32).view(rows, width)


def _paths(paths, t):
    out = torch.full((len(paths), t), -1, dtype=torch.int32)
    for row, p in enumerate(paths):
        out[row, :len(p)] = torch.tensor(p, dtype=torch.int32)
    return out


CASES = [
    (1, 1, 64, 4, torch.float16, "interleaved"),
    (3, 2, 128, 16, torch.bfloat16, "split"),
    (5, 8, 128, 32, torch.float16, "interleaved"),
    (2, 12, 64, 8, torch.bfloat16, "interleaved"),
    (2, 3, 40, 16, torch.float16, "split"),
    (2, 2, 64, 16, torch.float32, "interleaved"),
]


@pytest.mark.parametrize("layers,hkv,d,bs,dtype,layout", CASES)
def test_paths(layers, hkv, d, bs, dtype, layout):
    t, width = 40, 12 if bs >= 8 else 24
    paths = [[0, 1, 2, 3], [0, 2, 3, 4, 9], [0], [], [0, 39], [1, 2, 3, 4, 5], list(range(0, 40, 2)), list(range(20, 40)),
             list(range(40)), [0, 1, 3, 5, 7, 9, 11, 13, 15, 17, 18, 19, 30, 31]]
    starts = [0, 1, 5, 7, bs - 1, bs, 13, 2 * bs - 3, 3, 2 * bs]
    nb = len(paths) * width + 2
    pool, k, v = _pool(layers, hkv, d, bs, nb, dtype, layout)
    tables = _tables(len(paths), width, nb)
    lens = torch.full((len(paths),), -7, dtype=torch.int32, device=DEV)
    pool.keep_tokens(tables.to(DEV), torch.tensor(starts, device=DEV), _paths(paths, t).to(DEV),
                     torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV), lens_out=lens)
    got = _state(pool)
    assert torch.equal(got[0], oracle.keep_tokens(k, tables, starts, paths))
    assert torch.equal(got[1], oracle.keep_tokens(v, tables, starts, paths))
    assert lens.tolist() == [s + len(p) for s, p in zip(starts, paths)]
    pool.check_write_errors()


def test_paths_that_do_not_rise_and_places_outside():
    """Everything before the fault moves, nothing from there on; other rows are not touched by it."""
    bs, t, nb = 4, 10, 64
    pool, k, v = _pool(2, 2, 64, bs, nb)
    tables = _tables(5, 5, nb)
    path = torch.tensor([[0, 2, 2, 5] + [-1] * 6, [0, 3, 1, 6] + [-1] * 6, [0, 4, 12, 5] + [-1] * 6,
                         [0, 9, -1, -1] + [-1] * 6, [0, 2, 4, 6] + [-1] * 6], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 4, 4, 2, 4], dtype=torch.int32, device=DEV)
    starts = [3, 2, 0, 15, 7]  # row 3: token 15 + 9 is past its table of 20
    pool.keep_tokens(tables.to(DEV), torch.tensor(starts, dtype=torch.int32, device=DEV), path, counts)
    done = [[0, 2], [0, 3], [0, 4], [0], [0, 2, 4, 6]]
    got = _state(pool)
    assert torch.equal(got[0], oracle.keep_tokens(k, tables, starts, done))
    assert torch.equal(got[1], oracle.keep_tokens(v, tables, starts, done))
    with pytest.raises(IndexError):
        pool.check_write_errors()
    # a block id outside the pool, counts outside the path
    bad = tables.clone()
    bad[0, 1] = nb
    pool.keep_tokens(bad.to(DEV), torch.tensor([2] * 5, dtype=torch.int32, device=DEV),
                     torch.tensor([[0, 3, 4, 9] + [-1] * 6] + [[-1] * 10] * 4, dtype=torch.int32, device=DEV),
                     torch.tensor([4, 0, -5, 0, 0], dtype=torch.int32, device=DEV))
    with pytest.raises(IndexError):
        pool.check_write_errors()


def test_a_pool_on_the_cpu_does_the_same():
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    bs, t, nb, layers = 8, 12, 40, 3
    pool, k, v = _pool(layers, 2, 64, bs, nb)
    host = GpuKVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=layers, num_kv_heads=2, head_dim=64,
                          dtype=torch.float16, device="cpu")
    for i in range(layers):
        host.k_layer_view(i).copy_(k[i])
        host.v_layer_view(i).copy_(v[i])
    tables = _tables(3, 6, nb)
    args = [tables, torch.tensor([5, 0, 11]), _paths([[0, 1, 5, 6], [0, 3], [0, 2, 3, 4, 11]], t), torch.tensor([4, 2, 5])]
    lens = torch.zeros(3, dtype=torch.int32)
    host.keep_tokens(*args, lens_out=lens)
    pool.keep_tokens(*(a.to(DEV) for a in args))
    for a, b in zip(_state(pool), _state(host)):
        assert torch.equal(a, b)
    assert lens.tolist() == [9, 2, 16]


def test_captured_and_replayed():
    bs, t, nb = 16, 9, 30
    pool, k, v = _pool(4, 2, 128, bs, nb)
    tables = _tables(2, 5, nb).to(DEV)
    starts = torch.tensor([10, 30], dtype=torch.int32, device=DEV)
    path = _paths([[0, 5, 6, 8], [0, 1, 7]], t).to(DEV)
    counts = torch.tensor([4, 3], dtype=torch.int32, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        pool.keep_tokens(tables, starts, path, counts, lens_out=lens)
    paths, at = [[0, 5, 6, 8], [0, 1, 7]], [10, 30]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        k, v = (oracle.keep_tokens(x, tables.cpu(), at, paths) for x in (k, v))
        got = _state(pool)
        assert torch.equal(got[0], k) and torch.equal(got[1], v) and lens.tolist() == [a + len(p) for a, p in zip(at, paths)]
        starts.add_(1)
        at = [a + 1 for a in at]
