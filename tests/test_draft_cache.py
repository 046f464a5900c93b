"""CPU checks of a batch cache under drafts: which places a draft's forward writes and what the lengths become."""

from __future__ import annotations

import ctypes

import pytest
import torch

from runtime_amd.phase2 import _hip
from runtime_amd.phase2.paged_attention_hip import get_paged_decode_batch_metadata, set_paged_decode_batch_metadata
from runtime_amd.phase2.paged_kv_cache import BlockPagedBatchCache
from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool
from runtime_amd.phase2.speculative import DraftTree

HKV, D, BS, LAYERS, BLOCKS = 2, 8, 4, 2, 16


class _Cfg:
    num_hidden_layers = LAYERS


@pytest.fixture(autouse=True)
def _clear_metadata():
    set_paged_decode_batch_metadata(None)
    yield
    set_paged_decode_batch_metadata(None)


def _setup(rows, lens):
    """A filled pool, and a cache of rows with these blocks and lengths."""
    pool = GpuKVBlockPool(num_blocks=BLOCKS, block_size_tokens=BS, num_layers=LAYERS, num_kv_heads=HKV, head_dim=D,
                          dtype=torch.float32, device="cpu")
    g = torch.Generator().manual_seed(0)
    for layer in range(LAYERS):
        for view in (pool.k_layer_view(layer), pool.v_layer_view(layer)):
            view.copy_(torch.randn(view.shape, generator=g))
    width = max(len(r) for r in rows)
    tables = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32)
    return pool, BlockPagedBatchCache(_Cfg(), pool, block_tables=tables, seq_lens=torch.tensor(lens), block_ids_rows=rows)


def _pages(pool):
    return torch.stack([torch.stack((pool.k_layer_view(i), pool.v_layer_view(i))) for i in range(LAYERS)]).clone()


def _states(batch, t, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(batch, HKV, t, D, generator=g), torch.randn(batch, HKV, t, D, generator=g)) for _ in range(LAYERS)]


def _forward(cache, states, tree):
    cache.draft_tree = tree
    for layer, (k, v) in zip(cache.layers, states):
        layer.update(k, v)


def _expected(before, rows, lens, counts, states):
    """The pages with every row's nodes behind its context, token by token."""
    want = before.clone()
    for layer, kv in enumerate(states):
        for which, x in enumerate(kv):
            for b, row in enumerate(rows):
                for t in range(counts[b]):
                    at = lens[b] + t
                    want[layer, which, row[at // BS], :, at % BS] = x[b, :, t]
    return want


def test_nodes_past_a_rows_count_are_not_written():
    """The second row has one place left in its only block and one node: the other three would fall into block 0, the
    padding of its table, which is the first row's."""
    rows, lens, counts = [[0, 7], [5]], [4, 3], [4, 1]
    pool, cache = _setup(rows, lens)
    before, states = _pages(pool), _states(2, 4)
    _forward(cache, states, DraftTree.chain(4, "cpu", counts=torch.tensor(counts)))
    assert torch.equal(_pages(pool), _expected(before, rows, lens, counts, states))
    assert cache.seq_lens.tolist() == [8, 4]
    meta = get_paged_decode_batch_metadata()
    assert meta.block_tables.tolist() == [[0, 7], [5, -1]] and meta.block_tables.dtype == torch.int32


def test_nodes_without_a_block_of_their_row_are_refused():
    rows, lens = [[0, 7], [5]], [4, 3]
    pool, cache = _setup(rows, lens)
    before = _pages(pool)
    with pytest.raises(IndexError, match="out of range"):
        _forward(cache, _states(2, 4), DraftTree.chain(4, "cpu"))
    assert torch.equal(_pages(pool), before)


def test_rows_without_nodes_and_without_blocks():
    rows, lens, counts = [[0, 7], [], [3, 4, 9]], [5, 0, 9], [3, 0, 0]
    pool, cache = _setup(rows, lens)
    before, states = _pages(pool), _states(3, 3)
    _forward(cache, states, DraftTree.chain(3, "cpu", counts=torch.tensor(counts)))
    assert torch.equal(_pages(pool), _expected(before, rows, lens, counts, states))
    assert cache.seq_lens.tolist() == [8, 0, 9]
    cache.keep_drafted(torch.tensor([[0, 2, -1], [-1] * 3, [-1] * 3]), torch.tensor([2, 0, 0]))
    assert cache.seq_lens.tolist() == [7, 0, 9] and cache.layers[1]._row_seq_lens.tolist() == [7, 0, 9]


def test_drafts_follow_rows_whose_blocks_change():
    rows, lens = [[1, 2], [3]], [4, 2]
    pool, cache = _setup(rows, lens)
    _forward(cache, _states(2, 2), DraftTree.chain(2, "cpu"))
    cache.keep_drafted(torch.tensor([[0, 1], [0, 1]]), torch.tensor([2, 2]))
    cache.draft_tree = None
    cache.sync_block_ids_row(1, [3, 8, 6])
    before, states = _pages(pool), _states(2, 2, seed=2)
    _forward(cache, states, DraftTree.chain(2, "cpu"))
    assert torch.equal(_pages(pool), _expected(before, [[1, 2], [3, 8, 6]], [6, 4], [2, 2], states))
    assert get_paged_decode_batch_metadata().block_tables.tolist() == [[1, 2, -1], [3, 8, 6]]


def test_plain_writes_keep_the_tables_as_they_are():
    _, cache = _setup([[0, 7], [5]], [4, 3])
    for layer, (k, v) in zip(cache.layers, _states(2, 1)):
        layer.update(k, v)
    assert get_paged_decode_batch_metadata().block_tables.tolist() == [[0, 7], [5, 0]]


def test_batched_writes_with_counts():
    rows, lens, counts = [[1, 2], [3, 4], [5, 6]], [1, 3, 6], [3, 0, 2]
    pool, cache = _setup(rows, lens)
    before, states = _pages(pool), _states(3, 3)
    for layer, (k, v) in enumerate(states):
        pool.write_tokens_batch(layer, cache.block_tables, cache.seq_lens, k, v, counts=torch.tensor(counts))
    assert torch.equal(_pages(pool), _expected(before, rows, lens, counts, states))
    # counts below 0 and above the tokens are none and all of them
    pool.write_tokens_batch(0, cache.block_tables, torch.tensor([0, 0, 0]), *states[1], counts=torch.tensor([-2, 9, 0]))
    assert torch.equal(pool.k_layer_view(0)[3, :, :3], states[1][0][1])
    with pytest.raises(ValueError, match="counts"):
        pool.write_tokens_batch(0, cache.block_tables, cache.seq_lens, *states[0], counts=torch.tensor([1, 2]))


def test_append_with_counts_refuses_bad_arguments_before_it_launches():
    lib = _hip.load()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    v = dict(k=at, v=at, sb=512, sh=256, st=64, B=1, T=2, Hkv=2, D=64, bt=at, bt_sb=2, mb=2, start=at, counts=at, kp=at, vp=at,
             sblk=2048, shead=1024, bs=16, nb=4, err=None, used=None, stream=None)

    def call(**spoil):
        return lib.mx_kv_append_counts(*(v | spoil).values())

    for name in ("k", "v", "bt", "start", "counts", "kp", "vp"):
        assert call(**{name: None}) == _hip.MX_ERR_NULL
    for spoil in (dict(B=-1), dict(T=-1), dict(D=60), dict(nb=0), dict(mb=0)):
        assert call(**spoil) == _hip.MX_ERR_INVALID, spoil
    assert call(k=at + 2) == call(st=60) == _hip.MX_ERR_ALIGNMENT
    assert call(B=0, counts=None) == call(T=0) == _hip.MX_OK


@pytest.mark.parametrize("graph_safe", [False, True])
def test_counts_outside_the_tree_count_as_none_and_all(graph_safe):
    """As in the kernels: the length of a row grows by the nodes that it has."""
    rows, lens, counts = [[1, 2], [3, 4], [5, 6], [7, 8]], [2, 5, 3, 0], [0, -1, 3, 9]
    pool, cache = _setup(rows, lens)
    cache._graph_safe = graph_safe
    before, states = _pages(pool), _states(4, 2)
    _forward(cache, states, DraftTree.chain(2, "cpu", counts=torch.tensor(counts)))
    assert torch.equal(_pages(pool), _expected(before, rows, lens, [0, 0, 2, 2], states))
    assert cache.seq_lens.tolist() == [2, 5, 5, 2]
    assert all(layer._row_seq_lens.tolist() == [2, 5, 5, 2] for layer in cache.layers)
    assert get_paged_decode_batch_metadata().seq_lens.tolist() == [2, 5, 5, 2]


@pytest.mark.parametrize("counts", [[0, 3], [2, -1]])
def test_speculative_decode_refuses_rows_without_a_node(counts):
    """Such a row keeps nothing and would be drafted for ever. Refused ahead of the prefill: no model is asked."""
    from runtime_amd.phase2.hf_decode import speculative_decode

    pool = GpuKVBlockPool(num_blocks=8, block_size_tokens=4, num_layers=1, num_kv_heads=1, head_dim=8, dtype=torch.float32,
                          device="cpu")
    prompts = [torch.tensor([1, 2])] * 2
    with pytest.raises(ValueError, match="at least 1"):
        speculative_decode(None, pool, prompts, [[0, 1, 2], [3, 4, 5]], 2, DraftTree.chain(3, "cpu", counts=torch.tensor(counts)))
    with pytest.raises(ValueError, match="does not fit"):
        speculative_decode(None, pool, prompts, [[0, 1, 2], [3, 4, 5]], 2, DraftTree.from_parents([[-1, 0, 0]] * 3, "cpu"))


def test_host_drafts_are_refused():
    """On the host nothing attends over the pool: the nodes would see each other alone."""
    from oracle import model as om
    from runtime_amd.phase2.block_paged_attention import block_paged_attention_forward
    from runtime_amd.phase2.hf_decode import enable_block_paged_attention, paged_draft_step

    model = om.random_llama(seed=0, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                            intermediate_size=64, vocab_size=64, max_position_embeddings=64, head_dim=16)
    enable_block_paged_attention(model)
    pool = GpuKVBlockPool(num_blocks=8, block_size_tokens=4, num_layers=2, num_kv_heads=2, head_dim=16,
                          dtype=torch.float32, device="cpu")
    cache = BlockPagedBatchCache(model.config, pool, block_tables=torch.tensor([[1, 2]]), seq_lens=torch.tensor([3]),
                                 block_ids_rows=[[1, 2]])
    tokens, tree = torch.tensor([[5, 6]]), DraftTree.chain(2, "cpu")
    with pytest.raises(ValueError, match="16-bit pool on a ROCm device"):
        paged_draft_step(model, cache, tokens, tree)
    assert cache.seq_lens.tolist() == [3] and cache.draft_tree is None
    # ... and in the hook, for a model that is called by hand
    cache.draft_tree = tree
    with torch.no_grad(), pytest.raises(ValueError, match="device tensor"):
        model(input_ids=tokens, position_ids=tree.position_ids(cache.seq_lens), past_key_values=cache, use_cache=True)
    meta = get_paged_decode_batch_metadata()
    assert meta.tree is tree
    q = torch.zeros(1, 4, 2, 16)
    with pytest.raises(ValueError, match="device tensor"):
        block_paged_attention_forward(torch.nn.Module(), q, q[:, :2], q[:, :2], None, 0.25)


def test_a_plain_forward_follows_a_draft():
    """After a draft that was kept in part, and after one that was kept whole without a word; what is not kept any more
    cannot be kept later."""
    rows = [[1, 2, 3], [4, 5, 6]]
    pool, cache = _setup(rows, [2, 5])
    tree = DraftTree.from_parents([-1, 0, 0], "cpu")
    _forward(cache, _states(2, 3), tree)
    cache.draft_tree = None  # as paged_draft_step leaves it
    cache.keep_drafted(torch.tensor([[0, 2, -1], [0, -1, -1]]), torch.tensor([2, 1]))
    assert cache.seq_lens.tolist() == [4, 6]
    for layer, (k, v) in zip(cache.layers, _states(2, 1)):
        layer.update(k, v)
    assert cache.seq_lens.tolist() == [5, 7] and get_paged_decode_batch_metadata().tree is None
    _forward(cache, _states(2, 2), DraftTree.chain(2, "cpu"))
    cache.draft_tree = None
    for layer, (k, v) in zip(cache.layers, _states(2, 1)):
        layer.update(k, v)
    assert cache.seq_lens.tolist() == [8, 10]
    with pytest.raises(RuntimeError, match="follows"):
        cache.keep_drafted(torch.tensor([[0, 1]] * 2), torch.tensor([1, 1]))


@pytest.mark.parametrize("graph_safe", [False, True])
def test_a_draft_can_be_dropped_midway(graph_safe):
    pool, cache = _setup([[1, 2], [3, 4]], [2, 5])
    cache._graph_safe = graph_safe
    cache.draft_tree = DraftTree.chain(3, "cpu")
    cache.layers[0].update(*_states(2, 3)[0])
    assert cache.seq_lens.tolist() == [5, 8]
    cache.drop_drafted()
    cache.drop_drafted()
    assert cache.seq_lens.tolist() == [2, 5] and all(x._row_seq_lens.tolist() == [2, 5] for x in cache.layers)
    with pytest.raises(RuntimeError, match="follows"):
        cache.keep_drafted(torch.tensor([[0, 1, 2]] * 2), torch.tensor([1, 1]))
