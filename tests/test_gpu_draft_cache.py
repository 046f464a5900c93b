"""A batch cache under drafts on the device: which places a draft's forward writes, exactly, and what its attention and
the kept path then read."""

from __future__ import annotations

import pytest
import torch

from runtime_amd.phase2.paged_attention_hip import get_paged_decode_batch_metadata, set_paged_decode_batch_metadata
from runtime_amd.phase2.paged_kv_cache import BlockPagedBatchCache
from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool
from runtime_amd.phase2.speculative import DraftTree, paged_attention_tree

pytestmark = pytest.mark.gpu

DEV = "cuda"
HKV, D, BS, LAYERS, BLOCKS = 2, 64, 4, 2, 16


class _Cfg:
    num_hidden_layers = LAYERS


@pytest.fixture(autouse=True)
def _clear_metadata():
    set_paged_decode_batch_metadata(None)
    yield
    set_paged_decode_batch_metadata(None)


def _setup(rows, lens, width=None):
    pool = GpuKVBlockPool(num_blocks=BLOCKS, block_size_tokens=BS, num_layers=LAYERS, num_kv_heads=HKV, head_dim=D,
                          dtype=torch.float16, device=DEV)
    g = torch.Generator().manual_seed(0)
    for layer in range(LAYERS):
        for view in (pool.k_layer_view(layer), pool.v_layer_view(layer)):
            view.copy_(torch.randn(view.shape, generator=g))
    width = width or max(len(r) for r in rows)
    tables = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32)
    return pool, BlockPagedBatchCache(_Cfg(), pool, block_tables=tables, seq_lens=torch.tensor(lens), block_ids_rows=rows)


def _pages(pool):
    return torch.stack([torch.stack((pool.k_layer_view(i), pool.v_layer_view(i))) for i in range(LAYERS)]).cpu()


def _states(batch, t, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [tuple(torch.randn(batch, HKV, t, D, generator=g).half().to(DEV) for _ in range(2)) for _ in range(LAYERS)]


def _forward(cache, states, tree):
    cache.draft_tree = tree
    for layer, (k, v) in zip(cache.layers, states):
        layer.update(k, v)


def _expected(before, rows, lens, counts, states):
    want = before.clone()
    for layer, kv in enumerate(states):
        for which, x in enumerate(kv):
            for b, row in enumerate(rows):
                for t in range(counts[b]):
                    at = lens[b] + t
                    if at // BS < len(row):
                        want[layer, which, row[at // BS], :, at % BS] = x[b, :, t].cpu()
    return want


def test_nodes_past_a_rows_count_are_not_written():
    rows, lens, counts = [[0, 7], [5], [3, 9]], [4, 3, 1], [4, 1, 0]
    pool, cache = _setup(rows, lens)
    before, states = _pages(pool), _states(3, 4)
    _forward(cache, states, DraftTree.chain(4, DEV, counts=torch.tensor(counts)))
    assert torch.equal(_pages(pool), _expected(before, rows, lens, counts, states))
    pool.check_write_errors()
    assert cache.seq_lens.tolist() == [8, 4, 1]


def test_nodes_without_a_block_of_their_row_are_dropped_and_reported():
    """They are not written into block 0, which pads the tables, nor read or moved from there."""
    rows, lens = [[0, 7], [5]], [4, 3]
    pool, cache = _setup(rows, lens)
    before, states = _pages(pool), _states(2, 4)
    _forward(cache, states, DraftTree.chain(4, DEV))
    want = _expected(before, rows, lens, [4, 4], states)
    assert torch.equal(_pages(pool), want)
    with pytest.raises(IndexError, match="batched write"):
        pool.check_write_errors()
    meta = get_paged_decode_batch_metadata()
    q = torch.randn(2, 4, 4, D, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    out = paged_attention_tree(q, meta, 2, 0.125)
    # The second row's last nodes see its 4 tokens and no more: as a row that ends there.
    k, v = (want[1, i, 5].double().repeat_interleave(2, dim=0) for i in range(2))  # [heads, 4, D]
    for node in range(1, 4):
        p = torch.softmax(torch.matmul(k, q[1, :, node].cpu().double().unsqueeze(2)).squeeze(2) * 0.125, dim=1)
        exact = (p.unsqueeze(2) * v).sum(1)
        # rounded: the output 2^-11 of it, probabilities 2^-11 twice of sum p |v|, a score 64 products of 2^-24 and 2^-22 of
        # its size at most, twice, the rest 2^-16 of that sum
        reach = torch.matmul(k.abs(), q[1, :, node].cpu().double().abs().unsqueeze(2)).max() * 0.125
        score = (64 * 2.0 ** -24 + 2.0 ** -22) * reach
        tol = 2.0 ** -11 * exact.abs() + (2.0 ** -10 + 2 * score + 2.0 ** -16) * (p.unsqueeze(2) * v.abs()).sum(1)
        assert bool(((out[1, node].cpu().double() - exact).abs() <= tol).all())
    with pytest.raises(IndexError, match="attention"):
        pool.check_write_errors()
    cache.keep_drafted(torch.tensor([[0, 1, 3, -1], [0, 3, -1, -1]], dtype=torch.int32, device=DEV),
                       torch.tensor([3, 2], dtype=torch.int32, device=DEV))
    want[:, :, 7, :, 2] = want[:, :, 7, :, 3]  # node 3 of the first row to the third place
    assert torch.equal(_pages(pool), want)
    with pytest.raises(IndexError):
        pool.check_write_errors()


def test_a_captured_draft_follows_rows_whose_blocks_change():
    rows, lens = [[1, 2], [3]], [4, 2]
    pool, cache = _setup(rows, lens, width=3)
    cache._graph_safe = True
    states = _states(2, 2)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    path = torch.tensor([[0, 1], [0, 1]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    tree = DraftTree.chain(2, DEV)

    def step():
        _forward(cache, states, tree)
        cache.keep_drafted(path, counts)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for row, start in (([3, 8], 2), ([3, 8, 6], 7), ([5, 10], 3)):
        cache.sync_block_ids_row(1, row)
        cache._set_row_length(1, start)
        torch.cuda.synchronize()
        before = _pages(pool)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(_pages(pool), _expected(before, [[1, 2], row], [4, start], [2, 2], states))
        assert cache.seq_lens.tolist() == [4, start]
        pool.check_write_errors()
    cache._set_row_length(1, 7)  # its two nodes now end one place past [5, 10]
    torch.cuda.synchronize()
    before = _pages(pool)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(_pages(pool), _expected(before, [[1, 2], [5, 10]], [4, 7], [2, 2], states))
    with pytest.raises(IndexError):
        pool.check_write_errors()


def test_a_draft_is_not_captured_before_it_has_run():
    _, cache = _setup([[1, 2]], [3])
    states, tree = _states(1, 2), DraftTree.chain(2, DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph, stream=side):
            _forward(cache, states, tree)
    torch.cuda.synchronize()
    _forward(cache, states, tree)
    assert cache.seq_lens.tolist() == [5]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_batched_writes_with_counts(dtype):
    """Per-row counts, with used blocks marked for what was written only."""
    pool = GpuKVBlockPool(num_blocks=BLOCKS, block_size_tokens=BS, num_layers=1, num_kv_heads=HKV, head_dim=D, dtype=dtype,
                          device=DEV)
    tables = torch.tensor([[1, 2], [3, 4], [5, 6], [99, 99], [7, 8]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(5, HKV, 5, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    starts, counts = torch.tensor([1, 3, 6, 0, 0], device=DEV), torch.tensor([5, -1, 2, 0, 7], device=DEV)
    pool.write_tokens_batch(0, tables, starts, k, v, counts=counts)
    for x, view in ((k, pool.k_layer_view(0)), (v, pool.v_layer_view(0))):
        want = torch.zeros(view.shape, dtype=dtype)
        for b, (start, n) in enumerate(((1, 5), (3, 0), (6, 2), (0, 0), (0, 5))):
            for t in range(n):
                want[int(tables[b, (start + t) // BS]), :, (start + t) % BS] = x[b, :, t].cpu()
        assert torch.equal(view.cpu(), want)
    pool.check_write_errors()
    assert pool.allocated_block_count() == 5
    with pytest.raises(ValueError, match="counts"):
        pool.write_tokens_batch(0, tables, starts, k, v, counts=counts[:2])


def test_attention_of_counts_outside_the_tree():
    """A count above T is T, below 0 none: the outputs are those of the clipped counts, bit for bit."""
    rows, lens = [[1, 2], [3, 4], [5, 6]], [2, 5, 3]
    q = torch.randn(3, 4, 2, D, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    outs = []
    for counts in ([5, -1, 1], [2, 0, 1]):
        pool, cache = _setup(rows, lens)
        _forward(cache, _states(3, 2), DraftTree.chain(2, DEV, counts=torch.tensor(counts)))
        assert cache.seq_lens.tolist() == [4, 5, 4]
        outs.append(paged_attention_tree(q, get_paged_decode_batch_metadata(), 2, 0.125))
    assert torch.equal(*outs) and not outs[0][1].any() and not outs[0][2, 1].any() and outs[0][0].any()


@pytest.mark.parametrize("counts", [[0, 3], [2, -1]])
def test_speculative_decode_refuses_rows_without_a_node(counts):
    from runtime_amd.phase2.hf_decode import speculative_decode

    pool, _ = _setup([[0]], [0])
    with pytest.raises(ValueError, match="at least 1"):
        speculative_decode(None, pool, [torch.tensor([1, 2])] * 2, [[0, 1, 2], [3, 4, 5]], 2,
                           DraftTree.chain(3, DEV, counts=torch.tensor(counts)))


def test_drafts_over_an_8_bit_pool_are_refused_before_they_write():
    from runtime_amd.phase2.hf_decode import paged_draft_step
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool

    pool = Int8KVBlockPool(num_blocks=4, block_size_tokens=16, num_layers=2, num_kv_heads=2, head_dim=64,
                           dtype=torch.float16, device=DEV)
    cache = BlockPagedBatchCache(_Cfg(), pool, block_tables=torch.tensor([[1, 2]]), seq_lens=torch.tensor([3]),
                                 block_ids_rows=[[1, 2]])
    with pytest.raises(ValueError, match="16-bit"):
        paged_draft_step(None, cache, torch.zeros(1, 2, dtype=torch.int64, device=DEV), DraftTree.chain(2, DEV))
    assert cache.seq_lens.tolist() == [3] and cache.draft_tree is None


@pytest.fixture(scope="module")
def model():
    import copy

    from oracle import model as om
    from runtime_amd.phase2.hf_decode import enable_block_paged_attention

    model = om.random_llama(seed=0, hidden_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                            intermediate_size=512, vocab_size=1024, max_position_embeddings=512, head_dim=64)
    om.margin_controlled_(model, seed=0)
    model = om.to_device_dtype(copy.deepcopy(model), torch.device(DEV), torch.float16).eval()
    enable_block_paged_attention(model)
    return model


def _prompts(model):
    """Two rows in a batch cache and what greedy decoding makes of them."""
    from runtime_amd.phase2.hf_decode import greedy_decode, prefill_request

    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 1024, (n,), generator=g) for n in (5, 18)]
    rows = [[9, 2, 30], [4, 7, 1]]

    def pool():
        return GpuKVBlockPool(num_blocks=32, block_size_tokens=16, num_layers=2, num_kv_heads=2, head_dim=64,
                              dtype=torch.float16, device=DEV)

    want = greedy_decode(model, pool(), prompts, rows, 12).tolist()
    mine = pool()
    caches = [prefill_request(model, mine, r, p.view(1, -1).to(DEV))[0] for p, r in zip(prompts, rows)]
    return BlockPagedBatchCache.from_caches(caches, mine), want


def test_decode_steps_between_drafts(model):
    """Greedy tokens of drafts, kept in part, and of plain steps on the same cache in turn; a draft kept whole as well."""
    from runtime_amd.phase2.hf_decode import paged_decode_step, paged_draft_step

    cache, want = _prompts(model)
    tree = DraftTree.from_parents([-1, 0, 0, 2], DEV)
    at = 0  # tokens of `want` in the cache
    for _ in range(3):
        # the second branch is the answer, the first one is not; of the answer's two nodes one is kept
        tokens = torch.tensor([[w[at], (w[at + 1] + 1) % 1024, w[at + 1], w[at + 2]] for w in want], device=DEV)
        logits = paged_draft_step(model, cache, tokens, tree)
        assert cache.draft_tree is None
        best = logits.argmax(dim=-1).tolist()
        assert all([b[0], b[2], b[3]] == w[at + 1:at + 4] for b, w in zip(best, want))
        cache.keep_drafted(torch.tensor([[0, 2, -1, -1]] * 2, dtype=torch.int32, device=DEV),
                           torch.tensor([2, 2], dtype=torch.int32, device=DEV))
        at += 2
        logits = paged_decode_step(model, cache, torch.tensor([[w[at]] for w in want], device=DEV))
        at += 1
        assert logits.argmax(dim=-1).tolist() == [w[at] for w in want]
    # a chain that stays whole
    logits = paged_draft_step(model, cache, torch.tensor([w[at:at + 2] for w in want], device=DEV), DraftTree.chain(2, DEV))
    assert logits.argmax(dim=-1).tolist() == [w[at + 1:at + 3] for w in want]
    at += 2
    logits = paged_decode_step(model, cache, torch.tensor([[w[at]] for w in want], device=DEV))
    assert logits.argmax(dim=-1).tolist() == [w[at + 1] for w in want]
    with pytest.raises(RuntimeError, match="follows"):
        cache.keep_drafted(torch.tensor([[0, 1]] * 2, dtype=torch.int32, device=DEV),
                           torch.tensor([1, 1], dtype=torch.int32, device=DEV))


def test_a_forward_that_raises_leaves_the_lengths(model):
    from runtime_amd.phase2.hf_decode import paged_decode_step, paged_draft_step

    cache, want = _prompts(model)
    lens = cache.seq_lens.tolist()
    tokens = torch.tensor([w[:2] for w in want], device=DEV)
    layer = model.model.layers[1]

    def stop(*args):
        raise KeyError("stopped behind the first layer")

    hook = layer.register_forward_pre_hook(stop)
    try:
        with pytest.raises(KeyError):
            paged_draft_step(model, cache, tokens, DraftTree.chain(2, DEV))
    finally:
        hook.remove()
    assert get_paged_decode_batch_metadata() is None and cache.draft_tree is None
    assert cache.seq_lens.tolist() == lens and all(x._row_seq_lens.tolist() == lens for x in cache.layers)
    logits = paged_decode_step(model, cache, tokens[:, :1])
    assert logits.argmax(dim=-1).tolist() == [w[1] for w in want]


def test_a_gradient_is_refused_and_not_lost():
    """Where the query asks for one; under no_grad, or for a leaf that asks for none, the call is as ever."""
    import torch.autograd.forward_ad as fwad

    _, cache = _setup([[1, 2]], [3])
    _forward(cache, _states(1, 2), DraftTree.chain(2, DEV))
    meta = get_paged_decode_batch_metadata()
    q = torch.randn(1, 4, 2, D, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    want = paged_attention_tree(q, meta, 2, 0.125)
    leaf = q.clone().requires_grad_()
    for query in (leaf, leaf * 1):
        with pytest.raises(RuntimeError, match="no gradient"):
            paged_attention_tree(query, meta, 2, 0.125)
        with torch.no_grad():
            assert torch.equal(paged_attention_tree(query, meta, 2, 0.125), want)
        with torch.inference_mode():
            assert torch.equal(paged_attention_tree(query, meta, 2, 0.125), want)
    with fwad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        paged_attention_tree(fwad.make_dual(q, torch.ones_like(q)), meta, 2, 0.125)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: paged_attention_tree(x, meta, 2, 0.125), q, check_trace=False)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: paged_attention_tree(x, meta, 2, 0.125))(q.unsqueeze(0))
    assert torch.equal(paged_attention_tree(q, meta, 2, 0.125), want)


def test_a_captured_step_drafts_verifies_and_keeps(model):
    """One graph of the whole step over a cache whose lengths advance in place, replayed with eager work between."""
    from runtime_amd.phase2.hf_decode import paged_draft_step
    from runtime_amd.phase2.speculative import verify_draft

    cache, want = _prompts(model)
    cache._graph_safe, cache._cached_seq_len_py = True, None
    tree = DraftTree.from_parents([-1, 0, 0, 2], DEV)
    tokens, u = torch.zeros(2, 4, dtype=torch.int64, device=DEV), torch.full((2, 4), 0.5, device=DEV)
    lens = cache.seq_lens.clone()

    def step():
        verdict = verify_draft(paged_draft_step(model, cache, tokens, tree), tokens, tree, u, 0.0)
        cache.keep_drafted(verdict.path, verdict.counts)
        return verdict

    def draft(at):  # the answer by the second branch; for the second row its last node is another token
        tokens.copy_(torch.tensor([[w[a], (w[a + 1] + 1) % 1024, w[a + 1], (w[a + 2] + i) % 1024]
                                   for i, (a, w) in enumerate(zip(at, want))], device=DEV))

    side = torch.cuda.Stream()
    draft([0, 0])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            verdict = step()
    torch.cuda.synchronize()
    for target in (cache, *cache.layers):
        getattr(target, "seq_lens" if target is cache else "_row_seq_lens").copy_(lens)
    at = [0, 0]
    for _ in range(3):
        draft(at)
        graph.replay()
        torch.cuda.synchronize()
        assert verdict.counts.tolist() == [3, 2] and verdict.path.tolist() == [[0, 2, 3, -1], [0, 2, -1, -1]]
        assert verdict.tokens.tolist() == [want[0][at[0] + 1:at[0] + 4] + [-1], want[1][at[1] + 1:at[1] + 3] + [-1, -1]]
        at = [at[0] + 3, at[1] + 2]
        assert cache.seq_lens.tolist() == [n + a for n, a in zip(lens.tolist(), at)]
    cache.pool.check_write_errors()
