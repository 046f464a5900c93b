"""Speculative decoding of an HF model: draft, tree attention, verification and kept paths together.

The model's margins are large (``oracle.model.margin_controlled_``: greedy tokens that fp16 cannot flip), so at
temperature 0 the tokens have to be those of ``greedy_decode``, whatever is drafted."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

from oracle import model as om

pytestmark = pytest.mark.gpu

DEV = "cuda"
STEPS = 24


@pytest.fixture(scope="module")
def setup():
    from runtime_amd.phase2.hf_decode import enable_block_paged_attention, greedy_decode
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    model = om.random_llama(seed=0, hidden_size=256, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                            intermediate_size=512, vocab_size=1024, max_position_embeddings=512, head_dim=64)
    om.margin_controlled_(model, seed=0)
    model = om.to_device_dtype(copy.deepcopy(model), torch.device(DEV), torch.float16).eval()
    enable_block_paged_attention(model)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 1024, (n,), generator=g) for n in (5, 33, 17, 64)]

    def pool():
        return GpuKVBlockPool(num_blocks=64, block_size_tokens=16, num_layers=2, num_kv_heads=2, head_dim=64,
                              dtype=torch.float16, device=DEV)

    perm = torch.randperm(64, generator=g).tolist()
    blocks = [perm[16 * i:16 * i + 16] for i in range(4)]
    want = greedy_decode(model, pool(), prompts, blocks, STEPS).tolist()
    return model, pool, prompts, blocks, want


def _tree_with_the_answer(rows, prompts, want, parents, rng, hit):
    """Nodes' tokens: random ones, and where `hit` says so the greedy continuation along a random path."""
    out = []
    for row, prompt, answer in zip(rows, prompts, want):
        at = len(row) - len(prompt)
        tokens = [int(t) for t in rng.integers(0, 1024, len(parents))]
        tokens[0] = row[-1]
        node, k = 0, 0
        while True:
            children = [i for i in range(len(parents)) if parents[i] == node]
            if not children or at + k >= len(answer) or not hit(k):
                break
            node = int(rng.choice(children))
            tokens[node] = answer[at + k]
            k += 1
        out.append(tokens)
    return out


@pytest.mark.parametrize("kind", ["lookup", "chain", "tree", "wrong", "rows"])
def test_greedy_tokens_whatever_is_drafted(setup, kind):
    from runtime_amd.phase2.hf_decode import speculative_decode
    from runtime_amd.phase2.speculative import DraftTree

    model, make_pool, prompts, blocks, want = setup
    rng = np.random.default_rng(5)
    parents = {"chain": [-1, 0, 1, 2], "tree": [-1, 0, 0, 0, 1, 1, 2, 3, 3, 4, 6], "wrong": [-1, 0, 1],
               "rows": [-1, 0, 0, 1, 2, 2, 4]}.get(kind)
    if kind == "lookup":
        tokens, forwards = speculative_decode(model, make_pool(), prompts, blocks, STEPS, 5)
    else:
        tree = DraftTree.from_parents([parents] * 4 if kind == "rows" else parents, DEV)
        hit = (lambda k: False) if kind == "wrong" else (lambda k: rng.random() < 0.8)
        tokens, forwards = speculative_decode(
            model, make_pool(), prompts, blocks, STEPS, tree,
            lambda rows: _tree_with_the_answer(rows, prompts, want, parents, rng, hit))
    assert tokens == want
    assert forwards <= STEPS and (kind in ("wrong", "lookup") or forwards < STEPS * 3 // 4)


def test_ragged_trees(setup):
    """Rows with fewer nodes than the batch's tree."""
    from runtime_amd.phase2.hf_decode import speculative_decode
    from runtime_amd.phase2.speculative import DraftTree

    model, make_pool, prompts, blocks, want = setup
    rng = np.random.default_rng(6)
    parents = [-1, 0, 0, 1, 2]
    tree = DraftTree.from_parents(parents, DEV, counts=torch.tensor([5, 1, 3, 4]))
    tokens, _ = speculative_decode(model, make_pool(), prompts, blocks, STEPS, tree,
                                   lambda rows: _tree_with_the_answer(rows, prompts, want, parents, rng, lambda k: True))
    assert tokens == want


def test_sampling_is_reproducible_and_its_tokens_are_likely_ones(setup):
    """A temperature, a draft model's logits (here: the model's own at random): the same generator gives the same
    tokens; every one has a probability above 2^-24 of its step's distribution (a uniform fp32 cannot pick less)."""
    from runtime_amd.phase2.hf_decode import speculative_decode

    model, make_pool, prompts, blocks, _ = setup

    def propose(rows):
        g = torch.Generator(device=DEV).manual_seed(sum(len(r) for r in rows))
        logits = torch.randn(4, 4, 1024, device=DEV, generator=g).half()
        tokens = torch.distributions.Categorical(logits=logits.float()).sample().roll(1, dims=1)
        tokens[:, 0] = torch.tensor([r[-1] for r in rows], device=DEV)
        return tokens, logits

    runs = []
    for _ in range(2):
        torch.manual_seed(7)
        g = torch.Generator(device=DEV).manual_seed(1)
        runs.append(speculative_decode(model, make_pool(), prompts, blocks, 8, 4, propose, 0.7, g)[0])
    assert runs[0] == runs[1] and all(len(r) == 9 for r in runs[0])
    for prompt, row in zip(prompts, runs[0]):
        seq = torch.cat([prompt, torch.tensor(row)])[None].to(DEV)
        with torch.no_grad():
            model.config._attn_implementation = "eager"
            logits = model(input_ids=seq).logits[0].double()
            model.config._attn_implementation = "block_paged"
        p = torch.softmax(logits / 0.7, dim=-1)
        for i, t in enumerate(row):
            assert float(p[len(prompt) - 1 + i, t]) > 2.0 ** -24


def test_refusals(setup):
    from runtime_amd.phase2.hf_decode import paged_draft_step, speculative_decode
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool
    from runtime_amd.phase2.paged_kv_cache import BlockPagedBatchCache
    from runtime_amd.phase2.speculative import DraftTree

    model, make_pool, prompts, blocks, _ = setup
    with pytest.raises(ValueError, match="blocks"):
        speculative_decode(model, make_pool(), prompts, [b[:3] for b in blocks], STEPS, 4)
    with pytest.raises(ValueError, match="16-bit"):
        speculative_decode(model, Int8KVBlockPool(num_blocks=64, block_size_tokens=16, num_layers=2, num_kv_heads=2,
                                                  head_dim=64, dtype=torch.float16, device=DEV), prompts, blocks, STEPS, 4)
    cache = BlockPagedBatchCache.empty(model.config, make_pool(), max_batch_size=2, max_blocks=4)
    with pytest.raises(ValueError, match="tree"):
        paged_draft_step(model, cache, torch.zeros(2, 3, dtype=torch.int64, device=DEV), DraftTree.chain(4, DEV))
    with pytest.raises(RuntimeError, match="follows"):
        cache.keep_drafted(torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV))


def test_tokens_outside_the_vocabulary_and_logits_without_a_distribution(setup):
    """Neither reaches the embedding."""
    from runtime_amd.phase2.hf_decode import speculative_decode

    model, make_pool, prompts, blocks, _ = setup
    for bad in (-1, 1024):
        with pytest.raises(ValueError, match="drafted tokens"):
            speculative_decode(model, make_pool(), prompts, blocks, 4, 2, lambda rows: [[r[-1], bad] for r in rows])
    kept = model.lm_head.weight.data
    try:
        model.lm_head.weight.data = torch.full_like(kept, float("nan"))
        for temperature in (0.0, 1.0):
            with pytest.raises(ValueError, match="distribution"):
                speculative_decode(model, make_pool(), prompts, blocks, 4, 2, temperature=temperature)
    finally:
        model.lm_head.weight.data = kept
