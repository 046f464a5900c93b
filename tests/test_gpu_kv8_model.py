"""The native decode step over an 8-bit pool against the HF model oracle in fp32, reading the same cache.

Prompts' K and V come from the oracle; the pool quantises them. After each native step the rows are read back
(exactly the values that the cache stands for, the step's own token among them) and the oracle runs that token
with those keys and values in place of its own. What is compared is the step: projections, rotary, which slot
a token goes to, attention, MLP, lm_head. The rule is that of the 16-bit step's tests: a row's logits within
``max(1e-2, 1.25 x torch fp16's error)``, torch fp16 reading the same cache too.
"""

from __future__ import annotations

import copy

import pytest
import torch
from transformers import DynamicCache

from oracle import model as om

LOGIT_ATOL = 1e-2
YARDSTICK_SLACK = 1.25
BS, STEPS = 16, 4


class _Given(DynamicCache):
    """A cache whose layers answer an update with given keys and values."""

    given: list = []

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        super().update(key_states, value_states, layer_idx, *args, **kwargs)
        return self.given[layer_idx]


@torch.no_grad()
def _logits(model, kv, token):
    """fp32 logits after ``token``, the last of the ``kv`` [Hkv, n, D] of every layer."""
    p = next(model.parameters())
    cache = _Given(config=model.config)
    cache.given = []
    kv = [tuple(x.to(device=p.device, dtype=p.dtype)[None] for x in pair) for pair in kv]
    for li, (k, v) in enumerate(kv):
        DynamicCache.update(cache, k[:, :, :-1], v[:, :, :-1], li)
        cache.given.append((k, v))
    out = model(input_ids=torch.tensor([[int(token)]], device=p.device), past_key_values=cache, use_cache=True)
    return out.logits[0, -1].float().cpu()


def test_the_given_keys_and_values_are_what_the_oracle_reads():
    hf = om.random_qwen2(seed=6, num_hidden_layers=2, vocab_size=512)
    prompt = torch.randint(0, 512, (20,), generator=torch.Generator().manual_seed(0))
    kv, want = om.prefill_kv(hf, prompt)
    got = _logits(hf, kv, prompt[-1])
    assert (got - want).abs().max() <= 1e-3
    kv = [(k, torch.cat([v[:, 1:], v[:, :1]], dim=1)) for k, v in kv]
    assert (_logits(hf, kv, prompt[-1]) - want).abs().max() > 3 * LOGIT_ATOL


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("model,batch,lo,hi", [("qwen2", 16, 40, 200), ("qwen2", 3, 15, 40), ("llama", 4, 30, 120)])
def test_native_step_reads_what_the_cache_stands_for(model, batch, lo, hi):
    from runtime_amd.phase2.decode_step import Int8DecodeModel
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool

    dev = torch.device("cuda:0")
    make = om.random_qwen2 if model == "qwen2" else om.random_llama
    hf = make(seed=batch, num_hidden_layers=2, vocab_size=8192)
    ref = om.quantized_reference(hf, targets=om.PROJECTIONS + ("lm_head",))
    torch16 = om.to_device_dtype(copy.deepcopy(ref), dev, torch.float16).eval()
    native = Int8DecodeModel.from_hf(hf, device=dev, max_positions=512)
    s, g = native.shape, torch.Generator().manual_seed(batch)
    lens = torch.randint(lo, hi + 1, (batch,), generator=g).tolist()
    width = -(-(hi + STEPS) // BS)
    tables = torch.randperm(batch * width, generator=g).view(batch, width).int()
    pool = Int8KVBlockPool(num_blocks=batch * width, block_size_tokens=BS, num_layers=s.layers, num_kv_heads=s.kv_heads,
                           head_dim=s.head_dim, dtype=torch.float16, device=dev)
    tokens = []
    for b, n in enumerate(lens):
        kv, logits = om.prefill_kv(ref, torch.randint(0, 8192, (n,), generator=g))
        tokens.append(int(logits.argmax()))
        for li, (k, v) in enumerate(kv):
            pool.write_tokens(li, tables[b].tolist(), 0, k.half().to(dev), v.half().to(dev))
    tokens = torch.tensor(tokens, device=dev)
    seq_lens, tables_d = torch.tensor(lens, dtype=torch.int32, device=dev), tables.to(dev)
    for step in range(STEPS):
        nxt, logits = native.step(tokens, pool, tables_d, seq_lens, return_logits=True)
        logits = logits.float().cpu()
        for b, n in enumerate(lens):
            kv = [tuple(x[0].float().cpu() for x in pool.gather_layer(li, tables[b].tolist(), n + step + 1))
                  for li in range(s.layers)]
            want = _logits(ref, kv, tokens[b])
            err16 = float((_logits(torch16, kv, tokens[b]) - want).abs().max())
            err = float((logits[b] - want).abs().max())
            assert err <= max(LOGIT_ATOL, YARDSTICK_SLACK * err16), f"row {b} step {step}: {err:.3e}, torch16 {err16:.3e}"
        tokens.copy_(nxt)
    assert native.error_flag() == 0 and seq_lens.tolist() == [n + STEPS for n in lens]
