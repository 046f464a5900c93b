"""The exchange between the workgroups that walk a row (``verify_draft``): passes over nodes beyond the first launch's,
refusals, waits that run out. Answers are whole numbers and must be those of the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

from runtime_amd.phase2 import _hip

pytestmark = pytest.mark.gpu

DEV = "cuda"
NO_WAIT = 32


def _call(logits, tokens, parents, uniforms, temps, draft=None, flags=0):
    """``mx_verify_draft`` with flags of the caller's; fp32 logits."""
    b, t, v = logits.shape
    x = [a.to(DEV).contiguous() for a in (logits, tokens, uniforms, temps)]
    d = None if draft is None else draft.to(DEV).contiguous()
    up = torch.tensor(parents, dtype=torch.int32, device=DEV)
    out = (torch.empty(b, t, dtype=torch.int64, device=DEV), torch.empty(b, dtype=torch.int32, device=DEV),
           torch.empty(b, t, dtype=torch.int32, device=DEV))
    nbytes = _hip.verify_draft_workspace_bytes(b, t, v, int(draft is not None))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    _hip.check(_hip.load().mx_verify_draft(
        x[0].data_ptr(), t * v, v, None if d is None else d.data_ptr(), t * v, v, x[1].data_ptr(), t, up.data_ptr(), 0, None,
        x[2].data_ptr(), t, x[3].data_ptr(), 1, b, t, v, *(o.data_ptr() for o in out), ws.data_ptr(), nbytes,
        16 | flags, _hip.stream_handle(out[0].device)), "mx_verify_draft")
    return [o.cpu() for o in out]


def _refused_draft(b, v):
    """Rows whose one drafted token, 0, is refused: the target gives it a half and 17000 the other, the draft nearly all."""
    logits, draft = torch.full((b, 2, v), -40.0), torch.full((b, 2, v), -40.0)
    logits[..., 0] = logits[..., 17000] = 0.0
    draft[..., 0] = 0.0
    u = torch.zeros(b, 2)
    u[:, 1] = 0.9
    return logits, draft, torch.zeros(b, 2, dtype=torch.int64), u


def test_a_refusal_whose_wait_runs_out_ends_the_row():
    """And does not go on with the distribution as it was ahead of the refusal, whose first token is the refused one."""
    b, v = 64, 20000
    logits, draft, tokens, u = _refused_draft(b, v)
    temps = torch.ones(b)
    whole = _call(logits, tokens, [-1, 0], u, temps, draft)
    assert whole[0].tolist() == [[17000, -1]] * b and whole[1].tolist() == [1] * b
    cut = _call(logits, tokens, [-1, 0], u, temps, draft, NO_WAIT)
    assert set(cut[0][:, 0].tolist()) <= {17000, -1} and bool((cut[0][:, 0] == -1).any())
    assert cut[0][:, 1].tolist() == [-1] * b and cut[1].tolist() == [1] * b and cut[2].tolist() == [[0, -1]] * b


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_a_pass_whose_wait_runs_out_ends_the_row(temperature):
    """A chain whose nodes lie beyond the first launch's: what was kept stands, then -1."""
    b, t, v = 32, 6, 128256
    assert _hip.verify_draft_workspace_bytes(b, t - 1, v, 0) == _hip.verify_draft_workspace_bytes(b, t, v, 0)
    logits = torch.zeros(1, t, v)
    logits[..., 5] = 60.0
    logits = logits.expand(b, t, v)
    tokens, u = torch.full((b, t), 5, dtype=torch.int64), torch.full((b, t), 0.5)
    parents, temps = list(range(-1, t - 1)), torch.full((b,), temperature)
    whole = _call(logits, tokens, parents, u, temps)
    assert whole[0].tolist() == [[5] * t] * b and whole[1].tolist() == [t] * b
    cut = _call(logits, tokens, parents, u, temps, flags=NO_WAIT)
    for row, n, path in zip(*(x.tolist() for x in cut)):
        assert 1 <= n <= t and path == list(range(n)) + [-1] * (t - n)
        assert row == [5] * t if n == t and row[-1] == 5 else row == [5] * (n - 1) + [-1] * (t - n + 1)
    assert bool((cut[1] < t).any())


def _oracle(logits, tokens, parents, u, temps, draft=None):
    """What the 64-bit oracle makes of each row, as verify_draft's tokens and nodes."""
    from oracle import speculative as oracle

    t = tokens.shape[1]
    rows, nodes = [], []
    for b in range(tokens.shape[0]):
        kept, following = oracle.verify_row(logits[b].double().numpy(), tokens[b].tolist(), parents, t, u[b].tolist(),
                                            float(temps[b]), None if draft is None else draft[b].double().numpy())
        out = [int(tokens[b, i]) for i in kept[1:]] + [following]
        rows.append(out + [-1] * (t - len(out)))
        nodes.append(kept + [-1] * (t - len(kept)))
    return rows, nodes


def test_more_refusals_at_a_node_than_a_word_has_numbers():
    """Passes over two nodes with 510 refusals between them: the number that marks a word comes round, so a word that a
    refusal leaves alone would pass for one of the second node's."""
    v, a, n = 20011, 400, 511
    t = a + n + 8
    assert _hip.verify_draft_workspace_bytes(1, a, v, 1) == _hip.verify_draft_workspace_bytes(1, t, v, 1)
    g = torch.Generator().manual_seed(5)
    parents = [-1] * (a + 1) + [a] * n + list(range(a + n, t - 1))
    parents[a] = 0
    logits, tokens = 3 * torch.randn(1, t, v, generator=g), torch.randint(0, v, (1, t), generator=g)
    draft = logits + torch.randn(1, t, v, generator=g)
    u = torch.rand(1, t, generator=g)
    # Node a: the target is even over the upper half of the vocabulary, the draft over the lower one, whose tokens are refused.
    logits[0, a], draft[0, a] = -10.0, -10.0
    logits[0, a, v // 2:], draft[0, a, :v // 2] = 0.0, 0.0
    tokens[0, a + 1:a + n] = torch.arange(n - 1)
    tokens[0, a + n] = v // 2 + 77
    u[0, a:a + n] = 0.9
    u[0, a] = u[0, a + n] = 0.0
    for i in range(a + n, t - 1):  # ... and its last child is kept, and some behind it
        tokens[0, i + 1] = int(draft[0, i].argmax())
    temps = torch.ones(1)
    want = _oracle(logits, tokens, parents, u, temps, draft)
    assert want[1][0][:3] == [0, a, a + n]
    got = _call(logits, tokens, parents, u, temps, draft)
    assert (got[0].tolist(), got[2].tolist()) == want


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_more_passes_than_a_word_has_numbers(temperature):
    """A chain of 1000 nodes, all kept: 209 nodes in the first launch, the others a pass of the row's workgroups each."""
    v, t = 20011, 1000
    assert _hip.verify_draft_workspace_bytes(1, 250, v, 0) == _hip.verify_draft_workspace_bytes(1, t, v, 0)
    g = torch.Generator().manual_seed(6)
    logits, parents = 3 * torch.randn(1, t, v, generator=g), list(range(-1, t - 1))
    tokens, u = torch.zeros(1, t, dtype=torch.int64), torch.rand(1, t, generator=g)
    tokens[0, 1:] = logits[0, :-1].argmax(dim=-1)
    if temperature:
        u[0, 1:990] = 0.0
    temps = torch.tensor([temperature])
    want = _oracle(logits, tokens, parents, u, temps)
    assert want[1][0][989] == 989
    got = _call(logits, tokens, parents, u, temps)
    assert (got[0].tolist(), got[2].tolist()) == want
