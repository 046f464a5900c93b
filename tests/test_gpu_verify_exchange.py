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
