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


# Shapes whose first launch takes fewer nodes than the trees have (4 million logits of them, 12 of both kinds): the walk passes
# over the others with its workgroups together. b, t, v, draft, dtype, reach (1: chains), every which row is greedy (0: none).
BEYOND = [
    (8, 12, 128256, True, torch.float32, 2, 3),
    (8, 12, 128256, False, torch.float32, 3, 3),
    (8, 12, 128256, False, torch.bfloat16, 1, 1),
    (32, 6, 128256, True, torch.float16, 2, 4),
    (32, 6, 128256, False, torch.float16, 2, 4),
    (32, 6, 128256, False, torch.float16, 1, 1),
    (32, 6, 128256, False, torch.float32, 5, 0),
    (2, 70, 151936, True, torch.bfloat16, 2, 0),
    (2, 70, 100003, False, torch.float16, 4, 2),
    (600, 3, 8193, False, torch.float16, 1, 2),   # one workgroup a row
    (600, 5, 4099, True, torch.float16, 2, 3),
    (70, 40, 2049, False, torch.float32, 2, 3),   # slices of 1032 logits
    (1, 400, 151936, False, torch.float16, 3, 0),
]


def _likely_paths(seed, b, t, v, dtype, draft, reach, greedy):
    """Rows whose paths are long: a node's last child has the token that its target (draft) prefers, the ones before it likely
    ones that are refused often."""
    g = torch.Generator().manual_seed(seed)
    parents = [[-1] + [int(torch.randint(max(0, i - reach), i, (1,), generator=g)) for i in range(1, t)] for _ in range(b)]
    if t > 12:  # every reach-th node goes on, the others have no children
        parents = [[-1] + [(i - 1) // reach * reach for i in range(1, t)]] * b
    logits = (3 * torch.randn(b, t, v, generator=g)).to(dtype)
    q = (logits.float() + 0.5 * torch.randn(b, t, v, generator=g)).to(dtype) if draft else None
    temps = 0.2 + 0.3 * torch.rand(b, generator=g)
    if greedy:
        temps[::greedy] = 0.0
    tokens, u = torch.zeros(b, t, dtype=torch.int64), torch.rand(b, t, generator=g)
    top = (logits if q is None else q).float().topk(2, dim=-1).indices
    if draft and t > 12:  # of the likely ones those which the draft underrates and overrates most
        many = q.float().topk(8, dim=-1).indices
        over = q.float().gather(2, many) - logits.float().gather(2, many)
        top = many.gather(2, torch.stack((over.argmin(dim=-1), over.argmax(dim=-1)), dim=2))
    for row in range(b):
        last = {p: i for i, p in enumerate(parents[row])}
        for i in range(1, t):
            p = parents[row][i]
            tokens[row, i] = top[row, p, 0 if last[p] == i else 1]
            if last[p] == i:
                u[row, i] *= 0.5 if t <= 12 else 0.02
            elif t > 12:
                u[row, i] = 0.9 + 0.09 * u[row, i]
    return parents, logits, q, tokens, u, temps


@pytest.mark.parametrize("case", range(len(BEYOND)))
def test_nodes_beyond_the_first_launch(case):
    from runtime_amd.phase2.speculative import DraftTree, verify_draft
    from oracle import speculative as oracle

    b, t, v, draft, dtype, reach, greedy = BEYOND[case]
    # The workspace holds a place for every node of the first launch, so it grows with T up to their number.
    size = [_hip.verify_draft_workspace_bytes(b, n, v, int(draft)) for n in range(1, t + 1)]
    first = 1 + size.index(size[-1])
    assert first < t
    parents, logits, q, tokens, u, temps = _likely_paths(case, b, t, v, dtype, draft, reach, greedy)
    counts = torch.full((b,), t, dtype=torch.int32)
    if b > 1:
        counts[1::5] = t - 1
        counts[min(3, b - 1)] = 0
    tree = DraftTree.from_parents(parents, DEV, counts=counts)
    got = [x.cpu() for x in verify_draft(logits.to(DEV), tokens.to(DEV), tree, u.to(DEV), temps.to(DEV),
                                         draft_logits=None if q is None else q.to(DEV))]
    deepest = 0
    for row in range(b):
        kept, following = oracle.verify_row(_Rows(logits[row]), tokens[row].tolist(), parents[row], int(counts[row]),
                                            u[row].tolist(), float(temps[row]), None if q is None else _Rows(q[row]))
        want = [int(tokens[row, i]) for i in kept[1:]] + ([] if following is None else [following])
        assert got[2][row].tolist() == kept + [-1] * (t - len(kept)), row
        assert got[0][row].tolist() == want + [-1] * (t - len(want)), row
        assert int(got[1][row]) == len(kept)
        deepest = max(deepest, kept[-1] if kept else 0)
    assert deepest >= first, "no path reached the nodes beyond"


class _Rows:
    """Logits of a row's nodes in 64 bits, one at a time."""

    def __init__(self, x):
        self.x = x

    def __getitem__(self, i):
        return self.x[i].double().numpy()


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("draft", [False, True])
def test_nodes_without_a_distribution_beyond_the_first_launch(draft, temperature):
    """What makes a node of a later pass end its row: a NaN, nothing above -inf, with a temperature +inf."""
    b, t, v = 8, 14, 128256
    assert _hip.verify_draft_workspace_bytes(b, t - 1, v, int(draft)) == _hip.verify_draft_workspace_bytes(b, t, v, int(draft))
    logits, parents = torch.zeros(b, t, v), list(range(-1, t - 1))
    logits[..., 99999] = 40.0
    logits[0, 12, 128255] = float("nan")
    logits[1, 11] = -float("inf")
    logits[2, 12, 3] = float("inf")
    logits[3, 11, 0] = -float("inf")          # one token less
    logits[4, 12] = -float("inf")
    logits[4, 12, 70000] = -3.0               # one token left
    tokens, u = torch.full((b, t), 99999, dtype=torch.int64), torch.full((b, t), 0.25)
    temps, q = torch.full((b,), temperature), logits.clone() if draft else None
    if draft:
        q[5, 12, 17] = float("nan")           # a draft without a distribution: its children are not kept
        q[0:3] = q[6:7]                       # (those rows' drafts have one)
        q[4] = q[6]
    want = _oracle(logits, tokens, parents, u, temps, q)
    got = _call(logits, tokens, parents, u, temps, q)
    assert (got[0].tolist(), got[2].tolist()) == want
    greedy = temperature == 0.0
    assert got[1].tolist() == [13, 12, 13, 14, 13, 13 if draft and not greedy else 14, 14, 14]
    assert [r[n - 1] for r, n in zip(got[0].tolist(), got[1].tolist())] == [-1, -1, 3 if greedy else -1, 99999, 70000] + [99999] * 3


def test_wide_uniform_numbers_stay_below_1():
    """A token that is certain is kept whatever the number, also one that rounds to 1 in 32 bits."""
    from runtime_amd.phase2.speculative import DraftTree, verify_draft

    logits = torch.full((1, 3, 500), -float("inf"), device=DEV)
    logits[..., 7] = 1.0
    tokens, tree = torch.full((1, 3), 7, dtype=torch.int64, device=DEV), DraftTree.chain(3, DEV)
    u = torch.full((1, 3), 1 - 2.0 ** -40, dtype=torch.float64, device=DEV)
    for draft in (None, logits):
        out = verify_draft(logits, tokens, tree, u, 1.0, draft_logits=draft)
        assert out.tokens.tolist() == [[7, 7, 7]] and out.counts.tolist() == [3]
