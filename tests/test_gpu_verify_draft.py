"""Verification of drafted tokens (``verify_draft``) against the 64-bit oracle. Its answers are whole numbers and must be
equal: both sides work in 64 bits, where the chance that one of the uniform numbers used here lies within rounding
(some 1e-13 of the whole) of a border is below 1e-7 for all tests together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import speculative as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _run(logits, tokens, parents, uniforms, temps, draft=None, counts=None):
    from runtime_amd.phase2.speculative import DraftTree, verify_draft

    tree = DraftTree.from_parents(parents, DEV, counts=None if counts is None else torch.tensor(counts))
    out = verify_draft(logits.to(DEV), tokens.to(DEV), tree, uniforms.to(DEV),
                       temps.to(DEV) if isinstance(temps, torch.Tensor) else temps,
                       draft_logits=None if draft is None else draft.to(DEV))
    return [x.cpu() for x in out]


def _check(got, logits, tokens, parents, uniforms, temps, draft=None, counts=None):
    b, t = tokens.shape
    x = logits.double().numpy()
    q = None if draft is None else draft.double().numpy()
    lens = []
    for row in range(b):
        tree = parents[row] if isinstance(parents[0], list) else parents
        tau = float(temps[row]) if isinstance(temps, torch.Tensor) else float(temps)
        n = t if counts is None else max(0, min(t, counts[row]))
        kept, following = oracle.verify_row(x[row], tokens[row].tolist(), tree, n, uniforms[row].tolist(), tau,
                                            None if q is None else q[row])
        emitted = [int(tokens[row, i]) for i in kept[1:]] + ([] if following is None else [following])
        assert got[2][row].tolist() == kept + [-1] * (t - len(kept)), row
        assert got[0][row].tolist() == emitted + [-1] * (t - len(emitted)), row
        assert int(got[1][row]) == len(kept)
        lens.append(len(kept))
    return lens


def _draw(seed, b, t, v, dtype, draft, greedy_every, reach=3, peak=4.0):
    """Rows whose tree's tokens are likely ones; per-row trees."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    parents = [[-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, t)] for _ in range(b)]
    logits = (torch.randn(b, t, v, generator=g) * peak).to(dtype)
    q = (logits.float() + torch.randn(b, t, v, generator=g)).to(dtype) if draft else None
    tokens = torch.randint(0, v, (b, t), generator=g)
    temps = 0.5 + torch.rand(b, generator=g)
    if greedy_every:
        temps[::greedy_every] = 0.0
    for row in range(b):
        tau = float(temps[row]) or 1.0
        for i in range(1, t):
            src = (logits if q is None else q)[row, parents[row][i]].double() / tau
            tokens[row, i] = int(torch.multinomial(torch.softmax(src, 0), 1, generator=g)) if rng.random() < 0.7 \
                else int(src.argmax())
    return parents, logits, q, tokens, torch.rand(b, t, generator=g), temps


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("b,t,v", [(1, 1, 1), (3, 4, 7), (40, 9, 50), (5, 6, 4095), (4, 5, 4096), (3, 7, 8193), (2, 12, 20011)])
def test_random_trees(b, t, v, draft, dtype):
    parents, logits, q, tokens, u, temps = _draw(b * 1000 + t + v, b, t, v, dtype, draft, 3)
    got = _run(logits, tokens, parents, u, temps, q)
    _check(got, logits, tokens, parents, u, temps, q)


@pytest.mark.parametrize("draft", [False, True])
def test_chains_with_counts_and_one_temperature(draft):
    parents, logits, q, tokens, u, _ = _draw(5, 12, 8, 301, torch.float16, draft, 0, reach=1)
    counts = [8, 1, 0, 3, -2, 20, 2, 5, 8, 8, 4, 7]
    for temp in (0.8, 0.0, torch.tensor(1.3)):
        got = _run(logits, tokens, parents[0], u, temp, q, counts)
        _check(got, logits, tokens, parents[0], u, float(temp), q, counts)


@pytest.mark.parametrize("draft", [False, True])
def test_many_children_refused_one_after_the_other(draft):
    """One node with 40 children and uniform numbers near 1, which refuse most: r is what every refusal left."""
    t, v = 41, 500
    parents, logits, q, tokens, u, temps = _draw(6, 6, t, v, torch.float32, draft, 0, peak=1.0)
    parents = [-1] + [0] * (t - 1)
    u = 0.9 + 0.0999 * u
    u[:, 0] = torch.rand(6, generator=torch.Generator().manual_seed(1))
    _check(_run(logits, tokens, parents, u, temps, q), logits, tokens, parents, u, temps, q)


def test_a_token_drafted_twice_is_refused_the_second_time():
    v = 64
    logits = torch.zeros(1, 4, v)
    tokens = torch.tensor([[0, 5, 5, 6]])
    u = torch.tensor([[0.0, 0.5, 0.0, 0.999]])  # 0 < r(5) no longer holds
    got = _run(logits, tokens, [-1, 0, 0, 0], u, 1.0)
    _check(got, logits, tokens, [-1, 0, 0, 0], u, 1.0)
    assert got[0][0].tolist() == [0, -1, -1, -1]


def test_everything_refused_leaves_the_distribution_as_it_was():
    """The children are the whole vocabulary of positive weight."""
    logits = torch.full((1, 3, 5000), float("-inf"))
    logits[0, :, 4321] = 1.0
    u = torch.tensor([[0.7, 1.5, 1.5]])  # not below 1: refused whatever r is
    tokens = torch.tensor([[0, 4321, 4321]])
    got = _run(logits, tokens, [-1, 0, 0], u, 1.0)
    assert got[0][0].tolist() == [4321, -1, -1]
    q = logits.clone()
    got = _run(logits, tokens, [-1, 0, 0], u, 1.0, q)
    assert got[0][0].tolist() == [4321, -1, -1]


def test_draft_equal_to_the_target_is_always_kept():
    parents, logits, _, tokens, u, temps = _draw(9, 8, 6, 777, torch.bfloat16, False, 0, reach=1)
    got = _run(logits, tokens, parents[0], u, temps, logits.clone())
    assert got[1].tolist() == [6] * 8


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_ties_and_signed_zeros_go_to_the_first(dtype):
    logits = torch.zeros(2, 2, 9000, dtype=dtype)
    logits[0, 0, 8000] = logits[0, 0, 4100] = logits[0, 0, 300] = 2.0
    logits[1] = -0.0
    logits[1, :, 5000] = 0.0
    tokens = torch.tensor([[0, 300], [0, 0]])
    u = torch.full((2, 2), 0.5)
    got = _run(logits, tokens, [-1, 0], u, 0.0)
    _check(got, logits, tokens, [-1, 0], u, 0.0)
    assert got[1].tolist() == [2, 2]


def test_logits_without_a_distribution():
    inf, nan = float("inf"), float("nan")
    v = 5000
    logits = torch.zeros(6, 3, v)
    logits[0, 0, 4999] = nan
    logits[1, 0] = -inf
    logits[2, 0, 17] = inf
    logits[3, 1, 4500] = nan      # the child's
    logits[4, 0, :] = -inf
    logits[4, 0, 4200] = -3.0     # one token left
    logits[5, 0, 5] = nan
    tokens = torch.tensor([[0, 1, 1]] * 3 + [[0, 1, 1], [0, 4200, 1], [0, 1, 1]])
    u = torch.zeros(6, 3)
    temps = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.0])
    got = _run(logits, tokens, [-1, 0, 1], u, temps)
    _check(got, logits, tokens, [-1, 0, 1], u, temps)
    assert got[0][:, 0].tolist() == [-1, -1, -1, 1, 4200, -1] and got[0][3, 1] == -1
    greedy_inf = torch.zeros(1, 1, v)
    greedy_inf[0, 0, 4444] = inf
    assert _run(greedy_inf, tokens[:1, :1], [-1], u[:1, :1], 0.0)[0].tolist() == [[4444]]
    # a draft without a distribution: its children are not kept and r stays
    q = torch.zeros(1, 3, v)
    q[0, 0, 9] = nan
    base = torch.randn(1, 3, v, generator=torch.Generator().manual_seed(2))
    u = torch.tensor([[0.3, 0.0, 0.0]])
    got = _run(base, tokens[:1], [-1, 0, 1], u, 1.0, q)
    _check(got, base, tokens[:1], [-1, 0, 1], u, 1.0, q)
    assert got[1].tolist() == [1]


@pytest.mark.parametrize("draft", [False, True])
def test_tokens_outside_the_vocabulary_and_extreme_uniforms(draft):
    parents, logits, q, tokens, u, temps = _draw(11, 8, 5, 1000, torch.float16, draft, 0, reach=2)
    tokens[0, 1:] = 1000
    tokens[1, 1:] = -1
    tokens[2, 1] = 2 ** 40
    u[3] = 0.0
    u[4] = 1 - 2.0 ** -24
    u[5, 0] = 0.0
    u[6, 0] = 1 - 2.0 ** -24
    got = _run(logits, tokens, parents, u, temps, q)
    _check(got, logits, tokens, parents, u, temps, q)
    u[6, 0] = 1.0  # the last token there is
    assert int(_run(logits, tokens, parents, u, temps, q)[0].max()) < 1000


@pytest.mark.parametrize("temp", [1e-30, 1e-3, 1e4, 3e38])
def test_extreme_temperatures(temp):
    parents, logits, q, tokens, u, _ = _draw(12, 6, 4, 600, torch.float32, False, 0)
    _check(_run(logits, tokens, parents, u, temp), logits, tokens, parents, u, torch.full((6,), temp))


def test_strides_and_unaligned_rows():
    parents, logits, q, tokens, u, temps = _draw(13, 3, 5, 4099, torch.float16, True, 0)
    want = _run(logits, tokens, parents, u, temps, q)
    _check(want, logits, tokens, parents, u, temps, q)
    wide = torch.zeros(5, 3, 4107, dtype=torch.float16)
    wide[:, :, 3:4102] = logits.transpose(0, 1)
    tall = torch.zeros(3, 4099, 5, dtype=torch.float16)
    tall.copy_(q.transpose(1, 2))
    got = _run(wide.to(DEV)[:, :, 3:4102].transpose(0, 1), tokens.int(), parents, u.double(), temps.double(),
               tall.to(DEV).transpose(1, 2))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_parents_on_the_device_that_are_no_tree():
    """A parent that is not before its child counts as none: the node is never reached."""
    parents, logits, q, tokens, u, temps = _draw(14, 4, 6, 90, torch.float32, False, 2)
    sane = [-1, 0, -1, 1, -1, -1]
    odd = torch.tensor([-1, 0, 2, 1, 5, 99], device=DEV)
    got = _run(logits, tokens, odd, u, temps)
    _check(got, logits, tokens, sane, u, temps)


@pytest.mark.parametrize("draft", [False, True])
def test_the_tokens_are_distributed_as_the_target(draft):
    """20,000 rows that share their logits: the first emitted token is distributed as the target's softmax (every
    count within 5 standard deviations), for a tree whose draft is a different distribution."""
    n, v, t = 20000, 12, 4
    g = torch.Generator().manual_seed(21)
    logits = torch.randn(1, t, v, generator=g).expand(n, t, v)
    q = torch.randn(1, t, v, generator=g).expand(n, t, v) if draft else None
    parents = [-1, 0, 0, 1]
    tokens = torch.zeros(n, t, dtype=torch.int64)
    if draft:
        for i in range(1, t):
            p = torch.softmax(q[0, parents[i]].double(), 0)
            tokens[:, i] = torch.multinomial(p, n, replacement=True, generator=g)
    else:
        tokens[:] = torch.tensor([0, 3, 7, 2])
    got = _run(logits, tokens, parents, torch.rand(n, t, generator=g), 1.0, q)
    want = torch.softmax(logits[0, 0].double(), 0)
    share = torch.bincount(got[0][:, 0], minlength=v).double() / n
    sigma = (want * (1 - want) / n).sqrt()
    assert bool(((share - want).abs() < 5 * sigma).all()), (share, want)
    # and the second, given a first one that was kept
    on = (got[1] >= 2) & (got[2][:, 1] == 1)
    second = torch.bincount(got[0][on, 1], minlength=v).double() / int(on.sum())
    want = torch.softmax(logits[0, 1].double(), 0)
    sigma = (want * (1 - want) / int(on.sum())).sqrt()
    assert int(on.sum()) > 500 and bool(((second - want).abs() < 5 * sigma).all())


def test_two_graphs_on_two_streams():
    from runtime_amd.phase2.speculative import DraftTree, verify_draft

    parents, logits, q, tokens, u, temps = _draw(15, 6, 7, 9001, torch.float16, True, 3)
    tree = DraftTree.from_parents(parents, DEV)
    want = _run(logits, tokens, parents, u, temps, q)
    args = [x.to(DEV) for x in (logits, tokens, u, temps, q)]
    call = lambda: verify_draft(args[0], args[1], tree, args[2], args[3], draft_logits=args[4])  # noqa: E731
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(call())
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, stream in zip(graphs, (side, other)):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = call()
        torch.cuda.synchronize()
        for out in (*outs, eager):
            assert all(torch.equal(a.cpu(), w) for a, w in zip(out, want))
    args[2].uniform_()
    graphs[0].replay()
    torch.cuda.synchronize()
    _check([x.cpu() for x in outs[0]], logits, tokens, parents, args[2].cpu(), temps, q)
