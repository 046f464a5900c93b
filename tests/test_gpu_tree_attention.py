"""Attention of a tree of drafted tokens over the paged cache (``paged_attention_tree``) against the 64-bit oracle.

Tolerance, per element: with u = eps / 2 of the type, the output's own rounding is u |o|; every probability is
rounded to the type (relative u) in the numerator and, as the same number, in the denominator, together at most
2 u sum(p |v|); a score is a sum of D fp32 products, off by at most D 2^-24 sum|q k| scale, another 2^-22 |score|
from the fp32 scale and the exponential's argument, which enters numerator and denominator likewise; the rest
(fp32 sums of up to 2^13 terms in trees, exp2, joins) is below 2^-16 sum(p |v|)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import speculative as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _modules():
    from runtime_amd.phase2.paged_attention_hip import PagedDecodeBatchMetadata
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool
    from runtime_amd.phase2.speculative import DraftTree, paged_attention_tree

    return PagedDecodeBatchMetadata, GpuKVBlockPool, DraftTree, paged_attention_tree


class Case:
    """A pool with filled rows, queries and a tree."""

    def __init__(self, seed, lens, t, hkv=2, group=4, d=64, bs=16, dtype=torch.float16, layout="interleaved", width=None):
        _, pool_type, _, _ = _modules()
        g = torch.Generator().manual_seed(seed)
        self.lens, self.t, self.hkv, self.group, self.d, self.bs, self.dtype = lens, t, hkv, group, d, bs, dtype
        need = [-(-max(n, 1) // bs) for n in lens]
        nb = sum(need) + 3
        self.pool = pool_type(num_blocks=nb, block_size_tokens=bs, num_layers=2, num_kv_heads=hkv, head_dim=d, dtype=dtype,
                              device=DEV, kv_layout=layout)
        perm = torch.randperm(nb, generator=g).to(torch.int32)
        self.tables = torch.zeros(len(lens), width or max(need), dtype=torch.int32)
        at = 0
        for row, n in enumerate(need):
            n = min(n, self.tables.shape[1])
            self.tables[row, :n] = perm[at:at + n]
            at += n
        self.k = torch.randn(nb, hkv, bs, d, generator=g).to(dtype)
        self.v = torch.randn(nb, hkv, bs, d, generator=g).to(dtype)
        self.q = torch.randn(len(lens), hkv * group, t, d, generator=g).to(dtype)
        self.scale = d ** -0.5

    def slot(self, row, token):
        return int(self.tables[row, token // self.bs]), token % self.bs

    def run(self, tree=None, query=None, lens=None, shared=False):
        meta_type, _, _, attend = _modules()
        self.pool.k_layer_view(1).copy_(self.k.to(DEV))
        self.pool.v_layer_view(1).copy_(self.v.to(DEV))
        meta = meta_type(pool=self.pool, layer_idx=1, block_tables=self.tables.to(DEV),
                         seq_lens=torch.tensor(self.lens, dtype=torch.int32, device=DEV) if lens is None else lens,
                         shared_blocks=shared, tree=tree)
        return attend(self.q.to(DEV) if query is None else query, meta, self.group, self.scale)

    def check(self, out, see=None, counts=None):
        want, size, reach = oracle.tree_attention(self.q, self.k, self.v, self.tables, self.lens, see, counts, self.scale)
        u = torch.finfo(self.dtype).eps / 2
        score = self.d * 2.0 ** -24 * reach + 2.0 ** -22 * reach
        tol = u * want.abs() + (2 * u + 2 * score + 2.0 ** -16) * size
        got = out.cpu().double()
        assert got.shape == want.shape
        special = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[special & ~torch.isnan(want)], want[special & ~torch.isnan(want)])
        over = torch.where(special, 0.0, (got - want).abs() - tol)
        assert float(over.max()) <= 0, f"off by {float(over.max())} more than allowed"


def _tree(parents, counts=None):
    _, _, tree_type, _ = _modules()
    return tree_type.from_parents(parents, DEV, counts=None if counts is None else torch.tensor(counts))


def _random_parents(t, rng, reach):
    return [-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, t)]


CHAINS = [
    dict(lens=[1], t=1),
    dict(lens=[3, 70, 1], t=1, d=128, group=1),
    dict(lens=[2, 9, 64, 65], t=2, bs=4),
    dict(lens=[5, 130], t=5, d=128, bs=8, dtype=torch.bfloat16),
    dict(lens=[37, 300, 17], t=17, group=3, bs=32),                   # 51 query rows
    dict(lens=[100, 41], t=41, group=2, d=128, dtype=torch.bfloat16),  # 82 rows
    dict(lens=[150, 333], t=150, group=1, hkv=3),                     # 150 rows: a tile of 256
    dict(lens=[301, 320], t=301, group=4, hkv=1, d=128),              # 1204 rows: five tiles of query rows
    dict(lens=[64, 128, 192], t=64, group=2, bs=4),
]


@pytest.mark.parametrize("case", range(len(CHAINS)))
def test_chains(case):
    c = Case(case, **CHAINS[case])
    c.check(c.run())


TREES = [
    dict(lens=[4], t=4, d=128),
    dict(lens=[7, 90, 1000], t=7, group=7, dtype=torch.bfloat16),
    dict(lens=[25, 200], t=25, d=128, bs=32),
    dict(lens=[64, 129, 511], t=64, group=4, d=128),
    dict(lens=[70, 131], t=70, group=5, hkv=1, bs=8, dtype=torch.bfloat16),
    dict(lens=[100], t=100, group=8, hkv=1),                          # 800 rows: four tiles
]


@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_trees(case, per_row):
    c = Case(100 + case, **TREES[case])
    rng = np.random.default_rng(case)
    if per_row:
        parents = [_random_parents(c.t, rng, 6) for _ in c.lens]
        see = np.stack([oracle.visible(p) for p in parents])
    else:
        parents = _random_parents(c.t, rng, 6)
        see = oracle.visible(parents)
    c.check(c.run(_tree(parents)), see)


@pytest.mark.parametrize("t,group,d", [(6, 4, 128), (20, 7, 64), (40, 8, 128)])
def test_ragged_counts_and_empty_rows(t, group, d):
    counts = [t, 0, 1, t - 2, t + 5, -1]  # clipped to 0..T
    c = Case(7, lens=[t + 90, 40, 1, t - 2, t, 0], t=t, group=group, d=d)
    parents = _random_parents(t, np.random.default_rng(t), 4)
    out = c.run(_tree(parents, counts))
    c.check(out, oracle.visible(parents), counts)
    assert not out[1].any() and not out[5].any() and not out[2, 1:].any()
    c.check(c.run(_modules()[2].chain(t, DEV, counts=torch.tensor(counts))), None, counts)


def test_masks_that_leave_rows_empty():
    """An arbitrary mask: nodes that see nothing of an empty context give zeros, on any other they see the context."""
    t = 12
    c = Case(8, lens=[t, t + 33], t=t, d=128)
    rng = np.random.default_rng(1)
    see = rng.random((2, t, t)) < 0.3
    see[:, 3] = see[:, 7] = False
    tree = _tree([[-1] + [0] * (t - 1)] * 2)
    object.__setattr__(tree, "mask", torch.from_numpy(see).to(DEV))
    out = c.run(tree)
    c.check(out, see)
    assert not out[0, 3].any() and not out[0, 7].any() and out[1, 3].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,group", [(9, 1), (9, 4), (30, 4), (70, 4)])
def test_what_masked_places_hold_has_no_effect(dtype, t, group):
    """NaN and infinities past the end, in drafted siblings and, for a node that sees them, as the formula says."""
    c = Case(9, lens=[t + 50, t], t=t, group=group, d=128, dtype=dtype)
    parents = _random_parents(t, np.random.default_rng(2), 5)
    see = oracle.visible(parents)
    for row, n in enumerate(c.lens):
        for tok in range(n, c.tables.shape[1] * c.bs if row == 0 else -(-n // c.bs) * c.bs):
            b, o = c.slot(row, tok)
            c.k[b, :, o] = float("nan")
            c.v[b, :, o] = float("inf")
    ctx = [n - t for n in c.lens]
    leaf = [i for i in range(1, t) if i not in parents]
    marks = [float("nan"), float("inf"), -float("inf")]
    for row in range(2):
        for i, node in enumerate(leaf[:4]):
            b, o = c.slot(row, ctx[row] + node)
            c.v[b, i % 2, o, 5 + 9 * i] = marks[i % 3]
        b, o = c.slot(row, ctx[row] + leaf[-1])
        c.k[b, 0, o, 3] = float("nan")
    c.check(c.run(_tree(parents)), see)


@pytest.mark.parametrize("d,group,t", [(64, 4, 200), (128, 1, 300)])
def test_infinities_in_a_chain_of_several_tiles_of_query_rows(d, group, t):
    """Nodes of a later tile of query rows see a token whole that hides from the first ones'."""
    c = Case(23, [t + 30, t + 101], t, group=group, d=d)
    for row, ctx in enumerate((30, 101)):
        for node, sign in ((5, 1), (t // 2, 1), (t - 1, 1)):
            b, o = c.slot(row, ctx + node)
            c.v[b, 0, o, 3 + node % 5] = sign * float("inf")
            c.v[b, 1, o, 60] = float("nan")
    c.check(c.run())


def test_both_infinities_in_one_sum_give_nan():
    c = Case(10, lens=[40], t=6, d=64)
    for node, x in ((1, float("inf")), (2, -float("inf"))):
        b, o = c.slot(0, 34 + node)
        c.v[b, :, o, 7] = x
    parents = [-1, 0, 1, 2, 0, 4]
    out = c.run(_tree(parents))
    c.check(out, oracle.visible(parents))
    assert torch.isnan(out[0, 2, :, 7]).all() and torch.isposinf(out[0, 1, :, 7]).all()
    assert torch.isfinite(out[0, 5]).all()


def test_large_scores_and_a_single_winner():
    """Scores of hundreds, one token a row far above the rest, and the reference maximum rising tile after tile."""
    c = Case(11, lens=[700, 133], t=5, d=128)
    c.k *= 8
    c.q *= 4
    for row in range(2):
        for tok in range(0, c.lens[row], 64):
            b, o = c.slot(row, tok)
            c.k[b, :, o] *= 1 + tok / 300
    c.check(c.run())


@pytest.mark.parametrize("lens", [[3], [20, 40], [65, 90], [300]])
@pytest.mark.parametrize("t,sign", [(1, -1), (3, -1), (3, 1)])
def test_scores_far_from_zero(lens, t, sign):
    """All scores near +-2000 (the running reference has to go there, also below 0), in rows that leave some of a
    workgroup's waves without a token."""
    c = Case(21, lens=[n + t for n in lens], t=t, d=128, group=2)
    c.k *= 0.1
    c.q *= 0.1
    c.k[..., 0] = 150.0
    c.q[..., 0] = 150.0 * sign
    c.check(c.run())


def test_a_flat_tail_under_a_large_token_keeps_its_weight():
    """4000 tokens whose probabilities are 2^-24 of the largest's: their sum counts."""
    c = Case(12, lens=[4001], t=1, d=64, hkv=1, group=1)
    c.q.zero_()
    c.q[0, 0, 0, 0] = 8.0
    c.k.zero_()
    c.v.fill_(0.0)
    b, o = c.slot(0, 0)
    c.k[b, 0, o, 0] = 24 * 0.6931471805599453
    for tok in range(1, 4001):
        b, o = c.slot(0, tok)
        c.v[b, 0, o] = 512.0
    out = c.run()
    c.check(out)
    assert float(out[0, 0, 0, 0]) > 0.1


@pytest.mark.parametrize("bs,d,dtype", [(4, 64, torch.bfloat16), (32, 128, torch.float16)])
def test_long_rows_cut_into_many_pieces(bs, d, dtype):
    c = Case(13, lens=[5000, 257, 1], t=1 if bs == 4 else 11, d=d, bs=bs, hkv=1, group=2, dtype=dtype)
    c.lens[2] = c.t
    c.check(c.run())


def test_many_short_rows():
    lens = [3 + (i * 7) % 40 for i in range(150)]
    c = Case(14, lens=lens, t=3, hkv=1, group=2, d=64)
    c.check(c.run())


@pytest.mark.parametrize("seed", range(24))
def test_random_shapes(seed):
    """Row counts, nodes, heads, lengths (0 and below the nodes too), masks, pages and types drawn together."""
    rng = np.random.default_rng(1000 + seed)
    t = int(rng.choice([1, 2, 3, 5, 9, 17, 33, 70]))
    hkv, group = int(rng.integers(1, 4)), int(rng.choice([1, 2, 3, 4, 7, 8]))
    rows = int(rng.integers(1, max(2, min(70, 2400 // (t * hkv * group)))))
    lens = [int(rng.choice([0, t, int(rng.integers(0, 80)), int(rng.integers(t, t + 700))])) for _ in range(rows)]
    c = Case(seed, lens, t, hkv=hkv, group=group, d=int(rng.choice([64, 128])), bs=int(rng.choice([4, 8, 16, 32])),
             dtype=torch.bfloat16 if rng.random() < 0.4 else torch.float16)
    counts = [int(rng.integers(-1, t + 2)) for _ in range(rows)] if rng.random() < 0.5 else None
    see = None
    tree = _modules()[2].chain(t, DEV, counts=None if counts is None else torch.tensor(counts))
    if rng.random() < 0.7:
        parents = [_random_parents(t, rng, 5) for _ in range(rows)]
        see = np.stack([oracle.visible(p) for p in parents])
        tree = _tree(parents, counts)
    c.check(c.run(tree, shared=bool(rng.random() < 0.3)), see, counts)


def test_strides_layouts_and_shared_blocks():
    c = Case(15, lens=[90, 33], t=9, d=128, layout="split")
    want = c.run()
    c.check(want)
    wide = torch.zeros(2, 9, 12, 128, dtype=c.dtype, device=DEV)
    wide[:, :, 2:10] = c.q.transpose(1, 2).to(DEV)
    assert torch.equal(c.run(query=wide[:, :, 2:10].transpose(1, 2)), want)     # [B, T, heads, D] behind the view
    odd = torch.zeros(2 * 8 * 9 * 128 + 1, dtype=c.dtype, device=DEV)[1:].view(2, 8, 9, 128)
    odd.copy_(c.q.to(DEV))
    assert torch.equal(c.run(query=odd), want)                                  # rows that are not 16-byte aligned
    assert torch.equal(c.run(shared=True), want)
    assert torch.equal(c.run(lens=torch.tensor(c.lens, device=DEV)), want)      # int64 lengths
    # rows that share their blocks
    c.tables[1] = c.tables[0]
    c.lens = [90, 90]
    c.check(c.run(shared=True))


def test_a_block_outside_the_pool_is_skipped_and_reported():
    c = Case(16, lens=[100, 80], t=4, d=64)
    c.tables[0, 2] = 10 ** 6
    c.tables[1, 4] = -3
    c.v[0] = float("nan")  # what an id taken for 0 would bring in
    keep = [i for i in range(c.tables.numel()) if int(c.tables.view(-1)[i]) == 0]
    for i in keep:
        c.tables.view(-1)[i] = 1
    c.check(c.run())
    with pytest.raises(IndexError, match="attention"):
        c.pool.check_write_errors()
    c.pool.check_write_errors()


def test_a_table_narrower_than_its_row():
    c = Case(17, lens=[200], t=4, d=64, width=6)  # 96 tokens
    c.check(c.run())


def test_a_row_shorter_than_its_nodes():
    """seq_lens below the number of nodes: the first nodes have no place and the others count from the end."""
    c = Case(18, lens=[3, 6], t=8, d=64)
    c.check(c.run())


def test_streams_and_two_graphs():
    c = Case(19, lens=[75, 300], t=13, d=128, group=4)
    parents = _random_parents(13, np.random.default_rng(3), 4)
    tree = _tree(parents)
    meta_type, _, _, attend = _modules()
    want = c.run(tree)
    c.check(want, oracle.visible(parents))
    lens = torch.tensor(c.lens, dtype=torch.int32, device=DEV)
    q, tables = c.q.to(DEV), c.tables.to(DEV)
    meta = meta_type(pool=c.pool, layer_idx=1, block_tables=tables, seq_lens=lens, tree=tree)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(2):
            attend(q, meta, c.group, c.scale)
        side.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(attend(q, meta, c.group, c.scale))
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        other = torch.cuda.Stream()
        for graph, stream in zip(graphs, (side, other)):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = attend(q, meta, c.group, c.scale)
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and all(torch.equal(o, want) for o in outs)
    # the captured call follows what the tensors hold
    lens.sub_(torch.tensor([20, 150], dtype=torch.int32, device=DEV))
    graphs[0].replay()
    torch.cuda.synchronize()
    c.lens = [55, 150]
    c.check(outs[0], oracle.visible(parents))
