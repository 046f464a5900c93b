"""CPU checks of speculative decoding: the tree's shape, its refusals and those of the operators' entry points, the
64-bit oracle, a host pool's kept tokens, prompt lookup."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import speculative as oracle
from runtime_amd.phase2 import _hip
from runtime_amd.phase2.paged_attention_hip import PagedDecodeBatchMetadata
from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool
from runtime_amd.phase2.speculative import DraftTree, paged_attention_tree, verify_draft


# ---------------------------------------------------------------------------------------------
# The tree.
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("size", [1, 2, 3, 7, 16, 33, 64])
def test_tree_from_parents(size):
    rng = np.random.default_rng(size)
    for reach in (1, 2, 5, 64):
        rows = [[-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, size)] for _ in range(3)]
        tree = DraftTree.from_parents(rows, "cpu")
        assert tree.size == size and tree.parents.dtype == torch.int32
        for i, row in enumerate(rows):
            see = oracle.visible(row)
            if tree.mask is None:
                assert row == list(range(-1, size - 1))
                see_tree = np.tril(np.ones((size, size), dtype=bool))
            else:
                see_tree = tree.mask[i].numpy()
            assert (see_tree == see).all()
            depth = tree.depth[i if tree.rows > 1 else 0]
            assert depth.tolist() == (see.sum(1) - 1).tolist()
        one = DraftTree.from_parents(rows[0], "cpu")
        assert one.rows == 1 and one.position_ids(torch.tensor([4, 9])).tolist() == [
            [c + d for d in one.depth[0].tolist()] for c in (4, 9)]


def test_a_chain_needs_no_mask():
    assert DraftTree.from_parents([-1, 0, 1, 2], "cpu").mask is None
    assert DraftTree.from_parents([-1], "cpu").mask is None
    tree = DraftTree.chain(5, "cpu", counts=torch.tensor([2, 5]))
    assert tree.mask is None and tree.parents.tolist() == [[-1, 0, 1, 2, 3]] and tree.counts.dtype == torch.int32


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, -2], [-1, 0, 3], [[-1, 0], [0, 0]], [], [[]]])
def test_parents_that_are_no_tree_are_refused(parents):
    with pytest.raises(ValueError):
        DraftTree.from_parents(torch.tensor(parents, dtype=torch.int64), "cpu")


def test_other_trees_are_refused():
    with pytest.raises(TypeError):
        DraftTree.from_parents([-1.0, 0.0], "cpu")
    with pytest.raises(ValueError):
        DraftTree.chain(0, "cpu")
    with pytest.raises(ValueError):
        DraftTree.chain(3, "cpu", counts=[1, 2])
    tree = DraftTree.from_parents([[-1, 0], [-1, -1]], "cpu")
    tree.check_batch(2, 2, torch.device("cpu"))
    for batch, nodes in ((3, 2), (2, 3), (1, 2)):
        with pytest.raises(ValueError, match="does not fit"):
            tree.check_batch(batch, nodes, torch.device("cpu"))
    with pytest.raises(ValueError, match="device"):
        tree.check_batch(2, 2, torch.device("cuda:0"))
    with pytest.raises(ValueError, match="counts"):
        DraftTree.chain(2, "cpu", counts=torch.tensor([1, 2, 2])).check_batch(2, 2, torch.device("cpu"))
    bad = DraftTree(tree.parents, tree.depth, torch.zeros(2, 3, 3, dtype=torch.bool))
    with pytest.raises(ValueError, match="mask"):
        bad.check_batch(2, 2, torch.device("cpu"))


# ---------------------------------------------------------------------------------------------
# Refusals.
# ---------------------------------------------------------------------------------------------
def test_wrappers_refuse_cpu_tensors():
    pool = GpuKVBlockPool(num_blocks=4, block_size_tokens=16, num_layers=1, num_kv_heads=1, head_dim=64,
                          dtype=torch.float16, device="cpu")
    meta = PagedDecodeBatchMetadata(pool=pool, layer_idx=0, block_tables=torch.zeros(1, 2, dtype=torch.int32),
                                    seq_lens=torch.tensor([5]))
    with pytest.raises(ValueError, match="device tensor"):
        paged_attention_tree(torch.zeros(1, 1, 2, 64, dtype=torch.float16), meta, 1, 0.125)
    with pytest.raises(TypeError):
        paged_attention_tree(None, meta, 1, 0.125)
    with pytest.raises(ValueError, match="device tensor"):
        verify_draft(torch.zeros(1, 2, 10), torch.zeros(1, 2, dtype=torch.int64), DraftTree.chain(2, "cpu"),
                     torch.zeros(1, 2), 1.0)


class _Attn:
    """Arguments that ``mx_tree_attn`` takes, up to the launch; one at a time is spoilt."""

    def __init__(self):
        buf = ctypes.create_string_buffer(4096)
        self.buf, at = buf, (ctypes.addressof(buf) + 255) // 256 * 256
        self.v = dict(q=at, q_sb=512, q_sh=128, q_st=64, k=at, v=at, sblk=1024, shead=512, bt=at, bt_sb=4, max_blocks=4,
                      lens=at, mask=None, m_sb=0, m_st=0, counts=None, B=1, T=2, Hq=4, Hkv=2, D=64, bs=16, nb=4,
                      scale=0.125, out=at, o_sb=512, o_st=256, o_sh=64, ws=at, nbytes=1 << 40, err=None, flags=0,
                      stream=None)

    def call(self, **spoil):
        return _hip.load().mx_tree_attn(*(self.v | spoil).values())


def test_tree_attention_refuses_bad_arguments_before_it_launches():
    c = _Attn()
    lib = _hip.load()
    at = c.v["q"]
    for name in ("q", "k", "v", "bt", "lens", "out"):
        assert c.call(**{name: None}) == _hip.MX_ERR_NULL
    for spoil in (dict(B=-1), dict(T=-1), dict(Hq=3), dict(Hkv=0), dict(max_blocks=0), dict(nb=0), dict(flags=4),
                  dict(mask=at, m_sb=-1), dict(bt_sb=-1)):
        assert c.call(**spoil) == _hip.MX_ERR_INVALID, spoil
    for spoil in (dict(D=96), dict(D=256), dict(bs=24), dict(bs=64), dict(scale=0.0), dict(scale=-1.0),
                  dict(scale=float("nan")), dict(scale=3e38), dict(scale=float("inf")), dict(max_blocks=1 << 27),
                  dict(T=1 << 24, Hq=4)):
        assert c.call(**spoil) == _hip.MX_ERR_UNSUPPORTED, spoil
    for spoil in (dict(q=at + 8), dict(k=at + 2), dict(out=at + 4), dict(q_st=60), dict(o_sb=-64), dict(sblk=1020),
                  dict(ws=at + 8)):
        assert c.call(**spoil) == _hip.MX_ERR_ALIGNMENT, spoil
    need = lib.mx_tree_attn_workspace_bytes(1, 2, 4, 2, 64, 4, 16)
    assert need > 0
    for spoil in (dict(ws=None), dict(nbytes=need - 1)):
        assert c.call(**spoil) == _hip.MX_ERR_WORKSPACE, spoil
    assert c.call(B=0) == c.call(T=0) == _hip.MX_OK
    assert lib.mx_tree_attn_workspace_bytes(0, 2, 4, 2, 64, 4, 16) == 0
    # rows x heads x tiles past 32 bits
    assert c.call(B=1 << 20, T=1, max_blocks=1 << 20, bs=16) == _hip.MX_ERR_UNSUPPORTED


def test_verification_refuses_bad_arguments_before_it_launches():
    lib = _hip.load()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    v = dict(logits=at, l_sb=20, l_st=10, draft=None, d_sb=0, d_st=0, tokens=at, t_sb=2, parents=at, p_sb=0, counts=None,
             uniforms=at, u_sb=2, temps=at, temp_sb=0, B=1, T=2, V=10, tout=at, cout=at, pout=at, ws=at, nbytes=1 << 40,
             flags=0, stream=None)

    def call(**spoil):
        return lib.mx_verify_draft(*(v | spoil).values())

    for name in ("logits", "tokens", "parents", "uniforms", "temps", "tout", "cout", "pout"):
        assert call(**{name: None}) == _hip.MX_ERR_NULL
    for spoil in (dict(B=-1), dict(T=-1), dict(V=0), dict(flags=1), dict(flags=18), dict(l_sb=-1), dict(temp_sb=-1)):
        assert call(**spoil) == _hip.MX_ERR_INVALID, spoil
    for spoil in (dict(T=1025), dict(V=(1 << 22) + 1), dict(B=(1 << 20) + 1)):
        assert call(**spoil) == _hip.MX_ERR_UNSUPPORTED, spoil
    need = lib.mx_verify_draft_workspace_bytes(1, 2, 10, 0)
    for spoil in (dict(ws=None), dict(nbytes=need - 1)):
        assert call(**spoil) == _hip.MX_ERR_WORKSPACE, spoil
    assert call(ws=at + 8) == _hip.MX_ERR_ALIGNMENT
    assert call(B=0) == call(T=0) == _hip.MX_OK


def test_keeping_tokens_refuses_bad_arguments_before_it_launches():
    lib = _hip.load()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    v = dict(k=at, v=at, token=128, ls=4096, bs_=1024, hs=512, layers=1, Hkv=1, bs=4, nb=2, bt=at, bt_sb=2, mb=2, start=at,
             path=at, p_sb=3, counts=at + 64, B=1, T=3, lens=None, err=None, stream=None)

    def call(**spoil):
        return lib.mx_kv_keep_tokens(*(v | spoil).values())

    for name in ("k", "v", "bt", "start", "path", "counts"):
        assert call(**{name: None}) == _hip.MX_ERR_NULL
    for spoil in (dict(B=-1), dict(T=-1), dict(layers=0), dict(Hkv=0), dict(bs=0), dict(nb=0), dict(mb=0), dict(bt_sb=-1),
                  dict(p_sb=-1), dict(ls=-4096), dict(lens=at), dict(lens=at + 64)):
        assert call(**spoil) == _hip.MX_ERR_INVALID, spoil
    for spoil in (dict(token=8), dict(token=24), dict(B=65536)):
        assert call(**spoil) == _hip.MX_ERR_UNSUPPORTED, spoil
    for spoil in (dict(k=at + 8), dict(ls=8), dict(hs=4)):
        assert call(**spoil) == _hip.MX_ERR_ALIGNMENT, spoil
    assert call(B=0) == _hip.MX_OK


# ---------------------------------------------------------------------------------------------
# A pool on the host.
# ---------------------------------------------------------------------------------------------
def _host_pool(nb=12, bs=4, layers=2):
    pool = GpuKVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=layers, num_kv_heads=2, head_dim=8,
                          dtype=torch.float32, device="cpu")
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(layers, nb, 2, bs, 8, generator=g) for _ in range(2))
    for i in range(layers):
        pool.k_layer_view(i).copy_(k[i])
        pool.v_layer_view(i).copy_(v[i])
    return pool, k, v


def test_host_pool_keeps_paths():
    pool, k, v = _host_pool()
    tables = torch.tensor([[3, 1, 7, 0], [2, 5, 4, 6]])
    paths = [[0, 2, 3, 7], [1]]
    lens = torch.zeros(2, dtype=torch.int32)
    pool.keep_tokens(tables, torch.tensor([3, 6]), torch.tensor([[0, 2, 3, 7, -1, -1, -1, -1], [1] + [-1] * 7]),
                     torch.tensor([4, 1]), lens_out=lens)
    for got, was in ((pool.k_layer_view, k), (pool.v_layer_view, v)):
        want = oracle.keep_tokens(was, tables, [3, 6], paths)
        assert all(torch.equal(got(i), want[i]) for i in range(2))
    assert lens.tolist() == [7, 7]


def test_host_pool_refusals():
    pool, _, _ = _host_pool()
    tables, start = torch.tensor([[3, 1, 99]]), torch.tensor([2])
    path, counts = torch.tensor([[0, 1, 2, 3]]), torch.tensor([2])
    with pytest.raises(IndexError, match="rise"):
        pool.keep_tokens(tables, start, torch.tensor([[1, 1, 2, 3]]), counts)
    with pytest.raises(IndexError, match="rise"):
        pool.keep_tokens(tables, start, torch.tensor([[0, 4, 2, 3]]), counts)
    with pytest.raises(IndexError, match="out of range"):
        pool.keep_tokens(tables, torch.tensor([7]), torch.tensor([[0, 3, 2, 3]]), counts)
    with pytest.raises(IndexError, match="underrun"):
        pool.keep_tokens(tables, torch.tensor([11]), torch.tensor([[0, 3, 2, 3]]), counts)
    for bad in ((tables, start, path[0], counts), (tables, torch.tensor([2, 3]), path, counts),
                (tables, start, path, torch.tensor([1, 2])), (tables.float(), start, path, counts),
                (tables[0], start, path, counts)):
        with pytest.raises(ValueError):
            pool.keep_tokens(*bad)
    for lens in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="lens_out"):
            pool.keep_tokens(tables, start, path, counts, lens_out=lens)


# ---------------------------------------------------------------------------------------------
# The oracle and the drafts.
# ---------------------------------------------------------------------------------------------
def test_oracle_verification_by_hand():
    logits = np.log(np.array([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8], [0.25, 0.5, 0.25]]))
    # token 1 (r 0.3) refused at u 0.4; r = (5/7, 0, 2/7); token 0 taken at u 0.7 < 5/7; then from row 2 at u 0.6: token 1
    kept, following = oracle.verify_row(logits, [0, 1, 0], [-1, 0, 0], 3, [0.6, 0.4, 0.7], 1.0)
    assert (kept, following) == ([0, 2], 1)
    # the same at 0.72 refuses it too and leaves (0, 0, 1)
    kept, following = oracle.verify_row(logits, [0, 1, 0], [-1, 0, 0], 3, [0.6, 0.4, 0.72], 1.0)
    assert (kept, following) == ([0], 2)
    # greedy: the largest, whatever the numbers say
    kept, following = oracle.verify_row(logits, [0, 0, 2], [-1, 0, 1], 3, [0.0, 0.99, 0.99], 0.0)
    assert (kept, following) == ([0, 1, 2], 1)
    # drafted from q = (0.2, 0.2, 0.6): token 2 has r/q = 1/3; refused it leaves (0.3, 0.1, 0) / 0.4
    draft = np.log(np.array([[0.2, 0.2, 0.6]] * 3))
    kept, following = oracle.verify_row(logits, [0, 2, 2], [-1, 0, 1], 3, [0.74, 0.34, 0.0], 1.0, draft)
    assert (kept, following) == ([0], 0)
    kept, following = oracle.verify_row(logits, [0, 2, 2], [-1, 0, 1], 3, [0.76, 0.34, 0.0], 1.0, draft)
    assert (kept, following) == ([0], 1)


def test_oracle_attention_of_a_chain_is_causal_attention():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 4, 3, 16, generator=g)
    k, v = (torch.randn(4, 2, 4, 16, generator=g) for _ in range(2))
    tables = torch.tensor([[2, 0, 3]])
    out, _, _ = oracle.tree_attention(q, k, v, tables, [9], None, None, 0.25)
    keys, values = (x[[2, 0, 3]].permute(1, 0, 2, 3).reshape(2, 12, 16)[:, :9].double() for x in (k, v))
    for i in range(3):
        for h in range(4):
            p = torch.softmax(keys[h // 2, :7 + i] @ q[0, h, i].double() * 0.25, dim=0)
            assert torch.allclose(out[0, i, h], p @ values[h // 2, :7 + i], atol=1e-12)


def test_prompt_lookup():
    from runtime_amd.phase2.hf_decode import prompt_lookup

    rows = [[1, 2, 3, 4, 1, 2], [5, 5, 5], [7, 8, 9], [4]]
    assert prompt_lookup(rows, 4) == [[2, 3, 4, 1], [5, 5, 5, 5], [9, 9, 9, 9], [4, 4, 4, 4]]
    assert prompt_lookup(rows, 1) == [[2], [5], [9], [4]]
