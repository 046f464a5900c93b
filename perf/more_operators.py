"""The operators of a speculative decoding step, as cases that can be timed and compared.

A step drafts a tree of tokens for every row of a batch, runs the target model over all of them at once and
keeps the branch that the target agrees with. Three kinds of work, each in a plain form (elementary torch
operations) and through the entry points a program calls:

* ``attend`` - ``paged_attention_tree``: the ``T`` new tokens of every row, whose K and V stand behind the
  row's context in the paged cache, attend over the context and over their own ancestors in the tree (a chain
  of tokens, such as a chunk of a prompt, is the tree whose every node has one child);
* ``verify`` - ``verify_draft``: from the target's logits at every node, the drafted tokens, the temperatures
  and given uniform numbers, the path that is kept and the token that follows it;
* ``keep`` - ``GpuKVBlockPool.keep_tokens``: the K and V of the path's tokens moved, in every layer, to the
  places right behind the context.

Verification: node 0 is the last token that is already certain. The walk stands at a node whose target
distribution is ``r = softmax(logits / temperature)`` (at temperature 0 all of it at the largest logit, the
first on ties) and tries the node's children in the order of their indices. A child with token ``x`` is taken
where ``u * q(x) < r(x)``, ``u`` being its uniform number and ``q`` the distribution it was drafted from:
``softmax(draft_logits / temperature)`` at the parent, or all of it at ``x`` where there are no draft logits.
A child that is not taken leaves ``r = max(r - q, 0)``, scaled to a sum of 1 (without draft logits: ``r`` with
``x`` taken out), or ``r`` as it was where nothing remains. At a node none of whose children is taken the walk
ends and the following token is drawn from ``r``: the first whose running sum exceeds ``u0`` times the whole,
``u0`` the uniform number of node 0. Shapes are the Llama-3-8B and Qwen2-0.5B ones of ``decode_step.py``.
"""

from __future__ import annotations

import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "llm-serving-runtime_amd"))

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"
HEADS = [(8, 4, 128), (2, 7, 64), (4, 8, 128), (8, 5, 128), (12, 1, 64), (1, 8, 128)]
NEG = float("-inf")


def listed() -> list[dict]:
    return [
        # One request with a short chain of drafted tokens: latency. (branch 1: a chain; ragged: rows with fewer nodes.)
        dict(name="attend_b1_chain5", kind="attend", b=1, t=5, branch=1, ragged=False, lo=700, hi=700, hkv=8, group=4,
             d=128, bs=16, dtype="fp16"),
        # The benchmark's 32 rows of U[128, 4096] tokens, one tree of 16 nodes for all rows.
        dict(name="attend_b32_tree16", kind="attend", b=32, t=16, branch=2, ragged=False, lo=128, hi=4096, hkv=8,
             group=4, d=128, bs=16, dtype="fp16"),
        # A large tree on long rows: 256 query rows share each K and V, the matrix products count.
        dict(name="attend_b8_tree64", kind="attend", b=8, t=64, branch=3, ragged=False, lo=4096, hi=8192, hkv=8,
             group=4, d=128, bs=16, dtype="fp16"),
        # A small bf16 batch, an odd group, every row with a tree and a number of nodes of its own, pages of 32.
        dict(name="attend_b7_ragged_bf16", kind="attend", b=7, t=13, branch=0, ragged=True, lo=97, hi=1501, hkv=2,
             group=7, d=64, bs=32, dtype="bf16"),
        # One document of 131,071 tokens: few rows, a long axis to share out.
        dict(name="attend_b1_long", kind="attend", b=1, t=25, branch=3, ragged=False, lo=131071, hi=131071, hkv=8,
             group=4, d=128, bs=16, dtype="fp16"),
        # A chunk of 509 tokens of two prompts over what is cached of them.
        dict(name="attend_b2_chunk", kind="attend", b=2, t=509, branch=1, ragged=False, lo=2048, hi=4096, hkv=8,
             group=4, d=128, bs=16, dtype="bf16"),
        # One request, a chain found by prompt lookup (no draft logits), the small model's vocabulary: latency.
        dict(name="verify_b1_chain5", kind="verify", b=1, t=5, branch=1, ragged=False, vocab=151936, draft=False,
             greedy=0, dtype="fp16"),
        # The benchmark's 32 rows with trees of 16 nodes, every fourth row greedy.
        dict(name="verify_b32_tree16", kind="verify", b=32, t=16, branch=2, ragged=False, vocab=128256, draft=False,
             greedy=4, dtype="fp16"),
        # Chains sampled from a draft model whose logits are at hand, bf16, rows with chains of their own length.
        dict(name="verify_b8_draft_bf16", kind="verify", b=8, t=7, branch=1, ragged=True, vocab=128256, draft=True,
             greedy=0, dtype="bf16"),
        # Large trees on a full batch: half a gigabyte of logits, of which a row's path visits a few.
        dict(name="verify_b32_tree64", kind="verify", b=32, t=64, branch=4, ragged=False, vocab=128256, draft=False,
             greedy=4, dtype="fp16"),
        # One row of the small model: a path of 4 of 5 nodes kept in 24 layers.
        dict(name="keep_b1_small", kind="keep", b=1, t=5, layers=24, hkv=2, d=64, bs=16, hi=2048, dtype="fp16"),
        # 64 rows after trees of 64 nodes, 16 layers of the large model (one of two pipeline stages).
        dict(name="keep_b64_tree64", kind="keep", b=64, t=64, layers=16, hkv=8, d=128, bs=16, hi=4096, dtype="fp16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["attend", "attend", "attend", "verify", "verify", "keep"])
    if kind == "verify":
        vocab = rng.choice([32000, 128256, 151936, rng.randint(1000, 160000)])
        b = _log(rng, 1, 32)
        t = _log(rng, 1, max(1, min(64, 2**28 // 2 // (b * vocab))))
        return dict(kind=kind, b=b, t=t, branch=rng.choice([0, 1, 1, 2, 3, 4]), ragged=rng.random() < 0.3, vocab=vocab,
                    draft=t <= 32 and rng.random() < 0.4, greedy=rng.choice([0, 0, 1, 4]),
                    dtype=rng.choice(["fp16", "fp16", "bf16", "fp32"]))
    hkv, group, d = rng.choice(HEADS)
    c = dict(kind=kind, hkv=hkv, d=d, bs=rng.choice([4, 8, 16, 16, 32]), dtype=rng.choice(["fp16", "fp16", "bf16"]))
    if kind == "keep":
        c |= dict(b=_log(rng, 1, 64), t=_log(rng, 2, 64), layers=_log(rng, 1, 24), hi=_log(rng, 8, 4096))
        return c
    b = _log(rng, 1, 64)
    t = _log(rng, 1, max(1, min(512, 2048 // b)))
    # at most 36 GFLOP of products and 380 MB of K and V
    most = min(36e9 / (4 * b * t * hkv * group * d), 380e6 / (4 * b * hkv * d), 131071)
    hi = _log(rng, 1, max(1, int(most)))
    c |= dict(group=group, b=b, t=t, branch=1 if t > 64 else rng.choice([0, 1, 1, 2, 3, 4]),
              ragged=rng.random() < 0.3, lo=rng.randint(1, hi), hi=hi)
    return c


# ---------------------------------------------------------------------------------------------
# Inputs. Each from one generator in a fixed order, so that exact() can make the same ones.
# ---------------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32).to(DEV)


def _spread(lo: int, hi: int, b: int) -> list[int]:
    """``b`` lengths spread evenly over lo..hi: the same for every seed, so that the work is the case's."""
    return [lo + int((hi - lo) * (i + 0.5) / b) for i in range(b)]


def _trees(c: dict, seed: int) -> tuple[list[list[int]], list[int]]:
    """Parents of the nodes of each tree (one for all rows, or one a row with ``branch`` 0), in level order, and
    each row's number of nodes."""
    g = torch.Generator().manual_seed(seed + 1)
    rows = c["b"] if c["branch"] == 0 else 1
    parents = []
    for _ in range(rows):
        k = c["branch"] or int(torch.randint(1, 5, (1,), generator=g))
        jitter = torch.randint(0, 2, (c["t"],), generator=g).tolist()
        row = [-1]
        for i in range(1, c["t"]):
            near = max(0, (i - 1) // k - (jitter[i] if c["branch"] == 0 else 0))
            row.append(near if k == 1 else max(near, max(row[-1], 0)))
        parents.append(row if k > 1 else [i - 1 for i in range(c["t"])])
    counts = [c["t"]] * c["b"]
    if c["ragged"]:
        counts = _spread(1, c["t"], c["b"])
        counts = [counts[i] for i in torch.randperm(c["b"], generator=g).tolist()]
    return parents, counts


def _tables(lens: list[int], first: list[int], bs: int, seed: int) -> tuple[torch.Tensor, int]:
    """Disjoint block tables of rows of ``lens`` tokens in a seeded block order, and the pool's blocks. Only the
    pages from token ``first`` of each row on have a block of their own."""
    g = torch.Generator().manual_seed(seed + 2)
    need = [-(-n // bs) for n in lens]
    skip = [f // bs for f in first]
    blocks = sum(n - s for n, s in zip(need, skip)) + 8
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    tables, used = torch.zeros(len(lens), max(need), dtype=torch.int32), 0
    for row, (n, s) in enumerate(zip(need, skip)):
        tables[row, s:n] = perm[used:used + n - s]
        used += n - s
    return tables, blocks


def _attend_inputs(c: dict, seed: int):
    """Every row's K and V (context, then its nodes), the queries of its T nodes."""
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    parents, counts = _trees(c, seed)
    order = torch.randperm(c["b"], generator=torch.Generator().manual_seed(seed)).tolist()
    ctx = [_spread(c["lo"], c["hi"], c["b"])[i] for i in order]
    big = 1 + 7 * (torch.rand(c["hkv"], 1, c["d"], generator=g, device=DEV) < 0.02)  # a few channels of K are large
    rows = []
    for n, m in zip(ctx, counts):
        k = torch.randn(c["hkv"], n + m, c["d"], generator=g, device=DEV) * big
        rows.append((k.to(dt), torch.randn(c["hkv"], n + m, c["d"], generator=g, device=DEV).to(dt)))
    q = torch.randn(c["b"], c["hkv"] * c["group"], c["t"], c["d"], generator=g, device=DEV).to(dt)
    return parents, counts, ctx, rows, q


def _verify_inputs(c: dict, seed: int):
    """Logits in which a node's children are likely tokens (with draft logits: drawn from them), as a draft that is
    worth its while gives them."""
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    parents, counts = _trees(c, seed)
    b, t, v = c["b"], c["t"], c["vocab"]
    temps = 0.6 + 0.6 * torch.rand(b, generator=g, device=DEV)
    if c["greedy"]:
        temps[:: c["greedy"]] = 0.0
    tau = torch.where(temps > 0, temps, 1.0)
    tokens = torch.randint(0, v, (b, t), generator=g, device=DEV)
    uniforms = torch.rand(b, t, generator=g, device=DEV)
    up = torch.tensor(parents, device=DEV).expand(b, t)                         # parent of every node
    logits = torch.empty(b, t, v, dtype=dt, device=DEV)
    draft = torch.empty(b, t, v, dtype=dt, device=DEV) if c["draft"] else None
    # softmax's logsumexp over 2 * randn at temperature tau is about log(v) + 2 / tau**2
    whole = math.log(v) * tau + 2.0 / tau
    rank = torch.zeros(b, t, device=DEV)
    for i in range(1, t):
        same = (up[:, 1:i] == up[:, i:i + 1]).sum(dim=1)
        rank[:, i] = same.float()
    for row in range(b):
        x = 2.0 * torch.randn(t, v, generator=g, device=DEV)
        if draft is None:
            if t > 1:
                x[up[row, 1:], tokens[row, 1:]] = whole[row] + tau[row] * (0.7 - 1.2 * rank[row, 1:])
            logits[row] = x.to(dt)
            continue
        x.scatter_add_(1, torch.randint(0, v, (t, 24), generator=g, device=DEV),
                       tau[row] * 12.0 * torch.rand(t, 24, generator=g, device=DEV))
        logits[row] = x.to(dt)
        draft[row] = (x + 0.6 * torch.randn(t, v, generator=g, device=DEV)).to(dt)
        if t > 1:
            noise = -torch.log(-torch.log(torch.rand(t - 1, v, generator=g, device=DEV).clamp(1e-20, 1 - 1e-7)))
            tokens[row, 1:] = (draft[row][up[row, 1:]].float() / tau[row] + noise).argmax(dim=1)
    return parents, counts, logits, tokens, uniforms, temps, draft


def _keep_path(c: dict, row: int) -> list[int]:
    """The nodes kept of a row: the same for every seed. As in a tree in level order, a kept node either stands
    where it belongs or comes from behind every kept place."""
    n = 1 + (row * 5 + 3) % min(8, c["t"])
    path = list(range(n))
    far = list(range(n, c["t"]))[: n // 2 + 1]
    for i, node in zip(range(n - len(far[: n - 1]), n), far[: n - 1]):
        path[i] = node
    return path


def _keep_inputs(c: dict, seed: int):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    start = _spread(1, c["hi"], c["b"])
    start = [start[i] for i in torch.randperm(c["b"], generator=torch.Generator().manual_seed(seed)).tolist()]
    tables, blocks = _tables([s + c["t"] for s in start], start, c["bs"], seed)
    shape = (c["layers"], blocks, c["hkv"], c["bs"], c["d"])
    k, v = (torch.randn(shape, generator=g, device=DEV, dtype=dt) for _ in range(2))
    paths = [_keep_path(c, i) for i in range(c["b"])]
    return start, tables, blocks, paths, k, v


def _pool(c: dict, blocks: int, layers: int):
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    return GpuKVBlockPool(num_blocks=blocks, block_size_tokens=c["bs"], num_layers=layers, num_kv_heads=c["hkv"],
                          head_dim=c["d"], dtype=DTYPES[c["dtype"]], device=DEV)


def _visible(parents: list[list[int]]) -> torch.Tensor:
    """bool ``[trees, T, T]``: node i sees node j, an ancestor of its or itself."""
    t = len(parents[0])
    see = torch.zeros(len(parents), t, t, dtype=torch.bool)
    for m, row in zip(see, parents):
        for i, p in enumerate(row):
            if p >= 0:
                m[i] = m[p]
            m[i, i] = True
    return see


def prepare(case: dict, seed: int):
    kind = case["kind"]
    st = SimpleNamespace(kind=kind, case=case)
    if own:
        from runtime_amd.phase2.speculative import DraftTree
    if kind == "keep":
        start, tables, blocks, paths, k, v = _keep_inputs(case, seed)
        path = torch.full((case["b"], case["t"]), -1, dtype=torch.int32)
        for row, p in enumerate(paths):
            path[row, :len(p)] = torch.tensor(p, dtype=torch.int32)
        st.start, st.tables, st.path, st.counts = _ints(start), tables.to(DEV), path.to(DEV), _ints([len(p) for p in paths])
        if own:
            st.pool = _pool(case, blocks, case["layers"])
            for layer in range(case["layers"]):
                st.pool.k_layer_view(layer).copy_(k[layer])
                st.pool.v_layer_view(layer).copy_(v[layer])
            st.lens = torch.zeros(case["b"], dtype=torch.int32, device=DEV)
        else:
            st.k, st.v = k, v
        return st
    if kind == "verify":
        parents, counts, st.logits, st.tokens, st.uniforms, st.temps, st.draft = _verify_inputs(case, seed)
    else:
        parents, counts, ctx, rows, st.q = _attend_inputs(case, seed)
        st.scaling, st.group = case["d"] ** -0.5, case["group"]
        st.ctx, st.lens = _ints(ctx), _ints([n + m for n, m in zip(ctx, counts)])
        tables, blocks = _tables(st.lens.tolist(), [0] * case["b"], case["bs"], seed)
        st.tables = tables.to(DEV)
        if own:
            from runtime_amd.phase2.paged_attention_hip import PagedDecodeBatchMetadata

            st.pool = _pool(case, blocks, 1)
            for i, (k, v) in enumerate(rows):
                st.pool.write_tokens_batch(0, st.tables[i:i + 1], _ints([0]), k[None], v[None])
        else:
            st.k, st.v = (torch.zeros(blocks, case["hkv"], case["bs"], case["d"], dtype=st.q.dtype, device=DEV)
                          for _ in range(2))
            for i, kv in enumerate(rows):
                pos = torch.arange(kv[0].shape[1], device=DEV)
                page = st.tables[i].long()[pos // case["bs"]]
                for pages, x in zip((st.k, st.v), kv):
                    pages[page, :, pos % case["bs"]] = x.transpose(0, 1)
    st.node_counts = _ints(counts) if case["ragged"] else None
    if own:
        chain = case["branch"] == 1
        st.tree = (DraftTree.chain(case["t"], DEV, counts=st.node_counts) if chain
                   else DraftTree.from_parents(parents if case["branch"] == 0 else parents[0], DEV, counts=st.node_counts))
        if kind == "attend":
            st.meta = PagedDecodeBatchMetadata(pool=st.pool, layer_idx=0, block_tables=st.tables, seq_lens=st.lens,
                                               tree=st.tree)
    else:
        st.counts = _ints(counts)
        st.parents = torch.tensor(parents, dtype=torch.int32).to(DEV).expand(case["b"], case["t"])
        st.host_lens = [int(n) for n in st.lens.tolist()] if kind == "attend" else None
        if kind == "attend":
            st.see = _visible(parents).to(DEV)
    return st


# ---------------------------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------------------------
def _plain_attend(st) -> torch.Tensor:
    c = st.case
    b, t, hkv, group, d, bs = (c[n] for n in ("b", "t", "hkv", "group", "d", "bs"))
    out = torch.zeros(b, t, hkv * group, d, dtype=st.q.dtype, device=DEV)
    node = torch.arange(t, device=DEV)
    for row in range(b):
        n = st.host_lens[row]
        ids = st.tables[row, :-(-n // bs)].long()
        k, v = (x[ids].float().permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n] for x in (st.k, st.v))
        at = torch.arange(n, device=DEV) - st.ctx[row]                            # the node a token is, below 0: context
        see = st.see[row if len(st.see) > 1 else 0]
        live = (at[None] < 0) | see[:, at.clamp(min=0)]                           # [T, n]
        live = live & (node < st.counts[row])[:, None]
        qg = st.q[row].float().view(hkv, group * t, d)
        s = torch.matmul(qg, k.transpose(1, 2).contiguous()) * st.scaling
        s = torch.where(live[None, None], s.view(hkv, group, t, n), NEG)
        top = s.amax(dim=-1, keepdim=True)
        p = torch.exp(s - torch.where(top == NEG, 0.0, top))
        total = p.sum(dim=-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        o = torch.matmul(p.view(hkv, group * t, n), v.contiguous())
        out[row] = o.view(hkv * group, t, d).transpose(0, 1).to(st.q.dtype)
    return out


def _distribution(logits: torch.Tensor, temps: torch.Tensor) -> torch.Tensor:
    """softmax(logits / temperature) in 64 bits along the last of ``[B, ..., V]``."""
    shape = (-1,) + (1,) * (logits.dim() - 1)
    x = logits.double()
    tau = torch.where(temps > 0, temps, 1.0).double().view(shape)
    p = torch.exp((x - x.amax(dim=-1, keepdim=True)) / tau)
    p = p / p.sum(dim=-1, keepdim=True)
    first = torch.zeros_like(p).scatter_(-1, x.argmax(dim=-1, keepdim=True), 1.0)
    return torch.where((temps > 0).view(shape), p, first)


def _plain_verify(st):
    c = st.case
    b, t, v = c["b"], c["t"], c["vocab"]
    rows = torch.arange(b, device=DEV)
    at = torch.zeros(b, dtype=torch.long, device=DEV)
    r = _distribution(st.logits[:, 0], st.temps)
    q = _distribution(st.draft[:, 0], st.temps) if st.draft is not None else None
    path = torch.full((b, t), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    n = torch.ones(b, dtype=torch.int32, device=DEV)
    # Children stand behind their parents: one pass over the nodes meets every node's children in order.
    for i in range(1, t):
        tried = (st.parents[:, i] == at) & (i < st.counts)
        x = st.tokens[:, i]
        mine = r[rows, x]
        drafted = q[rows, x] if q is not None else torch.ones_like(mine)
        taken = tried & (st.uniforms[:, i].double() * drafted < mine)
        if q is not None:
            rest = torch.clamp(r - q, min=0.0)
        else:
            rest = r.clone()
            rest[rows, x] = 0.0
        mass = rest.sum(dim=1, keepdim=True)
        rest = torch.where(mass > 0, rest / torch.where(mass > 0, mass, 1.0), r)
        r = torch.where((tried & ~taken)[:, None], rest, r)
        r = torch.where(taken[:, None], _distribution(st.logits[:, i], st.temps), r)
        if q is not None:
            q = torch.where(taken[:, None], _distribution(st.draft[:, i], st.temps), q)
        at = torch.where(taken, i, at)
        path[rows, n.long() % t] = torch.where(taken, i, path[rows, n.long() % t])
        n = n + taken.int()
    run = r.cumsum(dim=1)
    following = (run <= st.uniforms[:, :1].double() * run[:, -1:]).sum(dim=1)
    last = v - 1 - (r > 0).flip(1).int().argmax(dim=1)
    following = torch.minimum(following, last)
    place = torch.arange(t, device=DEV)[None]
    drafted = st.tokens.gather(1, path.clamp(min=0).long()).roll(-1, dims=1)
    tokens = torch.where(place < n[:, None] - 1, drafted, -1)
    tokens = torch.where(place == n[:, None] - 1, following[:, None], tokens)
    return {"tokens": tokens, "counts": n, "path": path}


def _plain_keep(st):
    c = st.case
    bs = c["bs"]
    place = torch.arange(c["t"], device=DEV)[None]
    row, j = torch.nonzero(place < st.counts[:, None], as_tuple=True)
    of, to = st.start[row] + st.path[row, j], st.start[row] + j
    src, dst = (st.tables[row, (p // bs).long()].long() for p in (of, to))
    for x in (st.k, st.v):
        x[:, dst, :, (to % bs).long()] = x[:, src, :, (of % bs).long()]
    return {"k": list(st.k.unbind()), "v": list(st.v.unbind()), "lens": st.start + st.counts}


# ---------------------------------------------------------------------------------------------
# The framework's calls.
# ---------------------------------------------------------------------------------------------
def _own_run(st):
    if st.kind == "attend":
        from runtime_amd.phase2.speculative import paged_attention_tree

        return paged_attention_tree(st.q, st.meta, st.group, st.scaling)
    if st.kind == "verify":
        from runtime_amd.phase2.speculative import verify_draft

        out = verify_draft(st.logits, st.tokens, st.tree, st.uniforms, st.temps, draft_logits=st.draft)
        return {"tokens": out.tokens, "counts": out.counts, "path": out.path}
    st.pool.keep_tokens(st.tables, st.start, st.path, st.counts, lens_out=st.lens)
    views = range(st.case["layers"])
    return {"k": [st.pool.k_layer_view(i) for i in views], "v": [st.pool.v_layer_view(i) for i in views], "lens": st.lens}


@torch.no_grad()
def run(st):
    if own:
        return _own_run(st)
    return {"attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[st.kind](st)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without, and the exact answer.
# ---------------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    b, t = case["b"], case["t"]
    if case["kind"] == "keep":
        moved = sum(sum(i != p for i, p in enumerate(_keep_path(case, row))) for row in range(b))
        token = case["layers"] * case["hkv"] * case["d"] * 4
        return {"bytes": 2 * moved * token + 4 * b * (t + 3), "flops": 0}
    counts = _spread(1, t, b) if case["ragged"] else [t] * b
    if case["kind"] == "verify":
        # A row visits the nodes of its path, and reads no other logits: a child is taken about 3 times in 4.
        size = 4 if case["dtype"] == "fp32" else 2
        visited = sum(1 + min(2.0, (n - 1) * 0.75 / max(1, case["branch"])) for n in counts)
        row = case["vocab"] * (2 if case["draft"] else 1)
        return {"bytes": int(visited * row * size) + b * t * 28, "flops": int(visited * row * 4)}
    h, d, hq = case["hkv"], case["d"], case["hkv"] * case["group"]
    ctx = _spread(case["lo"], case["hi"], b)
    tokens = sum(ctx) + sum(counts)
    # a node sees the context and, of the nodes, at most those before it
    seen = sum(n * m for n, m in zip(ctx, counts)) + sum(m * (m + 1) // 2 for m in counts if case["branch"] == 1)
    pages = sum(-(-(n + m) // case["bs"]) for n, m in zip(ctx, counts))
    return {"bytes": 4 * tokens * h * d + 4 * pages + 4 * b * t * hq * d, "flops": 4 * seen * hq * d}


def _exact_attend(case: dict, seed: int) -> torch.Tensor:
    parents, counts, ctx, rows, q = _attend_inputs(case, seed)
    t, group, d = case["t"], case["group"], case["d"]
    out = torch.zeros(case["b"], t, case["hkv"] * group, d, dtype=torch.float64, device=DEV)
    for row, ((k, v), n, m) in enumerate(zip(rows, ctx, counts)):
        tree = parents[row % len(parents)] if len(parents) > 1 else parents[0]
        hide = torch.ones(m, n + m, dtype=torch.bool)
        hide[:, :n] = False
        for i in range(m):
            j = i
            while j >= 0:
                hide[i, n + j] = False
                j = tree[j]
        hide = hide.to(DEV)
        for h in range(case["hkv"]):
            kd, vd = k[h].double(), v[h].double()
            for e in range(group):
                s = torch.matmul(q[row, h * group + e, :m].double(), kd.t().contiguous()) / math.sqrt(d)
                out[row, :m, h * group + e] = torch.matmul(torch.softmax(s.masked_fill(hide, NEG), dim=-1), vd)
    return out


def _exact_verify(case: dict, seed: int) -> dict:
    parents, counts, logits, tokens, uniforms, temps, draft = _verify_inputs(case, seed)
    b, t = case["b"], case["t"]
    out = torch.full((b, t), -1, dtype=torch.int64)
    path = torch.full((b, t), -1, dtype=torch.int32)
    us, ts, taus = uniforms.tolist(), tokens.tolist(), temps.tolist()

    def dist(x: torch.Tensor, tau: float) -> torch.Tensor:
        x = x.double()
        if tau > 0:
            return torch.softmax(x / tau, dim=0)
        one = torch.zeros_like(x)
        one[int(torch.nonzero(x == x.max())[0])] = 1.0
        return one

    lens = []
    for row in range(b):
        tree, node, kept = parents[row] if len(parents) > 1 else parents[0], 0, [0]
        while True:
            r = dist(logits[row, node], taus[row])
            q = dist(draft[row, node], taus[row]) if draft is not None else None
            step = None
            for child in (i for i in range(1, counts[row]) if tree[i] == node):
                x = ts[row][child]
                if us[row][child] * (1.0 if q is None else float(q[x])) < float(r[x]):
                    step = child
                    break
                if q is None:
                    rest = r.clone()
                    rest[x] = 0.0
                else:
                    rest = (r - q).clamp(min=0.0)
                if float(rest.sum()) > 0:
                    r = rest / rest.sum()
            if step is None:
                break
            node = step
            kept.append(step)
        upto = torch.cumsum(r, dim=0)
        beyond = torch.nonzero(upto > us[row][0] * float(upto[-1]))
        following = int(beyond[0]) if len(beyond) else int(torch.nonzero(r > 0)[-1])
        lens.append(len(kept))
        path[row, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
        out[row, :len(kept)] = torch.tensor([ts[row][i] for i in kept[1:]] + [following])
    return {"tokens": out.to(DEV), "counts": _ints(lens), "path": path.to(DEV)}


def exact(case: dict, seed: int):
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(case, seed)
    start, tables, _, paths, k, v = _keep_inputs(case, seed)
    out = {"k": k.double(), "v": v.double()}
    bs = case["bs"]
    for row, kept in enumerate(paths):
        for x, was in ((out["k"], k), (out["v"], v)):
            for j, node in enumerate(kept):
                of, to = start[row] + node, start[row] + j
                x[:, int(tables[row, to // bs]), :, to % bs] = was[:, int(tables[row, of // bs]), :, of % bs].double()
    return {"k": list(out["k"].unbind()), "v": list(out["v"].unbind()),
            "lens": _ints([s + len(p) for s, p in zip(start, paths)])}
