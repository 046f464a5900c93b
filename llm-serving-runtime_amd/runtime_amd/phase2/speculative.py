"""Speculative decoding over the paged cache: attention of a tree of drafted tokens, and its verification.

The reference drafts tokens and verifies them greedily, one after the other, through its decode path
(``runtime/phase2/worker_server.py:1010-1075``). Here a step runs the target model once over all drafted
tokens of all rows:

* :class:`DraftTree` - the shape of the drafts: each node's parent, who sees whom, each node's depth;
* :func:`paged_attention_tree` - the nodes' attention over the paged cache (``mx_tree_attn``): the row's
  context and the node's own ancestors. A chain (:meth:`DraftTree.chain`) is causal attention of several
  new tokens, such as a chunk of a prompt;
* :func:`verify_draft` - the path that the target's distributions accept, and the token that follows it
  (``mx_verify_draft``), from uniform numbers that the caller gives;
* ``GpuKVBlockPool.keep_tokens`` - the path's K and V moved right behind the context, in every layer.

The drafted tokens' K and V stand in the cache behind the row's context in the order of the nodes
(``write_tokens_batch`` at the context's length), whatever their depth; a node's rotary position is the
context's length plus its depth (:meth:`DraftTree.position_ids`). ``hf_decode.speculative_decode`` puts the
pieces together for an HF model.

All take device tensors and enqueue on the current stream of their device; no call synchronises or keeps
anything between calls (workspaces come from torch's allocator, so calls on several streams and in several
graphs need no care). Errors raise ``ValueError`` or ``TypeError`` (bad arguments) or ``RuntimeError``.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _hip
from .kv8 import _lengths, _tables
from .paged_attention_hip import _DTYPE_FLAGS, MX_PA_BF16, MX_PA_SHARED_BLOCKS, PagedDecodeBatchMetadata

MX_LOGITS_FP32 = 16
_LOGITS_FLAGS = {torch.float16: 0, torch.bfloat16: MX_PA_BF16, torch.float32: MX_LOGITS_FP32}


@dataclass(frozen=True, eq=False)
class DraftTree:
    """The shape of the trees of ``size`` nodes that a batch drafts: one for all rows, or one a row.

    Node 0 is the last token that is already certain; every other node stands behind its parent. Built by
    :meth:`chain` or :meth:`from_parents`.
    """

    parents: torch.Tensor            # int32 [1 or B, T]; -1: no parent
    depth: torch.Tensor              # int64 [1 or B, T]; ancestors of each node
    mask: torch.Tensor | None        # bool [1 or B, T, T]: node i sees node j; None: a chain
    counts: torch.Tensor | None = None  # int32 [B]: nodes of each row (below 0: none, above T: T); None: all T

    @property
    def size(self) -> int:
        return int(self.parents.shape[1])

    @property
    def rows(self) -> int:
        """1 where all rows have the same tree, else how many there are."""
        return int(self.parents.shape[0])

    @classmethod
    def chain(cls, size: int, device: torch.device | str, counts: torch.Tensor | None = None) -> "DraftTree":
        """Every node the only child of the one before it."""
        if size < 1:
            raise ValueError("a tree has at least one node")
        depth = torch.arange(size, dtype=torch.int64).to(device).unsqueeze(0)
        return cls((depth - 1).to(torch.int32), depth, None, _node_counts(counts, depth.device))

    @classmethod
    def from_parents(cls, parents, device: torch.device | str | None = None, counts: torch.Tensor | None = None
                     ) -> "DraftTree":
        """From each node's parent: a list or int tensor ``[T]``, or ``[B, T]`` with a tree a row. Node 0 has
        none (-1), every other one a node before it or -1 (it then sees the context and itself only).

        Lists and host tensors are checked (``ValueError``). A device tensor is used as it stands, without a
        host sync: a parent that is not a node before its child counts as none.
        """
        t = torch.as_tensor(parents)
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
            raise TypeError(f"parents must be whole numbers, got {t.dtype}")
        t = t.unsqueeze(0) if t.dim() == 1 else t
        if t.dim() != 2 or t.shape[0] < 1 or t.shape[1] < 1:
            raise ValueError("parents must be [T] or [B, T] with at least one node")
        size = int(t.shape[1])
        is_chain = False
        if t.device.type == "cpu":
            before = torch.arange(size)
            if bool(((t < -1) | (t >= before)).any()):
                raise ValueError("a node's parent must be a node before it, or -1; node 0 has none")
            is_chain = bool((t == before - 1).all())
            t = t.to(torch.device(device) if device is not None else torch.device("cuda"))
        elif device is not None and torch.device(device) not in (t.device, torch.device(t.device.type)):
            t = t.to(device)
        if is_chain:
            return cls.chain(size, t.device, counts)
        node = torch.arange(size, dtype=torch.int64, device=t.device)
        parent = t.to(torch.int64)
        parent = torch.where((parent >= 0) & (parent < node), parent, -1)
        # reach[i, j]: j is i or an ancestor at most 2^k steps above; squared until 2^k covers every chain
        reach = ((parent.unsqueeze(2) == node) | (node.unsqueeze(1) == node)).float()
        steps = 1
        while steps < size - 1:
            reach = (torch.bmm(reach, reach) > 0).float()
            steps *= 2
        mask = reach > 0
        return cls(parent.to(torch.int32), mask.sum(dim=2) - 1, mask, _node_counts(counts, t.device))

    def position_ids(self, context_lens: torch.Tensor) -> torch.Tensor:
        """int64 ``[B, T]``: the position of each node behind contexts of ``context_lens [B]`` tokens."""
        return context_lens.to(torch.int64).unsqueeze(1) + self.depth

    def check_batch(self, batch: int, nodes: int, device: torch.device) -> None:
        """Raise ``ValueError`` unless this is the shape of ``batch`` rows of ``nodes`` drafted tokens on ``device``."""
        if self.size != nodes or self.rows not in (1, batch):
            raise ValueError(f"a draft of {batch} rows of {nodes} nodes does not fit a tree of {self.size} nodes in "
                             f"{self.rows} rows")
        t = self.parents
        if t.device != device or t.dtype != torch.int32 or t.stride(1) != 1 and nodes > 1:
            raise ValueError("a tree's parents must be int32 with unit inner stride on the draft's device")
        if self.mask is not None and (self.mask.dtype != torch.bool or self.mask.shape[1:] != (nodes, nodes)
                                      or self.mask.shape[0] not in (1, batch) or self.mask.device != device
                                      or self.mask.stride(2) != 1 and nodes > 1):
            raise ValueError("a tree's mask must be bool [1 or B, T, T] with unit inner stride on the draft's device")
        if self.counts is not None and (self.counts.shape != (batch,) or self.counts.dtype != torch.int32
                                        or self.counts.device != device or not self.counts.is_contiguous()):
            raise ValueError("a tree's counts must be contiguous int32 [B] on the draft's device")


def _node_counts(counts: torch.Tensor | None, device: torch.device) -> torch.Tensor | None:
    if counts is None:
        return None
    if not isinstance(counts, torch.Tensor) or counts.dim() != 1:
        raise ValueError("counts must be a tensor [B]")
    return counts.to(device=device, dtype=torch.int32).contiguous()


def _aligned_rows(t: torch.Tensor) -> tuple[int, int, int] | None:
    """Strides of ``[B, H, T, D]`` for 16-byte loads (0 for a dimension of one, whose stride may be anything), or None."""
    (b, h, n, _), (sb, sh, st, unit) = t.shape, t.stride()
    out = (sb if b > 1 else 0, sh if h > 1 else 0, st if n > 1 else 0)
    return None if unit != 1 or t.data_ptr() % 16 or out[0] % 8 or out[1] % 8 or out[2] % 8 else out


def paged_attention_tree(query: torch.Tensor, metadata: PagedDecodeBatchMetadata, num_kv_groups: int, scaling: float
                         ) -> torch.Tensor:
    """Attention of the nodes of ``metadata.tree``: ``query [B, heads, T, dim]`` -> ``[B, T, heads, dim]``.

    The nodes' K and V are in the pool behind the row's context; ``metadata.seq_lens`` counts them (the
    context's length plus ``T``, or plus the row's ``tree.counts``). Without a tree the T tokens are a chain.
    Nodes past a row's count, and nodes that see nothing, give zeros. fp16 or bf16 query and 16-bit pool of
    one dtype, head_dim in {64, 128}, block size in {4, 8, 16, 32}, any GQA group. A block id outside the
    pool is skipped and reported by ``pool.check_write_errors()``. There is no gradient: a query that asks for one
    (call it under ``torch.no_grad()``) or is being traced raises ``RuntimeError``.
    """
    _hip.require_device_tensor(query, "query")
    if query.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 or torch.jit.is_tracing():
        raise RuntimeError("tree attention has no gradient and cannot be traced: the result would be a constant")
    if query.dim() != 4:
        raise ValueError("query must be [B, heads, T, dim]")
    bsz, hq, nodes, d = query.shape
    pool = metadata.pool
    if getattr(pool, "kv_bits", 16) != 16:
        raise ValueError("tree attention reads a 16-bit pool")
    if bsz != metadata.block_tables.shape[0]:
        raise ValueError("query batch size must match block_tables rows")
    k_layer, v_layer = pool.k_layer_view(metadata.layer_idx), pool.v_layer_view(metadata.layer_idx)
    if query.dtype not in _DTYPE_FLAGS or k_layer.dtype != query.dtype:
        raise ValueError(f"tree attention takes fp16 or bf16 query and pool of one dtype, got {query.dtype}/{k_layer.dtype}")
    device = query.device
    if k_layer.device != device:
        raise ValueError("query and pool must be on one device")
    nb, hkv, bs, dk = k_layer.shape
    if dk != d:
        raise ValueError(f"head_dim mismatch: query {d} vs pool {dk}")
    if hkv * num_kv_groups != hq:
        raise ValueError(f"num_heads {hq} != num_kv_heads {hkv} * num_kv_groups {num_kv_groups}")
    tables = _tables(metadata.block_tables, bsz, device)
    lens = _lengths(metadata.seq_lens, bsz, device)
    tree = metadata.tree
    mask = counts = None
    mask_sb = mask_st = 0
    if tree is not None:
        tree.check_batch(bsz, nodes, device)
        mask, counts = tree.mask, tree.counts
        if mask is not None:
            mask_sb, mask_st = mask.stride(0) if mask.shape[0] > 1 else 0, mask.stride(1)
    out = torch.empty((bsz, nodes, hq, d), dtype=query.dtype, device=device)
    if bsz == 0 or nodes == 0:
        return out
    strides = _aligned_rows(query)
    if strides is None:
        query = query.contiguous() if query.stride(3) != 1 or not query.is_contiguous() else query.clone()
        if query.data_ptr() % 16:
            query = query.clone()
        strides = _aligned_rows(query)
    key = (bsz, nodes, hq, hkv, d, tables.shape[1], bs)
    nbytes = _hip.tree_attn_workspace_bytes(*key)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    k_strides = k_layer.stride()
    with _hip.on_device(device):
        rc = _hip.load().mx_tree_attn(
            query.data_ptr(), *strides, k_layer.data_ptr(), v_layer.data_ptr(), k_strides[0], k_strides[1],
            tables.data_ptr(), tables.stride(0), tables.shape[1], lens.data_ptr(),
            None if mask is None else mask.data_ptr(), mask_sb, mask_st, None if counts is None else counts.data_ptr(),
            bsz, nodes, hq, hkv, d, bs, nb, float(scaling), out.data_ptr(), nodes * hq * d, hq * d, d, ws.data_ptr(),
            nbytes, pool._write_err.data_ptr(),
            _DTYPE_FLAGS[query.dtype] | (MX_PA_SHARED_BLOCKS if metadata.shared_blocks else 0), _hip.stream_handle(device))
        _hip.check(rc, "mx_tree_attn")
    return out


class DraftVerdict(NamedTuple):
    """What :func:`verify_draft` returns, on the device."""

    tokens: torch.Tensor  # int64 [B, T]: the kept drafted tokens, then the one that follows, then -1
    counts: torch.Tensor  # int32 [B]: nodes kept, node 0 among them: as many tokens as the row goes on by
    path: torch.Tensor    # int32 [B, T]: the nodes kept, from node 0, then -1


def _rows_of(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be a tensor of shape {list(shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on the logits' device")
    if t.dtype != dtype:
        if dtype.is_floating_point != t.dtype.is_floating_point:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        t = t.to(dtype)
    return t if t.dim() == 0 or t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _logit_strides(t: torch.Tensor) -> tuple[int, int]:
    return t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0


def verify_draft(logits: torch.Tensor, tokens: torch.Tensor, tree: DraftTree, uniforms: torch.Tensor,
                 temperature: torch.Tensor | float, draft_logits: torch.Tensor | None = None) -> DraftVerdict:
    """The path of each row's tree that the target accepts, and the token that follows it.

    ``logits [B, T, V]`` (fp16, bf16 or fp32) are the target's at every node, ``tokens [B, T]`` the nodes'
    tokens, ``uniforms [B, T]`` numbers in [0, 1) (``torch.rand``), ``temperature`` a number or ``[B]``.
    ``draft_logits [B, T, V]`` are the draft model's at the nodes whose children were drawn, independently,
    from ``softmax(draft_logits / temperature)``; without them a child stands for a draft that was certain of
    it (prompt lookup, the largest logits of a draft model).

    At a node with ``r = softmax(logits / temperature)`` the children are tried in the order of their indices:
    one with token ``x`` is kept where ``uniforms[child] * q(x) < r(x)``; one that is not leaves
    ``r = max(r - q, 0)`` (without draft logits: ``r`` without ``x``), scaled to a sum of 1. Where none is kept
    the following token is drawn from ``r``: the first whose running sum exceeds ``uniforms[node 0]``. So the
    tokens are distributed as the target's own samples. At temperature 0 (or below) ``r`` is all at the largest
    logit, the first on ties: greedy decoding. The arithmetic is in 64 bits (sums over parts of the vocabulary are
    joined with 44 of their 52).

    A drafted token outside the vocabulary is not kept. A node whose logits hold a NaN, nothing above -inf or
    (with a temperature) +inf keeps nothing and is followed by -1.
    """
    _hip.require_device_tensor(logits, "logits")
    if logits.dim() != 3 or logits.dtype not in _LOGITS_FLAGS:
        raise ValueError(f"logits must be fp16, bf16 or fp32 [B, T, V], got {logits.dtype} {list(logits.shape)}")
    b, t, v = logits.shape
    dev = logits.device
    if v < 1:
        raise ValueError("logits must have a vocabulary")
    if draft_logits is not None:
        _hip.require_device_tensor(draft_logits, "draft_logits")
        if draft_logits.shape != logits.shape or draft_logits.dtype != logits.dtype or draft_logits.device != dev:
            raise ValueError("draft_logits must have the logits' shape, dtype and device")
        if draft_logits.stride(2) != 1 and v > 1:
            draft_logits = draft_logits.contiguous()
    if logits.stride(2) != 1 and v > 1:
        logits = logits.contiguous()
    tokens = _rows_of(tokens, "tokens", (b, t), torch.int64, dev)
    wide = isinstance(uniforms, torch.Tensor) and uniforms.dtype == torch.float64
    uniforms = _rows_of(uniforms, "uniforms", (b, t), torch.float32, dev)
    if wide:  # the largest ones would be rounded to 1, at which what is certain is refused
        uniforms = uniforms.clamp(max=1 - 2.0 ** -24)
    tree.check_batch(b, t, dev)
    if isinstance(temperature, torch.Tensor):
        if temperature.dim() == 0:
            temperature = temperature.expand(b)
        temperature = _rows_of(temperature, "temperature", (b,), torch.float32, dev)
        temp_sb = temperature.stride(0) if b > 1 else 0
    else:
        temperature = torch.full((1,), float(temperature), dtype=torch.float32, device=dev)
        temp_sb = 0
    out = DraftVerdict(torch.empty((b, t), dtype=torch.int64, device=dev), torch.empty(b, dtype=torch.int32, device=dev),
                       torch.empty((b, t), dtype=torch.int32, device=dev))
    if b == 0:
        return out
    if t == 0:
        raise ValueError("a tree has at least one node")
    nbytes = _hip.verify_draft_workspace_bytes(b, t, v, int(draft_logits is not None))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _hip.on_device(dev):
        _hip.check(_hip.load().mx_verify_draft(
            logits.data_ptr(), *_logit_strides(logits),
            None if draft_logits is None else draft_logits.data_ptr(),
            *((0, 0) if draft_logits is None else _logit_strides(draft_logits)), tokens.data_ptr(), tokens.stride(0),
            tree.parents.data_ptr(), tree.parents.stride(0) if tree.rows > 1 else 0,
            None if tree.counts is None else tree.counts.data_ptr(), uniforms.data_ptr(), uniforms.stride(0),
            temperature.data_ptr(), temp_sb, b, t, v, out.tokens.data_ptr(), out.counts.data_ptr(), out.path.data_ptr(),
            ws.data_ptr(), nbytes, _LOGITS_FLAGS[logits.dtype], _hip.stream_handle(dev)), "mx_verify_draft")
    return out
