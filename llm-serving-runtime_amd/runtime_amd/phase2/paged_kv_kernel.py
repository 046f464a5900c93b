"""Block-paged KV storage read by the HIP paged-attention decode kernel.

Keeps the reference's ``GpuKVBlockPool`` API (``runtime/phase2/paged_kv_kernel.py:24-315``):
``k_layer_view(l)`` / ``v_layer_view(l)`` are ``[num_blocks, Hkv, bs, D]`` per
layer with every (block, kv-head) one contiguous ``bs*D`` run (4 KiB at bs=16,
D=128, fp16), and token ``pos`` of a row is stored in block
``table[pos // bs]`` at offset ``pos % bs`` (``:163-174``, ``:217-227``).

MI355X-first differences:

* Layer-major storage, K beside V. The reference stores K and V in two
  ``[num_blocks, num_layers, Hkv, bs, D]`` tensors (``:101-107``), so one
  layer's blocks are spread over the whole pool, one ``Hkv*bs*D`` run every
  ``num_layers`` runs. Here one tensor ``[num_layers, num_blocks, Hkv, 2, bs,
  D]`` holds both: a layer is one contiguous region (``num_blocks * 64 KiB``
  for Llama-3-8B's 8 KV heads), so the decode kernel's random block reads for a
  layer stay inside a region the GPU's address-translation caches cover instead
  of landing on a different 2 MiB page almost every time across a 17 GB pool,
  and the K and V runs of a (block, kv-head) are one run. The views keep the
  reference's shape and per-block contents; only the strides of the first two
  dimensions differ, and every consumer takes strides from the view
  (``kv_layout="split"`` keeps K and V in two layer-major tensors).
* The reference grows its slabs lazily 8 blocks at a time and copies the
  whole slab on every growth (``:86-115``). Here the first use allocates all
  ``num_blocks`` at once (288 GB of HBM per GPU makes that the cheap choice),
  so tensor addresses never change after ``_ensure_pools`` and a captured HIP
  graph stays valid.
* ``write_tokens_batch`` on a device pool makes no host round trip. The
  reference checks the table bounds with ``.item()`` and records the written
  blocks with ``unique().tolist()`` on every call (``:221,229-231``), four
  syncs per layer per step. Here the one ``mx_kv_append`` launch skips a slot
  outside the table or the pool and sets the pool's device error word, and
  marks the blocks it writes in a device byte map. The ``IndexError`` the
  reference raises is raised by :meth:`check_write_errors` (one sync, called
  once per decode step by the decode loop), and ``allocated_block_count`` /
  ``peak_allocated_block_count`` read the byte map when asked. A caller that
  relies on the reference's raise at the write itself sets
  ``sync_write_checks`` (or ``PHASE2_KV_SYNC_CHECKS=1`` before the pool is
  built): every batched write then checks the word right away (one host sync
  per call, skipped while a HIP graph is being captured).
* ``copy_blocks`` on a device pool is one ``mx_kv_copy_pages`` launch per 448
  pages whose ids travel with it; beside it stand ``move_blocks`` (compaction:
  pages to other ids, the block tables that name them renamed) and
  ``free_blocks``. The reference has neither: its pool only ever adds to its
  used blocks.
"""

from __future__ import annotations

import array
import math
import os
import threading
from dataclasses import dataclass

import torch

from . import _hip

KV_LAYOUTS = ("split", "interleaved")

# Held while a pool makes its tensors: threads that use one first at the same time get the same ones.
_alloc_lock = threading.Lock()


@dataclass(frozen=True)
class PoolShape:
    num_blocks: int
    block_size_tokens: int
    num_layers: int
    num_kv_heads: int
    head_dim: int


def settle(device: torch.device) -> None:
    """Wait until a pool's tensors, filled on the current stream, hold what they begin with: its next use may be on
    another stream. (Under capture the fills are part of the graph.)"""
    with _hip.on_device(device):
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream().synchronize()


# Entries of one launch over pairs that depend on each other: a pair each, and one more for a cycle.
MAX_DEPENDENT = 448


def dependent_batches(src, dst) -> list[tuple[list[int], list[int]]]:
    """The copies page dst[i] = page src[i], all at once (of several with one dst the last), as lists that do the
    same one after the other, each within ``MAX_DEPENDENT``: a page is read before it is written. A longer cycle
    goes in shorter ones, whose shared page passes on the bytes that the next one needs."""
    of = {d: s for s, d in zip(src, dst)}
    of = {d: s for d, s in of.items() if s != d}
    readers = dict.fromkeys(of, 0)
    for s in of.values():
        if s in readers:
            readers[s] += 1
    ready, pairs = [d for d, n in readers.items() if n == 0], []
    while ready:
        d = ready.pop()
        s = of.pop(d)
        pairs.append((s, d))
        if s in of:
            readers[s] -= 1
            if readers[s] == 0:
                ready.append(s)
    batches = [pairs[i:i + MAX_DEPENDENT] for i in range(0, len(pairs), MAX_DEPENDENT)]
    room = 0  # entries left in the last batch, which takes cycles
    while of:  # cycles, every page read once
        d, s = of.popitem()
        ring = [d, s]  # ring[i] = page ring[i + 1], the last = the first
        while of[ring[-1]] != d:
            ring.append(of.pop(ring[-1]))
        del of[ring[-1]]
        while ring:
            part = ring[:MAX_DEPENDENT - 1]
            if len(part) + 1 > room:
                batches.append([])
                room = MAX_DEPENDENT
            batches[-1] += list(zip(part[1:] + part[:1], part))
            room -= len(part) + 1
            ring = part[-1:] + ring[len(part):] if len(ring) > len(part) else []
    return [([s for s, _ in b], [d for _, d in b]) for b in batches]


def _share_entries(tables: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether an entry of ``out`` is another one of its own or of ``tables`` (both of one shape and unit inner
    stride): renaming would read what it wrote. ``out`` may be ``tables`` itself."""
    rows, width = out.shape
    a, b = tables.stride(0) if rows > 1 else width, out.stride(0) if rows > 1 else width
    if rows == 0 or width == 0:
        return False
    if b < width:
        return True
    delta = (out.data_ptr() - tables.data_ptr()) // 4
    if (delta == 0 and a == b) or delta >= (rows - 1) * a + width or -delta >= (rows - 1) * b + width:
        return False
    return a != b or not width <= delta % b <= b - width  # columns of their own side by side in wider rows


def _ids(block_ids) -> list[int]:
    return list(map(int, block_ids))


class GpuKVBlockPool:
    """Shared block pool; same constructor and methods as the reference's."""

    kv_bits = 16  # of a stored K or V element (Int8KVBlockPool: 8)

    def __init__(self, *, num_blocks: int, block_size_tokens: int, num_layers: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype, device: str | torch.device, kv_layout: str = "interleaved") -> None:
        if num_blocks <= 0 or block_size_tokens <= 0:
            raise ValueError("num_blocks and block_size_tokens must be positive")
        if kv_layout not in KV_LAYOUTS:
            raise ValueError(f"kv_layout must be one of {KV_LAYOUTS}, got {kv_layout!r}")
        # "interleaved" (default): one tensor [L, nb, Hkv, 2, bs, D] whose K and V runs of a
        # (block, kv-head) are adjacent, one 2*bs*D run that the decode kernel reads as a unit; the
        # layer views keep the shape [nb, Hkv, bs, D] with strides (Hkv*2*bs*D, 2*bs*D, D, 1).
        # Measured on MI355X at the Llama-3-8B batch-32 step: attention 56.7-57.0 -> 54.6-55.4 us
        # per call, 7,773-7,817 -> 7,921-7,929 tokens/s. "split": K and V in two [L, nb, Hkv, bs, D]
        # tensors, each (block, kv-head) run bs*D elements.
        self.kv_layout = kv_layout
        self.shape = PoolShape(num_blocks=num_blocks, block_size_tokens=block_size_tokens, num_layers=num_layers,
                               num_kv_heads=num_kv_heads, head_dim=head_dim)
        self.dtype = dtype
        self.device = torch.device(device)
        self._k_pool: torch.Tensor | None = None
        self._v_pool: torch.Tensor | None = None
        self._k_views: tuple[torch.Tensor, ...] = ()  # k_layer_view's, made once: a step asks 2 L times
        self._v_views: tuple[torch.Tensor, ...] = ()
        self._regions: list[torch.Tensor] = []  # the tensors [L, num_blocks, ...] that hold the pages
        self._used_blocks: set[int] = set()
        self._peak_allocated_blocks = 0
        self._used_map: torch.Tensor | None = None    # uint8 [num_blocks]: blocks written on the device
        self._write_err: torch.Tensor | None = None   # int32 [1]: kv append error bits since the last check
        # True: write_tokens_batch raises IndexError at the call, as the reference does (:221-222),
        # at one host sync per call; False: at the next check_write_errors().
        self.sync_write_checks = os.getenv("PHASE2_KV_SYNC_CHECKS", "0").strip() == "1"

    @property
    def block_size_tokens(self) -> int:
        return self.shape.block_size_tokens

    def _sync_used_map(self) -> None:
        """Fold the device byte map of written blocks into the host set (one host sync)."""
        if self._used_map is None:
            return
        ids = torch.nonzero(self._used_map).flatten().tolist()
        if ids:
            self._used_blocks.update(int(i) for i in ids)
            self._peak_allocated_blocks = max(self._peak_allocated_blocks, len(self._used_blocks))

    def allocated_block_count(self) -> int:
        self._sync_used_map()
        return len(self._used_blocks)

    def peak_allocated_block_count(self) -> int:
        self._sync_used_map()
        return self._peak_allocated_blocks

    def check_write_errors(self) -> None:
        """Raise ``IndexError`` if a device KV write (or :meth:`keep_tokens`, or tree attention) met a slot
        outside its block table or the pool since the last check (the reference's ``:221-222`` check,
        deferred to one host sync); the error word is cleared."""
        if self._write_err is None:
            return
        bits = int(self._write_err.item())
        if bits:
            self._write_err.zero_()
            where = " and ".join(name for name, hit in (("batched write", bits & ~4), ("attention", bits & 4)) if hit)
            raise IndexError(f"block table underrun or physical block id out of range during {where}")

    def bytes_per_block(self) -> int:
        s = self.shape
        elems = s.num_layers * s.num_kv_heads * s.block_size_tokens * s.head_dim * 2
        return elems * torch.empty((), dtype=self.dtype).element_size()

    def bytes_for_blocks(self, block_count: int) -> int:
        return block_count * self.bytes_per_block()

    def peak_allocated_bytes(self) -> int:
        return self.bytes_for_blocks(self.peak_allocated_block_count())

    def _ensure_pools(self) -> None:
        if self._k_pool is None:
            with _alloc_lock:
                if self._k_pool is None:
                    self._make_pools()

    def _make_pools(self) -> None:
        """The pool's tensors; ``_k_pool``, by which other threads see that they are there, comes last."""
        s = self.shape
        if self.kv_layout == "interleaved":
            kv = torch.zeros(s.num_layers, s.num_blocks, s.num_kv_heads, 2, s.block_size_tokens, s.head_dim,
                             dtype=self.dtype, device=self.device)
            k_pool, v_pool = kv[:, :, :, 0], kv[:, :, :, 1]
            self._regions = [kv]
        else:
            shape = (s.num_layers, s.num_blocks, s.num_kv_heads, s.block_size_tokens, s.head_dim)
            k_pool = torch.zeros(shape, dtype=self.dtype, device=self.device)
            v_pool = torch.zeros(shape, dtype=self.dtype, device=self.device)
            self._regions = [k_pool, v_pool]
        self._k_views, self._v_views = (tuple(pool.select(0, i) for i in range(s.num_layers))
                                        for pool in (k_pool, v_pool))
        if self.device.type == "cuda":
            self._used_map = torch.zeros(s.num_blocks, dtype=torch.uint8, device=self.device)
            self._write_err = torch.zeros(1, dtype=torch.int32, device=self.device)
            settle(self._write_err.device)
        self._v_pool, self._k_pool = v_pool, k_pool

    def _touch_block(self, physical: int) -> None:
        if physical < 0 or physical >= self.shape.num_blocks:
            raise IndexError(f"physical block id out of range: {physical}")
        self._used_blocks.add(physical)
        self._peak_allocated_blocks = max(self._peak_allocated_blocks, len(self._used_blocks))

    def _touch_blocks(self, physical_ids: torch.Tensor) -> None:
        self._touch_ids(physical_ids.unique().tolist())

    def _touch_ids(self, ids: list[int]) -> None:
        """:meth:`_touch_block` of every id."""
        distinct = set(ids)
        if distinct and (min(distinct) < 0 or max(distinct) >= self.shape.num_blocks):
            for physical in ids:  # raises at the first id out of range
                self._touch_block(int(physical))
        self._used_blocks |= distinct
        self._peak_allocated_blocks = max(self._peak_allocated_blocks, len(self._used_blocks))

    def _gathers_on_device(self, tokens: int) -> bool:
        """Whether rows of ``tokens`` come out of the pool by ``mx_kv_gather``: 16-bit elements in 16-byte
        chunks, whose number in a row is a 32-bit index there."""
        return (self.device.type == "cuda" and self.dtype in (torch.float16, torch.bfloat16)
                and self.shape.head_dim % 8 == 0 and tokens * (self.shape.head_dim // 8) <= 0x7fffff00)

    def k_layer_view(self, layer_idx: int) -> torch.Tensor:
        """Per-layer K blocks: ``[num_blocks, num_kv_heads, block_size, head_dim]``."""
        self._ensure_pools()
        return self._k_views[layer_idx]

    def v_layer_view(self, layer_idx: int) -> torch.Tensor:
        """Per-layer V blocks: ``[num_blocks, num_kv_heads, block_size, head_dim]``."""
        self._ensure_pools()
        return self._v_views[layer_idx]

    def write_tokens(self, layer_idx: int, block_ids: list[int], start_pos: int, key_states: torch.Tensor,
                     value_states: torch.Tensor) -> None:
        """Write K/V for positions ``[start_pos, start_pos + kv_len)`` of one row (``:136-174``)."""
        if key_states.dim() == 3:
            key_states = key_states.unsqueeze(0)
            value_states = value_states.unsqueeze(0)
        if key_states.shape[0] != 1:
            raise ValueError("write_tokens takes a single row; use write_tokens_batch")
        kv_len = int(key_states.shape[-2])
        block_size = self.block_size_tokens
        n_logical = math.ceil((start_pos + kv_len) / block_size)
        if n_logical > len(block_ids):
            raise IndexError(f"block table underrun at pos={start_pos + kv_len - 1}: need block {n_logical - 1}, "
                             f"have {len(block_ids)}")
        table = torch.tensor([list(block_ids)], device=self.device, dtype=torch.int32)
        starts = torch.tensor([start_pos], device=self.device, dtype=torch.int64)
        self.write_tokens_batch(layer_idx, table, starts, key_states, value_states)

    def write_tokens_batch(self, layer_idx: int, block_tables: torch.Tensor, start_positions: torch.Tensor,
                           key_states: torch.Tensor, value_states: torch.Tensor,
                           counts: torch.Tensor | None = None) -> None:
        """KV write: tables ``[B, max_blocks]``, starts ``[B]``, states ``[B, Hkv, kv_len, D]``.

        Same semantics as the reference (``:176-227``). On a device pool it is
        one ``mx_kv_append`` launch (no per-token loop) and no host sync: a slot
        outside the table or the pool is skipped and recorded in the pool's
        error word, which :meth:`check_write_errors` turns into the reference's
        ``IndexError`` (``:221-222``); written blocks are marked in a device map
        for the usage accounting. A pool on the CPU (host-side tests of the
        cache bookkeeping) checks on the host and takes an indexed torch store.

        ``counts [B]`` (optional): tokens of each row; those from there on are neither written nor looked up.
        """
        if key_states.shape != value_states.shape:
            raise ValueError("key_states and value_states must match shape")
        batch_size = int(key_states.shape[0])
        kv_len = int(key_states.shape[-2])
        if block_tables.shape[0] != batch_size or start_positions.shape[0] != batch_size:
            raise ValueError("batch dimension mismatch in write_tokens_batch")
        if counts is not None and counts.shape != (batch_size,):
            raise ValueError("counts must be [B]")
        if kv_len == 0 or batch_size == 0:
            return
        self._ensure_pools()
        assert self._k_pool is not None and self._v_pool is not None
        device = self.device
        bs = self.block_size_tokens
        k_layer = self._k_pool[layer_idx]
        v_layer = self._v_pool[layer_idx]
        if device.type == "cuda":
            from .decode_glue import kv_append

            if key_states.dtype != self.dtype or value_states.dtype != self.dtype:
                key_states, value_states = key_states.to(self.dtype), value_states.to(self.dtype)
            kv_append(k_layer, v_layer, block_tables, start_positions, key_states, value_states, err=self._write_err,
                      used_blocks=self._used_map, counts=counts)
            if self.sync_write_checks and not torch.cuda.is_current_stream_capturing():
                self.check_write_errors()
            return
        tables = block_tables.to(device=device, dtype=torch.int64)
        pos = start_positions.to(device=device, dtype=torch.int64).view(-1, 1) + torch.arange(
            kv_len, device=device, dtype=torch.int64).view(1, -1)  # [B, T]
        logical = torch.div(pos, bs, rounding_mode="floor")
        live = None
        if counts is not None:
            live = torch.arange(kv_len, device=device).view(1, -1) < counts.to(device).view(-1, 1)
            if not bool(live.any()):
                return
            logical, pos = logical.masked_fill(~live, 0), pos.masked_fill(~live, 0)
        if int(logical.max().item()) >= tables.shape[1] or int(pos.min().item()) < 0:
            raise IndexError("block table underrun during batched write")
        physical = torch.gather(tables, 1, logical)  # [B, T]
        if live is not None:  # the rows' tokens, side by side
            physical, pos = physical[live].view(1, -1), pos[live].view(1, -1)
            key_states, value_states = (x.permute(1, 0, 2, 3)[:, live].unsqueeze(0) for x in (key_states, value_states))
        if int(physical.min().item()) < 0 or int(physical.max().item()) >= self.shape.num_blocks:
            raise IndexError("physical block id out of range during batched write")
        self._touch_blocks(physical)
        offset = (pos % bs).reshape(-1)
        phys = physical.reshape(-1)
        # pool[physical, layer, :, offset, :] = states[b, :, t, :]
        k_layer[phys, :, offset, :] = key_states.to(self.dtype).permute(0, 2, 1, 3).reshape(
            -1, key_states.shape[1], key_states.shape[3])
        v_layer[phys, :, offset, :] = value_states.to(self.dtype).permute(0, 2, 1, 3).reshape(
            -1, value_states.shape[1], value_states.shape[3])

    def keep_tokens(self, block_tables: torch.Tensor, start_positions: torch.Tensor, path: torch.Tensor,
                    counts: torch.Tensor, lens_out: torch.Tensor | None = None) -> None:
        """Keep a path of drafted tokens: of every row, token ``start + path[j]`` becomes token ``start + j`` for
        ``j < counts``, in all layers, every source as it was before the call.

        ``block_tables [B, max_blocks]``, ``start_positions [B]`` (the context's length), ``path [B, T]`` rising
        within [0, T) and ``counts [B]`` as ``speculative.verify_draft`` gives them, all on the pool's device: one
        launch, no host sync. ``lens_out`` (int32 ``[B]``, a tensor of its own) gets ``start + counts``, the
        rows' new lengths. A path that does not rise moves nothing from there on; that and a token outside its
        table or the pool are reported by :meth:`check_write_errors`. Rows own the blocks behind their context.
        A pool on the CPU checks on the host (``IndexError``).
        """
        if self.kv_bits != 16:
            raise ValueError("keep_tokens moves tokens of a 16-bit pool: a token of an 8-bit page has no scale of its own")
        b = int(block_tables.shape[0])
        if block_tables.dim() != 2 or path.dim() != 2 or path.shape[0] != b or counts.shape != (b,) \
                or start_positions.shape != (b,):
            raise ValueError("keep_tokens takes block_tables [B, max_blocks], start_positions [B], path [B, T], counts [B]")
        if any(t.dtype.is_floating_point or t.dtype == torch.bool for t in (block_tables, start_positions, path, counts)):
            raise ValueError("block_tables, start_positions, path and counts must be whole numbers")
        if lens_out is not None and (lens_out.dtype != torch.int32 or lens_out.shape != (b,) or not lens_out.is_contiguous()):
            raise ValueError("lens_out must be a contiguous int32 tensor [B]")
        if b == 0:
            return
        self._ensure_pools()
        k, v = self._k_pool, self._v_pool
        if self.device.type != "cuda":
            self._keep_on_host(block_tables, start_positions, path, counts, lens_out)
            return
        device = k.device
        if any(t.device != device for t in (block_tables, start_positions, path, counts) + (
                () if lens_out is None else (lens_out,))):
            raise ValueError("keep_tokens takes tensors on the pool's device")
        tables = block_tables if block_tables.dtype == torch.int32 and block_tables.stride(1) == 1 \
            else block_tables.to(torch.int32).contiguous()
        path = path if path.dtype == torch.int32 and path.stride(1) == 1 else path.to(torch.int32).contiguous()
        starts, counts = (t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()
                          for t in (start_positions, counts))
        s, size = self.shape, k.element_size()
        with _hip.on_device(device):
            _hip.check(_hip.load().mx_kv_keep_tokens(
                k.data_ptr(), v.data_ptr(), s.head_dim * size, k.stride(0) * size, k.stride(1) * size, k.stride(2) * size,
                s.num_layers, s.num_kv_heads, s.block_size_tokens, s.num_blocks, tables.data_ptr(), tables.stride(0),
                tables.shape[1], starts.data_ptr(), path.data_ptr(), path.stride(0), counts.data_ptr(), b, path.shape[1],
                None if lens_out is None else lens_out.data_ptr(), self._write_err.data_ptr(),
                _hip.stream_handle(device)), "mx_kv_keep_tokens")

    def _keep_on_host(self, block_tables, start_positions, path, counts, lens_out) -> None:
        bs, width = self.block_size_tokens, int(path.shape[1])
        src, dst, lens = [], [], []
        for table, start, row, n in zip(block_tables.tolist(), start_positions.tolist(), path.tolist(), counts.tolist()):
            n = min(max(n, 0), width)
            lens.append(start + n)
            nodes = row[:n]
            if any(not a < b < width for a, b in zip([-1] + nodes, nodes)):
                raise IndexError("the path of a row does not rise within its nodes")
            for j, node in enumerate(nodes):
                for pos, out in ((start + node, src), (start + j, dst)) if node != j else ():
                    if pos < 0 or pos // bs >= len(table) or not 0 <= table[pos // bs] < self.shape.num_blocks:
                        raise IndexError("block table underrun or physical block id out of range during keep_tokens")
                    out.append((table[pos // bs], pos % bs))
        if src:
            (sp, so), (dp, do) = (torch.tensor(x).unbind(1) for x in (src, dst))
            for pool in (self._k_pool, self._v_pool):
                pool[:, dp, :, do] = pool[:, sp, :, so]
        if lens_out is not None:
            lens_out.copy_(torch.tensor(lens, dtype=torch.int32))

    def copy_blocks(self, src_block_ids: list[int], dst_block_ids: list[int]) -> None:
        """Copy full physical blocks (all layers) from src ids to dst ids (``:233-250``), every source as
        it was before the call; of several pairs with one destination the last counts."""
        if len(src_block_ids) != len(dst_block_ids):
            raise ValueError(f"copy_blocks length mismatch: src={len(src_block_ids)} dst={len(dst_block_ids)}")
        pairs = [(s, d) for s, d in zip(_ids(src_block_ids), _ids(dst_block_ids)) if s != d]
        self._touch_ids([i for pair in pairs for i in pair])
        if pairs:
            self._copy_pages(array.array("i", [s for s, _ in pairs]), array.array("i", [d for _, d in pairs]))

    def move_blocks(self, src_block_ids: list[int], dst_block_ids: list[int],
                    block_tables: torch.Tensor | None = None, out: torch.Tensor | None = None
                    ) -> torch.Tensor | None:
        """Move blocks (all layers) from src ids to dst ids, which leaves the src ids free: a pool's live
        blocks brought together. Returns ``block_tables`` (int32 ``[B, max_blocks]`` on the pool's device)
        with every src id replaced by its dst id, as a new tensor or in ``out`` (which may be
        ``block_tables`` itself). No id may occur twice, neither among nor between the two lists.
        """
        src, dst = list(src_block_ids), list(dst_block_ids)
        if len(src) != len(dst):
            raise ValueError(f"move_blocks length mismatch: src={len(src)} dst={len(dst)}")
        if block_tables is None:
            if out is not None:
                raise ValueError("out goes with block_tables")
        else:
            if (block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.stride(1) != 1
                    or block_tables.device != self._page_regions()[0].device):
                raise ValueError("block_tables must be int32 [B, max_blocks] with unit inner stride on the pool's device")
            if block_tables.numel() >= 1 << 31:  # before a page moves: the renaming launch takes no more
                raise ValueError("block_tables must have fewer than 2**31 entries")
            if out is None:
                out = torch.empty(block_tables.shape, dtype=torch.int32, device=block_tables.device)
            elif (out.dtype != torch.int32 or out.shape != block_tables.shape or out.stride(1) != 1
                  or out.device != block_tables.device):
                raise ValueError("out must be int32 of block_tables' shape, device and unit inner stride")
            elif _share_entries(block_tables, out):
                raise ValueError("out must be block_tables itself or share no entry with it, and have rows of its own")
        on_device = self.device.type == "cuda"
        if not on_device:
            self._check_move(src, dst)
        if src:
            try:
                a, b = array.array("i", src), array.array("i", dst)
                self._copy_pages(a, b, move=True)
            except (ValueError, OverflowError):
                self._check_move(src, dst)
                raise
            held = self._used_blocks.intersection(src)  # the device map's marks move with the pages
            if held:
                self._used_blocks.update([d for s, d in zip(src, dst) if s in held])
                self._used_blocks -= held
            if block_tables is not None:
                self._rename(block_tables, out, a, b)
        elif block_tables is not None and out is not block_tables:
            out.copy_(block_tables)
        return out

    def _check_move(self, src: list[int], dst: list[int]) -> None:
        for i in src + dst:
            if not 0 <= i < self.shape.num_blocks:
                raise IndexError(f"physical block id out of range: {i}")
        if len(set(src).union(dst)) != 2 * len(src):
            raise ValueError("move_blocks takes every block id once")

    def free_blocks(self, block_ids: list[int]) -> None:
        """Give blocks back: they no longer count as allocated (and an 8-bit pool's stand for 0). A block
        written on the device and freed before the counts are read is not seen by the peak."""
        ids = sorted(set(_ids(block_ids)))
        if ids and (ids[0] < 0 or ids[-1] >= self.shape.num_blocks):
            raise IndexError(f"physical block id out of range: {ids[0] if ids[0] < 0 else ids[-1]}")
        self._used_blocks.difference_update(ids)
        if not ids or self._used_map is None:
            return
        codes, dev = self._freed_codes(), self._used_map.device
        arr = array.array("i", ids)
        with _hip.on_device(dev):
            _hip.check(_hip.load().mx_kv_clear_pages(
                codes.data_ptr() if codes is not None else None, codes[0, 0].numel() if codes is not None else 0,
                codes.stride(0) if codes is not None else 0, self.shape.num_layers, self._used_map.data_ptr(),
                self.shape.num_blocks, arr.buffer_info()[0], len(ids), _hip.stream_handle(dev)),
                "mx_kv_clear_pages")

    def _freed_codes(self) -> torch.Tensor | None:
        """What a freed block's bytes are cleared in (uint8 ``[L, num_blocks, ...]``); nothing in 16 bits."""
        return None

    def _page_regions(self) -> list[torch.Tensor]:
        self._ensure_pools()
        return self._regions

    def _copy_pages(self, src: array.array, dst: array.array, move: bool = False) -> None:
        """Page dst[i] = page src[i] in every layer, all at once (the lists as ``move_blocks`` or
        ``copy_blocks`` takes them)."""
        regions = self._page_regions()
        if self.device.type == "cuda":
            args: list = []
            for t in (*regions, None)[:2]:
                args += [None, 0, 0] if t is None else [t.data_ptr(), t[0, 0].numel() * t.element_size(),
                                                        t.stride(0) * t.element_size()]
            dev = regions[0].device

            def copy(of: array.array, to: array.array) -> int:
                return _hip.load().mx_kv_copy_pages(
                    *args, self.shape.num_layers, self.shape.num_blocks, of.buffer_info()[0], to.buffer_info()[0],
                    len(of), self._used_map.data_ptr(), int(move), _hip.stream_handle(dev))

            with _hip.on_device(dev):
                rc = copy(src, dst)
                if rc == _hip.MX_ERR_UNSUPPORTED and not move:  # more copies that depend on each other than a launch takes
                    for of, to in dependent_batches(src, dst):
                        _hip.check(copy(array.array("i", of), array.array("i", to)), "mx_kv_copy_pages")
                else:
                    _hip.check(rc, "mx_kv_copy_pages")
            return
        last = dict(zip(dst, src))
        to = torch.tensor(list(last), device=self.device, dtype=torch.long)
        of = torch.tensor(list(last.values()), device=self.device, dtype=torch.long)
        for t in regions:
            t[:, to] = t[:, of]

    def _rename(self, tables: torch.Tensor, out: torch.Tensor, src: array.array, dst: array.array) -> None:
        if self.device.type != "cuda":
            name = dict(zip(src, dst))
            out.copy_(torch.tensor([[name.get(i, i) for i in row] for row in tables.tolist()],
                                   dtype=torch.int32).view(tables.shape))
            return
        with _hip.on_device(tables.device):
            _hip.check(_hip.load().mx_kv_rename_pages(
                tables.data_ptr(), tables.stride(0), out.data_ptr(), out.stride(0), tables.shape[0], tables.shape[1],
                src.buffer_info()[0], dst.buffer_info()[0], len(src), _hip.stream_handle(tables.device)),
                "mx_kv_rename_pages")

    def gather_layer(self, layer_idx: int, block_ids: list[int], seq_len: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Gather one row as ``[1, Hkv, seq_len, D]`` (prefill / parity, ``:252-283``)."""
        if seq_len <= 0:
            raise ValueError("seq_len must be positive")
        bs = self.block_size_tokens
        n_logical = math.ceil(seq_len / bs)
        if n_logical > len(block_ids):
            raise IndexError("block table underrun during gather")
        self._ensure_pools()
        ids_list = [int(b) for b in list(block_ids)[:n_logical]]
        self._touch_ids(ids_list)
        if self._gathers_on_device(seq_len):
            table = torch.tensor([ids_list], dtype=torch.int32).to(self.device)
            return self._gather_table(layer_idx, table, seq_len)
        assert self._k_pool is not None and self._v_pool is not None
        ids = torch.tensor(ids_list, device=self.device, dtype=torch.long)
        s = self.shape
        k = self._k_pool[layer_idx, ids].permute(1, 0, 2, 3).reshape(s.num_kv_heads, n_logical * bs, s.head_dim)
        v = self._v_pool[layer_idx, ids].permute(1, 0, 2, 3).reshape(s.num_kv_heads, n_logical * bs, s.head_dim)
        return k[:, :seq_len].unsqueeze(0), v[:, :seq_len].unsqueeze(0)

    def _gather_table(self, layer_idx: int, table: torch.Tensor, tokens: int, seq_lens: torch.Tensor | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows of a device table (ids checked by the caller) as ``[B, Hkv, tokens, D]``, one launch."""
        from .decode_glue import kv_gather

        return kv_gather(self.k_layer_view(layer_idx), self.v_layer_view(layer_idx), table, tokens, seq_lens)

    def gather_layer_batch(self, layer_idx: int, block_tables: torch.Tensor, seq_lens: torch.Tensor
                           ) -> tuple[torch.Tensor, torch.Tensor]:
        """Gather rows as zero-padded ``[B, Hkv, max_seq, D]`` (batched prefill, ``:285-309``)."""
        batch_size = int(block_tables.shape[0])
        lens = [int(x) for x in seq_lens.tolist()]
        max_seq = max(lens) if lens else 0
        if max_seq <= 0:
            raise ValueError("seq_len must be positive")
        if len(lens) < batch_size:
            raise IndexError(f"{batch_size} block-table rows but {len(lens)} lengths")
        if self._gathers_on_device(max_seq):
            for row, n in zip(block_tables.tolist(), lens):
                if n <= 0:
                    raise ValueError("seq_len must be positive")
                n_logical = math.ceil(n / self.block_size_tokens)
                if n_logical > len(row):
                    raise IndexError("block table underrun during gather")
                self._touch_ids([int(i) for i in row[:n_logical]])
            return self._gather_table(layer_idx, block_tables, max_seq, seq_lens[:batch_size])
        s = self.shape
        keys = torch.zeros(batch_size, s.num_kv_heads, max_seq, s.head_dim, device=self.device, dtype=self.dtype)
        values = torch.zeros_like(keys)
        for b in range(batch_size):
            n_logical = math.ceil(lens[b] / self.block_size_tokens)
            row_ids = [int(x) for x in block_tables[b, :n_logical].tolist()]
            k, v = self.gather_layer(layer_idx, row_ids, lens[b])
            keys[b, :, : lens[b]] = k[0]
            values[b, :, : lens[b]] = v[0]
        return keys, values

    def reset(self) -> None:
        self._k_pool = None
        self._v_pool = None
        self._k_views = self._v_views = ()
        self._regions = []
        self._used_map = None
        self._write_err = None
        self._used_blocks.clear()
        self._peak_allocated_blocks = 0
