"""A block pool whose K and V are held in 8 bits: :class:`Int8KVBlockPool`.

It stands where a :class:`GpuKVBlockPool` does: the cache adapters (``paged_kv_cache.py``), the attention
hook and ``paged_attention_decode_batched`` (``runtime/phase2/paged_attention_triton.py:745-775``), the HF
decode loop and ``Int8DecodeModel.step`` take either. It holds the same tokens in half the bytes (and one
byte per page and head), so a decode step's attention reads half of them; ``dtype`` is the 16-bit type of
the states written and of the rows read back.

Differences from the 16-bit pool:

* device memory only: there is no CPU form;
* ``k_layer_view`` / ``v_layer_view`` raise ``ValueError`` (no 16-bit K or V exists to view);
  :meth:`layer_store` gives a layer's bytes and codes, ``gather_layer`` its rows in 16 bits;
* a write that begins inside a page keeps the tokens before it and drops what stood behind it; the kept
  ones may be rounded to a larger scale (``kv8.py``), so a prompt written at once and one written token by
  token can differ by a step;
* :meth:`check_write_errors` also reports a block id outside the pool that attention met.
"""

from __future__ import annotations

import torch

from .kv8 import BLOCK_SIZES, HEAD_DIMS, Kv8Layer, kv8_append, kv8_attention_decode, kv8_gather
from .paged_attention_hip import _DTYPE_FLAGS
from .paged_kv_kernel import GpuKVBlockPool, _alloc_lock, settle

ZERO_BYTE = 128  # q = 0


class Int8KVBlockPool(GpuKVBlockPool):
    """The 8-bit form of :class:`GpuKVBlockPool`; same constructor (without ``kv_layout``) and methods."""

    kv_bits = 8

    def __init__(self, *, num_blocks: int, block_size_tokens: int, num_layers: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype, device: str | torch.device) -> None:
        super().__init__(num_blocks=num_blocks, block_size_tokens=block_size_tokens, num_layers=num_layers,
                         num_kv_heads=num_kv_heads, head_dim=head_dim, dtype=dtype, device=device)
        if dtype not in _DTYPE_FLAGS:
            raise ValueError(f"an 8-bit pool holds fp16 or bf16 values, got {dtype}")
        if head_dim not in HEAD_DIMS or block_size_tokens not in BLOCK_SIZES:
            raise ValueError(f"an 8-bit pool needs head_dim in {HEAD_DIMS} and block_size_tokens in {BLOCK_SIZES}, got "
                             f"{head_dim} and {block_size_tokens}")
        if self.device.type != "cuda":
            raise ValueError(f"an 8-bit pool lives on a ROCm device (got {self.device}); it has no CPU form")
        self._data: torch.Tensor | None = None
        self._codes: torch.Tensor | None = None
        self._stores: list[Kv8Layer] = []

    def bytes_per_block(self) -> int:
        s = self.shape
        return s.num_layers * s.num_kv_heads * 2 * (s.block_size_tokens * s.head_dim + 1)

    def _ensure_pools(self) -> None:
        if self._data is None:
            with _alloc_lock:
                if self._data is None:
                    self._make_pools()

    def _make_pools(self) -> None:
        s = self.shape
        run = s.block_size_tokens * s.head_dim
        data = torch.full((s.num_layers, s.num_blocks, s.num_kv_heads, 2, run), ZERO_BYTE, dtype=torch.uint8,
                          device=self.device)
        codes = torch.zeros((s.num_layers, s.num_blocks, s.num_kv_heads, 2), dtype=torch.uint8, device=self.device)
        self._used_map = torch.zeros(s.num_blocks, dtype=torch.uint8, device=self.device)
        self._write_err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._stores = [Kv8Layer(data[i], codes[i], s.block_size_tokens, s.head_dim, self.dtype)
                        for i in range(s.num_layers)]
        settle(data.device)
        self._codes, self._data = codes, data

    def layer_store(self, layer_idx: int) -> Kv8Layer:
        """A layer's pages as the functions of ``kv8.py`` take them."""
        self._ensure_pools()
        return self._stores[layer_idx]

    def k_layer_view(self, layer_idx: int) -> torch.Tensor:
        raise ValueError("an 8-bit pool has no 16-bit K to view; use layer_store or gather_layer")

    def v_layer_view(self, layer_idx: int) -> torch.Tensor:
        raise ValueError("an 8-bit pool has no 16-bit V to view; use layer_store or gather_layer")

    def check_write_errors(self) -> None:
        """Raise ``IndexError`` if a write or an attention call met a slot outside its block table or the
        pool since the last check (one host sync); the error word is cleared."""
        if self._write_err is None:
            return
        bits = int(self._write_err.item())
        if bits:
            self._write_err.zero_()
            where = " and ".join(name for name, hit in (("batched write", bits & ~4), ("attention", bits & 4)) if hit)
            raise IndexError(f"block table underrun or physical block id out of range during {where}")

    def write_tokens_batch(self, layer_idx: int, block_tables: torch.Tensor, start_positions: torch.Tensor,
                           key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """KV write: tables ``[B, max_blocks]``, starts ``[B]``, states ``[B, Hkv, kv_len, D]``; one launch,
        no host sync (``sync_write_checks`` as in the 16-bit pool)."""
        if key_states.shape != value_states.shape:
            raise ValueError("key_states and value_states must match shape")
        batch_size = int(key_states.shape[0])
        if block_tables.shape[0] != batch_size or start_positions.shape[0] != batch_size:
            raise ValueError("batch dimension mismatch in write_tokens_batch")
        if key_states.shape[-2] == 0 or batch_size == 0:
            return
        if key_states.dtype != self.dtype or value_states.dtype != self.dtype:
            key_states, value_states = key_states.to(self.dtype), value_states.to(self.dtype)
        kv8_append(self.layer_store(layer_idx), block_tables, start_positions, key_states, value_states,
                   err=self._write_err, used_blocks=self._used_map)
        if self.sync_write_checks and not torch.cuda.is_current_stream_capturing():
            self.check_write_errors()

    def attend(self, layer_idx: int, query: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
               scaling: float, num_kv_groups: int, shared_blocks: bool = False) -> torch.Tensor:
        """One decode step's attention over a layer (``kv8_attention_decode``); a block id outside the pool
        is reported by :meth:`check_write_errors`."""
        return kv8_attention_decode(query, self.layer_store(layer_idx), block_tables, seq_lens, scaling,
                                    num_kv_groups, err=self._write_err, shared_blocks=shared_blocks)

    def _gathers_on_device(self, tokens: int) -> bool:
        return True

    def _gather_table(self, layer_idx: int, table: torch.Tensor, tokens: int, seq_lens: torch.Tensor | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor]:
        return kv8_gather(self.layer_store(layer_idx), table, tokens, seq_lens)

    def _page_regions(self) -> list[torch.Tensor]:
        self._ensure_pools()
        return [self._data, self._codes]

    def _freed_codes(self) -> torch.Tensor | None:
        return self._codes

    def reset(self) -> None:
        super().reset()
        self._data = None
        self._codes = None
        self._stores = []
