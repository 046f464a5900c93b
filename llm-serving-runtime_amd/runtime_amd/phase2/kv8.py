"""Host wrappers of the 8-bit KV cache's kernels: write, read back, rotary + write, decode attention.

The cache holds K and V of a page (a block and kv-head) as 8-bit ``q`` in [-127, 127] and one power of
two as their scale (the format is in ``include/mxdecode.h``); :class:`~.kv8_pool.Int8KVBlockPool` owns
its tensors and hands out a layer as :class:`Kv8Layer`. A decode step reads half the bytes of the 16-bit
pool; a value is off by at most half a scale step when it is written (an fp16 magnitude above 65280, where the
scale is at its cap of 2**9, by at most 480), and by less than one step of the page's last scale however often
that grows while tokens are appended.

* :func:`kv8_append` - new K/V states into a layer's pages (the 8-bit form of ``kv_append``);
* :func:`kv8_rope_append` - a decode step's fused QKV rows: q rotated out, k and v into their pages
  (of ``qkv_rope_append`` and ``qkv_rope_append_splits``);
* :func:`kv8_gather` - whole rows back in 16 bits, exactly the values that the pages stand for (of
  ``kv_gather``);
* :func:`kv8_attention_decode` - one decode step's attention (of ``mx_paged_attn_decode``).

All take device tensors and enqueue on the current stream of the cache's device; no call synchronises.
Errors raise ``ValueError`` (bad arguments) or ``RuntimeError``. A page must not stand in two rows'
written ranges of one call. What a page holds behind the tokens of the last write to it is lost.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import _hip
from .decode_glue import _i32, _lens_ptr, _used_ptr
from .paged_attention_hip import _DTYPE_FLAGS, MX_PA_SHARED_BLOCKS

HEAD_DIMS = (64, 128)
BLOCK_SIZES = (4, 8, 16, 32)


@dataclass(frozen=True, eq=False)
class Kv8Layer:
    """One layer's pages: ``data`` uint8 ``[num_blocks, Hkv, 2, bs * D]`` and ``codes`` uint8
    ``[num_blocks, Hkv, 2]``, contiguous; ``dtype`` is the 16-bit type their values are numbers of."""

    data: torch.Tensor
    codes: torch.Tensor
    block_size: int
    head_dim: int
    dtype: torch.dtype
    num_blocks: int = field(init=False)
    num_kv_heads: int = field(init=False)
    device: torch.device = field(init=False)
    pointers: tuple[int, int] = field(init=False)  # of data and codes
    flags: int = field(init=False)                 # MX_PA_BF16 or 0

    def __post_init__(self) -> None:
        data, codes = self.data, self.codes
        if self.dtype not in _DTYPE_FLAGS:
            raise ValueError(f"an 8-bit cache layer stands for fp16 or bf16 values, got {self.dtype}")
        if self.head_dim not in HEAD_DIMS or self.block_size not in BLOCK_SIZES:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS} and block_size one of {BLOCK_SIZES}, got "
                             f"{self.head_dim} and {self.block_size}")
        if (data.dtype != torch.uint8 or data.dim() != 4 or data.shape[2:] != (2, self.block_size * self.head_dim)
                or not data.is_contiguous()):
            raise ValueError("data must be contiguous uint8 [num_blocks, Hkv, 2, block_size * head_dim]")
        if codes.dtype != torch.uint8 or codes.shape != data.shape[:3] or not codes.is_contiguous():
            raise ValueError("codes must be contiguous uint8 [num_blocks, Hkv, 2]")
        if codes.device != data.device:
            raise ValueError("data and codes must be on one device")
        _hip.require_device_tensor(data, "data")
        object.__setattr__(self, "num_blocks", int(data.shape[0]))
        object.__setattr__(self, "num_kv_heads", int(data.shape[1]))
        object.__setattr__(self, "device", data.device)
        object.__setattr__(self, "pointers", (data.data_ptr(), codes.data_ptr()))
        object.__setattr__(self, "flags", _DTYPE_FLAGS[self.dtype])


def _tables(block_tables: torch.Tensor, rows: int, device: torch.device) -> torch.Tensor:
    if block_tables.dim() != 2 or block_tables.shape[0] != rows:
        raise ValueError("block_tables must be [B, max_blocks]")
    if block_tables.dtype != torch.int32 or block_tables.device != device or block_tables.stride(1) != 1:
        block_tables = block_tables.to(device=device, dtype=torch.int32).contiguous()
    return block_tables


def _lengths(t: torch.Tensor, rows: int, device: torch.device) -> torch.Tensor:
    """``rows`` lengths or positions as contiguous int32 on the device."""
    t = _i32(t if t.dim() == 1 else t.reshape(-1), device)
    if t.shape[0] != rows:
        raise ValueError(f"{rows} rows but {t.shape[0]} lengths or positions")
    return t


def _err_ptr(err: torch.Tensor | None, device: torch.device):
    if err is None:
        return None
    if err.dtype != torch.int32 or err.numel() < 1 or err.device != device:
        raise ValueError("err must be an int32 tensor on the cache's device")
    return err.data_ptr()


def _strides(t: torch.Tensor) -> tuple[int, int, int] | None:
    """(row, head, token) strides of ``[B, H, T, D]`` states the kernel reads with 16-byte loads (0 for
    a dimension of one, whose stride may be anything), or None."""
    (b, h, n, _), (sb, sh, st, unit) = t.shape, t.stride()
    out = (sb if b > 1 else 0, sh if h > 1 else 0, st if n > 1 else 0)
    return None if unit != 1 or t.data_ptr() % 16 or out[0] % 8 or out[1] % 8 or out[2] % 8 else out


def kv8_append(layer: Kv8Layer, block_tables: torch.Tensor, start_pos: torch.Tensor, key_states: torch.Tensor,
               value_states: torch.Tensor, err: torch.Tensor | None = None,
               used_blocks: torch.Tensor | None = None) -> None:
    """Write ``key/value_states [B, Hkv, T, D]`` at positions ``start_pos[b] + t`` of each row.

    A write that begins inside a page keeps the tokens before it (the page's scale only grows); one
    that begins at a page's first slot starts it anew. Slots outside the table or the pool are skipped
    and flagged in ``err`` (an int32 device word, OR-ed with 1) when given; ``used_blocks`` (uint8
    ``[num_blocks]``, optional) gets 1 at every block a token was written to.
    """
    _hip.require_device_tensor(key_states, "key_states")
    _hip.require_device_tensor(value_states, "value_states")
    dev = layer.device
    if key_states.shape != value_states.shape or key_states.dim() != 4:
        raise ValueError("key_states and value_states must both be [B, Hkv, T, D]")
    b, hkv, t, d = key_states.shape
    if key_states.dtype != layer.dtype or value_states.dtype != layer.dtype:
        raise ValueError(f"the cache takes {layer.dtype} states, got {key_states.dtype} and {value_states.dtype}")
    if (hkv, d) != (layer.num_kv_heads, layer.head_dim):
        raise ValueError("states do not match the cache's heads and head_dim")
    if key_states.device != dev or value_states.device != dev:
        raise ValueError("states must be on the cache's device")
    starts = _lengths(start_pos, b, dev)
    tables = _tables(block_tables, b, dev)
    strides = _strides(key_states)
    if strides is None or strides != _strides(value_states):
        key_states, value_states = key_states.contiguous(), value_states.contiguous()
        if key_states.data_ptr() % 16 or value_states.data_ptr() % 16:
            key_states, value_states = key_states.clone(), value_states.clone()
        strides = _strides(key_states)
    with _hip.on_device(dev):
        rc = _hip.load().mx_kv8_write(
            key_states.data_ptr(), value_states.data_ptr(), *strides, b, t, hkv, d, tables.data_ptr(),
            tables.stride(0), tables.shape[1], starts.data_ptr(), *layer.pointers,
            layer.block_size, layer.num_blocks, _err_ptr(err, dev), _used_ptr(used_blocks, layer.num_blocks, dev),
            layer.flags, _hip.stream_handle(dev))
    if rc != _hip.MX_OK:
        _hip.check(rc, "mx_kv8_write")


def kv8_gather(layer: Kv8Layer, block_tables: torch.Tensor, tokens: int, seq_lens: torch.Tensor | None = None,
               err: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The first ``tokens`` tokens of each row of ``block_tables [B, max_blocks]``: K and V as contiguous
    ``[B, Hkv, tokens, D]`` of the layer's dtype, zero past ``seq_lens[b]`` when given and where a block
    is outside the table or the pool (flagged in ``err``)."""
    dev = layer.device
    b = int(block_tables.shape[0]) if block_tables.dim() == 2 else -1
    tables = _tables(block_tables, b, dev)
    lens = _lengths(seq_lens, b, dev) if seq_lens is not None else None
    if tokens < 0:
        raise ValueError("tokens must be >= 0")
    k = torch.empty((b, layer.num_kv_heads, tokens, layer.head_dim), dtype=layer.dtype, device=dev)
    v = torch.empty_like(k)
    with _hip.on_device(dev):
        rc = _hip.load().mx_kv8_gather(
            *layer.pointers, tables.data_ptr(), tables.stride(0), tables.shape[1],
            lens.data_ptr() if lens is not None else None, b, tokens, layer.num_kv_heads, layer.head_dim,
            layer.block_size, layer.num_blocks, k.data_ptr(), v.data_ptr(), _err_ptr(err, dev),
            layer.flags, _hip.stream_handle(dev))
    if rc != _hip.MX_OK:
        _hip.check(rc, "mx_kv8_gather")
    return k, v


def kv8_rope_append(qkv: torch.Tensor | None, rope: torch.Tensor, positions: torch.Tensor, q_out: torch.Tensor,
                    layer: Kv8Layer, block_tables: torch.Tensor, num_heads: int, *,
                    partials: torch.Tensor | None = None, splits: int = 0, bias: torch.Tensor | None = None,
                    err: torch.Tensor | None = None, lens_out: torch.Tensor | None = None,
                    used_blocks: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q, k of ``qkv [B, (Hq + 2 Hkv) * D]`` at ``positions [B]``; q -> ``q_out``, k, v -> the cache.

    With ``qkv=None`` the rows are the projection's fp32 split ``partials [splits, B, width]`` plus
    ``bias`` (``int8_linear_partials``), rounded as its own output would be. ``rope`` is the fp32
    ``[max_pos, D/2, 2]`` table of ``rope_table``. ``lens_out`` (int32 ``[B]``, optional) receives
    ``positions + 1``; ``err`` is OR-ed with 1 (a slot outside the table or the pool, skipped) or 2 (a
    position outside ``rope``: zeros in ``q_out``, nothing written).
    """
    dev, d, hkv = layer.device, layer.head_dim, layer.num_kv_heads
    width = (num_heads + 2 * hkv) * d
    if (qkv is None) == (partials is None):
        raise ValueError("give exactly one of qkv and partials")
    _hip.require_device_tensor(q_out, "q_out")
    if q_out.dim() < 2 or q_out.dtype != layer.dtype or q_out.device != dev or q_out.shape[-1] != num_heads * d:
        raise ValueError("q_out must be [B, Hq * D] of the cache's dtype and device")
    q2 = q_out if q_out.dim() == 2 else q_out.view(-1, num_heads * d)
    b = int(q2.shape[0])
    if q2.stride(1) != 1 or (b > 1 and q2.stride(0) < num_heads * d):
        raise ValueError("q_out must have rows of their own with unit stride")
    x = None
    if qkv is not None:
        _hip.require_device_tensor(qkv, "qkv")
        if qkv.shape[-1] != width or qkv.dtype != layer.dtype or qkv.device != dev:
            raise ValueError("qkv must be [B, (Hq + 2 Hkv) * D] of the cache's dtype and device")
        x = qkv if qkv.dim() == 2 else qkv.reshape(-1, width)
        if x.stride(1) != 1:
            x = x.contiguous()
        if x.shape[0] != b:
            raise ValueError("batch dimension mismatch")
    else:
        _hip.require_device_tensor(partials, "partials")
        if (partials.dtype != torch.float32 or not partials.is_contiguous() or splits < 1
                or partials.numel() < splits * b * width or partials.device != dev):
            raise ValueError("partials must be contiguous fp32 [splits, B, (Hq + 2 Hkv) * D]")
    if bias is not None and (partials is None or bias.dtype != layer.dtype or bias.numel() != width
                             or not bias.is_contiguous() or bias.device != dev):
        raise ValueError("bias goes with partials: (Hq + 2 Hkv) * D entries of the cache's dtype")
    if (rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[1:] != (d // 2, 2) or not rope.is_contiguous()
            or rope.device != dev):
        raise ValueError("rope must be a contiguous fp32 [max_pos, D/2, 2] table")
    pos = _lengths(positions, b, dev)
    if lens_out is not None and (lens_out.device != dev or abs(lens_out.data_ptr() - pos.data_ptr()) < 4 * b):
        raise ValueError("lens_out must be on the cache's device and not the positions themselves")
    tables = _tables(block_tables, b, dev)
    with _hip.on_device(dev):
        rc = _hip.load().mx_kv8_rope_append(
            x.data_ptr() if x is not None else None, x.stride(0) if x is not None else 0,
            partials.data_ptr() if partials is not None else None, splits, bias.data_ptr() if bias is not None else None,
            b, num_heads, hkv, d, rope.data_ptr(), rope.shape[0], pos.data_ptr(), q2.data_ptr(), q2.stride(0),
            tables.data_ptr(), tables.stride(0), tables.shape[1], *layer.pointers,
            layer.block_size, layer.num_blocks, _err_ptr(err, dev), _lens_ptr(lens_out, b),
            _used_ptr(used_blocks, layer.num_blocks, dev), layer.flags, _hip.stream_handle(dev))
    if rc != _hip.MX_OK:
        _hip.check(rc, "mx_kv8_rope_append")
    return q_out


def _aligned_heads(t: torch.Tensor) -> bool:
    """Whether ``t [B, H, 1, D]`` has 16-byte aligned rows (a dimension of one may have any stride)."""
    (b, h, _, _), (sb, sh, _, unit) = t.shape, t.stride()
    return unit == 1 and t.data_ptr() % 16 == 0 and (b == 1 or sb % 8 == 0) and (h == 1 or sh % 8 == 0)


def kv8_attention_decode(query: torch.Tensor, layer: Kv8Layer, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                         scaling: float, num_kv_groups: int, out: torch.Tensor | None = None,
                         err: torch.Tensor | None = None, shared_blocks: bool = False) -> torch.Tensor:
    """``query [B, heads, 1, dim]`` against each row's first ``seq_lens[b]`` cached tokens.

    Rows of length 0 give zeros. A block id outside the pool is skipped and OR-s 4 into ``err`` (an
    int32 device word) when given. ``shared_blocks`` says that rows may share pages (the loads then keep
    them in the caches; the result is the same). A page that a value not finite was written to makes the outputs of
    its heads NaN.
    """
    _hip.require_device_tensor(query, "query")
    if query.dim() != 4 or query.shape[2] != 1:
        raise ValueError("paged decode expects a query [B, heads, 1, dim]")
    b, hq, _, d = query.shape
    dev, hkv = layer.device, layer.num_kv_heads
    if query.dtype != layer.dtype or query.device != dev:
        raise ValueError(f"query must be {layer.dtype} on {dev}, got {query.dtype} on {query.device}")
    if d != layer.head_dim:
        raise ValueError(f"head_dim mismatch: query {d} vs cache {layer.head_dim}")
    if hq != hkv * num_kv_groups:
        raise ValueError(f"num_heads {hq} != num_kv_heads {hkv} * num_kv_groups {num_kv_groups}")
    tables = _tables(block_tables, b, dev)
    lens = _lengths(seq_lens, b, dev)
    if not _aligned_heads(query):
        query = query.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty((b, hq, 1, d), dtype=query.dtype, device=dev)
    elif tuple(out.shape) != (b, hq, 1, d) or out.dtype != query.dtype or out.device != dev or not _aligned_heads(out):
        raise ValueError("out must be a [B, heads, 1, dim] tensor of the query dtype with 16-byte aligned rows")
    if b == 0:
        return out
    width = int(tables.shape[1])
    nbytes = _hip.kv8_attn_workspace_bytes(b, hq, hkv, d, width, layer.block_size)
    # The workspace is the call's own: the caching allocator gives calls on other streams, and graphs
    # being captured, memory of theirs.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    (q_sb, q_sh, _, _), (o_sb, o_sh, _, _) = query.stride(), out.stride()
    one_row, one_head = b == 1, hq == 1
    with _hip.on_device(dev):
        rc = _hip.load().mx_kv8_attn_decode(
            query.data_ptr(), 0 if one_row else q_sb, 0 if one_head else q_sh, *layer.pointers, tables.data_ptr(),
            tables.stride(0), width, lens.data_ptr(), b, hq, hkv, d,
            layer.block_size, layer.num_blocks, float(scaling), out.data_ptr(), 0 if one_row else o_sb,
            0 if one_head else o_sh, ws.data_ptr() if ws is not None else None, nbytes, _err_ptr(err, dev),
            layer.flags | (MX_PA_SHARED_BLOCKS if shared_blocks else 0), _hip.stream_handle(dev))
    if rc != _hip.MX_OK:
        _hip.check(rc, "mx_kv8_attn_decode")
    return out
