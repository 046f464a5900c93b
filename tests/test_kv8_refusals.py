"""CPU checks of the 8-bit cache's and the page operators' arguments: every refusal comes before a launch."""

from __future__ import annotations

import array
import ctypes

import pytest
import torch

from runtime_amd.phase2 import _hip
from runtime_amd.phase2.kv8 import Kv8Layer, kv8_append, kv8_attention_decode, kv8_gather, kv8_rope_append
from runtime_amd.phase2.kv8_pool import Int8KVBlockPool
from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
OFF = ctypes.c_void_p(4098)


def _status(rc: int, expected: int) -> None:
    assert rc == expected, (rc, _hip.load().mx_last_error())
    assert _hip.load().mx_last_error().decode()


def _write(k=FAKE, v=FAKE, sb=2048, sh=1024, st=64, B=1, T=3, hkv=2, d=64, bt=FAKE, mb=4, start=FAKE, data=FAKE,
           codes=FAKE, bs=16, nb=8, flags=0):
    return _hip.load().mx_kv8_write(k, v, sb, sh, st, B, T, hkv, d, bt, 4, mb, start, data, codes, bs, nb, None, None,
                                    flags, None)


def _gather(data=FAKE, codes=FAKE, bt=FAKE, mb=4, B=1, S=3, hkv=2, d=64, bs=16, nb=8, out=FAKE, flags=0):
    return _hip.load().mx_kv8_gather(data, codes, bt, 4, mb, None, B, S, hkv, d, bs, nb, out, out, None, flags, None)


def _token(qkv=FAKE, part=None, splits=0, B=1, hq=4, hkv=2, d=64, rope=FAKE, max_pos=64, pos=FAKE, q=FAKE, bt=FAKE,
           mb=4, data=FAKE, codes=FAKE, bs=16, nb=8, flags=0):
    return _hip.load().mx_kv8_rope_append(qkv, 512, part, splits, None, B, hq, hkv, d, rope, max_pos, pos, q, 256, bt, 4,
                                          mb, data, codes, bs, nb, None, None, None, flags, None)


def _attend(q=FAKE, q_sb=256, q_sh=64, data=FAKE, codes=FAKE, bt=FAKE, mb=4, lens=FAKE, B=1, hq=4, hkv=2, d=64, bs=16,
            nb=8, out=FAKE, o_sh=64, ws=FAKE, wsb=1 << 40, flags=0):
    return _hip.load().mx_kv8_attn_decode(q, q_sb, q_sh, data, codes, bt, 4, mb, lens, B, hq, hkv, d, bs, nb, 0.125, out,
                                          256, o_sh, ws, wsb, None, flags, None)


@pytest.mark.parametrize("call", [_write, _gather, _token, _attend])
def test_entry_points_refuse_bad_arguments(call):
    assert call(B=0) == _hip.MX_OK
    _status(call(B=-1), _hip.MX_ERR_INVALID)
    _status(call(data=None), _hip.MX_ERR_NULL)
    _status(call(codes=None), _hip.MX_ERR_NULL)
    _status(call(bt=None), _hip.MX_ERR_NULL)
    _status(call(data=OFF), _hip.MX_ERR_ALIGNMENT)
    for d in (0, 32, 96, 256):
        _status(call(d=d), _hip.MX_ERR_UNSUPPORTED)
    for bs in (0, 2, 12, 64):
        _status(call(bs=bs), _hip.MX_ERR_UNSUPPORTED)
    _status(call(hkv=0), _hip.MX_ERR_INVALID)
    _status(call(nb=0), _hip.MX_ERR_INVALID)
    _status(call(mb=0), _hip.MX_ERR_INVALID)
    _status(call(flags=4), _hip.MX_ERR_INVALID)


def test_entry_points_refuse_what_is_theirs():
    assert _write(T=0) == _hip.MX_OK and _gather(S=0) == _hip.MX_OK
    _status(_write(T=-1), _hip.MX_ERR_INVALID)
    _status(_write(k=None), _hip.MX_ERR_NULL)
    _status(_write(start=None), _hip.MX_ERR_NULL)
    _status(_write(v=OFF), _hip.MX_ERR_ALIGNMENT)
    for stride in ("sb", "sh", "st"):
        _status(_write(**{stride: 68}), _hip.MX_ERR_ALIGNMENT)
    _status(_write(B=1 << 30, T=1 << 30), _hip.MX_ERR_UNSUPPORTED)
    _status(_write(B=1 << 25, T=1), _hip.MX_ERR_UNSUPPORTED)  # 2**27 waves: 2**33 threads
    _status(_gather(S=-1), _hip.MX_ERR_INVALID)
    _status(_gather(out=None), _hip.MX_ERR_NULL)
    _status(_gather(out=OFF), _hip.MX_ERR_ALIGNMENT)
    _status(_gather(B=1 << 30, S=1 << 30), _hip.MX_ERR_UNSUPPORTED)
    _status(_gather(B=1 << 26, S=1), _hip.MX_ERR_UNSUPPORTED)
    _status(_token(qkv=None), _hip.MX_ERR_INVALID)
    _status(_token(part=FAKE, splits=2), _hip.MX_ERR_INVALID)  # both sources
    _status(_token(qkv=None, part=FAKE, splits=0), _hip.MX_ERR_INVALID)
    _status(_token(rope=None), _hip.MX_ERR_NULL)
    _status(_token(rope=ctypes.c_void_p(4100)), _hip.MX_ERR_ALIGNMENT)
    _status(_token(hq=0), _hip.MX_ERR_INVALID)
    _status(_token(max_pos=0), _hip.MX_ERR_INVALID)
    _status(_token(B=1 << 28), _hip.MX_ERR_UNSUPPORTED)
    _status(_attend(hq=5), _hip.MX_ERR_INVALID)
    _status(_attend(lens=None), _hip.MX_ERR_NULL)
    _status(_attend(q=OFF), _hip.MX_ERR_ALIGNMENT)
    _status(_attend(q_sh=60), _hip.MX_ERR_ALIGNMENT)
    _status(_attend(o_sh=68), _hip.MX_ERR_ALIGNMENT)
    _status(_attend(B=65536), _hip.MX_ERR_UNSUPPORTED)
    _status(_attend(codes=ctypes.c_void_p(4097)), _hip.MX_ERR_ALIGNMENT)
    _status(_attend(mb=1 << 27), _hip.MX_ERR_UNSUPPORTED)           # 2**31 tokens in a row
    _status(_attend(mb=1 << 20, B=1024, hkv=4), _hip.MX_ERR_UNSUPPORTED)  # 2**32 chunks
    # A wide table shares rows out between waves: room for their pieces, aligned, is asked for.
    need = _hip.load().mx_kv8_attn_workspace_bytes(1, 4, 2, 64, 4096, 16)
    assert need == 2 * 2048 * 2 * (64 + 2) * 4
    _status(_attend(mb=4096, ws=None, wsb=0), _hip.MX_ERR_WORKSPACE)
    _status(_attend(mb=4096, wsb=need - 1), _hip.MX_ERR_WORKSPACE)
    _status(_attend(mb=4096, ws=ctypes.c_void_p(4096 + 128)), _hip.MX_ERR_ALIGNMENT)
    assert _hip.load().mx_kv8_attn_workspace_bytes(1, 4, 2, 64, 4, 16) == 0
    assert _hip.load().mx_kv8_attn_workspace_bytes(1, 5, 2, 64, 4096, 16) == 0


def _arr(*ids):
    a = array.array("i", ids)
    return a, a.buffer_info()[0]


def test_page_entry_points_refuse_bad_arguments():
    lib = _hip.load()
    keep, ids = _arr(0, 1, 2)

    def copy(base=FAKE, pb=1024, ls=8192, base2=None, pb2=0, ls2=0, layers=2, pages=8, src=(0, 1), dst=(2, 3), move=0):
        (a, s), (b, d) = _arr(*src), _arr(*dst)
        return lib.mx_kv_copy_pages(base, pb, ls, base2, pb2, ls2, layers, pages, s, d, len(a), None, move, None)

    assert lib.mx_kv_copy_pages(FAKE, 1024, 8192, None, 0, 0, 2, 8, ids, ids, 0, None, 0, None) == _hip.MX_OK
    _status(lib.mx_kv_copy_pages(FAKE, 1024, 8192, None, 0, 0, 2, 8, None, ids, 1, None, 0, None), _hip.MX_ERR_NULL)
    _status(lib.mx_kv_copy_pages(FAKE, 1024, 8192, None, 0, 0, 2, 8, ids, ids, -1, None, 0, None), _hip.MX_ERR_INVALID)
    _status(copy(base=None), _hip.MX_ERR_NULL)
    _status(copy(base=OFF), _hip.MX_ERR_ALIGNMENT)
    _status(copy(ls=8200), _hip.MX_ERR_ALIGNMENT)
    _status(copy(pb=0), _hip.MX_ERR_INVALID)
    _status(copy(base2=FAKE, pb2=0), _hip.MX_ERR_INVALID)
    _status(copy(layers=0), _hip.MX_ERR_INVALID)
    _status(copy(layers=70000), _hip.MX_ERR_INVALID)
    _status(copy(src=(0, 8)), _hip.MX_ERR_INVALID)
    _status(copy(dst=(2, -1)), _hip.MX_ERR_INVALID)
    _status(copy(src=(0, 2), move=1), _hip.MX_ERR_INVALID)  # page 2 is a source and a destination
    n = 500  # one chain, longer than a launch takes
    _status(copy(src=range(n), dst=range(1, n + 1), pages=n + 1), _hip.MX_ERR_UNSUPPORTED)

    def rename(tables=FAKE, rows=2, width=4, of=(1, 2), to=(3, 4)):
        (a, s), (b, d) = _arr(*of), _arr(*to)
        return lib.mx_kv_rename_pages(tables, 4, FAKE, 4, rows, width, s, d, len(a), None)

    assert rename(rows=0) == _hip.MX_OK and rename(width=0) == _hip.MX_OK
    _status(rename(rows=-1), _hip.MX_ERR_INVALID)
    _status(rename(tables=None), _hip.MX_ERR_NULL)
    _status(rename(of=(1, 1)), _hip.MX_ERR_INVALID)
    _status(rename(of=(1, -1)), _hip.MX_ERR_INVALID)
    for src, dst in (((0, 0), (2, 3)), ((0, 1), (2, 2)), ((0, 1), (0, 2))):
        _status(copy(src=src, dst=dst, move=1), _hip.MX_ERR_INVALID)  # a page that occurs twice
    _status(rename(to=(3, 1)), _hip.MX_ERR_INVALID)
    _status(rename(rows=1 << 29, width=4), _hip.MX_ERR_UNSUPPORTED)
    many = (1 << 24) + 1  # refused before the lists are read
    _status(lib.mx_kv_rename_pages(FAKE, 4, FAKE, 4, 2, 4, ids, ids, many, None), _hip.MX_ERR_UNSUPPORTED)
    _status(lib.mx_kv_copy_pages(FAKE, 1024, 8192, None, 0, 0, 2, 8, ids, ids, many, None, 0, None), _hip.MX_ERR_UNSUPPORTED)
    assert lib.mx_kv_clear_pages(FAKE, 4, 64, 2, FAKE, 8, ids, 0, None) == _hip.MX_OK
    _status(lib.mx_kv_clear_pages(FAKE, 4, 64, 2, FAKE, 2, ids, 3, None), _hip.MX_ERR_INVALID)
    _status(lib.mx_kv_clear_pages(None, 4, 64, 2, None, 8, ids, 3, None), _hip.MX_ERR_NULL)
    _status(lib.mx_kv_clear_pages(FAKE, 0, 64, 2, None, 8, ids, 3, None), _hip.MX_ERR_INVALID)
    del keep


def test_wrappers_and_the_pool_refuse_host_memory_and_bad_shapes():
    with pytest.raises(ValueError, match="ROCm device"):
        Kv8Layer(torch.zeros(2, 1, 2, 1024, dtype=torch.uint8), torch.zeros(2, 1, 2, dtype=torch.uint8), 16, 64,
                 torch.float16)
    bad = dict(data=torch.zeros(2, 1, 2, 1000, dtype=torch.uint8), codes=torch.zeros(2, 1, 2, dtype=torch.uint8),
               block_size=16, head_dim=64, dtype=torch.float16)
    with pytest.raises(ValueError, match="contiguous uint8"):
        Kv8Layer(**bad)
    for change in (dict(dtype=torch.float32), dict(block_size=12), dict(head_dim=80)):
        with pytest.raises(ValueError):
            Kv8Layer(**(bad | change))
    args = dict(num_blocks=4, block_size_tokens=16, num_layers=1, num_kv_heads=2, head_dim=64, dtype=torch.float16)
    with pytest.raises(ValueError, match="no CPU form"):
        Int8KVBlockPool(**args, device="cpu")
    for change in (dict(dtype=torch.float32), dict(block_size_tokens=64), dict(head_dim=96), dict(num_blocks=0)):
        with pytest.raises(ValueError):
            Int8KVBlockPool(**(args | change), device="cuda")
    pool = Int8KVBlockPool(**args, device="cuda")  # nothing is allocated before the first use
    assert pool.bytes_per_block() == 2 * 2 * (16 * 64 + 1)
    for view in (pool.k_layer_view, pool.v_layer_view):
        with pytest.raises(ValueError, match="8-bit pool"):
            view(0)
    host = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    for call in (lambda: kv8_append(None, None, None, host, host),
                 lambda: kv8_attention_decode(host, None, None, None, 1.0, 1)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    assert callable(kv8_gather) and callable(kv8_rope_append)


def _cpu_pool(layout="interleaved", blocks=9):
    pool = GpuKVBlockPool(num_blocks=blocks, block_size_tokens=4, num_layers=2, num_kv_heads=2, head_dim=8,
                          dtype=torch.float32, device="cpu", kv_layout=layout)
    for li in range(2):
        for view in (pool.k_layer_view(li), pool.v_layer_view(li)):
            view.copy_(torch.randn(view.shape))
    return pool


def _snapshot(pool):
    return [[view(li).clone() for li in range(2)] for view in (pool.k_layer_view, pool.v_layer_view)]


@pytest.mark.parametrize("layout", ["interleaved", "split"])
@pytest.mark.parametrize("src,dst", [([0, 0], [1, 2]), ([1, 2], [2, 3]), ([1, 2, 3], [2, 3, 1]), ([4, 5], [6, 6]),
                                     ([3, 4], [3, 5]), ([1, 2, 2], [2, 1, 7])])
def test_copy_blocks_reads_every_source_first_on_the_cpu_pool(layout, src, dst):
    pool = _cpu_pool(layout)
    was = _snapshot(pool)
    pool.copy_blocks(src, dst)
    of = {d: s for s, d in zip(src, dst) if s != d}
    for a, b in zip(_snapshot(pool), was):
        for now, old in zip(a, b):
            assert torch.equal(now, old[[of.get(i, i) for i in range(9)]])


def test_move_and_free_blocks_on_the_cpu_pool():
    pool = _cpu_pool()
    was = _snapshot(pool)
    pool._touch_ids([3, 7, 8])
    tables = torch.tensor([[7, 3, 0], [8, 7, 5]], dtype=torch.int32)
    got = pool.move_blocks([7, 8], [1, 2], tables)
    assert got.tolist() == [[1, 3, 0], [2, 1, 5]] and tables.tolist()[0] == [7, 3, 0]
    for a, b in zip(_snapshot(pool), was):
        for now, old in zip(a, b):
            assert torch.equal(now, old[[0, 7, 8, 3, 4, 5, 6, 7, 8]])
    assert pool._used_blocks == {1, 2, 3} and pool.peak_allocated_block_count() == 3
    pool.move_blocks([5], [6])  # nothing was written to block 5
    assert pool._used_blocks == {1, 2, 3}
    pool.free_blocks([1, 2, 2])
    assert pool.allocated_block_count() == 1
    assert pool.move_blocks([], [], tables).tolist() == tables.tolist()
    assert pool.move_blocks([1], [2]) is None
    for src, dst in (([1], [1]), ([1, 1], [2, 3]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([1], [])):
        with pytest.raises(ValueError):
            pool.move_blocks(src, dst, tables)
    with pytest.raises(ValueError):
        pool.move_blocks([1], [2], tables.long())
    with pytest.raises(ValueError):
        pool.move_blocks([1], [2], out=tables)
    for call in (lambda: pool.move_blocks([1], [9]), lambda: pool.move_blocks([2**31], [1]), lambda: pool.copy_blocks([-1], [2]), lambda: pool.free_blocks([9])):
        with pytest.raises(IndexError):
            call()


def test_token_counts_at_the_top_of_32_bits_are_refused():
    for t in (2**31 - 1, 2**31 - 3, 2**31 - 31):  # more pages than a launch has waves for
        for bs in (4, 32):
            _status(_write(T=t, bs=bs), _hip.MX_ERR_UNSUPPORTED)
            _status(_gather(S=t, bs=bs), _hip.MX_ERR_UNSUPPORTED)


def test_pools_whose_byte_offsets_leave_64_bits_are_refused():
    big = dict(hkv=1 << 19, nb=2**31 - 1, bs=32, d=128)  # 2**63 bytes
    _status(_write(**big), _hip.MX_ERR_UNSUPPORTED)
    _status(_gather(**big), _hip.MX_ERR_UNSUPPORTED)
    _status(_token(**big), _hip.MX_ERR_UNSUPPORTED)
    _status(_attend(hq=1 << 19, **big), _hip.MX_ERR_UNSUPPORTED)


@pytest.mark.parametrize("bits,where", [(1, "batched write"), (4, "attention"), (5, "batched write and attention")])
def test_write_errors_name_every_kind_met(bits, where):
    pool = Int8KVBlockPool(num_blocks=4, block_size_tokens=16, num_layers=1, num_kv_heads=2, head_dim=64,
                           dtype=torch.float16, device="cuda")
    pool.check_write_errors()  # nothing allocated, nothing met
    pool._write_err = torch.tensor([bits], dtype=torch.int32)
    with pytest.raises(IndexError, match=f"during {where}$"):
        pool.check_write_errors()
    pool.check_write_errors()  # reported once


def test_move_blocks_refuses_tables_it_could_not_rename():
    pool = _cpu_pool()
    was = _snapshot(pool)
    flat = torch.arange(60, dtype=torch.int32) % 9
    tables = flat[:12].view(3, 4)
    row = torch.zeros(1, 1 << 15, dtype=torch.int32)
    with pytest.raises(ValueError, match=r"2\*\*31"):
        many = row.expand(1 << 16, -1)
        pool.move_blocks([1], [2], many, out=many)
    for out in (flat[:4].expand(3, 4), flat[1:13].view(3, 4), flat[8:20].view(3, 4), flat[:18].view(3, 6)[:, :4],
                flat[40:].as_strided((3, 4), (3, 1))):
        with pytest.raises(ValueError, match="share no entry"):
            pool.move_blocks([1], [2], tables, out=out)
    for a, b in zip(_snapshot(pool), was):
        for now, old in zip(a, b):
            assert torch.equal(now, old)


def test_move_blocks_takes_tables_beside_each_other():
    flat = torch.arange(60, dtype=torch.int32) % 9
    wide = flat.view(3, 20)
    for tables, out in ((flat[:12].view(3, 4), flat[12:24].view(3, 4)), (wide[:, :4], wide[:, 4:8]), (wide[:, 9:13], wide[:, 3:7]),
                        (wide[:, :4], wide[:, :4]), (flat[:4].expand(3, 4), flat[4:16].view(3, 4)),
                        (wide[:1, :4], flat[4:8].view(1, 4)), (wide[:0, :4], wide[:0, :4])):
        want = [[{1: 2}.get(i, i) for i in r] for r in tables.tolist()]
        assert _cpu_pool().move_blocks([1], [2], tables, out=out) is out
        assert out.tolist() == want
