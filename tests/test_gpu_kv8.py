"""The 8-bit KV cache on the GPU against its definition in float64 (``oracle/kv8.py``): writes, rows read
back, rotary + write, decode attention, and the paths that use them together.

Bars: what the cache stands for is bit-identical (scales are powers of two: every product and rounding of
the format is exact). Attention is within 6 u of the largest |value| that a head averages, u half a step
of the 16-bit type: the weights are rounded to it in the numerator and the denominator alike (2 u each way
at most: 4 u), the output once (u), and u covers scores and sums in fp32 and pieces joined in 32 bits.
"""

from __future__ import annotations

import pytest
import torch

from oracle.kv8 import Kv8Cache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = [(2, 16, 64, "fp16"), (1, 16, 128, "bf16"), (3, 4, 128, "fp16"), (2, 8, 64, "bf16"), (1, 32, 128, "fp16"),
         (2, 4, 64, "bf16"), (1, 8, 128, "fp16"), (2, 32, 64, "bf16")]


def _gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def _pool(nb, hkv, bs, d, dtype, layers=1):
    from runtime_amd.phase2.kv8_pool import Int8KVBlockPool

    return Int8KVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=layers, num_kv_heads=hkv, head_dim=d,
                           dtype=dtype, device=DEV)


def _states(b, hkv, t, d, dtype, g, spread=True):
    x = torch.randn(b, hkv, t, d, generator=g)
    if spread:  # tokens of very different sizes, so that scales grow and kept tokens are rounded again
        x = x * torch.exp2(torch.randint(-6, 7, (b, hkv, t, 1), generator=g))
    return x.to(dtype)


def _int(x):
    return torch.tensor(x, dtype=torch.int32)


def _same(pool, cache, tables, tokens, lens=None, layer=0):
    from runtime_amd.phase2.kv8 import kv8_gather

    got = kv8_gather(pool.layer_store(layer), tables.to(DEV), tokens, None if lens is None else _int(lens).to(DEV))
    for a, b in zip(got, cache.gather(tables, tokens, lens)):
        assert torch.equal(torch.nan_to_num(a.cpu().double(), nan=1e30), torch.nan_to_num(b, nan=1e30))


@pytest.mark.parametrize("hkv,bs,d,dt", SIZES)
def test_writes_and_rows_match_the_definition(hkv, bs, d, dt):
    dtype, g = DTYPES[dt], _gen(bs + d)
    pool, cache = _pool(24, hkv, bs, d, dtype), Kv8Cache(24, hkv, bs, d, dtype)
    tables = torch.randperm(24, generator=g)[:21].view(3, 7).int()
    starts = [0, 0, 0]
    # A prompt, single tokens across a page's end, chunks that begin inside a page and at its first slot.
    for t in (2 * bs + 3, 1, 1, bs - 3, 2, bs, 1):
        k, v = _states(3, hkv, t, d, dtype, g), _states(3, hkv, t, d, dtype, g)
        pool.write_tokens_batch(0, tables.to(DEV), _int(starts).to(DEV), k.to(DEV), v.to(DEV))
        assert cache.write(tables, starts, k, v)
        starts = [s + t for s in starts]
        _same(pool, cache, tables, starts[0], starts)
    pool.check_write_errors()
    _same(pool, cache, tables, 7 * bs, [1, 0, starts[0]])  # zeros past each row's length
    starts = [0, bs + 1, 3 * bs]  # rows rewritten from elsewhere: what stood behind is dropped
    k, v = _states(3, hkv, 2, d, dtype, g), _states(3, hkv, 2, d, dtype, g)
    pool.write_tokens_batch(0, tables.to(DEV), _int(starts).to(DEV), k.to(DEV), v.to(DEV))
    cache.write(tables, starts, k, v)
    _same(pool, cache, tables, 7 * bs, [s + 2 for s in starts])
    k, v = pool.gather_layer(0, tables[1].tolist(), bs + 3)
    want = cache.gather(tables[1:2], bs + 3)
    assert torch.equal(k.cpu().double(), want[0]) and torch.equal(v.cpu().double(), want[1])


@pytest.mark.parametrize("bs,d,dt,t", [(32, 128, "fp16", 8603), (32, 64, "bf16", 17001)])
def test_a_prompt_past_32_mib_of_states(bs, d, dt, t):
    """States that the streaming loads read (8 heads, 4 bytes a K/V element pair), from inside a page on."""
    dtype, g, hkv, start = DTYPES[dt], _gen(t), 8, 5
    assert 8 * t * d * 4 > 32 << 20
    nb = -(-(start + t) // bs)
    pool, cache = _pool(nb, hkv, bs, d, dtype), Kv8Cache(nb, hkv, bs, d, dtype)
    tables = torch.randperm(nb, generator=g).int()[None]
    for at, n in ((0, start), (start, t)):
        k, v = _states(1, hkv, n, d, dtype, g), _states(1, hkv, n, d, dtype, g)
        pool.write_tokens_batch(0, tables.to(DEV), _int([at]).to(DEV), k.to(DEV), v.to(DEV))
        cache.write(tables, [at], k, v)
    _same(pool, cache, tables, start + t)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_extreme_values(dt):
    """The largest and smallest numbers of the type, zeros, halfway cases, and values that are not finite."""
    dtype, hkv, bs, d = DTYPES[dt], 1, 4, 64
    info = torch.finfo(dtype)
    sub = torch.tensor(1, dtype=torch.int16).view(dtype).item()  # the smallest subnormal number
    cols = [info.max, -info.max, info.tiny, sub, -sub, 0.0, 127.5, 127.0, 254.5, 1.9921875, 1.984375, 0.5, -0.4980469]
    x = torch.zeros(len(cols) + 3, d)
    for i, c in enumerate(cols):
        x[i, i % d], x[i, (i + 9) % d] = c, c / 3
    x[len(cols), 5], x[len(cols) + 1, 6], x[len(cols) + 2, 7] = float("inf"), float("-inf"), float("nan")
    x = x.to(dtype)
    n = len(x)  # one row per token: each has a page of its own
    pool, cache = _pool(n, hkv, bs, d, dtype), Kv8Cache(n, hkv, bs, d, dtype)
    tables = torch.arange(n).view(n, 1).int()
    k = x.view(n, 1, 1, d)
    for at in (0, 1, 2):  # the same values again in the page, then ones that keep the scale
        pool.write_tokens_batch(0, tables.to(DEV), torch.full((n,), at, device=DEV, dtype=torch.int32), k.to(DEV), k.to(DEV))
        cache.write(tables, [at] * n, k, k)
        _same(pool, cache, tables, at + 1)
        k = k if at == 0 else torch.ones_like(k)
    pool.write_tokens_batch(0, tables.to(DEV), torch.zeros(n, device=DEV, dtype=torch.int32), k.to(DEV), k.to(DEV))
    cache.write(tables, [0] * n, k, k)
    _same(pool, cache, tables, 1)


def test_strided_and_unaligned_states():
    from runtime_amd.phase2.kv8 import kv8_append

    hkv, bs, d, dtype, g = 2, 16, 64, torch.float16, _gen(5)
    tables = torch.arange(6).view(2, 3).int()
    rows = torch.randn(2, 19, hkv, d + 8, generator=g).to(dtype)
    flat = torch.randn(2 * hkv * 19 * d + 1, generator=g).to(dtype)
    for make in (lambda x: x[..., :d].transpose(1, 2),                                  # as a decoder layer makes it
                 lambda x: flat.to(x.device)[1:].view(2, hkv, 19, d),                   # off by one element
                 lambda x: x[:, :, :, :d].transpose(1, 2).transpose(2, 3).contiguous().transpose(2, 3)):
        pool, cache = _pool(6, hkv, bs, d, dtype), Kv8Cache(6, hkv, bs, d, dtype)
        x, y = make(rows), make(rows.to(DEV))
        kv8_append(pool.layer_store(0), tables.to(DEV), _int([3, 0]).to(DEV), y, y.flip(0))
        cache.write(tables, [3, 0], x, x.flip(0))
        _same(pool, cache, tables, 22, [22, 19])


def test_slots_outside_the_table_or_the_pool_are_skipped_and_reported():
    hkv, bs, d, dtype, g = 1, 4, 64, torch.float16, _gen(6)
    pool, cache = _pool(8, hkv, bs, d, dtype), Kv8Cache(8, hkv, bs, d, dtype)
    tables = _int([[0, 1, 2], [3, 8, 4], [5, -1, 6]])
    for starts in ([9, 1, 2], [-2, 0, 0], [2**31 - 3, -(2**31), 1]):
        k, v = _states(3, hkv, 6, d, dtype, g), _states(3, hkv, 6, d, dtype, g)
        pool.write_tokens_batch(0, tables.to(DEV), _int(starts).to(DEV), k.to(DEV), v.to(DEV))
        assert not cache.write(tables, starts, k, v)
        with pytest.raises(IndexError, match="batched write"):
            pool.check_write_errors()
        pool.check_write_errors()
        _same(pool, cache, _int([[0, 1, 2, 3, 4, 5, 6, 7]]), 32, [4 if starts[0] == 9 else 2])
    assert pool.allocated_block_count() >= 3
    from runtime_amd.phase2.kv8 import kv8_gather

    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, _ = kv8_gather(pool.layer_store(0), tables.to(DEV), 14, err=err)  # two tokens past the table
    assert int(err) == 1 and (k[1:, :, 4:8] == 0).all() and (k[:, :, 12:] == 0).all()


def test_empty_calls():
    from runtime_amd.phase2.kv8 import kv8_attention_decode, kv8_gather

    pool = _pool(4, 2, 16, 64, torch.float16)
    layer = pool.layer_store(0)
    none = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    k, v = kv8_gather(layer, none, 5)
    assert k.shape == (0, 2, 5, 64) and kv8_gather(layer, torch.zeros(2, 1, dtype=torch.int32, device=DEV), 0)[0].numel() == 0
    q = torch.zeros(0, 4, 1, 64, dtype=torch.float16, device=DEV)
    assert kv8_attention_decode(q, layer, none, torch.zeros(0, dtype=torch.int32, device=DEV), 1.0, 2).shape == q.shape
    pool.write_tokens_batch(0, none, none[:, 0], torch.zeros(0, 2, 1, 64, device=DEV), torch.zeros(0, 2, 1, 64, device=DEV))
    pool.check_write_errors()


def test_a_pool_past_32_bits_of_bytes():
    hkv, bs, d, dtype, g = 8, 16, 128, torch.float16, _gen(8)
    nb = 140_000  # 4.6e9 bytes
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    pool = _pool(nb, hkv, bs, d, dtype)
    far = Kv8Cache(3, hkv, bs, d, dtype)  # pages 0..2 stand for nb - 1, nb - 2, 1
    ids = _int([[nb - 1, nb - 2, 1]])
    k, v = _states(1, hkv, 45, d, dtype, g, False), _states(1, hkv, 45, d, dtype, g, False)
    pool.write_tokens_batch(0, ids.to(DEV), _int([0]).to(DEV), k.to(DEV), v.to(DEV))
    far.write(_int([[0, 1, 2]]), [0], k, v)
    kk, vv = pool.gather_layer(0, ids[0].tolist(), 45)
    want = far.gather(_int([[0, 1, 2]]), 45)
    assert torch.equal(kk.cpu().double(), want[0]) and torch.equal(vv.cpu().double(), want[1])
    q = torch.randn(1, 16, 1, d, generator=g).to(dtype)
    out = kv8_attention_decode(q.to(DEV), pool.layer_store(0), ids.to(DEV), _int([45]).to(DEV), d ** -0.5, 2)
    _near(out, *far.attend(q[:, :, 0], _int([[0, 1, 2]]), [45], d ** -0.5))
    pool.copy_blocks([nb - 1, nb - 2], [7, 8])
    kk, _ = pool.gather_layer(0, [7, 8], 32)
    assert torch.equal(kk.cpu().double(), want[0][:, :, :32])


def _rope(n, d):
    from runtime_amd.phase2.decode_glue import rope_table

    return rope_table(n, d, 10000.0, DEV)


@pytest.mark.parametrize("hkv,bs,d,dt", SIZES)
@pytest.mark.parametrize("groups", [1, 3])
def test_rotary_and_write(hkv, bs, d, dt, groups):
    """k heads repeat q head 0, so the rotated k is known to the bit; v and the scales follow the
    definition; in fp16 q is the 16-bit path's bit for bit."""
    from runtime_amd.phase2.decode_glue import qkv_rope_append
    from runtime_amd.phase2.kv8 import kv8_rope_append
    from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool

    dtype, g, b, hq = DTYPES[dt], _gen(d + bs), 4, hkv * groups
    nb, rope = 4 * b, _rope(3 * bs, d)
    pool, cache = _pool(nb, hkv, bs, d, dtype), Kv8Cache(nb, hkv, bs, d, dtype)
    tables = torch.randperm(nb, generator=g)[:3 * b].view(b, 3).int()
    pos = [0, bs - 2, bs, 2 * bs - 1]
    k, v = _states(b, hkv, 2 * bs, d, dtype, g), _states(b, hkv, 2 * bs, d, dtype, g)
    pool.write_tokens_batch(0, tables.to(DEV), _int([0] * b).to(DEV), k.to(DEV), v.to(DEV))
    cache.write(tables, [0] * b, k, v)
    err, lens = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(b, dtype=torch.int32, device=DEV)
    used = torch.zeros(nb, dtype=torch.uint8, device=DEV)
    for _ in range(3):
        x = _states(b, hq + 2 * hkv, 1, d, dtype, g)[:, :, 0]
        x[:, hq:hq + hkv] = x[:, :1]
        q = torch.empty(b, hq * d, dtype=dtype, device=DEV)
        kv8_rope_append(x.reshape(b, -1).to(DEV), rope, _int(pos).to(DEV), q, pool.layer_store(0), tables.to(DEV), hq,
                        err=err, lens_out=lens, used_blocks=used)
        rot = q.cpu().view(b, hq, d)
        assert lens.tolist() == [p + 1 for p in pos] and int(err) == 0
        assert used.nonzero().flatten().tolist() == sorted({int(tables[i, p // bs]) for i, p in enumerate(pos)} |
                                                           set(used.nonzero().flatten().tolist()))
        cs = rope.cpu()[pos].double()
        a, c = x[:, :hq].double().chunk(2, dim=-1)
        cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
        want = torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1)
        # one rounding to the type, and fp32 products and sums of two terms before it
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -22 * torch.cat([a.abs() + c.abs()] * 2, dim=-1) + 2.0 ** -24
        assert ((rot.double() - want).abs() <= bound).all()
        cache.write(tables, pos, rot[:, :1].repeat(1, hkv, 1)[:, :, None], x[:, hq + hkv:, None])
        _same(pool, cache, tables, 3 * bs, [p + 1 for p in pos])
        if dtype == torch.float16:
            p16 = GpuKVBlockPool(num_blocks=nb, block_size_tokens=bs, num_layers=1, num_kv_heads=hkv, head_dim=d,
                                 dtype=dtype, device=DEV)
            q16 = torch.empty_like(q)
            qkv_rope_append(x.reshape(b, -1).to(DEV), rope, _int(pos).to(DEV), q16, p16.k_layer_view(0),
                            p16.v_layer_view(0), tables.to(DEV), hq, hkv)
            assert torch.equal(q, q16)
        pos = [p + 1 for p in pos]


def test_rotary_from_split_partials_and_its_errors():
    from runtime_amd.phase2.kv8 import kv8_rope_append

    hkv, hq, bs, d, dtype, g, b = 2, 4, 16, 128, torch.float16, _gen(11), 5
    width = (hq + 2 * hkv) * d
    part = torch.randn(3, b, width, generator=g)
    bias = torch.randn(width, generator=g).half()
    rows = (((bias.float() + part[0]) + part[1]) + part[2]).half()
    tables = _int([[i, 9] for i in range(4)] + [[77, 9]])  # the last row's page is outside the pool
    pos = [3, 15, -1, 64, 2]                               # two positions outside the rope table
    outs = []
    for partials in (False, True):
        pool = _pool(10, hkv, bs, d, dtype)
        q = torch.full((b, hq * d), 7.0, dtype=dtype, device=DEV)
        err, rope = torch.zeros(1, dtype=torch.int32, device=DEV), _rope(64, d)
        kv8_rope_append(None if partials else rows.to(DEV), rope, _int(pos).to(DEV), q, pool.layer_store(0),
                        tables.to(DEV), hq, partials=part.to(DEV) if partials else None, splits=3 if partials else 0,
                        bias=bias.to(DEV) if partials else None, err=err)
        assert int(err) == 3
        outs.append((q, pool._data, pool._codes))
    for a, c in zip(*outs):
        assert torch.equal(a, c)
    q, _, codes = outs[0]
    assert (q[2:4] == 0).all() and (q[[0, 1, 4]] != 7.0).any(dim=1).all()
    assert codes[0].amax(dim=(1, 2)).nonzero().flatten().tolist() == [0, 1]


def _near(got, want, most, dtype=torch.float16):
    got = got.cpu().double().view(want.shape)
    bound = 6 * torch.finfo(dtype).eps / 2 * most[..., None] + 2.0 ** -24
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - bound).max()
    assert worst <= 0, f"{float(worst)} over the bound"


def _cached(b, lens, hkv, bs, d, dtype, g, extra=2, spread=False):
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + extra
    pool, cache = _pool(nb, hkv, bs, d, dtype), Kv8Cache(nb, hkv, bs, d, dtype)
    perm, at = torch.randperm(nb, generator=g).int(), 0
    tables = torch.full((b, max(max(need), 1) + 1), -1, dtype=torch.int32)  # the tail ids are never read
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
        if lens[i]:
            k, v = _states(1, hkv, lens[i], d, dtype, g, spread), _states(1, hkv, lens[i], d, dtype, g, spread)
            pool.write_tokens_batch(0, tables[i:i + 1].to(DEV), _int([0]).to(DEV), k.to(DEV), v.to(DEV))
            cache.write(tables[i:i + 1], [0], k, v)
    return pool, cache, tables


ATTEND = [(h, bs, d, dt, grp) for (h, bs, d, dt), grp in zip(SIZES, (4, 8, 3, 7, 1, 16, 5, 2))] + [
    (1, 16, 128, "fp16", 17), (1, 16, 64, "bf16", 33), (2, 16, 128, "fp16", 4)]


@pytest.mark.parametrize("hkv,bs,d,dt,group", ATTEND)
def test_attention_matches_float64(hkv, bs, d, dt, group):
    from runtime_amd.phase2.paged_attention_hip import PagedDecodeBatchMetadata, paged_attention_decode_batched

    dtype, g = DTYPES[dt], _gen(group)
    lens = [0, 1, bs - 1, bs, bs + 1, 15, 16, 17, 63, 64, 65, 130, 300]
    b = len(lens)
    pool, cache, tables = _cached(b, lens, hkv, bs, d, dtype, g)
    q = torch.randn(b, hkv * group, 1, d, generator=g).to(dtype)
    want = cache.attend(q[:, :, 0], tables, lens, d ** -0.5)
    for table in (tables, _widen(tables, 140_000 // bs)):  # a workgroup per segment; shared out between waves
        meta = PagedDecodeBatchMetadata(pool=pool, layer_idx=0, block_tables=table.to(DEV), seq_lens=_int(lens).to(DEV))
        out = paged_attention_decode_batched(q.to(DEV), meta, group, d ** -0.5)
        _near(out, *want, dtype)
        shared = pool.attend(0, q.to(DEV), table.to(DEV), _int(lens).to(DEV), d ** -0.5, group, shared_blocks=True)
        assert torch.equal(shared, out)
        assert (out[0] == 0).all()
    pool.check_write_errors()


@pytest.mark.parametrize("hkv,bs,d,dt,group,lens", [
    (2, 16, 128, "fp16", 4, [5000]), (1, 32, 64, "bf16", 7, [3001, 17]), (8, 16, 128, "fp16", 2, [1025, 2047, 1]),
    (1, 4, 64, "fp16", 2, [2500]), (1, 8, 128, "bf16", 3, [1111, 0, 900])])
def test_attention_over_long_and_ragged_rows(hkv, bs, d, dt, group, lens):
    """Rows long enough to be shared out and joined; sizes of K and V that differ from page to page."""
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    dtype, g, b = DTYPES[dt], _gen(sum(lens)), len(lens)
    pool, cache, tables = _cached(b, lens, hkv, bs, d, dtype, g, spread=True)
    q = (torch.randn(b, hkv * group, 1, d, generator=g) * 0.05).to(dtype)
    out = kv8_attention_decode(q.to(DEV), pool.layer_store(0), tables.to(DEV), _int(lens).to(DEV), d ** -0.5, group)
    _near(out, *cache.attend(q[:, :, 0], tables, lens, d ** -0.5), dtype)


def _widen(tables, blocks):
    """The same rows in a table of ``blocks`` entries, the new ones outside the pool and never read."""
    return torch.cat([tables, torch.full((len(tables), blocks - tables.shape[1]), -7, dtype=torch.int32)], dim=1)


@pytest.mark.parametrize("b", [63, 64, 65, 150, 300])
@pytest.mark.parametrize("wide", [0, 5000])
def test_many_short_rows(b, wide):
    """A workgroup per row (narrow table) and rows shared out between waves (wide table), with rows
    without tokens in runs, also first and last, around the 64 rows that a wave takes at once."""
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    hkv, bs, d, dtype, g = 1, 16, 64, torch.float16, _gen(3)
    lens = [0 if i < 3 or i % 64 in (62, 63, 0) or i == b - 1 else (37 * i) % 90 for i in range(b)]
    pool, cache, tables = _cached(b, lens, hkv, bs, d, dtype, g)
    q = torch.randn(b, 2, 1, d, generator=g).to(dtype)
    want = cache.attend(q[:, :, 0], tables, lens, 0.125)
    tables = _widen(tables, wide) if wide else tables
    out = kv8_attention_decode(q.to(DEV), pool.layer_store(0), tables.to(DEV), _int(lens).to(DEV), 0.125, 2)
    _near(out, *want, dtype)


def test_no_row_has_tokens():
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    pool = _pool(4, 2, 16, 128, torch.bfloat16)
    q = torch.randn(70, 8, 1, 128).bfloat16().to(DEV)
    for width in (1, 9000):
        out = kv8_attention_decode(q, pool.layer_store(0), torch.zeros(70, width, dtype=torch.int32, device=DEV),
                                   torch.zeros(70, dtype=torch.int32, device=DEV), 1.0, 4)
        assert (out == 0).all()


def test_v_of_every_size():
    """V pages from the smallest to the largest scale side by side: in fp16 the scales above 2^5 leave a
    factor to the weights."""
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    for dtype, exps in ((torch.float16, (-24, -10, 0, 5, 6, 8, 9)), (torch.bfloat16, (-126, -20, 0, 119, 120, 121))):
        for bs in (4, 16):
            g, d = _gen(17), 64
            n = 16 * len(exps)
            pool, cache = _pool(n // bs, 1, bs, d, dtype), Kv8Cache(n // bs, 1, bs, d, dtype)
            tables = torch.arange(n // bs)[None].int()
            k = torch.randn(1, 1, n, d, generator=g).to(dtype)
            ints = torch.randint(-127, 128, (1, 1, n, d), generator=g).double()
            ints[..., 0] = 127
            v = (ints.view(1, 1, -1, 16, d) * torch.tensor([2.0 ** e for e in exps], dtype=torch.float64)[:, None, None])
            v = v.view(1, 1, n, d).to(dtype)
            pool.write_tokens_batch(0, tables.to(DEV), _int([0]).to(DEV), k.to(DEV), v.to(DEV))
            cache.write(tables, [0], k, v)
            # Each query is a key, so that its weights lie on one page or another.
            q = (8 * k[0, 0, 3::16][:len(exps)])[None, :, None].contiguous()
            out = kv8_attention_decode(q.to(DEV), pool.layer_store(0), tables.to(DEV), _int([n]).to(DEV), 1.0, len(exps))
            _near(out, *cache.attend(q[:, :, 0], tables, [n], 1.0), dtype)


def test_large_scores_and_one_token_that_takes_all():
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    hkv, bs, d, dtype, g = 1, 16, 64, torch.float16, _gen(4)
    pool, cache, tables = _cached(2, [200, 700], hkv, bs, d, dtype, g, spread=True)
    q = (torch.randn(2, 4, 1, d, generator=g) * 30).to(dtype)
    for scale in (1.0, -1.0, 0.0):
        out = kv8_attention_decode(q.to(DEV), pool.layer_store(0), tables.to(DEV), _int([200, 700]).to(DEV), scale, 4)
        want, most = cache.attend(q[:, :, 0], tables, [200, 700], scale)
        # Scores reach 30 * 64 * 64 * sqrt(64) ~ 1e6: an fp32 sum of D products of which the largest is that
        # size is off by up to D 2^-24 of it, so a weight may be wrong by more than its rounding.
        k = torch.stack([cache.row(tables[i], n, 0, 0)[0].abs().max() for i, n in ((0, 200), (1, 700))])
        err = float(d * 2.0 ** -23 * k.max() * q.double().abs().sum(dim=-1).max()) if scale else 0.0
        got = out.cpu().double().view(want.shape)
        assert ((got - want).abs() <= (6 * 2.0 ** -11 + 2 * min(1.0, err)) * most[..., None]).all()


def test_blocks_outside_the_pool_and_poisoned_pages():
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    hkv, bs, d, dtype, g = 2, 16, 64, torch.float16, _gen(9)
    lens = [90, 40, 20]
    pool, cache, tables = _cached(3, lens, hkv, bs, d, dtype, g)
    tables[0, 2], tables[2, :2] = cache.nb, -5  # one page of row 0, all of row 2
    q = torch.randn(3, 4, 1, d, generator=g).to(dtype)

    def run(table=tables):
        return kv8_attention_decode(q.to(DEV), pool.layer_store(0), table.to(DEV), _int(lens).to(DEV), 0.125, 2,
                                    err=pool._write_err)

    _near(run(_widen(tables, 9000)), *cache.attend(q[:, :, 0], tables, lens, 0.125))
    with pytest.raises(IndexError, match="attention"):
        pool.check_write_errors()
    out = run()
    _near(out, *cache.attend(q[:, :, 0], tables, lens, 0.125))
    assert (out[2] == 0).all()
    with pytest.raises(IndexError, match="attention"):
        pool.check_write_errors()
    x = torch.ones(1, hkv, 1, d).half()
    bad = x.clone()
    bad[0, 1, 0, 3] = float("nan")
    for kv in ((bad, x), (x, bad)):  # K, then V, of head 1 in row 1's last page
        pool.write_tokens_batch(0, tables[1:2].to(DEV), _int([39]).to(DEV), kv[0].to(DEV), kv[1].to(DEV))
        for out in (run(), run(_widen(tables, 9000))):
            assert torch.isnan(out[1, 2:]).all() and torch.isfinite(out[1, :2]).all()
            assert torch.isfinite(out[[0, 2]]).all()
        pool.write_tokens_batch(0, tables[1:2].to(DEV), _int([32]).to(DEV), x.expand(1, hkv, 8, d).to(DEV),
                                x.expand(1, hkv, 8, d).to(DEV))
        assert torch.isfinite(run()).all()


def test_lengths_past_the_table_strided_query_and_given_output():
    from runtime_amd.phase2.kv8 import kv8_attention_decode

    hkv, bs, d, dtype, g = 2, 16, 128, torch.bfloat16, _gen(10)
    pool, cache, tables = _cached(3, [64, 33, 48], hkv, bs, d, dtype, g)
    narrow = tables[:, :3].contiguous()  # 48 tokens at most
    wide = torch.randn(3, 1, 12, d + 8, generator=g).to(dtype)
    q = wide[:, :, ::2, :d].transpose(1, 2)  # [3, 6, 1, d]
    out = torch.full((3, 6, 2, d), 5.0, dtype=dtype, device=DEV)[:, :, :1]
    lens = [2**31 - 1, 33, 0]
    got = kv8_attention_decode(wide.to(DEV)[:, :, ::2, :d].transpose(1, 2), pool.layer_store(0), narrow.to(DEV),
                               _int(lens).to(DEV), 0.1, 3, out=out)
    assert got is out and (out._base[:, :, 1] == 5.0).all()
    _near(got, *cache.attend(q[:, :, 0], narrow, lens, 0.1), dtype)
    odd = torch.randn(3 * 6 * d + 1, generator=g).to(dtype)[1:].view(3, 6, 1, d)
    dev = torch.empty(3 * 6 * d + 1, dtype=dtype, device=DEV)[1:].view(3, 6, 1, d).copy_(odd)
    _near(kv8_attention_decode(dev, pool.layer_store(0), narrow.to(DEV), _int([-3, 33, 1]).to(DEV), 0.1, 3),
          *cache.attend(odd[:, :, 0], narrow, [-3, 33, 1], 0.1), dtype)


def test_wrappers_refuse_on_the_device():
    from runtime_amd.phase2.kv8 import kv8_append, kv8_attention_decode, kv8_gather, kv8_rope_append

    pool = _pool(4, 2, 16, 64, torch.float16)
    layer = pool.layer_store(0)
    t, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 2, 1, 64, dtype=torch.float16, device=DEV)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device=DEV)
    row, qo = torch.zeros(1, 8 * 64, dtype=torch.float16, device=DEV), torch.zeros(1, 4 * 64, dtype=torch.float16, device=DEV)
    rope = torch.zeros(8, 32, 2, device=DEV)
    calls = [
        lambda: kv8_append(layer, t, n, x, x[:, :1]), lambda: kv8_append(layer, t, n, x.float(), x.float()),
        lambda: kv8_append(layer, t[0], n, x, x), lambda: kv8_append(layer, t, n.repeat(2), x, x),
        lambda: kv8_append(layer, t, n, x[..., :32], x[..., :32]), lambda: kv8_append(layer, t, n, x[0], x[0]),
        lambda: kv8_append(layer, t, n, x, x, used_blocks=torch.zeros(3, dtype=torch.uint8, device=DEV)),
        lambda: kv8_append(layer, t, n, x, x, err=torch.zeros(1, device=DEV)),
        lambda: kv8_gather(layer, t, -1), lambda: kv8_gather(layer, t, 3, n.repeat(2)), lambda: kv8_gather(layer, t[0], 3),
        lambda: kv8_attention_decode(q[:, :3], layer, t, n, 1.0, 2), lambda: kv8_attention_decode(q.bfloat16(), layer, t, n, 1.0, 2),
        lambda: kv8_attention_decode(q[..., :32], layer, t, n, 1.0, 2), lambda: kv8_attention_decode(q, layer, t, n.repeat(2), 1.0, 2),
        lambda: kv8_attention_decode(q.repeat(1, 1, 2, 1), layer, t, n, 1.0, 2),
        lambda: kv8_attention_decode(q, layer, t, n, 1.0, 2, out=q.float()),
        lambda: kv8_rope_append(row, rope, n, qo, layer, t, 5), lambda: kv8_rope_append(row[:, :64], rope, n, qo, layer, t, 4),
        lambda: kv8_rope_append(None, rope, n, qo, layer, t, 4), lambda: kv8_rope_append(row, rope.half(), n, qo, layer, t, 4),
        lambda: kv8_rope_append(row, rope, n.repeat(2), qo, layer, t, 4), lambda: kv8_rope_append(row, rope, n, qo.float(), layer, t, 4),
        lambda: kv8_rope_append(row, rope, n, qo, layer, t, 4, bias=row[0]),
        lambda: kv8_rope_append(None, rope, n, qo, layer, t, 4, partials=row.float(), splits=2),
        lambda: kv8_rope_append(row, rope, n, qo, layer, t, 4, lens_out=n), lambda: kv8_rope_append(row, rope, n, qo, layer, t, 4, lens_out=n.cpu()),
        lambda: kv8_append(layer, t, n, x, x, err=torch.zeros(1, dtype=torch.int32)),
        lambda: kv8_attention_decode(q, layer, t[:, :0], n, 1.0, 2), lambda: kv8_gather(layer, t[:, :0], 3),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_side_stream_and_graph_replays():
    """A captured step (rotary + write, attention) replayed as rows grow, beside eager work on the same
    pool's other layer; every replay against eager calls on a pool of its own."""
    from runtime_amd.phase2.kv8 import kv8_attention_decode, kv8_rope_append

    hkv, hq, bs, d, dtype, g, b = 2, 8, 16, 128, torch.float16, _gen(12), 3
    lens0, steps = [30, 500, 0], 6
    tables = torch.randperm(120, generator=g)[:3 * 36].view(3, 36).int()
    k, v = _states(b, hkv, 500, d, dtype, g), _states(b, hkv, 500, d, dtype, g)
    rows = [torch.randn(b, (hq + 2 * hkv) * d, generator=g).half().to(DEV) for _ in range(steps)]
    rope = _rope(1024, d)

    def fresh():
        pool = _pool(120, hkv, bs, d, dtype, layers=2)
        for li in range(2):
            pool.write_tokens_batch(li, tables.to(DEV), _int([0] * b).to(DEV), k.to(DEV), v.to(DEV))
        return pool

    def step(pool, row, pos, lens, q, out):
        layer = pool.layer_store(0)
        kv8_rope_append(row, rope, pos, q, layer, tables_d, hq, lens_out=lens)
        kv8_attention_decode(q.view(b, hq, 1, d), layer, tables_d, lens, d ** -0.5, hq // hkv, out=out)

    tables_d = tables.to(DEV)

    def buffers():
        return (torch.empty(b, hq * d, dtype=dtype, device=DEV), torch.empty(b, hq, 1, d, dtype=dtype, device=DEV),
                _int(lens0).to(DEV), torch.zeros(b, dtype=torch.int32, device=DEV))

    eager, want = fresh(), []
    q, out, pos, lens = buffers()
    for row in rows:
        step(eager, row, pos, lens, q, out)
        want.append((q.clone(), out.clone()))
        pos.add_(1)
    pool, row = fresh(), rows[0].clone()
    q, out, pos, lens = buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the first step, eagerly on another stream
        step(pool, row, pos, lens, q, out)
        assert torch.equal(out, want[0][1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(pool, row, pos, lens, q, out)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(steps):
        row.copy_(rows[i])
        q.zero_(), out.zero_()
        graph.replay()
        other = torch.empty_like(out)
        kv8_attention_decode(q.view(b, hq, 1, d), pool.layer_store(1), tables_d, lens, d ** -0.5, hq // hkv, out=other)
        assert torch.equal(q, want[i][0]) and torch.equal(out, want[i][1]) and torch.isfinite(other).all()
        pos.add_(1)
        torch.cuda.synchronize()
    assert torch.equal(pool._data[0], eager._data[0]) and torch.equal(pool._codes[0], eager._codes[0])


def test_cache_layer_prompt_then_decode_through_the_hook():
    """A prompt through ``BlockPagedLayer.update`` and the attention hook, then decode steps: the rows the
    prompt's attention reads are the cache's values, and every step's output is float64's over them."""
    from types import SimpleNamespace

    from runtime_amd.phase2.block_paged_attention import block_paged_attention_forward
    from runtime_amd.phase2.paged_kv_cache import BlockPagedLayer

    hkv, grp, bs, d, dtype, g = 2, 4, 16, 64, torch.float16, _gen(13)
    pool, cache = _pool(12, hkv, bs, d, dtype), Kv8Cache(12, hkv, bs, d, dtype)
    table = torch.randperm(12, generator=g)[:8].int()
    layer = BlockPagedLayer(pool, 0)
    layer.set_block_ids(table.tolist())
    module = SimpleNamespace(num_key_value_groups=grp, training=False)
    n = 0
    for t in (37, 1, 1, 20, 1):
        k, v = _states(1, hkv, t, d, dtype, g, False), _states(1, hkv, t, d, dtype, g, False)
        q = torch.randn(1, hkv * grp, t, d, generator=g).to(dtype)
        keys, values = layer.update(k.to(DEV), v.to(DEV))
        cache.write(table[None], [n], k, v)
        n += t
        if t > 1:
            want = cache.gather(table[None], n)
            assert torch.equal(keys.cpu().double(), want[0]) and torch.equal(values.cpu().double(), want[1])
        out, _ = block_paged_attention_forward(module, q.to(DEV), keys, values, None, d ** -0.5)
        assert out.shape == (1, t, hkv * grp, d)
        if t == 1:
            _near(out, *cache.attend(q[:, :, 0], table[None], [n], d ** -0.5))
    pool.check_write_errors()


def test_rotation_in_place():
    """q_out may be the q part of the fused rows themselves."""
    from runtime_amd.phase2.kv8 import kv8_rope_append

    for d in (64, 128):
        hkv, hq, b, g = 2, 6, 5, _gen(d)
        rows = torch.randn(b, (hq + 2 * hkv) * d, generator=g).half().to(DEV)
        pos, rope = _int([3, 0, 17, 40, 16]).to(DEV), _rope(64, d)
        tables = torch.arange(3 * b).view(b, 3).int().to(DEV)
        pools, q = [_pool(3 * b, hkv, 16, d, torch.float16) for _ in range(2)], torch.empty(b, hq * d, dtype=torch.float16, device=DEV)
        kv8_rope_append(rows, rope, pos, q, pools[0].layer_store(0), tables, hq)
        kv8_rope_append(rows, rope, pos, rows[:, :hq * d], pools[1].layer_store(0), tables, hq)
        assert torch.equal(rows[:, :hq * d], q) and torch.equal(pools[0]._data, pools[1]._data)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_hf_model_decodes_over_an_8_bit_pool(dt):
    """The worker's paths over an 8-bit pool: prompts and ragged decode steps through the cache adapters, with
    and without a captured graph, agree to the bit; the single-row entry point and the warm-up take it."""
    from oracle import model as om
    from runtime_amd.phase2.hf_decode import (DecodeRequest, DecodeState, PagedDecoder, enable_block_paged_attention,
                                              prefill_request)
    from runtime_amd.phase2.hip_graph_decode import CudaGraphDecodeManager
    from runtime_amd.phase2.paged_attention_hip import paged_attention_decode, warmup_paged_attention_kernel

    dtype, g = DTYPES[dt], _gen(21)
    hf = om.random_llama(seed=3, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         intermediate_size=512, vocab_size=512, max_position_embeddings=256)
    om.to_device_dtype(hf, DEV, dtype).eval()
    enable_block_paged_attention(hf)
    prompts = [torch.randint(0, 512, (n,), generator=g) for n in (21, 16, 40)]
    runs = []
    for graphs in (False, True):
        pool = _pool(24, 2, 16, 64, dtype, layers=2)
        warmup_paged_attention_kernel(pool, num_heads=4, num_kv_groups=2, head_dim=64, block_ids=[0, 1])
        manager = CudaGraphDecodeManager(model=hf, device=DEV, warmup_steps=1, enabled=True) if graphs else None
        worker, states = PagedDecoder(hf, pool, max_active=4, graph_mgr=manager), []
        for i, ids in enumerate(prompts):
            cache, logits = prefill_request(hf, pool, list(range(8 * i, 8 * i + 8)), ids.view(1, -1).to(DEV))
            states.append(DecodeState(DecodeRequest(str(i)), cache, int(logits.argmax()), []))
        steps = []
        for _ in range(6):
            worker.decode_step(states)
            steps.append(worker.last_logits.float().clone())
        assert not graphs or manager.stats()["graphs"][0]["replays"] >= 4
        runs.append((torch.stack(steps), [s.generated_token_ids for s in states], pool))
    assert torch.equal(runs[0][0], runs[1][0]) and runs[0][1] == runs[1][1]
    assert torch.isfinite(runs[0][0]).all() and torch.equal(runs[0][2]._data, runs[1][2]._data)
    pool = runs[0][2]
    q = torch.randn(1, 4, 1, 64, generator=g).to(dtype).to(DEV)
    k, v = (x.double().cpu() for x in pool.gather_layer(1, list(range(8, 16)), 20))
    out = paged_attention_decode(q, pool, 1, list(range(8, 16)), 20, 2, 0.125).cpu().double()
    for h in range(4):
        want = torch.softmax(k[0, h // 2] @ q[0, h, 0].cpu().double() * 0.125, 0) @ v[0, h // 2]
        assert (out[0, h, 0] - want).abs().max() <= 6 * torch.finfo(dtype).eps / 2 * v[0, h // 2].abs().max() + 2.0 ** -24


@pytest.mark.parametrize("batch", [2, 16, 40])
def test_native_step_over_an_8_bit_pool(batch):
    """``Int8DecodeModel.step`` over an 8-bit pool is its parts called one by one, bit for bit: the
    QKV projection as whole rows here, in the step as split partials where the batch's shape splits K."""
    from runtime_amd.phase2.decode_step import DecoderShape, Int8DecodeModel
    from runtime_amd.phase2.kv8 import kv8_attention_decode, kv8_rope_append

    shape = DecoderShape(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, intermediate=512, vocab=1024,
                         qkv_bias=True)
    model = Int8DecodeModel(shape, device=DEV, seed=batch, max_positions=256)
    g = _gen(batch)
    tables = torch.randperm(batch * 4, generator=g).view(batch, 4).int().to(DEV)
    tokens = torch.randint(0, 1024, (batch,), generator=g).to(DEV)
    lens0 = torch.randint(0, 50, (batch,), generator=g).int()
    pools = [_pool(batch * 4, 2, 16, 64, torch.float16, layers=2) for _ in range(2)]
    k, v = _states(batch, 2, 50, 64, torch.float16, g, False), _states(batch, 2, 50, 64, torch.float16, g, False)
    for pool in pools:
        for li in range(2):
            pool.write_tokens_batch(li, tables, _int([0] * batch).to(DEV), k.to(DEV), v.to(DEV))
    seen = []

    def spy(buf, layer, pool, li, block_tables, seq_lens, lens_out, timers):
        x = buf.x.clone()
        real(buf, layer, pool, li, block_tables, seq_lens, lens_out, timers)
        seen.append((x, buf.attn.clone()))

    real, model._attend_kv8 = model._attend_kv8, None
    model._attend_kv8 = spy
    lens = lens0.to(DEV)
    model.step(tokens, pools[0], tables, lens)
    assert torch.equal(lens.cpu(), lens0 + 1) and model.error_flag() == 0
    from runtime_amd.phase2.int8_linear import int8_linear

    for li, (x, attn) in enumerate(seen):
        packed, scale, n, bias = model.layers[li].qkv
        rows = int8_linear(x, packed, scale, bias, n)
        q, out_lens = torch.empty(batch, 512, dtype=torch.float16, device=DEV), torch.zeros(batch, dtype=torch.int32, device=DEV)
        store = pools[1].layer_store(li)
        kv8_rope_append(rows, model.rope, lens0.to(DEV), q, store, tables, 8, lens_out=out_lens)
        out = kv8_attention_decode(q.view(batch, 8, 1, 64), store, tables, out_lens, 64 ** -0.5, 4)
        assert torch.equal(out, attn)
    assert torch.equal(pools[0]._data, pools[1]._data) and torch.equal(pools[0]._codes, pools[1]._codes)
    used = pools[0]._used_map.nonzero().flatten()
    assert len(used) == batch * 4
