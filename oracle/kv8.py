"""The 8-bit KV cache restated in float64 on the CPU: one page at a time, from the format's definition.

No counterpart in the reference, whose pool is 16-bit (``runtime/phase2/paged_kv_kernel.py:24-315``); the
slots a token goes to are its (``:163-174,217-227``). A page (block, kv-head, K or V) holds integers ``q``
and an exponent ``e``: the smallest for which every rounded ``x / 2**e`` is at most 127 in magnitude, within
``EXPONENTS``; ``None`` while nothing is written, ``"nan"`` once a value that is not finite was.
"""

from __future__ import annotations

import math

import torch

# Exponents whose multiples up to 127 are numbers of the element type.
EXPONENTS = {torch.float16: (-24, 9), torch.bfloat16: (-126, 121)}


def exponent(amax: float, dtype: torch.dtype):
    """The scale's exponent of a page whose largest magnitude is ``amax``."""
    lo, hi = EXPONENTS[dtype]
    if not math.isfinite(amax):
        return "nan"
    e = lo
    while e < hi and round(math.ldexp(amax, -e)) > 127:  # Python rounds halves to even
        e += 1
    return e


class Kv8Cache:
    """One layer: ``q [nb, Hkv, 2, bs, D]`` (float64 integers) and ``exps[(block, head, kind)]``."""

    def __init__(self, num_blocks: int, hkv: int, bs: int, d: int, dtype: torch.dtype) -> None:
        self.nb, self.hkv, self.bs, self.d, self.dtype = num_blocks, hkv, bs, d, dtype
        self.q = torch.zeros(num_blocks, hkv, 2, bs, d, dtype=torch.float64)
        self.exps: dict[tuple[int, int, int], object] = {}

    def write(self, tables, starts, keys: torch.Tensor, values: torch.Tensor) -> bool:
        """``keys``/``values [B, Hkv, T, D]`` at ``starts[b] + t``; False if a slot was skipped."""
        ok = True
        for b in range(keys.shape[0]):
            t = keys.shape[2]
            blocks: dict[int, list[int]] = {}
            for i in range(t):
                pos = int(starts[b]) + i
                lb = pos // self.bs
                if pos < 0 or lb >= tables.shape[1] or not 0 <= int(tables[b, lb]) < self.nb:
                    ok = False
                else:
                    blocks.setdefault(lb, []).append(i)
            for lb, toks in blocks.items():
                phys = int(tables[b, lb])
                o = (int(starts[b]) + toks[0]) % self.bs
                for kind, x in ((0, keys), (1, values)):
                    for h in range(self.hkv):
                        self._write_page(phys, h, kind, o, x[b, h, toks].double())
        return ok

    def _write_page(self, phys: int, h: int, kind: int, o: int, x: torch.Tensor) -> None:
        key, page = (phys, h, kind), self.q[phys, h, kind]
        old = self.exps.get(key) if o > 0 else None
        need = exponent(float("nan") if not torch.isfinite(x).all() else float(x.abs().max()), self.dtype)
        if "nan" in (old, need):
            self.exps[key] = "nan"
            return
        now = need if old is None else max(old, need)
        page[:o] = 0.0 if old is None else torch.round(page[:o] * 2.0 ** (old - now))
        page[o:o + len(x)] = torch.round(x * 2.0 ** -now).clamp(-127, 127)
        self.exps[key] = now

    def values(self, phys: int, h: int, kind: int) -> torch.Tensor:
        e = self.exps.get((phys, h, kind))
        if e is None:
            return torch.zeros(self.bs, self.d, dtype=torch.float64)
        if e == "nan":
            return torch.full((self.bs, self.d), float("nan"), dtype=torch.float64)
        return self.q[phys, h, kind] * 2.0 ** e

    def row(self, table, n: int, h: int, kind: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The first ``n`` tokens of a row for one head, and which of them lie in the pool."""
        parts, live = [], []
        for lb in range(-(-n // self.bs)):
            phys = int(table[lb])
            inside = 0 <= phys < self.nb
            parts.append(self.values(phys, h, kind) if inside else torch.zeros(self.bs, self.d, dtype=torch.float64))
            live.append(torch.full((self.bs,), inside))
        if not parts:
            return torch.zeros(0, self.d, dtype=torch.float64), torch.zeros(0, dtype=torch.bool)
        return torch.cat(parts)[:n], torch.cat(live)[:n]

    def gather(self, tables, tokens: int, lens=None) -> tuple[torch.Tensor, torch.Tensor]:
        out = []
        for kind in (0, 1):
            x = torch.zeros(len(tables), self.hkv, tokens, self.d, dtype=torch.float64)
            for b in range(len(tables)):
                n = min(tokens, tables.shape[1] * self.bs, tokens if lens is None else max(0, int(lens[b])))
                for h in range(self.hkv):
                    x[b, h, :n] = self.row(tables[b], n, h, kind)[0]
            out.append(x)
        return out[0], out[1]

    def attend(self, q: torch.Tensor, tables, lens, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
        """``q [B, Hq, D]``: the output and, per (row, head), the largest |value| it averages."""
        b_, hq, d = q.shape
        out = torch.zeros(b_, hq, d, dtype=torch.float64)
        most = torch.zeros(b_, hq, dtype=torch.float64)
        for b in range(b_):
            n = min(max(0, int(lens[b])), tables.shape[1] * self.bs)
            for h in range(hq):
                kv = h // (hq // self.hkv)
                k, live = self.row(tables[b], n, kv, 0)
                v, _ = self.row(tables[b], n, kv, 1)
                k, v = k[live], v[live]
                if not len(k):
                    continue
                p = torch.softmax(k @ q[b, h].double() * scale, dim=0)
                out[b, h] = p @ v
                most[b, h] = v.abs().max()
        return out, most
