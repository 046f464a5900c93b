"""Speculative decoding restated on the CPU in 64 bits: attention of drafted tokens over a paged cache, the
verification of a tree of drafted tokens, and the moves that keep a path. Test infrastructure only.

The reference verifies one drafted token after the other (``runtime/phase2/worker_server.py:1010-1075``); the
formulas here are those of a whole tree at once."""

from __future__ import annotations

import numpy as np
import torch


def visible(parents) -> np.ndarray:
    """bool [T, T]: node i sees node j, an ancestor of its or itself."""
    t = len(parents)
    see = np.zeros((t, t), dtype=bool)
    for i in range(t):
        j = i
        while j >= 0:
            see[i, j] = True
            j = int(parents[j])
    return see


def row_tokens(pages: torch.Tensor, table, n: int) -> tuple[torch.Tensor, np.ndarray]:
    """Tokens 0..n of a row from pages [nb, H, bs, D] as float64 [H, n, D], and which of them a block holds."""
    nb, h, bs, d = pages.shape
    out, held = torch.zeros(h, n, d, dtype=torch.float64), np.zeros(n, dtype=bool)
    for j in range(n):
        block = int(table[j // bs])
        if 0 <= block < nb:
            out[:, j] = pages[block, :, j % bs].double()
            held[j] = True
    return out, held


def tree_attention(q, k_pages, v_pages, tables, seq_lens, see, counts, scale: float):
    """q [B, Hq, T, D]; see: bool [T, T] or one a row, or None (a chain). Returns out [B, T, Hq, D] and the sums of
    p |v| and the largest sum of |q k| * scale that a tolerance needs, all in 64 bits."""
    bsz, hq, t, d = q.shape
    _, hkv, bs, _ = k_pages.shape
    group = hq // hkv
    out = torch.zeros(bsz, t, hq, d, dtype=torch.float64)
    size = torch.zeros_like(out)
    reach = 0.0
    for b in range(bsz):
        count = t if counts is None else max(0, min(t, int(counts[b])))
        s = max(0, int(seq_lens[b]))
        n = min(s, tables.shape[1] * bs)
        ctx = s - count
        if n == 0:
            continue
        k, held = row_tokens(k_pages, tables[b], n)
        v, _ = row_tokens(v_pages, tables[b], n)
        m = np.tril(np.ones((t, t), dtype=bool)) if see is None else (see[b] if np.ndim(see) == 3 else see)
        for i in range(count):
            live = np.array([held[j] and (j < ctx or (j - ctx < count and m[i, j - ctx])) for j in range(n)])
            idx = torch.from_numpy(np.nonzero(live)[0])
            if len(idx) == 0:
                continue
            for h in range(hq):
                kk, vv = k[h // group][idx], v[h // group][idx]
                x = q[b, h, i].double()
                p = torch.softmax((kk @ x) * scale, dim=0)
                out[b, i, h] = p @ vv
                size[b, i, h] = p @ vv.abs()
                reach = max(reach, float((kk.abs() @ x.abs()).max()) * scale)
    return out, size, reach


def distribution(logits: np.ndarray, temperature: float) -> np.ndarray | None:
    """float64 [V], or None where the logits have none."""
    x = logits.astype(np.float64)
    if np.isnan(x).any() or not (x > -np.inf).any():
        return None
    if not temperature > 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p
    if np.isposinf(x).any():
        return None
    w = np.exp((x - x.max()) / float(temperature))
    return w / w.sum()


def verify_row(logits, tokens, parents, count: int, uniforms, temperature: float, draft=None):
    """logits [T, V]; returns the nodes kept and the token that follows (-1: none)."""
    if count <= 0:
        return [], None
    greedy = not temperature > 0
    node, kept = 0, [0]
    while True:
        r = distribution(logits[node], temperature)
        q = None if draft is None or greedy else distribution(draft[node], temperature)
        step = None
        for c in range(node + 1, count):
            if parents[c] != node or r is None:
                continue
            x = int(tokens[c])
            if not 0 <= x < len(r) or (draft is not None and not greedy and q is None):
                continue
            if float(uniforms[c]) * (1.0 if q is None else q[x]) < r[x]:
                step = c
                break
            if greedy:
                continue
            if q is None:
                rest = r.copy()
                rest[x] = 0.0
            else:
                rest = np.maximum(r - q, 0.0)
            if rest.sum() > 0:
                r = rest / rest.sum()
        if step is None:
            break
        node = step
        kept.append(step)
    if r is None:
        return kept, -1
    run = np.cumsum(r)
    beyond = np.nonzero(run > float(uniforms[0]) * run[-1])[0]
    return kept, int(beyond[0]) if len(beyond) else int(np.nonzero(r > 0)[0][-1])


def keep_tokens(pages: torch.Tensor, tables, starts, paths) -> torch.Tensor:
    """pages [L, nb, H, bs, D]; paths: the nodes kept of each row."""
    out = pages.clone()
    bs = pages.shape[3]
    for table, start, path in zip(tables, starts, paths):
        for j, node in enumerate(path):
            src, dst = int(start) + int(node), int(start) + j
            out[:, int(table[dst // bs]), :, dst % bs] = pages[:, int(table[src // bs]), :, src % bs]
    return out
