"""K and V in pages, in torch and 64 bits (TEST INFRASTRUCTURE ONLY; the product never imports it).

Rows by a table of pages, the rotation of pairs of columns, and softmax attention of new tokens over their sequences' rows, as
``include/diffcache_hip.h`` defines them (``dc_paged_store``, ``dc_paged_tokens``).  The reference has no pages: PARITY UNPINNED there.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch


def spans(n_b: int, start: Optional[Sequence[int]], cu: Optional[Sequence[int]], counts: Optional[Sequence[int]],
          max_new: int, n_tokens: int) -> List[Tuple[int, int, int]]:
    """(place of the first token, tokens, rows held before) of every sequence."""
    out = []
    for b in range(n_b):
        if cu is not None:
            first = min(max(cu[b], 0), n_tokens)
            count = min(min(max(cu[b + 1], first), n_tokens) - first, max_new)
        else:
            first = b * max_new
            count = max_new if counts is None else min(max(counts[b], 0), max_new)
        out.append((first, count, 0 if start is None else min(max(start[b], 0), 1 << 30)))
    return out


def rotate(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
           sections: Optional[Sequence[int]] = None) -> torch.Tensor:
    """x (tokens, heads, hd) rotated by pos (tokens, axes), in 64 bits."""
    half = inv_freq.numel()
    out = x.double().clone()
    axis = [0] * half if sections is None else [i for i, n in enumerate(sections) for _ in range(n)]
    for f in range(half):
        t = pos[:, axis[f]].double() * inv_freq[f].double()
        a, b = (2 * f, 2 * f + 1) if interleaved else (f, f + half)
        xa, xb = x[..., a].double(), x[..., b].double()
        c, s = t.cos()[:, None], t.sin()[:, None]
        out[..., a], out[..., b] = xa * c - xb * s, xb * c + xa * s
    return out


def place(table_row: Sequence[int], row: int, page: int, n_pages: int) -> Optional[Tuple[int, int]]:
    """(page, row there) of a sequence's row; None where there is none."""
    i = row // page
    if i >= len(table_row) or not 0 <= table_row[i] < n_pages:
        return None
    return table_row[i], row % page


def attended(p: int, table_row: Sequence[int], page: int, n_pages: int, n_rows: int, n_sink: int = 0, window: int = 0) -> List[int]:
    """The rows that a token at row p attends to."""
    rows = range(min(p + 1, n_rows))
    return [r for r in rows if (window == 0 or r > p - window or r < n_sink) and place(table_row, r, page, n_pages) is not None]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """q (heads, hd) over k, v (rows, hd), all in 64 bits: out, lse, and sum of p |v|, what errors of weights are relative to."""
    if k.shape[0] == 0:
        zero = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return zero, torch.full(q.shape[:1], -math.inf, dtype=torch.float64, device=q.device), zero
    s = (q @ k.t()) * scale
    p = torch.softmax(s, -1)
    return p @ v, torch.logsumexp(s, -1), p @ v.abs()


def attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, span, n_rows: int, scale: float,
           n_sink: int = 0, window: int = 0):
    """q (tokens, heads, hd) packed or padded -> out, lse, weight of the tokens that count (NaN elsewhere)."""
    n_pages, h, page, hd = k_pages.shape
    group = q.shape[1] // h
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    weight, lse = out.clone(), out[..., 0].clone()
    for b, (first, count, start) in enumerate(span):
        row = table[b].tolist()
        for i in range(count):
            keep = attended(start + i, row, page, n_pages, n_rows, n_sink, window)
            at = [place(row, r, page, n_pages) for r in keep]
            ids = torch.tensor([a for a, _ in at], dtype=torch.long, device=q.device)
            slots = torch.tensor([s for _, s in at], dtype=torch.long, device=q.device)
            for j in range(h):
                mine = slice(j * group, (j + 1) * group)
                o, s, w = attention(q[first + i, mine].double(), k_pages[ids, j, slots].double(), v_pages[ids, j, slots].double(), scale)
                out[first + i, mine], lse[first + i, mine], weight[first + i, mine] = o, s, w
    return out, lse, weight
