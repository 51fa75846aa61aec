"""CPU restatement, in 64 bits, of the operators that serve many continuations of shared prompts (test
infrastructure only): cache append, attention over shared prefixes, the draw of tokens.

They have no counterpart in the reference; every function states its operator's definition.
"""

from __future__ import annotations

import math

import numpy as np
import torch

DIM = 128
PAGE = 64


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """``x`` [..., 128] f64 with angles [..., R / 2]: the first R dims turned in pairs."""
    half = cos.shape[-1]
    lo = torch.arange(half) * (2 if interleaved else 1)
    hi = lo + (1 if interleaved else half)
    y = x.clone()
    y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return y


def append_rows(x, q_heads, kv_heads, g_q, g_k, eps, cos, sin, positions, interleaved):
    """``x`` [tokens, heads * 128] -> q, k, v [tokens, heads, 128] in f64, before any rounding."""
    x = x.double().reshape(x.shape[0], -1, DIM)
    at = positions.clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]

    def head(y, g):
        if g is not None:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * (1 + g.double())
        return rope(y, c, s, interleaved)

    return head(x[:, :q_heads], g_q), head(x[:, q_heads : q_heads + kv_heads], g_k), x[:, q_heads + kv_heads :]


def cache_values(cache: torch.Tensor) -> torch.Tensor:
    return cache.view(torch.float8_e4m3fn).double()


def attend(q, k_cache, v_cache, q_start, page_table, lens, group_start, prefix_table, prefix_lens, k_scale, v_scale, sm_scale):
    """Returns (out f64 [tokens, q_heads, 128], weight-averaged |v| likewise, largest sum |q_i k_i| of a token's keys in
    score units [tokens, q_heads], keys seen [tokens]); rows of no sequence are NaN in ``out``."""
    n_pages, _, hk, _ = k_cache.shape
    kc, vc = cache_values(k_cache) * k_scale, cache_values(v_cache) * v_scale
    tokens, hq, _ = q.shape
    G = hq // hk
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    mag, big, seen = torch.zeros_like(out), torch.zeros(tokens, hq, dtype=torch.float64), torch.zeros(tokens, dtype=torch.int64)

    def keys(table, count):
        """Existing (page, offset) pairs of the first ``count`` keys, and their positions."""
        pos = torch.arange(min(count, len(table) * PAGE))
        page = table[pos // PAGE].long()
        ok = (page >= 0) & (page < n_pages)
        return page[ok], pos[ok] % PAGE, pos[ok]

    for b in range(len(lens)):
        t0, t1 = int(q_start[b]), int(q_start[b + 1])
        n, ln = t1 - t0, min(int(lens[b]), page_table.shape[1] * PAGE)
        pre = None
        for g in range(0 if prefix_lens is None else len(prefix_lens)):
            if int(group_start[g]) <= b < int(group_start[g + 1]):
                pre = keys(prefix_table[g], int(prefix_lens[g]))
        own = keys(page_table[b], ln)
        for t in range(t0, t1):
            vis = own[2] < ln - n + 1 + (t - t0)
            page, at = own[0][vis], own[1][vis]
            if pre is not None:
                page, at = torch.cat([pre[0], page]), torch.cat([pre[1], at])
            seen[t] = len(page)
            k, v = kc[page, at], vc[page, at]
            for h in range(hq):
                if not len(page):
                    out[t, h] = 0
                    continue
                qh = q[t, h].double()
                s = k[:, h // G] @ qh * sm_scale
                p = torch.softmax(s, 0)
                out[t, h] = p @ v[:, h // G]
                mag[t, h] = p @ v[:, h // G].abs()
                big[t, h] = (k[:, h // G].abs() @ qh.abs()).max() * sm_scale
    return out, mag, big, seen


def sample_row(x: np.ndarray, u: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0):
    """(token, logprob, least relative distance of u from a border of the drawn token's share) of one row."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    best = int(np.argmax(x))
    if x[best] == -np.inf:
        return -1, -math.inf, 1.0
    greedy = not temperature > 0
    t = 1.0 if greedy else float(temperature)
    with np.errstate(invalid="ignore"):
        w = np.where(x == x[best], 1.0, np.where(x == -np.inf, 0.0, np.exp((x - x[best]) / t)))
    z = math.fsum(w)
    token, gap = best, 1.0
    if not greedy:
        order = np.argsort(-x, kind="stable")
        ahead = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        front = np.ones(len(x), bool)
        if top_k >= 1:
            front &= np.arange(len(x)) < top_k
        if top_p < 1:
            front &= ahead < max(top_p, 0.0) * z
        if min_p > 0:
            front &= w[order] >= min_p
        front[0] = True
        kept = np.sort(order[front])
        c = np.cumsum(w[kept])
        u = 0.0 if not u > 0 else u
        # u = 1 and above draws the last token of the running sum
        at = int(np.searchsorted(c, u * c[-1], side="right")) if u < 1 else int(np.searchsorted(c, c[-1], side="left"))
        at = min(at, len(kept) - 1)
        token = int(kept[at])
        gap = float(np.min(np.abs(c - u * c[-1])) / c[-1])
    if x[token] == x[best]:
        y = 0.0
    else:
        y = (x[token] - x[best]) / t
    return token, y - math.log(z), gap
