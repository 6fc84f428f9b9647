"""Paged-cache oracle (CPU, float64): the append of new tokens' keys and values (q / k RMSNorm, |temperature|, rotary
embedding) and the attention of a chunk of new tokens, over ragged batches described by page_table, cache_seqlens and
cu_seqlens_q.

The same attention core as ``oracle.attention`` and the pinned whole-LM oracle (norms, interleaved rotary, query head h
reading KV head h // (Hq / Hkv), scale head_dim ** -0.5, causal mask), written out per token from the definition. Test
infrastructure only (see ``oracle/__init__.py``).
"""

from __future__ import annotations

import math

import torch


def requests(cu, seqlens):
    """(request, first row, rows, keys) of every request with rows."""
    for b in range(len(seqlens)):
        first, rows = int(cu[b]), int(cu[b + 1]) - int(cu[b])
        if rows > 0:
            yield b, first, rows, int(seqlens[b])


def _slot(table, pages, page_size, b, j):
    """(page, row) of key position j of request b, or None when no page of the cache holds it."""
    if j < 0 or j // page_size >= table.shape[1]:
        return None
    page = int(table[b, j // page_size])
    return (page, j % page_size) if 0 <= page < pages else None


def append(proj, k_cache, v_cache, table, seqlens, cu, *, heads, kv_heads, temp=None, eps=1e-6, theta=10000.0,
           rotary=None, interleaved=True, positions=None):
    """q [N, heads, hd] float64; k_cache and v_cache ([pages, page_size, kv_heads, hd] float64) updated in place. Also
    the magnitude sqrt(a^2 + b^2) of every q and k element's rotation pair, for error bounds: (q, q magnitude,
    k magnitude cache)."""
    pages, page_size, _, hd = k_cache.shape
    rotary = hd if rotary is None else rotary
    N = proj.shape[0]
    q = torch.zeros(N, heads, hd, dtype=torch.float64)
    q_mag, k_mag = torch.zeros_like(q), torch.zeros_like(k_cache)
    for b, first, rows, keys in requests(cu, seqlens):
        for i in range(rows):
            t, j = first + i, keys - rows + i
            x = proj[t, : (heads + 2 * kv_heads) * hd].double().view(heads + 2 * kv_heads, hd)
            qk = x[: heads + kv_heads].clone()
            if eps is not None:
                qk /= (qk.square().mean(-1, keepdim=True) + eps).sqrt()
            if temp is not None:
                qk[:heads] *= temp.double().abs()[:, None]
            mag = qk.abs()
            at = j if positions is None else int(positions[t])
            for pair in range(rotary // 2):
                lo, hi = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + rotary // 2)
                angle = at * theta ** (-2.0 * pair / rotary)
                c, s = math.cos(angle), math.sin(angle)
                a, d = qk[:, lo].clone(), qk[:, hi].clone()
                qk[:, lo], qk[:, hi] = a * c - d * s, a * s + d * c
                mag[:, lo] = mag[:, hi] = (a * a + d * d).sqrt()
            q[t], q_mag[t] = qk[:heads], mag[:heads]
            slot = _slot(table, pages, page_size, b, j)
            if slot is not None:
                k_cache[slot], v_cache[slot] = qk[heads:], x[heads + kv_heads:]
                k_mag[slot] = mag[heads:]
    return q, q_mag, k_mag


def chunk(q, k_cache, v_cache, table, seqlens, cu, *, scale=None, causal=True, window=0, sinks=0, gate=None):
    """(out, spread, lse, size): out [N, Hq, hd] float64 (with a window the first ``sinks`` keys stay visible); spread = sum_j p_j |v_j| (gated), the scale of out's rounding
    errors; lse [N, Hq]; size = max_j scale * sum_d |q_d k_jd|, the scale of a score's rounding error."""
    N, Hq, hd = q.shape
    pages, page_size, Hkv, _ = k_cache.shape
    scale = hd ** -0.5 if scale is None else scale
    out, spread = torch.zeros(N, Hq, hd, dtype=torch.float64), torch.zeros(N, Hq, hd, dtype=torch.float64)
    lse, size = torch.full((N, Hq), -math.inf, dtype=torch.float64), torch.zeros(N, Hq, dtype=torch.float64)
    for b, first, rows, keys in requests(cu, seqlens):
        slots = [(j, _slot(table, pages, page_size, b, j)) for j in range(keys)]
        live = [(j, s) for j, s in slots if s is not None]
        if not live:
            continue
        at = torch.tensor([j for j, _ in live])
        page, row = torch.tensor([s[0] for _, s in live]), torch.tensor([s[1] for _, s in live])
        key, value = k_cache[page, row].double(), v_cache[page, row].double()  # [n, Hkv, hd]
        for i in range(rows):
            p = keys - rows + i
            seen = torch.ones(len(at), dtype=torch.bool)
            if causal:
                seen &= at <= p
            if window:
                seen &= (at > p - window) | (at < sinks)
            if not seen.any():
                continue
            for h in range(Hq):
                kk, vv = key[seen, h // (Hq // Hkv)], value[seen, h // (Hq // Hkv)]
                x = q[first + i, h].double()
                s = (kk @ x) * scale
                lse[first + i, h] = torch.logsumexp(s, 0)
                size[first + i, h] = ((kk * x).abs().sum(-1) * scale).max()
                w = torch.exp(s - lse[first + i, h])
                g = 1.0 if gate is None else torch.sigmoid(gate[first + i, h].double())
                out[first + i, h], spread[first + i, h] = (w @ vv) * g, (w @ vv.abs()) * g
    return out, spread, lse, size
