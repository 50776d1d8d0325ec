"""Drafted trees, their commit, beam selection and copies in the cache, written out plainly in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import torch


def line_of(parent, x):
    """Node x and its ancestors, x first."""
    out = [x]
    while parent[out[-1]] >= 0:
        out.append(parent[out[-1]])
    return out


def tree_attention(q, k_pool, v_pool, parents, cached, tables, page_size, num_kv_heads, scale, window=None, sink=None, softcap=None):
    """q [T, Hq, D]; pools [pages, Hkv, P, D]; parents: a list per segment; tables: page ids per segment.  Returns float64 [T, Hq, D] and,
    per (node, head), the scores' error scale sum_d |q_d k_d| at its largest over the visible keys."""
    q, k_pool, v_pool = q.double(), k_pool.double(), v_pool.double()
    G = q.shape[1] // num_kv_heads
    out, size, t = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64), 0
    for parent, c, table in zip(parents, cached, tables):
        for x in range(len(parent)):
            line = line_of(parent, x)
            p = c + len(line) - 1
            slots = [j for j in range(c) if not window or j > p - window] + [c + y for i, y in enumerate(line) if not window or i < window]
            pages, rows = [table[j // page_size] for j in slots], [j % page_size for j in slots]
            k, v = k_pool[pages, :, rows], v_pool[pages, :, rows]             # [keys, Hkv, D]
            for h in range(q.shape[1]):
                prods = k[:, h // G] * q[t, h]
                s = prods.sum(-1) * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                m = s.max()
                w = torch.exp(s - m)
                total = w.sum() + (math.exp(float(sink[h]) - float(m)) if sink is not None else 0.0)
                out[t, h] = (w[:, None] * v[:, h // G]).sum(0) / total
                size[t, h] = prods.abs().sum(-1).max() * scale
            t += 1
    return out, size


def walk(tokens, parent, sampled):
    path = [0]
    while True:
        x = path[-1]
        children = [y for y in range(len(parent)) if parent[y] == x and tokens[y] == sampled[x]]
        if not children:
            return path
        path.append(min(children))


def commit(pool, tables, cached, paths, page_size):
    """The pool [layers, 2, pages, heads, P, n] (or [layers, pages, P, n]) behind the moves, from a copy."""
    old, new = pool.clone(), pool.clone()
    for table, c, path in zip(tables, cached, paths):
        for i, x in enumerate(path):
            (ps, rs), (pd, rd) = divmod(c + x, page_size), divmod(c + i, page_size)
            if i == x or table[ps] < 0 or table[pd] < 0:
                continue
            if pool.dim() == 6:
                new[:, :, table[pd], :, rd] = old[:, :, table[ps], :, rs]
            else:
                new[:, table[pd], rd] = old[:, table[ps], rs]
    return new


def beam_select(logits, scores, beams, keep):
    """Per request the best (total, beam, token), in float64, ties to the lowest (beam, token)."""
    x, scores = logits.double().numpy(), scores.double().numpy()
    V, out = x.shape[1], []
    with np.errstate(all="ignore"):
        for r in range(x.shape[0] // beams):
            rows = x[r * beams:(r + 1) * beams]
            top = rows.max(1, keepdims=True)
            total = scores[r * beams:(r + 1) * beams, None] + (rows - top - np.log(np.exp(rows - top).sum(1, keepdims=True)))
            total[~np.isfinite(scores[r * beams:(r + 1) * beams])] = -np.inf
            total = np.where(np.isnan(total), -np.inf, total).reshape(-1)
            order = np.argsort(-total, kind="stable")[:keep]
            out.append([(float(total[i]), int(i // V), int(i % V)) for i in order])
    return out


def copy_pages(pool, src, dst, rows):
    out = pool.clone()
    for a, b, n in zip(src, dst, rows):
        if a < 0 or b < 0 or n <= 0:
            continue
        if pool.dim() == 6:
            out[:, :, b, :, :n] = pool[:, :, a, :, :n]
        else:
            out[:, b, :n] = pool[:, a, :n]
    return out
