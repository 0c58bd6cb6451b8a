"""Speculative decoding over the paged cache, in 64 bits on the CPU: attention
of draft trees, their verification, and the cache moves, written from the
definitions (csrc/tree_attention.cu, csrc/verify.cu) one element after another.
"""
from __future__ import annotations

import math

import torch


def tree_attention(q, pool, tables, q_start, q_len, ctx_len, masks, hq, hkv, hd):
    """``(out, spread)`` float64 ``[rows, hq * hd]``: the attention of every
    draft node and softmax-weighted ``|v|`` (what roundings of the weights
    are relative to).  ``masks[row]``: Python int, bit j = node j is seen.
    Rows of no sequence are NaN; keys a row does not see are left out, not
    multiplied by zero."""
    bs, G = pool.shape[3], hq // hkv
    out = torch.full((q.shape[0], hq * hd), math.nan, dtype=torch.float64)
    spread = out.clone()
    pool, q = pool.double(), q.double()
    for a, k, c, table in zip(q_start, q_len, ctx_len, tables):
        if k == 0:
            continue
        kv = torch.cat([pool[b] for b in table[:-(-c // bs)]], 2)[:, :, :c] if c else None
        for i in range(k):
            seen = list(range(c - k)) + [c - k + j for j in range(k) if masks[a + i] >> j & 1]
            for h in range(hq):
                cols = slice(h * hd, (h + 1) * hd)
                if not seen:
                    out[a + i, cols] = spread[a + i, cols] = 0.0
                    continue
                key, val = kv[0, h // G, seen], kv[1, h // G, seen]
                p = torch.softmax(key @ q[a + i, cols] / math.sqrt(hd), 0)
                out[a + i, cols] = p @ val
                spread[a + i, cols] = p @ val.abs()
    return out, spread


def verify_greedy(ids, parents, q_start, q_len, target_ids, width):
    took, paths, nexts = [], [], []
    for a, k in zip(q_start, q_len):
        path = [0] if k else []
        while path and len(path) < width:
            kids = [i for i in range(1, k) if parents[a + i] == path[-1]
                    and ids[a + i] == target_ids[a + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        took.append(max(0, len(path) - 1))
        nexts.append(target_ids[a + path[-1]] if path else -1)
        paths.append(path + [-1] * (width - len(path)))
    return took, paths, nexts


def verify(ids, parents, q_start, q_len, probs, uniforms, width, draft_probs=None, draft_rows=None):
    """Speculative sampling over draft trees (the formulas of csrc/verify.cu)."""
    took, paths, nexts = [], [], []
    for a, k in zip(q_start, q_len):
        if k == 0:
            took.append(0), paths.append([-1] * width), nexts.append(-1)
            continue
        path = [0]
        while True:
            c, accepted = path[-1], None
            r = probs[a + c].double().clone()
            row = -1 if draft_rows is None else int(draft_rows[a + c])
            d0 = draft_probs[row].double().clone() if row >= 0 else None
            gone = 0.0
            kids = [i for i in range(1, k) if parents[a + i] == c] if len(path) < width else []
            for i in kids:
                x, u = int(ids[a + i]), float(uniforms[a + i])
                if d0 is None:
                    if r[x] > 0 and u * (1 - gone) < r[x]:
                        accepted = i
                        break
                    gone += float(r[x])
                    r[x] = 0
                    continue
                left = 1 - gone
                share = float(d0[x]) / left if left > 0 else 0.0
                if share <= 0:
                    continue
                if u * share < r[x]:
                    accepted = i
                    break
                rest = (r - d0 / left).clamp(min=0)
                if rest.sum() > 0:
                    r = rest / rest.sum()
                gone += float(d0[x])
                d0[x] = 0
            if accepted is None:
                break
            path.append(accepted)
        cdf = r.cumsum(0)
        over = (cdf > float(uniforms[a]) * cdf[-1]).nonzero()
        took.append(len(path) - 1)
        paths.append(path + [-1] * (width - len(path)))
        nexts.append(int(over[0]) if len(over) else -1)
    return took, paths, nexts


def keep_path(pools, tables, q_len, ctx_len, paths, n_accepted):
    """The pools after every accepted node moved to its place behind the root."""
    pools = [p.clone() for p in pools]
    for pool in pools:
        bs, old = pool.shape[3], pool.clone()
        for table, k, c, path, n in zip(tables, q_len, ctx_len, paths, n_accepted):
            for j in range(1, n + 1):
                s, d = c - k + path[j], c - k + j
                pool[table[d // bs], :, :, d % bs] = old[table[s // bs], :, :, s % bs]
    return pools
