"""Plain 64-bit definitions of the serving operators, sequence by sequence, for the tests."""
from __future__ import annotations

import math

import torch


def lengths_to_offsets(new, device="cuda:0"):
    off = [0]
    for n in new:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int32, device=device)


def attention_rows(q, k, v, n, length, scale, causal=True):
    """(out [n, H, d], lse [n, H]) of the last n of `length` tokens over keys k / v
    [length, KV, d]; rows that see nothing get 0 and -inf.  Hidden keys take no part, whatever
    they hold."""
    h, kv = q.shape[1], k.shape[1]
    g = h // kv
    out = torch.zeros(n, h, q.shape[2], dtype=torch.float64, device=q.device)
    lse = torch.full((n, h), -math.inf, dtype=torch.float64, device=q.device)
    for i in range(n):
        m = max(0, length - n + i + 1) if causal else length
        if m == 0:
            continue
        for c in range(kv):
            s = (q[i, c * g:(c + 1) * g].double() @ k[:m, c].double().t()) * scale
            out[i, c * g:(c + 1) * g] = torch.softmax(s, 1) @ v[:m, c].double()
            lse[i, c * g:(c + 1) * g] = torch.logsumexp(s, 1)
    return out, lse


def attention_block(q, k, v, n, length, scale, causal=True):
    """attention_rows without the loop over rows (finite values only)."""
    h, kv, d = q.shape[1], k.shape[1], q.shape[2]
    g = h // kv
    hidden = torch.zeros(n, length, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.ones(n, length, dtype=torch.bool, device=q.device).triu(length - n + 1)
    s = torch.einsum("nhd,mhd->hnm", q.double(), k.double().repeat_interleave(g, 1)) * scale
    s.masked_fill_(hidden, -math.inf)
    return (torch.einsum("hnm,mhd->nhd", torch.softmax(s, 2), v.double().repeat_interleave(g, 1)),
            torch.logsumexp(s, 2).t())


def cache_rows(cache, page_table, b, length):
    """The first `length` slots of sequence b as [length, KV, d]."""
    page = cache.shape[1]
    slot = torch.arange(length, device=cache.device)
    return cache[page_table[b].long()[slot // page], slot % page]


def evict_choice(mass, pos, length, keep, recent):
    """(hole, mover) slots of one head, lists of equal length, by the definition."""
    if length <= keep:
        return [], []
    w, p = mass[:length].tolist(), pos[:length].tolist()
    edge = max(p) - recent
    w = [math.inf if p[j] > edge else (-math.inf if math.isnan(w[j]) else w[j]) for j in range(length)]
    best = sorted(range(length), key=lambda j: (-w[j], j))[:keep]
    kept = set(best)
    return [j for j in range(keep) if j not in kept], sorted(j for j in best if j >= keep)
