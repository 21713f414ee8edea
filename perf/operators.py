"""The serving operators' cases: what they are measured and compared on.

Five operators that serve a prompt and what follows it: causal attention over packed
prompts with grouped heads, the append of new keys and values to a paged cache, the
attention of a chunk of new tokens (or single ones) over that cache, the attention
weight that each cached token has gathered, and the eviction of the tokens that gathered
least.  ``run`` computes a case either in plain form, elementary torch operations in
fp32, or, with ``own`` set, by the calls a user makes of the package's operators.

Layouts, the same for both: tokens of all sequences packed one after another, sequence b
at rows seq_offsets[b] .. seq_offsets[b + 1]; a cache of pages [pages, page, kv heads,
head_dim] with a table [sequences, pages per sequence] of page numbers; cache_lens counts
the tokens in the cache, the new ones included, so new token i of n is at slot
len - n + i and sees the slots up to its own.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # One short prompt, as an interactive request brings it: latency counts.
        {"name": "prompt_one_short", "op": "prompt", "dtype": "fp16", "batch": 1, "heads": 16,
         "kv_heads": 4, "head_dim": 64, "len_lo": 77, "len_hi": 77},
        # A batch of ragged prompts of the length and width of the framework's widest stack.
        {"name": "prompt_ragged_256", "op": "prompt", "dtype": "fp16", "batch": 256, "heads": 16,
         "kv_heads": 4, "head_dim": 64, "len_lo": 128, "len_hi": 256},
        # Long documents, wide heads shared by four query heads each.
        {"name": "prompt_long", "op": "prompt", "dtype": "bf16", "batch": 2, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "len_lo": 3001, "len_hi": 4096},
        # Single tokens of a few conversations: the smallest decode step.
        {"name": "step_few", "op": "attend", "dtype": "fp16", "batch": 4, "heads": 16,
         "kv_heads": 4, "head_dim": 64, "page": 16, "new_lo": 1, "new_hi": 1, "len_lo": 200,
         "len_hi": 1000},
        # Single tokens of a full batch, conversations of very different lengths.
        {"name": "step_batch", "op": "attend", "dtype": "bf16", "batch": 64, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "new_lo": 1, "new_hi": 1, "len_lo": 100,
         "len_hi": 8192},
        # Chunks of prompts whose beginning is in the cache already.
        {"name": "chunk_512", "op": "attend", "dtype": "bf16", "batch": 4, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "new_lo": 300, "new_hi": 512, "len_lo": 2000,
         "len_hi": 8192},
        # The new keys and values of a decode step, with the bookkeeping that eviction wants.
        {"name": "append_step", "op": "append", "dtype": "bf16", "batch": 64, "kv_heads": 8,
         "head_dim": 128, "page": 64, "new_lo": 1, "new_hi": 1, "len_lo": 100, "len_hi": 2048},
        # Those of whole prompts.
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "batch": 8, "kv_heads": 8,
         "head_dim": 128, "page": 64, "new_lo": 2000, "new_hi": 4096, "len_lo": 4096,
         "len_hi": 4096},
        # What a decode step adds to the weight of every cached token.
        {"name": "mass_step", "op": "mass", "dtype": "bf16", "batch": 32, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "new_lo": 1, "new_hi": 1, "len_lo": 1000,
         "len_hi": 4096},
        # What the chunks of prompts add.
        {"name": "mass_chunk", "op": "mass", "dtype": "bf16", "batch": 4, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "new_lo": 300, "new_hi": 512,
         "len_lo": 2000, "len_hi": 8192},
        # A budget kept while decoding: a few tokens above it are dropped now and then.
        {"name": "evict_budget", "op": "evict", "dtype": "bf16", "batch": 64, "kv_heads": 8,
         "head_dim": 128, "page": 64, "len_lo": 1025, "len_hi": 1152, "keep": 1024, "recent": 128},
        # A long prompt cut down once.
        {"name": "evict_prompt", "op": "evict", "dtype": "bf16", "batch": 2, "kv_heads": 8,
         "head_dim": 128, "page": 64, "len_lo": 20000, "len_hi": 32768, "keep": 4096,
         "recent": 256},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(("prompt", "attend", "attend", "append", "mass", "evict"))
    case = {"op": op, "dtype": rng.choice(("fp16", "bf16")), "head_dim": rng.choice((32, 64, 64, 128, 128, 256)),
            "kv_heads": rng.choice((1, 2, 3, 4, 8))}
    if op in ("prompt", "attend", "mass"):
        case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 4, 5, 8))
    if op != "prompt":
        case["page"] = rng.choice((16, 32, 64, 128))
    d, hkv = case["head_dim"], case["kv_heads"]
    if op == "prompt":
        hi = _log_int(rng, 1, 4096)
        # padded scores of the plain form: at most those of the largest listed case
        case["batch"] = max(1, min(_log_int(rng, 1, 256), int(1.0e9 / (case["heads"] * hi * hi))))
        case["len_hi"], case["len_lo"] = hi, max(1, int(hi * rng.uniform(0.1, 1)))
    elif op in ("attend", "mass"):
        hi = _log_int(rng, 16, 8192)
        new = 1 if rng.random() < 0.5 else min(hi, _log_int(rng, 2, 512))
        most = min(5.0e8 / (case["heads"] * hi * new), 64 * 8192 * 8 * 128 / (hi * hkv * d))
        case["batch"] = max(1, min(_log_int(rng, 1, 96), int(most)))
        case["new_lo"], case["new_hi"] = max(1, int(new * rng.uniform(0.1, 1))), new
        case["len_hi"], case["len_lo"] = hi, max(new, int(hi * rng.uniform(0.1, 1)))
    elif op == "append":
        hi = _log_int(rng, 16, 4096)
        new = 1 if rng.random() < 0.5 else min(hi, _log_int(rng, 2, 4096))
        case["batch"] = max(1, min(_log_int(rng, 1, 96), int(8 * 4096 * 8 * 128 / (hi * hkv * d))))
        case["new_lo"], case["new_hi"] = max(1, int(new * rng.uniform(0.1, 1))), new
        case["len_hi"], case["len_lo"] = hi, max(new, int(hi * rng.uniform(0.3, 1)))
    else:
        hi = _log_int(rng, 64, 32768)
        case["batch"] = max(1, min(_log_int(rng, 1, 64), int(2 * 32768 * 8 * 128 / (hi * hkv * d))))
        case["len_hi"], case["len_lo"] = hi, max(1, int(hi * rng.uniform(0.3, 1)))
        case["keep"] = max(1, int(hi * rng.uniform(0.1, 0.95)))
        case["recent"] = int(case["keep"] * rng.uniform(0, 0.5))
    return case


def _lengths(case):
    """Tokens per sequence (new ones, cached ones), from the case alone: spread evenly
    over the case's range, in an order that is not sorted."""
    b = case["batch"]

    def spread(lo, hi, step):
        return [lo + (hi - lo) * ((i * step + b - 1) % b) // max(1, b - 1) for i in range(b)]

    if case["op"] == "prompt":
        n = spread(case["len_lo"], case["len_hi"], 1 if b < 3 else 2 * (b // 4) + 1)
        return n, n
    total = spread(case["len_lo"], case["len_hi"], 1 if b < 3 else 2 * (b // 4) + 1)
    if case["op"] == "evict":
        return [0] * b, total
    return spread(case["new_lo"], case["new_hi"], 1), total


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op, b, hkv, d = case["op"], case["batch"], case["kv_heads"], case["head_dim"]
    new, total = _lengths(case)
    state = {"op": op, "dtype": dtype, "max_new": max(new), "max_len": max(total)}

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    state["seq_offsets"] = ints(offsets)
    t = offsets[-1]
    if "heads" in case:
        # q | k | v of a token side by side, as one projection writes them.
        h = case["heads"]
        qkv = normal(t, (h + 2 * hkv) * d)
        q, k, v = qkv.split((h * d, hkv * d, hkv * d), dim=1)
        # Scores of a standard deviation of 1.5: attention that looks at some tokens more.
        q.mul_(1.5)
        state["q"] = q.view(t, h, d)
        state["k"], state["v"] = k.view(t, hkv, d), v.view(t, hkv, d)
    elif op == "append":
        kv = normal(t, 2 * hkv * d)
        state["k"], state["v"] = kv[:, : hkv * d].view(t, hkv, d), kv[:, hkv * d:].view(t, hkv, d)
    if op == "prompt":
        return state
    page = case["page"]
    per_seq = -(-max(total) // page)
    pages = b * per_seq + 3
    state["k_cache"] = normal(pages, page, hkv, d)
    state["v_cache"] = normal(pages, page, hkv, d)
    # Pages in the order in which an allocator that has run for a while hands them out.
    order = torch.randperm(pages, device=dev, generator=g)[: b * per_seq]
    state["page_table"] = order.to(torch.int32).view(b, per_seq).contiguous()
    state["cache_lens"] = ints(total)
    cap = per_seq * page
    slot = torch.arange(cap, device=dev)
    live = slot[None, None, :] < state["cache_lens"][:, None, None]
    if op in ("append", "mass", "evict"):
        # Gathered weights: a few tokens have most of it, some have none.
        mass = torch.exp(2 * torch.randn(b, hkv, cap, device=dev, generator=g))
        mass = mass * (torch.rand(b, hkv, cap, device=dev, generator=g) > 0.1)
        state["mass"] = torch.where(live, mass, torch.zeros_like(mass)).contiguous()
    if op in ("append", "evict"):
        # Earlier evictions have mixed the slots: positions rise, with gaps, in an order of their own.
        keys = torch.rand(b, hkv, cap, device=dev, generator=g).masked_fill_(~live, 2.0)
        rank = keys.argsort(dim=2).argsort(dim=2)
        state["positions"] = torch.where(live, 3 * rank, torch.full_like(rank, -1)).to(torch.int32).contiguous()
        state["seen"] = (3 * state["cache_lens"] + 1).to(torch.int32)
    if op == "mass":
        # The log-sum-exp that the attention of the same queries returned.
        state["lse"] = _attend_plain(state, want_out=False)
    if op == "evict":
        state["keep"], state["recent"] = case["keep"], case["recent"]
    return state


# ------------------------------------------------------------------------- plain forms
def _padded(x, state):
    """Packed rows [T, heads, d] as [B, heads, most new tokens, d] in fp32, and which of them are there."""
    off = state["seq_offsets"].long()
    i = torch.arange(state["max_new"], device=off.device)
    there = i[None, :] < (off[1:] - off[:-1])[:, None]
    rows = (off[:-1, None] + i[None, :]).clamp_(max=x.shape[0] - 1)
    return x[rows].float().transpose(1, 2), there, rows


def _slots(state):
    """Page and slot inside it of every cached token [B, longest], and which of them are there."""
    table, page = state["page_table"].long(), state["k_cache"].shape[1]
    j = torch.arange(state["max_len"], device=table.device)
    return table[:, j // page], j % page, j[None, :] < state["cache_lens"][:, None]


def _cached(cache, state):
    pages, slots, _ = _slots(state)
    return cache[pages, slots[None, :].expand_as(pages)].float().transpose(1, 2)


def _grouped(q, hkv):
    b, h, n, d = q.shape
    return q.reshape(b, hkv, (h // hkv) * n, d)


def _masked_scores(state, q, k, there, lens):
    """Scores [B, heads, new, keys] of the scaled product, -inf where a token sees no key."""
    b, h, n, d = q.shape
    s = torch.matmul(_grouped(q, k.shape[1]) * d**-0.5, k.transpose(2, 3)).view(b, h, n, k.shape[2])
    new = there.sum(1)
    at = (lens - new)[:, None] + torch.arange(n, device=q.device)[None, :]
    j = torch.arange(k.shape[2], device=q.device)
    seen = (j[None, None, :] <= at[:, :, None]) & there[:, :, None]
    return s.masked_fill_(~seen[:, None], float("-inf"))


def _softmax_product(s, v, there, want_out=True):
    top = s.amax(dim=3, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(s.sub_(top))
    total = e.sum(dim=3, keepdim=True)
    lse = (torch.log(total) + top).squeeze(3)
    if not want_out:
        return None, lse
    b, h, n, _ = e.shape
    o = torch.matmul(_grouped(e, v.shape[1]), v).view(b, h, n, v.shape[3])
    return o / torch.where(total > 0, total, torch.ones_like(total)), lse


def _attend_plain(state, want_out=True):
    q, there, rows = _padded(state["q"], state)
    if state["op"] == "prompt":
        k, v = _padded(state["k"], state)[0], _padded(state["v"], state)[0]
        lens = there.sum(1)
    else:
        k, v = _cached(state["k_cache"], state), _cached(state["v_cache"], state)
        v = v.masked_fill(~_slots(state)[2][:, None, :, None], 0)
        lens = state["cache_lens"].long()
    s = _masked_scores(state, q, k, there, lens)
    o, lse = _softmax_product(s, v, there, want_out)
    lse = lse.transpose(1, 2)[there]
    return (o.transpose(1, 2)[there].to(state["dtype"]), lse) if want_out else lse


def _append_plain(state):
    off, lens = state["seq_offsets"].long(), state["cache_lens"].long()
    new = off[1:] - off[:-1]
    b = torch.repeat_interleave(torch.arange(len(new), device=off.device), new, output_size=state["k"].shape[0])
    i = torch.arange(state["k"].shape[0], device=off.device) - off[b]
    slot = lens[b] - new[b] + i
    page = state["k_cache"].shape[1]
    at = state["page_table"].long()[b, slot // page]
    state["k_cache"][at, slot % page] = state["k"]
    state["v_cache"][at, slot % page] = state["v"]
    state["positions"][b, :, slot] = (state["seen"].long()[b] - new[b] + i).to(torch.int32)[:, None]
    state["mass"][b, :, slot] = 0.0
    return {"k_cache": state["k_cache"], "v_cache": state["v_cache"], "positions": state["positions"],
            "mass": state["mass"]}


def _mass_plain(state):
    q, there, rows = _padded(state["q"], state)
    k = _cached(state["k_cache"], state)
    s = _masked_scores(state, q, k, there, state["cache_lens"].long())
    lse = state["lse"][rows].transpose(1, 2).masked_fill(~there[:, None, :], 0)
    b, h, n, keys = s.shape
    w = torch.exp(s.sub_(lse[..., None])).view(b, k.shape[1], -1, keys).sum(dim=2)
    out = state["mass"].clone()
    out[:, :, :keys] += w
    return out


def _evict_plain(state):
    mass, pos, lens, keep = state["mass"], state["positions"], state["cache_lens"], state["keep"]
    b, hkv, cap = mass.shape
    slot = torch.arange(cap, device=mass.device)
    live = slot[None, None, :] < lens[:, None, None]
    newest = pos.masked_fill(~live, -1).amax(dim=2, keepdim=True)
    value = torch.where(torch.isnan(mass), torch.full_like(mass, float("-inf")), mass)
    value = value.masked_fill(pos > newest - state["recent"], float("inf"))
    value = value.masked_fill(~live, float("-inf"))  # behind the live ones, which the stable order keeps first
    order = value.sort(dim=2, descending=True, stable=True).indices
    chosen = torch.zeros(b, hkv, cap, dtype=torch.bool, device=mass.device)
    chosen.scatter_(2, order[:, :, :keep], True)
    chosen &= live
    over = (lens > keep)[:, None, None]
    hole = over & ~chosen & (slot < keep)
    mover = over & chosen & (slot >= keep)
    # The i-th mover fills the i-th hole: both lists are in the order of (sequence, head, slot).
    hb, hh, hs = hole.nonzero(as_tuple=True)
    mb, mh, ms = mover.nonzero(as_tuple=True)
    page, table = state["k_cache"].shape[1], state["page_table"].long()
    for cache in (state["k_cache"], state["v_cache"]):
        cache[table[hb, hs // page], hs % page, hh] = cache[table[mb, ms // page], ms % page, mh]
    new_mass, new_pos = mass.clone(), pos.clone()
    new_mass[hb, hh, hs], new_pos[hb, hh, hs] = mass[mb, mh, ms], pos[mb, mh, ms]
    lens = lens.clamp(max=keep)
    gone = slot[None, None, :] >= lens[:, None, None]
    return {"mass": new_mass.masked_fill_(gone, 0.0), "positions": new_pos.masked_fill_(gone, -1),
            "cache_lens": lens, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _run_own(state):
    import optimized_transformer  # noqa: F401  (registers the package)
    from tttj_2026_b200 import ops

    op = state["op"]
    if op == "prompt":
        return ops.prompt_attention(state["q"], state["k"], state["v"], state["seq_offsets"], return_lse=True)
    if op == "append":
        ops.cache_append(state["k"], state["v"], state["k_cache"], state["v_cache"], state["page_table"],
                         state["seq_offsets"], state["cache_lens"], positions=state["positions"],
                         mass=state["mass"], seen=state["seen"])
        return {"k_cache": state["k_cache"], "v_cache": state["v_cache"], "positions": state["positions"],
                "mass": state["mass"]}
    if op == "attend":
        return ops.cache_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"],
                                   state["seq_offsets"], state["cache_lens"], max_new=state["max_new"],
                                   return_lse=True)
    if op == "mass":
        return ops.cache_mass(state["q"], state["lse"], state["k_cache"], state["page_table"],
                              state["seq_offsets"], state["cache_lens"], state["mass"],
                              max_new=state["max_new"])
    mass, positions, lens = ops.cache_evict(state["mass"], state["positions"], state["k_cache"],
                                            state["v_cache"], state["page_table"], state["cache_lens"],
                                            state["keep"], recent=state["recent"])
    return {"mass": mass, "positions": positions, "cache_lens": lens, "k_cache": state["k_cache"],
            "v_cache": state["v_cache"]}


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op in ("prompt", "attend"):
        return _attend_plain(state)
    return {"append": _append_plain, "mass": _mass_plain, "evict": _evict_plain}[op](state)


# --------------------------------------------------------------------------- the floor
def work(case):
    new, total = _lengths(case)
    op, hkv, d = case["op"], case["kv_heads"], case["head_dim"]
    t = sum(new)
    h = case.get("heads", 0)
    # Keys that the tokens of a sequence see, together.
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, total))
    row = hkv * d * 2  # one token's keys or values
    if op == "prompt":
        return {"bytes": 2 * t * h * d * 2 + 2 * t * row + 4 * t * h, "flops": 4 * d * h * pairs}
    table = sum(-(-m // case["page"]) for m in total) * 4
    if op == "attend":
        return {"bytes": 2 * t * h * d * 2 + 2 * sum(total) * row + 4 * t * h + table, "flops": 4 * d * h * pairs}
    if op == "append":
        return {"bytes": 4 * t * row + 8 * t * hkv, "flops": 0}
    if op == "mass":
        return {"bytes": t * h * d * 2 + 4 * t * h + sum(total) * row + 8 * sum(total) * hkv + table,
                "flops": 2 * d * h * pairs}
    # Rows that move: at least as many as tokens are kept from behind the budget; taken at
    # the share that a choice by chance leaves there.
    moved = sum(max(0, m - case["keep"]) * min(case["keep"], m) / m for m in total) * hkv
    return {"bytes": 16 * sum(total) * hkv + moved * 4 * d * 2, "flops": 0}


# ------------------------------------------------------------------ 64-bit definitions
def exact(case, seed):
    state = prepare(case, seed)
    new, total = _lengths(case)
    op, hkv, d = case["op"], case["kv_heads"], case["head_dim"]
    off, dev = [0], torch.device("cuda")
    for n in new:
        off.append(off[-1] + n)

    def rows_of(b, slots):
        """Row numbers of the cache seen as [pages * page, kv heads, d]."""
        page = case["page"]
        s = torch.tensor(slots, dtype=torch.long, device=dev)
        return state["page_table"][b].long()[s // page] * page + s % page

    if op in ("prompt", "attend", "mass"):
        group = case["heads"] // hkv
        t = off[-1]
        out = torch.zeros(t, case["heads"], d, dtype=torch.float64, device=dev)
        lse = torch.zeros(t, case["heads"], dtype=torch.float64, device=dev)
        mass = state["mass"].double() if op == "mass" else None
        for b, (n, m) in enumerate(zip(new, total)):
            mine = slice(off[b], off[b + 1])
            if op == "prompt":
                keys, values = state["k"][mine].double(), state["v"][mine].double()
            else:
                at = rows_of(b, list(range(m)))
                keys = state["k_cache"].flatten(0, 1)[at].double()
                values = state["v_cache"].flatten(0, 1)[at].double()
            hidden = torch.ones(n, m, dtype=torch.bool, device=dev).triu(m - n + 1)
            for g in range(hkv):
                heads = slice(g * group, (g + 1) * group)
                s = torch.einsum("nhd,md->hnm", state["q"][mine, heads].double(), keys[:, g]) / math.sqrt(d)
                s.masked_fill_(hidden, -math.inf)
                if op == "mass":
                    given = state["lse"][mine, heads].double().t()
                    mass[b, g, :m] += torch.exp(s - given[:, :, None]).sum((0, 1))
                else:
                    out[mine, heads] = torch.einsum("hnm,md->nhd", torch.softmax(s, 2), values[:, g])
                    lse[mine, heads] = torch.logsumexp(s, 2).t()
        return mass if op == "mass" else (out, lse)
    kc, vc = state["k_cache"].clone(), state["v_cache"].clone()
    kr, vr = kc.flatten(0, 1), vc.flatten(0, 1)
    mass, pos = state["mass"].clone(), state["positions"].clone()
    if op == "append":
        for b, (n, m) in enumerate(zip(new, total)):
            at = rows_of(b, list(range(m - n, m)))
            kr[at], vr[at] = state["k"][off[b]:off[b + 1]], state["v"][off[b]:off[b + 1]]
            first = int(state["seen"][b]) - n
            pos[b, :, m - n:m] = torch.arange(first, first + n, dtype=torch.int32, device=dev)
            mass[b, :, m - n:m] = 0
        return {"k_cache": kc, "v_cache": vc, "positions": pos, "mass": mass.double()}
    keep, lens = case["keep"], []
    for b, m in enumerate(total):
        lens.append(min(m, keep))
        for g in range(hkv):
            if m > keep:
                w, p = mass[b, g, :m].tolist(), pos[b, g, :m].tolist()
                edge = max(p) - case["recent"]
                w = [math.inf if p[j] > edge else w[j] for j in range(m)]
                best = sorted(range(m), key=lambda j: (-w[j], j))[:keep]
                kept = set(best)
                hole = [j for j in range(keep) if j not in kept]
                mover = sorted(j for j in best if j >= keep)
                to, src = rows_of(b, hole), rows_of(b, mover)
                kr[to, g], vr[to, g] = kr[src, g], vr[src, g]
                hole = torch.tensor(hole, dtype=torch.long, device=dev)
                mover = torch.tensor(mover, dtype=torch.long, device=dev)
                mass[b, g, hole], pos[b, g, hole] = mass[b, g, mover], pos[b, g, mover]
            mass[b, g, lens[b]:], pos[b, g, lens[b]:] = 0, -1
    return {"mass": mass.double(), "positions": pos, "k_cache": kc, "v_cache": vc,
            "cache_lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
