"""The operators of steps whose requests share cached tokens, and what they are measured on.

`attention`: one token per sequence over the paged cache, for batches in which groups of sequences begin with the same cached
tokens (samples of one prompt, requests under one system prompt): the keys of a group's prefix are read once for all its
sequences.  `tables`: the block tables, slot maps and positions of a step, built on the device from the requests' lengths and
the pages handed out in this step.

Head layouts are those of this repository's model sizes.  Pages of 16 tokens (the engine's default) and others lie in random
order; slots behind a sequence's last token hold what an earlier request left.  The plain forms compute in 32 bits.
"""
import math
import random
import zlib

import torch

own = False
DEVICE = "cuda:0"
F64 = torch.float64
HEADS = {"8b": (32, 8, 128), "7b": (28, 4, 128), "0.5b": (14, 2, 64), "2k": (16, 4, 128)}       # query heads, key/value heads, head size


# -------------------------------------------------------------------------------------------------------------- cases
def _attention(name, heads, groups, members, single, prefix_lo, prefix_hi, own_lo, own_hi, dtype="bfloat16", page=16, extras=False):
    return {"name": name, "kind": "attention", "heads": heads, "groups": groups, "members": members, "single": single,
            "prefix_lo": prefix_lo, "prefix_hi": prefix_hi, "own_lo": own_lo, "own_hi": own_hi, "dtype": dtype, "page": page,
            "extras": extras}


def _tables(name, seqs, portions, longest_portion, ctx_lo, ctx_hi, groups, page=16, rows=0):
    return {"name": name, "kind": "tables", "seqs": seqs, "portions": portions, "longest_portion": longest_portion, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "groups": groups, "page": page, "rows": rows or seqs + seqs // 4 + 1}


def listed():
    return [
        # two samples of a short question on a small model: launches and latency
        _attention("two samples, short", "0.5b", 1, 2, 0, 33, 33, 1, 9),
        # eight samples of an article, some way into their answers
        _attention("eight samples", "7b", 1, 8, 0, 1003, 1003, 30, 200),
        # a full batch under one system prompt, with chats of very different lengths behind it
        _attention("batch under one prompt", "8b", 1, 64, 0, 2048, 2048, 1, 700),
        # four prompts' samples beside requests that share nothing
        _attention("four prompts and others", "8b", 4, 12, 9, 400, 3500, 5, 400),
        # a document that 256 short questions are asked about: the prefix's arithmetic is what counts
        _attention("questions on a document", "8b", 1, 256, 0, 16384, 16384, 1, 160),
        # a long context for a few samples: the prefix's bytes are what counts
        _attention("long context, four samples", "8b", 1, 4, 0, 32768, 32768, 1, 1000),
        # capped scores, a sink and a gate per head
        _attention("capped scores, sink, gate", "2k", 2, 16, 1, 500, 1500, 1, 250, extras=True),
        # the 32-bit path, in which correctness is judged
        _attention("float32", "7b", 1, 16, 1, 777, 777, 1, 64, "float32"),
        # the tables of a decode step of a small batch
        _tables("tables, eight decode", 8, 0, 1, 40, 2048, 1),
        # of 64 requests with long contexts
        _tables("tables, 64 long contexts", 64, 0, 1, 500, 32767, 1),
        # of prompt portions beside decoded tokens, on a model with windows beside full attention
        _tables("tables, portions", 40, 16, 2048, 30, 8000, 2),
        # of a server's largest step
        _tables("tables, 1,024 requests", 1024, 24, 1500, 100, 32767, 2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.3:
        seqs = _log(rng, 1, 1000)
        ctx_hi = _log(rng, 16, 32000)
        portions = rng.choice((0, _log(rng, 1, 24)))
        c = _tables("", seqs, min(portions, seqs), _log(rng, 2, 1500), _log(rng, 1, ctx_hi), ctx_hi, rng.randint(1, 2), rng.choice((8, 16, 16, 32, 64)))
        return {k: v for k, v in c.items() if k != "name"}
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    groups = rng.choice((1, 1, 2, 5))
    members = _log(rng, 2, 32 if dtype == "float32" else 128 // groups)
    prefix_hi = _log(rng, 16, 2000 if dtype == "float32" else 24000 // groups)
    own_hi = _log(rng, 1, 100 if dtype == "float32" else 800)
    c = _attention("", rng.choice(tuple(HEADS)), groups, members, rng.randint(0, 5), _log(rng, max(1, prefix_hi // 4), prefix_hi), prefix_hi,
                   _log(rng, 1, own_hi), own_hi, dtype, rng.choice((8, 16, 16, 32, 64)), rng.random() < 0.3)
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(case):
    """The lengths of a case: they belong to it, and do not depend on a seed."""
    rng = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    if case["kind"] == "attention":
        prefix = [case["prefix_hi"]] + [_log(rng, case["prefix_lo"], case["prefix_hi"]) for _ in range(case["groups"] - 1)]
        seqs = [g for g in range(case["groups"]) for _ in range(case["members"])] + [-1] * case["single"]
        rng.shuffle(seqs)                                                     # arrival order: groups lie mixed in the batch
        own_lens = [_log(rng, case["own_lo"], case["own_hi"]) for _ in seqs]
        return prefix, seqs, own_lens
    q = [1] * (case["seqs"] - case["portions"]) + [rng.randint(2, case["longest_portion"]) for _ in range(case["portions"])]
    starts = [_log(rng, case["ctx_lo"], case["ctx_hi"]) - 1 for _ in q]
    fresh = [i for i, n in enumerate(q) if n > 1 and rng.random() < 0.5]      # first portions start at 0
    for i in fresh:
        starts[i] = 0
    return starts, q


def _spans(case):
    """(window, chunk) per group of layers, 0: none."""
    return [(0, 0), (1024, 0)][:case["groups"]]


def _live(start, window, chunk, page):
    first = max(0, start - window + 1) if window else 0
    return max(first, start // chunk * chunk if chunk else 0) // page


# -------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    page = case["page"]
    blocks = lambda n: (n + page - 1) // page  # noqa: E731
    if case["kind"] == "tables":
        starts, q = _lengths(case)
        G, B, R = case["groups"], len(q), case["rows"]
        ends = [s + n for s, n in zip(starts, q)]
        rows = torch.randperm(R, generator=host)[:B]
        pads = B // 8                                    # a captured batch is filled up with rows that stand for no request
        if pads:
            rows[B - pads:] = -1
        used = [blocks(e) if int(r) >= 0 else 0 for e, r in zip(ends, rows)]
        held = [min(u, blocks(s)) for u, s in zip(used, starts)]
        width = max(blocks(max(ends)), 1)
        pages = sum(u for u in used) + R
        perm = torch.stack([torch.randperm(pages, generator=host) for _ in range(G)]).to(torch.int32)
        new = torch.cat([perm[g, :sum(used) - sum(held)] for g in range(G)]) if sum(used) > sum(held) else torch.zeros(0, dtype=torch.int32)
        table = torch.randint(0, pages, (G, R, width + 5), generator=host, dtype=torch.int32)    # the longest request may be elsewhere
        return {"kind": "tables", "page_table": table.to(DEVICE), "rows": rows.to(torch.int32).to(DEVICE), "held": i32([held] * G),
                "starts": i32(starts), "q_lens": i32(q), "new_pages": new.to(DEVICE), "spans": i32(_spans(case)), "num_tokens": sum(q),
                "max_blocks": width, "page": page}
    prefix, seqs, own_lens = _lengths(case)
    nh, nkv, hd = HEADS[case["heads"]]
    dtype = getattr(torch, case["dtype"])
    B = len(seqs)
    ctx = [(prefix[g] if g >= 0 else 0) + n for g, n in zip(seqs, own_lens)]
    mb = blocks(max(ctx))
    # a group's whole pages have several holders; the page in which a prefix ends is each sequence's own copy
    whole = [p // page for p in prefix]
    total = sum(whole) + sum(blocks(c) - (whole[g] if g >= 0 else 0) for c, g in zip(ctx, seqs)) + 3
    order = torch.randperm(total, generator=host).to(torch.int32)
    cache = torch.empty((total, 2, nkv, page, hd), dtype=dtype, device=DEVICE)
    for part in cache.split(max(1, (1 << 26) // (2 * nkv * page * hd))):
        part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE))
    table = torch.full((B, mb), -1, dtype=torch.int32)
    at, shared_pages = 0, []
    for w in whole:
        shared_pages.append(order[at:at + w])
        at += w
    first = {}
    for b, g in enumerate(seqs):
        w = whole[g] if g >= 0 else 0
        n = blocks(ctx[b]) - w
        if w:
            table[b, :w] = shared_pages[g]
        table[b, w:w + n] = order[at:at + n]
        at += n
        if g >= 0 and prefix[g] % page:
            if g in first:                               # the copy of the page in which the prefix ends
                cache[int(table[b, w]), :, :, :prefix[g] % page] = cache[int(table[first[g], w]), :, :, :prefix[g] % page]
            else:
                first[g] = b
    groups = [([b for b, x in enumerate(seqs) if x == g], prefix[g]) for g in range(case["groups"])]
    q = (torch.randn((B, nh * hd), generator=gen, device=DEVICE) * 2.5).to(dtype)
    s = {"kind": "attention", "q": q, "cache": cache, "tables": table.to(DEVICE), "ctx": i32(ctx), "max_ctx": max(ctx), "page": page,
         "max_own": max(own_lens), "heads": (nh, nkv, hd), "scale": hd ** -0.5,
         "softcap": 30.0 if case["extras"] else None,
         "sinks": torch.randn((nh,), generator=gen, device=DEVICE) if case["extras"] else None,
         "gate": torch.sigmoid(torch.randn((B, nh), generator=gen, device=DEVICE)) if case["extras"] else None}
    # every sequence belongs to a group for the plain form: one that shares nothing is a group of its own without a prefix
    every = groups + [([b], 0) for b, g in enumerate(seqs) if g < 0]
    widest = max(len(m) for m, _ in every)
    s["members"] = torch.tensor([m + [m[0]] * (widest - len(m)) for m, _ in every], device=DEVICE)
    place = [0] * B
    for g, (m, _) in enumerate(every):
        for i, b in enumerate(m):
            place[b] = g * widest + i
    s["place"] = torch.tensor(place, device=DEVICE)
    s["group_prefix"] = torch.tensor([p for _, p in every], device=DEVICE)
    s["prefix"] = torch.tensor([prefix[g] if g >= 0 else 0 for g in seqs], device=DEVICE)
    s["max_prefix"] = max(prefix)
    if own:
        from rvllm_b200.kernels import AttentionMeta, SharedPrefixes, get_library
        s["kernels"] = get_library(DEVICE)
        s["meta"] = AttentionMeta(s["tables"], torch.arange(B + 1, dtype=torch.int32, device=DEVICE), s["ctx"],
                                  torch.arange(B, dtype=torch.int32, device=DEVICE), None, B, 1, max(ctx), page, B)
        s["shared"] = SharedPrefixes(groups, B, nh, nkv, DEVICE)
    return s


# -------------------------------------------------------------------------------------------------------------- passes
def run(s):
    if s["kind"] == "tables":
        return _run_tables(s)
    nh, nkv, hd = s["heads"]
    if own:
        return s["kernels"].shared_prefix_attention(s["q"], s["cache"], s["meta"], s["shared"], nh, nkv, hd, s["scale"], softcap=s["softcap"],
                                                    sinks=s["sinks"], gate=s["gate"], max_own=s["max_own"])
    return _plain_attention(s)


def _capped(scores, cap):
    return scores if cap is None else cap * torch.tanh(scores / cap)


def _keys(s, tables, positions, plane):
    """[rows, positions, kv heads, head size] in 32 bits; positions [rows, n]."""
    pages = tables.gather(1, torch.div(positions, s["page"], rounding_mode="floor")).clamp(min=0)
    return s["cache"][:, plane].transpose(1, 2)[pages.long(), positions % s["page"]].float()


def _plain_attention(s):
    """Scores of the prefixes by group and of what lies behind them by sequence, one softmax over both."""
    nh, nkv, hd = s["heads"]
    B, per = s["q"].shape[0], nh // nkv
    q = s["q"].float().view(B, nkv, per, hd)
    groups, members = s["members"].shape
    # the prefixes: [groups, kv heads, members x heads of the group, keys]
    at = torch.arange(max(s["max_prefix"], 1), device=q.device).expand(groups, -1)
    seen = at < s["group_prefix"][:, None]
    first = s["tables"][s["members"][:, 0]]
    at = torch.minimum(at, (s["group_prefix"][:, None] - 1).clamp(min=0))
    rows = q[s["members"]].permute(0, 2, 1, 3, 4).reshape(groups, nkv, members * per, hd)
    k = _keys(s, first, at, 0).permute(0, 2, 3, 1)
    a = _capped(torch.matmul(rows, k) * s["scale"], s["softcap"]).masked_fill(~seen[:, None, None], float("-inf"))
    a_top = a.amax(-1)
    # what each sequence has behind its prefix
    own_at = s["prefix"][:, None] + torch.arange(s["max_own"], device=q.device)
    own_seen = own_at < s["ctx"][:, None]
    own_at = torch.minimum(own_at, s["ctx"][:, None].long() - 1)
    k = _keys(s, s["tables"], own_at, 0).permute(0, 2, 3, 1)
    c = _capped(torch.matmul(q, k) * s["scale"], s["softcap"]).masked_fill(~own_seen[:, None, None], float("-inf"))
    c_top = c.amax(-1)
    # the sequences' own order for the prefixes' part
    back = lambda x: x.unflatten(2, (members, per)).transpose(1, 2).flatten(0, 1)[s["place"]]  # noqa: E731
    top = torch.maximum(c_top, back(a_top))
    if s["sinks"] is not None:
        top = torch.maximum(top, s["sinks"].view(1, nkv, per))
    by_group = top.new_zeros((groups * members, nkv, per)).index_copy(0, s["place"], top).view(groups, members, nkv, per)
    a = torch.exp(a - by_group.transpose(1, 2).flatten(2, 3)[..., None])
    c = torch.exp(c - top[..., None])
    total = c.sum(-1) + back(a.sum(-1))
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].view(1, nkv, per) - top)
    out = torch.matmul(c, _keys(s, s["tables"], own_at, 1).transpose(1, 2)) + back(torch.matmul(a, _keys(s, first, at, 1).transpose(1, 2)))
    out = out / total[..., None]
    if s["gate"] is not None:
        out = out * s["gate"].view(B, nkv, per, 1)
    return out.to(s["q"].dtype).view(B, nh * hd)


def _run_tables(s):
    if own:
        from rvllm_b200.kernels import get_library
        t = get_library(DEVICE).step_tables(s["page_table"], s["rows"], s["held"], s["starts"], s["q_lens"], s["new_pages"], s["spans"],
                                            s["num_tokens"], s["max_blocks"], s["page"])
        return {"page_table": s["page_table"], "block_tables": t.block_tables, "slot_mapping": t.slot_mapping, "positions": t.positions,
                "token_seq": t.token_seq, "cu_seqlens": t.cu_seqlens, "ctx_lens": t.ctx_lens}
    return _plain_tables(s)


def _plain_tables(s):
    table, page, T, MB = s["page_table"], s["page"], s["num_tokens"], s["max_blocks"]
    G, R, _ = table.shape
    B = s["rows"].shape[0]
    real = s["rows"] >= 0
    start, q, row = s["starts"].long(), s["q_lens"].long(), s["rows"].long().clamp(min=0)
    end = start + q
    used = torch.where(real, torch.div(end + page - 1, page, rounding_mode="floor"), 0)
    held = s["held"].long()
    count = (used - held).clamp(min=0) * real                                              # [G, B]
    offset = (count.flatten().cumsum(0) - count.flatten()).view(G, B)
    j = torch.arange(MB, device=table.device)
    is_new = (j >= held[..., None]) & (j < used[:, None]) & real[:, None]
    pages = torch.cat([s["new_pages"], s["new_pages"].new_zeros(1)])
    fresh = pages[torch.where(is_new, offset[..., None] + j - held[..., None], pages.shape[0] - 1)]
    entries = torch.where(is_new, fresh, table[:, row, :MB])
    # the table itself, row by row: which sequence of the step a row belongs to
    of_row = torch.full((R + 1,), -1, device=table.device).scatter_(0, torch.where(real, row, R), torch.arange(B, device=table.device))[:R]
    mine = (of_row >= 0)[:, None] & is_new[:, of_row.clamp(min=0)]
    table[:, :, :MB] = torch.where(mine, fresh[:, of_row.clamp(min=0)], table[:, :, :MB])
    window, chunk = s["spans"][:, 0, None].long(), s["spans"][:, 1, None].long()
    first = torch.where(window > 0, (start - window + 1).clamp(min=0), 0)
    first = torch.maximum(first, torch.where(chunk > 0, torch.div(start, chunk.clamp(min=1), rounding_mode="floor") * chunk, 0))
    live = torch.div(first, page, rounding_mode="floor")
    tables = torch.where((j < used[:, None]) & (j >= live[..., None]) & real[:, None], entries, -1).int()
    cu = torch.cat([q.new_zeros(1), q.cumsum(0)])
    t = torch.arange(T, device=table.device)
    seq = torch.searchsorted(cu[1:], t, right=True)
    pos = torch.where(real[seq], start[seq] + t - cu[seq], 0)
    at = entries[:, seq, torch.div(pos, page, rounding_mode="floor")].long() * page + pos % page
    return {"page_table": table, "block_tables": tables, "slot_mapping": torch.where(real[seq], at, -1).int(), "positions": pos.int(),
            "token_seq": seq.int(), "cu_seqlens": cu.int(), "ctx_lens": torch.where(real, end, 0).int()}


# -------------------------------------------------------------------------------------------------------------- floors
def work(case):
    if case["kind"] == "tables":
        starts, q = _lengths(case)
        page, G, B, T = case["page"], case["groups"], len(q), sum(q)
        pads = B // 8
        width = max((s + n + page - 1) // page for s, n in zip(starts, q))
        read = new = 0
        for window, chunk in _spans(case):
            for s, n in list(zip(starts, q))[:B - pads]:
                used, held = (s + n + page - 1) // page, (s + page - 1) // page
                read += used - min(used, _live(s, window, chunk, page))
                new += used - held
        return {"bytes": 4 * (read + new + G * B * (width + 1) + G * T + 2 * T + 5 * B + 1), "flops": G * (B * width + T)}
    prefix, seqs, own_lens = _lengths(case)
    nh, nkv, hd = HEADS[case["heads"]]
    el = 2 if case["dtype"] == "bfloat16" else 4
    B = len(seqs)
    keys = sum(prefix) + sum(own_lens)
    every = sum((prefix[g] if g >= 0 else 0) + n for g, n in zip(seqs, own_lens))
    extras = 4 * (nh + B * nh) if case["extras"] else 0
    tables = 4 * ((keys + case["page"] - 1) // case["page"] + B)
    return {"bytes": el * (2 * B * nh * hd + 2 * nkv * hd * keys) + extras + tables, "flops": 4 * nh * hd * every}


# ------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """Sequence by sequence, over all its keys, without any notion of a prefix."""
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    nh, nkv, hd = s["heads"]
    out = torch.empty((s["q"].shape[0], nh, hd), dtype=F64, device=DEVICE)
    for b, n in enumerate(s["ctx"].tolist()):
        kv = s["cache"][s["tables"][b, :(n + s["page"] - 1) // s["page"]].long()].transpose(1, 3)       # [pages, slot, kv head, plane, size]
        kv = kv.reshape(-1, nkv, 2, hd)[:n].to(F64)
        for g in range(nkv):
            heads = slice(g * (nh // nkv), (g + 1) * (nh // nkv))
            x = s["q"][b].view(nh, hd)[heads].to(F64) @ kv[:, g, 0].T * s["scale"]
            if s["softcap"] is not None:
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][heads, None].to(F64)], 1)
            p = torch.softmax(x, 1)[:, :n]
            out[b, heads] = p @ kv[:, g, 1]
            if s["gate"] is not None:
                out[b, heads] *= s["gate"][b, heads, None].to(F64)
    return out.view(-1, nh * hd)
