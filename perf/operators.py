"""Steps that carry several continuations of a request, operator by operator, as cases that can be timed and compared.

``tree_attention``  attention of a tree of drafted tokens per request over the paged cache, one layer
``tree_commit``     which drafted tokens hold, and their keys and values moved up in the cache, all layers
``beam_select``     the best continuations over a request's beams and the vocabulary
``copy_pages``      the first rows of cache pages copied to other pages, all layers: a beam that is carried on twice
``copy_slots``      per-request states copied from slot to slot, all layers: the same for models with states

Head counts, layers and vocabularies are those of ``bench.py`` and ``return_b200.benchmark`` (the 0.6B, 8B and 32B shapes, the
Pisatar design sizes).  Lengths within a case are worked out from the case alone (``_lengths``), contents come from the seed.
"""
import math
import types

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
PISATAR_HEAD = 128 * 128            # float32 values of one head's matrix state


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one user of a small model, eight drafted tokens: latency is all that counts
        {"name": "tree_one_short", "op": "tree_attention", "dtype": "bfloat16", "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16,
         "requests": 1, "ctx": 500, "spread": 0, "nodes": 8, "window": 0, "softcap": 0.0, "sink": False},
        # the decode headline's batch with sixteen drafted tokens a request
        {"name": "tree_8x2040", "op": "tree_attention", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "requests": 8, "ctx": 2040, "spread": 0, "nodes": 16, "window": 0, "softcap": 0.0, "sink": False},
        # a full batch of the 32B heads, ragged contexts up to 8,000, trees of up to 64: the largest
        {"name": "tree_32_ragged", "op": "tree_attention", "dtype": "bfloat16", "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 16,
         "requests": 32, "ctx": 8000, "spread": 75, "nodes": 64, "window": 0, "softcap": 0.0, "sink": False},
        # the true float32 path, a sliding window, odd sizes
        {"name": "tree_float32_window", "op": "tree_attention", "dtype": "float32", "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 8,
         "requests": 3, "ctx": 1901, "spread": 60, "nodes": 13, "window": 1000, "softcap": 0.0, "sink": False},
        # after the step of one user: 28 layers of the 0.6B model, three tokens hold
        {"name": "commit_one", "op": "tree_commit", "dtype": "bfloat16", "layers": 28, "kv_heads": 8, "head_dim": 128, "page": 16,
         "requests": 1, "ctx": 121, "spread": 0, "nodes": 8, "accept": 3},
        # after a full batch's step: 36 layers of the 8B model
        {"name": "commit_64", "op": "tree_commit", "dtype": "bfloat16", "layers": 36, "kv_heads": 8, "head_dim": 128, "page": 16,
         "requests": 64, "ctx": 200, "spread": 80, "nodes": 32, "accept": 6},
        # four beams of one request, the design sizes' vocabulary
        {"name": "beam_one_4", "op": "beam_select", "requests": 1, "beams": 4, "vocab": 32768, "keep": 8, "steps": 1 / 64, "dead": 0},
        # eight beams of sixteen requests, the 8B model's vocabulary
        {"name": "beam_16x8", "op": "beam_select", "requests": 16, "beams": 8, "vocab": 151936, "keep": 16, "steps": 0.0, "dead": 0},
        # beams of one request part ways: partly filled last pages of 28 layers
        {"name": "pages_4", "op": "copy_pages", "dtype": "bfloat16", "layers": 28, "kv_heads": 8, "head_dim": 128, "page": 16, "copies": 4},
        # sixteen requests of eight beams, 36 layers
        {"name": "pages_72", "op": "copy_pages", "dtype": "bfloat16", "layers": 36, "kv_heads": 8, "head_dim": 128, "page": 16, "copies": 72},
        # the states of beams of one request of the smaller Pisatar design size
        {"name": "slots_3", "op": "copy_slots", "layers": 8, "heads": 8, "more": 1536, "slots": 9, "copies": 3},
        # and of a full batch of the middle one
        {"name": "slots_32", "op": "copy_slots", "layers": 8, "heads": 16, "more": 0, "slots": 65, "copies": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tree_attention", "tree_attention", "tree_attention", "tree_commit", "beam_select", "beam_select", "copy_pages", "copy_slots"))
    if op == "tree_attention":
        heads, kv_heads = rng.choice(((16, 8), (32, 8), (64, 8), (16, 4), (5, 1), (8, 8)))
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        requests, nodes = _log(rng, 1, 32), _log(rng, 1, 80)
        most = min(8000, 160000 // requests) if dtype == "bfloat16" else min(2500, 200000 // (requests * nodes) + 20)
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice((128, 128, 128, 64, 48, 256)),
                "page": rng.choice((16, 16, 64, 8)), "requests": requests, "ctx": rng.choice((0, _log(rng, 1, most), _log(rng, 20, most), most)),
                "spread": rng.choice((0, 30, 90)), "nodes": nodes, "window": rng.choice((0, 0, 0, _log(rng, 2, 2000))),
                "softcap": rng.choice((0.0, 0.0, 0.0, 30.0)), "sink": rng.choice((False, False, True))}
    if op == "tree_commit":
        layers = rng.choice((28, 36, 8))
        return {"op": op, "dtype": rng.choice(("bfloat16", "bfloat16", "float32")), "layers": layers, "kv_heads": rng.choice((8, 4, 1)),
                "head_dim": rng.choice((128, 128, 64, 48)), "page": rng.choice((16, 16, 64, 8)), "requests": _log(rng, 1, 40),
                "ctx": rng.randint(0, 150), "spread": rng.choice((0, 50, 90)), "nodes": _log(rng, 1, 100), "accept": rng.randint(1, 9)}
    if op == "beam_select":
        requests, beams = _log(rng, 1, 16), rng.choice((1, 2, 3, 4, 5, 8))
        return {"op": op, "requests": requests, "beams": beams, "vocab": rng.choice((151936, 32768, _log(rng, 300, 150000))),
                "keep": rng.choice((1, beams, 2 * beams, 2 * beams, 2 * beams + 5)), "steps": rng.choice((0.0, 0.0, 1 / 64, 1 / 4)),
                "dead": rng.choice((0, 0, beams - 1))}
    if op == "copy_pages":
        return {"op": op, "dtype": rng.choice(("bfloat16", "bfloat16", "float32")), "layers": rng.choice((28, 36, 8)),
                "kv_heads": rng.choice((8, 4, 1)), "head_dim": rng.choice((128, 128, 64, 48)), "page": rng.choice((16, 16, 64, 8)),
                "copies": _log(rng, 1, 30)}
    slots = _log(rng, 2, 60)
    return {"op": op, "layers": rng.choice((8, 4, 3)), "heads": rng.choice((8, 16, 4)), "more": rng.choice((0, 1536, 1, 6144)),
            "slots": slots, "copies": rng.randint(1, max(1, slots // 2))}


def _lengths(case):
    """Cached tokens and drafted nodes of each request: contexts fall evenly by ``spread`` percent, trees by up to half."""
    n, ctx, nodes = case["requests"], case["ctx"], case["nodes"]
    cached = [ctx - ctx * case["spread"] * i // (100 * max(1, n - 1)) for i in range(n)]
    return cached, [nodes - (5 * i) % (nodes // 2 + 1) for i in range(n)]


def _size(case):
    return 4 if case["dtype"] == "float32" else 2


def work(case):
    op = case["op"]
    if op == "tree_attention":
        cached, nodes = _lengths(case)
        D, Hq, Hkv = case["head_dim"], case["heads"], case["kv_heads"]
        w = case["window"] or 1 << 30
        # the keys that a request's nodes see lie in the window of its root; a node sees at least itself
        keys = sum(min(c, w - 1) + n for c, n in zip(cached, nodes))
        pairs = sum(n * (min(c, max(0, w - n)) + 1) for c, n in zip(cached, nodes))
        return {"bytes": _size(case) * (2 * Hkv * D * keys + 2 * Hq * D * sum(nodes)), "flops": 4.0 * D * Hq * pairs}
    if op == "tree_commit":
        cached, nodes = _lengths(case)
        moved = sum(max(0, _accepted(n, case["accept"])[0] - _accepted(n, case["accept"])[1]) for n in nodes)
        row = case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * _size(case)
        return {"bytes": 2 * moved * row + 12 * sum(nodes) + 8 * case["requests"] * max(nodes), "flops": 0}
    if op == "beam_select":
        n = case["requests"] * case["beams"] * case["vocab"]
        return {"bytes": 4 * n + 12 * case["requests"] * case["keep"], "flops": 4.0 * n}
    if op == "copy_pages":
        rows = sum(_rows(case))
        return {"bytes": 2 * rows * case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * _size(case), "flops": 0}
    return {"bytes": 2 * 4 * case["copies"] * case["layers"] * (case["heads"] * PISATAR_HEAD + case["more"]), "flops": 0}


def _accepted(nodes, accept):
    """(nodes of the accepted path, how many of them lie in their place already).  The path begins at the root; what does not lie
    in place comes from behind the path's own slots, as where a branch that was not drafted first holds: a pass can then be
    repeated on the same cache."""
    count = max(1, min(accept, (nodes + 1) // 2))
    return count, (1 if count < 4 else 2)


def _rows(case):
    """Filled rows of the pages that are copied: 1 to a whole page."""
    return [1 + (7 * i + 4) % case["page"] for i in range(case["copies"])]


# ------------------------------------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


def _ints(values):
    return torch.tensor(np.asarray(values, dtype=np.int32), device=DEVICE)


def _pages(rs, total, page, spare=3):
    """A block table [n, blocks] for requests of ``total`` tokens, their pages strewn over a pool; -1 behind a request's last."""
    blocks = [(t + page - 1) // page for t in total]
    order = rs.permutation(sum(blocks) + spare).astype(np.int32)
    table, at = np.full((len(total), max(1, max(blocks))), -1, np.int32), 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += b
    return table, len(order)


def _batch(cached, nodes, parents, tokens):
    """The tables of a step of drafted trees, as the engine keeps them for its layers."""
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    host = types.SimpleNamespace(cu_q=cu, seg_pos0=np.asarray(cached, np.int32))
    return types.SimpleNamespace(host=host, scratch={}, num_tokens=int(cu[-1]), num_segments=len(nodes), cu_q=_ints(cu),
                                 seg_pos0=_ints(cached), tree_parent=_ints(parents), tokens=_ints(tokens))


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("tree_attention", "tree_commit"):
        cached, nodes = _lengths(case)
        table, n_pages = _pages(rs, [c + n for c, n in zip(cached, nodes)], case["page"])
        s["block_table"] = _ints(table)
        parents, tokens, sampled = [], [], []
        for n in nodes:
            parent = [-1] + [int(rs.randint(max(0, i - 6), i)) for i in range(1, n)]
            draft, target = rs.randint(0, 30000, n), rs.randint(30000, 60000, n)
            if op == "tree_commit":
                count, still = _accepted(n, case["accept"])
                path = list(range(still)) + sorted((count + rs.permutation(n - count)[:count - still]).tolist())
                for x, y in zip(path, path[1:]):
                    parent[y] = x
                    target[x] = draft[y]
            parents += parent
            tokens += draft.tolist()
            sampled += target.tolist()
        s["batch"] = _batch(cached, nodes, parents, tokens)
        s["sampled"] = _ints(sampled)
    if op == "tree_attention":
        D, Hq, Hkv, dt = case["head_dim"], case["heads"], case["kv_heads"], _dtype(case)
        # rows of projections: queries, then the step's keys and values, which are in the cache already
        s["qkv"] = torch.randn((sum(nodes), (Hq + 2 * Hkv) * D), generator=g, device=DEVICE).to(dt)
        s["k"], s["v"] = (torch.randn((n_pages, Hkv, case["page"], D), generator=g, device=DEVICE).to(dt) for _ in range(2))
        s["sink"] = torch.randn((Hq,), generator=g, device=DEVICE) if case["sink"] else None
    elif op in ("tree_commit", "copy_pages"):
        if op == "copy_pages":
            n_pages = 2 * case["copies"] + 3
            order = rs.permutation(n_pages)
            s["src"], s["dst"], s["rows"] = _ints(order[:case["copies"]]), _ints(order[case["copies"]:2 * case["copies"]]), _ints(_rows(case))
        shape = (case["layers"], 2, n_pages, case["kv_heads"], case["page"], case["head_dim"])
        s["pool"] = torch.empty(shape, dtype=_dtype(case), device=DEVICE).normal_(generator=g)
    elif op == "beam_select":
        B, V = case["requests"] * case["beams"], case["vocab"]
        x = torch.randn((B, V), generator=g, device=DEVICE) * 2.5
        if case["steps"]:                   # logits on a grid: many equal ones
            x = torch.round(x / case["steps"]) * case["steps"]
        s["logits"] = x
        s["scores"] = -20.0 * torch.rand((B,), generator=g, device=DEVICE)
        if case["dead"]:                    # a request's first step: one beam counts
            s["scores"].view(case["requests"], -1)[:, -case["dead"]:] = float("-inf")
    else:
        n = case["heads"] * PISATAR_HEAD + case["more"]
        s["states"] = [torch.randn((case["slots"], n), generator=g, device=DEVICE) for _ in range(case["layers"])]
        order = rs.permutation(case["slots"])
        s["dst"] = _ints(order[:case["copies"]])
        s["src"] = _ints(rs.choice(order[case["copies"]:], case["copies"]))       # one that lives on may have several copies
        if own:
            from return_b200.ext import ops
            s["table"] = ops.slot_table(s["states"])
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from return_b200.ext import ops
    case = s["case"]
    op = case["op"]
    if op == "tree_attention":
        Hq, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
        out = torch.empty((s["qkv"].shape[0], Hq * D), dtype=s["qkv"].dtype, device=DEVICE)
        ops.tree_attention(s["qkv"], s["k"], s["v"], s["batch"], s["block_table"], case["page"], out, Hq, Hkv, D, D ** -0.5,
                           window=case["window"] or None, sink=s["sink"], softcap=case["softcap"] or None)
        return out
    if op == "tree_commit":
        n, width = case["requests"], max(_lengths(case)[1])
        path, emitted = (torch.empty((n, width), dtype=torch.int32, device=DEVICE) for _ in range(2))
        count = torch.empty((n,), dtype=torch.int32, device=DEVICE)
        ops.tree_commit(s["sampled"], s["batch"], [(s["pool"], s["block_table"])], path, count, emitted)
        return path, count, emitted, s["pool"]
    if op == "beam_select":
        n, keep = case["requests"], case["keep"]
        scores = torch.empty((n, keep), dtype=torch.float32, device=DEVICE)
        beams, tokens = (torch.empty((n, keep), dtype=torch.int32, device=DEVICE) for _ in range(2))
        ops.beam_select(s["logits"], s["scores"], case["beams"], scores, beams, tokens)
        return scores, beams, tokens
    if op == "copy_pages":
        ops.copy_pages(s["pool"], s["src"], s["dst"], s["rows"])
        return s["pool"]
    ops.copy_slots(s["table"], s["src"], s["dst"])
    return s["states"]


def _run_plain(s):
    return {"tree_attention": _plain_attention, "tree_commit": _plain_commit, "beam_select": _plain_beams, "copy_pages": _plain_pages,
            "copy_slots": _plain_slots}[s["case"]["op"]](s)


def _padded(batch):
    """Rows of the packed step as [requests, longest tree], and which of them exist."""
    n = (batch.cu_q[1:] - batch.cu_q[:-1]).long()
    i = torch.arange(int(np.diff(batch.host.cu_q).max()), device=DEVICE)
    there = i[None] < n[:, None]
    return torch.where(there, batch.cu_q[:-1].long()[:, None] + i, 0), there


def _ancestors(parent):
    """[requests, M, M]: node j is i or an ancestor of i, from the parents [requests, M] (-1: none)."""
    M = parent.shape[1]
    reach = torch.eye(M, device=DEVICE) + (parent[:, :, None] == torch.arange(M, device=DEVICE)).float()
    for _ in range(max(1, M - 1).bit_length()):
        reach = (reach @ reach > 0).float()
    return reach > 0


def _places(table, slots, page):
    """Page and row in it of each slot [requests, m]."""
    return table.gather(1, torch.clamp(slots // page, max=table.shape[1] - 1)), slots % page


def _plain_attention(s):
    case, b = s["case"], s["batch"]
    Hq, Hkv, D, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    rows, there = _padded(b)
    parent = torch.where(there, b.tree_parent[rows], -1)
    seen = _ancestors(parent)
    depth = seen.sum(-1) - 1
    n, M = rows.shape
    c = b.seg_pos0.long()
    L = int((b.host.seg_pos0 + np.diff(b.host.cu_q)).max())
    j = torch.arange(L, device=DEVICE)[None]
    node = j - c[:, None]                                       # a slot's node; below zero: a cached key
    is_node = (node >= 0) & (node < there.sum(1)[:, None])
    at = torch.clamp(node, 0, M - 1)
    visible = torch.where((node < 0)[:, None], True, is_node[:, None] & seen.gather(2, at[:, None].expand(n, M, L)))
    if w:
        place = torch.where(node < 0, j, c[:, None] + depth.gather(1, at))
        visible = visible & (place[:, None] > (c[:, None] + depth)[:, :, None] - w)
    page, row = _places(s["block_table"].long(), j.expand(n, L), case["page"])
    page = torch.clamp(page, min=0)
    k, v = s["k"][page, :, row].float(), s["v"][page, :, row].float()         # [n, L, Hkv, D]
    v = torch.where(visible.any(1)[:, :, None, None], v, 0.0)
    q = s["qkv"][rows][:, :, :Hq * D].float().reshape(n, M, Hkv, Hq // Hkv, D)
    x = torch.einsum("nmhgd,nlhd->nhgml", q, k) * D ** -0.5
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x = x.masked_fill(~visible[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].reshape(1, Hkv, Hq // Hkv, 1, 1) - top)
    o = torch.einsum("nhgml,nlhd->nmhgd", p / total, v).reshape(n, M, Hq * D)
    return o[there].to(s["qkv"].dtype)


def _plain_commit(s):
    case, b, pool = s["case"], s["batch"], s["pool"]
    rows, there = _padded(b)
    n, M = rows.shape
    parent = torch.where(there, b.tree_parent[rows].long(), -1)
    token, sampled = b.tokens[rows], s["sampled"][rows]
    i = torch.arange(M, device=DEVICE)
    same = (parent[:, :, None] == parent[:, None]) & (token[:, :, None] == token[:, None]) & (i[None, :] < i[:, None])
    holds = ((parent < 0) | (token == sampled.gather(1, torch.clamp(parent, min=0)))) & ~same.any(-1)
    taken = ((_ancestors(parent) & ~holds[:, None]).sum(-1) == 0) & there
    count = taken.sum(1)
    path = torch.sort(torch.where(taken, i, M), dim=1).values          # a parent's index is below its children's
    ok = i[None] < count[:, None]
    src = torch.where(ok, path, 0)
    emitted = torch.where(ok, sampled.gather(1, src), -1)
    c, table = b.seg_pos0.long()[:, None], s["block_table"].long()
    (sp, sr), (dp, dr) = _places(table, c + src, case["page"]), _places(table, c + i[None], case["page"])
    pool[:, :, dp[ok], :, dr[ok]] = pool[:, :, sp[ok], :, sr[ok]]
    return torch.where(ok, path, -1).int(), count.int(), emitted.int(), pool


def _plain_beams(s):
    case = s["case"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - top
    total = s["scores"].double()[:, None] + (x - torch.log(torch.exp(x).sum(-1, keepdim=True)))
    total = torch.where(torch.isnan(total), float("-inf"), total).view(case["requests"], -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :case["keep"]], at[:, :case["keep"]]
    return best.float(), (at // case["vocab"]).int(), (at % case["vocab"]).int()


def _plain_pages(s):
    pool, page = s["pool"], s["case"]["page"]
    move, row = (torch.arange(page, device=DEVICE)[None] < s["rows"][:, None]).nonzero(as_tuple=True)
    pool[:, :, s["dst"].long()[move], :, row] = pool[:, :, s["src"].long()[move], :, row]
    return pool


def _plain_slots(s):
    src, dst = s["src"].long(), s["dst"].long()
    for t in s["states"]:
        t[dst] = t[src]
    return s["states"]


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    op = case["op"]
    if op in ("copy_pages", "copy_slots", "tree_commit"):
        return None                         # whole numbers, and rows that are moved as they are
    s = prepare(case, seed)
    if op == "beam_select":
        # row by row; the candidates of a request are merged from its rows' best
        V, keep, B, scores = case["vocab"], case["keep"], case["beams"], []
        for r in range(case["requests"]):
            merged = []
            for k in range(B):
                x = s["logits"][r * B + k].double()
                log_p = x - torch.logsumexp(x, 0) + s["scores"][r * B + k].double()
                merged.append(torch.topk(log_p, min(keep, V)).values)
            scores.append(torch.topk(torch.cat(merged), keep).values)
        return torch.stack(scores), None, None
    Hq, Hkv, D, P, w = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["window"]
    cached, nodes = _lengths(case)
    parent, table = s["batch"].tree_parent.tolist(), s["block_table"].tolist()
    out, at = [], 0
    for i, (c, n) in enumerate(zip(cached, nodes)):
        total = c + n
        pages = table[i][:(total + P - 1) // P]
        k, v = (torch.cat([s[name][p] for p in pages], dim=1)[:, :total].double() for name in ("k", "v"))     # [Hkv, total, D]
        seen, depth = np.zeros((n, total), bool), [0] * n
        for x in range(n):
            line = [x]
            while parent[at + line[-1]] >= 0:
                line.append(parent[at + line[-1]])
            depth[x] = len(line) - 1
            seen[x, :c] = True
            if w:
                seen[x, :max(0, c + depth[x] - w + 1)] = False
                line = line[:w]
            seen[x, [c + y for y in line]] = True
        q = s["qkv"][at:at + n, :Hq * D].double().view(n, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
        x = torch.bmm(q, k.transpose(1, 2)) * D ** -0.5
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        hidden = torch.from_numpy(~seen).to(DEVICE).repeat(Hq // Hkv, 1)
        x = torch.where(hidden, -math.inf, x)
        if s["sink"] is not None:           # a key without a value
            z = s["sink"].double().view(Hkv, Hq // Hkv, 1).expand(-1, -1, n).reshape(Hkv, -1, 1)
            p = torch.softmax(torch.cat([x, z], -1), -1)[..., :-1]
        else:
            p = torch.softmax(x, -1)
        out.append(torch.bmm(p, v).view(Hkv, Hq // Hkv, n, D).permute(2, 0, 1, 3).reshape(n, Hq * D))
        at += n
    return torch.cat(out)
