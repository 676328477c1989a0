"""Serving several chats from one paged KV cache, with drafted tokens: the
operators of one such step as cases to be timed.

A step of a server that drafts tokens and verifies them runs, in this order:

  * ``tables``  block tables, positions and cache slots from request lengths
    (``cw_block_tables``);
  * ``rope_kv`` q and k of the new rows rotated, k and v written to their
    slots (``cw_rope_kv_rows``); ``rope`` is the rotation alone
    (``cw_rope_rows``);
  * ``tree``    attention of every drafted token over its request's cached
    positions and its own ancestors (``cw_attention_tree``);
  * ``accept``  the accepted path's K and V rows moved to the positions that
    follow the cached ones (``cw_kv_accept``).

Widths are those of the Qwen3-8B and Qwen3-0.6B configurations that the tests
and the benchmark run (heads, kv heads, head size); contexts of a batch are
spread evenly over their logarithm, as chats of different ages are.
Activations, keys and values are unit normal (keys after their norm are), the
queries twice that, so that a row's softmax prefers some keys.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

# heads, kv heads, head size
SHAPES = {"8b": (32, 8, 128), "0.6b": (16, 8, 128)}


def listed():
    return [
        # one new token each of 32 chats: the queries' rotation, all latency
        {"name": "rope_decode_32", "kind": "rope", "rows": 32, "heads": 32, "head_dim": 128,
         "rot": 128, "layout": "halves", "scaling": "plain", "factor": 1.0, "far": 8000,
         "pad": 0},
        # q and k of long prompts inside their q|k|v rows, context stretched four times
        {"name": "rope_yarn_6000", "kind": "rope", "rows": 6000, "heads": 40, "head_dim": 128,
         "rot": 128, "layout": "halves", "scaling": "yarn", "factor": 4.0, "far": 131072,
         "pad": 1024},
        # one new token each of 48 chats into an f16 cache
        {"name": "rope_kv_decode_48", "kind": "rope_kv", "rows": 48, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "layout": "halves", "scaling": "plain", "factor": 1.0,
         "far": 8000, "kv": "f16", "page": 16},
        # a batch of prompts, 4,100 rows in all, into an f16 cache
        {"name": "rope_kv_prompts_4100", "kind": "rope_kv", "rows": 4100, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rot": 128, "layout": "halves", "scaling": "plain",
         "factor": 1.0, "far": 32768, "kv": "f16", "page": 64},
        # a decode step of 48 chats: a block here and there, three chats end
        {"name": "tables_decode_48", "kind": "tables", "seqs": 48, "lo": 40, "hi": 8000,
         "fresh_lo": 1, "fresh": 1, "page": 16, "tree": False, "spare": 80},
        # 600 requests with prompts of up to 400 tokens, rows left over for others
        {"name": "tables_prompts_600", "kind": "tables", "seqs": 600, "lo": 1, "hi": 3000,
         "fresh_lo": 1, "fresh": 400, "page": 16, "tree": False, "spare": 5000},
        # one chat, 61 drafted tokens as a tree, 4 K positions of an f16 cache
        {"name": "tree_1x61_at_4100", "kind": "tree", "seqs": 1, "nodes_lo": 61, "nodes": 61,
         "lo": 4100, "hi": 4100, "heads": 32, "kv_heads": 8, "head_dim": 128, "kv": "f16",
         "page": 16, "tree": True},
        # twelve chats with trees of 4 to 16 drafted tokens
        {"name": "tree_12x16_ragged", "kind": "tree", "seqs": 12, "nodes_lo": 4, "nodes": 16,
         "lo": 200, "hi": 12000, "heads": 32, "kv_heads": 8, "head_dim": 128, "kv": "f16",
         "page": 16, "tree": True},
        # 48 chats, one new token each and no drafts: batched decode
        {"name": "chain_48x1_ragged", "kind": "tree", "seqs": 48, "nodes_lo": 1, "nodes": 1,
         "lo": 100, "hi": 8000, "heads": 32, "kv_heads": 8, "head_dim": 128, "kv": "f16",
         "page": 64, "tree": False},
        # pieces of four prompts behind their earlier pieces, the small model's f32 cache
        {"name": "chunks_4x300_f32", "kind": "tree", "seqs": 4, "nodes_lo": 80, "nodes": 300,
         "lo": 700, "hi": 9000, "heads": 16, "kv_heads": 8, "head_dim": 128, "kv": "f32",
         "page": 32, "tree": False},
        # one chat's accepted path of five tokens
        {"name": "accept_1x5", "kind": "accept", "seqs": 1, "nodes": 61, "path": 5, "lo": 4100,
         "hi": 4100, "kv_heads": 8, "head_dim": 128, "kv": "f16", "page": 16},
        # 48 chats' accepted paths, the small model's f32 cache
        {"name": "accept_48x6_f32", "kind": "accept", "seqs": 48, "nodes": 24, "path": 6,
         "lo": 30, "hi": 900, "kv_heads": 8, "head_dim": 128, "kv": "f32", "page": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any of the kinds; rows, contexts, requests and tree
    sizes spread over their logarithm, every layout, scaling, page and type."""
    kind = rng.choice(["rope", "rope_kv", "tables", "tree", "tree", "tree", "accept"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv = rng.choice(["f16", "f16", "f32"])
    hd = rng.choice([128, 128, 64, 256])
    if kind in ("rope", "rope_kv"):
        scaling = rng.choice(["plain", "linear", "yarn", "bands"])
        heads, kv_heads = rng.choice([(32, 8), (16, 8), (16, 2), (8, 8), (7, 1)])
        case = {"kind": kind, "rows": _log(rng, 1, 4000), "heads": heads, "head_dim": hd,
                "rot": rng.choice([hd, hd, hd // 2, hd // 4]),
                "layout": rng.choice(["halves", "pairs"]), "scaling": scaling,
                "factor": 1.0 if scaling == "plain" else rng.uniform(1.5, 16.0),
                "far": _log(rng, 50, 1000000)}
        if kind == "rope":
            case["pad"] = rng.choice([0, 0, 4 * rng.randint(1, 300)])
        else:
            case.update(kv_heads=kv_heads, kv=kv, page=page)
        most = 4 * case["rows"] * hd * (2 * heads + 4 * kv_heads)
        if most > 240e6:
            case["rows"] = int(case["rows"] * 240e6 / most)
        return case
    if kind == "tables":
        tree = rng.random() < 0.4
        fresh = rng.randint(1, 64) if tree else _log(rng, 1, 300)
        return {"kind": kind, "seqs": _log(rng, 1, 500), "lo": rng.randint(1, 60),
                "hi": _log(rng, 100, 6000), "fresh_lo": rng.randint(1, fresh), "fresh": fresh,
                "page": page, "tree": tree, "spare": rng.choice([0, _log(rng, 1, 3000)])}
    lo = _log(rng, 1, 4000)
    hi = min(30000, lo + _log(rng, 1, 26000))
    if kind == "accept":
        path = rng.randint(1, 12)
        hi = min(hi, 1000)
        return {"kind": kind, "seqs": _log(rng, 1, 48), "nodes": rng.randint(path, 64),
                "path": path, "lo": min(lo, hi), "hi": hi, "kv_heads": rng.choice([1, 2, 8]),
                "head_dim": hd, "kv": kv, "page": page}
    tree = rng.random() < 0.6
    nodes = _log(rng, 1, 100) if tree else _log(rng, 1, 400)
    heads, kv_heads = rng.choice([(32, 8), (16, 8), (16, 2), (8, 8), (7, 1)])
    case = {"kind": kind, "seqs": _log(rng, 1, 48), "nodes_lo": rng.randint(1, nodes),
            "nodes": nodes, "lo": lo, "hi": hi, "heads": heads, "kv_heads": kv_heads,
            "head_dim": hd, "kv": kv, "page": page, "tree": tree}
    most = [work(c) for c in listed() if c["kind"] == "tree"]
    while True:  # no more than the largest listed ones
        w = work(case)
        if all(w[x] <= max(m[x] for m in most) for x in w):
            return case
        if case["seqs"] > 1:
            case["seqs"] = case["seqs"] * 3 // 4
        else:
            case["nodes"] = max(1, case["nodes"] * 3 // 4)
            case["nodes_lo"] = min(case["nodes_lo"], case["nodes"])


# ------------------------------------------------------------------ inputs

def _spread(n, lo, hi):
    """n whole numbers from lo to hi, even over their logarithm."""
    return np.rint(np.exp(np.linspace(math.log(lo), math.log(hi), n))).astype(np.int64)


def _lengths(case):
    """Cached positions and new rows of each request (-1: it has ended, as
    every 16th one of a ``tables`` case has)."""
    n = case["seqs"]
    cached = _spread(n, case["lo"], case["hi"]) if n > 1 else np.array([case["hi"]])
    key = "nodes" if "nodes" in case else "fresh"
    new = _spread(n, case.get(key + "_lo", case[key]), case[key])
    new = new[(np.arange(n) * 7 + 3) % n]
    if case["kind"] == "tables":
        new[15::16] = -1
    return cached, new


def _row_bytes(case):
    return case["kv_heads"] * case["head_dim"] * (2 if case["kv"] == "f16" else 4)


class _State:
    """A call's inputs on the device, and the buffers it fills."""


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype=dtype, device="cuda")


def _cache(s, case, g, slots):
    t = torch.float16 if case["kv"] == "f16" else torch.float32
    width = case["kv_heads"] * case["head_dim"]
    s.k = torch.randn(slots, width, generator=g, device="cuda").to(t)
    s.v = torch.randn(slots, width, generator=g, device="cuda").to(t)


def _trees(rng, new, words):
    """Ancestor bits of a random tree for each request: a node's parent is one
    of the eight before it, or the last cached token."""
    out = []
    for n in new:
        back = rng.integers(1, 9, n)
        seen = np.zeros((n, 32 * words), np.uint8)
        for i in range(n):
            if i - back[i] >= 0:
                seen[i] = seen[i - back[i]]
            seen[i, i] = 1
        out.append(np.packbits(seen, axis=1, bitorder="little").view(np.int32))
    return np.concatenate(out)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    rng = np.random.default_rng(int(seed) & 0x7FFFFFFF)
    s = _State()
    s.case, s.handles = case, None
    kind = case["kind"]
    if kind in ("rope", "rope_kv"):
        rows, heads, hd = case["rows"], case["heads"], case["head_dim"]
        width = (heads + 2 * case.get("kv_heads", 0)) * hd
        s.x = torch.randn(rows, width + case.get("pad", 0), generator=g, device="cuda")
        s.positions = _dev(rng.integers(0, case["far"], rows))
        s.freqs = _freqs(case)
        s.y = torch.empty(rows, heads * hd, device="cuda")
        if kind == "rope_kv":
            page = case["page"]
            s.blocks = (rows + page - 1) // page + 3
            _cache(s, case, g, s.blocks * page)
            s.slots = _dev(rng.permutation(s.blocks * page)[:rows])
        return s
    n, page = case["seqs"], case["page"]
    cached, new = _lengths(case)
    order = rng.permutation(n)
    cached, new = cached[order], new[order]
    s.most, s.longest = int(new.max()), int((cached + new).max())
    s.cached = _dev(cached)
    if kind == "tables":
        # blocks as the requests hold them before the step; unused table
        # entries are -1
        held = -(-cached // page)
        total = -(-(cached + np.maximum(new, 0)) // page)
        s.max_blocks = int(total.max()) + 1
        s.blocks = int(np.maximum(total, held).sum()) + 5
        ids = rng.permutation(s.blocks)
        tables = np.full((n, s.max_blocks), -1, np.int64)
        in_use = np.arange(s.max_blocks)[None] < held[:, None]
        tables[in_use] = ids[:held.sum()]
        free = np.full(s.blocks, -1, np.int64)
        left = s.blocks - int(held.sum())
        free[:left] = ids[held.sum():]
        s.fresh, s.held, s.tables, s.free = _dev(new), _dev(held), _dev(tables), _dev(free)
        s.n_free = _dev([left])
        s.rows = int(np.maximum(new, 0).sum()) + case["spare"]
        s.words = (s.most + 31) // 32
        s.mask = None
        if case["tree"]:
            bits = _trees(rng, np.maximum(new, 0), s.words)
            s.mask = _dev(np.pad(bits, ((0, case["spare"]), (0, 0))))
        s.held_out, s.n_free_out, s.status = (torch.empty_like(s.held),
                                              torch.empty_like(s.n_free),
                                              torch.empty_like(s.n_free))
        s.first_row = torch.empty(n + 1, dtype=torch.int32, device="cuda")
        s.positions, s.slots = (torch.empty(s.rows, dtype=torch.int32, device="cuda")
                                for _ in range(2))
        return s
    held = -(-(cached + new) // page)
    s.max_blocks = int(held.max()) + 2
    s.blocks = int(held.sum()) + 3
    tables = np.full((n, s.max_blocks), -1, np.int64)
    tables[np.arange(s.max_blocks)[None] < held[:, None]] = rng.permutation(s.blocks)[:held.sum()]
    s.tables = _dev(tables)
    _cache(s, case, g, s.blocks * page)
    s.rows = int(new.sum())
    s.first_row = _dev(np.concatenate([[0], np.cumsum(new)]))
    if kind == "accept":
        count = rng.integers(0, case["path"] + 1, n)
        count[0] = case["path"]
        path = np.sort(np.argsort(rng.random((n, case["nodes"])), axis=1)[:, :case["path"]], axis=1)
        s.path, s.count = _dev(path), _dev(count)
        s.cached_out = torch.empty_like(s.cached)
        return s
    heads, hd = case["heads"], case["head_dim"]
    s.q = 2.0 * torch.randn(s.rows, heads * hd, generator=g, device="cuda")
    s.words = (s.most + 31) // 32
    s.mask = _dev(_trees(rng, new, s.words)) if case["tree"] else None
    s.out = torch.empty_like(s.q)
    return s


# ------------------------------------------------------------- plain forms

# base of the rotary frequencies; where their scaled forms differ: trained
# length, turns over it (yarn), shortest and longest share of it (bands)
THETA, TRAINED, FAST, SLOW, LONG, SHORT = 1e6, 8192, 32.0, 1.0, 1.0, 4.0


def _freqs(case):
    """Angle per position of each rotated pair, in 64 bits."""
    rot, factor = case["rot"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = THETA ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return f / factor
    if case["scaling"] == "yarn":
        def dim(turns):
            return rot * math.log(TRAINED / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))
        lo, hi = max(math.floor(dim(FAST)), 0), min(math.ceil(dim(SLOW)), rot - 1)
        ramp = ((i - lo) / (hi - lo if hi > lo else 1e-3)).clamp(0.0, 1.0)
        return f / factor * ramp + f * (1.0 - ramp)
    if case["scaling"] == "bands":
        turns = TRAINED * f / (2.0 * math.pi)
        keep = ((turns - LONG) / (SHORT - LONG)).clamp(0.0, 1.0)
        return keep * f + (1.0 - keep) * f / factor
    return f


def _gain(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "yarn" else 1.0


def _rotate(s, x):
    """x [rows][heads][head_dim] rotated at the rows' positions."""
    rot, pairs = s.case["rot"], s.case["layout"] == "pairs"
    angle = s.positions.double()[:, None] * s.freqs
    c = (angle.cos() * _gain(s.case)).float()[:, None]
    d = (angle.sin() * _gain(s.case)).float()[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * c - b * d, b * c + a * d
    turned = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    c = s.case
    heads, hd = c["heads"], c["head_dim"]
    x = s.x[:, :heads * hd].reshape(-1, heads, hd)
    if c["kind"] == "rope":
        return _rotate(s, x).flatten(1)
    kv = c["kv_heads"]
    k, v = s.x[:, heads * hd:(heads + kv) * hd], s.x[:, (heads + kv) * hd:]
    s.k[s.slots.long()] = _rotate(s, k.reshape(-1, kv, hd)).flatten(1).to(s.k.dtype)
    s.v[s.slots.long()] = v.to(s.v.dtype)
    return {"q": _rotate(s, x).flatten(1), "k": s.k, "v": s.v}


def _plain_tables(s):
    page, n, width = s.case["page"], s.case["seqs"], s.max_blocks
    cached, fresh, held, n_free = (t.long() for t in (s.cached, s.fresh, s.held, s.n_free))
    ended = fresh < 0
    new = fresh.clamp(min=0)
    need = ((cached + new + page - 1) // page - held).clamp(min=0) * ~ended
    give = held * ended
    row_end, need_end, give_end = new.cumsum(0), need.cumsum(0), give.cumsum(0)
    top = n_free + give_end[-1]
    bad = (cached < 0).any() | (held < 0).any() | (held > width).any() | (n_free < 0) | \
        (top > s.blocks)
    status = torch.where(bad, 1, 2 * (row_end[-1] > s.rows) + 4 * (held + need > width).any() +
                         8 * (need_end[-1] > top))
    fine = status == 0
    # given back to the free list, then taken from its end
    j = torch.arange(width, device="cuda")
    put = ended[:, None] & (j < held[:, None]) & fine
    at = torch.where(put, n_free + (give_end - give)[:, None] + j, s.blocks)
    free = torch.cat([s.free, s.free[:1]]).scatter(0, at.flatten(), s.tables.flatten())[:-1]
    k = j - held[:, None]
    take = (k >= 0) & (k < need[:, None]) & fine
    at = (top - 1 - ((need_end - need)[:, None] + k)).clamp(0, s.blocks - 1)
    tables = torch.where(take, free[at], s.tables)
    first = torch.cat([row_end.new_zeros(1), row_end])
    r = torch.arange(s.rows, device="cuda")
    b = torch.searchsorted(row_end, r, right=True).clamp(max=n - 1)
    live = fine & (r < row_end[-1])
    at = cached[b] + r - first[b]
    block = tables[b, (at // page).clamp(0, width - 1)]
    slots = torch.where(live & (block >= 0) & (block < s.blocks), block * page + at % page, -1)
    depth = r - first[b]
    if s.mask is not None:
        bits = (s.mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        depth = (bits.sum((1, 2)) - 1).clamp(min=0)
    positions = torch.where(live, cached[b] + depth, -1)
    out = {"tables": tables, "free": free, "held": torch.where(fine, (held + need) * ~ended, held),
           "n_free": torch.where(fine, top - need_end[-1], n_free), "first_row": first * fine,
           "positions": positions, "slots": slots, "status": status}
    return {name: t.to(torch.int32) for name, t in out.items()}


def _plain_tree(s):
    c = s.case
    n, page, heads, kv, hd = c["seqs"], c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    group = heads // kv
    first, cached = s.first_row.long(), s.cached.long()
    p = torch.arange(s.longest, device="cuda")
    i = torch.arange(s.most, device="cuda")
    there = p < (cached + first[1:] - first[:-1])[:, None]
    slot = torch.where(there, s.tables.long()[:, p // page] * page + p % page, 0)
    k = s.k[slot].float().reshape(n, -1, kv, hd).permute(0, 2, 3, 1).contiguous()
    v = s.v[slot].float().reshape(n, -1, kv, hd).transpose(1, 2).contiguous()
    row = (first[:-1, None] + i).clamp(max=s.rows - 1)
    q = s.q[row].reshape(n, s.most, kv, group, hd).transpose(1, 2).reshape(n, kv, -1, hd)
    score = (q @ k).reshape(n, kv, s.most, group, -1) * hd ** -0.5
    j = p - cached[:, None]
    if s.mask is None:
        sees = j[:, None] <= i[:, None]
    else:
        word = (j >> 5).clamp(0, s.words - 1)[:, None].expand(n, s.most, -1)
        bits = s.mask[row].long().gather(2, word) >> (j & 31)[:, None]
        sees = (j < 0)[:, None] | ((bits & 1 == 1) & (j < 32 * s.words)[:, None])
    sees = (sees & there[:, None])[:, None, :, None]
    score = score.masked_fill(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    o = (e.reshape(n, kv, s.most * group, -1) @ v).reshape(n, kv, s.most, group, hd)
    o = torch.where(total > 0, o / total, 0.0).transpose(1, 2).reshape(n, s.most, heads * hd)
    r = torch.arange(s.rows, device="cuda")
    b = torch.searchsorted(first[1:], r, right=True)
    return o[b, r - first[b]]


def _plain_accept(s):
    page = s.case["page"]
    cached, count = s.cached.long()[:, None], s.count.long()[:, None]
    j = torch.arange(s.case["path"], device="cuda")
    src, dst = cached + torch.where(j < count, s.path.long(), j), cached + j
    tables = s.tables.long()
    src, dst = (tables.gather(1, p // page) * page + p % page for p in (src, dst))
    s.k[dst], s.v[dst] = s.k[src], s.v[src]
    return {"k": s.k, "v": s.v, "cached": s.cached + s.count}


# ------------------------------------------------------- the framework's calls

_CW = None


def _framework():
    """The binding and a context, loaded on first use."""
    global _CW
    if _CW is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "chat-wgpu_amd"))
        import cw
        _CW = cw, cw.Context(0)
    return _CW


def _handles(s):
    """The state's buffers as the binding takes them, made once."""
    cw, ctx = _framework()
    c, h = s.case, _State()
    for name, t in vars(s).items():
        if isinstance(t, torch.Tensor):
            setattr(h, name, cw.DeviceArray(ctx, tuple(t.shape), np.uint8, t.data_ptr()))
    h.mask = getattr(h, "mask", None)
    if c["kind"] in ("rope", "rope_kv"):
        h.spec = cw.rope_spec(c["rot"], THETA,
                              layout={"halves": cw.ROPE_HALVES, "pairs": cw.ROPE_PAIRS}[c["layout"]],
                              scaling={"plain": cw.ROPE_PLAIN, "linear": cw.ROPE_LINEAR,
                                       "yarn": cw.ROPE_YARN, "bands": cw.ROPE_BANDS}[c["scaling"]],
                              factor=c["factor"], trained=TRAINED, beta_fast=FAST, beta_slow=SLOW,
                              low_turns=LONG, high_turns=SHORT)
    if c["kind"] != "rope":
        kv_type = cw.CW_F32 if c.get("kv") == "f32" else cw.CW_F16
        h.kv = cw.kv_pages(getattr(h, "k", None), getattr(h, "v", None), kv_type,
                           c.get("kv_heads", 1), c.get("head_dim", 128), c["page"], s.blocks)
    if c["kind"] in ("tables", "tree", "accept"):
        h.batch = cw.batch(h.cached, c["seqs"], s.rows, h.first_row, h.tables, s.max_blocks,
                           mask=h.mask, mask_words=s.words if h.mask is not None else 0)
    return h


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if not own:
        return {"rope": _plain_rope, "rope_kv": _plain_rope, "tables": _plain_tables,
                "tree": _plain_tree, "accept": _plain_accept}[kind](s)
    _, ctx = _framework()
    if s.handles is None:
        s.handles = _handles(s)
    h = s.handles
    if kind == "rope":
        ctx.rope_rows(h.spec, h.x, h.positions, c["rows"], c["heads"], c["head_dim"],
                      x_stride=s.x.stride(0), y=h.y)
        return s.y
    if kind == "rope_kv":
        ctx.rope_kv_rows(h.spec, h.kv, h.x, h.positions, h.slots, c["rows"], c["heads"], q_out=h.y)
        return {"q": s.y, "k": s.k, "v": s.v}
    if kind == "tables":
        ctx.block_tables(h.kv, h.batch, h.fresh, h.held, h.held_out, h.free, h.n_free,
                         h.n_free_out, h.positions, h.slots, h.status)
        return {"tables": s.tables, "free": s.free, "held": s.held_out, "n_free": s.n_free_out,
                "first_row": s.first_row, "positions": s.positions, "slots": s.slots,
                "status": s.status}
    if kind == "tree":
        ctx.attention_tree(h.kv, h.batch, h.q, c["heads"], out=h.out)
        return s.out
    ctx.kv_accept(h.kv, h.batch, h.path, c["path"], h.count, cached_out=h.cached_out)
    return {"k": s.k, "v": s.v, "cached": s.cached_out}


# --------------------------------------------------------- floors and results

def work(case):
    kind = case["kind"]
    if kind == "rope":
        values = case["rows"] * case["heads"] * case["head_dim"]
        return {"bytes": 8 * values + 4 * case["rows"], "flops": 3 * values}
    if kind == "rope_kv":
        width = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        out = 4 * case["heads"] * case["head_dim"] + 2 * _row_bytes(case)
        return {"bytes": case["rows"] * (4 * width + out + 8), "flops": 3 * case["rows"] * width}
    cached, new = _lengths(case)
    if kind == "tables":
        # lengths and blocks held in and out, a table entry for each new block
        # and each block that rows fall into, two numbers for each row
        page, words = case["page"], (int(new.max()) + 31) // 32 if case["tree"] else 0
        new = np.maximum(new, 0)
        blocks = int((-(-(cached + new) // page) - cached // page).sum())
        rows = int(new.sum()) + case["spare"]
        return {"bytes": 20 * case["seqs"] + 8 * blocks + (8 + 4 * words) * rows, "flops": 4 * rows}
    if kind == "accept":
        rows = case["seqs"] * (case["path"] + 1) // 2
        return {"bytes": 4 * rows * _row_bytes(case) + 16 * case["seqs"], "flops": rows}
    pairs = int((new * (cached + 1)).sum()) if case["tree"] else \
        int((new * cached + new * (new + 1) // 2).sum())
    rows, heads, hd = int(new.sum()), case["heads"], case["head_dim"]
    return {"bytes": 2 * int((cached + new).sum()) * _row_bytes(case) + 8 * rows * heads * hd,
            "flops": 4 * heads * hd * pairs}


def _turn(case, x, positions):
    """Rows x [rows][heads][head_dim] in 64 bits, each pair as one complex number."""
    rot, f = case["rot"], []
    for i in range(rot // 2):
        w = 1.0 / THETA ** (2.0 * i / rot)
        if case["scaling"] == "linear":
            w /= case["factor"]
        elif case["scaling"] == "yarn":
            ends = [rot * math.log(TRAINED / (2 * math.pi * t)) / math.log(THETA) / 2
                    for t in (FAST, SLOW)]
            lo, hi = max(0, math.floor(ends[0])), min(rot - 1, math.ceil(ends[1]))
            share = min(1.0, max(0.0, (i - lo) / (hi - lo or 1e-3)))
            w = w * (1 - share) + w / case["factor"] * share
        elif case["scaling"] == "bands":
            length = 2 * math.pi / w
            if length > TRAINED / LONG:
                w /= case["factor"]
            elif length > TRAINED / SHORT:
                smooth = (TRAINED / length - LONG) / (SHORT - LONG)
                w = (1 - smooth) * w / case["factor"] + smooth * w
        f.append(w)
    gain = 1.0 + 0.1 * math.log(case["factor"]) if case["scaling"] == "yarn" else 1.0
    angle = torch.outer(positions.double(), torch.tensor(f, dtype=torch.float64, device="cuda"))
    z = torch.polar(torch.full_like(angle, gain), angle)[:, None]
    y = x.double().clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["layout"] == "pairs" else \
        (slice(0, rot // 2), slice(rot // 2, rot))
    turned = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = turned.real, turned.imag
    return y.flatten(1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("rope", "rope_kv"):
        heads, hd, kv = case["heads"], case["head_dim"], case.get("kv_heads", 0)
        x = s.x[:, :(heads + 2 * kv) * hd].reshape(case["rows"], -1, hd)
        q = _turn(case, x[:, :heads], s.positions)
        if kind == "rope":
            return q
        k, v = s.k.double(), s.v.double()
        k[s.slots.long()] = _turn(case, x[:, heads:heads + kv], s.positions)
        v[s.slots.long()] = x[:, heads + kv:].double().flatten(1)
        return {"q": q, "k": k, "v": v}
    page = case["page"]
    tables, cached = s.tables.tolist(), s.cached.tolist()
    if kind == "tables":
        free, held = s.free.tolist(), s.held.tolist()
        top = int(s.n_free)
        mask = None if s.mask is None else s.mask.cpu().numpy().view(np.uint32)
        fresh, first, positions, slots = s.fresh.tolist(), [0], [], []
        for b, new in enumerate(fresh):
            if new < 0:
                free[top:top + held[b]] = tables[b][:held[b]]
                top, held[b] = top + held[b], 0
        for b, new in enumerate(fresh):
            if new >= 0:
                while held[b] * page < cached[b] + new:
                    top -= 1
                    tables[b][held[b]] = free[top]
                    held[b] += 1
                for i in range(new):
                    at = cached[b] + i
                    row = len(slots)
                    depth = i if mask is None else max(0, int(np.unpackbits(
                        mask[row].view(np.uint8)).sum()) - 1)
                    slots.append(tables[b][at // page] * page + at % page)
                    positions.append(cached[b] + depth)
            first.append(len(slots))
        rest = [-1] * (s.rows - len(slots))
        out = {"tables": tables, "free": free, "held": held, "n_free": [top], "first_row": first,
               "positions": positions + rest, "slots": slots + rest, "status": [0]}
        return {name: torch.tensor(v, dtype=torch.int32) for name, v in out.items()}
    if kind == "accept":
        k, v = s.k.double(), s.v.double()
        path, count = s.path.tolist(), s.count.tolist()

        def slot(b, p):
            return tables[b][p // page] * page + p % page
        for b, c in enumerate(cached):
            for i in range(count[b]):
                a, z = slot(b, c + path[b][i]), slot(b, c + i)
                k[z], v[z] = k[a].clone(), v[a].clone()
        return {"k": k, "v": v, "cached": s.cached + s.count}
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    first, out = s.first_row.tolist(), []
    for b, c in enumerate(cached):
        n = first[b + 1] - first[b]
        slots = torch.tensor([tables[b][p // page] * page + p % page for p in range(c + n)],
                             device="cuda")
        keys, vals = (t[slots].double().reshape(c + n, kv, hd) for t in (s.k, s.v))
        hidden = torch.zeros(n, c + n, dtype=torch.bool, device="cuda")
        if s.mask is None:
            hidden[:, c:] = torch.ones(n, n, device="cuda").triu(1) > 0
        else:
            bits = s.mask[first[b]:first[b + 1]].cpu().numpy().view(np.uint8)
            bits = np.unpackbits(bits, axis=1, bitorder="little")[:, :n]
            hidden[:, c:] = torch.from_numpy(bits == 0).cuda()
        q = s.q[first[b]:first[b + 1]].double().reshape(n, heads, hd)
        o = torch.empty(n, heads, hd, dtype=torch.float64, device="cuda")
        for a in range(heads):
            g = a // (heads // kv)
            score = (q[:, a] @ keys[:, g].T.contiguous() / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            o[:, a] = score.softmax(-1) @ vals[:, g].contiguous()
        out.append(o.reshape(n, -1))
    return torch.cat(out)
