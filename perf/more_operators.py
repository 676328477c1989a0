"""What a step of a server needs around its paged cache and attention, from the
q | k | v rows to the next tokens, as cases to be timed:

  * ``norm``, ``norm_kv``  the norm of every query and key head with the rotary
    positions in the same pass, alone (``cw_qk_norm_rope_rows``) and with the
    cache write (``cw_qk_norm_rope_kv_rows``);
  * ``moe``     a whole mixture-of-experts layer over Q4_0 experts: router,
    choice, the chosen experts' products, their weighted sum (``cw_moe_rows``);
  * ``logits``  penalties for repeated tokens, biases and grammar masks, the
    likeliest token and its log probability (``cw_logits_rows``).

Heads, kv heads, head sizes, model widths and the vocabulary are those of the
Qwen3-8B and Qwen3-0.6B configurations that the tests and the benchmark run;
expert counts and widths are generic.  Activations are unit normal, as they are
behind a norm; expert weights are Q4_0 blocks of random nibbles that keep the
scale of what passes through; logits are normal with a few likely tokens, and
the tokens of a text repeat by a power law.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

VOCAB = 151936
EPS = 1e-6


def listed():
    return [
        # one new token each of 32 chats, q and k normed and rotated: all latency
        {"name": "norm_decode_32", "kind": "norm", "rows": 32, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "layout": "halves", "factor": 1.0, "far": 8000, "pad": 1024},
        # q and k of long prompts, context stretched four times
        {"name": "norm_yarn_6000", "kind": "norm", "rows": 6000, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "layout": "halves", "factor": 4.0, "far": 131072, "pad": 0},
        # one new token each of 48 chats into an f16 cache
        {"name": "norm_kv_decode_48", "kind": "norm_kv", "rows": 48, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot": 128, "layout": "halves", "factor": 1.0, "far": 8000,
         "kv": "f16", "page": 16},
        # a batch of prompts, 4,100 rows in all, into an f16 cache
        {"name": "norm_kv_prompts_4100", "kind": "norm_kv", "rows": 4100, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rot": 128, "layout": "halves", "factor": 1.0,
         "far": 32768, "kv": "f16", "page": 64},
        # one chat's decode step: its token alone is wanted
        {"name": "logits_1_greedy", "kind": "logits", "seqs": 1, "nodes": 1, "tree": False,
         "lo": 900, "hi": 900, "vocab": VOCAB, "bias": 0, "masks": False, "out": False},
        # 48 chats, every other one held to a grammar, some with biases; logits for a sampler
        {"name": "logits_48_masked", "kind": "logits", "seqs": 48, "nodes": 1, "tree": False,
         "lo": 100, "hi": 8000, "vocab": VOCAB, "bias": 40, "masks": True, "out": True},
        # one chat's 61 drafted tokens as a tree, each with the history of its own path
        {"name": "logits_tree_61", "kind": "logits", "seqs": 1, "nodes": 61, "tree": True,
         "lo": 4100, "hi": 4100, "vocab": VOCAB, "bias": 0, "masks": False, "out": False},
        # one chat's decode step through a layer of many small experts
        {"name": "moe_1_of_128x8", "kind": "moe", "rows": 1, "spare": 0, "dim": 2048, "hidden": 768,
         "experts": 128, "top": 8, "normalise": True, "residual": True},
        # the same for one chat with five drafted tokens
        {"name": "moe_6_of_128x8", "kind": "moe", "rows": 6, "spare": 0, "dim": 2048, "hidden": 768,
         "experts": 128, "top": 8, "normalise": True, "residual": True},
        # 45 chats in a batch recorded for 48
        {"name": "moe_48_of_128x8", "kind": "moe", "rows": 48, "spare": 3, "dim": 2048,
         "hidden": 768, "experts": 128, "top": 8, "normalise": True, "residual": True},
        # a piece of a prompt beside the chats
        {"name": "moe_500_of_128x8", "kind": "moe", "rows": 500, "spare": 0, "dim": 2048,
         "hidden": 768, "experts": 128, "top": 8, "normalise": True, "residual": True},
        # few experts as wide as the 8B model's feed-forward layer
        {"name": "moe_20_of_8x2_wide", "kind": "moe", "rows": 20, "spare": 0, "dim": 4096,
         "hidden": 12288, "experts": 8, "top": 2, "normalise": False, "residual": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any of the kinds; rows, histories and widths spread over
    their logarithm, odd ones among them."""
    kind = rng.choice(["norm", "norm_kv", "moe", "moe", "moe", "logits", "logits"])
    if kind in ("norm", "norm_kv"):
        hd = rng.choice([128, 128, 64, 256, 32])
        heads, kv_heads = rng.choice([(32, 8), (16, 8), (16, 2), (8, 8), (7, 1)])
        case = {"kind": kind, "rows": _log(rng, 1, 4000), "heads": heads, "kv_heads": kv_heads,
                "head_dim": hd, "rot": rng.choice([hd, hd, hd // 2, hd // 4]),
                "layout": rng.choice(["halves", "pairs"]),
                "factor": rng.choice([1.0, rng.uniform(1.5, 16.0)]), "far": _log(rng, 50, 1000000)}
        if kind == "norm":
            case["pad"] = rng.choice([0, 0, 4 * rng.randint(1, 300)])
        else:
            case.update(kv=rng.choice(["f16", "f16", "f32"]), page=rng.choice([16, 64, 256]))
    elif kind == "logits":
        nodes = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        lo = _log(rng, 1, 8000)
        seqs = _log(rng, 1, max(1, 64 // nodes))
        case = {"kind": kind, "seqs": seqs, "nodes": nodes, "tree": nodes > 1 and rng.random() < 0.7,
                "lo": lo, "hi": min(30000, lo + _log(rng, 1, 20000)),
                "vocab": rng.choice([VOCAB, VOCAB, _log(rng, 300, 160000)]),
                "bias": rng.choice([0, _log(rng, 1, 300)]), "masks": rng.random() < 0.5,
                "out": rng.random() < 0.5}
    else:
        dim, hidden = (32 * _log(rng, 8, 96) for _ in range(2))
        experts = _log(rng, 2, 200)
        case = {"kind": kind, "rows": _log(rng, 1, 500), "spare": 0, "dim": dim, "hidden": hidden,
                "experts": experts, "top": rng.randint(1, min(8, experts)),
                "normalise": rng.random() < 0.7, "residual": rng.random() < 0.5}
        case["spare"] = rng.choice([0, rng.randint(0, case["rows"] - 1)])
        while 3 * dim * hidden * case["experts"] > 1.0e9:
            case["experts"] = case["experts"] * 3 // 4
            case["top"] = min(case["top"], case["experts"])
    most = [work(c) for c in listed() if c["kind"] == kind]
    key = {"logits": "seqs"}.get(kind, "rows")
    while True:  # no more than the largest listed ones
        w = work(case)
        if case[key] == 1 or all(w[x] <= max(m[x] for m in most) for x in w):
            return case
        case[key] = case[key] * 3 // 4
        if "spare" in case:
            case["spare"] = min(case["spare"], case[key] - 1)


# ------------------------------------------------------------------ inputs

class _State:
    """A call's inputs on the device, and the buffers it fills."""


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype=dtype, device="cuda")


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, even over their logarithm."""
    if n == 1:
        return np.array([hi])
    return np.rint(np.exp(np.linspace(math.log(lo), math.log(hi), n))).astype(np.int64)


def _prepare_norm(s, case, g, rng):
    rows, heads, kv, hd = (case[x] for x in ("rows", "heads", "kv_heads", "head_dim"))
    cache = case["kind"] == "norm_kv"
    width = (heads + (2 if cache else 1) * kv) * hd
    # projections come out at other scales than 1, each head at its own
    size = 2.0 ** (2.0 * torch.randn(width // hd, generator=g, device="cuda"))
    s.x = torch.randn(rows, width + case.get("pad", 0), generator=g, device="cuda")
    s.x[:, :width] *= size.repeat_interleave(hd)
    s.q_gain, s.k_gain = (1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
    s.positions = _dev(rng.integers(0, case["far"], rows))
    s.y = torch.empty(rows, (heads if cache else heads + kv) * hd, device="cuda")
    if cache:
        page = case["page"]
        s.blocks = (rows + page - 1) // page + 3
        t = torch.float16 if case["kv"] == "f16" else torch.float32
        s.k, s.v = (torch.randn(s.blocks * page, kv * hd, generator=g, device="cuda").to(t)
                    for _ in range(2))
        s.slots = _dev(rng.permutation(s.blocks * page)[:rows])


def _q4(g, out_f, in_f, *lead):
    """Q4_0 blocks of random nibbles whose rows keep the scale of a unit input."""
    shape = (*lead, out_f, in_f // 32)
    d = torch.randn(shape, generator=g, device="cuda") * (1.0 / (4.6 * math.sqrt(in_f)))
    q = torch.randint(0, 256, (*shape, 16), generator=g, device="cuda", dtype=torch.uint8)
    return d.to(torch.float16), q


def _prepare_moe(s, case, g, rng):
    rows, dim, hidden, n = (case[x] for x in ("rows", "dim", "hidden", "experts"))
    s.x = torch.randn(rows, dim, generator=g, device="cuda")
    s.router = torch.randn(n, dim, generator=g, device="cuda") * (1.5 / math.sqrt(dim))
    (s.gate_s, s.gate_q), (s.up_s, s.up_q) = _q4(g, hidden, dim, n), _q4(g, hidden, dim, n)
    s.down_s, s.down_q = _q4(g, dim, hidden, n)
    s.residual = torch.randn(rows, dim, generator=g, device="cuda") if case["residual"] else None
    s.positions = None
    if case["spare"]:  # rows behind the last request's: of no position, holding anything
        at = rng.integers(0, 4000, rows)
        at[rows - case["spare"]:] = -1
        s.positions = _dev(at)
        s.x[rows - case["spare"]:] = math.nan
    s.y = torch.zeros(rows, dim, device="cuda")
    s.ids = torch.full((rows, case["top"]), -1, dtype=torch.int32, device="cuda")
    s.weights = torch.zeros(rows, case["top"], device="cuda")


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


def _logit_rows(case):
    """Nodes of each request."""
    n, nodes = case["seqs"], case["nodes"]
    return np.array([nodes]) if n == 1 else 1 + (np.arange(n) * 7 + nodes - 1) % nodes


def _prepare_logits(s, case, g, rng):
    n, vocab = case["seqs"], case["vocab"]
    new = _logit_rows(case)
    rows = s.rows = int(new.sum())
    s.first_row = _dev(np.concatenate([[0], np.cumsum(new)]))
    length = rng.permutation(_spread(n, case["lo"], case["hi"]))
    s.max_len = int(length.max())

    def text(*shape):  # the tokens of a text
        u = torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64)
        return (vocab * u ** 4).to(torch.int32).clamp(max=vocab - 1)
    s.tokens = text(n, s.max_len)
    s.cached = s.length = _dev(length)
    s.prompt = _dev(rng.integers(0, length + 1))
    s.node_token = text(rows) if case["nodes"] > 1 else None
    s.words = (int(new.max()) + 31) // 32
    s.mask = _dev(_trees(rng, new, s.words)) if case["tree"] else None
    s.repeat = _dev(rng.uniform(1.0, 1.4, n), torch.float32)
    s.presence = _dev(rng.uniform(0.0, 0.6, n), torch.float32)
    s.frequency = _dev(rng.uniform(0.0, 0.3, n), torch.float32)
    s.logits = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
    likely = text(rows, 6).long()
    s.logits.scatter_reduce_(1, likely, 8.0 + 4.0 * torch.rand(rows, 6, generator=g, device="cuda"),
                             "amax")
    s.bias_first = s.bias_token = s.bias = None
    if case["bias"]:
        count = rng.integers(0, case["bias"] + 1, n)
        count[0] = case["bias"]
        s.bias_first = _dev(np.concatenate([[0], np.cumsum(count)]))
        s.bias_token = text(int(count.sum()))
        s.bias = 4.0 * torch.randn(int(count.sum()), generator=g, device="cuda")
    s.allowed = s.allowed_row = None
    if case["masks"]:
        # grammars that allow few tokens and ones that allow most; one of 16
        # has come to its end and allows none
        w = s.allowed_words = (vocab + 31) // 32
        s.masks = rows // 2 + 1
        s.allowed = torch.zeros(s.masks, w, dtype=torch.int32, device="cuda")
        bits = torch.randint(-2 ** 31, 2 ** 31, (s.masks, 4, w), generator=g, device="cuda")
        few = bits[:, 0] & bits[:, 1] & bits[:, 2] & bits[:, 3]
        most = bits[:, 0] | bits[:, 1] | bits[:, 2] | bits[:, 3]
        k = torch.arange(s.masks, device="cuda")[:, None]
        s.allowed += torch.where(k % 16 == 11, 0, torch.where(k % 2 == 0, few, most)).int()
        use = np.where(np.arange(rows) % 2 == 0, np.arange(rows) // 2, -1)
        s.allowed_row = _dev(rng.permutation(use))
    s.out = torch.zeros(rows, vocab, device="cuda") if case["out"] else None
    s.token = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s.logprob = torch.zeros(rows, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    rng = np.random.default_rng(int(seed) & 0x7FFFFFFF)
    s = _State()
    s.case, s.handles = case, None
    {"norm": _prepare_norm, "norm_kv": _prepare_norm, "moe": _prepare_moe,
     "logits": _prepare_logits}[case["kind"]](s, case, g, rng)
    return s


# ------------------------------------------------------------- plain forms

# base of the rotary frequencies; of their stretched form (yarn) the trained
# length and the turns over it between which it sets in
THETA, TRAINED, FAST, SLOW = 1e6, 8192, 32.0, 1.0


def _plain_norm(s):
    c = s.case
    heads, kv, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rot"]
    cache = c["kind"] == "norm_kv"
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f, gain = THETA ** (-2.0 * i / rot), 1.0
    if c["factor"] != 1.0:
        ends = [rot * math.log(TRAINED / (t * 2.0 * math.pi)) / (2.0 * math.log(THETA))
                for t in (FAST, SLOW)]
        lo, hi = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rot - 1)
        ramp = ((i - lo) / (hi - lo if hi > lo else 1e-3)).clamp(0.0, 1.0)
        f, gain = f / c["factor"] * ramp + f * (1.0 - ramp), 0.1 * math.log(c["factor"]) + 1.0
    angle = s.positions.double()[:, None] * f
    co, si = ((t * gain).float()[:, None] for t in (angle.cos(), angle.sin()))
    x = s.x[:, :(heads + kv) * hd].reshape(-1, heads + kv, hd)
    g = torch.cat([s.q_gain.expand(heads, hd), s.k_gain.expand(kv, hd)])
    x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * g
    pairs = c["layout"] == "pairs"
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * co - b * si, b * co + a * si
    turned = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    x = torch.cat([turned, x[..., rot:]], -1)
    if not cache:
        return x.flatten(1)
    at = s.slots.long()
    s.k[at] = x[:, heads:].flatten(1).to(s.k.dtype)
    s.v[at] = s.x[:, (heads + kv) * hd:].to(s.v.dtype)
    return {"q": x[:, :heads].flatten(1), "k": s.k, "v": s.v}


def _weights(d, q):
    """The f32 matrices of split Q4_0 blocks."""
    w = torch.cat([q & 15, q >> 4], -1).float() - 8.0
    return (w * d.float()[..., None]).flatten(-2)


def _plain_moe(s):
    c = s.case
    rows, n, k = c["rows"], c["experts"], c["top"]
    live = torch.arange(rows, device="cuda")[:, None] < rows - c["spare"]
    x = torch.where(live, s.x, 0.0)
    # the choice between two experts is a border: in 64 bits
    score = x.double() @ s.router.double().T.contiguous()
    p, ids = score.softmax(-1).sort(dim=-1, descending=True, stable=True)
    p, ids = p[:, :k], ids[:, :k]
    p = (p / p.sum(-1, keepdim=True) if c["normalise"] else p).float()
    if rows * k < n:  # the chosen matrices alone
        e = ids.flatten()
        xs = x.repeat_interleave(k, 0)[:, :, None]
        g, u = (_weights(d[e], q[e]) @ xs for d, q in ((s.gate_s, s.gate_q), (s.up_s, s.up_q)))
        z = _weights(s.down_s[e], s.down_q[e]) @ (g * g.sigmoid() * u)
        y = (z.reshape(rows, k, -1) * p[..., None]).sum(1)
    else:  # every expert for every row, unchosen ones at no weight
        xt = x.T.contiguous()
        g, u = (_weights(d, q).flatten(0, 1) @ xt for d, q in ((s.gate_s, s.gate_q), (s.up_s, s.up_q)))
        h = (g * g.sigmoid() * u).reshape(n, -1, rows)
        dense = torch.zeros(rows, n, device="cuda").scatter_(1, ids, p)
        z = torch.bmm(_weights(s.down_s, s.down_q), h)
        y = z.mul_(dense.T[:, None]).sum(0).T
    if s.residual is not None:
        y = s.residual + y
    s.y.copy_(torch.where(live, y, s.y))
    s.ids.copy_(torch.where(live, ids.int(), s.ids))
    s.weights.copy_(torch.where(live, p, s.weights))
    return {"y": s.y, "experts": s.ids, "weights": s.weights}


def _plain_logits(s):
    c = s.case
    n, vocab, rows = c["seqs"], c["vocab"], s.rows
    first = s.first_row.long()
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(first[1:], r, right=True)
    at = torch.arange(s.max_len, device="cuda")
    there, made = at < s.length[:, None], at >= s.prompt[:, None]
    token = s.tokens.long()
    count = torch.zeros(n, vocab, device="cuda").scatter_add_(1, token, (there & made).float())[b]
    seen = torch.zeros(n, vocab, device="cuda").scatter_add_(1, token, there.float())[b]
    if s.node_token is not None:
        i, j = (r - first[b])[:, None], (r - first[b])[None]
        if s.mask is None:
            sees = j <= i
        else:
            sees = (s.mask.long()[:, j[0] >> 5] >> (j & 31)) & 1 == 1
        sees = (sees & (b[:, None] == b[None])).float()
        to = s.node_token.long().expand(rows, rows)
        count, seen = count.scatter_add(1, to, sees), seen.scatter_add(1, to, sees)
    x = s.logits
    repeat, presence, frequency = (t[b][:, None] for t in (s.repeat, s.presence, s.frequency))
    x = torch.where(seen > 0, torch.where(x > 0, x / repeat, x * repeat), x)
    x = x - frequency * count - presence * (count > 0)
    if s.bias is not None:
        e = torch.arange(len(s.bias), device="cuda")
        of = torch.searchsorted(s.bias_first.long()[1:], e, right=True)
        last = torch.full((n * vocab,), -1, device="cuda").scatter_reduce_(
            0, of * vocab + s.bias_token.long(), e, "amax").reshape(n, vocab)[b]
        x = x + torch.where(last >= 0, s.bias[last.clamp(min=0)], 0.0)
    if s.allowed is not None:
        v = torch.arange(vocab, device="cuda")
        use = s.allowed_row.long()
        bit = (s.allowed[use.clamp(min=0)][:, v >> 5] >> (v & 31).int()) & 1
        x = x.masked_fill((use[:, None] >= 0) & (bit == 0), -math.inf)
    top = x.amax(-1, keepdim=True)
    some = top[:, 0] > -math.inf
    v = torch.arange(vocab, device="cuda").expand(rows, vocab)
    best = torch.where(x == top, v, vocab).amin(-1)
    # the others' share of a likely token is small beside its 1: summed apart from it
    rest = (x.double() - top.double()).exp().scatter(1, best[:, None], 0.0).sum(-1)
    out = {"token": torch.where(some, best, -1).int(),
           "logprob": torch.where(some, -rest.log1p(), -math.inf).float()}
    return out if s.out is None else {"logits": x, **out}


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
        elif t is None:
            setattr(h, name, None)
    if c["kind"] in ("norm", "norm_kv"):
        scaling = {} if c["factor"] == 1.0 else dict(
            scaling=cw.ROPE_YARN, factor=c["factor"], trained=TRAINED, beta_fast=FAST, beta_slow=SLOW)
        h.spec = cw.rope_spec(c["rot"], THETA, layout={"halves": cw.ROPE_HALVES,
                                                       "pairs": cw.ROPE_PAIRS}[c["layout"]], **scaling)
    if c["kind"] == "norm_kv":
        h.kv = cw.kv_pages(h.k, h.v, cw.CW_F32 if c["kv"] == "f32" else cw.CW_F16, c["kv_heads"],
                           c["head_dim"], c["page"], s.blocks)
    if c["kind"] == "moe":
        h.moe = cw.moe(c["dim"], c["hidden"], c["experts"], c["top"], h.router, h.gate_s, h.gate_q,
                       h.up_s, h.up_q, h.down_s, h.down_q, normalise=c["normalise"])
    if c["kind"] == "logits":
        h.batch = cw.batch(h.cached, c["seqs"], s.rows, h.first_row, None, 0, mask=h.mask,
                           mask_words=s.words if h.mask is not None else 0)
        h.rules = cw.logit_rules(
            tokens=h.tokens, length=h.length, prompt=h.prompt, max_len=s.max_len,
            node_token=h.node_token, repeat=h.repeat, presence=h.presence, frequency=h.frequency,
            bias_first=h.bias_first, bias_token=h.bias_token, bias=h.bias,
            n_bias=0 if s.bias is None else len(s.bias), allowed=h.allowed,
            n_allowed=0 if s.allowed is None else s.masks,
            allowed_words=0 if s.allowed is None else s.allowed_words, allowed_row=h.allowed_row)
    return h


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if not own:
        return {"norm": _plain_norm, "norm_kv": _plain_norm, "moe": _plain_moe,
                "logits": _plain_logits}[kind](s)
    _, ctx = _framework()
    if s.handles is None:
        s.handles = _handles(s)
    h = s.handles
    if kind == "norm":
        ctx.qk_norm_rope_rows(h.spec, h.x, h.q_gain, h.k_gain, h.positions, c["rows"], c["heads"],
                              c["kv_heads"], c["head_dim"], EPS, x_stride=s.x.stride(0), y=h.y)
        return s.y
    if kind == "norm_kv":
        ctx.qk_norm_rope_kv_rows(h.spec, h.kv, h.x, h.q_gain, h.k_gain, h.positions, h.slots,
                                 c["rows"], c["heads"], EPS, q_out=h.y)
        return {"q": s.y, "k": s.k, "v": s.v}
    if kind == "moe":
        ctx.moe_rows(h.moe, h.x, c["rows"], residual=h.residual, positions=h.positions, y=h.y,
                     experts=h.ids, weights=h.weights)
        return {"y": s.y, "experts": s.ids, "weights": s.weights}
    ctx.logits_rows(h.rules, h.batch, h.logits, s.rows, c["vocab"], out=h.out, token=h.token,
                    logprob=h.logprob)
    out = {"token": s.token, "logprob": s.logprob}
    return out if s.out is None else {"logits": s.out, **out}


# --------------------------------------------------------- floors and results

def work(case):
    if case["kind"] in ("norm", "norm_kv"):
        heads, kv, hd, rows = (case[x] for x in ("heads", "kv_heads", "head_dim", "rows"))
        if case["kind"] == "norm":
            return {"bytes": rows * (8 * (heads + kv) * hd + 4) + 8 * hd,
                    "flops": 7 * rows * (heads + kv) * hd}
        out = 4 * heads * hd + 2 * kv * hd * (2 if case["kv"] == "f16" else 4)
        return {"bytes": rows * (4 * (heads + 2 * kv) * hd + out + 8) + 8 * hd,
                "flops": 7 * rows * (heads + kv) * hd}
    if case["kind"] == "moe":
        dim, hidden, n, k = (case[x] for x in ("dim", "hidden", "experts", "top"))
        rows = case["rows"] - case["spare"]
        chosen = n * (1.0 - (1.0 - k / n) ** rows)  # experts that any row chooses, on average
        expert = 3 * dim * hidden * 18 // 32
        return {"bytes": int(chosen * expert) + 4 * n * dim + 8 * rows * (dim + k) +
                (4 * rows * dim if case["residual"] else 0),
                "flops": 2 * rows * n * dim + 6 * rows * k * dim * hidden}
    vocab, n = case["vocab"], case["seqs"]
    rows = int(_logit_rows(case).sum())
    byte = rows * vocab * (8 if case["out"] else 4) + 4 * int(_spread(n, case["lo"], case["hi"]).sum())
    if case["masks"]:
        byte += (rows + 1) // 2 * ((vocab + 31) // 32 * 4)
    return {"bytes": byte + 4 * n * case["bias"] + 8 * rows, "flops": 6 * rows * vocab}


def _exact_norm(s):
    c = s.case
    heads, kv, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rot"]
    x = s.x.double()
    turned = []
    gain = 1.0 + 0.1 * math.log(c["factor"])  # 1 at factor 1
    ends = [rot * math.log(TRAINED / (2 * math.pi * t)) / math.log(THETA) / 2 for t in (FAST, SLOW)]
    lo, hi = max(0, math.floor(ends[0])), min(rot - 1, math.ceil(ends[1]))
    spin = []
    for i in range(rot // 2):
        w = 1.0 / THETA ** (2.0 * i / rot)
        share = min(1.0, max(0.0, (i - lo) / (hi - lo or 1e-3))) if c["factor"] != 1.0 else 0.0
        angle = s.positions.double() * (w * (1 - share) + w / c["factor"] * share)
        spin.append(torch.polar(torch.full_like(angle, gain), angle))
    spin = torch.stack(spin, -1)
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["layout"] == "pairs" else \
        (slice(0, rot // 2), slice(rot // 2, rot))
    for h in range(heads + kv):
        v = x[:, h * hd:(h + 1) * hd]
        v = v / ((v * v).sum(-1, keepdim=True) / hd + EPS).sqrt()
        v = v * (s.q_gain if h < heads else s.k_gain).double()
        z = torch.complex(v[:, first].contiguous(), v[:, second].contiguous()) * spin
        v[:, first], v[:, second] = z.real, z.imag
        turned.append(v)
    if c["kind"] == "norm":
        return torch.cat(turned, 1)
    k, v = s.k.double(), s.v.double()
    k[s.slots.long()] = torch.cat(turned[heads:], 1)
    v[s.slots.long()] = x[:, (heads + kv) * hd:]
    return {"q": torch.cat(turned[:heads], 1), "k": k, "v": v}


def _exact_moe(s):
    c = s.case
    rows, k = c["rows"] - c["spare"], c["top"]
    x, y = s.x[:rows].double(), s.y.double()
    ids, weights = s.ids.clone(), s.weights.double()
    if rows == 0:
        return {"y": y, "experts": ids, "weights": weights}
    score = (x @ s.router.double().T.contiguous()).cpu().numpy()
    order = np.argsort(-score, axis=1, kind="stable")[:, :k]
    e = np.exp(score - score.max(1, keepdims=True))
    p = np.take_along_axis(e, order, 1)
    p = p / (p.sum(1, keepdims=True) if c["normalise"] else e.sum(1, keepdims=True))
    ids[:rows] = torch.from_numpy(order).int().cuda()
    weights[:rows] = torch.from_numpy(p).cuda()
    y[:rows] = 0.0 if s.residual is None else s.residual[:rows].double()

    def product(x, d, q):
        d, q = d.double()[:, :, None], q.int()
        w = torch.cat([(q % 16 - 8) * d, (q // 16 - 8) * d], 2).flatten(1)
        return x @ w.T.contiguous()
    for a in sorted(set(order.flatten().tolist())):
        row, j = (torch.from_numpy(t).cuda() for t in np.nonzero(order == a))
        g = product(x[row], s.gate_s[a], s.gate_q[a])
        h = g / (1.0 + (-g).exp()) * product(x[row], s.up_s[a], s.up_q[a])
        y[row] += weights[row, j][:, None] * product(h, s.down_s[a], s.down_q[a])
    return {"y": y, "experts": ids, "weights": weights}


def _exact_logits(s):
    c, vocab = s.case, s.case["vocab"]
    first, length, prompt = (t.tolist() for t in (s.first_row, s.length, s.prompt))
    tokens = s.tokens.cpu().numpy()
    node = None if s.node_token is None else s.node_token.cpu().numpy()
    bits = None if s.mask is None else s.mask.cpu().numpy().view(np.uint32)
    x = s.logits.double().cpu().numpy()
    out, token, logprob = [], [], []
    for b in range(c["seqs"]):
        repeat, presence, frequency = (float(t[b]) for t in (s.repeat, s.presence, s.frequency))
        text = tokens[b, :length[b]]
        for r in range(first[b], first[b + 1]):
            made = list(text[prompt[b]:])
            if node is not None:
                for j in range(first[b + 1] - first[b]):
                    if j <= r - first[b] if bits is None else int(bits[r, j // 32]) >> (j % 32) & 1:
                        made.append(node[first[b] + j])
            count = np.bincount(np.array(made, np.int64), minlength=vocab)
            seen = count.copy()
            seen[text[:prompt[b]]] += 1
            l = x[r].copy()
            up, down = (seen > 0) & (l > 0), (seen > 0) & (l <= 0)
            l[up] /= repeat
            l[down] *= repeat
            l -= frequency * count
            l[count > 0] -= presence
            if s.bias is not None:
                lo, hi = s.bias_first[b:b + 2].tolist()
                l_bias = dict(zip(s.bias_token[lo:hi].tolist(), s.bias[lo:hi].tolist()))
                for v, value in l_bias.items():  # a token's last entry
                    l[v] += value
            if s.allowed is not None and int(s.allowed_row[r]) >= 0:
                word = s.allowed[int(s.allowed_row[r])].cpu().numpy().view(np.uint8)
                l[np.unpackbits(word, bitorder="little")[:vocab] == 0] = -np.inf
            best = int(l.argmax())
            fine = l[best] > -np.inf
            token.append(best if fine else -1)
            logprob.append(-math.log1p(np.exp(np.delete(l, best) - l[best]).sum()) if fine else -math.inf)
            out.append(l)
    got = {"token": torch.tensor(token, dtype=torch.int32),
           "logprob": torch.tensor(logprob, dtype=torch.float64)}
    return got if s.out is None else {"logits": torch.from_numpy(np.stack(out)), **got}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "norm_kv": _exact_norm, "moe": _exact_moe,
            "logits": _exact_logits}[case["kind"]](s)
