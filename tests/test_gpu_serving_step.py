"""A server's step through one layer, call by call as a server makes them: blocks
and positions, norm, q, k and v, head norms and rotation into the cache, attention,
its product, norm, experts, head, rules.

Each call's result is held to its definition in 64 bits on the inputs that the call
had, with the bounds of step_oracle and paged_oracle; a recording of the step gives
the bits of the same calls made one by one."""
import threading

import numpy as np
import pytest

import cw
import paged_oracle as po
import step_oracle as so
from test_gpu_paged import KV, i32, tables_state

pytestmark = pytest.mark.gpu

DIM, HEADS, KVH, HD, HIDDEN, EXPERTS, TOP, VOCAB, PAGE, EPS = 256, 4, 2, 64, 96, 12, 3, 3001, 16, 1e-6
WIDTH = (HEADS + 2 * KVH) * HD
ROWS, MAX_LEN, TABLE = 18, 64, 12


class Server:
    """Weights, cache and buffers of a step of three requests: a tree of drafted
    tokens, one token, a piece of a prompt."""

    def __init__(self, ctx, seed, kv):
        self.ctx, rng = ctx, np.random.default_rng(seed)
        self.kv_type, self.dt = KV[kv]
        self.norms = [(1 + 0.2 * rng.standard_normal(DIM)).astype(np.float32) for _ in range(3)]
        self.gains = [(1 + 0.2 * rng.standard_normal(HD)).astype(np.float32) for _ in range(2)]
        self.router = rng.standard_normal((EXPERTS, DIM)).astype(np.float32) / np.float32(8)
        self.w = {n: so.q4(rng, *shape, scale=0.2 / np.sqrt(shape[-1])) for n, shape in dict(
            qkv=(WIDTH, DIM), o=(DIM, HEADS * HD), gate=(EXPERTS, HIDDEN, DIM), up=(EXPERTS, HIDDEN, DIM),
            down=(EXPERTS, DIM, HIDDEN), head=(VOCAB, DIM)).items()}
        self.wd = {n: (ctx.storage(d.view(np.uint16)), ctx.storage(q)) for n, (d, q) in self.w.items()}
        self.nd, self.gd = [ctx.storage(a) for a in self.norms], [ctx.storage(a) for a in self.gains]
        self.moe = cw.moe(DIM, HIDDEN, EXPERTS, TOP, ctx.storage(self.router), *self.wd["gate"],
                          *self.wd["up"], *self.wd["down"])
        self.spec = cw.rope_spec(HD, 1e6)
        self.blocks = 40
        e = ctx.empty
        self.k, self.v = (e((self.blocks * PAGE, KVH, HD), self.dt) for _ in range(2))
        self.pages = cw.kv_pages(self.k, self.v, self.kv_type, KVH, HD, PAGE, self.blocks)
        self.ints = {n: e(s, np.int32) for n, s in dict(
            cached=3, fresh=3, held=3, tables=(3, TABLE), free=self.blocks, n_free=1, held_out=3,
            n_free_out=1, first=4, positions=ROWS, slots=ROWS, status=1, tokens=(3, MAX_LEN), length=3,
            prompt=3, node=ROWS, allowed_row=ROWS, path=(3, 3), path_len=3, cached_out=3).items()}
        self.mask, self.allowed = e((ROWS, 1), np.uint32), e((2, (VOCAB + 31) // 32), np.uint32)
        self.penalties = [e(3) for _ in range(3)]
        d = self.ints
        self.batch = cw.batch(d["cached"], 3, ROWS, d["first"], d["tables"], TABLE, self.mask, 1)
        self.rules = cw.logit_rules(d["tokens"], d["length"], d["prompt"], MAX_LEN, d["node"],
                                    *self.penalties, allowed=self.allowed, n_allowed=2,
                                    allowed_words=(VOCAB + 31) // 32, allowed_row=d["allowed_row"])
        self.buf = {n: e((ROWS, s)) for n, s in dict(
            x=DIM, h=DIM, qkv=WIDTH, q=HEADS * HD, att=HEADS * HD, o=DIM, x1=DIM, h1=DIM, y=DIM, h2=DIM,
            logits=VOCAB, out=VOCAB, weights=TOP).items()}
        self.ids, self.token, self.logprob = e((ROWS, TOP), np.int32), e(ROWS, np.uint32), e(ROWS)

    def draw(self, seed):
        """State before a step: host arrays, on the device too."""
        rng, s = np.random.default_rng(seed), {}
        s["cached"] = i32([rng.integers(20, 60), rng.integers(0, 40), rng.integers(0, 90)])
        s["fresh"] = i32([5, 1, rng.integers(0, 10)])
        s["tables"], s["held"], s["free"], n, used = tables_state(
            rng, s["cached"], s["fresh"], PAGE, TABLE, 2)
        s["free"] = i32(np.concatenate([s["free"], np.full(self.blocks - used, -1)]))
        s["n_free"] = i32([n])
        s["mask"] = np.zeros((ROWS, 1), np.uint32)
        s["mask"][:5] = po.tree(rng, 5, 1)
        s["mask"][5], s["mask"][6:] = 1, (2 << np.arange(ROWS - 6, dtype=np.uint32)[:, None]) - 1
        s["tokens"] = i32(rng.integers(0, VOCAB, (3, MAX_LEN)))
        s["length"], s["prompt"] = i32(rng.integers(0, MAX_LEN + 1, 3)), i32([9, 0, 64])
        s["node"] = i32(rng.integers(0, VOCAB, ROWS))
        s["allowed"] = rng.integers(0, 1 << 32, (2, (VOCAB + 31) // 32), dtype=np.uint32)
        s["allowed_row"] = i32(rng.integers(-1, 2, ROWS))
        s["path"], s["path_len"] = i32([[0, 2, 4], [0, 0, 0], [0, 0, 0]]), i32([rng.integers(0, 4), 1, 0])
        s["x"] = rng.standard_normal((ROWS, DIM)).astype(np.float32)
        s["k"], s["v"] = (rng.standard_normal((self.blocks * PAGE, KVH, HD)).astype(self.dt)
                          for _ in range(2))
        s["penalties"] = [np.float32(a) for a in ((1.2, 1.0, 1.1), (0.1, 0.0, 0.2), (0.3, 0.0, 0.05))]
        return s

    def upload(self, s):
        for n, d in self.ints.items():
            d.upload(s[n] if n in s else np.full(d.shape, -5, np.int32))
        for d, a in zip((self.mask, self.allowed, self.k, self.v, *self.penalties),
                        (s["mask"], s["allowed"], s["k"], s["v"], *s["penalties"])):
            d.upload(a)
        for n, d in self.buf.items():
            d.upload(s["x"] if n == "x" else np.full(d.shape, 7.5, np.float32))
        self.ids.upload(np.full((ROWS, TOP), -7, np.int32))
        self.token.upload(np.full(ROWS, 77, np.uint32))
        self.logprob.upload(np.full(ROWS, 7.5, np.float32))

    def calls(self):
        ctx, d, b, L = self.ctx, self.ints, self.buf, cw.lib()

        def norm(x, w, y):
            cw.check(L.cw_rmsnorm(ctx.h, b[x].ptr, w.ptr, ROWS, DIM, EPS, b[y].ptr))

        ctx.block_tables(self.pages, self.batch, d["fresh"], d["held"], d["held_out"], d["free"],
                         d["n_free"], d["n_free_out"], d["positions"], d["slots"], d["status"])
        norm("x", self.nd[0], "h")
        ctx.q4_gemm(b["h"], ROWS, *self.wd["qkv"], DIM, WIDTH, y=b["qkv"])
        ctx.qk_norm_rope_kv_rows(self.spec, self.pages, b["qkv"], *self.gd, d["positions"], d["slots"],
                                 ROWS, HEADS, EPS, q_out=b["q"])
        ctx.attention_tree(self.pages, self.batch, b["q"], HEADS, out=b["att"])
        ctx.q4_gemm(b["att"], ROWS, *self.wd["o"], HEADS * HD, DIM, y=b["o"])
        cw.check(L.cw_add(ctx.h, b["x"].ptr, b["o"].ptr, ROWS * DIM, b["x1"].ptr))
        norm("x1", self.nd[1], "h1")
        ctx.moe_rows(self.moe, b["h1"], ROWS, residual=b["x1"], positions=d["positions"], y=b["y"],
                     experts=self.ids, weights=b["weights"])
        norm("y", self.nd[2], "h2")
        ctx.q4_gemm(b["h2"], ROWS, *self.wd["head"], DIM, VOCAB, y=b["logits"])
        ctx.logits_rows(self.rules, self.batch, b["logits"], ROWS, VOCAB, out=b["out"], token=self.token,
                        logprob=self.logprob)
        ctx.kv_accept(self.pages, self.batch, d["path"], 3, d["path_len"], d["cached_out"])

    def results(self):
        r = {n: d.download() for n, d in (*self.buf.items(), *self.ints.items())}
        r.update(ids=self.ids.download(), token=self.token.download(), logprob=self.logprob.download(),
                 k=self.k.download(), v=self.v.download())
        return r

    def check(self, s, r):
        tables = po.block_tables(s["cached"], s["fresh"], s["held"], s["tables"], s["free"],
                                 int(s["n_free"][0]), PAGE, self.blocks, ROWS, s["mask"])
        assert r["status"][0] == 0 and tables[0] == 0
        for n, want in zip(("tables", "held_out", "free", "n_free_out", "first", "positions", "slots"),
                           tables[1:]):
            assert np.array_equal(r[n].ravel(), np.ravel(want)), n
        first, pos, slots = tables[5:]
        live = int(first[-1])
        assert np.all(pos[:live] >= 0) and np.all(pos[live:] < 0)

        def close(got, want, bound, n=live):
            assert np.all(np.abs(got[:n] - want[:n]) <= bound[:n])

        def norm(x, w, got):  # dim / 8 products in a chain, then sums; root, quotient, products
            want = so.head_norm(r[x].reshape(ROWS, 1, DIM), w, np.float32(EPS)).reshape(ROWS, DIM)
            close(r[got], want, (DIM / 8 + 20) * so.H * np.abs(want), ROWS)

        def product(x, w, got):
            x64 = r[x].astype(np.float64)
            close(r[got], *so._product(x64, so.weights(*self.w[w]), np.zeros(x64.shape)), ROWS)

        norm("x", self.norms[0], "h")
        product("h", "qkv", "qkv")
        gain = np.concatenate([np.tile(self.gains[0], (HEADS, 1)), np.tile(self.gains[1], (KVH, 1))])
        heads = r["qkv"].reshape(ROWS, HEADS + 2 * KVH, HD)
        want, bound = so.norm_rope(heads[:, :HEADS + KVH], gain, np.float32(EPS), pos,
                                   po.rope_freqs(HD, 1e6, "plain"), HD, False, 1.0)
        close(r["q"].reshape(ROWS, HEADS, HD), want[:, :HEADS], bound[:, :HEADS])
        assert np.all(r["q"][live:] == 7.5)
        # the cache as the rows were written, then as kv_accept moved the path's; an f16
        # row is half a step off (2^-11 relative, 2^-25 absolute)
        k, v = s["k"].astype(np.float64), s["v"].astype(np.float64)
        slack = np.zeros(k.shape)
        k[slots[:live]], v[slots[:live]] = want[:live, HEADS:], heads[:live, HEADS + KVH:].astype(self.dt)
        slack[slots[:live]] = bound[:live, HEADS:]
        if self.dt == np.float16:
            slack[slots[:live]] += 2.0**-11 * (np.abs(want) + bound)[:live, HEADS:] + 2.0**-25
        path = r["tables"], PAGE, s["cached"], s["path"], s["path_len"]
        k, v = po.accept(k, v, *path)
        slack, _ = po.accept(slack, slack, *path)
        assert np.all(np.abs(r["k"].astype(np.float64) - k) <= slack)
        assert np.array_equal(r["v"].astype(np.float64), v)
        if s["path_len"][0] < 2:  # no row of the cache moved
            want, bound = po.attention(r["q"].reshape(ROWS, HEADS, HD), r["k"], r["v"], r["tables"], PAGE,
                                       s["cached"], first, s["mask"])
            close(r["att"].reshape(ROWS, HEADS, HD), want, bound)
        assert np.all(r["att"][live:] == 7.5)
        product("att", "o", "o")
        x1 = r["x"].astype(np.float64) + r["o"]
        close(r["x1"], x1, so.H * np.abs(x1), ROWS)
        norm("x1", self.norms[1], "h1")
        want, bound, ids, p = so.moe(r["h1"][:live], self.router, self.w["gate"], self.w["up"],
                                     self.w["down"], TOP, True, r["x1"][:live])
        close(r["y"], want, bound)
        assert np.array_equal(r["ids"][:live], ids)
        assert np.all(np.abs(r["weights"][:live] - p) <= 4 * so.H * p)
        assert np.all(r["y"][live:] == 7.5) and np.all(r["ids"][live:] == -7)
        norm("y", self.norms[2], "h2")
        product("h2", "head", "logits")
        for i in range(ROWS):
            if i >= live:
                assert r["token"][i] == 77 and r["logprob"][i] == 7.5 and np.all(r["out"][i] == 7.5)
                continue
            b = int(np.searchsorted(first[1:], i, side="right"))
            r0 = int(first[b])
            nodes = [s["node"][r0 + j] for j in range(int(s["fresh"][b])) if po.sees(s["mask"], i, i - r0, j)]
            m = s["allowed_row"][i]
            allowed = None if m < 0 else np.unpackbits(s["allowed"][m].view(np.uint8),
                                                       bitorder="little")[:VOCAB].astype(bool)
            l, bound = so.logits(r["logits"][i], s["tokens"][b, :s["length"][b]], int(s["prompt"][b]), nodes,
                                 *(a[b] for a in s["penalties"]), allowed=allowed)
            no = ~np.isfinite(l)
            assert np.array_equal(r["out"][i][no], l[no])
            assert np.all(np.abs(r["out"][i][~no] - l[~no]) <= 1.001 * bound[~no])
            so.check_top(l, 1.001 * bound, r["token"][i], r["logprob"][i])
        assert np.array_equal(r["cached_out"], s["cached"] + s["path_len"])


def same(a, b):
    for n in a:
        assert np.array_equal(a[n], b[n]), n


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_a_step_call_by_call(ctx, kv):
    m = Server(ctx, 3, kv)
    for seed in range(4):
        s = m.draw(seed)
        if seed % 2 == 0:
            s["path_len"][0] = 0
        m.upload(s)
        m.calls()
        m.check(s, m.results())


def test_a_recorded_step(ctx):
    """Replays as the requests change, another server's work on the same context
    between them."""
    m, other = Server(ctx, 4, "f16"), Server(ctx, 5, "f32")
    m.upload(m.draw(0))
    m.calls()
    ctx.graph_begin()
    m.calls()
    g = ctx.graph_end()
    for seed in range(5):
        s = m.draw(seed)
        m.upload(s)
        g.launch()
        replayed = m.results()
        m.upload(s)
        m.calls()
        same(replayed, m.results())
        m.check(s, replayed)
        o = other.draw(seed)
        other.upload(o)
        other.calls()
        other.check(o, other.results())
    g.close()


def test_steps_of_two_contexts_at_once(ctx):
    """Two host threads with a context each: the bits of one alone."""
    m = Server(ctx, 6, "f16")
    want = []
    for seed in range(3):
        m.upload(m.draw(seed))
        m.calls()
        want.append(m.results())
    wrong = []

    def work():
        c = cw.Context(0)
        try:
            o = Server(c, 6, "f16")
            for i in range(6):
                o.upload(o.draw(i % 3))
                o.calls()
                same(o.results(), want[i % 3])
        except BaseException as e:  # noqa: BLE001 (reported by the test's thread)
            wrong.append(repr(e))
        finally:
            c.close()

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
