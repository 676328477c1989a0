"""The operators of several requests in one paged cache on the MI355X, each
against its definition in 64 bits (paged_oracle), and a run of them together.

Tolerances, counted in f32 half steps (2^-24) before the first run:
  * rotation: the angle's rest is off by pi/4 half steps, each series by two
    more, the gain by two, a product and a sum by one each: 7 half steps of
    gain (|x_a| + |x_b|), and the f64 angle itself by position * 1e-15;
  * f16 cache rows: half an f16 step more (2^-11 relative, 2^-25 absolute);
  * attention: paged_oracle.attention's bound;
  * tables, moves: exact.
"""
import numpy as np
import pytest

import cw
import paged_oracle as po

pytestmark = pytest.mark.gpu

H = 2.0**-24
LAYOUT = {"halves": cw.ROPE_HALVES, "pairs": cw.ROPE_PAIRS}
SCALING = {"plain": cw.ROPE_PLAIN, "linear": cw.ROPE_LINEAR, "yarn": cw.ROPE_YARN,
           "bands": cw.ROPE_BANDS}
KV = {"f16": (cw.CW_F16, np.float16), "f32": (cw.CW_F32, np.float32)}


def at(d, floats):
    """The device array d from its element `floats` on."""
    return cw.DeviceArray(d.ctx, d.shape, d.dtype, d.ptr + 4 * floats)


def i32(a):
    return np.ascontiguousarray(a, np.int32)


# ------------------------------------------------------------------ rotation

ROPE = [
    # rows, heads, hd, rot, layout, scaling, factor, x stride - width, shift, far
    (1, 1, 2, 2, "halves", "plain", 1.0, 0, 0, 9),
    (3, 5, 128, 128, "halves", "plain", 1.0, 0, 0, 40000),
    (7, 3, 128, 64, "pairs", "yarn", 4.0, 12, 0, 131072),
    (5, 2, 64, 64, "pairs", "bands", 8.0, 0, 0, 100000),
    (4, 9, 256, 256, "halves", "linear", 2.5, 4, 0, 30000),
    (2, 3, 256, 2, "pairs", "plain", 1.0, 0, 0, 500),       # 255 units of a head, one by one
    (6, 7, 96, 24, "halves", "yarn", 16.0, 0, 0, 1 << 24),
    (3, 4, 80, 20, "halves", "bands", 3.0, 3, 0, 70000),    # odd strides: element by element
    (9, 2, 64, 32, "pairs", "linear", 4.0, 0, 1, 70000),    # an unaligned start
    (700, 40, 128, 128, "halves", "yarn", 4.0, 1024, 0, 131072),
    (2100, 32, 128, 96, "halves", "linear", 2.0, 0, 0, 9000),  # past 32 MB of rows
    (1100, 64, 128, 128, "pairs", "plain", 1.0, 4, 0, 9000),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", ROPE)
def test_rope_rows(ctx, rng, case, in_place):
    rows, heads, hd, rot, layout, scaling, factor, pad, shift, far = case
    width, stride = heads * hd, heads * hd + pad
    x = rng.standard_normal((rows, stride)).astype(np.float32)
    pos = i32(rng.integers(0, far, rows))
    pos[0] = far - 1
    if rows > 2:
        pos[1] = -1
    spec = cw.rope_spec(rot, 1e6, LAYOUT[layout], SCALING[scaling], factor, 8192)
    xd = ctx.empty(rows * stride + 8)
    xd.upload(np.concatenate([np.zeros(shift), x.ravel(), np.zeros(8 - shift)]))
    y_stride = stride if in_place else width + 5 * shift
    yd = xd if in_place else ctx.storage(np.full(rows * y_stride + 8, 7.5, np.float32))
    ctx.rope_rows(spec, at(xd, shift), ctx.storage(pos), rows, heads, hd, x_stride=stride,
                  y=at(yd, shift), y_stride=y_stride)
    got = yd.download()[shift:shift + rows * y_stride].reshape(rows, y_stride)
    x3 = x[:, :width].reshape(rows, heads, hd)
    gain = po.rope_gain(scaling, factor)
    ref = po.rotate(x3, pos, po.rope_freqs(rot, 1e6, scaling, factor), rot, layout == "pairs", gain)
    mag = po.rotate(np.abs(x3), np.zeros(rows), np.zeros(rot // 2), rot, layout == "pairs", 1.0)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if layout == "pairs" else (slice(0, rot // 2),
                                                                          slice(rot // 2, rot))
    tol = np.zeros_like(ref)
    tol[..., a] = tol[..., b] = gain * (mag[..., a] + mag[..., b]) * \
        (7 * H + np.maximum(pos, 0)[:, None, None] * 1e-15)
    live = pos >= 0
    d = np.abs(got[:, :width].reshape(rows, heads, hd) - ref)
    assert np.all(d[live] <= tol[live]), float((d[live] - tol[live]).max())
    # padding rows, and what lies between rows, as they were
    before = x if in_place else np.full((rows, y_stride), 7.5, np.float32)
    assert np.array_equal(got[~live], before[~live])
    assert np.array_equal(got[:, width:], before[:, width:])


def test_rope_rows_matches_rope(ctx, rng):
    """The plain half layout is cw_rope at one position (two roundings apart
    in the cosines, 3 half steps each, and a fused product)."""
    x = rng.standard_normal((6, 128)).astype(np.float32)
    xd = ctx.storage(x)
    for pos in (0, 1, 4095):
        y = ctx.rope_rows(cw.rope_spec(128, 1e6), xd, ctx.storage(i32([pos])), 1, 6, 128).download()
        z = ctx.rope(xd, 6, 128, pos, 1e6).download().reshape(y.shape)
        s = np.abs(x) + np.abs(np.roll(x, 64, 1))
        assert np.all(np.abs(y - z).reshape(6, 128) <= 10 * H * s)


def test_rope_gain(ctx, rng):
    """An explicit gain replaces the formula's: at position 0 x times it."""
    x = rng.standard_normal((2, 64)).astype(np.float32)
    spec = cw.rope_spec(64, 1e4, scaling=cw.ROPE_YARN, factor=8.0, trained=4096, gain=1.25)
    y = ctx.rope_rows(spec, ctx.storage(x), ctx.storage(i32([0, 0])), 2, 1, 64).download()
    assert np.array_equal(y, x * np.float32(1.25))


ROPE_KV = [
    # rows, heads, kv heads, hd, rot, layout, kv, page, blocks, stride - width, in place
    (1, 4, 2, 16, 16, "halves", "f16", 16, 1, 0, False),
    (5, 32, 8, 128, 128, "halves", "f16", 16, 3, 0, False),
    (9, 6, 2, 128, 64, "pairs", "f32", 32, 2, 8, True),
    (33, 3, 1, 64, 48, "halves", "f16", 64, 1, 0, True),
    (17, 5, 5, 256, 256, "pairs", "f16", 16, 4, 4, False),
    (12, 0, 3, 32, 16, "halves", "f32", 100, 1, 0, False),   # the cache alone, no page rule
    (21, 2, 1, 32, 6, "pairs", "f16", 16, 2, 1, False),      # element by element
    (600, 16, 8, 128, 128, "halves", "f16", 16, 40, 0, False),
]


@pytest.mark.parametrize("case", ROPE_KV)
def test_rope_kv_rows(ctx, rng, case):
    rows, heads, kvh, hd, rot, layout, kv, page, blocks, pad, in_place = case
    kv_type, dt = KV[kv]
    width, qw = (heads + 2 * kvh) * hd, heads * hd
    stride, slots_n = width + pad, page * blocks
    x = rng.standard_normal((rows, stride)).astype(np.float32)
    pos = i32(rng.integers(0, 50000, rows))
    slots = i32(rng.permutation(slots_n + rows)[:rows])  # some lie past the cache
    if rows > 4:
        pos[2], slots[3], slots[4] = -1, -1, slots_n
    kc, vc = (rng.standard_normal((slots_n, kvh * hd)).astype(dt) for _ in range(2))
    kd, vd, xd = ctx.storage(kc), ctx.storage(vc), ctx.storage(x)
    pages = cw.kv_pages(kd, vd, kv_type, kvh, hd, page, blocks)
    spec = cw.rope_spec(rot, 1e6, LAYOUT[layout], cw.ROPE_YARN, 4.0, 8192)
    qd = None if not heads else xd if in_place else \
        ctx.storage(np.full((rows, qw), 7.5, np.float32))
    ctx.rope_kv_rows(spec, pages, xd, ctx.storage(pos), ctx.storage(slots), rows, heads,
                     stride=stride, q_out=qd, q_stride=stride if in_place else None)
    gain, freqs = po.rope_gain("yarn", 4.0), po.rope_freqs(rot, 1e6, "yarn", 4.0)
    x3 = x[:, :width].reshape(rows, -1, hd)
    ref = po.rotate(x3, pos, freqs, rot, layout == "pairs", gain)
    p = np.abs(x3)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if layout == "pairs" else (slice(0, rot // 2),
                                                                          slice(rot // 2, rot))
    tol = np.zeros_like(ref)
    tol[..., a] = tol[..., b] = gain * (p[..., a] + p[..., b]) * 7 * H + 5e-11 * gain * p.max()
    live = pos >= 0
    if heads:
        q = qd.download()
        d = np.abs(q[:, :qw].reshape(rows, heads, hd) - ref[:, :heads])
        assert np.all(d[live] <= tol[live, :heads])
        assert np.array_equal(q[~live, :qw], (x if in_place else np.full_like(q, 7.5))[~live, :qw])
        if in_place:
            assert np.array_equal(q[:, qw:], x[:, qw:])
    want_k, want_v, tol_k = kc.astype(np.float64), vc.copy(), np.zeros(kc.shape)
    for r in range(rows):
        if live[r] and 0 <= slots[r] < slots_n:
            want_k[slots[r]] = ref[r, heads:heads + kvh].ravel()
            tol_k[slots[r]] = tol[r, heads:heads + kvh].ravel()
            if kv == "f16":
                tol_k[slots[r]] += np.abs(want_k[slots[r]]) * 2.0**-11 + 2.0**-25
            want_v[slots[r]] = x3[r, heads + kvh:].ravel().astype(dt)
    assert np.all(np.abs(kd.download().astype(np.float64) - want_k) <= tol_k)
    assert np.array_equal(vd.download(), want_v)


# -------------------------------------------------------------- block tables

def tables_state(rng, cached, fresh, page, max_blocks, spare_blocks):
    n = len(cached)
    held = i32(-(-cached // page))
    need = -(-(cached + np.maximum(fresh, 0)) // page)
    blocks = int(np.maximum(need, held).sum()) + spare_blocks
    ids = rng.permutation(blocks)
    tables = np.full((n, max_blocks), -1, np.int32)
    free = np.full(blocks, -1, np.int32)
    used = 0
    for b in range(n):
        tables[b, :held[b]] = ids[used:used + held[b]]
        used += held[b]
    free[:blocks - used] = ids[used:]
    return tables, held, free, blocks - used, blocks


def run_tables(ctx, cached, fresh, held, tables, free, n_free, page, blocks, rows, mask=None,
               alias=False):
    d = {n: ctx.storage(i32(a)) for n, a in
         dict(cached=cached, fresh=fresh, held=held, tables=tables, free=free,
              n_free=[n_free]).items()}
    n = len(cached)
    held_out = d["held"] if alias else ctx.empty(n, np.int32)
    nf_out = d["n_free"] if alias else ctx.empty(1, np.int32)
    first, status = ctx.empty(n + 1, np.int32), ctx.empty(1, np.int32)
    pos, slots = ctx.empty(rows, np.int32), ctx.empty(rows, np.int32)
    md = None if mask is None else ctx.storage(mask)
    batch = cw.batch(d["cached"], n, rows, first, d["tables"], tables.shape[1], md,
                     0 if mask is None else mask.shape[1])
    ctx.block_tables(cw.kv_pages(None, None, 0, 0, 0, page, blocks), batch, d["fresh"], d["held"],
                     held_out, d["free"], d["n_free"], nf_out, pos, slots, status)
    got = (int(status.download()[0]), d["tables"].download(), held_out.download(),
           d["free"].download(), int(nf_out.download()[0]), first.download(), pos.download(),
           slots.download())
    if not alias:
        assert np.array_equal(d["held"].download(), held)
        assert int(d["n_free"].download()[0]) == n_free
    return got


def same_step(got, want):
    for name, g, w in zip(("status", "tables", "held", "free", "n_free", "first_row", "positions",
                           "slots"), got, want):
        assert np.array_equal(g, w), (name, g, w)


TABLES = [
    # requests, longest cached, longest new, page, spare rows, with a tree's mask
    (1, 1, 1, 16, 0, False), (1, 40, 3000, 16, 0, False), (7, 60, 5, 16, 3, True),
    (48, 900, 1, 16, 100, False), (130, 300, 40, 32, 0, True), (1025, 90, 9, 64, 7, False),
    (3000, 40, 2, 16, 1, False), (5, 5000, 700, 256, 2000, False),
]


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("n,most,new,page,spare,tree", TABLES)
def test_block_tables(ctx, rng, n, most, new, page, spare, tree, alias):
    cached = rng.integers(0, most + 1, n)
    fresh = rng.integers(0, new + 1, n)
    fresh[rng.random(n) < 0.1] = -1
    fresh[0] = new
    rows = int(np.maximum(fresh, 0).sum()) + spare
    words = (new + 31) // 32
    mask = None
    if tree:
        mask = np.concatenate([po.tree(rng, max(0, int(f)), words) for f in fresh] +
                              [np.zeros((spare, words), np.uint32)])
        mask[1] = 0  # a row that sees nothing keeps the first new position
    width = int((-(-(cached + np.maximum(fresh, 0)) // page)).max()) + 1
    tables, held, free, n_free, blocks = tables_state(rng, cached, fresh, page, width, 3)
    args = (i32(cached), i32(fresh), held, tables, free, n_free, page, blocks, rows, mask)
    want = po.block_tables(*args)
    assert want[0] == 0
    same_step(run_tables(ctx, *args, alias=alias), want)


def test_block_tables_keep_blocks_of_rejected_drafts(ctx, rng):
    """A request that holds more blocks than it needs takes none and gives none."""
    cached, fresh = np.array([17, 5]), np.array([3, 60])
    tables, held, free, n_free, blocks = tables_state(rng, np.array([90, 5]), fresh, 16, 8, 4)
    args = (i32(cached), i32(fresh), held, tables, free, n_free, 16, blocks, 63)
    want = po.block_tables(*args)
    assert want[2][0] == 6 and want[0] == 0
    same_step(run_tables(ctx, *args), want)


@pytest.mark.parametrize("rows_cap", [90, 4000])  # one launch, and two
@pytest.mark.parametrize("what", ["free", "table", "rows", "rows_table_free", "cached", "held",
                                  "held_over", "n_free", "back", "length"])
def test_block_tables_failures_change_nothing(ctx, rng, what, rows_cap):
    cached, fresh = np.array([30, 64, 5, 17]), np.array([20, 1, 40, -1])
    rows, width = rows_cap, 5
    tables, held, free, n_free, blocks = tables_state(rng, cached, fresh, 16, width, 0)
    cached, fresh = i32(cached), i32(fresh)
    if what == "free":
        n_free -= 3
    elif what == "table":
        fresh[2], rows = 90, rows_cap + 60
        free = np.concatenate([free, np.full(9, -1, np.int32)])
        free[n_free:n_free + 9] = np.arange(blocks, blocks + 9)
        blocks, n_free = blocks + 9, n_free + 9
    elif what == "rows":
        rows = 60
    elif what == "rows_table_free":
        fresh[2] = rows + 100
    elif what == "cached":
        cached[1] = -1
    elif what == "held":
        held[3] = -2
    elif what == "held_over":
        held[0] = width + 1
    elif what == "n_free":
        n_free = -1
    elif what == "back":
        n_free = blocks - 1
    elif what == "length":
        cached[2] = 2**31 - 5
    args = (cached, fresh, held, tables, free, n_free, 16, blocks, rows)
    want = po.block_tables(*args)
    assert want[0] == {"free": 8, "table": 4, "rows": 2, "rows_table_free": 14}.get(what, 1)
    same_step(run_tables(ctx, *args), want)


def test_block_tables_entries_that_are_no_block(ctx, rng):
    cached, fresh = np.array([40, 20]), np.array([4, 4])
    tables, held, free, n_free, blocks = tables_state(rng, cached, fresh, 16, 4, 2)
    tables[0, 2], tables[1, 1] = blocks, -7
    args = (i32(cached), i32(fresh), held, tables, free, n_free, 16, blocks, 8)
    want = po.block_tables(*args)
    assert want[0] == 0 and np.all(want[7][:8] == -1)
    same_step(run_tables(ctx, *args), want)


# ----------------------------------------------------------------- attention

class Batch:
    """A batch on the device: request b has cached[b] positions and new[b]
    nodes; every cache row that no request holds is NaN, and so are K and V of
    nodes that no row sees."""

    def __init__(self, ctx, rng, cached, new, heads, kvh, hd, kv, page, tree=False, contig=False,
                 spare_rows=0, mask=None, q_scale=1.0, v_scale=1.0):
        kv_type, dt = KV[kv]
        self.cached, self.new = i32(cached), i32(new)
        self.first = i32(np.concatenate([[0], np.cumsum(new)]))
        n, rows = len(cached), int(self.first[-1]) + spare_rows
        total = self.cached + self.new
        if contig:
            page, blocks = int(total.max()) + 3, n + 1
            self.tables, width = None, 0
        else:
            held = -(-total // page)
            blocks, width = int(held.sum()) + 2, int(held.max()) + 1
            ids = rng.permutation(blocks)
            self.tables = np.full((n, width), -1, np.int32)
            for b in range(n):
                self.tables[b, :held[b]] = ids[held[:b].sum():held[:b + 1].sum()]
        self.page, self.blocks, self.rows = page, blocks, rows
        k, v = (np.full((blocks * page, kvh, hd), np.nan, dt) for _ in range(2))
        for b in range(n):
            at_ = [po.slot_of(self.tables, page, b, p) for p in range(int(total[b]))]
            k[at_] = rng.standard_normal((len(at_), kvh, hd)).astype(dt)
            v[at_] = (v_scale * rng.standard_normal((len(at_), kvh, hd))).astype(dt)
        self.mask = mask
        if tree and mask is None:
            words = (max(1, int(self.new.max())) + 31) // 32
            self.mask = np.concatenate([po.tree(rng, int(m), words) for m in new] +
                                       [np.zeros((spare_rows, words), np.uint32)])
        self.k, self.v = k, v
        self.q = (q_scale * rng.standard_normal((rows, heads, hd))).astype(np.float32)
        self.dims = heads, kvh, hd, kv_type
        self.ctx = ctx

    def run(self, q_pad=0, out_pad=0):
        ctx, (heads, kvh, hd, kv_type) = self.ctx, self.dims
        w = heads * hd
        qb = np.full((self.rows, w + q_pad), np.nan, np.float32)
        qb[:, :w] = self.q.reshape(self.rows, w)
        kd, vd = ctx.storage(self.k), ctx.storage(self.v)
        out = ctx.storage(np.full((self.rows, w + out_pad), 7.5, np.float32))
        self.dev = cw.batch(ctx.storage(self.cached), len(self.cached), self.rows,
                            ctx.storage(self.first),
                            None if self.tables is None else ctx.storage(self.tables),
                            0 if self.tables is None else self.tables.shape[1],
                            None if self.mask is None else ctx.storage(self.mask),
                            0 if self.mask is None else self.mask.shape[1])
        self.pages = cw.kv_pages(kd, vd, kv_type, kvh, hd, self.page, self.blocks)
        self.qd, self.outd = ctx.storage(qb), out
        ctx.attention_tree(self.pages, self.dev, self.qd, heads, q_stride=w + q_pad, out=out,
                           out_stride=w + out_pad)
        got = out.download()
        live = int(self.first[-1])
        assert np.all(got[live:] == 7.5) and np.all(got[:, w:] == 7.5)
        return got[:live, :w].reshape(live, heads, hd)

    def check(self, got):
        ref, bound = po.attention(self.q, self.k, self.v, self.tables, self.page, self.cached,
                                  self.first, self.mask)
        live = int(self.first[-1])
        d = np.abs(got - ref[:live])
        worst = np.unravel_index(np.argmax(d - bound[:live]), d.shape)
        assert np.all(d <= bound[:live]), (worst, got[worst], ref[worst], bound[worst[0], worst[1]])


SHAPES = [
    # cached, new, heads, kv heads, hd, page
    ([0], [1], 1, 1, 128, 16), ([1], [1], 4, 1, 128, 16), ([15, 16, 17], [1, 1, 1], 8, 2, 128, 16),
    ([300], [61], 8, 2, 128, 16), ([63, 0, 130, 500], [5, 33, 1, 70], 4, 1, 128, 32),
    ([200, 64, 7], [16, 4, 9], 7, 1, 128, 64), ([90, 0, 31], [3, 0, 40], 6, 3, 64, 16),
    ([257], [130], 2, 2, 64, 256), ([33, 120], [20, 1], 4, 2, 256, 16),
    ([0, 70], [65, 2], 5, 5, 256, 32), ([18, 3, 200], [7, 1, 30], 4, 2, 16, 16),
    ([50, 129], [33, 2], 3, 1, 32, 64), ([1000, 1, 400, 0, 64], [1, 1, 1, 1, 1], 32, 8, 128, 64),
    # more tiles than workgroups: runs over several requests and heads
    ([1300, 700, 0, 999, 64, 411, 1280, 850, 37, 600], [1, 3, 2, 1, 5, 4, 1, 2, 3, 1], 16, 8, 128,
     32),
    ([500, 800, 300, 1000, 64, 640], [7, 6, 8, 7, 5, 9], 32, 8, 128, 64),
    ([900, 1300, 250, 700, 1100, 30], [20, 9, 33, 14, 25, 40], 16, 8, 128, 16),
    ([1500, 800], [61, 40], 32, 8, 128, 16), ([2000, 1500], [40, 9], 8, 8, 64, 32),
    ([1000, 1200, 500], [6, 2, 9], 16, 8, 256, 16),
]


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_tree(ctx, rng, shape, tree, kv):
    cached, new, heads, kvh, hd, page = shape
    b = Batch(ctx, rng, cached, new, heads, kvh, hd, kv, page, tree=tree, spare_rows=3)
    b.check(b.run())


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
def test_attention_without_tables_and_with_strides(ctx, rng, hd, kv):
    b = Batch(ctx, rng, [70, 0, 33], [9, 20, 1], 4, 2, hd, kv, 0, tree=True, contig=True)
    b.check(b.run(q_pad=8, out_pad=4))


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_attention_masked_values_stay_out(ctx, rng, hd, kv):
    """Rows that see nothing give zeros; NaN and infinities in the K and V of
    nodes reach only the rows that see them."""
    n = 40
    mask = np.concatenate([po.tree(rng, n, 2), po.tree(rng, n, 2)])
    mask[[3, n + 5]] = 0
    mask[:, 0] &= ~np.uint32(1 << 7 | 1 << 20)   # nodes 7 and 20 are seen by row 30 alone
    mask[[30, n + 30], 0] |= np.uint32(1 << 7 | 1 << 20)
    b = Batch(ctx, rng, [0, 45], [n, n], 4, 2, hd, kv, 16, mask=mask)
    for s in range(2):
        c = int(b.cached[s])
        for node, (kk, vv) in {7: (np.nan, np.inf), 20: (np.inf, np.nan)}.items():
            at_ = po.slot_of(b.tables, 16, s, c + node)
            b.k[at_], b.v[at_] = kk, vv
    got = b.run()
    assert np.all(got[3] == 0)  # request 0 has nothing cached
    assert np.all(np.isnan(got[[30, n + 30]]))
    keep = np.setdiff1d(np.arange(2 * n), [30, n + 30])
    ref, bound = po.attention(b.q, np.nan_to_num(b.k, posinf=0), np.nan_to_num(b.v, posinf=0),
                              b.tables, 16, b.cached, b.first, mask)
    assert np.all(np.abs(got - ref)[keep] <= bound[keep])


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("nodes", [[7, 20], range(24, 40), [39]])
@pytest.mark.parametrize("what", ["k", "v", "both"])
def test_attention_large_values_stay_out(ctx, rng, what, nodes, hd, kv):
    """Nodes of huge K or V cost the rows that do not see them no bits."""
    n = 40
    mask = np.concatenate([po.tree(rng, n, 2), po.tree(rng, n, 2)])
    bits = np.zeros(2, np.uint32)
    for i in nodes:
        bits[i // 32] |= np.uint32(1 << i % 32)
    mask &= ~bits
    mask[[30, n + 30]] |= bits
    b = Batch(ctx, rng, [0, 45], [n, n], 4, 2, hd, kv, 16, mask=mask)
    huge = {"f16": 3e4, "f32": 3e37}[kv]
    k, v = b.k.copy(), b.v.copy()
    for s in range(2):
        for i in nodes:
            at_ = po.slot_of(b.tables, 16, s, int(b.cached[s]) + i)
            if what != "v":
                b.k[at_] = (huge * rng.uniform(-1, 1, b.k[at_].shape)).astype(b.k.dtype)
            if what != "k":
                b.v[at_] = huge
    got = b.run()
    keep = np.setdiff1d(np.arange(2 * n), [30, n + 30])
    ref, bound = po.attention(b.q, k, v, b.tables, 16, b.cached, b.first, mask)
    assert np.all(np.abs(got - ref)[keep] <= bound[keep])


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_attention_infinite_values_of_seen_nodes(ctx, rng, kv):
    """A seen V of +inf gives +inf in its element, and nothing else changes."""
    b = Batch(ctx, rng, [20], [9], 2, 1, 128, kv, 16)
    at_ = po.slot_of(b.tables, 16, 0, 20 + 4)
    b.v[at_, 0, 17] = np.inf
    got = b.run()
    ref, bound = po.attention(b.q, b.k, np.nan_to_num(b.v, posinf=0), b.tables, 16, b.cached,
                              b.first, None)
    assert np.all(np.isposinf(got[4:, :, 17]))
    got[4:, :, 17] = ref[4:, :, 17]
    assert np.all(np.abs(got - ref) <= bound)


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("q_scale,v_scale", [(1e-6, 1.0), (300.0, 1.0), (3e5, 1e-3), (1e-30, 300.0)])
def test_attention_magnitudes(ctx, rng, q_scale, v_scale, kv):
    """Queries far from one: scores of any size, a softmax down to one key."""
    b = Batch(ctx, rng, [150, 4], [12, 3], 4, 2, 128, kv, 16, tree=True, q_scale=q_scale,
              v_scale=v_scale)
    b.check(b.run())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e-30, 1e-30, 1.0), (1.0, 0.0, 0.0), (1e18, 1e-19, 1e30),
                                                     (1e-12, 1e12, 1e-30)])
def test_attention_magnitudes_of_many_rows(ctx, rng, q_scale, k_scale, v_scale, hd):
    """Queries and an f32 cache far from one, more rows than 16."""
    b = Batch(ctx, rng, [150, 0], [40, 33], 4, 2, hd, "f32", 16, tree=True, q_scale=q_scale)
    b.k, b.v = b.k * np.float32(k_scale), b.v * np.float32(v_scale)
    b.check(b.run())


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_attention_bad_requests(ctx, rng, hd, kv):
    """A request with a block that is not in the cache gives NaN; one whose
    rows or lengths are out of range has no rows; the others are right."""
    b = Batch(ctx, rng, [40, 100, 20, 30], [3, 2, 4, 5], 4, 2, hd, kv, 16)
    got = b.run()
    b.check(got)
    good = got.copy()
    b.tables[1, 2] = b.blocks
    b.cached[2] = -1
    heads = b.dims[0]
    out = ctx.storage(np.full((b.rows, heads * hd), 7.5, np.float32))
    b.dev = cw.batch(ctx.storage(b.cached), 4, b.rows, ctx.storage(b.first),
                     ctx.storage(b.tables), b.tables.shape[1])
    ctx.attention_tree(b.pages, b.dev, b.qd, heads, out=out)
    got = out.download().reshape(good.shape)
    assert np.all(np.isnan(got[3:5]))
    assert np.all(got[5:9] == 7.5)
    assert np.array_equal(got[:3], good[:3]) and np.array_equal(got[9:], good[9:])
    # a length past the table's end, a row range past the rows
    b.cached[2], b.cached[1] = 20, 16 * b.tables.shape[1] - 1
    first = b.first.copy()
    first[4] = b.rows + 1
    b.dev = cw.batch(ctx.storage(b.cached), 4, b.rows, ctx.storage(first), ctx.storage(b.tables),
                     b.tables.shape[1])
    out = ctx.storage(np.full((b.rows, heads * hd), 7.5, np.float32))
    ctx.attention_tree(b.pages, b.dev, b.qd, heads, out=out)
    got = out.download().reshape(good.shape)
    assert np.all(np.isnan(got[3:5])) and np.all(got[9:] == 7.5)
    assert np.array_equal(got[5:9], good[5:9]) and np.array_equal(got[:3], good[:3])


def test_attention_same_bits_again(ctx, rng):
    b = Batch(ctx, rng, [700, 90, 0], [30, 7, 50], 8, 2, 128, "f16", 16, tree=True)
    first = b.run()
    for _ in range(3):
        assert np.array_equal(b.run(), first)


def test_attention_matches_the_single_query_one(ctx, rng):
    """One row of a request without drafts is cw_attention over its positions
    (either within the bound of the other's oracle)."""
    b = Batch(ctx, rng, [513], [1], 32, 8, 128, "f16", 16, contig=True)
    got = b.run()
    o = ctx.attention(ctx.storage(b.q[0].ravel()), ctx.storage(b.k[:514]), ctx.storage(b.v[:514]),
                      cw.CW_F16, 32, 8, 514, 128).download()
    _, bound = po.attention(b.q, b.k, b.v, None, b.page, b.cached, b.first)
    assert np.all(np.abs(got[0] - o.reshape(32, 128)) <= 2 * bound[0])


# ------------------------------------------------------------ accepted rows

@pytest.mark.parametrize("kv,kvh,hd,page,contig", [
    ("f16", 8, 128, 16, False), ("f32", 3, 64, 32, False), ("f16", 1, 16, 16, True),
    ("f32", 8, 256, 16, False)])
def test_kv_accept(ctx, rng, kv, kvh, hd, page, contig):
    n, nodes, most = 9, 50, 13
    cached, new = rng.integers(0, 200, n), np.full(n, nodes)
    b = Batch(ctx, rng, cached, new, kvh, kvh, hd, kv, page, contig=contig)
    path = i32(np.sort(np.argsort(rng.random((n, nodes)), axis=1)[:, :most], axis=1))
    path[0] = np.arange(most)           # nothing moves
    path[1] = np.arange(1, most + 1)    # every row moves onto the one before it
    count = i32(rng.integers(0, most + 1, n))
    count[:4] = most, most, 0, 1
    kd, vd = ctx.storage(b.k), ctx.storage(b.v)
    out = ctx.empty(n, np.int32)
    pages = cw.kv_pages(kd, vd, KV[kv][0], kvh, hd, b.page, b.blocks)
    batch = cw.batch(ctx.storage(b.cached), n, 1, None,
                     None if contig else ctx.storage(b.tables), 0 if contig else b.tables.shape[1])
    ctx.kv_accept(pages, batch, ctx.storage(path), most, ctx.storage(count), out)
    k, v = po.accept(b.k, b.v, b.tables, b.page, b.cached, path, count)
    assert kd.download().tobytes() == k.tobytes() and vd.download().tobytes() == v.tobytes()
    assert np.array_equal(out.download(), b.cached + count)


def test_kv_accept_leaves_out_what_is_not_there(ctx, rng):
    b = Batch(ctx, rng, [20, 20], [12, 12], 2, 2, 64, "f16", 16)
    b.tables[0, 1] = b.blocks  # request 0's nodes have no block
    kd, vd = ctx.storage(b.k), ctx.storage(b.v)
    pages = cw.kv_pages(kd, vd, cw.CW_F16, 2, 64, 16, b.blocks)
    batch = cw.batch(ctx.storage(b.cached), 2, 1, None, ctx.storage(b.tables), b.tables.shape[1])
    path, count = i32([[1, 2, 3], [-1, 5, 1 << 30]]), i32([3, 9])
    ctx.kv_accept(pages, batch, ctx.storage(path), 3, ctx.storage(count))
    k, v = b.k.copy(), b.v.copy()
    src, dst = (po.slot_of(b.tables, 16, 1, 20 + p) for p in (5, 1))
    k[dst], v[dst] = k[src], v[src]
    assert kd.download().tobytes() == k.tobytes() and vd.download().tobytes() == v.tobytes()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_a_step_with_drafts(ctx, rng, kv):
    """Tables, rotation with the cache write, tree attention and the accepted
    path, recorded once and replayed for three steps of two requests; after
    them each request's attention is cw_attention's over a cache written row
    by row (cw_rope, cw_kv_write)."""
    kv_type, dt = KV[kv]
    heads, kvh, hd, page, blocks, width, rows, words = 4, 2, 64, 16, 20, 8, 24, 1
    qw, total = heads * hd, (heads + 2 * kvh) * hd
    new = i32([7, 12])
    n = 2
    mask = np.zeros((rows, words), np.uint32)
    mask[:7], mask[7:19] = po.tree(rng, 7, 1), po.tree(rng, 12, 1)
    paths = []
    for s, r0 in ((0, 0), (1, 7)):  # the last node's ancestors and itself
        bits = int(mask[r0 + new[s] - 1, 0])
        paths.append([j for j in range(12) if bits >> j & 1])
    most = max(map(len, paths))
    path = i32([p + [0] * (most - len(p)) for p in paths])
    count = i32([len(p) for p in paths])

    kd, vd = (ctx.storage(np.full((blocks * page, kvh * hd), np.nan, dt)) for _ in range(2))
    pages = cw.kv_pages(kd, vd, kv_type, kvh, hd, page, blocks)
    z = lambda shape, t=np.int32: ctx.storage(np.zeros(shape, t))  # noqa: E731
    cached, cached_out, held, n_free = z(n), z(n), z(n), ctx.storage(i32([blocks]))
    first, tables, status = z(n + 1), z((n, width)), z(1)
    pos, slots, free = z(rows), z(rows), ctx.storage(i32(rng.permutation(blocks)))
    batch = cw.batch(cached, n, rows, first, tables, width, ctx.storage(mask), words)
    fresh, qkv = ctx.storage(new), z((rows, total), np.float32)
    q, out = z((rows, qw), np.float32), z((rows, qw), np.float32)
    pd, cd = ctx.storage(path), ctx.storage(count)
    spec = cw.rope_spec(hd, 1e6, scaling=cw.ROPE_PLAIN)

    def step():
        ctx.block_tables(pages, batch, fresh, held, held, free, n_free, n_free, pos, slots, status)
        ctx.rope_kv_rows(spec, pages, qkv, pos, slots, rows, heads, q_out=q)
        ctx.attention_tree(pages, batch, q, heads, out=out)
        ctx.kv_accept(pages, batch, pd, most, cd, cached_out)

    step()  # once before recording: scratch and the table of frequencies
    ctx.flush()
    for d, a in ((cached, np.zeros(n)), (held, np.zeros(n)), (n_free, [blocks])):
        d.upload(i32(a))
    ctx.graph_begin()
    step()
    g = ctx.graph_end()
    chains = [([], []) for _ in range(n)]  # accepted (k, v) rows of each request, row by row
    lengths = np.zeros(n, np.int64)
    for _ in range(3):
        x = rng.standard_normal((rows, total)).astype(np.float32)
        qkv.upload(x)
        g.launch()
        got, positions = out.download(), pos.download()
        assert status.download()[0] == 0
        for s, r0 in ((0, 0), (1, 7)):
            kc, vc = ctx.empty((width * page, kvh * hd), dt), ctx.empty((width * page, kvh * hd), dt)

            def put(p, kr, vr):
                ctx.kv_write(kc, vc, kv_type, p, kvh * hd, kr, vr)
            for p, (kr, vr) in enumerate(zip(*chains[s])):
                put(p, kr, vr)
            rotated = {}
            for j in paths[s]:
                r, p = r0 + j, int(lengths[s]) + paths[s].index(j)
                assert positions[r] == p
                kr = ctx.rope(ctx.storage(x[r, qw:qw + kvh * hd]), kvh, hd, p, 1e6)
                rotated[j] = kr, ctx.storage(x[r, qw + kvh * hd:])
                put(p, *rotated[j])
            # the path's last node sees exactly the path: one single-query call
            r, p = r0 + paths[s][-1], int(lengths[s]) + len(paths[s]) - 1
            qr = ctx.rope(ctx.storage(x[r, :qw]), heads, hd, p, 1e6)
            want = ctx.attention(qr, kc, vc, kv_type, heads, kvh, p + 1, hd).download()
            # K's rounding to the cache's type may fall on either side of a tie:
            # half a step of it on a few elements, else f32 sums
            assert np.max(np.abs(got[r] - want)) <= (2e-3 if kv == "f16" else 2e-5)
            chains[s][0].extend(rotated[j][0] for j in paths[s])
            chains[s][1].extend(rotated[j][1] for j in paths[s])
        lengths += count
        assert np.array_equal(cached_out.download(), lengths)
        cached.upload(i32(lengths))
    g.close()
