"""Values, masks and lengths at the edges of what the paged operators accept,
on the MI355X: each against its definition in 64 bits, with the bounds of
test_gpu_paged."""
import ctypes as C

import numpy as np
import pytest

import cw
import paged_oracle as po
import test_gpu_paged as tp
import test_gpu_paged_serving as ts
from test_gpu_paged import Batch, i32, run_tables, same_step, tables_state

pytestmark = pytest.mark.gpu

# kv, heads, kv heads, hd, new rows of the first of two requests (the second
# has two): few and many rows of a kv head, every head size
KERNELS = [
    ("f16", 2, 1, 64, 3), ("f16", 2, 1, 128, 3), ("f16", 8, 1, 128, 12), ("f16", 8, 1, 128, 90),
    ("f16", 2, 1, 256, 3), ("f16", 8, 1, 256, 90), ("f16", 2, 1, 32, 3), ("f16", 8, 1, 32, 90),
    ("f32", 2, 1, 64, 3), ("f32", 2, 1, 128, 3), ("f32", 8, 1, 64, 12), ("f32", 8, 1, 64, 90),
    ("f32", 8, 1, 128, 12), ("f32", 8, 1, 128, 90), ("f32", 2, 1, 32, 3), ("f32", 8, 1, 32, 90),
    ("f32", 2, 1, 256, 3), ("f32", 8, 1, 256, 90), ("f16", 2, 1, 16, 3), ("f16", 8, 1, 16, 90),
    ("f32", 2, 1, 16, 3), ("f32", 8, 1, 16, 90),
]


def free_block_0(b):
    """Block 0 is nobody's and holds NaN: its owner takes an unused one."""
    spare = int(np.setdiff1d(np.arange(b.blocks), b.tables)[-1])
    if spare == 0:
        return
    b.tables[b.tables == 0] = spare
    for a in (b.k, b.v):
        a[spare * b.page:(spare + 1) * b.page] = a[:b.page]
        a[:b.page] = np.nan


# ------------------------------------------------------- blocks that are missing

# (behind_inf: few rows are one row block, behind whose last tile nothing lies)
@pytest.mark.parametrize("case,what", [
    (c, w) for c in KERNELS for w in ("node", "cached", "cached_inf", "cached_far", "tile_inf",
                                      "behind_inf")[:None if c[4] == 90 else -1]])
def test_a_lost_block_is_nan_whatever_the_values(ctx, rng, case, what):
    """NaN for every row of a request with a block that is not there: also
    where block 0 holds NaN, a node's V is infinite (far from the block, in
    its tile, or before it), or a node is far from its neighbours."""
    kv, heads, kvh, hd, new = case
    cached = 100 if what == "tile_inf" else 70
    b = Batch(ctx, rng, [cached, 40], [new, 2], heads, kvh, hd, kv, 16)
    free_block_0(b)
    if what == "tile_inf":
        b.k[:16] = b.v[:16] = 1
    good = b.run()
    b.check(good)
    node = po.slot_of(b.tables, 16, 0, cached + 1)
    if what.endswith("inf"):
        b.v[node] = np.inf
    if what.endswith("far"):
        b.k[node], b.v[node] = b.k[node] * b.k.dtype.type(1e-4), 0
        b.v[node, 0, 3] = 1e-7
    entry = {"n": 4, "c": 1, "b": 9, "t": 4}[what[0]]  # positions 64 .., 16 .., 144 ..
    b.tables[0, entry] = -1 if hd != 64 else b.blocks
    got = b.run()
    assert np.all(np.isnan(got[:new])), np.argwhere(~np.isnan(got[:new]))[:3]
    assert np.array_equal(got[new:], good[new:])


# ------------------------------------------------------------------------ masks

@pytest.mark.parametrize("rows_cap", [0, 4000])  # one launch, and two
def test_block_tables_masks_of_more_bits_than_nodes(ctx, rng, rows_cap):
    """A row's position counts the nodes it sees of its request; bits behind
    the request's last node are no nodes."""
    fresh = np.array([5, 33, 1, 64, 0, -1, 31, 32, 70, 2])
    cached = rng.integers(0, 90, len(fresh))
    words = 3
    mask = np.concatenate([po.tree(rng, max(0, int(f)), words) for f in fresh])
    mask[4] = 0  # a row that sees nothing keeps the first new position
    wide, r = mask.copy(), 0
    for f in np.maximum(fresh, 0):
        for w in range(words):
            wide[r:r + f, w] |= np.uint32(0xffffffff << min(max(f - 32 * w, 0), 32) & 0xffffffff)
        r += f
    rows = max(r, rows_cap)
    mask, wide = (np.pad(m, ((0, rows - r), (0, 0))) for m in (mask, wide))
    width = int((-(-(cached + np.maximum(fresh, 0)) // 16)).max()) + 1
    tables, held, free, n_free, blocks = tables_state(rng, cached, fresh, 16, width, 3)
    args = (i32(cached), i32(fresh), held, tables, free, n_free, 16, blocks, rows)
    want = po.block_tables(*args, mask)
    assert want[0] == 0
    same_step(run_tables(ctx, *args, wide), want)


@pytest.mark.parametrize("case", KERNELS)
def test_attention_masks_of_more_bits_than_nodes(ctx, rng, case):
    """Bits behind a request's last node show nothing."""
    kv, heads, kvh, hd, new = case
    b = Batch(ctx, rng, [70, 40], [new, 2], heads, kvh, hd, kv, 16, tree=True)
    first = b.run()
    b.check(first)
    for r in range(new + 2):
        n = new if r < new else 2
        for w in range(b.mask.shape[1]):
            b.mask[r, w] |= np.uint32(0xffffffff << min(max(n - 32 * w, 0), 32) & 0xffffffff)
    assert np.array_equal(b.run(), first)


# ------------------------------------------------------------- the largest values

@pytest.mark.parametrize("hidden", [False, True])
@pytest.mark.parametrize("cached", [[150, 0], [0, 3100], [2047, 2046]])
@pytest.mark.parametrize("case", KERNELS)
def test_attention_of_the_largest_values(ctx, rng, case, cached, hidden):
    """V up to the type's largest: sums of many such values are past it, their
    mean is not.  hidden: beside a node of NaN that no row sees."""
    kv, heads, kvh, hd, new = case
    b = Batch(ctx, rng, cached, [new, 2], heads, kvh, hd, kv, 16, tree=hidden, q_scale=0.1)
    most = float(np.finfo(b.v.dtype).max) * 0.98
    held = ~np.isnan(b.v[:, 0, 0].astype(np.float32))
    b.v[held] = (most * rng.uniform(0.5, 1.0, b.v[held].shape)).astype(b.v.dtype)
    b.v[held, :, 1::2] *= -1
    if hidden:
        b.mask[:new, 0] &= ~np.uint32(1 << 1)
        at_ = po.slot_of(b.tables, 16, 0, int(b.cached[0]) + 1)
        b.k[at_] = b.v[at_] = np.nan
    b.check(b.run())


@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("case", [c for c in KERNELS if c[0] == "f32"])
def test_attention_of_cached_values_far_apart(ctx, rng, case, what):
    """Cached positions far below the ones beside them, which every row sees:
    the error counts from the largest."""
    kv, heads, kvh, hd, new = case
    b = Batch(ctx, rng, [333, 40], [new, 2], heads, kvh, hd, kv, 16, tree=True)
    for s in range(2):
        for p in range(int(b.cached[s])):
            f = np.float32(2.0 ** -int(rng.integers(0, 45)))
            at_ = po.slot_of(b.tables, 16, s, p)
            if what != "v":
                b.k[at_] *= f
            if what != "k":
                b.v[at_] *= f
    b.check(b.run())


# -------------------------------------------------------------------- row ranges

@pytest.mark.parametrize("case", KERNELS)
def test_a_bad_row_range_among_good_ones(ctx, rng, case):
    """A request whose rows lie behind the last has none, and neither has the
    one that would begin there; the others, before and behind, are right."""
    kv, heads, kvh, hd, new = case
    b = Batch(ctx, rng, [70, 40, 9, 33, 20], [new, 2, 4, 1, 5], heads, kvh, hd, kv, 16)
    good = b.run()
    b.check(good)
    first, heads = b.first.copy(), b.dims[0]
    first[2] = b.rows + 9
    b.dev = cw.batch(ctx.storage(b.cached), 5, b.rows, ctx.storage(first), ctx.storage(b.tables),
                     b.tables.shape[1])
    out = ctx.storage(np.full((b.rows, heads * hd), 7.5, np.float32))
    ctx.attention_tree(b.pages, b.dev, b.qd, heads, out=out)
    got = out.download().reshape(good.shape)
    assert np.all(got[new:new + 6] == 7.5)
    got[new:new + 6] = good[new:new + 6]
    b.check(got)


# ------------------------------------------------------------------ long requests

def test_kv_accept_past_a_billion_positions(rng):
    """Moves at positions past 2^30, which a request without tables can have."""
    page, hd = (1 << 30) + 4096, 16
    with cw.Context(0) as c:
        kd, vd = (c.empty((page, hd), np.float16) for _ in range(2))
        pages = cw.kv_pages(kd, vd, cw.CW_F16, 1, hd, page, 1)
        cached = (1 << 30) + 1000
        new = rng.standard_normal((2, 40, hd)).astype(np.float16)
        views = [cw.DeviceArray(c, (40, hd), np.float16, d.ptr + cached * hd * 2) for d in (kd, vd)]
        for d, a in zip(views, new):
            d.upload(a)
        path, out = [0, 3, 4, 17, 39], c.empty(1, np.int32)
        batch = cw.batch(c.storage(i32([cached])), 1, 1, None, None, 0)
        c.kv_accept(pages, batch, c.storage(i32([path])), 5, c.storage(i32([5])), out)
        for d, a in zip(views, new):
            want = a.copy()
            want[:5] = a[path]
            assert d.download().tobytes() == want.tobytes()
        assert out.download()[0] == cached + 5


# ------------------------------------------------------------------- head_dim 16

@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("check", [
    lambda *a: tp.test_attention_masked_values_stay_out(*a[:2], 16, a[2]),
    lambda *a: tp.test_attention_bad_requests(*a[:2], 16, a[2]),
    lambda *a: ts.test_attention_of_many_requests(*a[:2], 16, False, 4, a[2]),
    lambda *a: ts.test_attention_of_many_requests(*a[:2], 16, True, 4, a[2]),
    lambda *a: ts.test_attention_of_prompts(*a[:2], 7, 1, 16, a[2]),
    lambda *a: ts.test_a_lost_block_behind_the_first_rows(*a[:2], 1, 16, a[2]),
    lambda *a: ts.test_a_lost_block_behind_the_first_rows(*a[:2], 8, 16, a[2]),
    lambda *a: ts.test_a_length_behind_the_cache(*a[:2], 1, 16, False, a[2]),
    lambda *a: ts.test_a_length_behind_the_cache(*a[:2], 8, 16, True, a[2]),
], ids=["masked", "bad_requests", "many", "many_contig", "prompts", "lost_few", "lost_many",
        "length_few", "length_many"])
def test_head_dim_16(ctx, rng, check, kv):
    """What the other head sizes are held to, over few (row, head)s and many."""
    check(ctx, rng, kv)


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,cached,new,tree", [
    (8, 2, [300, 0, 17, 1000], [40, 30, 1, 9], True), (5, 5, [0, 63, 64], [1, 200, 0], False),
    (16, 1, [2500, 5], [33, 2], True)])
def test_head_dim_16_of_many_rows(ctx, rng, heads, kvh, cached, new, tree, kv):
    b = Batch(ctx, rng, cached, new, heads, kvh, 16, kv, 16, tree=tree, spare_rows=4)
    b.check(b.run(q_pad=4, out_pad=8))


# ----------------------------------------------------------- many specifications

def test_frequencies_of_many_specifications(ctx, rng):
    """A base that changes every step: each call is rotated by its own, a
    recording keeps its table, and the device's memory does not fill up."""
    rows, heads, hd = 5, 3, 64
    x = rng.standard_normal((rows, heads * hd)).astype(np.float32)
    pos = i32([0, 7, 900, 40000, 131071])
    xd, pd, y = ctx.storage(x), ctx.storage(pos), ctx.empty((rows, heads * hd))
    x3 = x.reshape(rows, heads, hd)
    pair = np.abs(x3) + np.abs(np.roll(x3, hd // 2, -1))
    tol = pair * (7 * tp.H + pos[:, None, None] * 1e-15)

    def check(theta):
        ref = po.rotate(x3, pos, po.rope_freqs(hd, theta, "plain"), hd, False, 1.0)
        assert np.all(np.abs(y.download().reshape(ref.shape) - ref) <= tol), theta

    def rotate(theta):
        ctx.rope_rows(cw.rope_spec(hd, theta), xd, pd, rows, heads, hd, y=y)

    rotate(3e5)
    ctx.graph_begin()
    rotate(3e5)
    g = ctx.graph_end()
    for i in range(150):
        rotate(1e4 + i)
        if i % 3 == 0:  # (else several are queued behind one another)
            check(1e4 + i)
        if i % 50 == 0:
            g.launch()
            check(3e5)
    rotate(1e4)
    check(1e4)

    def free():
        n = (C.c_size_t * 2)()
        assert cw.lib().hipMemGetInfo(C.byref(n, 0), C.byref(n, C.sizeof(C.c_size_t))) == 0
        return n[0]

    ctx.flush()
    before = free()
    for i in range(8000):
        rotate(2e4 + i)
    check(2e4 + 7999)
    g.launch()
    check(3e5)
    g.close()
    assert before - free() <= 4 << 20
