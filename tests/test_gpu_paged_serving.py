"""The paged operators as a server uses them on the MI355X: many requests, a
cache past 4 GB, recorded and replayed, two contexts at once.

Against the definitions in 64 bits with the bounds of test_gpu_paged; where the
same call runs twice its bits have to agree."""
import threading

import numpy as np
import pytest

import cw
import paged_oracle as po
from test_gpu_paged import KV, Batch, i32, run_tables, same_step, tables_state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("hd,contig,most", [(128, False, 4), (64, True, 4), (64, False, 40), (32, False, 4)])
def test_attention_of_many_requests(ctx, rng, hd, contig, most, kv):
    """More requests than lanes, some without a row, one with a long context."""
    n = 201
    cached, new = rng.integers(0, 90, n), rng.integers(0, most, n)
    cached[150], new[[0, 64, 200]] = 1700, 0
    b = Batch(ctx, rng, cached, new, 4, 2, hd, kv, 16, tree=True, contig=contig, spare_rows=5)
    b.check(b.run())


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 128), (7, 1, 128), (16, 1, 64), (7, 1, 256), (66, 1, 64), (3, 3, 32)])
def test_attention_of_prompts(ctx, rng, heads, kvh, hd, kv):
    """Prompts with little or nothing cached: later rows see more than earlier
    ones, and a block of rows only the positions up to its last."""
    b = Batch(ctx, rng, [0, 0, 5, 40, 0], [330, 64, 65, 129, 1], heads, kvh, hd, kv, 16, spare_rows=2)
    b.check(b.run())


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,hd", [(1, 128), (8, 128), (8, 64), (8, 256), (2, 32)])
def test_a_lost_block_behind_the_first_rows(ctx, rng, heads, hd, kv):
    """Every row of a request with a block that is not there is NaN, the rows
    too that come before it."""
    b = Batch(ctx, rng, [0, 30], [300, 9], heads, 1, hd, kv, 16)
    good = b.run()
    b.check(good)
    b.tables[0, 18] = -1  # positions 288 .. 299
    got = b.run()
    assert np.all(np.isnan(got[:300])) and np.array_equal(got[300:], good[300:])


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,hd,contig", [(1, 128, False), (8, 128, True), (8, 64, False), (8, 256, False),
                                             (2, 32, True)])
def test_a_length_behind_the_cache(ctx, rng, heads, hd, contig, kv):
    """A length of a billion positions that the cache does not have: NaN for that
    request's rows, the others as they were."""
    b = Batch(ctx, rng, [0, 30], [300, 9], heads, 1, hd, kv, 16, contig=contig)
    ref, bound = po.attention(b.q, b.k, b.v, b.tables, b.page, b.cached, b.first)
    b.cached[0] = (1 << 30) - 300
    got = b.run()
    assert np.all(np.isnan(got[:300])) and np.all(np.abs(got - ref)[300:] <= bound[300:])


@pytest.mark.parametrize("rows_cap", [300, 9000])
def test_tables_of_many_requests(ctx, rng, rows_cap):
    """More requests than the offsets in LDS hold."""
    n = 5000
    cached, fresh = rng.integers(0, 60, n), (rng.random(n) < 0.04).astype(np.int64)
    fresh[7], fresh[4999] = 40, 3
    fresh[rng.random(n) < 0.1] = -1
    tables, held, free, n_free, blocks = tables_state(rng, cached, fresh, 16, 8, 3)
    args = (i32(cached), i32(fresh), held, tables, free, n_free, 16, blocks, rows_cap)
    want = po.block_tables(*args)
    assert want[0] == 0
    same_step(run_tables(ctx, *args), want)


@pytest.mark.parametrize("kv,kvh,hd,rows", [("f16", 8, 128, 1), ("f16", 8, 128, 9), ("f16", 8, 128, 70),
                                            ("f32", 4, 128, 2), ("f32", 4, 128, 9), ("f32", 16, 32, 2)])
def test_cache_past_4_gb(ctx, rng, kv, kvh, hd, rows):
    """Slots whose bytes lie past 2^32: written, attended over, moved."""
    kv_type, dt = KV[kv]
    page, slots_n = 64, (1 << 32) // (kvh * hd * dt().itemsize) + 4096
    cached, n = 150, 150 + rows
    kd, vd = (ctx.empty((slots_n, kvh * hd), dt) for _ in range(2))
    pages = cw.kv_pages(kd, vd, kv_type, kvh, hd, page, slots_n // page)
    held = -(-n // page)
    tables = i32(slots_n // page - 1 - rng.permutation(60)[:held])[None]
    x = rng.standard_normal((n, 2 * kvh * hd)).astype(np.float32)
    slots = i32([po.slot_of(tables, page, 0, p) for p in range(n)])
    assert int(slots.min()) * kvh * hd * dt().itemsize > 1 << 32
    spec = cw.rope_spec(hd, 1e6, scaling=cw.ROPE_PLAIN)  # at position 0: as it is
    ctx.rope_kv_rows(spec, pages, ctx.storage(x), ctx.storage(np.zeros(n, np.int32)),
                     ctx.storage(slots), n, 0)
    xc = x.astype(dt).reshape(n, 2, kvh, hd)
    heads = 2 * kvh
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    first = i32([0, rows])
    batch = cw.batch(ctx.storage(i32([cached])), 1, rows, ctx.storage(first), ctx.storage(tables),
                     held)
    own = np.arange(held)[None]  # the oracle's cache: the request's positions alone
    k, v = (np.concatenate([xc[:, i], np.zeros((held * page - n, kvh, hd), dt)]) for i in range(2))
    for _ in range(2):
        got = ctx.attention_tree(pages, batch, ctx.storage(q), heads).download().reshape(q.shape)
        ref, bound = po.attention(q, k, v, own, page, [cached], first)
        assert np.all(np.abs(got - ref) <= bound)
        path = i32([[rows - 1]])
        ctx.kv_accept(pages, batch, ctx.storage(path), 1, ctx.storage(i32([1])))
        k, v = po.accept(k, v, own, page, [cached], path, [1])


@pytest.mark.parametrize("kv,heads,rows", [("f16", 4, 1), ("f16", 8, 40), ("f32", 4, 1), ("f32", 8, 40)])
def test_recorded_attention_follows_the_lengths(ctx, rng, kv, heads, rows):
    """One recording, replayed as lengths, tables and rows change on the device
    and other calls use the context's scratch between the replays."""
    kv_type, dt = KV[kv]
    kvh, hd, page, blocks, n = 2, 128, 16, 200, 3
    k, v = (rng.standard_normal((blocks * page, kvh, hd)).astype(dt) for _ in range(2))
    pages = cw.kv_pages(ctx.storage(k), ctx.storage(v), kv_type, kvh, hd, page, blocks)
    q = rng.standard_normal((n * rows, heads, hd)).astype(np.float32)
    qd, out = ctx.storage(q), ctx.empty(q.shape)
    cached_d, first_d = ctx.empty(n, np.int32), ctx.empty(n + 1, np.int32)
    tables_d = ctx.empty((n, 60), np.int32)
    batch = cw.batch(cached_d, n, n * rows, first_d, tables_d, 60)

    def draw():
        cached, new = rng.integers(0, 900, n), rng.integers(0, rows + 1, n)
        first = i32(np.concatenate([[0], np.cumsum(new)]))
        tables = i32(rng.permutation(blocks)[:n * 60].reshape(n, 60))
        for d, a in ((cached_d, cached), (first_d, first), (tables_d, tables)):
            d.upload(i32(a))
        return cached, first, tables

    draw()
    ctx.attention_tree(pages, batch, qd, heads, out=out)
    ctx.graph_begin()
    ctx.attention_tree(pages, batch, qd, heads, out=out)
    g = ctx.graph_end()
    ctx.graph_begin()
    ctx.attention_tree(pages, batch, qd, heads, out=out)
    g2 = ctx.graph_end()
    other = Batch(ctx, rng, [300, 20], [3, 9], 4, 2, 256, kv, 16)
    for i in range(6):
        cached, first, tables = draw()
        out.upload(np.full(q.shape, 7.5, np.float32))
        (g, g2)[i % 2].launch()
        got, live = out.download(), int(first[-1])
        ref, bound = po.attention(q, k, v, tables, page, cached, first)
        assert np.all(np.abs(got - ref)[:live] <= bound[:live])
        assert np.all(got[live:] == 7.5)
        eager = ctx.attention_tree(pages, batch, qd, heads).download().reshape(q.shape)
        assert np.array_equal(eager[:live], got[:live])
        if i == 2:  # larger scratch than any before: the recordings keep theirs
            other.check(other.run())
    g.close()
    g2.close()


def test_recording_needs_the_first_call(ctx):
    """A new table of frequencies is refused while recording, and made before."""
    x, pos = ctx.storage(np.ones((2, 64), np.float32)), ctx.storage(i32([1, 2]))
    spec = cw.rope_spec(64, 54321.0)
    y = ctx.empty((2, 64))
    ctx.graph_begin()
    with pytest.raises(cw.CwError, match="before cw_graph_begin"):
        ctx.rope_rows(spec, x, pos, 2, 1, 64, y=y)
    ctx.graph_end().close()
    want = ctx.rope_rows(spec, x, pos, 2, 1, 64, y=y).download()
    ctx.graph_begin()
    ctx.rope_rows(spec, x, pos, 2, 1, 64, y=y)
    g = ctx.graph_end()
    y.upload(np.zeros((2, 64), np.float32))
    g.launch()
    assert np.array_equal(y.download().reshape(want.shape), want)
    g.close()


def test_two_contexts_at_once(ctx, rng):
    """Two host threads with a context each, the same calls: the same bits."""
    cached, new = [400, 30, 900, 0], [20, 40, 7, 33]
    want = Batch(ctx, np.random.default_rng(5), cached, new, 8, 2, 128, "f16", 16, tree=True)
    ref = want.run()
    want.check(ref)
    wrong = []

    def work():
        c = cw.Context(0)
        try:
            b = Batch(c, np.random.default_rng(5), cached, new, 8, 2, 128, "f16", 16, tree=True)
            for _ in range(8):
                if not np.array_equal(b.run(), ref):
                    wrong.append("attention")
            x = c.storage(b.q.reshape(len(b.q), -1)[:, :512])
            pos = c.storage(i32(np.arange(len(b.q)) * 1000))
            for theta in (1e4, 1e5, 1e6):
                c.rope_rows(cw.rope_spec(128, theta), x, pos, len(b.q), 4, 128, y=x)
            y.append(x.download())
        except Exception as e:  # noqa: BLE001 (reported by the test's thread)
            wrong.append(repr(e))
        finally:
            c.close()

    y = []
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and np.array_equal(*y)
