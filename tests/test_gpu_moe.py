"""Mixture-of-experts layers against their definition in 64 bits; tolerances:
step_oracle.moe's bound.  The choice of experts is exact."""
import numpy as np
import pytest

import cw
import step_oracle as so
from test_gpu_paged import i32

pytestmark = pytest.mark.gpu


class Layer:
    """Random experts, on the host and on the device."""

    def __init__(self, ctx, rng, dim, hidden, n, k, normalise=True, shift=0):
        self.ctx, self.dim, self.k, self.normalise = ctx, dim, k, normalise
        self.router = (rng.standard_normal((n, dim)) * 1.5 / np.sqrt(dim)).astype(np.float32)
        self.gate, self.up = (so.q4(rng, n, hidden, dim, scale=0.2 / np.sqrt(dim)) for _ in range(2))
        self.down = so.q4(rng, n, dim, hidden, scale=0.2 / np.sqrt(hidden))
        self.hidden, self.n, self.shift = hidden, n, shift
        self.upload()

    def upload(self):
        ctx, d = self.ctx, []
        for s, q in (self.gate, self.up, self.down):
            # scales `shift` halves behind an aligned address
            buf = ctx.storage(np.concatenate([np.zeros(self.shift, np.uint16), s.view(np.uint16).ravel()]))
            d += [cw.DeviceArray(ctx, s.shape, np.uint16, buf.ptr + 2 * self.shift), ctx.storage(q)]
        self.moe = cw.moe(self.dim, self.hidden, self.n, self.k, ctx.storage(self.router), *d,
                          normalise=self.normalise)

    def run(self, x, residual=None, positions=None, y=None, in_place=False):
        ctx, rows = self.ctx, len(x)
        put = lambda a: None if a is None else ctx.storage(a)  # noqa: E731
        res = put(residual)
        yd = res if in_place else ctx.storage(np.full((rows, self.dim), 7.5, np.float32))
        ids = ctx.storage(np.full((rows, self.k), -7, np.int32))
        p = ctx.storage(np.full((rows, self.k), -7.0, np.float32))
        ctx.moe_rows(self.moe, ctx.storage(x), rows, residual=res, positions=put(positions), y=yd,
                     experts=ids, weights=p)
        return yd.download(), ids.download(), p.download()

    def check(self, x, got, residual=None, live=None):
        y, ids, p = got
        live = np.ones(len(x), bool) if live is None else live
        want, bound, we, wp = so.moe(x[live], self.router, self.gate, self.up, self.down, self.k,
                                     self.normalise, None if residual is None else residual[live])
        assert np.array_equal(ids[live], we)
        # (f32's values end in steps of 2^-149: a weight below them rounds to 0)
        assert np.all(np.abs(p[live] - wp) <= 4 * so.H * wp + 2.0**-149)
        d = np.abs(y[live] - want)
        assert np.all(d <= bound), (float(d.max()), float((d / bound).max()))


SHAPES = [
    # rows, dim, hidden, experts, top, normalise
    (1, 32, 32, 1, 1, True),
    (1, 256, 96, 7, 3, False),
    (1, 2048, 768, 32, 8, True),
    (2, 64, 64, 512, 32, True),
    (3, 96, 160, 5, 5, True),
    (5, 1024, 512, 64, 8, False),
    (8, 288, 224, 33, 4, True),
    (9, 512, 1056, 12, 2, True),
    (17, 2208, 544, 6, 2, False),
    (40, 256, 256, 128, 8, True),
    (70, 320, 480, 3, 1, True),
    (130, 128, 64, 2, 2, True),
    (300, 160, 96, 16, 4, False),
    (33, 4096, 128, 9, 3, True),
    (21, 128, 4128, 4, 2, True),
    (512, 256, 4096, 8, 4, True),
    (600, 4096, 256, 8, 8, False),
    (6, 1024, 512, 128, 8, True),
    (3, 160, 288, 100, 4, False),
]


@pytest.mark.parametrize("rows,dim,hidden,n,k,normalise", SHAPES)
def test_moe_rows(ctx, rng, rows, dim, hidden, n, k, normalise):
    m = Layer(ctx, rng, dim, hidden, n, k, normalise)
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    m.check(x, m.run(x))
    res = rng.standard_normal((rows, dim)).astype(np.float32)
    for in_place in (False, True):
        m.check(x, m.run(x, res, in_place=in_place), res)


@pytest.mark.parametrize("rows", [1, 3, 12, 50, 200])
def test_padding_rows_and_rows_that_are_not_finite(ctx, rng, rows):
    """Padding rows are left as they were, whatever they hold; a row of an
    infinity or a NaN is NaN and touches no other."""
    m = Layer(ctx, rng, 256, 128, 24, 4)
    x = rng.standard_normal((rows, 256)).astype(np.float32)
    pos = i32(rng.integers(0, 100, rows))
    pos[rng.random(rows) < 0.3] = -1
    if rows > 1:
        pos[0], pos[rows - 1] = 5, -1
    x[pos < 0] = np.nan
    bad = np.zeros(rows, bool)
    if rows > 2:
        pos[1] = 7
        x[1] = rng.standard_normal(256)
        x[1, 77] = np.inf if rows % 2 else np.nan
        bad[1] = True
    y, ids, p = m.run(x, positions=pos)
    live = (pos >= 0) & ~bad
    m.check(x, (y, ids, p), live=live)
    assert np.all(y[pos < 0] == 7.5) and np.all(ids[pos < 0] == -7) and np.all(p[pos < 0] == -7)
    assert np.all(np.isnan(y[bad])) and np.all((ids[bad] >= 0) & (ids[bad] < 24))
    assert all(len(set(r)) == 4 for r in ids[bad].tolist())


def test_no_row_at_all(ctx, rng):
    m = Layer(ctx, rng, 64, 32, 4, 2)
    for rows in (1, 30, 300):
        x = np.full((rows, 64), np.nan, np.float32)
        y, ids, _ = m.run(x, positions=np.full(rows, -1, np.int32))
        assert np.all(y == 7.5) and np.all(ids == -7)


@pytest.mark.parametrize("rows", [1, 4, 40, 260])
def test_equal_scores_go_to_the_lowest_experts(ctx, rng, rows):
    m = Layer(ctx, rng, 128, 64, 70, 6)
    m.router[:] = m.router[rng.integers(0, 3, 70)]
    m.upload()
    x = rng.standard_normal((rows, 128)).astype(np.float32)
    m.check(x, m.run(x))
    m.router[:] = 0.0
    m.upload()
    got = m.run(x)
    assert np.array_equal(got[1], np.tile(np.arange(6), (rows, 1)))
    m.check(x, got)


@pytest.mark.parametrize("rows", [6, 64, 400])
def test_every_row_takes_the_same_experts(ctx, rng, rows):
    """All rows on few of many experts: long lists beside empty ones."""
    m = Layer(ctx, rng, 96, 64, 100, 3)
    common = rng.standard_normal(96).astype(np.float32)
    x = (0.05 * rng.standard_normal((rows, 96)) + common).astype(np.float32)
    got = m.run(x)
    assert len(set(got[1].flatten().tolist())) < 12
    m.check(x, got)


@pytest.mark.parametrize("rows", [1, 7, 60, 280])
def test_scores_close_to_each_other(ctx, rng, rows):
    """Scores that differ by less than an f32 step are told apart."""
    m = Layer(ctx, rng, 64, 32, 40, 4)
    m.router[:] = 1.0
    m.router[:, 0] += rng.permutation(40) * np.float32(2.0**-23)
    m.upload()
    x = (1.0 + rng.random((rows, 64))).astype(np.float32) * 1000
    m.check(x, m.run(x))


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows", [1, 5, 20, 150])
def test_scales_at_any_address(ctx, rng, rows, shift):
    m = Layer(ctx, rng, 544, 288, 10, 2, shift=shift)
    x = rng.standard_normal((rows, 544)).astype(np.float32)
    m.check(x, m.run(x))


@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("dim,hidden", [(320, 448), (1984, 832), (64, 192), (1600, 2112)])
@pytest.mark.parametrize("rows,n,k", [(1, 9, 2), (2, 24, 5), (23, 6, 2), (90, 5, 2)])
def test_rows_of_an_even_number_of_blocks(ctx, rng, rows, n, k, dim, hidden, shift):
    """Rows that end within a group of four blocks, by every kernel; the last
    expert's last blocks are the last of their arrays."""
    m = Layer(ctx, rng, dim, hidden, n, k, shift=shift)
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    m.check(x, m.run(x))


@pytest.mark.parametrize("rows", [1, 6, 30, 170])
def test_large_and_small_values(ctx, rng, rows):
    """Rows of very different sizes, and elements far below their row's largest."""
    m = Layer(ctx, rng, 256, 128, 16, 4)
    x = rng.standard_normal((rows, 256)) * 2.0 ** rng.integers(-40, 20, (rows, 1))
    x[:, ::3] *= 2.0**-15
    x = x.astype(np.float32)
    x[0] = 0.0  # every score 0, y 0
    got = m.run(x)
    m.check(x, got)
    assert np.all(got[0][0] == 0.0)


def test_more_rows_than_go_through_together(ctx, rng):
    m = Layer(ctx, rng, 64, 32, 20, 2)
    x = rng.standard_normal((4500, 64)).astype(np.float32)
    pos = i32(np.where(np.arange(4500) % 7 == 3, -1, 1))
    got = m.run(x, x, positions=pos)
    m.check(x, got, x, pos >= 0)
    assert np.all(got[0][pos < 0] == 7.5)


@pytest.mark.parametrize("rows,dim,hidden,n,k", [(2500, 32, 64, 9, 2), (700, 32, 8192, 32, 32)])
def test_rows_in_pieces(ctx, rng, rows, dim, hidden, n, k):
    """More rows, or larger ones, than the workspace takes at once: each piece has
    its own positions, choices and residual, and rows that are padding."""
    m = Layer(ctx, rng, dim, hidden, n, k)
    x, res = (rng.standard_normal((rows, dim)).astype(np.float32) for _ in range(2))
    pos = i32(np.where(rng.random(rows) < 0.1, -1, 3))
    got = m.run(x, res, pos)
    live = pos >= 0
    m.check(x, got, res, live)
    assert np.all(got[0][~live] == 7.5) and np.all(got[1][~live] == -7) and np.all(got[2][~live] == -7.0)


@pytest.mark.parametrize("rows", [1, 6, 48, 300])
def test_the_same_bits_each_time_and_replayed(ctx, rng, rows):
    """Eager, recorded and replayed beside other work, with rows that come and go."""
    m = Layer(ctx, rng, 512, 256, 48, 6)
    other = Layer(ctx, rng, 256, 512, 8, 2)
    xd, y = ctx.empty((rows, 512)), ctx.empty((rows, 512))
    pos, ids = ctx.empty(rows, np.int32), ctx.empty((rows, 6), np.int32)

    def call():
        ctx.moe_rows(m.moe, xd, rows, positions=pos, y=y, experts=ids)
    xd.upload(np.zeros((rows, 512), np.float32)), pos.upload(np.zeros(rows, np.int32))
    call()
    graphs = []
    for _ in range(2):
        ctx.graph_begin()
        call()
        graphs.append(ctx.graph_end())
    for i in range(6):
        x = rng.standard_normal((rows, 512)).astype(np.float32)
        p = i32(np.where(rng.random(rows) < 0.2, -1, 3))
        xd.upload(x), pos.upload(p)
        got = []
        for do in (call, graphs[i % 2].launch, call):
            y.upload(np.full(y.shape, 7.5, np.float32)), ids.upload(np.full(ids.shape, -7, np.int32))
            do()
            got.append((y.download(), ids.download()))
            if i == 2:  # larger scratch than any before
                ox = rng.standard_normal((600, 256)).astype(np.float32)
                other.check(ox, other.run(ox))
        for g in got[1:]:
            assert np.array_equal(g[0], got[0][0]) and np.array_equal(g[1], got[0][1])
        want, bound, we, _ = so.moe(x[p >= 0], m.router, m.gate, m.up, m.down, 6, True)
        assert np.all(np.abs(got[0][0][p >= 0] - want) <= bound)
        assert np.array_equal(got[0][1][p >= 0], we) and np.all(got[0][0][p < 0] == 7.5)
    for g in graphs:
        g.close()


@pytest.mark.parametrize("hidden", [4224, 4128])
def test_experts_past_four_gigabytes(ctx, rng, hidden):
    """The last two of 512 experts, whose quants lie past 2^32 bytes; rows of whole
    groups of blocks and others."""
    n, dim, k = 512, 4096, 2
    two = Layer(ctx, rng, dim, hidden, k, k)
    two.router = np.abs(two.router)
    d = []
    for scales, quants in (two.gate, two.up, two.down):
        for a in (scales.view(np.uint16), quants):
            big = ctx.empty((n, *a.shape[1:]), a.dtype)
            skip = (n - k) * a[0].nbytes
            cw.DeviceArray(ctx, a.shape, a.dtype, big.ptr + skip).upload(a)
            d.append(big)
        assert skip > 1 << 32
    router = np.concatenate([np.zeros((n - k, dim), np.float32), two.router])
    two.moe = cw.moe(dim, hidden, n, k, ctx.storage(router), *d)
    for rows in (1, 3, 250):
        x = (0.1 + rng.random((rows, dim))).astype(np.float32)
        y, ids, p = two.run(x)
        assert ids.min() == n - k
        two.check(x, (y, ids - (n - k), p))
    for a in d:
        ctx.free(a)
