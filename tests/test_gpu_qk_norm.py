"""Norms of query and key heads with the rotation in the same pass, against
their definition in 64 bits.  Tolerances: step_oracle.norm_rope's bound; an f16
cache row half an f16 step more (2^-11 relative, 2^-25 absolute)."""
import numpy as np
import pytest

import cw
import paged_oracle as po
import step_oracle as so
from test_gpu_paged import KV, LAYOUT, SCALING, at, i32

pytestmark = pytest.mark.gpu

EPS = 1e-6


def gains(rng, hd):
    return [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]


def shifted(ctx, a, shift, pad=0.0):
    """a on the device, `shift` floats behind an aligned address."""
    d = ctx.empty(a.size + 8)
    return at(d.upload(np.concatenate([np.full(shift, pad), a.ravel(), np.full(8 - shift, pad)])), shift)


ROWS = [
    # rows, heads, kv heads, hd, rot, layout, scaling, factor, x stride - width, shift, far
    (1, 1, 0, 2, 2, "halves", "plain", 1.0, 0, 0, 9),
    (1, 0, 1, 8, 8, "pairs", "plain", 1.0, 0, 0, 9),
    (3, 5, 2, 128, 128, "halves", "plain", 1.0, 0, 0, 40000),
    (7, 3, 3, 128, 64, "pairs", "yarn", 4.0, 12, 0, 131072),
    (5, 2, 1, 64, 64, "pairs", "bands", 8.0, 0, 0, 100000),
    (4, 9, 2, 256, 256, "halves", "linear", 2.5, 4, 0, 30000),
    (2, 3, 1, 256, 2, "pairs", "plain", 1.0, 0, 0, 500),
    (2, 3, 2, 255, 254, "halves", "plain", 1.0, 0, 0, 500),
    (6, 7, 5, 96, 24, "halves", "yarn", 16.0, 0, 0, 1 << 24),   # 12 of 16 lanes
    (3, 4, 4, 80, 20, "halves", "bands", 3.0, 3, 0, 70000),     # a wave a head
    (9, 2, 1, 64, 32, "pairs", "linear", 4.0, 0, 1, 70000),     # an unaligned start
    (9, 2, 1, 40, 8, "halves", "linear", 4.0, 2, 3, 70000),
    (33, 17, 3, 32, 16, "pairs", "plain", 1.0, 0, 0, 3000),
    (700, 40, 8, 128, 128, "halves", "yarn", 4.0, 1024, 0, 131072),
    (2100, 32, 4, 128, 96, "halves", "linear", 2.0, 0, 0, 9000),  # past 32 MB of rows
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", ROWS)
def test_qk_norm_rope_rows(ctx, rng, case, in_place):
    rows, heads, kvh, hd, rot, layout, scaling, factor, pad, shift, far = case
    width, stride = (heads + kvh) * hd, (heads + kvh) * hd + pad
    x = (rng.standard_normal((rows, stride)) * 2.0 ** rng.integers(-8, 9, (rows, 1))).astype(np.float32)
    x[0, :hd] = 0.0  # a head of zeros stays zeros
    pos = i32(rng.integers(0, far, rows))
    pos[0] = far - 1
    if rows > 2:
        pos[1] = -1
    qg, kg = gains(rng, hd)
    spec = cw.rope_spec(rot, 1e6, LAYOUT[layout], SCALING[scaling], factor, 8192)
    xd = shifted(ctx, x, shift)
    y_stride = stride if in_place else width + 5 * shift
    yd = xd if in_place else shifted(ctx, np.full((rows, y_stride), 7.5, np.float32), shift)
    ctx.qk_norm_rope_rows(spec, xd, shifted(ctx, qg, shift) if heads else None,
                          shifted(ctx, kg, shift) if kvh else None, ctx.storage(pos), rows, heads,
                          kvh, hd, EPS, x_stride=stride, y=yd, y_stride=y_stride)
    got = at(yd, -shift).download()[shift:shift + rows * y_stride].reshape(rows, y_stride)
    gain = np.concatenate([np.tile(qg, (heads, 1)), np.tile(kg, (kvh, 1))])
    ref, tol = so.norm_rope(x[:, :width].reshape(rows, heads + kvh, hd), gain, np.float32(EPS), pos,
                            po.rope_freqs(rot, 1e6, scaling, factor), rot, layout == "pairs",
                            po.rope_gain(scaling, factor))
    live = pos >= 0
    d = np.abs(got[:, :width].reshape(ref.shape) - ref)
    assert np.all(d[live] <= tol[live]), float((d[live] - tol[live]).max())
    before = x if in_place else np.full((rows, y_stride), 7.5, np.float32)
    assert np.array_equal(got[~live], before[~live])
    assert np.array_equal(got[:, width:], before[:, width:])


KV_ROWS = [
    # rows, heads, kv heads, hd, rot, layout, kv, page, blocks, stride - width, in place, shift
    (1, 4, 2, 16, 16, "halves", "f16", 16, 1, 0, False, 0),
    (5, 32, 8, 128, 128, "halves", "f16", 16, 3, 0, False, 0),
    (9, 6, 2, 128, 64, "pairs", "f32", 32, 2, 8, True, 0),
    (33, 3, 1, 64, 48, "halves", "f16", 64, 1, 0, True, 0),
    (17, 5, 5, 256, 256, "pairs", "f16", 16, 4, 4, False, 0),
    (12, 0, 3, 32, 16, "halves", "f32", 100, 1, 0, False, 0),
    (21, 2, 1, 32, 6, "pairs", "f16", 16, 2, 1, False, 0),
    (21, 2, 1, 32, 8, "halves", "f16", 16, 2, 1, False, 2),
    (600, 16, 8, 128, 128, "halves", "f16", 16, 40, 0, False, 0),
]


@pytest.mark.parametrize("case", KV_ROWS)
def test_qk_norm_rope_kv_rows(ctx, rng, case):
    rows, heads, kvh, hd, rot, layout, kv, page, blocks, pad, in_place, shift = case
    kv_type, dt = KV[kv]
    width = (heads + 2 * kvh) * hd
    stride, slots_n = width + pad, page * blocks
    x = (3.0 * rng.standard_normal((rows, stride))).astype(np.float32)
    k0, v0 = (rng.standard_normal((slots_n, kvh, hd)).astype(dt) for _ in range(2))
    kd, vd = ctx.storage(k0), ctx.storage(v0)
    pos, slots = i32(rng.integers(0, 9000, rows)), i32(rng.permutation(slots_n)[:rows])
    if rows > 4:
        pos[1], slots[2], slots[3] = -1, -1, slots_n  # padding; rows without a slot
    qg, kg = gains(rng, hd)
    xd = shifted(ctx, x, shift)
    q_stride = stride if in_place else heads * hd + shift
    q0 = x if in_place else np.full((rows, q_stride), 7.5, np.float32)
    qd = xd if in_place else shifted(ctx, q0, shift)
    ctx.qk_norm_rope_kv_rows(cw.rope_spec(rot, 1e6, LAYOUT[layout]),
                             cw.kv_pages(kd, vd, kv_type, kvh, hd, page, blocks), xd,
                             shifted(ctx, qg, shift) if heads else None, shifted(ctx, kg, shift),
                             ctx.storage(pos), ctx.storage(slots), rows, heads, EPS, stride=stride,
                             q_out=qd if heads else None, q_stride=q_stride)
    gain = np.concatenate([np.tile(qg, (heads, 1)), np.tile(kg, (kvh, 1))])
    ref, tol = so.norm_rope(x[:, :(heads + kvh) * hd].reshape(rows, heads + kvh, hd), gain,
                            np.float32(EPS), pos, po.rope_freqs(rot, 1e6, "plain"), rot,
                            layout == "pairs", 1.0)
    live = pos >= 0
    if heads:
        got = at(qd, -shift).download()[shift:shift + rows * q_stride].reshape(rows, q_stride)
        d = np.abs(got[:, :heads * hd].reshape(rows, heads, hd) - ref[:, :heads])
        assert np.all(d[live] <= tol[live, :heads])
        assert np.array_equal(got[~live], q0[~live])
        assert np.array_equal(got[:, heads * hd:], q0[:, heads * hd:])
    held = live & (slots >= 0) & (slots < slots_n)
    k, v = kd.download(), vd.download()
    s = slots[held]
    r, t = ref[held, heads:], tol[held, heads:]
    if kv == "f16":
        t = t + np.abs(r) * 2.0**-11 + 2.0**-25
    assert np.all(np.abs(k[s].astype(np.float64) - r) <= t)
    assert np.array_equal(v[s], x[held, (heads + kvh) * hd:width].reshape(-1, kvh, hd).astype(dt))
    rest = np.ones(slots_n, bool)
    rest[s] = False
    assert np.array_equal(k[rest], k0[rest]) and np.array_equal(v[rest], v0[rest])


def test_norm_then_rotation_of_the_separate_calls(ctx, rng):
    """The same as cw_rmsnorm of every head and cw_rope_rows, to both's rounding."""
    rows, heads, hd = 6, 5, 128
    x = rng.standard_normal((rows, heads * hd)).astype(np.float32)
    g = gains(rng, hd)[0]
    spec, pos, gd = cw.rope_spec(hd, 1e6), ctx.storage(i32(rng.integers(0, 5000, rows))), ctx.storage(g)
    one = ctx.qk_norm_rope_rows(spec, ctx.storage(x), gd, None, pos, rows, heads, 0, hd, EPS).download()
    n = ctx.rmsnorm(ctx.storage(x), gd, rows * heads, hd, EPS)
    two = ctx.rope_rows(spec, n, pos, rows, heads, hd).download()
    n = np.abs(n.download().reshape(rows, heads, hd))
    mag = n + np.roll(n, hd // 2, 2)
    assert np.all(np.abs(one - two).reshape(mag.shape) <= 2 * 20 * so.H * mag)


def test_recorded(ctx, rng):
    """Replayed as positions and slots change on the device."""
    rows, heads, kvh, hd, page, blocks = 9, 4, 2, 64, 16, 4
    x = rng.standard_normal((rows, (heads + 2 * kvh) * hd)).astype(np.float32)
    qg, kg = (ctx.storage(g) for g in gains(rng, hd))
    kd, vd = (ctx.storage(np.zeros((page * blocks, kvh * hd), np.float16)) for _ in range(2))
    kv = cw.kv_pages(kd, vd, cw.CW_F16, kvh, hd, page, blocks)
    spec, xd, q = cw.rope_spec(hd, 7e5), ctx.storage(x), ctx.empty((rows, heads * hd))
    pos, slots = ctx.storage(i32(np.zeros(rows))), ctx.storage(i32(np.arange(rows)))

    def call():
        ctx.qk_norm_rope_kv_rows(spec, kv, xd, qg, kg, pos, slots, rows, heads, EPS, q_out=q)
    with pytest.raises(cw.CwError, match="before cw_graph_begin"):
        ctx.graph_begin()
        try:
            call()
        finally:
            ctx.graph_end().close()
    call()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()
    for _ in range(4):
        p, s = i32(rng.integers(-1, 9000, rows)), i32(rng.permutation(page * blocks)[:rows])
        pos.upload(p), slots.upload(s)
        start = rng.standard_normal(kd.shape).astype(np.float16)
        got = []
        for do in (call, g.launch):
            kd.upload(start), vd.upload(start), q.upload(np.full(q.shape, 7.5))
            do()
            got.append([d.download() for d in (q, kd, vd)])
        assert all(np.array_equal(a, b) for a, b in zip(*got))
        assert np.all(got[0][0][p < 0] == 7.5) and not np.any(got[0][0][p >= 0] == 7.5)
    g.close()
