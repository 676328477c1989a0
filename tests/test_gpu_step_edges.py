"""Values at the ends of f32's range in the operators of a step's rest."""
import numpy as np
import pytest

import cw
import paged_oracle as po
import step_oracle as so
from test_gpu_logits import Step
from test_gpu_moe import Layer
from test_gpu_paged import KV, LAYOUT, i32
from test_gpu_qk_norm import gains, shifted

pytestmark = pytest.mark.gpu

STEP = 2.0**-149  # f32's smallest


# ------------------------------------------------------------------ experts

def check_small(m, x, got, residual=None):
    """step_oracle.moe's bound, and f32's steps at its lower end.  Of h: its
    rounding, half a step, and the product's with gate or up half a step off, less
    than half a step for |gate|, |up| < 0.4: a step times the weights of down.  Of y:
    at most eight sums or 32 weighted products, each rounded twice: 32 steps."""
    y, ids, p = got
    want, bound, we, wp = so.moe(x, m.router, m.gate, m.up, m.down, m.k, m.normalise, residual)
    assert np.array_equal(ids, we)
    assert np.all(np.abs(p - wp) <= 4 * so.H * wp + STEP)
    down = np.abs(so.weights(*m.down)).sum(2)  # [experts, dim]
    bound = bound + STEP * ((wp[..., None] * down[we]).sum(1) + 32)
    d = np.abs(y - want)
    assert np.all(d <= bound), (float(d.max()), float((d / bound).max()))


@pytest.mark.parametrize("dim,hidden", [(256, 128), (96, 160), (512, 576)])
@pytest.mark.parametrize("size", [-45, -57, -60, -100, -114, -122, -126, -147])
@pytest.mark.parametrize("rows", [1, 6, 30, 170])
def test_rows_of_small_values(ctx, rng, rows, size, dim, hidden):
    """x, or h that is its square, down to the smallest values there are, beside
    ordinary rows."""
    m = Layer(ctx, rng, dim, hidden, 16, 4)
    x = rng.standard_normal((rows, dim)) * 2.0**size
    x[1::3] = rng.standard_normal((len(x[1::3]), dim))
    x = x.astype(np.float32)
    x[0, :2] = 2.0**size, 0.0
    check_small(m, x, m.run(x))
    res = rng.standard_normal((rows, dim)).astype(np.float32)
    check_small(m, x, m.run(x, res), res)


@pytest.mark.parametrize("hidden", [128, 96])
@pytest.mark.parametrize("rows,n", [(1, 500), (40, 500), (100, 500), (300, 70)])
def test_small_rows_under_small_weights(ctx, rng, rows, n, hidden):
    """h near f32's lower end, large matrices behind it, and p of 1 / n."""
    m = Layer(ctx, rng, 64, hidden, n, 3, normalise=False)
    m.down = so.q4(rng, n, 64, hidden, scale=90.0)
    m.upload()
    for size in (-56, -60, -62):
        x = (rng.standard_normal((rows, 64)) * 2.0**size).astype(np.float32)
        check_small(m, x, m.run(x))


# ------------------------------------------------------------------ logits

@pytest.mark.parametrize("vocab", [70, 4000, 5001, 40000, 700000])
def test_more_than_one_infinity(ctx, rng, vocab):
    """Two logits of infinity have no log softmax, wherever they lie."""
    at = [(3, 5), (0, 1), (2, 66), (vocab - 1, vocab - 2), (1, vocab - 1), (7, 8, 9), (vocab // 2, vocab // 2 + 4),
          (vocab - 3,)]
    for one in range(2):  # all rows, and each alone (slices of another size)
        s = Step(ctx, rng, vocab, [1] * len(at), 4, nodes=False, penalties=False)
        s.rules = cw.logit_rules()
        x = rng.standard_normal((len(at), vocab)).astype(np.float32)
        for i, a in enumerate(at):
            x[i, list(a)] = np.inf
        runs = [s.run(x[i:i + 1], rows=[i]) for i in range(len(at))] if one else [s.run(x)]
        token, logprob = (np.concatenate([r[k] for r in runs]) for k in (1, 2))
        assert token.tolist() == [min(a) for a in at]
        assert np.all(np.isnan(logprob[:-1])) and logprob[-1] == 0.0


def test_infinities_that_a_bias_makes(ctx, rng):
    vocab = 6000
    s = Step(ctx, rng, vocab, [1] * 3, 4, nodes=False, penalties=False, bias=2)
    s.bias_first, s.bias_token = i32([0, 2, 4, 6]), i32([8, 10, 8, 5000, 7, 8])
    s.bias = np.array([np.inf, np.inf, np.inf, np.inf, np.inf, 1.0], np.float32)
    s.upload()
    x = rng.standard_normal((3, vocab)).astype(np.float32)
    _, token, logprob = s.run(x)
    assert token.tolist() == [8, 8, 7] and np.all(np.isnan(logprob[:2])) and logprob[2] == 0.0


@pytest.mark.parametrize("vocab", [1000, 30001])
def test_repeat_penalties_of_any_size(ctx, rng, vocab):
    """l / repeat and l * repeat as f32 has them, where the nearest of 1 / repeat has
    lost bits too.  A step off where the quotient's remainder (2^-24 of l) or the result
    is below f32's normal range.  One below 2^-126 counts as that."""
    repeat = np.array([STEP, 2.0**-130, 3e-39, 2.0**-128, 0.0, -1.0, 2.0**-126, 1.3e-38, 1e-20, 0.7,
                       1.3, 1e20, 2.0**126, 1e38, 3.4e38, np.finfo(np.float32).max], np.float32)
    n = len(repeat)
    s = Step(ctx, rng, vocab, [1] * n, 600, nodes=False)
    s.tokens = i32(rng.integers(0, vocab, (n, 600)))
    s.length[:] = 600
    s.repeat, s.presence, s.frequency = repeat, None, None
    s.upload()
    x = (rng.standard_normal((n, vocab)) * 2.0 ** rng.integers(-149, 120, (n, vocab))).astype(np.float32)
    x[:, ::7] = np.float32(2.0) ** rng.integers(-149, -20, x[:, ::7].shape)
    x[:, 1::97], x[:, 2::97], x[:, 3::97], x[:, 4::97] = np.inf, -np.inf, 0.0, -0.0
    got = s.run(x)[0]
    repeat = np.maximum(repeat, np.float32(2.0**-126))
    seen = np.zeros((n, vocab), bool)
    np.put_along_axis(seen, s.tokens, True, 1)
    with np.errstate(all="ignore"):
        want = np.where(seen, np.where(x > 0, x / repeat[:, None], x * repeat[:, None]), x)
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
        normal = fine & (np.abs(want) >= 2.0**-126) & (np.abs(x) >= 2.0**-100)
        assert np.array_equal(got[normal], want[normal])
        off = np.abs(got.astype(np.float64) - want)
        assert np.all(off[fine] <= np.spacing(np.abs(want[fine])))


def test_zeros_keep_their_signs(ctx, rng):
    """A logit that no rule is for comes out as it went in."""
    vocab = 5000
    s = Step(ctx, rng, vocab, [1, 1], 3000, nodes=False, bias=30)
    s.tokens %= 1000
    s.upload()
    x = np.where(rng.random((2, vocab)) < 0.5, -0.0, 0.0).astype(np.float32)
    got = s.run(x)[0]
    free = np.ones((2, vocab), bool)
    for b in range(2):
        free[b, s.tokens[b, :s.length[b]]] = False
        listed = s.bias_token[s.bias_first[b]:s.bias_first[b + 1]]
        free[b, listed[(listed >= 0) & (listed < vocab)]] = False
    assert free.sum() > 6000
    assert np.array_equal(got.view(np.uint32)[free], x.view(np.uint32)[free])


# ------------------------------------------------------------------ norms

@pytest.mark.parametrize("hd,rot,layout,shift", [(128, 128, "halves", 0), (64, 32, "pairs", 0), (96, 96, "pairs", 1),
                                                 (80, 20, "halves", 0), (256, 2, "halves", 0)])
def test_norms_of_heads_of_any_size(ctx, rng, hd, rot, layout, shift):
    """Heads whose squares are past f32's range on either side, each head another."""
    sizes = [-147, -120, -100, -76, -62, -51, -30, 0, 30, 58, 61, 64, 90, 120]
    heads, rows = len(sizes), 5
    qg, kg = gains(rng, hd)
    pos = i32(rng.integers(0, 9000, rows))
    spec = cw.rope_spec(rot, 1e6, LAYOUT[layout])
    x = np.ldexp(rng.standard_normal((rows, heads, hd)), np.array(sizes)[:, None]).astype(np.float32)
    for eps in (0.0, 1e-38, 1e-30, 1e-6):
        xd = shifted(ctx, x, shift)
        got = ctx.qk_norm_rope_rows(spec, xd, shifted(ctx, qg, shift), None, ctx.storage(pos), rows, heads, 0, hd,
                                    eps).download().reshape(x.shape)
        ref, tol = so.norm_rope(x, np.tile(qg, (heads, 1)), np.float64(np.float32(eps)), pos,
                                po.rope_freqs(rot, 1e6, "plain"), rot, layout == "pairs", 1.0)
        # below f32's normal range: half a step for each of the pair's two by the root's factor, that
        # times the gain (under 3), half by the gain, the products and the sum: 5 steps
        assert np.all(np.abs(got - ref) <= tol + 8 * STEP), (eps, float((np.abs(got - ref) / (tol + 8 * STEP)).max()))


@pytest.mark.parametrize("hd,rot", [(128, 128), (32, 6)])
def test_norms_of_heads_of_any_size_into_a_cache(ctx, rng, hd, rot):
    sizes = [-140, -80, -60, 0, 62, 110]
    kvh, rows = len(sizes), 7
    kv_type, dt = KV["f32"]
    x = np.ldexp(rng.standard_normal((rows, 2 * kvh, hd)), np.array(sizes * 2)[:, None]).astype(np.float32)
    kd, vd = (ctx.storage(np.zeros((rows, kvh, hd), dt)) for _ in range(2))
    pos, kg = i32(rng.integers(0, 9000, rows)), gains(rng, hd)[1]
    ctx.qk_norm_rope_kv_rows(cw.rope_spec(rot, 1e6), cw.kv_pages(kd, vd, kv_type, kvh, hd, rows, 1),
                             ctx.storage(x), None, ctx.storage(kg), ctx.storage(pos),
                             ctx.storage(i32(np.arange(rows))), rows, 0, 0.0)
    ref, tol = so.norm_rope(x[:, :kvh], np.tile(kg, (kvh, 1)), 0.0, pos, po.rope_freqs(rot, 1e6, "plain"), rot,
                            False, 1.0)
    assert np.all(np.abs(kd.download() - ref) <= tol)
    assert np.array_equal(vd.download(), x[:, kvh:])
