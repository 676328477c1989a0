"""Logits under a server's rules against their definition in 64 bits, with
step_oracle's bounds; where every step is exact, to the bit."""
import numpy as np
import pytest

import cw
import paged_oracle as po
import step_oracle as so
from test_gpu_paged import at, i32

pytestmark = pytest.mark.gpu


class Step:
    """Requests with histories and a step's rows of logits."""

    def __init__(self, ctx, rng, vocab, new, longest, *, tree=False, nodes=True, penalties=True,
                 bias=0, masks=False, prompt=True, spare=0, hot=40):
        self.ctx, self.vocab, n = ctx, vocab, len(new)
        self.first = i32(np.concatenate([[0], np.cumsum(new)]))
        self.rows = int(self.first[-1]) + spare
        self.new, self.max_len = new, longest
        # few tokens often, and some outside the vocabulary
        self.tokens = i32(np.where(rng.random((n, longest)) < 0.5, rng.integers(0, min(hot, vocab), (n, longest)),
                                   rng.integers(-3, vocab + 3, (n, longest))))
        self.length = i32(rng.integers(0, longest + 1, n))
        self.length[0] = longest
        self.prompt = i32(rng.integers(0, self.length + 1)) if prompt else None
        self.node = i32(rng.integers(-1, min(hot, vocab) + 1, self.rows)) if nodes else None
        words = (max(max(new), 1) + 31) // 32
        self.mask = None
        if tree:
            self.mask = np.concatenate([po.tree(rng, k, words) for k in new] +
                                       [np.zeros((spare, words), np.uint32)])
        f32 = lambda lo, hi: rng.uniform(lo, hi, n).astype(np.float32)  # noqa: E731
        self.repeat, self.presence, self.frequency = (f32(1.0, 1.5), f32(-0.5, 1.0), f32(0.0, 0.4)) \
            if penalties else (None,) * 3
        self.bias = None
        if bias:
            k = rng.integers(0, bias + 1, n)
            k[0] = bias
            self.bias_first = i32(np.concatenate([[0], np.cumsum(k)]))
            self.bias_token = i32(rng.integers(-1, min(vocab, 2 * hot) + 1, self.bias_first[-1]))
            self.bias = (4 * rng.standard_normal(len(self.bias_token))).astype(np.float32)
        self.allowed, self.allowed_row = None, None
        if masks:
            w = (vocab + 31) // 32 + int(rng.integers(0, 2))
            bits = rng.integers(0, 1 << 32, (5, w), dtype=np.uint32)
            bits[0] &= bits[1] & bits[2]
            bits[3] = 0
            bits[4] = 0
            bits[4, (vocab - 1) // 32] = np.uint32(1) << np.uint32((vocab - 1) % 32)
            self.allowed, self.allowed_row = bits, i32(rng.integers(-1, 6, self.rows))
        self.upload()

    def upload(self):
        put = lambda a: None if a is None else self.ctx.storage(a)  # noqa: E731
        self.batch = cw.batch(None, len(self.new), self.rows, put(self.first), None, 0,
                              mask=put(self.mask), mask_words=0 if self.mask is None else self.mask.shape[1])
        kw = dict(tokens=put(self.tokens), length=put(self.length), prompt=put(self.prompt),
                  max_len=self.max_len, node_token=put(self.node), repeat=put(self.repeat),
                  presence=put(self.presence), frequency=put(self.frequency))
        if self.bias is not None:
            kw.update(bias_first=put(self.bias_first), bias_token=put(self.bias_token),
                      bias=put(self.bias), n_bias=len(self.bias))
        if self.allowed is not None:
            kw.update(allowed=put(self.allowed), n_allowed=len(self.allowed),
                      allowed_words=self.allowed.shape[1], allowed_row=put(self.allowed_row))
        self.rules = cw.logit_rules(**kw)

    def reference(self, x, i, r):
        """Row i of x as batch row r: (logits, bound), or None where it is padding."""
        own = [b for b in range(len(self.new)) if self.first[b] <= r < self.first[b + 1]]
        if not own:
            return None
        b = own[0]
        r0 = int(self.first[b])
        nodes = [] if self.node is None else \
            [self.node[r0 + j] for j in range(self.new[b]) if po.sees(self.mask, r, r - r0, j)]
        one = lambda a, none: none if a is None else a[b]  # noqa: E731
        bias = [] if self.bias is None else \
            [(self.bias_token[e], self.bias[e]) for e in range(self.bias_first[b], self.bias_first[b + 1])]
        allowed = None
        if self.allowed is not None and 0 <= self.allowed_row[i] < len(self.allowed):
            allowed = np.unpackbits(self.allowed[self.allowed_row[i]].view(np.uint8),
                                    bitorder="little")[:self.vocab].astype(bool)
        return so.logits(x[i], self.tokens[b, :self.length[b]], one(self.prompt, 0), nodes,
                         one(self.repeat, 1.0), one(self.presence, 0.0), one(self.frequency, 0.0),
                         bias, allowed)

    def run(self, x, rows=None, stride=None, out="other", out_stride=None, shift=0):
        """(logits, tokens, log probabilities) of the call; x [rows, vocab]."""
        ctx, n = self.ctx, len(x)
        stride = stride or self.vocab
        wide = np.full((n, stride), -77.0, np.float32)
        wide[:, :self.vocab] = x
        xd = at(ctx.empty(n * stride + 4).upload(np.concatenate(
            [np.zeros(shift), wide.ravel(), np.zeros(4 - shift)])), shift)
        od, out_stride = xd, out_stride or stride
        if out == "other":
            od = at(ctx.empty(n * out_stride + 4).upload(np.full(n * out_stride + 4, 7.5)), shift)
        token, logprob = ctx.storage(np.full(n, 77, np.uint32)), ctx.storage(np.full(n, 7.5, np.float32))
        ctx.logits_rows(self.rules, self.batch, xd, n, self.vocab,
                        at=None if rows is None else ctx.storage(i32(rows)), stride=stride,
                        out=od if out else None, out_stride=out_stride, token=token, logprob=logprob)
        got = at(od, -shift).download()[shift:shift + n * out_stride].reshape(n, out_stride)
        return got, token.download(), logprob.download()

    def check(self, x, got, rows=None, before=7.5):
        l, token, logprob = got
        for i in range(len(x)):
            ref = self.reference(x, i, i if rows is None else rows[i])
            if ref is None:
                assert token[i] == 77 and logprob[i] == 7.5
                if l is not None:
                    assert np.all(l[i, :self.vocab] == (x[i] if before is None else before))
                continue
            want, bound = ref
            if l is not None:
                g = l[i, :self.vocab].astype(np.float64)
                inf = ~np.isfinite(want)
                assert np.array_equal(g[inf], want[inf], equal_nan=True)
                assert np.all(np.abs(g[~inf] - want[~inf]) <= 1.001 * bound[~inf])
            so.check_top(want, 1.001 * bound, token[i], logprob[i])
        if l is not None:
            assert np.all(l[:, self.vocab:] == (-77.0 if before is None else before))


CASES = [
    # vocab, rows of each request, longest history, options
    (1, [1], 5, {}),
    (33, [1], 1, dict(masks=True)),
    (300, [1, 1, 1], 40, dict(bias=9, nodes=False)),
    (4096, [5], 300, dict(tree=True)),
    (4097, [3, 0, 2], 700, dict(bias=50, masks=True)),
    (5000, [1] * 9, 90, dict(penalties=False, bias=3, masks=True, nodes=False)),
    (12288, [40, 3], 10, dict(tree=True, bias=200)),
    (20011, [2, 65, 1], 33, dict(tree=True, spare=3)),
    (30000, [1] * 70, 200, dict(prompt=False)),
    (151936, [1, 1], 9000, dict(bias=300, masks=True, nodes=False)),
    (151936, [33], 500, dict()),
    (160001, [1, 4], 64, dict(masks=True, tree=True)),
]


def draw(rng, rows, vocab):
    x = (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] += rng.uniform(0, 20, rows).astype(np.float32)
    return x


@pytest.mark.parametrize("case", CASES)
def test_logits_rows(ctx, rng, case):
    vocab, new, longest, options = case
    s = Step(ctx, rng, vocab, new, longest, **options)
    x = draw(rng, s.rows, vocab)
    got = s.run(x)
    s.check(x, got)
    # odd strides and starts, in place, the token alone: the same bits
    for kw in (dict(stride=vocab + 3, out_stride=vocab + 5, shift=1), dict(stride=vocab + 4, out="same")):
        more = s.run(x, **kw)
        s.check(x, more, before=None if "out" in kw else 7.5)
        live = got[1] != 77
        assert np.array_equal(more[0][live, :vocab], got[0][live, :vocab])
    alone = s.run(x, out=None)
    assert np.array_equal(alone[1], got[1]) and np.array_equal(alone[2], got[2])


def test_rows_of_the_batch(ctx, rng):
    """Logits of some rows: each request's last, one twice, and rows of none."""
    s = Step(ctx, rng, 3000, [4, 0, 9], 60, tree=True, bias=5, masks=True, spare=2)
    rows = [3, 12, 3, -1, 13, 0, 1 << 30, 14]
    x = draw(rng, len(rows), 3000)
    s.check(x, s.run(x, rows), rows)


def test_no_rules_is_argmax(ctx, rng):
    s = Step(ctx, rng, 50000, [1, 1], 3, nodes=False, penalties=False)
    s.rules = cw.logit_rules()
    x = draw(rng, 2, 50000)
    got = s.run(x)
    assert np.array_equal(got[0], x)
    for i in range(2):
        assert got[1][i] == x[i].argmax() == ctx.argmax(ctx.storage(x[i]), 50000).download()[0]
        so.check_top(x[i].astype(np.float64), np.zeros(50000), got[1][i], got[2][i])


@pytest.mark.parametrize("vocab", [70, 5000, 40000])
def test_ties_infinities_and_rows_of_nothing(ctx, rng, vocab):
    s = Step(ctx, rng, vocab, [1] * 8, 4, nodes=False, penalties=False)
    s.rules = cw.logit_rules()
    x = np.zeros((8, vocab), np.float32)
    low = np.finfo(np.float32).min
    x[0, [vocab - 1, vocab // 2]] = 3.0        # equal: the lower index
    x[1] = -np.inf                             # nothing may follow
    x[2] = low                                 # the type's lowest value is a value
    x[3], x[3, vocab - 2] = -np.inf, low
    x[4, 7], x[4, 9] = np.nan, 1.0             # NaN is never the largest
    x[5] = np.nan
    x[6, 11] = np.inf
    x[7, 3], x[7, vocab - 1] = np.inf, np.inf
    got = s.run(x)
    assert np.array_equal(got[0], x, equal_nan=True)
    none = 0xffffffff
    assert got[1].tolist() == [vocab // 2, none, 0, vocab - 2, 9, none, 11, 3]
    assert got[2][1] == -np.inf and got[2][5] == -np.inf and got[2][3] == 0.0 and got[2][6] == 0.0
    assert np.isnan(got[2][4]) and np.isnan(got[2][7])
    assert abs(got[2][2] + np.log(vocab)) <= 4e-6 * np.log(vocab)


def test_what_is_not_allowed_does_not_reach_the_rest(ctx, rng):
    """NaN and infinities behind a mask, and a row whose grammar allows nothing."""
    vocab = 6000
    s = Step(ctx, rng, vocab, [1] * 4, 30, nodes=False, bias=20, masks=True)
    s.allowed_row = i32([1, 2, 3, 4])
    s.upload()
    x = draw(rng, 4, vocab)
    for i, bad in enumerate((np.nan, np.inf, np.nan, -np.inf)):
        bits = np.unpackbits(s.allowed[i + 1].view(np.uint8), bitorder="little")[:vocab]
        x[i, bits == 0] = bad
    got = s.run(x)
    s.check(x, got)
    assert got[1][2] == 0xffffffff and got[2][2] == -np.inf and np.all(got[0][2] == -np.inf)
    assert got[1][3] == vocab - 1 and got[2][3] == 0.0
    assert not np.any(np.isnan(got[2]))


def test_counts_are_whole(ctx, rng):
    """A token generated many times; in the prompt too; a last bias; exact steps."""
    vocab = 4500
    s = Step(ctx, rng, vocab, [2], 3000, spare=0)
    s.tokens[0] = 7
    s.tokens[0, :10] = [7, 8, 9, 4400, 4400, 1, 1, 1, 2, 3]
    s.length[0], s.prompt[0] = 3000, 5
    s.node = i32([8, 4400])
    s.repeat, s.presence, s.frequency = (np.array([v], np.float32) for v in (2.0, 0.5, 0.25))
    s.bias_first, s.bias_token = i32([0, 4]), i32([9, 2000, 9, 4499])
    s.bias = np.array([64.0, 3.0, -2.0, 1.5], np.float32)
    s.upload()
    x = rng.integers(-8, 9, (2, vocab)).astype(np.float32)
    got = s.run(x)
    for i in range(2):
        want, _ = s.reference(x, i, i)
        assert np.array_equal(got[0][i], want)
        assert got[1][i] == want.argmax()
    assert got[0][0][7] == (x[0, 7] / 2 if x[0, 7] > 0 else x[0, 7] * 2) - 0.5 - 2990 * 0.25
    # one node: generated once more in both rows or in the second alone
    assert got[0][1][4400] == (x[1, 4400] / 2 if x[1, 4400] > 0 else x[1, 4400] * 2) - 0.75


def test_bad_device_values_count_for_nothing(ctx, rng):
    """Lengths, list bounds and rows of requests out of their range."""
    s = Step(ctx, rng, 700, [2, 3, 1], 50, bias=6, masks=True)
    s.length[:] = [-5, 1 << 30, 20]
    s.prompt[:] = [3, -9, 1 << 30]
    s.upload()
    x = draw(rng, 6, 700)
    got = s.run(x)
    s.length[:] = [0, 50, 20]
    s.prompt[:] = [0, 0, 20]
    s.check(x, got)
    s.bias_first[1] = 1 << 30  # requests 0 and 1 have no list now
    s.upload()
    got = s.run(x)
    first = s.bias_first.copy()
    s.bias_first = i32([0, 0, first[2], first[3]])
    keep = s.bias_token.copy()
    s.bias_token = i32(np.where(np.arange(len(keep)) < first[2], -1, keep))
    s.check(x, got)
    good = s.first.copy()
    for first in ([0, 2, 1 << 30, 6], [-1, 2, 5, 6], [2, 1, 5, 6]):
        s.first = i32(first)
        s.upload()
        got = s.run(x)
        for i in range(6):
            owned = any(0 <= a <= i < z <= 6 for a, z in zip(first, first[1:]))
            assert (got[1][i] != 77) == owned
    s.first = good


def test_tokens_past_four_gigabytes(ctx, rng):
    """A request whose history lies past 2^32 bytes of the array."""
    max_len, n, vocab = 1 << 21, 520, 900
    big = ctx.empty((n, max_len), np.int32)
    hist = i32(rng.integers(0, vocab, 64))
    tail = cw.DeviceArray(ctx, (64,), np.int32, big.ptr + 4 * max_len * (n - 1))
    assert 4 * max_len * (n - 1) > 1 << 32
    tail.upload(hist)
    length = np.zeros(n, np.int32)
    length[n - 1] = 64
    first = np.zeros(n + 1, np.int32)
    first[n] = 1
    rules = cw.logit_rules(tokens=big, length=ctx.storage(length), max_len=max_len,
                           frequency=ctx.storage(np.full(n, 0.5, np.float32)))
    x = draw(rng, 1, vocab)
    out, token = ctx.empty((1, vocab)), ctx.empty(1, np.uint32)
    ctx.logits_rows(rules, cw.batch(None, n, 1, ctx.storage(first), None, 0), ctx.storage(x), 1,
                    vocab, out=out, token=token)
    want, bound = so.logits(x[0], hist, frequency=0.5)
    assert np.all(np.abs(out.download()[0] - want) <= bound)
    assert token.download()[0] == want.argmax()
    ctx.free(big)


def test_recorded(ctx, rng):
    """Replayed as histories, lengths and masks change on the device."""
    vocab = 9000
    s = Step(ctx, rng, vocab, [3, 2], 100, tree=True, bias=5, masks=True)
    x, out = ctx.empty((5, vocab)), ctx.empty((5, vocab))
    token, logprob = ctx.empty(5, np.uint32), ctx.empty(5)
    length, mask_row = ctx.empty(2, np.int32), ctx.empty(5, np.int32)
    s.rules.length, s.rules.allowed_row = length.ptr, mask_row.ptr

    def call():
        ctx.logits_rows(s.rules, s.batch, x, 5, vocab, out=out, token=token, logprob=logprob)
    length.upload(s.length), mask_row.upload(s.allowed_row), x.upload(draw(rng, 5, vocab))
    call()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()
    for _ in range(4):
        s.length, s.allowed_row = i32(rng.integers(0, 101, 2)), i32(rng.integers(-1, 6, 5))
        length.upload(s.length), mask_row.upload(s.allowed_row)
        h = draw(rng, 5, vocab)
        x.upload(h)
        ctx.argmax(x, 5 * vocab)  # other users of the scratch
        g.launch()
        got = out.download(), token.download(), logprob.download()
        s.check(h, got)
        call()
        for a, d in zip(got, (out, token, logprob)):
            assert np.array_equal(a, d.download())
    g.close()


def test_rows_of_many_requests(ctx, rng):
    """More requests than lanes, most without a row, and a table that does not ascend."""
    n, vocab = 9000, 500
    new = (rng.random(n) < 0.02).astype(int)
    new[[0, 64, n - 1]] = 1, 3, 2
    first = i32(np.concatenate([[0], np.cumsum(new)]))
    rows = int(first[-1]) + 3
    x = draw(rng, rows, vocab)
    frequency = rng.random(n).astype(np.float32)
    hist = i32(rng.integers(0, vocab, (n, 7)))
    rules = cw.logit_rules(tokens=ctx.storage(hist), length=ctx.storage(i32(np.full(n, 7))), max_len=7,
                           frequency=ctx.storage(frequency))
    for table in (first, np.concatenate([first[:1], first[:0:-1]])):  # the second: requests 0 only
        out = ctx.storage(np.full((rows, vocab), 7.5, np.float32))
        ctx.logits_rows(rules, cw.batch(None, n, rows, ctx.storage(i32(table)), None, 0), ctx.storage(x),
                        rows, vocab, out=out)
        got = out.download()
        for r in range(rows):
            own = [b for b in range(n) if table[b] <= r < table[b + 1]]
            if not own:
                assert np.all(got[r] == 7.5)
                continue
            want, bound = so.logits(x[r], hist[own[0]], frequency=float(frequency[own[0]]))
            assert np.all(np.abs(got[r] - want) <= 1.001 * bound)
