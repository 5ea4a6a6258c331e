"""The paged cache: decode attention over pages, copies between pages and dense planes, eviction -- against plain
restatements in 64 bits.  No counterpart in the reference, whose cache is one plane per sequence.

Tolerance of the attention, with u = 2^-24 (half a step of f32): a query element is off by at most 25 u of its rotation
pair's magnitude (norm: 11 u, sine and cosine and the rotation's three roundings: 8 u, two f16 that hold 22 bits: 6 u); a
score adds at most 17 products' partial sums and two factors, so with Z = scale * sum_i (|q_i| + |q_pair(i)|) |k_ji| it is
off by at most 46 u Z, a softmax weight by 2 * 46 u Z + 16 u of itself, and an output, whose sum runs over one step per 64
rows, the warps and the CTAs, by (100 Z + 80 + n / 16) u of sum_j P_j |v_j|.  The stored key is compared with its own
definition (half an f16 step) and then taken as it is."""
import numpy as np
import pytest

from tuckmill_b200 import cuda

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NONE = cuda.SEQ_NONE


def f32(buf, shape):
    return buf.download(0, int(np.prod(shape)) * 4, np.float32).reshape(shape)


def f16(buf, shape):
    return buf.download(0, int(np.prod(shape)) * 2, np.float16).reshape(shape)


def u32(buf, shape):
    return buf.download(0, int(np.prod(shape)) * 4, np.uint32).reshape(shape)


def status_of(buf):
    return int(buf.download(0, 4, np.uint32)[0])


class Paged:
    """A pool, its tables and one step's inputs, on the host and on the device.  Rows out of sight hold NaN and infinities,
    entries of pages that are not needed name none."""

    def __init__(self, ctx, lens, heads, kvh, hd, page, n_rot=None, window=0, dropped=0, weights=None, seed=0, pad=0,
                 max_pages=None, absent=()):
        g = np.random.default_rng(seed)
        self.ctx, self.lens, self.heads, self.kvh, self.hd, self.page = ctx, list(lens), heads, kvh, hd, page
        self.n_rot, self.window, self.S = n_rot or hd, window, len(lens)
        self.eps, self.scale = 1e-6, 1.0 / np.sqrt(np.float32(hd))
        live = [s for s in range(self.S) if s not in absent and lens[s] != NONE]
        need = {s: lens[s] // page + 1 for s in live}
        self.max_pages = max_pages or max(need.values()) + 1
        self.cap = self.max_pages * page
        live = [s for s in live if lens[s] < self.cap]
        self.live = live
        self.pages = sum(need[s] for s in live) + 3
        order = g.permutation(self.pages)
        self.table = np.full((self.S, self.max_pages), 0xFFFFFFFF, np.uint32)
        self.k = np.full((self.pages, kvh, page, hd), np.nan, np.float16)
        self.v = np.full((self.pages, kvh, page, hd), np.inf, np.float16)
        at = 0
        for s in live:
            for p in range(need[s]):
                self.table[s, p] = order[at]
                at += 1
        for s in live:
            lo = self.start(s)
            for p in range(lo // page):  # wholly before the window: given back
                self.table[s, p] = 0xFFFFFFFF
            for j in range(lo, lens[s]):
                self.k[self.table[s, j // page], :, j % page] = g.standard_normal((kvh, hd)).astype(np.float16)
                self.v[self.table[s, j // page], :, j % page] = g.standard_normal((kvh, hd)).astype(np.float16)
        self.width = (heads + 2 * kvh) * hd + pad
        self.qkv = g.standard_normal((self.S, self.width)).astype(np.float32)
        self.qn = (1 + 0.1 * g.standard_normal(hd)).astype(np.float32)
        self.kn = (1 + 0.1 * g.standard_normal(hd)).astype(np.float32)
        self.inv = (1e4 ** (-np.arange(self.n_rot // 2) * 2.0 / self.n_rot)).astype(np.float32)
        self.pos = np.array([0 if n == NONE else n + dropped for n in self.lens], np.uint32)
        self.w_in = None
        if weights:
            self.w_in = g.random((self.S, kvh, self.cap)).astype(np.float32)
        b = ctx.from_array
        self.bk, self.bv, self.btable = b(self.k), b(self.v), b(self.table)
        self.bqkv, self.bqn, self.bkn, self.binv = b(self.qkv), b(self.qn), b(self.kn), b(self.inv)
        self.bpos, self.blen = b(self.pos), b(np.array(self.lens, np.uint32))
        self.out0 = np.full((self.S, heads * hd), 7.5, np.float32)
        self.bout = b(self.out0)
        self.status = ctx.buffer(4, shared=True)
        self.status.zero()
        self.scratch = ctx.buffer(cuda.attention_paged_scratch_bytes(self.S, heads, kvh, hd, page, self.max_pages, bool(weights)))
        n = len(self.bqkv)
        self.views = [self.bqkv.view(o, n - o) for o in (0, heads * hd * 4, (heads + kvh) * hd * 4)]

    def start(self, s):
        n = self.lens[s] + 1
        return n - self.window if self.window and n > self.window else 0

    def call(self, w_in=None, w_out=None, **over):
        a = dict(q=self.views[0], k=self.views[1], v=self.views[2], q_norm=self.bqn, k_norm=self.bkn, inv_freq=self.binv,
                 k_pages=self.bk, v_pages=self.bv, table=self.btable, out=self.bout, scratch=self.scratch, pos_buf=self.bpos,
                 len_buf=self.blen, status=self.status, n_seq=self.S, heads=self.heads, kv_heads=self.kvh,
                 head_dim=self.hd, n_rot=self.n_rot, pages=self.pages, page_rows=self.page, max_pages=self.max_pages,
                 window=self.window, eps=self.eps, scale=self.scale, q_stride=self.width, kv_stride=self.width,
                 weights_in=w_in, weights_out=w_out)
        a.update(over)
        self.ctx.attention_decode_paged(**a)

    def turned(self, x, w, pos):
        """f64: x [heads][hd] normed and rotated, and the magnitude of each element's pair."""
        x = x.astype(np.float64)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + self.eps) * w
        angle = (np.float32(pos) * self.inv).astype(np.float64)
        h = self.n_rot // 2
        y, mag = x.copy(), np.abs(x)
        y[:, :h] = x[:, :h] * np.cos(angle) - x[:, h:2 * h] * np.sin(angle)
        y[:, h:2 * h] = x[:, :h] * np.sin(angle) + x[:, h:2 * h] * np.cos(angle)
        mag[:, :h] += np.abs(x[:, h:2 * h])
        mag[:, h:2 * h] += np.abs(x[:, :h])
        return y, mag

    def check(self, w_before=None, w_after=None, w_kept=None):
        """Outputs and pools after one call; with weights, what they were before and are now (`w_kept`: what the buffer
        held where the call leaves it)."""
        hd, kvh, group = self.hd, self.kvh, self.heads // self.kvh
        out, k, v = f32(self.bout, self.out0.shape), f16(self.bk, self.k.shape), f16(self.bv, self.v.shape)
        want_k, want_v = self.k.copy(), self.v.copy()
        for s in range(self.S):
            if s not in self.live:
                np.testing.assert_array_equal(out[s], self.out0[s])
                if w_after is not None:
                    np.testing.assert_array_equal(w_after[s], w_kept[s])
                continue
            n, lo = self.lens[s], self.start(s)
            x = self.qkv[s, :(self.heads + 2 * kvh) * hd].reshape(-1, hd)
            q, qmag = self.turned(x[:self.heads], self.qn, self.pos[s])
            kk, kmag = self.turned(x[self.heads:self.heads + kvh], self.kn, self.pos[s])
            page, row = self.table[s, n // self.page], n % self.page
            assert np.all(np.abs(k[page, :, row] - kk) <= 2.0 ** -11 * np.abs(kk) + 2.0 ** -25 + 25 * U * kmag)
            want_k[page, :, row] = k[page, :, row]
            want_v[page, :, row] = x[self.heads + kvh:].astype(np.float16)
            j = np.arange(lo, n + 1)
            keys = want_k[self.table[s, j // self.page], :, j % self.page].astype(np.float64)  # [rows][kvh][hd]
            vals = want_v[self.table[s, j // self.page], :, j % self.page].astype(np.float64)
            for h in range(kvh):
                qs = q[h * group:(h + 1) * group]
                z = qs @ keys[:, h].T * float(self.scale)
                Z = abs(float(self.scale)) * (qmag[h * group:(h + 1) * group] @ np.abs(keys[:, h]).T).max(-1)
                p = np.exp(z - z.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                got = out[s].reshape(self.heads, hd)[h * group:(h + 1) * group]
                tol = (100 * Z + 80 + len(j) / 16)[:, None] * U * (p @ np.abs(vals[:, h]))
                bad = np.abs(got - p @ vals[:, h]) / (tol + 1e-30)
                assert np.all(np.abs(got - p @ vals[:, h]) <= tol), f"sequence {s}, KV head {h}: {bad.max():.2f} tolerances"
                if w_after is not None:
                    w = np.zeros(n + 1)
                    w[:n] = w_before[s, h, :n]
                    w[lo:] += p.sum(0)
                    tol = U * (w + (100 * Z.max() + 80) * np.concatenate([np.zeros(lo), p.sum(0)]))
                    assert np.all(np.abs(w_after[s, h, :n + 1] - w) <= tol), f"weights of sequence {s}, KV head {h}"
                    np.testing.assert_array_equal(w_after[s, h, n + 1:], w_kept[s, h, n + 1:])
        np.testing.assert_array_equal(k.view(np.uint16), want_k.view(np.uint16))
        np.testing.assert_array_equal(v.view(np.uint16), want_v.view(np.uint16))


CASES = [
    # lens, heads, kvh, hd, page, more
    ([0], 1, 1, 128, 16, {}),
    ([0, 1, 15, 16, 17], 16, 8, 128, 16, {}),
    ([63, 64, 65, 127, 128, 129, 3], 4, 2, 64, 64, {}),
    ([700, 5, 300], 32, 8, 128, 128, {"dropped": 900}),
    ([2500], 8, 8, 128, 32, {}),
    ([1000, 0, 77], 5, 1, 256, 16, {"n_rot": 128}),
    ([333, 90], 4, 1, 256, 256, {"window": 100}),
    ([50, 200, 31, 32], 8, 4, 32, 32, {"window": 1}),
    ([600, 40, 16, 17], 6, 2, 128, 16, {"window": 17, "pad": 3}),
    ([150, 260], 20, 2, 64, 16, {"n_rot": 2}),  # ten heads a KV head: two blocks of columns
    ([90, 10], 32, 1, 128, 64, {"pad": 5}),
    ([40, 41], 17, 1, 32, 16, {}),
    ([i * 7 % 130 for i in range(70)], 4, 4, 64, 16, {}),
    ([20, NONE, 33], 4, 2, 128, 16, {}),
    # many heads in all: the join's uncut form, at every head size
    ([(i * 37) % 200 for i in range(40)], 8, 2, 128, 32, {}),
    ([(i * 53) % 150 for i in range(40)], 8, 1, 256, 16, {"window": 70}),
    ([(i * 11) % 90 for i in range(80)], 4, 4, 32, 16, {}),
    ([(i * 29) % 300 for i in range(160)], 2, 2, 64, 64, {"dropped": 5}),
    # more heads in all than find a place at once
    ([(i * 37) % 70 for i in range(75)], 8, 4, 32, 16, {}),
    ([(i * 37) % 90 for i in range(75)], 8, 2, 64, 32, {}),
    ([(i * 41) % 90 for i in range(75)], 8, 1, 128, 16, {}),
    ([(i * 43) % 70 for i in range(75)], 8, 2, 256, 16, {}),
    # pairs in many pieces
    ([1300], 4, 2, 32, 16, {}),
    ([1290, 30], 4, 1, 64, 16, {}),
    ([1500], 6, 2, 256, 64, {"dropped": 40}),
]
LONG = [  # pairs in many pieces, and many stretches of weights
    ([38000], 8, 8, 32, 256),
    ([38000], 16, 8, 64, 128),
    ([37000], 8, 8, 128, 64),
    ([31000], 8, 8, 256, 256),
]


@pytest.mark.parametrize("lens,heads,kvh,hd,page,more", CASES)
def test_attention_over_pages(ctx, lens, heads, kvh, hd, page, more):
    t = Paged(ctx, lens, heads, kvh, hd, page, **more)
    t.call()
    ctx.fence()
    assert status_of(t.status) == 0
    t.check()
    before = f32(t.bout, t.out0.shape).copy()
    t.call()  # the same step again: the same bits
    ctx.fence()
    np.testing.assert_array_equal(f32(t.bout, t.out0.shape), before)


@pytest.mark.parametrize("lens,heads,kvh,hd,page,more", CASES)
def test_attention_weights_are_counted(ctx, lens, heads, kvh, hd, page, more):
    t = Paged(ctx, lens, heads, kvh, hd, page, weights=True, seed=3, **more)
    held = np.full(t.w_in.shape, 0.25, np.float32)
    w_in, w_out = ctx.from_array(t.w_in), ctx.from_array(held)
    t.call(w_in, w_out)
    ctx.fence()
    t.check(t.w_in, f32(w_out, t.w_in.shape), held)
    np.testing.assert_array_equal(f32(w_in, t.w_in.shape), t.w_in)
    t.call(w_in, w_in)  # in place
    ctx.fence()
    t.check(t.w_in, f32(w_in, t.w_in.shape), t.w_in)
    w_out.upload(0, held)
    t.call(None, w_out)  # from zero
    ctx.fence()
    t.check(np.zeros_like(t.w_in), f32(w_out, t.w_in.shape), held)


@pytest.mark.parametrize("lens,heads,kvh,hd,page", LONG)
def test_attention_weights_of_long_sequences(ctx, lens, heads, kvh, hd, page):
    t = Paged(ctx, lens, heads, kvh, hd, page, weights=True)
    held = np.full(t.w_in.shape, 0.25, np.float32)
    w_in, w_out = ctx.from_array(t.w_in), ctx.from_array(held)
    t.call(w_in, w_out)
    ctx.fence()
    t.check(t.w_in, f32(w_out, t.w_in.shape), held)


def test_scale_of_either_sign_and_zero(ctx):
    for scale in (-0.3, 0.0, 2.0):
        t = Paged(ctx, [100, 3], 4, 2, 64, 16, seed=5)
        t.scale = scale
        t.call()
        ctx.fence()
        t.check()


def test_queries_of_any_size(ctx):
    """Norm weights that put queries far outside binary16."""
    for factor in (1e-9, 1e9):
        t = Paged(ctx, [100, 3], 4, 2, 64, 16, seed=6)
        t.qn = (t.qn * factor).astype(np.float32)
        t.bqn.upload(0, t.qn)
        t.scale = float(np.float32(0.125 / factor))
        t.call()
        ctx.fence()
        t.check()


@pytest.mark.parametrize("hd,heads,kvh,more", [(32, 8, 2, {}), (64, 16, 1, {"window": 150}), (128, 8, 2, {}), (256, 12, 4, {})])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinities_and_nan_in_sight(ctx, hd, heads, kvh, more, bad):
    """One in a key makes NaN of the heads that read it and of the weights that they count, one in a value of its own
    dimension of their outputs; all else has the bits that it has without."""
    group = heads // kvh
    for of_key in (True, False):
        t = Paged(ctx, [200, 70, 3], heads, kvh, hd, 16, weights=True, seed=13, **more)
        w_in, w_out = ctx.from_array(t.w_in), ctx.from_array(np.zeros_like(t.w_in))
        t.call(w_in, w_out)
        ctx.fence()
        t.check(t.w_in, f32(w_out, t.w_in.shape), np.zeros_like(t.w_in))
        want, want_w = f32(t.bout, t.out0.shape).copy().reshape(3, heads, hd), f32(w_out, t.w_in.shape).copy()
        for s, h, j, d in ((0, 0, 137, 5), (1, kvh - 1, 69, hd - 1), (2, 0, 0, 0)):
            t.k[t.table[s, j // 16], h, j % 16, d] = bad if of_key else t.k[t.table[s, j // 16], h, j % 16, d]
            t.v[t.table[s, j // 16], h, j % 16, d] = t.v[t.table[s, j // 16], h, j % 16, d] if of_key else bad
            if of_key:
                want[s, h * group:(h + 1) * group] = np.nan
                want_w[s, h, t.start(s):t.lens[s] + 1] = np.nan
            else:
                want[s, h * group:(h + 1) * group, d] = np.nan
        t.bk.upload(0, t.k)
        t.bv.upload(0, t.v)
        t.call(w_in, w_out)
        ctx.fence()
        np.testing.assert_array_equal(f32(t.bout, t.out0.shape).reshape(want.shape), want)
        np.testing.assert_array_equal(f32(w_out, t.w_in.shape), want_w)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_small_elements_of_a_query_beside_large_ones(ctx, hd):
    """Two elements of every query are 2^14 times the others, and meet zeros in every key: the small ones alone make the
    scores."""
    t = Paged(ctx, [3, 200], 4, 2, hd, 16, n_rot=2, seed=14)
    t.qn[:2], t.kn[:2] = 2.0 ** 14, 0
    t.k[..., :2] = 0
    for b, x in ((t.bqn, t.qn), (t.bkn, t.kn), (t.bk, t.k)):
        b.upload(0, x)
    t.call()
    ctx.fence()
    t.check()


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("octaves", [24.4, 30.7, 37.3])
def test_small_weights_beside_a_large_one(ctx, hd, octaves):
    """One row weighs 2^octaves times each of the others and its value is zero: the small weights alone make the output."""
    t = Paged(ctx, [300], 1, 1, hd, 16, n_rot=2, seed=15)
    q = t.turned(t.qkv[0, :hd].reshape(1, hd), t.qn, t.pos[0])[0][0]
    t.kn[:] = 0
    for j in range(300):
        t.k[t.table[0, j // 16], 0, j % 16] = 0
    t.k[t.table[0, 0], 0, 7] = octaves * np.log(2) / float(t.scale) / (q @ q) * q
    t.v[t.table[0, 0], 0, 7] = 0
    for b, x in ((t.bkn, t.kn), (t.bk, t.k), (t.bv, t.v)):
        b.upload(0, x)
    t.call()
    ctx.fence()
    t.check()


@pytest.mark.parametrize("hd,kvh", [(32, 32), (64, 16), (128, 8), (256, 4)])
def test_the_stored_key_is_right_in_every_bit(ctx, hd, kvh):
    """The new key in f16 is the definition's value in 64 bits, held in f32 and rounded to f16."""
    t = Paged(ctx, [i % 20 for i in range(64)], kvh, kvh, hd, 16, dropped=70001, seed=16)
    t.call()
    ctx.fence()
    k = f16(t.bk, t.k.shape)
    for s, n in enumerate(t.lens):
        want, _ = t.turned(t.qkv[s, kvh * hd:2 * kvh * hd].reshape(kvh, hd), t.kn, t.pos[s])
        np.testing.assert_array_equal(k[t.table[s, n // 16], :, n % 16], want.astype(np.float32).astype(np.float16))


def test_a_full_sequence_and_a_bad_page(ctx):
    t = Paged(ctx, [64, 30, 20], 4, 2, 64, 16, max_pages=4, seed=7)
    t.call()
    ctx.fence()
    assert status_of(t.status) == cuda.STATUS_PAST_CAPACITY
    assert t.live == [1, 2]
    t.check()
    # a page that is not there: its rows are zeros, the others are served as ever
    t = Paged(ctx, [70, 30], 4, 2, 64, 16, seed=8)
    gone = t.table[0, 2]
    t.table[0, 2] = t.pages
    t.btable.upload(0, t.table)
    t.call()
    ctx.fence()
    assert status_of(t.status) == cuda.STATUS_BAD_PAGE
    np.testing.assert_array_equal(f16(t.bk, t.k.shape)[gone].view(np.uint16), t.k[gone].view(np.uint16))
    t.table[0, 2] = gone
    t.k[gone] = t.v[gone] = 0
    t.bk.upload(gone * t.k[0].nbytes, t.k[gone])
    t.bv.upload(gone * t.v[0].nbytes, t.v[gone])
    t.check()
    # the new row's own page is not there: nothing is stored, the row is zeros like the page's others
    t = Paged(ctx, [17], 2, 2, 64, 16, seed=9)
    page = t.table[0, 1]
    t.k[page, :, 0] = t.v[page, :, 0] = 0
    t.bk.upload(0, t.k)
    t.bv.upload(0, t.v)
    t.btable.upload(4, np.array([0xFFFFFFFE], np.uint32))
    t.call()
    ctx.fence()
    assert status_of(t.status) == cuda.STATUS_BAD_PAGE
    np.testing.assert_array_equal(f16(t.bk, t.k.shape).view(np.uint16), t.k.view(np.uint16))
    t.k[page], t.v[page] = 0, 0  # keys of zeros weigh exp(0) each
    out = f32(t.bout, (2, 64))
    q, qmag = t.turned(t.qkv[0].reshape(-1, 64)[:2], t.qn, t.pos[0])
    for h in range(2):
        keys, vals = [np.concatenate([x[t.table[0, 0], h], x[page, h, :2]]).astype(np.float64) for x in (t.k, t.v)]
        p = np.exp(keys @ q[h] * float(t.scale))
        Z = float(t.scale) * (np.abs(keys) @ qmag[h]).max()
        assert np.all(np.abs(out[h] - p @ vals / p.sum()) <= (100 * Z + 82) * U * (p @ np.abs(vals) / p.sum()))


def test_a_recorded_step_grows_its_sequences(ctx):
    """One graph, replayed: lengths and positions advance on the device; equals the calls one by one."""
    def fresh():
        return Paged(ctx, [14, 60, NONE, 0], 4, 2, 128, 16, seed=11, max_pages=8)
    a, b = fresh(), fresh()
    spare = [p for p in range(a.pages) if p not in a.table]
    a.table[0, 1], a.table[1, 4] = spare[0], spare[1]
    for t in (a, b):
        t.btable.upload(0, a.table)
    got, want = [], []
    for i in range(4):
        a.call()
        ctx.fence()
        want.append(f32(a.bout, a.out0.shape).copy())
        a.blen.upload(0, np.array([15 + i, 61 + i, NONE, 1 + i], np.uint32))
        a.bpos.upload(0, np.array([15 + i, 61 + i, 0, 1 + i], np.uint32))
    ctx.begin_group()
    b.call()
    ctx.u32_add(b.blen, 0, 1)
    ctx.u32_add(b.blen, 1, 1)
    ctx.u32_add(b.blen, 3, 1)
    for s in (0, 1, 3):
        ctx.u32_add(b.bpos, s, 1)
    graph = ctx.end_group_retain()
    for i in range(4):
        graph.launch()
        ctx.fence()
        got.append(f32(b.bout, b.out0.shape).copy())
    graph.free()
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x, y)
    np.testing.assert_array_equal(f16(a.bk, a.k.shape).view(np.uint16), f16(b.bk, b.k.shape).view(np.uint16))


def test_pages_shared_by_a_prefix(ctx):
    """Two sequences read the same pages and store into their own."""
    t = Paged(ctx, [40, 45], 4, 2, 64, 16, seed=12)
    t.table[1, :2] = t.table[0, :2]
    t.btable.upload(0, t.table)
    t.call()
    ctx.fence()
    t.check()


def test_attention_refusals(ctx):
    t = Paged(ctx, [20, 3], 4, 2, 64, 16, weights=True)
    w = ctx.from_array(t.w_in)
    for over in (dict(head_dim=96), dict(head_dim=0), dict(page_rows=24), dict(page_rows=8), dict(heads=3), dict(heads=0),
                 dict(kv_heads=0), dict(heads=66), dict(n_rot=0), dict(n_rot=3), dict(n_rot=66), dict(n_seq=0),
                 dict(n_seq=1025), dict(n_seq=3), dict(pages=0), dict(max_pages=0), dict(pages=t.pages + 1),
                 dict(max_pages=t.max_pages + 1), dict(q_stride=1), dict(kv_stride=1), dict(q_stride=2 * t.width),
                 dict(weights_in=w), dict(max_pages=1 << 22), dict(pages=1 << 30)):
        with pytest.raises(cuda.CudaError) as e:
            t.call(**over)
        assert e.value.code in (-4, -5), over
    small = ctx.buffer(64)
    for over in (dict(out=small), dict(scratch=small), dict(k_pages=small), dict(v_pages=small), dict(table=ctx.buffer(4)),
                 dict(pos_buf=ctx.buffer(4)), dict(len_buf=ctx.buffer(4)), dict(weights_out=small)):
        with pytest.raises(cuda.CudaError):
            t.call(**over)
    # storage shared with what the call writes
    for over in (dict(out=t.bqkv), dict(v_pages=t.bk), dict(status=t.blen), dict(out=t.scratch), dict(weights_out=t.scratch),
                 dict(weights_in=w.view(16, len(w) - 16), weights_out=w)):
        with pytest.raises(cuda.CudaError) as e:
            t.call(**over)
        assert e.value.code in (-4, -5), over
    t.call(w_out=w)
    ctx.fence()


def test_a_pool_past_four_gigabytes(ctx):
    """Pages whose byte offsets pass 32 bits: what is stored, read, copied and moved there is what lies there."""
    heads, kvh, hd, page, pages, n = 4, 1, 256, 256, 33000, 300
    big = [ctx.buffer(pages * kvh * page * hd * 2) for _ in range(2)]
    size = kvh * page * hd * 2
    t = Paged(ctx, [n], heads, kvh, hd, page, seed=31, weights=True)
    ids = np.array([[32999, 32800, 5]], np.uint32)[:, :t.max_pages]
    for b, x in zip(big, (t.k, t.v)):
        for j in range(2):
            b.upload(int(ids[0, j]) * size, x[t.table[0, j]])
    table = ctx.from_array(ids)
    w = ctx.from_array(t.w_in)
    t.call(w, w, k_pages=big[0], v_pages=big[1], table=table, pages=pages)
    ctx.fence()
    for b, own in zip(big, (t.bk, t.bv)):  # the small pool gets what the large one holds now
        for j in range(2):
            own.upload(int(t.table[0, j]) * size, b.download(int(ids[0, j]) * size, size))
    t.check(t.w_in, f32(w, t.w_in.shape), t.w_in)
    # out to a dense plane, and back into other high pages
    dense = [ctx.buffer(kvh * 512 * hd * 2) for _ in range(2)]
    high = ctx.from_array(np.array([[32998, 32000, 7]], np.uint32)[:, :t.max_pages])
    for tb, to_pages in ((table, False), (high, True)):
        ctx.kv_pages_copy(dense[0], dense[1], big[0], big[1], tb, t.status, pages, page, t.max_pages, kvh, hd, 512, to_pages,
                          [(0, 0, 0, n)])
    ctx.fence()
    for b in big:
        np.testing.assert_array_equal(b.download(32998 * size, size), b.download(32999 * size, size))
        np.testing.assert_array_equal(b.download(32000 * size, (n - page) * hd * 2), b.download(32800 * size, (n - page) * hd * 2))
    kept, length = ctx.buffer(kvh * 40 * 4), ctx.from_array(np.array([n], np.uint32))
    before = [b.download(int(i) * size, size, np.uint16).reshape(page, hd) for b in big for i in ids[0, :2]]
    total = f32(w, t.w_in.shape).copy()
    ctx.kv_pages_evict(big[0], big[1], table, high, length, length, w, w, kept, t.status, 1, kvh, hd, pages, page, t.max_pages,
                       40, 2, 3)
    ctx.fence()
    rows = evicted([n], total, 40, 2, 3)[0, 0]
    np.testing.assert_array_equal(u32(kept, (40,)), rows)
    for x, b in enumerate(big):
        whole = np.concatenate(before[2 * x:2 * x + 2])
        np.testing.assert_array_equal(b.download(32998 * size, 40 * hd * 2, np.uint16).reshape(40, hd), whole[rows])
    assert status_of(t.status) == 0


def test_as_many_sequences_as_a_call_takes(ctx):
    """1024 short sequences, most of them absent."""
    g = np.random.default_rng(5)
    lens = [NONE if i % 3 else int(g.integers(0, 40)) for i in range(1024)]
    t = Paged(ctx, lens, 2, 1, 64, 16, seed=41)
    t.call()
    ctx.fence()
    assert status_of(t.status) == 0
    t.check()


def test_operands_that_are_views(ctx):
    """Every operand a view 16 bytes into a larger buffer."""
    t = Paged(ctx, [70, 3, 200], 6, 2, 64, 16, weights=True, seed=51)

    def inside(b):
        whole = ctx.buffer(len(b) + 48)
        v = whole.view(16, len(b))
        v.upload(0, b.download(0, len(b)))
        return v

    names = dict(k_pages="bk", v_pages="bv", table="btable", out="bout", pos_buf="bpos", len_buf="blen", q_norm="bqn", k_norm="bkn",
                 inv_freq="binv")
    for n in names.values():
        setattr(t, n, inside(getattr(t, n)))
    w = inside(ctx.from_array(t.w_in))
    t.scratch = ctx.buffer(len(t.scratch) + 16).view(16, len(t.scratch))
    t.call(w, w)
    ctx.fence()
    t.check(t.w_in, f32(w, t.w_in.shape), t.w_in)


def steps(ctx, how):
    """A prompt into its pages, two tokens, an eviction in place, another token and its choice: one operator after the other,
    each reading what the one before it has just written."""
    t = Paged(ctx, [40, 25], 8, 2, 64, 16, weights=True, max_pages=6, seed=61)
    g = np.random.default_rng(61)
    spare = [p for p in range(t.pages) if p not in t.table]
    t.table[0, 3:5], t.table[1, 2] = t.table[0, 2], spare[0]
    table = np.arange(12, dtype=np.uint32).reshape(2, 6)
    pool = np.zeros((12, 2, 16, 64), np.float16)
    k, v = ctx.from_array(pool), ctx.from_array(pool)
    dense = [ctx.from_array(g.standard_normal((2, 2, 48, 64)).astype(np.float16)) for _ in range(2)]
    btable, blen, bpos = ctx.from_array(np.full((2, 6), 99, np.uint32)), ctx.from_array(np.zeros(2, np.uint32)), ctx.from_array(np.zeros(2, np.uint32))
    w, kept = ctx.from_array(np.zeros((2, 2, 96), np.float32)), ctx.buffer(2 * 2 * 20 * 4)
    scratch = ctx.buffer(cuda.attention_paged_scratch_bytes(2, 8, 2, 64, 16, 6, True))
    log, spot = ctx.from_array(np.zeros((2, 8), np.uint32)), ctx.from_array(np.zeros(2, np.uint32))
    partial, pen = ctx.buffer(2 * cuda.LOGITS_PARTIAL_BYTES), ctx.from_array(np.array([[1.5, 0.1, 0.2]] * 2, np.float32))
    y = ctx.buffer(2 * 512 * 4)
    y.zero()
    ctx.fence()
    attend = dict(k_pages=k, v_pages=v, table=btable, len_buf=blen, pos_buf=bpos, scratch=scratch, pages=12, max_pages=6)

    def ops():
        yield lambda: btable.store_u32(table.reshape(-1))
        yield lambda: ctx.kv_pages_copy(dense[0], dense[1], k, v, btable, t.status, 12, 16, 6, 2, 64, 48, True, [(0, 0, 0, 40), (1, 1, 0, 25)])
        yield lambda: blen.store_u32([40, 25])
        yield lambda: bpos.store_u32([40, 25])
        for i in range(2):
            yield lambda: t.call(w, w, **attend)
            for b in (blen, bpos):
                yield lambda b=b: ctx.u32_add_sat(b, 0, 2, 1, 95)
        yield lambda: ctx.kv_pages_evict(k, v, btable, btable, blen, blen, w, w, kept, t.status, 2, 2, 64, 12, 16, 6, 20, 2, 4)
        yield lambda: t.call(w, w, **attend)
        yield lambda: ctx.logits_adjust_rows(t.bout, y, 2, 512, log, 8, 0, spot, pen, partial=partial)
        yield lambda: ctx.u32_add_sat(spot, 0, 2, 1, 7)
        yield lambda: ctx.logits_adjust_rows(y, y, 2, 512, log, 8, 0, spot, pen, partial=partial)

    if how in ("group", "burst"):
        ctx._call("begin_" + how)
    for op in ops():
        op()
        if how == "fence":
            ctx.fence()
    if how in ("group", "burst"):
        ctx._call("end_" + how)
    ctx.fence()
    return [k, v, w, kept, blen, t.bout, y, log, t.status]


def test_operators_one_after_the_other_see_each_others_results(ctx):
    alone = [b.download(0, len(b)) for b in steps(ctx, "fence")]
    assert int(alone[-1].view(np.uint32)[0]) == 0
    for how in ("queued", "group", "burst"):
        for x, b in zip(alone, steps(ctx, how)):
            np.testing.assert_array_equal(b.download(0, len(b)), x, err_msg=how)


def test_two_contexts_at_once(ctx):
    """A second context's calls on the same device, neither waiting for the other."""
    other = cuda.CudaContext(0)
    try:
        cases = [Paged(c, [900, 50, 333], 8, 2, 128, 32, weights=True, seed=71) for c in (ctx, other)]
        ws = [c.ctx.from_array(c.w_in) for c in cases]
        for c in cases:
            c.ctx.fence()
        for _ in range(5):
            for c, w in zip(cases, ws):
                c.call(w, w)
        for c in cases:
            c.ctx.fence()
        for a, b in ((cases[0].bout, cases[1].bout), (cases[0].bk, cases[1].bk), (ws[0], ws[1])):
            np.testing.assert_array_equal(a.download(0, len(a)), b.download(0, len(b)))
        with pytest.raises(cuda.CudaError):  # one context's buffer in another's call
            cases[0].call(out=cases[1].bout)
        del cases, ws, a, b, c, w
    finally:
        import gc
        gc.collect()
        other.close()


# ---------------------------------------------------------------- copies

@pytest.mark.parametrize("hd,page,kvh", [(32, 16, 3), (64, 256, 1), (128, 32, 2), (256, 64, 2)])
def test_runs_move_between_planes_and_pages(ctx, hd, page, kvh):
    g = np.random.default_rng(1)
    cap, max_pages, pages = 300, 300 // page + 1, 60
    runs = [(0, 2, 0, 300), (2, 0, 7, 1), (1, 1, 16, 65), (1, 1, 200, 100), (2, 3, 63, 2)]
    table = g.permutation(4 * max_pages).reshape(4, max_pages).astype(np.uint32) % pages if 4 * max_pages > pages else \
        g.permutation(pages)[:4 * max_pages].reshape(4, max_pages).astype(np.uint32)
    if 4 * max_pages > pages:  # every entry its own page
        pages = 4 * max_pages
        table = g.permutation(pages).reshape(4, max_pages).astype(np.uint32)
    dense = [g.integers(0, 65536, (3, kvh, cap, hd), dtype=np.uint16) for _ in range(2)]
    pool = [g.integers(0, 65536, (pages, kvh, page, hd), dtype=np.uint16) for _ in range(2)]
    status = ctx.buffer(4, shared=True)
    status.zero()
    for to_pages in (True, False):
        bd, bp = [ctx.from_array(x) for x in dense], [ctx.from_array(x) for x in pool]
        ctx.kv_pages_copy(bd[0], bd[1], bp[0], bp[1], ctx.from_array(table), status, pages, page, max_pages, kvh, hd, cap,
                          to_pages, runs)
        ctx.fence()
        for i in range(2):
            d, p = dense[i].copy(), pool[i].copy()
            for seq, at, lo, n in runs:
                for j in range(lo, lo + n):
                    if to_pages:
                        p[table[at, j // page], :, j % page] = dense[i][seq, :, j]
                    else:
                        d[seq, :, j] = pool[i][table[at, j // page], :, j % page]
            np.testing.assert_array_equal(bd[i].download(0, d.nbytes, np.uint16).reshape(d.shape), d)
            np.testing.assert_array_equal(bp[i].download(0, p.nbytes, np.uint16).reshape(p.shape), p)
    assert status_of(status) == 0
    # a page that is not there: zeros come out of it, nothing goes in
    bad = table.copy()
    bad[1, 16 // page] = pages
    bd, bp = [ctx.from_array(x) for x in dense], [ctx.from_array(x) for x in pool]
    ctx.kv_pages_copy(bd[0], bd[1], bp[0], bp[1], ctx.from_array(bad), status, pages, page, max_pages, kvh, hd, cap, True,
                      [(1, 1, 16, 1)])
    ctx.fence()
    assert status_of(status) == cuda.STATUS_BAD_PAGE
    np.testing.assert_array_equal(bp[0].download(0, pool[0].nbytes, np.uint16).reshape(pool[0].shape), pool[0])
    ctx.kv_pages_copy(bd[0], bd[1], bp[0], bp[1], ctx.from_array(bad), status, pages, page, max_pages, kvh, hd, cap, False,
                      [(1, 1, 16, 1)])
    ctx.fence()
    assert np.all(bd[0].download(0, dense[0].nbytes, np.uint16).reshape(dense[0].shape)[1, :, 16] == 0)


def test_copy_refusals(ctx):
    kvh, hd, page, cap, pages, max_pages = 2, 64, 16, 64, 10, 4
    d = [ctx.buffer(2 * kvh * cap * hd * 2) for _ in range(2)]
    p = [ctx.buffer(pages * kvh * page * hd * 2) for _ in range(2)]
    table, status = ctx.buffer(2 * max_pages * 4), ctx.buffer(4)
    table.zero()

    def call(runs=((0, 0, 0, 4),), to_pages=True, dk=d[0], dv=d[1], pk=p[0], pv=p[1], tb=table, st=status, pages=pages,
             page=page, max_pages=max_pages, kvh=kvh, hd=hd, cap=cap):
        ctx.kv_pages_copy(dk, dv, pk, pv, tb, st, pages, page, max_pages, kvh, hd, cap, to_pages, list(runs))

    for over in (dict(runs=()), dict(runs=[(0, 0, 0, 1)] * 65), dict(runs=[(0, 0, 0, 0)]), dict(runs=[(0, 0, 61, 4)]),
                 dict(runs=[(2, 0, 0, 1)]), dict(runs=[(0, 2, 0, 1)]), dict(runs=[(0xFFFFFFFF, 0, 0, 1)]),
                 dict(runs=[(0, 0, 0, 5), (1, 0, 4, 2)]), dict(runs=[(0, 0, 0, 5), (0, 1, 4, 2)], to_pages=False),
                 dict(cap=0), dict(hd=48), dict(page=17), dict(kvh=0), dict(pages=0), dict(pages=11), dict(max_pages=0),
                 dict(pk=p[1]), dict(dk=d[1], to_pages=False), dict(dk=p[0]), dict(st=table),
                 dict(runs=[(0xFFFFFFFE, 0, 0, 1)]), dict(runs=[(0, 0, 0xFFFFFFFF, 2)])):
        with pytest.raises(cuda.CudaError) as e:
            call(**over)
        assert e.value.code in (-4, -5), over
    for runs in ([(0, 0, 5)], [(0, 0, 0, 5), (1, 1)]):
        with pytest.raises(ValueError):
            call(runs=runs)
    call(runs=[(0, 0, 0, 5), (0, 1, 4, 2)])  # one dense row into two sequences is fine
    ctx.fence()


# ---------------------------------------------------------------- eviction

def evicted(lens, w, keep, first, recent):
    """kept [S][kvh][keep] by the definition: sort by (held first, weight, row)."""
    S, kvh = w.shape[:2]
    kept = np.full((S, kvh, keep), NONE, np.uint32)
    for s, n in enumerate(lens):
        for h in range(kvh):
            if n <= keep:
                rows = list(range(n))
            else:
                mid = sorted(range(first, n - recent),
                             key=lambda j: (1, 0.0, j) if np.isnan(w[s, h, j]) else (0, -float(w[s, h, j]), j))
                rows = sorted(list(range(first)) + mid[:keep - first - recent] + list(range(n - recent, n)))
            kept[s, h, :len(rows)] = rows
    return kept


EVICT = [
    # lens, kvh, hd, page, keep, first, recent
    ([100, 40, 7], 2, 64, 16, 40, 4, 8),
    ([33], 1, 128, 16, 1, 0, 0),
    ([33], 1, 128, 16, 1, 1, 0),
    ([70, 71], 3, 32, 32, 70, 10, 60),
    ([1500, 1400, 800], 2, 128, 64, 700, 0, 0),
    ([300, 0, 257], 1, 256, 256, 256, 3, 100),
    ([5000], 2, 64, 128, 2100, 4, 64),
    ([9000, 4096, 4097, 3000], 1, 32, 256, 2500, 1, 70),  # on both sides of what registers hold
    ([3000], 1, 32, 64, 1500, 0, 0),
    # few heads, long sequences: a cluster of 8, 4 or 2 CTAs a head, weights in its registers or read again
    ([20000, 0, 2049, 900], 2, 32, 256, 8000, 5, 33),
    ([32768], 1, 32, 256, 5000, 0, 0),
    ([40000, 32769, 100, 4100], 1, 32, 256, 6000, 0, 100),
    ([33000], 1, 32, 256, 700, 300, 400),
    ([16384, 16390], 20, 32, 256, 300, 3, 7),
    ([9000, 8192, 4097], 25, 32, 128, 257, 3, 7),
    ([4200], 150, 32, 256, 30, 1, 2),  # more heads than that: one CTA each
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,kvh,hd,page,keep,first,recent", EVICT)
def test_rows_that_drew_least_are_evicted(ctx, lens, kvh, hd, page, keep, first, recent, in_place):
    g = np.random.default_rng(2)
    S, max_pages = len(lens), max(max(lens), keep) // page + 1
    cap = max_pages * page
    pages = (1 if in_place else 2) * S * max_pages + 1
    order = g.permutation(pages).astype(np.uint32)
    table = order[:S * max_pages].reshape(S, max_pages).copy()
    to = table if in_place else order[S * max_pages:2 * S * max_pages].reshape(S, max_pages).copy()
    pool = [g.integers(0, 65536, (pages, kvh, page, hd), dtype=np.uint16) for _ in range(2)]
    w = np.round(g.random((S, kvh, cap)) ** 6, 2).astype(np.float32)  # many ties, many zeros
    w[g.random(w.shape) < 0.05] = -0.0
    w[g.random(w.shape) < 0.02] = np.nan
    w[g.random(w.shape) < 0.02] = np.inf
    w[g.random(w.shape) < 0.02] = -np.inf
    w[g.random(w.shape) < 0.02] = -1.5
    held = np.full(w.shape, 0.125, np.float32)
    bk, bv = ctx.from_array(pool[0]), ctx.from_array(pool[1])
    btable = ctx.from_array(table)
    bto = btable if in_place else ctx.from_array(to)
    blen = ctx.from_array(np.array(lens, np.uint32))
    blen_out = blen if in_place else ctx.from_array(np.zeros(S, np.uint32))
    bw = ctx.from_array(w)
    bw_out = bw if in_place else ctx.from_array(held)
    kept, status = ctx.buffer(S * kvh * keep * 4), ctx.buffer(4, shared=True)
    status.zero()
    ctx.kv_pages_evict(bk, bv, btable, bto, blen, blen_out, bw, bw_out, kept, status, S, kvh, hd, pages, page, max_pages,
                       keep, first, recent)
    ctx.fence()
    assert status_of(status) == 0
    want = evicted(lens, w, keep, first, recent)
    np.testing.assert_array_equal(u32(kept, want.shape), want)
    np.testing.assert_array_equal(u32(blen_out, (S,)), np.minimum(lens, keep))
    want_w = (w if in_place else held).copy()
    want_pool = [p.copy() for p in pool]
    for s, n in enumerate(lens):
        for h in range(kvh):
            for i in range(min(n, keep)):
                j = want[s, h, i]
                want_w[s, h, i] = w[s, h, j]
                for x in range(2):
                    want_pool[x][to[s, i // page], h, i % page] = pool[x][table[s, j // page], h, j % page]
    np.testing.assert_array_equal(f32(bw_out, w.shape).view(np.uint32), want_w.view(np.uint32))
    for b, p in zip((bk, bv), want_pool):
        np.testing.assert_array_equal(b.download(0, p.nbytes, np.uint16).reshape(p.shape), p)


def test_eviction_of_absent_full_and_bad_sequences(ctx):
    kvh, hd, page, max_pages, pages, keep = 2, 64, 16, 4, 20, 20
    g = np.random.default_rng(4)
    pool = [g.integers(0, 65536, (pages, kvh, page, hd), dtype=np.uint16) for _ in range(2)]
    table = np.arange(12, dtype=np.uint32).reshape(3, 4)
    w = g.random((3, kvh, 64)).astype(np.float32)
    for in_place in (False, True):
        bk, bv, bw = ctx.from_array(pool[0]), ctx.from_array(pool[1]), ctx.from_array(w)
        lens = np.array([NONE, 65, 64], np.uint32)  # absent; longer than its pages; exactly full
        blen, bt = ctx.from_array(lens), ctx.from_array(table)
        out = blen if in_place else ctx.from_array(np.zeros(3, np.uint32))
        to = bt if in_place else ctx.from_array(np.array([[12, 13, 20, 20], [14, 15, 20, 20], [16, 17, 20, 20]], np.uint32))
        kept, status = ctx.from_array(np.full((3, kvh, keep), 5, np.uint32)), ctx.buffer(4, shared=True)
        status.zero()
        ctx.kv_pages_evict(bk, bv, bt, to, blen, out, bw, bw, kept, status, 3, kvh, hd, pages, page, max_pages, keep, 2, 3)
        ctx.fence()
        assert status_of(status) == cuda.STATUS_PAST_CAPACITY
        np.testing.assert_array_equal(u32(out, (3,)), [NONE, 65, keep])
        got = u32(kept, (3, kvh, keep))
        assert np.all(got[:2] == 5)
        np.testing.assert_array_equal(got[2], evicted([64], w[2:], keep, 2, 3)[0])
        np.testing.assert_array_equal(f32(bw, w.shape)[:2], w[:2])
        k = bk.download(0, pool[0].nbytes, np.uint16).reshape(pool[0].shape)
        np.testing.assert_array_equal(k[:8], pool[0][:8])
        if not in_place:
            np.testing.assert_array_equal(k[12:16], pool[0][12:16])
    # pages that are not there: zeros come from one, nothing goes to one
    bad = table.copy()
    bad[2, 0] = 99
    bk, bv, bw = ctx.from_array(pool[0]), ctx.from_array(pool[1]), ctx.from_array(w)
    to = ctx.from_array(np.array([[12, 13, 20, 20], [14, 15, 20, 20], [16, 77, 20, 20]], np.uint32))
    status.zero()
    ctx.kv_pages_evict(bk, bv, ctx.from_array(bad), to, ctx.from_array(np.array([NONE, NONE, 64], np.uint32)),
                       ctx.buffer(12), bw, bw, kept, status, 3, kvh, hd, pages, page, max_pages, keep, 2, 3)
    ctx.fence()
    assert status_of(status) == cuda.STATUS_BAD_PAGE
    k = bk.download(0, pool[0].nbytes, np.uint16).reshape(pool[0].shape)
    np.testing.assert_array_equal(k[16, :, :2], np.zeros((kvh, 2, hd), np.uint16))
    np.testing.assert_array_equal(np.delete(k, 16, 0), np.delete(pool[0], 16, 0))


def test_eviction_refusals(ctx):
    kvh, hd, page, max_pages, pages, S = 2, 64, 16, 4, 8, 2
    b = dict(k=ctx.buffer(pages * kvh * page * hd * 2), v=ctx.buffer(pages * kvh * page * hd * 2),
             table=ctx.buffer(S * max_pages * 4), to=ctx.buffer(S * max_pages * 4), len=ctx.buffer(S * 4),
             out=ctx.buffer(S * 4), w=ctx.buffer(S * kvh * 64 * 4), w_out=ctx.buffer(S * kvh * 64 * 4),
             kept=ctx.buffer(S * kvh * 64 * 4), status=ctx.buffer(4))
    for x in b.values():
        x.zero()

    def call(S=S, kvh=kvh, hd=hd, pages=pages, page=page, max_pages=max_pages, keep=20, first=2, recent=3, **over):
        a = {**b, **over}
        ctx.kv_pages_evict(a["k"], a["v"], a["table"], a["to"], a["len"], a["out"], a["w"], a["w_out"], a["kept"], a["status"],
                           S, kvh, hd, pages, page, max_pages, keep, first, recent)

    for over in (dict(keep=0), dict(keep=65), dict(first=18), dict(recent=19), dict(recent=0xFFFFFFFF), dict(S=0), dict(S=3),
                 dict(S=40000), dict(kvh=0), dict(hd=80), dict(page=20), dict(pages=9), dict(pages=0), dict(max_pages=5),
                 dict(v=b["k"]), dict(kept=b["w"]), dict(status=b["len"]), dict(w_out=b["kept"]),
                 dict(w=b["w_out"].view(16, len(b["w_out"]) - 16)), dict(out=b["table"])):
        with pytest.raises(cuda.CudaError) as e:
            call(**over)
        assert e.value.code in (-4, -5), over
    call()
    ctx.fence()


# ---------------------------------------------------------------- together

def test_prompt_decode_eviction_and_more_decode(ctx):
    """A prompt's rows go from the dense planes into pages, tokens are decoded with their attention counted, the cache is
    cut in place by what was counted, and decoding goes on with positions ahead of the rows."""
    heads, kvh, hd, page, max_pages, n = 8, 2, 64, 16, 6, 50
    g = np.random.default_rng(21)
    t = Paged(ctx, [n], heads, kvh, hd, page, weights=True, max_pages=max_pages, seed=21)
    spare = [p for p in range(t.pages) if p not in t.table[0]]
    t.table[0, 4] = spare[0]  # room for rows 64 .. 79
    t.btable.upload(0, t.table)
    dense = [g.standard_normal((1, kvh, 64, hd)).astype(np.float16) for _ in range(2)]
    t.k[:], t.v[:] = np.nan, np.inf
    t.bk.upload(0, t.k)
    t.bv.upload(0, t.v)
    ctx.kv_pages_copy(ctx.from_array(dense[0]), ctx.from_array(dense[1]), t.bk, t.bv, t.btable, t.status, t.pages, page,
                      max_pages, kvh, hd, 64, True, [(0, 0, 0, n)])
    w = ctx.from_array(np.zeros_like(t.w_in))
    ctx.fence()
    t.k, t.v = f16(t.bk, t.k.shape).copy(), f16(t.bv, t.v.shape).copy()
    total = np.zeros_like(t.w_in)
    for i in range(3):
        t.lens, t.pos = [n + i], np.array([n + i], np.uint32)
        t.blen.upload(0, t.pos)
        t.bpos.upload(0, t.pos)
        t.call(w, w)
        ctx.fence()
        now = f32(w, total.shape).copy()
        t.check(total, now, total)
        total, t.k, t.v = now, f16(t.bk, t.k.shape).copy(), f16(t.bv, t.v.shape).copy()
    keep, rows = 30, n + 3
    t.blen.upload(0, np.array([rows], np.uint32))
    kept = ctx.buffer(kvh * keep * 4)
    ctx.kv_pages_evict(t.bk, t.bv, t.btable, t.btable, t.blen, t.blen, w, w, kept, t.status, 1, kvh, hd, t.pages, page,
                       max_pages, keep, 4, 8)
    ctx.fence()
    assert u32(t.blen, (1,))[0] == keep
    want = evicted([rows], total, keep, 4, 8)
    np.testing.assert_array_equal(u32(kept, want.shape), want)
    k, v, after = t.k.copy(), t.v.copy(), total.copy()
    for h in range(kvh):
        for i, j in enumerate(want[0, h]):
            k[t.table[0, i // page], h, i % page] = t.k[t.table[0, j // page], h, j % page]
            v[t.table[0, i // page], h, i % page] = t.v[t.table[0, j // page], h, j % page]
            after[0, h, i] = total[0, h, j]
    t.k, t.v, total = k, v, after
    t.lens, t.pos = [keep], np.array([rows], np.uint32)
    t.bpos.upload(0, t.pos)
    t.call(w, w)
    ctx.fence()
    t.check(total, f32(w, total.shape), total)
    assert status_of(t.status) == 0
