"""Penalties, bias maps, masks and the greedy choice on rows of logits, against a plain restatement.  Each step is rounded
to f32 by itself, so the restatement in f32 gives the same bits; its own steps are checked against 64 bits (four roundings
of at most 2^-24 of the largest magnitude on the way)."""
import numpy as np
import pytest

from tuckmill_b200 import cuda

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


def adjusted(x, log, pos, base, log_cap, prompt, pen, bias, mask, dtype):
    """y [rows][n] and the chosen tokens; bias: per row a list of (id, value)."""
    rows, n = x.shape
    y, chosen = x.astype(dtype), []
    for r in range(rows):
        end = min(base + int(pos[r]), log_cap) if log is not None else 0
        if pen is not None:
            rep, presence, freq = (dtype(v) for v in pen[r])
            ids = [int(t) for t in log[r, :end] if t < n]
            out = [int(t) for t in log[r, (prompt[r] if prompt is not None else 0):end] if t < n]
            for t in set(ids):
                y[r, t] = y[r, t] / rep if y[r, t] > 0 else y[r, t] * rep
            for t in set(out):
                y[r, t] = (y[r, t] - freq * dtype(out.count(t))) - presence
        for t, v in dict((t, v) for t, v in bias[r] if t < n).items() if bias is not None else ():
            y[r, t] = y[r, t] + dtype(v)
        allowed = np.ones(n, bool) if mask is None else \
            np.unpackbits(mask[r].view(np.uint8), bitorder="little")[:n].astype(bool)
        y[r, ~allowed] = -np.inf
        can = np.flatnonzero(allowed & ~np.isnan(y[r]))
        chosen.append(NONE if can.size == 0 else int(can[np.argmax(y[r, can])]))
    return y, chosen


CASES = [
    # rows, n, history, biases, mask, base
    (1, 1, 3, 2, True, 0),
    (1, 33, 40, 0, False, 1),
    (3, 1000, 700, 5, True, 0),
    (2, 1024, 1, 1500, True, 2),
    (5, 5003, 2000, 40, True, 1),
    (33, 32001, 90, 3, True, 0),
    (1, 151936, 3000, 300, True, 1),
    (1, 600001, 100, 10, False, 0),
    (70, 32000, 9, 2, True, 0),     # stretches of 4096 logits, rows in quads
    (70, 32001, 9, 2, True, 0),     # and not
    (150, 32004, 5, 1, True, 0),    # stretches of 8192
    (150, 32003, 5, 0, False, 0),
    (1, cuda.LOGITS_MAX, 50, 4, True, 0),
]


@pytest.mark.parametrize("rows,n,history,biases,mask,base", CASES)
def test_adjusted_logits_and_the_choice(ctx, rows, n, history, biases, mask, base):
    g = np.random.default_rng(n)
    stride = history + base + 5
    x = (4 * g.standard_normal((rows, n))).astype(np.float32)
    x[g.random(x.shape) < 0.01] = np.nan
    x[g.random(x.shape) < 0.01] = -np.inf
    x[g.random(x.shape) < 0.05] = 0.0
    x[g.random(x.shape) < 0.02] = -0.0
    log = g.integers(0, n, (rows, stride), dtype=np.uint32)
    log[:, ::7] = log[:, :1]  # one token many times
    log[g.random(log.shape) < 0.05] = NONE  # no token
    pos = np.array([history - r % 3 if history > 3 else history for r in range(rows)], np.uint32)
    prompt = np.array([(history * r) // rows for r in range(rows)], np.uint32)
    pen = np.stack([1 + g.random(rows), g.random(rows) - 0.3, g.random(rows) - 0.3], 1).astype(np.float32)
    ids = g.integers(0, n + 2, (rows, max(biases, 1)), dtype=np.uint32)
    if biases > 2:
        ids[:, -1] = ids[:, 0]  # named twice: the later value counts
    values = (5 * g.standard_normal(ids.shape)).astype(np.float32)
    count = np.array([0 if r == 1 else biases + 7 * (r == 2) for r in range(rows)], np.uint32)  # (more than there are)
    bits = g.integers(0, 1 << 32, (rows, (n + 31) // 32), dtype=np.uint32) if mask else None
    if mask and rows > 2:
        bits[2] = 0  # nothing is allowed
    b = ctx.from_array
    bx, blog, by = b(x), b(log), ctx.buffer(x.nbytes)
    partial = ctx.buffer(rows * cuda.LOGITS_PARTIAL_BYTES)
    mirror = ctx.buffer(log.nbytes, shared=True)
    mirror.zero()
    extra = dict(bias_ids=b(ids), bias_values=b(values), bias_count=b(count), bias_cap=biases) if biases else {}
    bias = [list(zip(ids[r].tolist(), values[r]))[:min(int(count[r]), biases)] for r in range(rows)] if biases else None
    bmask = b(bits) if mask else None
    ctx.logits_adjust_rows(bx, by, rows, n, blog, stride, base, b(pos), b(pen), prompt_len=b(prompt), mask=bmask,
                           partial=partial, log_cap=stride - 1, mirror=mirror, **extra)
    ctx.fence()
    want, chosen = adjusted(x, log, pos, base, stride - 1, prompt, pen, bias, bits, np.float32)
    got = by.download(0, x.nbytes, np.float32).reshape(x.shape)
    np.testing.assert_array_equal(got, want)
    wide, _ = adjusted(x.astype(np.float64), log, pos, base, stride - 1, prompt, pen, bias, bits, np.float64)
    top = np.abs(np.where(np.isfinite(x), x, 0)).max() * 2 + 1.3 + history + 25
    fine = np.isfinite(wide)
    assert np.all(np.abs(got[fine] - wide[fine]) <= 4 * 2.0 ** -24 * top)
    new_log = log.copy()
    for r in range(rows):
        if base + pos[r] < stride - 1:
            new_log[r, base + pos[r]] = chosen[r]
    np.testing.assert_array_equal(blog.download(0, log.nbytes, np.uint32).reshape(log.shape), new_log)
    seen = mirror.download(0, log.nbytes, np.uint32).reshape(log.shape)
    for r in range(rows):
        if base + pos[r] < stride - 1:
            assert seen[r, base + pos[r]] == chosen[r]
    # in place, without a choice: the log is left as it is
    blog.upload(0, log)
    ctx.logits_adjust_rows(bx, bx, rows, n, blog, stride, base, b(pos), b(pen), prompt_len=b(prompt), mask=bmask,
                           log_cap=stride - 1, **extra)
    ctx.fence()
    np.testing.assert_array_equal(bx.download(0, x.nbytes, np.float32).reshape(x.shape), want)
    np.testing.assert_array_equal(blog.download(0, log.nbytes, np.uint32).reshape(log.shape), log)


def test_each_part_alone(ctx):
    rows, n = 3, 700
    g = np.random.default_rng(0)
    x = g.standard_normal((rows, n)).astype(np.float32)
    log = g.integers(0, n, (rows, 50), dtype=np.uint32)
    pos = np.array([0, 20, 500], np.uint32)  # the last is past its log: all of it is history, nothing is written
    b = ctx.from_array
    bx, by, partial = b(x), ctx.buffer(x.nbytes), ctx.buffer(rows * cuda.LOGITS_PARTIAL_BYTES)

    def get():
        ctx.fence()
        return by.download(0, x.nbytes, np.float32).reshape(x.shape)

    ctx.logits_adjust_rows(bx, by, rows, n)
    np.testing.assert_array_equal(get(), x)
    blog = b(log)
    ctx.logits_adjust_rows(bx, by, rows, n, blog, 50, 0, b(pos), partial=partial)
    np.testing.assert_array_equal(get(), x)
    want = log.copy()
    want[0, 0], want[1, 20] = x[0].argmax(), x[1].argmax()
    np.testing.assert_array_equal(blog.download(0, log.nbytes, np.uint32).reshape(log.shape), want)
    pen = np.array([[1.5, 0.25, 0.125]] * rows, np.float32)
    ctx.logits_adjust_rows(bx, by, rows, n, b(log), 50, 0, b(pos), b(pen))
    np.testing.assert_array_equal(get(), adjusted(x, log, pos, 0, 50, None, pen, None, None, np.float32)[0])
    ids, val = np.array([[5, 5, 699]] * rows, np.uint32), np.array([[1, 2, 3]] * rows, np.float32)
    ctx.logits_adjust_rows(bx, by, rows, n, bias_ids=b(ids), bias_values=b(val), bias_count=b(np.array([3, 1, 2], np.uint32)), bias_cap=3)
    want = x.copy()
    want[0, 5] += 2
    want[0, 699] += 3
    want[1, 5] += 1
    want[2, 5] += 2
    np.testing.assert_array_equal(get(), want)
    bits = g.integers(0, 1 << 32, (rows, 22), dtype=np.uint32)
    ctx.logits_adjust_rows(bx, by, rows, n, mask=b(bits))
    np.testing.assert_array_equal(get(), adjusted(x, None, None, 0, 0, None, None, None, bits, np.float32)[0])


def test_a_recorded_step_appends_to_its_log(ctx):
    """Replayed with the position advancing on the device: each choice is penalised from the next step on."""
    n, steps = 500, 12
    g = np.random.default_rng(8)
    x = g.standard_normal((1, n)).astype(np.float32)
    log = np.full((1, 40), NONE, np.uint32)
    log[0, 0] = 17
    pen = np.array([[1.3, 0.5, 0.2]], np.float32)
    b = ctx.from_array
    bx, by, blog, bpos, bpen = b(x), ctx.buffer(x.nbytes), b(log), b(np.zeros(1, np.uint32)), b(pen)
    partial = ctx.buffer(cuda.LOGITS_PARTIAL_BYTES)
    ctx.begin_group()
    ctx.logits_adjust_rows(bx, by, 1, n, blog, 40, 1, bpos, bpen, partial=partial)
    ctx.u32_add(bpos, 0, 1)
    graph = ctx.end_group_retain()
    for _ in range(steps):
        graph.launch()
    ctx.fence()
    graph.free()
    for i in range(steps):
        log[0, 1 + i] = adjusted(x, log, np.array([i]), 1, 40, None, pen, None, None, np.float32)[1][0]
    np.testing.assert_array_equal(blog.download(0, log.nbytes, np.uint32).reshape(log.shape), log)


def test_the_choice_is_that_of_argmax_rows(ctx):
    rows, n = 4, 9001
    g = np.random.default_rng(3)
    x = np.round(g.standard_normal((rows, n)), 1).astype(np.float32)  # ties
    x[1] = -np.inf
    x[2] = np.nan
    x[3, :] = -0.0
    x[3, 5] = 0.0
    b = ctx.from_array
    one, two, pos = b(np.zeros((rows, 4), np.uint32)), b(np.zeros((rows, 4), np.uint32)), b(np.array([0, 1, 2, 3], np.uint32))
    bx = b(x)
    ctx.argmax_rows_dev(bx, rows, n, ctx.buffer(rows * 512), one, 4, 0, pos, 4)
    ctx.logits_adjust_rows(bx, ctx.buffer(x.nbytes), rows, n, two, 4, 0, pos, partial=ctx.buffer(rows * cuda.LOGITS_PARTIAL_BYTES))
    ctx.fence()
    np.testing.assert_array_equal(one.download(0, 64, np.uint32), two.download(0, 64, np.uint32))


def test_logits_refusals(ctx):
    rows, n = 2, 100
    f = ctx.buffer(rows * n * 4)
    y = ctx.buffer(rows * n * 4)
    log, pos, pen = ctx.buffer(rows * 10 * 4), ctx.buffer(rows * 4), ctx.buffer(rows * 12)
    part = ctx.buffer(rows * cuda.LOGITS_PARTIAL_BYTES)
    ids, val, cnt, mask = ctx.buffer(rows * 12), ctx.buffer(rows * 12), ctx.buffer(rows * 4), ctx.buffer(rows * 16)
    for x in (f, log, pos, pen, ids, val, cnt, mask):
        x.zero()
    full = dict(log=log, log_stride=10, base=0, pos_buf=pos, penalties=pen, prompt_len=cnt, bias_ids=ids, bias_values=val,
                bias_count=cnt, bias_cap=3, mask=mask, partial=part)

    def call(x=f, y=y, rows=rows, n=n, **over):
        ctx.logits_adjust_rows(x, y, rows, n, **{**full, **over})

    for over in (dict(rows=0), dict(rows=65536), dict(n=0), dict(n=cuda.LOGITS_MAX + 1), dict(n=101), dict(rows=3), dict(log=None),
                 dict(pos_buf=None), dict(log_cap=0), dict(log_cap=11), dict(log_stride=11), dict(penalties=None),
                 dict(partial=None, mirror=log), dict(bias_values=None), dict(bias_ids=None), dict(bias_count=None),
                 dict(bias_cap=0), dict(bias_cap=4), dict(bias_cap=cuda.LOGITS_MAX_BIASES + 1),
                 dict(log_cap=cuda.LOGITS_MAX_LOG + 1, log_stride=cuda.LOGITS_MAX_LOG + 1), dict(mask=cnt), dict(partial=pen), dict(mirror=cnt), dict(mirror=log),
                 dict(y=f.view(16, rows * n * 4 - 16)), dict(y=log), dict(partial=y), dict(x=part, n=4, y=part.view(16, 64))):
        with pytest.raises(cuda.CudaError) as e:
            call(**over)
        assert e.value.code in (-4, -5), over
    call()
    ctx.fence()


def test_buffers_of_another_context_are_refused(ctx):
    """A token log and positions that a call does not use are looked at no further than a buffer of its own, or refused."""
    other = cuda.CudaContext(0)
    try:
        n = 64
        x, y, mask = ctx.from_array(np.zeros((1, n), np.float32)), ctx.buffer(n * 4), ctx.from_array(np.full(2, 0xFFFFFFFF, np.uint32))
        own, foreign = ctx.buffer(16), other.buffer(16)
        for over in (dict(log=foreign), dict(pos_buf=foreign), dict(log=own, pos_buf=foreign), dict(log=foreign, pos_buf=own)):
            with pytest.raises(cuda.CudaError) as e:
                ctx.logits_adjust_rows(x, y, 1, n, log_stride=4, mask=mask, **over)
            assert e.value.code == -5, over
        ctx.logits_adjust_rows(x, y, 1, n, log=own, log_stride=4, pos_buf=own, mask=mask)
        ctx.fence()
        np.testing.assert_array_equal(y.download(0, n * 4, np.float32), np.zeros(n, np.float32))
        foreign.free()
    finally:
        other.close()
