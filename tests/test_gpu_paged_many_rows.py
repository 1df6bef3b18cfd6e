"""sl_hip_paged_window_attention in calls with so many query rows that the rows of
many tokens take the matrix-core tiles (a smaller call is left to the form for few query
rows whatever its shape), on the GPU against the definition in float64: a large
row beside small ones of every kind."""
import numpy as np
import pytest

from paged_tokens import Rows, assert_within, attention64, read_port
from starlight_amd.ir import Op
from starlight_amd.paged import PAGE_NONE
from test_gpu_paged_serving import Graph

pytestmark = pytest.mark.gpu


def large_row(window, heads, kv_heads):
    """(cached, new) tokens of a row that makes a call large: 32,000 queries (tokens times heads)
    behind a short window, 8,000 behind a longer one, and without one 1,600 per KV head that see
    2,600 keys and more."""
    if window == 0 or window > 2600:
        return 2600, 1600 * kv_heads // heads
    return (300, 32000 // heads) if window <= 500 else (2600, 8000 // heads)


def call(hip, rng, heads, kv_heads, dim, lens, news, page=16, window=0, layers=1, layer=0):
    """Rows of the given lengths with a large one in their midst."""
    past, new = large_row(window, heads, kv_heads)
    at = len(lens) // 2
    return Rows(hip, rng, heads, kv_heads, dim, lens[:at] + [past] + lens[at:], news[:at] + [new] + news[at:], page,
                layers=layers, layer=layer)


def queries(rows, factor=2.0):
    return (rows.rng.standard_normal((rows.total, rows.heads, rows.dim)) * factor).astype(np.float32)


def attend(rows, q, scale, window=0, sinks=0, offset=0):
    qr, out = rows.buffer(q, offset), rows.buffer(np.zeros_like(q), offset)
    rows.cache.window_attention(Op.causal_attention(rows.layer, rows.heads, rows.kv_heads, rows.dim, scale),
                                rows.tokens, qr, out, window, sinks)
    return read_port(rows.hip, out, q.shape)


def check(rows, window=0, sinks=0, scale=None, q=None, offset=0):
    scale = float(np.float32(rows.dim**-0.5 if scale is None else scale))
    q = queries(rows) if q is None else q
    want, bound = attention64(rows, q, scale, window, sinks)
    assert_within(attend(rows, q, scale, window, sinks, offset), want, bound)


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (32, 8, 128), (3, 3, 80), (6, 2, 16), (5, 1, 48),
                                                (40, 2, 96), (20, 1, 112)])
def test_head_layouts(hip, heads, kv_heads, dim):
    rng = np.random.default_rng(heads + dim)
    rows = call(hip, rng, heads, kv_heads, dim, [0, 37, 200, 16], [1, 50, 3, 90], window=200, layers=2, layer=1)
    check(rows, 200, 4)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (2, 3), (15, 0), (16, 16), (17, 1), (33, 20),
                                          (64, 500), (100, 4), (250, 15), (1000, 70), (5000, 4)])
@pytest.mark.parametrize("lens,news", [([0, 1, 40, 300], [33, 40, 257, 65]), ([0, 5, 130], [90, 0, 35])])
def test_windows_and_sinks(hip, window, sinks, lens, news):
    rng = np.random.default_rng(window * 31 + sinks)
    check(call(hip, rng, 4, 2, 64, lens, news, window=window), window, sinks)


@pytest.mark.parametrize("page", [32, 48, 112])
@pytest.mark.parametrize("window", [0, 60])
def test_page_sizes(hip, page, window):
    rng = np.random.default_rng(page)
    check(call(hip, rng, 8, 2, 128, [0, 95, 333], [70, 1, 17], page, window), window, 5)


@pytest.mark.parametrize("batch,large", [(63, 0), (64, -1), (65, 60), (65, -1), (150, 0), (150, 100)])
def test_many_rows(hip, batch, large):
    """The large row among the first 64 rows and behind them."""
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0, 100, batch)]
    news = [int(x) for x in rng.choice([0, 1, 3, 40, 70], batch)]
    lens[large], news[large] = large_row(40, 4, 1)
    check(Rows(hip, rng, 4, 1, 64, lens, news), 40, 2)


@pytest.mark.parametrize("offset,dim", [(1, 64), (2, 128), (3, 80), (4, 48)])
def test_ports_at_any_offset(hip, offset, dim):
    rng = np.random.default_rng(offset)
    check(call(hip, rng, 8, 2, dim, [40, 300], [3, 50], window=100), 100, 4, offset=offset)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_scales(hip, scale):
    rng = np.random.default_rng(3)
    check(call(hip, rng, 4, 2, 64, [40, 300], [3, 50], window=100), 100, 4, scale=scale)


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_pages_that_nothing_sees_are_not_read(hip, dim):
    rng = np.random.default_rng(4)
    window, sinks = 37, 5
    rows = call(hip, rng, 8, 2, dim, [200, 90, 0, 333], [1, 30, 50, 60], window=window)
    keep = np.zeros(rows.pool.shape[:2] + (rows.page,), bool)
    for b, (l, n) in enumerate(zip(rows.lens, rows.news)):
        first = max(l - window + 1, 0)
        seen = [j for j in range(l + n) if j >= first or j < sinks]
        for j in seen:
            keep[(0,) + rows.at(b, j)] = True
        pages = {j // rows.page for j in seen}
        for i in range(rows.table.shape[1]):
            if i not in pages:
                rows.table[b, i] = PAGE_NONE
    rows.pool[~np.broadcast_to(keep[:, :, None], (1, rows.pool.shape[1], 2, rows.page))] = np.nan
    rows.upload()
    check(rows, window, sinks)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_values_of_unseen_keys_do_not_matter(hip, value, dim):
    """A token in the midst of a chunk holds values that are not finite: the tokens
    before it come out as if it were not there."""
    rng = np.random.default_rng(5)
    rows = call(hip, rng, 4, 2, dim, [30, 2], [90, 9], window=100)
    q, scale = queries(rows), float(np.float32(dim**-0.5))
    want, bound = attention64(rows, q, scale, 100)
    starts = np.concatenate([[0], np.cumsum(rows.news)])
    clean = np.ones((rows.total, 4), bool)
    for b, i in ((0, 60), (1, 1000)):
        p, s = rows.at(b, rows.lens[b] + i)
        rows.pool[0, p, :, s, 1, 3] = value
        # the tokens that see it, on KV head 1
        clean[starts[b] + i:min(starts[b] + i + 100, starts[b + 1]), 2:] = False
    rows.upload()
    got = attend(rows, q, scale, 100)
    assert_within(got[clean], want[clean], bound[clean])
    # (a key of -inf may weigh nothing, its value's dimension is not finite then either)
    assert not np.isfinite(got[~clean][:, 3]).any()


@pytest.mark.parametrize("kv,qf", [(1e-6, 1.0), (1e-20, 1.0), (3e4, 1e-4), (1e15, 1e-15), (1e-3, 30.0)])
@pytest.mark.parametrize("dim", [64, 128])
def test_magnitudes(hip, kv, qf, dim):
    rng = np.random.default_rng(6)
    rows = call(hip, rng, 8, 2, dim, [70, 400], [50, 1], window=100)
    rows.pool *= np.float32(kv)
    rows.upload()
    check(rows, 100, 4, q=queries(rows, 2.0 * qf))


def test_values_that_grow_along_the_row(hip):
    """Each 16 positions' values 2^6 times the ones before, up to 2^60, then small
    again: the unit of the running result follows."""
    rng = np.random.default_rng(7)
    rows = call(hip, rng, 4, 2, 64, [0, 600], [160, 40])
    for b in range(3):
        for j in range(rows.lens[b] + rows.news[b]):
            p, s = rows.at(b, j)
            rows.pool[0, p, 1, s] *= np.float32(2.0**(6 * min(j // 16, 10) if j < 400 else 0))
            rows.pool[0, p, 0, s] *= np.float32(2.0**(-(j // 64 % 5)))
    rows.upload()
    check(rows)


def test_scores_that_rise_and_fall(hip):
    """Keys that grow and shrink along the row: the running maximum is followed
    late and early."""
    rng = np.random.default_rng(8)
    rows = call(hip, rng, 4, 2, 128, [0, 600], [160, 40])
    for b in range(3):
        for j in range(rows.lens[b] + rows.news[b]):
            p, s = rows.at(b, j)
            rows.pool[0, p, 0, s] *= np.float32(0.1 + 2.0 * abs(np.sin(j / 50)))
    rows.upload()
    check(rows)


FACTORS = [2.0**12, 2.0**15, 2.0**18, 2.0**30, 1e30]


@pytest.mark.parametrize("factor", FACTORS)
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("large", [False, True])
def test_large_values_of_unseen_keys_do_not_matter(hip, factor, dim, large):
    """Keys and values far larger than those beside them, of a token in the midst of a
    chunk: the tokens before it, and those whose window has left it behind, are as
    accurate as ever, and those that see it by their own values' measure."""
    rng = np.random.default_rng(9)
    rows = (call(hip, rng, 4, 2, dim, [30, 2], [90, 9], window=100) if large
            else Rows(hip, rng, 4, 2, dim, [30, 300, 2], [9, 1, 40]))
    for b, j in ((0, 35), (1, rows.lens[1] - 20), (2, 10)):
        k, v = (x[0] for x in rows.kv(b, [j]))
        rows.put(b, j, (k * factor).astype(np.float32), (v * factor).astype(np.float32))
    rows.upload()
    check(rows, 100 if large else 20)


@pytest.mark.parametrize("factor", FACTORS)
@pytest.mark.parametrize("dim,large", [(64, False), (64, True), (128, False), (128, True), (80, True), (192, False)])
def test_one_large_column(hip, factor, dim, large):
    """One dimension of the values far larger than the others."""
    rng = np.random.default_rng(10)
    rows = (call(hip, rng, 4, 2, dim, [30, 2], [90, 9], window=100) if large
            else Rows(hip, rng, 4, 2, dim, [30, 300, 2], [9, 1, 40]))
    rows.pool[:, :, 1, :, :, dim // 2 + 1] *= np.float32(factor)
    rows.pool[:, :, 1, :, :, 2] = 0
    rows.upload()
    check(rows, 100 if large else 20)


@pytest.mark.parametrize("dim,large", [(64, False), (64, True), (128, False), (128, True), (48, True), (192, False)])
def test_zeros_among_the_keys(hip, dim, large):
    """Rows of zeros, as a cleared cache holds, and whole pages of them."""
    rng = np.random.default_rng(11)
    rows = (call(hip, rng, 4, 2, dim, [30, 2], [90, 9], window=100) if large
            else Rows(hip, rng, 4, 2, dim, [30, 300, 2], [9, 1, 40]))
    for b in range(3):
        for j in range(rows.lens[b] + rows.news[b]):
            p, s = rows.at(b, j)
            if j % 5 == 3 or j // 16 % 3 == 1:
                rows.pool[0, p, 1, s] = 0
            if j % 7 == 2 or j // 16 % 4 == 1:
                rows.pool[0, p, 0, s] = 0
    rows.upload()
    check(rows, 100 if large else 0)


# prompts of a whole round of blocks of 256 query rows and part of another (32 and 128 of
# each KV head's fill 256 CUs): the part is split over the keys
@pytest.mark.parametrize("heads,kv_heads,dim,new", [(32, 8, 64, 2400), (32, 8, 128, 2100), (8, 2, 64, 8300),
                                                    (8, 2, 112, 9000)])
@pytest.mark.parametrize("lens,news", [([], []), ([900, 3, 0], [1, 70, 2])])
def test_the_last_round_of_blocks(hip, heads, kv_heads, dim, new, lens, news):
    rng = np.random.default_rng(new)
    check(Rows(hip, rng, heads, kv_heads, dim, lens[:1] + [70] + lens[1:], news[:1] + [new] + news[1:]), 150, 4)


def test_the_last_round_changes_between_replays(hip):
    """Captured for a prompt whose last round of blocks is split; replayed with its
    tokens in rows of other numbers, so that more, fewer or no blocks are left over."""
    rng = np.random.default_rng(12)
    news = [[2400, 0, 1], [1100, 1300, 1], [1, 2048, 352], [3, 2046, 352], [2394, 7, 0]]
    lens = [[30, 0, 500], [10, 600, 0], [900, 0, 3], [0, 0, 0], [5, 300, 0]]
    most = [max(l[b] + n[b] for l, n in zip(lens, news)) for b in range(3)]
    rows = Rows(hip, rng, 32, 8, 64, [m - 1 for m in most], [1] * 3)
    q = (rng.standard_normal((2401, 32, 64)) * 2).astype(np.float32)
    op = Op.causal_attention(0, 32, 8, 64, 0.125)
    qr, out = rows.buffer(q), rows.buffer(np.zeros_like(q))

    def put(i):
        rows.lens, rows.news = lens[i], news[i]
        hip.upload_u32(rows.cache.lens_buffer, np.asarray(rows.lens, np.uint32))
        rows.tokens.set(rows.news)

    put(0)
    graph = Graph(hip, lambda: rows.cache.window_attention(op, rows.tokens, qr, out, 150, 4))
    try:
        for i in (0, 1, 2, 3, 4, 0):
            put(i)
            want, bound = attention64(rows, q, 0.125, 150, 4)
            graph.launch()
            assert_within(read_port(hip, out, q.shape), want, bound)
            rows.cache.window_attention(op, rows.tokens, qr, out, 150, 4)
            assert_within(read_port(hip, out, q.shape), want, bound)
    finally:
        graph.close()
