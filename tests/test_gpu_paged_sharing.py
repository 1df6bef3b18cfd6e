"""sl_hip_paged_prefix_attention where reading the shared positions once pays
(24 MiB of keys and values saved: smaller batches are read row by row), and
sl_hip_paged_window_attention where rows of few and of many tokens are split
differently, on the GPU against the attention's definition in float64."""
import math

import numpy as np
import pytest

from paged_tokens import Rows, assert_within, attention64, read_port
from starlight_amd.device import HipDevice
from starlight_amd.ir import Op
from starlight_amd.paged import PAGE_NONE
from test_gpu_paged_serving import Graph

pytestmark = pytest.mark.gpu

SAVED = 24 << 20


def prefix_that_pays(batch, kv_heads, dim, past_multiple):
    """The least prefix that `batch` rows have to share, moved to `past_multiple`
    positions past a multiple of 16."""
    need = -(-SAVED // ((batch - 1) * kv_heads * dim * 8))
    return -(-need // 16) * 16 + past_multiple


def ragged(rng, batch, prefix, idle=0, most=2, beyond=70):
    lens = [prefix + int(x) for x in rng.integers(0, beyond, batch + idle)]
    news = [1 + int(x) for x in rng.integers(0, most, batch)]
    for i in range(idle):  # the first row among them
        news.insert((i * 7) % (batch + i), 0)
    return lens, news


def attend(rows, q, scale, prefix, offset=0):
    qr, out = rows.buffer(q, offset), rows.buffer(np.zeros_like(q), offset)
    rows.cache.prefix_attention(Op.causal_attention(rows.layer, rows.heads, rows.kv_heads, rows.dim, scale),
                                rows.tokens, qr, out, prefix)
    return read_port(rows.hip, out, q.shape)


def queries(rows):
    return (rows.rng.standard_normal((rows.total, rows.heads, rows.dim)) * 2).astype(np.float32)


def check(rows, prefix, offset=0):
    scale = float(np.float32(1.0 / math.sqrt(rows.dim)))
    q = queries(rows)
    want, bound = attention64(rows, q, scale)
    assert_within(attend(rows, q, scale, prefix, offset), want, bound)


# (heads, kv_heads, dim, batch): up to 64 query rows per KV head, more (one block of 256, more
# than one), and head_dim above 128
LAYOUTS = [(32, 8, 128, 8), (4, 4, 64, 40), (3, 3, 80, 50), (6, 2, 16, 21), (40, 2, 96, 3), (12, 4, 192, 12),
           (32, 8, 128, 40), (32, 8, 64, 60), (4, 4, 64, 90), (40, 2, 96, 24), (6, 2, 16, 110), (20, 1, 112, 30),
           (4, 4, 80, 300), (8, 1, 256, 30), (12, 4, 192, 40)]


@pytest.mark.parametrize("heads,kv_heads,dim,batch", LAYOUTS)
def test_head_layouts(hip, heads, kv_heads, dim, batch):
    rng = np.random.default_rng(heads + dim + batch)
    prefix = prefix_that_pays(batch, kv_heads, dim, 0)
    lens, news = ragged(rng, batch, prefix, idle=2)
    check(Rows(hip, rng, heads, kv_heads, dim, lens, news, prefix=prefix, layers=2, layer=1), prefix)


@pytest.mark.parametrize("past", [1, 5, 15, 17, 31, 63])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("batch", [9, 70])
def test_prefixes_end_anywhere(hip, past, page, batch):
    rng = np.random.default_rng(past + page)
    prefix = prefix_that_pays(batch, 2, 128, past)
    lens, news = ragged(rng, batch, prefix, most=4, beyond=3)
    check(Rows(hip, rng, 8, 2, 128, lens, news, page, prefix=prefix), prefix)


@pytest.mark.parametrize("batch,dim", [(9, 128), (70, 128), (40, 64)])
def test_one_row_with_many_tokens(hip, batch, dim):
    """A row's prompt over the shared positions beside decoding rows."""
    rng = np.random.default_rng(batch)
    prefix = prefix_that_pays(batch, 2, dim, 3)
    lens, news = ragged(rng, batch, prefix, idle=1)
    news[batch // 2] = 150
    check(Rows(hip, rng, 8, 2, dim, lens, news, prefix=prefix), prefix)


@pytest.mark.parametrize("batch", [9, 70])
def test_stale_values_are_not_read(hip, batch):
    """NaN in every slot that holds no position of a row, and no page at all in
    the tables of rows that sit the step out."""
    rng = np.random.default_rng(batch)
    prefix = prefix_that_pays(batch, 2, 128, 0)
    lens, news = ragged(rng, batch, prefix, idle=2)
    rows = Rows(hip, rng, 8, 2, 128, lens, news, prefix=prefix)
    keep = np.zeros((rows.pool.shape[1], rows.page), bool)
    for b in range(len(lens)):
        if news[b] == 0:
            rows.table[b] = PAGE_NONE
            continue
        for j in range(lens[b] + news[b]):
            keep[rows.at(b, j)] = True
    rows.pool[0].transpose(1, 0, 2, 3, 4)[:, ~keep] = np.nan
    rows.upload()
    check(rows, prefix)


@pytest.mark.parametrize("batch", [9, 70])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_values_that_are_not_finite(hip, batch, value):
    """In a shared value: that dimension of its KV head's queries and nothing
    else. In a later token's key: that token's row from it on."""
    rng = np.random.default_rng(batch)
    prefix = prefix_that_pays(batch, 2, 128, 7)
    lens, news = ragged(rng, batch, prefix)
    news[3] = 5
    rows = Rows(hip, rng, 8, 2, 128, lens, news, prefix=prefix)
    q = queries(rows)
    scale = float(np.float32(128**-0.5))
    want, bound = attention64(rows, q, scale)
    p, s = rows.at(0, 40)
    rows.pool[0, p, 1, s, 1, 9] = value
    p, s = rows.at(3, lens[3] + 2)
    rows.pool[0, p, 0, s, 0, 0] = np.nan
    rows.upload()
    got = attend(rows, q, scale, prefix)
    clean = np.ones(got.shape, bool)
    clean[:, 4:, 9] = False
    first = sum(news[:3])
    clean[first + 2:first + 5, :4] = False
    assert_within(got[clean], want[clean], bound[clean])
    assert not np.isfinite(got[~clean]).any()


@pytest.mark.parametrize("batch,dim", [(9, 128), (70, 128), (40, 64), (30, 256)])
def test_ports_at_any_offset(hip, batch, dim):
    rng = np.random.default_rng(batch)
    prefix = prefix_that_pays(batch, 2, dim, 9)
    lens, news = ragged(rng, batch, prefix)
    check(Rows(hip, rng, 8, 2, dim, lens, news, prefix=prefix), prefix, offset=1 + batch % 3)


@pytest.mark.parametrize("room", [65536, 6 << 20])
def test_small_workspace(hip, monkeypatch, room):
    """Without room for the partial results of both parts the rows are read one
    by one; with a little the longest are split as far as it goes."""
    monkeypatch.setenv("SL_HIP_WORKSPACE_BYTES", str(room))
    with HipDevice(0) as dev:
        rng = np.random.default_rng(7)
        prefix = prefix_that_pays(9, 8, 128, 0)
        lens, news = ragged(rng, 9, prefix)
        check(Rows(dev, rng, 32, 8, 128, lens, news, prefix=prefix), prefix)
        rows = Rows(dev, rng, 32, 8, 128, [9000, 50, 200], [1, 1, 90])
        check_window(rows)


@pytest.mark.parametrize("batch", [9, 70])
def test_captured_and_replayed_with_other_lengths(hip, batch):
    """Captured for one token each; replayed, between eager calls, with other
    lengths past the prefix and the same number of tokens dealt otherwise."""
    rng = np.random.default_rng(9)
    prefix = prefix_that_pays(batch, 2, 128, 5)
    many = [0] * batch
    many[2], many[batch - 1] = batch - 3, 3
    news = [[1] * batch, many, [1] * batch, [2] * (batch // 2) + [batch % 2] + [0] * (batch - batch // 2 - 1)]
    lens = [[prefix + x for x in row] for row in
            ([3] * batch, [17] * batch, [int(x) for x in rng.integers(0, 300, batch)], [i for i in range(batch)])]
    most = [max(l[b] + n[b] for l, n in zip(lens, news)) for b in range(batch)]
    rows = Rows(hip, rng, 8, 2, 128, [m - 1 for m in most], [1] * batch, prefix=prefix)
    q = (rng.standard_normal((batch, 8, 128)) * 2).astype(np.float32)
    scale = float(np.float32(128**-0.5))
    op = Op.causal_attention(0, 8, 2, 128, scale)
    qr, out = rows.buffer(q), rows.buffer(np.zeros_like(q))

    def work():
        rows.cache.prefix_attention(op, rows.tokens, qr, out, prefix)

    def put(i):
        rows.lens, rows.news = lens[i], news[i]
        hip.upload_u32(rows.cache.lens_buffer, np.asarray(rows.lens, np.uint32))
        rows.tokens.set(rows.news)

    put(0)
    graph = Graph(hip, work)
    try:
        for i in (0, 1, 2, 3, 2):
            put(i)
            graph.launch()
            want, bound = attention64(rows, q, scale)
            assert_within(read_port(hip, out, q.shape), want, bound)
            work()
            assert_within(read_port(hip, out, q.shape), want, bound)
    finally:
        graph.close()


def check_window(rows, window=0, sinks=0, work=None):
    scale = float(np.float32(rows.dim**-0.5))
    q = queries(rows)
    want, bound = attention64(rows, q, scale, window, sinks)
    qr, out = rows.buffer(q), rows.buffer(np.zeros_like(q))
    rows.cache.window_attention(Op.causal_attention(rows.layer, rows.heads, rows.kv_heads, rows.dim, scale),
                                rows.tokens, qr, out, window, sinks)
    assert_within(read_port(rows.hip, out, q.shape), want, bound)


# rows of few tokens split further than those of many, the other way round, one kind not at all
MIXED = [([5000, 100, 3000], [1, 300, 2]), ([100, 3000, 40], [1, 200, 3]), ([20, 4000], [1, 20]),
         ([7000, 0], [1, 40]), ([0, 6000, 30, 6100], [0, 1, 60, 8])]


@pytest.mark.parametrize("lens,news", MIXED)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (8, 2, 128), (6, 2, 80), (10, 1, 192)])
def test_rows_of_both_kinds(hip, lens, news, heads, kv_heads, dim):
    rng = np.random.default_rng(sum(lens) + dim)
    check_window(Rows(hip, rng, heads, kv_heads, dim, lens, news))


def test_a_prompt_that_fills_the_chip_beside_long_rows(hip):
    """The prompt's blocks are not split and write their results at once."""
    rng = np.random.default_rng(2)
    check_window(Rows(hip, rng, 32, 8, 64, [9000, 0, 2000], [1, 1700, 3]), 3000, 4)


def test_rows_change_their_kind_between_replays(hip):
    """Captured with one row of many tokens beside rows of one; replayed with the
    many in another row, and with all rows of one kind."""
    rng = np.random.default_rng(3)
    news = [[1, 100, 1], [100, 1, 1], [34, 34, 34], [94, 8, 0], [1, 100, 1]]
    lens = [[4000, 30, 900], [10, 4000, 0], [100, 2000, 3], [4000, 4000, 900], [0, 0, 4000]]
    most = [max(l[b] + n[b] for l, n in zip(lens, news)) for b in range(3)]
    rows = Rows(hip, rng, 8, 2, 64, [m - 1 for m in most], [1] * 3)
    q = (rng.standard_normal((102, 8, 64)) * 2).astype(np.float32)
    op = Op.causal_attention(0, 8, 2, 64, 0.125)
    qr, out = rows.buffer(q), rows.buffer(np.zeros_like(q))

    def put(i):
        rows.lens, rows.news = lens[i], news[i]
        hip.upload_u32(rows.cache.lens_buffer, np.asarray(rows.lens, np.uint32))
        rows.tokens.set(rows.news)

    put(0)
    graph = Graph(hip, lambda: rows.cache.window_attention(op, rows.tokens, qr, out))
    try:
        for i in (0, 1, 2, 3, 4, 0):
            put(i)
            graph.launch()
            want, bound = attention64(rows, q, 0.125)
            assert_within(read_port(hip, out, q.shape), want, bound)
            rows.cache.window_attention(op, rows.tokens, qr, out)
            assert_within(read_port(hip, out, q.shape), want, bound)
    finally:
        graph.close()


@pytest.mark.parametrize("batch", [64, 65, 130])
@pytest.mark.parametrize("news", [{-1: 1}, {0: 1, -1: 3}, {3: 2, 63: 1}, {60: 40, -1: 1}])
def test_long_rows_among_many_that_sit_out(hip, batch, news):
    """A few long rows, split over their keys, anywhere in a large batch whose others
    have no tokens."""
    rng = np.random.default_rng(batch)
    lens, counts = [0] * batch, [0] * batch
    for b, n in news.items():
        lens[b], counts[b] = 5000 + 100 * n, n
    check_window(Rows(hip, rng, 8, 2, 64, lens, counts))
    check_window(Rows(hip, rng, 8, 2, 64, lens, counts), 3000, 20)
