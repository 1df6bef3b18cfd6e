"""sl_hip_paged_window_attention on the GPU against its definition in float64:
ragged rows, windows and sinks of every relation to the lengths and pages, head
layouts, stale pages, masked values that are not finite, far-apart magnitudes."""
import math

import numpy as np
import pytest

from paged_tokens import Rows, assert_within, attention64, read_port
from starlight_amd.device import HipDevice
from starlight_amd.ir import Op
from starlight_amd.paged import PAGE_NONE

pytestmark = pytest.mark.gpu


def queries(rows, factor=2.0):
    return (rows.rng.standard_normal((rows.total, rows.heads, rows.dim)) * factor).astype(np.float32)


def attend(rows, q, scale, window=0, sinks=0, offset=0):
    qr, out = rows.buffer(q, offset), rows.buffer(np.zeros_like(q), offset)
    rows.cache.window_attention(Op.causal_attention(rows.layer, rows.heads, rows.kv_heads, rows.dim, scale),
                                rows.tokens, qr, out, window, sinks)
    return read_port(rows.hip, out, q.shape)


def check(rows, window=0, sinks=0, scale=None, q=None, offset=0):
    scale = float(np.float32(1.0 / math.sqrt(rows.dim) if scale is None else scale))
    q = queries(rows) if q is None else q
    want, bound = attention64(rows, q, scale, window, sinks)
    assert_within(attend(rows, q, scale, window, sinks, offset), want, bound)


LAYOUTS = [(4, 4, 64), (32, 8, 64), (32, 8, 128), (8, 1, 256), (12, 4, 192), (6, 2, 16), (3, 3, 80), (5, 1, 48),
           (40, 2, 96), (20, 1, 112)]


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_head_layouts(hip, heads, kv_heads, dim):
    rng = np.random.default_rng(heads + dim)
    check(Rows(hip, rng, heads, kv_heads, dim, [0, 37, 200, 16], [1, 1, 3, 40], layers=2, layer=1), 50, 4)


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 7), (1, 0), (1, 1), (2, 3), (15, 0), (16, 16), (17, 1),
                                          (33, 20), (64, 500), (100, 4), (250, 15), (5000, 4)])
@pytest.mark.parametrize("lens,news", [([0, 1, 40, 300], [1, 1, 1, 1]), ([0, 5, 130], [90, 33, 20])])
def test_windows_and_sinks(hip, window, sinks, lens, news):
    rng = np.random.default_rng(window * 31 + sinks)
    check(Rows(hip, rng, 4, 2, 64, lens, news), window, sinks)


@pytest.mark.parametrize("page", [16, 32, 48, 112])
def test_page_sizes(hip, page):
    rng = np.random.default_rng(page)
    check(Rows(hip, rng, 8, 2, 128, [0, 95, 333], [70, 1, 17], page), 60, 5)
    check(Rows(hip, rng, 8, 2, 128, [0, 95, 333], [70, 1, 17], page))


@pytest.mark.parametrize("lens,news", [([0], [1]), ([0], [2]), ([0], [17]), ([1], [1]), ([15], [1]), ([31], [2]),
                                       ([3, 0, 0, 9], [0, 1, 0, 2]), ([0] * 5, [1, 2, 3, 4, 5]),
                                       ([700, 3], [1, 300]), ([0], [513])])
def test_lengths(hip, lens, news):
    rng = np.random.default_rng(sum(lens) * 7 + sum(news))
    check(Rows(hip, rng, 8, 2, 64, lens, news))


@pytest.mark.parametrize("batch", [63, 64, 65, 150])
def test_many_rows(hip, batch):
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0, 100, batch)]
    news = [int(x) for x in rng.integers(0, 4, batch)]
    check(Rows(hip, rng, 4, 1, 64, lens, news), 40, 2)


@pytest.mark.parametrize("dim,lens,window", [(128, [20000], 0), (64, [9000, 12], 4096), (128, [30011, 17000], 5000)])
def test_long_rows_are_split(hip, dim, lens, window):
    rng = np.random.default_rng(dim)
    check(Rows(hip, rng, 8, 2, dim, lens, [1] * len(lens)), window, 4)


@pytest.mark.parametrize("offset", [1, 2, 3, 4])
def test_ports_at_any_offset(hip, offset):
    rng = np.random.default_rng(offset)
    check(Rows(hip, rng, 8, 2, 64, [40, 300], [3, 20]), 100, 4, offset=offset)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_scales(hip, scale):
    rng = np.random.default_rng(3)
    check(Rows(hip, rng, 4, 2, 64, [40, 300], [3, 20]), 100, 4, scale=scale, q=None)


def test_pages_that_nothing_sees_are_not_read(hip):
    """Behind the window every table entry is SL_PAGE_NONE; in the pages that are
    read, what lies before the window, past the last token and in every other
    page is NaN: none of it reaches a result."""
    rng = np.random.default_rng(4)
    window, sinks = 37, 5
    rows = Rows(hip, rng, 8, 2, 128, [200, 90, 0, 333], [1, 30, 5, 2])
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
    """A later token of the chunk holds values that are not finite: the tokens
    before it come out as if it were not there."""
    rng = np.random.default_rng(5)
    rows = Rows(hip, rng, 4, 2, dim, [30, 2], [9, 40])
    q, scale = queries(rows), float(np.float32(dim**-0.5))
    want, bound = attention64(rows, q, scale)
    for b, i in ((0, 6), (1, 25)):
        p, s = rows.at(b, rows.lens[b] + i)
        rows.pool[0, p, :, s, 1, 3] = value
    rows.upload()
    got = attend(rows, q, scale)
    clean = np.ones(got.shape[:2], bool)
    clean[6:9, 2:] = clean[9 + 25:, 2:] = False  # the tokens that see it, on KV head 1
    assert_within(got[clean], want[clean], bound[clean])


@pytest.mark.parametrize("kv,qf", [(1e-6, 1.0), (1e-20, 1.0), (3e4, 1e-4), (1e15, 1e-15), (1e-3, 30.0)])
def test_magnitudes(hip, kv, qf):
    rng = np.random.default_rng(6)
    rows = Rows(hip, rng, 8, 2, 64, [70, 400], [5, 1])
    rows.pool *= np.float32(kv)
    rows.upload()
    check(rows, 0, 0, q=queries(rows, qf))


def test_keys_and_values_of_far_apart_magnitudes(hip):
    """Rows of the cache from 2^-20 to 2^20 next to one another, in rising order
    for one row and mixed for the other."""
    rng = np.random.default_rng(16)
    rows = Rows(hip, rng, 4, 2, 64, [300, 300], [1, 4])
    for b in range(2):
        f = np.exp2(np.linspace(-20, 20, 304))
        for j, x in enumerate(f if b == 0 else rng.permutation(f)):
            if j < rows.lens[b] + rows.news[b]:
                p, s = rows.at(b, j)
                rows.pool[0, p, 1, s] *= np.float32(x)
                rows.pool[0, p, 0, s] *= np.float32(min(x, 4.0))
    rows.upload()
    check(rows)


def test_large_scores(hip):
    """Scores of +-10^4 and more: the largest one decides, nothing overflows."""
    rng = np.random.default_rng(11)
    rows = Rows(hip, rng, 4, 2, 64, [70, 500], [3, 1])
    q = queries(rows, 3000.0)
    scale = 1.0
    got = attend(rows, q, scale)
    want, _ = attention64(rows, q, scale)
    group = 2
    t = 0
    for b, (l, n) in enumerate(zip(rows.lens, rows.news)):
        for i in range(n):
            k, v = rows.kv(b, np.arange(l + i + 1))
            for h in range(4):
                s = k[:, h // group] @ q[t, h].astype(np.float64)
                two = np.sort(s)[-2:]
                err = (np.abs(k[:, h // group]) @ np.abs(q[t, h].astype(np.float64))).max() * 2.0**-20
                if two[1] - two[0] > err + 20:  # one key has all the weight
                    np.testing.assert_allclose(got[t, h], want[t, h], rtol=2.0**-20, atol=1e-8)
            t += 1
    assert np.isfinite(got).all()


def test_repeated_calls_give_the_same_bits(hip):
    rng = np.random.default_rng(12)
    rows = Rows(hip, rng, 32, 8, 128, [900, 3000, 17], [1, 1, 60])
    q = queries(rows)
    first = attend(rows, q, 0.09, 700, 4)
    for _ in range(3):
        np.testing.assert_array_equal(attend(rows, q, 0.09, 700, 4), first)


def test_small_workspace(hip, monkeypatch):
    """Without room for partial results the keys are not split."""
    monkeypatch.setenv("SL_HIP_WORKSPACE_BYTES", "65536")
    with HipDevice(0) as dev:
        rng = np.random.default_rng(13)
        check(Rows(dev, rng, 32, 8, 64, [2500, 40, 1200], [1, 30, 8]), 1500, 4)
