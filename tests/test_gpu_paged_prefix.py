"""sl_hip_paged_prefix_attention on the GPU against the attention's definition
in float64: rows that begin with the same pages."""
import math

import numpy as np
import pytest

from paged_tokens import Rows, assert_within, attention64, read_port
from starlight_amd.device import HipDevice
from starlight_amd.ir import Op
from starlight_amd.paged import PAGE_NONE

pytestmark = pytest.mark.gpu


def attend(rows, q, scale, prefix, offset=0):
    qr, out = rows.buffer(q, offset), rows.buffer(np.zeros_like(q), offset)
    rows.cache.prefix_attention(Op.causal_attention(rows.layer, rows.heads, rows.kv_heads, rows.dim, scale),
                                rows.tokens, qr, out, prefix)
    return read_port(rows.hip, out, q.shape)


def check(rows, prefix, offset=0):
    scale = float(np.float32(1.0 / math.sqrt(rows.dim)))
    q = (rows.rng.standard_normal((rows.total, rows.heads, rows.dim)) * 2).astype(np.float32)
    want, bound = attention64(rows, q, scale)
    assert_within(attend(rows, q, scale, prefix, offset), want, bound)


LAYOUTS = [(4, 4, 64), (32, 8, 64), (32, 8, 128), (8, 1, 256), (12, 4, 192), (6, 2, 16), (3, 3, 80), (40, 2, 96)]


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_head_layouts(hip, heads, kv_heads, dim):
    rng = np.random.default_rng(heads + dim)
    check(Rows(hip, rng, heads, kv_heads, dim, [160, 161, 300, 176], [1, 2, 1, 5], prefix=160, layers=2, layer=1), 160)


@pytest.mark.parametrize("prefix", [0, 1, 5, 15, 16, 17, 32, 100, 128, 144])
@pytest.mark.parametrize("page", [16, 32])
def test_prefixes_end_anywhere(hip, prefix, page):
    """The rows' tables agree for 144 positions' pages; any shorter prefix is as
    good, page boundary or not."""
    rng = np.random.default_rng(prefix + page)
    check(Rows(hip, rng, 8, 2, 64, [144, 150, 290], [1, 3, 1], page, prefix=144), prefix)


@pytest.mark.parametrize("batch,dim", [(1, 64), (2, 128), (16, 128), (17, 64), (40, 64), (64, 128), (70, 128)])
def test_batches(hip, batch, dim):
    rng = np.random.default_rng(batch)
    lens = [512 + int(x) for x in rng.integers(0, 60, batch)]
    news = [int(x) for x in rng.integers(0, 3, batch)]
    news[0] = 1
    check(Rows(hip, rng, 8, 2, dim, lens, news, prefix=512), 512)


def test_long_prefix(hip):
    rng = np.random.default_rng(1)
    check(Rows(hip, rng, 8, 2, 128, [9000, 9100, 9033], [1, 1, 2], prefix=8992), 8992)


def test_nothing_past_the_prefix_but_the_tokens(hip):
    rng = np.random.default_rng(2)
    check(Rows(hip, rng, 8, 2, 64, [64, 64, 64], [1, 1, 7], prefix=64), 64)


def test_rows_without_tokens_are_not_looked_at(hip):
    """Rows that sit the step out, the first among them, have no pages at all."""
    rng = np.random.default_rng(3)
    rows = Rows(hip, rng, 8, 2, 64, [96, 120, 96, 99], [0, 1, 0, 2], prefix=96)
    rows.table[[0, 2]] = PAGE_NONE
    rows.lens[0] = 0
    rows.upload()
    check(rows, 96)


def test_stale_values_are_not_read(hip):
    """NaN in every slot that holds no position of a row."""
    rng = np.random.default_rng(4)
    rows = Rows(hip, rng, 8, 2, 128, [70, 81, 90], [1, 2, 1], prefix=64)
    keep = np.zeros((rows.pool.shape[1], rows.page), bool)
    for b in range(3):
        for j in range(rows.lens[b] + rows.news[b]):
            keep[rows.at(b, j)] = True
    rows.pool[0].transpose(1, 0, 2, 3, 4)[:, ~keep] = np.nan
    rows.upload()
    check(rows, 64)


def test_values_of_unseen_keys_do_not_matter(hip):
    rng = np.random.default_rng(5)
    rows = Rows(hip, rng, 4, 2, 64, [64, 70], [5, 1], prefix=64)
    q = (rng.standard_normal((rows.total, 4, 64)) * 2).astype(np.float32)
    want, bound = attention64(rows, q, 0.125)
    p, s = rows.at(0, 67)
    rows.pool[0, p, :, s] = np.inf
    rows.upload()
    got = attend(rows, q, 0.125, 64)
    keep = [0, 1, 2, 5]  # tokens before the one that holds infinities, and the other row
    assert_within(got[keep], want[keep], bound[keep])
    assert not np.isfinite(got[3:5]).any()


@pytest.mark.parametrize("offset", [1, 3])
def test_ports_at_any_offset(hip, offset):
    rng = np.random.default_rng(6)
    check(Rows(hip, rng, 4, 2, 64, [64, 70], [5, 1], prefix=64), 64, offset)


def test_small_workspace(hip, monkeypatch):
    """Without room for the partial results of both parts the rows are read one
    by one."""
    monkeypatch.setenv("SL_HIP_WORKSPACE_BYTES", "65536")
    with HipDevice(0) as dev:
        rng = np.random.default_rng(7)
        check(Rows(dev, rng, 32, 8, 64, [600, 620, 601], [2, 1, 8], prefix=592), 592)
