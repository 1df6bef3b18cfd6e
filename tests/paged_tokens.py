"""What the tests of the operators on ragged new tokens over a paged cache
share: a cache on the device with a host copy of its pool, and the operators'
definitions in float64."""
import numpy as np

from starlight_amd.ir import BufferRef
from starlight_amd.paged import PAGE_NONE, PagedKvCache, PagedTokens, PagePool


class Rows:
    """Rows at `lens` cached positions with `news` new tokens each, pages in
    shuffled order, over a pool of `fill` values ("normal", or a constant)."""

    def __init__(self, hip, rng, heads, kv_heads, dim, lens, news, page=16, layers=1, layer=0, prefix=0, spare=3,
                 fill="normal", extra_entries=1):
        self.hip, self.rng, self.layer, self.layers, self.page = hip, rng, layer, layers, page
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.lens, self.news = list(lens), list(news)
        batch = len(lens)
        need = [-(-(l + n) // page) for l, n in zip(lens, news)]
        shared = -(-prefix // page)
        per_row = max(need) + extra_entries
        total = sum(max(n - shared, 0) for n in need) + shared + spare
        self.table = np.full((batch, per_row), PAGE_NONE, np.uint32)
        ids = list(rng.permutation(total))
        common = [ids.pop() for _ in range(shared)]
        for b, n in enumerate(need):
            row = common[:n] + [ids.pop() for _ in range(max(n - shared, 0))]
            self.table[b, :n] = row
        pool = PagePool(total, page, per_row, batch)
        self.cache = PagedKvCache(hip, layers, kv_heads, dim, pool)
        shape = (layers, total, 2, page, kv_heads, dim)
        self.pool = (rng.standard_normal(shape).astype(np.float32) if isinstance(fill, str)
                     else np.full(shape, fill, np.float32))
        self.tokens = PagedTokens(hip, batch)
        self.upload()

    def upload(self):
        self.hip.upload_f32(self.cache.pool_buffer, self.pool.ravel())
        self.hip.upload_u32(self.cache.table_buffer, self.table.ravel())
        self.hip.upload_u32(self.cache.lens_buffer, np.asarray(self.lens, np.uint32))
        self.tokens.set(self.news)

    @property
    def total(self):
        return sum(self.news)

    def device_pool(self):
        return self.hip.read_f32(self.cache.pool_buffer, self.pool.size).reshape(self.pool.shape)

    def at(self, b, j):
        """(page, slot) of position j of row b."""
        return int(self.table[b, j // self.page]), j % self.page

    def put(self, b, j, k, v):
        p, s = self.at(b, j)
        self.pool[self.layer, p, 0, s], self.pool[self.layer, p, 1, s] = k, v

    def kv(self, b, positions):
        """K and V rows [positions, kv_heads, dim] in float64."""
        pages = self.table[b, np.asarray(positions) // self.page].astype(np.int64)
        slots = np.asarray(positions) % self.page
        return (self.pool[self.layer, pages, 0, slots].astype(np.float64),
                self.pool[self.layer, pages, 1, slots].astype(np.float64))

    def buffer(self, values, offset=0):
        """`values` in a new buffer from `offset` on, sentinels around them."""
        values = np.asarray(values, np.float32).ravel()
        whole = np.full(values.size + offset + 5, SENTINEL, np.float32)
        whole[offset:offset + values.size] = values
        b = self.hip.upload_new_f32(whole)
        return BufferRef(b, offset, values.size)


SENTINEL = np.float32(-77.25)


def read_port(hip, ref, shape):
    """A port's values; what lies around them has to be as `buffer` left it."""
    whole = hip.read_f32(ref.buffer, ref.len + ref.offset + 5)
    assert (whole[:ref.offset] == SENTINEL).all() and (whole[ref.offset + ref.len:] == SENTINEL).all()
    return whole[ref.offset:ref.offset + ref.len].reshape(shape)


def visible(position, window, sinks):
    j = np.arange(position + 1)
    return j if window == 0 else j[(j > position - window) | (j < sinks)]


def attention64(rows, q, scale, window=0, sinks=0):
    """The attention of every new token in float64, and a bound on what an f32
    implementation with two fp16 parts per operand may be off, value by value.

    A score is off by at most 2^-20 of |scale| sum_d |q_d k_d|: 2 x 2^-22 from the
    parts of its operands and the product left out, 2^-22 from sums of up to
    256 terms rounded at 2^-24 in steps of 32, doubled. With d the largest such
    error of a query's keys, a weight is off by 2 d of itself (its numerator
    and the sum), and by 2^-20 for exp2, the weight's and the value's parts
    and the sums within a tile; each of the up to keys / 32 tiles and splits
    rounds the running sums once more (2^-23 with the rescale). The result is
    off by that share of sum_j w_j |v_j|."""
    group = rows.heads // rows.kv_heads
    out = np.zeros((rows.total, rows.heads, rows.dim))
    bound = np.zeros_like(out)
    t = 0
    for b, (past, new) in enumerate(zip(rows.lens, rows.news)):
        for i in range(new):
            j = visible(past + i, window, sinks)
            k, v = rows.kv(b, j)
            for h in range(rows.heads):
                x, kk, vv = q[t, h].astype(np.float64), k[:, h // group], v[:, h // group]
                s = scale * (kk @ x)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h] = w @ vv
                d = abs(scale) * (np.abs(kk) @ np.abs(x)).max() * 2.0**-20
                bound[t, h] = (w @ np.abs(vv)) * (2 * d + 2.0**-20 + (len(j) // 32 + 1) * 2.0**-23)
            t += 1
    return out, bound


def assert_within(got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= bound + 1e-37)
    assert not bad.any(), (f"{bad.sum()} of {bad.size} values off, first at {np.argwhere(bad)[0]}: "
                           f"{got[bad][0]!r} for {want[bad][0]!r}, {off[bad][0]:.3g} > {bound[bad][0]:.3g}")
