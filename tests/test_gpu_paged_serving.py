"""The operators on ragged new tokens as a serving loop uses them: prompts read
in chunks and decoded beside one another, against plain causal attention in
float64 of every sequence by itself; the same decode step through
sl_hip_paged_attention; HIP graphs captured from the device's stream and
replayed with other lengths; buffers shared with torch."""
import ctypes
import math

import numpy as np
import pytest

from paged_tokens import Rows, assert_within, attention64, read_port
from starlight_amd.device import DeviceError, HipDevice
from starlight_amd.ir import BufferRef, Op, RopeVariant
from starlight_amd.paged import PagedKvCache, PagedTokens, PagePool

pytestmark = pytest.mark.gpu

H, HKV, D, THETA = 8, 2, 64, 10_000.0
SCALE = float(np.float32(1.0 / math.sqrt(D)))


def rope64(x, positions):
    """NeoX rotation of [tokens, heads, D] in float64."""
    angle = positions[:, None] / THETA ** (2.0 * np.arange(D // 2) / D)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :D // 2].astype(np.float64), x[..., D // 2:].astype(np.float64)
    return np.concatenate([a * c - b * s, a * s + b * c], axis=-1)


def causal64(q, k, v, window, sinks):
    """Attention of a whole sequence, rotated, in float64."""
    n = len(q)
    pos = np.arange(n)
    qr, kr = rope64(q, pos), rope64(k, pos)
    out = np.zeros((n, H, D))
    for h in range(H):
        s = SCALE * qr[:, h] @ kr[:, h // (H // HKV)].T
        hidden = pos[None, :] > pos[:, None]
        if window:
            hidden |= (pos[None, :] <= pos[:, None] - window) & (pos[None, :] >= sinks)
        s[hidden] = -np.inf
        w = np.exp(s - s.max(axis=1, keepdims=True))
        out[:, h] = (w / w.sum(axis=1, keepdims=True)) @ v[:, h // (H // HKV)].astype(np.float64)
    return out


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_prompts_in_chunks_and_decode_together(hip, window, sinks):
    """Three sequences of 150, 77 and 20 tokens: each step takes some tokens of
    each (chunks, single tokens, none), appends and attends; every token's
    result is that of its sequence computed by itself. f32 rotations (2 roundings
    of |q| and |k|, so 2^-21 of a score's terms) add to the attention's own."""
    rng = np.random.default_rng(window)
    lengths = [150, 77, 20]
    data = [[rng.standard_normal((n, h, D)).astype(np.float32) for h in (H, HKV, HKV)] for n in lengths]
    want = [causal64(*d, window, sinks) for d in data]
    pool = PagePool(num_pages=30, page_size=16, pages_per_seq=12, max_batch=3)
    rng.shuffle(pool.free)
    cache = PagedKvCache(hip, 1, HKV, D, pool)
    tokens = PagedTokens(hip, 3)
    for b in range(3):
        pool.admit(b)
    attention, rope = Op.causal_attention(0, H, HKV, D, SCALE), Op.rope(RopeVariant.NEOX, THETA)
    steps = [[90, 0, 1], [1, 33, 0], [0, 1, 17], [1, 1, 1], [57, 41, 0], [1, 1, 1]]
    done = [0, 0, 0]
    for counts in steps:
        for b, n in enumerate(counts):
            pool.reserve(b, done[b] + n)
        cache.sync()
        tokens.set(counts)
        rows = [np.concatenate([data[b][i][done[b]:done[b] + n] for b, n in enumerate(counts)]) for i in range(3)]
        q, k, v = (hip.upload_new_f32(r) for r in rows)
        total = sum(counts)
        qr, out = hip.allocate_f32(rows[0].size, 256), hip.allocate_f32(rows[0].size, 256)
        ref = lambda buf, x: BufferRef(buf, 0, x.size)  # noqa: E731
        cache.append(attention, rope, tokens, ref(k, rows[1]), ref(v, rows[2]), ref(q, rows[0]), ref(qr, rows[0]))
        cache.window_attention(attention, tokens, ref(qr, rows[0]), ref(out, rows[0]), window, sinks)
        got = hip.read_f32(out, rows[0].size).reshape(total, H, D)
        at = 0
        for b, n in enumerate(counts):
            w = want[b][done[b]:done[b] + n]
            # scores up to |q||k| / 8: off by 2^-19 of that with the rotations; values up to 5
            np.testing.assert_allclose(got[at:at + n], w, rtol=0, atol=5 * 2.0**-16)
            at += n
            done[b] += n
            pool.lengths[b] = done[b]
    assert done == [150, 77, 20]


def test_a_decode_step_is_paged_attentions(hip):
    """One new token per row: append and window_attention (no window) give what
    sl_hip_paged_attention gives, the pool bit for bit."""
    rng = np.random.default_rng(3)
    rows = Rows(hip, rng, H, HKV, D, [5, 130, 64, 0], [1, 1, 1, 1])
    start = rows.pool.copy()
    q = rng.standard_normal((4, H, D)).astype(np.float32)
    k, v = (rng.standard_normal((4, HKV, D)).astype(np.float32) for _ in range(2))
    op = Op.causal_attention(0, H, HKV, D, SCALE)
    kr, vr, qr = rows.buffer(k), rows.buffer(v), rows.buffer(q)
    out = rows.buffer(np.zeros_like(q))
    rows.cache.append(op, None, rows.tokens, kr, vr)
    rows.cache.window_attention(op, rows.tokens, qr, out)
    got, pool = read_port(hip, out, q.shape), rows.device_pool()
    hip.upload_f32(rows.cache.pool_buffer, start.ravel())
    other = BufferRef(hip.allocate_f32(q.size, 256), 0, q.size)
    hip.paged_attention(op, qr, kr, vr, other, 4, rows.cache.c_struct())
    np.testing.assert_array_equal(rows.device_pool(), pool)
    rows.pool = pool
    want, bound = attention64(rows, q, SCALE)
    assert_within(got, want, bound)
    # (the other kernel's f32 sums are held to its own tests' tolerance)
    np.testing.assert_allclose(hip.read_f32(other.buffer, q.size).reshape(q.shape), got, rtol=0, atol=1e-5)


class Graph:
    """A HIP graph captured from a device's stream."""

    def __init__(self, dev, work):
        self.rt = ctypes.CDLL("libamdhip64.so")
        self.stream = ctypes.c_void_p(dev.stream)
        graph = ctypes.c_void_p()
        dev.synchronize()
        assert self.rt.hipStreamBeginCapture(self.stream, 1) == 0  # thread-local
        work()
        assert self.rt.hipStreamEndCapture(self.stream, ctypes.byref(graph)) == 0
        self.exec = ctypes.c_void_p()
        assert self.rt.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)) == 0
        self.graph = graph

    def launch(self):
        assert self.rt.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        self.rt.hipGraphExecDestroy(self.exec)
        self.rt.hipGraphDestroy(self.graph)


@pytest.mark.parametrize("kind", ["window", "full", "prefix"])
def test_captured_and_replayed_with_other_lengths(hip, kind):
    """Captured for rows of one token each at short lengths; replayed, between
    eager calls, with the same number of tokens dealt otherwise (one row then
    takes most of them) at longer lengths: every replay equals the definition."""
    rng = np.random.default_rng(9)
    prefix = 288 if kind == "prefix" else 0
    news = [[1] * 40, [1] * 40, [0] * 3 + [36] + [0] * 32 + [1] * 4, [2] * 20 + [0] * 20, [1] * 40]
    lens = [[prefix + x for x in row] for row in
            ([3] * 40, [int(x) for x in rng.integers(0, 900, 40)], [40] * 40, [i * 9 for i in range(40)], [0] * 40)]
    most = [max(l[b] + n[b] for l, n in zip(lens, news)) for b in range(40)]
    rows = Rows(hip, rng, H, HKV, D, [m - 1 for m in most], [1] * 40, prefix=prefix)
    q = (rng.standard_normal((40, H, D)) * 2).astype(np.float32)
    op = Op.causal_attention(0, H, HKV, D, SCALE)
    qr, out = rows.buffer(q), rows.buffer(np.zeros_like(q))
    window, sinks = (100, 5) if kind == "window" else (0, 0)

    def work():
        if kind == "prefix":
            rows.cache.prefix_attention(op, rows.tokens, qr, out, prefix)
        else:
            rows.cache.window_attention(op, rows.tokens, qr, out, window, sinks)

    def put(i):
        rows.lens, rows.news = lens[i], news[i]
        hip.upload_u32(rows.cache.lens_buffer, np.asarray(rows.lens, np.uint32))
        rows.tokens.set(rows.news)

    put(0)
    graph = Graph(hip, work)
    try:
        for i in (0, 1, 2, 3, 4, 1):
            put(i)
            graph.launch()
            want, bound = attention64(rows, q, SCALE, window, sinks)
            assert_within(read_port(hip, out, q.shape), want, bound)
            work()  # eager, between the replays
            assert_within(read_port(hip, out, q.shape), want, bound)
    finally:
        graph.close()


def test_append_captured_and_replayed(hip):
    rng = np.random.default_rng(10)
    rows = Rows(hip, rng, H, HKV, D, [60, 60, 60], [20, 1, 3])
    q = rng.standard_normal((6, H, D)).astype(np.float32)
    k, v = (rng.standard_normal((6, HKV, D)).astype(np.float32) for _ in range(2))
    op, rope = Op.causal_attention(0, H, HKV, D, SCALE), Op.rope(RopeVariant.GPTJ, THETA)
    ports = [rows.buffer(k), rows.buffer(v), rows.buffer(q), rows.buffer(np.zeros_like(q))]
    rows.tokens.set([2, 2, 2])
    graph = Graph(hip, lambda: rows.cache.append(op, rope, rows.tokens, *ports))
    try:
        for lens, news in (([0, 5, 15], [2, 2, 2]), ([60, 0, 31], [6, 0, 0]), ([17, 3, 60], [0, 5, 1])):
            rows.lens = lens
            hip.upload_u32(rows.cache.lens_buffer, np.asarray(lens, np.uint32))
            rows.tokens.set(news)
            hip.upload_f32(rows.cache.pool_buffer, rows.pool.ravel())
            graph.launch()
            replayed, rotated = rows.device_pool(), read_port(hip, ports[3], q.shape)
            assert (replayed != rows.pool).sum() > 6 * HKV * D  # K and V of six tokens
            hip.upload_f32(rows.cache.pool_buffer, rows.pool.ravel())
            rows.cache.append(op, rope, rows.tokens, *ports)
            np.testing.assert_array_equal(replayed, rows.device_pool())
            np.testing.assert_array_equal(rotated, read_port(hip, ports[3], q.shape))
    finally:
        graph.close()


def test_two_devices_handles_do_not_share_partials(hip):
    """Calls of two device handles, enqueued without waiting between them."""
    rng = np.random.default_rng(11)
    with HipDevice(0) as other:
        sides = [Rows(d, np.random.default_rng(20 + i), 32, 8, 128, [3000, 2500], [1, 2]) for i, d in
                 enumerate((hip, other))]
        qs = [(rng.standard_normal((3, 32, 128)) * 2).astype(np.float32) for _ in sides]
        scale = float(np.float32(1 / math.sqrt(128)))
        outs = []
        for rows, q in zip(sides, qs):
            outs.append((rows.buffer(q), rows.buffer(np.zeros_like(q))))
        for _ in range(4):
            for rows, (qr, out) in zip(sides, outs):
                rows.cache.window_attention(Op.causal_attention(0, 32, 8, 128, scale), rows.tokens, qr, out)
        for rows, q, (_, out) in zip(sides, qs, outs):
            want, bound = attention64(rows, q, scale)
            assert_within(read_port(rows.hip, out, q.shape), want, bound)


def test_buffers_shared_with_torch(hip):
    """A buffer filled and read through torch, in place; commands still logged
    have run before the view is given."""
    import torch

    a = hip.upload_new_f32(np.arange(12, dtype=np.float32))
    view = hip.view_f32(a, (3, 4))
    assert view.shape == (3, 4) and view.is_cuda and view.data_ptr() == hip.address(a)[0]
    view.mul_(2.0)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(hip.read_f32(a, 12), 2 * np.arange(12))
    assert hip.address(a)[1] == 12
    assert hip.view_f32(a, (2, 2), offset=8).flatten().tolist() == [16.0, 18.0, 20.0, 22.0]
    b = hip.allocate_f32(12, 256)
    from starlight_amd.ir import Value
    v = Value.f32([12])
    hip.dispatch(Op.scale_by(0.5), [BufferRef(a, 0, 12)], [v], [BufferRef(b, 0, 12)], [v])
    np.testing.assert_array_equal(hip.view_f32(b, (12,)).cpu().numpy(), np.arange(12))
    assert hip.view_f32(a, (0, 4)).shape == (0, 4)
    with pytest.raises(DeviceError) as e:
        hip.view_f32(a, (13,))
    assert e.value == DeviceError.invalid_range(a, 0, 13)
    u = hip.upload_new_u32(np.arange(4))
    with pytest.raises(DeviceError) as e:
        hip.address(u)
    assert e.value == DeviceError.invalid_buffer(u)
    empty = hip.allocate_f32(0, 256)
    assert hip.address(empty) == (0, 0)
