"""sl_hip_paged_append on the GPU: the new keys and values of ragged rows in
their pages, keys and queries rotated as the Rope operator rotates them (the
oracle's f64 angles; bit for bit against the operator on the same GPU), every
other value of the pool as it was."""
import numpy as np
import pytest

import oracle
from paged_tokens import Rows, read_port
from starlight_amd.device import DeviceError
from starlight_amd.ir import BufferRef, Op, RopeVariant, Value

pytestmark = pytest.mark.gpu


def operator_rope(hip, x, positions, theta, variant):
    """The Rope operator on [tokens, heads, dim] (as [1, heads, tokens, dim])."""
    t, heads, dim = x.shape
    src = np.ascontiguousarray(x.transpose(1, 0, 2))
    xb, pb = hip.upload_new_f32(src), hip.upload_new_u32(np.asarray(positions, np.uint32))
    ob = hip.allocate_f32(src.size, 256)
    v = Value.f32([1, heads, t, dim])
    hip.dispatch(Op.rope(variant, theta), [BufferRef(xb, 0, src.size), BufferRef(pb, 0, t)],
                 [v, Value.u32([1, t])], [BufferRef(ob, 0, src.size)], [v])
    return hip.read_f32(ob, src.size).reshape(heads, t, dim).transpose(1, 0, 2)


def run(hip, rows, theta, variant, offset=0, rotate=True, queries=True):
    rng, T = rows.rng, rows.total
    q = rng.standard_normal((T, rows.heads, rows.dim)).astype(np.float32)
    k = rng.standard_normal((T, rows.kv_heads, rows.dim)).astype(np.float32)
    v = rng.standard_normal((T, rows.kv_heads, rows.dim)).astype(np.float32)
    op = Op.causal_attention(rows.layer, rows.heads, rows.kv_heads, rows.dim, 1.0)
    rope = Op.rope(variant, theta) if rotate else None
    ports = [rows.buffer(k, offset), rows.buffer(v, offset)]
    if queries:
        ports += [rows.buffer(q, offset), rows.buffer(np.zeros_like(q), offset)]
    rows.cache.append(op, rope, rows.tokens, *ports)
    positions = np.concatenate([np.arange(l, l + n) for l, n in zip(rows.lens, rows.news)]).astype(np.int64)
    kr = operator_rope(hip, k, positions, theta, variant) if rotate else k
    at = 0
    for b, (l, n) in enumerate(zip(rows.lens, rows.news)):
        for i in range(n):
            rows.put(b, l + i, kr[at], v[at])
            at += 1
    np.testing.assert_array_equal(rows.device_pool(), rows.pool)
    if queries:
        want = operator_rope(hip, q, positions, theta, variant) if rotate else q
        np.testing.assert_array_equal(read_port(hip, ports[3], q.shape), want)
        if rotate:
            # and the oracle's rotation: f32 products and a difference of sines and
            # cosines rounded once, so 2 roundings of |x| + |y| apart at most
            flat = oracle.rope(q.transpose(1, 0, 2).ravel(), positions.astype(np.uint32), 1, rows.heads, T, rows.dim,
                               theta, "neox" if variant == RopeVariant.NEOX else "gptj")
            ref = np.asarray(flat).reshape(rows.heads, T, rows.dim).transpose(1, 0, 2)
            np.testing.assert_allclose(want, ref, rtol=0, atol=2.0**-22 * 2 * np.abs(q).max())
    return rows


LAYOUTS = [  # heads, kv_heads, dim, page
    (4, 4, 64, 16), (32, 8, 64, 16), (32, 8, 128, 16), (8, 1, 256, 32), (6, 2, 16, 48), (3, 3, 80, 16),
]


@pytest.mark.parametrize("variant", [RopeVariant.NEOX, RopeVariant.GPTJ])
@pytest.mark.parametrize("heads,kv_heads,dim,page", LAYOUTS)
def test_ragged_rows(hip, heads, kv_heads, dim, page, variant):
    """Rows of 0 to 70 tokens at positions 0 to 4,000, in the second of two
    layers: pages entered in their middle, crossed and just filled."""
    rng = np.random.default_rng(heads * dim + page)
    rows = Rows(hip, rng, heads, kv_heads, dim, [0, 15, 16, 31, 4000, 7], [33, 1, 16, 2, 70, 0], page, layers=2,
                layer=1)
    run(hip, rows, 10_000.0, variant)


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 130])
def test_one_token_per_row(hip, batch):
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0, 200, batch)]
    run(hip, Rows(hip, rng, 8, 2, 64, lens, [1] * batch), 500_000.0, RopeVariant.NEOX)


@pytest.mark.parametrize("offset", [1, 2, 3, 4])
def test_ports_at_any_offset(hip, offset):
    rng = np.random.default_rng(offset)
    run(hip, Rows(hip, rng, 4, 2, 48, [9, 0], [5, 20]), 10_000.0, RopeVariant.GPTJ, offset=offset)


def test_without_rotation_or_queries(hip):
    rng = np.random.default_rng(7)
    run(hip, Rows(hip, rng, 8, 2, 128, [3, 0, 40], [1, 30, 2]), 10_000.0, RopeVariant.NEOX, rotate=False)
    run(hip, Rows(hip, rng, 8, 2, 128, [3, 0, 40], [1, 30, 2]), 10_000.0, RopeVariant.NEOX, queries=False)
    run(hip, Rows(hip, rng, 8, 2, 128, [5], [6]), 10_000.0, RopeVariant.NEOX, rotate=False, queries=False)


def test_far_positions(hip):
    """Positions past 100,000, where an angle in f32 would be off by a percent."""
    rng = np.random.default_rng(8)
    run(hip, Rows(hip, rng, 2, 1, 64, [131_000, 100_003], [9, 1]), 10_000.0, RopeVariant.NEOX)


def test_no_tokens_is_a_no_op(hip):
    rng = np.random.default_rng(9)
    rows = Rows(hip, rng, 2, 1, 64, [5, 0], [1, 1])
    rows.tokens.set([0, 0])
    empty = BufferRef(hip.allocate_f32(16, 256), 0, 0)
    rows.cache.append(Op.causal_attention(0, 2, 1, 64, 1.0), None, rows.tokens, empty, empty)
    np.testing.assert_array_equal(rows.device_pool(), rows.pool)


def test_a_refused_call_changes_nothing(hip):
    rng = np.random.default_rng(10)
    rows = Rows(hip, rng, 2, 1, 64, [5, 20], [1, 1])
    rows.table[1, 1] = rows.table[0, 0]  # row 1 would append into row 0's page
    rows.upload()
    k = rows.buffer(np.ones(2 * 64))
    with pytest.raises(DeviceError) as e:
        rows.cache.append(Op.causal_attention(0, 2, 1, 64, 1.0), None, rows.tokens, k, k)
    assert e.value == DeviceError.execution("a row appends into a page another row reads")
    np.testing.assert_array_equal(rows.device_pool(), rows.pool)
