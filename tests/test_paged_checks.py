"""What the operators on ragged new tokens over a paged cache refuse, through
sl_hip_validate_paged (no GPU): arguments, shapes, buffers, row starts, lengths
and block tables."""
import dataclasses

import numpy as np
import pytest

from starlight_amd import device
from starlight_amd.device import PAGED_APPEND, PAGED_PREFIX, PAGED_WINDOW, DeviceError, validate_paged
from starlight_amd.ir import BufferRef, Op, RopeVariant
from starlight_amd.paged import PAGE_NONE, CPagedKv, CPagedTokens

H, HKV, D = 8, 2, 64
KINDS = [PAGED_APPEND, PAGED_WINDOW, PAGED_PREFIX]


class Call:
    """A call that is accepted: three rows, the first two sharing page 9 for
    positions 0-15, in a pool of 12 pages of 16 positions."""

    def __init__(self, kind):
        self.kind = kind
        self.op = Op.causal_attention(1, H, HKV, D, 0.125)
        self.rope = Op.rope(RopeVariant.NEOX, 10_000.0)
        self.starts = [0, 2, 2, 5]
        self.lens = [20, 40, 30]
        self.table = np.array([[9, 1, PAGE_NONE], [9, 2, 3], [9, 5, 6]], np.uint32)
        self.kv = dict(pool=0, block_table=1, seq_lens=2, layers=2, num_pages=12, page_size=16, pages_per_seq=3)
        self.tokens = dict(batch=3, tokens=5, row_starts=3)
        self.q = BufferRef(4, 0, 5 * H * D)
        self.k = BufferRef(5, 0, 5 * HKV * D)
        self.v = BufferRef(6, 7, 5 * HKV * D)
        self.out = BufferRef(7, 0, 5 * H * D)
        self.window, self.sinks = (16, 0) if kind == PAGED_PREFIX else (10, 4)
        f32, u32 = lambda n: {"kind": "f32", "elements": n}, lambda n: {"kind": "u32", "elements": n}
        self.buffers = [f32(2 * 12 * 2 * 16 * HKV * D), u32(9), u32(3), u32(4), f32(5 * H * D), f32(5 * HKV * D),
                        f32(5 * HKV * D + 8), f32(5 * H * D)]

    def run(self):
        k = self.k if self.kind == PAGED_APPEND else None
        v = self.v if self.kind == PAGED_APPEND else None
        return validate_paged(self.buffers, self.kind, self.op, CPagedTokens(**self.tokens, reserved=0),
                              CPagedKv(**self.kv, reserved=0), self.starts, self.lens, self.table, self.q, k, v,
                              self.out, self.rope if self.kind == PAGED_APPEND else None, self.window, self.sinks)


def execution(text):
    return DeviceError.execution(text)


@pytest.mark.parametrize("kind", KINDS)
def test_accepted(kind):
    assert Call(kind).run() is None


def test_append_takes_queries_or_none_and_no_rotation():
    c = Call(PAGED_APPEND)
    c.rope = None
    assert c.run() is None
    c.q = c.out = None
    assert c.run() is None
    c.q = BufferRef(4, 0, 5 * H * D)
    assert c.run() == execution("queries and rotated queries are given together")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("change,error", [
    (dict(code=Op.rope(RopeVariant.NEOX, 1.0).code), DeviceError("UnsupportedOp", op=5)),
    (dict(heads=7), execution("heads must be a multiple of kv_heads")),
    (dict(kv_heads=0), execution("heads must be a multiple of kv_heads")),
    (dict(heads=0), execution("heads must be a multiple of kv_heads")),
    (dict(head_dim=0), DeviceError.unimplemented("paged operators need head_dim a multiple of 16 up to 256")),
    (dict(head_dim=72), DeviceError.unimplemented("paged operators need head_dim a multiple of 16 up to 256")),
    (dict(head_dim=272), DeviceError.unimplemented("paged operators need head_dim a multiple of 16 up to 256")),
    (dict(heads=1026), DeviceError.unimplemented("paged operators take at most 1024 heads")),
    (dict(layer=2), execution("layer is out of range")),
    (dict(kv_heads=4), execution("page pool size does not match its layout")),
])
def test_op(kind, change, error):
    c = Call(kind)
    c.op = dataclasses.replace(c.op, **change)
    assert c.run() == error


@pytest.mark.parametrize("kind", [PAGED_WINDOW, PAGED_PREFIX])
@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_scale(kind, scale):
    c = Call(kind)
    c.op = dataclasses.replace(c.op, scale=scale)
    assert c.run() == execution("attention scale must be finite")


@pytest.mark.parametrize("rope,error", [
    (Op.silu(), DeviceError("UnsupportedOp", op=6)),
    (Op.rope(RopeVariant.NEOX, 0.0), execution("rope theta must be positive and finite")),
    (Op.rope(RopeVariant.GPTJ, -3.0), execution("rope theta must be positive and finite")),
    (Op.rope(RopeVariant.NEOX, float("nan")), execution("rope theta must be positive and finite")),
    (Op.rope(RopeVariant.NEOX, float("inf")), execution("rope theta must be positive and finite")),
])
def test_rope(rope, error):
    c = Call(PAGED_APPEND)
    c.rope = rope
    assert c.run() == error


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("change,error", [
    (dict(page_size=0), DeviceError.unimplemented("page_size must be a nonzero multiple of 16")),
    (dict(page_size=24), DeviceError.unimplemented("page_size must be a nonzero multiple of 16")),
    (dict(num_pages=0), execution("the page pool is empty")),
    (dict(pages_per_seq=0), execution("the page pool is empty")),
    (dict(layers=0), execution("layer is out of range")),
    (dict(num_pages=13), execution("page pool size does not match its layout")),
    (dict(pages_per_seq=4), execution("block table or lengths buffer is too small for the batch")),
    (dict(pages_per_seq=0xFFFFFFFF), DeviceError.unimplemented("a block table covers more than 2^31 - 1 positions")),
    (dict(pool=1), DeviceError.invalid_buffer(1)),
    (dict(pool=99), DeviceError.invalid_buffer(99)),
    (dict(block_table=0), DeviceError.invalid_buffer(0)),
    (dict(seq_lens=4), DeviceError.invalid_buffer(4)),
])
def test_cache(kind, change, error):
    c = Call(kind)
    c.kv.update(change)
    assert c.run() == error


@pytest.mark.parametrize("kind", KINDS)
def test_token_counts(kind):
    c = Call(kind)
    c.tokens["row_starts"] = 7
    assert c.run() == DeviceError.invalid_buffer(7)
    c = Call(kind)
    c.buffers[3]["elements"] = 3
    assert c.run() == execution("row starts buffer is too small for the batch")
    c = Call(kind)
    c.buffers[2]["elements"] = 2
    assert c.run() == execution("block table or lengths buffer is too small for the batch")
    c = Call(kind)
    c.buffers[1]["elements"] = (1 << 22) + 1
    assert c.run() == DeviceError.unimplemented("block table, lengths and row starts must be u32 buffers of at most "
                                                "16 MiB")
    c = Call(kind)
    c.tokens["tokens"] = 1 << 29
    assert c.run() == DeviceError.unimplemented("too many tokens or rows for one call")
    for starts in ([1, 2, 2, 5], [0, 3, 2, 5], [0, 2, 2, 4], [0, 6, 2, 5]):
        c = Call(kind)
        c.starts = starts
        assert c.run() == execution("row starts must rise from 0 to the number of tokens")


@pytest.mark.parametrize("kind", KINDS)
def test_ports(kind):
    for name in ("q", "out") + (("k", "v") if kind == PAGED_APPEND else ()):
        c = Call(kind)
        setattr(c, name, dataclasses.replace(getattr(c, name), len=getattr(c, name).len - 1))
        assert c.run() == execution("paged operator port has the wrong length")
        c = Call(kind)
        r = getattr(c, name)
        setattr(c, name, dataclasses.replace(r, offset=9))
        assert c.run() == DeviceError.invalid_range(r.buffer, 9, r.len)
        c = Call(kind)
        setattr(c, name, dataclasses.replace(r, buffer=3))
        assert c.run() == DeviceError.invalid_buffer(3)
        c = Call(kind)
        setattr(c, name, dataclasses.replace(r, buffer=0))
        assert c.run() == execution("a command output aliases an overlapping input range")
    c = Call(kind)
    c.buffers[4]["elements"] *= 2
    c.out = BufferRef(4, 5 * H * D - 1, 5 * H * D)
    assert c.run() == execution("a command output aliases an overlapping input range")
    c.out = BufferRef(4, 5 * H * D, 5 * H * D)
    assert c.run() is None


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_past_the_table(kind):
    c = Call(kind)
    c.lens[2] = 45
    assert c.run() is None
    c.lens[2] = 46
    assert c.run() == execution("paged KV length exceeds the row's block table")
    c.lens[2] = 0xFFFFFFFF
    assert c.run() == execution("paged KV length exceeds the row's block table")


@pytest.mark.parametrize("kind,row,entry,bad", [
    (PAGED_APPEND, 0, 1, True), (PAGED_APPEND, 0, 2, False),   # row 0 writes positions 20, 21: entry 1
    (PAGED_APPEND, 2, 1, True), (PAGED_APPEND, 2, 2, True),    # row 2 writes 30 .. 32
    (PAGED_APPEND, 1, 0, False),                               # row 1 writes nothing
    (PAGED_WINDOW, 0, 0, True),                                # row 0 sees 11 .. 21 and the sinks
    (PAGED_WINDOW, 0, 2, False), (PAGED_WINDOW, 1, 1, False),
    (PAGED_WINDOW, 2, 1, True), (PAGED_WINDOW, 2, 2, True),    # row 2 sees 21 .. 32
    (PAGED_PREFIX, 0, 1, True), (PAGED_PREFIX, 2, 2, True), (PAGED_PREFIX, 1, 0, False),
])
@pytest.mark.parametrize("value", [12, PAGE_NONE])
def test_page_ids(kind, row, entry, bad, value):
    c = Call(kind)
    c.table[row, entry] = value
    assert c.run() == (execution("page id out of range") if bad else None)


def test_entries_behind_the_window_may_be_anything():
    c = Call(PAGED_WINDOW)
    c.sinks = 0
    c.window = 8  # row 2 sees 23 .. 32
    c.table[2, 0] = 77
    assert c.run() is None
    c.sinks = 1
    assert c.run() == execution("page id out of range")
    c.window = 0
    assert c.run() == execution("page id out of range")


def test_append_refuses_pages_of_two_rows():
    twice = execution("a row appends into a page another row reads")
    c = Call(PAGED_APPEND)
    c.table[2, 2] = 1            # both rows write page 1
    assert c.run() == twice
    c = Call(PAGED_APPEND)
    c.table[2, 1] = 9            # row 2 writes the page that all read
    assert c.run() == twice
    c = Call(PAGED_APPEND)
    c.table[2, 1] = 2            # a page that row 1, which writes nothing, has cached
    assert c.run() == twice
    c = Call(PAGED_APPEND)
    c.table[2, 2] = 5            # the same page twice in one row
    assert c.run() == twice
    c = Call(PAGED_APPEND)
    c.table[2, 0] = 5            # a page the row has cached and writes
    assert c.run() == twice
    c = Call(PAGED_APPEND)
    c.table[1] = PAGE_NONE       # rows whose pages are gone
    assert c.run() is None


def test_prefix_pages_have_to_agree():
    c = Call(PAGED_PREFIX)
    c.table[2, 0] = 4
    assert c.run() == execution("a row does not begin with the shared prefix's pages")
    c = Call(PAGED_PREFIX)
    c.window = 17
    assert c.run() == execution("a row does not begin with the shared prefix's pages")
    c = Call(PAGED_PREFIX)
    c.lens[0] = 15
    assert c.run() == execution("a row is shorter than the shared prefix")
    c = Call(PAGED_PREFIX)
    c.lens[1] = 3                # a row without tokens
    assert c.run() is None
    c = Call(PAGED_PREFIX)
    c.table[:, 0] = 12
    assert c.run() == execution("page id out of range")


@pytest.mark.parametrize("kind", KINDS)
def test_null_arguments(kind):
    null = execution("paged operator received a null argument")
    for name in ("k", "v") if kind == PAGED_APPEND else ("q", "out"):
        c = Call(kind)
        setattr(c, name, None)
        assert c.run() == null
    c = Call(kind)
    c.kind = 3
    assert c.run() == null


@pytest.mark.parametrize("kind", KINDS)
def test_empty_batches(kind):
    c = Call(kind)
    c.tokens.update(batch=0, tokens=0)
    c.starts, c.lens, c.table = [0], [0], [0]
    for name in ("q", "k", "v", "out"):
        setattr(c, name, dataclasses.replace(getattr(c, name), len=0))
    assert c.run() is None


def test_tokens_of_more_rows_than_there_are():
    from starlight_amd.paged import PagedTokens

    class Fake:
        def allocate_u32(self, n, align):
            return 0

        def upload_u32(self, buffer, data):
            self.data = data

    fake = Fake()
    t = PagedTokens(fake, 3)
    t.set([2, 0])
    assert list(fake.data) == [0, 2, 2, 2] and (t.c_struct.batch, t.c_struct.tokens) == (2, 2)
    for bad in ([1, 1, 1, 1], [1, -1]):
        with pytest.raises(ValueError):
            t.set(bad)
    assert device.PAGED_PREFIX == 2


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,batch,heads,refused", [
    ((1 << 25) // H, 3, H, False), ((1 << 25) // H + 1, 3, H, True),
    ((1 << 24) - 1, 3, 1, False), (1 << 24, 3, 1, True),
    (5, (1 << 22) // HKV, H, False), (5, (1 << 22) // HKV + 1, H, True)])
def test_what_the_launches_can_count(kind, tokens, batch, heads, refused):
    """The limits themselves: one below is refused for the buffers' sizes, which a call
    of that size would need."""
    c = Call(kind)
    c.op = Op.causal_attention(1, heads, min(heads, HKV), D, 0.125)
    c.tokens.update(tokens=tokens, batch=batch)
    c.buffers[0]["elements"] = 2 * 12 * 2 * 16 * min(heads, HKV) * D
    error = c.run()
    assert (error == DeviceError.unimplemented("too many tokens or rows for one call")) == refused
    assert error is not None
