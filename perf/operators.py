"""The paged-cache operators whose time this repository is judged by.

A serving step over a paged KV cache has rows (sequences) at lengths of their
own, each with some new tokens: one while it decodes, a few when it checks a
draft, hundreds or thousands while its prompt is read. The tokens of all rows
lie one after the other ([tokens, heads, head_dim], the layout the projections
write and the output projection reads). Three operators serve such a step:

  append  rotates the new keys and queries to their positions and stores keys
          and values in their pages (`PagedKvCache.append`)
  window  attention of every new token over the cached positions its sliding
          window and the first few (sink) positions leave visible
          (`PagedKvCache.window_attention`; without a window, all of them)
  prefix  attention of a batch whose rows begin with the same pages, the
          shared positions read once for all rows
          (`PagedKvCache.prefix_attention`)

Models are the repository's own shapes (TINY, the 1B class, the 8B shape), f32
throughout, pages of 16 positions handed out in shuffled order.
"""
from __future__ import annotations

import math
import weakref

import numpy as np
import torch

own = False  # whether `run` calls the framework's operators or computes their plain form

# heads, kv_heads, head_dim, theta
SHAPES = {"tiny": (4, 4, 64, 10_000.0), "1b": (32, 8, 64, 500_000.0), "8b": (32, 8, 128, 500_000.0)}
PAGE = 16


def _case(op, shape, batch, past, new, window=0, sinks=0, prefix=0, variant="neox", layers=1, name=None):
    """`past` and `new`: (least, most) cached positions and new tokens of a
    row, spread over the batch. A prefix counts among the cached positions."""
    c = dict(op=op, shape=shape, batch=batch, past_lo=past[0], past_hi=past[1], new_lo=new[0], new_hi=new[1],
             window=window, sinks=sinks, prefix=prefix, variant=variant, layers=layers)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a few users decoding: a call of one layer is launches and host work
        _case("append", "8b", 8, (320, 1312), (1, 1), layers=2, name="append decode 8b x8"),
        # one long prompt
        _case("append", "8b", 1, (0, 0), (2000, 2000), name="append prompt 8b 2000"),
        # prompts and decoding rows in one step, the other rotation
        _case("append", "1b", 24, (0, 2900), (1, 400), variant="gptj", layers=2, name="append mixed 1b x24"),
        # one user of a small model
        _case("window", "1b", 1, (700, 700), (1, 1), 256, 4, layers=2, name="window decode 1b x1"),
        # long conversations decoding together behind a window
        _case("window", "8b", 16, (1000, 20000), (1, 1), 4096, 4, name="window decode 8b x16"),
        # prompts' chunks and decoding rows in one step
        _case("window", "8b", 12, (10, 2500), (1, 300), 1024, 16, name="window mixed 8b x12"),
        # a long document on a small model
        _case("window", "1b", 1, (0, 0), (3001, 3001), 1000, 4, name="window prompt 1b 3001"),
        # a later chunk of a long document
        _case("window", "8b", 1, (6000, 6000), (2048, 2048), 4096, 4, name="window chunk 8b 2048"),
        # three samples of one short prompt on a small model
        _case("prefix", "1b", 3, (512, 530), (1, 1), prefix=512, layers=2, name="prefix decode 1b x3"),
        # users of one system prompt with their own questions
        _case("prefix", "8b", 16, (2010, 2500), (1, 1), prefix=2000, name="prefix decode 8b x16"),
        # many users of a long shared document
        _case("prefix", "8b", 64, (16400, 17300), (1, 1), prefix=16384, name="prefix decode 8b x64"),
        # drafts of a few tokens checked over a shared prompt
        _case("prefix", "8b", 8, (4100, 4700), (3, 6), prefix=4096, name="prefix drafts 8b x8"),
    ]


def _log_between(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "window", "window", "prefix"])
    shape = rng.choice(["tiny", "1b", "8b", "8b"])
    layers = rng.choice([1, 2])
    variant = rng.choice(["neox", "neox", "gptj"])
    if op == "append":
        if rng.random() < 0.5:  # decoding rows
            batch, top = _log_between(rng, 1, 100), _log_between(rng, 20, 3000)
            return _case(op, shape, batch, (top // 3, top), (1, 1), variant=variant, layers=layers)
        batch = _log_between(rng, 1, 20)
        most = _log_between(rng, 8, 4000 // batch)
        past = _log_between(rng, 1, 2000) - 1
        return _case(op, shape, batch, (past // 2, past), (max(1, most // 9), most), variant=variant, layers=layers)
    if op == "window":
        sinks = rng.choice([0, 1, 4, 4, 37])
        if rng.random() < 0.5:  # decoding rows
            batch = _log_between(rng, 1, 24)
            window = rng.choice([0, _log_between(rng, 16, 4500)])
            top = _log_between(rng, 20, 16000 if window else 60000 // batch)
            return _case(op, shape, batch, (top // 4, top), (1, 1), window, sinks if window else 0, layers=layers)
        batch = _log_between(rng, 1, 8)
        window = rng.choice([0, _log_between(rng, 16, 2500)])
        most = _log_between(rng, 5, 3000 // batch)
        past = _log_between(rng, 1, 3000 // batch) - 1
        return _case(op, shape, batch, (past // 2, past), (max(1, most // 7), most), window, sinks if window else 0,
                     layers=layers)
    batch = _log_between(rng, 2, 48)
    prefix = PAGE * _log_between(rng, 2, 900)
    own_most = _log_between(rng, 1, 700)
    new = rng.choice([1, 1, 1, 2, 5])
    return _case(op, shape, batch, (prefix + own_most // 8, prefix + own_most), (1, new), prefix=prefix, layers=layers)


# ------------------------------------------------------------------ inputs --


def _rows(case):
    """(cached positions, new tokens) of every row: by the case alone, the
    lengths evenly spread, the tokens evenly over their logarithm, neither in
    order."""
    b = case["batch"]
    g = np.random.default_rng([b, case["past_hi"], case["new_hi"], case["window"]])
    at = np.linspace(0.0, 1.0, b) if b > 1 else np.ones(1)
    past = np.rint(case["past_lo"] + (case["past_hi"] - case["past_lo"]) * g.permutation(at)).astype(np.int64)
    new = np.rint(case["new_lo"] * (case["new_hi"] / case["new_lo"]) ** g.permutation(at)).astype(np.int64)
    return past, new


def _tables(case, seed):
    """Block tables [batch, pages_per_seq] and the number of pages: every
    row's pages in shuffled order, the prefix's the same for all."""
    past, new = _rows(case)
    pages = -(-(past + new) // PAGE)
    shared = case["prefix"] // PAGE
    per_row = int(pages.max()) + 1
    num_pages = int((pages - shared).sum()) + shared + 3
    ids = np.random.default_rng([int(seed), 8]).permutation(num_pages)
    table = np.zeros((case["batch"], per_row), np.int64)
    table[:, :shared] = ids[:shared]
    at = shared
    for b, n in enumerate(pages):
        table[b, shared:n] = ids[at:at + n - shared]
        at += n - shared
    return table, num_pages


def _tensors(case, seed):
    """The pool and the new tokens' rows: scores of a few units, as trained
    attention has them."""
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    table, num_pages = _tables(case, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2 + 1)
    tokens = int(_rows(case)[1].sum())

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    d = dict(pool=normal(case["layers"], num_pages, 2, PAGE, kv_heads, dim), q=normal(tokens, heads, dim) * 2.0)
    if case["op"] == "append":
        d.update(k=normal(tokens, kv_heads, dim), v=normal(tokens, kv_heads, dim))
    return d, table, num_pages


_open = None  # the process's HipDevice, as long as a state uses it


def _device():
    global _open
    device = _open() if _open is not None else None
    if device is None:
        from starlight_amd.device import HipDevice
        device = HipDevice(0)
        _open = weakref.ref(device)
    return device


def _scale(case):
    return float(np.float32(1.0 / math.sqrt(SHAPES[case["shape"]][2])))


def prepare(case, seed):
    tensors, table, num_pages = _tensors(case, seed)
    past, new = _rows(case)
    starts = np.concatenate([[0], np.cumsum(new)])
    state = dict(case=case, past=past, new=new)
    if own:  # the same inputs in the device's buffers, behind the cache and tokens that a serving program keeps
        from starlight_amd.ir import BufferRef, Op, RopeVariant
        from starlight_amd.paged import PagedKvCache, PagedTokens, PagePool
        heads, kv_heads, dim, theta = SHAPES[case["shape"]]
        device = _device()
        pool = PagePool(num_pages, PAGE, table.shape[1], case["batch"])
        cache = PagedKvCache(device, case["layers"], kv_heads, dim, pool)
        for b in range(case["batch"]):
            pool.admit(b)
            pool.pages[b] = [int(p) for p in table[b, :-(-int(past[b] + new[b]) // PAGE)]]
            pool.lengths[b] = int(past[b])
        cache.sync()
        state["tokens"] = PagedTokens(device, case["batch"])
        state["tokens"].set([int(n) for n in new])
        tensors["out"] = torch.empty_like(tensors["q"])
        for name, t in tensors.items():
            buffer = cache.pool_buffer if name == "pool" else device.allocate_f32(t.numel(), 256)
            state[name] = BufferRef(buffer, 0, t.numel())
            state[name + "_view"] = device.view_f32(buffer, t.shape)
            state[name + "_view"].copy_(t)
        state["attention"] = Op.causal_attention(case["layers"] - 1, heads, kv_heads, dim, _scale(case))
        state["rope"] = Op.rope(RopeVariant.NEOX if case["variant"] == "neox" else RopeVariant.GPTJ, theta)
        return dict(state, cache=cache, device=device)
    state.update(tensors, table=torch.from_numpy(table).cuda(), lens=torch.from_numpy(past).cuda(),
                 starts=torch.from_numpy(starts).cuda())
    return state


# --------------------------------------------------------- the plain forms --


def _places(state):
    """Row and position of every new token."""
    starts = state["starts"]
    token = torch.arange(int(state["new"].sum()), device="cuda")
    row = torch.searchsorted(starts, token, right=True) - 1
    return row, token - starts[row]


def _plain_append(state):
    case, pool, k, v = state["case"], state["pool"], state["k"], state["v"]
    dim, theta = SHAPES[case["shape"]][2:]
    row, at = _places(state)
    position = state["lens"][row] + at
    pair = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
    angle = position.double()[:, None] / theta ** (2.0 * pair / dim)
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def rotate(x):
        if case["variant"] == "neox":
            a, b = x[..., :dim // 2], x[..., dim // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)

    page, slot, layer = state["table"][row, position // PAGE], position % PAGE, case["layers"] - 1
    pool[layer, page, 0, slot] = rotate(k)
    pool[layer, page, 1, slot] = v
    return rotate(state["q"]), pool


def _padded(state):
    """The queries as [batch, kv_heads, tokens * group, head_dim], rows with
    fewer tokens padded, and where each token went."""
    q, new = state["q"], state["new"]
    heads, kv_heads, dim, _ = SHAPES[state["case"]["shape"]]
    b, most, group = len(new), int(new.max()), heads // kv_heads
    row, at = _places(state)
    padded = torch.zeros(b, most, heads, dim, device="cuda")
    padded[row, at] = q
    padded = padded.view(b, most, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    return padded.reshape(b, kv_heads, most * group, dim), row, at


def _gathered(state, key, which):
    """K (0) or V (1) rows [batch, kv_heads, keys, head_dim] of the positions
    `key` [batch, keys]."""
    page = torch.gather(state["table"], 1, key // PAGE)
    return state["pool"][state["case"]["layers"] - 1, page, which, key % PAGE].transpose(1, 2).contiguous()


def _unpadded(x, state, row, at):
    heads, kv_heads, dim, _ = SHAPES[state["case"]["shape"]]
    b, most = len(state["new"]), int(state["new"].max())
    x = x.view(b, kv_heads, most, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(b, most, heads, dim)
    return x[row, at]


def _plain_window(state):
    case, past, new, lens = state["case"], state["past"], state["new"], state["lens"]
    heads, kv_heads = SHAPES[case["shape"]][:2]
    window, sinks = case["window"], case["sinks"]
    group, most = heads // kv_heads, int(new.max())
    end = lens + torch.from_numpy(new).cuda()
    # each row's visible positions: its sinks, then from the first that its first query's window holds
    first = (lens - window + 1).clamp(min=sinks) if window else torch.zeros_like(lens)
    sinks = sinks if window else 0
    span = past + new - (np.maximum(past - window + 1, sinks) if window else 0) + sinks
    slot = torch.arange(int(span.max()), device="cuda")[None, :]
    key = torch.where(slot < sinks, slot, first[:, None] + slot - sinks)
    q, row, at = _padded(state)
    inside = key < end[:, None]
    key = torch.minimum(key, end[:, None] - 1)
    scores = torch.matmul(q, _gathered(state, key, 0).transpose(2, 3)) * _scale(case)
    position = lens[:, None] + torch.arange(most, device="cuda")[None, :]
    seen = key[:, None, :] <= position[:, :, None]
    if window:
        seen &= (key[:, None, :] > position[:, :, None] - window) | (key[:, None, :] < sinks)
    seen &= inside[:, None, :]
    # (padded tokens see position 0, so that no row of the mask is empty)
    seen |= (torch.arange(most, device="cuda")[None, :] >= (end - lens)[:, None])[:, :, None]
    seen = seen.repeat_interleave(group, dim=1)[:, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    weight = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    weight = weight / weight.sum(dim=-1, keepdim=True)
    return _unpadded(torch.matmul(weight, _gathered(state, key, 1)), state, row, at)


def _plain_prefix(state):
    case, past, new, lens = state["case"], state["past"], state["new"], state["lens"]
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    b, most, group, prefix, layer = len(new), int(new.max()), heads // kv_heads, case["prefix"], case["layers"] - 1
    q, row, at = _padded(state)
    # the prefix's rows once: [kv_heads, prefix, head_dim], against the queries of all rows together
    shared = state["pool"][layer, state["table"][0, :prefix // PAGE]]
    shared = shared.permute(1, 3, 0, 2, 4).reshape(2, kv_heads, prefix, dim)
    stacked = q.transpose(0, 1).reshape(kv_heads, b * most * group, dim)
    s0 = torch.matmul(stacked, shared[0].transpose(1, 2)).view(kv_heads, b, most * group, prefix).transpose(0, 1)
    key = prefix + torch.arange(int((past + new).max()) - prefix, device="cuda")[None, :].expand(b, -1)
    end = lens + torch.from_numpy(new).cuda()
    read = torch.minimum(key, end[:, None] - 1)
    s1 = torch.matmul(q, _gathered(state, read, 0).transpose(2, 3))
    position = lens[:, None] + torch.arange(most, device="cuda")[None, :]
    seen = (key[:, None, :] <= position[:, :, None]).repeat_interleave(group, dim=1)[:, None]
    scores = torch.cat([s0, s1.masked_fill(~seen, float("-inf"))], dim=-1) * _scale(case)
    weight = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    weight = weight / weight.sum(dim=-1, keepdim=True)
    w0 = weight[..., :prefix].transpose(0, 1).reshape(kv_heads, b * most * group, prefix)
    o = torch.matmul(w0, shared[1]).view(kv_heads, b, most * group, dim).transpose(0, 1)
    return _unpadded((o + torch.matmul(weight[..., prefix:], _gathered(state, read, 1))).contiguous(), state, row, at)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        cache, tokens = state["cache"], state["tokens"]
        if op == "append":
            cache.append(state["attention"], state["rope"], tokens, state["k"], state["v"], state["q"], state["out"])
            return state["out_view"], state["pool_view"]
        if op == "window":
            cache.window_attention(state["attention"], tokens, state["q"], state["out"], case["window"],
                                   case["sinks"])
        else:
            cache.prefix_attention(state["attention"], tokens, state["q"], state["out"], case["prefix"])
        return state["out_view"]
    return {"append": _plain_append, "window": _plain_window, "prefix": _plain_prefix}[op](state)


# ---------------------------------------------------- what a pass is held to --


def _visible(case):
    """Positions of each row that at least one of its queries sees, and the
    (query, key) pairs of the batch."""
    past, new = _rows(case)
    window, sinks = case["window"], case["sinks"]
    union, pairs = [], 0
    for p, n in zip(past.tolist(), new.tolist()):
        position = np.arange(p, p + n)
        if window:
            first = np.maximum(position - window + 1, 0)
            pairs += int((position + 1 - first + np.minimum(first, sinks)).sum())
            union.append(p + n - int(first[0]) + min(int(first[0]), sinks))
        else:
            pairs += int((position + 1).sum())
            union.append(p + n)
    return union, pairs


def work(case):
    """append: q read and written, k and v read and stored. Attention: every
    visible position's K and V rows read once (a shared prefix's once for the
    batch), q read, the result written; a product and a sum per pair and
    dimension, for the scores and for the result."""
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    tokens = int(_rows(case)[1].sum())
    if case["op"] == "append":
        values = tokens * (2 * heads + 4 * kv_heads) * dim
        return {"bytes": 4 * values, "flops": 3 * tokens * (heads + kv_heads) * dim}
    union, pairs = _visible(case)
    rows = sum(union) - (len(union) - 1) * case["prefix"]
    return {"bytes": 4 * (rows * 2 * kv_heads * dim + 2 * tokens * heads * dim), "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    """The operators' definitions in float64, a row at a time."""
    tensors, table, _ = _tensors(case, seed)
    heads, kv_heads, dim, theta = SHAPES[case["shape"]]
    past, new = _rows(case)
    f64, layer = torch.float64, case["layers"] - 1
    starts = np.concatenate([[0], np.cumsum(new)])
    pool = tensors["pool"].to(f64) if case["op"] == "append" else tensors["pool"]
    q = tensors["q"].to(f64)
    out = torch.empty_like(q)
    step = torch.arange(0, dim, 2, device="cuda", dtype=f64) / dim
    frequency = torch.exp(-step * math.log(theta))
    scale = _scale(case)
    for b in range(case["batch"]):
        lo, hi, n, p = int(starts[b]), int(starts[b + 1]), int(new[b]), int(past[b])
        if case["op"] == "append":
            where = torch.arange(p, p + n, device="cuda")
            turn = torch.polar(torch.ones(n, dim // 2, device="cuda", dtype=f64), where[:, None] * frequency)[:, None]

            def rotated(x):
                if case["variant"] == "neox":
                    z = torch.complex(x[..., :dim // 2].contiguous(), x[..., dim // 2:].contiguous()) * turn
                    return torch.cat([z.real, z.imag], dim=-1)
                return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)

            pages = torch.from_numpy(table[b]).cuda()[where // PAGE]
            pool[layer, pages, 0, where % PAGE] = rotated(tensors["k"][lo:hi].to(f64))
            pool[layer, pages, 1, where % PAGE] = tensors["v"][lo:hi].to(f64)
            out[lo:hi] = rotated(q[lo:hi])
            continue
        pages = torch.from_numpy(table[b, :-(-(p + n) // PAGE)]).cuda()
        kv = pool[layer, pages].to(f64).permute(1, 3, 0, 2, 4).reshape(2, kv_heads, -1, dim)[:, :, :p + n]
        key = torch.arange(p + n, device="cuda")
        group = heads // kv_heads
        most = max(1, (1 << 28) // (group * (p + n)))
        for t in range(0, n, most):
            at = torch.arange(p + t, p + min(n, t + most), device="cuda")[:, None]
            hidden = key > at
            if case["window"]:
                hidden = hidden | ((key <= at - case["window"]) & (key >= case["sinks"]))
            for g in range(kv_heads):
                x = q[lo + t:lo + t + len(at), g * group:(g + 1) * group]
                s = (x.reshape(-1, dim) @ kv[0, g].t()).view(len(at), group, -1) * scale
                w = torch.softmax(s.masked_fill(hidden[:, None, :], float("-inf")), dim=-1)
                out[lo + t:lo + t + len(at), g * group:(g + 1) * group] = (
                    w.view(-1, p + n) @ kv[1, g]).view(len(at), group, dim)
    return (out, pool) if case["op"] == "append" else out
