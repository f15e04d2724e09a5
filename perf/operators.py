"""Attention over keys and values held in 4 bits, the store that fills that
cache, and the block tables it is reached through: the cases that are timed.

Formats (the framework's 16-row block columns are the pages of the cache):

  page      16 tokens (or graph nodes).  pages: uint8 [num_pages, kv_heads,
            16 * d + 128]; a record holds, in this order,
              K codes  8 * d bytes: int32 words [16 tokens, d / 8]; the word of
                       channels 8 w ... 8 w + 7 has the code of channel
                       8 w + 2 n + h in bits 4 n + 16 h ... + 3
              V codes  8 * d bytes: 16-bit halves [2, 8, 4, d / 32, 2]; half
                       (p, g, t, w, l) belongs to token 8 p + 2 t + l and has
                       the code of channel g * d / 8 + 4 w + n in bits 4 n ... + 3
              scales   fp16 [8, 2, 2, 2]: (token % 8, token / 8, K or V, scale
                       or zero)
  value     scale * (code - zero), code and zero whole numbers 0 ... 15
  slot      page * 16 + row in the page; -1: nowhere
"""
import math
import random

import torch

own = False

PAGE = 16
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def record_bytes(d):
    return PAGE * d + 128


# ---------------------------------------------------------------- cases --

def listed():
    return [
        # one decoding step of a busy server: every request adds one token
        {"name": "tables decode", "kind": "tables", "requests": 256, "max_context": 8191, "max_new": 1},
        # prompts arriving, some of them behind a shared or earlier part
        {"name": "tables prompts", "kind": "tables", "requests": 41, "max_context": 3001, "max_new": 1777},
        # the new token's keys and values of 61 decoding requests, and their read-back
        {"name": "store decode", "kind": "store", "tokens": 61, "kv_heads": 8, "d": 128, "dtype": "bf16"},
        # prompts of 16,381 tokens together, and their read-back (an export of a prefix)
        {"name": "store prompts", "kind": "store", "tokens": 16381, "kv_heads": 8, "d": 128, "dtype": "bf16"},
        # node features of a graph, compressed once per layer and read back
        {"name": "store nodes", "kind": "store", "tokens": 50003, "kv_heads": 4, "d": 64, "dtype": "fp16"},
        # a single stream: the latency of one token over a middling context
        {"name": "attend one", "kind": "attend", "requests": 1, "max_context": 4099, "max_new": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "dtype": "bf16"},
        # ordinary batched decoding
        {"name": "attend decode", "kind": "attend", "requests": 64, "max_context": 8190, "max_new": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "dtype": "bf16"},
        # a few drafted tokens per request to verify, groups of 8 heads
        {"name": "attend verify", "kind": "attend", "requests": 23, "max_context": 2047, "max_new": 6, "heads": 16,
         "kv_heads": 2, "d": 64, "dtype": "fp16"},
        # prompts, ragged, behind contexts already cached
        {"name": "attend prompts", "kind": "attend", "requests": 5, "max_context": 1201, "max_new": 1999, "heads": 32,
         "kv_heads": 8, "d": 128, "dtype": "bf16"},
        # a citation graph: 2,708 nodes in one head
        {"name": "graph small", "kind": "graph", "nodes": 2708, "heads": 1, "kv_heads": 1, "d": 64, "mean_blocks": 40,
         "dtype": "fp16"},
        # a batch of larger graphs, 8 heads, a few windows with very many blocks
        {"name": "graph large", "kind": "graph", "nodes": 131057, "heads": 8, "kv_heads": 8, "d": 64,
         "mean_blocks": 22, "dtype": "fp16"},
        # wide heads shared in groups, denser windows
        {"name": "graph wide", "kind": "graph", "nodes": 40009, "heads": 4, "kv_heads": 2, "d": 128, "mean_blocks": 80,
         "dtype": "bf16"},
    ]


def spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "store", "attend", "attend", "graph"])
    dtype = rng.choice(["fp16", "bf16"])
    d = rng.choice([64, 128])
    if kind == "tables":
        requests = spread(rng, 1, 256)
        new = rng.choice([1, spread(rng, 2, 1777)])
        if requests * new > 70000:
            new = 1
        return {"kind": kind, "requests": requests, "max_context": spread(rng, 1, 8191), "max_new": new}
    if kind == "store":
        kv_heads = rng.choice([1, 2, 4, 8])
        most = 16381 * 8 * 128 // (kv_heads * d)
        return {"kind": kind, "tokens": spread(rng, 1, most), "kv_heads": kv_heads, "d": d, "dtype": dtype}
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8])
        new = rng.choice([1, 1, rng.randint(2, 8), spread(rng, 9, 2047)])
        context = spread(rng, 1, 8190)
        # no more cached tokens, and no more scores, than the largest listed cases have
        most = max(1, min(64, 64 * 8190 // (context + new), int(8e8 / (new * (context + new) * kv_heads * group))))
        return {"kind": kind, "requests": spread(rng, 1, most), "max_context": context, "max_new": new,
                "heads": kv_heads * group, "kv_heads": kv_heads, "d": d, "dtype": dtype}
    kv_heads = rng.choice([1, 2, 4])
    group = rng.choice([1, 2])
    mean_blocks = spread(rng, 2, 80)
    most = 131057 * 22 * 8 * 64 // (mean_blocks * kv_heads * group * d)
    return {"kind": kind, "nodes": spread(rng, 16, min(131057, most)), "heads": kv_heads * group, "kv_heads": kv_heads,
            "d": d, "mean_blocks": mean_blocks, "dtype": dtype}


def lengths(case):
    """(context, new) of every request: the same for all seeds but for their order."""
    rng = random.Random("%(requests)d %(max_context)d %(max_new)d" % case)
    got = []
    for i in range(case["requests"]):
        if case["max_new"] == 1:
            got.append((rng.randint(case["max_context"] // 4, case["max_context"]), 1))
        else:
            context = rng.choice([0, rng.randint(0, case["max_context"])])
            got.append((context, rng.randint(max(1, case["max_new"] // 4), case["max_new"])))
    return got


def block_counts(case):
    """Active blocks of every window: the same for all seeds but for their order.  A heavy tail, as in power-law graphs."""
    windows = -(-case["nodes"] // PAGE)
    rng = random.Random("%(nodes)d %(mean_blocks)d" % case)
    return [min(windows, 4096, max(1, int(case["mean_blocks"] * 0.4 * rng.paretovariate(1.6)))) for _ in range(windows)]


def pages_of(n):
    return -(-n // PAGE)


def work(case):
    if case["kind"] == "tables":
        ls = lengths(case)
        tokens = sum(n for _, n in ls)
        old = sum(n if n < PAGE else 1 for _, n in ls)  # table entries looked up
        new = sum(pages_of(c + n) - pages_of(c) for c, n in ls)
        return {"bytes": 8 * len(ls) + 4 * old + 8 * new + 8 * tokens + 4 * len(ls) + 12, "flops": 0}
    if case["kind"] == "store":
        values, rows = 2 * case["tokens"] * case["kv_heads"] * case["d"], 2 * case["tokens"] * case["kv_heads"]
        # values in, codes and scales out; then slots, codes and scales in, values out
        return {"bytes": 2 * values + 2 * (values // 2 + 4 * rows) + 8 * case["tokens"] + 2 * values, "flops": 6 * values}
    d, heads, kv_heads = case["d"], case["heads"], case["kv_heads"]
    if case["kind"] == "attend":
        ls = lengths(case)
        cached, tokens = sum(c + n for c, n in ls), sum(n for _, n in ls)
        seen = sum(n * c + n * (n + 1) // 2 for c, n in ls)
        return {"bytes": cached * kv_heads * (d + 8) + 2 * 2 * tokens * heads * d + 4 * sum(pages_of(c + n) for c, n in ls),
                "flops": 4 * seen * heads * d}
    counts = block_counts(case)
    return {"bytes": len(counts) * kv_heads * record_bytes(d) + 2 * 2 * case["nodes"] * heads * d + 4 * sum(counts) + 4 * len(counts),
            "flops": 4 * PAGE * PAGE * d * heads * sum(counts)}


# --------------------------------------------------------------- inputs --

def random_pages(gen, num_pages, kv_heads, d):
    """A filled cache: codes of every value, scales and zeros as keys and values of about unit size have them."""
    dev = gen.device
    pages = torch.randint(0, 256, (num_pages, kv_heads, record_bytes(d)), generator=gen, device=dev, dtype=torch.uint8)
    scales = torch.rand((num_pages, kv_heads, 32, 1), generator=gen, device=dev) * 0.2 + 0.15
    zeros = torch.randint(5, 11, (num_pages, kv_heads, 32, 1), generator=gen, device=dev).float()
    tail = torch.cat([scales, zeros], -1).half().reshape(num_pages, kv_heads, 64)
    pages[..., PAGE * d:] = tail.view(torch.uint8)
    return pages


def int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def prepare_tables(case, gen, seed):
    dev = gen.device
    ls = lengths(case)
    random.Random(seed).shuffle(ls)
    context, new = int32([c for c, _ in ls], dev), int32([n for _, n in ls], dev)
    width = max(pages_of(c + n) for c, n in ls) + 3
    held, needed = sum(pages_of(c) for c, _ in ls), sum(pages_of(c + n) for c, n in ls)
    num_pages = needed + 5
    ids = torch.randperm(num_pages, generator=gen, device=dev).int()
    # the pages that the requests hold already, row by row; then what is free
    old = (context + PAGE - 1) // PAGE
    column = torch.arange(width, device=dev)
    filled = column[None, :] < old[:, None]
    tables = torch.full((len(ls), width), -1, dtype=torch.int32, device=dev)
    tables[filled] = ids[:held]
    free = torch.cat([torch.full((2,), -1, dtype=torch.int32, device=dev), ids[held:]])
    return {"context": context, "new": new, "tables": tables, "free": free, "begin": int32([2], dev),
            "tokens": sum(n for _, n in ls), "num_pages": num_pages, "most_new": max(n for _, n in ls),
            "most_pages": max(pages_of(c + n) for c, n in ls)}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    kind = case["kind"]
    if kind == "tables":
        return {"case": case, **prepare_tables(case, gen, seed)}
    d, kv_heads, dtype = case["d"], case["kv_heads"], DTYPES[case["dtype"]]
    if kind == "store":
        tokens = case["tokens"]
        num_pages = pages_of(tokens) + 2
        # per-channel sizes differ, as keys' do
        size = torch.exp(torch.randn((1, kv_heads, d), generator=gen, device=dev) * 0.5)
        k, v = ((torch.randn((tokens, kv_heads, d), generator=gen, device=dev) * size).to(dtype) for _ in range(2))
        # consecutive rows of pages in any order, as a slot map has them
        order = torch.randperm(num_pages, generator=gen, device=dev)
        row = torch.arange(tokens, device=dev) + 5
        slots = (order[row // PAGE] * PAGE + row % PAGE).int()
        return {"case": case, "k": k, "v": v, "slots": slots,
                "pages": torch.zeros((num_pages, kv_heads, record_bytes(d)), dtype=torch.uint8, device=dev)}
    if kind == "attend":
        state = prepare_tables(case, gen, seed)
        q = torch.randn((state["tokens"], case["heads"], d), generator=gen, device=dev).to(dtype)
        return {"case": case, **state, "q": q, "scale": d ** -0.5,
                "pages": random_pages(gen, state["num_pages"], kv_heads, d)}
    counts = block_counts(case)
    random.Random(seed).shuffle(counts)
    windows = len(counts)
    count = torch.tensor(counts, device=dev)
    offsets = torch.zeros(windows + 1, dtype=torch.int64, device=dev)
    offsets[1:] = count.cumsum(0)
    window = torch.repeat_interleave(torch.arange(windows, device=dev), count)
    rank = torch.arange(window.numel(), device=dev) - offsets[window]
    step = (windows // count)[window]
    jump = (torch.rand(window.numel(), generator=gen, device=dev) * step).long().clamp(max=step - 1)
    columns = (rank * step + jump).int()
    order = torch.argsort(count, descending=True, stable=True).int()
    q = torch.randn((case["nodes"], case["heads"], d), generator=gen, device=dev).to(dtype)
    return {"case": case, "q": q, "offsets": offsets.int(), "columns": columns, "order": order, "scale": d ** -0.5,
            "pages": random_pages(gen, windows, kv_heads, d)}


# ---------------------------------------------------------- plain forms --

def codes_of_k(pages, d):
    """[..., 16, d] codes of the K half of page records."""
    words = pages[..., :8 * d].contiguous().view(torch.int32).unflatten(-1, (PAGE, d // 8))
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=pages.device)
    return ((words[..., None] >> shifts) & 15).flatten(-2)


def codes_of_v(pages, d):
    halves = pages[..., 8 * d:PAGE * d].contiguous().view(torch.int16).unflatten(-1, (2, 8, 4, d // 32, 2))
    halves = halves.movedim((-5, -3, -1), (-5, -4, -3))  # token (p, t, l), channel (g, w)
    shifts = torch.tensor([0, 4, 8, 12], dtype=torch.int16, device=pages.device)
    return ((halves[..., None] >> shifts) & 15).flatten(-6, -4).flatten(-3)


def values_of(pages, d, number):
    """K and V [..., 16, d] that page records stand for, as `number`s."""
    tail = pages[..., PAGE * d:].contiguous().view(torch.float16).unflatten(-1, (8, 2, 2, 2)).to(number)
    tail = tail.transpose(-4, -3).flatten(-4, -3)  # token, K or V, scale or zero
    k = tail[..., 0, 0, None] * (codes_of_k(pages, d).to(number) - tail[..., 0, 1, None])
    v = tail[..., 1, 0, None] * (codes_of_v(pages, d).to(number) - tail[..., 1, 1, None])
    return k, v


def quantised(x, number):
    """What rows of x stand for once held in 4 bits."""
    x = x.to(number)
    top, low = x.amax(-1, keepdim=True).clamp(min=0), x.amin(-1, keepdim=True).clamp(max=0)
    fifteen = torch.full((), 15.0, dtype=number, device=x.device)
    scale = ((top - low) / fifteen).half().clamp(min=2.0 ** -24, max=65504.0).to(number)
    zero = (-low / scale).round().clamp(0, 15)
    return scale * ((x / scale).round().add(zero).clamp(0, 15) - zero)


def plain_tables(state):
    """Query offsets, positions, slots, the tables with the new pages in, and the first page that is still free."""
    context, new, dev = state["context"].long(), state["new"].long(), state["context"].device
    requests = torch.arange(context.numel(), device=dev)
    offsets = torch.zeros(context.numel() + 1, dtype=torch.int64, device=dev)
    offsets[1:] = new.cumsum(0)
    old, all_pages = (context + PAGE - 1) // PAGE, (context + new + PAGE - 1) // PAGE
    taken = torch.zeros(context.numel() + 1, dtype=torch.int64, device=dev)
    taken[1:] = (all_pages - old).cumsum(0)
    column = torch.arange(state["tables"].shape[1], device=dev)[None, :]
    fresh = (column >= old[:, None]) & (column < all_pages[:, None])
    at = (state["begin"].long() + taken[:-1, None] + column - old[:, None]).clamp(0, state["free"].numel() - 1)
    tables = torch.where(fresh, state["free"][at], state["tables"])
    request = torch.repeat_interleave(requests, new, output_size=state["tokens"])
    position = context[request] + torch.arange(state["tokens"], device=dev) - offsets[request]
    slots = tables[request, position // PAGE] * PAGE + position % PAGE
    return {"query_offsets": offsets.int(), "positions": position.int(), "slots": slots.int(), "tables": tables,
            "free_begin": state["begin"] + taken[-1:].int()}


def plain_attend(state, number):
    case = state["case"]
    d, kv_heads, group = case["d"], case["kv_heads"], case["heads"] // case["kv_heads"]
    got = plain_tables(state)
    requests, most, width = state["context"].numel(), state["most_new"], state["most_pages"]
    pages = state["pages"][got["tables"][:, :width].long().clamp(min=0)]
    k, v = (x.movedim(2, 1).flatten(2, 3) for x in values_of(pages, d, number))  # [requests, kv_heads, tokens, d]
    step = torch.arange(most, device=k.device)
    row = (got["query_offsets"][:-1, None].long() + step).clamp(max=state["tokens"] - 1)
    q = state["q"][row].to(number).unflatten(2, (kv_heads, group)).movedim(2, 1).flatten(2, 3)  # [., ., most * group, d]
    scores = torch.matmul(q, k.transpose(2, 3)) * state["scale"]
    limit = (state["context"][:, None] + step).repeat_interleave(group, 1)
    hidden = torch.arange(k.shape[2], device=k.device) > limit[:, None, :, None]
    scores.masked_fill_(hidden, -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(scores, v) / scores.sum(-1, keepdim=True)
    out = out.unflatten(2, (most, group)).movedim(1, 2).flatten(2, 3)  # [requests, most, heads, d]
    return out[step < state["new"][:, None]]


def plain_graph(state, number):
    case = state["case"]
    nodes, d, heads, kv_heads = case["nodes"], case["d"], case["heads"], case["kv_heads"]
    windows, dev = state["offsets"].numel() - 1, state["q"].device
    k, v = values_of(state["pages"], d, number)  # [windows, kv_heads, 16, d]
    q = torch.zeros((windows * PAGE, heads, d), dtype=number, device=dev)
    q[:nodes] = state["q"].to(number)
    q = q.unflatten(0, (windows, PAGE)).movedim(1, 2)  # [windows, heads, 16, d]
    counts = (state["offsets"][1:] - state["offsets"][:-1]).long()
    window, column = torch.repeat_interleave(torch.arange(windows, device=dev), counts), state["columns"].long()
    group = heads // kv_heads
    qb = q[window].unflatten(1, (kv_heads, group)).flatten(2, 3)  # [blocks, kv_heads, group * 16, d]
    scores = torch.matmul(qb, k[column].transpose(2, 3)) * state["scale"]
    beyond = column[:, None] * PAGE + torch.arange(PAGE, device=dev) >= nodes
    scores.masked_fill_(beyond[:, None, None, :], -math.inf)
    rows = scores.amax(-1)
    top = torch.full((windows,) + rows.shape[1:], -math.inf, dtype=number, device=dev)
    top.scatter_reduce_(0, window[:, None, None].expand_as(rows), rows, "amax")
    scores = torch.exp(scores - top[window][..., None])
    total = torch.zeros_like(top).index_add_(0, window, scores.sum(-1))
    out = torch.zeros((windows, kv_heads, group * PAGE, d), dtype=number, device=dev)
    out.index_add_(0, window, torch.matmul(scores, v[column]))
    out = out / total[..., None]
    out = out.unflatten(2, (group, PAGE)).flatten(1, 2)  # [windows, heads, 16, d]
    return out.movedim(1, 2).flatten(0, 1)[:nodes]


# ------------------------------------------------------------------ run --

def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "tables":
            return plain_tables(state)
        if kind == "store":
            return [quantised(state[name], torch.float32).to(state[name].dtype) for name in ("k", "v")]
        plain = plain_attend if kind == "attend" else plain_graph
        return plain(state, torch.float32).to(state["q"].dtype)
    import fused3s_b200 as F
    if kind == "tables":
        bt = F.build_block_tables(state["context"], state["new"], state["tables"], state["free"], state["begin"],
                                  state["tokens"])
        return {"query_offsets": bt.query_offsets, "positions": bt.positions, "slots": bt.slots, "tables": bt.tables,
                "free_begin": bt.free_begin}
    cache = F.KV4Cache(state["pages"])
    if kind == "store":
        F.store_kv4(state["k"], state["v"], state["slots"], cache)
        return list(F.load_kv4(cache, state["slots"], state["k"].dtype))
    if kind == "attend":
        bt = F.build_block_tables(state["context"], state["new"], state["tables"], state["free"], state["begin"],
                                  state["tokens"], heads=case["heads"], kv_heads=case["kv_heads"])
        return F.attention_kv4(state["q"], cache, bt, scale=state["scale"])
    fmt = F.BlockSparseFormat(state["offsets"].numel() - 1, state["offsets"], state["columns"], case["nodes"])
    return F.fused3s_forward_kv4(state["q"], cache, fmt, order=state["order"], scale=state["scale"],
                                 out_dtype=state["q"].dtype)


# ---------------------------------------------------------------- exact --

def exact_values(pages, d):
    """K and V [pages, kv_heads, 16, d] in 64 bits, code by code from the description of the format."""
    dev = pages.device
    token, channel = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None, :]
    k_bit = 4 * ((channel % 8) // 2) + 16 * (channel % 2)
    k_at = token * (d // 2) + (channel // 8) * 4 + k_bit // 8
    g, w, n = channel // (d // 8), channel % (d // 8) // 4, channel % 4
    half = (((token // 8 * 8 + g) * 4 + token % 8 // 2) * (d // 32) + w) * 2 + token % 2
    v_at = 8 * d + 2 * half + n // 2
    tail = pages[..., PAGE * d:].contiguous().view(torch.float16).double()
    place = (token[:, 0] % 8) * 8 + token[:, 0] // 8 * 4
    got = []
    for at, bit, which in ((k_at, k_bit % 8, 0), (v_at, 4 * (n % 2) + 0 * token, 2)):
        code = torch.bitwise_and(torch.bitwise_right_shift(pages[..., at], bit.to(torch.uint8)), 15).double()
        got.append(tail[..., place + which, None] * (code - tail[..., place + which + 1, None]))
    return got


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None
    state = prepare(case, seed)
    if kind == "store":
        return [exact_rows(state[name].double()) for name in ("k", "v")]
    d, heads = case["d"], case["heads"]
    group = heads // case["kv_heads"]
    k, v = exact_values(state["pages"], d)
    q = state["q"].double()
    out = torch.zeros_like(q)
    if kind == "attend":
        tables, first = plain_tables(state)["tables"].cpu(), 0
        for i, (context, new) in enumerate(zip(state["context"].tolist(), state["new"].tolist())):
            length = context + new
            at = tables[i, :pages_of(length)].long().to(q.device)
            kr, vr = (x[at].transpose(0, 1).flatten(1, 2)[:, :length] for x in (k, v))
            for r in range(first, first + new, 512):
                rows = torch.arange(r, min(r + 512, first + new), device=q.device)
                s = torch.einsum("nhgd,htd->hgnt", q[rows].unflatten(1, (-1, group)), kr) * state["scale"]
                s = s.masked_fill(torch.arange(length, device=q.device)[None, :] > (rows - first + context)[:, None], -math.inf)
                out[rows] = torch.einsum("hgnt,htd->nhgd", torch.softmax(s, -1), vr).flatten(1, 2)
            first += new
        return out
    # the windows with as many blocks as each other at a time
    counts = (state["offsets"][1:] - state["offsets"][:-1]).long()
    nodes = case["nodes"]
    for count in counts.unique().tolist():
        same = torch.nonzero(counts == count)[:, 0]
        share = max(1, int(2e8) // (count * PAGE * max(d, PAGE) * heads))
        for part in same.split(share):
            columns = state["columns"][state["offsets"][part].long()[:, None] + torch.arange(count, device=q.device)].long()
            kr, vr = (x[columns].transpose(1, 2).flatten(2, 3) for x in (k, v))  # [part, kv_heads, count * 16, d]
            node = part[:, None] * PAGE + torch.arange(PAGE, device=q.device)
            qr = q[node.clamp(max=nodes - 1)].unflatten(2, (-1, group))
            s = torch.einsum("wrhgd,whtd->whgrt", qr, kr) * state["scale"]
            beyond = (columns[:, :, None] * PAGE + torch.arange(PAGE, device=q.device)).flatten(1) >= nodes
            s = s.masked_fill(beyond[:, None, None, None, :], -math.inf)
            o = torch.einsum("whgrt,whtd->wrhgd", torch.softmax(s, -1), vr).flatten(2, 3)
            out[node[node < nodes]] = o[node < nodes]
    return out


def exact_rows(x):
    """The values of quantised rows: the scale is the row's range with zero in it over 15, held in fp16."""
    low, top = x.min(-1, keepdim=True).values.clamp(max=0), x.max(-1, keepdim=True).values.clamp(min=0)
    scale = ((top - low) / 15).to(torch.float16).clamp(2.0 ** -24, 65504.0).double()
    zero = torch.round(-low / scale).clamp(0, 15)
    return scale * (torch.clamp(torch.round(x / scale) + zero, 0, 15) - zero)
