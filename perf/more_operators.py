"""A key/value cache kept in pages, as calls whose speed counts: its tables, the rows that go into it, the attention that reads it.

Pages hold `page` tokens each (a power of two).  The pages of a sequence stand in its row of an int32 table, those of nobody on a
stack `free`, of which `free_count` are there.  Keys and values are [pages, kv_heads, page, size]; `layout` says which way a page lies
in memory: "heads", the tokens of a head together, or "tokens", the heads of a token together.

A case names an operator by `op`:

    "extend"     sequences of lengths n grow by c = counts tokens (at most `rows` each, none more than the table holds): pages
                 are taken from the top of the stack, in the order of the sequences as long as there are enough; slots[b, t] =
                 page * `page` + place of new token t, -1 where there is none
    "cut"        sequences keep their first `keep` tokens, and the pages behind go back onto the stack, in order
    "write"      keys and values of new tokens, out of a packed projection, to their slots
    "attention"  the last `queries` tokens of every sequence over its pages: query at p sees key j if j <= p and (j >= p - left
                 or j < sinks); a bound of -1 is none.  Heads share keys and values in groups of heads / kv_heads.  Tokens
                 before the first give zeros.  "dropped": pages that the window has passed have left the table (-1)

Sizes are those of the two model configurations (12 or 16 heads of 64) and generic ones.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}


def _extend(name, batch, rows, limit, page, ragged=True, scarce=False):
    """limit: tokens that a table's row has room for; ragged: counts spread from 0 to `rows` (or all `rows`); scarce: pages for about
    half of what is asked for, and sequences that their tables have no more room for"""
    return {"name": name, "op": "extend", "batch": batch, "rows": rows, "limit": limit, "page": page, "ragged": ragged, "scarce": scarce}


def _cut(name, batch, limit, page, ends):
    """ends: the share of the sequences that end (the others give up a few tokens, as proposals that were refused)"""
    return {"name": name, "op": "cut", "batch": batch, "limit": limit, "page": page, "ends": ends}


def _write(name, dtype, batch, rows, heads, kv_heads, size, page, layout="heads"):
    return {"name": name, "op": "write", "dtype": dtype, "batch": batch, "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "size": size, "page": page, "layout": layout}


def _attention(name, dtype, batch, queries, keys, heads, kv_heads, size, page, left=-1, sinks=0, shortest=0.1, limit=None, layout="heads",
               dropped=False):
    """keys: the longest sequence (lengths are spread evenly from `shortest` times that on); limit: tokens that a table's row has room for"""
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "size": size, "page": page, "left": left, "sinks": sinks, "shortest": shortest,
            "limit": max(keys, limit or 0), "layout": layout, "dropped": dropped}


def listed():
    return [
        # a step of decoding: a token more for each of 256 sequences, of which one in 16 needs a page
        _extend("extend 256x1", 256, 1, 8192, 16, ragged=False),
        # a batch of prompts comes in, behind what some sequences have already
        _extend("extend 64x2048", 64, 2048, 8192, 16),
        # between two steps: one of eight sequences has ended
        _cut("cut 8", 8, 4096, 16, 0.125),
        # a large batch of long sequences is cleared but for a few
        _cut("cut 512", 512, 8192, 16, 0.9),
        # a token for each of eight sequences of the base model
        _write("write f32 8x1", "f32", 8, 1, 12, 12, 64, 16),
        # a prompt of odd length, with its padding, the heads of a token together
        _write("write f16 7x513", "f16", 7, 513, 16, 16, 64, 32, layout="tokens"),
        # prompts of a model with shared heads
        _write("write f16 16x2048", "f16", 16, 2048, 32, 8, 128, 16),
        # one short sequence, a token: the shortest call there is, all of it latency
        _attention("attention f16 1x1 of 64", "f16", 1, 1, 64, 12, 12, 64, 16, shortest=1.0, limit=512),
        # five proposed tokens of each of nine sequences of the base model checked at once
        _attention("attention f32 9x5", "f32", 9, 5, 1000, 12, 12, 64, 16, limit=2048),
        # 64 sequences a token each, lengths from a few tokens to 4096 in tables for 8192, four heads to a key head
        _attention("attention f16 64x1", "f16", 64, 1, 4096, 16, 4, 128, 16, shortest=0.01, limit=8192),
        # 32 sequences a token each, window of 4096 and four sinks, the heads of a token together
        _attention("attention f16 32x1 window", "f16", 32, 1, 8192, 16, 4, 128, 64, left=4095, sinks=4, layout="tokens"),
        # one long sequence a token at a time: few rows, a long axis
        _attention("attention f16 1x1 of 131072", "f16", 1, 1, 131072, 16, 2, 128, 128, shortest=1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_size(c) for c in listed())
    while True:
        c = _drawn(rng)
        if _size(c) <= most:
            c.pop("name")
            return c


def _drawn(rng):
    op = rng.choice(("extend", "cut", "write", "attention", "attention", "attention"))
    dtype = rng.choice(("f32", "f16"))
    page = rng.choice((16, 16, 32, 64, 128, 256))
    layout = rng.choice(("heads", "tokens"))
    if op == "extend":
        rows = rng.choice((1, _log(rng, 2, 8), _log(rng, 9, 4096)))
        batch = _log(rng, 1, min(2048, (1 << 18) // rows))
        return _extend("", batch, rows, max(rows, _log(rng, 64, 60000)), page, rng.random() < 0.6, rng.random() < 0.2)
    if op == "cut":
        return _cut("", _log(rng, 1, 1024), _log(rng, 64, 30000), page, rng.choice((0.0, 0.05, 0.5, 1.0)))
    kv, size = rng.choice((1, 2, 4, 8, 12)), rng.choice((32, 64, 128))
    heads = kv * rng.choice((1, 2, 4, 7, 8))
    if op == "write":
        rows = rng.choice((1, _log(rng, 2, 4096)))
        batch = _log(rng, 1, 64)
        batch = max(1, min(batch, 100_000_000 // (rows * (heads + 2 * kv) * size)))
        return _write("", dtype, batch, rows, heads, kv, size, page, layout)
    queries = rng.choice((1, 1, 1, rng.randint(2, 8)))
    keys = _log(rng, 1, 60000)
    batch = max(1, min(_log(rng, 1, 128), 40_000_000 // (kv * keys * size), 60_000_000 // (heads * queries * keys)))
    left = rng.choice((-1, -1, _log(rng, 16, 4096)))
    sinks = rng.choice((0, 1, 4, 70)) if left >= 0 else 0
    return _attention("", dtype, batch, queries, keys, heads, kv, size, page, left, sinks, rng.choice((0.0, 0.1, 0.6, 1.0)),
                      rng.choice((None, 2 * keys)), layout, left >= 0 and sinks == 0 and rng.random() < 0.5)


# ---------------------------------------------------------------------------- inputs


def _up(n, page):
    return -(-n // page)


def _lengths(case):
    """The lengths of a case's sequences, from the longest to the shortest (which of them has which goes by the seed)."""
    b, keys = case["batch"], case["keys"]
    short = min(keys, int(math.ceil(keys * case["shortest"])))
    return [keys if b == 1 else keys - (keys - short) * i // (b - 1) for i in range(b)]


def _counts(case):
    b, rows = case["batch"], case["rows"]
    return [rows if not case.get("ragged", True) or b == 1 else rows * (b - 1 - i) // (b - 1) for i in range(b)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lengths, width, page, pages, g):
    """A row of `width` entries per sequence with the pages that hold its tokens, any of `pages` and none twice, and those of nobody."""
    order = torch.randperm(pages, generator=g, device="cuda").int()
    held = (lengths.long() + page - 1) // page
    start = held.cumsum(0) - held
    i = torch.arange(width, device="cuda")
    table = torch.where(i < held[:, None], order[(start[:, None] + i).clamp_(max=pages - 1)], -1)
    return table, order[int(held.sum()):]


def _pools(case, pages, g):
    t = TYPES[case["dtype"]]
    shape = (pages, case["kv_heads"], case["page"], case["size"])
    if case["layout"] == "tokens":
        shape = (pages, case["page"], case["kv_heads"], case["size"])
    pools = [torch.empty(shape, device="cuda", dtype=t).normal_(generator=g) for _ in range(2)]
    return [p if case["layout"] == "heads" else p.permute(0, 2, 1, 3) for p in pools]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state, page, batch = dict(case), case["page"], case["batch"]

    def whole(high, n):  # 0 .. high
        return (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * (high + 1)).floor().clamp_(max=high).int()

    order = torch.randperm(batch, generator=g, device="cuda")
    if case["op"] == "extend":
        width = _up(case["limit"], page)
        counts = _ints(_counts(case))[order]
        lengths = whole(case["limit"] - (0 if case["scarce"] else case["rows"]), batch)
        need = (lengths.long() + counts + page - 1) // page - (lengths.long() + page - 1) // page
        held = int(((lengths.long() + page - 1) // page).sum())
        there = int(need.sum()) // 2 if case["scarce"] else int(need.sum()) + 64
        table, free = _table(lengths, width, page, held + there + 1, g)
        stack = torch.full((batch * width + 64,), -1, device="cuda", dtype=torch.int32)
        stack[:there] = free[:there]
        state.update(table=table, lengths=lengths, counts=counts, free=stack, free_count=_ints([there]))
    elif case["op"] == "cut":
        width = _up(case["limit"], page)
        lengths = whole(case["limit"], batch)
        ends = _ints([1 if i < round(case["ends"] * batch) else 0 for i in range(batch)])[order]
        keep = torch.where(ends != 0, 0, lengths - whole(4, batch))
        pages = batch * width + 64
        table, free = _table(lengths, width, page, pages, g)
        stack = torch.full((pages,), -1, device="cuda", dtype=torch.int32)
        stack[:free.numel()] = free
        state.update(table=table, lengths=lengths, keep=keep, free=stack, free_count=_ints([free.numel()]))
    elif case["op"] == "write":
        rows, heads, kv, size = case["rows"], case["heads"], case["kv_heads"], case["size"]
        packed = torch.empty(batch, rows, heads + 2 * kv, size, device="cuda", dtype=TYPES[case["dtype"]]).normal_(generator=g)
        before = whole(2 * page, batch)
        counts = _ints(_counts(case))[order]
        lengths = before + counts
        width = _up(rows + 2 * page, page)
        pages = sum(_up(n, page) for n in _counts(case)) + 2 * batch + 1
        table, _ = _table(lengths, width, page, pages, g)
        at = before.long()[:, None] + torch.arange(rows, device="cuda")
        slots = table.gather(1, at // page) * page + at % page
        slots = torch.where(torch.arange(rows, device="cuda") < counts[:, None], slots, -1).int()
        k_pages, v_pages = _pools(case, pages, g)
        state.update(k=packed[:, :, heads:heads + kv], v=packed[:, :, heads + kv:], slots=slots, k_pages=k_pages, v_pages=v_pages)
    else:
        lengths = _ints(_lengths(case))[order]
        pages = int(((lengths.long() + page - 1) // page).sum()) + 8
        table, _ = _table(lengths, _up(case["limit"], page), page, pages, g)
        if case["dropped"]:
            passed = (lengths.long() - case["queries"] - case["left"]).clamp_(min=0) // page
            table = torch.where(torch.arange(table.shape[1], device="cuda") < passed[:, None], -1, table)
        state["q"] = torch.randn(batch, case["queries"], case["heads"], case["size"], generator=g, device="cuda").to(TYPES[case["dtype"]])
        state["k_pages"], state["v_pages"] = _pools(case, pages, g)
        state.update(table=table, lengths=lengths)
    return state


# ---------------------------------------------------------------------------- one pass


def _run_extend(s):
    page, table, free = s["page"], s["table"], s["free"]
    if own:
        from cubert_amd import kernels
        slots, lengths, free_count = kernels.paged_extend(table, s["lengths"], s["counts"], free, s["free_count"], page, s["rows"])
        return slots, lengths, free_count, table
    width = table.shape[1]
    n, c = s["lengths"].long(), s["counts"].long().clamp(0, s["rows"])
    held = (n + page - 1) // page
    fits = n + c <= width * page
    need = torch.where(fits, (n + c + page - 1) // page - held, 0)
    through = need.cumsum(0)
    granted = fits & ((need == 0) | (through <= s["free_count"]))
    t = torch.arange(s["rows"], device="cuda")
    at = n[:, None] + t
    index = at // page
    fresh = index >= held[:, None]
    taken = s["free_count"].long() - 1 - (through - need)[:, None] - (index - held[:, None])
    pages = torch.where(fresh, free[taken.clamp(0, free.numel() - 1)], table.gather(1, index.clamp(max=width - 1)))
    there = (t < c[:, None]) & granted[:, None]
    slots = torch.where(there, pages * page + at % page, -1).int()
    # the pages of tables' rows from `held` on, so many of each as were taken
    i = torch.arange(width, device="cuda")
    taken = s["free_count"].long() - 1 - (through - need)[:, None] - (i - held[:, None])
    more = (i >= held[:, None]) & (i < (held + need)[:, None]) & granted[:, None]
    table.copy_(torch.where(more, free[taken.clamp(0, free.numel() - 1)], table))
    return (slots, torch.where(granted, n + c, n).int(), (s["free_count"] - torch.where(granted, need, 0).sum()).int(), table)


def _run_cut(s):
    page, table, free = s["page"], s["table"], s["free"]
    if own:
        from cubert_amd import kernels
        lengths, free_count = kernels.paged_cut(table, s["lengths"], s["keep"], free, s["free_count"], page)
        return lengths, free_count, free
    n = s["lengths"].long()
    keep = torch.minimum(s["keep"].long().clamp(min=0), n)
    i = torch.arange(table.shape[1], device="cuda")
    gone = (i >= ((keep + page - 1) // page)[:, None]) & (i < ((n + page - 1) // page)[:, None]) & (table >= 0)
    place = s["free_count"].long() + gone.view(-1).cumsum(0).view(gone.shape) - 1
    # entries that stay take turns at a place behind the stack's last
    room = torch.cat((free, free[:1]))
    room.scatter_(0, torch.where(gone, place, free.numel()).view(-1), table.view(-1))
    free.copy_(room[:-1])
    return keep.int(), (s["free_count"] + gone.sum()).int(), free


def _run_write(s):
    k_pages, v_pages, slots = s["k_pages"], s["v_pages"], s["slots"]
    if own:
        from cubert_amd import kernels
        kernels.paged_write(s["k"], s["v"], slots, k_pages, v_pages)
        return k_pages, v_pages
    kept = slots >= 0
    at = slots[kept].long()
    for rows, pool in ((s["k"], k_pages), (s["v"], v_pages)):
        pool.transpose(1, 2)[at // s["page"], at % s["page"]] = rows[kept]
    return k_pages, v_pages


def _run_attention(s):
    q, k_pages, v_pages, table, lengths = s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"]
    if own:
        from cubert_amd import kernels
        return kernels.attention_paged(q, k_pages, v_pages, table, lengths, s["left"], s["sinks"])
    b, nq, heads, size = q.shape
    kv, page = s["kv_heads"], s["page"]
    share = heads // kv
    # whoever plans the batch knows its longest sequence: that many pages of each, one behind the other
    table = table[:, :_up(s["keys"], page)]
    nk = table.shape[1] * page

    def rows_of(pool):
        return pool[table.clamp(min=0)].permute(0, 2, 1, 3, 4).reshape(b, kv, nk, size).float()

    p = (lengths.long() - nq)[:, None, None] + torch.arange(nq, device="cuda")[:, None]
    j = torch.arange(nk, device="cuda")
    seen = (j <= p) & (p >= 0) & (table >= 0).repeat_interleave(page, 1)[:, None, :]
    if s["left"] >= 0:
        seen = seen & ((j >= p - s["left"]) | (j < s["sinks"]))
    # the heads that share keys are rows of one product
    rows = q.float().view(b, nq, kv, share, size).permute(0, 2, 3, 1, 4).reshape(b, kv, share * nq, size)
    scores = rows @ rows_of(k_pages).transpose(2, 3) * (1 / math.sqrt(size))
    scores = scores.view(b, kv, share, nq, nk).masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(4, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(4, keepdim=True)
    out = (e.view(b, kv, share * nq, nk) @ rows_of(v_pages)).view(b, kv, share, nq, size) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4).reshape(b, nq, heads, size).to(q.dtype)


def run(state):
    return {"extend": _run_extend, "cut": _run_cut, "write": _run_write, "attention": _run_attention}[state["op"]](state)


# ---------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    page, batch = case["page"], case["batch"]
    if case["op"] == "extend":
        slots = sum(_counts(case))
        # a page for every `page` new tokens, from the stack to the table
        return {"bytes": 12 * batch + 4 * batch * case["rows"] + 8 * (slots // page), "flops": slots}
    if case["op"] == "cut":
        ends = round(case["ends"] * batch)
        pages = ends * case["limit"] // 2 // page
        return {"bytes": 12 * batch + 8 * pages, "flops": pages + batch}
    if case["op"] == "write":
        tokens, e = sum(_counts(case)), 4 if case["dtype"] == "f32" else 2
        n = 2 * tokens * case["kv_heads"] * case["size"]
        return {"bytes": 2 * n * e + 4 * batch * case["rows"], "flops": n}
    e = 4 if case["dtype"] == "f32" else 2
    left, sinks, pairs, reached, rows = case["left"], case["sinks"], 0, 0, 0
    for n in _lengths(case):
        low = n
        for p in range(max(0, n - case["queries"]), n):
            begin = max(0, p - left) if left >= 0 else 0
            pairs += p + 1 - begin + min(sinks, begin)
            low, rows = min(low, begin), rows + 1
        reached += n - low + min(sinks, low)
    size, heads, kv = case["size"], case["heads"], case["kv_heads"]
    moved = rows * heads * size * e + batch * case["queries"] * heads * size * e + 2 * reached * kv * size * e
    return {"bytes": moved + 4 * (reached // page) + 4 * batch, "flops": 4 * size * heads * pairs}


# ---------------------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] in ("extend", "cut"):
        table, lengths, stack = s["table"].tolist(), s["lengths"].tolist(), s["free"].tolist()
        left = int(s["free_count"])
        after = list(lengths)
        if case["op"] == "cut":
            for b, keep in enumerate(s["keep"].tolist()):
                after[b] = min(max(keep, 0), lengths[b])
                for i in range(_up(after[b], page), _up(lengths[b], page)):
                    if table[b][i] >= 0:
                        stack[left] = table[b][i]
                        left += 1
            return [torch.tensor(x, dtype=torch.int32) for x in (after, [left], stack)]
        slots = [[-1] * case["rows"] for _ in lengths]
        refused = False
        for b, count in enumerate(s["counts"].tolist()):
            count = min(max(count, 0), case["rows"])
            if lengths[b] + count > len(table[b]) * page:
                continue
            more = range(_up(lengths[b], page), _up(lengths[b] + count, page))
            refused = refused or len(more) > left
            if refused and len(more):
                continue
            for i in more:
                left -= 1
                table[b][i] = stack[left]
            after[b] += count
            slots[b][:count] = [table[b][at // page] * page + at % page for at in range(lengths[b], after[b])]
        return [torch.tensor(x, dtype=torch.int32) for x in (slots, after, [left], table)]
    if case["op"] == "write":
        out = []
        slots = s["slots"].reshape(-1).long()
        places = case["page"] * s["k_pages"].shape[0]
        # where every place of the pool has its row from, if it has a new one
        source = torch.full((places + 1,), -1, device="cuda", dtype=torch.int64)
        source[torch.where(slots < 0, places, slots)] = torch.arange(slots.numel(), device="cuda")
        source = source[:places].view(-1, page)
        for rows, pool in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            new = rows.reshape(slots.numel(), case["kv_heads"], case["size"])[source.clamp(min=0)].permute(0, 2, 1, 3)
            out.append(torch.where((source >= 0)[:, None, :, None], new, pool).double())
        return out
    q, table, lengths = s["q"], s["table"].long(), s["lengths"].tolist()
    nq, heads, share = case["queries"], case["heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        for i in range(nq):
            p = n - nq + i
            if p < 0:
                continue
            keys = torch.arange(p + 1, device="cuda")
            if case["left"] >= 0:
                keys = keys[(p - keys <= case["left"]) | (keys < case["sinks"])]
            pages = table[b][keys // page]
            keys, pages = keys[pages >= 0], pages[pages >= 0]
            if keys.numel() == 0:
                continue
            k = s["k_pages"][pages, :, keys % page].double().permute(1, 0, 2).contiguous()
            v = s["v_pages"][pages, :, keys % page].double().permute(1, 0, 2).contiguous()
            rows = q[b, i].double().view(case["kv_heads"], share, case["size"])
            z = torch.matmul(rows, k.transpose(1, 2).contiguous()) / math.sqrt(case["size"])
            z = (z - torch.logsumexp(z, 2, keepdim=True)).exp()
            out[b, i] = torch.matmul(z, v).view(heads, case["size"])
    return out
