"""A key/value cache in pages against its definition: tables and slots, which are whole numbers, against a plain walk through the sequences;
rows in pages bit for bit; attention over pages against its formula in 64 bits; and a run of them as a server makes it.

Tolerances count roundings.  u = 2^-24 is half a step of fp32 relative to the value, 2^-11 of fp16; a sum of n terms that
are added in fp32 in any order is off by at most (n - 1) u times the sum of their magnitudes."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}
SMALL = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25}   # half a step among the subnormals
TYPES = {"f32": torch.float32, "f16": torch.float16}


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the -m gpu tests must run on the MI355X box")
    from cubert_amd import kernels
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def up(n, page):
    return -(-n // page)


# ---------------------------------------------------------------------------- tables


def extend_reference(table, lengths, counts, free, free_count, page, rows, there=None):
    """What paged_extend gives, by a walk through the sequences: (slots, lengths, free_count, table)."""
    width, pages = len(table[0]) if table else 1, ((1 << 31) - 1) // page if there is None else there
    table, after = [list(r) for r in table], []
    top, refused = min(max(free_count, 0), len(free)), False
    slots = [[-1] * rows for _ in lengths]
    for b, n in enumerate(lengths):
        n = min(max(n, 0), width * page)
        count = min(max(counts[b], 0), rows) if counts is not None else rows
        after.append(n)
        if n + count > width * page:
            continue
        need = up(n + count, page) - up(n, page)
        refused = refused or need > top
        if refused and need:
            continue
        for i in range(up(n, page), up(n + count, page)):
            top -= 1
            table[b][i] = free[top]
        after[b] += count
        for t in range(count):
            own = table[b][(n + t) // page]
            slots[b][t] = own * page + (n + t) % page if 0 <= own < pages else -1
    return slots, after, top, table


def cut_reference(table, lengths, keep, free, free_count, page, there=None):
    """(lengths, free_count, free) of paged_cut."""
    width, pages = len(table[0]) if table else 1, ((1 << 31) - 1) // page if there is None else there
    free, top, after = list(free), min(max(free_count, 0), len(free)), []
    for b, n in enumerate(lengths):
        n = min(max(n, 0), width * page)
        left = min(max(keep[b], 0), n) if keep is not None else 0
        after.append(left)
        for i in range(up(left, page), up(n, page)):
            if 0 <= table[b][i] < pages and top < len(free):
                free[top] = table[b][i]
                top += 1
    return after, top, free


def tables(seed, batch, width, page, pages, longest, held=True):
    """Lengths up to `longest`, a table with pages that belong to nobody else, and a stack of the others."""
    r = random.Random(seed)
    order = list(range(pages))
    r.shuffle(order)
    lengths = [r.randint(0, longest) for _ in range(batch)]
    table = [[-1] * width for _ in range(batch)]
    for b in range(batch):
        for i in range(up(lengths[b], page)):
            table[b][i] = order.pop()
    return table, lengths, order + [-7] * (pages - len(order)), len(order)


# batch, rows, width, page, longest, pages to spare (of the stack), counts
EXTEND = {
    "one token": (1, 1, 4, 16, 40, 5, "rows"),
    "one token that needs a page": (1, 1, 4, 1, 3, 5, "rows"),
    "steps": (300, 1, 9, 16, 143, 300, "any"),
    "steps of nobody": (40, 1, 9, 16, 100, 10, "none"),
    "steps of four": (77, 4, 12, 16, 150, 100, "any"),
    "short stack": (100, 5, 12, 4, 40, 30, "any"),
    "empty stack": (100, 3, 12, 16, 150, 0, "any"),
    "full tables": (64, 9, 5, 8, 40, 500, "any"),
    "full tables and a short stack": (1500, 2, 5, 2, 10, 400, "any"),
    "prompts": (7, 1000, 70, 16, 90, 700, "any"),
    "prompts and a short stack": (9, 1000, 200, 16, 2000, 250, "any"),
    "long prompts": (3, 5000, 400, 32, 7000, 500, "rows"),
    "pages of one": (33, 20, 50, 1, 30, 660, "any"),
    "large pages": (20, 300, 3, 1024, 2500, 20, "any"),
    "many sequences": (5000, 1, 3, 16, 47, 5000, "any"),
    "counts beyond the rows": (50, 6, 9, 16, 100, 100, "wild"),
    "no rows": (20, 0, 4, 16, 60, 10, "any"),
    "exactly one workgroup": (1024, 1, 4, 16, 60, 1024, "rows"),
    "exactly two workgroups": (2, 1024, 70, 16, 60, 200, "rows"),
}


def counts_of(kind, batch, rows, seed):
    r = random.Random(seed + 1)
    if kind == "rows":
        return None
    if kind == "none":
        return [0] * batch
    if kind == "wild":
        return [r.choice((-5, rows + 3, 1 << 30, -(1 << 31), (1 << 31) - 1, r.randint(0, rows))) for _ in range(batch)]
    return [r.choice((0, rows, r.randint(0, rows))) for _ in range(batch)]


@pytest.mark.parametrize("name", list(EXTEND))
def test_extend(K, name):
    batch, rows, width, page, longest, spare, kind = EXTEND[name]
    table, lengths, _, _ = tables(len(name), batch, width, page, batch * width, longest)
    pages = sum(up(n, page) for n in lengths) + spare + 3
    table, lengths, free, there = tables(len(name), batch, width, page, pages, longest)
    there = min(there, spare)
    counts = counts_of(kind, batch, rows, len(name))
    on = [ints(table), ints(lengths), None if counts is None else ints(counts), ints(free), ints([there])]
    before = [None if x is None else x.clone() for x in on]
    slots, after, left = K.paged_extend(*on, page, rows)
    want = extend_reference(table, lengths, counts, free, there, page, rows)
    assert slots.tolist() == want[0] and after.tolist() == want[1] and left.tolist() == [want[2]] and on[0].tolist() == want[3]
    for x, y in zip(on[1:], before[1:]):                   # what it reads stays as it is
        assert x is None or torch.equal(x, y)
    assert [x.tolist() for x in K.paged_extend(*on, page, rows)] == [x.tolist() for x in (slots, after, left)]  # (and so a call may be repeated)


def test_extend_of_what_no_program_hands_over(K):
    """Lengths, heights and pages outside their ranges: cut to what there is, and never followed."""
    page, low, high = 16, -(1 << 31), (1 << 31) - 1
    table = [[5, -1, 3, 2], [high, low, 1, 0], [10, 9, 8, 7], [4, 4, 4, 4], [0, 1, 2, 3]]
    lengths, counts = [low, 20, high, 17, 30], [3, 40, 1, 4, 34]
    free = [6, -1, 11, high, low, 20, 0, 1, 2, 3, 4, 5]
    for there in (12, 6, 4, 0, -5, high):
        for pages in (12, None, 5, 1000):
            got_table = ints(table)
            slots, after, left = K.paged_extend(got_table, ints(lengths), ints(counts), ints(free), ints([there]), page, 40, pages)
            want = extend_reference(table, lengths, counts, free, there, page, 40, pages)
            assert (slots.tolist(), after.tolist(), left.tolist()[0], got_table.tolist()) == want


def test_tables_with_rows_apart(K):
    """Tables that are a part of a larger one."""
    table, lengths, free, there = tables(5, 30, 6, 16, 400, 70)
    whole = torch.full((30, 11), -9, dtype=torch.int32, device="cuda")
    part = whole[:, 2:8]
    part.copy_(ints(table))
    want = extend_reference(table, lengths, None, free, there, 16, 20)
    slots, after, left = K.paged_extend(part, ints(lengths), None, ints(free), ints([there]), 16, 20)
    assert (slots.tolist(), after.tolist(), left.tolist()[0], part.tolist()) == want
    assert bool((whole[:, :2] == -9).all()) and bool((whole[:, 8:] == -9).all())
    stack = ints(free)
    after, left = K.paged_cut(part, ints(lengths), None, stack, ints([there]), 16)
    assert (after.tolist(), left.tolist()[0], stack.tolist()) == cut_reference(want[3], lengths, None, free, there, 16)
    assert part.tolist() == want[3] and bool((whole[:, 8:] == -9).all())


def test_tables_of_nobody(K):
    for call in (lambda t, n, f, c: K.paged_extend(t, n, n, f, c, 16, 3)[1:], lambda t, n, f, c: K.paged_cut(t, n, n, f, c, 16)):
        for there in (3, 9, -4, 100):
            after, left = call(torch.zeros(0, 4, dtype=torch.int32, device="cuda"), ints([]), ints([0] * 9), ints([there]))
            assert after.shape == (0,) and left.tolist() == [min(max(there, 0), 9)]


CUT = {
    "one page": (1, 4, 16, 16, "none"),
    "a few end": (8, 40, 16, 600, "few"),
    "all end": (300, 20, 8, 160, "none"),
    "proposals": (100, 12, 16, 190, "near"),
    "anything": (70, 50, 4, 200, "any"),
    "one long": (1, 9000, 16, 140000, "any"),
    "few long": (5, 3000, 16, 48000, "none"),
    "many": (3000, 3, 16, 48, "any"),
    "pages of one": (20, 300, 1, 300, "any"),
    "wild": (200, 7, 16, 100, "wild"),
    "as many as one workgroup takes": (64, 512, 1, 512, "any"),
    "a sequence more": (65, 504, 1, 504, "any"),
    "a page more": (64, 513, 1, 513, "any"),
    "a few that are wild": (17, 40, 16, 640, "wild"),
}


@pytest.mark.parametrize("name", list(CUT))
@pytest.mark.parametrize("holes", [False, True])
def test_cut(K, name, holes):
    batch, width, page, longest, kind = CUT[name]
    r = random.Random(len(name))
    table, lengths, free, there = tables(len(name), batch, width, page, batch * width + 9, longest)
    if holes:                                              # pages that a window has passed, and entries that are nothing
        for b in range(batch):
            for i in range(width):
                if r.random() < 0.3:
                    table[b][i] = r.choice((-1, -(1 << 31), len(free), (1 << 31) - 1))
    keep = {"none": [0] * batch, "few": [n if r.random() < 0.8 else 0 for n in lengths], "near": [n - r.randint(0, 5) for n in lengths],
            "any": [r.randint(0, n) for n in lengths], "wild": [r.choice((-1, 1 << 30, n + 1, -(1 << 31))) for n in lengths]}[kind]
    if kind == "none" and holes:
        keep = None
    stack, on = ints(free), (ints(table), ints(lengths))
    pages = len(free) if holes or len(name) % 2 else None
    after, left = K.paged_cut(*on, None if keep is None else ints(keep), stack, ints([there]), page, pages)
    want = cut_reference(table, lengths, keep, free, there, page, pages)
    assert after.tolist() == want[0] and left.tolist() == [want[1]] and stack.tolist() == want[2]
    assert on[0].tolist() == table and on[1].tolist() == lengths


def test_cut_of_more_than_the_stack_holds(K):
    """Tables that have a page twice, and heights that are none: what there is no room for is left out, and nothing is written elsewhere."""
    table = [[i % 10 for i in range(30)] for _ in range(7)]
    lengths = [300, 480, 17, 480, (1 << 31) - 1, -3, 480]
    for there in (0, 8, 10, 40, -1):
        room = torch.full((30,), -8, dtype=torch.int32, device="cuda")
        stack = room[10:20]
        after, left = K.paged_cut(ints(table), ints(lengths), None, stack, ints([there]), 16)
        want = cut_reference(table, lengths, None, [-8] * 10, there, 16)
        assert after.tolist() == want[0] and left.tolist() == [want[1]] and stack.tolist() == want[2]
        assert bool((room[:10] == -8).all()) and bool((room[20:] == -8).all())


def test_a_stack_of_fewer_places_than_pages(K):
    """Some of a pool's pages are not the stack's: their numbers are beyond its places."""
    table, free = [[700, 3, -1, -1], [5, 900, 901, -1], [-1] * 4], [7, 999, 2, 0, 0]
    on = ints(table)
    slots, after, left = K.paged_extend(on, ints([20, 40, 0]), ints([13, 3, 2]), ints(free), ints([3]), 16, 13)
    assert (slots.tolist(), after.tolist(), left.tolist()[0], on.tolist()) == extend_reference(table, [20, 40, 0], [13, 3, 2], free, 3, 16, 13)
    assert slots[1, :3].tolist() == [901 * 16 + 8, 901 * 16 + 9, 901 * 16 + 10] and slots[2, 0] == 999 * 16
    stack = ints(free)
    after, left = K.paged_cut(on, after, ints([0, 16, 0]), stack, left, 16)
    assert stack.tolist() == [7, 700, 3, 2, 900] and left.tolist() == [5]


@pytest.mark.parametrize("page", [1, 16, 64])
def test_pages_come_and_go(K, page):
    """Steps of a server, growing and cutting back: no page belongs to two, none is lost."""
    r = random.Random(page)
    batch, width, pages = 40, 12, 200
    table, stack, count = torch.full((batch, width), -1, dtype=torch.int32, device="cuda"), ints(list(range(pages))), ints([pages])
    lengths = ints([0] * batch)
    for step in range(25):
        rows = r.choice((1, 1, 4, 3 * page))
        counts = [r.randint(0, rows) for _ in range(batch)]
        want = extend_reference(table.tolist(), lengths.tolist(), counts, stack.tolist(), int(count), page, rows)
        slots, lengths, count = K.paged_extend(table, lengths, ints(counts), stack, count, page, rows)
        assert (slots.tolist(), lengths.tolist(), int(count), table.tolist()) == want
        keep = [r.choice((n, n, n - 1, 0, r.randint(0, max(n, 1)))) for n in want[1]]
        want = cut_reference(want[3], want[1], keep, stack.tolist(), want[2], page)
        lengths, count = K.paged_cut(table, lengths, ints(keep), stack, count, page)
        assert (lengths.tolist(), int(count), stack.tolist()) == want
        held = [p for row, n in zip(table.tolist(), lengths.tolist()) for p in row[:up(n, page)]]
        assert sorted(held + stack.tolist()[:int(count)]) == list(range(pages))


# ---------------------------------------------------------------------------- rows into pages


def pool_of(layout, pages, kv_heads, page, size, t, seed):
    """Two pools [pages, kv_heads, page, size] in memory as `layout` has it, and all of the memory around them."""
    g = gen(seed)
    if layout == "heads":
        whole = normal(g, 2, pages, kv_heads, page, size).to(t)
        return whole[0], whole[1], whole
    if layout == "tokens":
        whole = normal(g, 2, pages, page, kv_heads, size).to(t)
        return whole[0].transpose(1, 2), whole[1].transpose(1, 2), whole
    if layout == "by turns":                               # keys and values of a page behind each other
        whole = normal(g, pages, 2, kv_heads, page, size).to(t)
        return whole[:, 0], whole[:, 1], whole
    if layout == "heads first":
        whole = normal(g, 2, kv_heads, pages, page, size).to(t)
        return whole[0].transpose(0, 1), whole[1].transpose(0, 1), whole
    assert layout == "apart"                               # rows with something between them
    whole = normal(g, 2, pages + 1, kv_heads + 1, page + 3, size + 8).to(t)
    return whole[0, 1:, :kv_heads, 2:page + 2, :size], whole[1, 1:, :kv_heads, 2:page + 2, :size], whole


LAYOUTS = ["heads", "tokens", "by turns", "heads first", "apart"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("batch,rows,heads,kv_heads,size,page", [(1, 1, 1, 1, 64, 16), (3, 1, 4, 2, 128, 16), (2, 37, 4, 4, 32, 1), (5, 200, 2, 12, 64, 32),
                                                                 (1, 3, 1, 3, 8, 4), (2, 50, 3, 1, 80, 64)])
def test_write(K, layout, t, batch, rows, heads, kv_heads, size, page):
    t, g = TYPES[t], gen(rows)
    pages = up(2 * batch * rows, page) + 2
    k_pages, v_pages, whole = pool_of(layout, pages, kv_heads, page, size, t, 3)
    packed = normal(g, batch, rows, heads + 2 * kv_heads, size).to(t)
    k, v = packed[:, :, heads:heads + kv_heads], packed[:, :, heads + kv_heads:]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:batch * rows].int().view(batch, rows)
    slots.view(-1)[1::5] = -1
    if batch * rows > 20:                                  # slots that no pool has
        slots.view(-1)[[2, 7, 12]] = ints([pages * page, (1 << 31) - 1, -(1 << 31)])
    want_k, want_v, want = pool_of(layout, pages, kv_heads, page, size, t, 3)
    for b in range(batch):
        for i in range(rows):
            s = int(slots[b, i])
            if 0 <= s < pages * page:
                want_k[s // page, :, s % page], want_v[s // page, :, s % page] = k[b, i], v[b, i]
    assert K.paged_write(k, v, slots, k_pages, v_pages) is not None
    assert torch.equal(whole, want)                        # and nothing else has changed


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_write_of_a_large_prompt(K, t):
    """So much that it goes past the caches: 64 MB and more, all of it there for what reads it next."""
    t, g = TYPES[t], gen(8)
    batch, rows, kv, size, page = 3, 7001, 8, 128 if t == torch.float16 else 64, 64
    pages = up(batch * rows, page) + 1
    k_pages, v_pages, _ = pool_of("heads", pages, kv, page, size, t, 3)
    packed = torch.randn(batch, rows, 3 * kv, size, generator=g, device="cuda").to(t)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:batch * rows].int().view(batch, rows)
    slots[1, 5000:] = -1
    want_k, want_v = k_pages.clone(), v_pages.clone()
    kept = slots >= 0
    at = slots[kept].long()
    for want, rows_of in ((want_k, packed[:, :, kv:2 * kv]), (want_v, packed[:, :, 2 * kv:])):
        want.transpose(1, 2)[at // page, at % page] = rows_of[kept]
    K.paged_write(packed[:, :, kv:2 * kv], packed[:, :, 2 * kv:], slots, k_pages, v_pages)
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


def test_write_refuses(K):
    pool, q = torch.zeros(4, 2, 16, 64, device="cuda"), torch.zeros(2, 3, 4, 64, device="cuda")
    slots = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    assert K.paged_write(q[:, :, :2, :], q[:, :, 2:], slots - 1, pool, pool + 0) is not None
    assert K.paged_write(q[:0, :, :2], q[:0, :, 2:], slots[:0], pool, pool + 0) is not None
    odd = torch.zeros(2, 3, 2, 66, device="cuda")
    assert K.paged_write(odd, odd, slots, torch.zeros(4, 2, 16, 66, device="cuda"), torch.zeros(4, 2, 16, 66, device="cuda")) is None
    whole = torch.zeros(4 * 2 * 16 * 64 + 1, device="cuda")[1:].view(4, 2, 16, 64)
    assert K.paged_write(q[:, :, :2], q[:, :, 2:], slots, whole, whole) is None
    with pytest.raises(RuntimeError):                      # all heads of a page in one place
        K.paged_write(q[:, :, :2], q[:, :, 2:], slots, pool[:, :1].expand(4, 2, 16, 64), pool[:, :1].expand(4, 2, 16, 64))


# ---------------------------------------------------------------------------- attention over pages

# batch, q_rows, heads, kv_heads, page, left, sinks, lengths, first (None: the last ones)
ATTENTION = {
    "one key": (1, 1, 1, 1, 16, -1, 0, (1,), None),
    "one query": (2, 1, 4, 2, 16, -1, 0, (300, 77), None),
    "no keys": (3, 1, 4, 1, 16, -1, 0, (0, 5, 0), None),
    "nobody": (2, 1, 12, 12, 16, -1, 0, (0, 0), None),
    "around a page": (9, 1, 3, 3, 16, -1, 0, (15, 16, 17, 31, 32, 33, 1, 2, 64), None),
    "around large pages": (6, 1, 8, 2, 64, -1, 0, (63, 64, 65, 127, 129, 300), None),
    "a few tokens": (4, 5, 8, 2, 16, -1, 0, (1000, 999, 64, 5), None),
    "seven heads to one": (3, 3, 7, 1, 32, 50, 4, (333, 100, 2), None),
    "many heads to one": (2, 1, 40, 1, 16, -1, 0, (500, 40), None),
    "many rows": (2, 9, 16, 2, 16, 100, 1, (700, 7), None),
    "a window": (3, 1, 4, 2, 16, 40, 0, (500, 41, 12), None),
    "a window and sinks": (3, 2, 4, 2, 16, 100, 5, (500, 300, 12), None),
    "a window of one": (2, 4, 2, 2, 16, 0, 0, (100, 17), None),
    "sinks alone": (2, 3, 2, 1, 16, 0, 40, (300, 35), None),
    "sinks up to the window": (2, 1, 2, 1, 16, 20, 70, (90, 95), None),
    "sinks of everything": (2, 2, 4, 4, 32, 3, 1000, (90, 200), None),
    "before the sequence": (3, 20, 2, 2, 16, 10, 1, (64, 7, 0), None),
    "padded tokens": (4, 6, 4, 2, 16, -1, 0, (50, 51, 52, 53), (44, 50, 52, 60)),
    "tokens in the middle": (2, 3, 4, 2, 16, 30, 2, (200, 100), (90, 20)),
    "long": (1, 1, 4, 1, 16, -1, 0, (4999,), None),
    "long of two heads": (2, 1, 16, 2, 128, -1, 0, (9000, 100), None),
    "long window": (2, 2, 8, 1, 256, 4095, 4, (9000, 4500), None),
    "unlike lengths": (33, 1, 4, 4, 16, -1, 0, tuple((37 * i * i) % 1500 for i in range(33)), None),
    "many short": (300, 1, 2, 2, 16, -1, 0, tuple(i % 40 for i in range(300)), None),
    "many and one long": (70, 1, 2, 1, 16, -1, 0, (3000,) + (3,) * 69, None),
    "many and a long one at the end": (260, 1, 4, 2, 16, -1, 0, (3,) * 259 + (5000,), None),
    "a prompt": (2, 130, 4, 2, 16, -1, 0, (130, 100), None),
}


def paged(name, t, size, layout="heads", seed=0, wide=3):
    """Inputs of a case (a name or the case itself), and its keys and values as they would stand without pages."""
    batch, q_rows, heads, kv_heads, page, left, sinks, lengths, first = ATTENTION.get(name, name)
    g = gen(seed + size + len(name))
    longest = max(max(lengths), 1)
    width = up(longest, page) + wide
    pages = sum(up(n, page) for n in lengths) + 3
    q = normal(g, batch, q_rows, heads, size).to(t)
    k, v = (normal(g, batch, longest, kv_heads, size).to(t) for _ in "kv")
    order = torch.randperm(pages, generator=g, device="cuda").int().tolist()
    rows = []
    for n in lengths:
        rows.append([order.pop() for _ in range(up(n, page))])
        rows[-1] += [-1] * (width - len(rows[-1]))
    table = ints(rows)
    k_pages, v_pages, _ = pool_of(layout, pages, kv_heads, page, size, t, seed + 1)
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        own = table[b].long()[at // page]
        k_pages[own, :, at % page], v_pages[own, :, at % page] = k[b, :n], v[b, :n]
    at = dict(left=left, sinks=sinks, lengths=ints(lengths), first=None if first is None else ints(first))
    return q, k_pages, v_pages, table, k, v, page, at


def visible(q, k, page, left, sinks, lengths, first, table=None, pages=None):
    """[batch, q_rows, keys]"""
    q_rows, keys = q.shape[1], k.shape[1]
    n = lengths.long()[:, None, None]
    p = ((n[:, 0] - q_rows if first is None else first.long()[:, None]) + torch.arange(q_rows, device="cuda"))[:, :, None]
    j = torch.arange(keys, device="cuda")
    seen = (j <= p) & (j < n) & (p >= 0) & (p < n)
    if left >= 0:
        seen = seen & ((j >= p - left) | (j < sinks))
    if table is not None:
        there = (table >= 0) & (table < pages)
        seen = seen & there.repeat_interleave(page, 1)[:, None, :keys]
    return seen


def reference(q, k, v, seen, alpha=None):
    """The formula in 64 bits, and how far a kernel may be off it."""
    t, size = q.dtype, q.shape[3]
    alpha = size ** -0.5 if alpha is None else alpha
    share = q.shape[2] // k.shape[2]
    hold = seen.any(1)[:, :, None, None]                   # keys that nobody sees may hold anything
    k, v = torch.where(hold, k, 0), torch.where(hold, v, 0)
    seen = seen[:, None]
    Q, KT = q.double().permute(0, 2, 1, 3), k.double().repeat_interleave(share, 2).permute(0, 2, 3, 1)
    V = v.double().repeat_interleave(share, 2).permute(0, 2, 1, 3)
    z = torch.where(seen, (Q @ KT) * alpha, -math.inf)
    top = z.amax(3, keepdim=True)
    e = torch.where(seen, torch.exp(z - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(3, keepdim=True)
    some = torch.where(total > 0, total, 1.0)
    out = (e @ V) / some
    # A score is a sum of `size` products of which each is rounded once and each sum once, 2 size u of the products' magnitudes; the factor
    # alpha log2(e) has 2 roundings, the difference to a maximum one and its product with the factor one, of at most twice the largest.
    products = (Q.abs() @ KT.abs()) * abs(alpha)
    slip = torch.where(seen, products, 0.0).amax(3, keepdim=True) * (2 * size + 8) * U
    # An exponential is off by 2^-22 of itself, and sums are scaled anew by some (once for 16 keys, twice when they are joined); sums have as
    # many terms as keys are seen, and a product each.
    count = seen.double().sum(3, keepdim=True)
    each = torch.expm1(2 * slip) + 3 * 2.0 ** -22 + (2 * count + 16) * U + (count / 16 + 2) * 2.0 ** -22
    off = each * ((e @ V.abs()) / some)
    bound = off + (out.abs() + off) * (HALF[t] + 4 * U) + SMALL[t]
    back = lambda x: x.permute(0, 2, 1, 3)                 # noqa: E731
    return back(out), back(bound)


def within(got, want, bound, what):
    """|got - want| <= bound element by element (want and bound in 64 bits)."""
    torch.cuda.synchronize()
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), "%s: off by %.3g where %.3g is allowed, %d of %d elements" % (
        what, float(off.nan_to_num(math.inf).max()), float(bound.flatten()[off.nan_to_num(math.inf).argmax()]),
        int((~(off <= bound)).sum()), off.numel())


@pytest.mark.parametrize("name", list(ATTENTION))
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_paged(K, name, t, size):
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], size)
    seen = visible(q, k, page, **at)
    want, bound = reference(q, k, v, seen)
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    within(got, want, bound, name)
    assert bool((got[~seen.any(2)] == 0).all())
    assert torch.equal(got, K.attention_paged(q, k_pages, v_pages, table, **at))     # the same call gives the same bits


@pytest.mark.parametrize("name", ["many rows", "many heads to one", "before the sequence", "padded tokens", "a prompt", "unlike lengths", "nobody", "long"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("filler", [None, math.nan])
def test_attention_paged_with_wide_tables(K, name, t, size, filler):
    """Tables with room for far longer sequences than there are: as calls on long ones are cut, and their rows."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], size, wide=20000)
    seen = visible(q, k, page, **at)
    want, bound = reference(q, k, v, seen)
    if filler is not None:
        keep = torch.zeros(k_pages.shape[0] * page, dtype=torch.bool, device="cuda")
        b, j = seen.any(1).nonzero(as_tuple=True)
        keep[table[b, j // page].long() * page + j % page] = True
        k_pages, v_pages = (torch.where(keep.view(-1, 1, page, 1), p, filler) for p in (k_pages, v_pages))
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    within(got, want, bound, name)
    assert bool((got[~seen.any(2)] == 0).all())


@pytest.mark.parametrize("batch,q_rows,left", [(64, 1, -1), (65, 1, -1), (128, 3, 40), (200, 20, -1), (256, 1, -1), (257, 1, -1), (300, 40, 100), (512, 1, -1),
                                               (513, 2, -1), (700, 1, -1), (1025, 1, -1), (2048, 1, -1), (2049, 1, -1)])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("at_end", [False, True])
def test_attention_paged_of_many_sequences(K, batch, q_rows, left, t, at_end):
    """Sequences among which a workgroup has to find its own, all but one in a few short."""
    r = random.Random(batch)
    lengths = [r.choice((0, 1, 9, 40, 70)) if r.random() < 0.97 else 600 for _ in range(batch)]
    lengths[-1 if at_end else 0] = 640
    case = (batch, q_rows, 2, 1, 16, left, 0, tuple(lengths), None)
    q, k_pages, v_pages, table, k, v, page, at = paged(case, TYPES[t], 32, wide=4000)
    want, bound = reference(q, k, v, visible(q, k, page, **at))
    within(K.attention_paged(q, k_pages, v_pages, table, **at), want, bound, "many")


@pytest.mark.parametrize("name", ["one query", "a few tokens", "a window and sinks", "long", "unlike lengths"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("layout", LAYOUTS[1:])
@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_paged_in_any_layout(K, name, t, layout, size):
    """Pools of other strides, queries out of a packed projection, another scale."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], size, layout)
    packed = torch.zeros(q.shape[0], q.shape[1], q.shape[2] + 3, size, dtype=q.dtype, device="cuda")
    packed[:, :, 1:-2] = q
    want, bound = reference(q, k, v, visible(q, k, page, **at), alpha=-0.03)
    within(K.attention_paged(packed[:, :, 1:-2], k_pages, v_pages, table, alpha=-0.03, **at), want, bound, name)


FEW = ["one query", "no keys", "around a page", "around large pages", "a few tokens", "seven heads to one", "a window and sinks", "sinks alone",
       "before the sequence", "tokens in the middle", "long", "long window", "unlike lengths", "many short", "many rows"]


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("heads,q_rows", [(8, 1), (8, 4), (8, 9)])
def test_attention_paged_of_a_large_pool(K, t, size, heads, q_rows):
    """Pools of 96 MB and more, which are read past the caches, with sequences in a part of them."""
    t, g = TYPES[t], gen(18)
    page, kv = 64, 4
    pages = (96 << 20) // (2 * page * kv * size * t.itemsize) + 1
    k_pages, v_pages, _ = pool_of("heads", pages, kv, page, size, t, 7)
    q, lengths = normal(g, 3, q_rows, heads, size).to(t), ints([1900, 77, 1])
    table = torch.randperm(pages, generator=g, device="cuda").int()[:90].view(3, 30).contiguous()
    k, v = (p.transpose(1, 2)[table.long()].reshape(3, 30 * page, kv, size) for p in (k_pages, v_pages))
    at = dict(left=-1, sinks=0, lengths=lengths, first=None)
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    within(got, *reference(q, k, v, visible(q, k, page, **at)), "large pool")


@pytest.mark.parametrize("name", FEW)
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("filler", [math.nan, math.inf, -math.inf])
def test_attention_paged_past_what_it_sees(K, name, t, filler):
    """What no query sees may hold anything: the rest of a last page, what a window has passed, pages of nobody; and tables anything behind
    the pages that are read."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], 64)
    seen = visible(q, k, page, **at)
    want, bound = reference(q, k, v, seen)
    keep = torch.zeros(k_pages.shape[0] * page, dtype=torch.bool, device="cuda")
    b, j = seen.any(1).nonzero(as_tuple=True)
    keep[table[b, j // page].long() * page + j % page] = True
    keep = keep.view(-1, 1, page, 1)
    k_pages, v_pages = torch.where(keep, k_pages, filler), torch.where(keep, v_pages, filler)
    need = torch.zeros(table.shape, dtype=torch.bool, device="cuda")
    need[b, j // page] = True
    wild = ints([-1, k_pages.shape[0], (1 << 31) - 1, -(1 << 31)]).repeat(table.numel() // 4 + 1)[:table.numel()].view(table.shape)
    within(K.attention_paged(q, k_pages, v_pages, torch.where(need, table, wild), **at), want, bound, name)


@pytest.mark.parametrize("name", FEW)
@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_paged_without_some_pages(K, name, t):
    """An entry that is no page takes its keys out of sight."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], 64)
    gone = torch.rand(table.shape, generator=gen(4), device="cuda") < 0.3
    gone[0] = True                                         # nothing left of the first sequence
    table = torch.where(gone, ints([-1, k_pages.shape[0], (1 << 31) - 1, -(1 << 31)]).repeat(table.numel() // 4 + 1)[:table.numel()].view(table.shape), table)
    seen = visible(q, k, page, table=table, pages=k_pages.shape[0], **at)
    want, bound = reference(q, k, v, seen)
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    within(got, want, bound, name)
    assert bool((got[~seen.any(2)] == 0).all())


@pytest.mark.parametrize("name", ["one query", "a few tokens", "long", "a window and sinks", "seven heads to one", "unlike lengths"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("where", ["q", "k"])
def test_attention_paged_of_no_number(K, name, t, where):
    """What is no number in a query or a key makes none of the results that take it, and of no others."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], 64)
    seen, share = visible(q, k, page, **at), q.shape[2] // k.shape[2]
    want, bound = reference(q, k, v, seen)
    b, i = (int(x) for x in seen.any(2).nonzero()[seen.any(2).sum() // 2])
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    if where == "q":
        q[b, i, 1, 5] = math.nan
        bad[b, i, 1] = True
    else:
        j = int(seen[b, i].nonzero()[0])
        k_pages[int(table[b, j // page]), 0, j % page, 63] = math.nan
        bad[b, :, :share] = seen[b, :, j, None]
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    assert bool(torch.isnan(got[bad]).all())
    within(torch.where(bad[..., None], 0, got), torch.where(bad[..., None], 0.0, want), bound, name)


@pytest.mark.parametrize("name", ["one query", "a few tokens", "long", "a window and sinks", "seven heads to one", "unlike lengths"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("alpha", [0.125, -0.125])
def test_attention_paged_of_infinite_keys(K, name, t, size, alpha):
    """An infinite key is a score of -infinity for a query of the other sign, as if it were not there, and no number for the others."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], size)
    q[..., 5] = torch.where(q[..., 5] < 0, -0.5, 0.5).to(q.dtype)
    seen, share = visible(q, k, page, **at), q.shape[2] // k.shape[2]
    b, i = (int(x) for x in seen.any(2).nonzero()[seen.any(2).sum() // 2])
    j = int(seen[b, i].nonzero()[0])
    without = seen.clone()
    without[b, :, j] = False
    want, bound = reference(q, k, v, seen, alpha=alpha)
    want_without, bound_without = reference(q, k, v, without, alpha=alpha)
    meets = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    meets[b, :, :share] = seen[b, :, j, None]
    none = meets & (q[..., 5] * alpha > 0)
    want, bound = torch.where(meets[..., None], want_without, want), torch.where(meets[..., None], bound_without, bound)
    k_pages[int(table[b, j // page]), 0, j % page, 5] = math.inf
    got = K.attention_paged(q, k_pages, v_pages, table, alpha=alpha, **at)
    assert bool(torch.isnan(got[none]).all())
    within(torch.where(none[..., None], 0, got), torch.where(none[..., None], 0.0, want), bound, name)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("at_key", [0, 17, 2999])
def test_attention_paged_of_infinite_values(K, t, at_key):
    """Infinite values reach the results of the heads that share them, in their column, and nothing else."""
    t, g = TYPES[t], gen(15)
    k_pages, v_pages, _ = pool_of("heads", 200, 2, 16, 64, t, 5)
    table = torch.randperm(200, generator=g, device="cuda").int()[:190].view(1, -1).contiguous()
    q, lengths = normal(g, 1, 1, 4, 64).to(t), ints([3000])
    clean = K.attention_paged(q, k_pages, v_pages, table, lengths)
    v_pages[int(table[0, at_key // 16]), 1, at_key % 16, 7] = -math.inf
    got = K.attention_paged(q, k_pages, v_pages, table, lengths)
    assert bool((got[0, 0, 2:, 7] == -math.inf).all())
    got[0, 0, 2:, 7] = clean[0, 0, 2:, 7]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_paged_of_large_scores(K, t, size):
    """Scores far apart and far from zero, up to the largest that there are: the softmax picks single keys, and nothing leaves the range."""
    t, g = TYPES[t], gen(10)
    largest = 60000.0 if t == torch.float16 else 1e18
    for q_by, k_by, alpha in ((30, 30, None), (30, 30, -0.7), (1000, 50, 0.3), (0, 0, None)):
        k_pages, v_pages, _ = pool_of("heads", 60, 2, 16, size, t, 5)
        k_pages *= k_by
        if k_by == 0:                                      # one number each, of the largest there are, the others zero
            k_pages[..., 3] = largest
            k_pages[7, :, 5, 3] = largest / 2
        table = torch.randperm(60, generator=g, device="cuda").int()[:50].view(2, 25).contiguous()
        q = (q_by * normal(g, 2, 3, 4, size)).to(t)
        if q_by == 0:
            q[..., 3] = largest / 4
        at = dict(left=-1, sinks=0, lengths=ints([400, 333]), first=None)
        own = table.long()
        k, v = (p.transpose(1, 2)[own].reshape(2, 400, 2, size) for p in (k_pages, v_pages))
        got = K.attention_paged(q, k_pages, v_pages, table, alpha=alpha, **at)
        assert bool(torch.isfinite(got).all())
        want, bound = reference(q, k, v, visible(q, k, 16, **at), alpha=alpha)
        within(got, want, bound, "%g %g" % (q_by, k_by))


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_paged_keeps_apart_what_rows_see(K, t, size):
    """Values as large as there are in keys that only the last of a few queries sees, or only the first: the others have none of them."""
    t, g = TYPES[t], gen(16)
    largest = 65504.0 if t == torch.float16 else 1e30
    k_pages, v_pages, _ = pool_of("heads", 40, 2, 16, size, t, 5)
    v_pages *= 1e-4
    table = torch.randperm(40, generator=g, device="cuda").int()[:33].view(1, -1).contiguous()
    q = normal(g, 1, 5, 4, size).to(t)
    at = dict(left=200, sinks=0, lengths=ints([520]), first=None)
    for j in (519, 315):                                   # the last token, and the first one of the first query's window
        v_pages[int(table[0, j // 16]), :, j % 16] = largest
    k, v = (p.transpose(1, 2)[table.long()].reshape(1, 528, 2, size)[:, :520] for p in (k_pages, v_pages))
    want, bound = reference(q, k, v, visible(q, k, 16, **at))
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    within(got, want, bound, "apart")
    assert bool((got[0, 1:4].abs() < 1e-2).all()) and bool((got[0, [0, 4]].abs() > 1).any())


@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_paged_of_the_largest_numbers(K, size):
    """Values near fp32's largest under scores that rise all the way, and scores near its least."""
    g = gen(17)
    k_pages, v_pages, _ = pool_of("heads", 40, 1, 16, size, torch.float32, 5)
    table = torch.randperm(40, generator=g, device="cuda").int()[:32].view(1, -1).contiguous()
    place = torch.arange(512, device="cuda")
    for scores, values, alpha in ((place.float() / 2, 1e38, 1.0), (place.float() * 30, 3e38, 1.0), (-3.39e38 + place.float() * 1e32, 1.0, 1e-32),
                                  (torch.full((512,), -3.35e38, device="cuda"), 1.0, 1.0)):
        k_pages.zero_(), v_pages.zero_()
        own = table[0, place // 16].long()
        k_pages[own, 0, place % 16, 1] = scores
        v_pages[own, 0, place % 16] = values * (torch.rand(512, size, generator=g, device="cuda") - 0.5)
        q = torch.zeros(1, 1, 2, size, device="cuda")
        q[..., 1] = 1
        at = dict(left=-1, sinks=0, lengths=ints([512]), first=None)
        k, v = (p.transpose(1, 2)[table.long()].reshape(1, 512, 1, size) for p in (k_pages, v_pages))
        # (bounds go by the scores, so they are wide for some of these; that results are numbers is the point)
        want, bound = reference(q, k, v, visible(q, k, 16, **at), alpha=alpha)
        got = K.attention_paged(q, k_pages, v_pages, table, alpha=alpha, **at)
        assert bool(torch.isfinite(got).all())
        within(got, want, bound, "%g" % values)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_paged_without_scores(K, t):
    """A scale of 0: the mean of what is seen."""
    for name in FEW:
        q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], 64)
        want, bound = reference(q, k, v, visible(q, k, page, **at), alpha=0.0)
        within(K.attention_paged(q, k_pages, v_pages, table, alpha=0.0, **at), want, bound, name)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_paged_keeps_a_long_axis_next_to_one_key(K, t):
    """One key of a large score and very many of a small one, whose probabilities add up to as much."""
    t, n, size = TYPES[t], 60000, 64
    k_pages, v_pages, _ = pool_of("heads", n // 16, 1, 16, size, t, 5)
    k_pages.zero_()
    v_pages.fill_(1)
    q = torch.zeros(1, 1, 2, size, dtype=t, device="cuda")
    q[..., 0] = 1
    table = torch.randperm(n // 16, generator=gen(3), device="cuda").int().view(1, -1).contiguous()
    for where in (0, 30000, n - 1):
        k_pages.zero_(), v_pages.fill_(1)
        own = int(table[0, where // 16])
        k_pages[own, 0, where % 16, 0] = 11.0
        v_pages[own, 0, where % 16] = -1
        got = K.attention_paged(q, k_pages, v_pages, table, ints([n]), alpha=1.0)
        e = math.exp(11.0)
        want = torch.full(got.shape, (n - 1 - e) / (n - 1 + e), dtype=torch.float64, device="cuda")
        # (its terms cancel in part: 1 - 2 e / (n - 1 + e); sums of n terms, and the roundings of 11 in multiples of log 2)
        within(got, want, torch.full_like(want, 2 * (2 * n + 64) * U + 2 * 2.0 ** -22 * n / 16) + want.abs() * HALF[t], "at %d" % where)


def test_attention_paged_lengths_that_no_table_holds(K):
    """Lengths and positions come from the device: ones beyond the table are cut to what it holds."""
    low, high = -(1 << 31), (1 << 31) - 1
    q, k_pages, v_pages, table, k, v, page, at = paged("a few tokens", torch.float16, 64, wide=0)
    n = table.shape[1] * page
    table = torch.where(table < 0, 0, table)
    k, v = (p.transpose(1, 2)[table.long()].reshape(4, n, 2, 64) for p in (k_pages, v_pages))
    at["lengths"], at["first"] = ints([high, 2000000000, -5, 5]), ints([995, 990, 0, low])
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    at["lengths"], at["first"] = ints([n, n, 0, 5]), ints([995, 990, 0, -100])
    want, bound = reference(q, k, v, visible(q, k, page, **at))
    within(got, want, bound, "cut")
    for first in ([high] * 4, [low] * 4, [n] * 4):
        assert bool((K.attention_paged(q, k_pages, v_pages, table, at["lengths"], first=ints(first)) == 0).all())


def test_attention_paged_far_into_a_pool(K):
    """Pages more than 2^31 elements in, keys and values by turns."""
    pages, kv, page, size = 70000, 8, 32, 128              # 4.6e9 elements, 9.2 GB
    pool = torch.zeros(pages, 2, kv, page, size, dtype=torch.float16, device="cuda")
    k_pages, v_pages = pool[:, 0], pool[:, 1]
    g = gen(11)
    table = ints([[69999, 1, 35000, 69998, 32768, 65537, 0]])
    for own in table[0].tolist():
        pool[own] = normal(g, 2, kv, page, size).half()
    q, lengths = normal(g, 1, 2, 16, size).half(), ints([7 * page - 3])
    k, v = (p.transpose(1, 2)[table.long()].reshape(1, 7 * page, kv, size) for p in (k_pages, v_pages))
    at = dict(left=150, sinks=3, lengths=lengths, first=None)
    want, bound = reference(q, k, v, visible(q, k, page, **at))
    within(K.attention_paged(q, k_pages, v_pages, table, **at), want, bound, "far")
    row = normal(g, 1, 1, 2 * kv, size).half()
    K.paged_write(row[:, :, :kv], row[:, :, kv:], ints([[69997 * page + 5]]), k_pages, v_pages)
    assert torch.equal(pool[69997, :, :, 5].reshape(-1, size), row[0, 0])
    pool[69997] = 0
    assert bool((pool[69990:69998] == 0).all())


def test_attention_paged_cut_and_uncut(K):
    """A call without room for its pieces runs uncut, with the same result within its bound."""
    from cubert_amd._lib import lib
    for t in (torch.float32, torch.float16):
        for name in ("long", "long of two heads", "long window", "one query", "a few tokens", "unlike lengths", "many and one long", "many rows", "nobody"):
            q, k_pages, v_pages, table, k, v, page, at = paged(name, t, 64)
            want, bound = reference(q, k, v, visible(q, k, page, **at))
            out = torch.full_like(q, math.nan)
            batch, q_rows, heads, size = q.shape
            rc = getattr(lib(), "cubert_attention_paged_" + ("f32" if t == torch.float32 else "f16"))(
                q.data_ptr(), heads * size, k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], table.data_ptr(), table.shape[1], table.shape[1],
                at["lengths"].data_ptr(), None, out.data_ptr(), heads * size, size ** -0.5, batch, heads, k_pages.shape[1], q_rows, k_pages.shape[0], page,
                size, at["left"], at["sinks"], None, 0, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            within(out, want, bound, name)


def test_attention_paged_declines(K):
    pool, q = torch.zeros(4, 2, 16, 64, device="cuda"), torch.zeros(2, 3, 4, 64, device="cuda")
    table, n = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints([0, 0])
    assert K.attention_paged(q[..., :48].contiguous(), pool[..., :48], pool[..., :48], table, n) is None
    assert K.attention_paged(q, pool[:, :, :8].contiguous(), pool[:, :, :8].contiguous(), table, n) is None
    assert K.attention_paged(q[:0], pool, pool, table[:0], n[:0]).shape == (0, 3, 4, 64)
    assert K.attention_paged(q[:, :0], pool, pool, table, n).shape == (2, 0, 4, 64)
    assert bool((K.attention_paged(q + 1, pool, pool, table, n) == 0).all())
    with pytest.raises(RuntimeError):
        K.attention_paged(q, pool[:, :1].expand(4, 2, 16, 64), pool[:, :1].expand(4, 2, 16, 64), table, n)


# ---------------------------------------------------------------------------- streams, graphs, a run of them


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_paged_in_two_graphs(K, t):
    """Calls over a long cache, two captured and one eager on another stream, each with its own partial sums, at once."""
    calls = [paged(name, TYPES[t], size, seed=seed) for name, size, seed in (("long", 64, 1), ("long of two heads", 64, 2), ("long window", 128, 3))]

    def run(c):
        return K.attention_paged(*c[:4], **c[7])

    for c in calls:
        run(c)
    torch.cuda.synchronize()
    graphs = []
    for c in calls[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(c)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        for c in calls:
            c[0].copy_(normal(gen(70 + turn), *c[0].shape))
        torch.cuda.synchronize()
        got = []
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = run(calls[2])
        torch.cuda.synchronize()
        got = [out.clone() for _, out in graphs] + [eager]
        for out, c in zip(got, calls):
            assert torch.equal(out, run(c))
            within(out, *reference(c[0], c[4], c[5], visible(c[0], c[4], c[6], **c[7])), "turn %d" % turn)


class Server(object):
    """A layer's cache in pages and, next to it, the same rows as attention_window has them."""

    heads, kv, size, page, width, pages, window, sinks = 4, 2, 64, 16, 12, 14, 60, 3

    def __init__(self, K, t, batch, seed):
        g = gen(seed)
        self.K, self.t, self.batch = K, t, batch
        self.k_pages, self.v_pages, _ = pool_of("heads", self.pages, self.kv, self.page, self.size, t, seed)
        self.k, self.v = (normal(g, batch, self.width * self.page, self.kv, self.size).to(t) for _ in "kv")
        self.table = torch.full((batch, self.width), -1, dtype=torch.int32, device="cuda")
        self.free, self.free_count = torch.randperm(self.pages, generator=g, device="cuda").int(), ints([self.pages])
        self.lengths, self.counts, self.keep = ints([0] * batch), ints([0] * batch), ints([0] * batch)

    def step(self, qkv):
        """`counts` new tokens of each sequence, and then a cut back to `keep`; everything is read on the device."""
        K, rows = self.K, qkv.shape[1]
        q, k, v = qkv[:, :, :self.heads], qkv[:, :, self.heads:self.heads + self.kv], qkv[:, :, self.heads + self.kv:]
        slots, after, left = K.paged_extend(self.table, self.lengths, self.counts, self.free, self.free_count, self.page, rows)
        K.paged_write(k, v, slots, self.k_pages, self.v_pages)
        out = K.attention_paged(q, self.k_pages, self.v_pages, self.table, after, self.window, self.sinks, first=self.lengths)
        kept, left = K.paged_cut(self.table, after, self.keep, self.free, left, self.page)
        self.lengths.copy_(kept)
        self.free_count.copy_(left)
        return out, after, kept

    def plain_step(self, qkv, before, after):
        """The attention of the same step over rows that stand one behind the other."""
        q, k, v = qkv[:, :, :self.heads], qkv[:, :, self.heads:self.heads + self.kv], qkv[:, :, self.heads + self.kv:]
        for b, (n, m) in enumerate(zip(before, after)):
            self.k[b, n:m], self.v[b, n:m] = k[b, :m - n], v[b, :m - n]
        at = dict(left=self.window, sinks=self.sinks, lengths=ints(after), first=ints(before))
        plain = self.K.attention_window(q, self.k, self.v, self.window, 0, self.sinks, first=at["first"], lengths=at["lengths"])
        return plain, at


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_a_server_step_by_step(K, t):
    """Prompts, tokens, proposals that are taken back, sequences that end and others in their place, with too few pages at times."""
    t, r = TYPES[t], random.Random(5)
    server = Server(K, t, 6, 31)
    refused = 0
    for step in range(30):
        rows = r.choice((1, 1, 1, 5, 40))
        before = server.lengths.tolist()
        counts = [r.choice((rows, rows, 0)) if n or rows > 1 else rows for n in before]
        server.counts.copy_(ints(counts))
        server.keep.copy_(ints([r.choice((1000, 1000, 1000, n + 1, 0)) for n in before]))
        qkv = normal(gen(step), 6, rows, server.heads + 2 * server.kv, server.size).to(t)
        got, after, kept = server.step(qkv)
        refused += sum(1 for n, c, m in zip(before, counts, after.tolist()) if m != n + c)
        plain, at = server.plain_step(qkv, before, after.tolist())
        q = qkv[:, :, :server.heads]
        want, bound = reference(q, server.k, server.v, visible(q, server.k, server.page, **at))
        within(got, want, bound, "step %d" % step)
        # (attention_window's probabilities have 22 bits in fp16, and both sides a rounding at the end)
        within(got, plain.double(), 4 * bound + 2 * HALF[t] * want.abs(), "against rows in one piece, step %d" % step)
        held = [p for row, n in zip(server.table.tolist(), kept.tolist()) for p in row[:up(n, server.page)]]
        assert sorted(held + server.free.tolist()[:int(server.free_count)]) == list(range(server.pages))
    assert 0 < refused < 60


def test_a_captured_server(K):
    """A step as a graph, replayed while lengths and tables change, with eager steps of another server in between, on another stream."""
    t = torch.float16
    servers = [Server(K, t, 3, 41), Server(K, t, 3, 41)]   # the same twice: one captured, one eager
    other = Server(K, t, 5, 42)
    qkv = normal(gen(1), 3, 1, 8, 64).to(t)
    for s in servers:
        s.counts.fill_(1)
        s.keep.fill_(1000)
    servers[0].step(qkv), servers[1].step(qkv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, after, kept = servers[0].step(qkv)
    stream = torch.cuda.Stream()
    for turn in range(70):
        qkv.copy_(normal(gen(100 + turn), *qkv.shape))
        for s in servers:
            s.keep.copy_(ints([0 if turn % 50 == 40 else 1000, 1000, turn % 9 * 8]))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        other.counts.fill_(2)
        other.keep.fill_(100)
        other.step(normal(gen(turn), 5, 3, 8, 64).to(t))
        want = servers[1].step(qkv)
        torch.cuda.synchronize()
        for a, b in zip((out, after, kept, servers[0].table, servers[0].free, servers[0].k_pages),
                        want + (servers[1].table, servers[1].free, servers[1].k_pages)):
            assert torch.equal(a, b), turn


# ---------------------------------------------------------------------------- probabilities far below the largest

# heads, kv_heads, q_rows, entries of the table behind the last page (with very many of them 20 rows share a tile)
SHARED = {"one row": (1, 1, 1, 3), "a few rows": (4, 2, 3, 3), "twenty rows": (20, 1, 1, 20000), "twenty rows of five": (8, 2, 5, 20000)}


def next_to_one_key(heads, kv_heads, q_rows, wide, t, size, gap, where, n=600, seed=21):
    """One sequence in which a key stands `gap` above all others and has nothing in its value; scores are exact in fp32 and all values positive."""
    g = gen(seed)
    page, width = 16, up(n, 16) + wide
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :up(n, page)] = torch.randperm(up(n, page), generator=g, device="cuda").int()
    k_pages, v_pages, _ = pool_of("heads", up(n, page), kv_heads, page, size, t, seed)
    k, v = torch.zeros(1, n, kv_heads, size, dtype=t, device="cuda"), (1 + torch.rand(1, n, kv_heads, size, generator=g, device="cuda")).mul(2.0 ** 14).to(t)
    k[0, :, :, 0] = -(torch.arange(n, device="cuda") % 8 / 8)[:, None].to(t)
    k[0, where, :, 0], v[0, where] = gap, 0
    at = torch.arange(n, device="cuda")
    own = table[0].long()[at // page]
    k_pages[own, :, at % page], v_pages[own, :, at % page] = k[0], v[0]
    q = torch.zeros(1, q_rows, heads, size, dtype=t, device="cuda")
    q[..., 0] = 1
    return q, k_pages, v_pages, table, k, v, page, dict(left=-1, sinks=0, lengths=ints([n]), first=None)


@pytest.mark.parametrize("rows", list(SHARED))
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("where", [0, 21, 599])
def test_attention_paged_next_to_a_key_without_value(K, rows, t, size, where):
    """A key that has nearly all of the weight and nothing to give, as a first token often has: the result is made of probabilities that are a
    2^12th to a 2^50th of the largest, and these are as exact, each by itself."""
    for gap in (8.0, 12.0, 17.0, 19.5, 21.5, 24.0, 28.0, 34.0):
        q, k_pages, v_pages, table, k, v, page, at = next_to_one_key(*SHARED[rows], TYPES[t], size, gap, where)
        seen = visible(q, k, page, **at)
        want, _ = reference(q, k, v, seen, alpha=1.0)
        got = K.attention_paged(q, k_pages, v_pages, table, alpha=1.0, **at)
        # Scores and their differences are exact.  The factor log2(e) has 2 roundings, the product with it and 12 added to it one: of x = 1.45 gap
        # + 14 as a power of two, so an exponential is off by log(2) 3 x u, and by 2^-22; fp16's terms leave out 2^-21.  Sums have n terms,
        # products, and are scaled anew as often as in `reference`.  All terms are positive, so a sum is off by no more than they are.
        n = 600
        each = 3 * (1.45 * gap + 14) * U + 3 * 2.0 ** -22 + 2.0 ** -21 + (2 * n + 16) * U + (n / 16 + 2) * 2.0 ** -22
        bound = want.abs() * (each + (1 + each) * (HALF[TYPES[t]] + 4 * U)) + SMALL[TYPES[t]]
        within(got, want, bound, "gap %g" % gap)


@pytest.mark.parametrize("rows", list(SHARED))
@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_paged_of_infinite_values_among_small_probabilities(K, rows, size):
    """An infinite value of the key that has nearly all of the weight stays infinite, what is no number stays none, in their columns alone."""
    for gap in (17.0, 24.0):
        q, k_pages, v_pages, table, k, v, page, at = next_to_one_key(*SHARED[rows], torch.float16, size, gap, 21)
        clean = K.attention_paged(q, k_pages, v_pages, table, alpha=1.0, **at)
        own = int(table[0, 21 // page])
        v_pages[own, :, 21 % page, 3], v_pages[own, :, 21 % page, 4], v_pages[own, :, 21 % page, 9] = math.inf, -math.inf, math.nan
        v_pages[int(table[0, 590 // page]), :, 590 % page, 11] = math.nan
        got = K.attention_paged(q, k_pages, v_pages, table, alpha=1.0, **at)
        assert bool((got[..., 3] == math.inf).all()) and bool((got[..., 4] == -math.inf).all())
        assert bool(torch.isnan(got[..., [9, 11]]).all())
        got[..., [3, 4, 9, 11]] = clean[..., [3, 4, 9, 11]]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("batch", [5, 400])
def test_cut_over_what_is_kept(K, batch):
    """The lengths afterwards may go over `keep`, in one launch and in two."""
    from cubert_amd._lib import lib
    table, lengths, free, there = tables(3, batch, 9, 16, batch * 9 + 4, 140)
    r = random.Random(batch)
    keep = [r.choice((0, n, n + 5, -3, r.randint(0, n))) for n in lengths]
    on, stack, count, left = [ints(x) for x in (table, lengths, keep)], ints(free), ints([there]), ints([0])
    work = torch.zeros(batch, dtype=torch.int32, device="cuda")
    rc = lib().cubert_paged_cut(on[0].data_ptr(), 9, 9, on[1].data_ptr(), on[2].data_ptr(), stack.data_ptr(), count.data_ptr(), len(free), len(free), 16, batch,
                                on[2].data_ptr(), left.data_ptr(), work.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (on[2].tolist(), left.tolist()[0], stack.tolist()) == cut_reference(table, lengths, keep, free, there, 16)


# batch, rows, page, pages to spare: more slots than 2048 workgroups of 1024 have
LARGE_EXTEND = {"long prompts": (5, 700000, 64, 60000), "many prompts": (3001, 900, 16, 200000), "many prompts and a short stack": (3001, 900, 16, 90000),
                "as many sequences as there may be": (1 << 18, 9, 4, 700000)}


@pytest.mark.parametrize("name", list(LARGE_EXTEND))
def test_extend_of_very_many_slots(K, name):
    """A workgroup takes several times its 1024 slots, and carries on what it has added up."""
    batch, rows, page, spare = LARGE_EXTEND[name]
    r = random.Random(batch)
    lengths, counts = [r.randint(0, 3 * page) for _ in range(batch)], [r.choice((0, rows, r.randint(0, rows))) for _ in range(batch)]
    width = up(rows, page) + 3
    table, held = [], 0
    for n in lengths:
        table.append(list(range(held, held + up(n, page))) + [-1] * (width - up(n, page)))
        held += up(n, page)
    free = list(range(held, held + spare))
    r.shuffle(free)
    on = ints(table)
    slots, after, left = K.paged_extend(on, ints(lengths), ints(counts), ints(free), ints([spare]), page, rows)
    want = extend_reference(table, lengths, counts, free, spare, page, rows)
    assert torch.equal(slots.cpu(), torch.tensor(want[0], dtype=torch.int32)) and after.tolist() == want[1] and left.tolist() == [want[2]]
    assert torch.equal(on.cpu(), torch.tensor(want[3], dtype=torch.int32))


def test_extend_of_very_many_slots_in_time(K):
    """As many workgroups as there are thousands of slots would add up all sequences each: fifty times as long as it takes to write the slots (2048
    workgroups: six times)."""
    batch, rows = 1 << 17, 2048
    table, lengths, free = torch.zeros(batch, 2, dtype=torch.int32, device="cuda"), ints(list(range(2048))).repeat(batch // 2048), ints(list(range(2 * batch)))

    def least(call):
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    slots = torch.empty(batch, rows, dtype=torch.int32, device="cuda")
    count = ints([2 * batch])
    assert least(lambda: K.paged_extend(table, lengths, None, free, count, rows, rows)) < 20 * least(lambda: slots.fill_(-1))


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("name", ["long", "a few tokens", "many heads to one", "many rows", "a window and sinks"])
@pytest.mark.parametrize("wide", [3, 20000])
def test_attention_paged_is_the_same_in_a_larger_pool(K, name, t, size, wide):
    """Pages of nobody, 96 MB and more of them, change how pools are read, where tables have room for as much, and no bit of the results."""
    q, k_pages, v_pages, table, k, v, page, at = paged(name, TYPES[t], size, wide=wide)
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    more = (100 << 20) // (2 * page * k_pages.shape[1] * size * q.element_size())
    k_large, v_large = (torch.cat([p, torch.full((more,) + p.shape[1:], math.nan, dtype=p.dtype, device="cuda")]) for p in (k_pages, v_pages))
    assert torch.equal(got, K.attention_paged(q, k_large, v_large, table, **at))
    within(got, *reference(q, k, v, visible(q, k, page, **at)), name)


@pytest.mark.parametrize("batch,q_rows", [(600, 1), (767, 2), (768, 1), (769, 1), (1280, 1), (1281, 1)])
@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_paged_of_as_many_sequences_as_are_cut(K, batch, q_rows, t):
    """1280 sequences are the most that are cut into pieces: five chunks of 64 for each of a workgroup's wavefronts to look through."""
    r = random.Random(batch)
    lengths = [r.choice((0, 1, 9, 40, 70)) if r.random() < 0.97 else 1600 for _ in range(batch)]
    lengths[0], lengths[-1] = 900, 1700
    q, k_pages, v_pages, table, k, v, page, at = paged((batch, q_rows, 2, 1, 16, -1, 0, tuple(lengths), None), TYPES[t], 32, wide=4000)
    want, bound = reference(q, k, v, visible(q, k, page, **at))
    within(K.attention_paged(q, k_pages, v_pages, table, **at), want, bound, "many")


# ---------------------------------------------------------------------------- tiles of 32 rows

# More than 16 rows share a tile of 32 where tables and window have room for 768 KB of K and V for a sequence and key head, and 24 MB (fp16) or
# 96 MB (fp32) of all.  Cases as above; those without a window have tables for 320000 keys, which is as much for two key heads of the smallest size.
TILES = {
    "seventeen rows": (2, 1, 17, 1, 16, -1, 0, (500, 40), None),
    "twenty rows": (2, 5, 8, 2, 16, -1, 0, (1000, 333), None),
    "thirty-two rows": (3, 8, 8, 2, 64, -1, 0, (700, 0, 130), None),
    "padded": (4, 5, 8, 2, 16, -1, 0, (50, 51, 52, 53), (44, 50, 52, 60)),
    "before the sequence": (3, 20, 2, 2, 16, -1, 0, (64, 7, 0), None),
    "tokens in the middle": (2, 3, 16, 2, 16, -1, 0, (600, 1000), (90, 20)),
    "three tiles": (2, 9, 18, 2, 16, -1, 0, (700, 45), None),
    "unlike lengths": (33, 3, 8, 1, 16, -1, 0, tuple((37 * i * i) % 1500 for i in range(33)), None),
    "long": (1, 8, 8, 2, 16, -1, 0, (9000,), None),
}
# key heads and window by type and size, so that the window's keys are as many bytes
WINDOWS = {("f16", 32): (36, 6200), ("f16", 64): (30, 3500), ("f16", 128): (26, 2100), ("f32", 32): (128, 3300), ("f32", 64): (104, 2100),
           ("f32", 128): (100, 1100)}


def tiles_case(name, t, size, layout="heads"):
    if name != "window":
        return paged(TILES[name], TYPES[t], size, layout, wide=20000)
    kv, left = WINDOWS[t, size]                            # (in two sequences, one of them within the window)
    return paged((2, 5, 2 * kv, kv // 2, 16, left, 3, (left + 700, 40), None), TYPES[t], size, layout, wide=0)


def in_pool(pool, *pages):
    """Pools as they are, or behind so many pages of nobody that the pool is read past the caches."""
    if pool == "own":
        return pages
    more = (100 << 20) // (2 * pages[0][0].numel() * pages[0].element_size()) + 1
    return tuple(torch.cat([p, torch.full((more,) + p.shape[1:], math.nan, dtype=p.dtype, device="cuda")]) for p in pages)


def attention_uncut(q, k_pages, v_pages, table, left, sinks, lengths, first, alpha=None):
    """attention_paged without memory for partial sums."""
    from cubert_amd._lib import lib
    batch, q_rows, heads, size = q.shape
    out = torch.full_like(q, math.nan, memory_format=torch.contiguous_format)
    rc = getattr(lib(), "cubert_attention_paged_" + ("f32" if q.dtype == torch.float32 else "f16"))(
        q.data_ptr(), q.stride(1) if q_rows > 1 else heads * size, k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], table.data_ptr(),
        table.shape[1], table.shape[1], lengths.data_ptr(), None if first is None else first.data_ptr(), out.data_ptr(), heads * size,
        size ** -0.5 if alpha is None else alpha, batch, heads, k_pages.shape[1], q_rows, k_pages.shape[0], k_pages.shape[2], size, left, sinks, None, 0,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out


@pytest.mark.parametrize("name", list(TILES) + ["window"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("pool", ["own", "large"])
def test_attention_paged_in_tiles_of_32_rows(K, name, t, size, pool):
    """Cut and uncut, with the same bits each time."""
    q, k_pages, v_pages, table, k, v, page, at = tiles_case(name, t, size)
    k_pages, v_pages = in_pool(pool, k_pages, v_pages)
    seen = visible(q, k, page, **at)
    want, bound = reference(q, k, v, seen)
    got = K.attention_paged(q, k_pages, v_pages, table, **at)
    within(got, want, bound, name)
    assert bool((got[~seen.any(2)] == 0).all())
    assert torch.equal(got, K.attention_paged(q, k_pages, v_pages, table, **at))
    got = attention_uncut(q, k_pages, v_pages, table, **at)
    within(got, want, bound, name + " uncut")
    assert bool((got[~seen.any(2)] == 0).all())


@pytest.mark.parametrize("name", ["seventeen rows", "padded", "tokens in the middle", "three tiles", "unlike lengths", "window"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("pool", ["own", "large"])
def test_attention_paged_in_tiles_of_32_rows_without_some_pages(K, name, t, size, pool):
    """Entries that are no pages, and no numbers in all that no query sees."""
    q, k_pages, v_pages, table, k, v, page, at = tiles_case(name, t, size)
    gone = torch.rand(table.shape, generator=gen(4), device="cuda") < 0.3
    wild = ints([-1, 1 << 30, (1 << 31) - 1, -(1 << 31)]).repeat(table.numel() // 4 + 1)[:table.numel()].view(table.shape)
    table = torch.where(gone, wild, table)
    seen = visible(q, k, page, table=table, pages=k_pages.shape[0], **at)
    keep = torch.zeros(k_pages.shape[0] * page, dtype=torch.bool, device="cuda")
    b, j = seen.any(1).nonzero(as_tuple=True)
    keep[table[b, j // page].long() * page + j % page] = True
    k_pages, v_pages = in_pool(pool, *(torch.where(keep.view(-1, 1, page, 1), p, math.nan) for p in (k_pages, v_pages)))
    want, bound = reference(q, k, v, seen)
    for got in (K.attention_paged(q, k_pages, v_pages, table, **at), attention_uncut(q, k_pages, v_pages, table, **at)):
        within(got, want, bound, name)
        assert bool((got[~seen.any(2)] == 0).all())


@pytest.mark.parametrize("name", ["twenty rows", "three tiles", "window"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("layout", LAYOUTS[1:])
def test_attention_paged_in_tiles_of_32_rows_in_any_layout(K, name, t, size, layout):
    """Pools of other strides, queries out of a packed projection, a scale below 0."""
    q, k_pages, v_pages, table, k, v, page, at = tiles_case(name, t, size, layout)
    packed = torch.zeros(q.shape[0], q.shape[1], q.shape[2] + 3, size, dtype=q.dtype, device="cuda")
    packed[:, :, 1:-2] = q
    want, bound = reference(q, k, v, visible(q, k, page, **at), alpha=-0.03)
    within(K.attention_paged(packed[:, :, 1:-2], k_pages, v_pages, table, alpha=-0.03, **at), want, bound, name)


@pytest.mark.parametrize("name", ["twenty rows", "thirty-two rows", "window"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("pool", ["own", "large"])
def test_attention_paged_in_tiles_of_32_rows_of_no_number(K, name, t, size, pool):
    """What is no number in a query, and an infinite key: the results that take it, and no others."""
    q, k_pages, v_pages, table, k, v, page, at = tiles_case(name, t, size)
    q[..., 5] = torch.where(q[..., 5] < 0, -0.5, 0.5).to(q.dtype)
    seen, share = visible(q, k, page, **at), q.shape[2] // k.shape[2]
    b, i = (int(x) for x in seen.any(2).nonzero()[seen.any(2).sum() // 2])
    j = int(seen[b, i].nonzero()[0])
    without = seen.clone()
    without[b, :, j] = False
    want, bound = reference(q, k, v, seen)
    want_without, bound_without = reference(q, k, v, without)
    meets = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    meets[b, :, :share] = seen[b, :, j, None]
    none = meets & (q[..., 5] > 0)
    want, bound = torch.where(meets[..., None], want_without, want), torch.where(meets[..., None], bound_without, bound)
    k_pages[int(table[b, j // page]), 0, j % page, 5] = math.inf
    q[b, i, -1, 2] = math.nan
    none[b, i, -1] = True
    k_pages, v_pages = in_pool(pool, k_pages, v_pages)
    for got in (K.attention_paged(q, k_pages, v_pages, table, **at), attention_uncut(q, k_pages, v_pages, table, **at)):
        assert bool(torch.isnan(got[none]).all())
        within(torch.where(none[..., None], 0, got), torch.where(none[..., None], 0.0, want), bound, name)


# ---------------------------------------------------------------------------- every key of a long axis, once

LONG_ROWS = {"one row": (1, 1, 1, 3), "heads of two": (8, 2, 1, 3), "sixteen rows": (4, 1, 4, 3), "twenty rows": (20, 1, 1, 20000), "two tiles": (20, 1, 2, 20000)}


def alike(heads, kv_heads, q_rows, wide, t, size, n, page, seed=23):
    """A sequence of n keys with the same score, of which the last q_rows queries see n - q_rows + 1 to n, and pools of zeros for its values."""
    width = up(n, page) + wide * 16 // page
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :up(n, page)] = torch.randperm(up(n, page), generator=gen(seed), device="cuda").int()
    k_pages = torch.zeros(up(n, page), kv_heads, page, size, dtype=t, device="cuda")
    q = torch.zeros(1, q_rows, heads, size, dtype=t, device="cuda")
    return q, k_pages, torch.zeros_like(k_pages), table, ints([n])


def exactly(got, want, t, what):
    """Probabilities are powers of two and values too, or nothing: their sums are exact in fp32.  What is left is fp32's reciprocal of the number of keys, the
    product with it, and the storage type's rounding; in fp16 the second terms of the probabilities, 2^-36 of them."""
    within(got, want, want.abs() * (HALF[t] + 5 * U) + SMALL[t], what)


@pytest.mark.parametrize("rows", list(LONG_ROWS))
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("cut", [True, False])
def test_attention_paged_counts_every_key_once(K, rows, t, size, cut):
    """Column d counts the keys j with j % size = d, about 300 each, so a key more or less is 7 roundings of fp16; and then those of the d-th stretch."""
    t, (heads, kv, q_rows, wide), page, n = TYPES[t], LONG_ROWS[rows], 16, 300 * size + 77
    q, k_pages, v_pages, table, lengths = alike(heads, kv, q_rows, wide, t, size, n, page)
    at, seen = torch.arange(n, device="cuda"), n - q_rows + 1 + torch.arange(q_rows, device="cuda")
    for of in (at % size, at // up(n, size)):
        column = torch.zeros(n, size, dtype=torch.float64, device="cuda")
        column[at, of] = 1
        v_pages[table[0].long()[at // page], :, at % page] = column.to(t)[:, None]
        want = (column.cumsum(0)[seen - 1] / seen[:, None])[None, :, None].expand(1, q_rows, heads, size)
        call = dict(left=-1, sinks=0, lengths=lengths, first=None)
        exactly(K.attention_paged(q, k_pages, v_pages, table, **call) if cut else attention_uncut(q, k_pages, v_pages, table, **call), want, t, rows)


@pytest.mark.parametrize("rows", list(LONG_ROWS))
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("n,page", [(60000, 16), (131072, 256)])
def test_attention_paged_takes_each_key_of_a_long_axis(K, rows, t, size, n, page):
    """A column for each of some keys: on either side of what a wavefront has on its way together (16 or 32), of the pages it looks up at once (512 or
    1024 keys), of pages, and of pieces wherever these may begin; and the first and the last."""
    t, (heads, kv, q_rows, wide) = TYPES[t], LONG_ROWS[rows]
    q, k_pages, v_pages, table, lengths = alike(heads, kv, q_rows, wide, t, size, n, page)
    r = random.Random(n)
    keys = [0, 15, 16, 31, 32, 511, 512, 1023, 1024, 2047, 2048, n // 2 - 1, n // 2, n - 1025, n - 33, n - 32, n - 17, n - 16, n - q_rows - 1]
    for pieces in (226, 232, 240, 254, 255, 448, 512):      # (whole units to each)
        for i in (1, pieces // 2, pieces - 1):
            edge = n // 32 * i // pieces * 32
            keys += [edge - 32, edge - 1, edge, edge + 31]
    keys += [r.randrange(n - q_rows) for _ in range(-len(keys) % size)]
    seen = n - q_rows + 1 + torch.arange(q_rows, device="cuda")
    for i in range(0, len(keys), size):
        v_pages.zero_()
        column = torch.arange(size, device="cuda")
        key = torch.tensor(keys[i:i + size], device="cuda")
        v_pages[table[0].long()[key // page], :, key % page, column] = 2.0 ** 15
        want = torch.zeros(n, size, dtype=torch.float64, device="cuda")
        want[key, column] = 2.0 ** 15
        want = (want.cumsum(0)[seen - 1] / seen[:, None])[None, :, None].expand(1, q_rows, heads, size)
        exactly(K.attention_paged(q, k_pages, v_pages, table, lengths), want, t, "keys %d" % i)


# ---------------------------------------------------------------------------- calls at the edges of what is allowed


def test_results_of_nothing_overlap_nothing(K):
    """No rows, or no sequences: pointers that nothing is written to may be any."""
    from cubert_amd._lib import lib
    table, lengths, free, count, after, left = ints([[3, -1], [4, -1]]), ints([5, 9]), ints([1, 2, 0, 0]), ints([2]), ints([7, 7]), ints([7])
    stream = torch.cuda.current_stream().cuda_stream
    rc = lib().cubert_paged_extend(table.data_ptr(), 2, 2, lengths.data_ptr(), None, free.data_ptr(), count.data_ptr(), 4, 5, 16, 2, 0, lengths.data_ptr() + 4,
                                   after.data_ptr(), left.data_ptr(), stream)
    assert rc == 0 and after.tolist() == [5, 9] and left.tolist() == [2]
    left.fill_(7)
    for call in (lambda: lib().cubert_paged_extend(table.data_ptr(), 2, 2, lengths.data_ptr(), None, free.data_ptr(), count.data_ptr(), 4, 5, 16, 0, 3,
                                                   lengths.data_ptr(), lengths.data_ptr(), left.data_ptr(), stream),
                 lambda: lib().cubert_paged_cut(table.data_ptr(), 2, 2, lengths.data_ptr(), None, free.data_ptr(), count.data_ptr(), 4, 5, 16, 0,
                                                lengths.data_ptr(), left.data_ptr(), None, stream)):
        assert call() == 0 and left.tolist() == [2] and lengths.tolist() == [5, 9]
        left.fill_(7)


@pytest.mark.parametrize("name", ["one query", "a few tokens", "long", "nobody", "many rows"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("wide", [3, 20000])
@pytest.mark.parametrize("cut", [True, False])
def test_attention_paged_between_other_columns(K, name, t, wide, cut):
    """Results in the middle of wider rows: what is beside them stays, and so do the bits."""
    from cubert_amd._lib import lib
    q, k_pages, v_pages, table, _, _, page, at = paged(name, TYPES[t], 64, wide=wide)
    batch, q_rows, heads, size = q.shape
    floats = lib().cubert_attention_paged_partials(int(t == "f16"), batch, heads, k_pages.shape[1], q_rows, table.shape[1], page, size, at["left"], at["sinks"])
    partials = torch.full((floats,), math.nan, device="cuda") if cut else None
    whole = torch.full((batch * q_rows + 2, heads * size + 24), -7.0, dtype=q.dtype, device="cuda")
    out = whole[1:-1, 8:-16]
    rc = getattr(lib(), "cubert_attention_paged_" + t)(
        q.data_ptr(), heads * size, k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], table.data_ptr(), table.shape[1], table.shape[1],
        at["lengths"].data_ptr(), None, out.data_ptr(), heads * size + 24, size ** -0.5, batch, heads, k_pages.shape[1], q_rows, k_pages.shape[0], page, size,
        at["left"], at["sinks"], partials.data_ptr() if floats and cut else None, floats if cut else 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    want = K.attention_paged(q, k_pages, v_pages, table, **at) if cut else attention_uncut(q, k_pages, v_pages, table, **at)
    assert torch.equal(out.reshape(q.shape), want)
    out.fill_(-7.0)
    assert bool((whole == -7.0).all())


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("page,lengths", [(4096, (5000, 1, 4096, 8191)), (65536, (70000, 65535, 30)), (1 << 20, (3000,))])
def test_attention_paged_of_very_large_pages(K, t, size, page, lengths):
    q, k_pages, v_pages, table, k, v, page, at = paged((len(lengths), 2, 4, 2, page, 1500, 5, lengths, None), TYPES[t], size, wide=1)
    want, bound = reference(q, k, v, visible(q, k, page, **at))
    within(K.attention_paged(q, k_pages, v_pages, table, **at), want, bound, "large pages")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("cut", [True, False])
def test_attention_paged_of_sixteen_million_keys(K, t, cut):
    """A table that has a few pages over and over (reading allows it), up to the last of 2^24 keys; sums of powers of two are exact in fp32."""
    t, n, page, size, pages = TYPES[t], 1 << 24, 16, 32, 9
    g = gen(29)
    table = torch.randint(pages, (1, n // page), generator=g, device="cuda").int()
    k_pages = torch.zeros(pages, 1, page, size, dtype=t, device="cuda")
    v_pages = (torch.rand(pages, 1, page, size, generator=g, device="cuda") < 0.3).to(t)
    q = torch.zeros(1, 1, 2, size, dtype=t, device="cuda")
    call = dict(left=-1, sinks=0, lengths=ints([n]), first=None)
    count = torch.bincount(table[0].long(), minlength=pages).double()
    want = ((v_pages[:, 0].double().sum(1) * count[:, None]).sum(0) / n).expand(1, 1, 2, size)
    exactly(K.attention_paged(q, k_pages, v_pages, table, **call) if cut else attention_uncut(q, k_pages, v_pages, table, **call), want, t, "all of them")
