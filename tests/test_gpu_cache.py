"""The paged cache on the GPU against its definition (tests/paged.py): the
bookkeeping as whole numbers, the pages' bytes as copies and as roundings of
the appended rows."""
import random

import pytest

import common  # noqa: F401  (the path of the binding)
import paged
from paged import FULL, LIST, PAGE, Book

pytestmark = pytest.mark.gpu
SHAPES = [(16, 1, 512, 0, True), (32, 2, 64, 64, False), (64, 3, 128, 128, True),
          (256, 1, 256, 256, False), (128, 2, 256, 0, True)]


@pytest.fixture(scope="module")
def env():
    import torch
    import dsv4_gpu
    return dict(torch=torch, lib=dsv4_gpu.lib(), gpu=dsv4_gpu, dev=torch.device("cuda:0"))


def ints(env, v):
    return env["torch"].tensor(list(v), dtype=env["torch"].int32, device=env["dev"])


def starts_of(env, counts):
    return ints(env, [sum(counts[:i]) for i in range(len(counts) + 1)])


def new_cache(env, shape, layers=2, pages=40, seqs=9, cols=12):
    ps, kvh, k, v, fp8 = shape
    c = env["gpu"].PagedCache.new(layers, pages, ps, kvh, k, v, seqs, cols,
                                  "fp8" if fp8 else "bf16", env["dev"])
    g = env["torch"].Generator(device=env["dev"]).manual_seed(1)
    c.pages.copy_(env["torch"].randint(0, 256, c.pages.shape, generator=g, device=env["dev"],
                                       dtype=env["torch"].uint8))
    return c, Book(pages, seqs, cols, ps)


def check(env, c, book, image, status=True):
    assert c.ref.tolist() == book.ref
    assert c.length.tolist() == book.len
    assert c.table.tolist() == book.table
    if image is not None:
        assert env["torch"].equal(c.pages, image)
    if status:
        assert env["lib"].cache_status(c) == book.status
        book.status = 0


def moved(image, moves):
    out = image.clone()
    for a, b in moves:
        out[:, b] = image[:, a]
    return out


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_random_bookkeeping(env, shape, seed):
    """Two hundred calls drawn at random, refused ones among them, on a pool
    that is often full; state and pages equal after each."""
    lib, rng = env["lib"], random.Random(seed)
    c, book = new_cache(env, shape)
    n, ps = len(book.len), book.ps
    image = c.pages.clone()
    for step in range(120):
        some = rng.sample(range(n), rng.randint(1, 5))
        what = rng.random()
        if what < 0.45:
            counts = [rng.choice((0, 1, 5, ps, rng.randint(0, 3 * ps))) for _ in some]
            if rng.random() < 0.05:
                some[-1] = some[0] if len(some) > 1 else n
            if rng.random() < 0.05:
                counts[0] = 13 * ps
            lib.cache_reserve(c, starts_of(env, counts), ints(env, some))
            if any(x < 0 for x in counts):
                continue
            image = moved(image, book.reserve(some, counts))
        elif what < 0.7:
            parents = [rng.randrange(n) for _ in some]
            lib.cache_fork(c, ints(env, parents), ints(env, some))
            book.fork(parents, some)
        elif what < 0.95:
            to = [rng.choice((0, book.len[s], rng.randint(0, book.len[s]), book.len[s] + 1))
                  if rng.random() < 0.3 else rng.randint(0, book.len[s]) for s in some]
            whole = rng.random() < 0.2
            lib.cache_free(c, ints(env, some), None if whole else ints(env, to))
            book.free(some, [0] * len(some) if whole else to)
        else:
            used = ints(env, [-5])
            lib.cache_compact(c, used)
            image = moved(image, book.compact())
            assert used.tolist() == [sum(r > 0 for r in book.ref)]
        check(env, c, book, image)


def test_copy_on_write_of_many(env):
    """Four sequences that share a partly filled page all grow: three copy (the
    first ones of the list), the last one keeps the page; contents equal."""
    lib = env["lib"]
    c, book = new_cache(env, SHAPES[0])
    image = c.pages.clone()
    for fn, a in ((lib.cache_reserve, ([20], [0])),):
        fn(c, starts_of(env, a[0]), ints(env, a[1]))
        book.reserve(a[1], a[0])
    lib.cache_fork(c, ints(env, [0, 0, 0]), ints(env, [1, 2, 3]))
    book.fork([0, 0, 0], [1, 2, 3])
    lib.cache_reserve(c, starts_of(env, [1, 1, 1, 1]), ints(env, [3, 1, 0, 2]))
    moves = book.reserve([3, 1, 0, 2], [1, 1, 1, 1])
    assert len(moves) == 3
    check(env, c, book, moved(image, moves))


def test_full_pool_changes_nothing_and_blocks(env):
    torch, lib = env["torch"], env["lib"]
    c, book = new_cache(env, SHAPES[1], pages=6)
    lib.cache_reserve(c, starts_of(env, [100]), ints(env, [0]))
    book.reserve([0], [100])
    check(env, c, book, None)
    image = c.pages.clone()
    lib.cache_reserve(c, starts_of(env, [10, 200]), ints(env, [0, 1]))
    # blocked until the status is read: append, attention and another reserve
    st = starts_of(env, [5])
    k = torch.randn(5, 2, 64, device=env["dev"])
    lib.cache_append(c, 0, k, k, st, ints(env, [0]))
    lib.cache_reserve(c, st, ints(env, [0]))
    out = torch.full((5, 4, 64), 7.0, dtype=torch.bfloat16, device=env["dev"])
    lse = torch.full((5, 4), 7.0, device=env["dev"])
    lib.attention(c, 0, out.clone(), st, ints(env, [0]), out=out, lse=lse)
    assert (out == 7).all() and (lse == 7).all()
    book.status = FULL
    check(env, c, book, image)
    lib.cache_reserve(c, st, ints(env, [0]))  # works again
    book.reserve([0], [5])
    check(env, c, book, image)


def test_large_pool_and_table(env):
    """More pages than one step of the scan, found near the end."""
    torch, lib = env["torch"], env["lib"]
    c, book = new_cache(env, (16, 1, 64, 64, True), layers=1, pages=20011, seqs=3, cols=20011)
    lib.cache_reserve(c, starts_of(env, [16 * 20000]), ints(env, [1]))
    book.reserve([1], [16 * 20000])
    lib.cache_reserve(c, starts_of(env, [100, 3]), ints(env, [0, 2]))
    book.reserve([0, 2], [100, 3])
    lib.cache_free(c, ints(env, [1]), ints(env, [5000]))
    book.free([1], [5000])
    image = c.pages.clone()
    check(env, c, book, image)
    lib.cache_compact(c)
    check(env, c, book, moved(image, book.compact()))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_append(env, shape, kind):
    """Ragged counts with zeros, strided rows, rows in front of and behind the
    listed ones, values that round, overflow the group's scale, NaN and
    infinities; the other layer, slots and sequences stay as they were."""
    torch, lib = env["torch"], env["lib"]
    ps, kvh, kd, vd, fp8 = shape
    c, book = new_cache(env, shape, cols=6)
    g = torch.Generator(device=env["dev"]).manual_seed(3)
    held, counts, seqs = [5, 0, ps, 2 * ps - 1], [7, 0, 1, ps + 3], [4, 1, 0, 7]
    lib.cache_reserve(c, starts_of(env, held), ints(env, seqs))
    lib.cache_reserve(c, starts_of(env, counts), ints(env, seqs))
    book.reserve(seqs, held), book.reserve(seqs, counts)
    front, rows = 2, sum(counts) + 2 + 3
    starts = starts_of(env, counts) + front
    dt = getattr(torch, kind)
    wide = [torch.randn(rows, kvh * d + 16, generator=g, device=env["dev"]) * 3 for d in (kd, vd)]
    for w in wide:
        w[3] *= 1e-6       # below the scale's floor
        w[4] *= 1e30
        w[5, ::7] = 0
        w[6, 3], w[6, 70 % w.shape[1]], w[6, 5] = float("nan"), float("inf"), float("-inf")
    k, v = [w.to(dt)[:, :kvh * d].unflatten(1, (kvh, d)) if d else None
            for w, d in zip(wide, (kd, vd))]
    image = c.pages.clone()
    lib.cache_append(c, 1, k, v, starts, ints(env, seqs))
    check(env, c, book, None)
    size, v_off, ks, vs = paged.page_layout(ps, kvh, kd, vd, fp8)
    want = image.clone()
    for new, d, at, sat in ((k, kd, 0, ks), (v, vd, v_off, vs)):
        if new is None:
            continue
        x = new.float().cpu()
        if fp8:
            x = x.unflatten(-1, (-1, 64))
            fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
            r = fin.amax(-1).clamp(min=1e-4) * torch.tensor(1 / 448)
            bits = r.view(torch.int32)
            code = (bits >> 23) + ((bits & 0x7FFFFF) != 0)
            q = (x / (code << 23).view(torch.float32)[..., None])
            byte = q.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            byte = torch.where(torch.isfinite(x), byte, byte | 0x7F).flatten(-2)
            code = code.to(torch.uint8)
        else:
            byte = x.to(torch.bfloat16).contiguous().view(torch.uint8)
        u = 1 if fp8 else 2
        for i, (s, n) in enumerate(zip(seqs, counts)):
            for j in range(n):
                row = int(starts[i]) + j
                pos = held[i] + j
                page, slot = book.table[s][pos // ps], pos % ps
                for h in range(kvh):
                    e = (h * ps + slot) * d
                    want[1, page, at + u * e:at + u * (e + d)] = byte[row, h].to(env["dev"])
                    if fp8:
                        want[1, page, sat + e // 64:sat + (e + d) // 64] = \
                            code[row, h].to(env["dev"])
    if not fp8:  # a NaN is a NaN, whatever its bits
        a, b = c.pages.view(torch.bfloat16), want.view(torch.bfloat16)
        same = (a.view(torch.int16) == b.view(torch.int16)) | (a.isnan() & b.isnan())
    else:
        same = c.pages == want
        nan = ((c.pages & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F)
        same |= nan
    assert same.all(), (~same).nonzero()[:5]


def test_append_refuses_on_device(env):
    """A sequence listed twice, one out of range, more new tokens than the
    sequence holds, a table entry that is no page: not written, a status bit."""
    torch, lib = env["torch"], env["lib"]
    c, book = new_cache(env, SHAPES[1])
    lib.cache_reserve(c, starts_of(env, [40, 40, 40]), ints(env, [0, 1, 2]))
    book.reserve([0, 1, 2], [40, 40, 40])
    check(env, c, book, None)
    k = torch.randn(6, 2, 64, device=env["dev"])
    for seqs, counts, bit in (([0, 0], [2, 2], LIST), ([1, 9], [0, 3], LIST),
                              ([-1], [3], LIST), ([2], [41], LIST), ([3], [1], LIST)):
        image = c.pages.clone()
        big = torch.randn(sum(counts), 2, 64, device=env["dev"])
        lib.cache_append(c, 0, big, big, starts_of(env, counts), ints(env, seqs))
        assert lib.cache_status(c) == bit, seqs
        if len(seqs) == 1 and counts[0] <= 40:
            assert torch.equal(c.pages, image)
    for entry in (-1, 40, 2 ** 31 - 1, -2 ** 31):
        c.table[1, 1] = entry
        image = c.pages.clone()
        lib.cache_append(c, 0, k, k, starts_of(env, [6]), ints(env, [1]))
        assert lib.cache_status(c) == PAGE
        assert torch.equal(c.pages, image)


def test_bookkeeping_in_a_graph(env):
    """A captured fork - reserve - free of the child, replayed with eager work
    between: every replay leaves what the eager calls leave."""
    torch, lib = env["torch"], env["lib"]
    c, book = new_cache(env, SHAPES[2])
    lib.cache_reserve(c, starts_of(env, [70, 9]), ints(env, [0, 1]))
    book.reserve([0, 1], [70, 9])
    ws = torch.empty(lib.cache_workspace_bytes(c), dtype=torch.uint8, device=env["dev"])
    kids, olds, st = ints(env, [5, 6]), ints(env, [0, 1]), starts_of(env, [4, 60])
    back = ints(env, [72, 9])

    def step():
        lib.cache_fork(c, olds, kids)
        lib.cache_reserve(c, st, kids, workspace=ws)
        lib.cache_free(c, kids, back)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        lib.cache_free(c, kids)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    book.fork([0, 1], [5, 6])
    moves = book.reserve([5, 6], [4, 60])
    book.free([5, 6], [72, 9])
    for i in range(4):
        image = c.pages.clone()
        graph.replay()
        check(env, c, book, moved(image, moves))
        lib.cache_free(c, kids)
        (c.pages.float().sum() * i).item()


def rows(env, n, c, seed):
    """New tokens' keys and values for a cache, float32."""
    torch, s = env["torch"], c.struct
    g = torch.Generator(device=env["dev"]).manual_seed(seed)
    return [torch.randn(n, s.kv_heads, d, generator=g, device=env["dev"]) if d else None
            for d in (s.k_dim, s.v_dim)]


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[1]], ids=str)
def test_append_skips_whole_entries(env, shape):
    """An entry with more new tokens than its sequence holds, with rows outside
    the call's or with a length beyond its table, one listed twice: none of
    its rows is written, pages shared with a fork among them, and the entries
    beside it are as in a call without it."""
    torch, lib = env["torch"], env["lib"]
    c, book = new_cache(env, shape)
    lib.cache_reserve(c, starts_of(env, [40, 70, 9]), ints(env, [0, 1, 2]))
    lib.cache_fork(c, ints(env, [0]), ints(env, [5]))
    assert lib.cache_status(c) == 0
    clean = c.pages.clone()
    k, v = rows(env, 120, c, 4)

    def call(seqs, starts, n=120):
        lib.cache_append(c, 1, k[:n], None if v is None else v[:n], ints(env, starts),
                         ints(env, seqs))

    def reset():
        c.pages.copy_(clean)

    for seqs, starts, good, good_starts, n in (
            ([0], [0, 41], None, None, 120),              # more than it holds
            ([5, 1], [0, 41, 111], [1], [41, 111], 120),
            ([1, 0], [3, 10, 90], [1], [3, 10], 120),
            ([0, 0], [0, 5, 9], None, None, 120),         # twice
            ([2, 0, 1, 0], [0, 9, 20, 60, 61], [2, 1], [0, 9], 120),
            ([1, 2], [0, 20, 29], [1], [0, 20], 25),      # its end behind the rows
            ([1, 2], [0, 20, 29], [1], [0, 20], 20),      # all of it
            ([2, 1], [-3, 6, 50], [1], [6, 50], 120),     # its start before them
            ([2, 1], [-9, 0, 50], [1], [0, 50], 120),
            ([-1, 1], [0, 4, 50], [1], [4, 50], 120), ([9, 1], [0, 4, 50], [1], [4, 50], 120),
            ([3, 1], [0, 4, 50], [1], [4, 50], 120),      # holds nothing
            ([1, 2], [10, 5, 14], None, None, 120),       # starts that fall
            ([1, 2, 0], [0, 20, 10, 30], None, None, 120)):
        reset()
        if good:
            if seqs[0] == 2 and len(seqs) == 4:           # the good ones are not neighbours
                call([2], [0, 9])
                call([1], [20, 60])
            else:
                call(good, good_starts, n)
            assert lib.cache_status(c) == 0
        want = c.pages.clone()
        reset()
        call(seqs, starts, n)
        assert lib.cache_status(c) == LIST, (seqs, starts)
        assert torch.equal(c.pages, want), (seqs, starts)
    for length in (-1, 12 * shape[0] + 1, 2 ** 31 - 1):
        reset()
        c.length[2] = length
        call([2], [0, 1])
        assert lib.cache_status(c) == LIST
        assert torch.equal(c.pages, clean)


@pytest.mark.parametrize("bad", ["list", "page"])
def test_append_writes_what_stands_beside_a_refused_entry(env, bad):
    """Thousands of valid tokens behind a refused entry, in several layers: all
    of them are written whatever waves of the call have met it, and so in
    the appends that follow; reserve, append and attention are blocked as soon
    as a reserve has met the refusal, until the status is read."""
    torch, lib = env["torch"], env["lib"]
    c, book = new_cache(env, (16, 1, 64, 64, False), layers=3, pages=1100, seqs=5, cols=500)
    counts, seqs = [33, 4000, 5000, 7000], [0, 1, 2, 3]
    lib.cache_reserve(c, starts_of(env, counts), ints(env, seqs))
    book.reserve(seqs, counts)
    k, v = rows(env, sum(counts), c, 5)
    starts = starts_of(env, counts)
    if bad == "page":
        c.table[0, 1:] = 5000
    else:
        lib.cache_free(c, ints(env, [0]), ints(env, [20]))
        book.free([0], [20])
    assert lib.cache_status(c) == 0
    clean = c.pages.clone()
    for layer in range(3):  # the valid ones alone
        lib.cache_append(c, layer, k, v, starts[1:].contiguous(), ints(env, seqs[1:]))
    want = c.pages.clone()
    for _ in range(5):
        c.pages.copy_(clean)
        for layer in range(3):
            lib.cache_append(c, layer, k, v, starts, ints(env, seqs))
        got = c.pages.clone()
        if bad == "page":  # the rows that its first page takes
            got[:, book.table[0][0]] = want[:, book.table[0][0]]
        assert torch.equal(got, want)
        image = c.pages.clone()
        out = torch.full((3, 2, 64), 7.0, dtype=torch.bfloat16, device=env["dev"])
        st = ints(env, [0, 3])
        lib.attention(c, 0, out.clone(), st, ints(env, [1]), out=out)
        lib.cache_reserve(c, st, ints(env, [1]))
        lib.cache_append(c, 1, k, v, starts[1:].contiguous(), ints(env, [3, 2, 1]))
        assert (out == 7).all() and c.length.tolist() == book.len
        assert torch.equal(c.pages, image)
        assert lib.cache_status(c) == (PAGE if bad == "page" else LIST)
    assert lib.cache_status(c) == 0


def test_fork_skips_a_parent_with_a_bad_entry(env):
    """A parent whose table names no page: its child stays empty and no page's
    count changes; the other pairs of the list are forked."""
    lib = env["lib"]
    c, book = new_cache(env, SHAPES[1])
    lib.cache_reserve(c, starts_of(env, [100, 70]), ints(env, [0, 1]))
    book.reserve([0, 1], [100, 70])
    for entry in (-1, 40, 2 ** 31 - 1, -2 ** 31):
        for at in (0, 3):
            good = book.table[0][at]
            c.table[0, at] = book.table[0][at] = entry
            lib.cache_fork(c, ints(env, [0, 1, 0]), ints(env, [4, 5, 6]))
            book.fork([1], [5])
            book.status = PAGE
            check(env, c, book, None)
            c.table[0, at] = book.table[0][at] = good
            lib.cache_free(c, ints(env, [5]))
            book.free([5], [0])
            check(env, c, book, None)


def test_free_skips_a_sequence_with_a_bad_entry(env):
    """A sequence whose table names no page behind the cut: its length, its row
    and the pages' counts stay as they were; the others of the list are cut.
    Entries in front of the cut are not looked at."""
    lib = env["lib"]
    c, book = new_cache(env, SHAPES[1])
    lib.cache_reserve(c, starts_of(env, [100, 70]), ints(env, [0, 1]))
    book.reserve([0, 1], [100, 70])
    for entry in (-1, 40, 2 ** 31 - 1, -2 ** 31):
        for at in (1, 3):
            good = book.table[0][at]
            c.table[0, at] = book.table[0][at] = entry
            lib.cache_fork(c, ints(env, [1]), ints(env, [5]))
            book.fork([1], [5])
            lib.cache_free(c, ints(env, [0, 5]), ints(env, [32, 32]))
            book.free([5], [32])
            book.status = PAGE
            check(env, c, book, None)
            lib.cache_free(c, ints(env, [5]))
            book.free([5], [0])
            c.table[0, at] = book.table[0][at] = good
            check(env, c, book, None)
    good = book.table[0][0]
    c.table[0, 0] = book.table[0][0] = -1
    lib.cache_free(c, ints(env, [0]), ints(env, [40]))
    book.free([0], [40])
    check(env, c, book, None)


def test_the_largest_lists(env):
    """As many sequences as a list may name, in any order: forked, grown and cut
    back together, and appended to; lists that are wrong at any place of it."""
    torch, lib = env["torch"], env["lib"]
    n, rng = 1024, random.Random(3)
    c, book = new_cache(env, (16, 1, 64, 64, True), layers=1, pages=4100, seqs=2 * n, cols=4)
    order = rng.sample(range(n), n)
    counts = [rng.choice((0, 1, 2, 16, 30)) for _ in order]
    lib.cache_reserve(c, starts_of(env, counts), ints(env, order))
    book.reserve(order, counts)
    kids = [n + s for s in order]
    lib.cache_fork(c, ints(env, order), ints(env, kids))
    book.fork(order, kids)
    image = c.pages.clone()
    some = rng.sample(kids, n)
    more = [rng.choice((0, 1, 3, 17)) for _ in some]
    lib.cache_reserve(c, starts_of(env, more), ints(env, some))
    image = moved(image, book.reserve(some, more))
    check(env, c, book, image)
    # appended as one list, and one sequence after the other
    k, v = rows(env, sum(more), c, 6)
    starts = starts_of(env, more)
    for i, s in enumerate(some[:300]):
        lib.cache_append(c, 0, k, v, starts[i:i + 2].contiguous(), ints(env, [s]))
    rest = starts[300:].contiguous()
    lib.cache_append(c, 0, k, v, rest, ints(env, some[300:]))
    want = c.pages.clone()
    c.pages.copy_(image)
    lib.cache_append(c, 0, k, v, starts, ints(env, some))
    assert lib.cache_status(c) == 0 and torch.equal(c.pages, want)
    c.pages.copy_(image)
    for at in (1, 63, 64, 65, 128, 1000, 1023):  # starts that fall there
        bad = starts.clone()
        bad[at] = bad[at - 1] - 1 if at > 1 else bad[at + 1] + 1
        lib.cache_append(c, 0, k, v, bad, ints(env, some))
        assert lib.cache_status(c) == LIST and torch.equal(c.pages, image), at
    for i, j in ((0, 64), (63, 1023), (5, 6)):   # a sequence twice
        twice = list(some)
        twice[j] = twice[i]
        lib.cache_append(c, 0, k, v, starts, ints(env, twice))
        want_bit = LIST if more[i] or more[j] else 0
        assert lib.cache_status(c) == want_bit
        for entry in (i, j):
            page = {p for p in book.table[some[entry]] if p >= 0}
            for p in page:
                if book.ref[p] == 1:
                    assert torch.equal(c.pages[:, p], image[:, p]), (i, j, entry)
        c.pages.copy_(image)
    to = [rng.randint(0, book.len[s]) for s in some]
    lib.cache_free(c, ints(env, some), ints(env, to))
    book.free(some, to)
    check(env, c, book, image)
