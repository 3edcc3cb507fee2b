"""dsv4g_attention against the softmax of its definition in 64 bits, and the
whole path around it: reserve, append, attention, head, scores, rollback.
Bounds: tests/paged.py (attend_bounds)."""
import math
import random

import pytest

import common  # noqa: F401  (the path of the binding)
import paged
from paged import LIST, PAGE

pytestmark = pytest.mark.gpu
# heads, kv heads, key width, value width
LATENT, SHARD, LAT256 = (64, 1, 512, 0), (5, 1, 512, 0), (12, 2, 256, 0)
GQA, ONE, ODD, WIDE, MHA = ((32, 8, 128, 128), (4, 1, 64, 64), (10, 2, 128, 128),
                            (6, 2, 256, 256), (3, 3, 64, 64))


@pytest.fixture(scope="module")
def env():
    import torch
    import dsv4_gpu
    return dict(torch=torch, lib=dsv4_gpu.lib(), gpu=dsv4_gpu, dev=torch.device("cuda:0"))


def ints(env, v):
    return env["torch"].tensor(list(v), dtype=env["torch"].int32, device=env["dev"])


class Setup:
    """A cache whose sequences hold past[i] + new[i] tokens of random rows in
    randomly ordered pages; every other byte of the pool is NaN or what extra
    says."""

    def __init__(self, env, shape, ps, fp8, past, new, seed=0, layers=2, layer=1, spare=3,
                 order=None, fill=0xFF):
        torch, dev = env["torch"], env["dev"]
        self.env, self.shape, self.ps, self.fp8 = env, shape, ps, fp8
        self.heads, kvh, kd, vd = shape
        self.past, self.new, self.layer = past, new, layer
        total = [p + n for p, n in zip(past, new)]
        need = [-(-t // ps) for t in total]
        n, cols = len(past), max(1, max(need)) + 1
        pages = sum(need) + spare
        rng = random.Random(seed)
        self.c = c = env["gpu"].PagedCache.new(layers, pages, ps, kvh, kd, vd, n, cols,
                                               "fp8" if fp8 else "bf16", dev)
        c.pages.fill_(fill)  # 0xFF: NaN as BF16, as E4M3 and as a scale
        order = order or rng.sample(range(pages), sum(need))
        table, at = [[-1] * cols for _ in range(n)], 0
        for i, k in enumerate(need):
            table[i][:k] = order[at:at + k]
            at += k
        c.table.copy_(torch.tensor(table, dtype=torch.int32))
        c.length.copy_(torch.tensor(total, dtype=torch.int32))
        c.ref[torch.tensor(order[:at], dtype=torch.long, device=dev)] = 1
        self.table = table
        g = torch.Generator(device=dev).manual_seed(seed)
        # the whole contents by append itself (tested on its own)
        st = ints(env, [sum(total[:i]) for i in range(n + 1)])
        rows = max(1, sum(total))
        self.k = torch.randn(rows, kvh, kd, generator=g, device=dev)
        self.v = torch.randn(rows, kvh, vd, generator=g, device=dev) if vd else None
        if sum(total):
            env["lib"].cache_append(c, layer, self.k, self.v, st)
        self.starts = ints(env, [sum(new[:i]) for i in range(n + 1)])
        self.q = (2 * torch.randn(max(1, sum(new)), self.heads, kd, generator=g,
                                  device=dev)).to(torch.bfloat16)

    def check(self, out, lse, window=0, sink=None, scale=None, rows=None, q=None):
        torch = self.env["torch"]
        heads, kvh, kd, vd = self.shape
        scale = kd ** -0.5 if scale is None else scale
        q = (self.q if q is None else q).to(torch.bfloat16).double().cpu()
        host = self.c.pages[self.layer].cpu()
        sink = None if sink is None else sink.double().cpu()
        out, lse = out.double().cpu(), lse.double().cpu()
        starts, r = self.starts.tolist(), 0
        for b, (p, n) in enumerate(zip(self.past, self.new)):
            keys, vals = paged.rows64(host, self.table[b], p + n, self.ps, kvh, kd, vd, self.fp8)
            for i in range(n):
                r = starts[b] + i
                if rows is not None and r not in rows:
                    continue
                o, e, mass, most = paged.attend64(q[r], keys, vals, p + i, scale, window, sink)
                tol, tol_lse = paged.attend_bounds(o, mass, most, kd)
                assert ((out[r] - o).abs() <= tol).all(), \
                    (b, i, ((out[r] - o).abs() / tol).max().item())
                assert ((lse[r] - e).abs() <= tol_lse + 2.0 ** -22 * e.abs()).all(), (b, i)

    def run(self, **kw):
        return self.env["lib"].attention(self.c, self.layer, self.q, self.starts, with_lse=True,
                                         **kw)


@pytest.mark.parametrize("shape", [LATENT, SHARD, LAT256, GQA, ONE, ODD, WIDE, MHA], ids=str)
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("window", [0, 20])
def test_shapes(env, shape, fp8, window):
    """Every head layout, page format: ragged chunks with an empty one, an
    empty cache, lengths of one; the rest of the pool NaN."""
    torch = env["torch"]
    s = Setup(env, shape, 16, fp8, [0, 37, 5, 0, 130, 64], [1, 3, 0, 40, 9, 1], seed=1)
    sink = torch.randn(shape[0], device=env["dev"]) if window else None
    out, lse = s.run(window=window, sink=sink)
    assert env["lib"].cache_status(s.c) == 0
    s.check(out, lse, window, sink)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("shape", [LATENT, GQA], ids=str)
def test_lengths(env, ps, shape):
    """Lengths around the tile's, the page's and the split's borders at decode
    (one token each)."""
    past = [0, 1, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 126, 127, 128, 254, 255, 256, 257,
            510, 511, 512, 513, 1000]
    s = Setup(env, shape, ps, False, past, [1] * len(past), seed=2)
    s.check(*s.run())
    s.check(*s.run(max_q=1, max_kv=1001))


@pytest.mark.parametrize("shape,fp8,past,new,window", [
    (LATENT, False, [5000], [1], 0), (LATENT, True, [9001, 100], [1, 1], 0),
    (GQA, False, [20011], [1], 0), (GQA, True, [3000, 7, 4097], [5, 5, 5], 0),
    (LATENT, False, [4000], [5], 128), (ONE, False, [30000], [3], 0),
    (WIDE, False, [2500], [2], 1000), (LAT256, True, [6000], [1], 0)], ids=str)
def test_split_over_the_cache(env, shape, fp8, past, new, window):
    """Few rows over a long cache: the cache is split and joined."""
    torch = env["torch"]
    s = Setup(env, shape, 64, fp8, past, new, seed=3)
    sink = torch.randn(shape[0], device=env["dev"])
    s.check(*s.run(max_q=max(new), window=window), window)
    s.check(*s.run(max_q=max(new), window=window, sink=sink), window, sink)


@pytest.mark.parametrize("shape", [LATENT, GQA, ODD, ONE], ids=str)
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_chunks(env, shape, fp8):
    """Prompt chunks: many rows, causal inside the chunk; sampled rows."""
    s = Setup(env, shape, 32, fp8, [300, 0], [333, 150], seed=4)
    rows = set(random.Random(1).sample(range(483), 40)) | {0, 1, 332, 333, 334, 482}
    for window in (0, 100):
        out, lse = s.run(window=window, max_q=333)
        s.check(out, lse, window, rows=rows)


def test_peaked_scores(env):
    """Scores in the hundreds: one token takes all, far from the running
    maximum of the tiles before it."""
    torch = env["torch"]
    s = Setup(env, LATENT, 64, False, [900], [4], seed=5)
    s.q.mul_(16)
    s.check(*s.run())
    s.check(*s.run(scale=0.5), scale=0.5)
    s.check(*s.run(scale=-0.04), scale=-0.04)
    s.check(*s.run(scale=0.0), scale=0.0)
    sink = torch.full((64,), 300.0, device=env["dev"])
    s.check(*s.run(sink=sink), sink=sink)


@pytest.mark.parametrize("shape", [LATENT, GQA, ONE], ids=str)
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("new", [5, 200])
def test_hidden_tokens_have_no_influence(env, shape, fp8, new):
    """NaN and infinities in later tokens of the chunk and in tokens behind
    the window: rows that do not see them are as without; rows that do hold
    them (as the 64-bit definition says) are not finite."""
    torch, lib = env["torch"], env["lib"]
    bad_new, window = new - 2, 150
    s = Setup(env, shape, 16, fp8, [300], [new], seed=6)
    clean, clean_lse = s.run(window=window)
    s.check(clean, clean_lse, window, rows=set(range(0, new, 17)))
    # token 299 - 150 - 3: no row of the chunk sees it; token bad_new of the
    # chunk: its rows bad_new, bad_new + 1 do
    hidden = 300 - window - 3
    k = torch.zeros(1, *s.k.shape[1:], device=env["dev"])
    for value in (float("nan"), float("inf"), float("-inf")):
        if fp8 and not math.isnan(value):
            continue  # held as NaN
        k.fill_(value)
        v = None if s.v is None else k.clone()
        for pos in (hidden, 300 + bad_new):
            s.c.length.fill_(pos + 1)
            lib.cache_append(s.c, 1, k, v, ints(env, [0, 1]))
        s.c.length.fill_(300 + new)
        out, lse = s.run(window=window)
        assert torch.equal(out[:bad_new], clean[:bad_new]), value
        assert torch.equal(lse[:bad_new], clean_lse[:bad_new])
        assert (~torch.isfinite(out[bad_new:].float())).any(-1).all()


@pytest.mark.parametrize("shape", [LATENT, SHARD, LAT256, GQA, ONE, ODD, WIDE, MHA], ids=str)
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("window", [0, 45])
def test_items_whole_and_dealt_out(env, shape, fp8, window):
    """The same batches under a close bound of their lengths (whole items) and
    under a wide one, which has their stages dealt out over the chip: decode,
    drafts and a chunk, with sequences that have nothing new between them."""
    gpu, lib = env["gpu"], env["lib"]
    for past, new in (([70, 0, 3, 200, 129], [1, 1, 1, 1, 0]), ([100, 31, 0], [5, 0, 5]),
                      ([40, 7], [150, 61])):
        s = Setup(env, shape, 16, fp8, past, new, seed=len(past))
        n, heads, kvh, kd, vd = len(past), *shape
        table = env["torch"].full((n, 4096), -1, dtype=env["torch"].int32, device=env["dev"])
        table[:, :s.c.table.shape[1]] = s.c.table
        c = gpu.PagedCache(s.c.pages, s.c.ref, table, s.c.length, s.c.status, 16, kvh, kd, vd,
                           "fp8" if fp8 else "bf16")
        most = [max(p + m for p, m in zip(past, new)), 65536]
        rows = set(range(0, sum(new), 13)) | {sum(new) - 1}
        need = [lib.attention_workspace_bytes(c, heads, n, sum(new), max(new), kv) for kv in most]
        assert need[1] > 0
        for kv in most:
            out, lse = lib.attention(c, 1, s.q, s.starts, max_q=max(new), max_kv=kv,
                                     window=window, with_lse=True)
            s.check(out, lse, window, rows=rows)
        assert lib.cache_status(c) == 0


@pytest.mark.parametrize("shape,fp8", [(LATENT, False), (GQA, True)], ids=str)
def test_window_that_no_length_passes(env, shape, fp8):
    """The largest windows are no window, in tiles whose first rows see
    nothing of the last stages."""
    s = Setup(env, shape, 32, fp8, [60, 0], [90, 33], seed=8)
    out, lse = s.run()
    s.check(out, lse, rows={0, 1, 40, 89, 90, 122})
    for window in (2**31 - 1, 2**31 - 200, 65536, 150):
        again, again_lse = s.run(window=window)
        assert env["torch"].equal(out, again) and env["torch"].equal(lse, again_lse), window


@pytest.mark.parametrize("shape", [LATENT, GQA], ids=str)
def test_scale_of_zero(env, shape):
    """Every visible token weighs the same, however large the products are."""
    torch = env["torch"]
    s = Setup(env, shape, 16, False, [70, 3], [5, 1], seed=9)
    s.q *= 1e16
    starts, total = [0, 75], [75, 4]
    for value in (1.0, 1e16):
        env["lib"].cache_append(s.c, 1, s.k * value, s.v, ints(env, [0, 75, 79]))
        out, lse = s.run(scale=0.0)
        rows = (s.k * value if s.v is None else s.v).to(torch.bfloat16).double()
        for r, (b, p) in enumerate([(0, 70), (0, 71), (0, 72), (0, 73), (0, 74), (1, 3)]):
            seen = rows[starts[b]:starts[b] + p + 1]
            want = seen.mean(0).repeat_interleave(shape[0] // shape[1], 0)
            mass = seen.abs().mean(0).repeat_interleave(shape[0] // shape[1], 0)
            # weights exactly 1, sums in fp32; the result rounded once
            tol = 2.0 ** -8 * want.abs() + (p + 8) * 2.0 ** -24 * mass
            assert ((out[r].double() - want).abs() <= tol).all(), (value, r)
            assert ((lse[r].double() - math.log(p + 1)).abs() <= 1e-6).all()


def test_values_not_finite_in_seen_places(env):
    """Separate values with an infinity in one column: rows that see it are not
    finite there, rows that do not see it are as without."""
    torch, lib = env["torch"], env["lib"]
    s = Setup(env, GQA, 16, False, [100], [40], seed=7)
    v = torch.randn(1, 8, 128, device=env["dev"])
    k = s.k[117:118]
    s.c.length.fill_(118)
    lib.cache_append(s.c, 1, k, v, ints(env, [0, 1]))
    s.c.length.fill_(140)
    clean, _ = s.run()
    v[:, :, 5] = float("inf")
    s.c.length.fill_(118)
    lib.cache_append(s.c, 1, k, v, ints(env, [0, 1]))
    s.c.length.fill_(140)
    out, lse = s.run()
    assert torch.equal(out[:17], clean[:17])
    assert not torch.isfinite(out[17:, :, 5].float()).any()


def test_rows_behind_the_last_and_strides(env):
    """Rows in front of the first sequence and behind the last stay as they
    were; q and out are columns of wider buffers; float32 activations."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    s = Setup(env, GQA, 16, False, [50, 3], [4, 2], seed=8)
    starts = s.starts + 3
    wide = torch.zeros(14, 32 * 128 + 64, dtype=torch.bfloat16, device=dev)
    q = wide[:, 64:].unflatten(1, (32, 128))
    q[3:9] = s.q
    obuf = torch.full((14, 32 * 128 + 8), 3.0, dtype=torch.bfloat16, device=dev)
    out = obuf[:, :32 * 128].unflatten(1, (32, 128))
    lse = torch.full((14, 32), 3.0, device=dev)
    lib.attention(s.c, 1, q, starts, out=out, lse=lse)
    s.check(out[3:9], lse[3:9])
    for t in (obuf, lse):
        assert (t[:3] == 3).all() and (t[9:] == 3).all()
    assert (obuf[:, 32 * 128:] == 3).all()
    f, fl = lib.attention(s.c, 1, s.q.float(), s.starts, with_lse=True)
    assert f.dtype == torch.float32
    want, wl = s.run()
    assert torch.equal(f, want.float()) and torch.equal(fl, wl)


@pytest.mark.parametrize("shape", [LATENT, SHARD, LAT256, GQA, ONE, ODD, WIDE, MHA], ids=str)
@pytest.mark.parametrize("kv", [64, 65536])
def test_chunks_in_wider_buffers(env, shape, kv):
    """As above for chunks, whose last tiles are not full: columns beside the
    heads and rows around the sequences stay as they were, in both types."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    heads, kvh, kd, vd = shape
    s = Setup(env, shape, 16, False, [9, 0, 1], [37, 0, 53], seed=10)
    dv, n = vd or kd, 90
    want, wl = lib.attention(s.c, 1, s.q, s.starts, max_q=53, max_kv=kv, with_lse=True)
    s.check(want, wl, rows={0, 1, 17, 36, 37, 60, 88, 89})
    for t in (torch.bfloat16, torch.float32):
        obuf = torch.full((n + 7, heads * dv + 8), 3.0, dtype=t, device=dev)
        out = obuf[:, :heads * dv].unflatten(1, (heads, dv))
        lse = torch.full((n + 7, heads), 3.0, device=dev)
        q = torch.zeros(n + 7, heads * kd + 16, dtype=t, device=dev)
        q = q[:, 16:].unflatten(1, (heads, kd))
        q[5:5 + n] = s.q
        lib.attention(s.c, 1, q, s.starts + 5, max_q=53, max_kv=kv, out=out, lse=lse)
        assert torch.equal(out[5:5 + n], want.to(t)) and torch.equal(lse[5:5 + n], wl)
        for x in (obuf, lse):
            assert (x[:5] == 3).all() and (x[5 + n:] == 3).all()
        assert (obuf[:, heads * dv:] == 3).all()


def test_many_sequences_and_repeats(env):
    """More sequences than a wave has lanes, listed in another order, some
    twice."""
    torch, lib = env["torch"], env["lib"]
    rng = random.Random(9)
    past = [rng.randint(0, 90) for _ in range(150)]
    s = Setup(env, ODD, 16, True, past, [rng.randint(0, 2) for _ in past], seed=9)
    out, lse = s.run()
    s.check(out, lse, rows=set(range(0, sum(s.new), 11)))
    a, b = [i for i, n in enumerate(s.new) if n == 2][:2]
    st = s.starts.tolist()
    q = torch.cat([s.q[st[a]:st[a] + 2], s.q[st[b]:st[b] + 2], s.q[st[a]:st[a] + 2]])
    two, two_lse = lib.attention(s.c, 1, q, ints(env, [0, 2, 4, 6]), ints(env, [a, b, a]),
                                 with_lse=True)
    assert torch.equal(two[:2], two[4:])
    out[st[a]:st[a] + 2], lse[st[a]:st[a] + 2] = two[:2], two_lse[:2]
    out[st[b]:st[b] + 2], lse[st[b]:st[b] + 2] = two[2:4], two_lse[2:4]
    s.check(out, lse, rows={st[a], st[a] + 1, st[b], st[b] + 1})


def test_device_refusals(env):
    """A list, length or table entry that cannot be: a status bit, the other
    sequences' rows right."""
    torch, lib = env["torch"], env["lib"]
    s = Setup(env, LATENT, 16, False, [40, 60], [2, 2], seed=10)
    good, _ = s.run()
    for seqs in ([-1, 1], [2, 1], [2 ** 31 - 1, 1]):
        out = torch.zeros_like(good)
        lib.attention(s.c, 1, s.q, s.starts, ints(env, seqs), out=out)
        assert lib.cache_status(s.c) == LIST
    for n in (1, -5, 2 ** 31 - 1):  # shorter than the chunk, or longer than the bound
        s.c.length[0] = n
        s.run()
        assert lib.cache_status(s.c) == LIST
    s.c.length[0] = 42
    s.run(max_kv=41)
    assert lib.cache_status(s.c) == LIST
    s.run(max_q=1)
    assert lib.cache_status(s.c) == LIST
    for entry in (-1, s.c.pages.shape[1], 2 ** 31 - 1, -2 ** 31):
        s.c.table[0, 1] = entry
        s.run()
        assert lib.cache_status(s.c) == PAGE
    s.c.table[0, 1] = s.table[0][1]
    assert torch.equal(s.run()[0], good)


def test_offsets_beyond_32_bits(env):
    """Pages more than 4 GiB behind the pool's start (their number times their
    size, and a layer's offset)."""
    torch = env["torch"]
    for layers, layer in ((1, 0), (30, 29)):
        pages = 80000 // layers
        s = Setup(env, LATENT, 64, False, [150, 70], [3, 1], seed=11, layers=layers, layer=layer,
                  spare=pages, order=[pages, pages - 3, pages - 1, pages + 2, pages - 7])
        assert s.c.pages.numel() > 1 << 32
        s.check(*s.run())
        del s
        torch.cuda.empty_cache()


def test_graph_and_streams(env):
    """A captured decode step (reserve, append, attention over the split
    cache), replayed with eager work between, against eager calls; two
    captured graphs that share a workspace, replayed one after the other."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    made = [Setup(env, LATENT, 64, True, [700, 90], [1, 1], seed=12, spare=8) for _ in range(2)]
    g = torch.Generator(device=dev).manual_seed(3)
    k = torch.randn(2, 1, 512, generator=g, device=dev)
    q = torch.randn(2, 64, 512, generator=g, device=dev).to(torch.bfloat16)
    st = ints(env, [0, 1, 2])
    need = lib.attention_workspace_bytes(made[0].c, 64, 2, 2, 1, 900)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    cws = torch.empty(lib.cache_workspace_bytes(made[0].c), dtype=torch.uint8, device=dev)

    def step(c, out, lse, ws):
        lib.cache_reserve(c, st, workspace=cws)
        lib.cache_append(c, 1, k, None, st)
        lib.attention(c, 1, q, st, max_q=1, max_kv=900, out=out, lse=lse, workspace=ws)

    bufs = [(torch.empty(2, 64, 512, dtype=torch.bfloat16, device=dev),
             torch.empty(2, 64, device=dev)) for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s, b in zip(made, bufs):
            step(s.c, *b, ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(bufs[0][0], bufs[1][0])
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            lib.attention(made[0].c, 1, q, st, max_q=1, max_kv=900, out=bufs[2 + i][0],
                          lse=bufs[2 + i][1], workspace=ws, window=64 * i)
    whole = torch.cuda.CUDAGraph()
    with torch.cuda.graph(whole):
        step(made[0].c, *bufs[0], ws)
    for i in range(4):
        k.copy_(torch.randn(2, 1, 512, generator=g, device=dev))
        q.copy_(torch.randn(2, 64, 512, generator=g, device=dev))
        whole.replay()
        step(made[1].c, *bufs[1], None)  # a workspace of its own
        torch.cuda.synchronize()
        assert torch.equal(bufs[0][0], bufs[1][0]) and torch.equal(bufs[0][1], bufs[1][1])
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(bufs[2][0], bufs[1][0])
        want = lib.attention(made[1].c, 1, q, st, window=64, max_q=1, max_kv=900)
        assert torch.equal(bufs[3][0], want)
    assert lib.cache_status(made[0].c) == lib.cache_status(made[1].c) == 0


def test_two_streams_at_once(env):
    torch, lib = env["torch"], env["lib"]
    s = Setup(env, LATENT, 64, False, [3000], [2], seed=13)
    t = Setup(env, GQA, 16, False, [2000, 10], [1, 70], seed=14)
    want = s.run()[0], t.run()[0]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            a = s.run()[0]
        b = t.run()[0]
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_speculative_step(env):
    """The path as an engine runs it, float32 activations as the library's
    other entries give them: a prompt, then a draft on a fork of the sequence,
    scored behind a head, cut back to what was accepted, a fork of that and
    more tokens on both sides, compaction; every layer's output and score
    against the definition over the tokens that the sequence then stands for."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    heads, vocab, kd = 8, 1000, 512
    g = torch.Generator(device=dev).manual_seed(15)
    bf = lambda *s: torch.randn(*s, generator=g, device=dev).to(torch.bfloat16).float()  # noqa: E731
    head = (torch.randn(vocab, kd, generator=g, device=dev) * 0.1).to(torch.bfloat16)
    c = env["gpu"].PagedCache.new(2, 24, 16, 1, kd, 0, 4, 10, "fp8", dev)
    latents, queries = bf(2, 80, 1, kd), bf(2, 80, heads, kd)
    given = torch.randint(0, vocab, (80,), generator=g, device=dev, dtype=torch.int32)
    holds = {0: [], 1: [], 2: [], 3: []}    # the rows that each sequence stands for
    # what the cache holds of each row: 8-bit, by its definition
    kept = latents.cpu().double().unflatten(-1, (-1, 64))
    scale = torch.exp2(torch.ceil(torch.log2(kept.abs().amax(-1, keepdim=True) / 448)))
    kept = ((kept / scale).float().to(torch.float8_e4m3fn).double() * scale).flatten(-2)

    def take(seq, tokens):
        st, sq = ints(env, [0, len(tokens)]), ints(env, [seq])
        lib.cache_reserve(c, st, sq)
        before = len(holds[seq])
        holds[seq] = holds[seq] + tokens
        for layer in range(2):
            lib.cache_append(c, layer, latents[layer, tokens], None, st, sq)
            o = lib.attention(c, layer, queries[layer, tokens], st, sq)
            rows = kept[layer, holds[seq]]
            for i in (0, len(tokens) // 2, len(tokens) - 1):
                want, _, mass, most = paged.attend64(
                    queries[layer, tokens[i]].double().cpu(), rows, rows, before + i,
                    kd ** -0.5, 0, None)
                tol, _ = paged.attend_bounds(want, mass, most, kd)
                assert ((o[i].double().cpu() - want).abs() <= tol).all(), (seq, layer, i)
        logits = lib.gemv_bf16(o[:, 3].contiguous(), head.view(torch.int16), kd, vocab)
        lp, en, rank, ids, top = lib.logprobs(logits, given[tokens].contiguous(), top=5)
        host = logits.double().cpu().numpy()
        for i in range(len(tokens)):
            w = paged.score64(host[i], int(given[tokens[i]]), 5)
            assert abs(lp[i].item() - w[0]) < 1e-4 and abs(en[i].item() - w[1]) < 1e-4
            assert rank[i].item() == w[2] and ids[i].tolist() == w[3]

    rows = list(range(80))
    take(0, rows[:37])                                  # the prompt
    lib.cache_fork(c, ints(env, [0]), ints(env, [1]))
    holds[1] = list(holds[0])
    take(1, rows[37:45])                                # a draft of eight on the fork
    lib.cache_free(c, ints(env, [1]), ints(env, [40]))  # three accepted
    holds[1] = holds[1][:40]
    lib.cache_fork(c, ints(env, [1]), ints(env, [2]))
    holds[2] = list(holds[1])
    take(1, rows[60:63])
    take(0, rows[50:54])
    take(3, rows[70:])
    take(2, rows[63:65])
    lib.cache_free(c, ints(env, [0, 3]))
    lib.cache_compact(c)
    take(2, rows[45:60])
    take(1, rows[40:60])
    assert lib.cache_status(c) == 0
    used = {e for r in (1, 2) for e in c.table[r].tolist() if e >= 0}
    assert {i for i, r in enumerate(c.ref.tolist()) if r} == used


def wide_table(s, cols=4096):
    """The cache of a Setup under a table wide enough for any bound of lengths."""
    torch = s.env["torch"]
    _, kvh, kd, vd = s.shape
    table = torch.full((len(s.past), cols), -1, dtype=torch.int32, device=s.env["dev"])
    table[:, :s.c.table.shape[1]] = s.c.table
    return s.env["gpu"].PagedCache(s.c.pages, s.c.ref, table, s.c.length, s.c.status, s.ps, kvh,
                                   kd, vd, "fp8" if s.fp8 else "bf16")


@pytest.mark.parametrize("shape", [LATENT, LAT256, GQA, ONE, WIDE], ids=str)
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_scores_of_any_size(env, shape, fp8):
    """Scores up to the end of fp32's range, single tokens and long ranges
    among the rows, items whole and dealt out, with and without a sink. Every
    query has one column that is not zero, a power of two, so that q.k is exact
    in fp32. What is left are the scaling's roundings, relative to the distance
    to the row's maximum: 2^-22 of it, and e^-d d 2^-22 < 2^-23 of a weight,
    within the bound's 2^-18 for a score of no size (attend_bounds)."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    heads, kvh, kd, vd = shape
    past, new = [0, 700, 40, 0], [1, 3, 0, 70]
    s = Setup(env, shape, 16, fp8, past, new, seed=21)
    c = wide_table(s)
    tokens, n = sum(new), len(past)
    starts = s.starts.tolist()
    host = s.c.pages[1].cpu()
    held = [paged.rows64(host, s.table[b], past[b] + new[b], 16, kvh, kd, vd, fp8)
            for b in range(n)]
    g = torch.Generator(device=dev).manual_seed(5)
    at = torch.randint(0, kd, (tokens, heads, 1), generator=g, device=dev)
    rows = [0, 1, 3, 4, 73]
    for exponent, scale in ((3, 1.0), (20, 1.0), (25, -0.7), (28, 1.0), (30, 1.3), (33, 1.0),
                            (33, -1.0), (40, 1.0), (77, 0.3), (100, -1.0), (124, 1.0),
                            (124, 3.0), (-100, 1e38), (-100, -2e38), (10, 1e-30)):
        s.q.zero_()
        s.q.scatter_(2, at, 2.0 ** exponent)
        q, given = s.q.double().cpu(), float(torch.tensor(scale, dtype=torch.float32))
        # the sink of each head is its first row's one score
        own = given * held[0][0][0].repeat_interleave(heads // kvh, 0).gather(
            1, at[0].cpu())[:, 0] * 2.0 ** exponent
        for sink in (None, own.float()):
            want = {}
            for r in rows:
                b = max(i for i in range(n) if starts[i] <= r and new[i])
                want[r] = paged.attend64_far(q[r], *held[b], past[b] + r - starts[b], given,
                                             None if sink is None else sink.double())
            for kv in (773, 65536):
                out, lse = lib.attention(c, 1, s.q, s.starts, max_q=max(new), max_kv=kv,
                                         scale=scale, with_lse=True,
                                         sink=None if sink is None else sink.to(dev))
                out, lse = out.double().cpu(), lse.double().cpu()
                for r, (o, e, mass) in want.items():
                    tol, tol_lse = paged.attend_bounds(o, mass, torch.zeros_like(e), kd)
                    where = (exponent, scale, kv, r)
                    assert ((out[r] - o).abs() <= tol).all(), where
                    assert ((lse[r] - e).abs() <= tol_lse + 2.0 ** -22 * e.abs()).all(), where
    assert lib.cache_status(c) == 0


def test_single_tokens_with_large_scores(env):
    """A row that sees one token is that token's value, and its lse the score,
    whatever the score's size: random rows, their products summed in fp32."""
    torch, lib = env["torch"], env["lib"]
    s = Setup(env, LATENT, 16, False, [0] * 40, [1] * 40, seed=22)
    keys = s.k.to(torch.bfloat16).double()[:40]  # [sequence][1][512]
    for size in (1.0, 1e6, 1e9, 3e9, 1e11, 1e20, 1e30):
        q = (s.q.double() * size).to(torch.bfloat16)
        out, lse = lib.attention(s.c, 1, q, s.starts, with_lse=True, scale=1.0)
        assert torch.equal(out.double(), keys.expand(40, 64, 512)), size
        z = (q.double() * keys).sum(2)
        # 512 exact products summed in fp32, scaled once more
        tol = 520 * 2.0 ** -24 * (q.double() * keys).abs().sum(2) + 1e-6
        assert ((lse.double() - z).abs() <= tol).all(), size


@pytest.mark.parametrize("shape", [LATENT, GQA], ids=str)
@pytest.mark.parametrize("kv", [64, 65536], ids=["whole", "dealt out"])
def test_a_blocked_call_adds_no_status(env, shape, kv):
    """A pool without room for a new sequence: the attention that follows leaves
    the refusal as it is, though the sequence holds less than it is to have."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    heads, kvh, kd, vd = shape
    c = env["gpu"].PagedCache.new(1, 4, 16, kvh, kd, vd, 2, 4096, "bf16", dev)
    lib.cache_reserve(c, ints(env, [0, 40]), ints(env, [0]))
    starts = ints(env, [0, 1, 31])
    assert (lib.attention_workspace_bytes(c, heads, 2, 31, 30, kv) > 0) == (kv > 64)
    lib.cache_reserve(c, starts)
    q = torch.zeros(31, heads, kd, dtype=torch.bfloat16, device=dev)
    out = torch.full((31, heads, vd or kd), 5.0, dtype=torch.bfloat16, device=dev)
    lib.attention(c, 0, q, starts, max_q=30, max_kv=kv, out=out)
    assert lib.cache_status(c) == paged.FULL
    assert (out == 5).all() and c.length.tolist() == [40, 0]


@pytest.mark.parametrize("shape", [LATENT, SHARD, LAT256, GQA, ONE, ODD, WIDE, MHA], ids=str)
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_one_batch_under_both_plans(env, shape, fp8):
    """A batch that takes no workspace under a close bound (its items are whole)
    and one under a wide bound (its stages are dealt out)."""
    lib = env["lib"]
    past, new = [60, 0, 33, 71, 12], [2, 1, 0, 2, 2]
    s = Setup(env, shape, 16, fp8, past, new, seed=17)
    c, heads = wide_table(s), shape[0]
    need = [lib.attention_workspace_bytes(c, heads, 5, 7, 2, kv) for kv in (73, 65536)]
    assert need[0] == 0 and need[1] > 0
    for kv in (73, 65536):
        out, lse = lib.attention(c, 1, s.q, s.starts, max_q=2, max_kv=kv, with_lse=True)
        s.check(out, lse)
    assert lib.cache_status(c) == 0


@pytest.mark.parametrize("shape", [LATENT, LAT256, GQA, ONE, WIDE], ids=str)
def test_products_at_both_ends_of_fp32(env, shape):
    """Products near the largest number of either sign, whose difference no fp32
    number holds, under scales that bring them close to each other."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    heads, kvh, kd, vd = shape
    past, new = [300, 0, 33], [2, 1, 40]
    s = Setup(env, shape, 16, False, past, new, seed=23)
    sign = torch.randint(0, 2, (s.k.shape[0], kvh, 1), device=dev,
                         generator=torch.Generator(device=dev).manual_seed(6)) * 2.0 - 1
    s.k[:, :, 7:8] = 3.5 * sign
    lib.cache_append(s.c, 1, s.k, s.v, ints(env, [0, 302, 303, 376]))
    s.q.zero_()
    s.q[:, :, 7] = 2.0 ** 126   # products of +-2.98e38
    c = wide_table(s)
    for scale in (0.0, 1e-38, -1e-38, 3e-39, 1e-37):
        for kv in (302, 65536):
            out, lse = lib.attention(c, 1, s.q, s.starts, max_q=40, max_kv=kv, scale=scale,
                                     with_lse=True)
            out, lse = out.double().cpu(), lse.double().cpu()
            host, q = s.c.pages[1].cpu(), s.q.double().cpu()
            for r, b in ((0, 0), (1, 0), (2, 1), (3, 2), (42, 2)):
                held = paged.rows64(host, s.table[b], past[b] + new[b], 16, kvh, kd, vd, False)
                o, e, mass = paged.attend64_far(q[r], *held, past[b] + r - s.starts[b].item(),
                                                float(torch.tensor(scale, dtype=torch.float32)),
                                                None)
                tol, tol_lse = paged.attend_bounds(o, mass, torch.zeros_like(e), kd)
                assert ((out[r] - o).abs() <= tol).all(), (scale, kv, r)
                assert ((lse[r] - e).abs() <= tol_lse).all(), (scale, kv, r)


@pytest.mark.parametrize("kv", [102, 65536])
def test_sinks_that_are_not_finite(env, kv):
    """A sink of -inf is none, one of inf takes everything, a NaN is one; heads
    beside them are as without."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    s = Setup(env, GQA, 16, False, [100, 0], [2, 1], seed=24)
    c = wide_table(s)
    run = lambda sink: lib.attention(c, 1, s.q, s.starts, max_q=2, max_kv=kv, sink=sink,  # noqa: E731
                                     with_lse=True)
    plain, plain_lse = run(None)
    sink = torch.full((32,), float("-inf"), device=dev)
    out, lse = run(sink)
    assert torch.equal(out, plain) and torch.equal(lse, plain_lse)
    sink[3], sink[17] = float("inf"), float("nan")
    out, lse = run(sink)
    others = [h for h in range(32) if h not in (3, 17)]
    assert torch.equal(out[:, others], plain[:, others])
    assert torch.equal(lse[:, others], plain_lse[:, others])
    assert (out[:, 3] == 0).all() and (lse[:, 3] == float("inf")).all()
    assert out[:, 17].isnan().all() and lse[:, 17].isnan().all()
    assert lib.cache_status(c) == 0
