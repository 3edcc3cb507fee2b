"""dsv4g_logprobs against its definition in 64 bits: ranks and ids exact (the
order is that of the fp32 products scale * logit), log probabilities within
fp32 rounding. Bounds: a sum of e^(z - m) in fp32 over at most 2^18 terms, each
within 2^-21 (the argument of e^x rounded, |z - m| < 2^5 where it counts, and
the hardware's exponential), joined pairwise: log s within 2^-20, doubled twice
over; z - m and the difference to log s round once each (2^-24 of themselves).
The entropy's second sum has terms at most 2^5 times as large."""
import numpy as np
import pytest

import common  # noqa: F401  (the path of the binding)
from paged import score64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import dsv4_gpu
    return dict(torch=torch, lib=dsv4_gpu.lib(), dev=torch.device("cuda:0"))


def check(env, z, tokens, k, scale, rows=None):
    """z: device tensor [n][vocab]."""
    torch, lib = env["torch"], env["lib"]
    tok = None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device=env["dev"])
    got = lib.logprobs(z, tok, top=k, scale=scale)
    got = [None if g is None else g.cpu().numpy() for g in got]
    host = (z.float().cpu().numpy() * np.float32(scale)).astype(np.float64)
    for r in (range(z.shape[0]) if rows is None else rows):
        lp, en, rank, ids, top = score64(host[r], -1 if tokens is None else tokens[r], k)

        def near(a, b, more=1.0):
            assert (np.isnan(a) and np.isnan(b)) or a == b or \
                abs(a - b) <= more * (2.0 ** -18 + 2.0 ** -21 * abs(b)), (r, a, b)
        near(got[1][r], en, 32.0)
        if tokens is not None:
            near(got[0][r], lp)
            assert got[2][r] == rank, r
        if k:
            assert got[3][r].tolist() == ids, r
            for a, b in zip(got[4][r], top):
                near(a, b)


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 1000, 4095, 4096, 4097, 8193, 50257,
                                   129280])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_sizes(env, vocab, kind):
    torch = env["torch"]
    g = torch.Generator(device=env["dev"]).manual_seed(vocab)
    for n, k, scale in ((1, 20, 1.0), (3, 64, 0.7), (5, 1, 1.0), (2, 0, 3.0)):
        z = (torch.randn(n, vocab, generator=g, device=env["dev"]) * 3).to(getattr(torch, kind))
        tokens = torch.randint(0, vocab, (n,), generator=g, device=env["dev"]).tolist()
        check(env, z, tokens, k, scale)


@pytest.mark.parametrize("n", [1, 7])
def test_orders_and_ties(env, n):
    """Ascending, descending, all equal, few distinct values, -0 and 0."""
    torch, dev = env["torch"], env["dev"]
    v = 20000
    up = torch.arange(v, device=dev, dtype=torch.float32) / 512
    g = torch.Generator(device=dev).manual_seed(5)
    few = torch.randint(0, 7, (v,), generator=g, device=dev).float()
    zeros = torch.where(torch.arange(v, device=dev) % 3 == 0, -0.0, 0.0)
    late = torch.zeros(v, device=dev)
    late[-70:] = 1
    for row in (up, up.flip(0), torch.full((v,), 2.5, device=dev), few, zeros, late):
        z = row.repeat(n, 1)
        check(env, z, [0, v - 1, 77, 5000, 4096, 4095, 19999][:n], 20, 1.0, rows=[0, n - 1])
        check(env, z, [13] * n, 64, 1.0, rows=[0])


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_equal_values_around_the_token(env, kind):
    """Ranks of tokens whose value also stands in the tiles before and behind
    theirs: zeros of both signs, the values next to them, infinities, the
    type's lowest value; whole rows per workgroup and rows in segments."""
    torch, dev = env["torch"], env["dev"]
    t = getattr(torch, kind)
    info = torch.finfo(t)
    tiny = torch.nextafter(torch.zeros((), dtype=t), torch.ones((), dtype=t)).item()
    some = torch.tensor([0.0, -0.0, tiny, -tiny, 1.0, -1.0, info.min, float("-inf")], dtype=t,
                        device=dev)
    v = 3 * 4096 + 5
    g = torch.Generator(device=dev).manual_seed(12)
    for n in (2050, 3):
        z = some[torch.randint(0, 8, (n, v), generator=g, device=dev)]
        tokens = [(4096 * (r % 4) + [0, 4, 4095, -1][r // 4 % 4]) % v for r in range(n)]
        # every value in turn at the token's place
        z[torch.arange(n, device=dev), torch.tensor(tokens, device=dev)] = \
            some[torch.arange(n, device=dev) % 8]
        check(env, z, tokens, 3, 1.0, rows=[r for r in range(0, 64) if r < n])


def test_banned_and_bad_values(env):
    torch, dev = env["torch"], env["dev"]
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device=dev).manual_seed(6)
    z = torch.randn(9, 9001, generator=g, device=dev)
    z[0, 10:] = -inf           # fewer than k that can be taken
    z[1, :] = -inf             # none
    z[2, 4500] = inf
    z[3, 17] = nan
    z[4, 1:] = -inf            # one
    z[5, :8192] = -inf         # whole tiles of a segment
    z[6, :] = torch.finfo(torch.float32).min  # a mask of the type's lowest value, everywhere
    z[7, 100:] = torch.finfo(torch.float32).min
    z[8, :] = nan
    for tokens in ([3, 5, 4500, 17, 0, 8999, 9, 3, 0], [20, 0, 0, 0, 5, 4, 9000, 200, 9000],
                   [-1, 9001, 2 ** 31 - 1, -2 ** 31, 9001, -1, -7, 9001, 9001]):
        for k in (0, 5, 40):
            check(env, z, tokens, k, 1.0)
    check(env, z, None, 3, 0.5)
    check(env, z[:, :37], [3, 5, 6, 17, 0, 30, 9, 3, 0], 64, 1.0)  # k above vocab


def test_views(env):
    """Rows of a wider buffer that start at any element."""
    torch, dev = env["torch"], env["dev"]
    g = torch.Generator(device=dev).manual_seed(7)
    for kind in (torch.float32, torch.bfloat16):
        buf = torch.randn(4, 10007, generator=g, device=dev).to(kind)
        for at, v in ((1, 10001), (3, 4096), (5, 9973)):
            check(env, buf[:, at:at + v], [0, 1, v - 1, 55], 8, 1.25)


def test_many_rows(env):
    torch, dev = env["torch"], env["dev"]
    g = torch.Generator(device=dev).manual_seed(8)
    z = torch.randn(2500, 1333, generator=g, device=dev) * 4
    tokens = torch.randint(0, 1333, (2500,), generator=g, device=dev).tolist()
    check(env, z, tokens, 10, 1.0, rows=range(0, 2500, 83))


def test_beside_argmax(env):
    """The first alternative is the greedy pick, and its rank 0."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    g = torch.Generator(device=dev).manual_seed(9)
    z = (torch.randn(33, 129280, generator=g, device=dev) * 2).to(torch.bfloat16).float()
    pick = lib.argmax(z)
    lp, _, rank, ids, top = lib.logprobs(z, pick, top=3)
    assert (rank == 0).all() and torch.equal(ids[:, 0], pick) and torch.equal(top[:, 0], lp)


def test_graph_and_streams(env):
    """Captured, and replayed on new logits with eager work between; two calls
    at once on two streams, each with its own workspace."""
    torch, lib, dev = env["torch"], env["lib"], env["dev"]
    g = torch.Generator(device=dev).manual_seed(10)
    z = torch.randn(2, 129280, generator=g, device=dev)
    tok = torch.tensor([5, 77], dtype=torch.int32, device=dev)
    ws = [torch.empty(lib.logprobs_workspace_bytes(129280, 2, 20), dtype=torch.uint8, device=dev)
          for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lib.logprobs(z, tok, top=20, workspace=ws[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lib.logprobs(z, tok, top=20, workspace=ws[0])
    for _ in range(4):
        z.copy_(torch.randn(2, 129280, generator=g, device=dev) * 3)
        graph.replay()
        torch.cuda.synchronize()
        want = lib.logprobs(z, tok, top=20, workspace=ws[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    other = torch.randn(3, 100000, generator=g, device=dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = lib.logprobs(other, None, top=4)
    b = lib.logprobs(z, tok, top=20)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(b, want))
    assert all(torch.equal(x, y) for x, y in zip(a[3:], lib.logprobs(other, None, top=4)[3:]))


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [3, 2050], ids=["segments", "whole rows"])
def test_values_of_any_size(env, kind, n):
    """Masks of every size beside ordinary logits, rows of nothing but masks (of
    one size, of two), largest values up to the end of fp32's range: a value
    is as far from the largest as its difference says."""
    torch, dev = env["torch"], env["dev"]
    t = getattr(torch, kind)
    v, low = 9001, torch.finfo(t).min
    g = torch.Generator(device=dev).manual_seed(13)
    some = torch.randn(v, generator=g, device=dev) * 3
    first = torch.arange(v, device=dev) < 4500   # whole segments and places of a thread
    third = torch.arange(v, device=dev) % 3 == 0
    one = torch.arange(v, device=dev) == 8000
    rows = []
    for m in (-1e4, -1e6, -1e9, -1e10, -3e10, -1e20, -1e30, -1e37, -1e38, -3e38, low):
        rows += [torch.where(first, m, some), torch.where(third, some, m),
                 torch.where(one, some, m), torch.full_like(some, m),
                 torch.where(third, m, low), torch.where(one, m, 3 * m if m > -1e38 else low)]
    for m in (1e6, 1.7e7, 1e9, 1e10, 1e30, 2.3e38, 3e38):
        rows += [torch.where(one, m, some), torch.full_like(some, m), torch.where(third, m, -m),
                 torch.where(third, m, 0.999 * m), some + m]
    # fp32 and BF16 steps around one large value
    rows += [torch.where(third, 4e9, 4e9 - 256), torch.where(first, 1.7e7, 1.7e7 - 1)]
    rows = torch.stack(rows).to(t)
    tokens = [(0, 8000, 4501, 3, 9000)[i % 5] for i in range(len(rows))]
    for i in range(0, len(rows), n):
        z, tok = rows[i:i + n], tokens[i:i + n]
        more = n - len(z) if n > len(rows) else 0   # fill the call with copies
        check(env, torch.cat([z, z[:1].expand(more, v)]), tok + tok[:1] * more, 5, 1.0,
              rows=range(len(z)))
    check(env, rows[:n], tokens[:n], 0, 0.7)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [3, 2050], ids=["segments", "whole rows"])
def test_products_that_vanish(env, kind, n):
    """Logits whose products with the scale round to zero, of either sign: they
    are equal, and go by their index."""
    torch, dev = env["torch"], env["dev"]
    t = getattr(torch, kind)
    tiny = torch.nextafter(torch.zeros((), dtype=t), torch.ones((), dtype=t)).item()
    some = torch.tensor([0.0, -0.0, tiny, -tiny, 3 * tiny, -3 * tiny], dtype=t, device=dev)
    v = 2 * 4096 + 77
    g = torch.Generator(device=dev).manual_seed(14)
    # 2^-151, 0.75 2^-149 and the like: zero, and one last place of the least number
    for scale in ((0.25, 0.75, 0.4) if kind == "float32" else (2.0 ** -18, 0.75 * 2.0 ** -16)):
        z = some[torch.randint(0, 6, (n, v), generator=g, device=dev)]
        z[1] = -tiny
        z[1, 100:] = -0.0
        z[2] = -tiny
        tokens = [(4096 * (r % 3) + [0, 50, 4000, 76][r // 3 % 4]) % v for r in range(n)]
        z[torch.arange(n, device=dev), torch.tensor(tokens, device=dev)] = \
            some[torch.arange(n, device=dev) % 6]
        check(env, z, tokens, 20, scale, rows=[r for r in range(36) if r < n])
