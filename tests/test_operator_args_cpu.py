"""Refusals of the paged cache, the attention over it and the scoring entries:
every argument that the host can check, through the C ABI, without a GPU (the
checks come before any launch)."""
import ctypes as C

import pytest

import common  # noqa: F401  (the binding's path)
import dsv4_gpu
from paged import page_layout

P = 1 << 20  # an aligned address that nothing dereferences
BF16, F32, E4M3, F16 = 2, 4, 7, 3


@pytest.fixture(scope="module")
def raw():
    return dsv4_gpu.GpuLib().lib


def cache(**kw):
    s = dsv4_gpu.DSV4GCache()
    base = dict(pages=P, ref=P, table=P, len=P, status=P, n_layers=2, n_pages=64, page_size=16,
                kv_heads=2, k_dim=128, v_dim=128, dtype=BF16, n_seqs=4, max_pages=8)
    for k, v in dict(base, **kw).items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kvh,k,v", [(1, 512, 0), (3, 256, 0), (8, 128, 128), (5, 64, 64),
                                     (2, 256, 256)])
@pytest.mark.parametrize("fp8", [False, True])
def test_page_bytes(raw, ps, kvh, k, v, fp8):
    c = cache(page_size=ps, kv_heads=kvh, k_dim=k, v_dim=v, dtype=E4M3 if fp8 else BF16)
    assert raw.dsv4g_cache_page_bytes(C.byref(c)) == page_layout(ps, kvh, k, v, fp8)[0]
    assert raw.dsv4g_cache_workspace_bytes(C.byref(c)) >= 3 * 64 * 4


BAD_SHAPES = [dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(k_dim=96, v_dim=96),
              dict(k_dim=512, v_dim=512), dict(k_dim=128, v_dim=64), dict(k_dim=128, v_dim=0),
              dict(k_dim=64, v_dim=0), dict(kv_heads=0), dict(n_layers=0), dict(n_pages=0),
              dict(n_pages=(1 << 20) + 1), dict(n_seqs=0), dict(max_pages=0), dict(dtype=F32),
              dict(dtype=F16), dict(max_pages=1 << 27)]


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_bad_shape(raw, bad):
    c = cache(**bad)
    assert raw.dsv4g_cache_page_bytes(C.byref(c)) == 0
    assert raw.dsv4g_cache_workspace_bytes(C.byref(c)) == 0
    assert raw.dsv4g_cache_init(C.byref(c), None) == 1
    assert b"cache shape" in raw.dsv4g_last_error()


@pytest.mark.parametrize("bad", [dict(pages=0), dict(ref=0), dict(table=0), dict(len=0),
                                 dict(status=0), dict(pages=P + 128)], ids=str)
def test_bad_pointer(raw, bad):
    c = cache(**bad)
    st = C.c_uint(0)
    assert raw.dsv4g_cache_init(C.byref(c), None) == 1
    assert raw.dsv4g_cache_status(C.byref(st), C.byref(c), None) == 1
    assert raw.dsv4g_cache_reserve(C.byref(c), P, P, 2, P, 1 << 20, None) == 1
    assert raw.dsv4g_cache_fork(C.byref(c), P, P, 2, None) == 1
    assert raw.dsv4g_cache_free(C.byref(c), P, P, 2, None) == 1
    assert raw.dsv4g_cache_compact(C.byref(c), P, P, 1 << 20, None) == 1


@pytest.mark.parametrize("seqs,starts,n,ws,size", [
    (P, None, 2, P, 1 << 20), (P, P, 0, P, 1 << 20), (P, P, 1025, P, 1 << 20),
    (P, P, 2, None, 1 << 20), (P, P, 2, P + 16, 1 << 20), (P, P, 2, P, 16)])
def test_reserve_refusals(raw, seqs, starts, n, ws, size):
    c = cache()
    assert raw.dsv4g_cache_reserve(C.byref(c), seqs, starts, n, ws, size, None) == 1


def test_list_refusals(raw):
    c = cache()
    for n in (0, -1, 1025):
        assert raw.dsv4g_cache_fork(C.byref(c), P, P, n, None) == 1
        assert raw.dsv4g_cache_free(C.byref(c), P, P, n, None) == 1
    assert raw.dsv4g_cache_fork(C.byref(c), None, P, 1, None) == 1
    assert raw.dsv4g_cache_fork(C.byref(c), P, None, 1, None) == 1
    assert raw.dsv4g_cache_status(None, C.byref(c), None) == 1
    for ws, size in ((None, 1 << 20), (P + 64, 1 << 20), (P, 64)):
        assert raw.dsv4g_cache_compact(C.byref(c), None, ws, size, None) == 1


GOOD_APPEND = dict(layer=0, k=P, ks=256, v=P, vs=256, dt=F32, seqs=P, starts=P, n=2, tokens=5)


@pytest.mark.parametrize("bad", [
    dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(dt=F16), dict(dt=E4M3),
    dict(starts=None), dict(n=0), dict(tokens=0), dict(ks=255), dict(ks=258), dict(vs=252),
    dict(k=P + 4), dict(v=P + 8), dict(dt=BF16, ks=260)], ids=str)
def test_append_refusals(raw, bad):
    a = dict(GOOD_APPEND, **bad)
    c = cache()
    assert raw.dsv4g_cache_append(C.byref(c), a["layer"], a["k"], a["ks"], a["v"], a["vs"],
                                  a["dt"], a["seqs"], a["starts"], a["n"], a["tokens"], None) == 1


def test_launches_too_large(raw):
    c = C.byref(cache())
    assert raw.dsv4g_cache_append(c, 0, P, 256, P, 256, F32, P, P, 2, 1 << 26, None) == 1
    assert b"2^26" in raw.dsv4g_last_error()
    for n, vocab in ((1 << 24, 8), (1, (1 << 30) + 1)):
        assert raw.dsv4g_logprobs(P, P, P, P, P, P, F32, vocab, n, vocab, P, 1, 1.0, P, 1 << 40,
                                  None) == 1
        assert b"2^24" in raw.dsv4g_last_error()
    # 2^24 items: as many (sequence, kv head) pairs
    a = GOOD_ATT
    assert raw.dsv4g_attention(P, a["os"], P, P, a["qs"], BF16, c, 1, 8, P, P, 1 << 23, 1 << 23,
                               1, 100, 0.1, 0, P, P, 1 << 40, None) == 1
    assert b"too many rows" in raw.dsv4g_last_error()


def test_append_values_of_a_latent_cache(raw):
    c = cache(k_dim=512, v_dim=0, kv_heads=1)
    a = GOOD_APPEND
    assert raw.dsv4g_cache_append(C.byref(c), 0, P, 512, P, 512, F32, P, P, 2, 5, None) == 1
    assert a["v"]


GOOD_ATT = dict(out=P, os=1024, lse=P, q=P, qs=1024, dt=BF16, layer=1, heads=8, seqs=P, starts=P,
                n=2, tokens=5, max_q=5, max_kv=100, scale=0.1, window=0, sink=P, ws=P,
                size=1 << 30)


@pytest.mark.parametrize("bad", [
    dict(out=None), dict(q=None), dict(starts=None), dict(n=0), dict(tokens=0), dict(layer=2),
    dict(layer=-1), dict(heads=0), dict(heads=7), dict(max_q=0), dict(max_kv=0), dict(window=-1),
    dict(dt=F16), dict(qs=1016), dict(os=1023), dict(qs=1028), dict(q=P + 8), dict(out=P + 2),
    dict(scale=float("nan")), dict(scale=float("inf"))], ids=str)
def test_attention_refusals(raw, bad):
    a = dict(GOOD_ATT, **bad)
    c = cache()
    assert raw.dsv4g_attention(a["out"], a["os"], a["lse"], a["q"], a["qs"], a["dt"], C.byref(c),
                               a["layer"], a["heads"], a["seqs"], a["starts"], a["n"],
                               a["tokens"], a["max_q"], a["max_kv"], a["scale"], a["window"],
                               a["sink"], a["ws"], a["size"], None) == 1


GOOD_SCORE = dict(lp=P, en=P, rank=P, ids=P, top=P, z=P, dt=F32, vocab=5000, n=3, stride=5000,
                  tokens=P, k=4, scale=1.0, ws=P, size=1 << 30)


@pytest.mark.parametrize("bad", [
    dict(z=None), dict(vocab=0), dict(n=0), dict(stride=4999), dict(k=-1), dict(k=65),
    dict(dt=F16), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(tokens=None), dict(tokens=None, lp=None), dict(z=P + 2),
    dict(ws=None), dict(ws=P + 8), dict(size=64)], ids=str)
def test_score_refusals(raw, bad):
    a = dict(GOOD_SCORE, **bad)
    assert raw.dsv4g_logprobs(a["lp"], a["en"], a["rank"], a["ids"], a["top"], a["z"], a["dt"],
                              a["vocab"], a["n"], a["stride"], a["tokens"], a["k"], a["scale"],
                              a["ws"], a["size"], None) == 1


def test_score_workspace(raw):
    need = raw.dsv4g_logprobs_workspace_bytes
    assert need(100, 1, 64) == 0            # one segment
    assert need(129280, 1, 20) > 0
    assert need(129280, 1, 0) < need(129280, 1, 20)
    assert need(129280, 4096, 20) == 0      # enough rows for the chip
    assert need(0, 1, 0) == need(1, 0, 0) == need(10, 1, 65) == 0


def test_wrapper_refusals():
    """The binding's own checks, on CPU tensors (which no entry takes)."""
    import torch
    lib = dsv4_gpu.lib()
    z = torch.zeros(2, 10)
    with pytest.raises(ValueError, match="one GPU"):
        lib.logprobs(z, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="contiguous rows"):
        lib.logprobs(z.t(), None)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="dtype"):
        dsv4_gpu.PagedCache(torch.zeros(1, 2, 256, dtype=torch.uint8), i(2), i(1, 2), i(1), i(1),
                            16, 1, 64, 64, "fp16")
    with pytest.raises(ValueError, match="uint8"):
        dsv4_gpu.PagedCache(torch.zeros(1, 2, 256), i(2), i(1, 2), i(1), i(1), 16, 1, 64, 64)
    with pytest.raises(ValueError, match="one GPU"):
        dsv4_gpu.PagedCache(torch.zeros(1, 2, 256, dtype=torch.uint8), i(2), i(1, 2), i(1), i(1),
                            16, 1, 64, 64)
    with pytest.raises(ValueError, match="not a cache shape"):
        dsv4_gpu.PagedCache.new(1, 4, 17, 1, 64, 64, 1, 2, device="cpu")


def test_scales_beyond_fp32_in_base_2(raw):
    """A scale whose product with log2 e is no fp32 number is refused; the
    largest that is one passes this check (and fails the next, its workspace)."""
    c, a = C.byref(cache(max_pages=4096)), GOOD_ATT
    top = 3.4028234663852886e38 / 1.4426950408889634
    for scale, why in ((top * 1.001, b"scale"), (-3.4e38, b"scale"), (top * 0.999, b"workspace"),
                       (-top * 0.999, b"workspace")):
        assert raw.dsv4g_attention(P, a["os"], P, P, a["qs"], BF16, c, 1, 8, P, P, 2, 5, 5, 8192,
                                   scale, 0, P, P, 0, None) == 1
        assert why in raw.dsv4g_last_error(), scale


def test_no_descriptor(raw):
    """NULL in place of the descriptor: no size, and a refusal."""
    assert raw.dsv4g_cache_page_bytes(None) == 0
    assert raw.dsv4g_cache_workspace_bytes(None) == 0
    assert raw.dsv4g_attention_workspace_bytes(None, 8, 2, 5, 5, 100) == 0
    a = GOOD_ATT
    for rc in (raw.dsv4g_cache_init(None, None), raw.dsv4g_cache_fork(None, P, P, 1, None),
               raw.dsv4g_cache_reserve(None, P, P, 2, P, 1 << 20, None),
               raw.dsv4g_cache_append(None, 0, P, 256, P, 256, F32, P, P, 2, 5, None),
               raw.dsv4g_cache_free(None, P, P, 2, None),
               raw.dsv4g_cache_compact(None, P, P, 1 << 20, None),
               raw.dsv4g_cache_status(P, None, None),
               raw.dsv4g_attention(P, a["os"], P, P, a["qs"], BF16, None, 1, 8, P, P, 2, 5, 5, 100,
                                   0.1, 0, P, P, 1 << 30, None)):
        assert rc == 1 and b"cache shape" in raw.dsv4g_last_error()


def test_sizes_beyond_every_launch(raw):
    """Products of sizes that pass 64 bits are refused as too many rows, and
    take no workspace; the same for lists that no counter of the device holds."""
    c, a = C.byref(cache(kv_heads=1024, k_dim=64, v_dim=64)), GOOD_ATT
    for heads, n_seqs, tokens in ((1024, 1 << 30, 0x7FFFFF00), (1024, 1 << 29, 0x7FFFFF00),
                                  (1024, 2**31 - 1, 1), (1 << 30, 1, 2**31 - 1),
                                  (1 << 30, 2**31 - 1, 2**31 - 1)):
        assert raw.dsv4g_attention_workspace_bytes(c, heads, n_seqs, tokens, tokens, 128) == 0
        assert raw.dsv4g_attention(P, heads * 64, P, P, heads * 64, BF16, c, 1, heads, P, P,
                                   n_seqs, tokens, tokens, 128, 0.1, 0, P, P, 1 << 62, None) == 1
        assert b"too many rows" in raw.dsv4g_last_error(), (heads, n_seqs, tokens)
    c = C.byref(cache())
    for n in (1 << 26, 2**31 - 1):
        assert raw.dsv4g_cache_append(c, 0, P, 256, P, 256, F32, P, P, n, 5, None) == 1
        assert b"2^26" in raw.dsv4g_last_error()
