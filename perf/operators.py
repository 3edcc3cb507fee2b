"""The measured work of the attention half's cache, the attention over it, and
the scoring of given tokens: what an engine that serves several sequences has
the library do between a layer's projections and after its vocabulary head.

Kinds of case (one field "kind"):

  attend     dsv4g_attention: a chunk of new tokens per sequence (one at
             decode, a few of a draft, a prompt's chunk) over the paged cache
             that already holds them
  append     dsv4g_cache_append: the new tokens' rows into the cache's pages
  branch     dsv4g_cache_fork, _reserve, _free: sequences forked (pages
             shared), the children extended by a draft (shared pages that the
             draft writes into are copied) and cut back to what was accepted
  compact    dsv4g_cache_compact: the live pages moved to the front of the pool
  score      dsv4g_logprobs: log probabilities of given tokens, with entropy,
             rank and the top alternatives

A page holds page_size tokens of one layer: [kv_heads][page_size][k_dim] keys,
then the values likewise (v_dim 0: the values are the keys, one latent row per
token), BF16, or E4M3 codes followed by one E8M0 scale code per 64 columns.
Scores are scale * q.k in base e; a token sees the cache up to itself (and no
further back than the window), a head's sink joins the sum of its softmax.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

GROUP = 64                 # columns per E8M0 scale of an 8-bit page
VOCAB = 129280
# heads, kv heads, key width, value width (0: the values are the keys): the
# latent attention behind the projections (wq_b 32768 = 64 x 512 rows, wkv 512),
# a quarter of its heads (as sharded over GPUs), and grouped heads
LATENT, SHARD = (64, 1, 512, 0), (16, 1, 512, 0)
GQA, SMALL, ODD, WIDE = (32, 8, 128, 128), (8, 8, 64, 64), (40, 8, 128, 128), (16, 2, 256, 256)


def _layout(shape):
    return dict(zip(("heads", "kv_heads", "k_dim", "v_dim"), shape))


def listed():
    return [
        # plain decode of one sequence, some way into an answer: latency
        {"name": "attend_decode_1", "kind": "attend", "seqs": 1, "q": 1, "q_min": 1,
         "past": 1777, "past_min": 1777, "window": 0, "sink": False, "fp8": False, "page": 64,
         **_layout(LATENT)},
        # a serving batch at decode, contexts of every length, 8-bit cache
        {"name": "attend_decode_64_fp8", "kind": "attend", "seqs": 64, "q": 1, "q_min": 1,
         "past": 8100, "past_min": 130, "window": 0, "sink": True, "fp8": True, "page": 64,
         **_layout(LATENT)},
        # speculative verify: drafts of five over grouped heads
        {"name": "attend_verify_8x5", "kind": "attend", "seqs": 8, "q": 5, "q_min": 5,
         "past": 16000, "past_min": 900, "window": 0, "sink": False, "fp8": False, "page": 16,
         **_layout(GQA)},
        # prompts of ragged length within the sliding window
        {"name": "attend_window_3x777", "kind": "attend", "seqs": 3, "q": 777, "q_min": 150,
         "past": 300, "past_min": 1, "window": 128, "sink": True, "fp8": False, "page": 32,
         **_layout(LATENT)},
        # a chunk of a long prompt, behind 14k tokens
        {"name": "attend_chunk_2048", "kind": "attend", "seqs": 1, "q": 2048, "q_min": 2048,
         "past": 14336, "past_min": 14336, "window": 0, "sink": False, "fp8": False, "page": 64,
         **_layout(LATENT)},
        # one decode step's rows, 8-bit
        {"name": "append_decode_64_fp8", "kind": "append", "seqs": 64, "q": 1, "q_min": 1,
         "past": 70, "past_min": 1, "fp8": True, "f32": True, "page": 64, **_layout(LATENT)},
        # the largest prefill chunk, several prompts packed
        {"name": "append_prefill_4096", "kind": "append", "seqs": 5, "q": 1500, "q_min": 400,
         "past": 40, "past_min": 1, "fp8": False, "f32": True, "page": 16, **_layout(GQA)},
        # tree drafts: every sequence branched, extended by five, cut back
        {"name": "branch_16x5", "kind": "branch", "seqs": 16, "past": 1900, "past_min": 100,
         "draft": 5, "layers": 43, "pages": 512, "fp8": True, "page": 64, **_layout(LATENT)},
        # a pool after many sequences have ended, every layer's pages moved
        {"name": "compact_2048", "kind": "compact", "seqs": 40, "past": 3000, "past_min": 60,
         "layers": 16, "pages": 2048, "fp8": False, "page": 32, **_layout((8, 1, 512, 0))},
        # the sampled token of one sequence, with alternatives: latency
        {"name": "score_1_top20", "kind": "score", "rows": 1, "vocab": VOCAB, "top": 20,
         "bf16": False, "banned": 0},
        # a verify batch under a grammar that bans most tokens
        {"name": "score_64", "kind": "score", "rows": 64, "vocab": VOCAB, "top": 0,
         "bf16": False, "banned": 90000},
        # a prompt chunk scored, with alternatives, narrow logits
        {"name": "score_2048_bf16_top8", "kind": "score", "rows": 2048, "vocab": VOCAB, "top": 8,
         "bf16": True, "banned": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """Scores of the padded batch (what the plain form holds) and its cache."""
    most = c["past"] + c["q"]
    return (c["seqs"] * c["q"] * c["heads"] * most,
            c["seqs"] * most * c["kv_heads"] * (c["k_dim"] + c["v_dim"]))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "append", "branch", "compact", "score",
                       "score"))
    if kind == "score":
        vocab = rng.choice((VOCAB, _log(rng, 500, 200000)))
        return {"kind": kind, "rows": min(_log(rng, 1, 2048), 264000000 // vocab),
                "vocab": vocab, "top": rng.choice((0, 1, 5, 20, rng.randint(2, 64))),
                "bf16": rng.random() < 0.4,
                "banned": int(vocab * rng.choice((0, 0, 0.1, 0.9)))}
    lay = _layout(rng.choice((LATENT, LATENT, SHARD, GQA, SMALL, ODD, WIDE)))
    fp8, page = rng.random() < 0.5, rng.choice((16, 32, 64, 128, 256))
    if kind == "attend":
        while True:
            mode = rng.choice(("decode", "draft", "chunk"))
            q = 1 if mode == "decode" else rng.randint(2, 16) if mode == "draft" \
                else _log(rng, 17, 2048)
            past = _log(rng, 1, 16000)
            c = {"kind": kind, "seqs": _log(rng, 1, 64), "q": q,
                 "q_min": rng.choice((q, max(1, q // 3), 0)), "past": past,
                 "past_min": rng.choice((past, max(1, past // 10), 0)),
                 "window": rng.choice((0, 0, 128, _log(rng, 1, 4000))),
                 "sink": rng.random() < 0.4, "fp8": fp8, "page": page, **lay}
            scores, cache = _cost(c)
            if scores <= 2000000000 and cache <= 2000000000 \
                    and work(c)["flops"] <= 4.0e12:
                return c
    if kind == "append":
        q = rng.choice((1, rng.randint(2, 16), _log(rng, 17, 3000)))
        seqs = min(_log(rng, 1, 128), max(1, 9000 // q))
        past = _log(rng, 1, 600)
        return {"kind": kind, "seqs": seqs, "q": q, "q_min": rng.choice((q, 0)),
                "past": past, "past_min": rng.choice((past, 0)), "fp8": fp8,
                "f32": rng.random() < 0.6, "page": page, **lay}
    lay = _layout(rng.choice((LATENT, (8, 1, 128, 128), (8, 2, 64, 64))))
    c = {"kind": kind, "fp8": fp8, "page": page, **lay, "layers": rng.randint(1, 43)}
    most = 700000000 // (c["layers"] * _page_bytes(c))
    if kind == "branch":
        past = _log(rng, 20, 3000)
        c.update(past=past, past_min=rng.choice((past, max(1, past // 20))),
                 draft=rng.randint(1, 40))
        each = -(-past // page) + -(-c["draft"] // page) + 2
        c["seqs"] = min(_log(rng, 1, 64), max(1, (most - 1) // each))
        c["pages"] = max(each * c["seqs"], min(most, _log(rng, 64, 8192)))
        return c
    c["pages"] = max(16, min(most, _log(rng, 64, 16384)))
    past = min(_log(rng, 20, 4000), page * (c["pages"] // 4))
    c.update(past=past, past_min=rng.choice((past, max(1, past // 20))))
    c["seqs"] = min(_log(rng, 1, 200), max(1, c["pages"] * 2 // (3 * -(-past // page))))
    return c


# ---------------------------------------------------------------- sizes

def _page_bytes(c):
    row = c["kv_heads"] * (c["k_dim"] + c["v_dim"])
    used = c["page"] * (row + row // GROUP if c["fp8"] else 2 * row)
    return (used + 255) // 256 * 256


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly over their logarithm."""
    if n == 1:
        return [hi]
    return [min(hi, max(lo, round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1))) - 1))
            for i in range(n)]


def _lengths(c):
    """(tokens before the new ones, new tokens) of each sequence."""
    past = _spread(c["seqs"], c["past_min"], c["past"])
    if "q" not in c:
        return past, [c.get("draft", 0)] * c["seqs"]
    new = _spread(c["seqs"], c["q_min"], c["q"])
    half = len(new) // 2  # long chunks behind middling contexts
    return past, new[half:] + new[:half]


def _seen(past, new, window):
    """Pairs (new token, token it sees) of one sequence."""
    total = 0
    full = new if not window else max(0, min(new, window - past))
    total += full * past + full * (full + 1) // 2
    return total + (new - full) * window


def work(case):
    c, kind = case, case["kind"]
    if kind == "score":
        size, n = 2 if c["bf16"] else 4, c["rows"]
        return {"bytes": n * (c["vocab"] * size + 16 + 8 * c["top"]),
                "flops": 6 * n * c["vocab"]}
    row = c["kv_heads"] * (c["k_dim"] + c["v_dim"])
    row_bytes = row + row // GROUP if c["fp8"] else 2 * row
    past, new = _lengths(c)
    if kind == "append":
        return {"bytes": sum(new) * (row * (4 if c["f32"] else 2) + row_bytes),
                "flops": 4 * sum(new) * row}
    if kind == "attend":
        v_dim = c["v_dim"] or c["k_dim"]
        pairs = sum(_seen(p, n, c["window"]) for p, n in zip(past, new))
        cached = sum(p + n if not c["window"] else min(p + n, c["window"] + n - 1)
                     for p, n in zip(past, new) if n)
        io = sum(new) * c["heads"] * (2 * c["k_dim"] + 2 * v_dim + 4)
        return {"bytes": cached * row_bytes + io,
                "flops": 2 * pairs * c["heads"] * (c["k_dim"] + v_dim)}
    page_bytes, table = _page_bytes(c), -(-(c["past"] + c.get("draft", 0)) // c["page"])
    if kind == "branch":
        copies = sum(1 for p in past if p % c["page"])
        return {"bytes": 2 * copies * c["layers"] * page_bytes + 4 * c["pages"]
                + 16 * c["seqs"] * table, "flops": 4 * c["seqs"] * table}
    # live pages are scattered evenly: a share of them sits behind the first live ones
    live = sum(-(-p // c["page"]) for p in past)
    moved = live * (c["pages"] - live) // c["pages"]
    return {"bytes": 2 * moved * c["layers"] * page_bytes + 8 * c["pages"]
            + 8 * c["seqs"] * table, "flops": 2 * c["pages"]}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(c, g, layers):
    """Pages of every layer as earlier sequences left them: rows of N(0, 1)
    in the page's own format, those that hold no token now too."""
    n, page_bytes = c["pages"], _page_bytes(c)
    row = c["page"] * c["kv_heads"] * (c["k_dim"] + c["v_dim"])
    pages = torch.zeros(layers, n, page_bytes, dtype=torch.uint8, device="cuda")
    vals = torch.randn(layers, n, row, generator=g, device="cuda", dtype=torch.bfloat16)
    if c["fp8"]:
        pages[..., :row] = (vals * 80).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        pages[..., row:row + row // GROUP] = torch.randint(
            119, 122, (layers, n, row // GROUP), generator=g, device="cuda",
            dtype=torch.uint8)
    else:
        pages[..., :2 * row] = vals.view(torch.uint8)
    return pages


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": dict(case)}
    if c["kind"] == "score":
        # a trained head's logits: a few tokens far above the rest
        z = torch.randn(c["rows"], c["vocab"], generator=g, device="cuda") * 2.5
        if c["banned"]:
            z[:, torch.randperm(c["vocab"], generator=g, device="cuda")[:c["banned"]]] = -math.inf
        s["logits"] = z.to(torch.bfloat16) if c["bf16"] else z
        # tokens that were sampled: Gumbel noise on the logits
        noise = torch.rand(c["rows"], c["vocab"], generator=g, device="cuda").clamp_(1e-20)
        s["tokens"] = (z - noise.log_().neg_().log_()).argmax(1).to(torch.int32)
        return s
    past, new = _lengths(c)
    n, page = c["seqs"], c["page"]
    total = [p + k for p, k in zip(past, new)]
    if c["kind"] in ("attend", "append"):
        held, layers = total, 2
        c = dict(c, pages=sum(-(-t // page) for t in total) + 7)
        rows, cols = n, max(1, -(-max(total) // page))
    else:
        held, layers = past, c["layers"]
        rows = 2 * n if c["kind"] == "branch" else n
        cols = -(-max(total) // page)
    s["pages"] = _pool(c, g, layers)
    # one buffer for the bookkeeping: users of each page, the sequences' page
    # tables and lengths, the status word
    book = torch.zeros(c["pages"] + rows * cols + rows + 1, dtype=torch.int32, device="cuda")
    s["ref"], table, s["len"], s["status"] = book.split([c["pages"], rows * cols, rows, 1])
    s["table"] = table.view(rows, cols)
    s["table"].fill_(-1)
    counts = _ints([-(-t // page) for t in held])
    mine = torch.arange(cols, device="cuda")[None] < counts[:, None]
    used = int(sum(-(-t // page) for t in held))
    some = torch.randperm(c["pages"], generator=g, device="cuda")[:used].to(torch.int32)
    s["table"][:n][mine] = some
    s["ref"][some.long()] = 1
    s["len"][:n] = _ints(held)
    s["book"], s["book0"] = book, book.clone()
    s["starts"] = _ints([sum(new[:i]) for i in range(n + 1)])
    tokens = sum(new)
    if c["kind"] == "attend":
        # queries that pick some tokens out: scores of standard deviation 2
        s["q"] = (2 * torch.randn(tokens, c["heads"], c["k_dim"], generator=g,
                                  device="cuda")).to(torch.bfloat16)
        s["sink"] = torch.randn(c["heads"], generator=g, device="cuda") if c["sink"] else None
        s["seqs"] = torch.arange(n, dtype=torch.int32, device="cuda")
    elif c["kind"] == "append":
        kind = torch.float32 if c["f32"] else torch.bfloat16
        for name, width in (("k", c["k_dim"]), ("v", c["v_dim"])):
            s[name] = torch.randn(tokens, c["kv_heads"], width, generator=g,
                                  device="cuda").to(kind) if width else None
        s["seqs"] = torch.arange(n, dtype=torch.int32, device="cuda")
    elif c["kind"] == "branch":
        s["parents"] = torch.arange(n, dtype=torch.int32, device="cuda")
        s["children"] = s["parents"] + n
        took = torch.randint(0, c["draft"] + 1, (n,), generator=g, device="cuda")
        s["kept"] = (_ints(past) + took).to(torch.int32)
    return s


# ---------------------------------------------------- the framework's calls

def _cache(s):
    """The cache's handle over the state's tensors, as a program keeps it."""
    if "cache" not in s:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(
            __file__))), "deepseek-v4-flash-0731-in-c_amd", "python"))
        import dsv4_gpu
        s["lib"] = dsv4_gpu.lib()
        c = s["case"]
        s["cache"] = None if c["kind"] == "score" else dsv4_gpu.PagedCache(
            s["pages"], s["ref"], s["table"], s["len"], s["status"], c["page"], c["kv_heads"],
            c["k_dim"], c["v_dim"], "fp8" if c["fp8"] else "bf16")
        s["ws"] = None
        if c["kind"] == "attend":
            s["ws"] = torch.empty(max(1, s["lib"].attention_workspace_bytes(
                s["cache"], c["heads"], c["seqs"], s["q"].shape[0], c["q"],
                c["past"] + c["q"])), dtype=torch.uint8, device="cuda")
        elif c["kind"] in ("branch", "compact"):
            s["ws"] = torch.empty(s["lib"].cache_workspace_bytes(s["cache"]), dtype=torch.uint8,
                                  device="cuda")
        elif c["kind"] == "score":
            s["ws"] = torch.empty(max(1, s["lib"].logprobs_workspace_bytes(
                c["vocab"], c["rows"], c["top"])), dtype=torch.uint8, device="cuda")
    return s["lib"], s["cache"]


def _run_own(s):
    lib, cache = _cache(s)
    c = s["case"]
    if c["kind"] == "attend":
        out, lse = lib.attention(cache, 1, s["q"], s["starts"], s["seqs"], max_q=c["q"],
                                 max_kv=c["past"] + c["q"], window=c["window"], sink=s["sink"],
                                 with_lse=True, workspace=s["ws"])
        return {"out": out, "lse": lse}
    if c["kind"] == "append":
        lib.cache_append(cache, 1, s["k"], s["v"], s["starts"], s["seqs"])
        return _held(s)
    if c["kind"] == "branch":
        s["book"].copy_(s["book0"])
        lib.cache_fork(cache, s["parents"], s["children"])
        lib.cache_reserve(cache, s["starts"], s["children"], workspace=s["ws"])
        lib.cache_free(cache, s["children"], s["kept"])
        return _state(s)
    if c["kind"] == "compact":
        s["book"].copy_(s["book0"])
        lib.cache_compact(cache, workspace=s["ws"])
        return _state(s)
    logprob, entropy, rank, ids, top = lib.logprobs(s["logits"], s["tokens"], top=c["top"],
                                                    scale=1 / 0.8, workspace=s["ws"])
    return {"logprob": logprob, "entropy": entropy, "rank": rank, "ids": ids, "top": top}


# ------------------------------------------------------------- plain forms

def _parts(c, pages):
    """Views of pages [..., page_bytes]: keys, values, their scale codes, each
    [..., kv_heads, page, width] (None where there is none)."""
    page, h = c["page"], c["kv_heads"]
    size, at, got = 1 if c["fp8"] else 2, 0, []
    for width, dtype, bytes_ in ((c["k_dim"], None, size), (c["v_dim"], None, size),
                                 (c["k_dim"] // GROUP, torch.uint8, 1),
                                 (c["v_dim"] // GROUP, torch.uint8, 1)):
        n = h * page * width * bytes_
        if not n or (dtype is not None and not c["fp8"]):
            got.append(None)
            continue
        part = pages[..., at:at + n]
        part = part.view(dtype or (torch.float8_e4m3fn if c["fp8"] else torch.bfloat16))
        got.append(part.unflatten(-1, (h, page, width)))
        at += n
    return got


def _held(s):
    """The layer's keys and values as the pages hold them (8-bit: the codes'
    values, and the scales' exponents)."""
    return dict(zip(("k", "v", "k_exp", "v_exp"), _parts(s["case"], s["pages"][1])))


def _state(s):
    return {"ref": s["ref"], "table": s["table"], "len": s["len"], "status": s["status"],
            "pages": s["pages"].view(torch.int32)}


def _rows(s, layer, dtype):
    """Keys and values of every table entry: [seqs, kv_heads, tokens, width]."""
    c = s["case"]
    k, v, ks, vs = _parts(c, s["pages"][layer][s["table"].clamp(min=0).long()])

    def wide(x, codes):
        x = x.to(dtype)
        if codes is not None:
            scale = torch.exp2(codes.to(dtype) - 127)
            x = (x.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)
        return x.transpose(1, 2).flatten(2, 3).contiguous()

    k = wide(k, ks)
    return k, (k if v is None else wide(v, vs))


def _attend_plain(s):
    c = s["case"]
    heads, kvh, dim = c["heads"], c["kv_heads"], c["k_dim"]
    g, n, most = heads // kvh, c["seqs"], c["q"]
    k, v = _rows(s, 1, torch.float32)
    length, starts = s["len"].long(), s["starts"].long()
    count = starts[1:] - starts[:-1]
    step = torch.arange(most, device="cuda")
    at = (starts[:-1, None] + step).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().view(n, most, kvh, g, dim).transpose(1, 2).reshape(n, kvh, most * g,
                                                                              dim)
    z = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(dim)).view(n, kvh, most, g, -1)
    pos = (length - count)[:, None] + step
    token = torch.arange(k.shape[2], device="cuda")
    hidden = token > torch.minimum(pos, length[:, None] - 1)[..., None]
    if c["window"]:
        hidden |= token <= pos[..., None] - c["window"]
    z.masked_fill_(hidden[:, None, :, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, kvh, 1, g, 1)
        m = torch.maximum(m, sink)
    m = m.clamp(min=torch.finfo(torch.float32).min)
    z = z.sub_(m).exp_()
    total = z.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + (sink - m).exp()
    out = torch.matmul(z.view(n, kvh, most * g, -1), v).view(n, kvh, most, g, -1) \
        / torch.where(total > 0, total, 1)
    lse = torch.where(total > 0, m + total.log(), -math.inf)
    row = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    i = row - starts[b]
    return {"out": out[b, :, i].flatten(1, 2).to(torch.bfloat16),
            "lse": lse[b, :, i].flatten(1).contiguous()}


def _append_plain(s):
    c, page = s["case"], s["case"]["page"]
    starts, length = s["starts"].long(), s["len"].long()
    row = torch.arange(s["k"].shape[0], device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    pos = length[b] - starts[b + 1] + row
    to, slot = s["table"].long()[b, pos // page], pos % page
    parts = _parts(c, s["pages"][1])
    for new, held, codes in ((s["k"], parts[0], parts[2]), (s["v"], parts[1], parts[3])):
        if new is None:
            continue
        x = new.float()
        if not c["fp8"]:
            held[to, :, slot] = x.to(torch.bfloat16)
            continue
        x = x.unflatten(-1, (-1, GROUP))
        ratio = x.abs().amax(-1).clamp(min=1e-4) * torch.tensor(1 / 448, device="cuda")
        bits = ratio.view(torch.int32)
        code = (bits >> 23) + ((bits & 0x7FFFFF) != 0)
        scale = (code << 23).view(torch.float32)
        x = (x / scale[..., None]).clamp(-448, 448).flatten(-2)
        held.view(torch.uint8)[to, :, slot] = x.to(torch.float8_e4m3fn).view(torch.uint8)
        codes[to, :, slot] = code.to(torch.uint8)
    return _held(s)


def _branch_plain(s):
    c, page = s["case"], s["case"]["page"]
    s["book"].copy_(s["book0"])
    ref, table, length = s["ref"], s["table"], s["len"]
    old, kids = s["parents"].long(), s["children"].long()
    # fork: the children hold the parents' pages
    mine = table[old]
    table[kids] = mine
    length[kids] = length[old]
    ref.index_add_(0, mine.clamp(min=0).flatten().long(), (mine >= 0).flatten().to(torch.int32))
    # reserve: pages for the draft, and a page of its own where a shared one
    # would be written into
    have = length[kids].long()
    count = (s["starts"][1:] - s["starts"][:-1]).long()
    last = table[kids, (have // page).clamp(max=table.shape[1] - 1)].long()
    part = (have % page > 0) & (count > 0)
    before = ((last[:, None] == last[None]) & part[None] & part[:, None]).tril(-1).sum(1)
    cow = part & (ref[last.clamp(min=0)] - before > 1)
    first = (have + page - 1) // page
    need = (have + count + page - 1) // page - first
    want = need + cow
    offset = want.cumsum(0) - want
    free = torch.nonzero(ref == 0).flatten()
    copied = free[offset.clamp(max=free.shape[0] - 1)]
    s["pages"][:, copied[cow]] = s["pages"][:, last[cow]]
    ref.index_add_(0, last.clamp(min=0), -cow.to(torch.int32))
    table[kids[cow], (have // page)[cow]] = copied[cow].to(torch.int32)
    ref[copied[cow]] = 1
    col = torch.arange(table.shape[1], device="cuda")
    fresh = (col >= first[:, None]) & (col < (first + need)[:, None])
    which = (offset + cow)[:, None] + col - first[:, None]
    given = free[which.clamp(0, free.shape[0] - 1)]
    table[kids] = torch.where(fresh, given.to(torch.int32), table[kids])
    ref[given[fresh]] = 1
    length[kids] += count.to(torch.int32)
    # free: back to what was accepted
    keep = (s["kept"].long() + page - 1) // page
    mine = table[kids]
    drop = (col >= keep[:, None]) & (mine >= 0)
    ref.index_add_(0, mine.clamp(min=0).flatten().long(), -drop.flatten().to(torch.int32))
    table[kids] = mine.masked_fill(drop, -1)
    length[kids] = s["kept"]
    return _state(s)


def _compact_plain(s):
    s["book"].copy_(s["book0"])
    ref, table = s["ref"], s["table"]
    live = ref > 0
    index = torch.arange(ref.shape[0], device="cuda")
    front = index < live.sum()
    to, src = torch.nonzero(front & ~live).flatten(), torch.nonzero(~front & live).flatten()
    s["pages"][:, to] = s["pages"][:, src]
    index[src] = to
    table.copy_(torch.where(table >= 0, index[table.clamp(min=0).long()].to(torch.int32), table))
    ref[to] = ref[src]
    ref[src] = 0
    return _state(s)


def _score_plain(s):
    c = s["case"]
    z = s["logits"].float() * (1 / 0.8) + 0.0
    t = s["tokens"].long()[:, None]
    index = torch.arange(c["vocab"], device="cuda")
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    total = e.sum(1, keepdim=True)
    mean = (e * torch.where(e > 0, z - m, 0)).sum(1, keepdim=True) / total
    lse = m + total.log()
    mine = z.gather(1, t)
    rank = ((z > mine) | ((z == mine) & (index < t))).sum(1).to(torch.int32)
    ids = top = None
    if c["top"]:
        # unique whole-number keys: larger logit first, then the lower index
        bits = z.view(torch.int32)
        bits = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        key = torch.topk((bits << 32) | (0xFFFFFFFF - index), min(c["top"], c["vocab"]), 1)[0]
        ids = (0xFFFFFFFF - (key & 0xFFFFFFFF)).to(torch.int32)
        top = z.gather(1, ids.long()) - lse
    return {"logprob": (mine - lse)[:, 0], "entropy": (total.log() - mean)[:, 0], "rank": rank,
            "ids": ids, "top": top}


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend_plain, "append": _append_plain, "branch": _branch_plain,
            "compact": _compact_plain, "score": _score_plain}[state["case"]["kind"]](state)


# ---------------------------------------------------------- in 64 bits

def exact(case, seed):
    if case["kind"] == "attend":
        return _attend_exact(prepare(case, seed))
    if case["kind"] == "score":
        return _score_exact(prepare(case, seed))
    if case["kind"] == "append":
        return _append_exact(prepare(case, seed))
    return None


def _append_exact(s):
    """Row after row: the values in units of their scale, not rounded to the
    page's format (8-bit: the scale is the power of two that brings the
    largest of 64 columns to 448 or less, and its exponent a whole number)."""
    c, page = s["case"], s["case"]["page"]
    parts = _parts(c, s["pages"][1])
    got = [None if x is None else x.double() for x in parts[:2]]
    lens, starts, table = s["len"].tolist(), s["starts"].tolist(), s["table"].tolist()
    for held, new in zip(got, (s["k"], s["v"])):
        if held is None:
            continue
        x = new.double().unflatten(-1, (-1, GROUP))
        if c["fp8"]:
            most = x.abs().amax(-1, keepdim=True).clamp(min=1e-4)
            x = x / torch.exp2(torch.ceil(torch.log2(most / 448)))
        x = x.flatten(-2)
        for b, n in enumerate(lens):
            for r in range(starts[b], starts[b + 1]):
                p = n - starts[b + 1] + r
                held[table[b][p // page], :, p % page] = x[r]
    return {"k": got[0], "v": got[1], "k_exp": None, "v_exp": None}


def _attend_exact(s):
    """One sequence after the other, some rows at a time: softmax over the
    tokens that a row sees, by its definition."""
    c = s["case"]
    heads, kvh, dim, page = c["heads"], c["kv_heads"], c["k_dim"], c["page"]
    g, v_dim = heads // kvh, c["v_dim"] or c["k_dim"]
    tokens = s["q"].shape[0]
    out = torch.zeros(tokens, heads, v_dim, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device="cuda")
    starts, lens = s["starts"].tolist(), s["len"].tolist()
    for b in range(c["seqs"]):
        n, new = lens[b], starts[b + 1] - starts[b]
        one = {"case": c, "pages": s["pages"],
               "table": s["table"][b:b + 1, :max(1, -(-n // page))]}
        keys, values = _rows(one, 1, torch.float64)
        step = max(1, int(4e8 // (max(n, 1) * heads)))
        for r0 in range(0, new, step):
            r1 = min(new, r0 + step)
            pos = n - new + torch.arange(r0, r1, device="cuda")
            low = max(0, n - new + r0 - c["window"] + 1) if c["window"] else 0
            high = n - new + r1
            token = torch.arange(low, high, device="cuda")
            seen = token[None] <= pos[:, None]
            if c["window"]:
                seen &= token[None] > pos[:, None] - c["window"]
            for h in range(kvh):
                q = s["q"][starts[b] + r0:starts[b] + r1, h * g:(h + 1) * g].double()
                z = (q.flatten(0, 1) @ keys[0, h, low:high].T / math.sqrt(dim)).view(
                    r1 - r0, g, -1)
                z = torch.where(seen[:, None], z, -math.inf)
                if s["sink"] is not None:
                    z = torch.cat([z, s["sink"][h * g:(h + 1) * g].double()[None, :, None]
                                   .expand(r1 - r0, g, 1)], 2)
                p = torch.softmax(z, 2)[..., :high - low]
                rows = slice(starts[b] + r0, starts[b] + r1)
                out[rows, h * g:(h + 1) * g] = (p.reshape(-1, high - low)
                                                @ values[0, h, low:high]).view(r1 - r0, g, -1)
                lse[rows, h * g:(h + 1) * g] = torch.logsumexp(z, 2)
                del z, p
    return {"out": out, "lse": lse}


def _score_exact(s):
    c = s["case"]
    got = {"logprob": [], "entropy": [], "top": []}
    for r0 in range(0, c["rows"], 128):
        # the scale is the fp32 number that the call is given
        z = s["logits"][r0:r0 + 128].double() * float(torch.tensor(1 / 0.8))
        logp = torch.log_softmax(z, 1)
        p = logp.exp()
        got["entropy"].append(-(p * logp.clamp(min=-1e300)).sum(1))
        got["logprob"].append(logp.gather(1, s["tokens"][r0:r0 + 128].long()[:, None])[:, 0])
        if c["top"]:
            got["top"].append(logp.sort(1, descending=True)[0][:, :min(c["top"], c["vocab"])])
    return {"logprob": torch.cat(got["logprob"]), "entropy": torch.cat(got["entropy"]),
            "rank": None, "ids": None, "top": torch.cat(got["top"]) if c["top"] else None}
