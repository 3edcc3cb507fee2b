"""Plain implementations (64 bits, whole numbers) of the paged cache, the
attention over it and the scoring of tokens, for their tests: one sequence and
one token after the other, as the entries' documentation defines them."""
import math

import numpy as np
import torch

GROUP = 64
FULL, LIST, PAGE = 1, 2, 4


def page_layout(ps, kvh, k_dim, v_dim, fp8):
    """(page bytes, offset of the values, of the keys' scales, of the values')."""
    kn, vn = kvh * ps * k_dim, kvh * ps * v_dim
    if not fp8:
        return (2 * (kn + vn) + 255) // 256 * 256, 2 * kn, 0, 0
    used = kn + vn + (kn + vn) // GROUP
    return (used + 255) // 256 * 256, kn, kn + vn, kn + vn + kn // GROUP


class Book:
    """The bookkeeping as Python lists; moves are returned as (from, to) pairs."""

    def __init__(self, n_pages, n_seqs, max_pages, ps):
        self.ref, self.len = [0] * n_pages, [0] * n_seqs
        self.table = [[-1] * max_pages for _ in range(n_seqs)]
        self.ps, self.status = ps, 0

    def cdiv(self, n):
        return -(-n // self.ps)

    def reserve(self, seqs, counts):
        if self.status:
            return []
        room = len(self.table[0]) * self.ps
        ok = [0 <= s < len(self.len) and c >= 0 and seqs.count(s) == 1 and self.len[s] + c <= room
              for s, c in zip(seqs, counts)]
        if not all(ok):
            self.status |= LIST
            return []
        # one after the other on a copy: all of it or nothing
        ref, moves, cells = list(self.ref), [], []
        free = [i for i, r in enumerate(ref) if r == 0]
        for s, c in zip(seqs, counts):
            n = self.len[s]
            if c and n % self.ps:
                page = self.table[s][n // self.ps]
                if ref[page] > 1:
                    if not free:
                        self.status |= FULL
                        return []
                    new = free.pop(0)
                    ref[page] -= 1
                    ref[new] = 1
                    moves.append((page, new))
                    cells.append((s, n // self.ps, new))
            for k in range(self.cdiv(n), self.cdiv(n + c)):
                if not free:
                    self.status |= FULL
                    return []
                new = free.pop(0)
                ref[new] = 1
                cells.append((s, k, new))
        self.ref = ref
        for s, k, page in cells:
            self.table[s][k] = page
        for s, c in zip(seqs, counts):
            self.len[s] += c
        return moves

    def fork(self, parents, children):
        n = len(self.len)
        old_len = list(self.len)
        for p, c in zip(parents, children):
            if not (0 <= p < n and 0 <= c < n) or children.count(c) > 1 or c in parents \
                    or old_len[c]:
                self.status |= LIST
                continue
            held = self.cdiv(self.len[p])
            self.table[c] = self.table[p][:held] + [-1] * (len(self.table[p]) - held)
            self.len[c] = self.len[p]
            for e in self.table[c][:held]:
                self.ref[e] += 1

    def free(self, seqs, new_len):
        for s, to in zip(seqs, new_len):
            if not 0 <= s < len(self.len) or seqs.count(s) > 1 or to < 0 or to > self.len[s]:
                self.status |= LIST
                continue
            for k in range(self.cdiv(to), self.cdiv(self.len[s])):
                self.ref[self.table[s][k]] -= 1
                self.table[s][k] = -1
            self.len[s] = to

    def compact(self):
        used = sum(r > 0 for r in self.ref)
        holes = [i for i in range(used) if self.ref[i] == 0]
        tails = [i for i in range(used, len(self.ref)) if self.ref[i] > 0]
        to = dict(zip(tails, holes))
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        self.table = [[to.get(e, e) for e in row] for row in self.table]
        return list(to.items())


def rows64(pages_layer, table_row, n, ps, kvh, k_dim, v_dim, fp8):
    """The first n tokens' keys and values [n][kvh][dim] in 64 bits, from one
    layer's pages on the host (uint8 [n_pages][page_bytes])."""
    _, v_off, ks, vs = page_layout(ps, kvh, k_dim, v_dim, fp8)
    idx = torch.tensor([table_row[j] for j in range(-(-n // ps))], dtype=torch.long)
    got = []
    for width, at, sat in ((k_dim, 0, ks), (v_dim, v_off, vs)):
        if not width:
            got.append(got[0])
            continue
        count = kvh * ps * width
        if fp8:
            x = pages_layer[idx, at:at + count].contiguous().view(torch.float8_e4m3fn).double()
            e = pages_layer[idx, sat:sat + count // GROUP].double() - 127
            x = (x.view(-1, GROUP) * torch.exp2(e).view(-1, 1)).view(len(idx), kvh, ps, width)
        else:
            x = pages_layer[idx, at:at + 2 * count].contiguous().view(torch.bfloat16).double() \
                .view(len(idx), kvh, ps, width)
        got.append(x.permute(0, 2, 1, 3).reshape(-1, kvh, width)[:n])
    return got


def attend64(q, keys, values, pos, scale, window, sink):
    """One new token at position pos: q [heads][dim] over keys, values
    [n][kvh][dim] (64 bits). (out [heads][v], lse [heads], sum of p |v|,
    largest scale * sum |q||k|)."""
    heads, kvh = q.shape[0], keys.shape[1]
    g = heads // kvh
    low = max(0, pos - window + 1) if window else 0
    k, v = keys[low:pos + 1], values[low:pos + 1]
    out = torch.zeros(heads, values.shape[2], dtype=torch.float64)
    lse = torch.full((heads,), -math.inf, dtype=torch.float64)
    mass, most = torch.zeros_like(out), torch.zeros(heads, dtype=torch.float64)
    for h in range(heads):
        z = scale * (k[:, h // g] @ q[h])
        all_z = z if sink is None else torch.cat([z, sink[h:h + 1]])
        if all_z.numel() == 0:
            continue
        lse[h] = torch.logsumexp(all_z, 0)
        p = torch.exp(z - lse[h])
        out[h] = p @ v[:, h // g]
        mass[h] = p @ v[:, h // g].abs()
        if z.numel():
            most[h] = abs(scale) * (k[:, h // g].abs() @ q[h].abs()).max()
    return out, lse, mass, most


def attend64_far(q, keys, values, pos, scale, sink):
    """attend64 without a window for scores of any size: every term relative to
    the largest one (beyond 2^53 the sum's logarithm is lost beside a score
    even in 64 bits). (out, lse, sum of p |v|)."""
    g = q.shape[0] // keys.shape[1]
    k, v = (x[:pos + 1].permute(1, 0, 2).repeat_interleave(g, 0) for x in (keys, values))
    z = scale * torch.matmul(k, q[:, :, None])[:, :, 0]
    if sink is not None:
        z = torch.cat([z, sink[:, None]], 1)
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    p = (p / total)[:, None, :pos + 1]
    return (torch.matmul(p, v)[:, 0], (top + total.log())[:, 0],
            torch.matmul(p, v.abs())[:, 0])


def attend_bounds(out, mass, most, dim):
    """How far a BF16 result may be from out, and lse from its own.

    Scores: dim products, exact in fp32 (BF16 times BF16), summed in any order
    and scaled: |dz| <= (dim + 4) 2^-24 most, doubled for the maximum's; e^z by
    the hardware's exp2 and the running rescaling add less than 2^-18 relative.
    Each weight is rounded to BF16 for the matrix unit (2^-8 of it), and the
    result once (2^-8 of it)."""
    dz = (dim + 4) * 2.0 ** -24 * 2 * most + 2.0 ** -18
    rel = torch.expm1(dz)
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 3 * rel)[:, None] * mass + 1e-30, rel + 1e-6


def score64(z, token, k):
    """Definition of dsv4g_logprobs for one row of scaled logits (the fp32
    products, as float64 numpy): logprob, entropy, rank, ids, their logprobs."""
    nan = float("nan")
    order = sorted(range(len(z)), key=lambda i: (-(z[i] if z[i] == z[i] else -math.inf), i))
    ids = (order + [-1] * k)[:k]
    bad = np.isnan(z).any() or np.isinf(z.max())
    if bad:
        return nan, nan, -1, ids, [nan] * k
    # relative to the maximum, which may be the type's lowest value
    d = z - z.max()
    ls = math.log(np.exp(d).sum())
    p = np.exp(d - ls)
    entropy = ls - (p * np.where(p > 0, d, 0)).sum()
    ok = 0 <= token < len(z)
    rank = int((z > z[token]).sum() + (z[:token] == z[token]).sum()) if ok else -1
    return (d[token] - ls if ok else nan, entropy, rank, ids,
            [d[i] - ls if i >= 0 else nan for i in ids])
