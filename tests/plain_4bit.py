"""A cache in 4 bits stated plainly: rounding, layout, attention, sums of weights and eviction, in 64 bits, one token at a time where
that is clearest.  Used by the tests only."""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch


def groups(D):
    """The fewest equal groups of at most 64 channels, each of whole words of 8."""
    g = 1
    while D // g > 64 or D % g or (D // g) % 8:
        g += 1
    return g


def page_bytes(D, page):
    raw = page * (D + 8 * groups(D))
    return raw + (-raw) % 16


def bf16_toward(x, up):
    """The bfloat16 next to each float64 of ``x`` that is not above (``up``: not below) it."""
    near = x.to(torch.bfloat16)
    wrong = near.double() < x if up else near.double() > x
    step = torch.full_like(near, math.inf if up else -math.inf)
    return torch.where(wrong, torch.nextafter(near, step), near)


def quantise(rows):
    """float32 ``[N, D]`` -> numbers ``[N, D]`` (int64), scales and minima ``[N, G]`` (bfloat16)."""
    N, D = rows.shape
    G = groups(D)
    x = rows.double().view(N, G, D // G)
    ok = torch.isfinite(x).all(-1)
    z = bf16_toward(torch.where(ok[..., None], x, torch.zeros_like(x)).amin(-1), up=False)
    spread = (torch.where(ok[..., None], x, torch.zeros_like(x)).amax(-1) - z.double()).float()
    # the division in float32, as the definition says: (maximum - minimum) / 15 rounded to nearest, then outwards
    s = bf16_toward((spread / torch.full_like(spread, 15.0)).double(), up=True)
    ok &= torch.isfinite(s.float()) & torch.isfinite(z.float())
    d = torch.where((s.double() > 0) & ok, s.double(), torch.ones_like(s.double()))
    n = torch.round(((x - z.double()[..., None]).float() / d.float()[..., None]).double()).clamp(0, 15)
    n = torch.where((ok & (s.double() > 0))[..., None], n, torch.zeros_like(n))
    nan = torch.full_like(s, math.nan)
    return n.reshape(N, D).long(), torch.where(ok, s, nan), torch.where(ok, z, nan)


def value(n, s, z):
    """What numbers stand for, float64."""
    size = n.shape[-1] // s.shape[-1]
    return z.double().repeat_interleave(size, -1) + n.double() * s.double().repeat_interleave(size, -1)


def _row_bytes(n, s, z):
    """Bytes of one row's codes and parameters."""
    D, G = n.numel(), s.numel()
    code = []
    for i in range(D // 8):
        first = (i % G) * (D // G) + 8 * (i // G)
        word = sum(int(n[first + c]) << (4 * c) for c in range(8))
        code += [(word >> (8 * b)) & 255 for b in range(4)]
    pair = torch.stack([s, z], -1).contiguous().view(torch.int16).flatten().tolist()
    par = [b for v in pair for b in ((v & 0xFFFF) & 255, (v & 0xFFFF) >> 8)]
    return torch.tensor(code, dtype=torch.uint8), torch.tensor(par, dtype=torch.uint8)


def places_in(D, page, row):
    """Where a row's key codes, value codes, key parameters and value parameters lie in a record: (first byte, bytes) each."""
    half, par = D // 2, 4 * groups(D)
    return ((row * half, half), ((page + row) * half, half), (2 * page * half + row * par, par),
            (2 * page * half + (page + row) * par, par))


def write(pages, page_id, head, row, page, k, v):
    """One token's key and value (float32 ``[D]`` each) into its record."""
    D = k.numel()
    at = places_in(D, page, row)
    for x, c, p in ((k, at[0], at[2]), (v, at[1], at[3])):
        n, s, z = quantise(x[None])
        code, par = _row_bytes(n[0], s[0], z[0])
        pages[page_id, head, c[0]:c[0] + c[1]] = code
        pages[page_id, head, p[0]:p[0] + p[1]] = par


def read(record, D, page, row):
    """(key, value) of one row, as numbers, scales and minima."""
    G = groups(D)
    at = places_in(D, page, row)
    out = []
    for c, p in ((at[0], at[2]), (at[1], at[3])):
        code = record[c[0]:c[0] + c[1]].long()
        n = torch.zeros(D, dtype=torch.long)
        for i in range(D // 8):
            first = (i % G) * (D // G) + 8 * (i // G)
            word = sum(int(code[4 * i + b]) << (8 * b) for b in range(4))
            for c8 in range(8):
                n[first + c8] = (word >> (4 * c8)) & 15
        par = record[p[0]:p[0] + p[1]].contiguous().view(torch.bfloat16).view(G, 2)
        out.append((n, par[:, 0].clone(), par[:, 1].clone()))
    return out


class Cache:
    """Random sequences in pages, filled at once: the same layout as :func:`write`, made with tensors.  ``spare`` pages more than are
    used; what no token uses is poisoned (codes of 15, parameters that are NaN)."""

    def __init__(self, lens, G, D, page, seed=0, k_scale=1.0, width=None, mutate=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.G, self.D, self.page = list(lens), G, D, page
        need = [-(-n // page) for n in lens]
        self.width = width or max(1, max(need, default=1))
        count = sum(need) + 1
        order = torch.randperm(count, generator=g).tolist()
        self.table = torch.full((len(lens), self.width), order[-1], dtype=torch.int32)
        self.pages = torch.full((count, G, page_bytes(D, page)), 255, dtype=torch.uint8)
        self.k, self.v = [], []  # (n, s, z) of every sequence: [G, L, D], [G, L, groups] x 2
        half, par, at = D // 2, 4 * groups(D), 0
        for b, n in enumerate(lens):
            self.table[b, : need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
            at += need[b]
            k, v = torch.randn((G, n, D), generator=g) * k_scale, torch.randn((G, n, D), generator=g)
            if mutate:
                mutate(b, k, v)
            for which, (x, out) in enumerate(((k, self.k), (v, self.v))):
                q = [y.view(G, n, -1) for y in quantise(x.reshape(G * n, D))]
                out.append(q)
                if n == 0:
                    continue
                words = q[0].view(G, n, groups(D), -1, 8).transpose(2, 3).reshape(G, n, D)
                code = (words[..., 0::2] | (words[..., 1::2] << 4)).to(torch.uint8)
                params = torch.stack([q[1], q[2]], -1).reshape(G, n, -1).contiguous().view(torch.uint8)
                for i in range(need[b]):
                    rows = slice(i * page, min((i + 1) * page, n))
                    m = rows.stop - rows.start
                    rec = self.pages[int(self.table[b, i])]
                    rec[:, which * page * half:(which * page + m) * half] = code[:, rows].reshape(G, -1)
                    base = 2 * page * half + which * page * par
                    rec[:, base:base + m * par] = params[:, rows].reshape(G, -1)

    def values(self, b):
        """(keys, values) ``[G, L, D]`` of one sequence in float64."""
        return value(*self.k[b]), value(*self.v[b])


def step_of(new, lens, page, device="cuda", captured_width=0):
    """What attention reads of a step: sequences with ``lens`` tokens, the last ``new`` of them brought by the step."""
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    singles = [b for b, n in enumerate(new) if n == 1]
    return SimpleNamespace(
        num_tokens=cu[-1], num_seqs=len(new), cu_seqlens=dev(cu), kv_lens=dev(list(lens)), kv_longest=dev([max(lens, default=0)]),
        token_seq=dev([b for b, n in enumerate(new) for _ in range(n)]),
        positions=dev([L - n + i for n, L in zip(new, lens) for i in range(n)]), max_query_len=max(new, default=0), max_kv_len=max(lens, default=0),
        decode_only=all(n == 1 for n in new), single_seqs=dev(singles), num_single=len(singles), host_cu_seqlens=cu,
        host_kv_lens=list(lens), captured_width=captured_width, choices={})


def attention(q, cache, new, lens, scale, window=None):
    """float64: ``[T, H, D]`` results, ``[T, H]`` log sums, and per sequence the weights ``[n, H, L]``."""
    T, H, D = q.shape
    R = H // cache.G
    out, lse, weights, t = torch.zeros((T, H, D), dtype=torch.float64), torch.zeros((T, H), dtype=torch.float64), [], 0
    for b, (n, L) in enumerate(zip(new, lens)):
        k, v = cache.values(b)
        w = torch.zeros((n, H, L), dtype=torch.float64)
        for i in range(n):
            last = L - n + i
            first = max(0, last - window + 1) if window else 0
            for h in range(H):
                x = (k[h // R, first:last + 1] @ q[t, h].double()) * scale
                lse[t, h] = torch.logsumexp(x, 0)
                w[i, h, first:last + 1] = torch.softmax(x, 0)
                out[t, h] = w[i, h, first:last + 1] @ v[h // R, first:last + 1]
            t += 1
        weights.append(w)
    return out, lse, weights


def evict(mass, place, keep, first, recent):
    """One (sequence, head): the slot whose token each of the first ``keep`` slots holds afterwards."""
    n = len(mass)
    if n <= keep:
        return list(range(n))
    newest = max(place)
    forced = [p < first or p > newest - recent for p in place]
    rank = lambda i: (0 if forced[i] else 1, -math.inf if math.isnan(mass[i]) else -mass[i],  # noqa: E731
                      0 if math.isnan(mass[i]) else 1, i)
    stays = sorted(sorted(range(n), key=rank)[:keep])
    movers = [i for i in stays if i >= keep]
    kept = set(stays)
    return [i if i in kept else movers.pop(0) for i in range(keep)]


def values_of(pages, D, page):
    """What whole records ``[.., bytes]`` stand for: keys and values ``[.., page, D]`` in float32, by tensors."""
    G, half, par = groups(D), D // 2, 4 * groups(D)
    out = []
    for which in range(2):
        code = pages[..., which * page * half:(which + 1) * page * half].unflatten(-1, (page, half))
        n = torch.stack([code & 15, code >> 4], -1).flatten(-2)  # [.., page, D] in the order of words
        n = n.unflatten(-1, (-1, G, 8)).transpose(-3, -2).flatten(-3).float()
        base = 2 * page * half + which * page * par
        sz = pages[..., base:base + page * par].contiguous().view(torch.bfloat16).float().unflatten(-1, (page, G, 2))
        s, z = (x.repeat_interleave(D // G, -1) for x in (sz[..., 0], sz[..., 1]))
        out.append(z + n * s)
    return out
