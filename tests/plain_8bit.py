"""A cache in 8 bits stated plainly: rounding, layout, writing and attention, in 64 bits, one number or one token at a time where that is
clearest.  Used by the tests only."""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

LEAST = -100  # exponent of the least scale


def page_bytes(D, page):
    return 2 * page * D + 16


def four_bits(x):
    """float64 values rounded to 4 significant bits, half ways to even; NaN where they or the result are not finite in float32."""
    mantissa, exponent = torch.frexp(x.double())
    y = torch.ldexp(torch.round(mantissa * 16), exponent - 4)  # (round: half ways to even)
    return torch.where(x.double().isfinite() & (y.abs() < 2.0**128), y, torch.full_like(y, math.nan))


def scale_exponent(rounded):
    """The exponent of the scale of values of 4 significant bits (any shape)."""
    most = float(rounded[rounded.isfinite()].abs().max()) if bool(rounded.isfinite().any()) else 0.0
    e = LEAST
    while most > 448.0 * 2.0**e:
        e += 1
    return e


def held(rounded, e):
    """What values of 4 significant bits stand for under the scale 2^e."""
    y = rounded / 2.0**e
    return torch.where(y.abs() < 2.0**-6, torch.trunc(y * 512) / 512, y) * 2.0**e


def code_of(value, e):
    """The byte of a held value (a float) under 2^e."""
    sign = 128 if math.copysign(1.0, value) < 0 else 0
    y = abs(value) / 2.0**e
    if math.isnan(y):
        return sign | 127
    if y < 2.0**-6:
        return sign | int(y * 512)
    mantissa, exponent = math.frexp(y)  # in [0.5, 1)
    return sign | ((exponent - 1 + 7) << 3) | int(mantissa * 16 - 8)


def value_of(code):
    """What a byte stands for without the scale."""
    exponent, mantissa = (code >> 3) & 15, code & 7
    y = math.nan if code & 127 == 127 else (1 + mantissa / 8) * 2.0 ** (exponent - 7) if exponent else mantissa * 2.0**-9
    return -y if code & 128 else y


VALUES = torch.tensor([value_of(c) for c in range(256)], dtype=torch.float64)


def channel_at(D, row):
    """Where each channel of a row lies in it."""
    mask = {64: 3, 128: 7, 256: 7}.get(D, 0)
    d = torch.arange(D)
    return ((d // 16) ^ (row & mask)) * 16 + d % 16


def write_rows(pages, page_id, head, page, which, rows):
    """The first ``len(rows)`` rows (4 significant bits, float64 ``[n, D]``) of the keys (0) or values (1) of a record, written at once."""
    n, D = rows.shape
    e = scale_exponent(rows)
    y = held(rows, e)
    for r in range(n):
        at = (which * page + r) * D + channel_at(D, r)
        pages[page_id, head, at] = torch.tensor([code_of(v, e) for v in y[r].tolist()], dtype=torch.uint8)
    at = 2 * page * D + 4 * which
    pages[page_id, head, at:at + 4] = torch.tensor([2.0**e], dtype=torch.float32).view(torch.uint8)
    return y


def read_rows(record, D, page, which, n):
    """(values ``[n, D]``, the scale) of the first ``n`` rows of a record."""
    at = 2 * page * D + 4 * which
    s = float(record[at:at + 4].contiguous().view(torch.float32)[0])
    out = torch.empty((n, D), dtype=torch.float64)
    for r in range(n):
        out[r] = VALUES[record[(which * page + r) * D + channel_at(D, r)].long()] * s
    return out, s


def values_of(pages, D, page):
    """What whole records ``[.., bytes]`` stand for: keys and values ``[.., page, D]`` in float32, by tensors."""
    order = torch.stack([channel_at(D, r) for r in range(page)])
    scale = pages[..., 2 * page * D:2 * page * D + 8].contiguous().view(torch.float32)
    out = []
    for which in range(2):
        code = pages[..., which * page * D:(which + 1) * page * D].unflatten(-1, (page, D))
        out.append((VALUES[code.gather(-1, order.expand(code.shape)).long()] * scale[..., which, None, None]).float())
    return out


class Cache:
    """Random sequences in pages, filled at once.  A spare page more than are used; what no token uses is poisoned (codes and scales that are
    no numbers).  ``mutate(b, k, v)`` may change a sequence's keys and values before they are rounded."""

    def __init__(self, lens, G, D, page, seed=0, k_scale=1.0, width=None, mutate=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.G, self.D, self.page = list(lens), G, D, page
        need = [-(-n // page) for n in lens]
        self.width = width or max(1, max(need, default=1))
        count = sum(need) + 1
        order = torch.randperm(count, generator=g).tolist()
        self.table = torch.full((len(lens), self.width), order[-1], dtype=torch.int32)
        self.pages = torch.full((count, G, page_bytes(D, page)), 255, dtype=torch.uint8)
        self.kv, self.scales, at = [], [], 0  # per sequence: [2, G, L, D] and [2, G, pages]
        place = torch.stack([channel_at(D, r) for r in range(page)])
        for b, n in enumerate(lens):
            self.table[b, : need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
            at += need[b]
            k, v = torch.randn((G, n, D), generator=g) * k_scale, torch.randn((G, n, D), generator=g)
            if mutate:
                mutate(b, k, v)
            rows = four_bits(torch.stack([k, v]))
            scales = torch.zeros((2, G, need[b]), dtype=torch.float64)
            for i in range(need[b]):
                part = rows[:, :, i * page:(i + 1) * page]
                m = part.shape[2]
                for which in range(2):
                    for h in range(G):
                        e = scale_exponent(part[which, h])
                        y = part[which, h] = held(part[which, h], e)
                        scales[which, h, i] = 2.0**e
                        code = (y / 2.0**e).float().to(torch.float8_e4m3fn).view(torch.uint8)
                        code = torch.where(y.isnan(), torch.full_like(code, 127), code)
                        rec = self.pages[int(self.table[b, i]), h]
                        rec[which * page * D:(which * page + m) * D] = torch.empty_like(code).scatter_(1, place[:m], code).flatten()
                        rec[2 * page * D + 4 * which:2 * page * D + 4 * which + 4] = torch.tensor([2.0**e], dtype=torch.float32).view(torch.uint8)
            self.kv.append(rows)
            self.scales.append(scales)

    def values(self, b):
        """(keys, values) ``[G, L, D]`` of one sequence in float64."""
        return self.kv[b][0], self.kv[b][1]


def step_of(new, lens, page, device="cuda", captured_width=0):
    """What the operators read of a step: sequences with ``lens`` tokens, the last ``new`` of them brought by the step."""
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
        host_kv_lens=list(lens), captured_width=captured_width, choices={}, extras={})


def seen(last, window=None, keep_first=0):
    """The keys that a token at place ``last`` sees."""
    lo = max(0, last - window + 1) if window else 0
    return [j for j in range(last + 1) if j >= lo or j < keep_first]


def attention(q, cache, new, lens, scale, window=None, keep_first=0):
    """float64: ``[T, H, D]`` results, and per sequence the weights ``[n, H, L]``."""
    T, H, D = q.shape
    R = H // cache.G
    out, weights, t = torch.zeros((T, H, D), dtype=torch.float64), [], 0
    for b, (n, L) in enumerate(zip(new, lens)):
        k, v = cache.values(b)
        w = torch.zeros((n, H, L), dtype=torch.float64)
        for i in range(n):
            at = torch.tensor(seen(L - n + i, window, keep_first))
            kk, vv = k[:, at].repeat_interleave(R, 0), v[:, at].repeat_interleave(R, 0)
            p = torch.softmax(torch.einsum("hd,hjd->hj", q[t].double(), kk) * scale, -1)
            w[i][:, at] = p
            out[t] = torch.einsum("hj,hjd->hd", p, vv)
            t += 1
        weights.append(w)
    return out, weights
