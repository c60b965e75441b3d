"""The operators around a key/value cache that is held in 8 bits, as cases that can be timed and compared.

A page of such a cache keeps, for each of its key/value heads, one record: the keys' codes, the values' codes (a byte a channel, 8-bit
floats with 4 exponent and 3 mantissa bits), and the keys' and the values' scale (float32, powers of two), rounded up to 16 bytes.  A row's
16-byte pieces stand in the order ``piece ^ (row & mask)``, ``mask`` 3 for heads of 64 channels, 7 for 128 and 256, else 0.

A number is rounded to 4 significant bits; the scale is the least power of two that brings all numbers of the page's tokens to 448 at most
(2^-100 at least); numbers below 2^-6 of the scale are cut to multiples of 2^-9 of it.  Cutting composes: tokens that come one by one, under a scale
that grows, end as those that came together.

* ``store``     -- a step's queries, keys and values behind the projection: norm, rotation, the cache write; then the sequences'
                   keys and values as the attention over prompts reads them
* ``attention`` -- every token of a step over its sequence's tokens: single tokens, portions of prompts, or both
* ``window``    -- the same where a token sees the last ``window`` tokens and the sequence's first ``first`` ones
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    b8 = ",".join(["4096"] * 8)
    return [
        # eight requests' next tokens written behind short contexts: the smallest write
        dict(name="store_decode", kind="store", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="40,41,42,43,44,45,46,47", new="1,1,1,1,1,1,1,1"),
        # a step that takes several prompts at once, one of them a later portion
        dict(name="store_prompts", kind="store", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="0,0,2048,0", new="1500,701,1024,33"),
        # one user reading along: the least work, where latency counts
        dict(name="attention_one", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16", context="512", new="1"),
        # the package's default benchmark point: eight requests behind 4,096 tokens each
        dict(name="attention_batch", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context=b8, new=",".join(["1"] * 8)),
        # a continuous batch: 48 requests of unequal lengths
        dict(name="attention_ragged", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context=",".join(str(64 + 83 * i) for i in range(48)), new=",".join(["1"] * 48)),
        # a few requests behind long documents: the largest case
        dict(name="attention_long", kind="attention", heads=64, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="32768,32768,31111,29999,32768,17001,32000,30001", new="1,1,1,1,1,1,1,1"),
        # prompts: two new ones, a later portion of a third, and a request that decodes beside them
        dict(name="attention_prompts", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="0,0,2048,700", new="1500,701,1000,1"),
        # the 32-bit path, which checks the 16-bit one
        dict(name="attention_float32", kind="attention", heads=16, kv_heads=4, dim=64, page=16, dtype="float32",
             context="300,77", new="20,1"),
        # chats that went on for long, cut to a window and their first tokens
        dict(name="window_decode", kind="window", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context=",".join(str(900 + 1117 * i) for i in range(16)), new=",".join(["1"] * 16), window=4096, first=4),
        # prompts under a window: one that fits it, one that does not, a later portion of a third
        dict(name="window_prompts", kind="window", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="0,0,5000", new="700,2048,500", window=1024, first=16),
    ]


# query heads, key/value heads, head size
_HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (16, 4, 128), (16, 8, 64), (40, 8, 128), (16, 2, 256), (16, 1, 64), (20, 4, 80)]


def _spread(rng, low, high):
    """A whole number in low..high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    kind = rng.choice(["store", "store", "attention", "attention", "attention", "window", "window"])
    H, G, D = rng.choice(_HEADS)
    case = dict(kind=kind, heads=H, kv_heads=G, dim=D, page=rng.choice([16, 16, 16, 8, 32, 64, 24, 5]), dtype="bfloat16")
    if rng.random() < 0.5:  # next tokens
        n = _spread(rng, 1, 64)
        most = _spread(rng, 64, min(32768, 131072 // n)) if kind != "store" else 200
        case.update(context=_text(rng.randint(most // 8, most) for _ in range(n)), new=_text([1] * n))
    else:  # portions of prompts, single tokens among them
        n = rng.randint(1, 4)
        case.update(context=_text(rng.choice([0, 0, rng.randint(1, 2000)]) for _ in range(n)),
                    new=_text(rng.choice([1, _spread(rng, 2, 40), _spread(rng, 17, 1000), _spread(rng, 17, 1000)]) for _ in range(n)))
    if kind == "window":
        case.update(window=_spread(rng, 1, 4096), first=rng.choice([0, 1, 4, 16, rng.randint(1, 100)]))
    if rng.random() < 0.2:
        case.update(dtype="float32", context=_text(min(int(c), rng.randint(50, 700)) for c in case["context"].split(",")),
                    new=_text(min(int(c), 100) for c in case["new"].split(",")))
    return case


# ---- sizes ---------------------------------------------------------------------------------------------------------------


def _numbers(text):
    return [int(x) for x in text.split(",")]


def _lengths(case):
    """Cached tokens and new tokens of every sequence."""
    return _numbers(case["context"]), _numbers(case["new"])


def _record(D, page):
    """Bytes of one page and head."""
    return 2 * D * page + 16


def _seen(case, place):
    """How many tokens a token at that place sees."""
    window, first = case.get("window") or 0, case.get("first") or 0
    return place + 1 if not window else min(place + 1, window) + min(first, max(0, place + 1 - window))


def work(case):
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    e = 4 if case["dtype"] == "float32" else 2
    token = G * (2 * D + 8 / page)  # bytes of a cached token's keys and values, its share of the scales with them
    context, new = _lengths(case)
    T = sum(new)
    if case["kind"] == "store":
        # the projection read, queries and the new tokens' codes written; then every token read and its keys and values written
        kv = sum(context) + T
        return {"bytes": int(T * ((2 * H + 2 * G) * D * e + token) + kv * (token + 2 * G * D * e)), "flops": 8 * T * (H + 2 * G) * D}
    read = pairs = 0
    for c, n in zip(context, new):
        first, window = case.get("first") or 0, case.get("window") or 0
        reach = max(0, c - window + 1) if window else 0  # the first token that the first new one's window holds
        read += c + n - reach + min(first, reach)
        pairs += sum(_seen(case, c + i) for i in range(n))
    return {"bytes": int(read * token + 2 * T * H * D * e), "flops": 4 * H * D * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------------


def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    context, new = _lengths(case)
    kv = [c + n for c, n in zip(context, new)]
    B, T = len(kv), sum(new)
    need = [-(-n // page) for n in kv]
    width = -(-max(need) // 8) * 8
    count = sum(need)
    order = torch.randperm(count, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table = torch.full((B, width), count, dtype=torch.int32)  # what no token uses names the spare page
    window, first = case.get("window") or 0, case.get("first") or 0
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        if window:  # pages that every new token's window has passed were given back
            table[b, -(-first // page): max(0, context[b] - window + 1) // page] = -1
        at += n
    table = table.to(DEV)
    pages = torch.empty((count + 1, G, _record(D, page)), dtype=torch.uint8, device=DEV)
    pages.fill_(255)  # the spare page, pages without a token, and rows behind a sequence's last one: nothing that is a number
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    # the tokens that the cache holds before the step (with the new ones, where the step does not write them itself)
    held = torch.tensor(context, dtype=torch.int32, device=DEV) if case["kind"] == "store" else lens
    place = torch.arange(width, device=DEV)
    b, i = ((place * page < held[:, None]) & (table >= 0) & (place < torch.tensor(need, device=DEV)[:, None])).nonzero(as_tuple=True)
    loud = 1.0 + 3.0 * (torch.rand((1, 1, 1, D), generator=g, device=DEV) < 0.05)  # some channels are larger than others, as keys' are
    for lo in range(0, len(b), 2048):  # in portions: less memory
        part = slice(lo, lo + 2048)
        rows = [torch.randn((len(b[part]), G, page, D), generator=g, device=DEV) for _ in range(2)]
        rows[0] *= loud
        there = (i[part, None] * page + torch.arange(page, device=DEV) < held[b[part], None])[:, None, :, None].expand(-1, G, -1, 1)
        _write_pages(pages, table[b[part], i[part]].long(), [_four_bits(x) for x in rows], there, None)
    state = dict(case=case, kv=kv, new=new, context=context, table=table, lens=lens, pages=pages)
    state["positions"] = torch.tensor([c + j for c, n in zip(context, new) for j in range(n)], dtype=torch.int32, device=DEV)
    state["token_seq"] = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], dtype=torch.int32, device=DEV)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    singles = [b for b, n in enumerate(new) if n == 1]
    state.update(host_cu=cu, cu=torch.tensor(cu, dtype=torch.int32, device=DEV), longest=torch.tensor([max(kv)], dtype=torch.int32, device=DEV),
                 singles=torch.tensor(singles, dtype=torch.int32, device=DEV), num_singles=len(singles))
    state["qkv"] = torch.randn((T, (H + 2 * G) * D), generator=g, device=DEV).to(_dtype(case))
    if case["kind"] == "store":
        state["q_weight"] = 1.0 + 0.1 * torch.randn((D,), generator=g, device=DEV)
        state["k_weight"] = 1.0 + 0.1 * torch.randn((D,), generator=g, device=DEV)
        angle = torch.arange(max(kv), device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# ---- the framework's calls ---------------------------------------------------------------------------------------------------


def _ops(keep=[]):  # one kernel table for the program
    if not keep:
        from qwen3_runtime_b200.ops.cuda import CudaOps

        keep.append(CudaOps())
    return keep[0]


def _step(s):
    from qwen3_runtime_b200.parts.base import StepContext

    n = s["new"]
    return StepContext(num_tokens=sum(n), num_seqs=len(n), token_ids=s["positions"], positions=s["positions"], token_seq=s["token_seq"],
                       cu_seqlens=s["cu"], kv_lens=s["lens"], state_slots=s["lens"], block_tables=[s["table"]], logit_rows=s["positions"],
                       num_logit_rows=0, max_query_len=max(n), max_kv_len=max(s["kv"]), decode_only=max(n) == 1, kv_longest=s["longest"],
                       single_seqs=s["singles"], num_single=s["num_singles"], host_cu_seqlens=s["host_cu"], host_kv_lens=s["kv"])


def _run_own(s):
    ops, case, step = _ops(), s["case"], _step(s)
    H, D, qkv = case["heads"], case["dim"], s["qkv"]
    sizes = dict(num_kv_heads=case["kv_heads"], head_dim=D, page_size=case["page"], pages=s["pages"], block_table=s["table"])
    out = torch.empty((qkv.shape[0], H * D), dtype=qkv.dtype, device=DEV)
    if case["kind"] == "store":
        ops.qk_norm_rope_store_8bit(qkv, num_heads=H, q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, cos=s["cos"], sin=s["sin"],
                                    step=step, q_out=out, **sizes)
        return (out, *ops.unpack_8bit(kv_lens=s["lens"], max_kv_len=max(s["kv"]), dtype=qkv.dtype, **sizes))
    ops.paged_attention_8bit(qkv, qkv.stride(0), num_heads=H, out=out, scale=D ** -0.5, window=case.get("window"),
                             keep_first=case.get("first") or 0, step=step, **sizes)
    return out


# ---- the plain form ------------------------------------------------------------------------------------------------------------


def _pieces(D, page):
    """Where channel d of row r lies in the row, ``[page, D]``."""
    mask = {64: 3, 128: 7, 256: 7}.get(D, 0)
    row, d = torch.arange(page, device=DEV)[:, None], torch.arange(D, device=DEV)
    return ((d // 16) ^ (row & mask)) * 16 + d % 16


def _four_bits(x):
    """float32 rounded to 4 significant bits, half ways to even; NaN where it or the result is not finite."""
    bits = x.contiguous().view(torch.int32)
    y = ((bits + 0x7FFFF + ((bits >> 20) & 1)) & ~0xFFFFF).view(torch.float32)
    return torch.where(torch.isfinite(x) & torch.isfinite(y), y, float("nan"))


def _parts(pages, D, page):
    """Views of the pages' codes ``[pages, heads, page, D]`` (keys', values') and scales ``[pages, heads, 2]``."""
    keys, values = [pages[:, :, k * page * D:(k + 1) * page * D].unflatten(2, (page, D)) for k in range(2)]
    return keys, values, pages[:, :, 2 * page * D:2 * page * D + 8]


def _write_pages(pages, at, rows, there, new):
    """Pages ``at`` get ``rows`` (keys and values ``[n, heads, page, D]`` of 4 significant bits) where ``there`` ``[n, heads, page, 1]``;
    ``new``: which of them the step brings (None: all of them); the scale of a page that held others before grows if it has to."""
    heads, page, D = rows[0].shape[1:]
    keys, values, scales = _parts(pages, D, page)
    held = scales[at].contiguous().view(torch.float32)  # [n, heads, 2]
    order = _pieces(D, page).expand(len(at), heads, page, D)
    grown = []
    for k, (part, x) in enumerate(zip((keys, values), rows)):
        most = torch.where(there & torch.isfinite(x), x.abs(), 0.0).amax((2, 3))
        mantissa, exponent = torch.frexp(most)
        power = torch.where(most > 0, exponent - 9 + (mantissa > 0.875).int(), -100).clamp(min=-100)  # 448 = 0.875 * 2^9
        s = torch.ldexp(torch.ones_like(most), power)
        if new is not None:
            s = torch.where((there & ~new).any(2)[..., 0], torch.maximum(s, held[..., k]), s)
        y = x / s[..., None, None]
        y = torch.where(y.abs() < 2.0**-6, (y * 512).trunc() / 512, y)
        code = y.to(torch.float8_e4m3fn).view(torch.uint8)
        code = torch.where(torch.isnan(y), (code & 0x80) | 0x7F, code)
        part[at] = torch.where(there, torch.empty_like(code).scatter_(3, order, code), part[at])
        grown.append(s)
    scales[at] = torch.stack(grown, -1).contiguous().view(torch.uint8)


def _values(pages, D, page):
    """Keys and values ``[pages, heads, page, D]`` in float32."""
    keys, values, scales = _parts(pages, D, page)
    scale = scales.contiguous().view(torch.float32)
    order = _pieces(D, page).expand(*keys.shape)
    return [part.gather(3, order).view(torch.float8_e4m3fn).float() * scale[:, :, k, None, None] for k, part in enumerate((keys, values))]


def _rotated(x, weight, cos, sin):
    """Rows ``[tokens, heads, D]``: RMS norm, then element i and i + D / 2 turn by the token's angles."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_store(s):
    case = s["case"]
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    at = s["positions"].long()
    x = s["qkv"].float().unflatten(1, (-1, D))
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = _rotated(x[:, :H], s["q_weight"], cos, sin)
    k = _rotated(x[:, H:H + G], s["k_weight"], cos, sin)
    # the pages that get tokens, in the order of (sequence, page): what they hold, with the new tokens put in
    width = s["table"].shape[1]
    where, index = (s["token_seq"].long() * width + at // page).unique(return_inverse=True)
    ids = s["table"].flatten()[where].long()
    past = s["lens"][where // width] - s["cu"].diff()[where // width]  # the sequence's tokens before the step
    slot = torch.arange(page, device=DEV)
    old = ((where % width)[:, None] * page + slot < past[:, None])[:, None, :, None].expand(-1, G, -1, 1)
    fresh = torch.zeros_like(old)
    fresh[index, :, at % page] = True
    rows = [torch.where(old, held, 0.0) for held in _values(s["pages"][ids], D, page)]
    for part, y in zip(rows, (k, x[:, H + G:])):
        part[index, :, at % page] = _four_bits(y)
    _write_pages(s["pages"], ids, rows, old | fresh, fresh)
    n = -(-max(s["kv"]) // page)
    table = s["table"][:, :n].long().flatten()
    keep = (torch.arange(n * page, device=DEV) < s["lens"][:, None]).view(-1, 1, page, 1)
    return (q.flatten(1).to(_dtype(case)), *[torch.where(keep, y, 0.0).to(_dtype(case)) for y in _values(s["pages"][table], D, page)])


def _run_attention(s):
    case = s["case"]
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    R = H // G
    B, n, L = len(s["kv"]), max(s["new"]), max(s["kv"])
    slot = torch.arange(L, device=DEV)
    table = s["table"][:, : -(-L // page)]
    live = (slot[None, :] < s["lens"][:, None]) & (table[:, slot // page] >= 0)
    k, v = [torch.where(live[:, None, :, None], x.unflatten(0, (B, -1)).transpose(1, 2).flatten(2, 3)[:, :, :L], 0.0)
            for x in _values(s["pages"][table.clamp(min=0).long().flatten()], D, page)]  # [B, G, L, D]
    seq, at = s["token_seq"].long(), s["positions"].long()
    place = torch.arange(at.numel(), device=DEV) - s["cu"].long()[seq]  # a token's row among its sequence's new ones
    q = torch.zeros((B, n, H, D), device=DEV)
    q[seq, place] = s["qkv"][:, : H * D].float().unflatten(1, (H, D))
    where = torch.full((B, n), -1, dtype=torch.long, device=DEV)
    where[seq, place] = at
    sees = live[:, None] & (slot <= where[..., None])  # [B, n, L]
    if case.get("window"):
        sees = sees & ((slot > where[..., None] - case["window"]) | (slot < case["first"]))
    q = q.unflatten(2, (G, R)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, G, R n, D]
    score = (q @ k.transpose(2, 3)).mul_(D ** -0.5).unflatten(2, (R, n))
    score.masked_fill_(~sees[:, None, None], float("-inf"))
    score = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    score.div_(score.sum(-1, keepdim=True).clamp(min=1e-30))
    return (score.flatten(2, 3) @ v).unflatten(2, (R, n)).permute(0, 3, 1, 2, 4)[seq, place].flatten(1).to(_dtype(case))


def run(state):
    if own:
        return _run_own(state)
    return _run_store(state) if state["case"]["kind"] == "store" else _run_attention(state)


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------------


def _cache64(pages, table, length, D, page):
    """Keys and values ``[heads, length, D]`` of one sequence, read from the bytes; zero where it has no page."""
    ids = table[: -(-length // page)].long()
    rows = pages[ids.clamp(min=0)]
    swap = {64: 3, 128: 7, 256: 7}.get(D, 0)
    out = []
    for which in range(2):
        code = rows[:, :, which * page * D:(which + 1) * page * D].reshape(*rows.shape[:2], page, D // 16, 16).long()
        straight = torch.empty_like(code)
        for r in range(page):
            for p in range(D // 16):
                straight[:, :, r, p] = code[:, :, r, p ^ (r & swap)]
        straight = straight.flatten(-2)
        sign = 1.0 - 2.0 * (straight // 128).double()
        exponent, mantissa = (straight // 8) % 16, (straight % 8).double()
        value = torch.where(exponent > 0, (1.0 + mantissa / 8) * 2.0 ** (exponent - 7).double(), mantissa * 2.0**-9)
        value = torch.where(straight % 128 == 127, math.nan, sign * value)
        at = 2 * page * D + 4 * which
        scale = rows[:, :, at:at + 4].contiguous().view(torch.float32).double()
        value = torch.where((ids >= 0)[:, None, None, None], value * scale[..., None], 0.0)
        out.append(value.permute(1, 0, 2, 3).reshape(rows.shape[1], -1, D)[:, :length])
    return out


def _held64(x, page):
    """What a sequence's tokens ``[heads, length, D]`` stand for once they are held (those that were held before stay, or are cut)."""
    mantissa, exponent = torch.frexp(x)
    x = torch.ldexp(torch.round(mantissa * 16.0), exponent - 4)
    length = x.shape[1]
    tiles = torch.nn.functional.pad(x, (0, 0, 0, -length % page)).unflatten(1, (-1, page))
    most = tiles.abs().amax((2, 3), keepdim=True)
    power = torch.full_like(most, -100.0)
    some = most > 0
    power[some] = torch.ceil(torch.log2(most[some] / 448.0)).clamp(min=-100)
    s = 2.0**power
    y = tiles / s
    y = torch.where(y.abs() < 2.0**-6, torch.trunc(y * 512.0) / 512.0, y) * s
    return y.flatten(1, 2)[:, :length]


def _exact_store(s):
    case = s["case"]
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    width = -(-max(s["kv"]) // page)
    q, keys, values = [], [], []
    for b, (c, n) in enumerate(zip(s["context"], s["new"])):
        x = s["qkv"][s["host_cu"][b]:s["host_cu"][b] + n].double().reshape(n, H + 2 * G, D)
        turned = []
        for rows, weight in ((x[:, :H], s["q_weight"]), (x[:, H:H + G], s["k_weight"])):
            y = rows / (rows.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
            cos, sin = s["cos"][c:c + n].double()[:, None], s["sin"][c:c + n].double()[:, None]
            first, second = y[..., : D // 2], y[..., D // 2:]
            turned.append(torch.cat((first * cos - second * sin, first * sin + second * cos), -1))
        q.append(turned[0].reshape(n, H * D))
        old = _cache64(s["pages"], s["table"][b], c, D, page) if c else [x.new_zeros((G, 0, D))] * 2
        for all_rows, past, fresh in ((keys, old[0], turned[1]), (values, old[1], x[:, H + G:])):
            held = _held64(torch.cat((past, fresh.transpose(0, 1)), 1), page)
            held = torch.nn.functional.pad(held, (0, 0, 0, width * page - c - n))
            all_rows.append(held.reshape(G, width, page, D).transpose(0, 1))
    return torch.cat(q), torch.cat(keys), torch.cat(values)


def _exact_attention(s):
    case = s["case"]
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    window, kept, scale = case.get("window") or 0, case.get("first") or 0, 1.0 / math.sqrt(D)
    outs = []
    for b, (c, n) in enumerate(zip(s["context"], s["new"])):
        k, v = _cache64(s["pages"], s["table"][b], c + n, D, page)
        key = torch.arange(c + n, device=DEV)
        if window:  # what no new token sees is left out
            key = key[(key > c - window) | (key < kept)]
            k, v = k[:, key], v[:, key]
        q = s["qkv"][s["host_cu"][b]:s["host_cu"][b] + n, : H * D].double().reshape(n, G, H // G, D)
        me = torch.arange(c, c + n, device=DEV)[:, None]
        hidden = key > me
        if window:
            hidden = hidden | ((key <= me - window) & (key >= kept))
        rows = torch.empty((n, G, H // G, D), dtype=torch.float64, device=DEV)
        for h in range(G):
            score = torch.einsum("nrd,kd->nrk", q[:, h], k[h]) * scale
            weight = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1)
            rows[:, h] = torch.einsum("nrk,kd->nrd", weight, v[h])
        outs.append(rows.reshape(n, H * D))
    return torch.cat(outs)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_store(s) if case["kind"] == "store" else _exact_attention(s)
