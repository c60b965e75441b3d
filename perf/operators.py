"""The operators around a key/value cache that is held in 4 bits, as cases that can be timed and compared.

A page of such a cache keeps, for each of its key/value heads, one record: the keys' codes, the values' codes, the keys' parameters
and the values' parameters of its tokens.  A head of ``D`` channels is ``G`` equal groups (the fewest of at most 64 channels, each of
whole words of 8); a group is 4-bit numbers ``n`` and a scale and a minimum in bfloat16, and stands for ``minimum + n * scale``.
A token's codes are ``D / 8`` words of 32 bits: word ``i`` holds channels ``8 (i // G)`` to ``8 (i // G) + 7`` of group ``i % G``,
the first in its lowest bits.

* ``store``    -- a step's queries, keys and values behind the projection: norm, rotation, the cache write; then the sequences'
                  values as the attention over prompts reads them
* ``attention`` -- every token of a step over its sequence's tokens: single tokens, portions of prompts, or both
* ``mass``     -- attention, and the weights that the step's last tokens give to each cached token added to its sum
* ``evict``    -- sequences that hold more than a budget keep their first and last tokens and those with the largest sums;
                  then the kept tokens' values
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    b8 = ",".join(["4096"] * 8)
    ragged = ",".join(str(64 + 83 * i) for i in range(48))
    return [
        # eight requests' next tokens written behind short contexts: the smallest write
        dict(name="store_decode", kind="store", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="40,41,42,43,44,45,46,47", new="1,1,1,1,1,1,1,1"),
        # a step that takes several prompts at once, one of them a later portion
        dict(name="store_prompts", kind="store", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="0,0,2048,0", new="1500,701,1024,33"),
        # one user reading along: the least work, where latency counts
        dict(name="attention_one", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16", context="512", new="1", window=0),
        # the package's default benchmark point: eight requests behind 4,096 tokens each
        dict(name="attention_batch", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context=b8, new=",".join(["1"] * 8), window=0),
        # a few requests behind long documents, what a cache in 4 bits is made for: the largest case
        dict(name="attention_long", kind="attention", heads=64, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="32768,32768,31111,29999,32768,17001,32000,30001", new="1,1,1,1,1,1,1,1", window=0),
        # prompts: two new ones, a later portion of a third, and a request that decodes beside them
        dict(name="attention_prompts", kind="attention", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context="0,0,2048,700", new="1500,701,1000,1", window=0),
        # the 32-bit path, which checks the 16-bit one
        dict(name="attention_float32", kind="attention", heads=16, kv_heads=4, dim=64, page=16, dtype="float32",
             context="300,77", new="20,1", window=0),
        # decoding with sums: requests of unequal lengths
        dict(name="mass_decode", kind="mass", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16", context=ragged,
             new=",".join(["1"] * 48), observe=1),
        # a prompt whose last tokens' weights are summed
        dict(name="mass_prompt", kind="mass", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16", context="0", new="2048", observe=32),
        # one request that has passed its budget by a little
        dict(name="evict_one", kind="evict", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16", context="1088", keep=1024,
             first=4, recent=64),
        # many requests behind prompts of unequal lengths, cut to a budget
        dict(name="evict_batch", kind="evict", heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16",
             context=",".join(str(900 + 467 * i) for i in range(16)), keep=2000, first=16, recent=256),
    ]


# query heads, key/value heads, head size
_HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (16, 4, 128), (16, 8, 64), (40, 8, 128), (16, 2, 256), (16, 1, 64), (20, 4, 80)]


def _spread(rng, low, high):
    """A whole number in low..high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    kind = rng.choice(["store", "attention", "attention", "attention", "mass", "mass", "evict"])
    H, G, D = rng.choice(_HEADS)
    case = dict(kind=kind, heads=H, kv_heads=G, dim=D, page=rng.choice([16, 16, 16, 8, 32, 64, 24, 5]), dtype="bfloat16")
    if kind == "evict":
        n = _spread(rng, 1, 16)
        keep = _spread(rng, 64, 4096)
        first = rng.choice([0, 1, 4, 16])
        return dict(case, context=_text(rng.randint(max(1, keep // 2), 3 * keep) for _ in range(n)), keep=keep, first=first,
                    recent=rng.randint(1, keep // 2))
    if rng.random() < 0.5:  # next tokens
        n = _spread(rng, 1, 64)
        most = _spread(rng, 64, min(32768, 131072 // n)) if kind != "store" else 200
        case.update(context=_text(rng.randint(most // 8, most) for _ in range(n)), new=_text([1] * n))
    else:  # portions of prompts, single tokens among them
        n = rng.randint(1, 4)
        case.update(context=_text(rng.choice([0, 0, rng.randint(1, 2000)]) for _ in range(n)),
                    new=_text(rng.choice([1, _spread(rng, 2, 40), _spread(rng, 17, 1000), _spread(rng, 17, 1000)]) for _ in range(n)))
    if kind == "attention":
        case["window"] = rng.choice([0, 0, 0, rng.randint(1, 2000)])
        if rng.random() < 0.2:
            case.update(dtype="float32", context=_text(min(int(c), 700) for c in case["context"].split(",")),
                        new=_text(min(int(c), 100) for c in case["new"].split(",")))
    if kind == "mass":
        case["observe"] = rng.choice([1, 8, 32, 64])
    return case


# ---- sizes ---------------------------------------------------------------------------------------------------------------


def _numbers(text):
    return [int(x) for x in text.split(",")]


def _lengths(case):
    """Cached tokens and new tokens of every sequence."""
    context = _numbers(case["context"])
    return context, _numbers(case["new"]) if "new" in case else [0] * len(context)


def _groups(D):
    words = D // 8
    return next(g for g in range(-(-D // 64), words + 1) if words % g == 0)


def _record(D, page):
    """Bytes of one page and head."""
    return -(-page * (D + 8 * _groups(D)) // 16) * 16


def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    e = 4 if case["dtype"] == "float32" else 2
    token = G * (D + 8 * _groups(D))  # bytes of a cached token's keys and values
    context, new = _lengths(case)
    T = sum(new)
    kv = [c + n for c, n in zip(context, new)]
    if case["kind"] == "store":
        # the projection read, queries and the new tokens' records written; then every token read and its values written
        return {"bytes": T * ((2 * H + 2 * G) * D * e + token) + sum(kv) * (token + 2 * G * D * e), "flops": 8 * T * (H + 2 * G) * D}
    if case["kind"] == "evict":
        moved = kept = 0
        for c in kv:
            kept += min(c, case["keep"])
            if c > case["keep"]:  # as many leave the first places as the share of tokens that goes
                moved += (case["keep"] - case["first"]) * (c - case["keep"]) / c
        return {"bytes": sum(kv) * G * 8 + 2 * moved * (token + 8 * G) + kept * (token + 2 * G * D * e), "flops": sum(kv) * G}
    window = case.get("window") or 0
    pairs = read = 0
    for c, n in zip(context, new):
        read += min(c + n, window + n - 1) if window else c + n
        pairs += sum(min(c + i + 1, window) if window else c + i + 1 for i in range(n))
    out = {"bytes": read * token + 2 * T * H * D * e, "flops": 4 * H * D * pairs}
    if case["kind"] == "mass":
        seen = sum(c + i + 1 for c, n in zip(context, new) for i in range(max(0, n - case["observe"]), n))
        out["bytes"] += sum(kv) * G * 8
        out["flops"] += H * seen
    return out


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
    at = 0
    window = case.get("window") or 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        if window:  # pages that every new token's window has passed were given back
            table[b, : max(0, context[b] - window + 1) // page] = -1
        at += n
    pages = torch.empty((count + 1, G, _record(D, page)), dtype=torch.uint8, device=DEV)
    pages.fill_(255)  # the spare page, and rows behind a sequence's last token: codes of 15, parameters that are not numbers
    loud = 1.0 + 3.0 * (torch.rand((1, 1, D), generator=g, device=DEV) < 0.05)  # some channels are larger than others, as keys' are
    for lo in range(0, count, 2048):  # in portions: less memory
        n = min(2048, count - lo)
        rows = [torch.randn((n * page, G, D), generator=g, device=DEV) for _ in range(2)]
        rows[0] *= loud
        _write(pages, lo + torch.arange(n * page, device=DEV) // page, torch.arange(n * page, device=DEV) % page, rows[0], rows[1], page)
    table = table.to(DEV)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    state = dict(case=case, kv=kv, new=new, context=context, table=table, lens=lens)
    # the rows behind each sequence's last token (the new tokens' own, where the step writes them)
    end = lens if case["kind"] != "store" else torch.tensor(context, dtype=torch.int32, device=DEV)
    slot = torch.arange(width * page, device=DEV)
    blank = (slot[None, :] >= end[:, None]) & (slot[None, :] < torch.tensor(need, device=DEV)[:, None] * page)
    b, s = blank.nonzero(as_tuple=True)
    at = table[b, s // page].long()
    for part in _sections(pages, D, page):
        part[at, :, s % page] = 255
    state["pages"] = pages
    if case["kind"] == "evict":
        # sums as many steps leave them: a few tokens with much, most with little, ties among those with none
        mass = torch.rand((count + 1, G, page), generator=g, device=DEV)
        mass = torch.where(mass < 0.1, torch.zeros_like(mass), -torch.log(mass) ** 3)
        places = torch.full((count + 1, G, page), -1, dtype=torch.int32, device=DEV)
        b, s = (slot[None, :] < lens[:, None]).nonzero(as_tuple=True)
        places[table[b, s // page].long(), :, s % page] = s.int()[:, None]
        return dict(state, mass=mass.abs(), places=places)
    state["positions"] = torch.tensor([c + i for c, n in zip(context, new) for i in range(n)], dtype=torch.int32, device=DEV)
    state["token_seq"] = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], dtype=torch.int32, device=DEV)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    singles = [b for b, n in enumerate(new) if n == 1]
    state.update(host_cu=cu, cu=torch.tensor(cu, dtype=torch.int32, device=DEV), longest=torch.tensor([max(kv)], dtype=torch.int32, device=DEV),
                 singles=torch.tensor(singles, dtype=torch.int32, device=DEV), num_singles=len(singles))
    rows = torch.randn((T, (H + 2 * G) * D), generator=g, device=DEV)
    state["qkv"] = rows.to(_dtype(case))
    if case["kind"] == "store":
        state["q_weight"] = 1.0 + 0.1 * torch.randn((D,), generator=g, device=DEV)
        state["k_weight"] = 1.0 + 0.1 * torch.randn((D,), generator=g, device=DEV)
        angle = torch.arange(max(kv), device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    if case["kind"] == "mass":
        state["mass"] = torch.rand((count + 1, G, page), generator=g, device=DEV)
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
    ops, case = _ops(), s["case"]
    sizes = dict(num_kv_heads=case["kv_heads"], head_dim=case["dim"], page_size=case["page"])
    if case["kind"] == "evict":
        mass, places = s["mass"].clone(), s["places"].clone()
        ops.evict_4bit(pages=s["pages"], mass=mass, places=places, block_table=s["table"], kv_lens=s["lens"], max_kv_len=max(s["kv"]),
                       keep=case["keep"], first=case["first"], recent=case["recent"], **sizes)
        k, v = ops.unpack_4bit(s["pages"], block_table=s["table"], kv_lens=s["lens"], max_kv_len=min(max(s["kv"]), case["keep"]),
                               dtype=_dtype(case), **sizes)
        return mass, places, k, v
    H, D = case["heads"], case["dim"]
    qkv, T = s["qkv"], s["qkv"].shape[0]
    if case["kind"] == "store":
        q = torch.empty((T, H * D), dtype=qkv.dtype, device=DEV)
        ops.qk_norm_rope_store_4bit(qkv, num_heads=H, q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, cos=s["cos"], sin=s["sin"],
                                    positions=s["positions"], token_seq=s["token_seq"], block_table=s["table"], pages=s["pages"], q_out=q,
                                    **sizes)
        return (q, *ops.unpack_4bit(s["pages"], block_table=s["table"], kv_lens=s["lens"], max_kv_len=max(s["kv"]), dtype=qkv.dtype, **sizes))
    step, scale = _step(s), D ** -0.5
    out = torch.empty((T, H * D), dtype=qkv.dtype, device=DEV)
    lse = None
    if case["kind"] == "mass" and step.decode_only and ops.decode_4bit_ok(qkv, H, case["kv_heads"], D):  # (other sizes have no log sums)
        lse = torch.empty((T, H), dtype=torch.float32, device=DEV)
    ops.paged_attention_4bit(qkv, qkv.stride(0), num_heads=H, pages=s["pages"], block_table=s["table"], out=out, scale=scale,
                             window=case.get("window") or None, step=step, lse=lse, **sizes)
    if case["kind"] == "attention":
        return out
    mass = s["mass"].clone()
    ops.attention_mass_4bit(qkv, qkv.stride(0), num_heads=H, pages=s["pages"], mass=mass, block_table=s["table"], scale=scale, step=step,
                            observe=case["observe"], lse=lse, **sizes)
    return out, mass


# ---- the plain form ------------------------------------------------------------------------------------------------------------


def _sections(pages, D, page):
    """Views of the pages' four parts: key codes, value codes ``[pages, heads, page, D / 2]`` and both parameters ``[.., 4 * groups]``, in bytes."""
    half, par = D // 2, 4 * _groups(D)
    ends = [0, page * half, 2 * page * half, page * (2 * half + par), page * (2 * half + 2 * par)]
    return [pages[:, :, a:b].unflatten(2, (page, -1)) for a, b in zip(ends, ends[1:])]


def _toward(x, up):
    """The nearest bfloat16 that is not above (``up``: not below) each float32, as float32."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    away = (bits != cut) & ((x > 0) if up else (x < 0))  # cutting goes towards zero
    return torch.where(torch.isfinite(x), cut + away.int() * 65536, bits).view(torch.float32)


def _codes(x):
    """4-bit numbers, scales and minima of rows ``[..., D]``."""
    rows = x.float().unflatten(-1, (_groups(x.shape[-1]), -1))
    low, high = rows.amin(-1, keepdim=True), rows.amax(-1, keepdim=True)
    z = _toward(low, up=False)
    s = _toward((high - z) / torch.full_like(z, 15.0), up=True)  # a division: the inverse of 15 has no end, and exact quotients are common
    bad = ~torch.isfinite(s) | ~torch.isfinite(z)
    n = torch.where(bad | (s == 0), 0.0, ((rows - z) / s)).round().clamp(0, 15).to(torch.uint8)
    nan = torch.full_like(s, float("nan"))
    return n, torch.where(bad, nan, s), torch.where(bad, nan, z)


def _write(pages, page_of, row_of, k, v, page):
    """Rows ``[tokens, heads, D]`` into their pages."""
    D = k.shape[-1]
    kc, vc, kp, vp = _sections(pages, D, page)
    n, s, z = _codes(torch.stack([k, v]))
    words = n.unflatten(-1, (-1, 8)).transpose(-3, -2).flatten(-3)  # the groups' words in turn
    code = words[..., 0::2] | (words[..., 1::2] << 4)
    par = torch.cat([s, z], -1).to(torch.bfloat16).flatten(-2).contiguous().view(torch.uint8)
    kc[page_of, :, row_of], vc[page_of, :, row_of] = code[0], code[1]
    kp[page_of, :, row_of], vp[page_of, :, row_of] = par[0], par[1]


def _values(pages, D, page):
    """Keys and values ``[pages, heads, page, D]`` in float32."""
    kc, vc, kp, vp = _sections(pages, D, page)
    out = []
    for code, par in ((kc, kp), (vc, vp)):
        n = torch.stack([code & 15, code >> 4], -1).flatten(-2)
        n = n.unflatten(-1, (-1, _groups(D), 8)).transpose(-3, -2).flatten(-2).float()
        s, z = par.contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2)).split(1, -1)
        out.append((z + n * s).flatten(-2))
    return out


def _unpacked(s, lens, pages_of, D, page):
    """Values of every sequence's pages, one after the other; zero behind a sequence's last token."""
    table = s["table"][:, :pages_of].clamp(min=0).long().flatten()
    row = torch.arange(pages_of * page, device=DEV)
    keep = (row[None, :] < lens[:, None]).view(-1, 1, page, 1)
    return [torch.where(keep, x, 0.0).to(_dtype(s["case"])) for x in _values(s["pages"][table], D, page)]


def _run_evict(s):
    case = s["case"]
    D, page, keep = case["dim"], case["page"], case["keep"]
    mass, places = s["mass"].clone(), s["places"].clone()
    table, lens = s["table"], s["lens"]
    slot = torch.arange(max(s["kv"]), device=DEV)
    page_of, row_of = table[:, slot // page].long(), slot % page  # [B, L], [L]
    live = (slot[None, :] < lens[:, None])[:, None]  # [B, 1, L]
    held = mass[page_of, :, row_of].transpose(1, 2)  # [B, heads, L]
    place = places[page_of, :, row_of].transpose(1, 2)
    newest = torch.where(live, place, -1).amax(-1, keepdim=True)
    forced = live & ((place < case["first"]) | (place > newest - case["recent"]))
    key = torch.where(forced, float("inf"), torch.where(live, held, -1.0))
    order = key.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    kept = live & (rank < keep)
    over = (lens > keep)[:, None, None]
    hole, mover = over & ~kept & (slot < keep) & live, over & kept & (slot >= keep)
    b, h, to = hole.nonzero(as_tuple=True)
    b2, h2, at = mover.nonzero(as_tuple=True)  # as many in every (sequence, head), in the same order
    src, dst = (page_of[b2, at], h2, at % page), (page_of[b, to], h, to % page)
    for part in (*_sections(s["pages"], D, page), mass, places):
        part[dst] = part[src]
    left = lens.clamp(max=keep)
    return (mass, places, *_unpacked(s, left, -(-min(max(s["kv"]), keep) // page), D, page))


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
    _write(s["pages"], s["table"][s["token_seq"].long(), at // page].long(), at % page, k, x[:, H + G:], page)
    return (q.flatten(1).to(_dtype(case)), *_unpacked(s, s["lens"], -(-max(s["kv"]) // page), D, page))


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
        sees = sees & (slot > where[..., None] - case["window"])
    q = q.unflatten(2, (G, R)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, G, R n, D]
    score = (q @ k.transpose(2, 3)).mul_(D ** -0.5).unflatten(2, (R, n))
    score.masked_fill_(~sees[:, None, None], float("-inf"))
    score = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    score.div_(score.sum(-1, keepdim=True).clamp(min=1e-30))
    out = (score.flatten(2, 3) @ v).unflatten(2, (R, n)).permute(0, 3, 1, 2, 4)[seq, place].flatten(1).to(_dtype(case))
    if case["kind"] == "attention":
        return out
    count = s["cu"].long().diff()
    seen = (torch.arange(n, device=DEV) >= (count - case["observe"])[:, None]).float()  # [B, n]
    share = (score * seen[:, None, None, :, None]).sum((2, 3))  # [B, G, L]
    mass = s["mass"].clone()
    b, j = live.nonzero(as_tuple=True)
    mass[table[b, j // page].long(), :, j % page] += share[b, :, j]
    return out, mass


def run(state):
    if own:
        return _run_own(state)
    return {"store": _run_store, "evict": _run_evict}.get(state["case"]["kind"], _run_attention)(state)


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------------


def _codes64(x):
    """What rows ``[rows, D]`` stand for once they are held in 4 bits."""
    D = x.shape[-1]
    x = x.reshape(x.shape[0], _groups(D), D // _groups(D))

    def bf16(v, up):
        mantissa, exponent = torch.frexp(v)
        m = mantissa * 256.0
        return torch.ldexp(torch.ceil(m) if up else torch.floor(m), exponent - 8)

    z = bf16(x.min(-1, keepdim=True).values, False)
    s = bf16((x.max(-1, keepdim=True).values - z) / 15.0, True)
    n = torch.round((x - z) / torch.where(s > 0, s, torch.ones_like(s))).clamp(0, 15)
    return (z + n * s).reshape(-1, D)


def _cache64(pages, table, length, D, page, dead=0):
    """Keys and values ``[heads, length, D]`` of one sequence, read from the bytes; the first ``dead`` rows' pages are gone."""
    G, half, words = _groups(D), D // 2, D // 8
    size = D // G
    channel = np.empty((words, 8), dtype=np.int64)  # which channel each 4-bit place holds
    for i in range(words):
        channel[i] = (i % G) * size + 8 * (i // G) + np.arange(8)
    channel = torch.from_numpy(channel.reshape(-1)).to(pages.device)
    rows = pages[table[: -(-length // page)].clamp(min=0).long()]
    out = []
    for which in range(2):
        code = rows[:, :, which * page * half:(which + 1) * page * half].reshape(*rows.shape[:2], page, half).to(torch.int64)
        n = torch.zeros((*code.shape[:3], D), dtype=torch.float64, device=pages.device)
        n[..., channel[0::2]] = (code % 16).double()
        n[..., channel[1::2]] = (code // 16).double()
        base = 2 * page * half + which * page * 4 * G
        par = rows[:, :, base:base + page * 4 * G].reshape(*rows.shape[:2], page, G, 4).to(torch.int64)
        s, z = [((par[..., 2 * i] + 256 * par[..., 2 * i + 1]) << 16).to(torch.int32).view(torch.float32).double() for i in range(2)]
        value = z.repeat_interleave(size, -1) + n * s.repeat_interleave(size, -1)
        out.append(value.permute(1, 0, 2, 3).reshape(rows.shape[1], -1, D)[:, :length])
    return out


def _pages64(per_sequence, width, page):
    """Sequences' rows ``[heads, length, D]`` laid out in pages ``[sequences * width, heads, page, D]``, zero behind each."""
    out = []
    for x in per_sequence:
        x = torch.nn.functional.pad(x, (0, 0, 0, width * page - x.shape[1]))
        out.append(x.reshape(x.shape[0], width, page, -1).transpose(0, 1))
    return torch.cat(out)


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
            held = _codes64(fresh.transpose(0, 1).reshape(G * n, D)).reshape(G, n, D)
            all_rows.append(torch.cat((past, held), 1))
    return (torch.cat(q), _pages64(keys, width, page), _pages64(values, width, page))


def _exact_attention(s):
    case = s["case"]
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    window, scale = case.get("window") or 0, 1.0 / math.sqrt(D)
    outs = []
    mass = s["mass"].double() if "mass" in s else None
    for b, (c, n) in enumerate(zip(s["context"], s["new"])):
        k, v = _cache64(s["pages"], s["table"][b], c + n, D, page)
        first = max(0, c - window + 1) if window else 0
        k, v = k[:, first:], v[:, first:]
        q = s["qkv"][s["host_cu"][b]:s["host_cu"][b] + n, : H * D].double().reshape(n, G, H // G, D)
        key = torch.arange(first, c + n, device=DEV)
        me = torch.arange(c, c + n, device=DEV)[:, None]
        hidden = (key > me) | ((key <= me - window) if window else torch.zeros_like(key, dtype=torch.bool))
        total = torch.zeros((G, c + n - first), dtype=torch.float64, device=DEV)
        rows = torch.empty((n, G, H // G, D), dtype=torch.float64, device=DEV)
        for h in range(G):
            score = torch.einsum("nrd,kd->nrk", q[:, h], k[h]) * scale
            weight = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1)
            rows[:, h] = torch.einsum("nrk,kd->nrd", weight, v[h])
            if mass is not None:
                total[h] = weight[max(0, n - case["observe"]):].sum((0, 1))
        outs.append(rows.reshape(n, H * D))
        if mass is not None:
            for h in range(G):
                mass[s["table"][b, key // page].long(), h, key % page] += total[h]
    return torch.cat(outs) if mass is None else (torch.cat(outs), mass)


def _exact_evict(s):
    case = s["case"]
    G, D, page, keep = case["kv_heads"], case["dim"], case["page"], case["keep"]
    mass, places = s["mass"].cpu().numpy().copy(), s["places"].cpu().numpy().copy()
    table = s["table"].cpu().numpy()
    width = -(-min(max(s["kv"]), keep) // page)
    keys, values = [], []
    for b, length in enumerate(s["kv"]):
        k, v = _cache64(s["pages"], s["table"][b], length, D, page)
        source = np.tile(np.arange(min(length, keep)), (G, 1))  # the slot whose token each kept slot holds afterwards
        if length > keep:
            slot = np.arange(length)
            at = (table[b, slot // page], slot % page)
            for h in range(G):
                m, p = mass[at[0], h, at[1]], places[at[0], h, at[1]]
                stays = (p < case["first"]) | (p > p.max() - case["recent"])
                rest = slot[~stays]
                best = rest[np.lexsort((rest, -m[rest]))][: keep - int(stays.sum())]
                stays[best] = True
                source[h, np.flatnonzero(~stays[:keep])] = keep + np.flatnonzero(stays[keep:])
                to = (at[0][:keep], h, at[1][:keep])
                mass[to], places[to] = m[source[h]], p[source[h]]
        source = torch.from_numpy(source).to(DEV)[..., None].expand(-1, -1, D)
        keys.append(k.gather(1, source))
        values.append(v.gather(1, source))
    return (torch.from_numpy(mass).double(), torch.from_numpy(places), _pages64(keys, width, page), _pages64(values, width, page))


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "evict": _exact_evict}.get(case["kind"], _exact_attention)(s)
