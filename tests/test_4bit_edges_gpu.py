"""A cache in 4 bits on the GPU, at its edges: tokens that have no place, scores far from zero, single tokens of every head size from attention to
sums.  The tolerances are those of tests/test_4bit_gpu.py."""


import math

import pytest
import torch

import plain_4bit as p4
import test_4bit_gpu as t4
from test_4bit_gpu import BF16, F32, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("copies", [1, 400])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 80)])
@pytest.mark.parametrize("window", [None, 300])
def test_a_token_without_a_place_is_zero(ops, copies, dtype, D, window):  # noqa: F811
    """A token of no sequence, or whose place lies behind or in front of the table, sees nothing, whether a block goes through its slices
    or a second kernel joins them (few tokens); the others are as ever."""
    H, G, lens = 4, 2, [700, 700, 1100, 700, 900]
    c = p4.Cache(lens, G, D, 16, seed=D)
    n, new = len(lens) * copies, [1] * len(lens) * copies
    q = t4.queries(n, H, D, 3, dtype)
    table = c.table.repeat(copies, 1)
    args = dict(dtype=dtype, table=table, window=window)
    want = t4.attend(ops, c, q, new, lens * copies, H, D ** -0.5, **args)
    step = p4.step_of(new, lens * copies, 16)
    step.token_seq[0], step.token_seq[1] = -1, n
    step.positions[2], step.positions[3] = table.shape[1] * 16, -2
    got = t4.attend(ops, c, q, new, lens * copies, H, D ** -0.5, step=step, **args)
    assert bool((got[:4] == 0).all()) and torch.equal(got[4:], want[4:])


@pytest.mark.parametrize("H,G,D,dtype,slices", [(8, 2, 128, BF16, 1), (8, 2, 128, BF16, 3), (8, 2, 128, BF16, -3), (8, 1, 64, BF16, 2),
                                                (4, 2, 256, BF16, -2), (4, 2, 80, BF16, None), (4, 2, 64, F32, None), (4, 1, 128, F32, None)])
@pytest.mark.parametrize("sign", [-1, 1])
def test_scores_that_all_lie_far_from_zero(ops, H, G, D, dtype, slices, sign):  # noqa: F811
    """All scores of a row near -10^33 (or 10^33): the largest takes the row, as it does anywhere else.  A score is off by 2^-23 (D + 8) of
    the row's largest product sum (``score_error``); here the best key is twice as far from the next as two such errors, so it weighs one."""
    lens, scale = [70, 700], D ** -0.5

    def mutate(b, k, v):
        k.abs_()
        k *= sign * 1e16
        k[:, 33] *= 0.5 if sign < 0 else 2.0  # (the best key of most rows)

    c = p4.Cache(lens, G, D, 16, seed=D, mutate=mutate)
    q = (t4.queries(2, H, D, 3, F32).abs() * 1e17).to(dtype)
    rows = q.view(2, H, D)
    log_sums = dtype == BF16 and D in (64, 128, 256)
    got = t4.attend(ops, c, q, [1, 1], lens, H, scale, dtype=dtype, lse=log_sums, slices=slices)
    got, lse = got if log_sums else (got, None)
    for b in range(2):
        k, v = c.values(b)
        err = t4.score_error(rows[b:b + 1], c, b, scale)[0]
        num, s, z = (x.double() for x in c.v[b])
        s, z = s.repeat_interleave(D // s.shape[-1], -1), z.repeat_interleave(D // z.shape[-1], -1)
        spread = (z + 8 * s).abs() + s * (num - 8).abs()
        for h in range(H):
            x = (k[h // (H // G)] @ rows[b, h].double()) * scale
            best, next_best = x.topk(2).values.tolist()
            j = int(x.argmax())
            assert best - next_best > 4 * float(err[h])
            want = v[h // (H // G), j]
            tol = 2.0 ** -22 * spread[h // (H // G), j] if dtype == F32 else (2 * t4.U + 2.0 ** -14) * spread[h // (H // G), j] + t4.U * want.abs()
            assert bool(((got[b, h].double() - want).abs() <= tol).all()), (b, h)
            if log_sums:
                assert abs(float(lse[b, h]) - best) <= float(err[h]) + 2.0 ** -20 * abs(best)
    # a log sum of such rows is known to 2^-23 of itself only: sums stay within what the rows can give, none is lost to infinity
    for given in {None, lse}:
        mass = t4.mass_of(ops, c, q, [1, 1], lens, H, scale, 1, lse=None if given is None else given.cuda())
        assert bool((mass >= 0).all()) and bool((mass <= H // G).all()) and math.isfinite(float(mass.sum()))


@pytest.mark.parametrize("H,G,D,dtype", [(8, 2, 128, BF16), (8, 2, 64, BF16), (4, 2, 256, BF16), (20, 4, 80, BF16), (20, 1, 128, BF16), (4, 2, 16, BF16),
                                         (6, 2, 240, BF16), (8, 2, 128, F32), (4, 2, 80, F32)])
def test_single_tokens_from_attention_to_sums(ops, H, G, D, dtype):  # noqa: F811
    """As a layer under a token budget calls them: log sums are asked for where the decode kernel has them, elsewhere the sums make their own."""
    lens, page = [1, 16, 100, 333], 16
    c = p4.Cache(lens, G, D, page, seed=D)
    q = t4.queries(len(lens), H, D, 6, dtype)
    rows, new, scale = q.view(-1, H, D), [1] * len(lens), D ** -0.5
    ok = ops.decode_4bit_ok(q.cuda(), H, G, D)
    assert ok == (dtype == BF16 and D in (64, 128, 256) and H // G <= 16)
    got = t4.attend(ops, c, q, new, lens, H, scale, dtype=dtype, lse=ok)
    got, lse = got if ok else (got, None)
    t4.check_rows(got, rows, c, new, lens, scale, wide=not ok, dtype=dtype)
    start = torch.rand((c.pages.shape[0], G, page), generator=torch.Generator().manual_seed(1))
    mass = t4.mass_of(ops, c, q, new, lens, H, scale, 1, lse=None if lse is None else lse.cuda(), start=start)
    t4.check_mass(mass, rows, c, new, lens, scale, 1, start=start, dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [128, 256])
def test_the_order_of_a_writes_sums(ops, dtype, D):  # noqa: F811
    """Heads of 128 and 256, number for number: squares are summed four neighbours at a time, then eight channels of either half of the head
    with their counterparts, then by halves; products and sums of norm and rotation are rounded one by one.  Stated here by element-wise
    operations, which leave no order open."""
    H, G, page, T = 3, 2, 16, 400
    g = torch.Generator().manual_seed(D)
    qkv = torch.randn((T, (H + 2 * G) * D), generator=g).to(dtype).cuda()
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).cuda() for _ in range(2))
    angle = torch.arange(T)[:, None] * 1e4 ** (-torch.arange(0, D, 2) / D)
    cos, sin = angle.cos().contiguous().cuda(), angle.sin().contiguous().cuda()
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    table = torch.randperm(T // page, generator=g).int()[None].cuda()
    pages = torch.zeros((T // page, G, p4.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    q = torch.empty((T, H * D), dtype=dtype, device="cuda")
    ops.qk_norm_rope_store_4bit(qkv, num_heads=H, num_kv_heads=G, head_dim=D, q_weight=qw, k_weight=kw, eps=1e-6, cos=cos, sin=sin, positions=pos,
                                token_seq=torch.zeros_like(pos), block_table=table, pages=pages, page_size=page, q_out=q)
    x = qkv.float().view(T, -1, D)
    square = (x * x).unflatten(-1, (-1, 4))
    fours = square[..., 0] + square[..., 1]
    fours = fours + square[..., 2]
    fours = fours + square[..., 3]  # [T, heads, D / 4]: of channels 4i .. 4i + 3
    first, second = fours.chunk(2, -1)
    lanes = (first + second).unflatten(-1, (-1, 2))  # of each eight channels of a half: their first four, their last four
    while lanes.shape[-2] > 1:
        low, high = lanes.chunk(2, -2)
        lanes = low + high
    mean = (lanes[..., 0, 0] + lanes[..., 0, 1])[..., None] / D
    y = x * torch.rsqrt(mean + 1e-6)
    for rows, weight, name in ((y[:, :H], qw, "q"), (y[:, H:H + G], kw, "k")):
        a, b = (rows * weight).chunk(2, -1)
        c, s = cos[:, None], sin[:, None]
        left, right = a * c, b * s
        top = left - right
        left, right = b * c, a * s
        turned = torch.cat([top, left + right], -1)
        if name == "q":
            assert torch.equal(q.view(T, H, D), turned.to(dtype))
        else:
            keys = turned
    got = pages[table[0].long()]
    half, par = D // 2, 4 * p4.groups(D)
    for which, rows in enumerate((keys, x[:, H + G:])):
        n, scale, low = p4.quantise(rows.transpose(0, 1).reshape(G * T, D).cpu())
        words = n.view(G, T, p4.groups(D), -1, 8).transpose(2, 3).reshape(G, T, D)
        code = (words[..., 0::2] | (words[..., 1::2] << 4)).to(torch.uint8)
        params = torch.stack([scale, low], -1).reshape(G, T, -1).contiguous().view(torch.uint8)
        have = got[:, :, which * page * half:(which + 1) * page * half].reshape(-1, G, page, half).transpose(0, 1).reshape(G, T, half)
        base = 2 * page * half + which * page * par
        have_par = got[:, :, base:base + page * par].reshape(-1, G, page, par).transpose(0, 1).reshape(G, T, par)
        assert torch.equal(have.cpu(), code) and torch.equal(have_par.cpu(), params)
