"""A cache in 4 bits on the GPU: every kernel against the plain statements in tests/plain_4bit.py, at the sizes and masks where they can
go wrong.

Tolerances.  u = 2^-8 is half a step of bfloat16 relative to the value.  A decoded row rounds each weight times scale once (u s|n - 8| p)
and each weight once (u |z + 8 s| p) -- together at most 2 u p (|z + 8 s| + s |n - 8|) -- and the result once (u |o|).  A score is a sum of D
products in float32: it is off by at most ``score_error`` below, which moves a weight by a factor of exp(2 error).  Prompts read keys and values rounded to bfloat16 (u each) and round the weights and the result (u each)."""

import math

import pytest
import torch

import plain_4bit as p4

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from qwen3_runtime_b200.ops.cuda import CudaOps

    return CudaOps()


def sizes(c):
    return dict(num_kv_heads=c.G, head_dim=c.D, page_size=c.page)


def queries(T, H, D, seed, dtype=BF16, extra=0):
    """``[T, H * D + extra]`` rows (a projection's row may be wider than its queries)."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, H * D + extra), generator=g).to(dtype)


def score_error(q, cache, b, scale):
    """Bound of a score's error ``[T, H]``: D additions of float32 to sums of |q| s n, n at most 15, and of |q z|, whatever their order."""
    D = q.shape[2]
    s = cache.k[b][1].double().nan_to_num().amax()
    z = cache.k[b][2].double().abs().nan_to_num().amax()
    total = q.double().abs().sum(-1)
    return scale * 2.0 ** -23 * (D + 8) * total * (s * 16 + z)


def attend(ops, c, q, new, lens, H, scale, *, window=None, lse=False, slices=None, dtype=BF16, table=None, step=None):
    step = step or p4.step_of(new, lens, c.page)
    dev = q.cuda()
    T = dev.shape[0]
    out = torch.full((T, H * c.D), math.nan, dtype=dtype, device="cuda")
    sums = torch.full((T, H), math.nan, device="cuda") if lse else None
    ops.paged_attention_4bit(dev, dev.stride(0), num_heads=H, pages=c.pages.cuda(), block_table=(c.table if table is None else table).cuda(),
                             out=out, scale=scale, step=step, window=window, lse=sums, decode_slices=slices, **sizes(c))
    ops.raise_if_kernel_error()
    out = out.cpu().view(T, H, c.D)
    return (out, sums.cpu()) if lse else out


def check_rows(got, q, c, new, lens, scale, window=None, wide=False, dtype=BF16):
    """Every row of ``got`` within its bound."""
    want, lse, weights = p4.attention(q, c, new, lens, scale, window)
    R, t = q.shape[1] // c.G, 0
    for b, n in enumerate(new):
        k, v = c.values(b)
        num, s, z = (x.double() for x in c.v[b])
        size = c.D // s.shape[-1]
        s, z = s.repeat_interleave(size, -1), z.repeat_interleave(size, -1)
        spread = (z + 8 * s).abs() + s * (num - 8).abs()  # >= |v|
        for i in range(n):
            row = q[t]
            err = score_error(row[None], c, b, scale)[0]
            if wide:
                err = err + scale * U * row.double().abs().sum(-1) * k.abs().amax()
            if dtype == F32:
                err = scale * 2.0 ** -22 * (c.D + 8) * row.double().abs().sum(-1) * k.abs().amax()
            for h in range(q.shape[1]):
                w = weights[b][i, h]
                grow = math.expm1(min(20.0, 2 * float(err[h]))) * (w @ v[h // R].abs())
                if dtype == F32:
                    tol = grow + 2.0 ** -20 * (w @ v[h // R].abs()) + 2.0 ** -23 * want[t, h].abs()
                else:
                    tol = grow + (2 * U + 2.0 ** -14) * (w @ spread[h // R]) + U * want[t, h].abs() + 1e-30
                diff = (got[t, h].double() - want[t, h]).abs()
                assert bool((diff <= tol).all()), (b, i, h, float((diff / tol).max()))
            t += 1
    return want, lse, weights


# ---- rounding and layout -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 16), (256, 8), (16, 4), (32, 3), (48, 16), (80, 5), (176, 16), (240, 7)])
def test_values_are_written_by_the_definition(ops, dtype, D, page):
    """Without norm and rotation what is written is the projection itself: the same bytes as the plain form's, row by row, and nothing
    else is touched."""
    H, G, lens = 4, 2, [2 * page + 1, 3]
    g = torch.Generator().manual_seed(D)
    T = 7
    qkv = torch.randn((T, (H + 2 * G) * D), generator=g).to(dtype)
    qkv[0, H * D:H * D + 8] = 3.0  # some equal ones
    qkv[1, H * D:(H + 1) * D] = 0.75  # a group of one value: scale zero
    qkv[2, H * D:(H + 1) * D] = 0.0
    qkv[3, (H + G) * D:(H + G + 1) * D] *= 1e-30
    qkv[4, (H + G) * D + 5] = 1e30
    seq = [0, 0, 0, 1, 1, 0, 1]
    pos = [0, page, 2 * page, 0, 1, page - 1, 2]
    table = torch.tensor([[5, 1, 4], [2, -1, 0]], dtype=torch.int32)
    pages = torch.randint(0, 256, (7, G, p4.page_bytes(D, page)), generator=g, dtype=torch.uint8)
    want = pages.clone()
    for t in range(T):
        for h in range(G):
            k = qkv[t, (H + h) * D:(H + h + 1) * D].float()
            v = qkv[t, (H + G + h) * D:(H + G + h + 1) * D].float()
            p4.write(want, int(table[seq[t], pos[t] // page]), h, pos[t] % page, page, k, v)
    dev = pages.cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = qkv.cuda()
    mass, places = torch.full((7, G, page), 2.0, device="cuda"), torch.full((7, G, page), -9, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_store_4bit(x, num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                positions=i32([100 + i for i in range(T)]), token_seq=i32(seq), block_table=table.cuda(), pages=dev,
                                page_size=page, slots=i32(pos), mass=mass, places=places)
    assert torch.equal(dev.cpu(), want)
    assert torch.equal(x.cpu(), qkv), "queries without norm and rotation stay as they are"
    for t in range(T):
        at = (int(table[seq[t], pos[t] // page]), slice(None), pos[t] % page)
        assert bool((mass[at] == 0).all()) and bool((places[at] == 100 + t).all())
    assert int((mass == 0).sum()) == T * G and int((places >= 0).sum()) == T * G
    k, v = ops.unpack_4bit(dev, num_kv_heads=G, head_dim=D, page_size=page, block_table=table[:1].cuda(), kv_lens=i32(lens[:1]),
                           max_kv_len=lens[0], dtype=F32)
    for t in range(T):
        if seq[t] == 0:
            for h in range(G):
                num = [p4.value(n[None], s[None], z[None])[0] for n, s, z in p4.read(want[int(table[0, pos[t] // page]), h], D, page, pos[t] % page)]
                assert torch.equal(k[pos[t] // page, h, pos[t] % page].cpu(), num[0].float())
                assert torch.equal(v[pos[t] // page, h, pos[t] % page].cpu(), num[1].float())
    assert bool((k[2, :, 1:] == 0).all()) and bool((v[2, :, 1:] == 0).all()), "zero behind the last token"


def test_no_value_is_off_by_more_than_half_a_step(ops):
    D, page, G, T = 128, 16, 4, 200
    g = torch.Generator().manual_seed(3)
    qkv = (torch.randn((T, (1 + 2 * G) * D), generator=g) * torch.exp(3 * torch.randn((T, 1), generator=g))).cuda()
    pages = torch.zeros((T // page + 1, G, p4.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    table = torch.arange(T // page + 1, dtype=torch.int32, device="cuda")[None]
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_store_4bit(qkv, num_heads=1, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                positions=pos, token_seq=torch.zeros_like(pos), block_table=table, pages=pages, page_size=page)
    k, v = ops.unpack_4bit(pages, num_kv_heads=G, head_dim=D, page_size=page, block_table=table, kv_lens=pos[-1:] + 1, max_kv_len=T, dtype=F32)
    for got, want in ((k, qkv[:, D:(1 + G) * D]), (v, qkv[:, (1 + G) * D:])):
        got = got.transpose(1, 2).reshape(-1, G, 2, 64)[:T].double()
        want = want.view(T, G, 2, 64).double()
        low = want.amin(-1, keepdim=True)
        # the scale: up to bfloat16 (2^-7) of (maximum - minimum) / 15, whose minimum was rounded down by 2^-7 of itself at most
        step = (want.amax(-1, keepdim=True) - low + low.abs() * 2.0 ** -7) / 15 * (1 + 2.0 ** -7)
        # float32: the quotient's rounding moves a border by 2^-24 * 16 steps, the sum is rounded by 2^-24 of itself
        assert bool(((got - want).abs() <= step * (0.5 + 2.0 ** -19) + got.abs() * 2.0 ** -23).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, "spread"])
def test_what_is_not_finite_makes_its_group_nan_and_nothing_else(ops, bad):
    D, page, G = 128, 16, 2
    qkv = torch.randn((1, (1 + 2 * G) * D), generator=torch.Generator().manual_seed(1))
    if bad == "spread":
        qkv[0, D + 3], qkv[0, D + 9] = 3e38, -3e38
    else:
        qkv[0, D + 3] = bad
    pages = torch.zeros((1, G, p4.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_store_4bit(qkv.cuda(), num_heads=1, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                positions=zero, token_seq=zero, block_table=zero[None], pages=pages, page_size=page)
    k, v = ops.unpack_4bit(pages, num_kv_heads=G, head_dim=D, page_size=page, block_table=zero[None], kv_lens=zero + 1, max_kv_len=1, dtype=F32)
    assert bool(k[0, 0, 0, :64].isnan().all()) and bool(k[0, 0, 0, 64:].isfinite().all())
    assert bool(k[0, 1, 0].isfinite().all()) and bool(v.isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,rot,pairing", [(128, 128, "half"), (64, 64, "interleaved"), (256, 256, "half"), (128, 64, "half"), (80, 80, "half"),
                                           (48, 32, "interleaved")])
def test_norm_and_rotation_are_those_of_the_wide_cache(ops, dtype, D, rot, pairing):
    """Queries within a rounding of ``qk_norm_rope_store``'s; keys: a step of the group's scale at most from quantising its float32 keys
    (a key within float32's rounding of a border may fall on either side of it)."""
    H, G, page, T = 6, 2, 8, 37
    g = torch.Generator().manual_seed(D + rot)
    qkv = torch.randn((T, (H + 2 * G) * D + 16), generator=g).to(dtype).cuda()[:, : (H + 2 * G) * D]
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).cuda() for _ in range(2))
    ang = torch.arange(64)[:, None] * 1e4 ** (-torch.arange(0, rot, 2) / rot)
    cos, sin = ang.cos().contiguous().cuda(), ang.sin().contiguous().cuda()
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    table = torch.randperm(8, generator=g).int()[None].cuda()
    args = dict(num_heads=H, num_kv_heads=G, head_dim=D, q_weight=qw, k_weight=kw, eps=1e-6, cos=cos, sin=sin, positions=pos,
                token_seq=torch.zeros_like(pos), block_table=table, page_size=page, pairing=pairing)
    wide = qkv.float().contiguous()
    kp, vp = (torch.zeros((8, G, page, D), device="cuda") for _ in range(2))
    ops.qk_norm_rope_store(wide, k_pages=kp, v_pages=vp, write_kv=True, **args)
    pages = torch.zeros((8, G, p4.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    q = torch.full((T, H * D), math.nan, dtype=dtype, device="cuda")
    before = qkv.clone()
    ops.qk_norm_rope_store_4bit(qkv, pages=pages, q_out=q, **args)
    assert torch.equal(qkv, before), "with q_out the projection stays as it is"
    # a turned element is a difference of two products, each at most the pair's length, which turning keeps and which is at most
    # sqrt(2) times the head's largest element: the two ways round those products and the norm (a few units of 2^-24), and store the
    # result rounded to its own type
    want = wide[:, : H * D].view(T, H, D)
    err = (q.float().view(T, H, D) - want).abs()
    assert bool((err <= 2.0 ** -20 * 2 ** 0.5 * want.abs().amax(-1, keepdim=True) + (U * want.abs() if dtype == BF16 else 0)).all())
    k, v = ops.unpack_4bit(pages, num_kv_heads=G, head_dim=D, page_size=page, block_table=table, kv_lens=pos[-1:] + 1, max_kv_len=T, dtype=F32)
    used = -(-T // page)
    for got, src in ((k, kp), (v, vp)):
        rows = src[table[0, :used].long()].cpu().view(-1, D)
        n, s, z = p4.quantise(rows)
        want = p4.value(n, s, z)
        live = torch.arange(used * page).view(used, 1, page).expand(used, G, page).reshape(-1) < T
        diff = (got.cpu().view(-1, D).double() - want).abs()[live]
        step = s.double().repeat_interleave(D // s.shape[1], -1)[live]
        assert bool((diff <= step * (1 + 2.0 ** -7) + 1e-6).all())
        assert float((diff > 1e-5).float().mean()) < 1e-3
    # in place, and without writing keys
    again = qkv.clone()
    ops.qk_norm_rope_store_4bit(again, pages=pages, **args)
    assert torch.equal(again[:, : H * D], q)
    kept = pages.clone()
    ops.qk_norm_rope_store_4bit(qkv[:, : H * D], pages=pages, q_out=q, write_kv=False, **args)
    assert torch.equal(pages, kept)


def test_positions_outside_the_tables_write_nothing_and_are_reported(ops):
    from qwen3_runtime_b200.ops.cuda import KernelError

    for D in (128, 48):
        pages = torch.zeros((2, 1, p4.page_bytes(D, 16)), dtype=torch.uint8, device="cuda")
        qkv = torch.randn((2, 3 * D), device="cuda")
        cos = torch.ones((4, D // 2), device="cuda")
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        args = dict(num_heads=1, num_kv_heads=1, head_dim=D, q_weight=None, k_weight=None, eps=0.0, token_seq=i32([0, 0]), pages=pages,
                    page_size=16)
        with pytest.raises(KernelError, match="rotation tables"):
            ops.qk_norm_rope_store_4bit(qkv.clone(), cos=cos, sin=cos, positions=i32([4, -1]), slots=i32([0, 1]), block_table=i32([[0]]), **args)
            ops.raise_if_kernel_error()
        half = p4.places_in(D, 16, 0)[0][1]
        assert bool((pages[0, :, : 2 * half] == 0).all()), "no key"
        pages.zero_()
        # places without a page in the table: nothing is written
        ops.qk_norm_rope_store_4bit(qkv.clone(), cos=None, sin=None, positions=i32([0, 1]), slots=i32([16, -3]), block_table=i32([[0]]), **args)
        ops.qk_norm_rope_store_4bit(qkv.clone(), cos=None, sin=None, positions=i32([0, 1]), block_table=i32([[-1]]), **args)
        ops.raise_if_kernel_error()
        assert not bool(pages.any())


# ---- attention --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("H,G,D,page", [(8, 2, 128, 16), (4, 4, 128, 16), (16, 2, 128, 32), (12, 1, 128, 16), (16, 1, 64, 16), (2, 2, 64, 8),
                                        (6, 2, 256, 16), (16, 1, 256, 64), (8, 2, 128, 5), (8, 2, 64, 24), (5, 1, 128, 48), (8, 1, 256, 3)])
@pytest.mark.parametrize("slices", [None, 1, 3, -3, 8, 9, 16, 40])
def test_decoded_tokens(ops, H, G, D, page, slices):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 611]
    c = p4.Cache(lens, G, D, page, seed=H + D, k_scale=1.5)
    new = [1] * len(lens)
    q = queries(len(lens), H, D, 7, extra=8)
    got, lse = attend(ops, c, q, new, lens, H, D ** -0.5, lse=True, slices=slices)
    q = q[:, : H * D].view(-1, H, D)
    _want, want_lse, _w = check_rows(got, q, c, new, lens, D ** -0.5)
    for b in range(len(lens)):
        err = score_error(q[b:b + 1], c, b, D ** -0.5)[0]
        assert bool(((lse[b].double() - want_lse[b]).abs() <= err + 2.0 ** -20 * (1 + want_lse[b].abs())).all())


@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 5000])
@pytest.mark.parametrize("page,D", [(16, 128), (8, 64), (5, 128)])
def test_decoded_tokens_behind_a_window(ops, window, page, D):
    """Pages that the window has passed are gone (-1)."""
    lens = [1, 40, 64, 333, 500]
    c = p4.Cache(lens, 2, D, page, seed=window)
    table = c.table.clone()
    for b, n in enumerate(lens):
        table[b, : max(0, n - window) // page] = -1
    q = queries(len(lens), 8, D, 3)
    for slices in (None, 4):
        got = attend(ops, c, q, [1] * len(lens), lens, 8, D ** -0.5, window=window, table=table, slices=slices)
        check_rows(got, q.view(-1, 8, D), c, [1] * len(lens), lens, D ** -0.5, window=window)


def test_a_long_cache(ops):
    lens = [20011, 9000]
    c = p4.Cache(lens, 1, 128, 16, seed=5, k_scale=2.0)
    q = queries(2, 4, 128, 3)
    for slices in (None, 1, 16, -16, 64):
        got, lse = attend(ops, c, q, [1, 1], lens, 4, 128 ** -0.5, lse=True, slices=slices)
        check_rows(got, q.view(-1, 4, 128), c, [1, 1], lens, 128 ** -0.5)


def test_offsets_beyond_32_bits(ops):
    """Pages whose bytes lie more than 2^31 (and 2^32) behind the first."""
    G, D, page = 8, 128, 16
    c = p4.Cache([40], G, D, page, seed=8)
    rec = p4.page_bytes(D, page)
    count = (1 << 32) // (G * rec) + 8
    big = torch.zeros((count, G, rec), dtype=torch.uint8, device="cuda")
    ids = [count - 1, (1 << 31) // (G * rec) + 3, count - 4]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    for i, page_id in enumerate(ids):
        big[page_id] = c.pages[int(c.table[0, i])].cuda()
    q = queries(1, 16, D, 2)
    step = p4.step_of([1], [40], page)
    dev = q.cuda()
    out, lse = torch.empty((1, 16 * D), dtype=BF16, device="cuda"), torch.empty((1, 16), device="cuda")
    ops.paged_attention_4bit(dev, dev.stride(0), num_heads=16, pages=big, block_table=table, out=out, scale=D ** -0.5, step=step, lse=lse,
                             **sizes(c))
    check_rows(out.cpu().view(1, 16, D), q.view(1, 16, D), c, [1], [40], D ** -0.5)
    k, _v = ops.unpack_4bit(big, block_table=table, kv_lens=step.kv_lens, max_kv_len=40, dtype=F32, **sizes(c))
    assert torch.equal(k.transpose(1, 2).reshape(-1, G, D)[:40].cpu(), c.values(0)[0].transpose(0, 1).float())
    mass = torch.zeros((count, G, page), device="cuda")
    ops.attention_mass_4bit(dev, dev.stride(0), num_heads=16, pages=big, mass=mass, block_table=table, scale=D ** -0.5, step=step, **sizes(c))
    assert abs(float(mass.sum()) - 16) < 1e-3 and abs(float(mass[table[0].long()].sum()) - 16) < 1e-3
    places = torch.full((count, G, page), -1, dtype=torch.int32, device="cuda")
    for i, page_id in enumerate(ids):
        places[page_id] = torch.arange(i * page, (i + 1) * page, device="cuda")
    mass[ids[0]] = 0.0
    ops.evict_4bit(pages=big, mass=mass, places=places, block_table=table, kv_lens=step.kv_lens, max_kv_len=40, keep=24, first=0, recent=1, **sizes(c))
    assert torch.equal(big[ids[0], :, : 8 * 64].cpu(), c.pages[int(c.table[0, 1]), :, 8 * 64:16 * 64])  # tokens 24 .. 31 fill places 0 .. 7


def test_a_key_or_value_that_is_not_finite_stays_with_its_head(ops):
    def mutate(b, k, v):
        if b == 1:
            k[0, 7, 3] = math.nan
            v[1, 9, 100] = math.inf

    lens = [30, 30]
    c = p4.Cache(lens, 3, 128, 16, seed=1, mutate=mutate)
    q = queries(2, 6, 128, 5)
    for slices in (1, 2):
        got = attend(ops, c, q, [1, 1], lens, 6, 128 ** -0.5, slices=slices)
        assert bool(got[0].isfinite().all()) and bool(got[1, 4:].isfinite().all())
        assert bool(got[1, :2].isnan().all()), "a key that is not a number: the row's weights are none"
        assert bool(got[1, 2:4, :64].isfinite().all()) and bool(got[1, 2:4, 64:].isnan().all()), "its group of channels"


def test_far_scores_and_zero_queries(ops):
    """Rows whose weights lie on one token, rows of equal weights, and scores far apart between the slices."""
    lens = [300, 300, 300]
    def mutate(b, k, v):
        if b == 1:
            k[:, 250] *= 30
            k[:, 10] *= -20
    c = p4.Cache(lens, 2, 128, 16, seed=2, mutate=mutate)
    q = queries(3, 4, 128, 9).view(3, 4, 128)
    q[0, 1] = 0
    q[1] *= 8
    q[2, 0, 5:] = 0
    q[2, 1] *= 2.0 ** -20
    q[2, 2, ::2] *= 2.0 ** -12
    for slices in (1, 4):
        got = attend(ops, c, q.view(3, -1), [1] * 3, lens, 4, 128 ** -0.5, slices=slices)
        check_rows(got, q, c, [1] * 3, lens, 128 ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,G,D,page,window", [(8, 2, 128, 16, None), (8, 2, 64, 8, None), (8, 2, 128, 16, 20), (4, 2, 256, 16, None),
                                               (4, 1, 80, 5, None), (20, 1, 128, 16, None), (4, 2, 48, 16, 9)])
def test_portions_of_prompts_and_single_tokens_in_one_step(ops, dtype, H, G, D, page, window):
    new, lens = [1, 33, 1, 5, 18], [70, 33, 1, 90, 50]
    c = p4.Cache(lens, G, D, page, seed=D, width=9 if page == 16 else None)
    q = queries(sum(new), H, D, 4, dtype, extra=16)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, dtype=dtype)
    check_rows(got, q[:, : H * D].view(-1, H, D), c, new, lens, D ** -0.5, window=window, wide=True, dtype=dtype)


@pytest.mark.parametrize("H,G,D,dtype", [(20, 1, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32)])
def test_single_tokens_of_other_sizes(ops, H, G, D, dtype):
    lens = [1, 17, 130]
    c = p4.Cache(lens, G, D, 16, seed=D)
    q = queries(3, H, D, 4, dtype)
    got = attend(ops, c, q, [1] * 3, lens, H, D ** -0.5, dtype=dtype)
    check_rows(got, q.view(-1, H, D), c, [1] * 3, lens, D ** -0.5, wide=True, dtype=dtype)


# ---- sums of weights ----------------------------------------------------------------------------------------------------------


def mass_of(ops, c, q, new, lens, H, scale, observe, lse=None, start=None, repeat=1):
    step = p4.step_of(new, lens, c.page)
    dev = q.cuda()
    mass = (torch.zeros((c.pages.shape[0], c.G, c.page)) if start is None else start).cuda()
    for _ in range(repeat):
        ops.attention_mass_4bit(dev, dev.stride(0), num_heads=H, pages=c.pages.cuda(), mass=mass, block_table=c.table.cuda(), scale=scale,
                                step=step, observe=observe, lse=lse, **sizes(c))
    return mass.cpu()


def check_mass(got, q, c, new, lens, scale, observe, start=None, dtype=BF16, times=1):
    _o, _l, weights = p4.attention(q, c, new, lens, scale)
    R = q.shape[1] // c.G
    want = torch.zeros(got.shape, dtype=torch.float64) if start is None else start.double().clone()
    tol = want.abs() * 2.0 ** -23
    t = 0
    for b, (n, L) in enumerate(zip(new, lens)):
        err = float(score_error(q[t:t + n], c, b, scale).max()) + 2.0 ** -20 * 12
        w = weights[b][max(0, n - (observe or n)):].view(-1, c.G, R, L).sum((0, 2)) * times  # [G, L]
        for j in range(L):
            at = (int(c.table[b, j // c.page]), slice(None), j % c.page)
            want[at] += w[:, j]
            tol[at] += w[:, j] * math.expm1(2 * err) + 1e-30
        t += n
    diff = (got.double() - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol.clamp(min=1e-37)).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,G,D,page", [(8, 2, 128, 16), (16, 1, 64, 8), (6, 2, 256, 16), (20, 1, 128, 5), (4, 2, 80, 16), (3, 3, 48, 7)])
@pytest.mark.parametrize("observe", [1, 4, None])
def test_sums_of_weights(ops, dtype, H, G, D, page, observe):
    new, lens = [1, 19, 1, 40, 3], [70, 19, 1, 170, 300]
    c = p4.Cache(lens, G, D, page, seed=H)
    q = queries(sum(new), H, D, 4, dtype)
    g = torch.Generator().manual_seed(2)
    start = torch.rand((c.pages.shape[0], G, page), generator=g)
    got = mass_of(ops, c, q, new, lens, H, D ** -0.5, observe, start=start)
    check_mass(got, q.view(-1, H, D), c, new, lens, D ** -0.5, observe, start=start, dtype=dtype)
    again = mass_of(ops, c, q, new, lens, H, D ** -0.5, observe, start=start)
    assert torch.equal(got, again), "the same bits every time"


@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (16, 1, 64), (4, 2, 256)])
def test_sums_of_decoded_tokens_from_the_attentions_log_sums(ops, H, G, D):
    lens = [1, 16, 100, 1000]
    c = p4.Cache(lens, G, D, 16, seed=H)
    q = queries(4, H, D, 4)
    _out, lse = attend(ops, c, q, [1] * 4, lens, H, D ** -0.5, lse=True)
    got = mass_of(ops, c, q, [1] * 4, lens, H, D ** -0.5, 1, lse=lse.cuda(), repeat=2)
    check_mass(got, q.view(-1, H, D), c, [1] * 4, lens, D ** -0.5, 1, times=2)
    assert abs(float(got.sum()) - 2 * 4 * H) < 1e-2


# ---- eviction --------------------------------------------------------------------------------------------------------------------


def check_eviction(ops, lens, G, D, page, keep, first, recent, layers=0, mass_of=None, seed=0, places_of=None):
    c = p4.Cache(lens, G, D, page, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    L = max(1, layers)
    shape = (L, *c.pages.shape[:2], page)
    pages = torch.stack([c.pages.roll(i, 1) for i in range(L)])  # (other heads' bytes in other layers)
    mass = torch.rand(shape, generator=g) if mass_of is None else mass_of(shape, g)
    places = torch.full(shape, -5, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(n):
            places[:, int(c.table[b, j // page]), :, j % page] = j if places_of is None else places_of(b, j)
    want = [pages.clone(), mass.clone(), places.clone()]
    for layer in range(L):
        for b, n in enumerate(lens):
            at = [(int(c.table[b, j // page]), j % page) for j in range(n)]
            for h in range(G):
                m = [float(mass[layer, p, h, r]) for p, r in at]
                pl = [int(places[layer, p, h, r]) for p, r in at]
                for to, src in enumerate(p4.evict(m, pl, keep, first, recent)):
                    if to != src:
                        for (a, w), (a2, _w) in zip(p4.places_in(D, page, at[to][1]), p4.places_in(D, page, at[src][1])):
                            want[0][layer, at[to][0], h, a:a + w] = pages[layer, at[src][0], h, a2:a2 + w]
                        want[1][layer, at[to][0], h, at[to][1]] = mass[layer, at[src][0], h, at[src][1]]
                        want[2][layer, at[to][0], h, at[to][1]] = places[layer, at[src][0], h, at[src][1]]
    have = [x.cuda() if layers else x[0].cuda() for x in (pages, mass, places)]
    ops.evict_4bit(pages=have[0], mass=have[1], places=have[2], block_table=c.table.cuda(),
                   kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), max_kv_len=max(lens), keep=keep, first=first, recent=recent,
                   **sizes(c))
    for got, w in zip(have, want):
        assert torch.equal(got.cpu().nan_to_num(7e7) if got.is_floating_point() else got.cpu(),
                           (w if layers else w[0]).nan_to_num(7e7) if got.is_floating_point() else (w if layers else w[0]))


@pytest.mark.parametrize("D,page", [(128, 16), (64, 8), (256, 16), (80, 5), (16, 3)])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 0, 1), (40, 4, 8), (40, 40, 0), (40, 0, 40), (64, 0, 0), (1000, 2, 3)])
def test_eviction(ops, D, page, keep, first, recent):
    check_eviction(ops, [1, 39, 40, 41, 64, 65, 200], 2, D, page, keep, first, recent, seed=keep + D)


def test_eviction_of_equal_and_strange_sums(ops):
    def strange(shape, g):
        m = torch.randint(0, 4, shape, generator=g).float()
        pick = torch.rand(shape, generator=g)
        m[pick < 0.1] = math.nan
        m[(pick > 0.1) & (pick < 0.15)] = math.inf
        m[(pick > 0.15) & (pick < 0.2)] = -math.inf
        m[(pick > 0.2) & (pick < 0.3)] = -0.0
        m[(pick > 0.3) & (pick < 0.4)] = -1.5
        m[(pick > 0.4) & (pick < 0.5)] = 1e-42
        return m

    for keep in (5, 30, 60, 99):
        check_eviction(ops, [100, 77], 3, 64, 16, keep, 2, 3, mass_of=strange, seed=keep)
    check_eviction(ops, [100], 1, 64, 16, 50, 0, 0, mass_of=lambda shape, g: torch.zeros(shape))


def test_eviction_of_many_layers_and_blocks_of_threads(ops):
    check_eviction(ops, [2100, 1024, 1025, 1500], 2, 64, 16, 1024, 4, 100, layers=3, seed=3)


def test_eviction_again_after_tokens_have_moved(ops):
    """Places no longer in order: the newest tokens are known by their positions, not by where they lie."""
    check_eviction(ops, [120, 60], 2, 64, 16, 50, 3, 20, places_of=lambda b, j: (j * 37) % 120 if b == 0 else (j * 7) % 60)


def test_eviction_of_more_tokens_than_shared_memory_holds(ops):
    n = ops.EVICT_KEYS + 1000
    G, D, page = 1, 64, 16
    count = -(-n // page)
    g = torch.Generator().manual_seed(4)
    mass = torch.randint(0, 5000, (count, G, page), generator=g).float()
    places = torch.arange(count * page, dtype=torch.int32).view(count, G, page)
    pages = torch.randint(0, 256, (count, G, p4.page_bytes(D, page)), generator=g, dtype=torch.uint8)
    keep, first, recent = 40000, 10, 500
    dev = [x.cuda() for x in (pages, mass, places)]
    table = torch.arange(count, dtype=torch.int32, device="cuda")[None]
    ops.evict_4bit(pages=dev[0], mass=dev[1], places=dev[2], block_table=table, kv_lens=torch.tensor([n], dtype=torch.int32, device="cuda"),
                   max_kv_len=n, keep=keep, first=first, recent=recent, num_kv_heads=G, head_dim=D, page_size=page)
    src = p4.evict(mass.flatten()[:n].tolist(), places.flatten()[:n].tolist(), keep, first, recent)
    assert dev[2].cpu().flatten()[:keep].tolist() == src
    assert torch.equal(dev[1].cpu().flatten()[:keep], mass.flatten()[src])
    code = lambda x: x[:, 0, : page * 32].reshape(-1, 32)  # noqa: E731
    assert torch.equal(code(dev[0].cpu())[:keep], code(pages)[src])


# ---- how they are called ---------------------------------------------------------------------------------------------------


def test_another_stream_and_captured_steps(ops):
    """Two captured steps of unequal sizes replayed in turn, then after their lengths have changed; the first call on a side stream."""
    H, G, D, page = 8, 2, 128, 16
    caches = [p4.Cache([200, 90], G, D, page, seed=1, width=16), p4.Cache([33, 150, 7], G, D, page, seed=2, width=16)]
    made = []
    for i, c in enumerate(caches):
        B = len(c.lens)
        q = queries(B, H, D, 3 + i)
        step = p4.step_of([1] * B, c.lens, page, captured_width=16)
        t = dict(q=q.cuda(), pages=c.pages.cuda(), table=c.table.cuda(), out=torch.zeros((B, H * D), dtype=BF16, device="cuda"),
                 lse=torch.zeros((B, H), device="cuda"), mass=torch.zeros((c.pages.shape[0], G, page), device="cuda"))

        def run(t=t, c=c, step=step):
            ops.paged_attention_4bit(t["q"], t["q"].stride(0), num_heads=H, pages=t["pages"], block_table=t["table"], out=t["out"],
                                     scale=D ** -0.5, step=step, lse=t["lse"], decode_slices=5, **sizes(c))
            ops.attention_mass_4bit(t["q"], t["q"].stride(0), num_heads=H, pages=t["pages"], mass=t["mass"], block_table=t["table"],
                                    scale=D ** -0.5, step=step, lse=t["lse"], **sizes(c))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        pool = made[0]["graph"].pool() if made else None
        with torch.cuda.graph(graph, pool=pool):
            run()
        made.append(dict(t=t, graph=graph, q=q, c=c, step=step))
    for lens in ([[200, 90], [33, 150, 7]], [[31, 64], [2, 149, 7]]):
        for m, n in zip(made, lens):
            m["step"].kv_lens.copy_(torch.tensor(n, dtype=torch.int32))
            m["step"].kv_longest.fill_(max(n))
            m["t"]["out"].zero_()
            m["t"]["mass"].zero_()
        for _ in range(2):
            for m in made:
                m["graph"].replay()
        torch.cuda.synchronize()
        for m, n in zip(made, lens):
            cut = p4.Cache.__new__(p4.Cache)
            cut.__dict__.update(m["c"].__dict__)
            cut.k = [[x[:, :L] for x in k] for k, L in zip(m["c"].k, n)]
            cut.v = [[x[:, :L] for x in v] for v, L in zip(m["c"].v, n)]
            q = m["q"].view(-1, H, D)
            check_rows(m["t"]["out"].cpu().view(-1, H, D), q, cut, [1] * len(n), n, D ** -0.5)
            check_mass(m["t"]["mass"].cpu(), q, cut, [1] * len(n), n, D ** -0.5, 1, times=2)


def test_a_cache_that_is_written_attended_summed_and_cut(ops):
    """The operators as a decoder's layer uses them: a prompt, then token after token, cut to a budget on the way; against the plain
    statements over the same numbers."""
    H, G, D, page, keep, first, recent = 8, 2, 128, 16, 48, 4, 16
    R, scale, total = H // G, D ** -0.5, 75
    g = torch.Generator().manual_seed(11)
    x = torch.randn((total, (H + 2 * G) * D), generator=g).to(BF16)
    pages = torch.zeros((6, G, p4.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    mass, places = torch.zeros((6, G, page), device="cuda"), torch.zeros((6, G, page), dtype=torch.int32, device="cuda")
    table = torch.tensor([[3, 0, 5, 1, 4]], dtype=torch.int32, device="cuda")
    rows = [[] for _ in range(G)]  # plain: per head (position, key, value, sum)
    held, at = 0, 0
    for n in [60] + [1] * 15:
        if held + n > 64:
            ops.evict_4bit(pages=pages, mass=mass, places=places, block_table=table, kv_lens=torch.tensor([held], dtype=torch.int32, device="cuda"),
                           max_kv_len=held, keep=keep, first=first, recent=recent, num_kv_heads=G, head_dim=D, page_size=page)
            # sums that nearly tie may go either way: the plain rows follow the sums that the kernels made, checked below
            m = mass[table[0].long()].transpose(0, 1).reshape(G, -1)[:, :held].cpu()
            for h in range(G):
                kept = places[table[0].long(), h].flatten()[:keep].tolist()
                by = {r[0]: r for r in rows[h]}
                newest = max(by)
                assert len(set(kept)) == keep and all(p in kept for p in by if p < first or p > newest - recent)
                gone = [r[3] for p, r in by.items() if p not in kept]
                stay = [r[3] for p, r in by.items() if p in kept and first <= p <= newest - recent]
                assert max(gone) <= min(stay) * (1 + 1e-4)
                rows[h] = [by[p] for p in kept]
            held = keep
        step = p4.step_of([n], [held + n], page)
        xs = x[at:at + n].cuda()
        pos = torch.arange(at, at + n, dtype=torch.int32, device="cuda")
        q = torch.empty((n, H * D), dtype=BF16, device="cuda")
        ops.qk_norm_rope_store_4bit(xs, num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                    positions=pos, slots=step.positions, token_seq=step.token_seq, block_table=table, pages=pages,
                                    page_size=page, q_out=q, mass=mass, places=places)
        out, lse = torch.empty_like(q), torch.empty((n, H), device="cuda") if n == 1 else None
        args = dict(num_heads=H, num_kv_heads=G, head_dim=D, pages=pages, block_table=table, page_size=page, scale=scale, step=step)
        ops.paged_attention_4bit(q, q.stride(0), out=out, lse=lse, **args)
        ops.attention_mass_4bit(q, q.stride(0), mass=mass, lse=lse, **args)
        for h in range(G):
            k = x[at:at + n, (H + h) * D:(H + h + 1) * D].float()
            v = x[at:at + n, (H + G + h) * D:(H + G + h + 1) * D].float()
            k, v = (p4.value(*p4.quantise(y)) for y in (k, v))
            rows[h] += [[at + i, k[i], v[i], 0.0] for i in range(n)]
        got = out.cpu().view(n, H, D).double()
        for i in range(n):
            for h in range(H):
                seen = rows[h // R][: held + i + 1]
                w = torch.softmax(torch.stack([r[1] for r in seen]) @ x[at + i, h * D:(h + 1) * D].double() * scale, 0)
                want = w @ torch.stack([r[2] for r in seen])
                assert float((got[i, h] - want).norm() / want.norm()) < 0.03
                for r, y in zip(seen, w.tolist()):
                    r[3] += y
        held, at = held + n, at + n
    m = mass[table[0].long()].transpose(0, 1).reshape(G, -1)[:, :held].cpu().double()
    for h in range(G):
        want = torch.tensor([r[3] for r in rows[h]], dtype=torch.float64)
        assert bool(((m[h] - want).abs() <= 1e-4 * want).all())


@pytest.mark.parametrize("page,D", [(48, 128), (80, 64), (160, 128), (256, 256), (67, 128)])
def test_pages_larger_than_what_a_block_takes_at_a_time(ops, page, D):
    """A block's next keys lie in the same page, or further on than one page behind."""
    H, G, lens = 8, 2, [1, 47, 48, 161, 700]
    c = p4.Cache(lens, G, D, page, seed=page)
    q = queries(len(lens), H, D, 5)
    rows, new = q.view(-1, H, D), [1] * len(lens)
    for slices in (None, 3, -3):
        got, lse = attend(ops, c, q, new, lens, H, D ** -0.5, lse=True, slices=slices)
        check_rows(got, rows, c, new, lens, D ** -0.5)
        check_mass(mass_of(ops, c, q, new, lens, H, D ** -0.5, 1, lse=lse.cuda()), rows, c, new, lens, D ** -0.5, 1)
    check_mass(mass_of(ops, c, q, new, lens, H, D ** -0.5, 1), rows, c, new, lens, D ** -0.5, 1)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 20]])
@pytest.mark.parametrize("shift,extra", [(0, 4), (1, 0), (1, 3), (4, 8)])
def test_rows_of_queries_that_begin_anywhere(ops, new, shift, extra):
    """``shift`` elements behind a multiple of 16 bytes, rows ``extra`` elements apart."""
    H, G, D, lens = 8, 2, 128, [9, 40, 33]
    c = p4.Cache(lens, G, D, 16, seed=3)
    q = queries(sum(new), H, D, 4)
    T, width = q.shape[0], H * D + extra
    dev = torch.zeros(shift + T * width, dtype=BF16, device="cuda")[shift:].view(T, width)
    dev[:, : H * D] = q.cuda()
    out = torch.zeros(2 + T * H * D, dtype=BF16, device="cuda")[2:].view(T, H * D) if shift == 1 else torch.zeros_like(q, device="cuda")
    ops.paged_attention_4bit(dev, width, num_heads=H, pages=c.pages.cuda(), block_table=c.table.cuda(), out=out, scale=D ** -0.5,
                             step=p4.step_of(new, lens, 16), **sizes(c))
    check_rows(out.cpu().view(T, H, D), q.view(T, H, D), c, new, lens, D ** -0.5, wide=True)


@pytest.mark.parametrize("slices", [1, 4, -4])
def test_sequences_without_keys(ops, slices):
    """Length zero: results are zero, log sums minus infinity, no sum moves; the others are as ever."""
    H, G, D, lens, page = 8, 2, 128, [20, 700, 31], 16
    c = p4.Cache(lens, G, D, page, seed=6)
    q = queries(3, H, D, 5)
    step = p4.step_of([1] * 3, lens, page)
    step.kv_lens[0] = 0
    got, lse = attend(ops, c, q, [1] * 3, lens, H, D ** -0.5, lse=True, slices=slices, step=step)
    assert bool((got[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    whole = attend(ops, c, q, [1] * 3, lens, H, D ** -0.5, slices=slices)
    assert torch.equal(got[1:], whole[1:])
    for sums in (lse.cuda(), None):
        mass = torch.zeros((c.pages.shape[0], G, page), device="cuda")
        ops.attention_mass_4bit(q.cuda(), H * D, num_heads=H, pages=c.pages.cuda(), mass=mass, block_table=c.table.cuda(), scale=D ** -0.5,
                                step=step, lse=sums, **sizes(c))
        assert bool((mass[c.table[0, :2].long().cuda()] == 0).all()) and abs(float(mass.sum()) - 2 * H) < 1e-2


@pytest.mark.parametrize("page", [16, 32, 5])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 20]])
def test_entries_that_are_no_pages_are_read_nowhere(ops, page, new):
    H, G, D, lens = 8, 2, 128, [90, 70, 60]
    c = p4.Cache(lens, G, D, page, seed=3)
    q = queries(sum(new), H, D, 4)
    table = c.table.clone()
    table[0, 0], table[0, 1] = -7, c.pages.shape[0]
    for slices in (1, 3):
        got, whole = (attend(ops, c, q, new, lens, H, D ** -0.5, table=t, slices=slices) for t in (table, c.table))
        assert torch.equal(got[new[0]:], whole[new[0]:])
    step, dev = p4.step_of(new, lens, page), q.cuda()
    masses = []
    for t in (table, c.table):
        masses.append(torch.zeros((c.pages.shape[0], G, page), device="cuda"))
        ops.attention_mass_4bit(dev, H * D, num_heads=H, pages=c.pages.cuda(), mass=masses[-1], block_table=t.cuda(), scale=D ** -0.5, step=step,
                                **sizes(c))
    others = c.table[1:].flatten().long().unique()
    others = others[~torch.isin(others, c.table[0].long())].cuda()
    assert torch.equal(masses[0][others], masses[1][others])
    assert bool((masses[0][c.table[0, :2].long().cuda()] == 0).all()), "what the table does not name is left alone"


def test_two_streams_at_once(ops):
    """Unequal steps under way together, each with workspaces of its own."""
    H, G, D = 8, 2, 128
    caches = [p4.Cache([5000, 1200], G, D, 16, seed=1), p4.Cache([3000, 64, 900], G, D, 16, seed=2)]
    made, alone = [], []
    for i, c in enumerate(caches):
        q = queries(len(c.lens), H, D, i)
        made.append((c, q.cuda(), c.pages.cuda(), c.table.cuda(), p4.step_of([1] * len(c.lens), c.lens, 16), torch.cuda.Stream()))
        alone.append(attend(ops, c, q, [1] * len(c.lens), c.lens, H, D ** -0.5, slices=-9))
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (c, q, pages, table, step, stream) in enumerate(made):
            with torch.cuda.stream(stream):
                out = torch.empty_like(q)
                ops.paged_attention_4bit(q, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=D ** -0.5, step=step,
                                         decode_slices=-9, **sizes(c))
                outs[i].append(out)
    torch.cuda.synchronize()
    for got, want in zip(outs, alone):
        assert all(torch.equal(x.cpu().view(want.shape), want) for x in got)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("keep", [40, 700])
def test_a_captured_eviction(ops, keep, shift):
    """Replayed with other lengths, some within the budget; sums and positions that do not begin at 16 bytes."""
    G, D, page, lens = 2, 64, 16, [1500, 64, 900]
    c = p4.Cache(lens, G, D, page, seed=9)
    g = torch.Generator().manual_seed(1)
    shape = (c.pages.shape[0], G, page)
    count = shape[0] * G * page
    mass = torch.rand(shape, generator=g)
    places = torch.full(shape, -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(n):
            places[int(c.table[b, j // page]), :, j % page] = j
    dev = [c.pages.cuda(), torch.zeros(count + shift, device="cuda")[shift:].view(shape),
           torch.zeros(count + shift, dtype=torch.int32, device="cuda")[shift:].view(shape)]
    table, kv_lens = c.table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    run = lambda: ops.evict_4bit(pages=dev[0], mass=dev[1], places=dev[2], block_table=table, kv_lens=kv_lens, max_kv_len=1500,  # noqa: E731
                                 keep=keep, first=4, recent=10, **sizes(c))
    graph = torch.cuda.CUDAGraph()
    run()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run()
    for now in (lens, [keep + 1, 20, 0], [1499, 64, keep]):
        for d, x in zip(dev, (c.pages, mass, places)):
            d.copy_(x)
        kv_lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate(now):
            rows = c.table[b].long()
            for h in range(G):
                m, p = (x[rows, h].flatten()[:n].tolist() for x in (mass, places))
                src = p4.evict(m, p, keep, 4, 10) if n > keep else list(range(n))
                assert dev[2].cpu()[rows, h].flatten()[: len(src)].tolist() == [p[i] for i in src]
                assert dev[1].cpu()[rows, h].flatten()[: len(src)].tolist() == [m[i] for i in src]


def test_steps_of_nothing(ops):
    G, D, page = 2, 128, 16
    c = p4.Cache([20], G, D, page)
    pages, table = c.pages.cuda(), c.table.cuda()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    qkv = torch.zeros((0, (4 + 2 * G) * D), dtype=BF16, device="cuda")
    ops.qk_norm_rope_store_4bit(qkv, num_heads=4, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, positions=none, token_seq=none,
                                block_table=table, pages=pages, **sizes(c))
    k, v = ops.unpack_4bit(pages, block_table=table, kv_lens=torch.tensor([20], dtype=torch.int32, device="cuda"), max_kv_len=0, dtype=BF16, **sizes(c))
    assert k.shape == v.shape == (0, G, page, D)
    k, v = ops.unpack_4bit(pages, block_table=table[:0], kv_lens=none, max_kv_len=20, dtype=BF16, **sizes(c))
    assert k.shape == v.shape == (0, G, page, D)
    torch.cuda.synchronize()
    assert torch.equal(pages.cpu(), c.pages)
    for dtype in (BF16, F32):
        step, q = p4.step_of([], [], page), torch.zeros((0, 4 * D), dtype=dtype, device="cuda")
        out, mass = torch.empty_like(q), torch.zeros((pages.shape[0], G, page), device="cuda")
        args = dict(num_heads=4, pages=pages, block_table=table[:0], scale=1.0, step=step, **sizes(c))
        ops.paged_attention_4bit(q, 4 * D, out=out, **args)
        ops.attention_mass_4bit(q, 4 * D, mass=mass, **args)
    ops.evict_4bit(pages=pages, mass=mass, places=torch.zeros_like(mass, dtype=torch.int32), block_table=table[:0], kv_lens=none, max_kv_len=20,
                   keep=4, first=0, recent=0, **sizes(c))
    torch.cuda.synchronize()
    assert torch.equal(pages.cpu(), c.pages) and not bool(mass.any())


@pytest.mark.parametrize("D,dtype", [(64, F32), (80, BF16), (208, F32)])
def test_slices_joined_by_a_block_or_by_a_second_kernel(ops, D, dtype):
    """The same bits either way: a token alone (a block a slice), and among so many that each block goes through its token's slices."""
    H, G, lens = 4, 2, [700, 1100] + [3] * 400
    c = p4.Cache(lens, G, D, 16, seed=D)
    q = queries(len(lens), H, D, 4, dtype)
    got = attend(ops, c, q, [1] * len(lens), lens, H, D ** -0.5, dtype=dtype)
    few = attend(ops, c, q[:2], [1, 1], lens[:2], H, D ** -0.5, dtype=dtype, table=c.table[:2])
    assert torch.equal(got[:2], few)
    two = p4.Cache.__new__(p4.Cache)
    two.__dict__.update(c.__dict__)
    check_rows(got[:2], q[:2].view(2, H, D), two, [1, 1], lens[:2], D ** -0.5, wide=True, dtype=dtype)
