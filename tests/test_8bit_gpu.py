"""A cache in 8 bits on the GPU: every kernel against the plain statements in tests/plain_8bit.py, at the sizes and masks where they can
go wrong.

Tolerances.  U = 2^-8 is half a step of bfloat16 relative to the value, H = 2^-11 of half precision.  A score is a sum of D products in float32:
it is off by at most ``score_error`` below, which moves a weight by a factor of exp(2 error).  A decoded row rounds each weight (times a power of
two) to half precision: H of itself, and where that leaves the normal numbers, below 2^-20 of the largest contribution's weight, 2^-31 of
that at most, each times a code of up to 448; its other roundings are those of float32 sums of up to a few thousand numbers and of exponentials good to
2^-22, together below H / 2 of the sum of weight times |value|; and the result (U |o|).  Prompts round the weights to bfloat16 (U each) and
the result.  float32 rounds sums only."""

import math

import pytest
import torch

import plain_8bit as p8

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -8, 2.0 ** -11
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from qwen3_runtime_b200.ops.cuda import CudaOps

    return CudaOps()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def sizes(c):
    return dict(num_kv_heads=c.G, head_dim=c.D, page_size=c.page)


def queries(T, H, D, seed, dtype=BF16, extra=0):
    """``[T, H * D + extra]`` rows (a projection's row may be wider than its queries)."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, H * D + extra), generator=g).to(dtype)


def attend(ops, c, q, new, lens, H, scale, *, window=None, keep_first=0, slices=None, dtype=BF16, table=None, step=None):
    step = step or p8.step_of(new, lens, c.page)
    dev = q.cuda()
    T = dev.shape[0]
    out = torch.full((T, H * c.D), math.nan, dtype=dtype, device="cuda")
    ops.paged_attention_8bit(dev, dev.stride(0), num_heads=H, pages=c.pages.cuda(), block_table=(c.table if table is None else table).cuda(),
                             out=out, scale=scale, step=step, window=window, keep_first=keep_first, decode_slices=slices, **sizes(c))
    ops.raise_if_kernel_error()
    return out.cpu().view(T, H, c.D)


def score_error(row, k, scale, dtype):
    """Bound of a score's error ``[H]``: D additions of float32 to sums of |q k|, whatever their order."""
    D = row.shape[-1]
    return abs(scale) * 2.0 ** (-22 if dtype == F32 else -23) * (D + 8) * row.double().abs().sum(-1) * k.abs().amax()


def check_rows(got, q, c, new, lens, scale, window=None, keep_first=0, wide=False, dtype=BF16):
    """Every row of ``got`` within its bound.  ``wide``: some rows may come from the kernels for wide pages."""
    want, weights = p8.attention(q, c, new, lens, scale, window, keep_first)
    R, t = q.shape[1] // c.G, 0
    for b, n in enumerate(new):
        k, v = c.values(b)
        v = v.repeat_interleave(R, 0)  # [H, L, D]
        largest = c.scales[b][1].repeat_interleave(c.page, 1)[:, : lens[b]].repeat_interleave(R, 0) * 448  # [H, L]
        for i in range(n):
            w = weights[b][i]  # [H, L]
            spread = torch.einsum("hl,hld->hd", w, v.abs())
            grow = torch.expm1((2 * score_error(q[t], k, scale, dtype)).clamp(max=20.0))[:, None] * spread
            if dtype == F32:
                tol = grow + 2.0 ** -20 * spread + 2.0 ** -23 * want[t].abs()
            else:
                floor = 2.0 ** -31 * lens[b] * (w * largest).amax(-1)[:, None]
                tol = grow + ((U if wide else HALF) + HALF / 2) * spread + floor + U * want[t].abs() + 1e-30
            diff = (got[t].double() - want[t]).abs()
            assert bool((diff <= tol).all()), (b, i, float((diff / tol).max()))
            t += 1
    return want


# ---- rounding and layout -------------------------------------------------------------------------------------------------


def strange(qkv, H, G, D):
    """Rows with equal numbers, zeros, half ways, and numbers far apart."""
    T = qkv.shape[0]
    qkv[0, H * D:H * D + 8] = 3.0
    qkv[1 % T, H * D:(H + 1) * D] = 0.0
    qkv[2 % T, (H + G) * D:(H + G + 1) * D] *= 1e-30
    qkv[3 % T, (H + G) * D + 5] = 1e30
    qkv[4 % T, H * D:H * D + 4] = torch.tensor([1.0625, -1.1875, 0.96875, 2.125])  # half ways between numbers of 4 bits
    qkv[5 % T, H * D + 9] = -0.0
    return qkv


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 16), (256, 8), (16, 4), (32, 3), (48, 16), (80, 5), (176, 16), (240, 7), (128, 100), (256, 70)])
def test_values_are_written_by_the_definition(ops, dtype, D, page):
    """Without norm and rotation what is written is the projection itself: the same bytes as the plain form's, and nothing else is touched; the
    second step goes on behind the first, in the middle of pages."""
    H, G = 4, 2
    g = torch.Generator().manual_seed(D)
    steps = [([page + 2, 1, page], [page + 2, 1, page]), ([3, 2, 1], [page + 5, 3, page + 1]), ([1, 1, 1], [page + 6, 4, page + 2])]
    table = torch.tensor([[5, 1, 4], [2, -1, 0], [7, 3, 6]], dtype=torch.int32)
    if page < 8:  # (more pages)
        table = torch.tensor([[5, 1, 4, 8, 9], [2, 10, 0, 11, 12], [7, 3, 6, 13, 14]], dtype=torch.int32)
    pages = torch.randint(0, 256, (16, G, p8.page_bytes(D, page)), generator=g, dtype=torch.uint8)
    want, dev = pages.clone(), pages.cuda()
    rows = [torch.zeros((2, G, 0, D), dtype=torch.float64) for _ in range(3)]
    for new, lens in steps:
        T = sum(new)
        qkv = strange(torch.randn((T, (H + 2 * G) * D), generator=g), H, G, D).to(dtype)
        at = 0
        for b, n in enumerate(new):
            kv = qkv[at:at + n, H * D:].float().view(n, 2, G, D).permute(1, 2, 0, 3)
            rows[b] = torch.cat([rows[b], p8.four_bits(kv)], 2)
            at += n
            for i in range((lens[b] - n) // page, (lens[b] - 1) // page + 1):
                if table[b, i] >= 0:
                    for which in range(2):
                        for h in range(G):
                            p8.write_rows(want, int(table[b, i]), h, page, which, rows[b][which, h, i * page:(i + 1) * page])
        x = qkv.cuda()
        ops.qk_norm_rope_store_8bit(x, num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                    step=p8.step_of(new, lens, page), block_table=table.cuda(), pages=dev, page_size=page)
        assert torch.equal(dev.cpu(), want)
        assert torch.equal(x.cpu().view(torch.uint8), qkv.view(torch.uint8)), "queries without norm and rotation stay as they are"
    lens = steps[-1][1]
    for out in (F32, BF16):
        k, v = ops.unpack_8bit(dev, num_kv_heads=G, head_dim=D, page_size=page, block_table=table[::2].contiguous().cuda(), kv_lens=i32(lens[::2]),
                               max_kv_len=max(lens), dtype=out)
        n = k.shape[0] // 2
        for s, b in enumerate((0, 2)):
            for got, which in ((k, 0), (v, 1)):
                got = got[s * n:(s + 1) * n].transpose(1, 2).reshape(-1, G, D).transpose(0, 1).double().cpu()
                whole = torch.zeros((G, n * page, D), dtype=torch.float64)
                for i in range(-(-lens[b] // page)):
                    m = min(page, lens[b] - i * page)
                    for h in range(G):
                        whole[h, i * page:i * page + m] = p8.read_rows(want[int(table[b, i]), h], D, page, which, m)[0]
                assert torch.equal(got, whole), "exact in both types, zero behind the last token"


@pytest.mark.parametrize("D,page,dtype", [(128, 16, F32), (64, 32, BF16), (80, 5, F32), (256, 24, F32)])
def test_tokens_one_by_one_end_as_tokens_at_once(ops, D, page, dtype):
    """Whatever the portions, a page holds the same bytes in the end: magnitudes that grow from token to token make scales grow on the way."""
    H, G, T = 1, 2, 3 * page + 2
    g = torch.Generator().manual_seed(page)
    grow = torch.exp(torch.randn((T, 1), generator=g) * 8)
    qkv = (torch.randn((T, (H + 2 * G) * D), generator=g) * grow * torch.exp(3 * torch.randn((T, (H + 2 * G) * D), generator=g))).to(dtype)
    qkv[5, D + 3] = math.inf
    table = torch.randperm(4, generator=g).int()[None].cuda()
    results = []
    for cuts in ([T], [1] * T, [2, 7, 1, 1, page, T]):
        pages = torch.zeros((4, G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
        at = 0
        for n in cuts:
            n = min(n, T - at)
            if n < 1:
                break
            ops.qk_norm_rope_store_8bit(qkv[at:at + n].cuda(), num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None,
                                        sin=None, step=p8.step_of([n], [at + n], page), block_table=table, pages=pages, page_size=page)
            at += n
        while at < T:
            ops.qk_norm_rope_store_8bit(qkv[at:at + 1].cuda(), num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0,
                                        cos=None, sin=None, step=p8.step_of([1], [at + 1], page), block_table=table, pages=pages, page_size=page)
            at += 1
        results.append(pages)
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


def test_how_far_values_are_off(ops):
    """Half a step of 4 significant bits, 2^-4 of the value, or less than 2^-9 of the scale; the scale is at most 2 / 448 of the largest."""
    D, page, G, T = 128, 16, 4, 200
    g = torch.Generator().manual_seed(3)
    qkv = (torch.randn((T, (1 + 2 * G) * D), generator=g) * torch.exp(4 * torch.randn((T, (1 + 2 * G) * D), generator=g))).cuda()
    pages = torch.zeros((T // page + 1, G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    table = torch.arange(T // page + 1, dtype=torch.int32, device="cuda")[None]
    step = p8.step_of([T], [T], page)
    ops.qk_norm_rope_store_8bit(qkv, num_heads=1, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                step=step, block_table=table, pages=pages, page_size=page)
    k, v = ops.unpack_8bit(pages, num_kv_heads=G, head_dim=D, page_size=page, block_table=table, kv_lens=step.kv_lens, max_kv_len=T, dtype=F32)
    for got, want in ((k, qkv[:, D:(1 + G) * D]), (v, qkv[:, (1 + G) * D:])):
        want = torch.nn.functional.pad(want.reshape(T, G, D), (0, 0, 0, 0, 0, -T % page)).view(-1, page, G, D).transpose(1, 2).double()
        scale = want.abs().amax((2, 3), keepdim=True) * (1 + 2.0 ** -4) * 2 / 448
        assert bool(((got.double() - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -4 * want.abs() + 2.0 ** -9 * scale
                                                                  * (want.abs() < 2.0 ** -6 * scale))).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3.4e38])
def test_what_is_not_finite_becomes_nan_and_nothing_else(ops, bad):
    D, page, G = 128, 16, 2
    qkv = torch.randn((1, (1 + 2 * G) * D), generator=torch.Generator().manual_seed(1))
    clean = qkv.clone()
    qkv[0, D + 3] = bad
    clean[0, D + 3] = 0.0
    both = []
    for x in (qkv, clean):
        pages = torch.zeros((1, G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
        step = p8.step_of([1], [1], page)
        ops.qk_norm_rope_store_8bit(x.cuda(), num_heads=1, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                    step=step, block_table=i32([[0]]), pages=pages, page_size=page)
        both.append(ops.unpack_8bit(pages, num_kv_heads=G, head_dim=D, page_size=page, block_table=i32([[0]]), kv_lens=step.kv_lens, max_kv_len=1, dtype=F32))
    (k, v), (k0, v0) = both
    assert bool(k[0, 0, 0, 3].isnan()), "(3.4e38 rounds beyond float32)"
    k[0, 0, 0, 3] = 0.0
    assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [128, 64, 256, 48])
def test_numbers_that_round_beyond_float32_under_the_largest_scale(ops, D, dtype):
    """3.2e38 rounds to 1.875 * 2^127 and makes the scale 2^120, under which 3.4e38 (bfloat16: 3.39e38), which rounds beyond float32, is no more than 256
    scales: not a number like elsewhere, also among large numbers; by the same bytes at every size, in the step that makes the scale and later."""
    G, page, T = 2, 8, 5
    g = torch.Generator().manual_seed(D)
    qkv = (torch.rand((T, (1 + 2 * G) * D), generator=g) + 0.5) * 1e37
    qkv[0, 2 * D + 3], qkv[2, D + 9] = 3.2e38, -3.2e38
    for row, col in ((0, 2 * D + 1), (1, D + 1), (2, 2 * D + 17), (3, D + 10), (4, 2 * D + 30), (4, 3 * D + 30)):
        qkv[row, col] = 3.4e38 if dtype == F32 else 3.39e38
    qkv[4, D + 5] = -3.39e38
    qkv = qkv.to(dtype)
    want = torch.zeros((1, G, p8.page_bytes(D, page)), dtype=torch.uint8)
    rows = p8.four_bits(qkv[:, D:].float().view(T, 2, G, D).permute(1, 2, 0, 3))
    assert int(rows.isnan().sum()) == 7 and p8.scale_exponent(rows[0, 1]) == 120
    for which in range(2):
        for h in range(G):
            p8.write_rows(want, 0, h, page, which, rows[which, h])
    for cuts in ([5], [3, 1, 1]):
        pages, at = torch.zeros_like(want).cuda(), 0
        for n in cuts:
            ops.qk_norm_rope_store_8bit(qkv[at:at + n].cuda(), num_heads=1, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None,
                                        sin=None, step=p8.step_of([n], [at + n], page), block_table=i32([[0]]), pages=pages, page_size=page)
            at += n
        assert torch.equal(pages.cpu(), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,rot,pairing", [(128, 128, "half"), (64, 64, "interleaved"), (256, 256, "half"), (128, 64, "half"), (80, 80, "half"),
                                           (48, 32, "interleaved"), (32, 32, "half")])
def test_norm_and_rotation_are_those_of_the_wide_cache(ops, dtype, D, rot, pairing):
    """Queries within a rounding of ``qk_norm_rope_store``'s; keys: those of its float32 keys, but where one lies within float32's rounding of a
    border between two numbers, which are 2^-3 of it apart."""
    H, G, page, T = 6, 2, 8, 37
    g = torch.Generator().manual_seed(D + rot)
    qkv = torch.randn((T, (H + 2 * G) * D + 16), generator=g).to(dtype).cuda()[:, : (H + 2 * G) * D]
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).cuda() for _ in range(2))
    ang = torch.arange(64)[:, None] * 1e4 ** (-torch.arange(0, rot, 2) / rot)
    cos, sin = ang.cos().contiguous().cuda(), ang.sin().contiguous().cuda()
    step = p8.step_of([T], [T], page)
    step.positions += 3  # (angles go by positions, places by the lengths)
    table = torch.randperm(8, generator=g).int()[None].cuda()
    wide = qkv.float().contiguous()
    kp, vp = (torch.zeros((8, G, page, D), device="cuda") for _ in range(2))
    same = dict(num_heads=H, num_kv_heads=G, head_dim=D, q_weight=qw, k_weight=kw, eps=1e-6, cos=cos, sin=sin, page_size=page, pairing=pairing)
    rows = torch.arange(1, dtype=torch.int32, device="cuda").expand(T).contiguous() * 0
    pos_table = torch.zeros((1, 8), dtype=torch.int32, device="cuda")  # page size 8: the wide cache places tokens by their positions
    pos_table[0] = torch.arange(8)
    ops.qk_norm_rope_store(wide, k_pages=kp, v_pages=vp, write_kv=True, positions=step.positions, token_seq=rows, block_table=pos_table, **same)
    args = dict(same, step=step, block_table=table)
    pages = torch.zeros((8, G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    q = torch.full((T, H * D), math.nan, dtype=dtype, device="cuda")
    before = qkv.clone()
    ops.qk_norm_rope_store_8bit(qkv, pages=pages, q_out=q, **args)
    assert torch.equal(qkv, before), "with q_out the projection stays as it is"
    # a turned element is a difference of two products, each at most the pair's length, which turning keeps and which is at most
    # sqrt(2) times the head's largest element: the two ways round those products and the norm (a few units of 2^-24), and store the
    # result rounded to its own type
    want = wide[:, : H * D].view(T, H, D)
    err = (q.float().view(T, H, D) - want).abs()
    assert bool((err <= 2.0 ** -20 * 2 ** 0.5 * want.abs().amax(-1, keepdim=True) + (U * want.abs() if dtype == BF16 else 0)).all())
    k, v = ops.unpack_8bit(pages, num_kv_heads=G, head_dim=D, page_size=page, block_table=table, kv_lens=step.kv_lens, max_kv_len=T, dtype=F32)
    for got, src, exact in ((k, kp, False), (v, vp, True)):
        got = got.transpose(1, 2).reshape(-1, G, D)[:T].cpu().double()
        src = src.transpose(1, 2).reshape(-1, G, D)[3:3 + T].cpu()
        rounded = p8.four_bits(src)
        want = torch.empty_like(rounded)
        for i in range(0, T, page):
            for h in range(G):
                want[i:i + page, h] = p8.held(rounded[i:i + page, h], p8.scale_exponent(rounded[i:i + page, h]))
        diff = (got - want).abs()
        if exact:
            assert torch.equal(got, want)
        else:  # a step of 2^-3 at most (and what is cut), where the key lies next to a border
            step_size = 2.0 ** -3 * want.abs() * (1 + 2.0 ** -3) + 2.0 ** -8 * src.abs().amax() / 224
            assert bool((diff <= step_size).all()) and float((diff > 0).float().mean()) < 1e-3
    # in place, and without writing keys
    again = qkv.clone()
    ops.qk_norm_rope_store_8bit(again, pages=pages, **args)
    assert torch.equal(again[:, : H * D], q)
    kept = pages.clone()
    ops.qk_norm_rope_store_8bit(qkv[:, : H * D], pages=pages, q_out=q, write_kv=False, **args)
    assert torch.equal(pages, kept)


def test_positions_outside_the_tables_write_nothing_and_are_reported(ops):
    from qwen3_runtime_b200.ops.cuda import KernelError

    for D in (128, 48):
        pages = torch.zeros((2, 1, p8.page_bytes(D, 16)), dtype=torch.uint8, device="cuda")
        qkv = torch.randn((2, 3 * D), device="cuda")
        cos = torch.ones((4, D // 2), device="cuda")
        args = dict(num_heads=1, num_kv_heads=1, head_dim=D, q_weight=None, k_weight=None, eps=0.0, pages=pages, page_size=16)
        step = p8.step_of([2], [2], 16)
        step.positions = i32([4, -1])
        with pytest.raises(KernelError, match="rotation tables"):
            ops.qk_norm_rope_store_8bit(qkv.clone(), cos=cos, sin=cos, step=step, block_table=i32([[0]]), **args)
            ops.raise_if_kernel_error()
        assert bool((pages[0, :, : 16 * D] == 0).all()), "no key"
        pages.zero_()
        # places without a page in the table, and tables that name none: nothing is written
        ops.qk_norm_rope_store_8bit(qkv.clone(), cos=None, sin=None, step=p8.step_of([2], [34], 16), block_table=i32([[0, 1]]), **args)
        ops.qk_norm_rope_store_8bit(qkv.clone(), cos=None, sin=None, step=p8.step_of([2], [2], 16), block_table=i32([[-1]]), **args)
        ops.qk_norm_rope_store_8bit(qkv.clone(), cos=None, sin=None, step=p8.step_of([1, 1], [1, 1], 16), block_table=i32([[2], [-5]]), **args)
        gone = p8.step_of([1, 1], [1, 1], 16)
        gone.kv_lens.zero_()  # (sequences of nothing, although they bring a token)
        ops.qk_norm_rope_store_8bit(qkv.clone(), cos=None, sin=None, step=gone, block_table=i32([[0], [1]]), **args)
        ops.raise_if_kernel_error()
        assert not bool(pages.any())


def test_a_page_that_is_used_again_starts_anew(ops):
    """Whatever a page holds, its first token makes its scale; what lies behind the last token says nothing."""
    D, page = 128, 16
    pages = torch.full((1, 1, p8.page_bytes(D, page)), 255, dtype=torch.uint8, device="cuda")
    x = torch.randn((3, 3 * D), generator=torch.Generator().manual_seed(0)).cuda()
    args = dict(num_heads=1, num_kv_heads=1, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, block_table=i32([[0]]), page_size=page)
    for scale in (1e6, 1.0, 1e-6):
        fresh = torch.full_like(pages, 255)
        for p in (pages, fresh):
            for n in (1, 2):
                ops.qk_norm_rope_store_8bit(x[n - 1:2 * n - 1] * scale, step=p8.step_of([n], [2 * n - 1], page), pages=p, **args)
        assert torch.equal(*(torch.stack(ops.unpack_8bit(p, num_kv_heads=1, head_dim=D, page_size=page, block_table=i32([[0]]), kv_lens=i32([3]),
                                                         max_kv_len=3, dtype=F32)) for p in (pages, fresh)))


@pytest.mark.parametrize("new,single", [([1] * 70, True), ([2, 1] * 40, False)])
def test_many_sequences(ops, new, single):
    """More sequences than a warp scans at a time; some bring nothing."""
    H, G, D, page = 2, 1, 64, 16
    if not single:
        new = [n * (i % 5 != 3) for i, n in enumerate(new)]
    lens = [(7 * i) % 40 + n for i, n in enumerate(new)]
    g = torch.Generator().manual_seed(1)
    whole = [torch.randn((n, (H + 2 * G) * D), generator=g) for n in lens]
    table = torch.randperm(4 * len(new), generator=g).int().view(len(new), 4).cuda()
    both = []
    for steps in ([(lens, lens)], [([n - m for n, m in zip(lens, new)],) * 2, (new, lens)]):
        pages = torch.zeros((4 * len(new), G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
        for brings, upto in steps:
            x = torch.cat([w[L - n:L] for w, n, L in zip(whole, brings, upto)])
            step = p8.step_of(brings, upto, page)
            ops.qk_norm_rope_store_8bit(x.cuda(), num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                        step=step, block_table=table, pages=pages, page_size=page)
        both.append(pages)
    assert torch.equal(*both)


# ---- attention --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("H,G,D,page", [(8, 2, 128, 16), (4, 4, 128, 16), (16, 2, 128, 32), (12, 1, 128, 16), (16, 1, 64, 16), (2, 2, 64, 8),
                                        (6, 2, 256, 16), (16, 1, 256, 64), (8, 2, 128, 5), (8, 2, 64, 24), (5, 1, 128, 48), (8, 1, 256, 3)])
@pytest.mark.parametrize("slices", [None, 1, 3, -3, 8, 9, 16, 40])
def test_decoded_tokens(ops, H, G, D, page, slices):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 611]
    c = p8.Cache(lens, G, D, page, seed=H + D, k_scale=1.5)
    new = [1] * len(lens)
    q = queries(len(lens), H, D, 7, extra=8)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, slices=slices)
    check_rows(got, q[:, : H * D].view(-1, H, D), c, new, lens, D ** -0.5)


@pytest.mark.parametrize("keep_first", [0, 1, 16, 40, 300])
@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 5000])
@pytest.mark.parametrize("page,D", [(16, 128), (8, 64), (5, 128), (32, 256)])
def test_decoded_tokens_behind_a_window(ops, window, keep_first, page, D):
    """Pages that the window has passed are gone (-1), but for those of the first tokens."""
    lens = [1, 40, 64, 333, 500]
    c = p8.Cache(lens, 2, D, page, seed=window)
    table = c.table.clone()
    for b, n in enumerate(lens):
        table[b, -(-keep_first // page): max(0, n - window) // page] = -1
    q = queries(len(lens), 8, D, 3)
    for slices in (None, 4, -4):
        got = attend(ops, c, q, [1] * len(lens), lens, 8, D ** -0.5, window=window, keep_first=keep_first, table=table, slices=slices)
        check_rows(got, q.view(-1, 8, D), c, [1] * len(lens), lens, D ** -0.5, window=window, keep_first=keep_first)


def test_a_long_cache(ops):
    lens = [20011, 9000]
    c = p8.Cache(lens, 1, 128, 16, seed=5, k_scale=2.0)
    q = queries(2, 4, 128, 3)
    for slices in (None, 1, 16, -16, 64):
        got = attend(ops, c, q, [1, 1], lens, 4, 128 ** -0.5, slices=slices)
        check_rows(got, q.view(-1, 4, 128), c, [1, 1], lens, 128 ** -0.5)
    got = attend(ops, c, q, [1, 1], lens, 4, 128 ** -0.5, window=7000, keep_first=2000)
    check_rows(got, q.view(-1, 4, 128), c, [1, 1], lens, 128 ** -0.5, window=7000, keep_first=2000)


def test_a_page_as_large_as_they_come(ops):
    """Codes that end just in front of 2^31: those that were there are cut to the last, and no others."""
    D, page, new = 256, (1 << 23) - 1, 5
    pages = torch.full((1, 1, p8.page_bytes(D, page)), 0x38, dtype=torch.uint8, device="cuda")  # ones
    pages[0, 0, 2 * page * D:2 * page * D + 8] = torch.tensor([1.0, 1.0]).view(torch.uint8).cuda()
    x = torch.full((new, 3 * D + 1), 2.0, device="cuda")[:, : 3 * D]  # (rows that do not begin at 16 bytes: the form for all sizes)
    x[:, ::D] = 1000.0  # rounds to 1024: under a scale of 4
    ops.qk_norm_rope_store_8bit(x, num_heads=1, num_kv_heads=1, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                step=p8.step_of([new], [page], page), block_table=i32([[0]]), pages=pages, page_size=page)
    ops.raise_if_kernel_error()
    assert pages[0, 0, 2 * page * D:2 * page * D + 8].cpu().view(torch.float32).tolist() == [4.0, 4.0]
    for codes in pages[0, 0, : 2 * page * D].view(2, page, D):
        assert bool((codes[: page - new] == 0x28).all()), "a quarter"
        for row in range(page - new, page):
            want = torch.full((D,), 0x30, dtype=torch.uint8)
            want[p8.channel_at(D, row)[0]] = 0x78
            assert torch.equal(codes[row].cpu(), want)


def test_offsets_beyond_32_bits(ops):
    """Pages whose bytes lie more than 2^31 (and 2^32) behind the first."""
    G, D, page = 8, 128, 16
    c = p8.Cache([40], G, D, page, seed=8)
    rec = p8.page_bytes(D, page)
    count = (1 << 32) // (G * rec) + 8
    big = torch.zeros((count, G, rec), dtype=torch.uint8, device="cuda")
    ids = [count - 1, (1 << 31) // (G * rec) + 3, count - 4]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    for i, page_id in enumerate(ids):
        big[page_id] = c.pages[int(c.table[0, i])].cuda()
    q = queries(1, 16, D, 2)
    step = p8.step_of([1], [40], page)
    dev, out = q.cuda(), torch.empty((1, 16 * D), dtype=BF16, device="cuda")
    args = dict(num_heads=16, pages=big, block_table=table, scale=D ** -0.5, **sizes(c))
    ops.paged_attention_8bit(dev, dev.stride(0), out=out, step=step, **args)
    check_rows(out.cpu().view(1, 16, D), q.view(1, 16, D), c, [1], [40], D ** -0.5)
    k, _v = ops.unpack_8bit(big, block_table=table, kv_lens=step.kv_lens, max_kv_len=40, dtype=F32, **sizes(c))
    assert torch.equal(k.transpose(1, 2).reshape(-1, G, D)[:40].cpu(), c.values(0)[0].transpose(0, 1).float())
    q = queries(2, 16, D, 2, F32)
    got = torch.empty((2, 16 * D), device="cuda")
    ops.paged_attention_8bit(q.cuda(), 16 * D, out=got, step=p8.step_of([2], [40], page), **args)
    check_rows(got.cpu().view(2, 16, D), q.view(2, 16, D), c, [2], [40], D ** -0.5, dtype=F32)
    x = torch.randn((2, 18 * D), generator=torch.Generator().manual_seed(1))
    ops.qk_norm_rope_store_8bit(x.cuda(), num_heads=2, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                step=p8.step_of([2], [42], page), block_table=table, pages=big, page_size=page)
    for h in range(G):
        rows = torch.cat([c.values(0)[0][h, 32:], p8.four_bits(x[:, (2 + h) * D:(3 + h) * D])])
        want = p8.held(rows, p8.scale_exponent(rows))
        assert torch.equal(p8.read_rows(big[ids[2], h].cpu(), D, page, 0, 10)[0], want)


def test_a_key_or_value_that_is_not_finite_stays_with_its_head(ops):
    def mutate(b, k, v):
        if b == 1:
            k[0, 7, 3] = math.nan
            v[1, 9, 100] = math.inf

    lens = [30, 30]
    c = p8.Cache(lens, 3, 128, 16, seed=1, mutate=mutate)
    q = queries(2, 6, 128, 5)
    for slices in (1, 2):
        got = attend(ops, c, q, [1, 1], lens, 6, 128 ** -0.5, slices=slices)
        assert bool(got[0].isfinite().all()) and bool(got[1, 4:].isfinite().all())
        assert bool(got[1, :2].isnan().all()), "a key that is not a number: the row's weights are none"
        assert bool(got[1, 2:4, 100].isnan().all()), "its channel"
        got[1, 2:4, 100] = 0
        assert bool(got[1, 2:4].isfinite().all())
    hidden = attend(ops, c, q, [1, 1], lens, 6, 128 ** -0.5, window=20, keep_first=5)
    assert bool(hidden.isfinite().all()), "outside the window they are not seen"


def test_far_scores_and_zero_queries(ops):
    """Rows whose weights lie on one token, rows of equal weights, scores far apart between the slices, queries far apart in size."""
    lens = [300, 300, 300]

    def mutate(b, k, v):
        if b == 1:
            k[:, 250] *= 30
            k[:, 10] *= -20

    c = p8.Cache(lens, 2, 128, 16, seed=2, mutate=mutate)
    q = queries(3, 4, 128, 9).view(3, 4, 128)
    q[0, 1] = 0
    q[1] *= 8
    q[2, 0, 5:] = 0
    q[2, 1] *= 2.0 ** -20
    q[2, 2, ::2] *= 2.0 ** -12
    q[2, 3] *= 2.0 ** -90
    for slices in (1, 4):
        got = attend(ops, c, q.view(3, -1), [1] * 3, lens, 4, 128 ** -0.5, slices=slices)
        check_rows(got, q, c, [1] * 3, lens, 128 ** -0.5)


@pytest.mark.parametrize("spread", [10.0, 60.0, 2.0 ** 30])
def test_scales_that_lie_far_apart(ops, spread):
    """Pages whose values are a power of ``spread`` times as large as others', with the large ones on the tokens of little weight."""
    lens = [200, 130]

    def mutate(b, k, v):
        v[:, 16:32] *= spread
        v[:, 96:112] /= spread
        v[:, 48:64] = 0
        k[:, :16] *= 0.01
        k[:, 100] *= 3

    c = p8.Cache(lens, 2, 128, 16, seed=4, mutate=mutate)
    q = queries(2, 8, 128, 9).view(2, 8, 128)
    k = c.values(0)[0][:, 100]
    q[0, :4] = k[0].to(BF16) * 0.3
    q[1, 4:] *= 0
    for slices in (1, 3, -3):
        got = attend(ops, c, q.view(2, -1), [1] * 2, lens, 8, 128 ** -0.5, slices=slices)
        check_rows(got, q, c, [1] * 2, lens, 128 ** -0.5)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_beyond_all_measure(ops, sign):
    """Scores near +-10^33: one token has all the weight, rows whose scores all lie far below zero get their results."""
    D, lens = 128, [40]

    def mutate(b, k, v):
        k[:] = k.abs() * 1e16

    c = p8.Cache(lens, 1, D, 16, seed=3, mutate=mutate)
    q = (queries(1, 2, D, 1).view(1, 2, D).abs() * 1e16 * sign).to(BF16)
    want, weights = p8.attention(q, c, [1], lens, D ** -0.5)
    for slices in (1, 2):
        got = attend(ops, c, q.view(1, -1), [1], lens, 2, D ** -0.5, slices=slices)
        for h in range(2):
            top = weights[0][0, h].topk(2).values
            if float(top[0]) > 1 - 1e-9:  # (else two scores lie within float32's rounding)
                assert float((got[0, h].double() - want[0, h]).abs().max()) <= U * float(want[0, h].abs().max()) * 2


@pytest.mark.parametrize("first,end", [(0, 200), (200, 300), (128, 256), (0, 300)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_beyond_float32_in_one_slice(ops, dtype, first, end):
    """Products below -3.4e38 weigh nothing beside others, wherever slices end; where there are no others, the row is none."""
    H, G, D, lens = 4, 2, 128, [300]

    def mutate(b, k, v):
        k[:, :, 0] = 0
        k[:, first:end, 0] = -1e30

    c = p8.Cache(lens, G, D, 16, seed=4, mutate=mutate)
    q = torch.zeros((1, H, D), dtype=dtype)  # (the other tokens weigh alike: beside 1e30 a row's other numbers are rounded away)
    q[0, :, 0] = 1e30
    for slices in (1, 2, -2, 3, -3):
        got = attend(ops, c, q.view(1, -1), [1], lens, H, D ** -0.5, slices=slices, dtype=dtype)
        if end - first == 300:
            assert bool(got.isnan().all())
            continue
        keep = [j for j in range(300) if not first <= j < end]
        sub = p8.Cache([], G, D, 16)
        sub.kv, sub.scales = [c.kv[0][:, :, keep]], [torch.ones((2, G, 19), dtype=torch.float64)]
        check_rows(got, torch.zeros_like(q), sub, [1], [len(keep)], D ** -0.5, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,G,D,page,window,keep_first", [
    (8, 2, 128, 16, None, 0), (8, 2, 64, 8, None, 0), (8, 2, 128, 16, 20, 0), (8, 2, 128, 16, 20, 7), (4, 2, 256, 16, None, 0), (4, 2, 256, 16, 30, 20),
    (4, 1, 80, 5, None, 0), (20, 1, 128, 16, None, 0), (4, 2, 48, 16, 9, 3), (8, 2, 128, 8, 3, 70), (4, 2, 64, 24, 12, 30), (6, 2, 128, 16, 12, 30)])
def test_portions_of_prompts_and_single_tokens_in_one_step(ops, dtype, H, G, D, page, window, keep_first):
    new, lens = [1, 33, 1, 5, 18, 150], [70, 33, 1, 90, 50, 290]
    c = p8.Cache(lens, G, D, page, seed=D, width=20 if page == 16 else None)
    table = c.table.clone()
    if window:  # what every new token's window has passed is gone
        for b, (n, L) in enumerate(zip(new, lens)):
            table[b, -(-keep_first // page): max(0, L - n - window + 1) // page] = -1
    q = queries(sum(new), H, D, 4, dtype, extra=16)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first, dtype=dtype, table=table)
    check_rows(got, q[:, : H * D].view(-1, H, D), c, new, lens, D ** -0.5, window=window, keep_first=keep_first, wide=True, dtype=dtype)


@pytest.mark.parametrize("window,keep_first", [(1, 0), (63, 64), (64, 1), (65, 65), (128, 200), (300, 129), (1000, 5)])
def test_prompts_under_windows(ops, window, keep_first):
    """Windows and first tokens next to the borders of the tiles of 64 keys, long and short portions behind contexts."""
    H, G, D, page, new, lens = 8, 2, 128, 16, [400, 70, 2, 65], [400, 600, 333, 129]
    c = p8.Cache(lens, G, D, page, seed=window)
    table = c.table.clone()
    for b, (n, L) in enumerate(zip(new, lens)):
        table[b, -(-keep_first // page): max(0, L - n - window + 1) // page] = -1
    q = queries(sum(new), H, D, 4)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first, table=table)
    check_rows(got, q.view(-1, H, D), c, new, lens, D ** -0.5, window=window, keep_first=keep_first, wide=True)


@pytest.mark.parametrize("H,G,D,dtype", [(20, 1, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32), (6, 1, 16, F32), (3, 3, 240, BF16)])
@pytest.mark.parametrize("window,keep_first", [(None, 0), (100, 30)])
def test_single_tokens_of_other_sizes(ops, H, G, D, dtype, window, keep_first):
    lens = [1, 17, 130, 900]
    c = p8.Cache(lens, G, D, 16, seed=D)
    q = queries(4, H, D, 4, dtype)
    got = attend(ops, c, q, [1] * 4, lens, H, D ** -0.5, dtype=dtype, window=window, keep_first=keep_first)
    check_rows(got, q.view(-1, H, D), c, [1] * 4, lens, D ** -0.5, wide=True, dtype=dtype, window=window, keep_first=keep_first)


@pytest.mark.parametrize("window,keep_first", [(None, 0), (700, 0), (500, 300), (90, 600)])
def test_float32_is_the_same_in_every_company(ops, window, keep_first):
    """The same bits for a token alone, among others, and behind a longer table (slices joined by the block itself, or by the second kernel)."""
    H, G, D, page, lens = 4, 2, 64, 16, [1500, 40, 800]
    c = p8.Cache(lens, G, D, page, seed=3, width=100)
    q = queries(300, H, D, 4, F32)
    kw = dict(window=window, keep_first=keep_first, dtype=F32)
    together = attend(ops, c, q[:3], [1] * 3, lens, H, D ** -0.5, **kw)
    crowd = attend(ops, c, torch.cat([q[3:203], q[0:1], q[1:2], q[2:3]]), [201, 1, 1], lens, H, D ** -0.5, **kw)  # (enough blocks for one kernel)
    check_rows(together, q[:3].view(3, H, D), c, [1] * 3, lens, D ** -0.5, window=window, keep_first=keep_first, dtype=F32)
    for got, want in zip(crowd[-3:], together):
        assert torch.equal(got, want)


@pytest.mark.parametrize("page,D", [(48, 128), (80, 64), (160, 128), (256, 256), (67, 128)])
def test_pages_larger_than_what_a_block_takes_at_a_time(ops, page, D):
    """A block's next keys lie in the same page, or further on than one page behind."""
    H, G, lens = 8, 2, [1, 47, 48, 161, 700]
    c = p8.Cache(lens, G, D, page, seed=page)
    q = queries(len(lens), H, D, 5)
    rows, new = q.view(-1, H, D), [1] * len(lens)
    for slices in (None, 3, -3):
        check_rows(attend(ops, c, q, new, lens, H, D ** -0.5, slices=slices), rows, c, new, lens, D ** -0.5)
        got = attend(ops, c, q, new, lens, H, D ** -0.5, slices=slices, window=200, keep_first=90)
        check_rows(got, rows, c, new, lens, D ** -0.5, window=200, keep_first=90)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 20]])
@pytest.mark.parametrize("shift,extra", [(0, 4), (1, 0), (1, 3), (4, 8)])
def test_rows_of_queries_that_begin_anywhere(ops, new, shift, extra):
    """``shift`` elements behind a multiple of 16 bytes, rows ``extra`` elements apart."""
    H, G, D, lens = 8, 2, 128, [9, 40, 33]
    c = p8.Cache(lens, G, D, 16, seed=3)
    q = queries(sum(new), H, D, 4)
    T, width = q.shape[0], H * D + extra
    dev = torch.zeros(shift + T * width, dtype=BF16, device="cuda")[shift:].view(T, width)
    dev[:, : H * D] = q.cuda()
    out = torch.zeros(2 + T * H * D, dtype=BF16, device="cuda")[2:].view(T, H * D) if shift == 1 else torch.zeros_like(q, device="cuda")
    for window in (None, 12):
        ops.paged_attention_8bit(dev, width, num_heads=H, pages=c.pages.cuda(), block_table=c.table.cuda(), out=out, scale=D ** -0.5,
                                 step=p8.step_of(new, lens, 16), window=window, keep_first=2, **sizes(c))
        check_rows(out.cpu().view(T, H, D), q.view(T, H, D), c, new, lens, D ** -0.5, wide=True, window=window, keep_first=2 if window else 0)


@pytest.mark.parametrize("shift,extra", [(0, 4), (1, 0), (3, 5)])
def test_projections_that_begin_anywhere(ops, shift, extra):
    """Rows at any address and distance are written like aligned ones."""
    H, G, D, page, T = 2, 1, 128, 16, 20
    x = torch.randn((T, (H + 2 * G) * D), generator=torch.Generator().manual_seed(1)).to(BF16)
    width = x.shape[1] + extra
    dev = torch.zeros(shift + T * width, dtype=BF16, device="cuda")[shift:].view(T, width)[:, : x.shape[1]]
    dev.copy_(x)
    both, table = [], i32([[1, 0]])
    for y in (x.cuda(), dev):
        pages = torch.zeros((2, G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
        ops.qk_norm_rope_store_8bit(y, num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                    step=p8.step_of([T], [T], page), block_table=table, pages=pages, page_size=page)
        both.append(pages)
    assert torch.equal(*both)


@pytest.mark.parametrize("slices", [1, 4, -4])
def test_sequences_without_keys(ops, slices):
    """Length zero: results are zero; the others are as ever."""
    H, G, D, lens, page = 8, 2, 128, [20, 700, 31], 16
    c = p8.Cache(lens, G, D, page, seed=6)
    q = queries(3, H, D, 5)
    step = p8.step_of([1] * 3, lens, page)
    step.kv_lens[0] = 0
    got = attend(ops, c, q, [1] * 3, lens, H, D ** -0.5, slices=slices, step=step)
    assert bool((got[0] == 0).all())
    whole = attend(ops, c, q, [1] * 3, lens, H, D ** -0.5, slices=slices)
    assert torch.equal(got[1:], whole[1:])


def test_tokens_without_a_place_are_zero_in_the_general_form(ops):
    H, G, D, lens = 4, 2, 64, [20, 700, 31]
    c = p8.Cache(lens, G, D, 16, seed=6)
    q = queries(3, H, D, 5, F32)
    step = p8.step_of([1] * 3, lens, 16)
    step.positions = i32([-1, 699, 1 << 20])
    got = attend(ops, c, q, [1] * 3, lens, H, D ** -0.5, step=step, dtype=F32)
    assert bool((got[0] == 0).all()) and bool((got[2] == 0).all()) and bool(got[1].isfinite().all()) and bool(got[1].any())


@pytest.mark.parametrize("page", [16, 32, 5])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 20]])
def test_entries_that_are_no_pages_are_read_nowhere(ops, page, new):
    H, G, D, lens = 8, 2, 128, [90, 70, 60]
    c = p8.Cache(lens, G, D, page, seed=3)
    q = queries(sum(new), H, D, 4)
    table = c.table.clone()
    table[0, 0], table[0, 1] = -7, c.pages.shape[0]
    for slices in (1, 3):
        got, whole = (attend(ops, c, q, new, lens, H, D ** -0.5, table=t, slices=slices) for t in (table, c.table))
        assert torch.equal(got[new[0]:], whole[new[0]:])


def test_two_streams_at_once(ops):
    """Unequal steps under way together, each with workspaces of its own."""
    H, G, D = 8, 2, 128
    caches = [p8.Cache([5000, 1200], G, D, 16, seed=1), p8.Cache([3000, 64, 900], G, D, 16, seed=2)]
    made, alone = [], []
    for i, c in enumerate(caches):
        q = queries(len(c.lens), H, D, i)
        made.append((c, q.cuda(), c.pages.cuda(), c.table.cuda(), p8.step_of([1] * len(c.lens), c.lens, 16), torch.cuda.Stream()))
        alone.append(attend(ops, c, q, [1] * len(c.lens), c.lens, H, D ** -0.5, slices=-9))
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (c, q, pages, table, step, stream) in enumerate(made):
            with torch.cuda.stream(stream):
                out = torch.empty_like(q)
                ops.paged_attention_8bit(q, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=D ** -0.5, step=step,
                                         decode_slices=-9, **sizes(c))
                outs[i].append(out)
    torch.cuda.synchronize()
    for got, want in zip(outs, alone):
        assert all(torch.equal(x.cpu().view(want.shape), want) for x in got)


@pytest.mark.parametrize("window,keep_first", [(None, 0), (40, 6)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_steps(ops, dtype, window, keep_first):
    """Two captured steps of single tokens that share a pool of memory, replayed in turn with lengths that grow: each writes its tokens and attends
    to what is there, as uncaptured steps do."""
    H, G, D, page, width = 8, 2, 128, 16, 6
    g = torch.Generator().manual_seed(5)
    graphs, pool = [], None
    for i, lens in enumerate(([3, 40, 17], [30, 5])):
        B = len(lens)
        pages = torch.zeros((B * width, G, p8.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
        table = torch.randperm(B * width, generator=g).int().view(B, width).cuda()
        past = torch.randn((sum(lens), (H + 2 * G) * D), generator=g).to(dtype).cuda()
        step = p8.step_of([1] * B, [n + 1 for n in lens], page, captured_width=width)
        x = torch.zeros((B, (H + 2 * G) * D), dtype=dtype, device="cuda")
        out = torch.zeros((B, H * D), dtype=dtype, device="cuda")
        store = dict(num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, block_table=table, page_size=page)
        ops.qk_norm_rope_store_8bit(past, step=p8.step_of(lens, lens, page), pages=pages, **store)
        plain = pages.clone()

        def run(x=x, out=out, pages=pages, step=step, store=store, table=table):
            ops.qk_norm_rope_store_8bit(x, step=step, pages=pages, **store)
            ops.paged_attention_8bit(x, x.stride(0), num_heads=H, num_kv_heads=G, head_dim=D, pages=pages, block_table=table, out=out, page_size=page,
                                     scale=D ** -0.5, step=step, window=window, keep_first=keep_first, decode_slices=3)

        saved = pages.clone()
        run()
        torch.cuda.synchronize()
        pages.copy_(saved)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            run()
        pool = pool or graph.pool()
        graphs.append(dict(graph=graph, lens=list(lens), pages=pages, plain=plain, step=step, x=x, out=out, store=store, table=table))
    for turn in range(24):
        for s in graphs:
            row = torch.randn(s["x"].shape, generator=g).to(dtype)
            s["x"].copy_(row)
            now = [n + 1 for n in s["lens"]]
            s["step"].kv_lens.copy_(i32(now))
            s["step"].positions.copy_(i32(s["lens"]))
            s["step"].kv_longest.copy_(i32([max(now)]))
            s["graph"].replay()
            free = p8.step_of([1] * len(now), now, page)
            y, want = row.cuda(), torch.empty_like(s["out"])
            ops.qk_norm_rope_store_8bit(y, step=free, pages=s["plain"], **s["store"])
            ops.paged_attention_8bit(y, y.stride(0), num_heads=H, num_kv_heads=G, head_dim=D, pages=s["plain"], block_table=s["table"], out=want,
                                     page_size=page, scale=D ** -0.5, step=free, window=window, keep_first=keep_first, decode_slices=3)
            torch.cuda.synchronize()
            assert torch.equal(s["pages"], s["plain"])
            if dtype == F32:
                assert torch.equal(s["out"], want)
            else:  # (slices are cut by the same lengths)
                assert torch.equal(s["out"], want)
            s["lens"] = now


@pytest.mark.parametrize("dtype,H,G,D", [(BF16, 8, 2, 128), (BF16, 20, 4, 80), (BF16, 4, 2, 256), (F32, 4, 2, 64)])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
@pytest.mark.parametrize("new", [[1, 1], [700, 1]])
def test_any_scale(ops, dtype, H, G, D, scale, new):
    lens = [900, 300]
    c = p8.Cache(lens, G, D, 16, seed=6)
    q = queries(sum(new), H, D, 3, dtype)
    got = attend(ops, c, q, new, lens, H, scale, dtype=dtype)
    check_rows(got, q.view(-1, H, D), c, new, lens, scale, wide=True, dtype=dtype)


def test_steps_of_nothing(ops):
    c = p8.Cache([5], 2, 128, 16)
    pages, table = c.pages.cuda(), c.table.cuda()
    step = p8.step_of([], [], 16)
    out = torch.empty((0, 8 * 128), dtype=BF16, device="cuda")
    q = torch.empty((0, 12 * 128), dtype=BF16, device="cuda")
    args = dict(num_heads=8, pages=pages, block_table=table[:0], **sizes(c))
    before = pages.clone()
    ops.paged_attention_8bit(q, 12 * 128, out=out, scale=1.0, step=step, **args)
    ops.qk_norm_rope_store_8bit(q, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, step=step, **args)
    k, _v = ops.unpack_8bit(pages, block_table=table, kv_lens=i32([5]), max_kv_len=0, dtype=BF16, **sizes(c))
    assert k.shape[0] == 0 and torch.equal(pages, before)


def test_sequences_of_more_than_are_unpacked_at_a_time(ops):
    """Turns of sequences: the same results whatever they are."""
    H, G, D, page, new, lens = 8, 2, 128, 16, [9, 1, 30, 2, 17], [100, 70, 30, 64, 90]
    c = p8.Cache(lens, G, D, page, seed=9)
    q = queries(sum(new), H, D, 4)
    for kw in (dict(), dict(window=24, keep_first=4)):
        whole = attend(ops, c, q, new, lens, H, D ** -0.5, **kw)
        check_rows(whole, q.view(-1, H, D), c, new, lens, D ** -0.5, wide=True, **kw)
        ops.UNPACK_BYTES = 6 * 4 * G * page * D
        try:
            assert torch.equal(attend(ops, c, q, new, lens, H, D ** -0.5, **kw), whole)
        finally:
            del ops.UNPACK_BYTES


def test_a_cache_that_is_written_and_attended(ops):
    """The operators as a decoder's layer uses them: prompts in portions, then token after token, with norm and rotation; against the plain
    statements over the numbers that the cache holds."""
    H, G, D, page, scale = 8, 2, 128, 16, 128 ** -0.5
    g = torch.Generator().manual_seed(11)
    lens, total = [0, 0], [61, 40]
    x = [torch.randn((n, (H + 2 * G) * D), generator=g).to(BF16) for n in total]
    ang = torch.arange(80)[:, None] * 1e4 ** (-torch.arange(0, D, 2) / D)
    cos, sin = ang.cos().contiguous().cuda(), ang.sin().contiguous().cuda()
    w = (1 + 0.1 * torch.randn(D, generator=g)).cuda()
    pages = torch.full((9, G, p8.page_bytes(D, page)), 255, dtype=torch.uint8, device="cuda")
    table = torch.randperm(8, generator=g).int().view(2, 4).cuda()
    for new in ([30, 7], [9, 1], [1, 20], *[[1, 1]] * 12):
        lens = [a + n for a, n in zip(lens, new)]
        step = p8.step_of(new, lens, page)
        qkv = torch.cat([x[b][lens[b] - n:lens[b]] for b, n in enumerate(new)]).cuda()
        q = torch.empty((sum(new), H * D), dtype=BF16, device="cuda")
        ops.qk_norm_rope_store_8bit(qkv, num_heads=H, num_kv_heads=G, head_dim=D, q_weight=w, k_weight=w, eps=1e-6, cos=cos, sin=sin, step=step,
                                    block_table=table, pages=pages, page_size=page, q_out=q)
        out = torch.empty_like(q)
        ops.paged_attention_8bit(q, H * D, num_heads=H, num_kv_heads=G, head_dim=D, pages=pages, block_table=table, out=out, page_size=page,
                                 scale=scale, step=step)
        # what the cache holds now, as plain numbers
        c = p8.Cache([], G, D, page)
        bytes_now = pages.cpu()
        for b in range(2):
            kv, scales = torch.zeros((2, G, lens[b], D), dtype=torch.float64), torch.zeros((2, G, -(-lens[b] // page)), dtype=torch.float64)
            for i in range(scales.shape[2]):
                m = min(page, lens[b] - i * page)
                for which in range(2):
                    for h in range(G):
                        kv[which, h, i * page:i * page + m], scales[which, h, i] = p8.read_rows(bytes_now[int(table[b, i]), h], D, page, which, m)
            c.kv.append(kv)
            c.scales.append(scales)
        check_rows(out.cpu().view(-1, H, D), q.cpu().view(-1, H, D), c, new, lens, scale, wide=True)
        # and what it holds is what was projected, normed and turned, to 4 significant bits
        for b in range(2):
            rows = x[b][: lens[b], H * D:(H + G) * D].double().view(-1, G, D)
            y = rows / (rows.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.cpu().double()
            a = ang[: lens[b], None].double()
            y = torch.cat([y[..., :64] * a.cos() - y[..., 64:] * a.sin(), y[..., 64:] * a.cos() + y[..., :64] * a.sin()], -1).transpose(0, 1)
            assert bool(((c.kv[b][0] - y).abs() <= (2.0 ** -4 + 2.0 ** -18) * y.abs() + 2.0 ** -16 * y.abs().amax()).all())
