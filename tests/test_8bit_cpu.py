"""A cache in 8 bits, host side: sizes, the plain form's rounding, and what the kernel table refuses before it launches anything."""

import math
import random

import pytest
import torch

import plain_8bit as p8
from qwen3_runtime_b200.cache.layout import eight_bit_page_bytes
from qwen3_runtime_b200.ops.cuda import CudaOps, KernelError, unpacked_pages_4bit
from test_4bit_cpu import Table, i32
from test_4bit_steps_cpu import Elsewhere, elsewhere


def test_sizes():
    for D in range(16, 257, 16):
        for page in (1, 5, 16, 64):
            assert eight_bit_page_bytes(D, page) == p8.page_bytes(D, page) and eight_bit_page_bytes(D, page) % 16 == 0


def test_the_plain_codes_are_those_of_8_bit_floats():
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(p8.VALUES.nan_to_num(7e7), want.nan_to_num(7e7))
    for c in range(256):
        if c & 127 != 127:
            assert p8.code_of(p8.value_of(c) * 2.0 ** 5, 5) == c
    assert p8.code_of(math.nan, 3) & 127 == 127


def test_the_plain_rounding():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5000, generator=g) * torch.exp(9 * torch.randn(5000, generator=g))
    y = p8.four_bits(x)
    assert bool(((y - x.double()).abs() <= 2.0 ** -4 * x.double().abs()).all())
    # in float32's own bits, as the kernels do it
    bits = x.view(torch.int32)
    assert torch.equal(((bits + 0x7FFFF + ((bits >> 20) & 1)) & ~0xFFFFF).view(torch.float32).double(), y)
    e = p8.scale_exponent(y)
    assert float(y.abs().max()) <= 448 * 2.0 ** e and float(y.abs().max()) > 224 * 2.0 ** e
    z = p8.held(y, e)
    assert bool(((z - y).abs() < 2.0 ** (e - 9)).all()) and torch.equal(z[y.abs() >= 2.0 ** (e - 6)], y[y.abs() >= 2.0 ** (e - 6)])
    for more in (1, 3, 9, 40):  # cuts compose
        assert torch.equal(p8.held(p8.held(y, e), e + more), p8.held(y, e + more))
    assert p8.scale_exponent(torch.zeros(3, dtype=torch.float64)) == p8.LEAST
    assert bool(p8.four_bits(torch.tensor([math.inf, math.nan, 3.4e38])).isnan().all())


def test_the_cache_of_tensors_has_the_layout_of_single_rows():
    for D, page in ((80, 5), (64, 8), (128, 16), (256, 3)):
        c = p8.Cache([17, 3], 2, D, page, seed=1)
        whole = p8.values_of(c.pages, D, page)
        for b, n in enumerate(c.lens):
            for i in range(-(-n // page)):
                m = min(page, n - i * page)
                for h in range(2):
                    for which in range(2):
                        got, s = p8.read_rows(c.pages[int(c.table[b, i]), h], D, page, which, m)
                        want = c.kv[b][which, h, i * page:i * page + m]
                        assert torch.equal(got, want) and s == float(c.scales[b][which, h, i])
                        assert torch.equal(whole[which][int(c.table[b, i]), h, :m].double(), want)
                        again = c.pages.clone()
                        p8.write_rows(again, int(c.table[b, i]), h, page, which, want)
                        assert torch.equal(again, c.pages)


@pytest.fixture
def ops():
    table = Table()
    table._slices_cache = {}
    table._clusters_8bit = lambda D, wide, size: 9 * 148 * table.DECODE_8BIT_BLOCKS_PER_SM[D] // (10 * size)  # (about what a device holds)
    return table


def cache(D=128, page=16, G=2, count=4, layers=()):
    return torch.zeros((*layers, count, G, eight_bit_page_bytes(D, page)), dtype=torch.uint8)


def store_args(new=(3,), lens=(20,), H=4, G=2, D=128, page=16, step=None, **kw):
    T = sum(new)
    made = p8.step_of(list(new), list(lens), page, device="cpu")
    for name, value in (step or {}).items():
        setattr(made, name, value)
    return {**dict(qkv=torch.zeros((T, (H + 2 * G) * D)), num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0,
                   cos=None, sin=None, step=made, block_table=i32([[0, 1]] * len(new)), pages=cache(D, page, G), page_size=page), **kw}


@pytest.mark.parametrize("change,match", [
    (dict(head_dim=24), "multiples of 16"), (dict(head_dim=272), "multiples of 16"), (dict(page_size=0), "pages and heads"),
    (dict(num_kv_heads=0), "heads at least one"), (dict(pages=cache(page=8)), "dense uint8"), (dict(pages=cache().float()), "dense uint8"),
    (dict(pages=cache(layers=(2,))), "dense uint8"), (dict(pages=cache(G=4)[:, ::2]), "dense uint8"),
    (dict(block_table=i32([[0, 1]]).long()), "block table"), (dict(block_table=i32([0, 1])), "block table"),
    (dict(block_table=torch.zeros((1, 0), dtype=torch.int32)), "block table"), (dict(step=dict(positions=i32([0]))), "positions"),
    (dict(step=dict(positions=torch.arange(3))), "positions"), (dict(step=dict(kv_lens=torch.tensor([20]))), "lengths"),
    (dict(step=dict(kv_lens=i32([]))), "lengths"), (dict(step=dict(cu_seqlens=i32([0]))), "cu_seqlens"),
    (dict(step=dict(cu_seqlens=torch.tensor([0, 3]))), "cu_seqlens"), (dict(step=dict(host_cu_seqlens=[])), "host_cu_seqlens"),
    (dict(step=dict(host_cu_seqlens=[0, 2])), "host_cu_seqlens"), (dict(step=dict(num_seqs=2)), "a row per sequence"),
    (dict(step=dict(decode_only=True)), "single tokens"), (dict(q_weight=torch.zeros(64)), "norm weights"),
    (dict(k_weight=torch.zeros(128, dtype=torch.bfloat16)), "norm weights"), (dict(cos=torch.zeros((4, 64))), "together"),
    (dict(cos=torch.zeros((4, 65)), sin=torch.zeros((4, 65))), "rotation tables"), (dict(cos=torch.zeros((0, 64)), sin=torch.zeros((0, 64))), "rotation"),
    (dict(cos=torch.zeros((4, 64)).half(), sin=torch.zeros((4, 64)).half()), "rotation"), (dict(q_out=torch.zeros((3, 4 * 128)).bfloat16()), "queries"),
    (dict(q_out=torch.zeros((2, 4 * 128))), "queries"), (dict(qkv=torch.zeros((3, 7 * 128))), "projection"),
    (dict(qkv=torch.zeros((2, 8 * 128))), "a row per token"), (dict(qkv=torch.zeros((3, 8 * 128)).half()), "float32 and bfloat16"),
    (dict(qkv=torch.zeros((8 * 128, 3)).T), "unit-stride")])
def test_a_write_that_is_refused(ops, change, match):
    args = store_args(**change)
    with pytest.raises(KernelError, match=match):
        ops.qk_norm_rope_store_8bit(args.pop("qkv"), **args)
    assert not ops.calls


def test_writes_that_are_taken(ops):
    for args in (store_args(), store_args(new=(), lens=(), block_table=torch.zeros((0, 2), dtype=torch.int32)), store_args(D=80, page=5), store_args(new=(1, 1), lens=(1, 30)),
                 store_args(qkv=torch.zeros((3, 4 * 128)), write_kv=False)):
        ops.qk_norm_rope_store_8bit(args.pop("qkv"), **args)
    assert ops.calls == ["q3_store_8bit"] * 5


def test_pages_that_a_step_writes():
    """No fewer than any lengths touch, and one a sequence where each brings one token; asked once a step."""
    rnd = random.Random(1)
    for _ in range(300):
        page = rnd.randint(1, 20)
        new = [rnd.choice([0, 1, 1, rnd.randint(1, 60)]) for _ in range(rnd.randint(1, 6))]
        lens = [n + rnd.randint(0, 50) for n in new]
        step = p8.step_of(new, lens, page, device="cpu")
        units, most = CudaOps._written_pages("x", step, page)
        touched = sum((L - 1) // page - (L - n) // page + 1 for n, L in zip(new, lens) if n)
        assert units >= touched and most == max(1, *new) and (not step.decode_only or (units, most) == (len(new), 1))
        assert units <= sum(-(-n // page) + 1 for n in new if n)
        assert step.decode_only or CudaOps._written_pages("x", step, page) is CudaOps._written_pages("x", step, page)


def test_a_step_that_is_filled_anew_is_counted_anew():
    step = p8.step_of([3, 1], [3, 40], 16, device="cpu")
    assert CudaOps._written_pages("x", step, 16) == (3, 3)
    step.host_cu_seqlens[1:] = [1, 4]
    assert CudaOps._written_pages("x", step, 16) == (3, 3)
    step.host_cu_seqlens[1:] = [40, 41]
    step.num_tokens = 41
    assert CudaOps._written_pages("x", step, 16) == (5, 40)
    step.host_cu_seqlens = [0, 1, 41]
    assert CudaOps._written_pages("x", step, 16) == (5, 40)


def attention_args(new=(1, 1), lens=(20, 3), H=4, G=2, D=128, page=16, dtype=torch.bfloat16, **kw):
    step = p8.step_of(list(new), list(lens), page, device="cpu")
    T = sum(new)
    return {**dict(q=torch.zeros((T, H * D), dtype=dtype), q_stride=H * D, num_heads=H, num_kv_heads=G, head_dim=D, pages=cache(D, page, G),
                   block_table=i32([[0, 1], [2, 3]]), out=torch.zeros((T, H * D), dtype=dtype), page_size=page, scale=1.0, step=step), **kw}


@pytest.mark.parametrize("change,match", [
    (dict(lens=(33, 3)), "do not fit"), (dict(num_heads=3), "multiple of kv heads"), (dict(num_heads=0), "multiple of kv heads"),
    (dict(out=torch.zeros((2, 512))), "queries' type"),
    (dict(out=torch.zeros((2, 1024), dtype=torch.bfloat16)[:, :512]), "dense"), (dict(dtype=torch.float16), "float32 and bfloat16"),
    (dict(window=-1), "no fewer than none"), (dict(window=3, keep_first=-1), "no fewer than none"), (dict(window=1 << 30, keep_first=1), "no fewer"),
    (dict(pages=cache(page=8)), "dense uint8"), (dict(block_table=i32([[0], [1]])), "do not fit"), (dict(block_table=i32([[0, 1]])), "lengths|do not fit"),
    (dict(q=torch.zeros((1, 512), dtype=torch.bfloat16)), "a row per token"), (dict(q=torch.zeros((2, 504), dtype=torch.bfloat16)), "a row per token"),
    (dict(q_stride=504), "a row per token"), (dict(q_stride=1024), "a row per token"),
    (dict(q=torch.zeros((2, 1024), dtype=torch.bfloat16)[:, ::2], q_stride=1024), "a row per token"),
    (dict(pages=torch.zeros(cache().numel() + 1, dtype=torch.uint8)[1:].view(cache().shape)), "multiple of 16 bytes")])
def test_attention_that_is_refused(ops, change, match):
    args = attention_args(**change)
    with pytest.raises(KernelError, match=match):
        ops.paged_attention_8bit(args.pop("q"), args.pop("q_stride"), **args)
    assert not ops.calls


def far(T, columns, stride=1 << 31, dtype=torch.bfloat16):
    """Rows so far apart, without their memory."""
    return torch.empty_strided((T, columns), (stride, 1), dtype=dtype, device="meta")


def test_rows_and_sequences_beyond_32_bits_are_refused(ops):
    """What the kernels get of them are 32 bits: others would be somewhere else."""
    for change in (dict(qkv=far(3, 1024)), dict(q_out=far(3, 512, dtype=torch.float32))):
        args = store_args(**change)
        with pytest.raises(KernelError, match="elements apart"):
            ops.qk_norm_rope_store_8bit(args.pop("qkv"), **args)
    args = attention_args(q=far(2, 512), q_stride=1 << 31)
    with pytest.raises(KernelError, match="elements apart"):
        ops.paged_attention_8bit(args.pop("q"), args.pop("q_stride"), **args)
    assert not ops.calls
    for T in (1, 2):  # (a single row lies nowhere else)
        near = far(T, 1024, (1 << 31) - T)
        args = store_args(new=(1,) * T, lens=(20,) * T, qkv=near, block_table=i32([[0, 1], [2, 3]][:T]))
        ops.qk_norm_rope_store_8bit(args.pop("qkv"), **args)
    args = store_args(new=(1,), lens=(20,), qkv=far(1, 1024))
    ops.qk_norm_rope_store_8bit(args.pop("qkv"), **args)
    assert ops.calls == ["q3_store_8bit"] * 3
    wide = torch.empty((2, 1 << 27), dtype=torch.int32, device="meta")  # room for 2^31 tokens
    args = attention_args(block_table=wide)
    args["step"].max_kv_len = (1 << 30) + 1
    with pytest.raises(KernelError, match="do not fit"):
        ops.paged_attention_8bit(args.pop("q"), args.pop("q_stride"), **args)
    with pytest.raises(KernelError, match="does not fit"):
        ops.unpack_8bit(cache(), num_kv_heads=2, head_dim=128, page_size=16, block_table=wide, kv_lens=i32([1, 1]), max_kv_len=(1 << 30) + 1,
                        dtype=torch.float32)
    seen, taken = [], attention_args(block_table=wide)
    taken["step"].captured_width = 1 << 27
    call = ops._call
    ops._call = lambda group, name, *sizes: (seen.append(sizes), call(group, name, *sizes))
    ops.paged_attention_8bit(taken.pop("q"), taken.pop("q_stride"), **taken)
    assert 1 << 30 in seen[0] and 1 << 31 not in seen[0], "a captured step looks as far as it can"


class Here(Table):
    """A table whose own device is the CPU."""

    _check_here = CudaOps._check_here

    def __init__(self):
        super().__init__()
        self._device_index, self._slices_cache, self.prefill_attention = torch.zeros(1).get_device(), {}, "tcgen05"
        self._clusters_8bit = lambda *sizes: 0

    def paged_attention(self, *args, **kw):
        self.calls.append("paged_attention")


def call(new=(1, 1), kw={}, unpacked=None, **change):
    """The launches of an attention call; ``unpacked``: how portions are decided on (None: by their cost)."""
    ops, args = Here(), attention_args(new=new, **kw)
    if unpacked is not None:
        ops._prompts_unpacked = lambda *sizes: unpacked
    for name, value in change.items():
        setattr(args["step"], name, value)
    ops.paged_attention_8bit(args.pop("q"), args.pop("q_stride"), **args)
    return ops.calls


@pytest.mark.parametrize("change,match", [
    (dict(kv_longest=torch.tensor([20])), "kv_longest"), (dict(kv_longest=i32([])), "kv_longest"), (dict(kv_longest=elsewhere([20])), "launches on"),
    (dict(kv_lens=elsewhere([20, 3])), "launches on"), (dict(cu_seqlens=torch.tensor([0, 1, 2])), "cu_seqlens"), (dict(cu_seqlens=i32([0, 1])), "cu_seqlens"),
    (dict(cu_seqlens=elsewhere([0, 1, 2])), "launches on"),
    (dict(new=(1, 2), single_seqs=torch.tensor([0])), "single_seqs"), (dict(new=(1, 2), single_seqs=i32([])), "single_seqs"),
    (dict(new=(1, 2), decode_only=True), "single tokens"), (dict(new=(2, 1), kw=dict(D=80), decode_only=True), "single tokens"),
    (dict(new=(1, 2), single_seqs=None), "single_seqs"), (dict(new=(1, 2), single_seqs=elsewhere([0])), "launches on"),
    (dict(kw=dict(dtype=torch.float32), token_seq=i32([0])), "token_seq"), (dict(kw=dict(dtype=torch.float32), positions=torch.tensor([0, 1])), "positions")])
def test_what_attention_reads_of_a_step(change, match):
    with pytest.raises(KernelError, match=match):
        call(**change)


def test_tensors_on_another_device_are_refused():
    for name in ("qkv", "pages", "block_table"):
        ops, args = Here(), store_args()
        args[name] = args[name].as_subclass(Elsewhere)
        with pytest.raises(KernelError, match="launches on"):
            ops.qk_norm_rope_store_8bit(args.pop("qkv"), **args)


def test_which_kernels_attention_takes():
    f32, wide = dict(dtype=torch.float32), dict(H=34, G=2)
    decode, straight, general = "q3_decode_attention_8bit", "q3_prompts_attention_8bit", "q3_general_attention_8bit"
    unpacked = ["q3_unpack_8bit", "q3_prompts_tiles_8bit"]
    assert call() == call(kv_longest=None, single_seqs=None) == [decode]
    assert call(kw=f32) == call((2, 3), f32) == [general]
    assert call(kw=dict(D=80)) == call(kw=dict(D=80, H=16)) == [general] and call(kw=dict(D=80, H=18)) == [straight]
    assert call(kw=wide) == call((2, 3), wide) == call((2, 1), wide) == call((2, 1), dict(D=80)) == [straight]
    odd = dict(H=1, G=1, q=torch.zeros((3, 132), dtype=torch.bfloat16), q_stride=132)  # rows that do not begin at 16 bytes
    assert call((2, 1), odd) == [general]
    for kw in (dict(), dict(window=4, keep_first=1), dict(D=64), dict(page=20), dict(H=10)):
        assert call((2, 1), kw, True) == [decode, *unpacked] and call((2, 3), kw, True) == unpacked
        assert call((2, 1), kw, False) == [decode, straight] and call((2, 3), kw, False) == call((2, 3), kw) == [straight]
    assert call((2, 1), dict(D=256), True) == [decode, "q3_unpack_8bit", "q3_prompts_tiles_wide_8bit"] and call((2, 1), dict(D=48), True) == [straight]
    assert call((2, 1), dict(D=80), True) == call((2, 1), wide, True) == unpacked
    assert call((2, 3), dict(scale=0.0), True) == call((2, 3), dict(scale=-1.0), True) == [straight]
    assert call((1, 1), dict(D=80, H=18), True) == call((2, 1), dict(H=129, G=1), True) == [straight]


def test_which_portions_are_unpacked():
    """Long ones and those behind long contexts; prompts of a few tokens are not."""
    ops = Here()
    ops.SM_COUNT = 148
    cases = lambda news, kvs, D=128, window=0, first=0, group=4: ops._prompts_unpacked(  # noqa: E731
        [sum(news[:b]) for b in range(len(news) + 1)], kvs, group, 8, D, window, first)
    assert cases([2048], [2048]) and cases([512, 1, 700], [512, 9000, 900]) and cases([2048], [2048], 64) and cases([256], [4256]) and cases([64], [16064])
    assert not cases([16], [16]) and not cases([2, 1, 3], [1000, 5, 1003]) and not cases([1, 1], [9, 9])
    assert cases([2048], [9000], window=1024, first=4)


def test_slices_of_prompts():
    """No more items than SMs by slices, each of at least eight tiles (a block of 128 rows: four)."""
    ops = Here()
    ops.SM_COUNT = 148
    assert [ops._tile_splits(n, 16384, 64, 0, 0) for n in (1, 8, 74, 75, 148, 500)] == [16, 16, 2, 1, 1, 1]
    assert [ops._tile_splits(8, n, 64, 0, 0) for n in (1, 64, 1000, 1024, 3000)] == [1, 1, 2, 2, 5]
    assert ops._tile_splits(8, 16384, 64, 1000, 24) == 2 and ops._prompt_splits(8, 128, 1000, 24, 64, 16384) == 4
    assert [ops._prompt_splits(8, D, 0, 0, 64, 16384) for D in (64, 128)] == [32, 18]


def test_unpacking_more_than_the_table_holds_is_refused(ops):
    args = dict(num_kv_heads=2, head_dim=128, page_size=16, block_table=i32([[0, 1]]), kv_lens=i32([20]))
    for bad, dtype, match in ((33, torch.float32, "does not fit"), (-1, torch.float32, "does not fit"), (20, torch.float16, "float32 and bfloat16")):
        with pytest.raises(KernelError, match=match):
            ops.unpack_8bit(cache(), max_kv_len=bad, dtype=dtype, **args)
    ops.unpack_8bit(cache(), max_kv_len=20, dtype=torch.bfloat16, **args)
    assert ops.calls == ["q3_unpack_8bit"]


def test_pages_that_prompts_unpack_under_a_window():
    """The pages of every key that a new token sees, and no others; not exact: no fewer for any shorter length."""
    rnd = random.Random(2)
    for _ in range(400):
        page, window, first = rnd.randint(1, 20), rnd.choice([0, 1, rnd.randint(1, 60)]), rnd.choice([0, 1, rnd.randint(0, 50)])
        new = rnd.randint(1, 30)
        kv = new + rnd.randint(0, 150)
        keys = set()
        for last in range(kv - new, kv):
            keys |= {j // page for j in p8.seen(last, window, first if window else 0)}
        got = unpacked_pages_4bit([0, new], [kv], page, window, 1, True, first if window else 0)
        assert got == [len(keys)]
        assert unpacked_pages_4bit([0, new], [kv + rnd.randint(0, 100)], page, window, 1, False, first if window else 0)[0] >= got[0]


def test_slices_of_decode_attention(ops):
    """At least one, no more than the longest sequence has rounds; a launch that fills the device is not cut further than that helps its last
    blocks, one that leaves it idle is; clusters only where all their blocks run at once; asked again, the answer is kept."""
    for lens in ([1], [128], [129], [513], [4097] * 8, [32768], [1024] * 64, [512] * 128, [65 + 83 * i for i in range(48)]):
        for G, D, group in ((8, 128, 4), (8, 64, 2), (2, 256, 8), (1, 128, 16), (1, 256, 16)):
            s = ops.decode_slices_8bit(lens, G, D, None, group)
            slots = 148 * ops.DECODE_8BIT_BLOCKS_PER_SM[D]
            assert 1 <= abs(s) <= min(64, -(-max(lens) // 64)) and s != -1
            assert s < 0 or s == 1 or (s <= 16 and s * len(lens) * G <= slots)
            assert s == ops.decode_slices_8bit(lens, G, D, None, group)
    assert ops.decode_slices_8bit([1], 8, 128) == 1 and ops.decode_slices_8bit([], 8, 128) == 1
    assert abs(ops.decode_slices_8bit([32768], 8, 128)) >= 16 and abs(ops.decode_slices_8bit([4097], 8, 128)) >= 8
    assert ops.decode_slices_8bit([32768], 8, 128, 100) == 1
    assert abs(ops.decode_slices_8bit([32768], 8, 128, 100, 1, 4000)) > 4
