"""A cache in 4 bits, host side: sizes, the plain form's rounding, and what the kernel table refuses before it launches anything."""

import math

import pytest
import torch

import plain_4bit as p4
from qwen3_runtime_b200.cache.layout import four_bit_groups, four_bit_page_bytes, four_bit_token_bytes
from qwen3_runtime_b200.ops import cuda
from qwen3_runtime_b200.ops.cuda import KernelError


def test_sizes():
    for D in range(16, 257, 16):
        G = four_bit_groups(D)
        assert G == p4.groups(D) and D % G == 0 and (D // G) % 8 == 0 and D // G <= 64
        assert four_bit_token_bytes(D) == D + 8 * G
        for page in (1, 5, 16, 64):
            assert four_bit_page_bytes(D, page) == p4.page_bytes(D, page) and four_bit_page_bytes(D, page) % 16 == 0
    assert [four_bit_groups(D) for D in (64, 80, 128, 256)] == [1, 2, 2, 4]


def test_the_plain_rounding_covers_every_value():
    g = torch.Generator().manual_seed(0)
    x = torch.randn((500, 128), generator=g) * torch.exp(4 * torch.randn((500, 1), generator=g)) + torch.randn((500, 1), generator=g)
    n, s, z = p4.quantise(x)
    step = s.double().repeat_interleave(64, -1)
    assert bool(((p4.value(n, s, z) - x.double()).abs() <= step * (0.5 + 2.0 ** -19)).all())
    same = torch.full((1, 64), 0.75)
    assert bool((p4.value(*p4.quantise(same)) == 0.75).all())


def test_the_cache_of_tensors_has_the_layout_of_single_rows():
    c = p4.Cache([7, 3], 2, 80, 5, seed=1)
    for b, n in enumerate(c.lens):
        for j in range(n):
            for h in range(2):
                got = p4.read(c.pages[int(c.table[b, j // 5]), h], 80, 5, j % 5)
                for have, want in zip(got, (c.k[b], c.v[b])):
                    assert all(torch.equal(a, w[h, j]) for a, w in zip(have, want))


def test_plain_eviction():
    assert p4.evict([5.0, 1.0, 3.0, 2.0], [0, 1, 2, 3], 2, 0, 0) == [0, 2]
    assert p4.evict([5.0, 1.0, 3.0, 2.0], [0, 1, 2, 3], 2, 0, 1) == [0, 3]
    assert p4.evict([1.0, 1.0, 1.0, 1.0], [0, 1, 2, 3], 2, 0, 0) == [0, 1]
    assert p4.evict([0.0, math.nan, 9.0, math.inf], [0, 1, 2, 3], 2, 0, 0) == [3, 1]
    assert p4.evict([1.0, 2.0], [0, 1], 2, 0, 0) == [0, 1]


class Table(cuda.CudaOps):
    """The kernel table's checks without a device: a call is noted, not launched."""

    def __init__(self):
        self.timing, self.launches, self.calls, self._device_index = None, 0, [], 0
        self._err = torch.zeros(1, dtype=torch.int32)

    def _check_here(self, what, *tensors):
        pass

    def _call(self, group, name, what, *args):
        assert len(args) + 1 == len(cuda._SIGNATURES[group][name]), "every argument of the launcher, and the stream"
        self.calls.append(name)


@pytest.fixture
def ops():
    return Table()


def cache(D=128, page=16, G=2, count=4, layers=()):
    return torch.zeros((*layers, count, G, four_bit_page_bytes(D, page)), dtype=torch.uint8)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def store_args(T=3, H=4, G=2, D=128, page=16, **kw):
    pos = torch.arange(T, dtype=torch.int32)
    return {**dict(qkv=torch.zeros((T, (H + 2 * G) * D)), num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0,
                   cos=None, sin=None, positions=pos, token_seq=torch.zeros_like(pos), block_table=i32([[0, 1]]), pages=cache(D, page, G),
                   page_size=page), **kw}


@pytest.mark.parametrize("change,match", [
    (dict(head_dim=24), "multiples of 16"), (dict(head_dim=272), "multiples of 16"), (dict(page_size=0), "pages and heads"),
    (dict(pages=cache(page=8)), "dense uint8"), (dict(pages=cache().float()), "dense uint8"), (dict(pages=cache(layers=(2,))), "dense uint8"),
    (dict(pages=cache(G=4)[:, ::2]), "dense uint8"), (dict(block_table=i32([[0, 1]]).long()), "block table"),
    (dict(block_table=i32([0, 1])), "block table"), (dict(block_table=torch.zeros((1, 0), dtype=torch.int32)), "block table"),
    (dict(positions=i32([0])), "positions"), (dict(positions=torch.arange(3)), "positions"), (dict(slots=i32([0])), "slots"),
    (dict(token_seq=i32([0])), "token_seq"), (dict(q_weight=torch.zeros(64)), "norm weights"),
    (dict(k_weight=torch.zeros(128, dtype=torch.bfloat16)), "norm weights"), (dict(cos=torch.zeros((4, 64))), "together"),
    (dict(cos=torch.zeros((4, 65)), sin=torch.zeros((4, 65))), "rotation tables"), (dict(cos=torch.zeros((0, 64)), sin=torch.zeros((0, 64))), "rotation"),
    (dict(cos=torch.zeros((4, 64)).half(), sin=torch.zeros((4, 64)).half()), "rotation"), (dict(q_out=torch.zeros((3, 4 * 128)).bfloat16()), "queries"),
    (dict(q_out=torch.zeros((2, 4 * 128))), "queries"), (dict(qkv=torch.zeros((3, 7 * 128))), "projection"),
    (dict(qkv=torch.zeros((3, 8 * 128)).half()), "float32 and bfloat16"), (dict(qkv=torch.zeros((8 * 128, 3)).T), "unit-stride"),
    (dict(mass=torch.zeros((4, 2, 8))), "sums"), (dict(places=torch.zeros((4, 2, 16))), "sums")])
def test_a_write_that_is_refused(ops, change, match):
    args = store_args(**change)
    with pytest.raises(KernelError, match=match):
        ops.qk_norm_rope_store_4bit(args.pop("qkv"), **args)
    assert not ops.calls


def test_writes_that_are_taken(ops):
    for args in (store_args(), store_args(T=0), store_args(D=80, page=5), store_args(mass=torch.zeros((4, 2, 16)))):
        ops.qk_norm_rope_store_4bit(args.pop("qkv"), **args)
    assert ops.calls == ["q3_store_4bit"] * 4


def attention_args(new=(1, 1), lens=(20, 3), H=4, G=2, D=128, page=16, dtype=torch.bfloat16, **kw):
    step = p4.step_of(list(new), list(lens), page, device="cpu")
    T = sum(new)
    return {**dict(q=torch.zeros((T, H * D), dtype=dtype), q_stride=H * D, num_heads=H, num_kv_heads=G, head_dim=D, pages=cache(D, page, G),
                   block_table=i32([[0, 1], [2, 3]]), out=torch.zeros((T, H * D), dtype=dtype), page_size=page, scale=1.0, step=step), **kw}


@pytest.mark.parametrize("change,match", [
    (dict(lens=(33, 3)), "do not fit"), (dict(num_heads=3), "multiple of kv heads"), (dict(out=torch.zeros((2, 512))), "queries' type"),
    (dict(out=torch.zeros((2, 1024), dtype=torch.bfloat16)[:, :512]), "dense"), (dict(dtype=torch.float16), "float32 and bfloat16"),
    (dict(lse=torch.zeros((2, 3))), "log sums"), (dict(lse=torch.zeros((2, 4)).double()), "log sums"),
    (dict(new=(2, 1), lse=torch.zeros((3, 4))), "log sums come from"), (dict(D=80, lse=torch.zeros((2, 4))), "log sums come from"),
    (dict(dtype=torch.float32, lse=torch.zeros((2, 4))), "log sums come from"), (dict(pages=cache(page=8)), "dense uint8"),
    (dict(block_table=i32([[0], [1]])), "do not fit"), (dict(block_table=i32([[0, 1]])), "do not fit"),
    (dict(q=torch.zeros((1, 512), dtype=torch.bfloat16)), "a row per token"), (dict(q=torch.zeros((2, 504), dtype=torch.bfloat16)), "a row per token"),
    (dict(q_stride=504), "a row per token"), (dict(q_stride=1024), "a row per token"),
    (dict(q=torch.zeros((2, 1024), dtype=torch.bfloat16)[:, ::2], q_stride=1024), "a row per token"),
    (dict(pages=torch.zeros(cache().numel() + 1, dtype=torch.uint8)[1:].view(cache().shape)), "multiple of 16 bytes")])
def test_attention_that_is_refused(ops, change, match):
    args = attention_args(**change)
    with pytest.raises(KernelError, match=match):
        ops.paged_attention_4bit(args.pop("q"), args.pop("q_stride"), **args)
    assert not ops.calls


@pytest.mark.parametrize("change,match", [
    (dict(mass=torch.zeros((4, 2, 8))), "sums"), (dict(mass=torch.zeros((4, 2, 16)).double()), "sums"), (dict(observe=0), "observe"),
    (dict(lse=torch.zeros((2, 5))), "log sums"), (dict(num_heads=5), "multiple"), (dict(q_stride=516), "16 bytes"),
    (dict(q_stride=520), "a row per token"),
    (dict(q=torch.zeros((1, 512), dtype=torch.bfloat16)), "a row per token"), (dict(block_table=i32([[0, 1]])), "do not fit")])
def test_sums_that_are_refused(ops, change, match):
    args = {**attention_args(), "mass": torch.zeros((4, 2, 16)), **change}
    args.pop("out")
    with pytest.raises(KernelError, match=match):
        ops.attention_mass_4bit(args.pop("q"), args.pop("q_stride"), **args)
    assert not ops.calls


@pytest.mark.parametrize("change,match", [
    (dict(keep=0), "keep at least"), (dict(first=-1), "keep at least"), (dict(recent=-1), "keep at least"), (dict(first=5, recent=6), "keep at least"),
    (dict(max_kv_len=33), "does not fit"), (dict(mass=torch.zeros((4, 2, 15))), "sums"), (dict(places=torch.zeros((4, 2, 16))), "sums"),
    (dict(pages=cache(layers=(3,))), "sums"), (dict(kv_lens=i32([20])), "lengths"), (dict(kv_lens=torch.tensor([20, 3])), "lengths")])
def test_eviction_that_is_refused(ops, change, match):
    args = {**dict(pages=cache(), mass=torch.zeros((4, 2, 16)), places=torch.zeros((4, 2, 16), dtype=torch.int32), block_table=i32([[0, 1], [2, 3]]),
                   kv_lens=i32([20, 3]), max_kv_len=20, keep=10, first=2, recent=3, num_kv_heads=2, head_dim=128, page_size=16), **change}
    with pytest.raises(KernelError, match=match):
        ops.evict_4bit(**args)
    assert not ops.calls


def test_a_cache_within_its_budget_is_left_alone(ops):
    ops.evict_4bit(pages=cache(), mass=torch.zeros((4, 2, 16)), places=torch.zeros((4, 2, 16), dtype=torch.int32), block_table=i32([[0, 1]]),
                   kv_lens=i32([20]), max_kv_len=20, keep=20, first=2, recent=3, num_kv_heads=2, head_dim=128, page_size=16)
    assert not ops.calls


def test_unpacking_more_than_the_table_holds_is_refused(ops):
    with pytest.raises(KernelError, match="does not fit"):
        ops.unpack_4bit(cache(), num_kv_heads=2, head_dim=128, page_size=16, block_table=i32([[0, 1]]), kv_lens=i32([20]), max_kv_len=33,
                        dtype=torch.float32)
    with pytest.raises(KernelError, match="float32 and bfloat16"):
        ops.unpack_4bit(cache(), num_kv_heads=2, head_dim=128, page_size=16, block_table=i32([[0, 1]]), kv_lens=i32([20]), max_kv_len=20,
                        dtype=torch.float16)


def test_tensors_on_another_device_are_refused():
    table = Table()
    with pytest.raises(KernelError, match="launches on cuda:0"):
        cuda.CudaOps._check_here(table, "x", torch.zeros(1))


def test_slices_of_decode_attention():
    """At least one, no more than the longest sequence has rounds of 128 keys; a launch that fills the device is not cut further, one that
    leaves it idle is; clusters only where all their blocks run at once; asked again, the answer is kept."""
    table = Table()
    table._slices_cache = {}
    for lens in ([1], [128], [129], [513], [4097] * 8, [32768], [1024] * 64, [512] * 128, [65 + 83 * i for i in range(48)]):
        for G, D, group in ((8, 128, 4), (8, 64, 2), (2, 256, 8), (1, 128, 16), (1, 256, 16)):
            s = table.decode_slices_4bit(lens, G, D, None, group)
            slots = 148 * table.DECODE_4BIT_BLOCKS_PER_SM[D][int(group > 8)]
            assert 1 <= abs(s) <= min(64, -(-max(lens) // 128)) and s != -1
            assert s < 0 or s == 1 or (s <= table._most_clustered(D, group > 8) and s * len(lens) * G <= slots)
            assert s == table.decode_slices_4bit(lens, G, D, None, group)
    assert table.decode_slices_4bit([1024] * 64, 8, 128) == 1 and table.decode_slices_4bit([1], 8, 128) == 1
    assert table.decode_slices_4bit([32768], 8, 128) < -16 and 8 <= table.decode_slices_4bit([4097], 8, 128) <= 16
    assert table.decode_slices_4bit([32768], 8, 128, 100) == 1 and table.decode_slices_4bit([], 8, 128) == 1
