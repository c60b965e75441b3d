"""What attention over prompts unpacks from a cache in 4 bits, host side: which pages, in which turns, and what the pool leaves for them."""

import random

import pytest
import torch

import plain_4bit as p4
from qwen3_runtime_b200.cache.layout import CacheLayout, KVLayerSpec
from qwen3_runtime_b200.engine.factory import beside_unpacked
from qwen3_runtime_b200.ops.cuda import runs_within, unpacked_pages_4bit
from test_4bit_cpu import Table, cache


def test_the_pages_that_new_tokens_see():
    rnd = random.Random(1)
    for _ in range(300):
        page, window, least = rnd.choice([1, 3, 16]), rnd.choice([None, 1, 7, 16, 40]), rnd.choice([1, 2])
        new = [rnd.randint(0, 9) for _ in range(5)]
        lens = [max(1, n + rnd.choice([0, rnd.randint(0, 90)])) for n in new]
        cu = [sum(new[:b]) for b in range(6)]
        for b, got in enumerate(unpacked_pages_4bit(cu, lens, page, window, least)):
            seen = {j // page for t in range(lens[b] - new[b], lens[b]) for j in range(max(0, t - window + 1) if window else 0, t + 1)}
            assert got == (len(seen) if new[b] >= least else 0)
        bound = unpacked_pages_4bit(cu, [100] * 5, page, window, least, exact=False)
        assert all(a <= b for a, b in zip(unpacked_pages_4bit(cu, lens, page, window, least), bound))


def test_runs():
    assert runs_within([], 5) == [] and runs_within([0, 0], 5) == []
    assert runs_within([0, 2, 0, 3, 0, 1, 0], 5) == [(0, 5), (5, 7)]
    assert runs_within([2, 9, 0, 2, 2], 5) == [(0, 1), (1, 3), (3, 5)]
    assert runs_within([1, 1, 1], 0) == [(0, 1), (1, 2), (2, 3)]
    rnd = random.Random(2)
    for _ in range(300):
        counts, limit = [rnd.choice([0, 0, rnd.randint(1, 12)]) for _ in range(rnd.randint(0, 12))], rnd.randint(1, 20)
        runs = runs_within(counts, limit)
        assert [c for a, b in runs for c in counts[a:b] if c] == [c for c in counts if c]
        assert all(sum(counts[a:b]) <= limit or sum(c > 0 for c in counts[a:b]) == 1 for a, b in runs)


class Noting(Table):
    def __init__(self):
        super().__init__()
        self.steps, self._slices_cache = [], {}

    def paged_attention(self, q, q_stride, *, k_pages, block_table, step, token_seq, positions, out, **kw):
        self.steps.append((k_pages.shape[0], tuple(block_table.shape), step, q.shape[0], out.shape[0]))


@pytest.mark.parametrize("D", [128, 80])
def test_the_turns_are_steps_of_their_own(D):
    """Each turn is the step of its sequences, counted from zero; what it allocates is what its own sequences hold."""
    ops, page, G, H = Noting(), 16, 2, 4
    new, lens = [1, 5, 3, 1, 4], [500, 40, 33, 90, 17]
    step = p4.step_of(new, lens, page, device="cpu")
    table = torch.arange(5 * 32, dtype=torch.int32).view(5, 32)
    q = torch.zeros((14, H * D), dtype=torch.bfloat16)
    args = dict(num_heads=H, num_kv_heads=G, head_dim=D, pages=cache(D, page, G), block_table=table, out=torch.zeros_like(q), page_size=page,
                scale=1.0, step=step)
    per = [-(-n // page) for n in lens]
    split = D == 128
    counts = [c if n > 1 or not split else 0 for n, c in zip(new, per)]
    ops.paged_attention_4bit(q, H * D, **args)
    assert [(s[0], s[1][0], s[3]) for s in ops.steps] == [(sum(counts), 5, 14)]
    assert ops.calls.count("q3_decode_attention_4bit") == int(split) and ops.calls.count("q3_unpack_4bit") == 1
    ops.steps = []
    ops.UNPACK_BYTES = 6 * 4 * G * page * D
    ops.paged_attention_4bit(q, H * D, **args)
    runs = [(0, 4), (4, 5)] if split else [(0, 1), (1, 3), (3, 4), (4, 5)]  # pages 0 3 3 0 2, or 32 3 3 6 2
    assert len(ops.steps) == len(runs)
    for (pages, shape, part, rows, outs), (a, b) in zip(ops.steps, runs):
        assert pages == sum(counts[a:b]) and shape == (b - a, -(-max(n for n, c in zip(lens[a:b], counts[a:b]) if c) // page)) and rows == outs == sum(new[a:b])
        want = p4.step_of(new[a:b], lens[a:b], page, device="cpu")
        want.max_kv_len = max(n for n, c in zip(lens[a:b], counts[a:b]) if c)
        for name in ("cu_seqlens", "kv_lens", "token_seq", "positions"):
            assert torch.equal(getattr(part, name), getattr(want, name)), name
        assert (part.num_tokens, part.num_seqs, part.host_cu_seqlens, part.host_kv_lens, part.max_query_len, part.max_kv_len) == (
            want.num_tokens, want.num_seqs, want.host_cu_seqlens, want.host_kv_lens, want.max_query_len, want.max_kv_len)
        assert part.num_single == (0 if split else want.num_single)
        if part.num_single:
            assert torch.equal(part.single_seqs, want.single_seqs)
    assert step.num_seqs == 5 and step.num_single == 2, "the caller's step stays as it is"


@pytest.mark.parametrize("layers", [1, 2, 36])
@pytest.mark.parametrize("longest", [1000, 131072, 1 << 30])
@pytest.mark.parametrize("total", [1 << 20, 1 << 28, 100 << 30])
def test_the_pool_leaves_what_prompts_unpack(layers, longest, total):
    at_once, page = 1 << 30, 16
    layout = CacheLayout({i: KVLayerSpec(8, 128, bits=4) for i in range(layers)})
    got = beside_unpacked(total, layout, page, longest, at_once, 8, 256)
    held = got // sum(layout.page_bytes(page, 2)) * page
    need = max(min(at_once, held * 4096), min(longest, held) * 4096)
    assert 0 < got and got + need <= total
    assert got + need >= 0.9 * total, "and no more than that"
    assert layout.unpacked_bytes(10) == 10 * 4 * 8 * 128 and CacheLayout({0: KVLayerSpec(8, 128)}).unpacked_bytes(10) == 0
