"""Random calls of the operators around a cache in 8 bits, and random engine scenarios; each test's cases come from its seed alone.  The bounds are
those of tests/test_8bit_gpu.py."""

import random

import pytest
import torch

import engine_8bit_cases as ec
import plain_8bit as p8
import test_8bit_gpu as t8
from helpers import TINY, random_ids
from test_8bit_gpu import BF16, F32, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def sizes_of(rnd):
    D = rnd.choice([64, 128, 256, 64, 128, 256, 16, 32, 48, 80, 96, 112, 144, 176, 208, 240])
    page = rnd.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 16, 16, 24, 32, 48, 64, 100])
    return D, page, rnd.choice([1, 2, 3, 4]), rnd.choice([BF16, BF16, F32])


@pytest.mark.parametrize("seed", range(80))
def test_calls(ops, seed):  # noqa: F811
    rnd = random.Random(seed)
    for mode in ("decode", "mixed"):
        D, page, G, dtype = sizes_of(rnd)
        R, scale = rnd.choice([1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 20]), D ** -0.5
        top = rnd.choice([20, 90, 300])
        lens = [rnd.randint(1, top) for _ in range(rnd.randint(1, 5))]
        new = [1] * len(lens) if mode == "decode" else [rnd.randint(1, min(n, 60)) for n in lens]
        single = all(n == 1 for n in new)

        def mutate(b, k, v):
            v *= torch.exp(torch.randn(v.shape[1], 1, generator=torch.Generator().manual_seed(b)) * loud)

        loud = rnd.choice([0.0, 1.0, 4.0])
        c = p8.Cache(lens, G, D, page, seed=seed, k_scale=rnd.choice([0.5, 1.0, 2.0]), mutate=mutate)
        q = t8.queries(sum(new), G * R, D, seed + 1, dtype)
        window = rnd.choice([None, None, 1, 7, 50, 64, 200])
        first = rnd.choice([0, 1, 5, 16, 64, 130]) if window else 0
        table = c.table.clone()
        if window:
            for b, (n, L) in enumerate(zip(new, lens)):
                table[b, -(-first // page): max(0, L - n - window + 1) // page] = -1
        slices = rnd.choice([None, None, 1, 2, -2, 5, -5, 16, 20]) if single else None
        got = t8.attend(ops, c, q, new, lens, G * R, scale, window=window, keep_first=first, slices=slices, dtype=dtype, table=table)
        fast = dtype == BF16 and D in (64, 128, 256) and R <= 16 and single
        t8.check_rows(got, q.view(-1, G * R, D), c, new, lens, scale, window=window, keep_first=first, wide=not fast, dtype=dtype)


@pytest.mark.parametrize("seed", range(40))
def test_writes(ops, seed):  # noqa: F811
    """Tokens of several sequences in random portions: the bytes of the plain form at every step."""
    rnd = random.Random(seed)
    D, page, G, dtype = sizes_of(rnd)
    H, B = rnd.randint(1, 5), rnd.randint(1, 4)
    g = torch.Generator().manual_seed(seed)
    width = -(-60 // page)
    pages = torch.randint(0, 256, (B * width, G, p8.page_bytes(D, page)), generator=g, dtype=torch.uint8)
    table = torch.randperm(B * width, generator=g).int().view(B, width)
    dev, want, lens = pages.cuda(), pages.clone(), [0] * B
    rows = [torch.zeros((2, G, 0, D), dtype=torch.float64) for _ in range(B)]
    loud = rnd.choice([0.0, 2.0, 10.0])
    for _ in range(5):
        new = [min(60 - L, rnd.choice([0, 1, 1, rnd.randint(1, 20)])) for L in lens] if rnd.random() < 0.7 else [min(60 - L, 1) for L in lens]
        if not sum(new):
            continue
        lens = [L + n for L, n in zip(lens, new)]
        T = sum(new)
        x = (torch.randn((T, (H + 2 * G) * D), generator=g) * torch.exp(loud * torch.randn((T, 1), generator=g))).to(dtype)
        at = 0
        for b, n in enumerate(new):
            kv = x[at:at + n, H * D:].float().view(n, 2, G, D).permute(1, 2, 0, 3)
            rows[b], at = torch.cat([rows[b], p8.four_bits(kv)], 2), at + n
            for i in range((lens[b] - n) // page, -(-lens[b] // page) if n else 0):
                for which in range(2):
                    for h in range(G):
                        p8.write_rows(want, int(table[b, i]), h, page, which, rows[b][which, h, i * page:(i + 1) * page])
        ops.qk_norm_rope_store_8bit(x.cuda(), num_heads=H, num_kv_heads=G, head_dim=D, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None,
                                    step=p8.step_of(new, lens, page), block_table=table.cuda(), pages=dev, page_size=page)
        assert torch.equal(dev.cpu(), want), (new, lens, D, page, dtype)


@pytest.mark.parametrize("seed", range(8))
def test_engines(tmp_path, ops, seed):  # noqa: F811
    """Pools down to the smallest that can hold a request, portions of a few tokens: every request ends with its tokens, every page comes back; in
    float32 captured steps give the tokens of uncaptured ones."""
    rnd = random.Random(seed)
    for name in "ABCDE":
        page, vocab = TINY[name]["page_size"], TINY[name]["config"].vocab_size
        prompts = [random_ids(vocab, rnd.randint(1, 70), rnd.randint(0, 9999)) for _ in range(rnd.randint(1, 5))]
        count = rnd.randint(1, 30)
        least = -(-(max(len(p) for p in prompts) + count) // page) + 1
        kw = dict(pages=rnd.choice([least, least + 3, 120]), tokens=rnd.choice([5, 16, 64]), seqs=rnd.randint(1, 6), run_ahead=rnd.random() < 0.5)
        dtype, outs = rnd.choice(["float32", "float32", "bfloat16"]), []
        for graph in (False, True):
            eng = ec.engine(tmp_path, name, dtype, ops, "cuda", graph=graph, **kw)
            requests = [eng.get_request(eng.add_request(p, max_tokens=count)) for p in prompts]
            while not eng.is_finished():
                eng.step()
                eng.cache.check_invariants()
            assert eng.cache.num_free_pages == eng.cache.num_pages
            ops.raise_if_kernel_error()
            outs.append([r.output_token_ids for r in requests])
            assert [len(o) for o in outs[-1]] == [count] * len(prompts)
        if dtype == "float32":
            assert outs[0] == outs[1], (name, kw)
