"""Random calls of the operators around a cache in 4 bits, and random engine scenarios; each test's cases come from its seed alone.  The bounds are
those of tests/test_4bit_gpu.py."""

import random

import pytest

import engine_4bit_cases as ec
import plain_4bit as p4
import test_4bit_gpu as t4
from helpers import TINY, random_ids
from qwen3_runtime_b200 import TokenBudget
from test_4bit_gpu import BF16, F32, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(60))
def test_calls(ops, seed):  # noqa: F811
    rnd = random.Random(seed)
    for mode in ("decode", "mixed", "sums", "eviction"):
        D = rnd.choice([64, 128, 256, 64, 128, 256, 16, 32, 48, 80, 96, 112, 144, 176, 208, 240])
        G, R = rnd.choice([1, 2, 3, 4]), rnd.choice([1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 20])
        page, dtype, scale = rnd.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 16, 16, 24, 32, 48, 64, 100]), rnd.choice([BF16, BF16, F32]), D ** -0.5
        top = rnd.choice([20, 90, 300])
        lens = [rnd.randint(1, top) for _ in range(rnd.randint(1, 5))]
        if mode == "eviction":
            keep = rnd.randint(1, max(lens) + 3)
            first = rnd.randint(0, min(keep, 10))
            t4.check_eviction(ops, lens, G, D, page, keep, first, rnd.randint(0, keep - first), layers=rnd.choice([0, 2]), seed=seed)
            continue
        new = [1] * len(lens) if mode == "decode" else [rnd.randint(1, min(n, 30)) for n in lens]
        single = all(n == 1 for n in new)
        c = p4.Cache(lens, G, D, page, seed=seed, k_scale=rnd.choice([0.5, 1.0, 2.0]))
        q = t4.queries(sum(new), G * R, D, seed + 1, dtype)
        rows = q.view(-1, G * R, D)
        if mode == "sums":
            observe = rnd.choice([1, 2, 5, 32, None])
            t4.check_mass(t4.mass_of(ops, c, q, new, lens, G * R, scale, observe), rows, c, new, lens, scale, observe, dtype=dtype)
        else:
            window = rnd.choice([None, None, 1, 7, 50, 200])
            slices = rnd.choice([None, None, 1, 2, -2, 5, -5, 16, 20]) if single else None
            got = t4.attend(ops, c, q, new, lens, G * R, scale, window=window, slices=slices, dtype=dtype)
            fast = dtype == BF16 and D in (64, 128, 256) and R <= 16 and single
            t4.check_rows(got, rows, c, new, lens, scale, window=window, wide=not fast, dtype=dtype)


@pytest.mark.parametrize("seed", range(12))
def test_engines(tmp_path, ops, seed):  # noqa: F811
    """Pools down to the smallest that can hold a request, portions of a few tokens, budgets: every request ends with its tokens and within its
    budget, every page comes back; in float32 captured steps give the tokens of uncaptured ones."""
    rnd = random.Random(seed)
    for name in "ABCDE":
        page, vocab = TINY[name]["page_size"], TINY[name]["config"].vocab_size
        keep = rnd.randint(1, 60)
        first = rnd.randint(0, min(4, keep))
        budget = None if rnd.random() < 0.25 else TokenBudget(keep, first=first, recent=rnd.randint(0, keep - first), slack=rnd.randint(0, 20),
                                                              observe=rnd.choice([1, 4, 32]))
        prompts = [random_ids(vocab, rnd.randint(1, 70), rnd.randint(0, 9999)) for _ in range(rnd.randint(1, 5))]
        count = rnd.randint(1, 30)
        need = max(len(p) for p in prompts) + count
        least = -(-(need if budget is None else min(need, budget.keep + budget.slack + 1)) // page) + 1
        kw = dict(budget=budget, pages=rnd.choice([least, least + 3, 120]), tokens=rnd.choice([5, 16, 64]), seqs=rnd.randint(1, 6),
                  run_ahead=rnd.random() < 0.5)
        dtype, outs = rnd.choice(["float32", "float32", "bfloat16"]), []
        for graph in (False, True):
            eng = ec.engine(tmp_path, name, dtype, ops, "cuda", graph=graph, **kw)
            requests = [eng.get_request(eng.add_request(p, max_tokens=count)) for p in prompts]
            while not eng.is_finished():
                eng.step()
                eng.cache.check_invariants()
                assert budget is None or all(r.cache is None or r.cache.held <= keep + budget.slack for r in requests)
            assert eng.cache.num_free_pages == eng.cache.num_pages
            ops.raise_if_kernel_error()
            outs.append([r.output_token_ids for r in requests])
            assert [len(o) for o in outs[-1]] == [count] * len(prompts)
        if dtype == "float32":
            assert outs[0] == outs[1], (name, kw)
