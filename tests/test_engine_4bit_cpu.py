"""The engine with a cache in 4 bits on the CPU, its kernels replaced by their plain statements; and what it refuses."""

import pytest
import torch

import engine_4bit_cases as ec
import plain_4bit as p4
from emulated_4bit import TorchOps4
from helpers import make_model_dir
from qwen3_runtime_b200 import LLM, EngineConfig, TokenBudget
from qwen3_runtime_b200.cache.layout import KVLayerSpec, kept_for_readers
from qwen3_runtime_b200.cache.manager import CacheError, CacheManager, GroupSpec
from qwen3_runtime_b200.engine.factory import build_engine, build_model, load_model

OPS, DEV = TorchOps4(), "cpu"


def test_values_by_tensors_are_those_of_single_rows():
    for D, page in ((64, 16), (80, 5), (128, 8)):
        c = p4.Cache([7], 2, D, page, seed=1)
        k, v = p4.values_of(c.pages, D, page)
        for h in range(2):
            for j in range(7):
                for x, (n, s, z) in zip((k, v), p4.read(c.pages[int(c.table[0, j // page]), h], D, page, j % page)):
                    assert torch.equal(x[int(c.table[0, j // page]), h, j % page], p4.value(n[None], s[None], z[None])[0].float())


@pytest.mark.parametrize("name", ["A", "C"])
def test_schedules_agree(tmp_path, name):
    ec.case_schedules_agree(tmp_path, name, OPS, DEV, share=0.03)


def test_generation(tmp_path):
    ec.case_generation(tmp_path, "A", "float32", OPS, DEV)


@pytest.mark.parametrize("name", ["A", "B"])
def test_budget(tmp_path, name):
    a = ec.case_budget(tmp_path, name, "float32", OPS, DEV)
    assert a == ec.case_budget(tmp_path, name, "float32", OPS, DEV)


def test_a_roomy_budget_changes_nothing(tmp_path):
    ec.case_roomy_budget_changes_nothing(tmp_path, "A", OPS, DEV)


def test_the_budget_of_a_request():
    assert TokenBudget(100) == TokenBudget(100, first=4, recent=50, slack=12)
    assert TokenBudget(1) == TokenBudget(1, first=1, recent=0, slack=0)
    for bad in (dict(keep=0), dict(keep=4, first=3, recent=2), dict(keep=4, first=-1), dict(keep=4, recent=-1), dict(keep=4, slack=-1),
                dict(keep=4, observe=0)):
        with pytest.raises(ValueError, match="budget"):
            TokenBudget(**bad)


def test_the_manager_under_a_budget():
    m = CacheManager([GroupSpec("full"), GroupSpec("state")], 4, 8, 2, budget=TokenBudget(10, first=1, recent=2, slack=2))
    assert m.fits_at_all(1000) and not CacheManager([GroupSpec("full")], 4, 2, 1, budget=TokenBudget(10, slack=0)).fits_at_all(1000)
    rc = m.open("a")
    m.reserve(rc, 12)
    m.commit(rc, 12)
    assert rc.held == 12 and not m.over_budget(rc) and len(rc.tables[0]) == 3
    m.reserve(rc, 1)
    m.commit(rc, 1)
    assert m.over_budget(rc) and len(rc.tables[0]) == 4
    m.cut(rc)
    assert (rc.held, rc.num_computed, rc.num_evicted, len(rc.tables[0])) == (10, 13, 3, 3)
    with pytest.raises(CacheError, match="nothing to cut"):
        m.cut(rc)
    assert m.max_reservable(rc, 100) == 32 - 10 and m.new_pages_needed(rc, 3) == [1]
    m.reserve(rc, 3)  # reserved before it is cut again: its pages stay
    assert len(rc.tables[0]) == 4
    m.check_invariants()
    m.reset(rc)
    assert (rc.held, rc.num_evicted, m.num_free_pages) == (0, 0, [8])
    m.close(rc)
    with pytest.raises(ValueError, match="budget"):
        CacheManager([GroupSpec("window", 8)], 4, 8, 2, budget=TokenBudget(10))


def test_readers_of_a_layer_in_4_bits():
    own = KVLayerSpec(2, 64, bits=4)
    assert kept_for_readers(0, own, [own]) is own
    with pytest.raises(ValueError, match="differs"):
        kept_for_readers(0, own, [KVLayerSpec(2, 64)])
    assert kept_for_readers(0, KVLayerSpec(2, 64, 8, bits=4), [KVLayerSpec(2, 64, 16, bits=4)]) == KVLayerSpec(2, 64, 16, bits=4)


def test_what_is_refused(tmp_path):
    folder = make_model_dir(tmp_path, "A")
    args = dict(dtype="float32", device=DEV, ops=OPS)
    for bits in (8, 3, True, "4"):
        with pytest.raises(ValueError, match="kv_bits"):
            build_engine(folder, kv_bits=bits, **args)
    with pytest.raises(ValueError, match="needs kv_bits=4"):
        build_engine(folder, token_budget=100, **args)
    with pytest.raises(ValueError, match="needs kv_bits=4"):
        EngineConfig(token_budget=100)
    assert EngineConfig(kv_bits=4, token_budget=100).token_budget == TokenBudget(100)
    model, _cfg, _raw = load_model(folder, **args)
    with pytest.raises(ValueError, match="another cache"):
        build_engine(model=model, kv_bits=4, **args)
    model, _cfg, _raw = load_model(folder, kv_bits=4, **args)
    assert build_engine(model=model, num_kv_blocks=8, **args).config.kv_bits == 4
    for architecture in ("Logesun", "Puladra", "Medilix", "Tabisun", "Pevazen", "Timopel"):
        with pytest.raises(ValueError, match="4 bits"):
            LLM(None, architecture=architecture, kv_bits=4, dtype="float32", device=DEV, ops=OPS)


def test_a_window_cannot_have_a_budget():
    from qwen3_runtime_b200.config import PartSpec
    from qwen3_runtime_b200.parts.base import BuildContext, build_part

    spec = PartSpec("paged_attention", dict(hidden_size=32, num_heads=2, num_kv_heads=1, head_dim=16, window=8))
    ctx = dict(dtype=torch.float32, device=torch.device("cpu"), ops=OPS, kv_bits=4)
    assert build_part("mixer", spec, BuildContext(**ctx)).cache_spec() == KVLayerSpec(1, 16, 8, bits=4)
    with pytest.raises(ValueError, match="window"):
        build_part("mixer", spec, BuildContext(**ctx, kv_budget=TokenBudget(10)))


def test_the_python_entry(tmp_path):
    llm = LLM(make_model_dir(tmp_path, "A"), dtype="float32", device=DEV, ops=OPS, kv_bits=4, token_budget=TokenBudget(8, slack=1), block_size=4,
              num_kv_blocks=12, cuda_graph=False)
    assert len(llm.generate([1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], max_tokens=9)) == 9
    small = LLM(None, dtype="float32", device=DEV, ops=OPS, kv_bits=4, cuda_graph=False)
    assert small.engine.runtime.model.ctx.kv_bits == 4 and len(small.generate([1, 2, 3], max_tokens=2)) == 2


def test_bytes_of_a_page():
    from qwen3_runtime_b200.cache.layout import CacheLayout

    assert CacheLayout({0: KVLayerSpec(8, 128, bits=4), 1: KVLayerSpec(8, 128, bits=4)}).page_bytes(16, 2) == [2 * 8 * 2304]
    assert CacheLayout({0: KVLayerSpec(8, 128, bits=4, sums=True)}).page_bytes(16, 2) == [8 * (2304 + 128)]


def test_build_model_takes_the_number_of_tokens():
    from helpers import TINY
    from qwen3_runtime_b200.weights import DictSource
    from qwen3_runtime_b200.weights.random_init import random_state

    cfg = TINY["A"]["config"]
    model = build_model(cfg, DictSource(random_state(cfg, 0)), dtype="float32", device=DEV, ops=OPS, kv_bits=4, token_budget=64)
    assert model.ctx.kv_budget == TokenBudget(64)


def test_a_budget_is_a_number_of_tokens():
    for budget in (True, 1.5, "100"):
        with pytest.raises(ValueError, match="number of tokens"):
            EngineConfig(kv_bits=4, token_budget=budget)
    with pytest.raises(ValueError, match="at least one"):
        EngineConfig(kv_bits=4, token_budget=0)
