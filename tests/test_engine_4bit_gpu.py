"""The engine with a cache in 4 bits on the GPU: the cases of the CPU tests with the real kernels, captured steps, bfloat16, and the same
traces as the plain statements' engine."""

import pytest
import torch

import engine_4bit_cases as ec
from emulated_4bit import TorchOps4
from helpers import TINY, make_model_dir, random_ids, trace_portions
from qwen3_runtime_b200 import LLM, TokenBudget

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from qwen3_runtime_b200.ops.cuda import CudaOps

    return CudaOps()


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_schedules_agree_bit_for_bit_and_with_the_plain_statements(tmp_path, ops, name):
    got = ec.case_schedules_agree(tmp_path, name, ops, "cuda")
    want = ec.case_schedules_agree(tmp_path, name, TorchOps4(), "cpu", share=0.03) if name in "AC" else None
    if want is not None:
        for key, row in want.items():
            assert float((got[key] - row).abs().max()) <= 0.03 * float(row.abs().max())


@pytest.mark.parametrize("name", ["A", "C", "D", "E"])
def test_generation_in_float32(tmp_path, ops, name):
    ec.case_generation(tmp_path, name, "float32", ops, "cuda", graphs=(False, True))
    ops.raise_if_kernel_error()


@pytest.mark.parametrize("name", ["B", "D", "E"])
def test_generation_in_bfloat16(tmp_path, ops, name):
    ec.case_generation(tmp_path, name, "bfloat16", ops, "cuda", graphs=(False, True))
    ops.raise_if_kernel_error()


@pytest.mark.parametrize("name", ["D", "E"])
def test_bfloat16_logits_lie_near_those_of_the_plain_statements(tmp_path, ops, name):
    """The same bound as between a 16-bit and a 32-bit engine elsewhere: 16-bit activations move logits by about 1 %, a key that falls on the
    other side of a border by less than that."""
    reqs = ec.requests_of(name, (70, 33))
    want = ec.run_trace(ec.engine(tmp_path, name, "float32", ops, "cuda"), trace_portions(reqs))
    got = ec.run_trace(ec.engine(tmp_path, name, "bfloat16", ops, "cuda", graph=True), trace_portions(reqs))
    span = max(float(r.max() - r.min()) for r in want.values())
    assert max(float((got[k] - r).abs().max()) for k, r in want.items()) <= 0.1 * span


@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
@pytest.mark.parametrize("graph", [False, True])
def test_budget(tmp_path, ops, name, graph):
    a = ec.case_budget(tmp_path, name, "float32", ops, "cuda", graph=graph)
    assert a == ec.case_budget(tmp_path, name, "float32", ops, "cuda", graph=not graph)
    ec.case_budget(tmp_path, name, "bfloat16", ops, "cuda", graph=graph)
    ops.raise_if_kernel_error()


def test_a_roomy_budget_changes_nothing(tmp_path, ops):
    ec.case_roomy_budget_changes_nothing(tmp_path, "D", ops, "cuda")


def test_long_generation_under_a_small_budget_holds_few_pages(tmp_path):
    """More tokens than the pool could hold: the budget keeps the request within it."""
    name = "E"
    llm = LLM(make_model_dir(tmp_path, name), dtype="bfloat16", block_size=16, num_kv_blocks=8, max_num_batched_tokens=32, kv_bits=4,
              token_budget=TokenBudget(64, slack=32))
    out = llm.generate([random_ids(TINY[name]["config"].vocab_size, 90, 1)], max_tokens=400)
    assert len(out[0]) == 400 and llm.engine.cache.num_free_pages == [8]
    torch.cuda.synchronize()
    llm.engine.sampler.ops.raise_if_kernel_error()
