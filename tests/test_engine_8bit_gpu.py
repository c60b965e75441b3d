"""The engine with a cache in 8 bits on the GPU: the cases of the CPU tests with the real kernels, captured steps, bfloat16, and the same
traces as the plain statements' engine."""

import pytest
import torch

import engine_8bit_cases as ec
from emulated_8bit import TorchOps8
from helpers import TINY, make_model_dir, random_ids, trace_portions
from qwen3_runtime_b200 import LLM

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from qwen3_runtime_b200.ops.cuda import CudaOps

    return CudaOps()


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_schedules_agree_also_with_the_plain_statements(tmp_path, ops, name):
    got = ec.case_schedules_agree(tmp_path, name, ops, "cuda")
    if name in "AC":
        for key, row in ec.case_schedules_agree(tmp_path, name, TorchOps8(), "cpu").items():
            assert float((got[key] - row).abs().max()) <= 0.03 * float(row.abs().max())


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_portions_of_pages_are_the_whole_prompts_bit_for_bit(tmp_path, ops, name):
    ec.case_portions_of_pages(tmp_path, name, ops, "cuda")


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


@pytest.mark.parametrize("name", ["D", "E"])
def test_captured_steps_are_the_uncaptured_ones(tmp_path, ops, name):
    """bfloat16; four requests of unequal lengths, as many as a captured step has rows: the same kernels see the same numbers, so tokens and what the
    cache holds are the same bits."""
    vocab = TINY[name]["config"].vocab_size
    prompts = [random_ids(vocab, n, n) for n in (31, 5, 17, 50)]
    runs = []
    for graph in (False, True):
        eng = ec.engine(tmp_path, name, "bfloat16", ops, "cuda", graph=graph, tokens=128, seqs=4)
        requests = [eng.get_request(eng.add_request(p, max_tokens=24)) for p in prompts]
        while not eng.is_finished():
            eng.step()
        ops.raise_if_kernel_error()
        assert (eng.runner.graphs.replays if graph else 0) > 20 * graph - 1
        pages = list(range(eng.cache.num_pages[0]))  # (the scratch page is the padding rows')
        runs.append(([r.output_token_ids for r in requests], eng.runner.storage.tensors[0][:, pages].clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])


@pytest.mark.parametrize("name", ["D", "E"])
def test_captured_logits_are_the_uncaptured_ones(tmp_path, ops, name):
    """One request, portions and then single tokens with given ids."""
    reqs = ec.requests_of(name, (70,))
    a, b = (ec.run_trace(ec.engine(tmp_path, name, "bfloat16", ops, "cuda", graph=graph), trace_portions(reqs)) for graph in (False, True))
    assert a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)


def test_the_python_entry(tmp_path):
    name = "E"
    llm = LLM(make_model_dir(tmp_path, name), dtype="bfloat16", block_size=16, num_kv_blocks=40, max_num_batched_tokens=32, kv_bits=8)
    out = llm.generate([random_ids(TINY[name]["config"].vocab_size, 90, 1)], max_tokens=200)
    assert len(out[0]) == 200 and llm.engine.cache.num_free_pages == [40]
    torch.cuda.synchronize()
    llm.engine.sampler.ops.raise_if_kernel_error()
