"""Sums of attention weights in the engine's captured steps: the launch that a graph holds is the one that the live requests' lengths ask for."""

import pytest

import engine_4bit_cases as ec
from helpers import TINY, random_ids
from qwen3_runtime_b200 import TokenBudget
from qwen3_runtime_b200.ops.cuda import CudaOps

pytestmark = pytest.mark.gpu


class Ops(CudaOps):
    """Notes the sums' launches; a few hundred keys call for longer slices, as if the device held two blocks."""

    def __init__(self):
        super().__init__()
        self.sums = []

    def mass_slice_keys_4bit(self, kv_lens, num_kv_heads):
        return max(128, 1 << max(0, (sum(kv_lens) * num_kv_heads // 2).bit_length() - 1))

    def _call(self, group, name, what, *args):
        if name == "q3_attention_mass_4bit":
            self.sums.append((args[14], args[-1]))  # sequences, blocks for each of their kv heads
        return super()._call(group, name, what, *args)


@pytest.mark.parametrize("name", ["D", "E"])
def test_slices_of_captured_sums(tmp_path, name):
    """A step captured for requests of 200 tokens asks for their slices, not for those of the padding rows that it is captured with."""
    ops = Ops()
    page, vocab = TINY[name]["page_size"], TINY[name]["config"].vocab_size
    prompts = [random_ids(vocab, 200, s) for s in range(4)]
    eng = ec.engine(tmp_path, name, "bfloat16", ops, "cuda", budget=TokenBudget(400), graph=True, pages=80, tokens=900)
    out = eng.generate_batch(prompts, max_tokens=5)
    ops.raise_if_kernel_error()
    assert [len(o) for o in out] == [5] * 4
    heads = eng.runner.storage.layout.groups[0].layer_spec.num_kv_heads
    (bucket, width, choices), = eng.runner.graphs.captured
    keys = {name: n for (name, *_sizes), n in choices}["mass_slice_keys_4bit"]
    assert bucket == 4 and keys == ops.mass_slice_keys_4bit([201] * 4, heads) > 128
    captured = [few for sequences, few in ops.sums if sequences == bucket and few == -(-width * page // keys)]
    layers = len(eng.runner.storage.layout.groups[0].cache_ids)
    assert len(captured) >= 2 * layers, "warm-up and capture"
    assert -(-width * page // 128) not in {few for _s, few in ops.sums}
