"""The engine with a cache in 8 bits on the CPU, its kernels replaced by their plain statements; and what it refuses."""

import pytest
import torch

import engine_8bit_cases as ec
from emulated_4bit import TorchOps4
from emulated_8bit import TorchOps8
from helpers import make_model_dir
from qwen3_runtime_b200 import LLM, EngineConfig
from qwen3_runtime_b200.cache.layout import CacheLayout, KVLayerSpec, kept_for_readers
from qwen3_runtime_b200.engine.factory import beside_unpacked, build_engine, load_model

OPS, DEV = TorchOps8(), "cpu"


@pytest.mark.parametrize("name", ["A", "C"])
def test_schedules_agree(tmp_path, name):
    ec.case_schedules_agree(tmp_path, name, OPS, DEV)


def test_generation(tmp_path):
    ec.case_generation(tmp_path, "A", "float32", OPS, DEV)


def test_what_is_refused(tmp_path):
    folder = make_model_dir(tmp_path, "A")
    args = dict(dtype="float32", device=DEV, ops=OPS)
    for bits in (16, 3, True, "8"):
        with pytest.raises(ValueError, match="kv_bits must be 4 or 8"):
            build_engine(folder, kv_bits=bits, **args)
    with pytest.raises(ValueError, match="needs kv_bits=4"):
        build_engine(folder, kv_bits=8, token_budget=100, **args)
    with pytest.raises(ValueError, match="needs kv_bits=4"):
        EngineConfig(kv_bits=8, token_budget=100)
    assert EngineConfig(kv_bits=8).kv_bits == 8
    with pytest.raises(ValueError, match="no attention over a cache in 8 bits"):
        build_engine(folder, kv_bits=8, dtype="float32", device=DEV, ops=TorchOps4())
    model, _cfg, _raw = load_model(folder, **args)
    with pytest.raises(ValueError, match="another cache"):
        build_engine(model=model, kv_bits=8, **args)
    model, _cfg, _raw = load_model(folder, kv_bits=8, **args)
    assert build_engine(model=model, num_kv_blocks=8, **args).config.kv_bits == 8
    with pytest.raises(ValueError, match="another cache"):
        build_engine(model=model, kv_bits=4, **args)
    for architecture in ("Logesun", "Puladra", "Medilix", "Tabisun", "Pevazen", "Timopel"):
        with pytest.raises(ValueError, match="8 bits"):
            LLM(None, architecture=architecture, kv_bits=8, dtype="float32", device=DEV, ops=OPS)


def test_a_layer_with_a_window():
    from qwen3_runtime_b200.config import PartSpec
    from qwen3_runtime_b200.parts.base import BuildContext, build_part

    spec = PartSpec("paged_attention", dict(hidden_size=32, num_heads=2, num_kv_heads=1, head_dim=16, window=8))
    part = build_part("mixer", spec, BuildContext(dtype=torch.float32, device=torch.device("cpu"), ops=OPS, kv_bits=8))
    assert part.cache_spec() == KVLayerSpec(1, 16, 8, bits=8)
    assert {"cache_8bit", "attention_8bit"} <= set(part.kernel_groups())
    with pytest.raises(ValueError, match="differs"):
        kept_for_readers(0, part.cache_spec(), [KVLayerSpec(1, 16, 8, bits=4)])


def test_the_python_entry(tmp_path):
    llm = LLM(make_model_dir(tmp_path, "A"), dtype="float32", device=DEV, ops=OPS, kv_bits=8, block_size=4, num_kv_blocks=12, cuda_graph=False)
    assert len(llm.generate([1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], max_tokens=9)) == 9
    small = LLM(None, dtype="float32", device=DEV, ops=OPS, kv_bits=8, cuda_graph=False)
    assert small.engine.runtime.model.ctx.kv_bits == 8 and len(small.generate([1, 2, 3], max_tokens=2)) == 2


def test_bytes_of_a_page():
    layout = CacheLayout({0: KVLayerSpec(8, 128, bits=8), 1: KVLayerSpec(8, 128, bits=8)})
    assert layout.page_bytes(16, 2) == [2 * 8 * (4096 + 16)]
    assert layout.unpacked_bytes(10) == 10 * 4 * 8 * 128
    assert 0 < beside_unpacked(1 << 30, layout, 16, 100000, 1 << 28, 8, 256) < 1 << 30


def test_the_command_line_takes_it(tmp_path, capsys, monkeypatch):
    import qwen3_runtime_b200.cli as cli
    import qwen3_runtime_b200.engine.factory as factory

    seen = {}

    def fake(*args, **kw):
        seen.update(kw)
        raise SystemExit(0)

    monkeypatch.setattr(factory, "build_engine", fake)
    with pytest.raises(SystemExit):
        cli._generate(["--model", str(tmp_path), "--kv-bits", "8"])
    assert seen["kv_bits"] == 8
    with pytest.raises(SystemExit):
        cli._generate(["--model", str(tmp_path), "--kv-bits", "16"])
