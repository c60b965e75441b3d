"""Sums of attention weights in captured steps, host side: a step is captured with padding rows of one token, so the keys of a slice come from
the chooser that the step's key holds, not from those rows."""

import torch

import plain_4bit as p4
from qwen3_runtime_b200 import TokenBudget
from qwen3_runtime_b200.config import PartSpec
from qwen3_runtime_b200.ops.cuda import CudaOps
from qwen3_runtime_b200.parts.base import BuildContext, build_part
from test_4bit_cpu import Table, cache


class Noting(Table):
    def _call(self, group, name, what, *args):
        super()._call(group, name, what, *args)
        self.last = args


def test_keys_of_a_slice():
    table = Table()
    for lens in ([], [1], [40] * 8, [4096] * 8, [65 + 83 * i for i in range(48)], [32768] * 64, [131072] * 200):
        for heads in (1, 8):
            keys = table.mass_slice_keys_4bit(lens, heads)
            assert keys >= 128 and keys & (keys - 1) == 0
            blocks = sum(n * heads / keys for n in lens)
            assert keys == 128 or 4 * 148 <= blocks < 2 * 4 * 148 + 1e-9
    assert table.mass_slice_keys_4bit([65 + 83 * i for i in range(48)], 8) == 1024


def slices(ops, lens, **kw):
    """Blocks a (sequence, kv head) that the sums' launch asks for: its last argument."""
    G, H, D, page = 2, 4, 128, 16
    step = p4.step_of([1] * len(lens), lens, page, device="cpu", captured_width=kw.pop("captured_width", 0))
    table = torch.zeros((len(lens), 256), dtype=torch.int32)
    ops.attention_mass_4bit(torch.zeros((len(lens), H * D), dtype=torch.bfloat16), H * D, num_heads=H, num_kv_heads=G, head_dim=D, pages=cache(D, page, G),
                            mass=torch.zeros((4, G, page)), block_table=table, page_size=page, scale=1.0, step=step,
                            lse=torch.zeros((len(lens), H)), **kw)
    return ops.last[-1]


def test_a_captured_step_takes_the_slices_of_its_key():
    ops, lens = Noting(), [2000] * 400
    keys = ops.mass_slice_keys_4bit(lens, 2)
    assert keys == 2048 and slices(ops, lens) == 1
    assert slices(ops, [1] * 400, captured_width=256) == 4096 // 128, "padding rows alone: the shortest slices"
    assert slices(ops, [1] * 400, captured_width=256, slice_keys=keys) == 2


def test_the_mixer_asks_for_them_under_a_budget():
    class Ops(CudaOps):
        def __init__(self):
            self._slices_cache = {}

    spec = PartSpec("paged_attention", dict(hidden_size=256, num_heads=4, num_kv_heads=2, head_dim=128))
    for budget in (None, TokenBudget(100)):
        for dtype in (torch.bfloat16, torch.float32):
            part = build_part("mixer", spec, BuildContext(dtype=dtype, device=torch.device("cpu"), ops=Ops(), kv_bits=4, kv_budget=budget))
            found = {key[0]: fn([2000] * 400) for key, fn in part.step_choosers().items()}
            want = {} if dtype == torch.float32 else {"decode_slices_4bit"} | ({"mass_slice_keys_4bit"} if budget else set())
            assert set(found) == set(want) and found.get("mass_slice_keys_4bit", 2048) == 2048
