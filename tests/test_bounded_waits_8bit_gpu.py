"""The waits of attention over a cache in 8 bits, running out: as in tests/test_bounded_waits_gpu.py."""

from __future__ import annotations

import pytest
import torch

import plain_8bit as p8
import test_8bit_gpu as t8
from test_bounded_waits_gpu import _build

pytestmark = pytest.mark.gpu


def run(launch, *args):
    """The error word after a launch whose waits run out."""
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    code = launch(*args, word.data_ptr(), torch.cuda.current_stream().cuda_stream)
    stop.record()
    assert code == 0
    torch.cuda.synchronize()  # returns: every wait in the kernel is bounded
    assert start.elapsed_time(stop) < 2000.0
    return int(word.item())


@pytest.mark.parametrize("splits", [1, 2])
def test_decode_attention(splits):
    from qwen3_runtime_b200.ops.cuda import CudaOps

    ops = CudaOps()
    G, D, page, lens = 2, 128, 16, [300, 40]
    c = p8.Cache(lens, G, D, page, seed=3)
    q = t8.queries(2, 8, D, 1)
    dev, pages, table = q.cuda(), c.pages.cuda(), c.table.cuda()
    step, out = p8.step_of([1, 1], lens, page), torch.zeros((2, 8 * D), dtype=torch.bfloat16, device="cuda")
    launch = _build("attention_8bit", "q3_decode_attention_8bit")  # (compiled here the first time: not what is timed)
    assert run(launch, dev.data_ptr(), 8 * D, pages.data_ptr(), pages.shape[0], table.data_ptr(), table.shape[1], step.kv_lens.data_ptr(),
               step.cu_seqlens.data_ptr(), None, out.data_ptr(), None, None, 2, 8, G, D, page, D ** -0.5, 0, 0, splits, max(lens), None) == 22
    got = t8.attend(ops, c, q, [1, 1], lens, 8, D ** -0.5, slices=splits)  # the ordinary build afterwards
    t8.check_rows(got, q.view(2, 8, D), c, [1, 1], lens, D ** -0.5)


@pytest.mark.parametrize("D", [128, 256])
def test_prompts_under_a_window(D):
    from qwen3_runtime_b200.ops.cuda import CudaOps

    ops = CudaOps()
    H, G, page, new, lens = 8, 2, 16, [70, 200], [400, 200]
    per, group = (64, "prompts_tiles_8bit") if D == 128 else (32, "prompts_tiles_wide_8bit")
    c = p8.Cache(lens, G, D, page, seed=3)
    q = t8.queries(270, H, D, 1)
    step, dev, out = p8.step_of(new, lens, page), q.cuda(), torch.zeros((270, H * D), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((14, G, 64, D), dtype=torch.bfloat16, device="cuda")
    v, items = k.clone(), t8.i32([*([i, 70 * b, new[b], lens[b], 7 * b, 0, 0, 0] for b in range(2) for i in range(-(-new[b] // per))), [0] * 8])
    launch = _build(group, "q3_" + group)
    assert run(launch, dev.data_ptr(), H * D, 270, k.data_ptr(), v.data_ptr(), 14, items.data_ptr(), len(items) - 1, out.data_ptr(), H, G, D,
               D ** -0.5, 100, 20, 1, None, None, None, 2, 1) == 2
    got = t8.attend(ops, c, q, new, lens, H, D ** -0.5, window=100, keep_first=20)  # the ordinary build afterwards
    t8.check_rows(got, q.view(270, H, D), c, new, lens, D ** -0.5, window=100, keep_first=20, wide=True)
