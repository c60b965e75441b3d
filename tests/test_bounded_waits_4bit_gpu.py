"""The wait for the tiles of decode attention over a cache in 4 bits, running out: as in tests/test_bounded_waits_gpu.py."""

from __future__ import annotations

import pytest
import torch

import plain_4bit as p4
import test_4bit_gpu as t4
from test_bounded_waits_gpu import _build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("splits", [1, 2])
def test_decode_attention(splits):
    from qwen3_runtime_b200.ops.cuda import CudaOps

    ops = CudaOps()
    G, D, page, lens = 2, 128, 16, [300, 40]
    c = p4.Cache(lens, G, D, page, seed=3)
    q = t4.queries(2, 8, D, 1)
    dev, pages, table = q.cuda(), c.pages.cuda(), c.table.cuda()
    step, out = p4.step_of([1, 1], lens, page), torch.zeros((2, 8 * D), dtype=torch.bfloat16, device="cuda")
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    launch = _build("attention_4bit", "q3_decode_attention_4bit")  # (compiled here the first time: not what is timed)
    start.record()
    code = launch(
        dev.data_ptr(), 8 * D, pages.data_ptr(), pages.shape[0], table.data_ptr(), table.shape[1], step.kv_lens.data_ptr(),
        step.cu_seqlens.data_ptr(), None, out.data_ptr(), None, None, None, 2, 8, G, D, page, D ** -0.5, 0, splits, max(lens), None,
        word.data_ptr(), torch.cuda.current_stream().cuda_stream)
    stop.record()
    assert code == 0
    torch.cuda.synchronize()  # returns: every wait in the kernel is bounded
    assert start.elapsed_time(stop) < 2000.0 and int(word.item()) == 21
    got = t4.attend(ops, c, q, [1, 1], lens, 8, D ** -0.5, slices=splits)  # the ordinary build afterwards
    t4.check_rows(got, q.view(2, 8, D), c, [1, 1], lens, D ** -0.5)
