"""What the kernels around a cache in 4 bits read of a step is looked at before anything is launched: types, sizes, devices."""

import pytest
import torch

from qwen3_runtime_b200.ops.cuda import CudaOps, KernelError
from test_4bit_cpu import Table, attention_args, i32


class Elsewhere(torch.Tensor):
    """A tensor that says it lies on another device."""

    def get_device(self):
        return 7


class Here(Table):
    """A table whose own device is the CPU."""

    _check_here = CudaOps._check_here

    def __init__(self):
        super().__init__()
        self._device_index, self._slices_cache = torch.zeros(1).get_device(), {}

    def paged_attention(self, *args, **kw):
        pass


def call(sums, new=(1, 1), lse=None, **change):
    ops, args = Here(), attention_args(new=new)
    for name, value in change.items():
        setattr(args["step"], name, value)
    q, stride = args.pop("q"), args.pop("q_stride")
    if sums:
        args.pop("out")
        ops.attention_mass_4bit(q, stride, mass=torch.zeros((4, 2, 16)), lse=lse, **args)
    else:
        ops.paged_attention_4bit(q, stride, **args)
    return ops.calls


def elsewhere(x):
    return i32(x).as_subclass(Elsewhere)


@pytest.mark.parametrize("sums", [False, True])
@pytest.mark.parametrize("new", [(1, 1), (3, 1)])
@pytest.mark.parametrize("cu,match", [(torch.tensor([0, 1, 2]), "cu_seqlens"), (i32([0, 1]), "cu_seqlens"), (i32([0, 0, 1, 1, 2, 2])[::2], "cu_seqlens"),
                                      (elsewhere([0, 1, 2]), "launches on")])
def test_where_sequences_begin(sums, new, cu, match):
    with pytest.raises(KernelError, match=match):
        call(sums, new, cu_seqlens=cu)


@pytest.mark.parametrize("change,match", [
    (dict(kv_longest=torch.tensor([20])), "kv_longest"), (dict(kv_longest=i32([])), "kv_longest"), (dict(kv_longest=elsewhere([20])), "launches on"),
    (dict(kv_lens=elsewhere([20, 3])), "launches on"),
    (dict(new=(1, 2), single_seqs=torch.tensor([0])), "single_seqs"), (dict(new=(1, 2), single_seqs=i32([])), "single_seqs"),
    (dict(new=(1, 2), single_seqs=None), "single_seqs"), (dict(new=(1, 2), single_seqs=elsewhere([0])), "launches on")])
def test_what_else_attention_reads(change, match):
    with pytest.raises(KernelError, match=match):
        call(False, **change)


def test_log_sums_that_lie_elsewhere():
    with pytest.raises(KernelError, match="launches on"):
        call(True, lse=torch.zeros((2, 4)).as_subclass(Elsewhere))


def test_steps_without_what_they_do_not_need_are_taken():
    assert call(False, kv_longest=None, single_seqs=None) == ["q3_decode_attention_4bit"]
    assert call(True, kv_longest=None, single_seqs=None) == ["q3_attention_mass_4bit"]
    assert call(False, new=(2, 3), kv_longest=None, single_seqs=None) == ["q3_unpack_4bit"]
