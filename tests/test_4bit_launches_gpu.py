"""The kernel table's count of launches around a cache in 4 bits: as many as a captured call has kernels."""

import pytest
import torch

import plain_4bit as p4
import test_4bit_gpu as t4
from test_4bit_gpu import BF16, F32, ops, sizes  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def kernels_of(call):
    """Kernel nodes of a captured call (which has run once before)."""
    from cuda.bindings import runtime as rt

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    err, _none, count = rt.cudaGraphGetNodes(raw)
    err, nodes, _n = rt.cudaGraphGetNodes(raw, count)
    assert err == rt.cudaError_t.cudaSuccess
    return sum(rt.cudaGraphNodeGetType(n)[1] == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for n in nodes)


def check(ops, call):  # noqa: F811
    kernels = kernels_of(call)
    before = ops.launches
    call()
    torch.cuda.synchronize()
    assert ops.launches - before == kernels
    return kernels


@pytest.mark.parametrize("keep,want", [(50, 1), (1000, 2)])
def test_eviction(ops, keep, want):  # noqa: F811
    c = p4.Cache([keep + 600], 1, 64, 16)
    mass, places = torch.rand((c.pages.shape[0], 1, 16), device="cuda"), torch.zeros((c.pages.shape[0], 1, 16), dtype=torch.int32, device="cuda")
    pages, table, lens = c.pages.cuda(), c.table.cuda(), torch.tensor([keep + 600], dtype=torch.int32, device="cuda")
    assert check(ops, lambda: ops.evict_4bit(pages=pages, mass=mass, places=places, block_table=table, kv_lens=lens, max_kv_len=keep + 600,
                                             keep=keep, first=0, recent=0, **sizes(c))) == want


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 80), (F32, 64)])
@pytest.mark.parametrize("new", [[1, 1], [20, 1]])
@pytest.mark.parametrize("given", [False, True])
def test_sums_and_attention(ops, dtype, D, new, given):  # noqa: F811
    H, G, lens = 4, 2, [700, 90]
    c = p4.Cache(lens, G, D, 16)
    q, pages, table, step = t4.queries(sum(new), H, D, 1, dtype).cuda(), c.pages.cuda(), c.table.cuda(), p4.step_of(new, lens, 16)
    mass, lse = torch.zeros((c.pages.shape[0], G, 16), device="cuda"), torch.zeros((sum(new), H), device="cuda") if given else None
    out = torch.empty_like(q)
    args = dict(num_heads=H, pages=pages, block_table=table, scale=0.1, step=step, **sizes(c))
    assert check(ops, lambda: ops.attention_mass_4bit(q, H * D, mass=mass, lse=lse, **args)) == 1 + (not given)
    for slices in (1, 3, -3):
        check(ops, lambda: ops.paged_attention_4bit(q, H * D, out=out, decode_slices=slices, **args))
