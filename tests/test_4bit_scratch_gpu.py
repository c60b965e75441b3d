"""What attention over prompts unpacks from a cache in 4 bits, on the GPU: how much memory a step takes, and that sequences taken in turn get the
results of a step that takes them together.  The tolerances are those of tests/test_4bit_gpu.py."""

import pytest
import torch

import plain_4bit as p4
import test_4bit_gpu as t4
from test_4bit_gpu import BF16, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,G,D,page,window", [(8, 2, 128, 16, None), (8, 2, 128, 5, None), (8, 2, 64, 8, 20), (8, 2, 128, 16, 33), (4, 2, 256, 16, None),
                                               (4, 1, 80, 5, 9), (4, 2, 80, 16, None), (20, 1, 128, 16, None), (4, 2, 48, 16, 9)])
def test_sequences_in_turn(ops, H, G, D, page, window):  # noqa: F811
    """Pages that the windows have passed are gone; one sequence needs more than a turn's share, one brings nothing."""
    new, lens = [1, 33, 1, 5, 0, 18, 2, 1], [170, 33, 1, 290, 20, 50, 77, 60]
    c = p4.Cache(lens, G, D, page, seed=D)
    table = c.table.clone()
    if window:
        for b, (n, L) in enumerate(zip(new, lens)):
            table[b, : max(0, L - n - window + 1) // page] = -1
    q = t4.queries(sum(new), H, D, 4, extra=16)
    args = dict(window=window, table=table)
    whole = t4.attend(ops, c, q, new, lens, H, D ** -0.5, **args)
    t4.check_rows(whole, q[:, : H * D].view(-1, H, D), c, new, lens, D ** -0.5, window=window, wide=True)
    for pages in (8, 1):
        ops.UNPACK_BYTES = pages * 4 * G * page * D
        try:
            launches = ops.launches
            got = t4.attend(ops, c, q, new, lens, H, D ** -0.5, **args)
            assert ops.launches - launches >= 4
        finally:
            del ops.UNPACK_BYTES
        t4.check_rows(got, q[:, : H * D].view(-1, H, D), c, new, lens, D ** -0.5, window=window, wide=True)
        if D in (64, 128) and H // G <= 16:
            assert torch.equal(got, whole), "prompts' kernels do not look beyond a sequence"


@pytest.mark.parametrize("D,page,window", [(128, 16, None), (128, 16, 40), (80, 5, 40)])
def test_lengths_of_the_moment(ops, D, page, window):  # noqa: F811
    """A step that says how far its lengths may reach, or names none on the host: the device's lengths count, and no page is missing."""
    H, G, new, lens = 4, 2, [9, 1, 20, 3, 1], [100, 70, 20, 61, 1]
    c = p4.Cache(lens, G, D, page, seed=1, width=-(-200 // page))
    q = t4.queries(sum(new), H, D, 2)
    want = t4.attend(ops, c, q, new, lens, H, D ** -0.5, window=window)
    for change in (dict(captured_width=c.table.shape[1]), dict(host_kv_lens=[])):
        step = p4.step_of(new, lens, page)
        for name, x in change.items():
            setattr(step, name, x)
        got = t4.attend(ops, c, q, new, lens, H, D ** -0.5, window=window, step=step)
        t4.check_rows(got, q.view(-1, H, D), c, new, lens, D ** -0.5, window=window, wide=True)
        cu = step.host_cu_seqlens
        many = [t for b, n in enumerate(new) if n > 1 for t in range(cu[b], cu[b + 1])]
        assert torch.equal(got[many], want[many]), "(single tokens: other slices)"


@pytest.mark.parametrize("D", [128, 64, 256])
def test_a_captured_step_of_portions_and_single_tokens(ops, D):  # noqa: F811
    """Captured while its sequences are short, replayed when they are longer, up to the table that it was captured for."""
    H, G, page, new, short, long = 8, 2, 16, [1, 20, 1, 3], [5, 20, 9, 3], [250, 60, 140, 256]
    c = p4.Cache(long, G, D, page, seed=D, width=16)
    q = t4.queries(sum(new), H, D, 2)
    step = p4.step_of(new, short, page, captured_width=16)
    dev, pages, table, out = q.cuda(), c.pages.cuda(), c.table.cuda(), torch.zeros((sum(new), H * D), dtype=BF16, device="cuda")

    def run():
        ops.paged_attention_4bit(dev, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=D ** -0.5, step=step, **t4.sizes(c))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lens in (long, [n + 2 for n in short]):
        now = p4.step_of(new, lens, page)
        for name in ("kv_lens", "positions", "kv_longest"):
            getattr(step, name).copy_(getattr(now, name))
        graph.replay()
        torch.cuda.synchronize()
        ops.raise_if_kernel_error()
        cut = p4.Cache.__new__(p4.Cache)
        cut.__dict__.update(c.__dict__)
        cut.k, cut.v = ([[x[:, :n] for x in y] for y, n in zip(z, lens)] for z in (c.k, c.v))
        t4.check_rows(out.cpu().view(-1, H, D), q.view(-1, H, D), cut, new, lens, D ** -0.5, wide=True)


@pytest.mark.parametrize("new", [[1] + [20] * 31, [20] * 32])
@pytest.mark.parametrize("H,G,D", [(32, 8, 128), (8, 2, 256)])
def test_short_portions_beside_a_long_request_take_what_they_hold(ops, new, H, G, D):  # noqa: F811
    """31 portions of 20 tokens beside a request of 32,768: the long one's room once at most, and none when it decodes at 64 or 128."""
    lens, page = [32768] + [20] * 31, 16
    count = 32768 // page
    pages = torch.zeros((count + 1, G, p4.page_bytes(D, page)), dtype=torch.uint8, device="cuda")
    table = torch.arange(count, dtype=torch.int32, device="cuda").repeat(32, 1)
    step = p4.step_of(new, lens, page)
    q = torch.zeros((sum(new), H * D), dtype=BF16, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.paged_attention_4bit(q, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=0.1, step=step, num_kv_heads=G, head_dim=D,
                             page_size=page)
    torch.cuda.synchronize()
    own = 4 * G * D * page * (sum(-(-n // page) for n in lens[1:]) + (0 if D == 128 and new[0] == 1 else count))
    # beside the pages: tables of the longest sequence's width, the single tokens' slices and results
    assert torch.cuda.max_memory_allocated() - before <= own + 32 * count * 4 + (16 << 20)
    assert bool((out == 0).all())
    ops.raise_if_kernel_error()


def test_a_pool_sized_from_free_memory_leaves_room(tmp_path):
    """Pages and what prompts unpack beside them stay within the share of the free memory that the cache is given, and the engine runs."""
    import engine_4bit_cases as ec
    from helpers import TINY, random_ids
    from qwen3_runtime_b200.ops.cuda import CudaOps

    ops = CudaOps()
    torch.cuda.empty_cache()
    free, _total = torch.cuda.mem_get_info()
    share = 0.01
    eng = ec.engine(tmp_path, "E", "bfloat16", ops, "cuda", pages=None, kv_memory_fraction=share)
    layout, page = eng.runner.storage.layout, TINY["E"]["page_size"]
    held = eng.cache.num_pages[0] * page
    longest = min(held, eng.runtime.max_positions)
    room = max(min(ops.UNPACK_BYTES, layout.unpacked_bytes(held)), layout.unpacked_bytes(longest))
    assert 0.5 * share * free < eng.runner.storage.nbytes() + room <= share * free + (64 << 20)
    assert len(eng.generate(random_ids(TINY["E"]["config"].vocab_size, 40, 1), max_tokens=4)) == 4
    ops.raise_if_kernel_error()
