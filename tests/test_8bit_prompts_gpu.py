"""Attention of prompts over a cache in 8 bits, straight over the codes and over unpacked pages, each where the other would be chosen too; and single
tokens that take the way of prompts.  The bounds are those of tests/test_8bit_gpu.py."""

import math

import pytest
import torch

import plain_8bit as p8
from test_8bit_gpu import BF16, attend, check_rows, i32, ops, queries, sizes  # noqa: F401 (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["unpacked", "straight"])
def form(request, ops, monkeypatch):  # noqa: F811
    """Whichever form the rule on times would choose; ``used`` collects the entry points that ran."""
    used, call = [], ops._call
    monkeypatch.setattr(ops, "_prompts_unpacked", lambda *sizes: request.param, raising=False)
    monkeypatch.setattr(ops, "_call", lambda group, name, *args: (used.append(name), call(group, name, *args))[1], raising=False)
    return request.param, used


def check_form(form, D):
    unpacked, used = form
    names = set(used) - {"q3_decode_attention_8bit"}
    assert names == ({"q3_unpack_8bit", f"q3_prompts_tiles{'_wide' if D > 128 else ''}_8bit"} if unpacked and D >= 64 else {"q3_prompts_attention_8bit"})


@pytest.mark.parametrize("window,keep_first", [(None, 0), (1, 0), (40, 6), (70, 200)])
@pytest.mark.parametrize("H,G,D,page", [(8, 8, 64, 5), (6, 2, 64, 8), (5, 1, 80, 16), (20, 4, 80, 24), (10, 1, 96, 32), (14, 2, 112, 1), (40, 2, 128, 16),
                                        (8, 2, 128, 100), (12, 4, 128, 64), (128, 1, 64, 16), (100, 1, 128, 16), (70, 1, 144, 8), (16, 2, 256, 7), (6, 1, 32, 3), (3, 3, 208, 16)])
def test_portions(ops, form, H, G, D, page, window, keep_first):  # noqa: F811
    """Portions with and without tokens before them, that end inside a tile, a page and a block of rows; single tokens and sequences that bring none
    between them."""
    new, lens = [0, 33, 1, 70, 0, 2, 1, 5, 0], [20, 33, 90, 210, 0, 64, 1, 130, 300]
    c = p8.Cache(lens, G, D, page, seed=D + G)
    q = queries(sum(new), H, D, H)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first)
    check_rows(got, q.view(-1, H, D), c, new, lens, D ** -0.5, window=window, keep_first=keep_first, wide=True)
    check_form(form, D)


@pytest.mark.parametrize("window,keep_first", [(None, 0), (2000, 70)])
@pytest.mark.parametrize("new,lens", [([37], [4021]), ([5, 37, 1, 60, 3], [40, 3021, 900, 64, 1500])])
@pytest.mark.parametrize("H,G,D", [(20, 4, 80), (40, 2, 128), (8, 2, 128), (6, 3, 64), (2, 1, 256)])
def test_portions_behind_long_contexts(ops, form, H, G, D, new, lens, window, keep_first):  # noqa: F811
    """One portion behind thousands of tokens, by itself and among others that have a key for the first of its slices alone."""
    c = p8.Cache(lens, G, D, 16, seed=3)
    q = queries(sum(new), H, D, 2)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first)
    check_rows(got, q.view(-1, H, D), c, new, lens, D ** -0.5, window=window, keep_first=keep_first, wide=True)
    check_form(form, D)


@pytest.mark.parametrize("H,G,D", [(10, 2, 80), (40, 2, 128)])
def test_turns_of_sequences(ops, form, H, G, D):  # noqa: F811
    """More sequences than are unpacked at a time, single tokens among them: the same results."""
    new, lens, page = [9, 1, 30, 2, 17], [100, 70, 30, 64, 90], 24
    c = p8.Cache(lens, G, D, page, seed=9)
    q = queries(sum(new), H, D, 4)
    whole = attend(ops, c, q, new, lens, H, D ** -0.5)
    check_rows(whole, q.view(-1, H, D), c, new, lens, D ** -0.5, wide=True)
    ops.UNPACK_BYTES = 8 * 4 * G * 16 * D
    try:
        assert torch.equal(attend(ops, c, q, new, lens, H, D ** -0.5), whole)
    finally:
        del ops.UNPACK_BYTES


@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_what_is_not_finite_stays_with_its_sequence_and_head(ops, form, D):  # noqa: F811
    """A key or value that is no number: tokens that see it are none; other heads and sequences are untouched, and so are, by a key, the
    tokens before it and, by a value, other channels."""
    def mutate(b, k, v):
        if b == 1:
            k[0, 30, 3] = math.nan
            v[1, 31, D - 2] = math.inf

    H, G, new, lens = 6, 3, [20, 20, 20], [40, 40, 40]
    c = p8.Cache(lens, G, D, 16, seed=1, mutate=mutate)
    q = queries(60, H, D, 5)
    got = attend(ops, c, q, new, lens, H, D ** -0.5)
    assert bool(got[:20].isfinite().all()) and bool(got[40:].isfinite().all()) and bool(got[:, 4:].isfinite().all())
    assert bool(got[30:40, :2].isnan().all()) and bool(got[20:30, :2].isfinite().all()), "a key: tokens that see it, and no others"
    assert bool(got[31:40, 2:4, D - 2].isnan().all())
    got[20:40, 2:4, D - 2] = 0
    assert bool(got[20:40, 2:4].isfinite().all()), "a value: its channel"


@pytest.mark.parametrize("H,G,D,page", [(10, 1, 80, 16), (20, 2, 96, 5), (40, 2, 128, 16), (20, 4, 80, 16)])
def test_captured_single_tokens(ops, H, G, D, page):  # noqa: F811
    """Steps of single tokens that the decode kernel does not take, captured, replayed with lengths that grow."""
    width, lens = 400 // page, [3, 150, 17]
    c = p8.Cache([400] * 3, G, D, page, seed=7, width=width)
    pages, table = c.pages.cuda(), c.table.cuda()
    q = torch.zeros((3, H * D), dtype=BF16, device="cuda")
    out = torch.zeros_like(q)
    step = p8.step_of([1] * 3, lens, page, captured_width=width)

    def run(to, by):
        ops.paged_attention_8bit(q, H * D, num_heads=H, pages=pages, block_table=table, out=to, scale=D ** -0.5, step=by, **sizes(c))

    run(out, step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out, step)
    for turn in range(1, 200, 33):
        now = [n + turn for n in lens]
        rows = queries(3, H, D, turn)
        q.copy_(rows)
        step.kv_lens.copy_(i32(now))
        step.positions.copy_(i32([n - 1 for n in now]))
        graph.replay()
        torch.cuda.synchronize()
        sub = p8.Cache([], G, D, page)
        sub.kv = [x[:, :, :n] for x, n in zip(c.kv, now)]
        sub.scales = [s[:, :, : -(-n // page)] for s, n in zip(c.scales, now)]
        check_rows(out.cpu().view(3, H, D), rows.view(-1, H, D), sub, [1] * 3, now, D ** -0.5, wide=True)


def test_portions_on_another_stream(ops, form):  # noqa: F811
    """Two steps of portions under way together: each with pages and slices of its own."""
    H, G, D = 10, 2, 128
    made = []
    for i, (new, lens) in enumerate((([40, 3], [900, 300]), ([7, 90, 1], [40, 700, 60]))):
        c = p8.Cache(lens, G, D, 16, seed=i)
        q = queries(sum(new), H, D, i)
        made.append((c, q.cuda(), c.pages.cuda(), c.table.cuda(), p8.step_of(new, lens, 16), torch.cuda.Stream(), attend(ops, c, q, new, lens, H, D ** -0.5)))
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (c, q, pages, table, step, stream, _want) in enumerate(made):
            with torch.cuda.stream(stream):
                out = torch.empty_like(q)
                ops.paged_attention_8bit(q, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=D ** -0.5, step=step, **sizes(c))
                outs[i].append(out)
    torch.cuda.synchronize()
    for got, (*_, want) in zip(outs, made):
        assert all(torch.equal(x.cpu().view(want.shape), want) for x in got)


@pytest.mark.parametrize("window,keep_first", [(None, 0), (300, 20)])
def test_captured_portions(ops, form, window, keep_first):  # noqa: F811
    """A step of portions, captured, replayed with lengths that grow to all that its pages hold: what is counted from the lengths holds for any."""
    H, G, D, page, new = 10, 2, 128, 16, [40, 1, 7]
    width, lens = 2048 // page, [60, 90, 7]
    c = p8.Cache([2048] * 3, G, D, page, seed=8, width=width)
    pages, table = c.pages.cuda(), c.table.cuda()
    q = torch.zeros((48, H * D), dtype=BF16, device="cuda")
    out = torch.zeros_like(q)
    step = p8.step_of(new, lens, page, captured_width=width)

    def run():
        ops.paged_attention_8bit(q, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=D ** -0.5, step=step, window=window,
                                 keep_first=keep_first, **sizes(c))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for more in (0, 1, 63, 800, 1958):
        now = [min(2048, n + more) for n in lens]
        rows = queries(48, H, D, more)
        q.copy_(rows)
        step.kv_lens.copy_(i32(now))
        step.positions.copy_(i32([L - n + i for n, L in zip(new, now) for i in range(n)]))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        ops.raise_if_kernel_error()
        sub = p8.Cache([], G, D, page)
        sub.kv = [x[:, :, :n] for x, n in zip(c.kv, now)]
        sub.scales = [s[:, :, : -(-n // page)] for s, n in zip(c.scales, now)]
        check_rows(out.cpu().view(48, H, D), rows.view(-1, H, D), sub, new, now, D ** -0.5, window=window, keep_first=keep_first, wide=True)


@pytest.fixture
def sliced(ops, monkeypatch):  # noqa: F811
    """Into how many slices the launches' tiles were cut."""
    found = []
    for name in ("_prompt_splits", "_tile_splits"):
        call = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *args, call=call: (found.append(call(*args)), found[-1])[1], raising=False)
    return found


SLICED = pytest.mark.parametrize("H,G,D", [(20, 4, 80), (40, 2, 128), (8, 2, 128), (6, 3, 64), (2, 1, 256)])


@SLICED
@pytest.mark.parametrize("window,keep_first", [(None, 0), (2000, 70)])
def test_rows_that_are_no_numbers_in_slices(ops, form, sliced, H, G, D, window, keep_first):  # noqa: F811
    """A query that is none, of which one number is none, or infinite: its rows are none, all others the same bits as without it."""
    new, lens = [37, 2], [4021, 900]
    c = p8.Cache(lens, G, D, 16, seed=3)
    clean = queries(39, H, D, 2)
    q = clean.clone().view(39, H, D)
    q[3, H - 1] = math.nan
    q[20, 0, D - 1] = math.nan
    q[21, 1, 5] = math.inf
    q[38, 0, 0] = math.nan
    args = (new, lens, H, D ** -0.5)
    want = attend(ops, c, clean, *args, window=window, keep_first=keep_first)
    got = attend(ops, c, q.view(39, -1), *args, window=window, keep_first=keep_first)
    assert min(sliced) >= 1 and max(sliced) > 1
    bad = torch.zeros((39, H), dtype=torch.bool)
    bad[[3, 20, 21, 38], [H - 1, 0, 1, 0]] = True
    assert bool(got[bad].isnan().all())
    assert torch.equal(got[~bad], want[~bad]) and bool(want.isfinite().all())


@SLICED
@pytest.mark.parametrize("first,end", [(0, 4000), (1500, 2700), (64, 65)])
def test_keys_that_are_no_numbers_throughout_slices(ops, form, sliced, H, G, D, first, end):  # noqa: F811
    """Rows that see such a key are none, whatever part of their keys it is; other heads, and rows whose window begins behind it, are as ever."""
    def mutate(b, k, v):
        k[0, first:end] = math.nan

    new, lens, R = [37], [4021], H // G
    c, plain = p8.Cache(lens, G, D, 16, seed=3, mutate=mutate), p8.Cache(lens, G, D, 16, seed=3)
    q = queries(37, H, D, 2)
    for window, keep_first, hidden in ((None, 0, 0), (4000, 40, 0), (4021 - 20 - first, 0, 20)):
        got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first)
        want = attend(ops, plain, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first)
        assert torch.equal(got[:, R:], want[:, R:]) and bool(want.isfinite().all())
        # the last row that sees the last of these keys through its window
        sees = [window is None or max(0, lens[0] - 37 + i - window + 1) < end or first < keep_first for i in range(37)]
        assert all(bool(got[i, :R].isnan().all()) for i in range(37) if sees[i])
        assert all(torch.equal(got[i, :R], want[i, :R]) for i in range(37) if not sees[i])
    assert max(sliced) > 1


@SLICED
@pytest.mark.parametrize("lens", [[30], [4021]])
def test_rows_whose_scores_are_all_minus_infinity(ops, form, H, G, D, lens):  # noqa: F811
    """No weight can be made of them: none, in one slice and in many."""
    def mutate(b, k, v):
        k[:, :, 7] = -1.0

    c = p8.Cache(lens, G, D, 16, seed=4, mutate=mutate)
    q = queries(20, H, D, 3).view(20, H, D)
    q[4, 0, 7] = math.inf
    got = attend(ops, c, q.view(20, -1), [20], lens, H, D ** -0.5)
    assert bool(got[4, 0].isnan().all())
    got[4, 0] = 0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("window,keep_first", [(None, 0), (30, 6)])
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (40, 2, 128), (6, 3, 64), (20, 4, 80), (4, 2, 256), (6, 1, 32)])
@pytest.mark.parametrize("new,lens", [([70, 5, 40, 1], [20, 0, 300, 0]), ([100], [40]), ([130, 2], [1, 2]), ([40, 3], [0, 0]),
                                      ([70, 40, 1], [20, 4000, 0])])
def test_sequences_that_hold_fewer_tokens_than_they_bring(ops, form, H, G, D, new, lens, window, keep_first):  # noqa: F811
    """Tokens in front of a sequence's first key get zeros, those with keys what they always get; with values that are no numbers as well."""
    c = p8.Cache(lens, G, D, 16, seed=D)
    q = queries(sum(new), H, D, H)
    got = attend(ops, c, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first)
    there, at = torch.zeros(sum(new), dtype=torch.bool), 0
    for n, L in zip(new, lens):
        there[at + n - min(n, L):at + n] = True
        at += n
    assert bool((got[~there] == 0).all())
    check_rows(got[there], q.view(-1, H, D)[there], c, [min(n, L) for n, L in zip(new, lens)], lens, D ** -0.5, window=window, keep_first=keep_first,
               wide=True)

    def mutate(b, k, v):
        v[0, :1] = math.nan

    bad = p8.Cache(lens, G, D, 16, seed=D, mutate=mutate)
    assert bool((attend(ops, bad, q, new, lens, H, D ** -0.5, window=window, keep_first=keep_first)[~there] == 0).all())


@pytest.mark.parametrize("H,G,D", [(10, 2, 128), (4, 2, 256)])
def test_captured_portions_of_sequences_that_hold_fewer_tokens(ops, form, H, G, D):  # noqa: F811
    """What is captured for sequences that hold their tokens holds for ones that do not: those in front of the first key get zeros."""
    page, new = 16, [40, 1, 70]
    width, full = 1024 // page, [60, 90, 700]
    c = p8.Cache([1024] * 3, G, D, page, seed=8, width=width)
    pages, table = c.pages.cuda(), c.table.cuda()
    q = queries(111, H, D, 5)
    dev, out = q.cuda(), torch.zeros((111, H * D), dtype=BF16, device="cuda")
    step = p8.step_of(new, full, page, captured_width=width)

    def run():
        ops.paged_attention_8bit(dev, H * D, num_heads=H, pages=pages, block_table=table, out=out, scale=D ** -0.5, step=step, **sizes(c))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for now in (full, [0, 0, 0], [39, 1, 20], [0, 90, 1024], [1, 0, 69]):
        step.kv_lens.copy_(i32(now))
        step.positions.copy_(i32([L - n + i for n, L in zip(new, now) for i in range(n)]))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        ops.raise_if_kernel_error()
        got, there, at = out.cpu().view(111, H, D), torch.zeros(111, dtype=torch.bool), 0
        for n, L in zip(new, now):
            there[at + n - min(n, L):at + n] = True
            at += n
        assert bool((got[~there] == 0).all())
        sub = p8.Cache([], G, D, page)
        sub.kv = [x[:, :, :n] for x, n in zip(c.kv, now)]
        sub.scales = [s[:, :, : -(-n // page)] for s, n in zip(c.scales, now)]
        check_rows(got[there], q.view(-1, H, D)[there], sub, [min(n, L) for n, L in zip(new, now)], now, D ** -0.5, wide=True)
