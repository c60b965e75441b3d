"""The engine with a cache in 4 bits in bfloat16: captured steps against uncaptured ones, and the sums of attention weights against their plain
statement over what the engine's own layers read."""

import math

import pytest
import torch

import engine_4bit_cases as ec
import plain_4bit as p4
from helpers import TINY, random_ids, trace_portions
from qwen3_runtime_b200 import TokenBudget
from qwen3_runtime_b200.ops.cuda import CudaOps

pytestmark = pytest.mark.gpu


def sums_of(eng):
    mass, places = eng.runner.storage.sums[0]
    return mass.clone(), places.clone()


@pytest.mark.parametrize("name", ["D", "E"])
@pytest.mark.parametrize("budget", [None, TokenBudget(40, first=2, recent=10, slack=5)])
def test_captured_steps_are_the_uncaptured_ones(tmp_path, name, budget):
    """Four requests of unequal lengths, as many as a captured step has rows: the same kernels see the same numbers, so logits, tokens and sums are
    the same bits, cut or not."""
    ops, vocab = CudaOps(), TINY[name]["config"].vocab_size
    prompts = [random_ids(vocab, n, n) for n in (31, 5, 17, 50)]
    runs = []
    for graph in (False, True):
        eng = ec.engine(tmp_path, name, "bfloat16", ops, "cuda", budget=budget, graph=graph, tokens=128, seqs=4)
        requests = [eng.get_request(eng.add_request(p, max_tokens=24)) for p in prompts]
        while not eng.is_finished():
            eng.step()
        ops.raise_if_kernel_error()
        assert (eng.runner.graphs.replays if graph else 0) > 20 * graph - 1
        pages = list(range(eng.cache.num_pages[0]))  # (the scratch page is the padding rows')
        runs.append(([r.output_token_ids for r in requests], [x[:, pages] for x in sums_of(eng)] if budget else []))
    assert runs[0][0] == runs[1][0]
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


@pytest.mark.parametrize("name", ["D", "E"])
def test_captured_logits_are_the_uncaptured_ones(tmp_path, name):
    """One request, portions and then single tokens with given ids."""
    ops = CudaOps()
    reqs = ec.requests_of(name, (70,))
    a, b = (ec.run_trace(ec.engine(tmp_path, name, "bfloat16", ops, "cuda", graph=graph), trace_portions(reqs)) for graph in (False, True))
    assert a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)


class Noting(CudaOps):
    """Keeps what every call of the sums read and made."""

    def __init__(self):
        super().__init__()
        self.calls = []

    def attention_mass_4bit(self, q, q_stride, *, mass, pages, block_table, step, lse=None, observe=None, **kw):
        before = mass.clone()
        super().attention_mass_4bit(q, q_stride, mass=mass, pages=pages, block_table=block_table, step=step, lse=lse, observe=observe, **kw)
        self.calls.append(dict(q=q.clone(), pages=pages.clone(), table=block_table.clone(), cu=step.host_cu_seqlens, lens=step.host_kv_lens,
                               made=(mass.double() - before.double()).cpu(), base=before.double().cpu(), lse=lse, observe=observe, **kw))


@pytest.mark.parametrize("name", ["D", "E"])
def test_sums_are_those_of_what_a_layer_reads(tmp_path, name):
    """Every layer and step, with the attention's log sums handed on (single tokens) or not (portions), before and after cuts.  A score of the
    kernels is off by 2^-23 (D + 8) of its row's largest product sum, a log sum by as much and 2^-20 of its size; a sum is rounded once a step."""
    ops, vocab = Noting(), TINY[name]["config"].vocab_size
    budget = TokenBudget(24, first=2, recent=8, slack=4, observe=4)
    eng = ec.engine(tmp_path, name, "bfloat16", ops, "cuda", budget=budget, tokens=32, seqs=3, run_ahead=False)
    eng.generate_batch([random_ids(vocab, n, n) for n in (40, 7, 19)], max_tokens=12)
    handed = 0
    for call in ops.calls:
        H, G, D, page = call["num_heads"], call["num_kv_heads"], call["head_dim"], call["page_size"]
        keys = p4.values_of(call["pages"].cpu(), D, page)[0].double()  # [pages, heads, page, D]
        want, tol = torch.zeros_like(call["made"]), torch.zeros_like(call["made"])
        handed += call["lse"] is not None
        for b, L in enumerate(call["lens"]):
            at = torch.arange(L)
            pages, rows = call["table"][b].cpu().long()[at // page], at % page
            k = keys[pages, :, rows]  # [L, G, D]
            for t in range(max(call["cu"][b], call["cu"][b + 1] - call["observe"]), call["cu"][b + 1]):
                seen = L - (call["cu"][b + 1] - 1 - t)
                q = call["q"][t, : H * D].double().cpu().view(G, H // G, D)
                x = torch.einsum("lgd,grd->grl", k[:seen], q) * call["scale"]
                err = call["scale"] * 2.0 ** -23 * (D + 8) * float(q.abs().sum(-1).max()) * float(k[:seen].abs().max()) * 18
                w = torch.softmax(x, -1).sum(1)  # [G, seen]
                log_sum = float(torch.logsumexp(x, -1).abs().max())
                want[pages[:seen], :, rows[:seen]] += w.T
                tol[pages[:seen], :, rows[:seen]] += w.T * math.expm1(2 * (2 * err + 2.0 ** -20 * (1 + log_sum)))
        tol += 2.0 ** -23 * (call["base"].abs() + want) + 1e-30
        diff = (call["made"] - want).abs()
        scratch = eng.runner.storage.scratch_page[0]
        assert bool((diff <= tol)[:scratch].all())
    assert handed >= 8 * len(eng.runner.storage.layout.groups[0].cache_ids)
