"""The engine with a cache in 4 bits, with and without a budget of tokens: the same cases with the kernels and with their plain statements."""

from __future__ import annotations

import torch

from helpers import TINY, make_model_dir, random_ids, trace_mixed, trace_portions, trace_whole
from qwen3_runtime_b200 import TokenBudget
from qwen3_runtime_b200.engine.batch import StepEntry
from qwen3_runtime_b200.engine.factory import build_engine


def engine(tmp_path, name, dtype, ops, device, *, budget=None, graph=False, pages=64, tokens=64, seqs=6, **kw):
    return build_engine(make_model_dir(tmp_path, name), dtype=dtype, device=device, ops=ops, block_size=TINY[name]["page_size"],
                        num_kv_blocks=pages, max_num_seqs=seqs, max_num_batched_tokens=tokens, cuda_graph=graph, kv_bits=4,
                        token_budget=budget, **kw)


def run_trace(eng, trace):
    """Logits of every wanted place, by request and position."""
    cache, runner, live, out = eng.cache, eng.runner, {}, {}
    for step in trace:
        entries = []
        for e in step["entries"]:
            rc = live.get(e["id"])
            if rc is None:
                rc = live[e["id"]] = cache.open(e["id"])
            cache.reserve(rc, len(e["tokens"]))
            entries.append(StepEntry(rc, e["tokens"], e["want"]))
        starts = [e.cache.num_computed for e in entries]
        logits = runner.run(entries)
        rows = iter(logits.float().cpu() if logits is not None else [])
        for e, start, s in zip(entries, starts, step["entries"]):
            for w in e.want:
                out[(s["id"], start + w)] = next(rows)
        cache.check_invariants()
        for rid in step["end"]:
            cache.close(live.pop(rid))
    assert cache.num_free_pages == cache.num_pages
    return out


def requests_of(name, lengths, seed=0):
    vocab = TINY[name]["config"].vocab_size
    return {f"r{i}": random_ids(vocab, n, seed + i) for i, n in enumerate(lengths)}


def case_schedules_agree(tmp_path, name, ops, device, lengths=(40, 25, 9), share=0.0):
    """float32: every schedule of the same requests gives the same bits, as without 4 bits; pages that are used again leak nothing.
    ``share``: of the largest logit, how far rows may differ (products whose bits depend on the batch may put a key on the other side
    of the border between two numbers, a step of a 15th of its group's spread)."""
    reqs = requests_of(name, lengths)
    want = run_trace(engine(tmp_path, name, "float32", ops, device), trace_whole(reqs))
    for trace in (trace_portions(reqs), trace_mixed(reqs, seed=3)):
        eng = engine(tmp_path, name, "float32", ops, device, pages=24)
        eng.runner.storage.poison_pages(0, list(range(24)))
        got = run_trace(eng, trace)
        for key, row in got.items():
            assert float((row - want[key]).abs().max()) <= share * float(want[key].abs().max()), key
    return want


def case_generation(tmp_path, name, dtype, ops, device, graphs=(False,)):
    """Requests alone, batched, in portions, preempted, running ahead or not, from captured steps or not: the same tokens (float32)."""
    vocab = TINY[name]["config"].vocab_size
    prompts = [random_ids(vocab, n, 50 + n) for n in (5, 33, 18, 1)]
    alone = [engine(tmp_path, name, dtype, ops, device).generate(p, max_tokens=12) for p in prompts]
    for graph in graphs:
        for kw in (dict(), dict(tokens=9), dict(run_ahead=False), dict(pages=-(-60 // TINY[name]["page_size"]), seqs=4)):
            eng = engine(tmp_path, name, dtype, ops, device, graph=graph, **kw)
            got = eng.generate_batch(prompts, max_tokens=12)
            if dtype == "float32":
                assert got == alone, (graph, kw)
            assert eng.cache.num_free_pages == eng.cache.num_pages
    return alone


def case_budget(tmp_path, name, dtype, ops, device, graph=False):
    """Long generations under a budget: no request holds more than it allows, the first and the last tokens stay, every head's tokens are
    different ones, what is kept of the first layer is what was written; pages go back."""
    vocab, page = TINY[name]["config"].vocab_size, TINY[name]["page_size"]
    budget = TokenBudget(24, first=3, recent=7, slack=6, observe=4)
    eng = engine(tmp_path, name, dtype, ops, device, budget=budget, graph=graph, pages=30, tokens=20, seqs=3)
    whole = engine(tmp_path, name, dtype, ops, device, pages=64)
    prompt = random_ids(vocab, 50, 7)
    cache, st = eng.cache, eng.runner.storage
    reqs = [eng.get_request(eng.add_request(p, max_tokens=n)) for p, n in ((prompt, 40), (random_ids(vocab, 4, 8), 60), (random_ids(vocab, 23, 9), 3))]
    cuts, most = 0, 0
    while not eng.is_finished():
        before = {r.request_id: r.cache.num_evicted for r in reqs if r.cache is not None}
        assert eng.step()
        cache.check_invariants()
        for r in reqs:
            rc = r.cache
            if rc is None:
                continue
            assert rc.held <= budget.keep + budget.slack and len(rc.tables[0]) <= cache.pages_for(rc.num_reserved - rc.num_evicted)
            most = max(most, rc.held)
            if rc.num_evicted and rc.num_evicted != before.get(r.request_id, 0) and r is reqs[0]:
                cuts += 1
                mass, places = (x[:, torch.tensor(rc.tables[0], dtype=torch.long, device=x.device)].cpu() for x in st.sums[0])
                at = places.permute(0, 2, 1, 3).flatten(2)[:, :, : rc.held]  # [layers, heads, held]
                newest = rc.num_computed - 1
                for layer in at:
                    for head in layer.tolist():
                        assert len(set(head)) == rc.held and max(head) == newest and min(head) == 0
                        assert set(range(budget.first)) <= set(head)
                        assert set(range(newest - budget.recent + 1, newest + 1)) <= set(head)
                assert bool((mass >= 0).all())
                if cuts == 1:  # the first layer's keys and values depend on the token and its position alone
                    held = _first_layer(st, rc, rc.held, page)
                    other = whole.cache.open("x")
                    tokens = r.token_ids[: rc.num_computed]
                    whole.cache.reserve(other, len(tokens))
                    whole.runner.run([StepEntry(other, tokens, [])])
                    full = _first_layer(whole.runner.storage, other, len(tokens), page)
                    whole.cache.close(other)
                    for h, head in enumerate(at[0].tolist()):
                        for slot, position in enumerate(head):
                            for a, b in zip(held, full):
                                assert torch.equal(a[h][slot], b[h][position])
    assert cuts >= 3 and most > budget.keep
    assert [r.num_output_tokens for r in reqs] == [40, 60, 3]
    assert cache.num_free_pages == cache.num_pages
    return [r.output_token_ids for r in reqs]


def _first_layer(storage, rc, count, page):
    """Key codes, value codes and both parameters of the first layer, per head and place."""
    import plain_4bit as p4

    spec = storage.layout.groups[0].layer_spec
    rec = storage.tensors[0][0].cpu()
    out = [[[] for _ in range(spec.num_kv_heads)] for _ in range(4)]
    for j in range(count):
        for h in range(spec.num_kv_heads):
            for part, (a, n) in zip(out, p4.places_in(spec.head_dim, page, j % page)):
                part[h].append(rec[rc.tables[0][j // page], h, a:a + n])
    return out


def case_roomy_budget_changes_nothing(tmp_path, name, ops, device):
    vocab = TINY[name]["config"].vocab_size
    prompts = [random_ids(vocab, n, 50 + n) for n in (5, 33)]
    want = engine(tmp_path, name, "float32", ops, device).generate_batch(prompts, max_tokens=10)
    assert engine(tmp_path, name, "float32", ops, device, budget=200).generate_batch(prompts, max_tokens=10) == want
