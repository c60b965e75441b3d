"""The engine with a cache in 8 bits: the same cases with the kernels and with their plain statements."""

from __future__ import annotations

from engine_4bit_cases import requests_of, run_trace
from helpers import TINY, make_model_dir, random_ids, trace_mixed, trace_portions, trace_whole
from qwen3_runtime_b200.engine.factory import build_engine


def engine(tmp_path, name, dtype, ops, device, *, graph=False, pages=64, tokens=64, seqs=6, **kw):
    return build_engine(make_model_dir(tmp_path, name), dtype=dtype, device=device, ops=ops, block_size=TINY[name]["page_size"],
                        num_kv_blocks=pages, max_num_seqs=seqs, max_num_batched_tokens=tokens, cuda_graph=graph, kv_bits=8, **kw)


def case_schedules_agree(tmp_path, name, ops, device, lengths=(40, 25, 9), share=0.03):
    """float32: every schedule of the same requests gives nearly the same; pages that are used again leak nothing.  What may differ: a token sees
    numbers of its own page cut to the scale that later tokens of the same portion have made (by 2^-9 of it), and a key that this moves
    across the border between two numbers is off by an eighth of itself.  ``share``: of the largest logit, as between schedules of a cache in
    4 bits whose products depend on the batch, where a key moves by a 15th of its group's spread."""
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
    """Requests alone, batched, running ahead or not, from captured steps or not: the same tokens (float32).  In portions or preempted: as many, and
    every page comes back."""
    vocab = TINY[name]["config"].vocab_size
    prompts = [random_ids(vocab, n, 50 + n) for n in (5, 33, 18, 1)]
    alone = [engine(tmp_path, name, dtype, ops, device).generate(p, max_tokens=12) for p in prompts]
    for graph in graphs:
        for same, kw in ((True, dict()), (False, dict(tokens=9)), (True, dict(run_ahead=False)),
                         (False, dict(pages=-(-60 // TINY[name]["page_size"]), seqs=4))):
            eng = engine(tmp_path, name, dtype, ops, device, graph=graph, **kw)
            got = eng.generate_batch(prompts, max_tokens=12)
            if dtype == "float32" and same:
                assert got == alone, (graph, kw)
            assert [len(x) for x in got] == [12] * 4 and eng.cache.num_free_pages == eng.cache.num_pages
    return alone


def trace_of_pages(requests, page):
    """Portions of one to three whole pages (a request's last one ends where it ends), every request in every step while it lasts."""
    steps, at = [], dict.fromkeys(requests, 0)
    while at:
        entries, end = [], []
        for i, rid in enumerate(list(at)):
            tokens = requests[rid]
            n = min(len(tokens) - at[rid], page * (1 + (len(steps) + i) % 3))
            entries.append({"id": rid, "tokens": tokens[at[rid]:at[rid] + n], "want": list(range(n))})
            at[rid] += n
            if at[rid] == len(tokens):
                end.append(rid)
                del at[rid]
        steps.append({"step": len(steps), "entries": entries, "end": end})
    return steps


def case_portions_of_pages(tmp_path, name, ops, device, lengths=(40, 25, 9, 33)):
    """float32: portions that end where pages end give the bits of whole prompts, whatever their company.  A page's tokens then come together, and
    what makes schedules differ (``case_schedules_agree``) has no place.  (Not for the CPU, where a row of PyTorch's products depends on how many there are.)"""
    reqs = requests_of(name, lengths)
    want = run_trace(engine(tmp_path, name, "float32", ops, device), trace_whole(reqs))
    eng = engine(tmp_path, name, "float32", ops, device)
    eng.runner.storage.poison_pages(0, list(range(64)))
    got = run_trace(eng, trace_of_pages(reqs, TINY[name]["page_size"]))
    assert got.keys() == want.keys()
    for key, row in got.items():
        assert bool((row == want[key]).all()), key
