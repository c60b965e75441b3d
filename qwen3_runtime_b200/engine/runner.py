"""The step function.

``ModelRunner.run(entries)`` takes a batch of (request, its next tokens, wanted
places) -- portions of prompts beside single decoded tokens, cut anywhere -- runs
exactly those tokens as one batch against the cache that earlier steps left, stores
their keys and values, and returns float32 logits at the wanted places, in the order
of the entries and of each entry's ``want``.  It samples nothing: the engine samples
from what it returns, and trace replay writes it to disk.
Parity: qwen3_runtime/engine/model_runner.py:107-192 (``run`` / ``run_logits`` /
``_run_group``); there is no prefill/decode split here, one launch sequence serves
every mix.
"""

from __future__ import annotations

import torch

from ..cache.manager import CacheManager
from ..cache.storage import CacheStorage
from ..parts.model import DecoderModel
from .batch import BatchBuilder, StepEntry


class ModelRunner:
    def __init__(self, model: DecoderModel, cache: CacheManager, storage: CacheStorage, *,
                 max_positions: int, cuda_graph: bool = False, graph_batch_sizes=(1, 2, 4, 8, 16, 32, 64)):
        self.model = model
        self.cache = cache
        self.storage = storage
        self.device = model.ctx.device
        self.builder = BatchBuilder(cache, self.device, vocab_size=model.spec.vocab_size,
                                    max_positions=max_positions)
        self.graphs = None
        if cuda_graph:
            from .graph import DecodeGraphs

            self.graphs = DecodeGraphs(self, graph_batch_sizes)
        self.num_steps = 0

    def run(self, entries: list[StepEntry], device_tokens: torch.Tensor | None = None) -> torch.Tensor | None:
        """One step; returns logits ``[sum(len(want)), vocab]`` float32, or None.

        ``device_tokens`` (int32, one per entry, every entry bringing one token): the token ids
        are on the device only -- sampled by a step whose result the host has not read yet --
        and replace the placeholders in ``entries`` after the step's metadata is packed."""
        if device_tokens is not None and (any(len(e.tokens) != 1 for e in entries)
                                          or device_tokens.numel() != len(entries)):
            raise ValueError("device_tokens: one token per entry, every entry bringing exactly one")
        resets = [e.cache.slot for e in entries if e.cache.needs_state_reset]
        if resets:
            self.storage.zero_state_slots(resets)
            for e in entries:
                e.cache.needs_state_reset = False
        logits = None
        if self.graphs is not None:
            logits = self.graphs.try_run(entries, device_tokens)
        if logits is None:
            step = self.builder.build(entries, scratch_page=self.storage.scratch_page,
                                      scratch_slot=self.storage.scratch_slot)
            if device_tokens is not None:
                self.builder.last_token_ids.copy_(device_tokens)
            if step.decode_only:
                step.choices = self.model.step_choices(step.host_kv_lens)
            logits = self.model.forward(step, self.storage)
        else:
            logits = logits if logits.numel() else None
        for e in entries:
            self.cache.commit(e.cache, len(e.tokens))
        if self.cache.budget is not None:
            self.cut([e.cache for e in entries if self.cache.over_budget(e.cache)])
        self.num_steps += 1
        return logits

    def cut(self, requests) -> None:
        """Cut requests that hold more tokens than the budget allows: all layers at once, each kv head by its own sums.  What the
        next step reads lies in front; the pages behind it go back to the pool (later work on the stream comes after the moves)."""
        if not requests:
            return
        budget, page_size = self.cache.budget, self.cache.page_size
        width = max(len(t) for rc in requests for t in rc.tables)
        count, n_paged = len(requests), len(self.cache.paged_groups)
        host = torch.zeros((n_paged * count * width + count,), dtype=torch.int32, pin_memory=self.builder.pin)
        image = host.numpy()
        tables = image[: n_paged * count * width].reshape(n_paged, count, width)
        for g in range(n_paged):
            tables[g] = self.storage.scratch_page[g]
            for b, rc in enumerate(requests):
                tables[g, b, : len(rc.tables[g])] = rc.table_array(g)
        image[n_paged * count * width:] = [rc.held for rc in requests]
        dev = host.to(self.device, non_blocking=True)
        lens = dev[n_paged * count * width:]
        for g, gi in enumerate(self.cache.paged_groups):
            spec = self.storage.layout.groups[gi].layer_spec
            mass, places = self.storage.sums[gi]
            self.model.ops.evict_4bit(
                pages=self.storage.tensors[gi], mass=mass, places=places, kv_lens=lens, max_kv_len=max(rc.held for rc in requests),
                block_table=dev[g * count * width:(g + 1) * count * width].view(count, width), keep=budget.keep, first=budget.first,
                recent=budget.recent, num_kv_heads=spec.num_kv_heads, head_dim=spec.head_dim, page_size=page_size)
        for rc in requests:
            self.cache.cut(rc)
