"""The plain torch statements of the operators around a cache in 4 bits, beside those of tests/emulated_ops.py: with them the engine's host
logic runs on the CPU."""

from __future__ import annotations

import torch

import plain_4bit as p4
from emulated_ops import TorchOps


class TorchOps4(TorchOps):
    @staticmethod
    def decode_4bit_ok(q, num_heads, num_kv_heads, head_dim):
        return False

    def qk_norm_rope_store_4bit(self, qkv, *, num_heads, num_kv_heads, head_dim, q_weight, k_weight, eps, cos, sin, positions, token_seq,
                                block_table, pages, page_size, write_kv=True, pairing="half", q_out=None, slots=None, mass=None, places=None):
        T, G, D = qkv.shape[0], num_kv_heads, head_dim
        rows = qkv.clone()
        # wide pages of one token each, named by the token's position
        k, v = torch.zeros((T, G, 1, D)), torch.zeros((T, G, 1, D))
        table = torch.zeros((int(token_seq.max()) + 1, int(positions.max()) + 1), dtype=torch.int32)
        table[token_seq.long(), positions.long()] = torch.arange(T, dtype=torch.int32)
        self.qk_norm_rope_store(rows.float() if rows.dtype == torch.float32 else rows, num_heads=num_heads, num_kv_heads=G, head_dim=D,
                                q_weight=q_weight, k_weight=k_weight, eps=eps, cos=cos, sin=sin, positions=positions, token_seq=token_seq,
                                block_table=table, k_pages=k, v_pages=v, page_size=1, write_kv=write_kv, pairing=pairing)
        (qkv if q_out is None else q_out)[:, : num_heads * D] = rows[:, : num_heads * D]
        if not write_kv:
            return
        slots = positions if slots is None else slots
        for t in range(T):
            slot = int(slots[t])
            page = int(block_table[int(token_seq[t]), slot // page_size])
            for h in range(G):
                p4.write(pages, page, h, slot % page_size, page_size, k[t, h, 0], v[t, h, 0])
            if mass is not None:
                mass[page, :, slot % page_size] = 0.0
            if places is not None:
                places[page, :, slot % page_size] = int(positions[t])

    def unpack_4bit(self, pages, *, num_kv_heads, head_dim, page_size, block_table, kv_lens, max_kv_len, dtype):
        n = -(-max_kv_len // page_size)
        k, v = p4.values_of(pages[block_table[:, :n].long().clamp(min=0).flatten()], head_dim, page_size)
        live = torch.arange(n * page_size)[None] < kv_lens[:, None].clamp(max=max_kv_len)
        live = live.view(-1, 1, page_size, 1)
        return [torch.where(live, x, 0.0).to(dtype) for x in (k, v)]

    def paged_attention_4bit(self, q, q_stride, *, num_heads, num_kv_heads, head_dim, pages, block_table, out, page_size, scale, step,
                             window=None, decode_slices=None, lse=None):
        k, v = p4.values_of(pages, head_dim, page_size)
        return self.paged_attention(q, q_stride, num_heads=num_heads, num_kv_heads=num_kv_heads, head_dim=head_dim, k_pages=k, v_pages=v,
                                    block_table=block_table, token_seq=step.token_seq, positions=step.positions, out=out, page_size=page_size,
                                    scale=scale, window=window)

    def attention_mass_4bit(self, q, q_stride, *, num_heads, num_kv_heads, head_dim, pages, mass, block_table, page_size, scale, step,
                            observe=None, lse=None):
        k, _v = p4.values_of(pages, head_dim, page_size)
        group = num_heads // num_kv_heads
        for t in range(step.num_tokens):
            b = int(step.token_seq[t])
            if observe is not None and t < int(step.cu_seqlens[b + 1]) - observe:
                continue
            at = torch.arange(int(step.positions[t]) + 1)
            page, row = block_table[b, at // page_size].long(), at % page_size
            keys = k[page, :, row].repeat_interleave(group, dim=1)  # [n, heads, D]
            w = torch.softmax(torch.einsum("hd,nhd->hn", q[t, : num_heads * head_dim].view(num_heads, -1).float(), keys) * scale, -1)
            mass[page, :, row] += w.view(num_kv_heads, group, -1).sum(1).T

    def evict_4bit(self, *, pages, mass, places, block_table, kv_lens, max_kv_len, keep, first, recent, num_kv_heads, head_dim, page_size):
        if pages.dim() == 3:
            pages, mass, places = pages[None], mass[None], places[None]
        for layer in range(pages.shape[0]):
            old = [x[layer].clone() for x in (pages, mass, places)]
            for b in range(block_table.shape[0]):
                at = [(int(block_table[b, j // page_size]), j % page_size) for j in range(int(kv_lens[b]))]
                for h in range(num_kv_heads):
                    chosen = p4.evict([float(old[1][p, h, r]) for p, r in at], [int(old[2][p, h, r]) for p, r in at], keep, first, recent)
                    for to, src in enumerate(chosen):
                        (p, r), (p2, r2) = at[to], at[src]
                        for (a, w), (a2, _) in zip(p4.places_in(head_dim, page_size, r), p4.places_in(head_dim, page_size, r2)):
                            pages[layer, p, h, a:a + w] = old[0][p2, h, a2:a2 + w]
                        mass[layer, p, h, r], places[layer, p, h, r] = old[1][p2, h, r2], old[2][p2, h, r2]
