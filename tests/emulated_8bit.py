"""The plain torch statements of the operators around a cache in 8 bits, beside those of tests/emulated_ops.py: with them the engine's host
logic runs on the CPU."""

from __future__ import annotations

import torch

import plain_8bit as p8
from emulated_ops import TorchOps


class TorchOps8(TorchOps):
    def qk_norm_rope_store_8bit(self, qkv, *, num_heads, num_kv_heads, head_dim, q_weight, k_weight, eps, cos, sin, step, block_table, pages,
                                page_size, write_kv=True, pairing="half", q_out=None):
        T, G, D = qkv.shape[0], num_kv_heads, head_dim
        rows = qkv.clone()
        # wide pages of one token each, named by the token's position
        k, v = torch.zeros((T, G, 1, D)), torch.zeros((T, G, 1, D))
        table = torch.zeros((int(step.token_seq.max()) + 1, int(step.positions.max()) + 1), dtype=torch.int32)
        table[step.token_seq.long(), step.positions.long()] = torch.arange(T, dtype=torch.int32)
        self.qk_norm_rope_store(rows, num_heads=num_heads, num_kv_heads=G, head_dim=D, q_weight=q_weight, k_weight=k_weight, eps=eps, cos=cos,
                                sin=sin, positions=step.positions, token_seq=step.token_seq, block_table=table, k_pages=k, v_pages=v, page_size=1,
                                write_kv=write_kv, pairing=pairing)
        (qkv if q_out is None else q_out)[:, : num_heads * D] = rows[:, : num_heads * D]
        if not write_kv:
            return
        for b in range(step.num_seqs):
            t0, t1, L = int(step.cu_seqlens[b]), int(step.cu_seqlens[b + 1]), int(step.kv_lens[b])
            past = L - (t1 - t0)
            for i in range(past // page_size, -(-L // page_size)):
                page = int(block_table[b, i])
                old, upto = max(0, past - i * page_size), min(page_size, L - i * page_size)
                first = t0 + i * page_size + old - past
                for h in range(G):
                    for which, x in enumerate((k, v)):
                        new = p8.four_bits(x[first:first + upto - old, h, 0])
                        kept = p8.read_rows(pages[page, h], D, page_size, which, old)[0]
                        p8.write_rows(pages, page, h, page_size, which, torch.cat([kept, new]))

    def unpack_8bit(self, pages, *, num_kv_heads, head_dim, page_size, block_table, kv_lens, max_kv_len, dtype):
        n = -(-max_kv_len // page_size)
        k, v = p8.values_of(pages[block_table[:, :n].long().clamp(min=0).flatten()], head_dim, page_size)
        live = torch.arange(n * page_size)[None] < kv_lens[:, None].clamp(max=max_kv_len)
        live = live.view(-1, 1, page_size, 1)
        return [torch.where(live, x, 0.0).to(dtype) for x in (k, v)]

    def paged_attention_8bit(self, q, q_stride, *, num_heads, num_kv_heads, head_dim, pages, block_table, out, page_size, scale, step,
                             window=None, keep_first=0, decode_slices=None):
        k, v = p8.values_of(pages, head_dim, page_size)
        return self.paged_attention(q, q_stride, num_heads=num_heads, num_kv_heads=num_kv_heads, head_dim=head_dim, k_pages=k, v_pages=v,
                                    block_table=block_table, token_seq=step.token_seq, positions=step.positions, out=out, page_size=page_size,
                                    scale=scale, window=window)
