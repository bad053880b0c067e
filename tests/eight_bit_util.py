"""The test double of the kernel surface with a cache in 8 bits and trees of drafted tokens, and the plain implementation with
keys and values quantised."""

from contextlib import contextmanager

import torch

import plain_cache
import plain_qwen2 as plain
from distie_amd.kernels.interface import EightBitCache
from torch_ops import TorchOps


class EightBitOps(TorchOps):
    def rope_kv_write_e4m3(self, qkv, meta, group, cache, inv_freq, num_heads, num_kv_heads, head_dim, write):
        T = qkv.shape[0]
        x = qkv.double().view(T, -1, head_dim)
        if inv_freq is not None:
            x = torch.cat([plain_cache.rotated(x[:, :num_heads + num_kv_heads], meta.positions, inv_freq), x[:, num_heads + num_kv_heads:]], 1)
        if write:
            P = cache.k.shape[2]
            slots = meta.groups[group].slots.long()
            k, kb = plain_cache.quantised(x[:, num_heads:num_heads + num_kv_heads])
            v, vb = plain_cache.quantised(x[:, num_heads + num_kv_heads:])
            code = lambda values, power: (values / torch.exp2(power.double() - 127)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
            cache.k.view(torch.uint8)[slots // P, :, slots % P] = code(k, kb)
            cache.v.view(torch.uint8)[slots // P, :, :, slots % P] = code(v, vb)
            cache.k_scale[slots // P, :, slots % P] = kb.to(torch.uint8)
            cache.v_scale[slots // P, :, slots % P] = vb.to(torch.uint8)
        return x[:, :num_heads].reshape(T, -1).to(qkv.dtype)

    @staticmethod
    def _values(cache):
        if not isinstance(cache, EightBitCache):
            return cache
        power = lambda b: torch.exp2(b.double() - 127)
        return cache.k.double() * power(cache.k_scale)[..., None], cache.v.double() * power(cache.v_scale)[..., None, :]

    def paged_attention_e4m3(self, qkv, meta, group, cache, num_heads, num_kv_heads, head_dim, scale, window):
        return self.paged_attention(qkv, meta, group, *self._values(cache), num_heads, num_kv_heads, head_dim, scale, window)

    def tree_attention(self, qkv, meta, group, cache, num_heads, num_kv_heads, head_dim, scale, window):
        k_cache, v_cache = self._values(cache)
        P, T = k_cache.shape[2], meta.num_tokens
        table = meta.groups[group].block_table.long()
        if meta.table_rows is not None:
            table = table[meta.table_rows.long()]
        out = torch.zeros(T, num_heads, head_dim)
        cu = meta.cu_q.tolist()
        for t in range(T):
            b = int(meta.token_request[t])
            n = cu[b + 1] - cu[b]
            past = int(meta.kv_len[b]) - n
            where = torch.cat([torch.arange(past), meta.positions[cu[b]:cu[b + 1]].long()])
            bits = [int(meta.tree[t, i // 64]) >> (i % 64) & 1 for i in range(n)]
            seen = torch.tensor([1] * past + bits, dtype=torch.bool)
            if window is not None:
                seen &= int(meta.positions[t]) - where < window
            at = seen.nonzero()[:, 0]
            k = k_cache[table[b, at // P], :, at % P].double().repeat_interleave(num_heads // num_kv_heads, 1)
            v = v_cache[table[b, at // P], :, :, at % P].double().repeat_interleave(num_heads // num_kv_heads, 1)
            q = qkv[t, :num_heads * head_dim].view(num_heads, head_dim).double()
            w = torch.softmax((q * k).sum(-1) * scale, 0)
            out[t] = (w[..., None] * v).sum(0)
        return out.view(T, -1).to(qkv.dtype)

    def keep_drafted(self, slab, page_axis, table, table_rows, past, path):
        held = slab.movedim(page_axis, 2)
        P, old = held.shape[2], held.clone()
        for b in range(path.shape[0]):
            row = table[int(table_rows[b]) if table_rows is not None else b].tolist()
            begin = int(past[b])
            for d, i in enumerate(path[b].tolist()):
                if i < 0:
                    break
                to, source = begin + d, begin + i
                held[:, row[to // P], to % P] = old[:, row[source // P], source % P]


@contextmanager
def quantised_keys_and_values():
    """Within it the plain implementation attends over keys and values as a cache in 8 bits holds them."""
    attention = plain.attention

    def over_codes(q, k, v, window=None):
        held = lambda x: plain_cache.quantised(x.double())[0].to(x.dtype)
        return attention(q, held(k), held(v), window)

    plain.attention = over_codes
    try:
        yield
    finally:
        plain.attention = attention
