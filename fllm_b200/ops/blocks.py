"""Attention that reads only some blocks of the cache, selected for each query row and key head: the fp32 PyTorch statement of each op (``BlocksRef``,
mixed into the reference ops) and the wrappers of the sm_100a kernels (``BlocksNative``).

Bounds, int8 [blocks, kv heads, 2 * head_dim + 16], say of every full block between which values each channel of its keys lies: hi = ceil(max / 2^e),
lo = floor(min / 2^e), then e, the smallest exponent with which they fit (at least -120; 127: a value is not finite, or too large). With
u = sum_h max(q_h, 0) and w = sum_h max(-q_h, 0) over the heads of a key head's group, rounded to 7 bits in a unit of their own, a block's score
2^e (u . hi - w . lo) bounds sum_h q_h . k of its keys. It is computed in whole numbers, so equal inputs are answered equally everywhere.

A row whose text has more than ``count`` blocks reads the first ``lead``, the last ``tail`` (among them its own, the last one) and the best of the others,
ties to the lower block; a row with a shorter text reads all of it.
"""
from __future__ import annotations

import torch

from .kv4 import cache_values

BOUNDS_TAIL = 16
MOST_BLOCKS = 48 * 1024        # of a text that the kernel chooses from
NOT_FINITE = 127


def bounds_width(head_dim: int) -> int:
    return 2 * head_dim + BOUNDS_TAIL


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _unit(top):
    """The smallest e >= -120 with top <= 127 x 2^e (-120 for 0)."""
    e = (torch.frexp(top)[1] - 7).clamp(min=-120)
    return torch.where(top > 0, torch.where(top > 127 * _pow2(e.clamp(max=120)), e + 1, e), -120)


def code_bounds(k: torch.Tensor) -> torch.Tensor:
    """Keys [..., block_size, head_dim] in fp32 -> their bounds [..., 2 * head_dim + 16]."""
    fine = torch.isfinite(k).all(-1, keepdim=True).all(-2, keepdim=True)
    k = torch.where(fine, k, 0.0)
    hi, lo = k.amax(-2), k.amin(-2)
    e = _unit(torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True))
    fine = fine[..., 0] & (e <= 100)
    f = torch.where(fine, _pow2(-e.clamp(max=120)), 0.0)
    tail = torch.zeros(*e.shape[:-1], BOUNDS_TAIL, dtype=torch.int8, device=k.device)
    tail[..., :1] = torch.where(fine, e, NOT_FINITE).to(torch.int8)
    return torch.cat([torch.ceil(hi * f).to(torch.int8), torch.floor(lo * f).to(torch.int8), tail], -1)


def _check(hq, hkv, count, lead, tail, meta):
    if hq % hkv or lead < 0 or tail < 1 or count < lead + tail:
        raise ValueError("select_blocks: count must have room for the first and the last blocks, one of the last at least")
    if meta is None or meta.q_starts is None or meta.seq_lens is None:
        raise ValueError("select_blocks takes its rows from the step batch: q_starts, seq_lens and their bounds")


class BlocksRef:
    def kv_bounds(self, k_cache, bounds, slots):
        bs, head_dim = k_cache.shape[2], (bounds.shape[-1] - BOUNDS_TAIL) // 2
        full = slots[(slots >= 0) & (slots % bs == bs - 1)].long() // bs
        bounds[full] = code_bounds(cache_values(k_cache[full], head_dim))

    def _block_rows(self, meta):
        starts, lens = meta.q_starts.tolist(), meta.seq_lens.tolist()
        for b in range(meta.num_seqs):
            for r in range(starts[b], starts[b + 1]):
                yield b, r, max(0, lens[b] - (starts[b + 1] - r) + 1)          # sequence, row, tokens it sees

    def select_blocks(self, q, bounds, block_tables, hq, hkv, head_dim, block_size, count, meta, lead=1, tail=2):
        _check(hq, hkv, count, lead, tail, meta)
        picks = torch.full((q.shape[0], hkv, count), -1, dtype=torch.int32, device=q.device)
        for b, r, n in self._block_rows(meta):
            blocks = -(-n // block_size)
            if blocks <= count:
                picks[r, :, :blocks] = torch.arange(blocks, dtype=torch.int32, device=q.device)
                continue
            x = q[r].float().view(hkv, hq // hkv, head_dim)
            x = torch.where(torch.isfinite(x), x, 0.0)
            most = torch.finfo(torch.float32).max
            u = torch.cat([x.clamp(min=0).sum(1), (-x).clamp(min=0).sum(1)], -1).clamp(max=most)
            top = u.amax(-1, keepdim=True)
            u = torch.round(u * _pow2(-torch.where(top > 0, _unit(top), 0).clamp(max=126)))
            of = bounds[block_tables[b, :blocks].long()].transpose(0, 1).float()                # [hkv, blocks, 2 head_dim + 16]
            s = (u[:, None, :head_dim] * of[..., :head_dim]).sum(-1) - (u[:, None, head_dim:] * of[..., head_dim:2 * head_dim]).sum(-1)
            e = of[..., 2 * head_dim]
            s = torch.where(e == NOT_FINITE, float("inf"), s * _pow2(e.clamp(max=120)))[:, lead:blocks - tail]
            best = torch.argsort(s, dim=-1, descending=True, stable=True)[:, :count - lead - tail].sort(-1)[0] + lead
            ends = torch.arange(blocks, device=q.device).expand(hkv, -1)
            picks[r] = torch.cat([ends[:, :lead], best, ends[:, blocks - tail:]], -1).to(torch.int32)
        return picks

    def attention_blocks(self, q, k_cache, v_cache, block_tables, blocks, hq, hkv, head_dim, scale, meta, sinks=None, softcap=0.0):
        bs, g = k_cache.shape[2], hq // hkv
        out = torch.zeros(q.shape[0], hq * head_dim, dtype=q.dtype, device=q.device)
        for b, r, n in self._block_rows(meta):
            for h in range(hkv):
                tok = torch.tensor([i * bs + j for i in blocks[r, h].tolist() if i >= 0 for j in range(bs) if i * bs + j < n], dtype=torch.long, device=q.device)
                if not len(tok):
                    continue
                page = block_tables[b, tok // bs].long()
                k, v = (cache_values(c[page, h, tok % bs], head_dim) for c in (k_cache, v_cache))
                s = (q[r].float().view(hq, head_dim)[h * g:(h + 1) * g] @ k.T) * scale
                if softcap > 0:
                    s = softcap * torch.tanh(s / softcap)
                if sinks is not None:
                    s = torch.cat([s, sinks[h * g:(h + 1) * g].float()[:, None]], 1)
                p = torch.softmax(s, -1)[:, :len(tok)]
                out[r].view(hq, head_dim)[h * g:(h + 1) * g] = (p @ v).to(q.dtype)
        return out


class BlocksNative:
    def kv_bounds(self, k_cache, bounds, slots):
        """Bounds of the blocks that the step's rows complete: those of which a slot is the last (rows of the keys are in the cache by then)."""
        self.k.kv_bounds(k_cache, bounds, slots, self.status)
        self.launches += 1

    def select_blocks(self, q, bounds, block_tables, hq, hkv, head_dim, block_size, count, meta, lead=1, tail=2):
        """Blocks of its text that each row reads for each key head, int32 [rows, hkv, count]: rising, -1 behind the last. ``meta``: the step batch (a
        sequence's rows are its last ones; texts are at most ``max_kv_len`` long, those that are not are cut off and reported in ``status``)."""
        _check(hq, hkv, count, lead, tail, meta)
        picks, n = self.k.select_blocks(q, bounds, block_tables, meta.q_starts, meta.seq_lens, meta.num_seqs, meta.max_q_len, meta.max_kv_len, hq, hkv, head_dim,
                                        block_size, count, lead, tail, self.status)
        self.launches += n
        return picks

    def attention_blocks(self, q, k_cache, v_cache, block_tables, blocks, hq, hkv, head_dim, scale, meta, sinks=None, softcap=0.0):
        """Attention of which each row reads, of each key head, the blocks of its text that ``blocks`` [rows, hkv, count] names (each once, none behind the
        first negative one), up to its own position. Caches of bf16, e4m3 or 4-bit rows; head dims 64, 128 and 256, blocks of a multiple of 16 tokens."""
        return self._attention_span(q, k_cache, v_cache, block_tables, hq, hkv, head_dim, scale, 0, 0, sinks, softcap, meta, picks=blocks)
