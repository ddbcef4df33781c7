"""A KV cache held in 4 bits: the fp32 PyTorch statement of its rows (``Kv4Ref``, mixed into the reference ops) and the wrappers of the sm_100a
kernels (``Kv4Native``). Rotation and write in one (``rope_kv_write``) and attention take such a cache like any other.

A pool is uint8 [blocks, kv heads, block_size, head_dim / 2 + 4]. The row of a token and head holds codes of 0 to 15, dims 2i and 2i + 1 in the low
and the high half of byte i, then a step s and a lowest value z in bf16; code c stands for z + s c. Of bf16 values x: z = min x, s = (max x - z) / 15
rounded up to bf16, c = (x - z) / s rounded to nearest (ties to even). A row with an infinity or a NaN, or whose range fp32 does not hold, reads as NaN.
At a head dim of 128 a token takes 68 bytes a head, bf16 256.
"""
from __future__ import annotations

import torch

KV4_TAIL = 4


def kv4_width(head_dim: int) -> int:
    """Bytes of a token's row of one head."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"a 4-bit cache has head dims of 64, 128 or 256, not {head_dim}")
    return head_dim // 2 + KV4_TAIL


def is_kv4(cache: torch.Tensor, head_dim: int) -> bool:
    return cache.dtype == torch.uint8 and cache.shape[-1] == head_dim // 2 + KV4_TAIL


def kv4_encode(x: torch.Tensor) -> torch.Tensor:
    """Rows of bf16 values [..., head_dim] -> uint8 [..., head_dim / 2 + 4]."""
    x = x.to(torch.bfloat16).float()
    low = x.amin(-1, keepdim=True)
    span = x.amax(-1, keepdim=True) - low
    fine = torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(span)
    low, span = torch.where(fine, low, 0.0), torch.where(fine, span, 0.0)
    step = ((torch.div(span, torch.full_like(span, 15)).view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)
    code = torch.where((step > 0) & fine, torch.round((x - low) / step).clamp(max=15), 0.0).nan_to_num(0.0).to(torch.uint8)
    tail = (torch.cat([torch.where(fine, step, float("nan")), low], -1).view(torch.int32) >> 16).to(torch.int16).view(torch.uint8)      # (bf16 values already)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, tail], -1)


def kv4_decode(rows: torch.Tensor) -> torch.Tensor:
    """uint8 [..., head_dim / 2 + 4] -> fp32 [..., head_dim]."""
    half = rows.shape[-1] - KV4_TAIL
    par = rows[..., half:].contiguous().view(torch.bfloat16).float()
    code = torch.stack([rows[..., :half] & 15, rows[..., :half] >> 4], -1).flatten(-2).float()
    return par[..., 1:] + code * par[..., :1]


def cache_values(rows: torch.Tensor, head_dim: int) -> torch.Tensor:
    """fp32 values of rows of a cache of any kind."""
    return kv4_decode(rows) if is_kv4(rows, head_dim) else rows.float()


def cache_rows(x: torch.Tensor, cache: torch.Tensor) -> torch.Tensor:
    """Rows [..., head_dim] as what ``cache`` holds."""
    return kv4_encode(x) if is_kv4(cache, x.shape[-1]) else x.to(cache.dtype)


class Kv4Ref:
    def kv4_write(self, k, v, slots, k_cache, v_cache):
        hkv, bs = k_cache.shape[1], k_cache.shape[2]
        at = slots[slots >= 0].long()
        for x, cache in ((k, k_cache), (v, v_cache)):
            cache[at // bs, :, at % bs] = kv4_encode(x[slots >= 0].view(at.numel(), hkv, -1))

    def kv4_read(self, cache, slots):
        bs = cache.shape[2]
        at = slots.clamp(min=0).long()
        rows = kv4_decode(cache[at // bs, :, at % bs]).flatten(1)
        return torch.where(slots[:, None] >= 0, rows, torch.zeros_like(rows))


class Kv4Native:
    def kv4_write(self, k, v, slots, k_cache, v_cache):
        """Rows k and v [rows, hkv * head_dim] (bf16) to the places ``slots`` [rows] (int32: block * block_size + offset, none named twice; negative:
        the row is not kept) of a 4-bit cache. Slots behind the pool are skipped and reported in ``status``."""
        self.k.kv4_write(k, v, slots, k_cache, v_cache, self.status)
        self.launches += 1

    def kv4_read(self, cache, slots):
        """What the rows at ``slots`` of a 4-bit cache stand for, fp32 [rows, hkv * head_dim]; 0 where a slot is negative."""
        self.launches += 1
        return self.k.kv4_read(cache, slots, self.status)
