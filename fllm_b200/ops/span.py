"""Attention behind which the first tokens of the text stay visible when a window has moved past them, attention for the nodes of draft trees,
and moves inside the cache pools: the fp32 PyTorch statement of each op (``SpanRef``, mixed into the reference ops) and the wrappers of the
sm_100a kernels (``SpanNative``).

A row at place P of its text sees what stands at a place w <= P with P - w < window or w < first (window 0: everything). A draft tree's node i
is stored at position ``tree_base + i``, but its place is ``tree_base`` + its depth, and a row sees of the tree only what its mask names: its
ancestors and itself. Parents come before their children. Masks are int64 [rows], or [rows, words] with 64 nodes to a word, at most 256.

Moves take pools ``[planes, blocks, heads, block_size, width]`` of one number of blocks and one block size (``KVCache.pools``,
``RowCache.pools``): every plane is moved the same way.
"""
from __future__ import annotations

from typing import List, Sequence, Tuple

import torch


def ordered_copies(pairs: Sequence[Tuple[int, int]], blocks: int) -> List[List[Tuple[int, int]]]:
    """Copies of blocks that are meant one after the other, in groups that may run at once: no group writes a block that it reads or writes
    elsewhere."""
    out, reads, writes = [], set(), set()
    for src, dst in pairs:
        src, dst = int(src), int(dst)
        if not (0 <= src < blocks and 0 <= dst < blocks):
            raise ValueError(f"copy of block {src} to {dst}: the pool has {blocks}")
        if src == dst:
            continue
        if not out or src in writes or dst in writes or dst in reads:
            out.append([])
            reads, writes = set(), set()
        out[-1].append((src, dst))
        reads.add(src)
        writes.add(dst)
    return out


def _check_span(window, first, bidirectional=False):
    if window < 0 or first < 0:
        raise ValueError("window and first must not be negative")
    if first and bidirectional:
        raise ValueError("first tokens that stay visible belong to causal attention")


class SpanRef:
    def _span_rows(self, q, k_cache, v_cache, tables, seqs, lens, seen, hq, hkv, head_dim, scale, sinks, softcap):
        """Row t attends to the tokens of sequence seqs[t] that ``seen(t, tokens)`` names among its first lens[t]."""
        bs, g = k_cache.shape[2], hq // hkv
        out = torch.zeros(q.shape[0], hq * head_dim, dtype=q.dtype, device=q.device)
        for t, (s, n) in enumerate(zip(seqs, lens)):
            tok = torch.arange(n, device=q.device)
            tok = tok[seen(t, tok)]
            if not len(tok):
                continue                                   # nothing is seen: 0, whatever the sink
            page = tables[s, tok // bs].long()
            k = k_cache[page, :, tok % bs].float().repeat_interleave(g, 1)
            v = v_cache[page, :, tok % bs].float().repeat_interleave(g, 1)
            x = torch.einsum("hd,nhd->hn", q[t].float().view(hq, head_dim), k) * scale
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
            if sinks is not None:
                x = torch.cat([x, sinks.float()[:, None]], 1)
            p = torch.softmax(x, -1)[:, :len(tok)]
            out[t] = torch.einsum("hn,nhd->hd", p, v).reshape(-1).to(q.dtype)
        return out

    def attention_first(self, q, k_cache, v_cache, block_tables, row_seq, positions, hq, hkv, head_dim, scale, window, first, sinks=None,
                        softcap=0.0):
        pos = [int(p) for p in positions]
        seen = lambda t, tok: (tok > pos[t] - window) | (tok < first)
        return self._span_rows(q, k_cache, v_cache, block_tables, row_seq.tolist(), [p + 1 for p in pos], seen, hq, hkv, head_dim, scale, sinks, softcap)

    def attention_tree_span(self, q, k_cache, v_cache, block_tables, tree_mask, tree_base, hq, hkv, head_dim, scale, window, sinks, softcap, first, meta):
        starts, lens, base = meta.q_starts.tolist(), meta.seq_lens.tolist(), tree_base.tolist()
        seqs = [s for s in range(meta.num_seqs) for _ in range(starts[s], starts[s + 1])]
        words = tree_mask.view(tree_mask.shape[0], -1).tolist()
        bits = [sum((w & ((1 << 64) - 1)) << (64 * i) for i, w in enumerate(row)) for row in words]

        def seen(t, tok):
            b, n = base[t], lens[seqs[t]]
            nodes = [i for i in range(n - b) if bits[t] >> i & 1]
            place = {b + i: b + k for k, i in enumerate(nodes)}
            me = b + len(nodes) - 1
            at = [j if j < b else place.get(j, -1) for j in range(n)]
            return torch.tensor([w >= 0 and (not window or me - w < window or w < first) for w in at], dtype=torch.bool, device=tok.device)
        return self._span_rows(q, k_cache, v_cache, block_tables, seqs, [lens[s] for s in seqs], seen, hq, hkv, head_dim, scale, sinks, softcap)

    def kv_copy_blocks(self, pools, pairs):
        if isinstance(pairs, torch.Tensor):
            pairs = pairs.tolist()
        for group in ordered_copies(pairs, pools[0].shape[1]):
            src, dst = ([p[i] for p in group] for i in (0, 1))
            for t in pools:
                t[:, dst] = t[:, src]

    def kv_compact(self, pools, block_tables, base, path, counts):
        bs = pools[0].shape[3]
        for b, n in enumerate(counts.tolist()):
            for i, node in enumerate(path[b].tolist()[:max(n, 0)]):
                if node < i:
                    raise ValueError("a path's nodes rise, and none is below its place")
                src, dst = int(base[b]) + node, int(base[b]) + i
                if src != dst:
                    s, d = int(block_tables[b, src // bs]), int(block_tables[b, dst // bs])
                    for t in pools:
                        t[:, d, :, dst % bs] = t[:, s, :, src % bs]


class SpanNative:
    def _attention_span(self, q, k_cache, v_cache, block_tables, hq, hkv, head_dim, scale, window, first, sinks, softcap, meta, tree_mask=None, tree_base=None):
        if meta is None or meta.q_starts is None or meta.seq_lens is None:
            raise ValueError("this attention takes its rows from the step batch: q_starts, seq_lens and their bounds")
        out, n = self.k.attention_span(q, k_cache, v_cache, block_tables, meta.q_starts, meta.seq_lens, meta.num_seqs, meta.max_q_len, meta.min_q_len,
                                       meta.max_kv_len, hq, hkv, head_dim, scale, window, first, sinks, softcap, tree_mask, tree_base, self.status)
        self.launches += n
        return out

    def kv_copy_blocks(self, pools, pairs):
        """Blocks ``pairs[i][0]`` of all planes to ``pairs[i][1]``. A host list is carried out as if pair after pair; an int32 tensor [n, 2] on the
        device in one launch: it names no block as a destination twice, or as a source and a destination (pairs out of range are skipped and
        reported in ``status``). Both are queued without waiting for the stream, and may be captured: a graph keeps the pairs of a list, and
        reads those of a tensor when it is replayed."""
        if isinstance(pairs, torch.Tensor):
            self.launches += self.k.kv_copy_blocks(pools, pairs, self.status)
            return
        for g in ordered_copies(pairs, pools[0].shape[1] if pools else 0):
            self.launches += self.k.kv_copy_listed(pools, [b for pair in g for b in pair], self.status)

    def kv_compact(self, pools, block_tables, base, path, counts):
        """For every sequence b the row of position ``base[b] + path[b, i]`` to position ``base[b] + i``, for i < counts[b], in this order: what is
        left of a draft tree when its accepted path has been found. The nodes of a path rise and path[b, i] >= i. All int32 on the device;
        sequences do not share the blocks that are written."""
        self.launches += self.k.kv_compact(pools, block_tables, base, path, counts, self.status)
