"""Cases over caches held in 4 bits, made of those of span_oracle: what its pools hold, encoded; its keys and values, what the codes stand for.

Its bound holds here as well. Weights are f16, times a step s, for a product with codes that are counted from the middle of their range (at most 8 in
magnitude): an error of 2^-11 w s 8 for each token at most, and what is added to it for the middle of the range is exact in fp32. A row of bf16 values has
s <= (max - min) / 15 (1 + 2^-7), so 8 s 2^-11 <= 2^-11.8 (max - min): below 2^-8 A where A = sum_j w_j |v_j| >= (max - min) / 13 or so. The rows here are normal
values, of which no channel is near 0 in all tokens: A is about 0.8 where max - min is at most 8. Short rows see few tokens, whose weights are then large; the
bound's factor of 1.1 and `slack` (2^-11 x 8 s, summed over the weights) stand for those.

The kernel of prompts widens keys and values to f16 (times a power of two), each z + s c rounded once: relative 2^-11 of those within 2^-8 of a tile's largest,
2^-25 + 2^-26 of the unit in which that is above 2^-9 otherwise. Let o' be the formula's output for keys and values rounded to f16 as they are (normal values
here, for which that is 2^-11 as well); an error of either can be that of o' and, rounded the other way, twice it. The kernel's other errors are those of an
8-bit cache's kernel, so |y - o| <= bound' + 2 |o' - o|, both of which are computed here, and 2^-10 A for values whose roundings cancel in o' (A >= |o|, of
normal values about 0.8, is bound' / 2^-8 or less). Which kernel a row meets is the planner's
business: the other one's |y - o| <= bound is within that, up to bound - bound', so the larger of the two bounds is taken."""
from types import SimpleNamespace

import torch

import span_oracle as so
from fllm_b200.ops.kv4 import kv4_decode, kv4_encode


def setup(*args, **more):
    c = so.setup(*args, **more)
    c.k, c.v = kv4_encode(c.k), kv4_encode(c.v)
    c.steps = [kv4_encode(v)[..., -4:-2].contiguous().view(torch.bfloat16).float().amax().item() if len(v) else 0.0 for v in c.values]
    c.keys, c.values = [kv4_decode(kv4_encode(k)) if len(k) else k.float() for k in c.keys], [kv4_decode(kv4_encode(v)) if len(v) else v.float() for v in c.values]
    return c


def slack(c):
    return 2.0 ** -11 * 8 * max(c.steps)


def want(c, *args, **more):
    o, bound = so.want(c, *args, **more)
    rounded = SimpleNamespace(**{**vars(c), "keys": [k.half() for k in c.keys], "values": [v.half() for v in c.values]})
    o2, bound2 = so.want(rounded, *args, **more)
    return o, torch.maximum(bound, bound2) * (1 + 2.0 ** -2) + 2 * (o2 - o).abs() + slack(c)


def blocks_of_head(c, picks, block, row, head):
    """[tokens of the row's text] truth values: what the row reads of a key head."""
    s = int(c.row_seq[row])
    n = int(c.positions[row]) + 1
    seen = torch.zeros(c.lens[s], dtype=torch.bool)
    for b in picks[row, head].tolist():
        if b >= 0:
            seen[b * block:(b + 1) * block] = True
    seen[n:] = False
    return seen


def want_blocks(c, picks, scale, sinks=None, cap=0.0):
    """(outputs, bounds) [rows, hq * D] of attention over the blocks that ``picks`` names."""
    block, g = c.k.shape[2], c.hq // c.hkv
    outs, bounds = [], []
    for r in range(c.q.shape[0]):
        s = int(c.row_seq[r])
        o, b = [], []
        for h in range(c.hkv):
            q = c.q[r].view(c.hq, c.D)[h * g:(h + 1) * g][None]
            y, z = so.attend(q, c.keys[s][:, h:h + 1], c.values[s][:, h:h + 1], blocks_of_head(c, picks, block, r, h)[None], scale,
                             None if sinks is None else sinks[h * g:(h + 1) * g], cap)
            o.append(y.flatten())
            b.append(z.flatten())
        outs.append(torch.cat(o))
        bounds.append(torch.cat(b))
    return torch.stack(outs), torch.stack(bounds) + (slack(c) if hasattr(c, "steps") else 0.0)
