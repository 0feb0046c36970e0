"""Caches in 8 bits with scales for each block and head, their operators' definitions in 64 bits, and how far 16-bit
kernels may be from them."""
import math

import torch

FP8, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Cache:
    """Blocks of random codes whose scales differ, and tables of requests over them."""

    def __init__(self, codes, heads, width, block, lens, seed=0, spread=1.0, blocks=None):
        gen = torch.Generator().manual_seed(seed)
        need = [-(-n // block) for n in lens]
        nb = blocks or sum(need) + 3
        self.block, self.heads, self.width, self.lens = block, heads, width, list(lens)
        self.codes = random_codes((2, nb, block, heads, width), codes, gen)
        self.scales = torch.exp2(torch.round(spread * torch.randn(2, nb, heads, generator=gen)) - (7 if codes == FP8 else 6))
        order = torch.randperm(nb, generator=gen).int()
        self.tables = torch.zeros(len(lens), max(1, max(need, default=0)), dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.tables[r, :n] = order[at:at + n]
            at += n
        self.unused = order[at:]
        self.seq_lens = torch.tensor(lens, dtype=torch.int32)

    def to(self, dev):
        for n in ("codes", "scales", "tables", "seq_lens"):
            setattr(self, n, getattr(self, n).to(dev))
        return self

    def parts(self):
        return self.codes[0], self.codes[1], self.scales[0], self.scales[1]


def random_codes(shape, codes, gen):
    x = torch.randn(shape, generator=gen)
    if codes == INT8:
        return torch.round(40 * x).clamp(-127, 127).to(INT8)
    return (100 * x).clamp(-448, 448).to(FP8)


def attention(q, cache, q_lens, scale, window=0, first=0):
    """Definition in 64 bits: (outputs [T, Hq, D], sums of p |v| over sums of p, largest sums of |q k|, largest share of a
    key times its values' scale) for the rows of the requests, one behind the other."""
    q = q.double().cpu()
    codes, scales = cache.codes.cpu().float().double(), cache.scales.cpu().double()
    Hq, G = q.shape[1], q.shape[1] // cache.heads
    out, size, reach = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], Hq, dtype=torch.float64)
    top = torch.zeros_like(reach)
    at = 0
    for r, n in enumerate(q_lens):
        length = cache.lens[r]
        if n and length:
            pages = cache.tables[r, :-(-length // cache.block)].long().cpu()
            k, v = ((c[pages] * s[pages][:, None, :, None]).flatten(0, 1)[:length].transpose(0, 1)
                    for c, s in zip(codes, scales))
            k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
            rows = q[at:at + n].transpose(0, 1)
            pos, keys = torch.arange(length - n, length)[:, None], torch.arange(length)
            seen = keys <= pos
            if window:
                seen &= (keys > pos - window) | (keys < first)
            s = (rows @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where(seen.any(-1)[:, None], p, 0.0)
            out[at:at + n] = (p @ v).transpose(0, 1)
            size[at:at + n] = (p @ v.abs()).transpose(0, 1)
            unit = scales[1][pages].repeat_interleave(cache.block, 0)[:length].T.repeat_interleave(G, 0)
            top[at:at + n] = (p * unit[:, None]).amax(-1).T
            reach[at:at + n] = ((rows.abs() @ k.abs().transpose(1, 2)) * scale).masked_fill(~seen, 0.0).amax(-1).T
        at += n
    return out, size, reach, top


def allowed(out, size, reach, top, dtype, p_type, keys, width):
    """How far a kernel may be: half a step of the result's type; half a step of the probabilities' type each; scores in 32
    bits whose sum of ``width`` products and scale round by 2^-24 each (an error d of a score is one of 2 d of its
    probability's share); sums of ``keys`` terms in 32 bits, truncated.

    Where the codes meet 8-bit parts of a probability times its block's scale, the last part ends at a fixed place behind
    the largest of them, which is 1 or more: int8 digits of a multiple of 2^-26 are off by 2^-27; e4m3 parts of 16 times
    the number by half of the smallest step 2^-9 with weight 2^-8, 2^-18, which is 2^-22 of the number.  Each of ``keys``
    codes of at most 448 takes that part of ``top``.  (It shows where the keys that count have codes of 0.)"""
    p = torch.finfo(p_type).eps / 2 + 2 * (width + 8) * 2.0 ** -23 * reach[..., None] + (keys + 16) * 2.0 ** -22
    return size * p + keys * 448 * 2.0 ** -22 * top[..., None] + out.abs() * torch.finfo(dtype).eps / 2 * 1.01 + 1e-30 + torch.finfo(dtype).tiny


def check(got, q, cache, q_lens, scale, window, first, p_type):
    out, size, reach, top = attention(q, cache, q_lens, scale, window, first)
    n = sum(q_lens)
    far = (got[:n].double().cpu() - out[:n]).abs()
    may = allowed(out, size, reach, top, got.dtype, p_type, max(cache.lens, default=0), cache.width)[:n]
    assert torch.isfinite(got[:n]).all()
    worst = (far / may).max().item() if n else 0.0
    assert worst <= 1.0, worst
    return worst
