"""How exact states of a selective scan are to be: the recurrence in 64 bits beside what rounding can leave in each number,
and the recurrence by chunks with operands in parts of bf16, as products of tiles make it."""
from __future__ import annotations

import math

import torch

F64 = torch.float64
STEP = 2.0 ** -24                 # half a step of fp32

# A norm's bound of what a chunk's products leave in a state, as a part of the state's own: weights by a power of two that
# is off by 2 steps at most (2^-22), a sum of 8 products that is cut off by up to a step each time, on average half of
# one and while it is smaller than in the end (2^-21 at most), a weight's, an operand's and the state's own rounding
# (3 half steps).  2^-22 + 2^-21 + 3 * 2^-24 < 2^-20.
CHUNK = 2.0 ** -20
# Each further chunk: its decay's mean error (2e-8) and the rounding of what is kept, half a step.
FURTHER = 2e-8 + STEP


def heads_case(N, lens, kind, seed=0, H=3, P=64):
    """Tokens with rates per head, step sizes as they are in fp32: signs at random, strong decays in front of weak ones, or
    positive numbers that a state keeps for thousands of tokens."""
    g = torch.Generator().manual_seed(seed + N)
    T = sum(lens)
    row = torch.randn(T, H * P + 2 * N, generator=g).to(torch.bfloat16)
    dt = torch.exp(math.log(1e-3) + math.log(100) * torch.rand(T, H, generator=g))
    if kind == "strong":
        dt = 0.03 * dt
        dt[5::40] = 300.0
    if kind == "long":
        row, dt = row.abs(), 0.01 * dt
    a_log = torch.log(1 + 15 * torch.rand(H, generator=g))
    return dict(row=row, x=row[:, :H * P], b=row[:, H * P:H * P + N], c=row[:, H * P + N:], dt=dt, a_log=a_log,
                state=torch.randn(len(lens), H, P, N, generator=g))


def states(x, dt, b, a_log, groups, lens, starts, state):
    """(states, their bounds) behind portions whose slots are 0, 1, ... and whose step sizes are taken as they are.

    What a number is off by, token after token: what it was off by, decayed; a decay's error, of the number it decays: 2
    steps of the exponential, half of one of the product, 2e-8 that a power of two is corrected by, and of its argument's
    magnitude the rate's (2 steps of the exponential and half of one) and the product's half step; of the new term three
    roundings (two products, the sum)."""
    rates = a_log.shape[0]
    P, N = x.shape[1] // rates, b.shape[1] // groups
    A = -torch.exp(a_log.to(F64)).reshape(rates, -1)
    new, off, lo = [], [], 0
    for n, p, old in zip(lens, starts, state):
        S = old.to(F64).reshape(rates, P, N) if p else torch.zeros(rates, P, N, dtype=F64)
        E = torch.zeros_like(S)
        for t in range(lo, lo + n):
            arg = (dt[t].to(F64)[:, None] * A)[:, None]
            keep = torch.exp(arg)
            B = b[t].to(F64).view(groups, 1, N).repeat_interleave(rates // groups, 0)
            add = (dt[t].to(F64)[:, None] * x[t].to(F64).view(rates, P))[..., None] * B
            E = keep * E + keep * S.abs() * (4 * STEP + STEP + 2e-8 + 6 * STEP * arg.abs()) + 3 * STEP * add.abs() \
                + STEP * (keep * S + add).abs()
            S = keep * S + add
        new.append(S.view(old.shape))
        off.append(E.view(old.shape))
        lo += n
    return torch.stack(new), torch.stack(off)


def by_chunks(x, dt, b, a_log, lens, starts, state, parts=3, two_floats=True, rows=128):
    """The same states, rates per head, chunk after chunk: ``sum_j 2^(L_end - L_j) dt_j x_j B_j`` with the weighted x in
    ``parts`` parts of bf16 and the sums L in 64 bits or in one number of 32."""
    H, P, N, lo, new = a_log.shape[0], state.shape[2], state.shape[3], 0, []
    rate = -torch.exp(a_log.to(F64)) / math.log(2)
    for n, p, old in zip(lens, starts, state):
        h = old.clone() if p else torch.zeros_like(old)
        for t in range(lo, lo + n, rows):
            end = min(t + rows, lo + n)
            la = dt[t:end].to(F64) * rate
            L = la.cumsum(0) if two_floats else la.float().cumsum(0).to(F64)
            f = (torch.exp2(L[-1] - L).float() * dt[t:end])[..., None] * x[t:end].float().view(-1, H, P)
            S = torch.zeros(H, P, N, dtype=F64)
            for _ in range(parts):
                part = f.to(torch.bfloat16).float()
                S += torch.einsum("jhp,jn->hpn", part.to(F64), b[t:end].to(F64))
                f = f - part
            h = torch.exp2(L[-1]).float()[:, None, None] * h + S.float()
        new.append(h)
        lo += n
    return torch.stack(new)


def norm_error(got, want):
    """Of the heads of each state the largest error's norm, as a part of the state's."""
    d = got.detach().cpu().to(F64) - want
    return (d.flatten(-2).norm(dim=-1) / want.flatten(-2).norm(dim=-1)).max().item()


def chunk_bound(lens):
    return CHUNK + FURTHER * max((n + 127) // 128 - 1 for n in lens)
