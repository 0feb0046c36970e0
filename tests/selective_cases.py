"""Steps and definitions for the tests of a state-space mixer's operators: each operator's formula in 64 bits, token
by token, beside the sum of its terms' magnitudes, which bounds what rounding can do."""
from __future__ import annotations

import dataclasses
import math

import torch

F64 = torch.float64
NEW = 1e30                        # what a test finds where nothing was written


@dataclasses.dataclass
class Step:
    positions: torch.Tensor
    state_slots: torch.Tensor
    num_decode_tokens: int
    cu_q_prefill: torch.Tensor | None
    lens: list
    starts: list

    def to(self, dev):
        f = lambda t: None if t is None else t.to(dev)  # noqa: E731
        return dataclasses.replace(self, positions=f(self.positions), state_slots=f(self.state_slots),
                                   cu_q_prefill=f(self.cu_q_prefill))

    @property
    def tokens(self):
        return sum(self.lens)


def step(decodes=0, lens=(), starts=None, slots=None, behind=0):
    """``decodes`` single tokens, then portions; ``behind``: rows behind the last one."""
    lens = [1] * decodes + list(lens)
    starts = [3 + 5 * r if r % 3 else 0 for r in range(len(lens))] if starts is None else list(starts)
    pos = [torch.arange(s, s + n) for s, n in zip(starts, lens)] + [torch.zeros(behind, dtype=torch.long)]
    R = len(lens)
    order = torch.randperm(R, generator=torch.Generator().manual_seed(R)) if slots is None else torch.tensor(slots)
    cu = torch.tensor([0] + lens[decodes:]).cumsum(0).int() if R > decodes else None
    return Step(torch.cat(pos).long(), order.int(), decodes, cu, lens, starts)


def _places(md, num_slots, write):
    lo = 0
    write = md.state_slots if write is None else write
    for r, (n, p) in enumerate(zip(md.lens, md.starts)):
        if n:
            yield lo, lo + n, int(md.state_slots[r]), int(write[r]), p
        lo += n


def sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def conv(x, weight, bias, md, ring, act="silu", write=None):
    """(result, its terms' magnitudes, ring) in 64 bits."""
    back = weight.shape[0] - 1
    x64, w = x.to(F64), weight.to(F64)
    out, mag = torch.full_like(x64, NEW), torch.zeros_like(x64)
    new = None if ring is None else ring.clone()
    for lo, hi, slot, to, p in _places(md, 0, write):
        if ring is not None and not 0 <= slot < ring.shape[0]:
            out[lo:hi] = 0
            continue
        for t in range(lo, hi):
            s = torch.zeros_like(x64[0]) if bias is None else bias.to(F64)
            m = s.abs()
            for j in range(back + 1):
                src = t - back + j
                if src >= lo:
                    v = x64[src]
                elif ring is not None and p + src - lo >= 0:
                    v = ring[slot, (p + src - lo) % back].to(F64)
                else:
                    continue
                s, m = s + w[j] * v, m + (w[j] * v).abs()
            out[t], mag[t] = s * sigmoid(s) if act else s, m
        if ring is not None and 0 <= to < ring.shape[0]:
            for q in range(max(0, p + hi - lo - back), p + hi - lo):
                new[to, q % back] = x[lo + q - p] if q >= p else ring[slot, q % back]
    return out, mag, new


def scan(x, dt, b, c, a_log, groups, md, state, d=None, dt_bias=None, z=None, softplus=True,
         dt_limits=(0.0, math.inf), write=None):
    """(result, magnitudes, state, its magnitudes) in 64 bits."""
    T, rates = x.shape[0], a_log.shape[0]
    P, N = x.shape[1] // rates, b.shape[1] // groups
    x64 = x.to(F64).reshape(T, rates, P)
    v = dt.to(F64) + (0 if dt_bias is None else dt_bias.to(F64))
    v = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
    v = v.clamp(*dt_limits)
    A = -torch.exp(a_log.to(F64)).reshape(rates, -1)
    out, mag = torch.full((T, rates, P), NEW, dtype=F64), torch.zeros(T, rates, P, dtype=F64)
    new = None if state is None else state.to(F64).clone()
    smag = None if state is None else torch.zeros_like(new)
    for lo, hi, slot, to, p in _places(md, 0, write):
        if state is not None and not 0 <= slot < state.shape[0]:
            out[lo:hi] = 0
            continue
        S = torch.zeros(rates, P, N, dtype=F64)
        if state is not None and p:
            S = state[slot].to(F64).reshape(rates, P, N)
        M = S.abs()
        for t in range(lo, hi):
            B, C = (u[t].to(F64).view(groups, N).repeat_interleave(rates // groups, 0)[:, None] for u in (b, c))
            keep, add = torch.exp(v[t][:, None] * A)[:, None], (v[t][:, None] * x64[t])[..., None] * B
            S, M = keep * S + add, keep * M + add.abs()
            out[t], mag[t] = (S * C).sum(-1), (M * C.abs()).sum(-1)
            if d is not None:
                skip = d.to(F64)[:, None] * x64[t]
                out[t], mag[t] = out[t] + skip, mag[t] + skip.abs()
        if state is not None and 0 <= to < state.shape[0]:
            new[to], smag[to] = S.view(new[to].shape), M.view(new[to].shape)
    out, mag = out.reshape(T, -1), mag.reshape(T, -1)
    if z is not None:
        gate = z.to(F64) * sigmoid(z.to(F64))
        here = out != NEW
        out, mag = torch.where(here, out * gate, out), mag * gate.abs()
    return out, mag, new, smag


def norm(x, z, weight, groups, eps, bias=None, center=False, gate_after=False, act="silu"):
    """(result, its terms' magnitudes) in 64 bits."""
    f = {None: lambda u: u, "silu": lambda u: u * sigmoid(u), "sigmoid": sigmoid}[act]
    v = x.to(F64)
    g = torch.ones_like(v) if z is None else f(z.to(F64))
    v = v if gate_after else v * g
    v = v.view(*x.shape[:1], groups, -1)
    mean = v.mean(-1, keepdim=True) if center else torch.zeros_like(v[..., :1])
    scale = 1 / torch.sqrt((v - mean).square().mean(-1, keepdim=True) + eps)
    # a mean of n numbers is off by steps of the sum of their magnitudes over n, however small it is itself: |sum of (1 +
    # e_i) v_i - sum of v_i| <= max |e_i| sum |v_i|
    about = v.abs().mean(-1, keepdim=True) if center else mean
    m = ((v.abs() + about) * scale).flatten(1) * weight.to(F64).abs()
    v = ((v - mean) * scale).flatten(1) * weight.to(F64)
    if bias is not None:
        v, m = v + bias.to(F64), m + bias.to(F64).abs()
    if z is None:
        return f(v), m
    return (v * g, m * g.abs()) if gate_after else (v, m)


def near(got, want, dtype, rounding):
    """Every element: half a step of its type, and ``rounding`` for what was rounded on the way to it."""
    got = got.detach().cpu().to(F64)
    # (subnormal results of a 16-bit type are rounded to steps of its smallest number)
    lim = torch.finfo(dtype).eps / 2 * want.abs() + rounding + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert not torch.isnan(got).any()
    bad = (got - want).abs() > lim
    assert not bad.any(), (int(bad.sum()), got.shape, ((got - want).abs() / lim).max().item(), bad.nonzero()[:4].tolist())


def conv_case(C, taps, md, dtype, seed=0, pad=0, slots=None):
    g = torch.Generator().manual_seed(seed)
    T, S = md.positions.shape[0], slots or 2 * len(md.lens) + 1
    x = torch.randn(T, C + pad, generator=g).to(dtype)
    w, bias = torch.randn(taps, C, generator=g), torch.randn(C, generator=g)
    ring = torch.randn(S, taps - 1, C, generator=g).to(dtype)
    return x, w, bias, ring


def scan_case(form, H, P, N, G, md, dtype, seed=0, slots=None, dt32=False):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    T, S = md.positions.shape[0], slots or 2 * len(md.lens) + 1
    # x, B and C are views of one row; where their widths allow it, all of them lie on 16-byte boundaries
    row = rnd(T, H * P + 2 * G * N + (8 if H * P % 8 == 0 and G * N % 8 == 0 else 3)).to(dtype)
    parts = row[:, :H * P], row[:, H * P:H * P + G * N], row[:, H * P + G * N:H * P + 2 * G * N]
    dt = rnd(T, H) if dt32 else rnd(T, H).to(dtype)
    a_log = torch.log(1 + 7 * torch.rand(H, N, generator=g)) if form == "channels" else \
        torch.log(1 + 15 * torch.rand(H, generator=g))
    state = rnd(S, H, N) if form == "channels" else rnd(S, H, P, N)
    return dict(row=row, x=parts[0], b=parts[1], c=parts[2], dt=dt, a_log=a_log, d=rnd(H),
                dt_bias=rnd(H) - 2.0, z=rnd(T, H * P + 8).to(dtype)[:, :H * P], state=state)


def scan_rounding(md, N, mag):
    """What 32 bits can be off in a scan: each term of a sum passes at most as many products with decays as its
    portion has tokens, each off by the product's half step, the decay's (2 steps of expf and 1 of its argument, whose
    magnitude is below 16 wherever the decay counts: 8 half steps) and the sum's, then N sums of the read-out."""
    return mag * 2.0 ** -24 * (12 * max(md.lens) + N + 8)
