"""The operators of a state-space mixer, as cases that can be timed and checked.

Between a mixer's two projections a step runs three operators over its rows:

* ``conv``   short causal convolution with SiLU over a request's tokens; the last rows of a request lie
             in a ring in its state slot
* ``scan``   selective state space scan, either with one rate per head (``heads``: a state of P x N
             numbers per head) or with rates of its own for every channel (``channels``: N numbers each)
* ``norm``   group norm of a row with its gate's activation

A step holds single tokens of running requests and portions of prompts, one behind the other.  Requests read
their state in one slot and leave it in another, as a request does that is forked into several answers, so
that a pass can be made again.
"""
from __future__ import annotations

import math
import types

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64                        # tokens of a chunk of the plain scan
EPS = 1e-5


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    def conv(name, dtype, channels, taps, decodes, lens, started):
        return dict(name=name, op="conv", dtype=dtype, channels=channels, taps=taps, decodes=decodes, lens=lens,
                    started=started)

    def heads(name, dtype, H, P, N, groups, decodes, lens, started, gate=False):
        return dict(name=name, op="scan", form="heads", dtype=dtype, heads=H, width=P, states=N, groups=groups,
                    decodes=decodes, lens=lens, started=started, gate=gate)

    def channels(name, dtype, D, N, decodes, lens, started):
        return dict(name=name, op="scan", form="channels", dtype=dtype, heads=D, width=1, states=N, groups=1,
                    decodes=decodes, lens=lens, started=started, gate=True)

    def norm(name, dtype, rows, channels, groups, after, center):
        return dict(name=name, op="norm", dtype=dtype, rows=rows, channels=channels, groups=groups, after=after,
                    center=center)

    return [
        # a full token budget of prompts, some of them continued, rows of x, B and C side by side
        conv("conv-prompts", "bf16", 10240, 4, 0, "2048,2048,1531,997,800,513,250,5", True),
        # the decode step of a busy server
        conv("conv-step-128", "bf16", 4352, 4, 128, "", True),
        # one long prompt: a state of 64 x 128 numbers for each of 128 heads
        heads("heads-prompt-4096", "bf16", 128, 64, 128, 8, 0, "4096", False),
        # running requests beside the portions of a few prompts of odd lengths
        heads("heads-mixed", "bf16", 64, 64, 128, 1, 24, "1024,701,333,129,64,1,40", True),
        # one user waits for each token of an answer
        heads("heads-step-1", "bf16", 64, 64, 128, 1, 1, "", True),
        # the decode step of a busy server: every state is read and written
        heads("heads-step-96", "bf16", 80, 64, 128, 1, 96, "", True),
        # a trace replay in 32 bits, narrow odd heads with the gate in the scan
        heads("heads-replay", "fp32", 20, 40, 64, 2, 3, "300,77", True, gate=True),
        # a prompt through a mixer whose channels have rates of their own
        channels("channels-prompt-2048", "bf16", 8192, 16, 0, "2048", False),
        # several short prompts behind running requests
        channels("channels-mixed", "fp16", 2560, 16, 16, "200,350,17,128", True),
        # a decode step of the same mixers
        channels("channels-step-64", "bf16", 8192, 16, 64, "", True),
        # rows of a full token budget, eight groups, gate in front of the norm
        norm("norm-8192", "bf16", 8192, 8192, 8, False, False),
        # a decode step, one group as wide as the row, the gate behind a centred norm
        norm("norm-step-48", "fp16", 48, 4096, 1, True, True),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _step(rng, tokens: int) -> tuple[int, str]:
    """Single tokens and portions of a step of at most about ``tokens`` tokens."""
    kind = rng.choice(["prompts", "mixed", "step"])
    decodes = 0 if kind == "prompts" else _spread(rng, 1, 96)
    lens, left = [], 0 if kind == "step" else _spread(rng, 2, tokens)
    while left > 0 and len(lens) < 12:
        lens.append(_spread(rng, 1, left))
        left -= lens[-1]
    return decodes, ",".join(map(str, lens))


def draw(rng) -> dict:
    op = rng.choice(["conv", "heads", "channels", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        groups = rng.choice([1, 2, 4, 8])
        return dict(op="norm", dtype=dtype, rows=_spread(rng, 1, 4096), channels=groups * _spread(rng, 16, 8192 // groups),
                    groups=groups, after=rng.random() < 0.5, center=rng.random() < 0.5)
    started = rng.random() < 0.7
    if op == "conv":
        decodes, lens = _step(rng, 4096)
        return dict(op="conv", dtype=dtype, channels=_spread(rng, 64, 10240), taps=rng.choice([2, 3, 4, 4, 4]),
                    decodes=decodes, lens=lens, started=started)
    decodes, lens = _step(rng, 2048)
    if op == "channels":
        return dict(op="scan", form="channels", dtype=dtype, heads=_spread(rng, 64, 4096), width=1,
                    states=rng.choice([8, 16, 16, 16, 24]), groups=1, decodes=decodes, lens=lens, started=started,
                    gate=rng.random() < 0.7)
    groups = rng.choice([1, 1, 2, 8])
    return dict(op="scan", form="heads", dtype=dtype, heads=groups * _spread(rng, 1, 64 // groups),
                width=rng.choice([64, 64, 64, 128, 32, 40]) if dtype != "fp32" else rng.choice([64, 40, 33]),
                states=rng.choice([128, 128, 64, 16, 100]), groups=groups, decodes=decodes, lens=lens, started=started,
                gate=rng.random() < 0.3)


def _lens(case) -> list[int]:
    return [1] * case["decodes"] + [int(n) for n in case["lens"].split(",") if n]


def _starts(case) -> list[int]:
    """Position of each portion's first token: single tokens continue, of the prompts every second one where
    the case has started requests."""
    return [40 + 7 * r if r < case["decodes"] or case["started"] and (r - case["decodes"]) % 2 else 0
            for r in range(len(_lens(case)))]


def work(case) -> dict:
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["channels"]
        return {"bytes": 3 * n * e + 4 * case["channels"], "flops": 10 * n}
    lens, T = _lens(case), sum(_lens(case))
    kept = sum(s > 0 for s in _starts(case))
    if case["op"] == "conv":
        n, ring = T * case["channels"], case["channels"] * (case["taps"] - 1) * e
        return {"bytes": 2 * n * e + ring * (kept + len(lens)), "flops": (2 * case["taps"] + 4) * n}
    H, P, N = case["heads"], case["width"], case["states"]
    state = 4 * H * P * N
    row = (2 + case["gate"]) * H * P + H + 2 * case["groups"] * N
    return {"bytes": T * row * e + state * (kept + len(lens)), "flops": 5 * T * H * P * N}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev, dt_ = "cuda", TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    uni = lambda *s: torch.rand(*s, device=dev, generator=gen)  # noqa: E731
    s = types.SimpleNamespace(case=case)
    if case["op"] == "norm":
        T, C = case["rows"], case["channels"]
        s.x, s.z = rnd(T, C).to(dt_), rnd(T, C).to(dt_)
        s.weight, s.bias = 1 + 0.1 * rnd(C), 0.1 * rnd(C) if case["center"] else None
        s.out = torch.empty_like(s.x)
        return s
    lens, starts = _lens(case), _starts(case)
    T, R, nd = sum(lens), len(lens), case["decodes"]
    ends = torch.tensor(lens).cumsum(0)
    s.md = types.SimpleNamespace(
        positions=torch.cat([torch.arange(p, p + n) for p, n in zip(starts, lens)]).to(dev),
        state_slots=torch.randperm(R, generator=torch.Generator().manual_seed(seed)).int().to(dev),
        num_decode_tokens=nd,
        cu_q_prefill=(torch.tensor([0] + [int(e) - nd for e in ends[nd:]], dtype=torch.int32, device=dev)
                      if R > nd else None))
    s.write = s.md.state_slots + R
    # which request and which token of it a row is
    s.req = torch.repeat_interleave(torch.arange(R), torch.tensor(lens)).to(dev)
    s.first = torch.repeat_interleave(ends - torch.tensor(lens), torch.tensor(lens)).to(dev)
    s.ends, s.fresh = ends.to(dev), torch.tensor([p == 0 for p in starts], device=dev)
    if case["op"] == "conv":
        C, back = case["channels"], case["taps"] - 1
        s.x = rnd(T, C).to(dt_)
        s.weight, s.bias = rnd(back + 1, C) / math.sqrt(back + 1), 0.1 * rnd(C)
        s.ring = rnd(2 * R, back, C).to(dt_)
        s.ring[R:] = 0
        s.out = torch.empty_like(s.x)
        return s
    H, P, N, G = case["heads"], case["width"], case["states"], case["groups"]
    # x, B and C are parts of one convolved row, as the convolution leaves them
    pad = -(H * P) % 8
    row = torch.nn.functional.silu(rnd(T, H * P + pad + 2 * G * N)).to(dt_)
    s.x, s.b, s.c = row[:, :H * P], row[:, H * P + pad:H * P + pad + G * N], row[:, H * P + pad + G * N:]
    s.dt = rnd(T, H).to(dt_)
    step = torch.exp(math.log(1e-3) + uni(H) * math.log(1e2))     # step sizes from 1e-3 to 1e-1
    s.dt_bias = step + torch.log(-torch.expm1(-step))
    if case["form"] == "channels":
        s.a_log = torch.log(torch.arange(1, N + 1, device=dev, dtype=torch.float32)).repeat(H, 1)
    else:
        s.a_log = torch.log(1 + 15 * uni(H))
    s.d, s.z = 1 + 0.1 * rnd(H), rnd(T, H * P).to(dt_) if case["gate"] else None
    s.state = torch.zeros(2 * R, H, *([P] if case["form"] == "heads" else []), N, device=dev)
    s.state[:R] = 0.5 * rnd(*s.state[:R].shape)
    s.out = torch.empty(T, H * P, dtype=dt_, device=dev)
    # the plain scan goes by chunks: their rows (T: behind the end) and the first chunk of every request
    chunks = [(r, i) for r, n in enumerate(lens) for i in range(0, n, CHUNK)]
    at = [int(ends[r]) - lens[r] + i for r, i in chunks]
    stop = [int(ends[r]) for r, _ in chunks]
    rows = torch.tensor(at)[:, None] + torch.arange(CHUNK)
    s.rows = torch.where(rows < torch.tensor(stop)[:, None], rows, T).to(dev)
    s.chunk_req = torch.tensor([r for r, _ in chunks]).to(dev)
    s.chunk_first = torch.tensor([i == 0 for _, i in chunks]).to(dev)
    s.chunk_last = torch.tensor([i + CHUNK >= lens[r] for r, i in chunks]).nonzero()[:, 0].to(dev)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _silu(x):
    return x / (1 + torch.exp(-x))


def _linear(a, u):
    """h of h_t = a_t h_(t-1) + u_t along the first axis, distances doubled."""
    k = 1
    while k < u.shape[0]:
        u = torch.cat([u[:k], u[k:] + a[k:] * u[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return u


def _conv(s):
    n = s.weight.shape[0]
    back = n - 1
    T, t = s.x.shape[0], torch.arange(s.x.shape[0], device=s.x.device)
    src = t[:, None] + torch.arange(n, device=t.device) - back              # row of every tap
    pos = s.md.positions[:, None] + torch.arange(n, device=t.device) - back
    old = s.ring[s.md.state_slots[s.req].long()[:, None], pos % back].float()
    now = s.x.float()[src.clamp(min=0)]
    here = (src >= s.first[:, None])[..., None]
    rows = torch.where(here, now, torch.where((pos >= 0)[..., None], old, 0.0))
    s.out.copy_(_silu((rows * s.weight).sum(1) + s.bias))
    # rings: the old rows, then those that this step brings
    slots, write = s.md.state_slots.long(), s.write.long()
    keep = ~s.fresh
    s.ring[write[keep]] = s.ring[slots[keep]]
    last = (t >= s.ends[s.req] - back).nonzero()[:, 0]
    s.ring[write[s.req[last]], s.md.positions[last] % back] = s.x[last]
    return s.out, s.ring[s.ring.shape[0] // 2:]


def _steps(s):
    """Step sizes and rates."""
    z = s.dt.float() + s.dt_bias
    return torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())), -torch.exp(s.a_log)


def _finish(s, y):
    """Skip and gate, rounded once."""
    y = y + s.x.float() * s.d.repeat_interleave(s.x.shape[1] // s.d.shape[0])
    s.out.copy_(y if s.z is None else y * _silu(s.z.float()))
    return s.out, s.state[s.state.shape[0] // 2:]


def _channels(s):
    dt, A = _steps(s)
    a = torch.exp(dt[..., None] * A)                                        # [T, D, N]
    u = (dt * s.x.float())[..., None] * s.b.float()[:, None]
    head = (s.ends - torch.bincount(s.req))[~s.fresh]
    u[head] += a[head] * s.state[s.md.state_slots.long()[~s.fresh]]
    a[s.ends - torch.bincount(s.req)] = 0
    h = _linear(a, u)
    s.state[s.write.long()] = h[s.ends - 1]
    return _finish(s, (h * s.c.float()[:, None]).sum(-1))


def _heads(s):
    H, G = s.a_log.shape[0], s.case["groups"]
    P, N, T = s.case["width"], s.case["states"], s.x.shape[0]
    dt, A = _steps(s)
    h0 = s.state[s.md.state_slots.long()] * (~s.fresh)[:, None, None, None]
    if s.rows.shape[0] == T:                                                # single tokens
        x, b, c = s.x.float().view(T, H, P), s.b.float().view(T, G, N), s.c.float().view(T, G, N)
        b, c = (t.repeat_interleave(H // G, 1)[:, :, None] for t in (b, c))
        h = torch.exp(dt * A)[..., None, None] * h0 + (dt[..., None] * x)[..., None] * b
        s.state[s.write.long()] = h
        return _finish(s, (h * c).sum(-1).view(T, H * P))
    # rows behind a portion's end: zeros, which leave a state as it is
    pick = lambda t: torch.cat([t, t.new_zeros(1, t.shape[1])])[s.rows]  # noqa: E731
    x, dt = pick(s.x.float()).unflatten(-1, (H, P)), pick(dt)               # [K, Q, H, P], [K, Q, H]
    b, c = (pick(t.float()).unflatten(-1, (G, N)) for t in (s.b, s.c))
    far = torch.cumsum((dt * A).double(), 1)                                # log decay from a chunk's start
    gap = far[:, :, None] - far[:, None]                                    # [K, Q, Q, H]: from token j to token i
    seen = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=x.device).tril()[..., None]
    m = torch.where(seen, torch.exp(torch.where(seen, gap, 0.0)), 0.0).float() * dt[:, None]
    score = c.permute(0, 2, 1, 3) @ b.permute(0, 2, 3, 1)                   # [K, G, Q, Q]
    m = m.permute(0, 3, 1, 2) * score.repeat_interleave(H // G, 1)
    y = m @ x.permute(0, 2, 1, 3)                                           # [K, H, Q, P]
    # what a chunk adds to the state, and the state in front of every chunk
    left = (torch.exp(far[:, -1:] - far).float() * dt)[..., None] * x       # [K, Q, H, P]
    b, c = (t.repeat_interleave(H // G, 2).permute(0, 2, 1, 3) for t in (b, c))
    u = left.permute(0, 2, 3, 1) @ b                                        # [K, H, P, N]
    a = torch.exp(far[:, -1]).float()[..., None, None]
    start = torch.where(s.chunk_first[:, None, None, None], h0[s.chunk_req], 0.0)
    h = _linear(torch.where(s.chunk_first[:, None, None, None], 0.0, a), u + a * start)
    s.state[s.write.long()] = h[s.chunk_last]
    before = torch.where(s.chunk_first[:, None, None, None], start, torch.cat([h[:1], h[:-1]]))
    y = y + torch.exp(far).float().permute(0, 2, 1)[..., None] * (c @ before.transpose(-1, -2))
    rows = torch.empty(T + 1, H * P, device=x.device)
    rows[s.rows.flatten()] = y.permute(0, 2, 1, 3).reshape(-1, H * P)
    return _finish(s, rows[:T])


def _norm(s):
    G, gate = s.case["groups"], _silu(s.z.float())
    v = (s.x.float() if s.case["after"] else s.x.float() * gate).unflatten(-1, (G, -1))
    if s.case["center"]:
        v = v - v.mean(-1, keepdim=True)
    v = (v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)).flatten(-2) * s.weight
    if s.bias is not None:
        v = v + s.bias
    s.out.copy_(v * gate if s.case["after"] else v)
    return s.out


def run(s):
    case = s.case
    if own:
        from vllm_gcu_b200.ops import cuda as ops
        if case["op"] == "norm":
            return ops.group_norm_gate(s.x, s.z, s.weight, case["groups"], EPS, bias=s.bias, center=case["center"],
                                       gate_after=case["after"], out=s.out)
        if case["op"] == "conv":
            ops.causal_conv(s.x, s.weight, s.bias, s.md, s.ring, write_slots=s.write, out=s.out)
            return s.out, s.ring[s.ring.shape[0] // 2:]
        ops.selective_scan(s.x, s.dt, s.b, s.c, s.a_log, case["groups"], s.md, s.state, d=s.d, dt_bias=s.dt_bias,
                           z=s.z, write_slots=s.write, out=s.out)
        return s.out, s.state[s.state.shape[0] // 2:]
    if case["op"] == "norm":
        return _norm(s)
    if case["op"] == "conv":
        return _conv(s)
    return _channels(s) if case["form"] == "channels" else _heads(s)


# ---------------------------------------------------------------------------
# the definitions, token by token in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    if case["op"] == "norm":
        x, gate = wide(s.x), wide(s.z) * torch.sigmoid(wide(s.z))
        out = torch.empty_like(x)
        for part in torch.arange(case["channels"], device=x.device).chunk(case["groups"]):
            v = x[:, part] if case["after"] else x[:, part] * gate[:, part]
            mean = v.mean(1, keepdim=True) if case["center"] else 0.0
            r = (v - mean) * torch.rsqrt(((v - mean) ** 2).mean(1, keepdim=True) + EPS) * wide(s.weight)[part]
            r = r if s.bias is None else r + wide(s.bias)[part]
            out[:, part] = r * gate[:, part] if case["after"] else r
        return out
    lens, starts = _lens(case), _starts(case)
    R, lo = len(lens), 0
    slots = s.md.state_slots.tolist()
    if case["op"] == "conv":
        back, x, out, ring = case["taps"] - 1, wide(s.x), torch.empty_like(wide(s.x)), wide(s.ring)
        for r, (n, p) in enumerate(zip(lens, starts)):
            old = [ring[slots[r], q % back] if q >= 0 else torch.zeros_like(x[0]) for q in range(p - back, p)]
            seq = torch.cat([torch.stack(old), x[lo:lo + n]])
            c = wide(s.bias) + sum(wide(s.weight)[j] * seq[j:j + n] for j in range(back + 1))
            out[lo:lo + n] = c * torch.sigmoid(c)
            if p:
                ring[R + slots[r]] = ring[slots[r]]
            for i in range(max(0, n - back), n):
                ring[R + slots[r], (p + i) % back] = x[lo + i]
            lo += n
        return out, ring[R:]
    H, P, N, G = case["heads"], case["width"], case["states"], case["groups"]
    x = wide(s.x).view(-1, H, P)
    b, c = (wide(t).view(-1, G, N) for t in (s.b, s.c))
    dt = torch.nn.functional.softplus(wide(s.dt) + wide(s.dt_bias))
    A = -torch.exp(wide(s.a_log)).view(H, -1)
    y, out_state = torch.empty_like(x), torch.zeros(R, H, P, N, dtype=torch.float64, device=x.device)
    for r, (n, p) in enumerate(zip(lens, starts)):
        h = torch.zeros(H, P, N, dtype=torch.float64, device=x.device)
        if p:
            h = wide(s.state[slots[r]]).view(H, P, N)
        for t in range(lo, lo + n):
            bt, ct = (v[t].repeat_interleave(H // G, 0)[:, None] for v in (b, c))
            h = h * torch.exp(dt[t, :, None] * A)[:, None] + (dt[t, :, None] * x[t])[..., None] * bt
            y[t] = (h * ct).sum(-1)
        out_state[slots[r]] = h
        lo += n
    y = (y + wide(s.d)[:, None] * x).flatten(1)
    if s.z is not None:
        y = y * wide(s.z) * torch.sigmoid(wide(s.z))
    return y, out_state.view(s.state[R:].shape)
