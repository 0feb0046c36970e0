"""The operators of a key/value cache held in 8 bits with a scale for each block of tokens and head, as cases that can
be timed and checked.

A block (page) of such a cache holds the keys and values of ``block`` tokens of one request as 8-bit codes, fp8 e4m3
or int8; what a code stands for is the code times the scale of its block and head, a power of two.

* ``write``   a step's keys and values go into their blocks.  A block that takes its first token starts with the
              smallest scale that holds the new numbers; a block that goes on keeps its scale or, where a new number does not
              fit, takes a larger one and its earlier codes are rounded to that
* ``decode``  attention of one token of each request over its blocks, all keys or the last ``window`` ones and the
              ``first`` ones of the request
* ``prefill`` the same for portions of prompts, and for a few tokens of each request (checked drafts)
* ``pages``   requests are forked into answers that share their full blocks, the last one, partly filled, is copied
              (``fork``), and blocks are copied in pairs (``copy``); the layers of a cache and its scales at once
"""
from __future__ import annotations

import math
import types

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
         "fp8": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"fp8": 448.0, "int8": 127.0}
LOW, HIGH = -100, 121             # exponents of scales


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    def write(name, codes, dtype, heads, width, block, decodes, lens):
        return dict(name=name, op="write", codes=codes, dtype=dtype, kv_heads=heads, width=width, block=block,
                    decodes=decodes, lens=lens)

    def decode(name, codes, dtype, heads, group, width, block, lens, window=0, first=0):
        return dict(name=name, op="decode", codes=codes, dtype=dtype, kv_heads=heads, group=group, width=width,
                    block=block, lens=lens, window=window, first=first)

    def prefill(name, codes, dtype, heads, group, width, block, lens, before, window=0, first=0):
        return dict(name=name, op="prefill", codes=codes, dtype=dtype, kv_heads=heads, group=group, width=width,
                    block=block, lens=lens, before=before, window=window, first=first)

    def pages(name, op, codes, layers, heads, width, block, requests, answers, blocks):
        return dict(name=name, op=op, codes=codes, layers=layers, kv_heads=heads, width=width, block=block,
                    requests=requests, answers=answers, blocks=blocks)

    return [
        # a full token budget of prompts, the last ones behind what earlier steps left in their blocks
        write("write-prompts", "fp8", "bf16", 8, 128, 16, 0, "2048,2048,1531,997,800,513,250,5"),
        # one user waits for each token of an answer
        write("write-step-1", "fp8", "bf16", 8, 128, 16, 1, ""),
        # the step of a busy server with a few short prompts, heads of 64, blocks of 32
        write("write-step-192", "int8", "fp16", 4, 64, 32, 192, "33,70,1,15"),
        # one user's answer, 32 query heads over 8 key heads
        decode("decode-1", "fp8", "bf16", 8, 4, 128, 16, "1501"),
        # the decode step of a busy server: 256 answers behind prompts of 1024 tokens
        decode("decode-256", "fp8", "bf16", 8, 4, 128, 16, ",".join(str(1024 + (37 * i) % 256) for i in range(256))),
        # a few long documents, seven query heads a key head
        decode("decode-long", "int8", "fp16", 4, 7, 128, 16, "65536,120001,31007,98765"),
        # endless answers: each sees its last 1024 tokens and its first four
        decode("decode-window", "fp8", "bf16", 8, 4, 128, 64, ",".join(str(4000 + 97 * i) for i in range(64)), 1024, 4),
        # a full token budget of prompts
        prefill("prefill-prompts", "fp8", "bf16", 8, 4, 128, 16, "2048,1500,777,1024,130,33", "0,0,512,0,0,1024"),
        # a portion of a long document that sees its last 4096 tokens and its first 64
        prefill("prefill-window", "fp8", "bf16", 8, 4, 128, 16, "2048", "14336", 4096, 64),
        # drafts of four tokens are checked behind each of 32 answers
        prefill("prefill-checked", "int8", "fp16", 4, 7, 128, 16, ",".join(["4"] * 32),
                ",".join(str(1500 + 61 * i) for i in range(32))),
        # every beam of 16 requests goes on from one of its request's beams
        pages("fork-64", "fork", "fp8", 32, 4, 128, 16, 16, 64, 8),
        # copies of whole blocks in one layer of a cache, large blocks
        pages("copy-96", "copy", "int8", 1, 8, 128, 64, 96, 96, 1),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, total: int, count: int) -> list[int]:
    """``count`` lengths of together about ``total``, most of them near the mean."""
    parts = [math.exp(rng.gauss(0.0, 0.7)) for _ in range(count)]
    return [max(1, round(total * p / sum(parts))) for p in parts]


def draw(rng) -> dict:
    op = rng.choice(["write", "decode", "prefill", "fork", "copy"])
    case = dict(op=op, codes=rng.choice(["fp8", "fp8", "int8"]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                kv_heads=rng.choice([1, 2, 3, 4, 8]), width=rng.choice([128, 128, 128, 64]),
                block=rng.choice([16, 16, 32, 64]))
    join = lambda v: ",".join(map(str, v))  # noqa: E731
    if op in ("fork", "copy"):
        del case["dtype"]
        requests = _spread(rng, 1, 24)
        return dict(case, layers=_spread(rng, 1, 8), requests=requests, answers=requests * rng.choice([1, 2, 4]),
                    blocks=_spread(rng, 1, 64 // case["block"] + 1))
    if op == "write":
        kind = rng.choice(["prompts", "mixed", "step"])
        return dict(case, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    decodes=0 if kind == "prompts" else _spread(rng, 1, 192),
                    lens="" if kind == "step" else join(_lengths(rng, _spread(rng, 12, 7800), rng.randint(1, 12))))
    case["group"] = rng.choice([g for g in (1, 2, 4, 4, 5, 7, 8) if g * case["kv_heads"] <= 32])
    case["window"], case["first"] = rng.choice([(0, 0), (0, 0), (_spread(rng, 1, 4096), 0),
                                                (_spread(rng, 16, 4096), _spread(rng, 1, 200))])
    if op == "decode":
        return dict(case, lens=join(_lengths(rng, _spread(rng, 64, 262144), _spread(rng, 1, 128))))
    if rng.random() < 0.3:                                     # a few tokens of each request
        n = _spread(rng, 1, 64)
        lens, before = [rng.randint(2, 6) for _ in range(n)], [_spread(rng, 1, 2048) for _ in range(n)]
    else:
        lens = _lengths(rng, _spread(rng, 16, 1500), rng.randint(1, 6))
        before = [rng.choice([0, 0, _spread(rng, 1, 4096)]) for _ in lens]
    return dict(case, lens=join(lens), before=join(before))


def _ints(text: str) -> list[int]:
    return [int(n) for n in text.split(",") if n]


def _lens(case) -> tuple[list[int], list[int]]:
    """Tokens of a step for each request, and its tokens in front of them."""
    if case["op"] == "write":
        nd, lens = case["decodes"], _ints(case["lens"])
        # running requests stand anywhere in their blocks, of the prompts every second one goes on
        return [1] * nd + lens, [40 + 7 * r for r in range(nd)] + [(21 + 9 * r) * (r % 2) for r in range(len(lens))]
    if case["op"] == "decode":
        return [1] * len(_ints(case["lens"])), [n - 1 for n in _ints(case["lens"])]
    return _ints(case["lens"]), _ints(case["before"])


def _held(case) -> list[int]:
    """Tokens of each request that is forked: its blocks are full but the last one."""
    bs = case["block"]
    return [case["blocks"] * bs - (7 * r) % bs for r in range(case["requests"])]


def work(case) -> dict:
    H, D, bs = case["kv_heads"], case["width"], case["block"]
    if case["op"] == "copy":
        n = case["requests"] * case["layers"] * 2 * H
        return {"bytes": 2 * n * (bs * D + 4), "flops": 0}
    if case["op"] == "fork":
        held, row = _held(case), 2 * case["layers"] * H
        moved = sum(held[n % case["requests"]] % bs * D + 4 * (held[n % case["requests"]] % bs > 0)
                    for n in range(case["answers"])
                    if n >= case["requests"])
        return {"bytes": 2 * moved * row + 4 * (case["requests"] + case["answers"]) * (case["blocks"] + 1), "flops": 0}
    e = 4 if case["dtype"] == "fp32" else 2
    lens, before = _lens(case)
    if case["op"] == "write":
        blocks = sum((b + n - 1) // bs - b // bs + 1 for n, b in zip(lens, before))
        return {"bytes": sum(lens) * 2 * H * D * (e + 1) + blocks * 2 * H * 4, "flops": 3 * sum(lens) * 2 * H * D}
    w, f = case["window"] or 1 << 40, case["first"]
    seen, pairs, blocks = 0, 0, 0
    for n, b in zip(lens, before):
        lo = max(0, b + 1 - w)                                  # first key of the window of the first token
        keys = b + n - lo + min(f, lo)
        seen, blocks = seen + keys, blocks + -(-keys // bs)
        pairs += sum(min(p + 1, w) + min(f, max(0, p + 1 - w)) for p in range(b, b + n))
    Hq = H * case["group"]
    return {"bytes": seen * 2 * H * D + blocks * 2 * H * 4 + 2 * e * sum(lens) * Hq * D, "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def _power(e: torch.Tensor) -> torch.Tensor:
    """2 ** e in 32 bits for whole numbers e of normal results."""
    return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _scale_for(top: torch.Tensor, codes: str) -> torch.Tensor:
    """The smallest power of two, in the limits, whose largest code reaches ``top``."""
    m, e = torch.frexp(top)                                     # top = m 2^e, m in [0.5, 1)
    m_top, e_top = math.frexp(LARGEST[codes])
    e = e - e_top + (m > m_top).int()
    return _power(torch.where(top > 0, e, LOW).clamp(LOW, HIGH))


def _codes(x: torch.Tensor, codes: str) -> torch.Tensor:
    """Numbers of the codes' range, rounded to the nearest code, ties to even."""
    top = LARGEST[codes]
    x = torch.where(torch.isnan(x), 0.0, x).clamp(-top, top)
    return torch.round(x).to(torch.int8) if codes == "int8" else x.to(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    s = types.SimpleNamespace(case=case)
    H, D, bs, codes = case["kv_heads"], case["width"], case["block"], case["codes"]

    def cache(layers, nb):
        """Full blocks of numbers whose size differs between blocks and heads: codes, scales."""
        x = torch.empty(layers * 2, nb, bs, H, D, dtype=TYPES[codes], device=dev)
        scale = torch.empty(layers * 2, nb, H, device=dev)
        for plane in range(layers * 2):
            v = rnd(nb, bs, H, D) * torch.exp(0.5 * rnd(nb, 1, H, 1))
            scale[plane] = _scale_for(v.abs().amax((1, 3)), codes)
            x[plane] = _codes(v / scale[plane][:, None, :, None], codes)
        return x.view(layers, 2, nb, bs, H, D), scale.view(layers, 2, nb, H)

    if case["op"] in ("fork", "copy"):
        R, N, M = case["requests"], case["answers"], case["blocks"]
        nb = R * M + N + 3
        s.cache, s.scale = cache(case["layers"], nb)
        order = torch.randperm(nb, generator=host)
        s.tables = torch.zeros(R, M + 1, dtype=torch.int32)
        s.tables[:, :M] = order[:R * M].view(R, M)
        s.tables = s.tables.to(dev)
        s.lens = torch.tensor(_held(case), dtype=torch.int32, device=dev)
        s.parents = (torch.arange(N, dtype=torch.int32) % R).to(dev)
        # a request's first answer goes on in its blocks
        s.fresh = torch.where(torch.arange(N) < R, -1, order[R * M:R * M + N]).int().to(dev)
        s.pairs = torch.stack([order[:R], order[R * M:R * M + R]], 1).to(dev) if case["op"] == "copy" else None
        return s
    lens, before = _lens(case)
    T, R, e = sum(lens), len(lens), TYPES[case["dtype"]]
    total = [n + b for n, b in zip(lens, before)]
    need = [-(-n // bs) for n in total]
    nb = sum(need) + 5
    s.cache, s.scale = (t[0] for t in cache(1, nb))
    order = torch.randperm(nb, generator=host).int()
    s.tables = torch.zeros(R, max(need), dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        s.tables[r, :n] = order[at:at + n]
        at += n
    s.seq_lens = torch.tensor(total, dtype=torch.int32, device=dev)
    # which request a row belongs to, and its position
    req = torch.repeat_interleave(torch.arange(R), torch.tensor(lens))
    first = torch.tensor(lens).cumsum(0) - torch.tensor(lens)
    pos = torch.arange(T) - first[req] + torch.tensor(before)[req]
    s.slots = (s.tables[req, pos // bs].long() * bs + pos % bs).to(dev)
    s.tables = s.tables.to(dev)
    s.req, s.pos = req.to(dev), pos.to(dev)
    if case["op"] == "write":
        size = torch.exp(0.5 * rnd(T, H, 1))
        row = torch.cat([(rnd(T, H, D) * size).flatten(1), (rnd(T, H, D) * size).flatten(1)], 1).to(e)
        s.k, s.v = row[:, :H * D], row[:, H * D:]               # parts of a projection's row
        return s
    Hq = H * case["group"]
    s.q = rnd(T, Hq * D).to(e).view(T, Hq, D)
    s.out = torch.empty_like(s.q)
    s.lens, s.total = lens, total
    s.cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    s.row = (torch.arange(T) - first[req]).to(dev)              # row in its request
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _write(s):
    case, nb, bs = s.case, s.cache.shape[1], s.case["block"]
    H, D = case["kv_heads"], case["width"]
    x = torch.stack([s.k.float().view(-1, H, D), s.v.float().view(-1, H, D)])
    page, off = s.slots // bs, s.slots % bs
    row = torch.full((nb, bs), -1, device=off.device)           # which row a place takes
    row[page, off] = torch.arange(len(off), device=off.device)
    top = torch.where((row >= 0)[..., None], x.abs().amax(-1)[:, row], 0.0).amax(2)
    first = torch.where(row >= 0, torch.arange(bs, device=off.device), bs).amin(1)
    old = torch.where((first == 0)[:, None], 0.0, s.scale)      # a block that starts anew has no earlier tokens
    scale = torch.where((first < bs)[:, None], torch.maximum(old, _scale_for(top, case["codes"])), s.scale)
    # earlier tokens of blocks whose scale grew
    ratio = torch.where(scale > 0, s.scale / scale, 0.0)[:, :, None, :, None]
    again = _codes(s.cache.float() * ratio, case["codes"])
    held = (torch.arange(bs, device=off.device) < first[:, None])[None, :, :, None, None] & (first < bs)[:, None, None, None]
    s.cache.copy_(torch.where(held, again.float(), s.cache.float()).to(s.cache.dtype))
    new = _codes(x / scale[:, page][..., None], case["codes"])
    s.cache.view(torch.uint8)[:, page, off] = new.view(torch.uint8)
    s.scale.copy_(scale)
    return s.cache[0], s.cache[1], s.scale[0], s.scale[1]


def _seen(keys, pos, case):
    """Which keys a query at ``pos`` sees."""
    near = keys > pos - case["window"] if case["window"] else keys >= 0
    return (keys <= pos) & (near | (keys < case["first"]))


def _attention(s):
    case, R = s.case, len(s.lens)
    H, G, D, bs = case["kv_heads"], case["group"], case["width"], case["block"]
    n = max(s.lens)
    S = s.tables.shape[1] * bs
    pages = s.tables.long()
    k, v = (c[pages].float() * f[pages][:, :, None, :, None] for c, f in zip(s.cache, s.scale))
    k, v = (t.view(R, S, H, D).transpose(1, 2) for t in (k, v))             # [R, H, S, D]
    q = torch.zeros(R, n, H, G, D, device=k.device)
    q[s.req, s.row] = s.q.float().view(-1, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(R, H, G * n, D)
    pos = torch.full((R, n), -1, device=k.device)
    pos[s.req, s.row] = s.pos
    seen = _seen(torch.arange(S, device=k.device), pos[..., None], case)     # [R, n, S]
    score = (q @ k.transpose(2, 3)).view(R, H, G, n, S) * D ** -0.5
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.view(R, H, G * n, S) @ v).view(R, H, G, n, D) / torch.where(total > 0, total, 1.0)
    s.out.copy_(o.permute(0, 3, 1, 2, 4)[s.req, s.row].reshape(s.out.shape))
    return s.out


def _fork(s):
    bs = s.case["block"]
    rows = s.tables[s.parents.long()]
    lens = s.lens.long()[s.parents.long()]
    last, used, new = lens // bs, lens % bs, s.fresh >= 0
    at = torch.arange(len(lens), device=rows.device)
    src = rows[at, last].long()
    rows[at[new], last[new]] = s.fresh[new]
    move = new & (used > 0)
    src, dst, used = src[move], s.fresh.long()[move], used[move]
    keep = (torch.arange(bs, device=src.device) < used[:, None])[None, None, :, :, None, None]
    raw = s.cache.view(torch.uint8)
    raw[:, :, dst] = torch.where(keep, raw[:, :, src], raw[:, :, dst])
    s.scale[:, :, dst] = s.scale[:, :, src]
    return rows, s.cache, s.scale


def _copy(s):
    src, dst = s.pairs.unbind(1)
    raw = s.cache.view(torch.uint8)
    raw[:, :, dst] = raw[:, :, src]
    s.scale[:, :, dst] = s.scale[:, :, src]
    return s.cache, s.scale


def run(s):
    case = s.case
    if own:
        from vllm_gcu_b200.ops import cuda as ops
        if case["op"] in ("fork", "copy"):
            if not hasattr(s, "pages"):
                s.pages = ops.CachePages([*s.cache.flatten(0, 1), *s.scale.flatten(0, 1)], case["block"])
            if case["op"] == "fork":
                return s.pages.fork(s.tables, s.lens, s.parents, s.fresh), s.cache, s.scale
            s.pages.copy(s.pairs)
            return s.cache, s.scale
        held = (s.cache[0], s.cache[1], s.scale[0], s.scale[1])
        if case["op"] == "write":
            ops.block_scaled_cache(s.k, s.v, *held, s.slots)
            return held
        if case["op"] == "decode":
            return ops.block_scaled_decode(s.q, *held, s.tables, s.seq_lens, case["width"] ** -0.5, out=s.out,
                                           max_seq_len=max(s.total), window=case["window"], first=case["first"])
        return ops.block_scaled_prefill(s.q, *held, s.tables, s.cu, s.seq_lens, case["width"] ** -0.5, s.lens, s.total,
                                        out=s.out, window=case["window"], first=case["first"])
    return {"write": _write, "decode": _attention, "prefill": _attention, "fork": _fork, "copy": _copy}[case["op"]](s)


# ---------------------------------------------------------------------------
# the definitions, block by block and token by token, in 64 bits
# ---------------------------------------------------------------------------
def _nearest(x, codes):
    """The code nearest to x, ties to the even one."""
    if codes == "int8":
        return torch.round(x).clamp(-127, 127)
    # neighbours of a number in [2^e, 2^(e + 1)) are 2^(e - 3) apart, below 2^-6 all 2^-9
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x)[1].clamp(min=-5) - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)



def exact(case, seed):
    s = prepare(case, seed)
    bs, codes = case["block"], case["codes"]
    if case["op"] in ("fork", "copy"):
        cache, scale = s.cache.double(), s.scale.double()
        if case["op"] == "copy":
            for a, b in s.pairs.tolist():
                cache[:, :, b], scale[:, :, b] = cache[:, :, a], scale[:, :, a]
            return cache, scale
        rows = []
        for p, f in zip(s.parents.tolist(), s.fresh.tolist()):
            row, n = s.tables[p].clone(), int(s.lens[p])
            if f >= 0:
                a = int(row[n // bs])
                row[n // bs] = f
                if n % bs:
                    cache[:, :, f, :n % bs], scale[:, :, f] = cache[:, :, a, :n % bs], scale[:, :, a]
            rows.append(row)
        return torch.stack(rows), cache, scale
    H, D = case["kv_heads"], case["width"]
    cache, scale = s.cache.double(), s.scale.double()
    lens, before = _lens(case)
    if case["op"] == "write":
        x, at = torch.stack([s.k.double().view(-1, H, D), s.v.double().view(-1, H, D)]), 0
        for r, (n, b) in enumerate(zip(lens, before)):
            for page in range(b // bs, (b + n - 1) // bs + 1):
                lo, hi = max(b, page * bs), min(b + n, page * bs + bs)
                blk, off, new = int(s.tables[r, page]), lo - page * bs, x[:, at + lo - b:at + hi - b]
                m, e = torch.frexp(new.abs().amax((1, 3)).clamp(min=2.0 ** -200) / LARGEST[codes])
                e = torch.where(m == 0.5, e - 1, e)
                f = torch.ldexp(torch.ones_like(m), e.clamp(LOW, HIGH))
                if off:
                    f = torch.maximum(f, scale[:, blk])
                    cache[:, blk, :off] = _nearest(cache[:, blk, :off] * (scale[:, blk] / f)[:, None, :, None], codes)
                cache[:, blk, off:off + hi - lo] = _nearest(new / f[:, None, :, None], codes)
                scale[:, blk] = f
            at += n
        return cache[0], cache[1], scale[0], scale[1]
    q, G, out, at = s.q.double(), case["group"], [], 0
    for r, (n, b) in enumerate(zip(lens, before)):
        pages = s.tables[r, :-(-(b + n) // bs)].long()
        k, v = ((c[pages] * f[pages][:, None, :, None]).flatten(0, 1)[:b + n] for c, f in zip(cache, scale))
        pos = torch.arange(b, b + n, device=q.device)[:, None]
        keys = torch.arange(b + n, device=q.device)
        hidden = keys > pos
        if case["window"]:
            hidden |= (keys <= pos - case["window"]) & (keys >= case["first"])
        o = torch.empty(n, H * G, D, dtype=torch.float64, device=q.device)
        for h in range(H * G):
            t = q[at:at + n, h] @ k[:, h // G].T / math.sqrt(D)
            o[:, h] = torch.softmax(t.masked_fill(hidden, -math.inf), -1) @ v[:, h // G]
        out.append(o)
        at += n
    return torch.cat(out)
