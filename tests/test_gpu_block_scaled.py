"""Operators of a cache in 8 bits with a scale for each block and head against their definitions in 64 bits."""
import math

import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200.ops import cuda as C
from vllm_gcu_b200.ops import ref

pytestmark = pytest.mark.gpu
CODES = [K.FP8, K.INT8]


@pytest.fixture(autouse=True)
def _clean_status():
    from vllm_gcu_b200.ops import _native
    yield
    assert _native.take_status()[0] == 0


def _same(a, b):
    return torch.equal(a.view(torch.uint8).cpu(), b.view(torch.uint8).cpu())


def _write_both(dev, cpu, k, v, slots):
    C.block_scaled_cache(k.cuda(), v.cuda(), *dev, slots.cuda())
    ref.block_scaled_cache(k, v, *cpu, slots)
    assert all(_same(a, b) for a, b in zip(dev, cpu))


@pytest.mark.parametrize("dtype", [K.BF16, K.F16, K.F32])
@pytest.mark.parametrize("codes,H,D,bs", [(K.FP8, 1, 64, 16), (K.FP8, 5, 128, 16), (K.FP8, 2, 256, 48),
                                          (K.INT8, 3, 64, 64), (K.INT8, 2, 128, 32), (K.INT8, 1, 256, 16)])
def test_writes_step_by_step(dtype, codes, H, D, bs):
    """Portions and single tokens of three requests over several steps, sizes that grow: the oracle's bits."""
    gen = torch.Generator().manual_seed(D + bs)
    nb = 3 * (-(-300 // bs)) + 1
    dev = [torch.zeros(nb, bs, H, D, dtype=codes).cuda() for _ in range(2)] + [torch.zeros(nb, H).cuda() for _ in range(2)]
    cpu = [t.cpu() for t in dev]
    tables = torch.randperm(nb - 1, generator=gen).view(3, -1)
    at = [0, 0, 0]
    for step, lens in enumerate([(7, 100, 1), (1, 1, 1), (20, 1, 3), (1, 1, 1), (0, 33, 60), (1, 2, 1)]):
        slots, rows = [], sum(lens)
        for r, n in enumerate(lens):
            pos = torch.arange(at[r], at[r] + n)
            slots.append(tables[r, pos // bs] * bs + pos % bs)
            at[r] += n
        size = torch.exp(torch.randn(rows, H, 1, generator=gen) + 0.3 * step)
        k, v = ((torch.randn(rows, H, D, generator=gen) * size).to(dtype).flatten(1) for _ in range(2))
        _write_both(dev, cpu, k, v, torch.cat(slots))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("rows", [1, 40, 700])
def test_writes_of_views_and_rows_that_go_nowhere(codes, rows):
    """Parts of a row at an odd pitch and address, padding behind and between requests."""
    gen = torch.Generator().manual_seed(rows)
    H, D, bs = 2, 64, 16
    nb = rows // bs + 4
    dev = [torch.zeros(nb, bs, H, D, dtype=codes).cuda() for _ in range(2)] + [torch.zeros(nb, H).cuda() for _ in range(2)]
    cpu = [t.cpu() for t in dev]
    slots = torch.arange(rows)
    slots[rows // 3:rows // 3 + 2] = -1                     # (what follows goes on in the same block)
    if rows > 2:
        slots = torch.where(slots >= 0, slots, -1)
        slots[rows // 3 + 2:] += bs                        # ... in another one
    wide = torch.randn(rows, 2 * H * D + 3, generator=gen).to(K.BF16)
    gpu = wide.cuda()
    C.block_scaled_cache(gpu[:, 1:1 + H * D], gpu[:, 1 + H * D:1 + 2 * H * D], *dev, slots.cuda())
    ref.block_scaled_cache(wide[:, 1:1 + H * D], wide[:, 1 + H * D:1 + 2 * H * D], *cpu, slots)
    assert all(_same(a, b) for a, b in zip(dev, cpu))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [K.BF16, K.F16, K.F32])
def test_writes_of_extremes(codes, dtype):
    """Zeros, infinities, NaN, the type's largest and smallest numbers, powers of two at the codes' ends."""
    H, D, bs, top = 2, 128, 16, 448.0 if codes == K.FP8 else 127.0
    info = torch.finfo(dtype)
    rows = torch.randn(40, H * D)
    rows[0:3] = 0
    rows[16:19] = 0
    rows[17, 3] = info.tiny
    rows[20, 5], rows[21, 6], rows[22, 7] = math.inf, -math.inf, math.nan
    rows[33, 8] = info.max
    rows[3] = 0
    rows[3, 0] = top * 2 ** -5
    rows[4:16] = 0
    rows[7, D] = -top
    rows = rows.to(dtype)
    dev = [torch.zeros(4, bs, H, D, dtype=codes).cuda() for _ in range(2)] + [torch.zeros(4, H).cuda() for _ in range(2)]
    cpu = [t.cpu() for t in dev]
    _write_both(dev, cpu, rows, rows.flip(0), torch.arange(40))
    # a block that goes on behind what was never written, and scales that hold anything
    dev[2][3], cpu[2][3] = math.nan, math.nan
    _write_both(dev, cpu, rows[18:21], rows[18:21], torch.tensor([53, 54, 55]))


def test_writes_behind_4_gb():
    """Blocks whose bytes lie more than 2^32 behind the first."""
    H, D, bs, nb = 8, 256, 64, 36000                        # 4.7 GB for each of keys and values
    dev = [torch.zeros(nb, bs, H, D, dtype=K.INT8, device="cuda") for _ in range(2)] + \
          [torch.zeros(nb, H, device="cuda") for _ in range(2)]
    k = torch.randn(70, H * D, dtype=K.BF16, device="cuda")
    slots = torch.cat([torch.arange(64) + 35990 * bs, torch.arange(6) + 35999 * bs + 3]).cuda()
    C.block_scaled_cache(k, k, *dev, slots)
    for c, s in zip(dev[:2], dev[2:]):
        got = c.view(-1, H, D)[slots].float() * s[slots // bs][..., None]
        assert ((got - k.view(70, H, D).float()).abs() <= s[slots // bs][..., None] / 2).all()
        assert int((s != 0).sum()) == 2 * H
    q = torch.randn(1, 16, D, dtype=K.BF16, device="cuda")
    table, lens = torch.tensor([[35990]], dtype=torch.int32).cuda(), torch.tensor([64], dtype=torch.int32).cuda()
    cache = K.Cache(K.INT8, H, D, bs, [64])
    cache.codes, cache.scales = torch.stack([c[35990:35991] for c in dev[:2]]), torch.stack([s[35990:35991] for s in dev[2:]])
    cache.tables = torch.zeros(1, 1, dtype=torch.int32)
    K.check(C.block_scaled_decode(q, *dev, table, lens, D ** -0.5), q, cache, [1], D ** -0.5, 0, 0, K.F16)
    far = [d[35990:] for d in dev]
    assert torch.equal(C.block_scaled_decode(q, *dev, table, lens, D ** -0.5),
                       C.block_scaled_decode(q, *far, table - 35990, lens, D ** -0.5))
    pages = C.CachePages(dev, bs)
    pages.copy(torch.tensor([[35990, 7], [-1, -1]]).cuda())
    assert all(_same(d[7], d[35990]) for d in dev)


LENS = [1, 16, 0, 17, 255, 64, 1000, 5, 129, 33]


@pytest.mark.parametrize("dtype", [K.BF16, K.F16])
@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (40, 3), (130, 70), (16, 16), (100, 2000)])
@pytest.mark.parametrize("codes,H,G,D,bs", [(K.FP8, 2, 4, 128, 16), (K.INT8, 1, 7, 128, 32), (K.FP8, 3, 1, 64, 48),
                                            (K.INT8, 2, 16, 64, 16), (K.FP8, 1, 20, 128, 64), (K.INT8, 1, 3, 256, 16),
                                            (K.FP8, 1, 40, 256, 16)])
def test_decode(codes, H, G, D, bs, window, first, dtype):
    cache = K.Cache(codes, H, D, bs, LENS, seed=G).to("cuda")
    q = torch.randn(len(LENS), H * G, D, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    for splits in (0, 1, 3, 8, 13):
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, D ** -0.5, num_splits=splits,
                                    window=window, first=first)
        K.check(got, q, cache, [1] * len(LENS), D ** -0.5, window, first, K.F16)
        assert (got[2] == 0).all()


@pytest.mark.parametrize("dtype", [K.BF16, K.F16])
@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (50, 3), (300, 150), (128, 128), (200, 5000)])
@pytest.mark.parametrize("codes,H,G,D,bs", [(K.FP8, 2, 4, 128, 16), (K.INT8, 1, 7, 128, 32), (K.FP8, 3, 1, 64, 48),
                                            (K.INT8, 2, 2, 128, 64), (K.INT8, 1, 3, 256, 16)])
@pytest.mark.parametrize("few", [64, 0])
def test_prefill(codes, H, G, D, bs, window, first, dtype, few, monkeypatch):
    """Portions of one token to some hundred behind nothing or more, by either way, and by both ways in turn."""
    monkeypatch.setattr(C, "SCALED_ROWS", few)
    q_lens = [1, 130, 0, 4, 300, 17, 2, 129]
    lens = [n + b for n, b in zip(q_lens, [0, 0, 20, 700, 411, 1, 127, 640])]
    cache = K.Cache(codes, H, D, bs, lens, seed=G).to("cuda")
    T = sum(q_lens)
    gen = torch.Generator().manual_seed(4)
    row = torch.randn(T + 3, (H * G + 1) * D, generator=gen).to(dtype).cuda()
    q = row[:, :H * G * D].view(T + 3, H * G, D)            # a part of a wider row, rows of no request behind
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    out = torch.full((T + 3, H * G, D), 7.0, dtype=dtype, device="cuda")
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, q_lens, lens, out=out,
                                 window=window, first=first)
    assert got is out and (out[T:] == 7).all()
    p_type = K.F16 if few or D == 256 else dtype
    if few and any(n * G > 64 for n in q_lens) and D != 256:
        p_type = dtype
    K.check(got, q, cache, q_lens, D ** -0.5, window, first, p_type)


def test_prefill_in_parts(monkeypatch):
    """Requests whose keys do not fit the room for expanded ones together: the same bits."""
    q_lens, lens = [70, 150, 33, 64, 90], [200, 150, 700, 64, 333]
    cache = K.Cache(K.FP8, 2, 128, 16, lens).to("cuda")
    q = torch.randn(sum(q_lens), 8, 128, device="cuda", dtype=K.BF16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    monkeypatch.setattr(C, "SCALED_ROWS", 0)
    args = (q, *cache.parts(), cache.tables, cu, cache.seq_lens, 0.09, q_lens, lens)
    want = C.block_scaled_prefill(*args)
    for room in (1, 300, 900):
        monkeypatch.setattr(C, "SCALED_EXPANDED_KEYS", room)
        K.check(C.block_scaled_prefill(*args), q, cache, q_lens, 0.09, 0, 0, K.BF16)
    monkeypatch.setattr(C, "SCALED_EXPANDED_KEYS", 1 << 17)
    assert torch.equal(C.block_scaled_prefill(*args), want)


def test_many_requests_in_turn():
    """More changes between short and long portions than launches are worth."""
    q_lens = [3, 80, 2, 90, 1, 70, 4, 65]
    lens = [n + 30 * i for i, n in enumerate(q_lens)]
    cache = K.Cache(K.FP8, 1, 128, 16, lens).to("cuda")
    q = torch.randn(sum(q_lens), 8, 128, device="cuda", dtype=K.BF16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, 0.1, q_lens, lens)
    K.check(got, q, cache, q_lens, 0.1, 0, 0, K.BF16)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("window,first", [(0, 0), (90, 20)])
def test_what_no_query_sees_may_be_anything(codes, window, first):
    """Places behind the last key and blocks of no request hold the worst codes, scales and tables there as well."""
    lens = [5, 130, 77, 300]
    cache = K.Cache(codes, 2, 128, 16, lens)
    raw = cache.codes.view(torch.uint8)
    raw[:, cache.unused.long()] = 0x7f if codes == K.FP8 else 0x80
    cache.scales[:, cache.unused.long()] = math.nan
    for r, n in enumerate(lens):
        if n % 16:
            raw[:, cache.tables[r, n // 16].long(), n % 16:] = 0xff if codes == K.FP8 else 0x80
        cache.tables[r, -(-n // 16):] = 1 << 30
    if window:                                              # blocks in the gap between the first tokens and the window
        for r, n in enumerate(lens):
            for b in range(-(-first // 16), (n - 40 - window) // 16):
                raw[:, cache.tables[r, b].long()] = 0x7f
                cache.scales[:, cache.tables[r, b].long()] = math.inf
    clean = K.Cache(codes, 2, 128, 16, lens)                # what is seen is the same
    cache.to("cuda")
    q = torch.randn(4, 8, 128, device="cuda", dtype=K.BF16)
    for splits in (1, 4):
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, 0.09, num_splits=splits,
                                    window=window, first=first)
        K.check(got, q, clean, [1] * 4, 0.09, window, first, K.F16)
    q_lens = [5, 40, 1, 31]
    q = torch.randn(sum(q_lens), 8, 128, device="cuda", dtype=K.BF16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    for few in (64, 0):
        before, C.SCALED_ROWS = C.SCALED_ROWS, few
        try:
            got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, 0.09, q_lens, lens,
                                         window=window, first=first)
        finally:
            C.SCALED_ROWS = before
        K.check(got, q, clean, q_lens, 0.09, window, first, K.BF16)


@pytest.mark.parametrize("codes", CODES)
def test_scales_far_apart(codes):
    """Blocks whose values differ by 2^20: what the probabilities choose counts, not the largest block."""
    cache = K.Cache(codes, 1, 128, 16, [256, 200], spread=0.0)
    cache.scales[1] *= torch.exp2(torch.linspace(-20, 20, cache.scales.shape[1]).round())[:, None]
    cache.scales[0] *= torch.exp2(torch.linspace(3, -3, cache.scales.shape[1]).round())[:, None]
    cache.to("cuda")
    q = torch.randn(2, 4, 128, device="cuda", dtype=K.BF16)
    for splits in (1, 4, 12):
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, 0.3, num_splits=splits)
        K.check(got, q, cache, [1, 1], 0.3, 0, 0, K.F16)


def test_queries_of_all_sizes():
    """bf16 rows from 2^-90 to 2^60: scores in 32 bits."""
    cache = K.Cache(K.FP8, 1, 128, 16, [90] * 4, spread=0.0).to("cuda")
    q = torch.randn(4, 4, 128, device="cuda") * torch.tensor([2.0 ** -90, 1e-3, 30.0, 1.0], device="cuda")[:, None, None]
    q = q.to(K.BF16)
    K.check(C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, 0.05), q, cache, [1] * 4, 0.05, 0, 0, K.F16)
    # one key takes all of a row whose scores are far apart
    big = (q.float() * 2.0 ** 40).to(K.BF16)[3:]
    got = C.block_scaled_decode(big, *cache.parts(), cache.tables[3:].contiguous(), cache.seq_lens[3:], 1.0)
    assert torch.isfinite(got).all()


def test_rows_that_are_no_numbers_stay_alone():
    cache = K.Cache(K.FP8, 2, 128, 16, [300, 40, 90]).to("cuda")
    q = torch.randn(3, 8, 128, device="cuda", dtype=K.BF16)
    want = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, 0.09)
    q[1, 2, 5], q[0, 3, 7] = math.nan, math.inf
    for splits in (0, 1, 5, 11):
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, 0.09, num_splits=splits)
        assert got[1, 2].isnan().all() and got[0, 3].isnan().all()
        keep = torch.ones(3, 8, dtype=torch.bool)
        keep[1, 2] = keep[0, 3] = False
        assert torch.isfinite(got[keep.cuda()]).all()
    assert torch.isfinite(want).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("G", [1, 4, 7, 16, 24])
def test_shares_of_all_sizes(codes, G):
    """Requests of very different lengths, more of them than CTAs and fewer, shares that start and end anywhere."""
    for lens in ([1] * 700, [3, 0, 20000, 1, 129] + [40] * 90, [2500], list(range(1, 400, 7))):
        cache = K.Cache(codes, 2, 128, 16, lens, seed=G).to("cuda")
        q = torch.randn(len(lens), 2 * G, 128, device="cuda", dtype=K.BF16)
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, 0.09)
        K.check(got, q, cache, [1] * len(lens), 0.09, 0, 0, K.F16)


@pytest.mark.parametrize("codes,H,G,D", [(K.FP8, 1, 7, 128), (K.INT8, 1, 20, 128), (K.INT8, 3, 1, 128), (K.FP8, 2, 4, 64),
                                         (K.INT8, 2, 4, 256), (K.FP8, 9, 2, 256)])
def test_few_requests_of_many_keys(codes, H, G, D):
    """Keys of a request that many CTAs share, whose parts many CTAs merge; single tokens, and portions in several blocks of
    rows."""
    lens = [9000, 6200, 1]
    cache = K.Cache(codes, H, D, 16, lens, seed=G).to("cuda")
    q = torch.randn(3, H * G, D, device="cuda", dtype=K.BF16)
    got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, D ** -0.5)
    K.check(got, q, cache, [1] * 3, D ** -0.5, 0, 0, K.F16)
    q_lens = [4, 2, 1]
    q = torch.randn(7, H * G, D, device="cuda", dtype=K.F16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, q_lens, lens, window=7000,
                                 first=9)
    K.check(got, q, cache, q_lens, D ** -0.5, 7000, 9, K.F16)


def test_the_same_bits_again_and_on_another_stream():
    cache = K.Cache(K.FP8, 2, 128, 16, [5000, 3001, 77]).to("cuda")
    q = torch.randn(3, 8, 128, device="cuda", dtype=K.BF16)
    args = (q, *cache.parts(), cache.tables, cache.seq_lens, 0.09)
    for splits in (0, 1, 20):
        want = C.block_scaled_decode(*args, num_splits=splits)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [C.block_scaled_decode(*args, num_splits=splits) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(g, want) for g in got)


def test_captured_steps():
    """Writes, attention and a fork in two graphs that share no memory but the cache: replays follow what their inputs
    hold then."""
    H, G, D, bs, nb, M = 2, 4, 128, 16, 40, 8
    codes, scales = torch.zeros(2, nb, bs, H, D, dtype=K.FP8, device="cuda"), torch.zeros(2, nb, H, device="cuda")
    parts = (*codes, *scales)
    tables = torch.arange(2 * M, dtype=torch.int32, device="cuda").view(2, M)
    lens, slots = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    row = torch.zeros(2, (G + 2) * H * D, dtype=K.BF16, device="cuda")
    q, k, v = row.split([G * H * D, H * D, H * D], 1)
    pages = C.CachePages([*codes, *scales], bs)
    parents, fresh = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 1, 0], [-1, -1, 30]))

    def step():
        C.block_scaled_cache(k, v, *parts, slots)
        return C.block_scaled_decode(q.view(2, G * H, D), *parts, tables, lens, 0.1, num_splits=12)

    def fork():
        return pages.fork(tables, lens, parents, fresh)

    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), fork()
    torch.cuda.current_stream().wait_stream(side)
    for f in (step, fork):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    codes.zero_(), scales.zero_()
    cpu = [t.cpu() for t in parts]
    gen = torch.Generator().manual_seed(0)
    for p in range(20):
        new = torch.randn(row.shape, generator=gen).to(K.BF16)
        row.copy_(new)
        slots.copy_(torch.tensor([p, M * bs + p]))
        lens.fill_(p + 1)
        graphs[0].replay()
        ref.block_scaled_cache(*new[:, G * H * D:].split(H * D, 1), *cpu, torch.tensor([p, M * bs + p]))
        want = ref.block_scaled_attention(new[:, :G * H * D].view(2, G * H, D), *cpu, tables.cpu(), torch.tensor([0, 1, 2]),
                                          lens.cpu(), 0.1)
        assert (outs[0].cpu().float() - want.float()).abs().max() < 0.02
    assert all(_same(a, b) for a, b in zip(parts, cpu))
    graphs[1].replay()
    want = ref.fork_blocks([cpu[0], cpu[1], cpu[2], cpu[3]], bs, tables.cpu(), lens.cpu(), parents.cpu(), fresh.cpu())
    assert torch.equal(outs[1].cpu(), want) and all(_same(a, b) for a, b in zip(parts, cpu))


def _planes(gen, nb, bs):
    """Tensors of several types and widths; the last ones end at odd bytes."""
    return [torch.randn(nb, bs, 2, 64, generator=gen).to(K.FP8), torch.randn(nb, bs, 40, generator=gen).to(K.BF16),
            torch.randn(nb, 2, generator=gen), torch.randint(0, 99, (nb, bs, 3), generator=gen, dtype=torch.int8),
            torch.randint(0, 99, (nb, 5), generator=gen, dtype=torch.int8), torch.randn(nb, bs, generator=gen)]


@pytest.mark.parametrize("bs,n", [(16, 1), (48, 30), (5, 9)])
def test_copies_of_blocks(bs, n):
    gen = torch.Generator().manual_seed(n)
    cpu = _planes(gen, 2 * n + 2, bs)
    dev = [t.cuda() for t in cpu]
    order = torch.randperm(2 * n + 2, generator=gen)
    pairs = torch.stack([order[:n], order[n:2 * n]], 1)
    pairs[n // 2] = -1
    if n > 8:
        pairs[3, 0] = pairs[4, 0]                           # one block to two others
    C.CachePages(dev, bs).copy(pairs.cuda())
    ref.copy_blocks([c.view(torch.uint8) for c in cpu], pairs[pairs[:, 0] >= 0])
    assert all(_same(a, b) for a, b in zip(dev, cpu))


@pytest.mark.parametrize("bs", [16, 5])
def test_forks(bs):
    gen = torch.Generator().manual_seed(bs)
    nb, M = 60, 4
    cpu = _planes(gen, nb, bs)
    dev = [t.cuda() for t in cpu]
    order = torch.randperm(nb, generator=gen).int()
    tables = order[:5 * M].view(5, M).clone()
    lens = torch.tensor([0, bs, 2 * bs - 1, 4 * bs, 3 * bs + 1], dtype=torch.int32)
    parents = torch.tensor([4, 0, 1, 2, 2, 3, -1, 4, 4, 1, 2], dtype=torch.int32)
    fresh = order[5 * M:5 * M + 11].clone()
    fresh[[3, 7]] = -1
    got = C.CachePages(dev, bs).fork(tables.cuda(), lens.cuda(), parents.cuda(), fresh.cuda())
    want = ref.fork_blocks(cpu, bs, tables, lens, parents, fresh)
    assert torch.equal(got.cpu(), want) and all(_same(a, b) for a, b in zip(dev, cpu))


def test_pages_and_steps_without_anything():
    dev = [torch.zeros(3, 16, 2, 64, dtype=K.FP8, device="cuda"), torch.zeros(3, 2, device="cuda")]
    pages = C.CachePages(dev, 16)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    pages.copy(torch.zeros(0, 2, dtype=torch.int64, device="cuda"))
    assert pages.fork(torch.zeros(2, 4, dtype=torch.int32, device="cuda"), none.new_zeros(2), none, none).shape == (0, 4)
    with pytest.raises(ValueError, match="mapping"):
        pages.copy(torch.zeros(1, 2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="fresh"):
        pages.fork(torch.zeros(2, 4, dtype=torch.int32, device="cuda"), none.new_zeros(2), none.new_zeros(3), none)
    with pytest.raises(ValueError, match="blocks"):
        C.CachePages([dev[0], torch.zeros(4, 2, device="cuda")], 16)
    with pytest.raises(ValueError, match="tokens"):
        C.CachePages(dev, 8)
    cache = K.Cache(K.FP8, 2, 128, 16, [5]).to("cuda")
    q = torch.zeros(0, 4, 128, dtype=K.BF16, device="cuda")
    assert C.block_scaled_decode(q, *cache.parts(), cache.tables[:0], cache.seq_lens[:0], 0.1).shape == (0, 4, 128)
    C.block_scaled_cache(q[:, :2].reshape(0, 256), q[:, :2].reshape(0, 256), *cache.parts(), none.long())
    q = torch.ones(2, 4, 128, dtype=K.BF16, device="cuda")
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables[:0], none.new_zeros(1), cache.seq_lens[:0], 0.1, [], [],
                                 out=torch.full_like(q, 3))
    assert (got == 3).all()
