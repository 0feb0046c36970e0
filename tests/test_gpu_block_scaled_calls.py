"""Calls of the operators of a cache in 8 bits with block scales that meet each other or the ends of their ranges."""
import math
import threading

import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200.ops import cuda as C

pytestmark = pytest.mark.gpu
CODES = [K.FP8, K.INT8]


@pytest.fixture(autouse=True)
def _clean_status():
    from vllm_gcu_b200.ops import _native
    yield
    assert _native.take_status()[0] == 0


@pytest.mark.parametrize("few", [64, 0])
@pytest.mark.parametrize("D", [64, 128])
def test_two_threads_on_one_stream(D, few, monkeypatch):
    """Portions and single tokens from two threads that launch on the same stream: each gets what it gets alone."""
    monkeypatch.setattr(C, "SCALED_ROWS", few)
    jobs, wants, faults = [], [], []
    for seed in (1, 2):
        q_lens, lens = [70 + seed, 130, 33], [200, 700 + 9 * seed, 333]
        cache = K.Cache(K.FP8, 2, D, 16, lens, seed=seed).to("cuda")
        q = torch.randn(sum(q_lens), 8, D, device="cuda", dtype=K.BF16)
        cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
        single = torch.randn(3, 8, D, device="cuda", dtype=K.BF16)

        def job(q=q, cache=cache, cu=cu, q_lens=q_lens, lens=lens, single=single):
            return (C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, 0.09, q_lens, lens),
                    C.block_scaled_decode(single, *cache.parts(), cache.tables, cache.seq_lens, 0.09, num_splits=12))
        jobs.append(job)
        wants.append(job())
    torch.cuda.synchronize()

    def work(n):
        try:
            got = [jobs[n]() for _ in range(60)]
            torch.cuda.synchronize()
            assert all(torch.equal(g, w) for pair in got for g, w in zip(pair, wants[n]))
        except Exception as e:                            # (an assertion of a thread alone would be lost)
            faults.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults, faults[0]


@pytest.mark.parametrize("D", [64, 128, 256])
def test_queries_that_start_anywhere(D):
    """Contiguous rows behind one element, rows at an odd pitch, one row for all tokens: as the same numbers at 16 bytes."""
    lens = [300, 40, 129]
    cache = K.Cache(K.INT8, 2, D, 16, lens, seed=D).to("cuda")
    wide = torch.randn(3 * 8 * D + 40, device="cuda").to(K.BF16)
    rows = [wide[1:1 + 3 * 8 * D].view(3, 8, D), torch.as_strided(wide, (3, 8, D), (8 * D + 12, D, 1)),
            wide[:8 * D].view(1, 8, D).expand(3, 8, D)]
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    for q in rows:
        K.check(C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, D ** -0.5), q, cache, [1] * 3,
                D ** -0.5, 0, 0, K.F16)
        for few in (64, 0):
            before, C.SCALED_ROWS = C.SCALED_ROWS, few
            try:
                got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, [1] * 3, lens)
            finally:
                C.SCALED_ROWS = before
            K.check(got, q, cache, [1] * 3, D ** -0.5, 0, 0, K.F16 if few or D == 256 else K.BF16)


@pytest.mark.parametrize("first", [2 ** 31 - 1, 2 ** 31 - 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_all_tokens_as_first_ones(D, first):
    """A window beside first tokens without end hides nothing."""
    q_lens, lens = [3, 140, 20], [300, 700, 129]
    cache = K.Cache(K.FP8, 2, D, 16, lens, seed=D).to("cuda")
    q = torch.randn(sum(q_lens), 8, D, device="cuda", dtype=K.BF16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    got = C.block_scaled_decode(q[:3], *cache.parts(), cache.tables, cache.seq_lens, D ** -0.5, window=40, first=first)
    K.check(got, q[:3], cache, [1] * 3, D ** -0.5, 0, 0, K.F16)
    for few in (64, 0):
        before, C.SCALED_ROWS = C.SCALED_ROWS, few
        try:
            got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, q_lens, lens,
                                         window=40, first=first)
        finally:
            C.SCALED_ROWS = before
        K.check(got, q, cache, q_lens, D ** -0.5, 0, 0, K.BF16)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("late", [65504.0, -65504.0, math.inf])
def test_the_largest_numbers_of_fp16_in_expanded_values(codes, D, late, monkeypatch):
    """A code that stands for more than fp16 holds: rows in front of it keep their bits, rows that see it are finite and off
    by 2^-11 of its share (65504 in place of 65536) beside what they are allowed anyway; so are those that see an
    infinity, whose code is the largest."""
    monkeypatch.setattr(C, "SCALED_ROWS", 0)
    H, G, n, at = 2, 4, 200, 181
    gen = torch.Generator().manual_seed(D)
    cache = K.Cache(codes, H, D, 16, [n], seed=1).to("cuda")
    q = torch.randn(n, H * G, D, generator=gen).to(K.F16).cuda()
    cu, slots = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.arange(176, 192).cuda()
    slots = cache.tables[0, 11].long() * 16 + slots % 16
    args = (q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, [n], [n])
    k, v = (torch.randn(16, H * D, generator=gen).to(K.F16).cuda() for _ in range(2))
    C.block_scaled_cache(k, v, *cache.parts(), slots)
    want = C.block_scaled_prefill(*args)
    v[at - 176, ::5] = late
    C.block_scaled_cache(k, v, *cache.parts(), slots)
    got = C.block_scaled_prefill(*args)
    assert torch.isfinite(got).all() and torch.equal(got[:176], want[:176])
    if math.isinf(late):
        return
    out, size, reach, top = K.attention(q, cache, [n], D ** -0.5)
    may = K.allowed(out, size, reach, top, K.F16, K.F16, n, D) + size * 2.0 ** -11
    keep = out.abs() < 65000
    assert ((got.double().cpu() - out).abs()[keep] <= may[keep]).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("log2", [30, 60])
def test_zeros_beside_the_largest_values(codes, D, log2):
    """Blocks of zeros have the least scale: their keys count beside values of 2^30 or 2^60 times a code."""
    lens = [200, 64, 33]
    cache = K.Cache(codes, 2, D, 16, lens, seed=D, spread=0.0)
    cache.scales[1] = 2.0 ** log2
    for r, n in enumerate(lens):
        for b in range(0, -(-n // 16), 2):
            cache.scales[1, cache.tables[r, b].long()] = 2.0 ** -100
            cache.codes[1, cache.tables[r, b].long()] = 0
    cache.to("cuda")
    q = torch.randn(3, 8, D, device="cuda", dtype=K.BF16)
    for splits in (0, 1, 5, 12):
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, D ** -0.5, num_splits=splits)
        K.check(got, q, cache, [1] * 3, D ** -0.5, 0, 0, K.F16)


def test_types_and_drafters_that_are_refused():
    """Before the first step: activations in fp32, and a drafter whose heads have another size."""
    from vllm_gcu_b200 import LLM
    kw = dict(num_hidden_layers=1, max_num_seqs=2, max_num_batched_tokens=64, max_model_len=64, num_gpu_blocks=16,
              device="cuda", enforce_eager=True, kv_cache_dtype="fp8_block")
    with pytest.raises(ValueError, match="bf16 or fp16"):
        LLM("llama-3-8b", dtype="float32", **kw)
    llm = LLM("llama-3-8b", **kw)

    class Drafter:
        def kv_cache_spec(self):
            return {"type": "gqa", "layers": 1, "kv_heads": 2, "head_dim": 96}
    llm.engine.runner.drafter = Drafter()
    with pytest.raises(ValueError, match="not 96"):
        llm.engine.runner.init_kv_cache(16)
