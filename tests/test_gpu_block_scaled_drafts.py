"""Drafts over a cache in 8 bits with block scales: rows that are written, checked, rejected and written again."""
import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200 import LLM, SamplingParams
from vllm_gcu_b200.ops import _native
from vllm_gcu_b200.ops import cuda as C
from vllm_gcu_b200.ops import ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _native.take_status()[0] == 0


@pytest.mark.parametrize("codes,H,G,D", [(K.FP8, 2, 4, 128), (K.INT8, 1, 7, 128), (K.INT8, 2, 2, 64), (K.FP8, 1, 4, 256)])
def test_rows_that_are_written_again(codes, H, G, D):
    """Three requests, four drafts a step of which some are taken; rejected ones are larger, begin blocks and reach into the next
    one.  The cache holds the oracle's bits, and attention after each step is that of what it holds."""
    gen = torch.Generator().manual_seed(D)
    bs, M = 16, 8
    nb = 3 * M + 1
    dev = [torch.zeros(nb, bs, H, D, dtype=codes).cuda() for _ in range(2)] + [torch.zeros(nb, H).cuda() for _ in range(2)]
    cpu = [t.cpu() for t in dev]
    tables = torch.randperm(nb - 1, generator=gen)[:3 * M].view(3, M)
    at = [13, 30, 1]
    for r, n in enumerate(at):                              # prompts
        k, v = (torch.randn(n, H * D, generator=gen).to(K.BF16) for _ in range(2))
        slots = tables[r, torch.arange(n) // bs] * bs + torch.arange(n) % bs
        C.block_scaled_cache(k.cuda(), v.cuda(), *dev, slots.cuda())
        ref.block_scaled_cache(k, v, *cpu, slots)
    for taken in [(1, 5, 2), (3, 1, 1), (4, 1, 5), (1, 1, 3), (2, 4, 1), (5, 5, 5), (1, 2, 1)]:
        pos = [torch.arange(a, a + 5) for a in at]
        slots = torch.cat([tables[r, p // bs] * bs + p % bs for r, p in enumerate(pos)])
        size = torch.ones(15, 1)
        for r, n in enumerate(taken):
            size[5 * r + n:5 * r + 5] = 20.0
        k, v = ((torch.randn(15, H * D, generator=gen) * size).to(K.BF16) for _ in range(2))
        C.block_scaled_cache(k.cuda(), v.cuda(), *dev, slots.cuda())
        ref.block_scaled_cache(k, v, *cpu, slots)
        assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(dev, cpu))
        lens = [a + 5 for a in at]
        cache = K.Cache(codes, H, D, bs, lens, blocks=nb)
        cache.codes, cache.scales = torch.stack(dev[:2]), torch.stack(dev[2:])
        cache.tables, cache.seq_lens = tables.int().cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        q = torch.randn(15, H * G, D, generator=gen).to(K.F16).cuda()
        cu = torch.tensor([0, 5, 10, 15], dtype=torch.int32, device="cuda")
        got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, [5] * 3, lens)
        K.check(got, q, cache, [5] * 3, D ** -0.5, 0, 0, K.F16)
        at = [a + n for a, n in zip(at, taken)]


KW = dict(num_hidden_layers=2, max_num_seqs=4, max_num_batched_tokens=256, max_model_len=256, num_gpu_blocks=64,
          device="cuda", enforce_eager=True, enable_prefix_caching=False)


def _steps(llm, prompt, n):
    """Tokens of an answer, and the logits that each of them was taken from."""
    eng, rows = llm.engine, []
    eng.runner.keep_logits = True
    finish = eng._finish

    def kept(so, handle):
        for tokens in handle.token_ids().values():
            rows.extend(eng.runner.last_logits[:len(tokens)])
        return finish(so, handle)
    eng._finish = kept
    out = llm.generate([prompt], SamplingParams(max_tokens=n, temperature=0.0, ignore_eos=True))[0].outputs[0].token_ids
    eng._finish = finish
    _native.check_status()
    return list(out), rows[:n]


def _compare(plain, prompt, got):
    """Each token's logits are those of a run without drafts whose prompt ends in front of it, but for the scales that
    rejected rows have raised (codes of the block are rounded once more) and for the order of sums."""
    for i, row in enumerate(got[1]):
        want = _steps(plain, prompt + got[0][:i], 1)[1][0]
        assert torch.nn.functional.cosine_similarity(want, row, dim=0) > 0.99, i


@pytest.mark.parametrize("kvd", ["fp8_block", "int8_block"])
def test_drafts_that_are_taken_and_rejected(kvd):
    prompt = torch.randint(0, 128256, (29,), generator=torch.Generator().manual_seed(4)).tolist()
    plain = LLM("llama-3-8b", kv_cache_dtype=kvd, **KW)
    want = _steps(plain, prompt, 24)
    llm = LLM("llama-3-8b", kv_cache_dtype=kvd, speculative_method="ngram", num_speculative_tokens=3, **KW)

    class Proposer:
        """What comes next, the token wrong whose place is that of the step in turn."""
        def propose(self, tokens):
            i = len(tokens) - len(prompt)
            drafts = want[0][i:i + 3]
            if drafts and i % 4 < len(drafts):
                drafts[i % 4] = (drafts[i % 4] + 1) % 128256
            return drafts
    llm.engine.proposer = Proposer()
    got = _steps(llm, prompt, 24)
    m = llm.engine.spec_metrics
    assert 0 < m.num_accepted_tokens < m.num_draft_tokens
    _compare(plain, prompt, got)


def test_a_drafter_with_its_own_cache_and_the_answer_without_it():
    prompt = torch.randint(0, 128256, (29,), generator=torch.Generator().manual_seed(5)).tolist()
    llm = LLM("llama-3-8b", kv_cache_dtype="fp8_block", speculative_method="eagle", num_speculative_tokens=1, **KW)
    got = _steps(llm, prompt, 20)
    m = llm.engine.spec_metrics
    assert m.num_accepted_tokens < m.num_draft_tokens
    _compare(LLM("llama-3-8b", kv_cache_dtype="fp8_block", **KW), prompt, got)


@pytest.mark.parametrize("codes,H,G,D,bs", [(K.FP8, 2, 4, 128, 16), (K.INT8, 1, 7, 128, 32), (K.FP8, 3, 1, 64, 48),
                                            (K.INT8, 1, 3, 256, 16)])
@pytest.mark.parametrize("window,first", [(0, 0), (50, 3), (300, 150)])
def test_portions_by_the_way_that_each_takes(codes, H, G, D, bs, window, first, monkeypatch):
    """Few rows in front, long portions behind: each request is held to the rounding of probabilities of its own way."""
    monkeypatch.setattr(C, "_rows_pay", lambda *args: False)
    q_lens = [1, 4, 0, 8, 300, 129]
    lens = [n + b for n, b in zip(q_lens, [0, 700, 20, 127, 411, 640])]
    cache = K.Cache(codes, H, D, bs, lens, seed=G).to("cuda")
    gen = torch.Generator().manual_seed(4)
    q = torch.randn(sum(q_lens), H * G, D, generator=gen).to(K.BF16).cuda()
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, D ** -0.5, q_lens, lens,
                                 window=window, first=first).double().cpu()
    out, size, reach, top = K.attention(q, cache, q_lens, D ** -0.5, window, first)
    at = 0
    for n in q_lens:
        s = slice(at, at + n)
        at += n
        few = n * G <= 64 or D == 256
        may = K.allowed(out[s], size[s], reach[s], top[s], K.BF16, K.F16 if few else K.BF16, max(lens), D)
        assert ((got[s] - out[s]).abs() <= may).all(), n
