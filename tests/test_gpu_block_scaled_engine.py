"""The engine over a cache in 8 bits with a scale for each block and head: the layer's steps, graphs, swapping, checked
drafts, windows whose first tokens stay visible."""
import pytest
import torch

from vllm_gcu_b200 import LLM, SamplingParams
from vllm_gcu_b200.layers.attention import BlockScaledCache
from vllm_gcu_b200.ops import _native

pytestmark = pytest.mark.gpu
KW = dict(num_hidden_layers=2, max_num_seqs=8, max_num_batched_tokens=256, max_model_len=512, num_gpu_blocks=256)


def _prompts(lens, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 128256, (n,), generator=gen).tolist() for n in lens]


def _logits(prompts, sp, **kw):
    llm = LLM("llama-3-8b", device="cuda", **{**KW, "enforce_eager": True, **kw})
    llm.engine.runner.keep_logits = True
    out = llm.generate(prompts, sp)
    _native.check_status()
    return llm, out, llm.engine.runner.last_logits


@pytest.mark.parametrize("kvd", ["fp8_block", "int8_block"])
def test_logits_track_those_of_16_bits(kvd):
    prompts, sp = _prompts([200, 33, 120], 9), SamplingParams(max_tokens=3, temperature=0.0, ignore_eos=True)
    _, _, want = _logits(prompts, sp)
    llm, _, got = _logits(prompts, sp, kv_cache_dtype=kvd)
    assert isinstance(llm.engine.runner.kv_caches[0], BlockScaledCache)
    cos = torch.nn.functional.cosine_similarity(want.flatten(), got.flatten(), dim=0).item()
    rms = ((want - got).pow(2).mean().sqrt() / want.std()).item()
    assert cos > 0.97 and rms < 0.25, (cos, rms)


def test_a_window_with_first_tokens():
    """Prompts that fit the window give the same logits as without one; longer ones differ, and differ again with the
    first tokens visible."""
    sp = SamplingParams(max_tokens=3, temperature=0.0, ignore_eos=True)
    short, long = _prompts([60, 33], 2), _prompts([300, 200], 3)
    kw = dict(kv_cache_dtype="fp8_block")
    a = _logits(short, sp, **kw)[2]
    b = _logits(short, sp, sliding_window=64, sliding_window_first=4, **kw)[2]
    assert torch.equal(a, b)
    a = _logits(long, sp, **kw)[2]
    b = _logits(long, sp, sliding_window=64, **kw)[2]
    c = _logits(long, sp, sliding_window=64, sliding_window_first=4, **kw)[2]
    assert not torch.equal(a, b) and not torch.equal(b, c)
    with pytest.raises(ValueError, match="fp8_block"):
        LLM("llama-3-8b", device="cuda", sliding_window=64, sliding_window_first=4, enforce_eager=True, **KW)


def test_graphs_give_the_same_tokens():
    prompts, sp = _prompts([100, 17, 64, 31], 5), SamplingParams(max_tokens=24, temperature=0.0, ignore_eos=True)
    outs = [LLM("llama-3-8b", device="cuda", kv_cache_dtype="int8_block", enforce_eager=eager, **KW).generate(prompts, sp)
            for eager in (True, False)]
    same = sum(a.outputs[0].token_ids == b.outputs[0].token_ids for a, b in zip(*outs))
    assert same >= 3            # (other numbers of splits round otherwise)
    _native.check_status()


def test_swapped_requests_take_their_scales_along():
    """A pool too small for all requests: what is swapped out and in again gives the tokens of an ample pool."""
    prompts, sp = _prompts([90, 85, 95, 80], 6), SamplingParams(max_tokens=40, temperature=0.0, ignore_eos=True)
    kw = dict(KW, kv_cache_dtype="fp8_block", enforce_eager=True, enable_prefix_caching=False)
    want = LLM("llama-3-8b", device="cuda", **kw).generate(prompts, sp)
    kw.update(num_gpu_blocks=30, num_cpu_blocks=64)
    small = LLM("llama-3-8b", device="cuda", **kw)
    got = small.generate(prompts, sp)
    assert getattr(small.engine.runner, "cpu_caches", None) is not None, "nothing was swapped"
    same = sum(a.outputs[0].token_ids == b.outputs[0].token_ids for a, b in zip(want, got))
    assert same >= 3            # (steps of other requests round otherwise)
    _native.check_status()


def test_checked_drafts():
    prompts, sp = [[5, 6, 7, 8] * 12, [9, 10, 11] * 15], SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True)
    kw = dict(KW, kv_cache_dtype="fp8_block", enforce_eager=True)
    got = LLM("llama-3-8b", device="cuda", speculative_method="ngram", num_speculative_tokens=3, **kw).generate(prompts, sp)
    assert all(len(o.outputs[0].token_ids) == 12 for o in got)
    _native.check_status()


def test_sizes_that_are_refused():
    with pytest.raises(ValueError, match="fp8_block"):
        LLM("llama-3-8b", device="cuda", kv_cache_dtype="fp8_block", head_dim=96, enforce_eager=True, **KW)
    with pytest.raises(ValueError, match="int4_block"):
        LLM("llama-3-8b", device="cuda", kv_cache_dtype="int4_block", enforce_eager=True, **KW)


def test_prompts_in_portions_and_from_the_prefix_cache():
    """Prompts that take several steps, and prompts that start with another one's blocks: nearly the logits of a prompt at
    once (the blocks' scales grow with the portions)."""
    a = _prompts([400], 8)[0]
    sp = SamplingParams(max_tokens=2, temperature=0.0, ignore_eos=True)
    kw = dict(kv_cache_dtype="fp8_block")
    whole = _logits([a], sp, max_num_batched_tokens=512, **kw)[2]
    parts = _logits([a], sp, max_num_batched_tokens=64, **kw)[2]
    llm, _, _ = _logits([a], sp, **kw)
    again = llm.generate([a[:390] + a[:10]], sp)[0]
    assert again.num_cached_tokens >= 384
    cos = torch.nn.functional.cosine_similarity(whole.flatten(), parts.flatten(), dim=0).item()
    assert cos > 0.99
    _native.check_status()


def test_the_connector_refuses():
    llm = LLM("llama-3-8b", device="cuda", kv_cache_dtype="fp8_block", enforce_eager=True, **KW)
    with pytest.raises(ValueError, match="scales"):
        llm.engine.attach_kv_connector(object())


def test_models_that_are_refused():
    """Caches of another layout, and attention with distances among the scores, have no form with block scales."""
    with pytest.raises(ValueError, match="alike"):
        LLM("tiny-deepseek", device="cuda", kv_cache_dtype="fp8_block", enforce_eager=True, num_gpu_blocks=64)
    with pytest.raises(ValueError, match="ALiBi"):
        LLM("llama-3-8b", device="cuda", kv_cache_dtype="fp8_block", extra={"position_embedding": "ALIBI"},
            enforce_eager=True, **KW)


def test_a_drafter_with_its_own_cache():
    prompts, sp = _prompts([60, 33], 9), SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True)
    llm = LLM("llama-3-8b", device="cuda", kv_cache_dtype="fp8_block", speculative_method="eagle", num_speculative_tokens=1,
              enforce_eager=True, **KW)
    got = llm.generate(prompts, sp)
    assert all(len(o.outputs[0].token_ids) == 12 for o in got)
    assert all(type(c) is type(llm.engine.runner.kv_caches[0]) for c in llm.engine.runner.drafter_caches)
    _native.check_status()
