"""A cache in 8 bits with a scale for each block and head: the oracle's definitions, refusals, the attention layer."""
import math

import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200.layers.attention import AttentionMetadata, BlockScaledCache, PagedAttention
from vllm_gcu_b200.layers.basic import RotaryEmbedding
from vllm_gcu_b200.ops import cuda as C
from vllm_gcu_b200.ops import ref

CODES = [K.FP8, K.INT8]


@pytest.mark.parametrize("codes", CODES)
def test_scales_are_the_least_powers_of_two(codes):
    top = 448.0 if codes == K.FP8 else 127.0
    x = torch.cat([torch.tensor([0.0, 1e-42, 2.0 ** -92, 1.0, top, top * 1.0000001, 3.3e38]), torch.rand(200) * 1e3])
    s = ref.block_scale(x, codes == K.INT8).double()
    assert torch.equal(torch.exp2(torch.round(torch.log2(s))), s)
    assert ((x.double() <= top * s) | (s == 2.0 ** 121)).all()
    assert ((x.double() > top * s / 2) | (s == 2.0 ** -100)).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("steps", [[16], [5, 11], [1] * 16, [3, 20, 1, 8, 1, 1]])
def test_what_is_written_stands_for_the_rows(codes, steps):
    """Every number is off by half a step of its block's scale (fp8: half a step of the number's own where that is more),
    and by as much again for every time that the scale grew."""
    torch.manual_seed(1)
    H, D, bs, T = 2, 64, 16, sum(steps)
    k, v = (torch.randn(T, H * D) * torch.exp(torch.randn(T, 1)) for _ in range(2))
    kc = torch.zeros(2, 4, bs, H, D, dtype=codes)
    sc = torch.zeros(2, 4, H)
    table, at, grew = torch.tensor([2, 0, 3]), 0, 0
    for n in steps:
        pos = torch.arange(at, at + n)
        before = sc.clone()
        ref.block_scaled_cache(k[at:at + n], v[at:at + n], kc[0], kc[1], sc[0], sc[1], table[pos // bs] * bs + pos % bs)
        grew += int(((sc > before) & (before > 0)).any())
        at += n
    pages = table[:-(-T // bs)]
    for c, s, x in ((kc[0], sc[0], k), (kc[1], sc[1], v)):
        got = (c[pages].float() * s[pages][:, None, :, None]).flatten(0, 1)[:T].double()
        want, scale = x.view(T, H, D).double(), s[pages].repeat_interleave(bs, 0)[:T, :, None].double()
        step = scale / 2 if codes == K.INT8 else torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10)
        assert ((got - want).abs() <= step * (1 + grew) * 1.0001).all()


def test_what_is_no_number_does_not_set_the_scale():
    for codes, top in ((K.FP8, 448.0), (K.INT8, 127.0)):
        c, s = torch.zeros(2, 1, 16, 1, 64, dtype=codes), torch.zeros(2, 1, 1)
        x = torch.ones(2, 64)
        x[0, 0], x[0, 1], x[1, 2] = math.inf, math.nan, -math.inf
        ref.block_scaled_cache(x, x, *c, *s, torch.tensor([0, 1]))
        assert (s == ref.block_scale(torch.tensor(1.0), codes == K.INT8)).all()
        assert c[0, 0, 0, 0, 0].float() == top and c[0, 0, 0, 0, 1].float() == 0 and c[0, 0, 1, 0, 2].float() == -top


def test_fork_shares_full_blocks():
    caches = [torch.arange(8 * 4 * 3).view(8, 4, 3).float(), torch.arange(8.0).view(8, 1)]
    before = [c.clone() for c in caches]
    tables = torch.tensor([[5, 1, 0], [2, 0, 0]], dtype=torch.int32)
    got = ref.fork_blocks(caches, 4, tables, torch.tensor([6, 4], dtype=torch.int32),
                          torch.tensor([0, 0, 1, -1], dtype=torch.int32), torch.tensor([-1, 7, 6, 3], dtype=torch.int32))
    assert got.tolist() == [[5, 1, 0], [5, 7, 0], [2, 6, 0], [0, 0, 0]]
    assert torch.equal(caches[0][7, :2], before[0][1, :2]) and torch.equal(caches[0][7, 2:], before[0][7, 2:])
    assert caches[1][7] == 1 and caches[1][6] == 6
    caches[0][7, :2], caches[1][7] = before[0][7, :2], 7.0
    assert all(torch.equal(a, b) for a, b in zip(caches, before))


def _layer(**kw):
    rot = RotaryEmbedding(64, 64, 512, 10000.0, True, None, torch.float32, "cpu")
    return PagedAttention(4, 2, 64, 0.125, rot, **kw)


def _md(starts, q_lens, table, bs):
    pos = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, q_lens)])
    req = torch.repeat_interleave(torch.arange(len(q_lens)), torch.tensor(q_lens))
    nd = sum(n == 1 for n in q_lens)
    cu = torch.tensor([0] + q_lens[nd:]).cumsum(0).int()
    return AttentionMetadata(
        num_tokens=len(pos), num_decodes=nd, num_prefills=len(q_lens) - nd, num_decode_tokens=nd, positions=pos,
        slot_mapping=table[req, pos // bs].long() * bs + pos % bs, block_tables=table,
        seq_lens=torch.tensor([s + n for s, n in zip(starts, q_lens)], dtype=torch.int32), cu_q_prefill=cu,
        q_lens_cpu=list(q_lens), seq_lens_cpu=[s + n for s, n in zip(starts, q_lens)])


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("kw", [{}, dict(sliding_window=9), dict(sliding_window=9, window_first=3)])
def test_layer_over_scaled_blocks(codes, kw):
    """The layer's steps over a cache in 8 bits stay near those over one in 32 bits: e4m3 codes are off by 2^-4 of
    themselves, int8 ones by 2^-8 of the largest or twice that."""
    torch.manual_seed(0)
    layer = _layer(**kw)
    bs, table = 16, torch.tensor([[3, 1, 0], [4, 2, 5]], dtype=torch.int32)
    wide = torch.zeros(2, 6, bs, 2, 64)
    small = BlockScaledCache.zeros(6, bs, 2, 64, codes, "cpu")
    for starts, q_lens in (([0, 0], [13, 30]), ([13, 30], [1, 1]), ([14, 31], [1, 4]), ([15, 35], [7, 2])):
        md = _md(starts, q_lens, table, bs)
        x = torch.randn(md.num_tokens, 8 * 64)
        want, got = layer(x, wide, md), layer(x, small, md)
        assert (got - want).norm() / want.norm() < 0.12
    assert len(small.planes()) == 4 and small.planes()[2].shape == (6, 2)


def test_first_tokens_stay_visible():
    torch.manual_seed(2)
    q, kc, vc = torch.randn(1, 2, 64), torch.randn(3, 16, 2, 64), torch.randn(3, 16, 2, 64)
    tables, cu, lens = torch.tensor([[1, 0, 2]]), torch.tensor([0, 1]), torch.tensor([40])
    got = ref.varlen_prefill_attention(q, kc, vc, tables, cu, lens, 0.125, window=8, first=5)
    keep = [0, 1, 2, 3, 4] + list(range(32, 40))
    k, v = kc[tables[0]].flatten(0, 1)[keep], vc[tables[0]].flatten(0, 1)[keep]
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0], k) * 0.125, -1)
    assert torch.allclose(got[0], torch.einsum("hn,nhd->hd", p, v), atol=1e-5)


def _call(**change):
    c = K.Cache(K.FP8, 2, 64, 16, [20, 33])
    a = dict(q=torch.zeros(2, 4, 64, dtype=K.BF16), k_cache=c.codes[0], v_cache=c.codes[1], k_scale=c.scales[0],
             v_scale=c.scales[1], block_tables=c.tables, seq_lens=c.seq_lens, scale=0.125)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(2, 4, 64)), "bf16 or fp16"), (dict(q=torch.zeros(2, 3, 64, dtype=K.BF16)), "heads"),
    (dict(q=torch.zeros(2, 4, 128, dtype=K.BF16)), "heads of"), (dict(window=-1), "window"), (dict(first=-2), "window"),
    (dict(num_splits=33), "splits"), (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens"),
    (dict(block_tables=torch.zeros(3, 2, dtype=torch.int32)), "block_tables"),
    (dict(k_scale=torch.zeros(3, 2)), "k_scale"), (dict(v_scale=torch.zeros(2, dtype=torch.float64)), "v_scale"),
    (dict(k_cache=torch.zeros(3, 16, 2, 64)), "caches"), (dict(out=torch.zeros(2, 4, 64)), "out"),
])
def test_decode_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        C.block_scaled_decode(**_call(**change))


def test_caches_that_are_refused():
    for shape, dtype in (((3, 8, 2, 64), K.FP8), ((3, 16, 2, 80), K.FP8), ((3, 16, 2, 64), torch.uint8),
                         ((0, 16, 2, 64), K.INT8), ((3, 16, 64), K.INT8)):
        c, s = torch.zeros(shape).to(dtype), torch.zeros(shape[0], 2)
        with pytest.raises(ValueError):
            C.block_scaled_cache(torch.zeros(1, 128), torch.zeros(1, 128), c, c.clone(), s, s.clone(), torch.zeros(1).long())
    c = K.Cache(K.INT8, 2, 64, 16, [20])
    turned = c.codes[0].transpose(1, 2).contiguous().transpose(1, 2)
    with pytest.raises(ValueError, match="k_cache"):
        C.block_scaled_cache(torch.zeros(1, 128), torch.zeros(1, 128), turned, turned, *c.scales, torch.zeros(1).long())
    with pytest.raises(ValueError, match="slot_mapping"):
        C.block_scaled_cache(torch.zeros(1, 128), torch.zeros(1, 128), *c.parts(), torch.zeros(1).int())
    with pytest.raises(ValueError, match="k has|k:"):
        C.block_scaled_cache(torch.zeros(1, 64), torch.zeros(1, 128), *c.parts(), torch.zeros(1).long())
    with pytest.raises(ValueError, match="v is"):
        C.block_scaled_cache(torch.zeros(1, 128), torch.zeros(1, 128).half(), *c.parts(), torch.zeros(1).long())
    with pytest.raises(ValueError, match="GPU"):
        C.block_scaled_cache(torch.zeros(1, 128), torch.zeros(1, 128), *c.parts(), torch.zeros(1).long())


@pytest.mark.parametrize("q_lens,kv_lens,match", [([1, 2], [20, 33, 4], "portions"), ([1, 34], [20, 33], "portions"),
                                                  ([1, 2], [20, 49], "portions"), ([2, 2], [20, 33], "portions"),
                                                  ([1], [20], "block_tables"), ([-1, 2], [20, 33], "portions")])
def test_prefill_refuses(q_lens, kv_lens, match):
    with pytest.raises(ValueError, match=match):
        C.block_scaled_prefill(**_call(q=torch.zeros(3, 4, 64, dtype=K.BF16)), cu_q=torch.zeros(3, dtype=torch.int32),
                               q_lens=q_lens, kv_lens=kv_lens)


def test_output_that_shares_memory_is_refused():
    a = _call()
    with pytest.raises(ValueError, match="shares memory with q"):
        C.block_scaled_decode(**a, out=a["q"])
    with pytest.raises(ValueError, match="shares memory with the cache"):
        raw = a["k_cache"].flatten().view(torch.uint8)[:2 * 4 * 64 * 2]
        C.block_scaled_decode(**a, out=raw.view(K.BF16).view(2, 4, 64))


def test_expanded_tiles_cover_what_is_seen():
    for q, n, w, f in [(1, 1, 0, 0), (5, 700, 0, 9), (5, 700, 100, 0), (5, 700, 100, 200), (200, 1000, 300, 129),
                       (700, 700, 64, 5), (1, 513, 1, 1)]:
        seen = {k // 128 for p in range(n - q, n) for k in range(p + 1) if not w or k > p - w or k < f}
        assert C._expanded_tiles(q, n, w, f) == len(seen)


def test_pages_refuse():
    for tensors, bs in (([], 16), ([torch.zeros(4, 16, 3)], 16), ([torch.zeros(4, 3)], 0)):
        with pytest.raises(ValueError):
            C.CachePages(tensors, bs)


def test_splits_fill_the_device(monkeypatch):
    monkeypatch.setattr(C, "_sms", lambda: 148)
    assert C.block_scaled_splits(1, 8, 100) == 1 and C.block_scaled_splits(512, 8, 4096) == 1
    for b, h, n in [(1, 1, 300), (1, 8, 1501), (3, 8, 9000), (4, 4, 120001), (1, 1, 1 << 20)]:
        s = C.block_scaled_splits(b, h, n)
        assert 1 <= s <= 32 and (s == 1 or n // s >= 128)


def test_engine_config_knows_the_types():
    from vllm_gcu_b200.config import preset
    wide, small = (preset("llama-3-8b", kv_cache_dtype=t) for t in ("auto", "int8_block"))
    assert small.kv_bytes_per_token() * 2 == wide.kv_bytes_per_token()


def test_long_documents_leave_the_wide_kernel_idle(monkeypatch):
    """A few dozen rows behind one long document go by the kernel for few rows, a prompt does not."""
    monkeypatch.setattr(C, "_sms", lambda: 148)
    assert C._rows_pay([64], [250], 4, 8) and C._rows_pay([16] * 32, [16] * 32, 4, 8)
    assert not C._rows_pay([32] * 64, [8] * 64, 4, 4) and not C._rows_pay([2048], [16], 8, 4)
    assert not C._rows_pay([2048], [128], 8, 4)
