"""Keys far below one that takes nearly all of a row: what they add up to is kept, beside a value of 0 of that key.

The keys behind the first one have four scores, and values of one sign in each column, so that the rounding of a probability
or its loss is not averaged away by its neighbours'."""
import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200.ops import cuda as C

pytestmark = pytest.mark.gpu
GAPS = [4.0, 9.0, 12.0, 14.0, 16.0, 18.0]          # nats, a query head each: shares of 0.09 to 1 - 1e-5 at 600 keys


@pytest.fixture(autouse=True)
def _clean_status():
    from vllm_gcu_b200.ops import _native
    yield
    assert _native.take_status()[0] == 0


def _cache(codes, D, lens, H=2):
    cache = K.Cache(codes, H, D, 16, lens, seed=D, spread=0.0)
    gen = torch.Generator().manual_seed(5)
    nb = cache.codes.shape[1]
    keys = torch.zeros(nb, 16, H, D)
    keys[..., 0] = torch.randint(0, 4, (nb, 16, H), generator=gen).float()
    top = 448 if codes == K.FP8 else 127
    values = torch.randint(top // 2, top + 1, (nb, 16, H, D), generator=gen).float()
    values *= torch.where(torch.rand(D, generator=gen) < 0.5, -1.0, 1.0)
    for r, n in enumerate(lens):
        if n:
            keys[cache.tables[r, 0].long(), 0, :, 0] = 64.0
            values[cache.tables[r, 0].long(), 0] = 0.0
    cache.codes = torch.stack([keys, values]).to(codes)
    cache.scales[0], cache.scales[1] = 2.0 ** -6, 16.0
    return cache.to("cuda")


def _queries(T, D, scale, dtype, H=2):
    q = torch.zeros(T, H * len(GAPS), D, dtype=dtype, device="cuda")
    q[..., 0] = (torch.tensor(GAPS * H) / scale).to(dtype).cuda()
    return q


def _check(got, q, cache, q_lens, scale, window, first, rel, step):
    """``rel``: half a step of a probability relative to itself; ``step``: how far one may be off at least, of the largest
    one times its values' scale, which counts for each key with its code.  Scores, sums and the result as in
    ``block_scaled_cases.allowed``; an fp16 result ends at 2^-24."""
    out, size, reach, top = K.attention(q, cache, q_lens, scale, window, first)
    keys = max(cache.lens)
    most = 448 if cache.codes.dtype == K.FP8 else 127
    may = size * (rel + 2 * (cache.width + 8) * 2.0 ** -23 * reach[..., None] + (keys + 16) * 2.0 ** -22)
    may += keys * most * step * top[..., None] + out.abs() * torch.finfo(got.dtype).eps / 2 * 1.01
    may += 2.0 ** -25 if got.dtype == K.F16 else 1e-30
    far = (got.double().cpu() - out).abs()
    worst = (far / may).amax((0, 2))
    assert torch.isfinite(got).all() and (worst <= 1).all(), worst.tolist()


def _step(codes, D):
    """fp16 of 2^11 times a probability ends at 2^-24: half a step is 2^-36.  int8 digits of multiples of 2^-31."""
    return 2.0 ** -32 if codes == K.INT8 and D == 128 else 2.0 ** -36


EXPANDED = [(K.FP8, 64), (K.INT8, 128), (K.FP8, 128)]


@pytest.mark.parametrize("dtype", [K.F16, K.BF16])
@pytest.mark.parametrize("window,first", [(0, 0), (300, 3)])
@pytest.mark.parametrize("codes,D", EXPANDED)
def test_expanded_portions(codes, D, window, first, dtype, monkeypatch):
    monkeypatch.setattr(C, "SCALED_ROWS", 0)
    q_lens, lens = [130, 20, 200], [130, 600, 1500]
    cache, scale = _cache(codes, D, lens), D ** -0.5
    q = _queries(sum(q_lens), D, scale, dtype)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, scale, q_lens, lens, window=window,
                                 first=first)
    _check(got, q, cache, q_lens, scale, window, first, torch.finfo(dtype).eps / 2, 2.0 ** -36 if dtype == K.F16 else 0.0)


FEW = [(K.FP8, 64), (K.INT8, 64), (K.FP8, 256), (K.INT8, 256), (K.FP8, 128), (K.INT8, 128)]


@pytest.mark.parametrize("dtype", [K.F16, K.BF16])
@pytest.mark.parametrize("window,first", [(0, 0), (300, 3)])
@pytest.mark.parametrize("codes,D", FEW)
def test_single_tokens(codes, D, window, first, dtype):
    lens = [600, 40, 0, 1, 17, 5000]
    cache, scale = _cache(codes, D, lens), D ** -0.5
    q = _queries(len(lens), D, scale, dtype)
    for splits in (0, 1, 3, 12):
        got = C.block_scaled_decode(q, *cache.parts(), cache.tables, cache.seq_lens, scale, num_splits=splits,
                                    window=window, first=first)
        _check(got, q, cache, [1] * len(lens), scale, window, first, torch.finfo(K.F16).eps / 2, _step(codes, D))


@pytest.mark.parametrize("codes,D", FEW)
def test_portions_of_few_tokens(codes, D):
    q_lens, lens = [4, 1, 3, 10], [600, 40, 3, 2500]
    cache, scale = _cache(codes, D, lens), D ** -0.5
    q = _queries(sum(q_lens), D, scale, K.F16)
    cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    got = C.block_scaled_prefill(q, *cache.parts(), cache.tables, cu, cache.seq_lens, scale, q_lens, lens)
    _check(got, q, cache, q_lens, scale, 0, 0, torch.finfo(K.F16).eps / 2, _step(codes, D))
