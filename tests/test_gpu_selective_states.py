"""States of the selective scan as near to 64 bits as each of its kernels is to leave them: three parts of bf16 and sums in
two floats by tiles, a few roundings a token elsewhere, step sizes to the last bits of fp32."""
import pytest
import torch

import selective_cases as S
import selective_states as E

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _scan(k, lens, starts, slots=None, **kw):
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(0, lens, starts, slots=list(range(len(lens))) if slots is None else slots).to("cuda")
    kept = k["state"].cuda()
    K.selective_scan(**{n: k[n].cuda() for n in ("x", "dt", "b", "c", "a_log")}, md=md, state=kept,
                     **{**dict(groups=1, softplus=False), **kw})
    return kept


@pytest.mark.parametrize("kind,lens", [(kind, lens) for kind in ("signs", "strong") for lens in
                                       ([128], [129, 127], [400], [64, 1000])] + [("long", [4000]), ("long", [130])])
@pytest.mark.parametrize("N", [64, 128])
def test_states_by_tiles(N, kind, lens):
    k = E.heads_case(N, lens, kind, seed=len(lens))
    starts = [0 if kind == "long" else 5] * len(lens)
    want, _ = E.states(k["x"], k["dt"], k["b"], k["a_log"], 1, lens, starts, k["state"])
    assert E.norm_error(_scan(k, lens, starts), want) < E.chunk_bound(lens)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 40, 64), ("heads", 2, 64, 100), ("heads", 4, 16, 16), ("heads", 2, 64, 256),
                                        ("channels", 96, 1, 16), ("channels", 40, 1, 7), ("channels", 40, 1, 128)])
def test_states_token_after_token(form, H, P, N, dtype):
    lens, starts = [600, 45], [3, 0]
    g = torch.Generator().manual_seed(N)
    k = S.scan_case(form, H, P, N, 1, S.step(0, lens), dtype, slots=2)
    k["dt"] = torch.exp(-6.9 + 4.6 * torch.rand(sum(lens), H, generator=g))
    want, off = E.states(k["x"], k["dt"], k["b"], k["a_log"], 1, lens, starts, k["state"])
    got = _scan(k, lens, starts).cpu().to(E.F64)
    assert ((got - want).abs() <= off).all(), ((got - want).abs() / off).max().item()


@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 128), ("heads", 4, 16, 64), ("heads", 3, 7, 12), ("channels", 96, 1, 16),
                                        ("channels", 40, 1, 7)])
@pytest.mark.parametrize("decode", [True, False])
def test_states_of_single_tokens_and_short_portions(form, H, P, N, decode):
    """One portion cut into a call for each token or into short ones that many requests have beside it."""
    T = 60
    g = torch.Generator().manual_seed(N + 1)
    k = S.scan_case(form, H, P, N, 1, S.step(0, [T]), F32, slots=1)
    k["dt"] = torch.exp(-6.9 + 4.6 * torch.rand(T, H, generator=g))
    want, off = E.states(k["x"], k["dt"], k["b"], k["a_log"], 1, [T], [9], k["state"])
    from vllm_gcu_b200.ops import cuda as K
    kept, dev = k["state"].cuda(), {n: k[n].cuda() for n in ("x", "dt", "b", "c", "a_log")}
    step = 1 if decode else 4
    for t in range(0, T, step):
        md = (S.step(1, [], [9 + t], slots=[0]) if decode else S.step(0, [step], [9 + t], slots=[0])).to("cuda")
        K.selective_scan(**{n: v if n == "a_log" else v[t:t + step] for n, v in dev.items()}, groups=1, md=md, state=kept,
                         softplus=False)
    got = kept.cpu().to(E.F64)
    assert ((got - want).abs() <= off).all(), ((got - want).abs() / off).max().item()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("form", ["heads", "channels"])
def test_step_sizes(form, decode, dtype):
    """log(1 + e^v) of every kind of v: with x and B of 1 a state of zeros becomes the step size.  16-bit rows: a power of two
    that is off by 2 steps at most, a polynomial by 1.2e-8 and three roundings, 2^-22 + 1.2e-8 + 3 * 2^-24 < 2^-21; fp32 rows: 2
    steps each of the exponential and of the logarithm and a sum's rounding, less than 2^-20.8."""
    from vllm_gcu_b200.ops import cuda as K
    T, D, N = 64, 2048, 4
    v = torch.cat([torch.linspace(-85, 95, T * D // 2), torch.linspace(-4, 4, T * D // 4),
                   torch.logspace(-30, 0, T * D // 8, base=2), -torch.logspace(-30, 0, T * D // 8, base=2)])
    v = v[torch.randperm(T * D, generator=torch.Generator().manual_seed(0))].view(T, D)
    one = torch.ones(T, D, dtype=dtype, device="cuda")
    a_log = torch.zeros(D, N) if form == "channels" else torch.zeros(D)
    md = S.step(T if decode else 0, [] if decode else [1] * T, [0] * T, slots=list(range(T))).to("cuda")
    kept = torch.full((T, D, N) if form == "channels" else (T, D, 1, N), 7.0, device="cuda")
    K.selective_scan(one, v.cuda(), one[:, :N], one[:, :N], a_log.cuda(), 1, md, kept)
    want = torch.logaddexp(v.to(E.F64), torch.zeros(T, D, dtype=E.F64))
    for n in range(N):
        got = kept.view(T, D, N)[..., n].cpu().to(E.F64)
        off = (got / want - 1).abs().max().item()
        assert off < (2.0 ** -20.8 if dtype == F32 else 2.0 ** -21), off


@pytest.mark.parametrize("step", [1, 8, 4000])
@pytest.mark.parametrize("dtype,form,H,P,N", [(F32, "heads", 4, 8, 16), (F32, "heads", 4, 64, 64), (F16, "heads", 4, 40, 64),
                                              (F32, "heads", 3, 7, 5)])
def test_rates_per_head_over_thousands_of_tokens(dtype, form, H, P, N, step):
    """A prompt, short portions and single tokens whose states forget a part in 600 to 3000 a token.  Decays and sums
    are rounded by half a step (2^-25 on average over all roundings' sizes) either way, so that of some 3000 tokens
    that a state holds, two roundings each, sqrt(2 * 3000) * 2^-25 shows, 2.3e-6; twice that for the largest of a few
    hundred numbers, which share their decays.  A mean error of 1.5e-8 of a decay would leave 1500 times as much, 2.3e-5."""
    from vllm_gcu_b200.ops import cuda as K
    T = 4000
    g = torch.Generator().manual_seed(7)
    x, b = (torch.randn(T, n, generator=g).abs().to(dtype) for n in (H * P, N))
    dt = 1e-3 + 1e-3 * torch.rand(T, H, generator=g)
    a_log = torch.log(torch.linspace(0.2, 1.0, H))
    want, _ = E.states(x, dt, b, a_log, 1, [T], [0], torch.zeros(1, H, P, N))
    kept = torch.zeros(1, H, P, N, device="cuda")
    dev = [t.cuda() for t in (x, dt, b, b)]
    rates = a_log.cuda()
    for t in range(0, T, step):
        md = S.step(*((1, []) if step == 1 else (0, [step])), [t], slots=[0]).to("cuda")
        K.selective_scan(*(v[t:t + step] for v in dev), rates, 1, md, kept, softplus=False)
    worst = (kept.cpu().to(E.F64) / want - 1).abs().max().item()
    assert worst < 4.6e-6
