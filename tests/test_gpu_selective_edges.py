"""State-space operators at the ends of what their launchers allow."""
import math

import pytest
import torch

import selective_cases as S

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _on_gpu(k):
    """A case's tensors on the GPU, x, b and c as parts of one row again."""
    row, out = k["row"].cuda(), {n: v.cuda() for n, v in k.items() if n not in ("row", "x", "b", "c")}
    nx, nb = k["x"].shape[1], k["b"].shape[1]
    return dict(out, x=row[:, :nx], b=row[:, nx:nx + nb], c=row[:, nx + nb:nx + 2 * nb])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("decodes,lens", [(3, ()), (0, (140, 2)), (2, (5, 1))])
@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 128), ("heads", 2, 7, 5), ("channels", 40, 1, 16),
                                        ("channels", 20, 1, 7)])
def test_a_state_without_slots(form, H, P, N, decodes, lens, dtype):
    """Every slot lies outside a state or ring of no slots: rows of zeros."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(decodes, lens)
    dev = _on_gpu(S.scan_case(form, H, P, N, 1, md, dtype))
    state = dev.pop("state")[:0]
    got = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=state)
    assert got.shape == (md.tokens, H * P) and (got == 0).all()
    ring = torch.empty(0, 3, H * P, dtype=dtype, device="cuda")
    got = K.causal_conv(dev["x"], torch.randn(4, H * P, device="cuda"), torch.ones(H * P, device="cuda"), md.to("cuda"), ring)
    assert got.shape == (md.tokens, H * P) and (got == 0).all()


@pytest.mark.parametrize("dtype,H,P,N", [(F32, 4, 64, 128), (F16, 16, 64, 128), (BF16, 4, 64, 16), (BF16, 8, 32, 64)])
@pytest.mark.parametrize("many", [3, 9, 15])
def test_a_long_portion_beside_short_ones(many, dtype, H, P, N):
    """A portion that is long beside those of one token takes the way that it takes alone, where many tokens are not one
    slow walk: the same bits.  (The walk for short portions sums in another order.)"""
    from vllm_gcu_b200.ops import cuda as K
    long = 30 * many
    md = S.step(0, [long] + [1] * many, [5] * (many + 1), slots=list(range(many + 1)))
    k = S.scan_case("heads", H, P, N, 1, md, dtype)
    dev = _on_gpu(k)
    state = dev.pop("state")
    both, alone = state.clone(), state.clone()
    got = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=both)
    cut = {n: v[:long] if n in ("x", "b", "c", "dt", "z") else v for n, v in dev.items()}
    want = K.selective_scan(**cut, groups=1, md=S.step(0, [long], [5], slots=[0]).to("cuda"), state=alone)
    assert torch.equal(got[:long], want) and torch.equal(both[0], alone[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 64), ("channels", 40, 1, 16)])
@pytest.mark.parametrize("limits,softplus", [((-math.inf, math.inf), False), ((-1e300, 0.05), False), ((-0.01, 1e300), False),
                                             ((-math.inf, math.inf), True), ((-3.0, 0.2), True), ((-3.0, -0.01), True)])
def test_limits_of_step_sizes(limits, softplus, form, H, P, N, dtype):
    """Limits that limit nothing, on either side, and those below 0, as single tokens and portions take them."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [30, 150], [3, 0, 4, 0])
    k = S.scan_case(form, H, P, N, 1, md, dtype)
    k["a_log"] = torch.full_like(k["a_log"], -1.0)
    if not softplus:
        k["dt"], k["dt_bias"] = (0.02 * k["dt"].float()).to(dtype), None
    state, dev = k["state"], _on_gpu({n: v for n, v in k.items() if v is not None})
    dev.setdefault("dt_bias", None)
    more = dict(softplus=softplus, dt_limits=limits)
    want, mag, new, smag = S.scan(**{n: v for n, v in k.items() if n not in ("row", "state")}, groups=1, md=md, state=state,
                                  **more)
    kept = dev.pop("state")
    got = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=kept, **more)
    S.near(got, want, dtype, S.scan_rounding(md, N, mag) + (mag * (2.0 ** -15 + 4e-6) if dtype != F32 else 0))
    S.near(kept, new, F32, S.scan_rounding(md, N, smag))


@pytest.mark.parametrize("N", [64, 128])
def test_limits_below_zero_leave_softplus_its_way(N):
    """A softplus is not below 0, so a limit below 0 changes nothing: the same bits."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(0, [200], [0]).to("cuda")
    dev = _on_gpu(S.scan_case("heads", 2, 64, N, 1, md, BF16))
    state = dev.pop("state")
    a, b = (K.selective_scan(**dev, groups=1, md=md, state=state.clone(), dt_limits=(lo, math.inf)) for lo in (0.0, -1.0))
    assert torch.equal(a, b)
