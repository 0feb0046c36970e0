"""State-space operators of the torch formulation at the ends of their inputs' ranges."""
import pytest
import torch

import selective_cases as S
from vllm_gcu_b200.ops import ref

F32 = torch.float32


@pytest.mark.parametrize("form,H,P,N,G", [("heads", 2, 3, 4, 1), ("channels", 6, 1, 3, 3)])
def test_large_and_small_step_sizes(form, H, P, N, G):
    """Raw step sizes whose exponential 32 bits do not hold: log(1 + e^v) is v there, and e^v far below 0."""
    md = S.step(2, [7], [3, 0, 4])
    k = S.scan_case(form, H, P, N, G, md, F32)
    state = k.pop("state")
    k.pop("row")
    k["dt"][0], k["dt"][3], k["dt"][4], k["dt"][6] = 89.0, 120.0, 3e4, -30.0
    want, mag, new, smag = S.scan(**k, groups=G, md=md, state=state)
    kept = state.clone()
    got = ref.selective_scan(**k, groups=G, md=md, state=kept)
    S.near(got, want, F32, S.scan_rounding(md, N, mag))
    S.near(kept, new, F32, S.scan_rounding(md, N, smag))


@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 3, 4), ("channels", 6, 1, 3)])
def test_a_state_without_slots(form, H, P, N):
    md = S.step(2, [3])
    k = S.scan_case(form, H, P, N, 1, md, F32)
    k.pop("row")
    state = k.pop("state")[:0]
    assert (ref.selective_scan(**k, groups=1, md=md, state=state) == 0).all()
    x, w, bias, ring = S.conv_case(6, 4, md, F32)
    assert (ref.causal_conv(x, w, bias, md, ring[:0]) == 0).all()
