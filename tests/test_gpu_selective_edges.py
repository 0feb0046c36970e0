"""State-space operators at the ends of what their launchers allow."""
import pytest
import torch

import selective_cases as S

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


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
