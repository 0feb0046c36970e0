"""Operators of a state-space mixer on the CPU: the torch formulation against the formulas in 64 bits, portions against
whole prompts, forks, and what the launchers refuse."""
import math

import pytest
import torch

import selective_cases as S
from vllm_gcu_b200.ops import cuda as C, ref

F32, BF16 = torch.float32, torch.bfloat16


def steps():
    return [S.step(3), S.step(0, [7, 1, 20]), S.step(2, [5, 0, 3, 2], starts=[9, 0, 0, 4, 1, 2], behind=2),
            S.step(2, [4, 6], slots=[-1, 2, 9, 0])]


@pytest.mark.parametrize("taps", [1, 2, 4, 8])
@pytest.mark.parametrize("case", range(4))
def test_convolution(case, taps):
    md = steps()[case]
    x, w, bias, ring = S.conv_case(6, taps, md, F32, slots=5)
    for act, bi in (("silu", bias), (None, None)):
        want, mag, new = S.conv(x, w, bi, md, ring if taps > 1 else None, act)
        got, kept = torch.full_like(x, S.NEW), ring.clone()
        ref.causal_conv(x, w, bi, md, kept, out=got, act=act)
        S.near(got, want, F32, 2.0 ** -24 * (taps + 12) * mag)
        if taps > 1:
            assert torch.equal(kept, new)


def test_convolution_of_portions_and_forks():
    g = torch.Generator().manual_seed(1)
    x, w, bias = torch.randn(23, 5, generator=g), torch.randn(4, 5, generator=g), torch.randn(5, generator=g)
    whole, mag, _ = S.conv(x, w, bias, S.step(0, [23], [0]), torch.zeros(1, 3, 5))
    ring, at, got = torch.full((3, 3, 5), math.nan), 0, []
    for i, n in enumerate([1, 1, 5, 2, 1, 9, 4]):        # every portion reads one slot and writes another
        md = S.step(0, [n], [at], slots=[i % 3])
        got.append(ref.causal_conv(x[at:at + n], w, bias, md, ring,
                                   write_slots=torch.tensor([(i + 1) % 3], dtype=torch.int32)))
        at += n
    # (not to the bit: the CPU's vector exponential is another one than that of the elements behind the last vector)
    S.near(torch.cat(got), whole, F32, 2.0 ** -24 * 16 * mag)


@pytest.mark.parametrize("form,H,P,N,G", [("heads", 4, 3, 5, 2), ("channels", 6, 1, 4, 1), ("channels", 6, 1, 3, 3)])
@pytest.mark.parametrize("case", range(4))
def test_scan(case, form, H, P, N, G):
    md = steps()[case]
    k = S.scan_case(form, H, P, N, G, md, F32, slots=5)
    state = k.pop("state")
    k.pop("row")
    for drop, more in (((), {}), (("z", "d", "dt_bias"), dict(softplus=False, dt_limits=(1e-3, 0.4)))):
        kw = {n: None if n in drop else v for n, v in k.items()}
        want, mag, new, smag = S.scan(**kw, groups=G, md=md, state=state, **more)
        got, kept = torch.full_like(want, S.NEW, dtype=F32), state.clone()
        ref.selective_scan(**kw, groups=G, md=md, state=kept, out=got, **more)
        S.near(got, want, F32, S.scan_rounding(md, N, mag))
        S.near(kept, new, F32, S.scan_rounding(md, N, smag))


def test_scan_of_portions_and_forks():
    md = S.step(0, [19], [0])
    k = S.scan_case("heads", 2, 3, 4, 1, md, F32)
    k.pop("row"), k.pop("state")
    whole, mag, _, _ = S.scan(**k, groups=1, md=md, state=torch.full((1, 2, 3, 4), math.nan))
    state, at, got = torch.full((2, 2, 3, 4), math.nan), 0, []
    for i, n in enumerate([1, 4, 1, 13]):
        cut = {m: v[at:at + n] if m in ("x", "b", "c", "dt", "z") else v for m, v in k.items()}
        got.append(ref.selective_scan(**cut, groups=1, md=S.step(0, [n], [at], slots=[i % 2]), state=state,
                                      write_slots=torch.tensor([(i + 1) % 2], dtype=torch.int32)))
        at += n
    S.near(torch.cat(got), whole, F32, S.scan_rounding(md, 4, mag))
    # without a state a portion starts from zeros, wherever it says it is
    again = ref.selective_scan(**k, groups=1, md=S.step(0, [19], [7]), state=None)
    S.near(again, whole, F32, S.scan_rounding(md, 4, mag))


@pytest.mark.parametrize("groups,center,after,gate,act", [
    (1, False, False, True, "silu"), (4, False, False, True, "silu"), (3, True, True, True, "sigmoid"),
    (2, True, False, False, "silu"), (12, False, True, True, None), (1, True, False, False, None)])
def test_norm(groups, center, after, gate, act):
    g = torch.Generator().manual_seed(groups)
    x, z = torch.randn(5, 12, generator=g), torch.randn(5, 12, generator=g)
    w, bias = torch.randn(12, generator=g), torch.randn(12, generator=g) if center else None
    want, mag = S.norm(x, z if gate else None, w, groups, 1e-3, bias, center, after, act)
    got = ref.group_norm_gate(x, z if gate else None, w, groups, 1e-3, None, bias, center, after, act)
    # squares and their sum: 12 + 4 roundings of the variance, half of which reach the root; its inverse, the
    # products, the gate's exponential and quotient
    S.near(got, want, F32, 2.0 ** -24 * 32 * mag)


def test_refusals():
    md = S.step(1, [4])
    x, w, bias, ring = S.conv_case(8, 4, md, BF16)
    conv = lambda **k: C.causal_conv(**{**dict(x=x, weight=w, bias=bias, md=md, ring=ring), **k})  # noqa: E731
    many = torch.zeros(9, 8)
    for k, says in [(dict(weight=many), "9 taps"), (dict(x=x.double()), "bf16, fp16 or fp32"), (dict(act="gelu"), "gelu"),
                    (dict(bias=bias[:4]), "bias"), (dict(ring=ring.float()), "ring"), (dict(out=x), "shares memory"),
                    (dict(x=x.t().contiguous().t()), "apart"), (dict(out=torch.empty(5, 4, dtype=BF16)), "out"),
                    (dict(out=torch.empty(1, 8, dtype=BF16).expand(5, 8)), "apart"), (dict(weight=w.to(BF16)), "weight"),
                    (dict(write_slots=md.state_slots.long()), "write_slots"),
                    (dict(write_slots=md.state_slots[:1]), "write_slots"),
                    (dict(md=S.dataclasses.replace(md, state_slots=None)), "state_slots"),
                    (dict(md=S.dataclasses.replace(md, positions=md.positions.int())), "positions"),
                    (dict(md=S.dataclasses.replace(md, positions=md.positions[:2])), "positions"),
                    (dict(md=S.dataclasses.replace(md, cu_q_prefill=md.cu_q_prefill.long())), "cu_q"),
                    (dict(md=S.dataclasses.replace(md, num_decode_tokens=6)), "single tokens"), ({}, "on a GPU")]:
        with pytest.raises(ValueError, match=says):
            conv(**k)
    for form in ("heads", "channels"):
        P = 3 if form == "heads" else 1
        c = S.scan_case(form, 4, P, 4, 2, md, BF16)
        row = c.pop("row")
        scan = lambda **k: C.selective_scan(**{**c, **dict(groups=2, md=md), **k})  # noqa: E731
        for k, says in [(dict(groups=3), "groups"), (dict(x=c["x"].float()), "b is|z is|bfloat16"), (dict(groups=0), "groups"),
                        (dict(dt=c["dt"].half()), "dt is"), (dict(dt=c["dt"][:, :3]), "dt has"),
                        (dict(b=c["b"][:, :4]), "has shape|a_log|state"), (dict(c=c["c"][:3]), "c has"),
                        (dict(a_log=c["a_log"].double()), "a_log"), (dict(d=c["d"][:2]), "d:"),
                        (dict(dt_bias=c["dt_bias"].to(BF16)), "dt_bias"), (dict(state=c["state"][:, :, ..., :3]), "state"),
                        (dict(state=c["state"].to(BF16)), "state"), (dict(out=c["x"]), "shares memory with x"),
                        (dict(out=c["z"]), "shares memory with z"), (dict(dt_limits=(2.0, 1.0)), "dt_limits"),
                        (dict(x=c["x"][:, :-1]), "rates|has shape"),
                        (dict(b=torch.zeros(5, 2 * 300, dtype=BF16), c=torch.zeros(5, 2 * 300, dtype=BF16)), "300"),
                        ({}, "on a GPU")]:
            with pytest.raises(ValueError, match=says):
                scan(**k)
        # columns of one buffer that do not meet are no overlap
        wide = torch.zeros(5, row.shape[1] + 4 * P, dtype=BF16)
        meet = lambda u, v: C._overlap(*((t.data_ptr(), t.stride(0), *t.shape, 2) for t in (u, v)))  # noqa: E731
        assert not meet(wide[:, :4 * P], wide[:, 4 * P:]) and not meet(wide[:, 4 * P:], wide[:, :4 * P])
        assert meet(wide[:, :4 * P + 1], wide[:, 4 * P:]) and meet(wide[:, 4 * P:], wide[:, 1:4 * P + 1])
        assert not meet(wide[:2], wide[2:]) and meet(wide[:3], wide[2:]) and not meet(wide[:0], wide)
    z, w8 = torch.randn_like(x), torch.ones(8)
    norm = lambda **k: C.group_norm_gate(**{**dict(x=x, z=z, weight=w8, groups=2, eps=1e-5), **k})  # noqa: E731
    for k, says in [(dict(groups=3), "groups"), (dict(groups=0), "groups"), (dict(act="gelu"), "gelu"),
                    (dict(z=z.float()), "z is"), (dict(z=z[:4]), "z has"), (dict(weight=w8[:4]), "weight"),
                    (dict(bias=w8.to(BF16)), "bias"), (dict(x=x.double()), "bf16"), ({}, "on a GPU")]:
        with pytest.raises(ValueError, match=says):
            norm(**k)
    buf = torch.zeros(6, 8, dtype=BF16)
    with pytest.raises(ValueError, match="is not x"):
        norm(x=buf[:5], z=None, out=buf[1:])
    with pytest.raises(ValueError, match="on a GPU"):
        norm(out=x)                                          # in place is fine


def test_too_many_requests():
    T = 65536
    md = S.Step(torch.zeros(T, dtype=torch.int64), torch.zeros(T, dtype=torch.int32), T, None, [1] * T, [0] * T)
    one = torch.zeros(T, 1, dtype=BF16)
    with pytest.raises(ValueError, match="65536 requests"):
        C.selective_scan(one, one, one, one, torch.zeros(1), 1, md, None)
