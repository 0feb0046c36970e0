"""State-space operators of the torch formulation at the ends of their inputs' ranges."""
import math

import pytest
import torch

import selective_cases as S
import selective_states as E
from vllm_gcu_b200.ops import cuda as C, ref

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


def test_results_do_not_go_into_what_is_kept():
    """Rows of results that meet the ring or the state, which other requests read at the same time, are refused; a state
    between two rows of results is none of theirs."""
    md = S.step(1, [3])
    T = md.tokens
    x, w, bias, _ = S.conv_case(8, 4, md, F32)
    buf = torch.zeros(64 * 8)
    ring = buf[:6 * 3 * 8].view(6, 3, 8)
    conv = lambda out: C.causal_conv(x, w, bias, md, ring, out=out)  # noqa: E731
    last = buf[17 * 8 + 7:]
    for out in (buf[:T * 8].view(T, 8), last[:T * 8].view(T, 8), buf.as_strided((T, 8), (17 * 8, 1), 40)):
        with pytest.raises(ValueError, match="shares memory with ring"):
            conv(out)
    k = S.scan_case("heads", 2, 4, 4, 1, md, F32)
    k.pop("row"), k.pop("state")
    mem = torch.zeros(4096)
    state = mem[1000:1000 + 4 * 32].view(4, 2, 4, 4)
    scan = lambda out: C.selective_scan(**k, groups=1, md=md, state=state, out=out)  # noqa: E731
    for first, pitch in ((1000, 8), (993, 900), (0, 1000), (1127, 500), (500, 300)):
        with pytest.raises(ValueError, match="shares memory with state"):
            scan(mem.as_strided((T, 8), (pitch, 1), first))
    for first, pitch in ((992, 1128 - 992), (1128, 8), (968, 8), (0, 800)):
        with pytest.raises(ValueError, match="on a GPU"):
            scan(mem.as_strided((T, 8), (pitch, 1), first))
    # every place of four rows beside a block, against the elements themselves
    for pitch in (8, 11, 30):
        for lo in range(0, 140, 3):
            for size in (1, 5, 40):
                rows = {i * pitch + j + 20 for i in range(4) for j in range(8)}
                assert C._rows_meet(20, pitch, 4, 8, lo, size) == bool(rows & set(range(lo, lo + size)))


@pytest.mark.parametrize("kind", ["signs", "strong"])
@pytest.mark.parametrize("N", [64, 128])
@pytest.mark.parametrize("lens", [[128], [129, 127], [400]])
def test_bounds_of_states_tell_mistakes(lens, N, kind):
    """What the GPU tests ask of states by products of tiles holds for weighted x in three parts of bf16 and sums in two
    floats, not for two parts, and behind strong decays not for sums in one float."""
    k = E.heads_case(N, lens, kind)
    k.pop("row"), k.pop("c")
    starts = [5] * len(lens)
    args = dict(x=k["x"], dt=k["dt"], b=k["b"], a_log=k["a_log"], lens=lens, starts=starts, state=k["state"])
    want, off = E.states(**args, groups=1)
    bound = E.chunk_bound(lens)
    whole = E.by_chunks(**args)
    assert E.norm_error(whole, want) < bound / 4
    assert E.norm_error(E.by_chunks(**args, parts=2), want) > 1.5 * bound
    if kind == "strong":
        assert E.norm_error(E.by_chunks(**args, two_floats=False), want) > 50 * bound
    # and the torch formulation holds the bounds of each number
    md = S.step(0, lens, starts, slots=list(range(len(lens))))
    kept = k["state"].clone()
    ref.selective_scan(**{n: k[n] for n in ("x", "dt", "b", "a_log")}, c=k["b"], groups=1, md=md, state=kept, softplus=False)
    assert ((kept.to(E.F64) - want).abs() <= off).all()


def test_limits_of_step_sizes():
    md = S.step(0, [3])
    k = S.scan_case("heads", 2, 3, 4, 1, md, F32)
    k.pop("row")
    for limits, says in [((-math.inf, math.inf), "on a GPU"), ((-1e300, 0.5), "on a GPU"), ((0.0, 1e300), "on a GPU"),
                         ((math.inf, math.inf), "dt_limits"), ((-math.inf, -math.inf), "dt_limits"),
                         ((math.nan, 1.0), "dt_limits"), ((0.0, math.nan), "dt_limits"), ((1.0, 0.0), "dt_limits")]:
        with pytest.raises(ValueError, match=says):
            C.selective_scan(**k, groups=1, md=md, softplus=False, dt_limits=limits)


def test_arguments_without_dimensions_or_positions():
    md = S.step(1, [3])
    x, w, bias, ring = S.conv_case(8, 4, md, F32)
    conv = lambda **k: C.causal_conv(**{**dict(x=x, weight=w, bias=bias, md=md, ring=ring), **k})  # noqa: E731
    one = torch.tensor(1.0)
    none = S.dataclasses.replace(md, positions=None)
    for k, says in [(dict(weight=one), "0 taps"), (dict(ring=one), "ring"), (dict(bias=one), "bias"), (dict(x=one), "x:"),
                    (dict(md=none), "positions"), (dict(out=one), "out")]:
        with pytest.raises(ValueError, match=says):
            conv(**k)
    k = S.scan_case("heads", 2, 3, 4, 1, md, F32)
    k.pop("row")
    for more, says in [({n: one}, n) for n in ("x", "dt", "b", "c", "a_log", "d", "dt_bias", "z", "state")] + \
            [(dict(md=none), "positions")]:
        with pytest.raises(ValueError, match=says):
            C.selective_scan(**{**k, **dict(groups=1, md=md), **more})
    for more, says in [({n: one}, n) for n in ("x", "z", "weight", "bias")]:
        with pytest.raises(ValueError, match=says):
            C.group_norm_gate(**{**dict(x=x, z=x, weight=torch.ones(8), groups=2, eps=1e-5), **more})
