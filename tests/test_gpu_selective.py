"""Operators of a state-space mixer on the GPU against their formulas in 64 bits: types, head layouts, strides, odd
sizes, portions of one token and of none, slots and forks, neighbours full of infinities and NaN, graphs, and a
run of all of them as a mixer makes it."""
import math

import pytest
import torch

import selective_cases as S

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [BF16, F16, F32]


def _cuda(v):
    if isinstance(v, dict):
        return {k: _cuda(u) for k, u in v.items()}
    return v.cuda() if torch.is_tensor(v) else v


def _views(k):
    """x, b and c on the GPU as views of the one row that they are on the CPU."""
    row, out = k["row"].cuda(), _cuda({n: v for n, v in k.items() if n not in ("row", "x", "b", "c")})
    nx, nb = k["x"].shape[1], k["b"].shape[1]
    return dict(out, x=row[:, :nx], b=row[:, nx:nx + nb], c=row[:, nx + nb:nx + 2 * nb])


def _steps():
    return [S.step(1), S.step(5), S.step(0, [1]), S.step(0, [40, 1, 3, 17, 64]),
            S.step(3, [5, 0, 33, 2, 16], starts=[9, 0, 1, 0, 4, 1, 2, 70], behind=3),
            S.step(2, [4, 130], slots=[-1, 2, 9, 0])]


def _fill(shape, dtype):
    return torch.full(shape, S.NEW if dtype != F16 else 6e4, dtype=dtype, device="cuda")


# -- convolution ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,taps", [(64, 4), (37, 4), (1, 3), (1040, 2), (24, 8), (8, 1), (2056, 5)])
@pytest.mark.parametrize("case", range(6))
def test_convolution(case, C, taps, dtype):
    from vllm_gcu_b200.ops import cuda as K
    md = _steps()[case]
    x, w, bias, ring = S.conv_case(C, taps, md, dtype, pad=8 if C % 8 == 0 else 3, slots=2 * len(md.lens) + 1)
    R = len(md.lens)
    write = torch.where(md.state_slots >= 0, md.state_slots + R, -1).int() if case % 2 else None
    for act, bi in (("silu", bias), (None, None)):
        want, mag, new = S.conv(x[:, :C], w, bi, md, ring if taps > 1 else None, act, write)
        kept, got = ring.cuda(), _fill((x.shape[0], C), dtype)
        before = got.clone()
        K.causal_conv(x.cuda()[:, :C], w.cuda(), _cuda(bi), md.to("cuda"), kept, out=got, act=act,
                      write_slots=_cuda(write))
        n = md.tokens
        # products and sums of the taps, the exponential and the quotient (1e-6 in the fast forms)
        S.near(got[:n], want[:n], dtype, 2.0 ** -24 * (taps + 4 + 40 * (act is not None)) * (mag[:n] + 1))
        assert torch.equal(got[n:], before[n:])
        if taps > 1:
            assert torch.equal(kept.cpu(), new)


def test_convolution_portions_in_every_place():
    """Portions whose first rows lie on either side of the CTAs' strips, cut anywhere: the same bits as one prompt."""
    from vllm_gcu_b200.ops import cuda as K
    g = torch.Generator().manual_seed(3)
    w, bias = torch.randn(4, 40, generator=g).cuda(), torch.randn(40, generator=g).cuda()
    x = torch.randn(4, 70, 40, generator=g).to(BF16).cuda()
    whole = [K.causal_conv(x[i], w, bias, S.step(0, [70], [0]).to("cuda"), None) for i in range(4)]
    for cut in range(1, 36):
        ring = torch.full((4, 3, 40), math.nan, dtype=BF16, device="cuda")
        a = S.step(0, [cut, 70 - cut, 1, 33], [0] * 4, slots=[0, 1, 2, 3])
        rows = torch.cat([x[i, :n] for i, n in enumerate(a.lens)])
        one = K.causal_conv(rows, w, bias, a.to("cuda"), ring).split(a.lens)
        b = S.step(0, [70 - n for n in a.lens], a.lens, slots=[0, 1, 2, 3])
        rows = torch.cat([x[i, n:] for i, n in enumerate(a.lens)])
        two = K.causal_conv(rows, w, bias, b.to("cuda"), ring).split(b.lens)
        for i in range(4):
            assert torch.equal(torch.cat([one[i], two[i]]), whole[i]), (cut, i)


# -- scan -------------------------------------------------------------------------------
SHAPES = [("heads", 4, 64, 128, 1), ("heads", 4, 64, 64, 2), ("heads", 3, 40, 24, 1), ("heads", 2, 7, 5, 2),
          ("heads", 2, 128, 128, 2), ("heads", 1, 1, 1, 1), ("heads", 2, 33, 200, 1), ("heads", 2, 64, 256, 1),
          ("channels", 96, 1, 16, 1), ("channels", 33, 1, 16, 1), ("channels", 40, 1, 5, 2), ("channels", 64, 1, 64, 4),
          ("channels", 257, 1, 8, 1)]


def _rounding(md, N, mag, dtype, k=None):
    """See ``scan_rounding``; products of 16-bit tiles carry 2^-16 more (operands in two parts of 8 bits each, half a
    step of the lower part), and gates and step sizes of 16-bit rows go through fast exponentials (1e-6)."""
    return S.scan_rounding(md, N, mag) + (mag * (2.0 ** -15 + 4e-6) if dtype != F32 else 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,H,P,N,G", SHAPES)
@pytest.mark.parametrize("case", range(6))
def test_scan(case, form, H, P, N, G, dtype):
    from vllm_gcu_b200.ops import cuda as K
    md = _steps()[case]
    k = S.scan_case(form, H, P, N, G, md, dtype, dt32=case == 3)
    state, dev = k["state"], _views(k)
    del dev["state"]
    R = len(md.lens)
    write = torch.where(md.state_slots >= 0, md.state_slots + R, -1).int() if case % 2 else None
    for drop, more in (((), {}), (("z", "d", "dt_bias"), dict(softplus=False, dt_limits=(1e-3, 0.4)))):
        kw = {n: None if n in drop else v for n, v in k.items() if n not in ("row", "state")}
        want, mag, new, smag = S.scan(**kw, groups=G, md=md, state=state, write=write, **more)
        kept, got = state.cuda(), _fill((md.positions.shape[0], H * P), dtype)
        before = got.clone()
        K.selective_scan(**{n: None if n in drop else v for n, v in dev.items()}, groups=G, md=md.to("cuda"),
                         state=kept, out=got, write_slots=_cuda(write), **more)
        n = md.tokens
        S.near(got[:n], want[:n], dtype, _rounding(md, N, mag[:n], dtype))
        assert torch.equal(got[n:], before[n:])
        S.near(kept, new, F32, S.scan_rounding(md, N, smag))


@pytest.mark.parametrize("form,H,P,N,G", [("heads", 2, 64, 128, 1), ("heads", 2, 24, 16, 1), ("channels", 48, 1, 16, 1)])
@pytest.mark.parametrize("lens", [[127], [128], [129], [300], [1, 128, 2, 256, 65]])
def test_scan_of_longer_portions(lens, form, H, P, N, G):
    """Lengths at the edges of chunks, and strong decays: step sizes up to hundreds beside small ones."""
    from vllm_gcu_b200.ops import cuda as K
    for strong in (False, True):
        md = S.step(0, lens, [0 if i % 2 else 11 for i in range(len(lens))])
        k = S.scan_case(form, H, P, N, G, md, BF16, seed=len(lens))
        if strong:
            dt = k["dt"].float()
            some = torch.rand(dt.shape, generator=torch.Generator().manual_seed(1)) < 0.1
            k["dt"] = torch.where(some, 300.0, dt - 3).to(BF16)
        state, dev = k["state"], _views(k)
        kw = {n: v for n, v in k.items() if n not in ("row", "state")}
        want, mag, new, smag = S.scan(**kw, groups=G, md=md, state=state)
        kept = dev.pop("state")
        got = K.selective_scan(**dev, groups=G, md=md.to("cuda"), state=kept)
        S.near(got, want, BF16, _rounding(md, N, mag, BF16))
        S.near(kept, new, F32, S.scan_rounding(md, N, smag))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,H,P,N,G", [("heads", 2, 64, 128, 1), ("heads", 3, 10, 6, 1), ("channels", 40, 1, 16, 1)])
def test_neighbours_full_of_nan(form, H, P, N, G, dtype):
    """What belongs to other requests, lies in slots that nobody reads or behind the last row never shows."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [5, 70, 9], starts=[3, 4, 0, 0, 6], behind=4)
    k = S.scan_case(form, H, P, N, G, md, dtype)
    for bad in (math.nan, math.inf):
        row, dt, z = k["row"].clone(), k["dt"].clone(), k["z"].clone()
        bad_rows = list(range(77, md.positions.shape[0])) + [0]      # the last portion, what is behind it, a token
        row[bad_rows], z[bad_rows] = bad, bad
        dt[bad_rows] = math.nan
        state = k["state"].clone()
        for r in (0, 2, 3, 4):                                   # fresh portions and those of bad rows read nothing good
            state[md.state_slots[r]] = bad
        nx, nb = k["x"].shape[1], k["b"].shape[1]
        cut = lambda t: dict(x=t[:, :nx], b=t[:, nx:nx + nb], c=t[:, nx + nb:nx + 2 * nb])  # noqa: E731
        good = slice(1, 77)
        fine = S.step(1, [5, 70], starts=[4, 0, 0], slots=md.state_slots[1:4].tolist())
        kw = {n: v for n, v in k.items() if n not in ("row", "state", "x", "b", "c", "dt", "z")}
        want, mag, new, smag = S.scan(**cut(row[good]), dt=dt[good], z=z[good], **kw, groups=G, md=fine, state=state)
        kept = state.cuda()
        got = K.selective_scan(**cut(row.cuda()), dt=dt.cuda(), z=z.cuda(), **_cuda(kw), groups=G, md=md.to("cuda"),
                               state=kept)
        S.near(got[good], want, dtype, _rounding(fine, N, mag, dtype))
        for r in (1, 2, 3):
            at = int(md.state_slots[r])
            S.near(kept[at], new[at], F32, S.scan_rounding(fine, N, smag[at]))


@pytest.mark.parametrize("form,H,P,N,G", [("heads", 4, 64, 128, 1), ("channels", 80, 1, 16, 1)])
def test_without_a_state_and_with_write_slots_outside(form, H, P, N, G):
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [37, 5], starts=[4, 4, 4, 4])
    k = S.scan_case(form, H, P, N, G, md, BF16)
    dev, zero = _views(k), S.step(2, [37, 5], starts=[0] * 4)
    state = dev.pop("state")
    a = K.selective_scan(**dev, groups=G, md=md.to("cuda"), state=None)
    b = K.selective_scan(**dev, groups=G, md=zero.to("cuda"), state=state.clone())
    assert torch.equal(a, b)
    for out in (-1, state.shape[0]):
        kept = state.clone()
        K.selective_scan(**dev, groups=G, md=md.to("cuda"), state=kept,
                         write_slots=torch.full((4,), out, dtype=torch.int32, device="cuda"))
        assert torch.equal(kept, state)
    # one state read by two requests, left in two places: a fork
    same = S.dataclasses.replace(md, state_slots=torch.full_like(md.state_slots, 1)).to("cuda")
    kept, to = state.clone(), torch.tensor([4, 5, 6, 7], dtype=torch.int32, device="cuda")
    one = K.selective_scan(**dev, groups=G, md=same, state=kept, write_slots=to)
    assert torch.equal(kept[1], state[1])
    again = K.selective_scan(**dev, groups=G, md=same, state=kept, write_slots=to)
    assert torch.equal(one, again)


# -- norm -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,C,groups", [(1, 8, 1), (5, 96, 4), (3, 37, 1), (4, 111, 3), (7, 1024, 1), (2, 4096, 1),
                                        (3, 8192, 8), (2, 8200, 1), (2, 16384, 1), (1, 40008, 1), (130, 256, 8),
                                        (2, 5003, 1), (3, 2, 2)])
def test_norm(T, C, groups, dtype):
    from vllm_gcu_b200.ops import cuda as K
    g = torch.Generator().manual_seed(C)
    pad = 8 if C % 8 == 0 else 1
    x, z = (torch.randn(T, C + pad, generator=g).to(dtype)[:, :C] for _ in range(2))
    w, bias = torch.randn(C, generator=g), torch.randn(C, generator=g)
    for gate, after, center, bi, act in [(True, False, False, None, "silu"), (True, True, True, bias, "silu"),
                                         (False, False, True, bias, "silu"), (True, False, True, None, "sigmoid"),
                                         (True, True, False, None, None), (False, False, False, None, None)]:
        zz = z if gate else None
        want, mag = S.norm(x, zz, w, groups, 1e-3, bi, center, after, act)
        buf = torch.zeros(T, C + 16, dtype=dtype, device="cuda")
        # out of the way first: a part of wider rows, then in place of x
        got = K.group_norm_gate(x.cuda(), _cuda(zz), w.cuda(), groups, 1e-3, buf[:, 8:8 + C], _cuda(bi), center, after, act)
        # the sum of C / groups squares in a tree of at most C / groups / 32 + 10 steps, half of it under the root; gate,
        # products, mean; fast exponentials 2e-6 of the factor that they make
        S.near(got, want, dtype, (2.0 ** -24 * (C / groups / 32 + 30) + 4e-6 * (dtype != F32)) * mag)
        assert (buf[:, :8] == 0).all() and (buf[:, 8 + C:] == 0).all()
        xx = x.cuda()
        assert torch.equal(K.group_norm_gate(xx, _cuda(zz), w.cuda(), groups, 1e-3, xx, _cuda(bi), center, after, act), got)
    none = K.group_norm_gate(x.cuda()[:0], None, w.cuda(), groups, 1e-3)
    assert none.shape == (0, C)


# -- as a mixer uses them -----------------------------------------------------------------
class Mixer:
    """What lies between the projections of a state-space mixer."""

    def __init__(self, H, P, N, G, dtype, slots, channels=False, dev="cuda"):
        g = torch.Generator().manual_seed(0)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        D = H * P
        self.H, self.P, self.N, self.G, self.D, self.channels = H, P, N, G, D, channels
        self.w, self.bias = rnd(4, D + 2 * G * N) / 2, 0.1 * rnd(D + 2 * G * N)
        rates = D if channels else H
        self.a_log = torch.log(1 + 7 * torch.rand(*((D, N) if channels else (H,)), generator=g))
        self.d, self.dt_bias, self.norm = rnd(rates), rnd(rates) - 3, 1 + 0.1 * rnd(D)
        self.ring = torch.zeros(slots, 3, D + 2 * G * N, dtype=dtype)
        self.state = torch.zeros(slots, *((D, N) if channels else (H, P, N)))
        for n in ("w", "bias", "a_log", "d", "dt_bias", "norm", "ring", "state"):
            setattr(self, n, getattr(self, n).to(dev))

    def rows(self, T, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        steps = self.D if self.channels else self.H
        return torch.randn(T, 2 * self.D + 2 * self.G * self.N + steps, generator=g).to(dtype)

    def __call__(self, ops, row, md):
        D, gn = self.D, self.G * self.N
        z, xbc, dt = row[:, :D], row[:, D:2 * D + 2 * gn], row[:, 2 * D + 2 * gn:]
        y = ops.causal_conv(xbc, self.w, self.bias, md, self.ring)
        s = ops.selective_scan(y[:, :D], dt, y[:, D:D + gn], y[:, D + gn:], self.a_log, self.G, md, self.state, d=self.d,
                               dt_bias=self.dt_bias, z=z if self.channels else None)
        return s if self.channels else ops.group_norm_gate(s, z, self.norm, self.G, 1e-5)


@pytest.mark.parametrize("dtype,lim", [(BF16, 2.0 ** -6), (F32, 1e-4)])
@pytest.mark.parametrize("channels", [False, True])
def test_mixer_prompts_then_tokens(channels, dtype, lim):
    """Prompts in portions beside running requests, then single tokens, through all three operators; the torch
    formulation in 32 bits makes the same steps (rounding its rows to the type where the kernels do): each of the
    three roundings of a row shows with a few of its steps in the next."""
    from vllm_gcu_b200.ops import cuda as K, ref
    H, P, N, G = (96, 1, 16, 1) if channels else (4, 64, 64, 2)
    a, b = (Mixer(H, P, N, G, dtype, 5, channels, dev) for dev in ("cuda", "cpu"))
    plan = [S.step(0, [33, 140], [0, 0], [3, 1]), S.step(1, [50, 7], [33, 140, 0], [3, 1, 0]),
            S.step(3, [], [34, 190, 7], [3, 1, 0]), S.step(3, [], [35, 191, 8], [3, 1, 0])]
    for i, md in enumerate(plan):
        row = a.rows(md.tokens, dtype, i)
        got, want = a(K, row.cuda(), md.to("cuda")).float().cpu(), b(ref, row, md).float()
        assert (got - want).norm() < lim * want.norm(), (i, ((got - want).norm() / want.norm()).item())
    assert (a.state.cpu() - b.state).norm() < lim * b.state.norm()
    assert torch.isfinite(a.ring.float()).all() and torch.equal(a.ring.cpu(), b.ring)


@pytest.mark.parametrize("channels", [False, True])
def test_captured_steps_on_streams(channels):
    """A captured decode step replayed with new rows and positions, on a stream of its own; two such graphs that run at
    the same time share nothing."""
    from vllm_gcu_b200.ops import cuda as K
    H, P, N, G = (96, 1, 16, 1) if channels else (4, 64, 128, 1)
    lens = [[], [70, 9]]
    mixers = [[Mixer(H, P, N, G, BF16, 6, channels) for _ in range(2)] for _ in range(2)]
    mds = [S.step(2, lens[i], [4, 5] + [0] * len(lens[i]), list(range(2 + len(lens[i])))).to("cuda") for i in range(2)]
    rows = [mixers[i][0].rows(mds[i].tokens, BF16).cuda() for i in range(2)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        mixers[i][0](K, rows[i], mds[i])                        # warm up, then zeros again
        mixers[i][0].state.zero_(), mixers[i][0].ring.zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(mixers[i][0](K, rows[i], mds[i]))
        graphs.append(g)
    for turn in range(3):
        for i in range(2):
            rows[i].copy_(mixers[i][0].rows(mds[i].tokens, BF16, 10 * turn + i))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = mixers[i][1](K, rows[i], mds[i])
            assert torch.equal(outs[i], want)
            assert torch.equal(mixers[i][0].state, mixers[i][1].state)


def test_bits_repeat():
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(3, [200, 65], slots=list(range(5))).to("cuda")
    for form, H, P, N in (("heads", 8, 64, 128), ("channels", 200, 1, 16)):
        dev = _views(S.scan_case(form, H, P, N, 1, md, BF16))
        state = dev.pop("state")
        runs = []
        for _ in range(3):
            kept = state.clone()
            runs.append((K.selective_scan(**dev, groups=1, md=md, state=kept), kept))
        assert all(torch.equal(u, v) for r in runs[1:] for u, v in zip(runs[0], r))


# -- the far ends of what the launchers allow ---------------------------------------------
def _far_rows(rows, cols, seed=0):
    """Rows a megabyte and more apart: the last ones lie behind 2^31 elements."""
    pitch = 1 << 20
    wide = torch.empty(rows, pitch, dtype=BF16, device="cuda")
    view = wide[:, pitch - cols - 8:pitch - 8]
    view.copy_(torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(BF16))
    return view


def test_offsets_behind_32_bits():
    from vllm_gcu_b200.ops import cuda as K
    R, C = 2100, 72
    md = S.step(3, [1500, R - 1503], [5, 0, 9, 0, 3])
    x = _far_rows(R, C)
    out = _far_rows(R, C, 1)
    g = torch.Generator().manual_seed(2)
    w, bias, ring = torch.randn(4, C, generator=g), torch.randn(C, generator=g), torch.randn(5, 3, C, generator=g).to(BF16)
    K.causal_conv(x, w.cuda(), bias.cuda(), md.to("cuda"), ring.cuda(), out=out)
    near = K.causal_conv(x.contiguous(), w.cuda(), bias.cuda(), md.to("cuda"), ring.cuda())
    assert torch.equal(out, near)
    norm = K.group_norm_gate(x, x, torch.ones(C, device="cuda"), 3, 1e-5, out)
    assert torch.equal(norm, K.group_norm_gate(x.contiguous(), x.contiguous(), torch.ones(C, device="cuda"), 3, 1e-5))
    for form, H, P, N in (("heads", 1, 64, 64), ("heads", 2, 32, 8), ("channels", 64, 1, 16)):
        k = S.scan_case(form, H, P, N, 1, md, BF16)
        dev = _views(k)
        state = dev.pop("state")
        far = dict(dev, **{n: _far_rows(R, v.shape[1]) for n, v in dev.items() if n in ("x", "b", "c", "dt")})
        for n in ("x", "b", "c", "dt"):
            far[n].copy_(dev[n])
        s1, s2 = state.clone(), state.clone()
        a = K.selective_scan(**far, groups=1, md=md.to("cuda"), state=s1, out=_far_rows(R, H * P))
        b = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=s2)
        del far
        # (the far rows may go by other kernels than those that 16-byte boundaries allow)
        assert (a.float() - b.float()).norm() < 2.0 ** -8 * b.float().norm()
        assert (s1 - s2).norm() < 2e-6 * s2.norm()


@pytest.mark.parametrize("taps", [2, 4, 8])
def test_far_positions(taps):
    """A ring goes by positions of 64 bits."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [9, 3], [2 ** 33 + 5, 2 ** 31 - 1, 2 ** 40 + 1, 2 ** 31 + 6])
    x, w, bias, ring = S.conv_case(24, taps, md, BF16)
    want, mag, new = S.conv(x, w, bias, md, ring)
    kept = ring.cuda()
    got = K.causal_conv(x.cuda(), w.cuda(), bias.cuda(), md.to("cuda"), kept)
    S.near(got, want, BF16, 2.0 ** -24 * (taps + 44) * (mag + 1))
    assert torch.equal(kept.cpu(), new)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 64), ("channels", 40, 1, 16)])
def test_growing_states(form, H, P, N, dtype):
    """Step sizes below 0, where the limits allow them: states that grow."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [30, 150], [3, 0, 4, 0])
    k = S.scan_case(form, H, P, N, 1, md, dtype)
    k["a_log"] = torch.full_like(k["a_log"], -1.0)
    more = dict(softplus=False, dt_limits=(-0.02, 0.1))
    state, dev = k["state"], _views(k)
    want, mag, new, smag = S.scan(**{n: v for n, v in k.items() if n not in ("row", "state")}, groups=1, md=md, state=state,
                                  **more)
    kept = dev.pop("state")
    got = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=kept, **more)
    S.near(got, want, dtype, _rounding(md, N, mag, dtype))
    S.near(kept, new, F32, S.scan_rounding(md, N, smag))


@pytest.mark.parametrize("decodes,lens", [(6, ()), (0, (20, 3)), (2, (9,))])
@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 128), ("heads", 4, 16, 12), ("channels", 64, 1, 16),
                                        ("channels", 20, 1, 7)])
def test_weights_off_16_byte_boundaries(form, H, P, N, decodes, lens):
    """Rates, skips and biases that are parts of larger tensors, and rows that start anywhere."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(decodes, lens)
    k = S.scan_case(form, H, P, N, 1, md, BF16)
    state = k["state"]
    want, mag, new, smag = S.scan(**{n: v for n, v in k.items() if n not in ("row", "state")}, groups=1, md=md, state=state)

    def off(t):                                      # one element behind a boundary
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:].copy_(t.flatten())
        return buf[1:].view(t.shape)

    dev = {n: off(v) for n, v in k.items() if n in ("a_log", "d", "dt_bias")}
    for n in ("x", "b", "c", "dt", "z"):
        buf = torch.zeros(md.tokens, k[n].shape[1] + 5, dtype=BF16, device="cuda")
        buf[:, 3:-2] = k[n].cuda()
        dev[n] = buf[:, 3:-2]
    kept = state.cuda()
    got = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=kept)
    S.near(got, want, BF16, _rounding(md, N, mag, BF16))
    S.near(kept, new, F32, S.scan_rounding(md, N, smag))
    with pytest.raises(ValueError, match="16-byte boundary"):
        K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=off(state))


@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 128), ("heads", 2, 8, 8), ("channels", 32, 1, 16)])
def test_not_a_number_stays_one(form, H, P, N):
    """A step size that is no number leaves a state and results that are none, from its token on."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [140, 12], [4, 4, 4, 0])
    k = S.scan_case(form, H, P, N, 1, md, BF16)
    k["dt"][1], k["dt"][2 + 70] = math.nan, math.nan
    dev = _views(k)
    state = dev.pop("state")
    got = K.selective_scan(**dev, groups=1, md=md.to("cuda"), state=state).float()
    bad = torch.zeros(md.tokens, dtype=torch.bool)
    bad[1], bad[72:142] = True, True
    assert torch.isnan(got[bad.cuda()]).all() and not torch.isnan(got[~bad.cuda()]).any()
    nan = torch.isnan(state).flatten(1)
    for r, want in enumerate((False, True, True, False)):
        at = int(md.state_slots[r])
        assert bool(nan[at].all()) == want and bool(nan[at].any()) == want


def test_calls_on_another_stream_than_the_tensors():
    """Tensors made on one stream, used on another behind an event, given back to the allocator at once."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [150], [3, 4, 5]).to("cuda")
    dev = _views(S.scan_case("heads", 2, 64, 128, 1, md.to("cpu"), BF16))
    state = dev.pop("state")
    want_state, side = state.clone(), torch.cuda.Stream()
    want = K.selective_scan(**dev, groups=1, md=md, state=want_state)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.selective_scan(**dev, groups=1, md=md, state=state)
        norm = K.group_norm_gate(got, None, torch.ones(128, device="cuda"), 2, 1e-5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(state, want_state)
    assert torch.equal(norm, K.group_norm_gate(want, None, torch.ones(128, device="cuda"), 2, 1e-5))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("form,H,P,N,G", [("heads", 2, 64, 128, 1), ("heads", 2, 64, 64, 2), ("heads", 2, 8, 8, 1),
                                          ("channels", 32, 1, 16, 1)])
def test_later_tokens_never_show(form, H, P, N, G, bad):
    """A number of x, B or C that is none shows in its own token's results and, of x and B, in later ones', nowhere
    else: a token is masked from those in front of it, a column of x from the other ones."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(1, [200, 40], [3, 4, 0])
    k = S.scan_case(form, H, P, N, G, md, BF16)
    k["z"] = None
    good = _views({n: v for n, v in k.items() if v is not None})
    state = good.pop("state")
    kept = state.clone()
    want = K.selective_scan(**good, groups=G, md=md.to("cuda"), state=kept)
    first, end, col = 1 + 77, 201, 3                          # token 77 of the first portion
    for which in ("x", "b", "c"):
        dev = _views({n: v for n, v in k.items() if v is not None})
        new = dev.pop("state")
        dev[which][first, col] = bad
        got = K.selective_scan(**dev, groups=G, md=md.to("cuda"), state=new)
        hit = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
        per = H * P // G                                      # columns of B's and C's first group
        if which == "x":
            hit[first:end, col] = True
        else:
            hit[first:end if which == "b" else first + 1, :per] = True
        assert not torch.isfinite(got[hit]).any(), which
        assert torch.equal(got[~hit], want[~hit]), which
        slot = int(md.state_slots[1])
        a, b = new[slot].flatten(0, -2), kept[slot].flatten(0, -2)   # [columns, N]
        lost = torch.zeros(a.shape, dtype=torch.bool, device="cuda")
        if which == "x":
            lost[col] = True
        elif which == "b":
            lost[:per, col] = True
        assert not torch.isfinite(a[lost]).any() and torch.equal(a[~lost], b[~lost]), which


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,P,N,G", [(16, 64, 128, 2), (16, 64, 64, 1), (4, 16, 64, 1), (2, 64, 16, 1), (4, 32, 32, 2),
                                     (4, 12, 160, 1), (3, 7, 12, 1)])
def test_many_short_portions(H, P, N, G, dtype):
    """Many portions of a few tokens, some without any, beside single tokens; then two of them long enough for other
    kernels: states and results of the same formula."""
    from vllm_gcu_b200.ops import cuda as K
    for lens in ([1, 3, 0, 2, 5, 1, 1, 9, 4, 2, 0, 1], [2, 1, 140, 1], [31, 90]):
        md = S.step(3, lens, behind=2)
        k = S.scan_case("heads", H, P, N, G, md, dtype)
        state, dev = k["state"], _views(k)
        R = len(md.lens)
        write = (md.state_slots + R).int()
        want, mag, new, smag = S.scan(**{n: v for n, v in k.items() if n not in ("row", "state")}, groups=G, md=md,
                                      state=state, write=write)
        kept, got = dev.pop("state"), _fill((md.positions.shape[0], H * P), dtype)
        before = got.clone()
        K.selective_scan(**dev, groups=G, md=md.to("cuda"), state=kept, out=got, write_slots=write.cuda())
        n = md.tokens
        S.near(got[:n], want[:n], dtype, _rounding(md, N, mag[:n], dtype))
        assert torch.equal(got[n:], before[n:])
        S.near(kept, new, F32, S.scan_rounding(md, N, smag))


@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 128), ("heads", 2, 8, 16), ("channels", 32, 1, 16)])
def test_steps_of_zero_keep_the_state(form, H, P, N):
    """Tokens whose step size is 0 leave a state as it is, bit for bit; so do the places behind a portion's end."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(3, [40, 131, 1], [2, 5, 7, 1, 9, 4])
    dev = _views(S.scan_case(form, H, P, N, 1, md, F32 if P == 8 else BF16))
    state, kept = dev["state"].clone(), dev.pop("state")
    dev["dt"].zero_()
    K.selective_scan(**{**dev, "dt_bias": None}, groups=1, md=md.to("cuda"), state=kept, softplus=False)
    assert torch.equal(kept, state)


def test_long_memory():
    """A state that forgets over thousands of tokens: its decays' mean error would add up over 4000 of them."""
    from vllm_gcu_b200.ops import cuda as K
    T, D, N = 4000, 16, 16
    md = S.step(0, [T], [0])
    g = torch.Generator().manual_seed(5)
    x, b, c = (torch.randn(T, n, generator=g).abs().to(BF16) for n in (D, N, N))
    dt = torch.full((T, D), 1.5e-3)
    a_log = torch.log(torch.linspace(0.2, 1.0, N)).repeat(D, 1)
    kept = torch.zeros(1, D, N, device="cuda")
    K.selective_scan(x.cuda(), dt.cuda(), b.cuda(), c.cuda(), a_log.cuda(), 1, md.to("cuda"), kept, softplus=False)
    want = torch.zeros(D, N, dtype=S.F64)
    keep = torch.exp(-dt[0, 0].double() * torch.exp(a_log.double()))
    for t in range(T):
        want = keep * want + (dt[t].double() * x[t].double())[:, None] * b[t].double()
    # terms last 1 / (1 - keep) = 670 to 3300 tokens; a decay is off by half a step and less than that on average
    err = (kept[0].cpu().double() / want - 1).abs()
    assert err.max() < 3300 * 2.0 ** -25 + 2.0 ** -20, err.max().item()


@pytest.mark.parametrize("form,H,P,N", [("heads", 2, 64, 128), ("heads", 2, 32, 8), ("channels", 64, 1, 16)])
def test_rows_that_are_one(form, H, P, N):
    """Rows of an expanded tensor are all the same memory."""
    from vllm_gcu_b200.ops import cuda as K
    md = S.step(2, [150, 3]).to("cuda")
    dev = _views(S.scan_case(form, H, P, N, 1, md.to("cpu"), BF16))
    state, T = dev.pop("state"), md.tokens
    one = dict(dev, **{n: dev[n][:1].contiguous().expand(T, -1) for n in ("x", "b", "c", "dt", "z")})
    kept, want_kept = state.clone(), state.clone()
    got = K.selective_scan(**one, groups=1, md=md, state=kept)
    want = K.selective_scan(**{n: v.contiguous() if torch.is_tensor(v) else v for n, v in one.items()}, groups=1, md=md,
                            state=want_kept)
    # (another kernel may take them: each result is half a step of its type off, and states what 32 bits leave of sums)
    assert (got.float() - want.float()).norm() <= 2.0 ** -8 * want.float().norm()
    assert (kept - want_kept).norm() <= 2e-6 * want_kept.norm()
    x = one["x"]
    w, ones = torch.randn(4, x.shape[1], device="cuda"), torch.ones(x.shape[1], device="cuda")
    ring = torch.zeros(state.shape[0], 3, x.shape[1], dtype=BF16, device="cuda")
    assert torch.equal(K.causal_conv(x, w, None, md, ring), K.causal_conv(x.contiguous(), w, None, md, ring.zero_()))
    assert torch.equal(K.group_norm_gate(x, x, ones, 2, 1e-5), K.group_norm_gate(x.contiguous(), x.contiguous(), ones, 2, 1e-5))
