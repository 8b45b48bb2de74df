"""gated_scan, its gradient and gated_step against the recursion in 64 bits, with bounds carried through the recursion."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
# Roundings of a step, in half steps of float32: the gate and its rest each take exp (2, and as many as its argument's size, below 20
# here), a sum and a quotient or product; then two products and a sum.  A product of n gates is off by n times as much as one, which
# is what n steps in turn give as well, so the bound holds for any way of joining parts of a sequence.
STEP = 32.0


def _reference(x, gate, state, lengths, gy=None, gf=None):
    """float64: y, final, dx, dgate, dstate and a bound on each one's error, steps in turn."""
    x, g = x.double().cpu(), gate.double().cpu()
    B, T, D = x.shape
    n = torch.full((B,), T) if lengths is None else lengths.cpu().clamp(0, T)
    h = torch.zeros(B, D, dtype=torch.float64) if state is None else state.double().cpu()
    a, rest = torch.sigmoid(g), torch.sigmoid(-g)
    e = torch.zeros_like(h)
    y, ye, before, be = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        on = (t < n)[:, None]
        before[:, t], be[:, t] = h, e
        new = a[:, t] * h + rest[:, t] * x[:, t]
        new_e = a[:, t] * e + STEP * U * (a[:, t] * h.abs() + rest[:, t] * x[:, t].abs())
        h, e = torch.where(on, new, h), torch.where(on, new_e, e)
        y[:, t], ye[:, t] = torch.where(on, h, 0.0), torch.where(on, e, 0.0)
    out = {"y": (y, ye), "final": (h, e)}
    if gy is None and gf is None:
        return out
    gy = torch.zeros_like(x) if gy is None else gy.double().cpu()
    u = torch.zeros_like(h) if gf is None else gf.double().cpu()
    s = torch.zeros_like(h)                                  # error of u
    dx, dxe, dg, dge = (torch.zeros_like(x) for _ in range(4))
    for t in range(T - 1, -1, -1):
        on = (t < n)[:, None]
        w = u + gy[:, t]
        ws = s + U * STEP * (u.abs() + gy[:, t].abs())
        dx[:, t] = torch.where(on, rest[:, t] * w, 0.0)
        dxe[:, t] = torch.where(on, rest[:, t] * (ws + STEP * U * w.abs()), 0.0)
        lead, k = before[:, t] - x[:, t], a[:, t] * rest[:, t]
        dg[:, t] = torch.where(on, w * lead * k, 0.0)
        dge[:, t] = torch.where(on, k * (ws * lead.abs() + w.abs() * (be[:, t] + U * before[:, t].abs()) + 3 * STEP * U * (w * lead).abs()), 0.0)
        u, s = torch.where(on, a[:, t] * w, u), torch.where(on, a[:, t] * (ws + STEP * U * w.abs()), s)
    half, tiny = HALF[gate.dtype], TINY[gate.dtype]
    out.update(dx=(dx, dxe), dgate=(dg, dge + half * dg.abs() * 1.01 + tiny), dstate=(u, s))
    return out


def _close(got, want, what):
    value, bound = want
    bad = (got.double().cpu() - value).abs() > bound * 1.05 + 1e-38
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def _case(B, T, D, dtype=torch.float32, state=True, lengths=None, seed=0):
    gen = torch.Generator().manual_seed(seed + 31 * B + 7 * T + D)
    x = torch.exp(torch.rand(B, T, D, generator=gen)).to(DEV)
    gate = (1.5 + 2.0 * torch.randn(B, T, D, generator=gen)).to(dtype).to(DEV)
    s = torch.exp(torch.rand(B, D, generator=gen)).to(DEV) if state else None
    n = None
    if lengths == "ragged":
        n = torch.randint(0, T + 1, (B,), generator=gen)
        n[0] = 0
        if B > 1:
            n[1] = T
        n = n.to(DEV)
    return x, gate, s, n, torch.randn(B, T, D, generator=gen).to(DEV), torch.randn(B, D, generator=gen).to(DEV)


def _check(x, gate, s, n, gy, gf):
    import snntc_amd as snn
    want = _reference(x, gate, s, n, gy, gf)
    y, final = snn.gated_scan(x, gate, s, n)
    _close(y, want["y"], "y")
    _close(final, want["final"], "final")
    dx, dgate, dstate = snn.gated_scan_grad(gy, gf, x, gate, y, s, n)
    assert dgate.dtype == gate.dtype
    _close(dx, want["dx"], "dx")
    _close(dgate, want["dgate"], "dgate")
    _close(dstate, want["dstate"], "dstate")


@pytest.mark.parametrize("lengths", [None, "ragged"])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (3, 2, 5), (2, 17, 64), (5, 64, 33), (2, 129, 70), (4, 300, 257), (65, 31, 16)])
def test_scan_and_gradient(B, T, D, dtype, lengths):
    _check(*_case(B, T, D, dtype, lengths=lengths))


@pytest.mark.parametrize("B,T,D,lengths", [(1, 5000, 3, None), (2, 4097, 65, "ragged"), (1, 2048, 128, None), (3, 1500, 100, "ragged"),
                                           (1, 9001, 40, "ragged"), (2, 700, 4, None)])
def test_long_sequences(B, T, D, lengths):
    """Few channels and many steps: the work is split along the sequence."""
    _check(*_case(B, T, D, torch.bfloat16, lengths=lengths))


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("B,T,D", [(9, 70, 96), (11, 200, 160), (2, 700, 192)])
def test_rows_of_whole_and_half_lines(B, T, D, dtype):
    _check(*_case(B, T, D, dtype, lengths="ragged"))


@pytest.mark.parametrize("B,T,D", [(1, 24000, 1024), (24, 1000, 1024), (12, 1000, 1024), (3, 4001, 1024), (16, 1600, 992),
                                   (8, 1500, 1024), (8, 3000, 1024)])
def test_more_than_the_caches_hold(B, T, D):
    """Gates of 16-bit values in float32: the same results as from 16 bits, where the call touches less than 256 MB and stores otherwise."""
    import snntc_amd as snn
    gen = torch.Generator(device=DEV).manual_seed(T)
    x = torch.exp(torch.rand(B, T, D, generator=gen, device=DEV))
    gate = (1.5 + 2.0 * torch.randn(B, T, D, generator=gen, device=DEV)).to(torch.bfloat16)
    gy = torch.randn(B, T, D, generator=gen, device=DEV)
    n = torch.full((B,), T - 77, device=DEV)
    y, final = snn.gated_scan(x, gate, None, n)
    y32, final32 = snn.gated_scan(x, gate.float(), None, n)
    assert torch.equal(y, y32) and torch.equal(final, final32)
    dx, dgate, dstate = snn.gated_scan_grad(gy, None, x, gate, y, None, n)
    dx32, dgate32, dstate32 = snn.gated_scan_grad(gy, None, x, gate.float(), y, None, n)
    assert torch.equal(dx, dx32) and torch.equal(dstate, dstate32) and torch.equal(dgate, dgate32.to(torch.bfloat16))
    assert not y[:, T - 77:].any() and not dx[:, T - 77:].any() and not dgate[:, T - 77:].any()


def test_ends_of_the_lengths():
    """Lengths around every place where a sequence may be cut, negative ones and ones beyond T included."""
    x, gate, s, _, gy, gf = _case(40, 600, 8)
    n = torch.tensor([0, 1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 319, 320, 383, 384,
                      385, 447, 448, 511, 512, 513, 575, 576, 599, 600, 700], device=DEV)
    n[2] = -5
    _check(x, gate, s, n, gy, gf)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("B,T,D", [(3, 65, 31), (2, 128, 32), (2, 129, 33), (5, 255, 100), (4, 256, 64)])
def test_short_sequences_of_few_channels(B, T, D, dtype):
    for lengths in (None, "ragged"):
        _check(*_case(B, T, D, dtype, lengths=lengths))


@pytest.mark.parametrize("B,T,D,lengths", [(100, 520, 40, "ragged"), (60, 700, 100, None), (125, 450, 33, "ragged"), (130, 400, 70, None),
                                           (1, 384, 1030, "ragged"), (1, 385, 1030, None)])
def test_around_the_line_between_cut_and_whole(B, T, D, lengths):
    _check(*_case(B, T, D, torch.float16, lengths=lengths))


def test_ends_of_the_lengths_of_short_sequences():
    x, gate, s, _, gy, gf = _case(34, 256, 40, torch.bfloat16)
    n = torch.tensor([0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 71, 72, 73, 119, 120, 121, 127, 128, 129, 135, 136, 137, 191, 192,
                      193, 254, 255, 256, 300], device=DEV)
    n[2] = -1
    _check(x, gate, s, n, gy, gf)


@pytest.mark.parametrize("B,T", [(12, 190001), (3, 760003)])
def test_more_elements_than_32_bits_count(B, T):
    """The first and last sequence are the same, and come out the same."""
    import snntc_amd as snn
    gen = torch.Generator(device=DEV).manual_seed(T)
    x = 1.0 + torch.rand(B, T, 1024, generator=gen, device=DEV)
    gate = torch.empty(B, T, 1024, dtype=torch.bfloat16, device=DEV).normal_(1.5, 2.0, generator=gen)
    gy = torch.empty(B, T, 1024, device=DEV).normal_(generator=gen)
    for v in (x, gate, gy):
        v[-1] = v[0]
    y, final = snn.gated_scan(x, gate)
    assert torch.equal(y[0], y[-1]) and torch.equal(final[0], final[-1])
    # the last 300 steps by the formula, begun 300 steps earlier: what the state there is off by is multiplied by all gates in between
    last = slice(T - 600, T)
    want = _reference(x[-1:, last, :16], gate[-1:, last, :16], y[-1:, T - 601, :16], None)
    _close(y[-1:, T - 300:, :16], [v[:, 300:] for v in want["y"]], "y")
    _close(final[-1:, :16], want["final"], "final")             # (made by joining runs of steps, y step by step: each within its bound)
    dx, dgate, dstate = snn.gated_scan_grad(gy, None, x, gate, y)
    assert torch.equal(dx[0], dx[-1]) and torch.equal(dgate[0], dgate[-1]) and torch.equal(dstate[0], dstate[-1])
    assert not torch.equal(dx[0], dx[1]) and bool(torch.isfinite(dx[-1]).all())


def test_gates_at_their_ends():
    """Gates that keep everything, take everything, or mix: 1 - a keeps its precision where a is close to 1."""
    import snntc_amd as snn
    x, _, s, _, gy, gf = _case(1, 9, 4)
    gate = torch.tensor([0.0, 16.0, -16.0, 60.0, -60.0, 1e4, -1e4, float("inf"), -float("inf")], device=DEV).view(1, 9, 1).expand(1, 9, 4)
    y, final = snn.gated_scan(x, gate, s)
    want = _reference(x, gate, s, None, gy, gf)
    # at 60 and above exp's argument adds its own size in roundings to the rest of 1, which is 1e-26 there
    assert torch.allclose(y.double().cpu(), want["y"][0], rtol=1e-5, atol=0) and torch.isfinite(y).all()
    dx, dgate, dstate = snn.gated_scan_grad(gy, gf, x, gate, y, s)
    assert torch.isfinite(dx).all() and torch.isfinite(dgate).all() and torch.isfinite(dstate).all()
    assert torch.allclose(dx.double().cpu(), want["dx"][0], rtol=2e-5, atol=1e-30)


def test_what_lies_behind_a_length_is_not_read():
    import snntc_amd as snn
    x, gate, s, _, gy, gf = _case(3, 90, 20)
    n = torch.tensor([0, 41, 90], device=DEV)
    y, final = snn.gated_scan(x, gate, s, n)
    grads = snn.gated_scan_grad(gy, gf, x, gate, y, s, n)
    nan = float("nan")
    x2, gate2, gy2 = x.clone(), gate.clone(), gy.clone()
    for b in range(3):
        x2[b, n[b]:] = nan
        gate2[b, n[b]:] = nan
        gy2[b, n[b]:] = nan
    y2, final2 = snn.gated_scan(x2, gate2, s, n)
    assert torch.equal(y, y2) and torch.equal(final, final2) and torch.equal(final[0], s[0])
    for a, b in zip(grads, snn.gated_scan_grad(gy2, gf, x2, gate2, y2, s, n)):
        assert torch.equal(a, b)
    assert (y[1, 41:] == 0).all() and (grads[0][1, 41:] == 0).all() and (grads[1][0] == 0).all()


def test_a_nan_stays_in_its_channel():
    import snntc_amd as snn
    x, gate, s, _, _, _ = _case(2, 700, 70)
    y0, _ = snn.gated_scan(x, gate, s)
    x[1, 300, 5] = float("nan")
    gate[0, 650, 69] = float("nan")
    y, final = snn.gated_scan(x, gate, s)
    bad = torch.isnan(y)
    want = torch.zeros_like(bad)
    want[1, 300:, 5] = True
    want[0, 650:, 69] = True
    assert torch.equal(bad, want) and torch.equal(y[~bad], y0[~bad])


def test_optional_inputs_and_outputs():
    import snntc_amd as snn
    x, gate, s, n, gy, gf = _case(3, 200, 30, lengths="ragged")
    zero = torch.zeros_like(s)
    y, final = snn.gated_scan(x, gate, None, n)
    y2, final2 = snn.gated_scan(x, gate, zero, n)
    assert torch.equal(y, y2) and torch.equal(final, final2)
    full = snn.gated_scan_grad(gy, gf, x, gate, y, None, n)
    only = [snn.gated_scan_grad(gy, gf, x, gate, y, None, n, want_dx=i == 0, want_dgate=i == 1, want_dstate=i == 2) for i in range(3)]
    for i in range(3):
        assert torch.equal(only[i][i], full[i]) and all(only[i][k] is None for k in range(3) if k != i)
    for a, b in zip(snn.gated_scan_grad(None, gf, x, gate, y, None, n), snn.gated_scan_grad(torch.zeros_like(gy), gf, x, gate, y, None, n)):
        assert torch.equal(a, b)
    for a, b in zip(snn.gated_scan_grad(gy, None, x, gate, y, None, n), snn.gated_scan_grad(gy, zero, x, gate, y, None, n)):
        assert torch.equal(a, b)


def test_empty_sizes():
    import snntc_amd as snn
    s = torch.rand(3, 5, device=DEV)
    y, final = snn.gated_scan(torch.zeros(3, 0, 5, device=DEV), torch.zeros(3, 0, 5, device=DEV), s)
    assert y.shape == (3, 0, 5) and torch.equal(final, s)
    g = torch.rand(3, 5, device=DEV)
    z = torch.zeros(3, 0, 5, device=DEV)
    assert torch.equal(snn.gated_scan_grad(None, g, z, z, z, s)[2], g)
    y, final = snn.gated_scan(torch.zeros(0, 4, 5, device=DEV), torch.zeros(0, 4, 5, device=DEV))
    assert y.shape == (0, 4, 5) and final.shape == (0, 5)
    assert snn.gated_step(torch.zeros(0, 5, device=DEV), torch.zeros(0, 5, device=DEV)).shape == (0, 5)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (64, 800), (513, 33)])
def test_steps_are_the_scan(shape, dtype):
    import snntc_amd as snn
    B, D = shape
    x, gate, s, _, _, _ = _case(B, 3, D, dtype)
    want = _reference(x, gate, s, None)
    state = s.clone()
    for t in range(3):
        new = snn.gated_step(x[:, t], gate[:, t], state)
        assert snn.gated_step(x[:, t].contiguous(), gate[:, t].contiguous(), state, out=state) is not None
        assert torch.equal(new, state)                       # in place is the same
        _close(state, (want["y"][0][:, t], want["y"][1][:, t]), f"step {t}")
    assert torch.equal(snn.gated_step(x[:, 0], gate[:, 0]), snn.gated_step(x[:, 0], gate[:, 0], torch.zeros_like(s)))


def test_strides_and_alignment():
    import snntc_amd as snn
    x, gate, s, n, gy, gf = _case(3, 50, 12, lengths="ragged")
    y, final = snn.gated_scan(x, gate, s, n)
    tx = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert not tx.is_contiguous()
    y2, _ = snn.gated_scan(tx, gate, s, n)
    assert torch.equal(y, y2)
    shifted = [torch.empty(v.numel() + 1, device=DEV)[1:].view(v.shape).copy_(v) for v in (x, gate, gy, y)]
    y3, f3 = snn.gated_scan(shifted[0], shifted[1], s, n)
    assert torch.equal(y, y3) and torch.equal(final, f3)
    for a, b in zip(snn.gated_scan_grad(gy, gf, x, gate, y, s, n), snn.gated_scan_grad(shifted[2], gf, shifted[0], shifted[1], shifted[3], s, n)):
        assert torch.equal(a, b)


def test_refusals():
    import snntc_amd as snn
    x, gate, s, _, gy, gf = _case(2, 3, 4)
    with pytest.raises(ValueError, match="does not match x"):
        snn.gated_scan(x, gate[:, :2], s)
    with pytest.raises(ValueError, match="state must have shape"):
        snn.gated_scan(x, gate, s[:1])
    with pytest.raises(TypeError, match="float32"):
        snn.gated_scan(x.half(), gate)
    with pytest.raises(TypeError, match="gate must be"):
        snn.gated_scan(x, gate.double())
    with pytest.raises(ValueError, match="3 dimensions"):
        snn.gated_scan(x[0], gate[0])
    with pytest.raises(ValueError, match="one entry per sequence"):
        snn.gated_scan(x, gate, s, torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError, match="int64"):
        snn.gated_scan(x, gate, s, torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="grad_y must have shape"):
        snn.gated_scan_grad(gy[:1], gf, x, gate, x)
    with pytest.raises(ValueError, match="out must"):
        snn.gated_step(x[:, 0], gate[:, 0], s, out=torch.empty(4, 2, device=DEV))
    with pytest.raises(ValueError, match="contiguous"):
        snn.gated_step(x[:, 0], gate[:, 0], s, out=torch.empty(4, 2, device=DEV).t())
    with pytest.raises(ValueError, match=r"must be \[B,T,4\]"):
        snn.SNN_recurrence(4).to(DEV)(x[:, :, :3].contiguous())


def test_the_layer_and_its_steps():
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(1)
    layer = snn.SNN_recurrence(6, weight=torch.randn(7, 6, generator=gen).numpy()).to(DEV)
    x = torch.exp(torch.rand(3, 10, 6, generator=gen)).to(DEV).requires_grad_(True)
    s = torch.exp(torch.rand(3, 6, generator=gen)).to(DEV).requires_grad_(True)
    n = torch.tensor([10, 4, 0], device=DEV)
    y, final = layer(x, s, n, return_state=True)
    up, upf = torch.randn(3, 10, 6, generator=gen).to(DEV), torch.randn(3, 6, generator=gen).to(DEV)
    grads = torch.autograd.grad([y, final], [x, s, layer.weight], [up, upf])
    xd, sd, w = (v.detach().double().cpu().requires_grad_(True) for v in (x, s, layer.weight))
    a = torch.sigmoid(xd @ w[:-1] + w[-1])
    h, ys = sd, []
    for t in range(10):
        on = (t < n.cpu())[:, None]
        h = torch.where(on, a[:, t] * h + (1 - a[:, t]) * xd[:, t], h)
        ys.append(torch.where(on, h, torch.zeros_like(h)))
    wy = torch.stack(ys, 1)
    want = torch.autograd.grad([wy, h], [xd, sd, w], [up.double().cpu(), upf.double().cpu()])
    # values below 3, ten steps and products of six terms in float32: some hundred roundings of 2e-7
    assert torch.allclose(y.double().cpu(), wy, atol=2e-5) and torch.allclose(final.double().cpu(), h, atol=2e-5)
    for g, r in zip(grads, want):
        assert torch.allclose(g.double().cpu(), r, rtol=1e-4, atol=1e-4)
    state = s.detach()
    with torch.no_grad():
        ys2, _ = layer(x, s, return_state=True)
        for t in range(10):
            state = layer.step(x[:, t], state)
            assert torch.allclose(state, ys2[:, t], atol=2e-5)
    (only,) = torch.autograd.grad(layer(x, s, n, return_state=True)[1].sum(), [s])          # one of the two outputs
    assert torch.isfinite(only).all()
    y = layer(x)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
