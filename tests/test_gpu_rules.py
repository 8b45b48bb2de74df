"""Rules on times and the choice of tokens against plain implementations in 64 bits.

Tolerances.  A ruled time is at most a product (or quotient), a product and a sum for the occurrences, and two sums, each off by half a step
of float32, 2^-24 of a value no larger than the sum of the terms' magnitudes, and one rounding to the result's type, half a step of it.
A chosen token is compared where its uniform number lies further than 1e-5 from either end of its share: a sum of up to 2e5 exponentials of
float32, each off by 2^-22 of itself (argument and exponential) and added with errors of no more, is off by less than 2^-20 = 1e-6."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _plain(times, history=None, lengths=None, prompts=None, repetition=1.0, presence=0.0, frequency=0.0, delay=None, allowed=None):
    """(ruled times, a bound of the terms' magnitudes, factor of the gradient), float64 on the CPU, row by row."""
    J = times.shape[-1]
    t = times.detach().double().cpu().reshape(-1, J)
    N = t.shape[0]
    u, size, slope = t.clone(), t.abs(), torch.ones_like(t)
    num = lambda x, h: float(x.cpu()[h]) if isinstance(x, torch.Tensor) else float(torch.tensor(x, dtype=torch.float32))      # noqa: E731
    if history is not None:
        S, L = history.shape
        hist = history.cpu()
        for r in range(N):
            h = r // (N // S)
            seen = L if lengths is None else max(0, min(L, int(lengths.reshape(-1)[r])))
            start = 0 if prompts is None else max(0, min(L, int(prompts[h])))
            count = {}
            for i in range(seen):
                j = int(hist[h, i])
                if 0 <= j < J:
                    count[j] = count.get(j, 0) + (i >= start)
            rep, pres, freq = num(repetition, h), num(presence, h), num(frequency, h)
            for j, o in count.items():
                slope[r, j] = rep if t[r, j] > 0 else 1 / rep
                u[r, j] = t[r, j] * slope[r, j]
                size[r, j] = u[r, j].abs()
                if o:
                    u[r, j] += pres + freq * o
                    size[r, j] += abs(pres) + abs(freq) * o
    if delay is not None:
        d = delay.double().cpu().expand(times.shape).reshape(N, J)
        u, size = u + d, size + d.abs()
    if allowed is not None:
        j = torch.arange(J)
        words = allowed.cpu().expand(*times.shape[:-1], -1).reshape(N, -1)
        on = (words[:, j // 32] >> (j % 32) & 1) == 1
        u, size, slope = torch.where(on, u, math.inf), torch.where(on, size, 0.0), torch.where(on, slope, 0.0)
    return u.view(times.shape), size.view(times.shape), slope.view(times.shape)


def _check(got, want, size, dtype):
    assert got.dtype == dtype
    got = got.double().cpu()
    limit = 4 * 2.0 ** -24 * size + HALF[dtype] * (want.abs() + 4 * 2.0 ** -24 * size) + TINY[dtype]
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]) and bool(got[want.isnan()].isnan().all())
    assert bool(((got - want).abs() <= limit)[fine].all()), float(((got - want).abs() / limit)[fine].max())


def _inputs(seed, S, T, J, L, dtype, signed=False):
    gen = torch.Generator().manual_seed(seed)
    times = 1.0 + 12.0 * torch.rand(S, T, J, generator=gen)
    if signed:
        times = times * torch.randint(-1, 2, times.shape, generator=gen)              # negative times and zeros too
    k = dict(history=torch.randint(-2, J + 2, (S, L), generator=gen), prompts=torch.randint(-1, L + 2, (S,), generator=gen),
             lengths=torch.randint(-1, L + 2, (S, T), generator=gen),
             repetition=0.7 + torch.rand(S, generator=gen), presence=torch.randn(S, generator=gen), frequency=0.3 * torch.randn(S, generator=gen),
             delay=torch.randn(J, generator=gen) * (torch.rand(J, generator=gen) < 0.3),
             allowed=torch.randint(-(1 << 31), 1 << 31, (S, T, (J + 31) // 32), generator=gen).to(torch.int32))
    return times.to(dtype).to(DEV), {n: v.to(DEV) for n, v in k.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,T,J,L", [(1, 1, 1, 1), (3, 5, 7, 9), (2, 3, 255, 40), (2, 2, 513, 70), (1, 3, 4099, 300), (2, 1, 8192, 33),
                                     (1, 2, 20011, 17), (2, 2, 33, 700), (1, 1, 8200, 9000)])
def test_ruled_times_and_their_gradient(S, T, J, L, dtype):
    import snntc_amd as snn
    times, k = _inputs(J + L, S, T, J, L, dtype, signed=True)
    g = torch.randn(S, T, J, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    for leave in ((), ("allowed",), ("delay", "allowed"), ("lengths", "prompts"), ("history", "lengths", "prompts", "repetition", "presence", "frequency"),
                  ("presence", "frequency"), ("repetition",)):
        how = {n: v for n, v in k.items() if n not in leave}
        want, size, slope = _plain(times, **how)
        _check(snn.rule_times(times, **how), want, size, dtype)
        kept = {n: v for n, v in how.items() if n in ("history", "lengths", "repetition", "allowed")}
        d = g.double().cpu() * slope
        _check(snn.rule_times_grad(g, times, **kept), d, d.abs(), dtype)
        leaf = times.clone().requires_grad_()
        (got,) = torch.autograd.grad(snn.rule_times(leaf, **how), [leaf], [g])
        assert torch.equal(got, snn.rule_times_grad(g, times, **kept))


def test_numbers_for_all_rows_and_rows_of_their_own():
    import snntc_amd as snn
    times, k = _inputs(5, 2, 3, 100, 20, torch.float32)
    how = dict(history=k["history"], repetition=1.3, presence=0.25, frequency=-0.1)
    want, size, _ = _plain(times, **how)
    _check(snn.rule_times(times, **how), want, size, torch.float32)
    rows = torch.randn(2, 3, 100, generator=torch.Generator().manual_seed(2)).to(DEV)
    for how in (dict(delay=rows), dict(delay=rows[0, 0].contiguous(), allowed=k["allowed"][0, 0].contiguous()), dict(allowed=k["allowed"]), {}):
        want, size, _ = _plain(times, **how)
        _check(snn.rule_times(times, **how), want, size, torch.float32)
    assert torch.equal(snn.rule_times(times), times)


def test_masked_places_hold_anything():
    """NaN, infinities and a type's lowest value under a mask; a mask that leaves nothing; bits behind the row."""
    import snntc_amd as snn
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        times = (1.0 + torch.rand(4, 70, device=DEV)).to(dtype)
        mask = torch.rand(4, 70, device=DEV) < 0.5
        mask[2] = False
        words = snn.pack_allowed(mask) | snn.pack_allowed(torch.arange(96, device=DEV) >= 70)
        clean = snn.rule_times(times, delay=torch.ones(70, device=DEV), allowed=words)
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
            dirty = torch.where(mask, times, torch.full_like(times, bad))
            assert torch.equal(snn.rule_times(dirty, delay=torch.ones(70, device=DEV), allowed=words), clean)
            g = torch.where(mask, torch.ones_like(times), torch.full_like(times, bad))
            assert torch.equal(snn.rule_times_grad(g, dirty, allowed=words), mask.to(dtype))
        assert bool((clean[2] == math.inf).all())
        late = torch.where(mask[0], math.nan, torch.ones(70, device=DEV))
        assert torch.equal(snn.rule_times(times[:1], delay=late, allowed=words[:1] ^ -1)[~mask[:1]], (times[:1].float() + 1).to(dtype)[~mask[:1]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("J", [3, 130, 1001, 9001])
def test_views_that_start_anywhere(J, dtype):
    import snntc_amd as snn
    times, k = _inputs(J, 2, 2, J, 50, dtype)
    big = torch.empty(times.numel() + 9, dtype=dtype, device=DEV)
    delay = torch.empty(J + 3, device=DEV)
    delay[3:] = k["delay"]
    want = snn.rule_times(times, **k)
    u = torch.rand(2, 2, device=DEV)
    chosen = snn.choose_tokens(times, u, 0.9, **k)
    for shift in (1, 3, 9):
        there = big[shift:shift + times.numel()].view(times.shape)
        there.copy_(times)
        assert torch.equal(snn.rule_times(there, **{**k, "delay": delay[3:]}), want)
        tokens, logp = snn.choose_tokens(there, u, 0.9, **k)
        assert torch.equal(tokens, chosen[0]) and torch.equal(logp.nan_to_num(nan=1.0), chosen[1].nan_to_num(nan=1.0))
    turned = times.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(snn.rule_times(turned, **k), want)
    assert torch.equal(snn.rule_times_grad(turned, turned, k["history"], k["lengths"], 1.5), snn.rule_times_grad(times, times, k["history"], k["lengths"], 1.5))


def test_tokens_at_the_ends_of_their_type():
    import snntc_amd as snn
    times = 1.0 + torch.rand(1, 50, device=DEV)
    far = torch.tensor([[-(1 << 63), (1 << 63) - 1, 1 << 32, (1 << 32) + 3, -(1 << 32) + 3, 50, -1, 7]], device=DEV)
    want, size, _ = _plain(times, far, repetition=2.0, frequency=1.0)
    _check(snn.rule_times(times, far, repetition=2.0, frequency=1.0), want, size, torch.float32)
    lengths = torch.tensor([1 << 40], device=DEV)
    assert torch.equal(snn.rule_times(times, far, lengths, repetition=2.0), snn.rule_times(times, far, repetition=2.0))
    assert torch.equal(snn.rule_times(times, far, -lengths, repetition=2.0), times)
    empty = torch.zeros(1, 0, dtype=torch.int64, device=DEV)
    assert torch.equal(snn.rule_times(times, empty, repetition=2.0), times)
    assert torch.equal(snn.choose_tokens(times, None, 0.0, empty, repetition=2.0)[0], times.argmin(1))


def test_empty_sizes():
    import snntc_amd as snn
    none = torch.zeros(0, 5, device=DEV)
    assert snn.rule_times(none).shape == (0, 5) and snn.rule_times_grad(none, none).shape == (0, 5)
    t, p = snn.choose_tokens(none, none[:, 0])
    assert t.shape == p.shape == (0,) and t.dtype == torch.int64
    assert snn.rule_times(none, torch.zeros(0, 3, dtype=torch.int64, device=DEV), repetition=2.0).shape == (0, 5)
    with pytest.raises(ValueError, match="without outputs"):
        snn.choose_tokens(torch.zeros(3, 0, device=DEV), torch.zeros(3, device=DEV))


def _distribution(times, temperature, **how):
    """Shares and their logarithms in 64 bits, of the ruled times as they are stored."""
    import snntc_amd as snn
    v = -snn.rule_times(times, **how).double()
    heat = temperature.double()[..., None] if isinstance(temperature, torch.Tensor) else temperature
    return torch.softmax(v / heat, -1), torch.log_softmax(v / heat, -1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,T,J,L", [(4, 3, 2, 3), (40, 1, 10, 5), (6, 5, 257, 40), (3, 7, 2049, 100), (2, 5, 8191, 60), (1, 6, 8193, 60),
                                     (3, 2, 33000, 2000), (2, 2, 150001, 9000), (1, 2, 600000, 50)])
def test_chosen_tokens(S, T, J, L, dtype):
    import snntc_amd as snn
    times, k = _inputs(S + J, S, T, J, L, dtype)
    gen = torch.Generator().manual_seed(3)
    u = torch.rand(S, T, generator=gen).to(DEV)
    heat = (0.3 + 2 * torch.rand(S, T, generator=gen)).to(DEV)
    # with one output allowed, or none, there is nothing to draw
    for how, temperature in ((k, heat), ({}, 1.0), ({n: k[n] for n in ("history", "prompts", "frequency")}, 0.5), ({"delay": k["delay"]}, heat)):
        tokens, logp = snn.choose_tokens(times, u, temperature, **how)
        assert tokens.dtype == torch.int64 and tokens.shape == u.shape and logp.shape == u.shape
        p, lp = _distribution(times, temperature, **how)
        nothing = p.isnan().all(-1)
        assert torch.equal(tokens == -1, nothing) and torch.equal(logp.isnan(), nothing)
        at = tokens.clamp(min=0)
        # logp: a difference of two times over T and a logarithm of a sum of J terms that is off by 2^-20 of itself
        ref = lp.gather(-1, at[..., None])[..., 0]
        assert bool(((logp.double() - ref).abs() <= 2.0 ** -20 + 2.0 ** -23 * ref.abs())[~nothing].all())
        cum = torch.cumsum(p, -1)
        upto = cum.gather(-1, at[..., None])[..., 0]
        before = upto - p.gather(-1, at[..., None])[..., 0]
        assert bool(((before - 1e-6 <= u) & (u <= upto + 1e-6))[~nothing].all())
        assert bool((p.gather(-1, at[..., None])[..., 0] > 0)[~nothing].all())
        # well inside the share of a token that is drawn so: exactly that token
        pick = torch.searchsorted(cum, torch.rand(S, T, 1, dtype=torch.float64, generator=gen).to(DEV)).clamp(max=J - 1)
        pick = torch.where(p.gather(-1, pick) < 1e-4, p.argmax(-1, keepdim=True), pick)
        share = p.gather(-1, pick)[..., 0]
        inside = (cum.gather(-1, pick)[..., 0] - 0.5 * share)
        got, _ = snn.choose_tokens(times, inside.float(), temperature, **how)
        clear = ~nothing & (share >= 4e-5)
        assert torch.equal(got[clear], pick[..., 0][clear])


@pytest.mark.parametrize("J", [1, 5, 64, 3000, 9000, 70000])
def test_ends_of_the_uniform_numbers(J):
    """0 and less, NaN: the first possible output; 1 and more: the last."""
    import snntc_amd as snn
    times = 1.0 + torch.rand(6, J, device=DEV)
    mask = torch.rand(6, J, device=DEV) < 0.7
    mask[:, J // 2] = True
    u = torch.tensor([0.0, -3.0, math.nan, 1.0, 7.0, math.inf], device=DEV)
    tokens, _ = snn.choose_tokens(times, u, allowed=snn.pack_allowed(mask))
    j = torch.arange(J, device=DEV)
    first, last = torch.where(mask, j, J).amin(1), torch.where(mask, j, -1).amax(1)
    assert torch.equal(tokens, torch.cat([first[:3], last[3:]]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("J", [1, 6, 300, 5000, 40000])
def test_temperature_zero_takes_the_earliest(J, dtype):
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(J)
    times = torch.randint(1, 5, (9, J), generator=gen).to(dtype).to(DEV)              # equal times: the lowest index
    mask = torch.rand(9, J, generator=gen).to(DEV) < 0.5
    mask[:, -1] = True
    words = snn.pack_allowed(mask)
    ruled = torch.where(mask, times.double(), math.inf)
    want = torch.sort(ruled, dim=1, stable=True).indices[:, 0]
    tokens, logp = snn.choose_tokens(times, None, 0.0, allowed=words)
    ref = torch.log_softmax(-ruled, 1).gather(1, want[:, None])[:, 0]
    assert torch.equal(tokens, want) and bool(((logp.double() - ref).abs() <= 2.0 ** -20 + 2.0 ** -23 * ref.abs()).all())
    # rows of one call with temperatures of their own
    heat = torch.tensor([0.0, 1.0, 0.5, 0.0, 2.0, 0.0, 1e-38, 1.0, 0.0], device=DEV)
    u = torch.rand(9, generator=gen).to(DEV)
    both = snn.choose_tokens(times, u, heat, allowed=words)
    cold, warm = heat < 1e-37, heat >= 1e-37
    assert torch.equal(both[0][cold], tokens[cold]) and torch.equal(both[1][cold], logp[cold])
    one = [snn.choose_tokens(times[r:r + 1], u[r:r + 1], float(heat[r]), allowed=words[r:r + 1]) for r in torch.nonzero(warm)[:, 0].tolist()]
    assert torch.equal(both[0][warm], torch.cat([o[0] for o in one])) and torch.equal(both[1][warm], torch.cat([o[1] for o in one]))


@pytest.mark.parametrize("J", [4, 700, 20000])
def test_rows_without_a_choice(J):
    """All masked, all infinite, a NaN, minus infinity, temperatures that are none: token -1 and NaN, its neighbours as ever."""
    import snntc_amd as snn
    times = 1.0 + torch.rand(9, J, device=DEV)
    clean = snn.choose_tokens(times, torch.full((9,), 0.5, device=DEV))
    heat = torch.ones(9, device=DEV)
    words = snn.pack_allowed(torch.ones(9, J, dtype=torch.bool, device=DEV))
    words[0] = 0
    times[1] = math.inf
    times[2, J // 2] = math.nan
    times[3, J - 1] = -math.inf
    heat[4], heat[5], heat[6] = -1.0, math.nan, math.inf
    tokens, logp = snn.choose_tokens(times, torch.full((9,), 0.5, device=DEV), heat, allowed=words)
    assert bool((tokens[:7] == -1).all() and logp[:7].isnan().all())
    assert torch.equal(tokens[7:], clean[0][7:]) and torch.equal(logp[7:], clean[1][7:])
    greedy, _ = snn.choose_tokens(times, None, 0.0, allowed=words)
    assert bool((greedy[:4] == -1).all()) and torch.equal(greedy[4:], times[4:].argmin(1))
    times[2, J // 2] = 1.0
    times[8, 1:] = math.inf                                                           # one output left
    assert snn.choose_tokens(times[8:], torch.rand(1, device=DEV))[0].item() == 0
    never = torch.full((1, J), 1e5, device=DEV)                                       # neurons that do not fire are alike
    token, logp = snn.choose_tokens(never, torch.tensor([0.999], device=DEV))
    assert token.item() == min(J - 1, int(0.999 * J)) and abs(logp.item() + math.log(J)) < 1e-5


def test_log_probability_is_that_of_the_ruled_times():
    """What a policy loss takes as old: time_logp of the stored ruled times, in 16 bits too."""
    import snntc_amd as snn
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        times, k = _inputs(11, 3, 20, 5000, 80, dtype)
        u = torch.rand(3, 20, device=DEV)
        tokens, logp = snn.choose_tokens(times, u, 1.0, **k)
        again = snn.time_logp(snn.rule_times(times, **k), tokens)
        assert bool(((logp - again).abs() <= 2.0 ** -19 + 2.0 ** -22 * again.abs()).all())


def test_draws_follow_the_shares():
    """Every output's number of draws among 2^16 evenly spread uniform numbers is its share's, but for the two ends."""
    import snntc_amd as snn
    N, J = 1 << 16, 37
    times = (4.0 * torch.rand(J, generator=torch.Generator().manual_seed(0))).to(DEV).expand(N, J)
    u = (torch.arange(N, device=DEV) + 0.5) / N
    tokens, _ = snn.choose_tokens(times, u, 0.7)
    share = torch.softmax(-times[0].double() / 0.7, 0) * N
    assert bool(((torch.bincount(tokens, minlength=J).double() - share).abs() <= 1.5).all())
    assert bool((tokens[1:] >= tokens[:-1]).all())


def test_gradient_by_differences():
    import snntc_amd as snn
    times, k = _inputs(21, 2, 2, 40, 30, torch.float32, signed=True)
    times = torch.where(times == 0, torch.ones_like(times), times)
    c = torch.randn(times.shape, generator=torch.Generator().manual_seed(4)).to(DEV)
    on = torch.isfinite(snn.rule_times(times, **k))
    leaf = times.clone().requires_grad_()
    f = lambda t: torch.where(on, snn.rule_times(t, **k).double() * c, 0.0).sum()       # noqa: E731
    ruled = snn.rule_times(leaf, **k)
    (g,) = torch.autograd.grad(ruled, [leaf], [torch.where(on, c, torch.zeros_like(c))])
    v = torch.randn(times.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
    h = 2.0 ** -6                                                # piecewise linear: differences of any length that crosses no zero
    v = v.clamp(-8, 8)
    got, want = float((f(times + h * v) - f(times - h * v)) / (2 * h)), float((g.double() * v).sum())
    # 160 ruled times of at most 60, each off by 5 half steps, over 2 h
    assert abs(got - want) <= 160 * 60 * 3 * 5 * 2.0 ** -24 / (2 * h) * 2


def test_refusals():
    import snntc_amd as snn
    t = torch.rand(4, 6, device=DEV)
    h = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    words = torch.zeros(1, dtype=torch.int32, device=DEV)
    for call, error in (
            (lambda: snn.rule_times(t.double()), TypeError), (lambda: snn.rule_times(t[0]), ValueError), (lambda: snn.rule_times(t.int()), TypeError),
            (lambda: snn.rule_times(t, h.int()), TypeError), (lambda: snn.rule_times(t, h[0]), ValueError),
            (lambda: snn.rule_times(t, h[:1].expand(3, 3)), ValueError), (lambda: snn.rule_times(t, h.cpu()), snn.SnntcLibraryError),
            (lambda: snn.rule_times(t, h, torch.zeros(2, dtype=torch.int64, device=DEV)), ValueError),
            (lambda: snn.rule_times(t, h, None, torch.zeros(4, dtype=torch.int64, device=DEV)), ValueError),
            (lambda: snn.rule_times(t, None, torch.zeros(4, dtype=torch.int64, device=DEV)), ValueError),
            (lambda: snn.rule_times(t, repetition=torch.ones(4, device=DEV)), ValueError),
            (lambda: snn.rule_times(t, h, repetition=torch.ones(4, device=DEV)), ValueError),
            (lambda: snn.rule_times(t, h, repetition=torch.ones(2, device=DEV).double()), TypeError),
            (lambda: snn.rule_times(t, h, repetition=0.0), ValueError), (lambda: snn.rule_times(t, h, presence=math.nan), ValueError),
            (lambda: snn.rule_times(t, delay=t[:2]), ValueError), (lambda: snn.rule_times(t, delay=t[0, :5].contiguous()), ValueError),
            (lambda: snn.rule_times(t, allowed=words.long()), TypeError), (lambda: snn.rule_times(t, allowed=words.expand(2)), ValueError),
            (lambda: snn.rule_times(t, allowed=words.expand(2, 1)), ValueError), (lambda: snn.rule_times(t, allowed=words.cpu()), snn.SnntcLibraryError),
            (lambda: snn.rule_times_grad(t.bfloat16(), t), TypeError), (lambda: snn.rule_times_grad(t[:2], t), ValueError),
            (lambda: snn.choose_tokens(t, None), ValueError), (lambda: snn.choose_tokens(t, None, torch.zeros(4, device=DEV)), ValueError),
            (lambda: snn.choose_tokens(t, t[:, 0].double()), TypeError), (lambda: snn.choose_tokens(t, t[:2, 0]), ValueError),
            (lambda: snn.choose_tokens(t, t[:, 0], -1.0), ValueError), (lambda: snn.choose_tokens(t, t[:, 0], math.inf), ValueError),
            (lambda: snn.choose_tokens(t, t[:, 0], t[0]), ValueError)):
        with pytest.raises(error):
            call()
    for name, value in (("delay", t[0].clone()), ("repetition", torch.ones(2, device=DEV)), ("frequency", torch.ones(2, device=DEV))):
        with pytest.raises(ValueError, match="must not require a gradient"):
            snn.rule_times(t, h, **{name: value.requires_grad_()})
    leaf = t.clone().requires_grad_()
    (g,) = torch.autograd.grad((snn.rule_times(leaf, h, repetition=2.0) ** 2).sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once only"):
        g.sum().backward()
    assert not snn.choose_tokens(leaf, t[:, 0])[1].requires_grad


def test_graphs_of_autograd():
    """Saved tensors hooks, general paths, inference mode, changed inputs."""
    import snntc_amd as snn
    from snntc_amd import ops
    times, k = _inputs(2, 2, 3, 50, 20, torch.float32)
    for how in (k, {"delay": k["delay"]}, {"allowed": k["allowed"]}, dict(history=k["history"], repetition=1.4)):
        leaf = times.clone().requires_grad_()
        want = torch.autograd.grad(snn.rule_times(leaf, **how), [leaf], [times])[0]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
            out = snn.rule_times(leaf, **how)
        assert torch.equal(torch.autograd.grad(out, [leaf], [times])[0], want)
        order = ("history", "lengths", "prompts", "repetition", "presence", "frequency", "delay", "allowed")
        default = dict(repetition=1.0, presence=0.0, frequency=0.0)
        out = ops.GENERAL["rule_layer"](leaf, *[how.get(n, default.get(n)) for n in order])
        assert torch.equal(out, snn.rule_times(leaf, **how)) and torch.equal(torch.autograd.grad(out, [leaf], [times])[0], want)
        with torch.inference_mode():
            assert torch.equal(snn.rule_times(leaf, **how), out)
    leaf = times.clone().requires_grad_()
    x = leaf * 1.0
    out = snn.rule_times(x, k["history"], repetition=1.5)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    x = leaf * 1.0
    out = snn.rule_times(x, k["history"], frequency=1.5, delay=k["delay"])
    x.mul_(2.0)                                                  # the gradient does not read the times here
    out.sum().backward()
    assert torch.equal(leaf.grad, torch.ones_like(leaf))


@pytest.mark.parametrize("rows,J", [(70000, 40), (2200, 1000000)])
def test_more_elements_than_31_bits_count(rows, J):
    """Offsets of rows beyond 2^31 elements, and more workgroups than a small grid."""
    import snntc_amd as snn
    times = torch.rand(1, 64, device=DEV).to(torch.bfloat16).repeat(rows, -(-J // 64))[:, :J].contiguous()
    history = torch.randint(0, J, (rows, 4), device=DEV)
    ruled = snn.rule_times(times, history, repetition=2.0)
    r = torch.arange(rows, device=DEV)[:, None]
    assert torch.equal(ruled[r, history], (times[r, history].float() * 2.0).to(torch.bfloat16))
    ruled[r, history] = times[r, history]
    assert torch.equal(ruled, times)
    at = torch.randint(0, J, (rows,), device=DEV)
    times[r[:, 0], at] = -3.0
    assert torch.equal(snn.choose_tokens(times, None, 0.0)[0], at)
    if J > 64:
        times[r[:, 0], at] = -60.0
        assert torch.equal(snn.choose_tokens(times, torch.full((rows,), 0.5, device=DEV))[0], at)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("J", [65, 67, 513, 8193, 8197, 12295, 16387, 20481])
def test_ends_of_rows_under_rules(J, dtype):
    """Rows that end one element or a few into what a workgroup or a wavefront takes."""
    import snntc_amd as snn
    times, k = _inputs(J, 2, 2, J, 40, dtype, signed=True)
    k["history"][:, ::3] = torch.arange(J - 14, J, device=DEV)
    want, size, slope = _plain(times, **k)
    _check(snn.rule_times(times, **k), want, size, dtype)
    g = torch.randn(2, 2, J, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    d = g.double().cpu() * slope
    _check(snn.rule_times_grad(g, times, k["history"], k["lengths"], k["repetition"], k["allowed"]), d, d.abs(), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,J", [(3, 65), (5, 2049), (3, 8195), (530, 9001), (600, 16387), (260, 16389), (3, 32769), (3, 40961), (300, 40967), (1100, 33000)])
def test_tokens_from_the_ends_of_rows(rows, J, dtype):
    """Nearly all of the chance lies with the last seven elements, under every rule."""
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(J)
    times = 20.0 + torch.rand(rows, J, generator=gen)
    times[:, -7:] = torch.rand(rows, 7, generator=gen) - 5.0
    times = times.to(dtype).to(DEV)
    words = torch.randint(-(1 << 31), 1 << 31, (rows, (J + 31) // 32), generator=gen).to(torch.int32)
    words[:, (J - 4) // 32] |= torch.tensor((1 << (J - 4) % 32), dtype=torch.int64).to(torch.int32)          # one of them is allowed
    how = dict(history=torch.randint(J - 9, J, (rows, 11), generator=gen).to(DEV), prompts=torch.full((rows,), 3, device=DEV), repetition=1.2,
               presence=0.3, frequency=0.1, delay=torch.randn(J, generator=gen).to(DEV), allowed=words.to(DEV))
    ruled = snn.rule_times(times, **how).double()
    lp = torch.log_softmax(-ruled / 0.9, -1)
    cum = lp[:, -40:].exp().cumsum(-1)                                # what lies before the last forty has a chance of e^-20 40000 at most
    seen = set()
    for u in (0.02, 0.3, 0.6, 0.99):
        tokens, logp = snn.choose_tokens(times, torch.full((rows,), u, device=DEV), 0.9, **how)
        at = torch.searchsorted(cum, torch.full((rows, 1), u, dtype=torch.float64, device=DEV))[:, 0]
        edges = torch.cat([torch.zeros_like(cum[:, :1]), cum], 1)
        clear = ((edges - u).abs() > 1e-3).all(1)
        assert torch.equal(tokens[clear], (J - 40 + at)[clear]) and bool(clear.float().mean() > 0.5)
        ref = lp.gather(-1, tokens[:, None])[:, 0]
        assert bool(((logp.double() - ref).abs() <= 2.0 ** -20 + 2.0 ** -23 * ref.abs()).all())
        seen |= set((J - tokens).tolist())
    assert seen <= set(range(1, 8))
    assert torch.equal(snn.choose_tokens(times, None, 0.0, **how)[0], ruled.argmin(-1))


@pytest.mark.parametrize("L", [65535, 65536, 70000])
def test_occurrences_past_16_bits(L):
    import snntc_amd as snn
    times = 1.0 + torch.rand(1, 5000, device=DEV)
    history = torch.full((1, L), 4321, device=DEV)
    history[0, 17], history[0, 300] = 12, 13
    got = snn.rule_times(times, history, frequency=2.0 ** -10)
    want = times.clone()
    want[0, 4321] += 2.0 ** -10 * (L - 2)
    want[0, 12] += 2.0 ** -10
    want[0, 13] += 2.0 ** -10
    assert torch.equal(got, want)
    assert int(snn.choose_tokens(times, None, 0.0, history, frequency=-1.0)[0]) == 4321
