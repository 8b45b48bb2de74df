"""time_logp, policy_time_loss and preference_time_loss against their formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
CLIP, KL, BETA, SMOOTHING = (0.2, 0.3), 0.1, 0.3, 0.1


def _soft(times, tokens):
    """float64 on the CPU: logp, softmax, and a bound on the error of logp in float32."""
    v = -times.double().cpu()
    k = tokens.cpu()
    logs = torch.log_softmax(v, -1)
    p = logs.exp()
    logp = logs.gather(-1, k[..., None])[..., 0]
    top = v.amax(-1)
    away = (v - top[..., None]).abs()
    # every exponential: its argument's rounding and its product with log2(e) (two of its size), the result's two; the sum: at most
    # J / 64 terms in a lane and 32 more joins; the logarithm: two of its size; the token's difference and the last: two of theirs
    J = v.shape[-1]
    spread = torch.nan_to_num(p * away, nan=0.0).sum(-1)
    lse = logs.amax(-1).neg()
    tol = U * (2.0 * spread + 4.0 + J / 64 + 32.0 + 2.0 * lse.abs() + 2.0 * (v.gather(-1, k[..., None])[..., 0] - top).abs() + 2.0 * logp.abs())
    return logp, p, away, tol


def _grad(p, away, tokens, coef, coef_tol, tol, dtype):
    """The gradient coef (p - [j = token]) and a bound on its error."""
    hot = torch.zeros_like(p).scatter_(-1, tokens.cpu()[..., None], 1.0)
    g = coef[..., None] * (p - hot)
    # p: logsumexp's error, its argument's (two of its size), two of its own; then a difference and two products
    e = coef.abs()[..., None] * (p * (tol[..., None] + U * (2.0 * away + 2.0 * away.clamp(max=100.0) + 4.0)) + 4.0 * U * (p - hot).abs() + U * hot)
    return g, 1.05 * e + coef_tol[..., None] * (p - hot).abs() + HALF[dtype] * g.abs() * 1.05 + TINY[dtype]


def _close(got, want, tol, what):
    bad = ~((got.double().cpu() - want).abs() <= tol + 1e-38)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def _case(rows, J, dtype, seed=0, spread=8.0):
    gen = torch.Generator().manual_seed(seed + 17 * sum(rows) + J)
    times = (1.0 + spread * torch.rand(*rows, J, generator=gen)).to(dtype)
    tokens = torch.randint(0, J, rows, generator=gen)
    return times, tokens, gen


def _policy_inputs(times, tokens, gen):
    logp = torch.log_softmax(-times.double(), -1).gather(-1, tokens[..., None])[..., 0]
    step = 0.25 * torch.randn(logp.shape, generator=gen, dtype=torch.float64)
    for end in (1 - CLIP[0], 1 + CLIP[1]):                     # no ratio on an end of the clip, where the gradient jumps
        step = torch.where((step.exp() - end).abs() < 1e-2, torch.zeros_like(step), step)
    return (logp - step).float(), torch.randn(logp.shape, generator=gen), (logp + 0.5 * torch.randn(logp.shape, generator=gen)).float()


def _policy_reference(times, tokens, old, adv, ref, weight, kl=KL):
    logp, p, away, tol = _soft(times, tokens)
    ratio = torch.exp(logp - old.double())
    A = adv.double()
    plain, clipped = ratio * A, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * A
    loss, c = -torch.minimum(plain, clipped), -torch.where(plain <= clipped, plain, torch.zeros_like(plain))
    rt = tol + U * (2.0 * (logp - old.double()).abs() + 6.0)     # relative error of the ratio
    lt = ratio * A.abs() * rt + 4 * U * loss.abs()
    ct = c.abs() * (rt + 2 * U)
    if ref is not None:
        d = ref.double() - logp
        e = torch.expm1(d)
        et = (e.abs() + 1.0) * (tol + 4 * U * d.abs()) + 4 * U * e.abs()
        loss, c = loss + kl * (e - d), c - kl * e
        lt = lt + abs(kl) * (e.abs() * tol + 8 * U * (e.abs() + d.abs())) + 4 * U * loss.abs()
        ct = ct + abs(kl) * et + 4 * U * c.abs()
    w = torch.full_like(loss, 1.0 / loss.numel()) if weight is None else weight.double()
    on = (w != 0).double()
    g, gt = _grad(p, away, tokens, c * w, ct * w.abs() + 2 * U * (c * w).abs(), tol, times.dtype)
    return (loss * on, lt * on), (logp * on, tol * on), (g, gt), (loss * w).sum()


def _check_policy(times, tokens, old, adv, ref, weight, same=True):
    """same: one workgroup owns a row with and without its gradient, or several do, so that the losses are equal to the last digit."""
    import snntc_amd as snn
    dev = [None if v is None else v.to(DEV) for v in (times, tokens, old, adv, ref, weight)]
    loss, logp, grad = snn.policy_time_loss(*dev[:4], ref_logp=dev[4], weight=dev[5], clip=CLIP, kl_coef=KL)
    (wl, wp, wg, total) = _policy_reference(times, tokens, old, adv, ref, weight)
    assert grad.dtype == times.dtype
    _close(logp, *wp, "logp")
    _close(loss, *wl, "loss")
    _close(grad, *wg, "gradient")
    leaf = dev[0].clone().requires_grad_(True)
    objective = snn.policy_loss(leaf, *dev[1:4], ref_logp=dev[4], weight=dev[5], clip=CLIP, kl_coef=KL)
    bound = float((wl[1] * (1.0 / loss.numel() if weight is None else weight.abs().double())).sum()) + 40 * U * float(
        (wl[0].abs() * (1.0 / loss.numel() if weight is None else weight.abs().double())).sum())
    assert abs(float(objective.detach()) - float(total)) <= bound + 1e-30
    (g2,) = torch.autograd.grad(objective, [leaf], torch.tensor(-0.5, device=DEV))
    _close(g2, -0.5 * wg[0], 0.5 * wg[1] + TINY[times.dtype] + HALF[times.dtype] * wg[0].abs(), "gradient through autograd")
    quiet = snn.policy_time_loss(*dev[:4], ref_logp=dev[4], weight=dev[5], clip=CLIP, kl_coef=KL, want_grad=False)
    assert quiet[2] is None
    if same:
        assert torch.equal(quiet[0], loss) and torch.equal(quiet[1], logp)
    _close(quiet[1], *wp, "logp without the gradient")
    _close(quiet[0], *wl, "loss without the gradient")


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,J", [((1,), 1), ((1,), 2), ((3,), 10), ((257,), 10), ((5,), 63), ((4, 9), 65), ((33,), 1000), ((6,), 1027),
                                    ((7,), 2048), ((3,), 4099), ((5,), 8200), ((2,), 20001)])
def test_policy(rows, J, dtype):
    times, tokens, gen = _case(rows, J, dtype)
    old, adv, ref = _policy_inputs(times, tokens, gen)
    _check_policy(times, tokens, old, adv, ref, None)
    weight = torch.rand(rows, generator=gen) * (torch.rand(rows, generator=gen) < 0.7)
    _check_policy(times, tokens, old, adv, None, weight)


@pytest.mark.parametrize("rows,J,dtype", [((1,), 70000, torch.float32), ((3,), 131072, torch.bfloat16), ((2,), 100003, torch.float16),
                                          ((40,), 33000, torch.float32), ((300,), 5000, torch.bfloat16), ((5000,), 30, torch.float32),
                                          ((9000,), 129, torch.bfloat16)])
def test_policy_of_long_rows_and_many_rows(rows, J, dtype):
    times, tokens, gen = _case(rows, J, dtype, spread=20.0)
    old, adv, ref = _policy_inputs(times, tokens, gen)
    _check_policy(times, tokens, old, adv, ref, None)


@pytest.mark.parametrize("rows,J,dtype", [((64,), 32801, torch.float32), ((70,), 65536, torch.float32), ((192,), 65551, torch.float16),
                                          ((200,), 131072, torch.bfloat16)])
def test_long_rows_held_for_their_gradient(rows, J, dtype):
    """More than 8192 pieces of 16 bytes, in enough rows that one workgroup keeps each."""
    times, tokens, gen = _case(rows, J, dtype, spread=20.0)
    old, adv, ref = _policy_inputs(times, tokens, gen)
    _check_policy(times, tokens, old, adv, ref, None, same=False)


@pytest.mark.parametrize("J", [50, 251, 1003, 4001, 8005, 16001, 32003, 60001, 70001])
def test_gradients_larger_than_the_caches(J):
    """Rows do not know how many there are: both halves of a batch whose times and gradient are more than 256 MB, by themselves."""
    import snntc_amd as snn
    rows = 2 ** 25 // J + 2
    gen = torch.Generator(device=DEV).manual_seed(J)
    times = 1.0 + 8.0 * torch.rand(rows, J, generator=gen, device=DEV)
    tokens = torch.randint(0, J, (rows,), generator=gen, device=DEV)
    old, adv = torch.full((rows,), -math.log(J), device=DEV), torch.randn(rows, generator=gen, device=DEV)
    weight = (torch.rand(rows, generator=gen, device=DEV) - 0.2).clamp(min=0.0)
    whole = snn.policy_time_loss(times, tokens, old, adv, weight=weight)
    cut = rows // 8 * 4                                         # (4 J elements are whole pieces of 16 bytes: rows lie to those as they did)
    for part in (slice(0, cut), slice(cut, rows)):
        half = snn.policy_time_loss(times[part].clone(), tokens[part], old[part], adv[part], weight=weight[part])
        assert all(torch.equal(w[part], h) for w, h in zip(whole, half))


@pytest.mark.parametrize("J", [50, 251, 1003, 4001, 9001])
def test_preference_gradients_larger_than_the_caches(J):
    """Two pairs of long sequences and each by itself, where the mean over pairs makes its gradient twice as large."""
    import snntc_amd as snn
    T = 2 ** 23 // J // 4 * 4 + 4
    gen = torch.Generator(device=DEV).manual_seed(J)
    times = 1.0 + 8.0 * torch.rand(4, T, J, generator=gen, device=DEV)
    tokens = torch.randint(0, J, (4, T), generator=gen, device=DEV)
    ref = snn.time_logp(times, tokens).double().sum(1).float()[[2, 3, 0, 1]]
    weight = (torch.rand(4, T, generator=gen, device=DEV) < 0.8).float()
    beta = 1e-3
    whole = snn.preference_time_loss(times, tokens, ref, weight, beta)
    for pair in ([0, 2], [1, 3]):
        one = snn.preference_time_loss(times[pair], tokens[pair], ref[pair], weight[pair], beta)
        assert torch.equal(2.0 * whole[-1][pair], one[-1])
        assert torch.equal(whole[0][pair[:1]], one[0])


def test_rows_of_weight_zero_are_not_read():
    import snntc_amd as snn
    for J in (10, 900, 70000):
        times, tokens, gen = _case((6,), J, torch.float32)
        old, adv, ref = _policy_inputs(times, tokens, gen)
        weight = torch.tensor([0.5, 0.0, 1.0, 0.0, -0.25, 0.0])
        args = [v.to(DEV) for v in (times, tokens, old, adv)]
        a = snn.policy_time_loss(*args, ref_logp=ref.to(DEV), weight=weight.to(DEV), kl_coef=0.1)
        off = weight == 0
        times[off], old[off], adv[off], ref[off] = (float("nan"),) * 4
        tokens[off] = -100
        args = [v.to(DEV) for v in (times, tokens, old, adv)]
        b = snn.policy_time_loss(*args, ref_logp=ref.to(DEV), weight=weight.to(DEV), kl_coef=0.1)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert (a[0][off] == 0).all() and (a[1][off] == 0).all() and (a[2][off] == 0).all()
        none = snn.policy_time_loss(*args, ref_logp=ref.to(DEV), weight=torch.zeros(6, device=DEV))
        assert all((v == 0).all() for v in none)
        assert float(snn.policy_loss(*args, weight=torch.zeros(6, device=DEV))) == 0.0
        assert torch.equal(snn.time_logp(args[0], args[1], weight.to(DEV)), a[1])


def test_actions_outside_the_classes_are_visible():
    import snntc_amd as snn
    for J in (10, 3000, 70000):
        times, tokens, gen = _case((5,), J, torch.float32)
        old, adv, ref = (v.to(DEV) for v in _policy_inputs(times, tokens, gen))
        tokens[1], tokens[3] = J, -1
        loss, logp, grad = snn.policy_time_loss(times.to(DEV), tokens.to(DEV), old, adv)
        bad = torch.tensor([False, True, False, True, False], device=DEV)
        assert torch.equal(torch.isnan(loss), bad) and torch.equal(torch.isnan(logp), bad)
        assert torch.equal(torch.isnan(grad).any(1), bad) and torch.isnan(grad[bad]).all()
        assert torch.equal(torch.isnan(snn.time_logp(times.to(DEV), tokens.to(DEV))), bad)


@pytest.mark.parametrize("J", [5, 64, 1000, 9000, 70000])
def test_neurons_that_never_fire(J):
    """Times at MAX_SPIKE_TIME, the largest number and infinity; rows of nothing else."""
    import snntc_amd as snn
    big = torch.finfo(torch.float32).max
    times, tokens, _ = _case((6,), J, torch.float32)
    times[0, ::2] = 1e5
    times[1] = 1e5
    times[2] = big
    times[3, 1:] = math.inf
    times[4] = math.inf
    times[5, J // 2] = math.nan
    tokens[:] = 0
    tokens[0] = 1
    logp = snn.time_logp(times.to(DEV), tokens.to(DEV)).cpu()
    want = torch.log_softmax(-times.double(), -1).gather(-1, tokens[:, None])[:, 0]
    assert torch.allclose(logp[:4].double(), want[:4], rtol=1e-5, atol=1e-5)
    assert abs(float(logp[1]) + math.log(J)) < 1e-5 and abs(float(logp[2]) + math.log(J)) < 1e-5 and float(logp[3]) == 0.0
    assert torch.isnan(logp[4:]).all()
    ones = torch.ones(6, device=DEV)
    _, _, grad = snn.policy_time_loss(times.to(DEV), tokens.to(DEV), logp.to(DEV), ones, weight=ones)
    grad = grad.cpu()
    assert torch.isnan(grad[4]).any() and torch.isnan(grad[5]).any()
    hot = torch.zeros(6, J).scatter_(1, tokens[:, None], 1.0)
    p = torch.softmax(-times.double(), -1)
    assert torch.allclose(grad[:4].double(), -(p - hot)[:4], atol=1e-5)
    # an output that can never be chosen was: its log-probability is minus infinity, and the divergence from a reference infinite
    tokens[3] = 1
    loss, logp, _ = snn.policy_time_loss(times[3:4].to(DEV), tokens[3:4].to(DEV), ones[:1], ones[:1], ref_logp=ones[:1], kl_coef=0.1)
    assert float(logp) == -math.inf and float(loss) == math.inf


def _preference_reference(times, tokens, ref, weight, beta=BETA, smoothing=SMOOTHING):
    logp, p, away, tol = _soft(times, tokens)
    w = torch.ones_like(logp) if weight is None else weight.double()
    on = w != 0
    terms = torch.where(on, w * logp, 0.0)
    T = logp.shape[1]
    seq = terms.sum(1)
    seq_tol = torch.where(on, w.abs() * tol, 0.0).sum(1) + U * (T / 64 + 10.0) * terms.abs().sum(1)
    P = len(seq) // 2
    gain = seq - ref.double()
    m = beta * (gain[:P] - gain[P:])
    mt = abs(beta) * (seq_tol[:P] + seq_tol[P:] + 4 * U * (seq[:P].abs() + seq[P:].abs() + ref[:P].abs() + ref[P:].abs()))
    sp = torch.nn.functional.softplus
    loss = (1 - smoothing) * sp(-m) + smoothing * sp(m)
    lt = mt + 8 * U * (loss + m.abs())
    slope = beta / P * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m))
    st = abs(beta) / P * (mt + 12 * U * (1 + m.abs()))
    coef = torch.cat([slope, -slope])[:, None] * w
    ct = torch.cat([st, st])[:, None] * w.abs() + 2 * U * coef.abs()
    g, gt = _grad(torch.where(on[..., None], p, 0.0), away, tokens.clamp(0, p.shape[-1] - 1), coef, ct, tol, times.dtype)
    return (loss, lt), (seq, seq_tol), (torch.where(on[..., None], g, 0.0), torch.where(on[..., None], gt, 0.0))


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("P,T,J", [(1, 1, 2), (3, 5, 10), (2, 65, 33), (5, 13, 1000), (4, 200, 17), (2, 3, 5003), (1, 2, 40000)])
def test_preference(P, T, J, dtype):
    import snntc_amd as snn
    times, tokens, gen = _case((2 * P, T), J, dtype)
    logp = torch.log_softmax(-times.double(), -1).gather(-1, tokens[..., None])[..., 0]
    for masked in (False, True):
        weight = None
        if masked:
            n = torch.randint(0, T + 1, (2 * P,), generator=gen)
            n[0] = 0                                        # a sequence of nothing
            weight = (torch.arange(T)[None] < n[:, None]).float() * (0.5 + torch.rand(2 * P, T, generator=gen))
        ref = ((logp if weight is None else logp * weight).sum(1) + 2.0 * torch.randn(2 * P, generator=gen)).float()
        wl, ws, wg = _preference_reference(times, tokens, ref, weight)
        t, k, r, w = (None if v is None else v.to(DEV) for v in (times, tokens, ref, weight))
        loss, seq, grad = snn.preference_time_loss(t, k, r, w, BETA, SMOOTHING)
        _close(seq, *ws, "sequence log-probability")
        _close(loss, *wl, "loss")
        _close(grad, *wg, "gradient")
        leaf = t.clone().requires_grad_(True)
        objective = snn.preference_loss(leaf, k, r, w, BETA, SMOOTHING)
        assert abs(float(objective.detach()) - float(wl[0].mean())) <= float(wl[1].mean()) + 20 * U * float(wl[0].mean())
        (g2,) = torch.autograd.grad(objective * 3.0, [leaf])
        _close(g2, 3.0 * wg[0], 3.0 * wg[1] + TINY[dtype] + HALF[dtype] * wg[0].abs() * 3.0, "gradient through autograd")


def test_preference_far_from_indifference():
    """Margins of hundreds either way: the loss grows like the margin, its slope stays between 0 and beta."""
    import snntc_amd as snn
    times, tokens, _ = _case((4, 3), 7, torch.float32)
    seq = torch.log_softmax(-times.double(), -1).gather(-1, tokens[..., None])[..., 0].sum(1)
    ref = (seq + torch.tensor([3000.0, -3000.0, 0.0, 0.0], dtype=torch.float64)).float()
    loss, _, grad = snn.preference_time_loss(times.to(DEV), tokens.to(DEV), ref.to(DEV), beta=0.5)
    assert torch.allclose(loss.cpu(), torch.tensor([1500.0, 0.0]), rtol=1e-5, atol=1e-30) and torch.isfinite(grad).all()
    assert (grad[1] == 0).all() and (grad[3] == 0).all()


def test_empty_batches():
    import snntc_amd as snn
    k = torch.zeros(0, dtype=torch.int64, device=DEV)
    f = torch.zeros(0, device=DEV)
    loss, logp, grad = snn.policy_time_loss(torch.zeros(0, 5, device=DEV), k, f, f)
    assert loss.shape == logp.shape == (0,) and grad.shape == (0, 5)
    t = torch.zeros(4, 0, 5, device=DEV)                    # pairs of sequences without a step: no difference, log 2 each
    loss, seq, grad = snn.preference_time_loss(t, torch.zeros(4, 0, dtype=torch.int64, device=DEV), torch.zeros(4, device=DEV))
    assert torch.allclose(loss, torch.full((2,), math.log(2.0), device=DEV)) and (seq == 0).all() and grad.shape == (4, 0, 5)
    assert snn.preference_time_loss(t[:0], torch.zeros(0, 0, dtype=torch.int64, device=DEV), f)[0].shape == (0,)


def test_strides_and_alignment():
    import snntc_amd as snn
    for J, dtype in [(12, torch.float32), (1001, torch.bfloat16), (5000, torch.float32), (70001, torch.float16)]:
        times, tokens, gen = _case((5,), J, dtype)
        old, adv, _ = (v.to(DEV) for v in _policy_inputs(times, tokens, gen))
        t, k = times.to(DEV), tokens.to(DEV)
        want = snn.policy_time_loss(t, k, old, adv)
        wide = torch.zeros(5, 2 * J, dtype=dtype, device=DEV)
        wide[:, ::2] = t
        shifted = torch.empty(5 * J + 1, dtype=dtype, device=DEV)[1:].view(5, J).copy_(t)
        for other in (wide[:, ::2], shifted, t.t().contiguous().t()):
            got = snn.policy_time_loss(other, k, old, adv)
            for a, b in zip(got, want):                      # (rows may be read in other pieces: equal but for the order of sums)
                assert torch.allclose(a.float(), b.float(), rtol=max(4 * HALF[dtype], 6e-6), atol=1e-6)


def test_the_same_result_on_every_call():
    import snntc_amd as snn
    for rows, J in (((2000,), 33), ((3,), 90000)):
        times, tokens, gen = _case(rows, J, torch.bfloat16)
        old, adv, ref = (v.to(DEV) for v in _policy_inputs(times, tokens, gen))
        t, k = times.to(DEV), tokens.to(DEV)
        first = snn.policy_time_loss(t, k, old, adv, ref, kl_coef=0.1)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, snn.policy_time_loss(t, k, old, adv, ref, kl_coef=0.1)))


def test_more_elements_than_32_bits_count():
    """Rows that start behind 2^31 elements: the last rows of the batch against the same rows alone."""
    import snntc_amd as snn
    J, N = 131072, 16400
    times = torch.zeros(N, J, dtype=torch.bfloat16, device=DEV)
    times[-3:] = 1.0 + 8.0 * torch.rand(3, J, device=DEV)
    tokens = torch.full((N,), 77, device=DEV)
    weight = torch.zeros(N, device=DEV)
    weight[-3:] = 1.0
    weight[0] = 1.0
    old, adv = torch.full((N,), -12.0, device=DEV), torch.ones(N, device=DEV)
    loss, logp, grad = snn.policy_time_loss(times, tokens, old, adv, weight=weight)
    one = snn.policy_time_loss(times[-3:], tokens[-3:], old[-3:], adv[-3:], weight=weight[-3:])
    assert torch.allclose(loss[-3:], one[0], rtol=1e-4) and torch.allclose(logp[-3:], one[1], rtol=1e-5)
    assert torch.allclose(grad[-3:].float(), one[2].float(), rtol=2.0 ** -7, atol=1e-12)
    assert abs(float(logp[0]) + math.log(J)) < 1e-5 and (grad[1:-3] == 0).all()


def test_refusals():
    import snntc_amd as snn
    times, tokens, gen = _case((4, 3), 5, torch.float32)
    times, tokens = times.to(DEV), tokens.to(DEV)
    f = torch.zeros(4, 3, device=DEV)
    with pytest.raises(TypeError, match="int64"):
        snn.policy_time_loss(times, tokens.int(), f, f)
    with pytest.raises(ValueError, match="actions must have shape"):
        snn.policy_time_loss(times, tokens[:, :2], f, f)
    with pytest.raises(ValueError, match="advantage must have shape"):
        snn.policy_time_loss(times, tokens, f, f[:2])
    with pytest.raises(TypeError, match="times must be float32, bfloat16 or float16"):
        snn.policy_time_loss(times.double(), tokens, f, f)
    with pytest.raises(ValueError, match="at least 2 dimensions"):
        snn.time_logp(times[0, 0], tokens[0, 0])
    with pytest.raises(ValueError, match="outside its range"):
        snn.policy_time_loss(times, tokens, f, f, clip=(-0.1, 0.2))
    with pytest.raises(ValueError, match="outside its range"):
        snn.policy_time_loss(times, tokens, f, f, f, kl_coef=float("inf"))
    with pytest.raises(ValueError, match="must not require a gradient"):
        snn.policy_loss(times, tokens, f, f.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="2 pairs"):
        snn.preference_time_loss(times[:3], tokens[:3], f[0])
    with pytest.raises(ValueError, match="ref_logp must have shape"):
        snn.preference_time_loss(times, tokens, f[:3, 0])
    with pytest.raises(ValueError, match="outside its range"):
        snn.preference_time_loss(times, tokens, f[:, 0].contiguous(), smoothing=1.5)
    with pytest.raises(ValueError, match="without outputs"):
        snn.time_logp(times[..., :0], tokens)
    with pytest.raises(snn.SnntcLibraryError, match="lives on cpu"):
        snn.time_logp(times, tokens.cpu())


def test_gradient_by_differences():
    import snntc_amd as snn
    times, tokens, gen = _case((4, 3), 6, torch.float32)
    old, adv, ref = _policy_inputs(times, tokens, gen)
    leaf = times.to(DEV).requires_grad_(True)
    (g,) = torch.autograd.grad(snn.policy_loss(leaf, tokens.to(DEV), old.to(DEV), adv.to(DEV), ref.to(DEV), clip=CLIP, kl_coef=KL), [leaf])
    rl = torch.randn(4, generator=gen) - 5.0
    (h,) = torch.autograd.grad(snn.preference_loss(leaf, tokens.to(DEV), rl.to(DEV), beta=BETA), [leaf])
    for i in range(0, times.numel(), 5):
        ends, pref = [], []
        for s in (1e-6, -1e-6):
            t = times.double().clone()
            t.view(-1)[i] += s
            ends.append(_objective(t, tokens, old, adv, ref))
            pref.append(_preference_objective(t, tokens, rl))
        # differences: 1e-12 of the third derivative and 1e-16 / 1e-6 of rounding
        assert abs(float(g.view(-1)[i]) - (ends[0] - ends[1]) / 2e-6) < 1e-6 + 1e-5 * abs(float(g.view(-1)[i]))
        assert abs(float(h.view(-1)[i]) - (pref[0] - pref[1]) / 2e-6) < 1e-6 + 1e-5 * abs(float(h.view(-1)[i]))


def _objective(t, tokens, old, adv, ref):
    logp = torch.log_softmax(-t, -1).gather(-1, tokens[..., None])[..., 0]
    r, d = torch.exp(logp - old.double()), ref.double() - logp
    A = adv.double()
    return float((KL * (torch.exp(d) - d - 1) - torch.minimum(r * A, r.clamp(1 - CLIP[0], 1 + CLIP[1]) * A)).mean())


def _preference_objective(t, tokens, ref):
    seq = torch.log_softmax(-t, -1).gather(-1, tokens[..., None])[..., 0].sum(1) - ref.double()
    P = len(seq) // 2
    return float(torch.nn.functional.softplus(-BETA * (seq[:P] - seq[P:])).mean())


def test_a_graph_is_walked_twice_or_freed():
    import snntc_amd as snn
    times, tokens, gen = _case((4, 3), 6, torch.float32)
    leaf = times.to(DEV).requires_grad_(True)
    ref = torch.zeros(4, device=DEV)
    loss = snn.preference_loss(leaf, tokens.to(DEV), ref)
    a = torch.autograd.grad(loss, [leaf], retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(loss, [leaf])[0])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, [leaf])
    loss = snn.preference_loss(leaf, tokens.to(DEV), ref)
    with torch.no_grad():
        leaf.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
