"""The AdamW update, its states in 8 bits and the norm over all gradients against plain implementations in 64 bits.

Tolerances.  float32 states: m is two products and a sum over gradients that were scaled (and constants, each half a step off), 5 half steps of
the terms; v one more product, 7; a weight's change is m over a root: 5 + 7 / 2, root, sum, division, two constants, at most 16 half steps of what
it is with the terms of m in m's place, and the weight has two roundings of its own.  8-bit states are 64 bits wide between their
codes: the codes are those of the definition, the scales one rounding to float32."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = 2.0 ** -24
STEP16 = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
VALUES = {"m": np.array([c if c < 8 else (8 + c % 8) << (c // 8 - 1) for c in range(128)], np.float64),
          "v": np.array([c if c < 8 else (8 + c % 8) << (c // 8 - 1) for c in range(256)], np.float64)}


def _mix(x):
    x = ((x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)).astype(np.uint32)
    x = ((x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)).astype(np.uint32)
    return x ^ (x >> np.uint32(16))


def _bits(n, seed, step, tensor):
    key = np.zeros(1, np.uint32)
    for word in (tensor, step, seed >> 32, seed):
        key = _mix((key + np.uint32(word & 0xFFFFFFFF)).astype(np.uint32))
    return _mix((np.arange(n, dtype=np.uint64) * 0x9E3779B9 & 0xFFFFFFFF).astype(np.uint32) ^ key)


def _blocks(x):
    return np.concatenate([x, np.zeros(-len(x) % 256)]).reshape(-1, 256)


def _decode(codes, scale, which):
    c = codes.cpu().numpy().reshape(-1)
    value = VALUES[which] / VALUES[which][-1]
    sign = np.where(c >= 128, -1.0, 1.0) if which == "m" else 1.0
    return value[c % 128 if which == "m" else c] * sign * np.repeat(scale.cpu().numpy().astype(np.float64), 256)[:len(c)]


def _encode(x, part, which):
    """Codes by search in the list of values."""
    values = VALUES[which]
    scale = np.abs(_blocks(x)).max(1).astype(np.float32)
    s = np.repeat(scale.astype(np.float64), 256)[:len(x)]
    y = np.divide(np.abs(x) * values[-1], s, out=np.zeros_like(x), where=s > 0)
    low = np.clip(np.searchsorted(values, y, side="right") - 1, 0, len(values) - 2)
    up = (y - values[low]) / (values[low + 1] - values[low]) + (part + 0.5) / 65536 >= 1.0
    code = low + up
    return np.where((x < 0) & (which == "m"), code + 128, code).astype(np.uint8), scale


LR, B1, B2, EPS, DECAY = 3e-3, 0.9, 0.99, 1e-8, 0.05
SIZES = [(1,), (255,), (256,), (257,), (3, 171), (1024, 2), (2049,), (77, 131), (0, 5), (4096,)]


def _tensors(seed, dtype, sizes=SIZES, scale=0.1):
    gen = torch.Generator().manual_seed(seed)
    r = lambda s: torch.randn(s, generator=gen)                                       # noqa: E731
    ws, gs = [r(s).to(dtype).to(DEV) for s in sizes], [(scale * r(s) * torch.exp(r(s))).to(dtype).to(DEV) for s in sizes]
    ms, vs = [0.05 * r(s).to(DEV) for s in sizes], [0.01 * (r(s) ** 2).to(DEV) for s in sizes]
    return ws, gs, ms, vs


def _coded(seed, sizes):
    gen = torch.Generator().manual_seed(seed)
    codes = [[torch.randint(0, 256, s, generator=gen, dtype=torch.uint8).to(DEV) for s in sizes] for _ in range(2)]
    scales = [[(0.1 * torch.rand(-(-math.prod(s) // 256), generator=gen)).to(DEV) for s in sizes] for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def _f64(t):
    return t.detach().cpu().double().numpy().reshape(-1).copy()


def _expected(w, g, m, v, t, share=1.0):
    g = g * share
    m, terms = B1 * m + (1 - B1) * g, np.abs(B1 * m) + np.abs((1 - B1) * g)
    v = B2 * v + (1 - B2) * g * g
    d = LR / (1 - B1 ** t) / (np.sqrt(v / (1 - B2 ** t)) + EPS)
    return w * (1 - LR * DECAY) - d * m, m, v, terms, d


def _check_weights(got, want, before, moved, dtype, bits):
    got = _f64(got)
    limit = HALF * (3 * np.abs(before) + 16 * moved)
    if dtype == torch.float32:
        assert np.all(np.abs(got - want) <= limit)
        return
    # one of the two neighbours of the exact weight, and the one that the bits name where the place between them is clear
    size = np.maximum(np.abs(want), 2.0 ** (-126 if dtype == torch.bfloat16 else -14))
    step = np.exp2(np.floor(np.log2(size))) * STEP16[dtype]
    low = np.floor(np.abs(want) / step)
    place = np.abs(want) / step - low
    q = low + (place * 65536 > bits)
    near = np.abs(place * 65536 - bits) <= limit / step * 65536 + 1
    edge = (place < limit / step) | (place > 1 - limit / step)
    assert np.all((np.abs(got) == q * step) | near | edge) and near.mean() < 0.02
    assert np.all(np.abs(got - want) <= step + limit)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step,clip", [(1, False), (7, True)])
def test_a_step_with_states_in_32_bits(dtype, step, clip):
    import snntc_amd as snn
    ws, gs, ms, vs = _tensors(1, dtype)
    before = [[_f64(x) for x in t] for t in zip(ws, gs, ms, vs)]
    norm = snn.grad_norm(gs)
    exact = math.sqrt(sum(float((b[1] ** 2).sum()) for b in before))
    assert abs(float(norm) - exact) <= 2 * HALF * exact
    share = min(1.0, 2.0 / float(norm)) if clip else 1.0
    assert share < 1.0 or not clip
    version = [w._version for w in ws]
    snn.adamw_update(ws, gs, ms, vs, step, LR, (B1, B2), EPS, DECAY, norm=norm if clip else None, max_norm=2.0, seed=5)
    assert all(w._version > k for w, k in zip(ws, version))
    for i, (w, g, m, v) in enumerate(before):
        if not len(w):
            continue
        want, m1, v1, terms, d = _expected(w, g, m, v, step, share)
        assert np.all(np.abs(_f64(ms[i]) - m1) <= 5 * HALF * terms) and np.all(np.abs(_f64(vs[i]) - v1) <= 7 * HALF * v1)
        third = (_bits(len(w), 5, step, i).astype(np.uint64) * 0x9E3779B9 & 0xFFFFFFFF) >> 16
        _check_weights(ws[i], want, w, d * terms, dtype, third.astype(np.float64))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seed", [0, 3 + (9 << 32), (1 << 64) - 5])
def test_a_step_with_states_in_8_bits(dtype, seed):
    import snntc_amd as snn
    ws, gs, _, _ = _tensors(2, dtype)
    gs[3].zero_()
    m, v, ms, vs = _coded(3, SIZES)
    for lists in (m, v, ms, vs):
        lists[3].zero_()                                         # a tensor that begins, with no gradient: stays all zero
    before = [(_f64(w), _f64(g), _decode(a, c, "m"), _decode(b, d, "v")) for w, g, a, b, c, d in zip(ws, gs, m, v, ms, vs)]
    read = snn.adamw_moments(m, v, ms, vs)
    for i, b in enumerate(before):
        assert np.array_equal(read[0][i].cpu().numpy().reshape(-1), b[2].astype(np.float32))
        assert np.array_equal(read[1][i].cpu().numpy().reshape(-1), b[3].astype(np.float32))
    norm = snn.grad_norm(gs)
    share = min(1.0, 2.0 / float(norm))
    snn.adamw_update(ws, gs, m, v, 4, LR, (B1, B2), EPS, DECAY, norm, 2.0, ms, vs, seed)
    for i, (w, g, a, b) in enumerate(before):
        if not len(w):
            continue
        want, m1, v1, terms, d = _expected(w, g, a, b, 4, share)
        bits = _bits(len(w), seed, 4, i)
        for codes, scales, x, which, part in ((m[i], ms[i], m1, "m", bits & np.uint32(0xFFFF)), (v[i], vs[i], v1, "v", bits >> np.uint32(16))):
            c, s = _encode(x, part.astype(np.float64), which)
            assert np.array_equal(scales.cpu().numpy(), s)
            got = codes.cpu().numpy().reshape(-1)
            assert np.array_equal(np.where(c == 128, 0, c), np.where(got == 128, 0, got))        # (minus zero is zero)
        third = (bits.astype(np.uint64) * 0x9E3779B9 & 0xFFFFFFFF) >> 16
        _check_weights(ws[i], want, w, d * terms, dtype, third.astype(np.float64))
    assert not bool(m[3].any() or v[3].any() or ms[3].any() or vs[3].any())


def test_many_tensors_of_all_types_in_one_call():
    """More tensors than a launch takes, types mixed, as one by one."""
    import snntc_amd as snn
    sizes = [(1 + 37 * i % 700,) for i in range(150)]
    types = [(torch.float32, torch.bfloat16, torch.float16)[i % 3] for i in range(150)]
    ws, gs, ms, vs = _tensors(4, torch.float32, sizes)
    ws, gs = [w.to(t) for w, t in zip(ws, types)], [g.to(t) for g, t in zip(gs, types)]
    whole = [[x.clone() for x in t] for t in (ws, gs, ms, vs)]
    snn.adamw_update(*whole, 3, LR, (B1, B2), EPS, DECAY, seed=8)
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(float(snn.grad_norm(gs)) - exact) <= 2 * HALF * exact and torch.equal(snn.grad_norm(gs), snn.grad_norm(gs))
    for i in range(150):
        one = [[x[i].clone()] for x in (ws, gs, ms, vs)]
        if types[i] == torch.float32:
            snn.adamw_update(*one, 3, LR, (B1, B2), EPS, DECAY, seed=8)
            assert all(torch.equal(a[0], b[i]) for a, b in zip(one, whole))
        else:                                                    # (other places in the list have other random bits)
            assert torch.equal(snn.adamw_update(*one, 3, LR, (B1, B2), EPS, DECAY, seed=8) or one[2][0], whole[2][i])
            assert bool(((one[0][0].double() - whole[0][i].double()).abs() <= 2.0 ** -6 * whole[0][i].double().abs() + 1e-6).all())


def test_views_that_start_anywhere():
    """Parts of one buffer with no gap between them, at every place of their type."""
    import snntc_amd as snn
    sizes = [5, 1, 259, 1030, 2, 511]
    for dtype in (torch.float32, torch.bfloat16):
        for coded in (False, True):
            ws, gs, ms, vs = _tensors(6, dtype, [(n,) for n in sizes])
            states = list(_coded(7, [(n,) for n in sizes])) if coded else [ms, vs]
            bufs = [torch.cat(t) for t in (ws, gs, *states)]
            packed = []
            for buf, t in zip(bufs, (ws, gs, *states)):
                ends = np.cumsum([x.numel() for x in t])
                packed.append([buf[e - x.numel():e] for e, x in zip(ends, t)])
            for w, g, st in ((ws, gs, states), (packed[0], packed[1], packed[2:])):
                more = dict(first_scale=st[2], second_scale=st[3]) if coded else {}
                snn.adamw_update(w, g, st[0], st[1], 2, LR, (B1, B2), EPS, DECAY, norm=snn.grad_norm(g), max_norm=0.5, seed=1, **more)
            for a, b in zip((ws, *states), (bufs[0], *bufs[2:])):
                assert torch.equal(torch.cat(a), b)


def test_a_norm_that_is_no_number_leaves_everything():
    import snntc_amd as snn
    for coded in (False, True):
        for bad in (math.nan, math.inf, -math.inf):
            ws, gs, ms, vs = _tensors(9, torch.float32)
            states = list(_coded(7, SIZES)) if coded else [ms, vs]
            gs[4][0, 0] = bad
            kept = [[x.clone() for x in t] for t in (ws, *states)]
            more = dict(first_scale=states[2], second_scale=states[3]) if coded else {}
            count = torch.tensor(6, dtype=torch.int64, device=DEV)
            snn.adamw_update(ws, gs, states[0], states[1], count, norm=snn.grad_norm(gs), max_norm=1.0, **more)
            assert all(torch.equal(a, b) for t, k in zip((ws, *states), kept) for a, b in zip(t, k)) and int(count) == 7
    huge = [torch.full((1000,), 1e25, device=DEV), torch.full((1000,), 1e-30, device=DEV)]
    assert abs(float(snn.grad_norm(huge)) / (1e25 * math.sqrt(1000)) - 1) < 1e-6           # squares beyond float32
    assert abs(float(snn.grad_norm(huge[1:])) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    assert float(snn.grad_norm([torch.zeros(0, device=DEV)])) == 0.0


def test_a_nan_reaches_its_weight_without_a_norm():
    import snntc_amd as snn
    w, g = [torch.ones(600, device=DEV)], [torch.ones(600, device=DEV)]
    g[0][300] = math.nan
    m, v, ms, vs = _coded(1, [(600,)])
    snn.adamw_update(w, g, m, v, 1, first_scale=ms, second_scale=vs)
    assert bool(w[0][300].isnan()) and int(w[0].isnan().sum()) == 1
    first, second = snn.adamw_moments(m, v, ms, vs)
    assert bool(first[0][256:512].isnan().all()) and not bool(first[0][:256].isnan().any() or first[0][512:].isnan().any())


@pytest.mark.parametrize("coded", [False, True])
def test_steps_counted_on_the_device_and_replayed(coded):
    """A captured step, replayed with other gradients, with eager work and synchronisations between, follows the eager steps."""
    import snntc_amd as snn
    sides = []
    for _ in range(2):
        ws, gs, ms, vs = _tensors(12, torch.bfloat16)
        states = list(_coded(13, SIZES)) if coded else [ms, vs]
        sides.append((ws, gs, states, torch.tensor(3, dtype=torch.int64, device=DEV)))

    def step(ws, gs, states, number):
        more = dict(first_scale=states[2], second_scale=states[3]) if coded else {}
        norm = snn.grad_norm(gs)
        snn.adamw_update(ws, gs, states[0], states[1], number, LR, (B1, B2), EPS, DECAY, norm=norm, max_norm=1.0, seed=3, **more)
        return norm

    snn.grad_norm(sides[0][1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(*sides[0])
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = step(*sides[1][:3], 4 + i)                        # eager, the number from the host
        assert torch.equal(norm, want) and int(sides[0][3]) == 4 + i
        for a, b in zip((sides[0][0], *sides[0][2]), (sides[1][0], *sides[1][2])):
            for x, y in zip(a, b):
                if x.dtype == torch.bfloat16 or not x.is_floating_point():
                    # 1 - b^t of the device's and the host's power may differ by a rounding; codes and weights by a step then
                    assert float((x.double() - y.double()).abs().gt(0).double().mean() if x.numel() else 0.0) <= 1e-3
                else:
                    assert torch.equal(x, y)
        for a, b in zip(sides[0][0], sides[1][0]):
            b.copy_(a)
        for k in (0, 1):
            for g in sides[k][1]:
                g.mul_(0.9)


def test_small_changes_of_16_bit_weights_are_not_lost():
    """A change of a hundredth of what a weight can tell apart: on average it arrives."""
    import snntc_amd as snn
    n, steps = 1 << 16, 20
    for dtype in (torch.bfloat16, torch.float16):
        w, g = [torch.full((n,), 1.5, dtype=dtype, device=DEV)], [torch.ones(n, dtype=dtype, device=DEV)]
        m, v = [torch.zeros(n, device=DEV)], [torch.zeros(n, device=DEV)]
        lr = STEP16[dtype] / 100
        for t in range(1, steps + 1):
            snn.adamw_update(w, g, m, v, t, lr, weight_decay=0.0, seed=2)
        moved = 1.5 - float(w[0].double().mean())
        # each step's rounding has at most the variance (1/100)(99/100) of a step squared; five deviations of the mean
        assert abs(moved - steps * lr) <= 5 * STEP16[dtype] * math.sqrt(steps / 100 / n) + 1e-4 * steps * lr


def test_8_bit_states_move_where_gradients_vanish():
    """A block with one large gradient that goes on and others that stop: their v falls as b2^t, on average, though each step is a
    hundredth of the distance between two codes."""
    import snntc_amd as snn
    n, steps = 256 * 256, 300
    w, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 0.5, device=DEV)]
    g[0][::256] = 1.0
    m, v = [torch.zeros(n, dtype=torch.uint8, device=DEV)], [torch.zeros(n, dtype=torch.uint8, device=DEV)]
    ms, vs = [torch.zeros(n // 256, device=DEV)], [torch.zeros(n // 256, device=DEV)]
    snn.adamw_update(w, g, m, v, 1, betas=(0.9, 0.0), first_scale=ms, second_scale=vs, seed=4)            # v = g^2
    small = torch.ones(n, dtype=torch.bool, device=DEV)
    small[::256] = False
    start = float(snn.adamw_moments(m, v, ms, vs)[1][0][small].mean())
    assert abs(start - 0.25) < 0.01
    g[0][small] = 0.0
    for t in range(2, steps + 2):
        snn.adamw_update(w, g, m, v, t, betas=(0.9, 0.999), first_scale=ms, second_scale=vs, seed=4)
    second = snn.adamw_moments(m, v, ms, vs)[1][0]
    # a step's rounding has a variance of at most 0.001 v times the distance of two codes, an eighth of v: a deviation of 20 % of v after
    # 300 steps for an element, 0.08 % for the mean of 65280; five of them, and a little for the moving grid
    assert abs(float(second[small].mean()) / (start * 0.999 ** steps) - 1) < 0.02
    assert bool((second[::256] - 1.0).abs().max() < 1e-5)


def test_refusals():
    import snntc_amd as snn
    w, g, m, v = (torch.ones(6, device=DEV) for _ in range(4))
    c, d, cs, ds = torch.zeros(6, dtype=torch.uint8, device=DEV), torch.zeros(6, dtype=torch.uint8, device=DEV), torch.zeros(1, device=DEV), torch.zeros(1, device=DEV)
    f = lambda w=w, g=g, m=m, v=v, step=1, **how: snn.adamw_update([w], [g], [m], [v], step, **how)                    # noqa: E731
    for call, error in (
            (lambda: f(w=w.double(), g=g.double()), TypeError), (lambda: f(g=g.bfloat16()), ValueError), (lambda: f(g=g[:5]), ValueError),
            (lambda: f(w=torch.ones(6, 2, device=DEV)[:, 0]), ValueError), (lambda: f(m=m[:5]), ValueError), (lambda: f(m=m.half()), TypeError),
            (lambda: f(g=g.cpu()), snn.SnntcLibraryError), (lambda: f(m=m.cpu()), snn.SnntcLibraryError),
            (lambda: f(m=w), ValueError), (lambda: f(v=m), ValueError), (lambda: f(g=w), ValueError), (lambda: f(step=0), ValueError),
            (lambda: f(step=torch.ones(1, device=DEV)), TypeError), (lambda: f(step=1.5), TypeError), (lambda: f(lr=-1.0), ValueError),
            (lambda: f(betas=(1.0, 0.9)), ValueError), (lambda: f(eps=0.0), ValueError), (lambda: f(norm=w[0].clone(), max_norm=0.0), ValueError),
            (lambda: f(norm=w), TypeError), (lambda: f(m=c, v=d), TypeError), (lambda: f(m=c, v=d, first_scale=[cs]), ValueError),
            (lambda: f(m=c, v=d, first_scale=[cs], second_scale=[torch.zeros(2, device=DEV)]), ValueError),
            (lambda: f(m=c, v=d, first_scale=[cs], second_scale=[cs]), ValueError),
            (lambda: snn.adamw_update([w, w], [g, g], [m, v], [v, m], 1), ValueError), (lambda: snn.adamw_update([w], [], [m], [v], 1), ValueError),
            (lambda: snn.adamw_update([w], [g], [m, m], [v], 1), ValueError), (lambda: snn.grad_norm([g.double()]), TypeError),
            (lambda: snn.adamw_moments([c], [d], [cs], None), (ValueError, TypeError)), (lambda: snn.adamw_moments([m], [v], [cs], [ds]), TypeError)):
        with pytest.raises(error):
            call()
    assert all(bool((x == 1).all()) for x in (w, g, m, v))
    w.requires_grad_()
    y = (w * w).sum()
    f(w=w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        x = [torch.ones(3, device=DEV) for _ in range(4)]
        snn.adamw_update(x[:1], x[1:2], x[2:3], x[3:], 1)


# ---- the optimizer -------------------------------------------------------------------------------------------------------------------


def _nets(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(20, 33), torch.nn.Tanh(), torch.nn.Linear(33, 7)).to(DEV)


def _train(net, opt, steps, gen):
    losses = []
    for _ in range(steps):
        x = torch.randn(16, 20, generator=gen).to(DEV)
        opt.zero_grad(set_to_none=True)
        loss = (net(x) - 1.0).square().mean()
        loss.backward()
        opt.step()
        losses.append(float(loss))
    return losses


def test_optimizer_follows_the_stock_one():
    import snntc_amd as snn
    a, b = _nets(), _nets()
    ours, stock = snn.optim.AdamW(a.parameters(), 0.01, max_norm=0.3), torch.optim.AdamW(b.parameters(), 0.01)
    for k in range(30):
        x = torch.randn(16, 20, generator=torch.Generator().manual_seed(k)).to(DEV)
        for net in (a, b):
            net.zero_grad()
            (net(x) - 1.0).square().mean().backward()
        # the same gradients for both: what differs is the update alone
        for p, q in zip(a.parameters(), b.parameters()):
            q.grad.copy_(p.grad)
        torch.nn.utils.clip_grad_norm_(b.parameters(), 0.3)
        ours.step()
        stock.step()
        for p, q in zip(a.parameters(), b.parameters()):
            # an update is at most some 0.01 x 3, off by 32 half steps, and the clip's own 1e-6 in its divisor
            assert float((p - q).detach().abs().max()) <= (k + 1) * (0.03 * 1e-5 + 4 * HALF * float(q.detach().abs().max()))


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_saves_and_resumes(bits):
    import copy
    import snntc_amd as snn
    net = _nets(1).bfloat16() if bits == 8 else _nets(1)
    def run(net, opt, first, last):
        for k in range(first, last):
            gen = torch.Generator().manual_seed(100 + k)
            for p in net.parameters():
                p.grad = torch.randn(p.shape, generator=gen).to(DEV).to(p.dtype)
            opt.step()
    make = lambda n, **how: snn.optim.AdamW(n.parameters(), 0.02, state_bits=bits, max_norm=1.0, seed=5, **how)            # noqa: E731
    opt = make(net)
    run(net, opt, 0, 4)
    for capturable in (False, True):
        other = copy.deepcopy(net)
        again = make(other, capturable=capturable)
        again.load_state_dict(copy.deepcopy(opt.state_dict()))
        for p, q in zip(net.parameters(), other.parameters()):
            assert all(opt.state[p][k].dtype == again.state[q][k].dtype for k in ("first", "second"))
        mine = copy.deepcopy(net)
        straight = make(mine)
        straight.load_state_dict(opt.state_dict())
        run(other, again, 4, 7)
        run(mine, straight, 4, 7)
        for p, q in zip(mine.parameters(), other.parameters()):
            assert torch.allclose(p.float(), q.float(), rtol=2.0 ** -7 if bits == 8 else 1e-6, atol=1e-6)
        if capturable:
            assert {int(again.state[p]["step"]) for p in other.parameters()} == {7}
    with pytest.raises(ValueError, match="not of"):
        snn.optim.AdamW(net.parameters(), state_bits=40 - bits).load_state_dict(opt.state_dict())


def test_optimizer_with_groups_and_tensors_that_join_later():
    import snntc_amd as snn
    ps = [torch.nn.Parameter(torch.randn(50, generator=torch.Generator().manual_seed(i)).to(DEV)) for i in range(4)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    ours = snn.optim.AdamW([{"params": ps[:2], "lr": 0.1}, {"params": ps[2:], "weight_decay": 0.0}], 0.01)
    stock = torch.optim.AdamW([{"params": qs[:2], "lr": 0.1}, {"params": qs[2:], "weight_decay": 0.0}], 0.01)
    for k in range(5):
        for i, (p, q) in enumerate(zip(ps, qs)):
            g = torch.randn(50, generator=torch.Generator().manual_seed(10 * k + i)).to(DEV)
            p.grad, q.grad = (g, g.clone()) if i != 1 or k >= 2 else (None, None)
        ours.step()
        stock.step()
    for p, q in zip(ps, qs):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-5)
    assert snn.optim.AdamW([torch.nn.Parameter(torch.ones(2, device=DEV))]).step(lambda: 3) == 3       # no gradients: nothing to do


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_in_a_captured_step(bits):
    import snntc_amd as snn
    net, eager = _nets(2), _nets(2)
    opt, ref = (snn.optim.AdamW(n.parameters(), 0.01, state_bits=bits, max_norm=1.0, capturable=True, seed=1) for n in (net, eager))
    xs = torch.randn(6, 16, 20, generator=torch.Generator().manual_seed(0)).to(DEV)
    x = xs[0].clone()

    def step(n, o, x):
        o.zero_grad(set_to_none=False)
        (n(x) - 1.0).square().mean().backward()
        o.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(net, opt, x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(net, opt, x)
    step(eager, ref, xs[0])
    for k in range(1, 6):
        x.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        step(eager, ref, xs[k])
        for p, q in zip(net.parameters(), eager.parameters()):
            assert torch.allclose(p, q, rtol=1e-5, atol=1e-6), k
    uncounted = snn.optim.AdamW(net.parameters(), 0.01)
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            uncounted.step()


def test_moments_are_tensors_of_their_own():
    import snntc_amd as snn
    m, v, ms, vs = _coded(5, SIZES)
    first, second = snn.adamw_moments(m, v, ms, vs)
    kept = [x.clone() for x in first + second]
    assert all(x.shape == y.shape and x.is_contiguous() for x, y in zip(first + second, m + v))
    first[5].fill_(7.0)
    first[5].requires_grad_()
    (first[5] * 2).sum().backward()
    assert bool((first[5].grad == 2).all()) and not first[4].requires_grad
    for x, y in zip(first[:5] + first[6:] + second, kept[:5] + kept[6:]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("coded", [False, True])
def test_calls_larger_than_the_caches(coded):
    """The form that goes past the caches, against the other one on parts of the same tensors."""
    import snntc_amd as snn
    n = (1 << 24) + 1234                                      # 28 or 16 bytes an element: above 2^28 bytes in all
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda: torch.randn(n, generator=gen, device=DEV)                             # noqa: E731
    w, g = r(), r()
    if coded:
        states = [torch.randint(0, 256, (n,), generator=gen, device=DEV).to(torch.uint8) for _ in range(2)]
        states += [torch.rand(-(-n // 256), generator=gen, device=DEV) for _ in range(2)]
    else:
        states = [r(), r().square()]
    before = [x.clone() for x in (w, *states)]
    more = lambda s: dict(first_scale=[s[2]], second_scale=[s[3]]) if coded else {}   # noqa: E731
    snn.adamw_update([w], [g], [states[0]], [states[1]], 3, seed=1, **more(states))
    size = 1 << 20                                            # a multiple of 256; the first part has the same places of its elements
    part = [x[:size].clone() if i < 3 else x[:size // 256].clone() for i, x in enumerate(before)]
    snn.adamw_update([part[0]], [g[:size].clone()], [part[1]], [part[2]], 3, seed=1, **more(part[1:]))
    assert torch.equal(w[:size], part[0])
    for x, y in zip(states, part[1:]):
        assert torch.equal(x[:y.numel()], y)
    if coded:
        first, _ = snn.adamw_moments([states[0]] * 2, [states[1]] * 2, [states[2]] * 2, [states[3]] * 2)
        assert torch.equal(first[0], first[1])
        assert torch.equal(first[0][:size], snn.adamw_moments([part[1]], [part[2]], [part[3]], [part[4]])[0][0])
    # the rest, by the formula in 64 bits
    if not coded:
        m = 0.9 * before[1].double() + 0.1 * g.double()
        assert bool(((states[0] - m).abs() <= 5 * HALF * (before[1].abs() + g.abs())).all())


def _two_groups(n=4):
    return [torch.nn.Parameter(torch.randn(50, generator=torch.Generator().manual_seed(i)).to(DEV)) for i in range(n)]


def _give(ps, k, skip=()):
    for i, p in enumerate(ps):
        p.grad = None if i in skip else torch.randn(50, generator=torch.Generator().manual_seed(10 * k + i)).to(DEV)


def test_groups_that_resume_count_for_themselves():
    import snntc_amd as snn
    ps, qs = _two_groups(), _two_groups()
    make = lambda a, **how: snn.optim.AdamW([{"params": a[:2], "lr": 0.1}, {"params": a[2:]}], 0.01, **how)                # noqa: E731
    plain, counted = make(ps), make(qs, capturable=True)
    for k in range(2):
        _give(ps, k)
        _give(qs, k)
        plain.step()
        counted.step()
    again = make(qs, capturable=True)
    again.load_state_dict(counted.state_dict())
    for k in range(2, 5):
        _give(ps, k)
        _give(qs, k)
        plain.step()
        again.step()
        assert [int(again.state[q]["step"]) for q in qs] == [k + 1] * 4
    for p, q in zip(ps, qs):
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-6)


def test_a_tensor_without_a_gradient_does_not_count():
    """Tensors that began together share a counter on the device until one of them sits a step out."""
    import snntc_amd as snn
    ps, qs = _two_groups(), _two_groups()
    plain, counted = snn.optim.AdamW(ps, 0.01), snn.optim.AdamW(qs, 0.01, capturable=True)
    for k, skip in enumerate(((), (1,), (1, 2), (), (3,))):
        _give(ps, k, skip)
        _give(qs, k, skip)
        plain.step()
        counted.step()
    assert [int(counted.state[q]["step"]) for q in qs] == [plain.state[p]["step"] for p in ps] == [5, 3, 4, 4]
    for p, q in zip(ps, qs):
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-6)


def test_a_captured_step_has_its_states_already():
    import snntc_amd as snn
    ps = _two_groups()
    _give(ps, 0)
    opt = snn.optim.AdamW(ps, 0.01, capturable=True)
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    assert all(bool((p != b).any()) for p, b in zip(ps, before))
    _give(ps, 1, (1,))
    with pytest.raises(RuntimeError, match="before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()


def test_a_refused_step_does_not_count():
    import snntc_amd as snn
    ps = _two_groups()
    opt = snn.optim.AdamW(ps, 0.01)
    _give(ps, 0)
    opt.step()
    _give(ps, 1)
    opt.state[ps[1]]["first"] = opt.state[ps[1]]["first"][:-1]
    with pytest.raises(ValueError):
        opt.step()
    assert [opt.state[p]["step"] for p in ps] == [1] * 4
