"""The optimizer with states in 8 bits where gradients of a block lie far apart."""
import numpy as np
import pytest
import torch

from test_gpu_adamw import SIZES, _bits, _coded, _encode, _f64, _decode, _tensors, _expected, LR, B1, B2, EPS, DECAY

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _steps(bits, r, rare, count, blocks=64):
    """The largest single change of a weight, in learning rates, of blocks with one gradient of 1 and others of r, some of them 0."""
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(3)
    p = torch.nn.Parameter(torch.zeros(blocks * 256, device=DEV))
    opt = snn.optim.AdamW([p], 1e-3, weight_decay=0.0, state_bits=bits, seed=5)
    largest = 0.0
    for _ in range(count):
        g = r * torch.randn(p.numel(), generator=gen) * (torch.rand(p.numel(), generator=gen) >= rare)
        g[::256] = 1.0
        p.grad = g.to(DEV)
        before = p.detach().clone()
        opt.step()
        largest = max(largest, float((p.detach() - before).abs().max()) / 1e-3)
    return largest, p.detach().clone()


@pytest.mark.parametrize("r", [1e-1, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("rare,count", [(0.5, 200), (0.97, 200)])
def test_steps_of_8_bit_states_are_bounded(r, rare, count):
    """Of any gradients m <= (1 - b1) / sqrt((1 - b2) (1 - b1^2 / b2)) sqrt(v), 7.3 sqrt(v).  A rounding at most doubles what is held of m
    and halves what is held of v: 7.3 x 2 sqrt 2, and (1 - b1) / sqrt(1 - b2) = 3.2 of the newest gradient, 24 learning rates."""
    eight, moved = _steps(8, r, rare, count)
    full, whole = _steps(32, r, rare, count)
    assert full <= 7.3 and eight <= 24.0, (eight, full)
    # no weight drifts further than it would if each of its steps were the largest that 32 bits took
    assert float(moved.abs().max()) <= 1e-3 * count * full


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_codes_of_paired_states(dtype):
    """Blocks in which half of the second moments are too small for their block: the definition's codes, first ones with their second."""
    import snntc_amd as snn
    ws, gs, _, _ = _tensors(2, dtype)
    m, v, ms, vs = _coded(3, SIZES)
    gen = torch.Generator().manual_seed(8)
    for g, second in zip(gs, v):
        small = (torch.rand(g.shape, generator=gen) < 0.5).to(DEV)
        g.mul_(torch.where(small, 2e-5, 1.0))
        second.mul_(~small)
    before = [(_f64(w), _f64(g), _decode(a, c, "m"), _decode(b, d, "v")) for w, g, a, b, c, d in zip(ws, gs, m, v, ms, vs)]
    apart = [[x.clone() for x in t] for t in (ws, m, v, ms, vs)]
    snn.adamw_update(ws, gs, m, v, 4, LR, (B1, B2), EPS, DECAY, None, 1.0, ms, vs, 6, True)
    snn.adamw_update(apart[0], gs, apart[1], apart[2], 4, LR, (B1, B2), EPS, DECAY, None, 1.0, apart[3], apart[4], 6)
    dropped = 0
    for i, (w, g, a, b) in enumerate(before):
        assert all(torch.equal(x[i], y[i]) for x, y in zip((ws, v, ms, vs), (apart[0], *apart[2:])))
        assert torch.equal(m[i], torch.where(v[i] == 0, 0, apart[1][i]))
        if not len(w):
            continue
        _, m1, v1, _, _ = _expected(w, g, a, b, 4)
        bits = _bits(len(w), 6, 4, i)
        second, _ = _encode(v1, (bits >> np.uint32(16)).astype(np.float64), "v")
        first, _ = _encode(m1, (bits & np.uint32(0xFFFF)).astype(np.float64), "m")
        got = m[i].cpu().numpy().reshape(-1)
        assert np.array_equal(v[i].cpu().numpy().reshape(-1), second)
        assert np.array_equal(np.where(got == 128, 0, got), np.where((second == 0) | (first == 128), 0, first))
        dropped += int(((second == 0) & (first % 128 != 0)).sum())
    assert dropped > 1000


def test_states_from_elsewhere_are_paired_when_they_are_loaded():
    import snntc_amd as snn
    p = torch.nn.Parameter(torch.ones(700, device=DEV))
    opt = snn.optim.AdamW([p], 1e-3, weight_decay=0.0, state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()
    saved = opt.state_dict()
    saved["state"][0]["second"][10:20] = 0                       # as an update that rounds them apart can leave them
    again = snn.optim.AdamW([p], 1e-3, weight_decay=0.0, state_bits=8)
    again.load_state_dict(saved)
    before = p.detach().clone()
    p.grad = torch.zeros_like(p)
    again.step()
    assert float((p.detach() - before).abs().max()) <= 1e-3 and bool((p.detach() == before)[10:20].all())


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
def test_copies_of_an_optimizer_go_on(bits, capturable):
    """Copied, or written and read back, between two steps: its own numbers, states and counters, as the one it was copied from."""
    import copy
    import io
    import pickle
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in (300, 7)]
    gs = [[torch.randn(p.shape, generator=gen).to(DEV) for p in ps] for _ in range(4)]
    opt = snn.optim.AdamW(ps, 1e-2, state_bits=bits, max_norm=0.5, seed=9, capturable=capturable)

    def go(opt, steps):
        for k in steps:
            for p, g in zip(opt.param_groups[0]["params"], gs[k]):
                p.grad = g.clone()
            opt.step()
        return [p.detach().clone() for p in opt.param_groups[0]["params"]]

    go(opt, (0, 1))
    saved = copy.deepcopy(opt.state_dict())                     # (by itself it goes on with the optimizer)
    copies = [copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))]
    torch.save(opt, buf := io.BytesIO())
    copies.append(torch.load(io.BytesIO(buf.getvalue()), weights_only=False))
    want = go(opt, (2, 3))
    for other in copies:
        assert other.norm is None and other.param_groups[0]["params"][0] is not ps[0]
        got = go(other, (2, 3))
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(other.norm, opt.norm)
        assert [int(s["step"]) for s in other.state.values()] == [4, 4]
    copies[0].load_state_dict(saved)
    assert [int(s["step"]) for s in copies[0].state.values()] == [2, 2]


def test_numbers_on_the_device_lie_apart_from_what_is_updated():
    """A norm or a step's number in the memory of a weight, a state or each other: every workgroup would read what others write."""
    import snntc_amd as snn
    buf = torch.ones(8, 6, device=DEV)
    w, g, m, v, a, b = (buf[i] for i in range(6))
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    number = lambda t: t[2:4].view(torch.int64)                                         # noqa: E731
    call = lambda step=1, norm=None: snn.adamw_update([w], [g], [m], [v], step, norm=norm)               # noqa: E731
    for how in (dict(norm=w[3]), dict(norm=m[0]), dict(norm=v[5]), dict(step=number(w)), dict(step=number(g)), dict(step=number(v)),
                dict(step=number(a), norm=a[3])):
        with pytest.raises(ValueError, match="overlap"):
            call(**how)
    assert bool((buf == 1).all())
    call(step, a[0])
    call(number(b.zero_()), g[0])                                # beside them, or read on both sides: as ever
    assert int(step) == int(number(b)) == 1


def test_a_call_without_elements_still_counts():
    import snntc_amd as snn
    step, none = torch.tensor(4, dtype=torch.int64, device=DEV), [torch.zeros(0, device=DEV)]
    snn.adamw_update([], [], [], [], step)
    assert int(step) == 5
    snn.adamw_update(none, none, none, none, step)
    assert int(step) == 6
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.adamw_update([], [], [], [], step.cpu())
    with pytest.raises(ValueError, match="as many states"):
        snn.adamw_update([], [], none, none, step)
