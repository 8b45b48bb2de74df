"""The gated scan and its step at their limits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_step_of_nearly_all_elements_that_32_bits_count():
    import snntc_amd as snn
    torch.cuda.empty_cache()
    n = 2 ** 32 - 100
    if torch.cuda.mem_get_info()[0] < 10 * n + (4 << 30):
        pytest.skip("needs 45 GB of the card's memory")
    x = torch.ones(n, device=DEV)
    gate = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    x[-5:] = 3.0
    out = snn.gated_step(x, gate)
    assert (out[-5:] == 1.5).all()
    out[-5:] = 0.5
    assert all((part == 0.5).all() for part in out.split(2 ** 29))


U = 2.0 ** -24
GATES = torch.tensor([8.0, 9.0, 10.0, 11.0, 12.0, 13.0, 14.0, 15.0, 16.0, 17.0, 18.0])
# sequences cut along time, whole ones in groups of 32 channels, whole ones in groups of 64
FORMS = [(1, 40000), (2, 70001), (100, 30000), (200, 20000)]


def _constant(B, T):
    """Channels of one value throughout, none a power of two, and gates that keep nearly everything."""
    value = (1.0 + torch.arange(B * 11) * 0.00731).view(B, 11).to(DEV)
    return value, value[:, None].expand(B, T, 11).contiguous(), GATES.to(DEV).expand(B, T, 11).contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T", FORMS)
def test_a_mean_of_one_value_is_that_value(B, T, dtype):
    """The weights of a step add up to one within 2^-45 (64-bit sums and products, a reciprocal that is off by the square of a
    float32 one's error), and so 70001 of them leave less than 2^-28: not a half step of the value, which comes back as it was."""
    import snntc_amd as snn
    value, x, gate = _constant(B, T)
    y, final = snn.gated_scan(x, gate.to(dtype), value)
    assert torch.equal(final, value) and torch.equal(y, x)


def test_steps_of_one_value_stay_there():
    import snntc_amd as snn
    value, x, gate = _constant(3, 1)
    x, gate, state = x[:, 0].contiguous(), gate[:, 0].contiguous(), value.clone()
    for _ in range(20000):
        snn.gated_step(x, gate, state, out=state)
    assert torch.equal(state, value)


@pytest.mark.parametrize("B,T", FORMS)
def test_a_mean_lies_between_its_smallest_and_largest_value(B, T):
    import snntc_amd as snn
    gen = torch.Generator(device=DEV).manual_seed(T)
    x = 1.0 + 2.0 * torch.rand(B, T, 11, generator=gen, device=DEV)
    x[:, T // 2:] = x[:, T // 2, None]                           # a stretch of one value to come close to
    s = 1.0 + 2.0 * torch.rand(B, 11, generator=gen, device=DEV)
    gate = (GATES.to(DEV) - 8.0) + torch.randn(B, T, 11, generator=gen, device=DEV)
    y, final = snn.gated_scan(x, gate, s)
    for part in (slice(0, T), slice(0, T // 2)):
        low, high = torch.minimum(x[:, part].amin(1), s), torch.maximum(x[:, part].amax(1), s)
        assert (y[:, part] >= low[:, None]).all() and (y[:, part] <= high[:, None]).all()
    assert torch.equal(final, y[:, -1])


@pytest.mark.parametrize("B,T", FORMS)
def test_gradients_through_gates_that_keep_nearly_everything(B, T):
    """A gradient at the end reaches step t times a^(T - t).  1 - a = exp(-gate) / (1 + exp(-gate)) is off by at most seven half steps of float32
    (the exponential by two steps, the reciprocal by one, their product by a half): call it eight, then a power n of a is off by n (1 - a)
    times as many, and each result by four more roundings."""
    import snntc_amd as snn
    value, x, gate = _constant(B, T)
    y, _ = snn.gated_scan(x, gate, value)
    dx, dgate, dstate = snn.gated_scan_grad(None, torch.ones(B, 11, device=DEV), x, gate, y, value)
    g = GATES.double().to(DEV)
    rest = torch.sigmoid(-g)
    log_a = -torch.nn.functional.softplus(-g)
    n = torch.arange(T - 1, -1, -1, device=DEV, dtype=torch.float64)[:, None]
    want = rest * torch.exp(n * log_a)
    assert ((dx.double() - want).abs() <= U * want * (8.0 * (n * rest + 1.0) + 4.0)).all()
    end = torch.exp(T * log_a)
    assert ((dstate.double() - end).abs() <= U * end * (8.0 * T * rest + 4.0)).all()
    assert (dgate.abs() <= 1e-20).all()                          # the state is the input throughout


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,D", [(3, 200, 224), (2, 300, 1056), (8, 700, 1024), (1, 384, 4128), (5, 129, 1000)])
def test_half_lines_of_gates_shared_by_neighbours(B, T, D, dtype):
    """Groups of 32 channels of 16-bit gates are dealt to the dies in another order than groups of 32-bit ones: with the same values the
    results are the same."""
    import snntc_amd as snn
    gen = torch.Generator(device=DEV).manual_seed(D)
    x = torch.exp(torch.rand(B, T, D, generator=gen, device=DEV))
    gate = (1.5 + 2.0 * torch.randn(B, T, D, generator=gen, device=DEV)).to(dtype)
    gy, n = torch.randn(B, T, D, generator=gen, device=DEV), torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(D)).to(DEV)
    y, final = snn.gated_scan(x, gate, None, n)
    y32, final32 = snn.gated_scan(x, gate.float(), None, n)
    assert torch.equal(y, y32) and torch.equal(final, final32)
    dx, dgate, dstate = snn.gated_scan_grad(gy, None, x, gate, y, None, n)
    dx32, dgate32, dstate32 = snn.gated_scan_grad(gy, None, x, gate.float(), y, None, n)
    assert torch.equal(dx, dx32) and torch.equal(dstate, dstate32)
    if dtype == torch.float16:
        # the last product and its rounding are one instruction (a product rounded once); rounded to float32 and then to float16 it can
        # come out a step away, where the first rounding ends in the middle of two float16 numbers
        low, high = (torch.nextafter(dgate32.to(dtype), torch.full_like(dgate, e)) for e in (-float("inf"), float("inf")))
        assert ((dgate >= low) & (dgate <= high)).all() and float((dgate != dgate32.to(dtype)).float().mean()) < 2.0 ** -10
    else:
        assert torch.equal(dgate, dgate32.to(dtype))
