"""Losses over choices where a row, a pair or a limit is out of the ordinary."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("J", [10, 1000, 5001, 9000, 70000])
def test_rows_of_weight_zero_in_a_pair_without_a_margin(J, dtype):
    """A choice out of range makes its pair's margin NaN, and the gradient of the pair's rows; its rows of weight 0 are still not
    read and have none, and the other pair is as it was."""
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(J)
    times = (1.0 + 8.0 * torch.rand(4, 3, J, generator=gen)).to(dtype)
    tokens = torch.randint(0, J, (4, 3), generator=gen)
    ref = torch.tensor([-3.0, -4.0, -5.0, -6.0])
    weight = torch.tensor([[1.0, 0.0, 0.5], [1.0, 1.0, 0.0], [0.0, 2.0, 0.0], [0.0, 1.0, 1.0]])
    want = snn.preference_time_loss(*(v.to(DEV) for v in (times, tokens, ref, weight)))
    tokens[0, 2] = J
    times[weight == 0] = float("nan")
    tokens[weight == 0] = -7
    t, k, r, w = (v.to(DEV) for v in (times, tokens, ref, weight))
    loss, seq, grad = snn.preference_time_loss(t, k, r, w)
    leaf = t.clone().requires_grad_(True)
    (through,) = torch.autograd.grad(snn.preference_loss(leaf, k, r, w), [leaf])
    off = w == 0
    for g in (grad, through):
        assert (g[off] == 0).all()
        assert torch.isnan(g[0, [0, 2]]).all() and torch.isnan(g[2, 1]).all()
    assert torch.equal(grad[[1, 3]], want[2][[1, 3]])
    assert torch.equal(torch.isnan(loss), torch.tensor([True, False], device=DEV)) and torch.equal(loss[1], want[0][1])
    assert torch.equal(torch.isnan(seq), torch.tensor([True, False, False, False], device=DEV)) and torch.equal(seq[1:], want[1][1:])


@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
def test_sequences_that_cannot_occur(smoothing):
    """A sequence with an output that can never be chosen has log-probability minus infinity.  Where only the rejected one has, the
    margin is infinite: without smoothing the loss is 0, where only the preferred one has, infinite; a term of factor 0 is none."""
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(7)
    times = 1.0 + 8.0 * torch.rand(4, 3, 6, generator=gen)
    tokens = torch.zeros(4, 3, dtype=torch.int64)
    times[2, 1, 0] = math.inf                                   # the rejected one of pair 0
    times[1, 0, 0] = math.inf                                   # the preferred one of pair 1
    t, k, ref = times.to(DEV), tokens.to(DEV), torch.full((4,), -5.0, device=DEV)
    loss, seq, grad = snn.preference_time_loss(t, k, ref, beta=0.5, smoothing=smoothing)
    assert seq.tolist()[1:3] == [-math.inf, -math.inf]
    assert loss.tolist() == [0.0 if smoothing == 0.0 else math.inf, 0.0 if smoothing == 1.0 else math.inf]
    # d loss / d margin is the smoothing at plus infinity, the smoothing - 1 at minus infinity; times beta over the pairs
    slopes = torch.tensor([smoothing, smoothing - 1.0], dtype=torch.float64) * 0.5 / 2
    p = torch.softmax(-times.double(), -1)
    want = torch.cat([slopes, -slopes])[:, None, None] * (p - torch.nn.functional.one_hot(tokens, 6))
    assert torch.allclose(grad.double().cpu(), want, rtol=1e-5, atol=1e-7)


def _many_rows(rows, J):
    """Rows of weight 0, which are not read, but for the first and the last three; times that lie differently to 16 bytes than the
    gradient; None where the card has no room for both."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2 * rows * J * 2 + (4 << 30):
        return None
    gen = torch.Generator().manual_seed(J)
    times = torch.empty(rows * J + 1, dtype=torch.bfloat16, device=DEV)[1:].view(rows, J)
    some = torch.tensor([0, rows - 3, rows - 2, rows - 1], device=DEV)
    times[some] = (1.0 + 8.0 * torch.rand(4, J, generator=gen)).to(torch.bfloat16).to(DEV)
    tokens = torch.full((rows,), 77, device=DEV)
    weight = torch.zeros(rows, device=DEV)
    weight[some] = torch.tensor([1.0, 0.5, 0.25, 2.0], device=DEV)
    old, adv = torch.full((rows,), -8.0, device=DEV), torch.ones(rows, device=DEV)
    return [times, tokens, old, adv, weight], some


# Sums in another order and other pieces of a row: J / 64 + 40 roundings of 2^-24 at most on either side, and bfloat16's step.
def _like(a, b, dtype=torch.float32):
    return torch.allclose(a.float(), b.float(), rtol=2.0 ** -7 if dtype == torch.bfloat16 else 2e-5, atol=1e-12 if dtype == torch.bfloat16 else 2e-5)


def test_more_rows_than_a_grid_dimension_holds():
    """2^22 workgroups of 1024 threads."""
    import snntc_amd as snn
    made = _many_rows(2 ** 22 + 3, 1025)
    if made is None:
        pytest.skip("needs 22 GB of the card's memory")
    (times, tokens, old, adv, weight), some = made
    loss, logp, grad = snn.policy_time_loss(times, tokens, old, adv, weight=weight)
    one = snn.policy_time_loss(times[some], tokens[some], old[some], adv[some], weight=weight[some])
    assert _like(loss[some], one[0]) and _like(logp[some], one[1]) and _like(grad[some], one[2], torch.bfloat16)
    for v in (loss, logp, grad):
        v[some] = 0.0
        assert not v.any()


def test_more_slices_than_a_grid_dimension_holds():
    """The gradient from statistics of 2^23 rows of two slices each."""
    import snntc_amd as snn
    made = _many_rows(2 ** 23 + 3, 4097)
    if made is None:
        pytest.skip("needs 142 GB of the card's memory")
    (times, tokens, old, adv, weight), some = made
    leaf = times.requires_grad_(True)
    (grad,) = torch.autograd.grad(snn.policy_loss(leaf, tokens, old, adv, weight=weight), [leaf])
    one = snn.policy_time_loss(leaf.detach()[some], tokens[some], old[some], adv[some], weight=weight[some])
    assert _like(grad[some], one[2], torch.bfloat16)
    grad[some] = 0.0
    assert not any(part.any() for part in grad.split(2 ** 20))


@pytest.mark.parametrize("J", [100, 1000, 9000, 20000, 70000])
def test_float32_gradients_of_unlikely_outputs(J):
    """An element is a single exponential, times what its row has in common.  Of times in steps of 2^-10, whose differences are exact, it stands
    to the row's earliest output, whose exponential is 1, as exp of their difference: but for two steps of the exponential (4 half steps U of
    float32) and the product's rounding."""
    import snntc_amd as snn
    U = 2.0 ** -24
    gen = torch.Generator().manual_seed(J)
    times = (1.0 + torch.randint(0, 12 * 1024, (8, J), generator=gen) / 1024.0).float()
    times[:, :2] = 1.0
    want = torch.exp(1.0 - times.double())
    t, k = times.to(DEV), torch.zeros(8, dtype=torch.int64, device=DEV)
    old, adv = torch.full((8,), -3.0, device=DEV), -torch.ones(8, device=DEV)
    _, _, direct = snn.policy_time_loss(t, k, old, adv, clip=(1.0, 1e9))          # (never clipped)
    leaf = t.clone().requires_grad_(True)
    (saved,) = torch.autograd.grad(snn.policy_loss(leaf, k, old, adv, clip=(1.0, 1e9)), [leaf])
    for got in (direct, saved):
        g = got.double().cpu()
        error = (g[:, 2:] / (g[:, 1:2] * want[:, 2:]) - 1.0).abs().max()
        assert error <= 5.01 * U, f"{float(error / U):.1f} half steps"


@pytest.mark.parametrize("rows,J", [(191, 32801), (192, 32801), (200, 65536)])
def test_long_float32_rows_held_for_their_gradient(rows, J):
    """More than 8192 pieces of 16 bytes of float32, around the number of rows from which one workgroup keeps each."""
    from test_gpu_choice import _case, _check_policy, _policy_inputs
    times, tokens, gen = _case((rows,), J, torch.float32, spread=20.0)
    old, adv, ref = _policy_inputs(times, tokens, gen)
    _check_policy(times, tokens, old, adv, ref, None, same=False)
