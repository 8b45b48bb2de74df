"""Draws next to the borders of tokens' shares, under masks, in every form of the kernel.

The terms are exact: times are whole numbers and the temperature is 1 / ln 2 as the kernel has it, so that a term is a power of two and its
running sums in 64 bits are exact.  A lane's share ends every 4 (float32) or 8 (16-bit times) elements; around each end the uniform
numbers are tried that float32 sums of another order can mix up.

Tolerance of a draw, in half steps of float32 (2^-24) of the whole sum: a run's sum has 31 additions in a lane and 6 over lanes, 37; the pieces
before the token's, whose sums are subtracted, 7 + 6 together; the scan up to its lane 7 + 6, and a difference 1: 64, and 2 for what lies outside the run."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TEMPERATURE = 1.44269504


def _rows(n, J, dtype, width, gen):
    """Whole times, nearly all of the chance with the first 2048, and masks in runs of `width`."""
    times = torch.randint(0, 24, (n, J), generator=gen)
    times[:, 2048:] = 100
    mask = (torch.rand(n, -(-J // width), generator=gen) < 0.5).repeat_interleave(width, 1)[:, :J]
    mask[:, 5] = True
    return times.to(dtype).to(DEV), mask.to(DEV)


# one launch by 1, 4 and 16 wavefronts a row; slices of 512 and of 256 threads, joined by one wavefront and by four
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 8])
@pytest.mark.parametrize("J,n,rows", [(2048, 24, 8192), (5000, 12, 4096), (20000, 8, 250), (20000, 8, 2000), (40000, 6, 250), (40000, 6, 1000)])
def test_draws_next_to_a_border_are_allowed(J, n, rows, width, dtype):
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(J + rows + width)
    times, mask = _rows(n, J, dtype, width, gen)
    words = snn.pack_allowed(mask)
    p = torch.where(mask, torch.exp2(-times.double()), 0.0)
    cum = p.cumsum(1)
    step = 16 // times.element_size()
    for r in range(n):
        total = cum[r, -1]
        border = torch.round(cum[r, step - 1:2048:step] / total * 2.0 ** 24)
        u = torch.unique((border[:, None] + torch.arange(-2, 3, device=DEV)).clamp(0, 2.0 ** 24 - 1).reshape(-1)) / 2.0 ** 24
        for part in u.float().split(rows):
            k = part.numel()
            tokens, logp = snn.choose_tokens(times[r].expand(k, J), part, TEMPERATURE, allowed=words[r].expand(k, -1))
            assert bool((tokens >= 0).all()) and bool(mask[r][tokens].all()), part[~mask[r][tokens.clamp(min=0)]].tolist()
            assert bool((logp.double() - torch.log(p[r, tokens] / total)).abs().max() <= 64 * 2.0 ** -24 + 24 * 2.0 ** -23)
            at, upto = part.double() * total, cum[r, tokens]
            slack = 66 * 2.0 ** -24 * total
            assert bool(((upto - p[r, tokens] - slack <= at) & (at <= upto + slack)).all())


@pytest.mark.parametrize("J", [3, 700, 5000, 20000, 40000])
@pytest.mark.parametrize("rows", [6, 600])
def test_times_whose_quotient_by_the_temperature_is_no_float(J, rows):
    """Differences count, whatever their quotient: a far earlier time is drawn for sure, equal ones alike; times of infinity never are."""
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(J)
    u = torch.rand(rows, generator=gen).to(DEV)
    at = torch.randint(0, J, (rows,), generator=gen).to(DEV)
    for early, late, temperature in ((1e10, 2e10, 1e-29), (1e30, 2e30, 1e-10), (-1e38, 3e38, 1.0), (-3e38, 3e38, 0.5), (2.0, float("inf"), 1e-20)):
        times = torch.full((rows, J), late, device=DEV)
        times[torch.arange(rows, device=DEV), at] = early
        tokens, logp = snn.choose_tokens(times, u, temperature)
        assert torch.equal(tokens, at) and bool((logp == 0).all())
    for time, temperature in ((1e38, 0.01), (3e38, 1e-29), (-1e38, 1e-3)):
        times = torch.full((rows, J), time, device=DEV)
        times[:, 1::2] = float("inf")
        tokens, logp = snn.choose_tokens(times, u, temperature)
        n = (J + 1) // 2
        # equal terms of 1: sums of whole numbers are exact
        assert torch.equal(tokens, 2 * (u.double() * n).floor().long()) and bool((logp.double() + torch.log(torch.tensor(n, dtype=torch.float64))).abs().max() <= 2.0 ** -20)

def test_the_gradient_without_penalties_does_not_hold_the_times():
    """Delays and masks alone: the gradient reads neither the times nor their memory."""
    import snntc_amd as snn
    words = snn.pack_allowed(torch.arange(4096, device=DEV) % 3 > 0)
    leaf = torch.rand(1024, 4096, device=DEV, requires_grad=True)
    size = leaf.numel() * leaf.element_size()

    def ruled():
        return snn.rule_times(leaf * 1.0, allowed=words, delay=torch.ones(4096, device=DEV))

    ruled()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = ruled()
    assert torch.cuda.memory_allocated() - before < 1.5 * size               # the result, not the times beside it
    g = torch.rand_like(out)
    for grad in (g, g.t().contiguous().t(), g[:1].expand_as(g)):
        (got,) = torch.autograd.grad(out, [leaf], [grad], retain_graph=True)
        assert torch.equal(got, torch.where(torch.arange(4096, device=DEV) % 3 > 0, grad, 0.0))
