"""The token table's gradient and the lookup at their limits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("N,V", [(12289, 3), (30000, 700), (40000, 64), (70001, 5000), (131072, 300000)])
@pytest.mark.parametrize("runs", [1, 3, 64, 100])
def test_every_position_is_placed_once(N, V, runs):
    """Gradients that are small whole numbers, whose sums are exact: a position that the sort lost or placed twice shows.  Runs of one
    token put many equal digits into the 64 entries that a wavefront places together."""
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(N + V + runs)
    tok = torch.randint(0, V, (N // runs + 1,), generator=gen).repeat_interleave(runs)[:N].to(DEV)
    grad = torch.randint(-8, 9, (N, 4), generator=gen).float().to(DEV)
    grad[:, 3] = 1.0
    want = torch.zeros(V, 4, device=DEV, dtype=torch.float64).index_add_(0, tok, grad.double())
    assert torch.equal(snn.embed_tokens_grad(grad, tok, torch.zeros(V, 4, device=DEV)).double(), want)


@pytest.mark.parametrize("N,D", [(2 ** 28 + 5, 3), (2 ** 29 + 9, 4)])
def test_more_tokens_than_a_grid_dimension_holds(N, D):
    """Some 2^24 workgroups: rows read element by element, and four elements at a time."""
    import snntc_amd as snn
    table = torch.randint(-64, 65, (1000, D), device=DEV).float()
    tok = torch.randint(0, 1000, (N,), device=DEV, dtype=torch.int32)
    tok[-2] = -1
    z = snn.embed_tokens(tok, table, 0.5)
    for first in range(0, N, 2 ** 24):                          # (an indexing of 2^26 rows of four is refused by PyTorch itself)
        part = slice(first, min(N, first + 2 ** 24))
        want = 0.5 * table[tok[part].clamp(min=0).long()]
        if part.stop == N:
            assert torch.isnan(z[-2]).all()
            z[-2], want[-2] = 0.0, 0.0
        assert torch.equal(z[part], want)


def test_a_table_that_is_not_encoded_may_change_before_its_gradient():
    """scale * table: the gradient does not read the table, so an update in between is no error; encoded, it does and is."""
    import snntc_amd as snn
    table = torch.rand(20, 6, device=DEV, requires_grad=True)
    tok, up = torch.randint(0, 20, (40,), device=DEV), torch.randn(40, 6, device=DEV)
    want = snn.embed_tokens_grad(up, tok, table.detach(), 0.5)
    from snntc_amd import ops
    for f in (snn.SnnEmbed.apply, ops.GENERAL["embed_layer"]):
        z = f(tok, table, 0.5, False)
        with torch.no_grad():
            table.mul_(0.5)
        (d,) = torch.autograd.grad(z, [table], up, retain_graph=True)
        assert torch.equal(d, want) and torch.equal(torch.autograd.grad(z, [table], up)[0], want)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(z, [table], up)
        z = f(tok, table, 0.5, True)
        with torch.no_grad():
            table.mul_(0.5)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(z, [table], up)
        z = f(tok, table, 0.5, False)
        with torch.no_grad():
            tok.clamp_(max=19)                                    # the tokens are read
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(z, [table], up)


def test_encoded_times_are_off_by_less_than_one_and_a_half_steps():
    """The hardware's exponential is off by a step, what its argument has lost is put back, and the result is rounded once: of intensities in
    steps of 2^-12, whose distance from one is exact, 3 half steps at most (and the loss put back has its own roundings: a percent)."""
    import snntc_amd as snn
    e = torch.arange(-8192, 8193, device=DEV).float().view(-1, 1) / 4096.0
    z = snn.embed_tokens(torch.arange(len(e), device=DEV), e, 1.0, True).double()
    want = torch.exp(1.0 - e.double())
    step = 2.0 ** (torch.floor(torch.log2(want)) - 23)
    worst, mean = float(((z - want).abs() / step).max()), float(((z - want).abs() / step).mean())
    assert worst <= 1.515, f"{worst:.3f} steps, {mean:.3f} in the mean"
    print(f"{worst:.3f} steps, {mean:.3f} in the mean")


def test_gradient_of_half_a_billion_positions():
    """Small whole numbers, whose sums are exact; some 500000 positions a token, spread over all chunks."""
    import snntc_amd as snn
    torch.cuda.empty_cache()
    N, V = 2 ** 29 + 7, 1009
    if torch.cuda.mem_get_info()[0] < 24 * N + (8 << 30):
        pytest.skip("needs 21 GB of the card's memory")
    tok = torch.randint(0, V, (N,), device=DEV, dtype=torch.int32)
    grad = torch.randint(-8, 9, (N, 1), device=DEV).float()
    tok[-3:] = torch.tensor([V, -1, 5], device=DEV)
    d = snn.embed_tokens_grad(grad, tok, torch.zeros(V, 1, device=DEV))
    want = torch.zeros(V + 1, device=DEV, dtype=torch.float64)
    for first in range(0, N, 2 ** 26):
        part = slice(first, min(N, first + 2 ** 26))
        t = tok[part].long()
        want.index_add_(0, torch.where((t >= 0) & (t < V), t, V), grad[part, 0].double())
    assert torch.equal(d[:, 0].double(), want[:V])
