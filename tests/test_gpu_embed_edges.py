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
