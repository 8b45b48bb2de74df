"""Padded batches of tokens: what lies behind a sequence's length is in no result and in no gradient."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("pad", [-1, 50])
def test_padding_outside_the_table_reaches_no_gradient(pad):
    """Padding tokens that are in no table make rows of NaN times.  Behind the lengths nobody reads them: the recurrence's gates are made
    of every step's times, but those of these steps have no gradient, and the weights' gradient is none of NaN times 0."""
    import snntc_amd as snn
    rng = np.random.default_rng(3)
    embed = snn.SNN_embedding(50, 24, weight=rng.random((50, 24))).to(DEV)
    recur = snn.SNN_recurrence(24, weight=rng.standard_normal((25, 24)) * 0.1).to(DEV)
    gen = torch.Generator().manual_seed(1)
    tok = torch.randint(0, 50, (5, 30), generator=gen)
    n = torch.tensor([30, 0, 7, 29, 1])
    behind = torch.arange(30)[None] >= n[:, None]
    up, upf = torch.randn(5, 30, 24, generator=gen).to(DEV), torch.randn(5, 24, generator=gen).to(DEV)
    results = []
    for filler in (0, pad):
        t = torch.where(behind, filler, tok).to(DEV)
        x = embed(t)
        y, final = recur(x, None, n.to(DEV), return_state=True)
        results.append([y, final, *torch.autograd.grad([y, final], [recur.weight, embed.weight, x], [up, upf])])
    for a, b in zip(*results):
        assert torch.isfinite(b).all() and torch.equal(a, b)
    assert not results[1][-1][behind.to(DEV)].any()


def test_lengths_of_another_kind_are_refused_by_the_op():
    import snntc_amd as snn
    recur, x = snn.SNN_recurrence(4).to(DEV), torch.rand(3, 5, 4, device=DEV)
    with pytest.raises(ValueError, match="one entry per sequence"):
        recur(x, None, torch.tensor([5, 4], device=DEV))
    with pytest.raises(ValueError, match="one entry per sequence"):
        recur(x, None, torch.tensor([[5, 4, 1]], device=DEV))
    with pytest.raises(TypeError, match="int64"):
        recur(x, None, torch.tensor([5, 4, 1], device=DEV, dtype=torch.int32))
    with pytest.raises(snn.SnntcLibraryError, match="lives on cpu"):
        recur(x, None, torch.tensor([5, 4, 1]))
