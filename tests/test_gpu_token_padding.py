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
    with pytest.raises(TypeError, match="lengths must be a torch.Tensor"):
        recur(x, None, [5, 4, 1])


def test_a_padded_training_step_from_tokens_to_the_loss():
    """The whole path, padding behind the lengths and of weight 0 in the loss: the same loss and the same gradients whatever the padding is."""
    import snntc_amd as snn
    from snntc_amd import networks
    net = networks.build([("embed", 50, 24), ("recur", 24), ("steps",), ("dense", 24, 40), ("dense", 40, 30)],
                         rng=np.random.default_rng(0)).to(DEV)
    gen = torch.Generator().manual_seed(4)
    tok, act = torch.randint(0, 50, (6, 20), generator=gen), torch.randint(0, 30, (6, 20), generator=gen).to(DEV)
    n = torch.tensor([20, 3, 0, 11, 19, 1])
    behind = torch.arange(20)[None] >= n[:, None]
    weight = (~behind).float().to(DEV) / float((~behind).sum())
    results = []
    for filler in (0, -1, 1 << 40):
        x = net[1](net[0](torch.where(behind, filler, tok).to(DEV)), None, n.to(DEV))
        times = net[4](net[3](net[2](x))).view(6, 20, 30)
        loss = snn.policy_loss(times, act, torch.full((6, 20), -3.0, device=DEV), torch.ones(6, 20, device=DEV), weight=weight)
        results.append([loss, *torch.autograd.grad(loss, net.weights())])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.isfinite(b).all() and torch.equal(a, b)
