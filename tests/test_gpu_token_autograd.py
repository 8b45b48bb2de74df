"""The differentiable operators over tokens and choices as PyTorch sees them: with tangents, transforms and modes each behaves as the
torch.autograd.Function it stands for, which refuses what the native node refuses and gives the same bits."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _rand(*shape, seed=0):
    return torch.rand(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(DEV)


def _ops():
    """name -> (function of the differentiated inputs, those inputs)"""
    import snntc_amd as snn
    tok = torch.tensor([[1, 2, 2], [0, 8, 1]], device=DEV)
    n = torch.tensor([5, 2], device=DEV)
    k = torch.randint(0, 6, (4, 3), generator=torch.Generator().manual_seed(1)).to(DEV)
    old, adv, ref, weight = -2.0 - _rand(4, 3), _rand(4, 3, seed=1) - 0.5, -2.0 - _rand(4, 3, seed=2), _rand(4, 3, seed=3)
    return {
        "embed": (lambda t: snn.SnnEmbed.apply(tok, t, 0.5, True), (_rand(9, 4),)),
        "embed_scaled": (lambda t: snn.SnnEmbed.apply(tok, t, 0.5, False), (_rand(9, 4),)),
        "scan": (lambda x, g, s: snn.SnnGatedScan.apply(x, g, s, n)[0], (_rand(2, 5, 3), _rand(2, 5, 3, seed=1), _rand(2, 3))),
        "scan_final": (lambda x, g: snn.SnnGatedScan.apply(x, g, None, None)[1], (_rand(2, 5, 3), _rand(2, 5, 3, seed=1))),
        "policy": (lambda t: snn.policy_loss(t, k, old, adv, ref, weight, kl_coef=0.1), (4 * _rand(4, 3, 6),)),
        "preference": (lambda t: snn.preference_loss(t, k, ref[:, 0].contiguous(), weight), (4 * _rand(4, 3, 6),)),
    }


OPS = ["embed", "embed_scaled", "scan", "scan_final", "policy", "preference"]


@pytest.mark.parametrize("name", OPS)
def test_tangents_and_transforms_are_refused(name):
    f, inputs = _ops()[name]
    for i in range(len(inputs)):
        with fwAD.dual_level():
            args = [fwAD.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(inputs)]
            with pytest.raises(NotImplementedError):
                f(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                f(*args)
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(*[t if i == j else u for j, u in enumerate(inputs)]).sum())(inputs[i])
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(*[torch.stack([t, t]) for t in inputs])


def _run(f, inputs, watch):
    args = [t.clone().requires_grad_(True) for t in inputs]
    if watch:
        with _Watch():
            return f(*args), args
    return f(*args), args


@pytest.mark.parametrize("watch", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_a_second_derivative_is_refused_on_either_path(name, watch):
    """Whether the upstream gradient depends on the inputs or not: what is differentiated again has to say that it cannot be, where a
    constant in its place would leave terms out."""
    f, inputs = _ops()[name]
    for objective in (lambda out: (out * out).sum(), lambda out: out.sum()):
        out, args = _run(f, inputs, watch)
        first = torch.autograd.grad(objective(out), args, create_graph=True)
        again, others = _run(f, inputs, watch)
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(objective(again), others)))
        for g in first:
            with pytest.raises(RuntimeError, match="differentiated once only"):
                torch.autograd.grad((g * g).sum() + sum((a * a).sum() for a in args), args, retain_graph=True)


@pytest.mark.parametrize("watch", [False, True])
def test_losses_refuse_other_inputs_that_require_a_gradient(watch):
    """Only the times have one: None in its place would leave it out without a word."""
    import contextlib
    import snntc_amd as snn
    times = (4 * _rand(4, 3, 6)).requires_grad_(True)
    k = torch.zeros(4, 3, dtype=torch.int64, device=DEV)
    f = -_rand(4, 3)
    names = ("old_logp", "advantage", "ref_logp", "weight")
    for name in names:
        args = {n: f.clone().requires_grad_(n == name) for n in names}
        with _Watch() if watch else contextlib.nullcontext():
            with pytest.raises(ValueError, match=f"policy loss: {name} must not require a gradient"):
                snn.policy_loss(times, k, **args, kl_coef=0.1)
    for name in ("ref_logp", "weight"):
        args = {n: t.clone().requires_grad_(n == name) for n, t in (("ref_logp", f[:, 0]), ("weight", f))}
        with _Watch() if watch else contextlib.nullcontext():
            with pytest.raises(ValueError, match=f"preference loss: {name} must not require a gradient"):
                snn.preference_loss(times, k, **args)


@pytest.mark.parametrize("name", OPS)
def test_the_function_and_the_native_node_agree(name):
    f, inputs = _ops()[name]
    (a, native), (b, function) = _run(f, inputs, False), _run(f, inputs, True)
    assert type(a.grad_fn).__name__ != type(b.grad_fn).__name__ and torch.equal(a, b)
    up = _rand(1, *a.shape, seed=5)[0]
    for x, y in zip(torch.autograd.grad(a, native, up), torch.autograd.grad(b, function, up)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_16_bits_are_rounded_once_behind_the_upstream_factor(dtype):
    """A loss scale keeps float16 gradients above its smallest numbers, 2^-24: they are not rounded before it is in them."""
    import snntc_amd as snn
    k = torch.randint(0, 6, (4, 3), generator=torch.Generator().manual_seed(2)).to(DEV)
    times = (4 * _rand(4, 3, 6)).to(dtype)
    old, adv = -2.0 - _rand(4, 3), _rand(4, 3, seed=1) - 0.5
    weight = torch.full((4, 3), 2.0 ** -30, device=DEV)
    # (ratios that are never clipped: every row has a gradient)
    for loss in (lambda t: snn.policy_loss(t, k, old, adv, weight=weight, clip=(1.0, 1e9)), lambda t: snn.preference_loss(t, k, old[:, 0].contiguous(), weight)):
        grads = []
        for watch in (False, True):
            out, (leaf,) = _run(loss, (times,), watch)
            grads += torch.autograd.grad(out * 2.0 ** 30, [leaf])
        assert torch.equal(*grads) and float((grads[0] != 0).float().mean()) > 0.9


def test_nothing_of_the_times_size_but_the_times_is_kept():
    import snntc_amd as snn
    times = (4 * _rand(4, 3, 600)).requires_grad_(True)
    k, f = torch.zeros(4, 3, dtype=torch.int64, device=DEV), -_rand(4, 3)
    for loss in (lambda: snn.policy_loss(times, k, f, f), lambda: snn.preference_loss(times, k, f[:, 0].contiguous())):
        for watch in (False, True):
            kept = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
                if watch:
                    with _Watch():
                        loss()
                else:
                    loss()
            assert kept and all(t.data_ptr() == times.data_ptr() or t.numel() <= 2 * k.numel() for t in kept)
