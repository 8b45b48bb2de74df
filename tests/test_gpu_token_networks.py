"""Networks over tokens: embedding, recurrence, dense layers and the losses over choices together, as they are used -- gradients
against differences and stock ops, training steps, serving token by token, captured graphs, streams, threads."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SPEC = [("embed", 50, 24), ("recur", 24), ("steps",), ("dense", 24, 40), ("dense", 40, 30)]


def _net(seed=0):
    from snntc_amd import networks
    return networks.build(SPEC, rng=np.random.default_rng(seed)).to(DEV)


def _batch(seed=0, B=6, T=20):
    gen = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, 50, (B, T), generator=gen).to(DEV)
    act = torch.randint(0, 30, (B, T), generator=gen).to(DEV)
    weight = (torch.arange(T)[None] < torch.randint(1, T + 1, (B, 1), generator=gen)).float().to(DEV)
    return tok, act, weight


def _stock(net, tok):
    """The same network with stock ops around the dense layers."""
    emb, rec = net[0], net[1]
    x = torch.exp(1.0 - emb.scale * emb.weight[tok])
    a = torch.sigmoid(rec.gates(x))
    h, ys = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        ys.append(h)
    return net[4](net[3](torch.stack(ys, 1).reshape(-1, x.shape[2])))


def test_policy_gradients_equal_the_stock_composition():
    import snntc_amd as snn
    net = _net()
    tok, act, weight = _batch()
    with torch.no_grad():
        old = snn.time_logp(net(tok).view(6, 20, 30), act)
    gen = torch.Generator().manual_seed(5)
    adv = torch.randn(6, 20, generator=gen).to(DEV)
    ref = old + 0.3 * torch.randn(6, 20, generator=gen).to(DEV)
    weight = weight / weight.sum()
    loss = snn.policy_loss(net(tok).view(6, 20, 30), act, old - 0.05, adv, ref, weight, kl_coef=0.1)
    got = torch.autograd.grad(loss, net.weights())
    logp = torch.log_softmax(-_stock(net, tok).view(6, 20, 30), -1).gather(-1, act[..., None])[..., 0]
    ratio = torch.exp(logp - (old - 0.05))
    d = ref - logp
    want_loss = (weight * (0.1 * (torch.exp(d) - d - 1) - torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv))).sum()
    want = torch.autograd.grad(want_loss, net.weights())
    assert torch.allclose(loss, want_loss, rtol=1e-4, atol=1e-6)
    for g, w in zip(got, want):
        # two float32 chains of the same mathematics: causal sets may differ where two times are equal but for a rounding
        assert float((g - w).norm()) <= 1e-3 * float(w.norm())


def test_preference_training_step_updates_every_weight():
    import snntc_amd as snn
    from snntc_amd import train
    net, other = _net(), _net()
    tok, act, weight = _batch()
    with torch.no_grad():
        ref = (snn.time_logp(net(tok).view(6, 20, 30), act, weight) * weight).sum(1) + torch.tensor([1.0, 0, 2, 0, 0, 3], device=DEV)
    loss = train.preference_step(net, torch.optim.SGD(net.parameters(), lr=0.1), tok, act, ref, weight)
    want = snn.preference_loss(other(tok).view(6, 20, 30), act, ref, weight)
    grads = torch.autograd.grad(want, other.weights())
    assert torch.equal(loss, want.detach())
    for w, w0, g in zip(net.weights(), other.weights(), grads):
        assert torch.allclose(w, w0 - 0.1 * g, rtol=1e-6, atol=1e-7) and bool((g != 0).any())
    loss = train.policy_step(net, torch.optim.SGD(net.parameters(), lr=0.1), tok, act, snn.time_logp(net(tok).view(6, 20, 30), act),
                             torch.ones(6, 20, device=DEV), weight=weight / weight.sum())
    assert abs(float(loss) + 1.0) < 1e-4                    # ratios of one, advantages of one


def test_steps_take_times_of_any_layout():
    """A model whose times are a view that is no plain block of memory."""
    from snntc_amd import train

    class Turned(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.times = torch.nn.Parameter(1.0 + torch.rand(20, 6, 30, device=DEV))

        def forward(self, _):
            return self.times.transpose(0, 1)

    _, act, weight = _batch()
    for step in (lambda m, o: train.policy_step(m, o, None, act, torch.full((6, 20), -3.0, device=DEV), torch.ones(6, 20, device=DEV)),
                 lambda m, o: train.preference_step(m, o, None, act, torch.zeros(6, device=DEV), weight)):
        turned, plain = Turned(), Turned()
        plain.times = torch.nn.Parameter(turned.times.detach().transpose(0, 1).contiguous())
        plain.forward = lambda _, m=plain: m.times
        got, want = (step(m, torch.optim.SGD(m.parameters(), lr=0.1)) for m in (turned, plain))
        assert torch.equal(got, want) and torch.equal(turned.times.transpose(0, 1), plain.times)


def test_sgd_update_takes_the_gradients():
    import snntc_amd as snn
    net = _net()
    tok, act, _ = _batch()
    before = [w.detach().clone() for w in net.weights()]
    loss = snn.policy_loss(net(tok).view(6, 20, 30), act, torch.full((6, 20), -3.0, device=DEV), torch.ones(6, 20, device=DEV))
    grads = torch.autograd.grad(loss, net.weights())
    snn.sgd_update([w.detach() for w in net.weights()], grads, 0.1)
    for w, b, g in zip(net.weights(), before, grads):
        assert torch.allclose(w, b - 0.1 * g, rtol=1e-6, atol=1e-7)


def test_serving_token_by_token():
    net = _net().eval()
    tok, _, _ = _batch()
    with torch.no_grad():
        want = net(tok).view(6, 20, 30)
        whole, _ = net[1](net[0](tok), return_state=True)
        state = torch.zeros(6, 24, device=DEV)
        for t in range(20):
            net[1].step(net[0](tok[:, t]), state, out=state)
            assert torch.allclose(state, whole[:, t], atol=1e-4)
            times = net[4](net[3](state))
            # a float32 sum of 24 or 40 terms over a difference that may be small: compare where it is not
            assert float(((times - want[:, t]).abs() <= 1e-3 * want[:, t].abs() + 1e-3).float().mean()) > 0.98


def _everything():
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(9)
    tok = torch.randint(0, 300, (9000,), generator=gen).to(DEV)
    table = torch.rand(300, 50, generator=gen).to(DEV)
    grad = torch.randn(9000, 50, generator=gen).to(DEV)
    x = torch.exp(torch.rand(2, 3000, 20, generator=gen)).to(DEV)
    gate = torch.randn(2, 3000, 20, generator=gen).to(DEV)
    n = torch.tensor([3000, 1234], device=DEV)
    small, wide = torch.rand(64, 10, generator=gen).to(DEV) * 5, torch.rand(4, 70000, generator=gen).to(DEV) * 9
    ka, kb = torch.randint(0, 10, (64,), generator=gen).to(DEV), torch.randint(0, 70000, (4, 1), generator=gen).to(DEV)
    f = torch.randn(64, generator=gen).to(DEV)

    def step():
        z = snn.embed_tokens(tok, table, 1.0, True)
        d = snn.embed_tokens_grad(grad, tok, table, 1.0, True)
        y, final = snn.gated_scan(x, gate, None, n)
        dx, dg, ds = snn.gated_scan_grad(x, None, x, gate, y, None, n)
        s = snn.gated_step(x[0, 0], gate[0, 0])
        p = snn.policy_time_loss(small, ka, f - 2.0, f, f - 1.5, kl_coef=0.1)
        q = snn.preference_time_loss(wide.view(4, 1, 70000), kb, f[:4].contiguous())
        return [z, d, y, final, dx, dg, ds, s, *p, *q]

    return step, [table, x, wide]


def test_graph_replays_match_eager():
    """A captured run of all the operators, with eager work, other inputs and synchronisations between the replays."""
    step, inputs = _everything()
    kept = [v.clone() for v in inputs]
    ref = [v.clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    torch.cuda.synchronize()
    for i in range(4):
        for o in out:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for k, (o, r) in enumerate(zip(out, ref)):
            assert torch.equal(o, r), f"replay {i}: output {k} differs from the eager result"
        for v in inputs:
            v.mul_(1.25)
        step()                                              # eager, on other inputs
        graph.replay()
        torch.cuda.synchronize()
        for k, (o, r) in enumerate(zip(out, step())):
            assert torch.equal(o, r), f"replay {i}: output {k} does not follow its inputs"
        for v, k in zip(inputs, kept):
            v.copy_(k)


def test_two_graphs_of_one_pool():
    """Workspaces of two graphs that share a pool do not overlap with what the other still needs."""
    import snntc_amd as snn
    step, _ = _everything()
    ref = [v.clone() for v in step()]
    gen = torch.Generator().manual_seed(2)
    tok, grad = torch.randint(0, 1000, (40000,), generator=gen).to(DEV), torch.randn(40000, 64, generator=gen).to(DEV)
    table = torch.rand(1000, 64, generator=gen).to(DEV)
    ref2 = snn.embed_tokens_grad(grad, tok, table).clone()
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, pool=pool):
        out1 = step()
    with torch.cuda.graph(g2, pool=pool):
        out2 = snn.embed_tokens_grad(grad, tok, table)
    for i in range(3):
        g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(out1, ref)), f"round {i}"
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, ref2), f"round {i}"


def test_threads_with_streams_of_their_own():
    step, _ = _everything()
    ref = [v.clone() for v in step()]
    torch.cuda.synchronize()
    failures = []

    def run(turn):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for k in range(6):
                    out = step()
                    stream.synchronize()
                    bad = [i for i, (o, r) in enumerate(zip(out, ref)) if not torch.equal(o, r)]
                    if bad:
                        failures.append((turn, k, bad))
        except Exception as e:                              # noqa: BLE001 -- reported by the main thread
            failures.append((turn, repr(e)))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failures


def test_a_second_derivative_is_refused():
    import snntc_amd as snn
    table = torch.rand(9, 4, device=DEV, requires_grad=True)
    k = torch.tensor([[1, 2], [2, 3]], device=DEV)
    x = torch.rand(2, 2, 4, device=DEV, requires_grad=True)
    f = torch.zeros(2, 2, device=DEV)
    for out, leaf in ((snn.SnnEmbed.apply(k, table), table), (snn.SnnGatedScan.apply(x, x)[0], x),
                      (snn.policy_loss(x, k, f, f + 1), x), (snn.preference_loss(x, k, f[0]), x)):
        (g,) = torch.autograd.grad((out * out).sum(), [leaf], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once only"):
            g.sum().backward()


def test_saved_tensor_hooks_inference_mode_and_transforms():
    import snntc_amd as snn
    net = _net()
    tok, act, _ = _batch()
    want = torch.autograd.grad(snn.preference_loss(net(tok).view(6, 20, 30), act, torch.zeros(6, device=DEV)), net.weights())
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        loss = snn.preference_loss(net(tok).view(6, 20, 30), act, torch.zeros(6, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, net.weights()), want))
    with torch.inference_mode():
        assert torch.equal(snn.preference_loss(net(tok).view(6, 20, 30), act, torch.zeros(6, device=DEV)), loss.detach())
    with torch.no_grad():
        assert not snn.gated_scan(torch.rand(1, 2, 3, device=DEV), torch.rand(1, 2, 3, device=DEV))[0].requires_grad
    # PyTorch's own Function classes of the same ops, which calls with transforms or modes in them go through
    from snntc_amd import ops
    table = torch.rand(9, 4, device=DEV, requires_grad=True)
    t = torch.tensor([1, 2, 2], device=DEV)
    a = ops.GENERAL["embed_layer"](t, table, 0.5, True)
    b = snn.SnnEmbed.apply(t, table, 0.5, True)
    assert torch.equal(a, b) and torch.equal(*(torch.autograd.grad(v.sum(), [table])[0] for v in (a, b)))
    x, g, s = (torch.rand(*sh, device=DEV, requires_grad=True) for sh in ((2, 5, 3), (2, 5, 3), (2, 3)))
    for state, lengths in ((s, None), (None, torch.tensor([5, 2], device=DEV))):
        leaves = [x, g] + ([s] if state is not None else [])
        outs = [f(x, g, state, lengths) for f in (ops.GENERAL["gated_layer"], snn.SnnGatedScan.apply)]
        grads = [torch.autograd.grad(y.sum() + 2 * f.sum(), leaves) for y, f in outs]
        assert all(torch.equal(p, q) for p, q in zip(*grads))
    times = (torch.rand(4, 3, 6, device=DEV) * 4).requires_grad_(True)
    k, f = torch.zeros(4, 3, dtype=torch.int64, device=DEV), torch.zeros(4, 3, device=DEV)
    pairs = [(ops.GENERAL["policy_layer"](times, k, f - 2, f + 1, f - 2, None, 0.2, 0.2, 0.1), snn.policy_loss(times, k, f - 2, f + 1, f - 2, kl_coef=0.1)),
             (ops.GENERAL["preference_layer"](times, k, f[:, 0].contiguous(), None, 0.1, 0.0), snn.preference_loss(times, k, f[:, 0].contiguous()))]
    for p, q in pairs:
        assert torch.equal(p, q)
        gp, gq = (torch.autograd.grad(v, [times])[0] for v in (p, q))
        assert torch.allclose(gp, gq, rtol=1e-5, atol=1e-8)
