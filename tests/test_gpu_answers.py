"""Answers, losses over them and updates together, as they are used: tokens drawn by rules, a policy step through the same rules, AdamW."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SPEC = [("embed", 50, 24), ("recur", 24), ("steps",), ("dense", 24, 40), ("dense", 40, 50)]
RULES = dict(repetition=1.3, presence=0.2, frequency=0.1)


def _net(seed=0):
    from snntc_amd import networks
    return networks.build(SPEC, rng=np.random.default_rng(seed)).to(DEV)


def _drawn(seed=0, B=6, P=4, T=9, temperature=1.0):
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(seed)
    net = _net(seed)
    prompt = torch.randint(0, 50, (B, P), generator=gen).to(DEV)
    uniform = torch.rand(B, T, generator=gen).to(DEV)
    mask = torch.rand(B, 50, generator=gen).to(DEV) < 0.8
    mask[:, 0] = True
    rules = dict(RULES, allowed=snn.pack_allowed(mask), delay=(0.1 * torch.randn(50, generator=gen)).to(DEV))
    return net, prompt, uniform, mask, rules, snn.train.answer(net, prompt, uniform, temperature, **rules)


def test_answers_follow_rules_and_have_their_log_probabilities():
    import snntc_amd as snn
    net, prompt, _, mask, rules, (tokens, logp) = _drawn()
    assert tokens.shape == (6, 9) and bool(mask.gather(1, tokens).all())
    batch = snn.train.answer_batch(prompt, tokens, logp, torch.ones(6, device=DEV), **rules)
    with torch.no_grad():
        times = net(batch["inputs"]).view(6, 12, 50)
        again = snn.time_logp(snn.rule_times(times, **batch["rules"]), batch["actions"])
    # one pass over a sequence and steps through it sum in another order, and a causal set may differ where a time comes close to another
    close = (again[:, 3:] - logp).abs() <= 1e-2
    assert float(close.float().mean()) > 0.95
    assert torch.equal(batch["weight"] > 0, (torch.arange(12, device=DEV) >= 3).expand(6, 12)) and abs(float(batch["weight"].sum()) - 1) < 1e-5
    # at temperature 0 the earliest of the ruled times, but for what two ways of summing differ by
    greedy = snn.train.answer(net, prompt, torch.zeros(6, 1, device=DEV), 0.0, **rules)[0]
    with torch.no_grad():
        ruled = snn.rule_times(net(prompt).view(6, 4, 50)[:, -1], prompt, prompts=torch.full((6,), 4, device=DEV), **rules)
    assert bool((ruled.gather(1, greedy)[:, 0] <= ruled.amin(1) + 1e-2).all())


def test_policy_step_through_the_rules_equals_stock_operations():
    import snntc_amd as snn
    net, prompt, _, mask, rules, (tokens, logp) = _drawn(1)
    other = _net(1)
    gen = torch.Generator().manual_seed(5)
    advantage = torch.randn(6, generator=gen).to(DEV)
    batch = snn.train.answer_batch(prompt, tokens, logp, advantage, **rules)
    loss = snn.train.policy_step(net, torch.optim.SGD(net.parameters(), lr=0.1), **batch)
    times = other(batch["inputs"]).view(6, 12, 50)
    history = batch["rules"]["history"]
    seen, count = torch.zeros(6, 12, 50, device=DEV), torch.zeros(6, 12, 50, device=DEV)
    for r in range(12):
        for i in range(r + 1):
            seen[torch.arange(6), r, history[:, i]] = 1
            if i >= 4:
                count[torch.arange(6), r, history[:, i]] += 1
    u = torch.where(seen > 0, times * 1.3, times) + torch.where(count > 0, 0.2 + 0.1 * count, torch.zeros_like(count)) + rules["delay"]
    u = torch.where(mask[:, None], u, torch.full_like(u, float("inf")))
    lp = torch.log_softmax(-u, -1).gather(-1, batch["actions"][..., None])[..., 0]
    on = batch["weight"] > 0
    ratio = torch.exp(torch.where(on, lp - batch["old_logp"], torch.zeros_like(lp)))
    adv = batch["advantage"]
    want = -(torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) * batch["weight"]).sum()
    assert torch.allclose(loss, want.detach(), rtol=1e-4, atol=1e-5)
    for w, w0, g in zip(net.weights(), other.weights(), torch.autograd.grad(want, other.weights())):
        moved = (w0 - w).detach() / 0.1
        assert float((moved - g).norm()) <= 2e-3 * float(g.norm()) + 1e-5


@pytest.mark.parametrize("bits", [8, 32])
def test_rounds_of_answers_and_updates(bits):
    """Answer, policy step, AdamW: every weight moves, and a round with the same numbers gives the same weights."""
    import snntc_amd as snn
    ends = []
    for _ in range(2):
        net = _net(3)
        start = [w.detach().clone() for w in net.weights()]
        opt = snn.optim.AdamW(net.parameters(), 1e-3, state_bits=bits, max_norm=1.0, seed=9)
        gen = torch.Generator().manual_seed(4)
        for _ in range(3):
            prompt = torch.randint(0, 50, (8, 3), generator=gen).to(DEV)
            tokens, logp = snn.train.answer(net, prompt, torch.rand(8, 6, generator=gen).to(DEV), **RULES)
            reward = (tokens % 2 == 0).float().mean(1)
            snn.train.policy_step(net, opt, **snn.train.answer_batch(prompt, tokens, logp, reward - reward.mean(), **RULES))
            assert bool(torch.isfinite(opt.norm))
        assert all(bool((w != s).any() and torch.isfinite(w).all()) for w, s in zip(net.weights(), start))
        ends.append([w.detach().clone() for w in net.weights()])
    assert all(torch.equal(a, b) for a, b in zip(*ends))


def test_preference_step_through_rules():
    import snntc_amd as snn
    net, other = _net(2), _net(2)
    gen = torch.Generator().manual_seed(7)
    tok = torch.randint(0, 50, (4, 11), generator=gen).to(DEV)
    rules = dict(history=tok, lengths=torch.arange(1, 11, device=DEV).expand(4, 10), repetition=1.2)
    loss = snn.train.preference_step(net, torch.optim.SGD(net.parameters(), lr=0.1), tok[:, :-1], tok[:, 1:], torch.zeros(4, device=DEV), rules=rules)
    times = other(tok[:, :-1]).view(4, 10, 50)
    want = snn.preference_loss(snn.rule_times(times, **rules), tok[:, 1:], torch.zeros(4, device=DEV))
    assert torch.equal(loss, want.detach())
    for w, w0, g in zip(net.weights(), other.weights(), torch.autograd.grad(want, other.weights())):
        assert torch.allclose(w, w0 - 0.1 * g, rtol=1e-6, atol=1e-7)


def _everything():
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(9)
    f = lambda *s: torch.rand(*s, generator=gen).to(DEV)                                # noqa: E731
    small, wide = 1 + 5 * f(40, 30), 1 + 9 * f(5, 70000)
    hs, hw = torch.randint(0, 30, (40, 12), generator=gen).to(DEV), torch.randint(0, 70000, (5, 900), generator=gen).to(DEV)
    words = snn.pack_allowed(f(5, 70000) < 0.6)
    u, heat = f(40), 0.5 + f(5)
    w, g = [f(3000), f(17, 9)], [f(3000), f(17, 9)]
    count = torch.zeros((), dtype=torch.int64, device=DEV)

    def step():
        m, v = [torch.zeros_like(x) for x in w], [torch.zeros_like(x) for x in w]
        c, d = [torch.zeros(x.shape, dtype=torch.uint8, device=DEV) for x in w], [torch.zeros(x.shape, dtype=torch.uint8, device=DEV) for x in w]
        cs, ds = [torch.zeros(-(-x.numel() // 256), device=DEV) for x in w], [torch.zeros(-(-x.numel() // 256), device=DEV) for x in w]
        a, b = [x.clone() for x in w], [x.clone() for x in w]
        count.zero_()
        norm = snn.grad_norm(g)
        snn.adamw_update(a, g, m, v, count, norm=norm, max_norm=0.1)
        snn.adamw_update(b, g, c, d, count, norm=norm, max_norm=0.1, first_scale=cs, second_scale=ds, seed=3)
        first, second = snn.adamw_moments(c, d, cs, ds)
        return [snn.rule_times(small, hs, **RULES), snn.rule_times_grad(wide, wide, hw, None, 1.4, words),
                *snn.choose_tokens(small, u, 0.7, hs, **RULES), *snn.choose_tokens(wide, u[:5].contiguous(), heat, hw, allowed=words, **RULES),
                norm, *a, *m, *v, *b, *first, *second]

    return step, [small, wide, *g]


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
            o.fill_(-7)
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


def test_threads_with_streams_of_their_own():
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(1)
    times = (1 + 9 * torch.rand(20, 30000, generator=gen)).to(DEV)
    history, u = torch.randint(0, 30000, (20, 300), generator=gen).to(DEV), torch.rand(20, generator=gen).to(DEV)
    run = lambda: [snn.rule_times(times, history, **RULES), *snn.choose_tokens(times, u, 0.9, history, **RULES), snn.grad_norm([times])]   # noqa: E731
    ref = [v.clone() for v in run()]
    torch.cuda.synchronize()
    failures = []

    def work(turn):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for k in range(6):
                    out = run()
                    stream.synchronize()
                    bad = [i for i, (o, r) in enumerate(zip(out, ref)) if not torch.equal(o, r)]
                    if bad:
                        failures.append((turn, k, bad))
        except Exception as e:                              # noqa: BLE001 -- reported by the main thread
            failures.append((turn, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failures


def test_tangents_and_transforms_are_refused():
    import snntc_amd as snn
    import torch.autograd.forward_ad as fwad
    t = torch.rand(2, 5, device=DEV)
    h = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    with fwad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            snn.rule_times(fwad.make_dual(t, t), h, repetition=2.0)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(lambda x: snn.rule_times(x, h, repetition=2.0).sum())(t)


def test_a_sequence_that_nothing_is_allowed_for_has_no_weight():
    """A sequence that runs out of tokens neither counts nor spoils the step of the others."""
    import snntc_amd as snn
    net, prompt, uniform, mask, rules, _ = _drawn(6)
    mask[2] = False
    rules["allowed"] = snn.pack_allowed(mask)
    tokens, logp = snn.train.answer(net, prompt, uniform, **rules)
    assert bool((tokens[2] == -1).all() and logp[2].isnan().all()) and bool((tokens[[0, 1, 3, 4, 5]] >= 0).all())
    tokens[4, 5:], logp[4, 5:] = -1, float("nan")                       # (and one that ended)
    advantage = torch.randn(6, generator=torch.Generator().manual_seed(5)).to(DEV)
    batch = snn.train.answer_batch(prompt, tokens, logp, advantage, **rules)
    drawn = torch.zeros(6, 12, dtype=torch.bool, device=DEV)
    drawn[:, 3:] = tokens >= 0
    assert torch.equal(batch["weight"] > 0, drawn) and abs(float(batch["weight"].sum()) - 1) < 1e-5
    loss = snn.train.policy_step(net, torch.optim.SGD(net.parameters(), lr=0.1), **batch)
    others, rest = _net(6), [0, 1, 3, 4, 5]
    kept = dict(rules, allowed=snn.pack_allowed(mask[rest]))
    batch = snn.train.answer_batch(prompt[rest], tokens[rest].clamp(min=0), logp[rest].nan_to_num(0.0), advantage[rest], **kept)
    batch["weight"] = drawn[rest].float() / drawn.sum()
    want = snn.train.policy_step(others, torch.optim.SGD(others.parameters(), lr=0.1), **batch)
    assert bool(torch.isfinite(loss)) and torch.allclose(loss, want, rtol=1e-5, atol=1e-6)
    for a, b in zip(net.weights(), others.weights()):
        # (the sums over rows are in another order: at most 72 terms, each half a step off, of a gradient of a tenth the step's size)
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("bits", [8, 32])
def test_classifier_step_with_the_optimizer(bits):
    """The recipe's step on images, whose gradients come from its own kernels, updated by this optimizer."""
    import snntc_amd as snn
    rng = np.random.default_rng(3)
    layers = [snn.SNN_dense(12, 30, weight=(4.0 / 12 + rng.standard_normal((13, 30)) / 12 ** 0.5).astype(np.float32)),
              snn.SNN_dense(30, 7, weight=(4.0 / 30 + rng.standard_normal((31, 7)) / 30 ** 0.5).astype(np.float32))]
    net = torch.nn.Sequential(*layers).to(DEV)
    opt = snn.optim.AdamW(net.parameters(), 1e-2, state_bits=bits, weight_decay=0.1, seed=2)
    images, labels = torch.rand(64, 12, device=DEV), torch.randint(0, 7, (64,), device=DEV)
    before = [p.detach().double() for p in net.parameters()]
    loss, _ = snn.train.train_step(net, opt, images, labels, 7)
    assert bool(torch.isfinite(loss))
    for p, w in zip(net.parameters(), before):
        # the first step: m / (1 - b1) is g and v / (1 - b2) its square; the change of at most lr is off by some steps of float32
        g = p.grad.double()
        want = w * (1 - 1e-3) - 1e-2 * g / (g.abs() + 1e-8)
        assert float((p.detach().double() - want).abs().max()) <= 1e-2 * 2.0 ** -20 + 2.0 ** -23 * float(w.abs().max())
    assert float(snn.train.train_step(net, opt, images, labels, 7)[0]) != float(loss)
