"""The operators for sequences of tokens and for choices, as cases that can be timed one by one.

Four kinds, each through the package's public entry points where `own` is true, in elementary torch operations otherwise:

  embed       tokens to spike times (embed_tokens), and the table's gradient (embed_tokens_grad)
  gated       a gated running mean of spike times along a sequence (gated_scan, gated_scan_grad), and one step of it
              for rows that are served token by token (gated_step)
  policy      the clipped policy loss with a KL term over softmax(-times), with its gradient (policy_time_loss)
  preference  the loss of preferred against rejected sequences, with its gradient (preference_time_loss)

A case's sizes are plain numbers; `prepare` makes its inputs from a seed, `run` is one pass, `exact` the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CLIP = (0.2, 0.28)
KL = 0.05
BETA, SMOOTHING = 0.1, 0.05


def listed():
    return [
        # The next token of eight served sequences: launches and host work are all there is.
        _embed("embed_decode_n8", 8, 1000, 512, "f32", 64, True, "forward"),
        # A training batch of 128 sequences of 64 tokens in front of layers of 800 inputs.
        _embed("embed_train_n8192", 8192, 8192, 800, "f32", 64, True, "train"),
        # Odd sizes, a 16-bit table most of whose rows do not occur, plain scaling.
        _embed("embed_train_ragged", 5003, 50021, 777, "bf16", 32, False, "train"),
        # A large batch: most tokens occur again and again, the commonest thousands of times.
        _embed("embed_train_n131072", 131072, 32768, 1024, "bf16", 64, True, "train"),
        # One step of 64 served sequences.
        _gated("gated_step_b64", 64, 1, 800, "f32", False, "step"),
        # An ordinary training batch.
        _gated("gated_train_b32", 32, 256, 800, "f32", False, "train"),
        # Odd sizes, sequences of different lengths in a padded batch, gates from a 16-bit product.
        _gated("gated_train_ragged", 24, 333, 777, "bf16", True, "train"),
        # One long sequence: the only parallel work is along it.
        _gated("gated_train_t32768", 1, 32768, 1024, "f16", False, "train"),
        # Actions of a small classifier used as a policy, one batch.
        _policy("policy_b256", 256, 10, "f32", False),
        # Sampled tokens of a large vocabulary, a share of the rows masked.
        _policy("policy_n4096", 4096, 32000, "bf16", True),
        # Pairs of short sequences of different lengths over 1000 classes.
        _preference("preference_ragged", 12, 97, 1000, "f32", True),
        # Pairs of whole answers over a large vocabulary.
        _preference("preference_p8", 8, 512, 32768, "bf16", True),
    ]


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    while True:
        kind = rng.choice(["embed", "gated", "policy", "preference"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        if kind == "embed":
            c = _embed(None, _log(rng, 1, 131072), _log(rng, 50, 131072), _log(rng, 16, 2048), dtype, rng.choice([32, 64]),
                       rng.random() < 0.5, rng.choice(["forward", "train", "train"]))
            fits = c["tokens"] * c["dim"] <= 1 << 27 and c["rows"] * c["dim"] <= 1 << 26
        elif kind == "gated":
            if rng.random() < 0.25:
                c = _gated(None, _log(rng, 1, 512), 1, _log(rng, 16, 4096), dtype, False, "step")
            else:
                c = _gated(None, _log(rng, 1, 64), _log(rng, 2, 32768), _log(rng, 16, 2048), dtype, rng.random() < 0.5, "train")
            fits = c["batch"] * c["steps"] * c["dim"] <= 1 << 25
        elif kind == "policy":
            c = _policy(None, _log(rng, 1, 16384), _log(rng, 2, 131072), dtype, rng.random() < 0.5)
            fits = c["rows"] * c["classes"] <= 1 << 27
        else:
            c = _preference(None, _log(rng, 1, 32), _log(rng, 1, 1024), _log(rng, 2, 131072), dtype, rng.random() < 0.7)
            fits = 2 * c["pairs"] * c["steps"] * c["classes"] <= 1 << 27
        if fits:
            return c


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    s = {"case": case}
    kind = case["kind"]
    if kind == "embed":
        N, V, D = case["tokens"], case["rows"], case["dim"]
        # word frequencies: rank r with a share of about 1 / r, the ranks scattered over the table
        u = torch.rand(N, generator=gen, device=DEVICE, dtype=torch.float64)
        rank = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        s["tokens"] = torch.randperm(V, generator=gen, device=DEVICE)[rank].to(torch.int32 if case["token_bits"] == 32 else torch.int64)
        s["table"] = torch.rand(V, D, generator=gen, device=DEVICE).to(TYPES[case["dtype"]])
        s["scale"] = 1.0 if case["encode"] else 0.5
        if case["mode"] == "train":
            s["grad"] = torch.randn(N, D, generator=gen, device=DEVICE) / N
    elif kind == "gated":
        B, T, D = case["batch"], case["steps"], case["dim"]
        shape = (B, D) if case["mode"] == "step" else (B, T, D)
        s["x"] = torch.exp(torch.rand(shape, generator=gen, device=DEVICE))
        s["gate"] = (2.0 + 1.5 * torch.randn(shape, generator=gen, device=DEVICE)).to(TYPES[case["dtype"]])
        s["state"] = torch.exp(torch.rand(B, D, generator=gen, device=DEVICE))
        if case["mode"] == "train":
            s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device=DEVICE) if case["ragged"] else None
            s["grad_y"] = torch.randn(shape, generator=gen, device=DEVICE)
            s["grad_final"] = torch.randn(B, D, generator=gen, device=DEVICE)
    elif kind == "policy":
        N, J = case["rows"], case["classes"]
        s["times"], s["actions"], logp = _rows(gen, N, J, case["dtype"])
        # a few updates after the actions were drawn: ratios around one, some of them beyond the clip's ends (none on them)
        step = 0.2 * torch.randn(N, generator=gen, device=DEVICE, dtype=torch.float64)
        for end in (1.0 - CLIP[0], 1.0 + CLIP[1]):
            step = torch.where((torch.exp(step) - end).abs() < 1e-3, torch.zeros_like(step), step)
        s["old_logp"] = (logp - step).float()
        s["ref_logp"] = (logp + 0.3 * torch.randn(N, generator=gen, device=DEVICE, dtype=torch.float64)).float()
        s["advantage"] = torch.randn(N, generator=gen, device=DEVICE)
        s["weight"] = None
        if case["masked"]:
            keep = (torch.rand(N, generator=gen, device=DEVICE) < 0.8).float()
            s["weight"] = keep / keep.sum().clamp(min=1.0)
    else:
        P, T, J = case["pairs"], case["steps"], case["classes"]
        times, tokens, logp = _rows(gen, 2 * P * T, J, case["dtype"])
        s["times"], s["tokens"] = times.view(2 * P, T, J), tokens.view(2 * P, T)
        s["weight"] = None
        weight = torch.ones(2 * P, T, device=DEVICE)
        if case["ragged"]:
            lengths = torch.randint(0 if P > 4 else 1, T + 1, (2 * P,), generator=gen, device=DEVICE)
            weight = (torch.arange(T, device=DEVICE)[None, :] < lengths[:, None]).float()
            s["weight"] = weight
        s["ref_logp"] = ((logp.view(2 * P, T) * weight).sum(1)
                         + 5.0 * torch.randn(2 * P, generator=gen, device=DEVICE, dtype=torch.float64)).float()
    return s


def run(s):
    return (_run_own if own else _run_plain)[s["case"]["kind"]](s)


def work(case):
    kind = case["kind"]
    size = BYTES[case["dtype"]]
    if kind == "embed":
        N, V, D = case["tokens"], case["rows"], case["dim"]
        used = _expected_distinct(N, V)
        ids = N * case["token_bits"] // 8
        out = {"bytes": ids + used * D * size + N * D * 4, "flops": 2.0 * N * D}
        if case["mode"] == "train":
            out["bytes"] += N * D * 4 + V * D * size
            out["flops"] += 1.0 * N * D + 2.0 * used * D
        return out
    if kind == "gated":
        n, state = case["batch"] * case["steps"] * case["dim"], case["batch"] * case["dim"]
        if case["mode"] == "step":
            return {"bytes": n * (4 + size) + 2 * state * 4, "flops": 8.0 * n}
        part = 0.5 if case["ragged"] else 1.0                       # what lies behind a length is not read
        reads, writes = (4 + size + 4) * n * part + 2 * state * 4, (4 + 4 + size) * n + 2 * state * 4
        return {"bytes": reads + writes, "flops": 20.0 * n * part}
    rows = case["rows"] if kind == "policy" else 2 * case["pairs"] * case["steps"]
    part = 1.0
    if kind == "policy" and case["masked"]:
        part = 0.8
    if kind == "preference" and case["ragged"]:
        part = 0.5
    n = rows * case["classes"]
    return {"bytes": (1.0 + part) * n * size + 32.0 * rows, "flops": 8.0 * n * part}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed":
        tok, table, scale = s["tokens"].long(), s["table"].double(), s["scale"]
        z = torch.exp(1.0 - scale * table) if case["encode"] else scale * table
        outputs = [z.index_select(0, tok)]
        if case["mode"] == "train":
            # every token's rows stand together once sorted: their sum is a difference of running sums
            order = torch.argsort(tok, stable=True)
            run_sum = torch.cumsum(s["grad"].double().index_select(0, order), 0)
            ids = tok.index_select(0, order)
            last = torch.cat([ids[1:] != ids[:-1], torch.ones(1, dtype=torch.bool, device=DEVICE)])
            upto = run_sum[last]
            sums = torch.cat([upto[:1], upto[1:] - upto[:-1]])
            d = torch.zeros(table.shape, dtype=torch.float64, device=DEVICE)
            d[ids[last]] = sums
            outputs.append(-scale * z * d if case["encode"] else scale * d)
        return tuple(outputs)
    if kind == "gated":
        x, a, h = s["x"].double(), torch.sigmoid(s["gate"].double()), s["state"].double()
        if case["mode"] == "step":
            return h * a + x * (1.0 - a)
        T, lengths = case["steps"], s["lengths"]
        on = None if lengths is None else (torch.arange(T, device=DEVICE)[:, None, None] < lengths[None, :, None]).double()
        hs = []
        for t in range(T):
            new = torch.lerp(x[:, t], h, a[:, t])
            h = new if on is None else torch.lerp(h, new, on[t].expand_as(h))
            hs.append(h)
        u = s["grad_final"].double()
        us = [None] * T
        gy = s["grad_y"].double()
        for t in range(T - 1, -1, -1):
            us[t] = u + gy[:, t] if on is None else u + gy[:, t] * on[t]
            u = us[t] * a[:, t] if on is None else us[t] * torch.lerp(torch.ones_like(u), a[:, t], on[t].expand_as(u))
        hs, us = torch.stack(hs, 1), torch.stack(us, 1)
        before = torch.cat([s["state"].double()[:, None], hs[:, :-1]], 1)
        dx, dg = us * (1.0 - a), us * (before - x) * a * (1.0 - a)
        if on is not None:
            m = on.transpose(0, 1)
            final = hs[:, -1]
            return hs * m, final, dx * m, dg * m, u
        return hs, hs[:, -1], dx, dg, u
    times = s["times"].double().requires_grad_(True)
    tokens = s["actions"] if kind == "policy" else s["tokens"]
    logp = torch.log_softmax(-times, -1).gather(-1, tokens[..., None])[..., 0]
    if kind == "policy":
        ratio, away = torch.exp(logp - s["old_logp"].double()), s["ref_logp"].double() - logp
        adv = s["advantage"].double()
        gain = torch.minimum(ratio * adv, torch.clamp(ratio, 1.0 - CLIP[0], 1.0 + CLIP[1]) * adv)
        loss = KL * (torch.expm1(away) - away) - gain
        weight = torch.full_like(loss, 1.0 / loss.numel()) if s["weight"] is None else s["weight"].double()
        (grad,) = torch.autograd.grad((loss * weight).sum(), times)
        there = (weight != 0).double()
        return (loss * there).detach(), (logp * there).detach(), grad
    weight = torch.ones_like(logp) if s["weight"] is None else s["weight"].double()
    seq = (logp * weight).sum(1)
    gain = seq - s["ref_logp"].double()
    P = case["pairs"]
    m = BETA * (gain[:P] - gain[P:])
    loss = (1.0 - SMOOTHING) * torch.nn.functional.softplus(-m) + SMOOTHING * torch.nn.functional.softplus(m)
    (grad,) = torch.autograd.grad(loss.mean(), times)
    return loss.detach(), seq.detach(), grad


# ---- the framework's own operators -----------------------------------------------------------------------------------------------


def _snn():
    path = os.path.join(os.getcwd(), "snntc-2023_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import snntc_amd
    return snntc_amd


def _embed_own(s):
    snn, c = _snn(), s["case"]
    z = snn.embed_tokens(s["tokens"], s["table"], s["scale"], c["encode"])
    if c["mode"] == "forward":
        return (z,)
    return z, snn.embed_tokens_grad(s["grad"], s["tokens"], s["table"], s["scale"], c["encode"])


def _gated_own(s):
    snn = _snn()
    if s["case"]["mode"] == "step":
        return snn.gated_step(s["x"], s["gate"], s["state"])
    y, final = snn.gated_scan(s["x"], s["gate"], s["state"], s["lengths"])
    dx, dgate, dstate = snn.gated_scan_grad(s["grad_y"], s["grad_final"], s["x"], s["gate"], y, s["state"], s["lengths"])
    return y, final, dx, dgate, dstate


def _policy_own(s):
    return _snn().policy_time_loss(s["times"], s["actions"], s["old_logp"], s["advantage"], ref_logp=s["ref_logp"],
                                   weight=s["weight"], clip=CLIP, kl_coef=KL)


def _preference_own(s):
    return _snn().preference_time_loss(s["times"], s["tokens"], s["ref_logp"], weight=s["weight"], beta=BETA, smoothing=SMOOTHING)


# ---- the plain forms -------------------------------------------------------------------------------------------------------------


def _embed_plain(s):
    c, table, scale = s["case"], s["table"], s["scale"]
    tok = s["tokens"].long()
    z = table[tok].float() * scale
    if c["encode"]:
        z = torch.exp(1.0 - z)
    if c["mode"] == "forward":
        return (z,)
    d = torch.zeros(table.shape, dtype=torch.float32, device=table.device).index_add_(0, tok, s["grad"])
    if c["encode"]:
        d = d * (-scale * torch.exp(1.0 - scale * table.float()))
    else:
        d = d * scale
    return z, d.to(table.dtype)


def _running(a, b):
    """h[:, t] = a[:, t] * h[:, t - 1] + b[:, t] along dimension 1, h before the first being zero: distances double."""
    T, d = a.shape[1], 1
    while d < T:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _gated_plain(s):
    x, a, state = s["x"], 1.0 / (1.0 + torch.exp(-s["gate"].float())), s["state"]
    if s["case"]["mode"] == "step":
        return a * state + (1.0 - a) * x
    b = (1.0 - a) * x
    gy, lengths = s["grad_y"], s["lengths"]
    if lengths is not None:                                        # steps behind a length hold the state
        on = torch.arange(x.shape[1], device=x.device)[None, :, None] < lengths[:, None, None]
        a, b, gy = torch.where(on, a, 1.0), torch.where(on, b, 0.0), torch.where(on, gy, 0.0)
    b = torch.cat([b[:, :1] + a[:, :1] * state[:, None], b[:, 1:]], 1)
    h = _running(a, b)
    gy = torch.cat([gy[:, :-1], gy[:, -1:] + s["grad_final"][:, None]], 1)
    ahead = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    u = _running(ahead.flip(1), gy.flip(1)).flip(1)
    before = torch.cat([state[:, None], h[:, :-1]], 1)
    dx, dgate, dstate = (1.0 - a) * u, u * (before - x) * a * (1.0 - a), a[:, 0] * u[:, 0]
    y = h
    if lengths is not None:
        y, dx, dgate = torch.where(on, h, 0.0), torch.where(on, dx, 0.0), torch.where(on, dgate, 0.0)
    return y, h[:, -1].clone(), dx, dgate.to(s["gate"].dtype), dstate


def _logp_plain(times, tokens):
    """log softmax(-times) of each row's token, and the softmax."""
    v = -times.float()
    top = v.amax(-1, keepdim=True)
    e = torch.exp(v - top)
    total = e.sum(-1, keepdim=True)
    logp = (v.gather(-1, tokens[..., None]) - top - torch.log(total))[..., 0]
    return logp, e / total


def _logp_grad_plain(times, tokens, p, coef):
    g = p * coef[..., None]
    g.scatter_add_(-1, tokens[..., None], -coef[..., None])
    return g.to(times.dtype)


def _policy_plain(s):
    logp, p = _logp_plain(s["times"], s["actions"])
    weight = torch.full_like(logp, 1.0 / logp.numel()) if s["weight"] is None else s["weight"]
    lp, adv = logp.double(), s["advantage"].double()               # next to the clip's ends; differences of like numbers
    ratio, away = torch.exp(lp - s["old_logp"].double()), s["ref_logp"].double() - lp
    plain, clipped = ratio * adv, torch.clamp(ratio, 1.0 - CLIP[0], 1.0 + CLIP[1]) * adv
    loss = KL * (torch.exp(away) - away - 1.0) - torch.minimum(plain, clipped)
    slope = KL * (1.0 - torch.exp(away)) - torch.where(plain <= clipped, plain, torch.zeros_like(plain))
    there = weight != 0
    grad = _logp_grad_plain(s["times"], s["actions"], p, (slope * weight).float())
    return torch.where(there, loss.float(), 0.0), torch.where(there, logp, 0.0), grad


def _preference_plain(s):
    logp, p = _logp_plain(s["times"], s["tokens"])
    weight = torch.ones_like(logp) if s["weight"] is None else s["weight"]
    seq = (logp.double() * weight).sum(1)
    gain = seq - s["ref_logp"].double()
    P = gain.shape[0] // 2
    m = BETA * (gain[:P] - gain[P:])
    sig = 1.0 / (1.0 + torch.exp(-m))
    loss = (1.0 - SMOOTHING) * torch.log1p(torch.exp(-m)) + SMOOTHING * torch.log1p(torch.exp(m))
    slope = (BETA / P) * (SMOOTHING * sig - (1.0 - SMOOTHING) * (1.0 - sig))
    coef = torch.cat([slope, -slope])[:, None] * weight
    return loss.float(), seq.float(), _logp_grad_plain(s["times"], s["tokens"], p, coef.float())


_run_own = {"embed": _embed_own, "gated": _gated_own, "policy": _policy_own, "preference": _preference_own}
_run_plain = {"embed": _embed_plain, "gated": _gated_plain, "policy": _policy_plain, "preference": _preference_plain}


# ---- cases and inputs ------------------------------------------------------------------------------------------------------------


def _rows(gen, N, J, dtype):
    """Spike times of N rows of J outputs, one token per row drawn from softmax(-times), and its log-probability in 64 bits."""
    times = torch.rand(N, J, generator=gen, device=DEVICE).mul_(12.0).add_(1.0).to(TYPES[dtype])
    tokens = torch.empty(N, dtype=torch.int64, device=DEVICE)
    logp = torch.empty(N, dtype=torch.float64, device=DEVICE)
    step = max(1, (1 << 26) // J)                                  # rows at a time
    for r in range(0, N, step):
        v = -times[r:r + step].float()
        noise = torch.rand(v.shape, generator=gen, device=DEVICE).clamp_(min=1e-30)
        tokens[r:r + step] = torch.argmax(v - torch.log(-torch.log(noise).clamp_(min=1e-30)), 1)
        logp[r:r + step] = v.gather(1, tokens[r:r + step, None])[:, 0].double() - torch.logsumexp(v.double(), 1)
    return times, tokens, logp


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def _expected_distinct(N, V):
    """Distinct tokens among N of the law above, in expectation."""
    total = math.log(V + 1.0)
    out, r = 0.0, 0
    while r < V:
        span = max(1, r // 64)
        top = min(V, r + span)
        share = math.log((top + 1.0) / (r + 1.0)) / total / (top - r)
        out += (top - r) * -math.expm1(N * math.log1p(-min(share, 1.0 - 1e-12)))
        r = top
    return out


def _embed(name, tokens, rows, dim, dtype, token_bits, encode, mode):
    return _named(name, {"kind": "embed", "tokens": tokens, "rows": rows, "dim": dim, "dtype": dtype, "token_bits": token_bits,
                         "encode": encode, "mode": mode})


def _gated(name, batch, steps, dim, dtype, ragged, mode):
    return _named(name, {"kind": "gated", "batch": batch, "steps": steps, "dim": dim, "dtype": dtype, "ragged": ragged, "mode": mode})


def _policy(name, rows, classes, dtype, masked):
    return _named(name, {"kind": "policy", "rows": rows, "classes": classes, "dtype": dtype, "masked": masked})


def _preference(name, pairs, steps, classes, dtype, ragged):
    return _named(name, {"kind": "preference", "pairs": pairs, "steps": steps, "classes": classes, "dtype": dtype, "ragged": ragged})


def _named(name, case):
    return case if name is None else {"name": name, **case}
