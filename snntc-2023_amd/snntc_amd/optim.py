"""AdamW as a ``torch.optim.Optimizer`` over the update kernel, for the steps in train.py and any other loop (the reference takes its
framework's Adam, snntc-mnist.py:70)."""
import torch

from .ops import adamw_update, grad_norm

_BLOCK = 256                                             # elements of a state that share a scale


class AdamW(torch.optim.Optimizer):
    """AdamW over all tensors of a group in one launch (see ops.adamw_update for the formula).

      state_bits  32, or 8: codes with a scale for every 256 elements, a quarter of the memory.  An element whose second moment is too
                  small for its block (2^-34 of the largest) has no first moment either, so that steps stay those of 32 bits in size
      max_norm    None, or what the norm over all gradients of a step is scaled down to; a step whose norm is no finite number then
                  changes nothing but its number.  `norm` is the last step's, on the device
      seed        of the random bits by which codes and 16-bit weights are rounded, from [0, 2^32)
      capturable  the steps are counted on the device, so that a captured step counts by itself when it is replayed; learning
                  rate and the other numbers stay what they were when it was captured.  The step before has to have had the same
                  tensors' gradients, or there is no state yet that a replay could go on from

    Weights: contiguous float32, bfloat16 or float16 tensors on one ROCm device, with gradients of their types."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, max_norm=None, seed=0,
                 capturable=False):
        if state_bits not in (8, 32):
            raise ValueError(f"states are held in 8 or 32 bits, not in {state_bits}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive, or None: {max_norm}")
        if not 0 <= int(seed) < 1 << 32:
            raise ValueError(f"a seed is a number of 32 bits, not {seed}")
        self.state_bits, self.max_norm, self.seed, self.capturable = state_bits, max_norm, int(seed), bool(capturable)
        self.norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        """The base class carries weights, states and groups into a copy; what this class adds goes with them, but not the last norm."""
        own = {k: getattr(self, k) for k in ("state_bits", "max_norm", "seed", "capturable")}
        return {**super().__getstate__(), **own, "norm": None}

    def _begin(self, p, steps):
        """The state of a tensor that has its first gradient."""
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=p.device)                   # noqa: E731
        if self.state_bits == 8:
            blocks = -(-p.numel() // _BLOCK)
            state = {"first": zeros(p.shape, torch.uint8), "second": zeros(p.shape, torch.uint8),
                     "first_scale": zeros(blocks, torch.float32), "second_scale": zeros(blocks, torch.float32)}
        else:
            state = {"first": zeros(p.shape, torch.float32), "second": zeros(p.shape, torch.float32)}
        if self.capturable:
            if p.device not in steps:                    # one counter for all that begin in the same step
                steps[p.device] = zeros((), torch.int64)
            state["step"] = steps[p.device]
        else:
            state["step"] = 0
        self.state[p] = state

    def _parting(self, group, params):
        """Tensors with a gradient that share their counter with one that has none in this step: lists of them, by counter."""
        stepping, waiting = {}, set()
        with_gradient = {id(p) for p in params}
        for p in group["params"]:
            state = self.state.get(p)
            if state and id(p) in with_gradient:
                stepping.setdefault(id(state["step"]), []).append(p)
            elif state:
                waiting.add(id(state["step"]))
        return [tensors for counter, tensors in stepping.items() if counter in waiting]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        captured = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if captured and not self.capturable:
            raise RuntimeError("AdamW: a step that is captured into a graph needs capturable=True")
        groups = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if any(p.grad.is_sparse for p in params):
                raise RuntimeError("AdamW: sparse gradients are not supported")
            groups.append(params)
        grads = [p.grad for params in groups for p in params]
        if not grads:
            return loss
        parting = [self._parting(group, params) if self.capturable else [] for group, params in zip(self.param_groups, groups)]
        if captured and (any(parting) or any(not self.state.get(p) for params in groups for p in params)):
            raise RuntimeError("AdamW: before a step is captured, take one with gradients for the same tensors")
        self.norm = None if self.max_norm is None else grad_norm(grads)
        call = 0
        for group, params, apart in zip(self.param_groups, groups, parting):
            for tensors in apart:
                counter = self.state[tensors[0]]["step"].clone()
                for p in tensors:
                    self.state[p]["step"] = counter
            steps = {}
            for p in params:
                if not self.state[p]:
                    self._begin(p, steps)
            together = {}                                # tensors with the same number of steps behind them
            for p in params:
                n = self.state[p]["step"]
                together.setdefault(id(n) if self.capturable else n, []).append(p)
            for tensors in together.values():
                states = [self.state[p] for p in tensors]
                number = states[0]["step"] if self.capturable else states[0]["step"] + 1
                scales = ([s["first_scale"] for s in states], [s["second_scale"] for s in states]) if self.state_bits == 8 else (None, None)
                adamw_update([p.detach() for p in tensors], [p.grad for p in tensors], [s["first"] for s in states],
                             [s["second"] for s in states], number, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                             weight_decay=group["weight_decay"], norm=self.norm, max_norm=1.0 if self.max_norm is None else self.max_norm,
                             first_scale=scales[0], second_scale=scales[1], seed=self.seed + (call << 32), paired=self.state_bits == 8)
                if not self.capturable:
                    for s in states:
                        s["step"] = number
                call += 1
        return loss

    def load_state_dict(self, state_dict):
        """As the base class, but a state keeps the type it was saved with (the base class makes it the weights')."""
        super().load_state_dict(state_dict)
        params = [(g, p) for g, group in enumerate(self.param_groups) for p in group["params"]]
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        counters = {}                                    # of a group: every group is a call of its own
        for i, (g, p) in zip(saved, params):
            if i not in state_dict["state"]:
                continue
            old = state_dict["state"][i]
            if ("first_scale" in old) != (self.state_bits == 8):
                raise ValueError(f"AdamW: the saved states are not of {self.state_bits} bits")
            state = {k: v.detach().to(p.device, copy=True) for k, v in old.items() if k != "step"}
            if self.state_bits == 8:
                state["first"].mul_(state["second"] != 0)           # (as the update leaves them; codes from elsewhere need not be so)
            step = int(old["step"])
            if self.capturable:
                if (g, p.device, step) not in counters:
                    counters[g, p.device, step] = torch.tensor(step, dtype=torch.int64, device=p.device)
                step = counters[g, p.device, step]
            state["step"] = step
            self.state[p] = state
