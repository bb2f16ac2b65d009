"""AdamW over all parameters in one launch, with states in 32 or in 8 bits (``hiscache_backend.adamw_step``).

It makes the steps of ``torch.optim.AdamW(params, capturable=True)``: they are counted on the device, so that a recorded iteration
(``RecordedIteration``) replays them; with ``weight_decay=0`` it is Adam.  It has arguments of its own: none of ``amsgrad``, ``maximize``,
``foreach``, ``capturable`` and ``fused``; a group's parameters lie on one device.
"""
import torch

import hiscache_backend as _be


class AdamW(torch.optim.Optimizer):
    """lr: a number or one fp32 on the parameters' device.  ``state_bits`` 8: both moments take a byte an element (parameters
    of fewer than ``min_elements`` keep 32 bits: there is little to gain), rounded at random so that they are right in the mean over
    any number of steps and at any betas: over the elements the root of the second moment is within 1 % of that in 32 bits, for one element
    within 10 % (one standard deviation; up to 35 % while it falls to a hundredth), the first moment within 10 %.
    ``master``: parameters in half precision have a copy in fp32 that takes the steps; one that something else has changed since the
    last step (weights that were loaded, say) is taken as it is, an element that its copy still rounds to keeps the copy.  (A
    change through ``.data`` is not noticed, nor one between replays of a recorded step.)

    Parameters must be contiguous and on a GPU.  States are made by a parameter's first step, which cannot be recorded."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master=True,
                 min_elements=4096):
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not all(0 <= b < 1 for b in betas) or not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"betas must lie in [0, 1), eps and weight_decay must not be negative: got {betas}, {eps}, {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master=master, min_elements=min_elements))
        self._handles, self._versions = {}, {}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._handles, self._versions = {}, {}

    _PARTS = ("exp_avg", "exp_avg_sq", "step", "scale", "master")

    def _handle(self, p, group):
        """p's state as ``adamw_step`` takes it, made where there is none."""
        state, handle = self.state[p], self._handles.get(p)
        if not state:
            if not p.is_cuda:
                raise RuntimeError(f"parameters must live on the GPU (got {p.device})")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a parameter's first step makes its state and cannot be recorded: run one step before")
            made = _be.adamw_state(p, group["state_bits"] if p.numel() >= group["min_elements"] else 32,
                                   bool(group["master"]) and p.dtype is not torch.float32)
            state.update({k: getattr(made, k) for k in self._PARTS if getattr(made, k) is not None})
        if handle is None or any(getattr(handle, k) is not state.get(k) for k in self._PARTS):
            handle = self._handles[p] = _be.AdamWState(*(state.get(k) for k in self._PARTS))
        if handle.master is not None and not p.is_inference():
            # (of a parameter that this object has not stepped yet, one of a copied optimizer, say, nothing is known: it is looked at)
            if self._versions.get(p) != p._version:
                same = handle.master.to(p.dtype) == p
                handle.master.copy_(torch.where(same, handle.master, p.float()))
        return handle

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            states = [self._handle(p, group) for p in params]
            how = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                       rounding="random")
            with torch.cuda.device(params[0].device):
                _be.adamw_step(params, [p.grad for p in params], states, **how)
            for p, s in zip(params, states):
                if s.master is not None and not p.is_inference():
                    self._versions[p] = p._version
        return loss

    @torch.no_grad()
    def moments(self, p):
        """(first, second moment) of a parameter that has made a step, in fp32."""
        state = self.state[p]
        if "scale" not in state:
            return state["exp_avg"], state["exp_avg_sq"]
        with torch.cuda.device(p.device):
            (m, root), = _be.adamw_moments([_be.AdamWState(*(state.get(k) for k in self._PARTS))])
        return m, root * root

    def load_state_dict(self, state_dict):
        """What ``state_dict`` returned, in its own types (``Optimizer.load_state_dict`` would cast it to the parameters')."""
        super().load_state_dict(state_dict)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, i in zip(group["params"], saved["params"]):
                if i in state_dict["state"]:
                    self.state[p] = {k: v.to(device=p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                     for k, v in state_dict["state"][i].items()}
                    # (a copy that the loaded parameter does not round from gives way at the next step)
                    self._versions[p] = -1
        self._handles.clear()
