"""AdamW over all tensors of a network at once, moments in 32 or in 8 bits.

``HipAdamW`` is a ``torch.optim.Optimizer``: parameter groups, schedulers,
``zero_grad``, ``state_dict`` and ``load_state_dict`` work as they do there
(a 32 bit one loads the state of ``torch.optim.AdamW``).  With ``state_bits=8``
the two moments take 2.03 bytes an element instead of 8: codes in blocks of
256 elements, each block with a float32 scale per moment; see
:meth:`HipAdamW.moments` for their values.  No counterpart in the reference.
"""

import math

import torch

from .. import _lib

__all__ = ["HipAdamW"]

_NAMES = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
_OPTIONS = ("lr", "betas", "eps", "weight_decay", "state_bits")


def _check_options(group):
    if group["state_bits"] not in _NAMES:
        raise ValueError(f"`state_bits` has to be 32 or 8, got {group['state_bits']}.")
    lr, (beta1, beta2) = float(group["lr"]), group["betas"]
    if not (lr >= 0.0 and math.isfinite(lr)):
        raise ValueError(f"Invalid learning rate: {lr}")
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"Invalid betas, expected values in [0, 1): {group['betas']}")
    if not (group["eps"] >= 0.0 and group["weight_decay"] >= 0.0):
        raise ValueError(f"Invalid eps or weight decay: {group['eps']}, {group['weight_decay']}")


class _Loaded:
    """The state of one parameter on its way through torch's loading, which would
    convert its tensors to the parameter's type."""

    def __init__(self, held):
        self.held = held


class HipAdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay.

    Parameters are contiguous float32, bfloat16 or float16 tensors on one GPU,
    with dense gradients of their type; the step is computed in float32 and each
    parameter rounded once.  Parameters without a gradient are left as they are,
    and their count of steps with them.

    A step that is not the first (``moments()`` prepares that) can be captured in a
    HIP graph: each replay is a step of its own, with the options of the capture.
    The GPU counts steps from then on; counts in the state are those of the work that
    has been waited for, and ``state_dict()`` waits.  A load then changes the moments
    that the graph works on, and so does an edit of the state, from the next
    ``moments()`` or eager step on; the groups have to stay as they are.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32):
        if state_bits not in _NAMES:
            raise ValueError(f"`state_bits` has to be 32 or 8, got {state_bits}.")
        self._plan = None
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay,
                                  "state_bits": int(state_bits)})

    def add_param_group(self, param_group):
        options = {**self.defaults, **param_group}
        _check_options(options)
        if self.param_groups and options["state_bits"] != self.state_bits:
            raise ValueError("All parameter groups need the same `state_bits`.")
        super().add_param_group(param_group)

    def __getstate__(self):
        self._settle()
        return super().__getstate__()

    def __setstate__(self, state):
        plan = self.__dict__.get("_plan")  # (none in a copy)
        super().__setstate__(state)
        self._plan = plan if plan is not None and plan.captured() else None
        loaded = [key for key, held in self.state.items() if isinstance(held, _Loaded)]
        for key in loaded:
            self.state[key] = self.state[key].held
        if loaded or self._plan is not None:
            self._build()

    def _settle(self):
        """Wait for the counts that the GPU keeps."""

        if self._plan is not None and self._plan.captured():
            torch.cuda.synchronize(next(p.device for group in self.param_groups for p in group["params"]))

    def state_dict(self):
        self._settle()
        return super().state_dict()

    @property
    def state_bits(self):
        return self.param_groups[0]["state_bits"]

    @torch.no_grad()
    def _build(self):
        """Lay the moments of all parameters out, taking over what the state holds.
        A state that does not fit raises, and stays as it is."""

        bits, plan = self.state_bits, self._plan
        in_place = plan is not None and plan.captured()
        if in_place:
            # a graph works on the plan's memory
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("The state of a HipAdamW cannot be replaced while a graph is captured.")
            if not plan.same_groups(self.param_groups):
                raise RuntimeError("The groups of a HipAdamW have to stay as they are once a step was captured.")
            self._settle()
        else:
            plan = _lib.torch_ext().AdamWPlan([list(group["params"]) for group in self.param_groups], bits)
        steps, index = plan.steps(), 0
        laid_out, copies = [], {}
        for g, group in enumerate(self.param_groups):
            for k, p in enumerate(group["params"]):
                views = dict(zip(_NAMES[bits], plan.views(g, k)), step=steps[index])
                index += 1
                state = self.state.get(p, {})
                if in_place:
                    # (what is not there starts again; what is may be a view of what is written)
                    state = {name: torch.as_tensor(t).clone() for name, t in state.items()}
                    state = {**{name: torch.zeros_like(t) for name, t in views.items()}, **state}
                for name, held in state.items():
                    if name not in views:
                        raise ValueError(f"A state of {bits} bits has no `{name}`.")
                    held = torch.as_tensor(held)
                    to = views[name]
                    if name != "step" and (held.shape != to.shape or held.dtype != to.dtype):
                        raise ValueError(
                            f"`{name}` of a state of {bits} bits has to be {to.dtype} {tuple(to.shape)}, "
                            f"got {held.dtype} {tuple(held.shape)}."
                        )
                    to_all, held_all = copies.setdefault(to.dtype, ([], []))
                    to_all.append(to)
                    held_all.append(held)
                laid_out.append((p, views))
        for to_all, held_all in copies.values():
            torch._foreach_copy_(to_all, held_all)
        self.state.update(laid_out)
        plan.watch(self.state, self.param_groups)
        self._plan = plan

    def _current_plan(self):
        """The plan, made again where groups or state were replaced, cleared or added to."""

        if self._plan is None or not self._plan.current(self.state, self.param_groups):
            self._build()
        return self._plan

    def step(self, closure=None):
        """One step of all parameters that have a gradient, on the current stream."""

        # (nothing here is recorded for autograd, so no guard against it is entered)

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        plan = self._current_plan()
        for g, group in enumerate(self.param_groups):
            beta1, beta2 = group["betas"]
            plan.step(g, float(group["lr"]), beta1, beta2, group["eps"], group["weight_decay"])
        return loss

    def moments(self, param=None):
        """The moments ``(m, v)`` as float32 values: of one parameter, in its shape, or
        of all as two flat tensors in the order of the groups, each parameter from
        the next multiple of 256 elements (zeros between).  With 32 bits these are
        the state itself, with 8 bits what its codes stand for."""

        plan = self._current_plan()
        m, v = plan.moments() or (torch.zeros(0), torch.zeros(0))
        if param is None:
            return m, v
        for g, group in enumerate(self.param_groups):
            for k, p in enumerate(group["params"]):
                if p is param:
                    at = plan.first(g, k)
                    return tuple(t[at : at + p.numel()].view(p.shape) for t in (m, v))
        raise ValueError("The tensor is not one of the optimizer's parameters.")

    def load_state_dict(self, state_dict):
        """Take over options and moments as ``torch.optim.Optimizer`` does, hooks and
        all; the moments keep their types.  States of optimizers that step otherwise
        (``maximize``, ``amsgrad``, weight decay through the gradients) are refused.
        A load that fails changes nothing."""

        before = self.state, self.param_groups, self._plan
        # (the last hook: it sees what the user's have made of the state)
        handle = self.register_load_state_dict_pre_hook(HipAdamW._loadable)
        try:
            super().load_state_dict(state_dict)
        except BaseException:
            self.state, self.param_groups, self._plan = before
            raise
        finally:
            handle.remove()

    def _loadable(self, state_dict):
        """The state as torch's loading takes it, after checks."""

        groups, bits = [], self.state_bits
        if [len(g["params"]) for g in self.param_groups] != [len(g["params"]) for g in state_dict["param_groups"]]:
            raise ValueError("The loaded state has other parameter groups.")
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            if saved.get("state_bits", 32) != bits:
                raise ValueError(f"The loaded state has {saved.get('state_bits', 32)} bits, expected {bits}.")
            for name in ("maximize", "amsgrad"):
                if saved.get(name):
                    raise ValueError(f"The loaded state is of an optimizer with `{name}`, which HipAdamW has not.")
            if saved.get("decoupled_weight_decay") is False and saved.get("weight_decay"):
                raise ValueError("The loaded state's weight decay is part of its gradients; HipAdamW's is not.")
            groups.append({**{name: group[name] for name in _OPTIONS}, **saved})
            _check_options(groups[-1])
        state = {key: _Loaded(dict(held)) for key, held in state_dict["state"].items()}
        return {**state_dict, "state": state, "param_groups": groups}
