"""Optimizer of a training step on the CUDA backend.

``AdamW`` updates every weight of a model in one kernel launch (one more when gradients
are clipped or non-finite steps skipped), with moments in 32 or in 8 bits, and can keep
an exponential average of the weights in the same pass (the reference trainer's AdamW
and EMA, ``mace_ictc/training/train_loop.py``).
"""
from __future__ import annotations

import math
import operator
from array import array

import torch

from ictc_o3.backends.cuda.runtime import require_cuda_fp32

__all__ = ["AdamW"]


def _number(value, name, low, high=math.inf, open_low=False):
    if isinstance(value, bool) or not isinstance(value, (int, float)):
        raise TypeError(f"{name} must be a number")
    value = float(value)
    if not (low < value if open_low else low <= value) or not value < high:
        raise ValueError(f"{name} is outside its range")
    return value


def _check_seed(seed):
    if not isinstance(seed, int) or isinstance(seed, bool) or not 0 <= seed < 1 << 64:
        raise ValueError("seed must be an integer in [0, 2^64)")


def _hyperparameters(group):
    betas = group["betas"]
    if not isinstance(betas, (tuple, list)) or len(betas) != 2:
        raise ValueError("betas must be two numbers")
    eps = _number(group["eps"], "eps", 0.0, open_low=True)
    if eps < 1.2e-38:
        raise ValueError("eps must be a normal FP32 number")
    return {"lr": _number(group["lr"], "lr", 0.0),
            "betas": (_number(betas[0], "beta1", 0.0, 1.0), _number(betas[1], "beta2", 0.0, 1.0)),
            "eps": eps, "weight_decay": _number(group["weight_decay"], "weight_decay", 0.0)}


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over CUDA FP32 tensors on one device.

    Arithmetic and hyperparameters are those of ``torch.optim.AdamW``; each tensor
    counts its own steps, and one without a gradient is left as it is.

    ``state_bits``: 32 keeps both moments in FP32.  8 keeps one byte per value and moment and a
    power-of-two scale per 256 values (the last block of a tensor may be shorter), rounded
    stochastically from ``seed``, the tensor's step and the value's place, so that
    equal inputs give equal results.  A block whose new moments are not finite is left as it was.
    ``max_norm``: gradients are scaled by min(1, max_norm / (|g| + 1e-6)), |g| over all of them; a NaN among
    them makes that factor NaN (moments in 8 bits, and their weights, then stay as they were).
    ``skip_nonfinite``: a step with an infinite or NaN gradient changes nothing and is not counted.
    ``ema_decay``: keeps average = d average + (1 - d) weight in ``state[p]["ema"]``.
    ``state[p]`` holds views of the buffers that the kernels use: values may be written into them, not put
    in their place.

    ``step`` never waits for the device, allocates nothing for contiguous gradients and may be
    captured into a CUDA graph; addresses and hyperparameters are then those of the
    capture, and ``mark_updated()`` after a replay tells modules that keep state derived
    from the weights.  One step of an optimizer at a time: its workspace is shared.
    Weights, gradients and the current stream must be ordered by the caller, as for any operator.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 max_norm=None, skip_nonfinite=False, ema_decay=None, seed=0):
        if state_bits not in (8, 32) or isinstance(state_bits, bool):
            raise ValueError("state_bits must be 8 or 32")
        if not isinstance(skip_nonfinite, bool):
            raise TypeError("skip_nonfinite must be a boolean")
        _check_seed(seed)
        self.state_bits = state_bits
        self.skip_nonfinite = skip_nonfinite
        self.seed = seed
        self.max_norm = None if max_norm is None else _number(max_norm, "max_norm", 0.0, open_low=True)
        self.ema_decay = None if ema_decay is None else _number(ema_decay, "ema_decay", 0.0, 1.0)
        self._table = None
        super().__init__(params, {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay})
        self._build()

    # -- construction -------------------------------------------------------

    def add_param_group(self, param_group):
        if getattr(self, "_table", None) is not None:
            raise ValueError("parameter groups are fixed when the optimizer is built")
        super().add_param_group(param_group)

    def _build(self):
        from ictc_o3.backends.cuda import _native
        from ictc_o3.backends.cuda.adamw import BLOCK, TensorTable, blocks_of
        for group in self.param_groups:
            _hyperparameters(group)
        params = [p for group in self.param_groups for p in group["params"]]
        require_cuda_fp32(*params)
        if any(not p.is_contiguous() or p.is_neg() for p in params):
            raise ValueError("the optimizer requires contiguous parameters that are no lazily negated views")
        spans = sorted((p.data_ptr(), 4 * p.numel()) for p in params if p.numel())
        if len({id(p) for p in params}) != len(params) or any(a + n > b for (a, n), (b, _) in zip(spans, spans[1:])):
            raise ValueError("parameters must not repeat or share memory")
        device = params[0].device
        with torch.cuda.device(device):
            table = TensorTable([p.numel() for p in params], device)
            kind = torch.float32 if self.state_bits == 32 else torch.uint8
            flat = {"m": torch.zeros(table.values, dtype=kind, device=device),
                    "v": torch.zeros(table.values, dtype=kind, device=device), "m_scale": None, "v_scale": None,
                    "average": None, "steps": torch.zeros(len(params), dtype=torch.int64, device=device),
                    "rates": torch.zeros(len(params), 4, dtype=torch.int64, device=device)}
            if self.state_bits == 8:
                flat["m_scale"] = torch.ones(table.blocks, dtype=torch.uint8, device=device)
                flat["v_scale"] = torch.ones(table.blocks, dtype=torch.uint8, device=device)
            if self.ema_decay is not None:
                flat["average"] = torch.zeros(table.values, dtype=torch.float32, device=device)
            for i, (p, start) in enumerate(zip(params, table.starts)):
                place, first = slice(start, start + p.numel()), start // BLOCK
                entry = {"step": flat["steps"][i], "exp_avg": flat["m"][place].view(p.shape),
                         "exp_avg_sq": flat["v"][place].view(p.shape)}
                if self.state_bits == 8:
                    scales = slice(first, first + blocks_of(p.numel()))
                    entry["exp_avg_exponent"] = flat["m_scale"][scales]
                    entry["exp_avg_sq_exponent"] = flat["v_scale"][scales]
                if self.ema_decay is not None:
                    entry["ema"] = flat["average"][place].view(p.shape)
                    entry["ema"].copy_(p.detach())
                self.state[p] = entry
        self._params, self._flat, self._device = params, flat, device
        self._places = [None if flat[k] is None else flat[k].data_ptr()
                        for k in ("m", "v", "m_scale", "v_scale", "average", "steps", "rates")]
        self._sizes = array("q", [p.numel() for p in params])
        self._weights, self._grads = array("Q", [0] * len(params)), array("Q", [0] * len(params))
        try:
            self._host = _native.host_tensors()
        except _native.NativeError:      # not built here: the same in Python, 0.55 us instead of 0.03 per tensor
            self._host = None
        self._table = table
        self._empty = table.workspace.data_ptr()      # stands for the gradient of a tensor without values

    def __getstate__(self):
        raise TypeError("an optimizer of the CUDA backend is not copied or pickled; use state_dict()")

    # -- one step -----------------------------------------------------------

    def _check_groups(self):
        """The tables and host arrays are those of the parameters at construction."""
        first = 0
        for group in self.param_groups:
            part = group["params"]
            same = (self._host.holds(self._params, first, part) if self._host is not None and type(part) is list else
                    len(part) <= len(self._params) - first and all(map(operator.is_, self._params[first:], part)))
            if not same:
                break
            first += len(part)
        if first != len(self._params) or not same:
            raise ValueError("the parameters of the groups are fixed when the optimizer is built")

    def _gather(self):
        """Fill the arrays of addresses (0: no gradient); returns how many have a gradient, and
        temporaries that must outlive the launch."""
        weights, grads = self._weights, self._grads
        if self._host is not None:
            live = self._host.gather(self._params, self._sizes.buffer_info()[0], self._device.index,
                                     weights.buffer_info()[0], grads.buffer_info()[0], self._empty)
            if live >= 0:
                return live, None
        # some tensor is not what it was, or a gradient is not contiguous
        kept = [None if p.grad is None else p.grad.detach() for p in self._params]
        for i, (p, g, size) in enumerate(zip(self._params, kept, self._sizes)):
            if g is None:
                continue
            if (p.dtype is not torch.float32 or p.device != self._device or p.numel() != size or not p.is_contiguous()
                    or p.is_neg()):
                raise ValueError("a parameter has changed its type, device, size or layout since the optimizer was built")
            if (g.layout is not torch.strided or g.dtype is not torch.float32 or g.device != self._device
                    or g.numel() != size):
                raise ValueError("gradients must be dense CUDA FP32 tensors of their parameter's size")
            kept[i] = g.contiguous().resolve_neg()
        for i, (p, g) in enumerate(zip(self._params, kept)):
            weights[i] = 0 if g is None else p.data_ptr()
            grads[i] = 0 if g is None else g.data_ptr() if g.numel() else self._empty
        return sum(g is not None for g in kept), kept

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_groups()
        groups = [_hyperparameters(group) for group in self.param_groups]
        live, kept = self._gather()
        if not live:
            return loss
        w, g = self._weights.buffer_info()[0], self._grads.buffer_info()[0]
        use_norm = self.max_norm is not None or self.skip_nonfinite
        if use_norm:
            self._table.grad_norm(g, self.max_norm, self.skip_nonfinite)
        first = 0
        for group, values in zip(self.param_groups, groups):
            count = len(group["params"])
            self._table.step(w, g, first, count, self.state_bits, self._places, **values,
                             ema_decay=0.0 if self.ema_decay is None else self.ema_decay, seed=self.seed,
                             use_norm=use_norm)
            first += count
        del kept                     # copies of gradients: their memory is reused on this stream only
        if self._host is not None:
            self._host.changed(self._params, g)
        else:
            torch.autograd.graph.increment_version([p for p, at in zip(self._params, self._grads) if at])
        return loss

    def mark_updated(self):
        """Tell modules that keep state derived from the weights that these have changed (after
        replaying a captured step; ``step`` does it by itself)."""
        torch.autograd.graph.increment_version([p for p in self._params if p.grad is not None])

    # -- results ------------------------------------------------------------

    @property
    def grad_norm(self):
        """Norm of all gradients before clipping at the last step (a device scalar that the next
        step overwrites), with ``max_norm`` or ``skip_nonfinite``; else None."""
        return self._table.norm if self.max_norm is not None or self.skip_nonfinite else None

    def moments(self):
        """(exp_avg, exp_avg_sq) of all parameters one after another, each from a multiple of 256
        values on with zeros between: the state's own FP32 buffers, or the values that 8-bit states
        stand for (BF16; exact where a block's scale is at least 2^-99: below, its least codes leave
        BF16's range)."""
        if self.state_bits == 32:
            return self._flat["m"], self._flat["v"]
        return self._table.decode(self._flat)

    def averages(self):
        """The averaged weights in the same arrangement (the state's own buffer), or None."""
        return self._flat["average"]

    # -- checkpoints --------------------------------------------------------

    def state_dict(self):
        """The base class's, and with 8-bit states the ``seed`` of their rounding; ``max_norm``,
        ``skip_nonfinite`` and ``ema_decay`` belong to the constructor."""
        state_dict = super().state_dict()
        # dicts of their own: a value replaced in the optimizer's would part it from the buffers that the kernels use
        state_dict["state"] = {k: dict(v) if isinstance(v, dict) else v for k, v in state_dict["state"].items()}
        if self.state_bits == 8:
            state_dict["seed"] = self.seed
        return state_dict

    def load_state_dict(self, state_dict):
        """Copy a state dict of this class (same ``state_bits`` and, if it keeps one, an average), or
        one of ``torch.optim.AdamW`` for ``state_bits`` 32.  Parameters without an entry start anew.
        A ``seed`` among the entries becomes this optimizer's, so that 8-bit states go on as they would have.
        Hooks registered for loading run before (they may give another dict) and after it."""
        state_dict = dict(state_dict)      # hooks may change its entries
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        self._load(state_dict)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)

    @torch.no_grad()
    def _load(self, state_dict):
        groups, saved = state_dict["param_groups"], state_dict["state"]
        if len(groups) != len(self.param_groups) or any(len(a["params"]) != len(b["params"])
                                                        for a, b in zip(groups, self.param_groups)):
            raise ValueError("the state dict has other parameter groups")
        loaded = []
        for group in groups:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("amsgrad and maximize are not supported")
            values = {k: group[k] for k in ("lr", "betas", "eps", "weight_decay")}
            values["lr"] = float(values["lr"])
            _hyperparameters(values)
            loaded.append(values)
        seed = state_dict.get("seed", self.seed)
        _check_seed(seed)
        names, exponents = [name for group in groups for name in group["params"]], []
        for name, p in zip(names, self._params):
            entry, mine = saved.get(name), self.state[p]
            if entry is None:
                continue
            for key, value in mine.items():
                if key == "ema" and key not in entry:
                    continue
                if key not in entry:
                    raise ValueError(f"the state dict has no {key}; was it saved with other state_bits?")
                theirs = entry[key]
                if key == "step":
                    if int(theirs) < 0:
                        raise ValueError("a step count is negative")
                elif not isinstance(theirs, torch.Tensor) or theirs.dtype != value.dtype or theirs.shape != value.shape:
                    raise ValueError(f"{key} has another type or shape; was it saved with other state_bits?")
                elif key.endswith("exponent") and theirs.numel():
                    exponents.append(theirs.to(self._device))
        if exponents and not 1 <= int((all_of := torch.cat(exponents)).min()) <= int(all_of.max()) <= 253:
            raise ValueError("a scale exponent is outside 1..253")
        for group, theirs, values in zip(self.param_groups, groups, loaded):
            # other entries (a scheduler's initial_lr) come along
            group.update({k: v for k, v in theirs.items() if k != "params"}, **values)
            group["betas"] = tuple(values["betas"])
        self.seed = seed
        steps, to, values = [], [], []
        for name, p in zip(names, self._params):
            entry, mine = saved.get(name), self.state[p]
            steps.append(0 if entry is None else int(entry["step"]))
            for key, value in mine.items():
                if key == "step":
                    continue
                if entry is not None and key in entry:
                    to.append(value)
                    values.append(entry[key])
                elif key == "ema":
                    value.copy_(p)
                else:
                    value.fill_(1 if key.endswith("exponent") else 0)
        self._flat["steps"].copy_(torch.tensor(steps, dtype=torch.int64))
        if values and all(v.device == self._device for v in values):
            torch._foreach_copy_(to, values)
        else:
            for mine, value in zip(to, values):
                mine.copy_(value)
