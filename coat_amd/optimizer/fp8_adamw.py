"""CoatAdamW: AdamW whose first and second moments live in FP8 e4m3 with one scale per 128 elements and,
by default, Dynamic Range Expansion (per-group exponent k and centre c).

Drop-in for coat/optimizer/fp8_adamw.py:36-342 of the reference: same constructor, same ``state`` keys
(``step, exp_avg, scale_exp_avg, expand_exp_avg, sqrt_minmax_exp_avg, exp_avg_sq, scale_exp_avg_sq,
expand_exp_avg_sq, sqrt_minmax_exp_avg_sq``; reference :119-137), same state-dict dtype policy
(:231-262).  One fused HIP kernel per parameter tensor does the whole step (``qoptim_cuda`` shim).

Differences, all deliberate:
  * the per-group vectors are always fp32 (the reference allocates them in the parameter dtype, which
    only works for fp32 parameters because its kernel takes ``float*``, :124-137);
  * the kernels run on torch's current stream;
  * ``amsgrad=True`` raises (the reference's branch calls ``torch.zeros(p, ...)`` and cannot run, :133-135).
"""
from collections import defaultdict
from copy import deepcopy
from itertools import chain
from typing import Optional, Tuple

import torch
from torch.optim.optimizer import Optimizer

from ..utils._fp8_quantization_config import QuantizationConfig
from . import qoptim_cuda

convert_str_to_fp8 = {"E4M3": torch.float8_e4m3fn, "E5M2": torch.float8_e5m2}

_EXPAND_KEYS = ("expand_exp_avg", "sqrt_minmax_exp_avg", "expand_exp_avg_sq", "sqrt_minmax_exp_avg_sq")
_STATE_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2, torch.float32)


class CoatAdamW(Optimizer):
    def __init__(
        self,
        params,
        lr: float = 1e-3,
        betas: Tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        amsgrad: bool = False,
        qargs: QuantizationConfig = None,
        *,
        fused: Optional[bool] = None,
        multi_tensor: bool = True,
        state_bits: int = 8,
        master_weights: bool = False,
        max_grad_norm: Optional[float] = None,
    ):
        """``state_bits=32`` keeps both moments in fp32 (norm weights, embeddings); ``master_weights`` then also an fp32 copy of
        16-bit parameters (state key ``master``), made at the first step: what is written into the parameters from outside after
        that is lost at the next one.  Both may be given per parameter group.  ``max_grad_norm``: the gradients of all groups, on
        one device, are clipped to that global 2-norm of this process's gradients inside the step (``grad_norm`` then holds the
        norm of the last step, on the device, or None after a step without clipping or without gradients; the gradients themselves
        stay as they are).  It is kept in the parameter groups,
        where it may be changed between steps and where ``load_state_dict`` restores it, and is the same in all of them: ``step``
        raises otherwise.  None of the three is in the reference."""
        # multi_tensor (not in the reference): parameters of one dtype, device and step count share kernel launches
        self.multi_tensor = multi_tensor
        self.qargs = QuantizationConfig() if qargs is None else qargs
        assert self.qargs.first_order_expansion == self.qargs.second_order_expansion, (
            "We expect the first order and second order momentum to use dynamic range expansion at the same time.")
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if amsgrad:
            raise ValueError("CoatAdamW does not support amsgrad")
        for name in ("first_order_bit", "second_order_bit"):
            if getattr(self.qargs, name) != "E4M3":
                raise ValueError(f"{name} must be E4M3: the optimizer kernels store both moments in e4m3")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad, fused=fused)
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        # only what differs from the reference's optimizer shows in the parameter groups
        extra = dict(state_bits=(state_bits, 8), master_weights=(master_weights, False), max_grad_norm=(max_grad_norm, None))
        defaults.update({k: v for k, (v, plain) in extra.items() if v != plain})
        self.grad_norm = None
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        bits = param_group.get("state_bits", self.defaults.get("state_bits", 8))
        if bits not in (8, 32):
            raise ValueError(f"Invalid state_bits: {bits} (8 or 32)")
        if param_group.get("master_weights", self.defaults.get("master_weights", False)) and bits != 32:
            raise ValueError("master_weights needs state_bits=32")
        clip = (self.param_groups[0] if self.param_groups else self.defaults).get("max_grad_norm")
        if param_group.get("max_grad_norm", clip) != clip:
            raise ValueError("max_grad_norm is one for all parameter groups")
        if clip is not None or "max_grad_norm" in self.defaults:
            param_group["max_grad_norm"] = clip  # that of the groups there, which may have changed since construction
        super().add_param_group(param_group)

    # ------------------------------------------------------------------ state
    @property
    def use_expansion(self) -> bool:
        """Only "expansion" and "true" switch Dynamic Range Expansion on (reference :293)."""
        return self.qargs.first_order_expansion.lower() in ("expansion", "true")

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("amsgrad", False)
            group.setdefault("fused", None)
            for p in group["params"]:
                p_state = self.state.get(p, {})
                if len(p_state) != 0 and not torch.is_tensor(p_state["step"]):
                    p_state["step"] = torch.tensor(float(p_state["step"]), dtype=torch.float32)

    def _init_state(self, p, expand):
        """Fresh state: codes 0, scales 0, k = 1, c = 1 (reference :117-137)."""
        state = self.state[p]
        ngroups = (p.numel() + self.qargs.qgroup_size - 1) // self.qargs.qgroup_size
        state["step"] = torch.tensor(0.0)  # host tensor: reading it never syncs the device
        for name, bit in (("exp_avg", self.qargs.first_order_bit), ("exp_avg_sq", self.qargs.second_order_bit)):
            state[name] = torch.zeros_like(p, dtype=convert_str_to_fp8[bit], memory_format=torch.contiguous_format)
            state["scale_" + name] = torch.zeros(ngroups, device=p.device, dtype=torch.float32)
            if expand:
                state["expand_" + name] = torch.ones(ngroups, device=p.device, dtype=torch.float32)
                state["sqrt_minmax_" + name] = torch.ones(ngroups, device=p.device, dtype=torch.float32)
        return state

    def _init_state32(self, p):
        state = self.state[p]
        state["step"] = torch.tensor(0.0)
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
        return state

    @torch._disable_dynamo
    def load_state_dict(self, state_dict) -> None:
        """torch's Optimizer.load_state_dict casts every floating-point state tensor to the parameter dtype;
        FP8 codes and fp32 group vectors must keep theirs, so the mapping is redone here with that policy
        (reference :158-262): ``step`` is left alone, every other tensor must be e4m3 / e5m2 / fp32 and is
        only moved to the parameter's device.  Groups that say nothing of ``state_bits``, ``master_weights`` or ``max_grad_norm``
        (plain 8-bit ones, those of another optimizer) keep this optimizer's; moments that do not fit ``state_bits=32`` are refused."""
        state_dict = state_dict.copy()
        for pre_hook in self._optimizer_load_state_dict_pre_hooks.values():
            replaced = pre_hook(self, state_dict)
            if replaced is not None:
                state_dict = replaced

        groups, saved_groups = self.param_groups, deepcopy(state_dict["param_groups"])
        if len(groups) != len(saved_groups):
            raise ValueError("loaded state dict has a different number of parameter groups")
        if any(len(g["params"]) != len(s["params"]) for g, s in zip(groups, saved_groups)):
            raise ValueError("loaded state dict contains a parameter group that doesn't match the size of optimizer's group")
        for g, s in zip(groups, saved_groups):
            s.update({k: g[k] for k in ("state_bits", "master_weights", "max_grad_norm") if k in g and k not in s})
            bits = s.get("state_bits", 8)
            if s.get("master_weights", False) and bits != 32:
                raise ValueError("master_weights needs state_bits=32")
            for key in s["params"] if bits == 32 else ():
                held = [t.dtype for name, t in state_dict["state"].get(key, {}).items() if name in ("exp_avg", "exp_avg_sq")]
                if any(dtype != torch.float32 for dtype in held):
                    raise ValueError(f"loaded moments are {held[0]}, but the parameter group has state_bits=32")
        id_map = dict(zip(chain.from_iterable(s["params"] for s in saved_groups),
                          chain.from_iterable(g["params"] for g in groups)))

        def place(param, value, key=None):
            if isinstance(value, torch.Tensor):
                if key == "step":
                    return value
                assert value.dtype in _STATE_DTYPES, f"unexpected optimizer state dtype {value.dtype} for {key}"
                return value.to(device=param.device)
            if isinstance(value, dict):
                return {k: place(param, v, k) for k, v in value.items()}
            return value

        state = defaultdict(dict)
        for k, v in state_dict["state"].items():
            if k in id_map:
                state[id_map[k]] = place(id_map[k], v)
            else:  # a key outside the parameter mapping is kept as it is (torch.optim.Optimizer.load_state_dict does the same)
                state[k] = v
        for g, s in zip(groups, saved_groups):
            s["params"] = g["params"]
        self.__setstate__({"state": state, "param_groups": saved_groups})
        for post_hook in self._optimizer_load_state_dict_post_hooks.values():
            post_hook(self)

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        """Perform a single optimization step."""
        self._cuda_graph_capture_health_check()
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        max_grad_norm, scale = (self.param_groups[0].get("max_grad_norm") if self.param_groups else None), None
        if any(group.get("max_grad_norm") != max_grad_norm for group in self.param_groups):
            raise ValueError("max_grad_norm is one for all parameter groups")
        self.grad_norm = None
        if max_grad_norm is not None:
            grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
            if any(g.is_sparse for g in grads):
                raise RuntimeError("AdamW does not support sparse gradients")
            if grads:
                self.grad_norm, scale = qoptim_cuda.grad_norm_multi(grads, max_grad_norm)
        expand = self.use_expansion
        qgroup_size, expand_min = self.qargs.qgroup_size, self.qargs.expand_min
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            lr, wd, eps = group["lr"], group["weight_decay"], group["eps"]
            if isinstance(lr, torch.Tensor):
                lr = lr.item()
            # parameters of one dtype, device and step count are stepped together, 32 to a launch (the reference launches
            # once per parameter, :419-515); a parameter alone in its bucket takes the single-tensor entry point
            buckets = {}
            bits, masters = group.get("state_bits", 8), group.get("master_weights", False)
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                state = self.state[p]
                if len(state) == 0:
                    state = self._init_state(p, expand) if bits == 8 else self._init_state32(p)
                state["step"] += 1
                step = int(state["step"].item())
                grad = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                if not p.is_contiguous():
                    raise RuntimeError("CoatAdamW needs contiguous parameters (the state is laid out flat)")
                if masters and p.dtype != torch.float32 and "master" not in state:
                    state["master"] = p.detach().float()
                buckets.setdefault((p.dtype, p.device, step), []).append((p, grad, state))
            for (dtype, _, step), items in buckets.items():
                if bits == 32:
                    ps, gs, sts = map(list, zip(*items))
                    copies = [st["master"] for st in sts] if masters and dtype != torch.float32 else None
                    qoptim_cuda.adamw_step_multi(ps, gs, [st["exp_avg"] for st in sts], [st["exp_avg_sq"] for st in sts], beta1, beta2, lr,
                                                 wd, eps, step, masters=copies, grad_scale=scale)
                    continue
                if scale is None and (len(items) == 1 or not getattr(self, "multi_tensor", True)):
                    for p, grad, state in items:
                        if expand:
                            qoptim_cuda.fp8_adamw_expand_step(
                                p, grad, state["exp_avg"], state["scale_exp_avg"], state["expand_exp_avg"],
                                state["sqrt_minmax_exp_avg"], state["exp_avg_sq"], state["scale_exp_avg_sq"],
                                state["expand_exp_avg_sq"], state["sqrt_minmax_exp_avg_sq"],
                                beta1, beta2, lr, wd, eps, step, qgroup_size, expand_min)
                        else:
                            qoptim_cuda.fp8_adamw_step(
                                p, grad, state["exp_avg"], state["scale_exp_avg"], state["exp_avg_sq"],
                                state["scale_exp_avg_sq"], beta1, beta2, lr, wd, eps, step, qgroup_size)
                    continue
                ps, gs, sts = [i[0] for i in items], [i[1] for i in items], [i[2] for i in items]
                col = lambda key: [st[key] for st in sts]  # noqa: E731
                if expand:
                    qoptim_cuda.fp8_adamw_expand_step_multi(
                        ps, gs, col("exp_avg"), col("scale_exp_avg"), col("expand_exp_avg"), col("sqrt_minmax_exp_avg"),
                        col("exp_avg_sq"), col("scale_exp_avg_sq"), col("expand_exp_avg_sq"), col("sqrt_minmax_exp_avg_sq"),
                        beta1, beta2, lr, wd, eps, step, qgroup_size, expand_min, grad_scale=scale)
                else:
                    qoptim_cuda.fp8_adamw_step_multi(
                        ps, gs, col("exp_avg"), col("scale_exp_avg"), col("exp_avg_sq"), col("scale_exp_avg_sq"),
                        beta1, beta2, lr, wd, eps, step, qgroup_size, grad_scale=scale)
        return loss
