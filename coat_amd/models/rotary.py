"""Rotary positions with several axes (time, height, width of video, image and text tokens) on q and k together, beside the one-axis
rotary of the decoder layers (``coat_llama.fused_rotary``).  Kernel: coat_amd/csrc/rope_axes.hip; arguments are checked and outputs
allocated in coat_amd/csrc/binding.cpp."""
import math

import torch
from torch.autograd.function import once_differentiable

from .. import _hip


class RotaryAxes:
    """Which pair of a head turns with which axis, and how fast.

    ``sections``: pairs of each axis in turn; their sum P is the number of turning pairs, 2 P <= ``head_dim`` (the elements behind
    are passed through).  Pair j turns by ``position * theta ** -(j / P)``; with ``restart`` every section counts its own pairs,
    ``theta ** -(i / n)`` for pair i of a section of n.  Pair j is elements ``(j, j + P)`` of the head, the layout of the decoder
    layers; with ``pairs`` neighbours ``(2 j, 2 j + 1)``.  If CUDA is initialised, the tables are made on the device that is current
    at construction; another device gets its own at the first use there (which must not be inside a graph capture).  A copy, or a
    plan that was saved and loaded, makes its own tables in the same way.  A plan may be dropped while work that uses it is still
    queued, on any stream; a captured graph reads its tables at every replay and needs the plan alive."""

    def __init__(self, head_dim, sections, theta=10000.0, restart=False, pairs=False):
        self.head_dim, self.sections, self.theta = int(head_dim), tuple(int(n) for n in sections), float(theta)
        self.restart, self.pairs = bool(restart), bool(pairs)
        if not self.sections or min(self.sections) < 0 or sum(self.sections) < 1:
            raise ValueError(f"RotaryAxes: invalid sections {tuple(sections)}")
        if 2 * sum(self.sections) > self.head_dim:
            raise ValueError(f"RotaryAxes: sections {self.sections} hold more pairs than a head of {self.head_dim}")
        if not (self.theta > 0.0 and math.isfinite(self.theta)):
            raise ValueError(f"RotaryAxes: invalid theta {theta}")
        total = self.turning = sum(self.sections)  # P
        self._axis = [a for a, n in enumerate(self.sections) for _ in range(n)]
        exponent = [i / n for n in self.sections for i in range(n)] if self.restart else [j / total for j in range(total)]
        self._freq = [self.theta ** -e for e in exponent]  # radians a position, in 64 bits
        self._start_tables()

    def _start_tables(self):
        self._tables, self._home = {}, {}  # by device: the tables, and the handle of the stream whose order their memory follows
        if torch.cuda.is_initialized():
            self.tables(torch.device("cuda", torch.cuda.current_device()))

    def __getstate__(self):
        """Without the tables: loading moves tensors between devices, but not the keys that say where they are."""
        return {k: v for k, v in self.__dict__.items() if k not in ("_tables", "_home")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._start_tables()

    def tables(self, device):
        """(turns a position fp64 [P], axis int32 [P]) on ``device``."""
        if device not in self._tables:
            turns = torch.tensor([f / (2.0 * math.pi) for f in self._freq], dtype=torch.float64, device=device)
            axis = torch.tensor(self._axis, dtype=torch.int32, device=device)
            if type(turns) is not torch.Tensor:  # of a mode that computes without memory: not for later calls
                return turns, axis
            self._home[device] = _hip.raw_stream(device.index) if device.type == "cuda" else 0
            self._tables[device] = turns, axis  # last: another thread that finds the tables finds their stream
        return self._tables[device]

    def cos_sin(self, position_ids, dtype):
        """cos / sin [B, S, 2 P] of the first 2 P elements of a head from torch operations on any device, in the (j, j + P) layout;
        position_ids [axes, B, S]."""
        if self.pairs:
            raise ValueError("RotaryAxes.cos_sin: only for the (j, j + P) layout")
        if position_ids.dim() != 3 or position_ids.shape[0] != len(self.sections):
            raise ValueError(f"RotaryAxes: expected position_ids of shape [{len(self.sections)}, batch, seq], got {list(position_ids.shape)}")
        freq = torch.tensor(self._freq, dtype=torch.float64, device=position_ids.device)
        angle = position_ids[torch.tensor(self._axis, device=position_ids.device)].permute(1, 2, 0).double() * freq
        angle = torch.cat((angle, angle), -1)
        return angle.cos().to(dtype), angle.sin().to(dtype)


def _rotate(q, k, position_ids, plan, inverse):
    first = k if q is None else q
    if first is None:
        raise ValueError("rotary_axes: neither q nor k given")
    device = first.device
    turns, axis = plan.tables(device)
    return _hip.native().rotary_axes(q, k, position_ids, turns, axis, plan.head_dim, len(plan.sections), plan.turning, plan.pairs, inverse,
                                     plan._home.get(device, 0))


def rotary_axes_forward(q, k, position_ids, plan):
    """Rotates q [B, S, heads, head_dim] and k [B, S, kv_heads, head_dim] (either may be None; bf16, fp16 or fp32; any strides, such
    as slices of a fused projection) by position_ids [axes, B, S] (whole numbers, broadcast over B and S).  Returns new dense
    tensors of the same shapes.  Angles are taken in 64 bits, the rotation in fp32, rounded once."""
    return _rotate(q, k, position_ids, plan, False)


def rotary_axes_backward(dq, dk, position_ids, plan):
    """The gradients of ``rotary_axes_forward``'s q and k: the rotation by the negated angles."""
    return _rotate(dq, dk, position_ids, plan, True)


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, position_ids, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(position_ids)
        ctx.plan = plan
        return _rotate(q, k, position_ids, plan, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        dq, dk = (g if needed else None for g, needed in zip((dq, dk), ctx.needs_input_grad))
        if dq is None and dk is None:
            return None, None, None, None
        (position_ids,) = ctx.saved_tensors
        return (*_rotate(dq, dk, position_ids, ctx.plan, True), None, None)


def rotary_axes(q, k, position_ids, plan):
    """``rotary_axes_forward`` with reverse-mode autograd.  Forward-mode derivatives are refused (NotImplementedError);
    ``torch.jit.trace`` records the call as one step."""
    if torch._C._get_tracing_state() or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k)):
        return _RotaryAxes.apply(q, k, position_ids, plan)
    return rotary_axes_forward(q, k, position_ids, plan)
