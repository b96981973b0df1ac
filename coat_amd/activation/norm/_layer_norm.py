"""LayerNorm over the last dimension of bf16 / fp16 / fp32 tensors: the norms outside the FP8 blocks (a model's last norm, norms of
q / k heads).  The FP8 LayerNorm of the blocks is ``real_quantization.fp8_layernorm_*``.  Kernels: coat_amd/csrc/layer_norm.hip."""
import torch
from torch.autograd.function import once_differentiable

from ... import _hip


def _rows(t, N):
    """(t as [M, N], row pitch in elements): a view wherever the rows lie at one distance, else a copy."""
    if N > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    if t.dim() != 2:
        try:
            t = t.view(-1, N)
        except RuntimeError:
            t = t.reshape(-1, N)
    if t.shape[0] > 1 and t.stride(0) < N:  # rows that overlap or are one row repeated
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else N


def _dense_like(t):
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _check(who, x, weight, bias):
    if not x.is_cuda:
        raise RuntimeError("coat_amd kernels need tensors on the GPU (got a %s tensor)" % x.device.type)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{who}: expected a tensor with a last dimension to normalise over, got shape {tuple(x.shape)}")
    _hip.dt(x)
    if weight is None:
        if bias is not None:
            raise ValueError(f"{who}: a bias needs a weight")
        return
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != x.shape[-1:]:
            raise ValueError(f"{who}: {name} must have shape {tuple(x.shape[-1:])}, got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{who}: {name} is on {p.device}, x on {x.device}")
        _hip.dt(p)
    if bias is not None and bias.dtype != weight.dtype:
        raise ValueError(f"{who}: bias dtype {bias.dtype} differs from weight dtype {weight.dtype}")


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """Returns ``(y, mean, rstd)``: y of x's shape and dtype, mean and rstd fp32 of shape ``x.shape[:-1]``.  ``weight`` / ``bias``
    may have another dtype than x (fp32 parameters of a bf16 model)."""
    _check("layer_norm_forward", x, weight, bias)
    if not eps >= 0.0:
        raise ValueError(f"layer_norm_forward: invalid eps {eps}")
    N = x.shape[-1]
    y = _dense_like(x)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    x, pitch = _rows(x, N)
    w = weight if weight is None else weight.contiguous()
    b = bias if bias is None else bias.contiguous()
    _hip.launch("coat_layer_norm_forward", x.get_device(), x.data_ptr(), pitch, _hip.dt(x), None if w is None else w.data_ptr(),
                None if b is None else b.data_ptr(), 0 if w is None else _hip.dt(w), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                x.shape[0], N, float(eps), what="layer_norm_forward")
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias_grad=True, *, x_grad=True, weight_grad=True):
    """Returns ``(dx, dw, db)`` from the forward's x, mean, rstd and weight: dx in x's dtype, dw and db in the weight's; without a
    weight, or where the gradient is not asked for, None.  dw and db are summed in fp32 in a fixed order."""
    _check("layer_norm_backward", x, weight, None)
    N, shape, device = x.shape[-1], x.shape, x.device
    M = x.numel() // N
    if dy.shape != shape or dy.dtype != x.dtype or dy.device != device:
        raise ValueError("layer_norm_backward: dy must have x's shape, dtype and device")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.numel() != M or t.device != device or not t.is_contiguous():
            raise ValueError(f"layer_norm_backward: {name} must be contiguous fp32 with one element a row, on x's device")
    w = weight if weight is None else weight.contiguous()
    dx = _dense_like(x) if x_grad else None
    dw = torch.empty_like(w) if w is not None and weight_grad else None
    db = torch.empty_like(w) if w is not None and bias_grad else None
    parts, partial = 0, None
    wanted = (dw is not None) + (db is not None)
    if wanted:
        parts = _hip.lib().coat_layer_norm_partials(M, N)
        if parts < 0:
            _hip.check(parts, "layer_norm_backward")
        if parts > 1 or N > 16384:  # one block writes the sums themselves
            partial = x.new_empty((wanted, parts, N), dtype=torch.float32)
    x, x_pitch = _rows(x, N)
    dy, dy_pitch = _rows(dy, N)
    _hip.launch("coat_layer_norm_backward", x.get_device(), dy.data_ptr(), dy_pitch, x.data_ptr(), x_pitch, _hip.dt(x), mean.data_ptr(),
                rstd.data_ptr(), None if w is None else w.data_ptr(), 0 if w is None else _hip.dt(w),
                *(None if t is None else t.data_ptr() for t in (dx, dw, db, partial)), parts, M, N, what="layer_norm_backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, need_b, x_grad=need_x, weight_grad=need_w)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``torch.nn.functional.layer_norm`` over the last dimension, with autograd, as one kernel forward and one (and the reduction
    of the parameters' gradients) backward."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps)[0]
