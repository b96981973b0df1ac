"""LayerNorm over the last dimension of bf16 / fp16 / fp32 tensors: the norms outside the FP8 blocks (a model's last norm, norms of
q / k heads).  The FP8 LayerNorm of the blocks is ``real_quantization.fp8_layernorm_*``.  Kernels: coat_amd/csrc/layer_norm.hip;
arguments are checked and outputs allocated in coat_amd/csrc/binding.cpp."""
import torch
from torch.autograd.function import once_differentiable

from ... import _hip


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """Returns ``(y, mean, rstd)``: y of x's shape and dtype, mean and rstd fp32 of shape ``x.shape[:-1]``.  ``weight`` / ``bias``
    may have another dtype than x (fp32 parameters of a bf16 model).  Rows may be slices of a wider tensor; other strides are copied."""
    return _hip.native().layer_norm_forward(x, weight, bias, eps)


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias_grad=True, *, x_grad=True, weight_grad=True):
    """Returns ``(dx, dw, db)`` from the forward's x, mean, rstd and weight: dx in x's dtype, dw and db in the weight's; without a
    weight, or where the gradient is not asked for, None.  dw and db are summed in fp32 in a fixed order; each
    gradient has the same bits whichever others are asked for."""
    return _hip.native().layer_norm_backward(dy, x, mean, rstd, weight, x_grad, weight_grad, bias_grad)


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
    """``torch.nn.functional.layer_norm`` over the last dimension, with reverse-mode autograd, as one kernel forward and one (and the
    reduction of the parameters' gradients) backward.  Forward-mode derivatives are refused (NotImplementedError);
    ``torch.jit.trace`` records the call as one step."""
    if torch._C._get_tracing_state() or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps)[0]
