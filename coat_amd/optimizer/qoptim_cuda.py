"""Drop-in for the reference's pybind module ``qoptim_cuda`` (coat/optimizer/kernels/bindings.cpp:5-8).

``fp8_adamw_expand_step_multi`` / ``fp8_adamw_step_multi`` (no counterpart in the reference) take lists of the same tensors
and step them in one launch per 32 tensors, each tensor bit-identical to its own call.

Same two functions, same positional arguments (include/fp8_adamw.h:6-13, include/fp8_adamw_expand.h:6-17),
torch tensors in, everything updated in place; the work is done by libcoat_hip.so on the tensor's current
stream (the reference launches on the legacy default stream).  Errors the reference raises through
AT_ASSERTM surface as RuntimeError with the same message."""
import ctypes

import torch

from .. import _hip


def _common_checks(params, grads, exp_avg, exp_avg_sq, scales, qgroup_size):
    if qgroup_size != 128:
        raise RuntimeError("Only Support 128 per-group quantization currently")
    if not params.is_cuda:
        raise RuntimeError("qoptim_cuda: params must be on the GPU")
    if grads.dtype != params.dtype:
        raise RuntimeError(f"qoptim_cuda: grads dtype {grads.dtype} differs from params dtype {params.dtype}")
    for name, t in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)):
        if t.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"expected scalar type Float8_e4m3fn but found {t.dtype} ({name})")
    for t in scales:
        if t.dtype != torch.float32:
            raise RuntimeError(f"expected scalar type Float but found {t.dtype}")
    ngroups = (params.numel() + qgroup_size - 1) // qgroup_size
    if scales[0].numel() != ngroups:
        raise RuntimeError("grid_dim == scale_exp_avg.numel()")
    for t in (params, grads, exp_avg, exp_avg_sq, *scales):
        if not t.is_contiguous():
            raise RuntimeError("qoptim_cuda: tensors must be contiguous")
    return ngroups


def fp8_adamw_expand_step(params, grads, exp_avg, scale_exp_avg, expand_exp_avg, sqrtminmax_exp_avg, exp_avg_sq,
                          scale_exp_avg_sq, expand_exp_avg_sq, sqrtminmax_exp_avg_sq, beta1, beta2, lr, wd, eps, step,
                          qgroup_size, expand_min):
    """Update the quantized optimizer states, use polynomial expander (bindings.cpp:7)."""
    scales = (scale_exp_avg, expand_exp_avg, sqrtminmax_exp_avg, scale_exp_avg_sq, expand_exp_avg_sq,
              sqrtminmax_exp_avg_sq)
    ngroups = _common_checks(params, grads, exp_avg, exp_avg_sq, scales, qgroup_size)
    if scale_exp_avg_sq.numel() != ngroups:
        raise RuntimeError("grid_dim == scale_exp_avg_sq.numel()")
    p = _hip.ptr
    _hip.check(_hip.lib().coat_fp8_adamw_expand_step(
        p(params), p(grads), _hip.dt(params), p(exp_avg), p(scale_exp_avg), p(expand_exp_avg), p(sqrtminmax_exp_avg),
        p(exp_avg_sq), p(scale_exp_avg_sq), p(expand_exp_avg_sq), p(sqrtminmax_exp_avg_sq),
        beta1, beta2, lr, wd, eps, int(step), int(qgroup_size), int(expand_min), params.numel(), ngroups,
        _hip.stream(params.device)), "fp8_adamw_expand_step")


def fp8_adamw_step(params, grads, exp_avg, scale_exp_avg, exp_avg_sq, scale_exp_avg_sq, beta1, beta2, lr, wd, eps,
                   step, qgroup_size):
    """Update the quantized optimizer states (bindings.cpp:6)."""
    ngroups = _common_checks(params, grads, exp_avg, exp_avg_sq, (scale_exp_avg, scale_exp_avg_sq), qgroup_size)
    if scale_exp_avg_sq.numel() != ngroups:
        raise RuntimeError("grid_dim == scale_exp_avg_sq.numel()")
    p = _hip.ptr
    _hip.check(_hip.lib().coat_fp8_adamw_step(
        p(params), p(grads), _hip.dt(params), p(exp_avg), p(scale_exp_avg), p(exp_avg_sq), p(scale_exp_avg_sq),
        beta1, beta2, lr, wd, eps, int(step), int(qgroup_size), params.numel(), ngroups,
        _hip.stream(params.device)), "fp8_adamw_step")


def _check_grad_scale(what, grad_scale, index):
    if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.get_device() != index:
        raise RuntimeError(f"{what}: grad_scale must be one fp32 element on the parameters' device")


def _pointer_array(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _multi(expand, params, grads, exp_avg, exp_avg_sq, scale_lists, hyper, step, qgroup_size, expand_min, grad_scale):
    n = len(params)
    if not (len(grads) == len(exp_avg) == len(exp_avg_sq) == n and all(len(l) == n for l in scale_lists)):
        raise RuntimeError("qoptim_cuda: the tensor lists differ in length")
    if n == 0:
        return
    ngroups = []
    for i in range(n):
        if params[i].dtype != params[0].dtype or params[i].device != params[0].device:
            raise RuntimeError("qoptim_cuda: the tensors of one multi-tensor step share dtype and device")
        ngroups.append(_common_checks(params[i], grads[i], exp_avg[i], exp_avg_sq[i], tuple(l[i] for l in scale_lists), qgroup_size))
        if any(l[i].numel() != ngroups[-1] for l in scale_lists):
            raise RuntimeError("grid_dim == scale_exp_avg_sq.numel()")
    scaled, more = "", ()
    if grad_scale is not None:
        _check_grad_scale("qoptim_cuda", grad_scale, params[0].get_device())
        scaled, more = "_scaled", (_hip.ptr(grad_scale),)
    numel = (ctypes.c_int64 * n)(*[t.numel() for t in params])
    n_scale = (ctypes.c_int64 * n)(*ngroups)
    arrays = [_pointer_array(l) for l in scale_lists]
    beta1, beta2, lr, wd, eps = hyper
    lib, st = _hip.lib(), _hip.stream(params[0].device)
    if expand:
        sm, km, cm, sv, kv, cv = arrays
        rc = getattr(lib, "coat_fp8_adamw_expand_step_multi" + scaled)(
            n, _pointer_array(params), _pointer_array(grads), _hip.dt(params[0]), _pointer_array(exp_avg), sm, km, cm,
            _pointer_array(exp_avg_sq), sv, kv, cv, numel, n_scale, beta1, beta2, lr, wd, eps, int(step), int(qgroup_size),
            int(expand_min), *more, st)
    else:
        sm, sv = arrays
        rc = getattr(lib, "coat_fp8_adamw_step_multi" + scaled)(
            n, _pointer_array(params), _pointer_array(grads), _hip.dt(params[0]), _pointer_array(exp_avg), sm,
            _pointer_array(exp_avg_sq), sv, numel, n_scale, beta1, beta2, lr, wd, eps, int(step), int(qgroup_size), *more, st)
    _hip.check(rc, "fp8_adamw_expand_step_multi" if expand else "fp8_adamw_step_multi")


def fp8_adamw_expand_step_multi(params, grads, exp_avg, scale_exp_avg, expand_exp_avg, sqrtminmax_exp_avg, exp_avg_sq,
                                scale_exp_avg_sq, expand_exp_avg_sq, sqrtminmax_exp_avg_sq, beta1, beta2, lr, wd, eps, step,
                                qgroup_size, expand_min, grad_scale=None):
    """``fp8_adamw_expand_step`` on lists of tensors (one dtype, one device, one step count): one launch per 32 tensors.
    ``grad_scale``: a one-element fp32 tensor on the device that the gradients are multiplied by (``grad_norm_multi``)."""
    _multi(True, params, grads, exp_avg, exp_avg_sq,
           (scale_exp_avg, expand_exp_avg, sqrtminmax_exp_avg, scale_exp_avg_sq, expand_exp_avg_sq, sqrtminmax_exp_avg_sq),
           (beta1, beta2, lr, wd, eps), step, qgroup_size, expand_min, grad_scale)


def fp8_adamw_step_multi(params, grads, exp_avg, scale_exp_avg, exp_avg_sq, scale_exp_avg_sq, beta1, beta2, lr, wd, eps,
                         step, qgroup_size, grad_scale=None):
    """``fp8_adamw_step`` on lists of tensors: one launch per 32 tensors; ``grad_scale`` as above."""
    _multi(False, params, grads, exp_avg, exp_avg_sq, (scale_exp_avg, scale_exp_avg_sq), (beta1, beta2, lr, wd, eps), step,
           qgroup_size, 0, grad_scale)


# ------------------------------------------------------------------------------------------------ 32-bit states, clipping
def grad_norm_multi(grads, max_norm=None):
    """The 2-norm of all ``grads`` (fp32 / bf16 / fp16 GPU tensors) taken together, and the factor that clips them to ``max_norm``.

    Returns ``(norm, scale)``: 0-dim fp32 tensors on the device, ``scale = min(1, max_norm / (norm + 1e-6))``, or None without
    ``max_norm``.  The gradients are only read: pass ``scale`` as ``grad_scale`` to the step.  Squares are summed in 64 bits and a
    fixed order.  A norm that is infinite gives the factor 0, one that is not a number a factor that is not one, as
    ``torch.nn.utils.clip_grad_norm_`` does."""
    grads = list(grads)
    if max_norm is not None and not float(max_norm) >= 0.0:
        raise ValueError(f"grad_norm_multi: invalid max_norm {max_norm}")
    if not grads:
        raise ValueError("grad_norm_multi: no gradients")
    norm, scale = _hip.native().grad_norm_multi(grads, 0.0 if max_norm is None else float(max_norm)).unbind()
    return norm, None if max_norm is None else scale


def adamw_step_multi(params, grads, exp_avg, exp_avg_sq, beta1, beta2, lr, wd, eps, step, masters=None, grad_scale=None):
    """AdamW on lists of tensors with both moments in fp32, in place: one launch per 76 tensors, the formula of
    ``fp8_adamw_step``.  ``params`` share a dtype, ``grads`` have theirs or fp32.  ``masters``: fp32 copies of 16-bit parameters;
    they are stepped, and the parameters receive their rounding.  ``grad_scale``: a one-element fp32 tensor on the device that the
    gradients are multiplied by (``grad_norm_multi``).  ``step`` counts from 1 and is read on the host: a captured graph keeps it.
    Tensors that are stepped may share no memory with each other or with the gradients (RuntimeError)."""
    if len(params) == 0:
        return
    _hip.native().adamw_step_multi(params, grads, exp_avg, exp_avg_sq, masters, beta1, beta2, lr, wd, eps, int(step), grad_scale)
