"""Operators over the list of an optimisation's gradients, on the native engine (csrc/grads.hip): the norms of the whole list, its scaling to a
bound of one of them, the momentum step.

The gradient of an iPEPS is a list of on-site tensors, float64 or complex128, of which the driver (ad_optim_lbfgs_mod.optimize_state; reference
optim/ad_optim_lbfgs_mod.py:132-360) needs the 2-norm and the largest modulus in every evaluation.  The adjoint of a truncated decomposition grows
without limit next to degenerate singular values (linalg/svd_gesdd.py:209-328 regularises it), and one such evaluation can throw the state away:
`clip_grads` bounds what such a gradient may do to an optimiser that steps along it (gradient descent: `sgd_step` does it on the way; L-BFGS must not
be given scaled gradients, whose differences are no curvature: ad_optim_lbfgs_mod shortens its step instead).

    N2 = (sum over all tensors and elements of |x|^2)^1/2,   Ninf = max |x|,   c = 1 if N <= max_norm, else max_norm / N

All tensors of a list are on the engine's device and of one dtype; empty tensors, 0-dimensional tensors, strided views and empty lists are allowed.
Tensors that are written share no memory with any other tensor of the call (clip_grads: but the one of the same index); where one of them is a
strided view, two of them whose extents interleave (`m[:, :2]` and `m[:, 2:]`) are refused too.  A NaN anywhere, in one part of a complex element too, makes
both norms NaN and a clipped list all NaN; a norm that is infinite or beyond the largest double makes c = 0 (0 x inf = NaN).  The returned norms are
the head of the call's workspace, 35 kB and more: clone what is kept.  Calls run on the current stream, do not synchronise and may be captured into a
graph (after one call outside of it, which makes the native context); they are not differentiable.  As every call of an engine they are one thread's
at a time: another thread inside the same engine makes them raise NativeError."""
import torch
from backend import get_engine


def grad_norms(tensors):
    """[N2, Ninf] of a list of tensors: float64 device tensor of two elements.  Squares do not overflow or underflow."""
    return get_engine().grad_norms(tensors)


def clip_grads(tensors, max_norm, norm_type=2, out=None):
    """Scale a list of tensors by c, in place or into the list `out` (the raw list stays); norm_type 2 or inf.  Returns [N2, Ninf] of the raw list.
    In place a list inside the bound keeps its bits."""
    return get_engine().clip_grads(tensors, max_norm, norm_type=norm_type, out=out)


def clip_grad_norm_(parameters, max_norm, norm_type=2):
    """clip_grads, in place, of the `.grad` of a list of parameters (those without one are left out) or of one parameter."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, norm_type=norm_type)


def sgd_step(params, grads, bufs=None, lr=1.0, momentum=0.0, dampening=0.0, first=False, max_norm=None, norm_type=2):
    """Step of gradient descent with momentum on all tensors of a list, in place, the gradients scaled as by clip_grads on their way (`grads` is
    not written):  m <- c g (first) or momentum m + (1 - dampening) c g,  p <- p - lr m;  momentum 0: p <- p - lr c g.  Returns [N2, Ninf] of the raw
    gradients, None without `max_norm`."""
    return get_engine().sgd_step(params, grads, bufs, lr=lr, momentum=momentum, dampening=dampening, first=first, max_norm=max_norm,
                                 norm_type=norm_type)
