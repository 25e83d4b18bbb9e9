"""Backward passes whose results carry no graph of their own.

The framework's autograd functions compute their gradients in kernels.  Under
create_graph=True autograd would take such results for constants and drop what
passes through them from a second derivative without a word.  (torch's
once_differentiable does so too where the incoming gradient needs no gradient,
as in a gradient penalty on sum(y).)"""
import functools

import torch


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, name, _anchor):
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _grad):
        raise RuntimeError("%s has no second derivative: its gradients cannot be differentiated" % ctx.name)


def first_order(backward):
    """Decorator of an autograd function's backward (under @staticmethod): its
    results raise when they are differentiated in their turn."""
    name = backward.__qualname__.partition(".")[0]

    @functools.wraps(backward)
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        anchor = torch.empty(0, requires_grad=True)
        return tuple(_Refuse.apply(t, name, anchor) if isinstance(t, torch.Tensor) else t
                     for t in (out if isinstance(out, tuple) else (out,)))
    return run
