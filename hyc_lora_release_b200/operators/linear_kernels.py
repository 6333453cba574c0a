"""Products with bias, activation and residual in the epilogue, and their backward pass, on the tcgen05 kernels: the projections of
layers whose MLP is not the gated one of ``mlp`` (no counterpart in the reference's operators)."""
import torch

from .._lib import HycError, host

_ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _act(activation):
    if activation not in _ACTS:
        raise ValueError("activation must be one of %s, got %r" % (", ".join(_ACTS), activation))
    return _ACTS[activation]


def linear_act_forward(x, weight, bias=None, activation="none", residual=None, save_pre=False):
    """-> (y, pre or None): ``y = act(x @ weight.T + bias) + residual`` in one launch, ``pre`` the argument of the activation where
    ``save_pre`` asks for it.  fp32 inside, each result rounded once.

    x [.., K] bf16 or fp16; weight [N, K] as ``nn.Linear`` has it, bias [N], residual [.., N] of the same type.  N and K are multiples of
    8; rows may be any number and have strides of their own (what does not lie on 16 bytes is copied).  activation: "none", "relu" (slope 0 at 0),
    "gelu" (x Phi(x)), "gelu_tanh", "silu"."""
    return host.linear_act_forward(x, weight, bias, _act(activation), residual, bool(save_pre))


def linear_act_backward(dy, x, weight, activation="none", pre=None, needs_grad=(True, True, True)):
    """-> (grad_x, grad_weight, grad_bias), None where ``needs_grad`` does not ask for one (frozen weights: ``(True, False, False)``).
    ``pre`` as forward saved it (not needed without an activation); the residual's gradient is ``dy`` itself.  ``dy * act'(pre)`` is
    rounded to the operands' type before its two products, so that grad_x and grad_weight carry about 1.4 times the error of their own
    rounding (up to 1.5 with one to four tokens); its column sums, the bias gradient, are taken of the unrounded values."""
    need_x, need_w, need_b = needs_grad
    return host.linear_act_backward(dy, x, weight, _act(activation), pre, bool(need_x), bool(need_w), bool(need_b))


def raise_on_device_errors(device=None):
    """Waits for the device (default: the current one) and raises if a bounded wait inside these kernels gave up on it since the library
    was loaded."""
    if isinstance(device, (str, torch.device)):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("expected a CUDA device, got %s" % device)
        device = device.index
    status = host.linear_status(torch.cuda.current_device() if device is None else int(device))
    if status != 0:
        raise HycError("linear kernels: %s" % {1: "TMA producer wait timed out", 2: "MMA issuer wait timed out", 3: "epilogue wait timed out"}
                       .get(status, "status %d" % status))
