"""The training path's differentiable operators.  The autograd Functions are native (host/host.cpp): forward and
backward run on the library's kernels, and the backward without the interpreter; what is saved between them follows
the reference's Functions (fairseq/modules/norm_layer/timestep_norm.py:14-66, sequence_norm.py:12-52,
fairseq/modules/fused_ops/{fftconv,ema_parameters,ema_hidden}.py)."""
import torch
from torch.nn.modules.module import _has_any_global_hook

from . import _lib, ops


def needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def plain(module, *types):
    """Whether calling the module is its class's forward and nothing else: one of these classes itself (an adapter, a
    quantised or a sharded layer is another), no forward of its own, no hooks.  Only then may a path take the module's
    parameters instead of calling it."""
    d = module.__dict__
    return (type(module) in types and "forward" not in d
            and not (d["_forward_hooks"] or d["_forward_pre_hooks"] or d["_backward_hooks"] or d["_backward_pre_hooks"])
            and not _has_any_global_hook())


def ema(x, alpha, delta, third, gamma, omega, padding_mask, bidirectional, shift, truncation=None, complex_poles=False,
        silu=False, channels_last=False):
    """y = EMA(x) [then SiLU] for x (B, D, L), with ``channels_last`` (B, L, D), from the layer's raw parameters; ``third`` is beta (real poles) or
    theta (complex ones)."""
    return _lib.host().ema_train(x, alpha, delta, third, gamma, omega, padding_mask, ops._flags(bidirectional, shift, False),
                                 ops._trunc(truncation), complex_poles, silu, channels_last)


def timestep_norm(x, prior_count, prior_mean, prior_logv, weight, bias, padding_mask, num_groups, eps):
    """y = TimestepNorm(x (B, L, D)) from the module's parameters.  Per-feature statistics (channels contiguous) are
    taken again in the backward, so only the arguments are kept; otherwise the statistics of every step are."""
    return _lib.host().timestep_norm_train(x, prior_count, prior_mean, prior_logv, weight, bias, padding_mask,
                                           0 if num_groups is None else num_groups, eps)


def sequence_norm(x, weight, bias, padding_mask, eps, length_last, num_groups=None):
    """y = SequenceNorm(x), per channel or per channel group, from the module's parameters."""
    return _lib.host().sequence_norm_train(x, weight, bias, padding_mask, eps, length_last,
                                           0 if num_groups is None else num_groups)


def gated_recurrence(x, forget, input_gate=None, padding_mask=None, reset_mask=None, h_in=None, want_state=False, reverse=False):
    """ops.gated_recurrence_fwd with gradients of x, both gates and h_in (through y and through the state that leaves)."""
    r = _lib.host().gated_recurrence_train(x, forget, input_gate, padding_mask, reset_mask, h_in, want_state, reverse)
    return tuple(r) if want_state else r[0]


def gated_recurrence_packed(z, gated=False, padding_mask=None, reset_mask=None, h_in=None, want_state=False, reverse=False):
    """gated_recurrence on z (B, L, 2 D), x and the forget gate side by side (with ``gated`` (B, L, 3 D), the input gate behind
    them), as one projection leaves them; z's gradient is written in place of its parts."""
    r = _lib.host().gated_recurrence_packed(z, gated, padding_mask, reset_mask, h_in, want_state, reverse)
    return tuple(r) if want_state else r[0]


def group_norm(x, weight, bias, num_groups, padding_mask, eps, activation):
    """y = act(GroupNorm(x)) from the module's parameters (effective scale weight + 1)."""
    fn = _lib.host().group_norm_train if needs_grad(x, weight, bias) else _lib.host().group_norm
    return fn(x, weight, bias, num_groups, padding_mask, eps, ops._silu(activation))


def decayed_attention(q, k, v, forget, padding_mask=None, reset_mask=None, h_in=None, scale=1.0, want_state=False, reverse=False):
    """ops.decayed_attention_fwd with gradients of q, k, v, forget and h_in (through y and through the state that leaves)."""
    r = _lib.host().decayed_attention_train(q, k, v, forget, padding_mask, reset_mask, h_in, float(scale), want_state, reverse)
    return tuple(r) if want_state else r[0]


def decayed_attention_packed(z, num_heads, keys, padding_mask=None, reset_mask=None, h_in=None, scale=1.0, want_state=False, reverse=False):
    """decayed_attention on z (B, L, H (2 K + V + 1)): queries, keys, values and gates of all heads side by side, as one projection
    leaves them; z's gradient is written in place of its parts."""
    r = _lib.host().decayed_attention_packed(z, num_heads, keys, padding_mask, reset_mask, h_in, float(scale), want_state, reverse)
    return tuple(r) if want_state else r[0]


def rms_norm(x, weight, residual=None, num_groups=1, eps=1e-5):
    """ops.rms_norm_fwd with gradients of x, the residual and weight."""
    r = _lib.host().rms_norm_train(x, weight, residual, int(num_groups), float(eps))
    return r[0] if residual is None else tuple(r)
