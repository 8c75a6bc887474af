"""Gated linear recurrence: an EMA whose decay depends on the input.

MultiHeadEMA keeps a fixed decay per channel (fairseq/modules/exponential_moving_average.py:71-80); here a projection of the input
gives the decay of every step, on the same footing otherwise: (B, L, D) activations, padding masks, a running state under the
caller's ``incremental_state``, one token at a time or whole sequences.
"""
from typing import Dict, Optional

import torch
from torch import Tensor, nn

from .. import functions, ops
from ..functions import needs_grad
from ..incremental_state import IncrementalStateMixin


def gated_recurrence(x, forget, input_gate=None, padding_mask=None, reset_mask=None, h_in=None, want_state=False, reverse=False):
    """The operator by itself: see ops.gated_recurrence_fwd; differentiable in x, both gates and h_in."""
    fn = functions.gated_recurrence if needs_grad(x, forget, input_gate, h_in) else ops.gated_recurrence_fwd
    return fn(x, forget, input_gate, padding_mask, reset_mask, h_in, want_state, reverse)


class GatedRecurrence(IncrementalStateMixin, nn.Module):
    """y = recurrence(W_x u, W_f u [, W_i u]) for u (B, L, D); ``bidirectional``: the sum of a forward and a backward walk, each
    with gates of its own.  ``forget_bias`` is what the forget gates start from (sigmoid(3) = 0.95: a state of about 20 steps)."""

    def __init__(self, embed_dim, input_gate=False, bidirectional=False, forget_bias=3.0):
        super().__init__()
        self.embed_dim = embed_dim
        self.input_gate = input_gate
        self.bidirectional = bidirectional
        self.forget_bias = forget_bias
        self.parts = 3 if input_gate else 2
        rows = self.parts * embed_dim
        self.in_proj = nn.Linear(embed_dim, rows)
        self.back_proj = nn.Linear(embed_dim, rows) if bidirectional else None
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for proj in (self.in_proj, self.back_proj):
                if proj is not None:
                    nn.init.xavier_uniform_(proj.weight)
                    nn.init.zeros_(proj.bias)
                    proj.bias[self.embed_dim:2 * self.embed_dim] = self.forget_bias

    def _walk(self, proj, u, padding_mask, reset_mask, h_in, want_state, reverse):
        z = proj(u)
        if needs_grad(z, h_in):
            return functions.gated_recurrence_packed(z, self.input_gate, padding_mask, reset_mask, h_in, want_state, reverse)
        return ops.gated_recurrence_fwd(*self._parts(z), padding_mask, reset_mask, h_in, want_state, reverse)

    def _parts(self, z):
        parts = z.split(self.embed_dim, dim=-1)
        return parts if self.input_gate else (*parts, None)

    def forward(self, u: Tensor, padding_mask: Optional[Tensor] = None,
                incremental_state: Optional[Dict[str, Dict[str, Optional[Tensor]]]] = None,
                reset_mask: Optional[Tensor] = None) -> Tensor:
        """u (B, L, D); masks (B, L), non-zero = padded / first step of a document."""
        assert u.size(-1) == self.embed_dim
        if incremental_state is not None:
            assert not self.bidirectional, 'a bidirectional recurrence does not support incremental state'
            if needs_grad(u, *self.parameters()):
                raise NotImplementedError("the incremental state is an inference feature: use torch.no_grad()")
            saved = self._get_input_buffer(incremental_state)
            h = saved.get('prev_state')
            if u.size(1) == 1 and padding_mask is None and reset_mask is None:
                y, h = ops.gated_recurrence_step(*self._parts(self.in_proj(u).squeeze(1)), h)
                y = y.unsqueeze(1)
            else:
                y, h = self._walk(self.in_proj, u, padding_mask, reset_mask, h, True, False)
            saved['prev_state'] = h
            self._set_input_buffer(incremental_state, saved)
            return y
        y = self._walk(self.in_proj, u, padding_mask, reset_mask, None, False, False)
        if self.bidirectional:
            ends = None
            if reset_mask is not None:   # (walking back, a document starts where the next one is about to)
                ends = torch.ones_like(reset_mask)
                ends[:, :-1] = reset_mask[:, 1:]
            y = y + self._walk(self.back_proj, u, padding_mask, ends, None, False, True)
        return y

    # -- incremental state -------------------------------------------------------------------
    def _get_input_buffer(self, incremental_state):
        result = self.get_incremental_state(incremental_state, "recurrence_state")
        return result if result is not None else {}

    def _set_input_buffer(self, incremental_state, buffer):
        return self.set_incremental_state(incremental_state, "recurrence_state", buffer)

    def reorder_incremental_state(self, incremental_state, new_order: Tensor):
        return self._reorder_buffer(incremental_state, "recurrence_state", new_order)

    def extra_repr(self) -> str:
        return 'edim={}, input_gate={}, bidirectional={}'.format(self.embed_dim, self.input_gate, self.bidirectional)
