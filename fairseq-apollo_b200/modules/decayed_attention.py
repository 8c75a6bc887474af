"""Linear attention with a decay for each head: attention whose cost grows with the length, not with its square.

EfficientAttention (fairseq/modules/efficient_attention.py:11-60) weighs every pair of steps of a chunk by a softmax; here a head
keeps the sum of its keys' and values' products, which a gate of every step lets fade, so a sequence needs no chunks and one token
no cache: (B, L, D) activations, padding masks and a running state under the caller's ``incremental_state`` as in GatedRecurrence.
"""
from typing import Dict, Optional

import torch
from torch import Tensor, nn

from .. import functions, ops
from ..functions import needs_grad
from ..incremental_state import IncrementalStateMixin


def decayed_attention(q, k, v, forget, padding_mask=None, reset_mask=None, h_in=None, scale=1.0, want_state=False, reverse=False):
    """The operator by itself: see ops.decayed_attention_fwd; differentiable in q, k, v, forget and h_in."""
    fn = functions.decayed_attention if needs_grad(q, k, v, forget, h_in) else ops.decayed_attention_fwd
    return fn(q, k, v, forget, padding_mask, reset_mask, h_in, scale, want_state, reverse)


class DecayedAttention(IncrementalStateMixin, nn.Module):
    """y = attention(W_q u, W_k u, W_v u, W_f u) for u (B, L, D): ``zdim`` queries and keys and ``hdim`` values over ``num_heads``
    heads, y (B, L, hdim); ``bidirectional``: the sum of a forward and a backward walk, each with projections of its own.  ``scale``:
    1 / sqrt(keys of a head) where it is None; ``forget_bias`` is what the gates start from (sigmoid(3) = 0.95: about 20 steps)."""

    def __init__(self, embed_dim, num_heads, zdim=None, hdim=None, bidirectional=False, scale=None, forget_bias=3.0):
        super().__init__()
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.zdim = embed_dim if zdim is None else zdim
        self.hdim = embed_dim if hdim is None else hdim
        assert self.zdim % num_heads == 0 and self.hdim % num_heads == 0
        self.keys = self.zdim // num_heads
        self.scale = self.keys ** -0.5 if scale is None else scale
        self.bidirectional = bidirectional
        self.forget_bias = forget_bias
        rows = 2 * self.zdim + self.hdim + num_heads
        self.in_proj = nn.Linear(embed_dim, rows)
        self.back_proj = nn.Linear(embed_dim, rows) if bidirectional else None
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for proj in (self.in_proj, self.back_proj):
                if proj is not None:
                    nn.init.xavier_uniform_(proj.weight)
                    nn.init.zeros_(proj.bias)
                    proj.bias[-self.num_heads:] = self.forget_bias

    def _walk(self, proj, u, padding_mask, reset_mask, h_in, want_state, reverse):
        z = proj(u)
        if needs_grad(z, h_in):
            r = functions.decayed_attention_packed(z, self.num_heads, self.keys, padding_mask, reset_mask, h_in, self.scale, want_state,
                                                   reverse)
        else:
            r = ops.decayed_attention_fwd(*self._parts(z), padding_mask, reset_mask, h_in, self.scale, want_state, reverse)
        return (r[0].flatten(-2), r[1]) if want_state else r.flatten(-2)

    def _parts(self, z):
        q, k, v, f = z.split((self.zdim, self.zdim, self.hdim, self.num_heads), dim=-1)
        return (*(t.unflatten(-1, (self.num_heads, -1)) for t in (q, k, v)), f)

    def forward(self, u: Tensor, padding_mask: Optional[Tensor] = None,
                incremental_state: Optional[Dict[str, Dict[str, Optional[Tensor]]]] = None,
                reset_mask: Optional[Tensor] = None) -> Tensor:
        """u (B, L, D); masks (B, L), non-zero = padded / first step of a document."""
        assert u.size(-1) == self.embed_dim
        if incremental_state is not None:
            assert not self.bidirectional, 'bidirectional attention does not support incremental state'
            if needs_grad(u, *self.parameters()):
                raise NotImplementedError("the incremental state is an inference feature: use torch.no_grad()")
            saved = self._get_input_buffer(incremental_state)
            h = saved.get('prev_state')
            if u.size(1) == 1 and padding_mask is None and reset_mask is None:
                y, h = ops.decayed_attention_step(*self._parts(self.in_proj(u).squeeze(1)), h, self.scale)
                y = y.flatten(-2).unsqueeze(1)
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
        result = self.get_incremental_state(incremental_state, "attention_state")
        return result if result is not None else {}

    def _set_input_buffer(self, incremental_state, buffer):
        return self.set_incremental_state(incremental_state, "attention_state", buffer)

    def reorder_incremental_state(self, incremental_state, new_order: Tensor):
        return self._reorder_buffer(incremental_state, "attention_state", new_order)

    def extra_repr(self) -> str:
        return 'edim={}, heads={}, zdim={}, hdim={}, bidirectional={}'.format(self.embed_dim, self.num_heads, self.zdim, self.hdim,
                                                                            self.bidirectional)
