"""Layers around the gated delta rule: the attention layer with its projections, decays and gated norm, and a pre- and
post-norm stack of such layers with feed-forward blocks, for whole sequences and token by token.

Beside ``CausalLinearAttention`` and ``TransformerEncoder``: a causal model with a state of fixed size.  Everything
between the matrix products is in three operators: the rule (``delta_rule``), its single step, and the norms around a
block (``norms.residual_norm``), which also norms and gates the heads' outputs.
"""
import torch
import torch.nn.functional as F
from torch.nn import Linear, Module, ModuleList, Parameter

from ..delta_rule import gated_delta_rule, gated_delta_step
from ..norms import residual_norm


class GatedDeltaLayer(Module):
    """Projections to queries, keys, values, decays, write strengths and gates, the gated delta rule, the gated norm of
    every head's output, and the projection back.  ``n_key_heads`` (default ``n_heads``) key heads serve ``n_heads``
    value heads.  ``d_keys`` (default ``d_model // n_heads``) is at most 128; ``d_values`` (the same) is 3 to 512: every
    head's output is normalised."""

    def __init__(self, d_model, n_heads, d_keys=None, d_values=None, n_key_heads=None, eps=1e-6):
        super().__init__()
        d_keys = d_keys or d_model // n_heads
        d_values = d_values or d_model // n_heads
        n_key_heads = n_key_heads or n_heads
        if n_heads % n_key_heads:
            raise ValueError("n_heads must be a multiple of n_key_heads")
        if not (1 <= d_keys <= 128 and 3 <= d_values <= 512):
            raise ValueError("takes d_keys from 1 to 128 and d_values from 3 to 512, got %d and %d" % (d_keys, d_values))
        self.n_heads, self.n_key_heads, self.d_keys, self.d_values, self.eps = n_heads, n_key_heads, d_keys, d_values, eps
        self.query_projection = Linear(d_model, n_key_heads * d_keys, bias=False)
        self.key_projection = Linear(d_model, n_key_heads * d_keys, bias=False)
        self.value_projection = Linear(d_model, n_heads * d_values, bias=False)
        self.gate_projection = Linear(d_model, n_heads * d_values, bias=False)
        self.decay_projection = Linear(d_model, n_heads)
        self.beta_projection = Linear(d_model, n_heads)
        self.out_projection = Linear(n_heads * d_values, d_model, bias=False)
        # rates from 1/16 to 1: memories of one to sixteen positions at softplus(0), longer where the projection says so
        self.log_rate = Parameter(torch.linspace(-2.7726, 0.0, n_heads))
        self.norm_weight = Parameter(torch.ones(d_values))

    def _project(self, x):
        lead = x.shape[:-1]
        q = self.query_projection(x).view(*lead, self.n_key_heads, self.d_keys)
        k = self.key_projection(x).view(*lead, self.n_key_heads, self.d_keys)
        v = self.value_projection(x).view(*lead, self.n_heads, self.d_values)
        gate = self.gate_projection(x).view(*lead, self.n_heads, self.d_values)
        log_decay = -self.log_rate.float().exp() * F.softplus(self.decay_projection(x).float())
        beta = torch.sigmoid(self.beta_projection(x).float())
        return q, k, v, gate, log_decay, beta

    def _finish(self, out, gate):
        out, _ = residual_norm(out, gate=gate, after=("rms", self.norm_weight), activation="silu", eps=self.eps)
        return self.out_projection(out.reshape(*out.shape[:-2], -1))

    def new_state(self, batch):
        """The state of ``batch`` sequences before their first position."""
        w = self.norm_weight
        return torch.zeros(batch, self.n_heads, self.d_keys, self.d_values, device=w.device, dtype=torch.float32)

    def forward(self, x, length_mask=None, state=None, return_state=False):
        """``x``: ``(N, L, d_model)``; ``length_mask``: None or a ``LengthMask``; ``state``: None or what a call on
        the positions before returned."""
        q, k, v, gate, log_decay, beta = self._project(x)
        heads = lambda t: t.transpose(1, 2)  # noqa: E731  (N, L, H, ...) -> (N, H, L, ...), where they lie
        out, state = gated_delta_rule(heads(q), heads(k), heads(v), heads(log_decay), heads(beta), state, normalize=True,
                                      lengths=None if length_mask is None else length_mask.lengths, return_state=True)
        out = self._finish(out.transpose(1, 2), gate)
        return (out, state) if return_state else out

    def step(self, x, state):
        """One position: ``x`` ``(N, d_model)``; ``state`` is updated in place."""
        q, k, v, gate, log_decay, beta = self._project(x)
        return self._finish(gated_delta_step(q, k, v, log_decay, beta, state, normalize=True), gate)


class GatedDeltaEncoder(Module):
    """A causal stack: per layer a gated delta layer and a feed-forward block, each with a norm before it, a norm after
    it and a residual scale, all norms between two blocks in one pass (``residual_norm``).  The residual stream is kept
    in ``stream_type`` (float32 by default) whatever the parameters' type."""

    def __init__(self, n_layers, d_model, n_heads, d_ff=None, d_keys=None, d_values=None, n_key_heads=None, residual_scale=1.0,
                 eps=1e-6, stream_type=torch.float32):
        super().__init__()
        d_ff = d_ff or 4 * d_model
        if not 3 <= d_model <= 16384:
            raise ValueError("takes d_model from 3 to 16384, got %d" % d_model)
        self.attentions = ModuleList(GatedDeltaLayer(d_model, n_heads, d_keys, d_values, n_key_heads, eps)
                                     for _ in range(n_layers))
        self.up = ModuleList(Linear(d_model, d_ff) for _ in range(n_layers))
        self.down = ModuleList(Linear(d_ff, d_model) for _ in range(n_layers))
        # before block i (the last one: after the stack), and after it
        self.before = torch.nn.ParameterList(torch.ones(d_model) for _ in range(2 * n_layers + 1))
        self.after = torch.nn.ParameterList(torch.ones(d_model) for _ in range(2 * n_layers))
        self.residual_scale, self.eps, self.stream_type = residual_scale, eps, stream_type

    def _run(self, x, attend):
        h = residual_norm(x, before=("rms", self.before[0]), eps=self.eps)[1]
        stream = x.to(self.stream_type)
        for i in range(len(self.attentions)):
            for block, out in enumerate((attend, self._feed_forward)):
                at = 2 * i + block
                stream, h = residual_norm(out(i, h), stream, after=("rms", self.after[at]),
                                          before=("rms", self.before[at + 1]), scale=self.residual_scale, eps=self.eps)
        return h

    def _feed_forward(self, i, h):
        return self.down[i](F.silu(self.up[i](h)))

    def new_states(self, batch):
        return [layer.new_state(batch) for layer in self.attentions]

    def forward(self, x, length_mask=None, states=None, return_states=False):
        """``x``: ``(N, L, d_model)`` in the parameters' type; ``states``: None or one state a layer."""
        after = [None] * len(self.attentions)

        def attend(i, h):
            out, after[i] = self.attentions[i](h, length_mask, None if states is None else states[i], return_state=True)
            return out
        h = self._run(x, attend)
        return (h, after) if return_states else h

    def step(self, x, states):
        """One position of every sequence: ``x`` ``(N, d_model)``; the states are updated in place."""
        return self._run(x, lambda i, h: self.attentions[i].step(h, states[i]))


__all__ = ["GatedDeltaLayer", "GatedDeltaEncoder"]
