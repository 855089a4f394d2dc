"""``TropicalSSM`` drop-in (research/tsrn_dml.py:917-980) on the sm_100a scan.

Same constructor, parameters and initialisation (``A``, ``B_proj``, ``C_proj``,
``gate_B``, ``gate_out``, ``mix``), so reference checkpoints load unchanged.
The scan (research/tsrn_dml.py:961-972) changes: the reference evaluates
``h_t = max(A_c + h_{t-1}, u_t)`` (h_{-1} = 0, A_c = clamp(A, max=0)) through
the closed form ``t*A_c + cummax(u - t*A_c)``; here the recurrence itself runs
as one fused kernel (bit-exact with the sequential recurrence; it differs from
the closed form by O(T ulp) rounding).  Gradients follow the same argmax path
(input wins ties, as torch.cummax's last-index rule does).  The three
projections of the input (gate_B, B_proj, gate_out) run as one GEMM on the
stacked weights (in inference an fp32-accurate 3xTF32 tensor-core GEMM,
``ops.linear``).

:class:`GatedSSM` is its (plus, times) counterpart: the same block around the
gated linear recurrence ``h_t = f_t h_{t-1} + (1 - f_t) v_t`` with a forget gate
for every element, ``ops.gated_scan``, and a step for serving.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import ops
from .ops import tropical_scan


class TropicalSSM(nn.Module):
    def __init__(self, d_model: int, d_state: int = None):
        super().__init__()
        ds = d_state or d_model
        self.ds = ds
        self.A = nn.Parameter(torch.randn(ds) * 0.01)
        self.B_proj = nn.Linear(d_model, ds, bias=False)
        self.C_proj = nn.Linear(ds, d_model, bias=False)
        nn.init.zeros_(self.C_proj.weight)
        self.gate_B = nn.Linear(d_model, ds)
        self.gate_out = nn.Linear(d_model, d_model)
        nn.init.zeros_(self.gate_B.weight)
        nn.init.constant_(self.gate_B.bias, 2.0)
        nn.init.zeros_(self.gate_out.weight)
        nn.init.constant_(self.gate_out.bias, 2.0)
        self.mix = nn.Parameter(torch.tensor(0.0))

    def branch(self, x: Tensor):
        """(C_proj of the states, gate_out's logits): the branch before its output gate and
        ``sigmoid(mix)``, for a caller that folds those into its residual sum."""
        # the three projections of x (gate_B, B_proj, gate_out) as one GEMM on
        # the stacked weights; x is read once
        ds, d = self.ds, x.shape[-1]
        w = torch.cat((self.gate_B.weight, self.B_proj.weight, self.gate_out.weight), dim=0)
        b = torch.cat((self.gate_B.bias, self.gate_B.bias.new_zeros(ds), self.gate_out.bias))
        gb, bp, go = ops.linear(x, w, b).split((ds, ds, d), dim=-1)
        u = torch.sigmoid(gb) * bp
        A_c = self.A.clamp(max=0)
        H = tropical_scan(u.contiguous(), None, A_c, 0.0)
        return ops.linear(H, self.C_proj.weight), go

    def forward(self, x: Tensor) -> Tensor:
        o, go = self.branch(x)
        out = torch.sigmoid(go) * o
        return torch.sigmoid(self.mix) * out


class GatedSSM(nn.Module):
    """Gated linear recurrence in the frame of :class:`TropicalSSM`::

        f = sigmoid(gate(x)),  v = B_proj(x)
        h_t = f_t * h_{t-1} + (1 - f_t) * v_t            (ops.gated_scan)
        y = sigmoid(mix) * sigmoid(gate_out(x)) * C_proj(h)

    The gates' biases are spread over memories of about 2 to 1000 steps.  CUDA tensors
    (float32) only."""

    def __init__(self, d_model: int, d_state: int = None):
        super().__init__()
        ds = d_state or d_model
        self.ds = ds
        self.gate = nn.Linear(d_model, ds)
        self.B_proj = nn.Linear(d_model, ds, bias=False)
        self.C_proj = nn.Linear(ds, d_model, bias=False)
        nn.init.zeros_(self.C_proj.weight)
        self.gate_out = nn.Linear(d_model, d_model)
        nn.init.zeros_(self.gate.weight)
        with torch.no_grad():
            # a memory of n steps: f = 1 - 1 / n
            self.gate.bias.copy_(torch.log(torch.logspace(0.3, 3.0, ds) - 1.0))
        nn.init.zeros_(self.gate_out.weight)
        nn.init.constant_(self.gate_out.bias, 2.0)
        self.mix = nn.Parameter(torch.tensor(0.0))

    def init_state(self, batch: int) -> Tensor:
        """The float32 state [batch, d_state] before the first token."""
        return torch.zeros(batch, self.ds, device=self.gate.weight.device)

    def _project(self, x: Tensor):
        # gate, B_proj and gate_out as one GEMM on the stacked weights
        w = torch.cat((self.gate.weight, self.B_proj.weight, self.gate_out.weight), dim=0)
        b = torch.cat((self.gate.bias, self.gate.bias.new_zeros(self.ds), self.gate_out.bias))
        return ops.linear(x, w, b).split((self.ds, self.ds, x.shape[-1]), dim=-1)

    def branch(self, x: Tensor, state: Optional[Tensor] = None,
               lengths: Optional[Tensor] = None, return_state: bool = False):
        """(C_proj of the states, gate_out's logits[, the state at each row's end]); ``state``
        [B, d_state] goes on from an earlier segment, ``lengths`` [B] ends the rows of a padded
        batch (see ``ops.gated_scan``)."""
        z, v, go = self._project(x)
        h, last = ops.gated_scan(z, v, state, form="sigmoid", lengths=lengths, return_state=True)
        o = ops.linear(h, self.C_proj.weight)
        return (o, go, last) if return_state else (o, go)

    def forward(self, x: Tensor, state: Optional[Tensor] = None,
                lengths: Optional[Tensor] = None, return_state: bool = False):
        o, go, last = self.branch(x, state, lengths, return_state=True)
        y = torch.sigmoid(self.mix) * (torch.sigmoid(go) * o)
        return (y, last) if return_state else y

    @torch.no_grad()
    def step(self, x: Tensor, state: Tensor) -> Tensor:
        """One token of every sequence: x [B, d_model]; ``state`` [B, d_state] is updated in
        place."""
        z, v, go = self._project(x)
        h = ops.gated_scan_step(z, v, state, form="sigmoid")
        return torch.sigmoid(self.mix) * (torch.sigmoid(go) * ops.linear(h, self.C_proj.weight))
