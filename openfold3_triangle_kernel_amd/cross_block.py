"""Pre-norm cross attention of a query stream to an encoder's states, on the MI355X
operators: ``layer_norm`` and ``linear`` with their inputs kept in 8 bits,
``cross_attention``, the sigmoid gate of the pair-stack attention modules and an
output projection.

    x = LN(query), s = LN(states)
    q | g = x W_q^T | x W_g^T,  k | v = s W_k^T | s W_v^T
    out = (cross_attention(q, k, v, key_mask) * sigmoid(g)) W_o^T

A BF16 GPU call of supported sizes runs the kernels; another follows the package's
routing policy: it raises under strict mode and otherwise logs once and runs the
same formulas in PyTorch.
"""

from __future__ import annotations

import math

import torch
from torch import nn

from . import routing
from .activations import linear
from .attention import _device_supported
from .cross_attention import additive_f32, cross_attention
from .layernorm import layer_norm


class CrossAttention(nn.Module):
    """Cross attention with ``no_heads`` query heads of ``c_hidden`` channels on
    ``no_kv_heads`` kv heads (default: as many).

    ``activation_save`` is what the norms and projections keep for the backward:
    ``"int8"`` (8 bits a value) or ``"full"``.  For single tokens, ``project_states``
    forms the states' keys and values once and ``forward`` takes them as ``states``.
    """

    def __init__(self, c_q: int, c_kv: int, c_hidden: int, no_heads: int,
                 no_kv_heads: int | None = None, gating: bool = True,
                 activation_save: str = "int8", eps: float = 1e-5):
        super().__init__()
        no_kv_heads = no_heads if no_kv_heads is None else no_kv_heads
        if min(c_q, c_kv, c_hidden, no_heads, no_kv_heads) < 1 or no_heads % no_kv_heads:
            raise ValueError("sizes must be positive, the query heads a multiple of the kv heads")
        if activation_save not in ("int8", "full"):
            raise ValueError('activation_save must be "int8" or "full"')
        self.c_q, self.c_kv, self.c_hidden = c_q, c_kv, c_hidden
        self.no_heads, self.no_kv_heads = no_heads, no_kv_heads
        self.activation_save, self.eps = activation_save, eps
        self.layer_norm_q = nn.LayerNorm(c_q, eps=eps)
        self.layer_norm_kv = nn.LayerNorm(c_kv, eps=eps)
        hc, kc = no_heads * c_hidden, no_kv_heads * c_hidden
        self.linear_q = nn.Linear(c_q, hc, bias=False)
        self.linear_k = nn.Linear(c_kv, kc, bias=False)
        self.linear_v = nn.Linear(c_kv, kc, bias=False)
        self.linear_g = nn.Linear(c_q, hc, bias=False) if gating else None
        self.linear_o = nn.Linear(hc, c_q, bias=False)

    def _supported(self, *tensors) -> tuple[bool, str]:
        for t in tensors:
            if t.dtype != torch.bfloat16:
                return False, "activations must be BF16"
            ok, reason = _device_supported(t)
            if not ok:
                return False, reason
        if self.c_q % 8 or self.c_kv % 8 or self.c_hidden % 8 or self.c_hidden > 128:
            return False, "channel counts must be multiples of 8 and c_hidden at most 128"
        if any(p.dtype not in (torch.bfloat16, torch.float32) or p.device != tensors[0].device
               for p in self.parameters()):
            return False, "parameters must be BF16 or FP32 on the activations' device"
        return True, ""

    def _kernels(self, *tensors) -> bool:
        ok, reason = self._supported(*tensors)
        if not ok:
            routing.report_fallback(type(self).__qualname__, tuple(tensors[0].shape), reason)
            routing.note_stock_call()
        return ok

    def _norm(self, ln: nn.LayerNorm, x: torch.Tensor, kernels: bool) -> torch.Tensor:
        if kernels:
            return layer_norm(x, ln.weight, ln.bias, self.eps, save=self.activation_save)
        return nn.functional.layer_norm(x.float(), ln.normalized_shape, ln.weight.float(),
                                        ln.bias.float(), self.eps).to(x.dtype)

    def _project(self, x: torch.Tensor, layers, kernels: bool):
        """The layers' outputs of ``x`` from one product over their stacked weights."""
        w = layers[0].weight if len(layers) == 1 else torch.cat([m.weight for m in layers])
        y = linear(x, w, save=self.activation_save) if kernels else x.matmul(w.to(x.dtype).t())
        return y.split([m.weight.shape[0] for m in layers], -1)

    def _heads(self, t: torch.Tensor) -> torch.Tensor:
        return t.unflatten(-1, (-1, self.c_hidden)).transpose(-2, -3)  # [*, heads, N, c_hidden]

    def project_states(self, states: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[*, no_kv_heads, Nk, c_hidden]`` of ``states`` ``[*, Nk, c_kv]``."""
        kernels = self._kernels(states)
        s = self._norm(self.layer_norm_kv, states, kernels)
        return tuple(self._heads(t) for t in self._project(s, (self.linear_k, self.linear_v), kernels))

    def forward(self, x: torch.Tensor, kv: torch.Tensor | None = None,
                key_mask: torch.Tensor | None = None,
                states: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        """``x`` ``[*, Nq, c_q]`` to ``kv`` ``[*, Nk, c_kv]`` (or ``states`` from
        ``project_states``); ``key_mask`` as in ``cross_attention``."""
        if (kv is None) == (states is None):
            raise ValueError("give either kv or states")
        k, v = self.project_states(kv) if states is None else states
        kernels = self._kernels(x, k, v)
        layers = (self.linear_q,) if self.linear_g is None else (self.linear_q, self.linear_g)
        q, *gate = self._project(self._norm(self.layer_norm_q, x, kernels), layers, kernels)
        q = self._heads(q)
        if kernels:
            o = cross_attention(q, k, v, key_mask)
        else:
            o = _stock_cross_attention(q, k, v, key_mask)
        o = o.flatten(-2)
        if gate:
            o = o * torch.sigmoid(gate[0])
        return self._project(o, (self.linear_o,), kernels)[0]


def _stock_cross_attention(q, k, v, key_mask):
    """``cross_attention``'s formulas in PyTorch, [*, Nq, H, D]."""
    group = q.shape[-3] // k.shape[-3]
    k, v = (t.repeat_interleave(group, -3) for t in (k, v))
    if key_mask is not None:
        dead = (~key_mask if key_mask.dtype == torch.bool else torch.isneginf(key_mask))
        dead = dead[..., None, :, None]
        k, v = k.masked_fill(dead, 0.0), v.masked_fill(dead, 0.0)
    s = q.float() @ k.float().transpose(-1, -2).contiguous() / math.sqrt(q.shape[-1])
    if key_mask is not None:
        drop = key_mask[..., None, None, :]
        s = s.masked_fill(~drop, float("-inf")) if drop.dtype == torch.bool else s + additive_f32(drop)
    # The maximum only guards the exponentials; 0 for scores of -inf alone.
    top = s.detach().amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:-1] + (1,))
    p = torch.exp(s - top.masked_fill(torch.isneginf(top), 0.0))
    total = p.sum(-1, keepdim=True)
    if key_mask is not None:
        # Rows without a state give 0; rows whose scores are all -inf otherwise 0 / 0.
        total = total.masked_fill(dead.all(-2, keepdim=True), 1.0)
    p = p / total
    return (p @ v.float()).transpose(-2, -3).to(q.dtype)


__all__ = ["CrossAttention"]
