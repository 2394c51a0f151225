"""Pre-norm causal self-attention of a token stream, on the MI355X operators: ``layer_norm``
and ``linear`` with their inputs kept in 8 bits, ``qk_norm_rotary``, ``window_attention`` (or,
through a paged cache, ``append_kv`` and ``paged_attention``), the sigmoid gate of the
pair-stack attention modules and an output projection.

    h = LN(x),  q | k | v | g = h W^T
    q, k = rotation by position of RMSNorm(q), RMSNorm(k), head by head
    out = (window_attention(q, k, v, window, sinks, key_mask) * sigmoid(g)) W_o^T

A BF16 GPU call of supported sizes runs the kernels; another follows the package's
routing policy: it raises under strict mode and otherwise logs once and runs the
same formulas in PyTorch.
"""

from __future__ import annotations

import math
import warnings

import torch
from torch import nn

from .cross_block import AttentionBlock
from .paged import PagedCache, append_kv, paged_attention
from .rotary import qk_norm_rotary
from .window_attention import window_attention


class SelfAttention(AttentionBlock):
    """Causal self-attention with ``no_heads`` query heads of ``c_hidden`` channels on
    ``no_kv_heads`` kv heads (default: as many).

    Tokens see the ``window`` tokens up to themselves (None: all before them) and the first
    ``sinks``.  The first ``rotary_channels`` channels of a head (default: all) are turned by
    ``position * rotary_base^(-2 c / rotary_channels)``, or by ``position * frequencies[c]``
    where these are given; 0 leaves the rotation out.  A ``state_dict`` holds the frequencies;
    loading one keeps the block's own and warns if they differ.  ``qk_norm`` normalises the
    heads of q and k.  ``activation_save`` as in ``CrossAttention``.  ``step`` takes new tokens
    of many sequences through a paged cache.
    """

    def __init__(self, c_in: int, c_hidden: int, no_heads: int, no_kv_heads: int | None = None,
                 window: int | None = None, sinks: int = 0, rotary_channels: int | None = None,
                 rotary_base: float = 10000.0, frequencies: torch.Tensor | None = None,
                 interleaved: bool = False, qk_norm: bool = True, gating: bool = True,
                 activation_save: str = "int8", eps: float = 1e-5):
        super().__init__()
        no_kv_heads = no_heads if no_kv_heads is None else no_kv_heads
        if min(c_in, c_hidden, no_heads, no_kv_heads) < 1 or no_heads % no_kv_heads:
            raise ValueError("sizes must be positive, the query heads a multiple of the kv heads")
        if activation_save not in ("int8", "full"):
            raise ValueError('activation_save must be "int8" or "full"')
        if (window is not None and window < 1) or sinks < 0:
            raise ValueError("window must be positive or None, sinks not negative")
        if frequencies is None:
            turned = c_hidden // 2 * 2 if rotary_channels is None else rotary_channels
            if turned < 0 or turned % 2 or turned > c_hidden:
                raise ValueError("rotary_channels must be even and at most c_hidden")
            frequencies = torch.tensor([rotary_base ** (-2.0 * c / turned) for c in range(turned // 2)],
                                       dtype=torch.float64, device="cpu")
        elif frequencies.ndim != 1 or 2 * len(frequencies) > c_hidden:
            raise ValueError("frequencies must have one axis, at most half the head's channels")
        self.c_in, self.c_hidden = c_in, c_hidden
        self._widths = (c_in,)
        self.no_heads, self.no_kv_heads = no_heads, no_kv_heads
        self.window, self.sinks, self.interleaved = window, sinks, interleaved
        self.activation_save, self.eps = activation_save, eps
        # In 64 bits whatever type the module is cast to; copies by device.
        self._frequencies = {"cpu": frequencies.detach().to("cpu", torch.float64, copy=True)}
        self.layer_norm = nn.LayerNorm(c_in, eps=eps)
        hc, kc = no_heads * c_hidden, no_kv_heads * c_hidden
        self.linear_q = nn.Linear(c_in, hc, bias=False)
        self.linear_k = nn.Linear(c_in, kc, bias=False)
        self.linear_v = nn.Linear(c_in, kc, bias=False)
        self.linear_g = nn.Linear(c_in, hc, bias=False) if gating else None
        self.linear_o = nn.Linear(hc, c_in, bias=False)
        self.norm_q = nn.Parameter(torch.ones(c_hidden)) if qk_norm else None
        self.norm_k = nn.Parameter(torch.ones(c_hidden)) if qk_norm else None

    def new_cache(self, pages: int, page: int, device="cuda") -> PagedCache:
        """A cache of ``pages`` pages of ``page`` states for ``step``."""
        return PagedCache(pages, self.no_kv_heads, page, self.c_hidden, torch.bfloat16, device)

    def get_extra_state(self) -> torch.Tensor:
        return self._frequencies["cpu"].clone()

    def set_extra_state(self, state: torch.Tensor) -> None:
        """The block's own frequencies stay (a context may be scaled by others); that a
        checkpoint's differ, beyond roundings of a cast or a mean, is said."""
        mine, given = self._frequencies["cpu"], state.detach().to("cpu", torch.float64)
        if given.shape != mine.shape or not torch.allclose(
                mine, given, rtol=max(1e-6, torch.finfo(state.dtype).eps), atol=0.0):
            warnings.warn("SelfAttention: the checkpoint's block was made with other rotary frequencies; "
                          "this block keeps its own", stacklevel=2)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, *rest):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, *rest)
        key = prefix + "_extra_state"  # (earlier checkpoints have none)
        if key in missing_keys:
            missing_keys.remove(key)

    def _rotation(self, device):
        f = self._frequencies.get(str(device))
        if f is None:
            # (Outside inference mode, whose tensors a later backward could not keep.)
            with torch.inference_mode(False):
                f = self._frequencies[str(device)] = self._frequencies["cpu"].to(device)
        return f if len(f) else None

    def _streams(self, x: torch.Tensor, kernels: bool):
        """q, k, v [*, N, heads, c_hidden] and the gate (a list, empty without)."""
        layers = [self.linear_q, self.linear_k, self.linear_v] + (
            [] if self.linear_g is None else [self.linear_g])
        q, k, v, *gate = self._project(self._norm(self.layer_norm, x, kernels), layers, kernels)
        return [t.unflatten(-1, (-1, self.c_hidden)) for t in (q, k, v)], gate

    def _out(self, o: torch.Tensor, gate, kernels: bool) -> torch.Tensor:
        o = o.flatten(-2)
        if gate:
            o = o * torch.sigmoid(gate[0])
        return self._project(o, (self.linear_o,), kernels)[0]

    def forward(self, x: torch.Tensor, key_mask: torch.Tensor | None = None,
                positions: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` ``[*, N, c_in]``; ``key_mask`` as in ``window_attention``; ``positions`` turn
        the heads (default: 0 .. N - 1)."""
        kernels = self._kernels(x)
        (q, k, v), gate = self._streams(x, kernels)
        q, k, v = (t.transpose(-2, -3) for t in (q, k, v))
        turn = (positions, self._rotation(x.device), self.norm_q, self.norm_k,
                None if self.norm_q is None else self.eps, self.interleaved)
        if kernels:
            q, k = qk_norm_rotary(q, k, *turn)
            o = window_attention(q, k, v, self.window, self.sinks, key_mask)
        else:
            q, k = _stock_rotary(q, *turn, 2), _stock_rotary(k, *turn, 3)
            o = _stock_window(q, k, v, self.window, self.sinks, key_mask)
        return self._out(o, gate, kernels)

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: PagedCache, tables: torch.Tensor, starts: torch.Tensor,
             lengths: torch.Tensor) -> torch.Tensor:
        """New tokens ``x`` ``[T, c_in]`` of the sequences that ``tables``, ``starts`` and
        ``lengths`` describe (``append_kv``): their keys and values go into ``cache``, their
        rows are what ``forward`` gives for them among their sequences' tokens.  Inference,
        on the kernels alone; can be captured and replayed (after a first call on the device)."""
        ok, reason = self._supported(x)
        if not ok:
            raise ValueError(f"unsupported self-attention step: {reason}")
        (q, k, v), gate = self._streams(x, True)
        q = append_kv(cache, k, v, tables, starts, lengths, q, self._rotation(x.device), self.norm_q,
                      self.norm_k, None if self.norm_q is None else self.eps, self.interleaved)
        o = paged_attention(q, cache, tables, starts, lengths, self.window, self.sinks)
        return self._out(o, gate, True)


def _stock_rotary(x, positions, frequencies, q_weight, k_weight, eps, interleaved, side):
    """``qk_norm_rotary``'s formulas in PyTorch for x [*, H, N, D]; side 2: q, 3: k."""
    dtype, x = x.dtype, x.float()
    if eps is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        x = x * (q_weight if side == 2 else k_weight).float()
    if frequencies is None:
        return x.to(dtype)
    half = len(frequencies)
    if positions is None:
        positions = torch.arange(x.shape[-2], device=x.device)
    angle = (positions.double()[..., None] * frequencies).unsqueeze(-3)
    cos, sin = angle.cos().float(), angle.sin().float()
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((head, rest), -1).to(dtype)


def _stock_window(q, k, v, window, sinks, key_mask):
    """``window_attention``'s formulas in PyTorch, [*, N, H, D]."""
    group = q.shape[-3] // k.shape[-3]
    k, v = (t.repeat_interleave(group, -3) for t in (k, v))
    n = torch.arange(q.shape[-2], device=q.device)
    far = n[:, None] - n
    see = far >= 0
    if window is not None:
        see = see & ((far < window) | (n < sinks))
    if key_mask is not None:
        see = see & key_mask[..., None, None, :]
        k, v = (t.masked_fill(~key_mask[..., None, :, None], 0.0) for t in (k, v))
    s = q.float() @ k.float().transpose(-1, -2).contiguous() / math.sqrt(q.shape[-1])
    s = s.masked_fill(~see, float("-inf"))
    # The maximum only guards the exponentials; 0 for scores of -inf alone.
    top = s.detach().amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:-1] + (1,))
    p = torch.exp(s - top.masked_fill(torch.isneginf(top), 0.0))
    total = p.sum(-1, keepdim=True)
    # Rows that see no state give 0; rows whose scores are all -inf otherwise 0 / 0.
    total = total.masked_fill(~see.any(-1, keepdim=True), 1.0)
    return ((p / total) @ v.float()).transpose(-2, -3).to(q.dtype)


__all__ = ["SelfAttention"]
