"""Layers on the dense operators (dgsparse/dense.py), in the form the graph layers take them: node / token embeddings in front of a first
aggregation, the residual norm between layers, a gated update function behind an aggregation (``GINConv(apply_func=GatedFFN(...))``), and the
projection of a ``GCNConv`` in 8 bits for serving.  New: the reference's models use torch modules for these (dgsparse/nn/ginconv.py:73-112)."""
from typing import Optional, Tuple

import torch

from .. import dense
from .fused import spmm_sum_fused
from .gcnconv import GCNConv


class Embedding(torch.nn.Module):
    """``scale * weight[ids]``; negative ids are "no token" (dense.embedding)."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, scale: float = 1.0):
        super().__init__()
        if padding_idx is not None and not 0 <= padding_idx < num_embeddings:
            raise ValueError(f'dgsparse: padding_idx {padding_idx} is not a row of the table')
        self.padding_idx, self.scale = padding_idx, scale
        self.weight = torch.nn.Parameter(torch.randn(num_embeddings, embedding_dim))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx] = 0

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return dense.embedding(ids, self.weight, self.scale, self.padding_idx)


class RMSNorm(torch.nn.Module):
    """``rms_norm(x)``, or with a residual ``(rms_norm(x + residual), x + residual)``."""

    def __init__(self, size: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(size))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if residual is None:
            return dense.rms_norm(x, self.weight, self.eps)
        return dense.add_rms_norm(x, residual, self.weight, self.eps)


class GatedFFN(torch.nn.Module):
    """``down(act(x Wg^T) * (x Wu^T))``: the two projections, the activation and the product in one kernel, then a Linear."""

    def __init__(self, in_size: int, hidden_size: int, out_size: Optional[int] = None, activation: str = 'silu'):
        super().__init__()
        self.activation = activation
        self.w_gate = torch.nn.Parameter(torch.empty(hidden_size, in_size))
        self.w_up = torch.nn.Parameter(torch.empty(hidden_size, in_size))
        for w in (self.w_gate, self.w_up):
            torch.nn.init.kaiming_uniform_(w, a=5 ** 0.5)  # as torch.nn.Linear
        self.down = torch.nn.Linear(hidden_size, in_size if out_size is None else out_size, bias=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down(dense.gated_ffn(x, self.w_gate, self.w_up, self.activation))


class LinearFP8(torch.nn.Module):
    """A bias-free Linear whose weight is held in 8 bits with a scale for each 128 x 128 (serving: no gradient).  Takes float rows, or the pair
    ``(q, scale)`` that ``add_rms_norm_fp8`` leaves."""

    def __init__(self, weight: torch.Tensor, out_dtype: torch.dtype = torch.float32):
        super().__init__()
        q, scale = dense.quantize_fp8(weight.detach(), 128)
        self.register_buffer('weight', q)
        self.register_buffer('weight_scale', scale)
        self.out_dtype = out_dtype

    def requantize(self, weight: torch.Tensor) -> None:
        """The 8-bit values of another weight of the same shape, in place."""
        q, scale = dense.quantize_fp8(weight.detach(), 128)
        self.weight.view(torch.uint8).copy_(q.view(torch.uint8))
        self.weight_scale.copy_(scale)

    def _apply(self, fn, recurse=True):
        # half(), to(dtype) and their like change what is trained and multiplied in that type: the 8-bit values and their scales go along as the
        # whole numbers of their bits, which a change of device moves and a change of type leaves alone
        kept = {}
        for name in ('weight', 'weight_scale'):
            held = self._buffers[name]
            bits = held.view({1: torch.uint8, 4: torch.int32}[held.element_size()])
            moved = fn(bits)
            kept[name] = (moved if moved.dtype == bits.dtype else bits.to(moved.device)).view(held.dtype)
        super()._apply(fn, recurse)
        self._buffers.update(kept)
        return self

    def forward(self, x) -> torch.Tensor:
        q, scale = x if isinstance(x, tuple) else dense.quantize_fp8(x)
        return dense.matmul_fp8(q, scale, self.weight, self.weight_scale, self.out_dtype)


class ResidualGCN(torch.nn.Module):
    """A residual graph layer with its norms in front: ``m = relu(A_hat (norm(x + r) W))``, ``out = ffn(norm(m + s))`` -> ``(out, s')`` where ``s``, ``s'``
    are the running residuals.  ``quantize()`` puts the graph projection into 8 bits for serving: the norm then writes 8-bit rows, which the
    projection reads as they are.  The 8-bit weight is made from the weight, by ``quantize()`` and again behind
    ``load_state_dict``; it is no part of a state dict, and training drops it.  A weight that is written to by other means in between is quantized again by
    ``quantize()``."""

    def __init__(self, size: int, hidden_size: int, activation: str = 'silu', eps: float = 1e-6):
        super().__init__()
        self.norm1, self.norm2 = RMSNorm(size, eps), RMSNorm(size, eps)
        self.conv = GCNConv(size, size, activation='relu')
        self.ffn = GatedFFN(size, hidden_size, activation=activation)
        self.conv8 = None
        self.in_8_bits = False
        self.register_load_state_dict_post_hook(ResidualGCN._weight_loaded)

    def quantize(self) -> 'ResidualGCN':
        self.in_8_bits = True
        if self.conv8 is None:
            self.projection8()
        else:
            self.conv8.requantize(self.conv.W.weight)
        return self.eval()

    def projection8(self) -> LinearFP8:
        if self.conv8 is None:
            self.conv8 = LinearFP8(self.conv.W.weight)
            for name, held in list(self.conv8.named_buffers()):  # made of the weight: no part of a state dict
                self.conv8.register_buffer(name, held, persistent=False)
        return self.conv8

    def train(self, mode: bool = True) -> 'ResidualGCN':
        if mode:
            self.in_8_bits, self.conv8 = False, None
        return super().train(mode)

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        for key in [k for k in state_dict if k.startswith(prefix + 'conv8.')]:  # (written when they were a part of it)
            del state_dict[key]
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def _weight_loaded(self, _keys) -> None:
        if self.conv8 is not None and self.conv.W.weight.is_cuda:
            self.conv8.requantize(self.conv.W.weight)  # in place: a captured graph reads it where it is
        else:
            self.conv8 = None  # (made again where it is used)

    def forward(self, dcsr, x: torch.Tensor, residual: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        if self.in_8_bits:
            with torch.no_grad():
                q, scale, s = dense.add_rms_norm_fp8(x, residual, self.norm1.weight, self.norm1.eps)
                m = spmm_sum_fused(dcsr, self.projection8()((q, scale)), relu=True)
                y, s = self.norm2(m, s)
                return self.ffn(y), s
        y, s = self.norm1(x, residual)
        y, s = self.norm2(self.conv(dcsr, y), s)
        return self.ffn(y), s
