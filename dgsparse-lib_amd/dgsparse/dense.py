"""Dense operators around the sparse products: what a graph (or token) model computes before, between and behind its aggregations, as
hand-written gfx950 kernels (csrc/embedding.hip, rms_norm.hip, gated_ffn.hip, fp8_matmul.hip) behind the same C ABI as the sparse ones.

All of them take float32, float16 and bfloat16 tensors on the GPU (one type a call), run on the current stream of the tensors' device,
never synchronise, and may be captured into a graph.  Sums and row statistics are held in 32 bits; a result is rounded to its type once.
Where a gradient is offered it is that of the formula given, once (no gradient of a gradient, and no forward-mode derivative: both
raise).  New: the reference's layers call torch for all of this (dgsparse/nn/gcnconv.py:10-35, ginconv.py:9-70)."""
from typing import Optional, Tuple

import torch

from . import _ops  # noqa: F401  (registers torch.ops.dgsparse_spmm.*)

_op = torch.ops.dgsparse_spmm
_embedding, _rms_norm, _add_rms_norm, _add_rms_norm_fp8 = _op.embedding.default, _op.rms_norm.default, _op.add_rms_norm.default, _op.add_rms_norm_fp8.default
_gated_ffn, _quantize_fp8, _matmul_fp8 = _op.gated_ffn.default, _op.quantize_fp8.default, _op.matmul_fp8.default


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    r"""``scale * table[ids]``: the rows of ``table`` [tokens, features] named by ``ids`` (int32 or int64, any shape) -> ``[*ids.shape, features]``.

    A negative id stands for "no token" (a padded place of a batch): its row is zero and it takes no part in the gradient.  An id behind
    the table's end is a mistake that costs no memory access: its row is NaN.  ``padding_idx`` names a row that is looked up like any
    other but gets no gradient.

    Gradient of ``table``: every row is ``scale *`` the sum of the output's gradient over the places that hold its id, added up in a fixed
    order (the same bits on every run), zero for rows without a place."""
    if padding_idx is not None and padding_idx < 0:
        raise ValueError('dgsparse: padding_idx must not be negative (negative ids are "no token" already)')
    return _embedding(ids, table, scale, -1 if padding_idx is None else padding_idx)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    r"""``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension.  Gradients of ``x`` and ``weight``."""
    return _rms_norm(x, weight, eps)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""``s = x + residual`` (rounded to their type: the residual of the next layer) and ``y = rms_norm(s, weight)`` in one pass over the
    rows -> ``(y, s)``.  Gradients of all three inputs; those of ``x`` and ``residual`` are one tensor."""
    return _add_rms_norm(x, residual, weight, eps)


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) \
        -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    r"""``add_rms_norm`` with the normed rows in 8 bits, for :func:`matmul_fp8` -> ``(q, scale, s)``: ``q`` in ``float8_e4m3fn`` and, for each
    row and block of 128 features, ``scale = max |y| / 448``; ``y`` is ``q * scale``.  For serving: it records no gradient."""
    return _add_rms_norm_fp8(x, residual, weight, eps)


_ACTIVATIONS = {'silu': 0, 'gelu': 1, 'relu': 2}


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = 'silu',
              recompute: Optional[bool] = None) -> torch.Tensor:
    r"""``act(x @ w_gate.T) * (x @ w_up.T)`` in one kernel: both projections of a gated feed-forward block, the activation (``'silu'``, ``'gelu'``
    in its erf form, or ``'relu'``) and the product.  ``x`` [..., features], the weights [hidden, features] as ``torch.nn.Linear`` keeps them.

    Gradients of ``x`` and both weights; the two projections' gradients are rounded once to the operands' type.  For them the backward pass
    needs the projections: ``recompute=False`` keeps both in 32 bits, ``True`` makes them again, ``None`` keeps them where that is faster
    and takes no more than 1 GiB.  Both ways give results within the rounding of the other (the same bits from 65 rows on).

    In float32 a value takes part as the sum of three of 16 bits (products as close as ones rounded to 32 bits): beyond 64 rows
    an infinity in ``x`` or a weight (or a magnitude above 3.38e38) gives NaN, in the rows that it reaches."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f'dgsparse: activation must be one of {sorted(_ACTIVATIONS)}, not {activation!r}')
    return _gated_ffn(x, w_gate, w_up, _ACTIVATIONS[activation], -1 if recompute is None else int(not recompute))


def quantize_fp8(x: torch.Tensor, block_rows: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""``x`` [..., features] in 8 bits -> ``(q, scale)``: ``q`` in ``float8_e4m3fn`` and a float32 ``scale = max |x| / 448`` for each
    ``block_rows`` x 128 values; ``x`` is ``q * scale``.  ``block_rows=1`` (a scale for each row: activations) or ``128`` (weights; 2-D).
    It records no gradient."""
    if block_rows not in (1, 128):
        raise ValueError(f'dgsparse: block_rows must be 1 or 128, not {block_rows}')
    return _quantize_fp8(x, block_rows)


def matmul_fp8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    r"""``a @ b.T`` of 8-bit operands with a scale for each block of 128: ``a`` [..., K] with ``a_scale`` [..., ceil(K / 128)]
    (:func:`add_rms_norm_fp8`, ``quantize_fp8(x)``), ``b`` [N, K] with ``b_scale`` [ceil(N / 128), ceil(K / 128)] (``quantize_fp8(w, 128)``) ->
    [..., N] in ``out_dtype``.  Sums in 32 bits, one rounding; so is the product of a block's two scales, which has to lie in their normal range
    (largest values of a row and of a block of weights whose product is between 2e-33 and 6e43).  For serving: it records no gradient."""
    return _matmul_fp8(a, a_scale, b, b_scale, out_dtype)
