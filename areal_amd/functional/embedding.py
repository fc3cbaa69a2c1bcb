"""Rows of the ``[V, H]`` embedding weight for token ids: the other user of the weight that
``fused_lm_head_logprobs_entropy`` contracts with when a model ties the two. The kernels are
``csrc/embedding.hip``.
"""

from __future__ import annotations

import torch

from areal_amd import _lib

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def embed_tokens(
    input_ids: torch.Tensor,
    weight: torch.Tensor,
    scale: float = 1.0,
    *,
    padding_idx: int | None = None,
    out_dtype: torch.dtype | None = None,
    weight_grad_accum: torch.Tensor | None = None,
) -> torch.Tensor:
    """``scale * weight[input_ids]``, computed in fp32 and rounded once.

    Args:
        input_ids: ``[...]`` integer token ids. An id outside ``[0, V)`` gives zeros and no gradient (the
            rows that another shard of a vocabulary holds).
        weight: ``[V, H]``, fp32, bf16 or fp16.
        scale: multiplier of the rows (and of their gradient).
        padding_idx: an id whose row gets no gradient.
        out_dtype: type of the rows, the weight's by default: bf16 rows of an fp32 master weight need no bf16
            copy of the weight.
        weight_grad_accum: an fp32 ``[V, H]`` tensor (normally the ``.grad`` of an fp32 master weight, or the
            accumulator that ``fused_lm_head_logprobs_entropy`` was given for a tied weight) that the gradient is ADDED
            to; no gradient is then returned for ``weight``, which still has to require one.

    The gradient is summed in fp32 in an order that does not change from run to run, and has the weight's
    type. Each row of the weight that no token names is written as zeros, or with
    ``weight_grad_accum`` not touched.
    """
    if weight.ndim != 2 or weight.size(0) == 0 or weight.size(1) == 0:
        raise ValueError(f"weight must be [V, H], got {tuple(weight.shape)}")
    if weight.dtype not in _DTYPES:
        raise ValueError(f"weight must be fp32, bf16 or fp16, got {weight.dtype}")
    if out_dtype is not None and out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be fp32, bf16 or fp16, got {out_dtype}")
    if input_ids.is_floating_point() or input_ids.is_complex() or input_ids.dtype == torch.bool:
        raise ValueError(f"input_ids must be integers, got {input_ids.dtype}")
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"scale must be finite in fp32, got {scale}")
    if padding_idx is not None and not 0 <= padding_idx < weight.size(0):
        raise ValueError(f"padding_idx must lie in [0, {weight.size(0)}), got {padding_idx}")
    if weight_grad_accum is not None:
        if weight_grad_accum.dtype != torch.float32 or weight_grad_accum.shape != weight.shape:
            raise ValueError(
                "weight_grad_accum must be an fp32 tensor of the weight's shape, got "
                f"{weight_grad_accum.dtype} {tuple(weight_grad_accum.shape)}"
            )
        if not weight_grad_accum.is_contiguous():
            raise ValueError("weight_grad_accum must be contiguous")
        if not torch.is_grad_enabled():
            weight_grad_accum = None
        elif not weight.requires_grad:
            raise ValueError("weight_grad_accum needs a weight that requires a gradient")
    return _lib.host().embed_tokens(
        input_ids, weight, scale, -1 if padding_idx is None else padding_idx, out_dtype, weight_grad_accum
    )
