"""The one-shot all-reduce fused with what a transformer layer does to its result: the norm
behind the block, its gate, the scaled residual and the norm in front of the next block; and
the backward pass.  The reference stops at the reduce
(symm_mem_recipes/triton_one_shot_all_reduce.py:96-125); validation, handshake and ownership
are ``one_shot_all_reduce``'s.  Nothing here is recorded by autograd.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .mxfp4 import _call
from .symm_mem import EmulatedSymmetricMemory

_DTYPE_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_FP32}
_GATE_NONE, _GATE_CHANNEL, _GATE_TOKEN, _GATE_ELEMENT = range(4)
#: longest row the kernels keep in a workgroup's registers
MAX_COLS = 16384


class NormGradients(NamedTuple):
    """``partial`` is the gradient of every rank's partial sums; ``post_weight`` and ``gate``
    are None where the forward pass had none."""
    partial: torch.Tensor
    residual: torch.Tensor
    weight: torch.Tensor
    post_weight: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _check(like: torch.Tensor, weight, post_weight, gate, *same_shape) -> Tuple[int, int, int]:
    """Validates the operands of both passes; (rows, cols, gate kind)."""
    dtype, device, shape = like.dtype, like.get_device(), like.shape
    assert dtype in _DTYPE_CODE, "Only bfloat16 and float32 are supported for now."
    assert len(shape) >= 1 and 1 <= shape[-1] <= MAX_COLS, f"the last dimension must be 1..{MAX_COLS}"
    cols = shape[-1]
    rows = like.numel() // cols
    kind = _GATE_NONE
    others = [weight, *same_shape]
    for t in same_shape:
        assert t.shape == shape, "the tensors must have one shape"
    assert weight.shape == (cols,), "weights must be [cols]"
    if post_weight is not None:
        assert post_weight.shape == (cols,), "weights must be [cols]"
        others.append(post_weight)
    if gate is not None:
        gate_shape = gate.shape
        if gate_shape == shape and len(shape) > 1:
            kind = _GATE_ELEMENT
        elif gate_shape == (cols,):
            kind = _GATE_CHANNEL
        elif gate_shape == shape[:-1] + (1,):
            kind = _GATE_TOKEN
        else:
            raise AssertionError("gate must be [cols], [..., 1] or of the tensor's shape")
        others.append(gate)
    assert like.is_contiguous(), "tensor must be contiguous"
    for t in others:
        assert t.dtype is dtype, "the tensors must have one dtype"
        assert t.get_device() == device, "the tensors must be on one device"
        assert t.is_contiguous(), "tensor must be contiguous"
    assert device >= 0, "the tensors must be on a GPU"
    return rows, cols, kind


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def one_shot_all_reduce_norm(tensor: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                             post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                             residual_scale: float = 1.0, eps: float = 1e-6, barrier: bool = True,
                             return_sum: bool = False):
    """The calling rank's ``(normed, residual_out)`` or, with ``return_sum``, ``(normed,
    residual_out, summed)``, all fresh tensors of ``tensor``'s shape::

        summed       = the ranks' symmetric buffers added in rank order (one_shot_all_reduce)
        n            = summed * rsqrt(mean(summed ** 2) + eps) * post_weight     (post_weight None: n = summed)
        residual_out = residual_scale * residual + gate * n                      (gate None: 1)
        normed       = residual_out * rsqrt(mean(residual_out ** 2) + eps) * weight

    with means over the last dimension, everything in fp32 and each output rounded once (the
    norms are of the unrounded values; rows whose squares do not fit fp32 are scaled for them).

    ``tensor``    partial sums [..., cols], allocated via SymmetricMemory, bf16 or fp32, cols <= 16384
    ``residual``  of the same shape and dtype
    ``weight``, ``post_weight``  [cols]
    ``gate``      [cols] (one per channel), [..., 1] (one per token) or of ``tensor``'s shape; a
                  one-dimensional gate of a one-dimensional tensor is per channel
    ``barrier``   the blockwise handshake before the peers are read, as one_shot_all_reduce, and on the
                  same signal pads: calls on one allocation belong on one stream at a time.  None follows
                  the reads: a rank overwrites its buffer only behind its peers' calls
    ``return_sum`` keep the sum too: the backward pass needs it
    """
    rows, cols, kind = _check(tensor, weight, post_weight, gate, residual)
    if rows == 0:                  # an empty tensor has no address to look up, and there is nothing to reduce
        return tuple(torch.empty_like(tensor) for _ in range(3 if return_sum else 2))
    symm_mem = EmulatedSymmetricMemory.rendezvous(tensor)
    assert symm_mem is not None, "tensor must be allocated via SymmetricMemory"
    assert tensor.numel() * tensor.element_size() <= symm_mem.buffer_size, "tensor exceeds the symmetric buffer"
    normed = torch.empty_like(tensor)
    residual_out = torch.empty_like(tensor)
    summed = torch.empty_like(tensor) if return_sum else None
    _call(tensor.get_device(), "one_shot_all_reduce_norm", _lib.load().smr_all_reduce_norm, symm_mem.buffer_ptrs_host,
          symm_mem.signal_pad_ptrs_host if barrier else None, residual.data_ptr(), weight.data_ptr(), _ptr(post_weight),
          _ptr(gate), kind, normed.data_ptr(), residual_out.data_ptr(), _ptr(summed), rows, cols,
          _DTYPE_CODE[tensor.dtype], float(residual_scale), float(eps), symm_mem.rank, symm_mem.world_size,
          _lib.BARRIER_PROXY if barrier else _lib.BARRIER_NONE, symm_mem.status.data_ptr())
    return (normed, residual_out, summed) if return_sum else (normed, residual_out)


def one_shot_all_reduce_norm_backward(grad_normed: torch.Tensor, grad_residual_out: Optional[torch.Tensor],
                                      summed: torch.Tensor, residual_out: torch.Tensor, weight: torch.Tensor, *,
                                      post_weight: Optional[torch.Tensor] = None,
                                      gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                                      eps: float = 1e-6) -> NormGradients:
    """Gradients of :func:`one_shot_all_reduce_norm` with respect to its inputs, from the
    gradients of ``normed`` and ``residual_out`` (None: zero) and from the forward pass's
    ``summed`` and ``residual_out``; the other arguments as given there.  The gradients of the
    weights and of a broadcast gate are summed in fp32, in an order that depends on the sizes
    only, and rounded once.  Rows narrower than 16 bytes go through one workgroup (22 us per 1000)."""
    same = (summed, residual_out) if grad_residual_out is None else (grad_residual_out, summed, residual_out)
    rows, cols, kind = _check(grad_normed, weight, post_weight, gate, *same)
    grads = NormGradients(torch.empty_like(grad_normed), torch.empty_like(grad_normed), torch.empty_like(weight),
                          None if post_weight is None else torch.empty_like(post_weight),
                          None if gate is None else torch.empty_like(gate))
    if rows == 0:
        for g in grads:
            if g is not None:
                g.zero_()
        return grads
    lib = _lib.load()
    dtype = _DTYPE_CODE[grad_normed.dtype]
    need = lib.smr_norm_backward_scratch_bytes(rows, cols, dtype, post_weight is not None, kind)
    scratch = torch.empty(need // 4, dtype=torch.float32, device=grad_normed.device) if need else None
    _call(grad_normed.get_device(), "one_shot_all_reduce_norm_backward", lib.smr_norm_backward, grad_normed.data_ptr(),
          _ptr(grad_residual_out), summed.data_ptr(), residual_out.data_ptr(), weight.data_ptr(), _ptr(post_weight),
          _ptr(gate), kind, grads.partial.data_ptr(), grads.residual.data_ptr(), grads.weight.data_ptr(),
          _ptr(grads.post_weight), _ptr(grads.gate), _ptr(scratch), need, rows, cols, dtype, float(residual_scale), float(eps))
    return grads
