"""The operators of a training step around the NVFP4 cast, on torch tensors:
products of NVFP4 operands, layer norm forward and backward, AdamW.

Each function checks its tensors, allocates its outputs and any scratch with
torch (so both belong to the stream, and inside a capture to the graph), and
launches on the current stream of the tensors' device.  Bad arguments raise
ValueError here or NVFP4Error from the library.  The pointer-level forms, with
explicit streams and workspaces, are in ops.

The checks and calls of the step's own operators are compiled
(csrc/torch_binding.cpp): their smallest cases take a few microseconds on the
device."""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import ops
from ._native import check, load_binding

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32 = torch.float32
STATE_BLOCK = 128   # elements that share one scale byte of an 8-bit state


def _result(name: str, r):
    """What a compiled call returned: tensors, or the library's status."""
    if r.__class__ is int:
        check(name, r)
    return r


def matmul_nvfp4(a: torch.Tensor, a_scales: torch.Tensor, a_amax: torch.Tensor, b: torch.Tensor,
                 b_scales: torch.Tensor, b_amax: torch.Tensor, *,
                 bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                 activation: str = "none", out_dtype: torch.dtype = torch.bfloat16,
                 out: Optional[torch.Tensor] = None, with_aux: bool = False,
                 amax_out: Optional[torch.Tensor] = None):
    """act(A B^T + bias) + residual of two NVFP4 operands (codes [rows, k/2],
    scales [rows, k/16], amax, as the casts return them).  Returns (D [m, n],
    aux or None); aux is the activation's argument, for matmul_nvfp4_dact.
    `out` (may be `residual`) receives D in place of a new tensor; `amax_out`
    (one float32) receives max |D|."""
    code = _DTYPES.get(out_dtype)
    if code is None:
        raise ValueError(f"unexpected out_dtype {out_dtype}")
    return _result("nvfp4_gemm", load_binding().matmul(
        a, a_scales, a_amax, b, b_scales, b_amax, bias, residual, ops._activation(activation),
        code, out, with_aux, amax_out))


def matmul_nvfp4_dact(a: torch.Tensor, a_scales: torch.Tensor, a_amax: torch.Tensor,
                      b: torch.Tensor, b_scales: torch.Tensor, b_amax: torch.Tensor,
                      aux: torch.Tensor, *, activation: str, with_dbias: bool = False,
                      amax_out: Optional[torch.Tensor] = None):
    """(A B^T) act'(aux), of aux's type, and its column sums in fp32 (the bias
    gradient) or None."""
    return _result("nvfp4_gemm_dact", load_binding().matmul_dact(
        a, a_scales, a_amax, b, b_scales, b_amax, aux, ops._activation(activation), with_dbias,
        amax_out))


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor] = None,
              eps: float = 1e-5, *, amax_out: Optional[torch.Tensor] = None):
    """Layer norm over the last dimension of a 2-D tensor.  Returns (y, mean,
    rstd); `amax_out` (one float32) receives max |y| for the cast of y."""
    return _result("nvfp4_layernorm_fwd",
                   load_binding().layernorm(x, gamma, beta, eps, amax_out))


def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       gamma: torch.Tensor, *, residual: Optional[torch.Tensor] = None):
    """Gradients (dx, dgamma, dbeta) of layernorm; `residual` is added to dx
    (the gradient that reaches x past the norm).  dgamma and dbeta have
    gamma's type."""
    return _result("nvfp4_layernorm_bwd",
                   load_binding().layernorm_backward(dy, x, mean, rstd, gamma, residual))


class AdamW:
    """The tensors of an AdamW step, described once for any number of steps.

    params (float32 or bfloat16), grads, exp_avgs and exp_avg_sqs are lists of
    contiguous tensors, one entry per parameter.  float32 moments are held as
    they are; uint8 moments need the scale tensors (ceil(n / 128) uint8 each),
    rng_state (int64 {seed, offset} on the device) and, for each tensor, the
    position of its first element in the numbering that the random bits go by
    (`offsets`, multiples of 128; default: one tensor behind the other).
    `copies` (bfloat16) receive the rounded new parameters, `amax_out` (one
    float32 per tensor) their amax.  All memory is the caller's.

    What a step writes must not overlap, nor what it reads lie in it.  The tensors
    are held, and every step looks whether each still has the memory
    it had (after `p.data = ...`, set_ or resize_ it has not: ValueError).
    Gradients that are new tensors are passed to step, which then uses them until
    it gets others; a gradient that was its parameter's .grad when it was listed
    must still be that (ValueError otherwise)."""

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
                 exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], *,
                 exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
                 exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
                 copies: Optional[Sequence[torch.Tensor]] = None,
                 weight_decays: Optional[Sequence[float]] = None,
                 offsets: Optional[Sequence[int]] = None,
                 amax_out: Optional[torch.Tensor] = None,
                 rng_state: Optional[torch.Tensor] = None):
        count = len(params)
        if count == 0:
            raise ValueError("no parameters")
        for name, seq in (("grads", grads), ("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs),
                          ("exp_avg_scales", exp_avg_scales),
                          ("exp_avg_sq_scales", exp_avg_sq_scales), ("copies", copies),
                          ("weight_decays", weight_decays), ("offsets", offsets)):
            if seq is not None and len(seq) != count:
                raise ValueError(f"{name}: {len(seq)} entries for {count} parameters")
        self.device = params[0].device
        self.param_dtype, self.grad_dtype = params[0].dtype, grads[0].dtype
        self.eight = exp_avgs[0].dtype == torch.uint8
        if self.param_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"params: unexpected type {self.param_dtype}")
        if self.grad_dtype not in _DTYPES:
            raise ValueError(f"grads: unexpected type {self.grad_dtype}")
        if copies is not None and self.param_dtype != torch.float32:
            raise ValueError("copies are for float32 parameters")
        if self.eight and (exp_avg_scales is None or exp_avg_sq_scales is None
                           or rng_state is None):
            raise ValueError("8-bit moments need their scales and rng_state")
        if rng_state is not None and (rng_state.numel() != 2 or rng_state.dtype != torch.int64
                                      or not rng_state.is_contiguous()
                                      or rng_state.device != self.device):
            raise ValueError("rng_state: expected contiguous int64 {seed, offset} on the "
                             "parameters' device")
        if offsets is not None:
            offsets = [int(x) for x in offsets]
            if any(x < 0 or x >= 2 ** 62 or (self.eight and x % STATE_BLOCK) for x in offsets):
                raise ValueError(f"offsets: expected multiples of {STATE_BLOCK} from 0 on")
        self._table = load_binding().adamw_table(
            params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales if self.eight else None,
            exp_avg_sq_scales if self.eight else None, copies,
            None if weight_decays is None else [float(d) for d in weight_decays],
            offsets, amax_out, rng_state)
        self.count = count

    def step(self, step: int, *, lr: float, beta1: float = 0.9, beta2: float = 0.95,
             eps: float = 1e-8, grad_scale: Optional[torch.Tensor] = None,
             scalars: Optional[torch.Tensor] = None,
             grads: Optional[Sequence[torch.Tensor]] = None) -> None:
        """One step (`step` counts from 1) on the current stream.  `grads` take the
        place of the gradients listed so far (same sizes and type).  grad_scale
        (one float32 on the device) multiplies the gradients; scalars (three
        float32 on the device: lr, 1 - beta1^step, 1 - beta2^step) take the
        place of lr and step in a captured step."""
        _result("nvfp4_adamw_step", load_binding().adamw_step(
            self._table, lr, beta1, beta2, eps, step, grad_scale, scalars, grads))


def adamw_unpack_state(codes: torch.Tensor, scales: torch.Tensor, moment: str,
                       out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an 8-bit moment ("exp_avg" or "exp_avg_sq"), for a
    checkpoint in floating point or for inspection."""
    if out_dtype not in (_F32, torch.bfloat16):
        raise ValueError(f"unexpected out_dtype {out_dtype}")
    if moment not in ops.MOMENTS:
        raise ValueError(f"unknown moment {moment!r}: one of {', '.join(ops.MOMENTS)}")
    return _result("nvfp4_adamw_unpack_state", load_binding().adamw_unpack_state(
        codes, scales, ops.MOMENTS[moment], _DTYPES[out_dtype]))[0]
