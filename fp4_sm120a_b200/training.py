"""The operators of a training step around the NVFP4 cast, on torch tensors:
products of NVFP4 operands, layer norm forward and backward, AdamW.

Each function checks its tensors, allocates its outputs and any scratch with
torch (so both belong to the stream, and inside a capture to the graph), and
launches on the current stream of the tensors' device.  Bad arguments raise
ValueError here or NVFP4Error from the library.  The pointer-level forms, with
explicit streams and workspaces, are in ops."""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence

import torch

from . import ops
from ._native import AdamWTensor

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
STATE_BLOCK = 128   # elements that share one scale byte of an 8-bit state


def _on_device_of_first(fn):
    """Runs fn with the device of its first argument current (its streams and
    allocations follow)."""
    @functools.wraps(fn)
    def run(x, *args, **kw):
        if not isinstance(x, torch.Tensor) or not x.is_cuda:
            raise ValueError("expected a CUDA tensor")
        if x.device.index == torch.cuda.current_device():
            return fn(x, *args, **kw)
        with torch.cuda.device(x.device):
            return fn(x, *args, **kw)
    return run


def _same_device(x: torch.Tensor, *others) -> None:
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError(f"tensors on {x.device} and {t.device}")


def _rows(t: torch.Tensor, shape, dtype, name: str) -> int:
    """Row stride of a 2-D tensor with unit inner stride."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name}: expected {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the inner stride must be 1")
    # A single row has no row stride to speak of.
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _vector(t: torch.Tensor, n: int, name: str, dtypes=None) -> None:
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous values, got {tuple(t.shape)}")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name}: unexpected type {t.dtype}")


def _word(t: Optional[torch.Tensor], name: str, n: int = 1) -> None:
    if t is not None and (t.numel() != n or t.dtype != torch.float32 or not t.is_contiguous()):
        raise ValueError(f"{name}: expected {n} float32")


def _operand(codes: torch.Tensor, scales: torch.Tensor, amax: torch.Tensor, name: str):
    if codes.dim() != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise ValueError(f"{name}: codes are a contiguous 2-D uint8 tensor")
    rows, half = codes.shape
    if half % 16:
        raise ValueError(f"{name}: k must be a multiple of 32, got {2 * half}")
    if scales.shape != (rows, half // 8) or scales.element_size() != 1 or not scales.is_contiguous():
        raise ValueError(f"{name}: scales are contiguous bytes of shape {(rows, half // 8)}")
    _word(amax, f"{name}: amax")
    return rows, 2 * half


def _operands(a, a_scales, a_amax, b, b_scales, b_amax):
    _same_device(a, a_scales, a_amax, b, b_scales, b_amax)
    m, k = _operand(a, a_scales, a_amax, "a")
    n, kb = _operand(b, b_scales, b_amax, "b")
    if k != kb:
        raise ValueError(f"a and b differ in k: {k} and {kb}")
    return m, n, k


@_on_device_of_first
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
    m, n, k = _operands(a, a_scales, a_amax, b, b_scales, b_amax)
    _same_device(a, bias, residual, out, amax_out)
    if out is None:
        if out_dtype not in _DTYPES:
            raise ValueError(f"unexpected out_dtype {out_dtype}")
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
        ldd = n
    else:
        if out.dtype not in _DTYPES:
            raise ValueError(f"out: unexpected type {out.dtype}")
        ldd = _rows(out, (m, n), out.dtype, "out")
    if bias is not None:
        _vector(bias, n, "bias", _DTYPES)
    ldr = n if residual is None else _rows(residual, (m, n), out.dtype, "residual")
    _word(amax_out, "amax_out")
    aux = torch.empty((m, n), dtype=out.dtype, device=a.device) if with_aux else None
    nbytes = ops.gemm_nvfp4_workspace_bytes(m, n, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device) if nbytes else None
    ops.gemm_nvfp4(m, n, k, a, a_scales, a_amax, b, b_scales, b_amax, out, ldd, out.dtype, bias,
                   torch.float32 if bias is None else bias.dtype, residual, ldr, activation, aux,
                   n, amax_out, ws, nbytes)
    return out, aux


@_on_device_of_first
def matmul_nvfp4_dact(a: torch.Tensor, a_scales: torch.Tensor, a_amax: torch.Tensor,
                      b: torch.Tensor, b_scales: torch.Tensor, b_amax: torch.Tensor,
                      aux: torch.Tensor, *, activation: str, with_dbias: bool = False,
                      amax_out: Optional[torch.Tensor] = None):
    """(A B^T) act'(aux), of aux's type, and its column sums in fp32 (the bias
    gradient) or None."""
    m, n, k = _operands(a, a_scales, a_amax, b, b_scales, b_amax)
    _same_device(a, aux, amax_out)
    if aux.dtype not in _DTYPES:
        raise ValueError(f"aux: unexpected type {aux.dtype}")
    ldaux = _rows(aux, (m, n), aux.dtype, "aux")
    _word(amax_out, "amax_out")
    d = torch.empty((m, n), dtype=aux.dtype, device=a.device)
    dbias = None
    if with_dbias:
        dbias = torch.empty(n, dtype=torch.float32, device=a.device)
        nbytes = ops.gemm_nvfp4_dact_workspace_bytes(m, n, k)
    else:
        nbytes = ops.gemm_nvfp4_workspace_bytes(m, n, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device) if nbytes else None
    ops.gemm_nvfp4_dact(m, n, k, a, a_scales, a_amax, b, b_scales, b_amax, aux, ldaux, activation,
                        d, n, d.dtype, dbias, amax_out, ws, nbytes)
    return d, dbias


def _norm_shapes(x: torch.Tensor, gamma: torch.Tensor):
    if x.dim() != 2 or x.dtype not in _DTYPES:
        raise ValueError("x: expected a 2-D float32, bfloat16 or float16 tensor")
    rows, cols = x.shape
    _vector(gamma, cols, "gamma", (x.dtype, torch.float32))
    return rows, cols


@_on_device_of_first
def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor] = None,
              eps: float = 1e-5, *, amax_out: Optional[torch.Tensor] = None):
    """Layer norm over the last dimension of a 2-D tensor.  Returns (y, mean,
    rstd); `amax_out` (one float32) receives max |y| for the cast of y."""
    rows, cols = _norm_shapes(x, gamma)
    _same_device(x, gamma, beta, amax_out)
    ldx = _rows(x, x.shape, x.dtype, "x")
    if beta is not None:
        _vector(beta, cols, "beta", (gamma.dtype,))
    _word(amax_out, "amax_out")
    y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    mean, rstd = stats[0], stats[1]
    ops.layernorm_fwd(rows, cols, x, ldx, gamma, beta, x.dtype, gamma.dtype, eps, y, cols, mean,
                      rstd, amax_out)
    return y, mean, rstd


@_on_device_of_first
def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       gamma: torch.Tensor, *, residual: Optional[torch.Tensor] = None):
    """Gradients (dx, dgamma, dbeta) of layernorm; `residual` is added to dx
    (the gradient that reaches x past the norm).  dgamma and dbeta have
    gamma's type."""
    rows, cols = _norm_shapes(x, gamma)
    _same_device(x, dy, mean, rstd, gamma, residual)
    ldx = _rows(x, x.shape, x.dtype, "x")
    lddy = _rows(dy, x.shape, x.dtype, "dy")
    ldr = cols if residual is None else _rows(residual, x.shape, x.dtype, "residual")
    _vector(mean, rows, "mean", (torch.float32,))
    _vector(rstd, rows, "rstd", (torch.float32,))
    dx = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    grads = torch.empty((2, cols), dtype=gamma.dtype, device=x.device)
    dgamma, dbeta = grads[0], grads[1]
    nbytes = ops.layernorm_bwd_workspace_bytes(rows, cols)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    ops.layernorm_bwd(rows, cols, dy, lddy, x, ldx, mean, rstd, gamma, residual, ldr, x.dtype,
                      gamma.dtype, dx, cols, dgamma, dbeta, ws, nbytes)
    return dx, dgamma, dbeta


class AdamW:
    """The tensors of an AdamW step, described once for any number of steps.

    params (float32 or bfloat16), grads, exp_avgs and exp_avg_sqs are lists of
    contiguous tensors, one entry per parameter.  float32 moments are held as
    they are; uint8 moments need the scale tensors (ceil(n / 128) uint8 each),
    rng_state (int64 {seed, offset} on the device) and, for each tensor, the
    position of its first element in the numbering that the random bits go by
    (`offsets`, multiples of 128; default: one tensor behind the other).
    `copies` (bfloat16) receive the rounded new parameters, `amax_out` (one
    float32 per tensor) their amax.  All memory is the caller's."""

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
                                      or rng_state.device != self.device):
            raise ValueError("rng_state: expected int64 {seed, offset} on the parameters' device")
        _word(amax_out, "amax_out", count)
        if amax_out is not None and amax_out.device != self.device:
            raise ValueError("amax_out: not on the parameters' device")
        state = torch.uint8 if self.eight else torch.float32

        def take(seq, i, n, dtype, name):
            if seq is None:
                return 0
            t = seq[i]
            if (not t.is_cuda or t.device != self.device or t.dtype != dtype or t.numel() != n
                    or not t.is_contiguous()):
                raise ValueError(f"{name}[{i}]: expected {n} contiguous {dtype} on {self.device}")
            self._keep.append(t)
            return t.data_ptr()

        # The tensors are held as long as their addresses are.
        self._keep = [t for t in (amax_out, rng_state) if t is not None]
        self._table = (AdamWTensor * count)()
        at = 0
        for i, d in enumerate(self._table):
            n = params[i].numel()
            d.param = take(params, i, n, self.param_dtype, "params")
            d.grad = take(grads, i, n, self.grad_dtype, "grads")
            d.exp_avg = take(exp_avgs, i, n, state, "exp_avgs")
            d.exp_avg_sq = take(exp_avg_sqs, i, n, state, "exp_avg_sqs")
            if self.eight:
                blocks = -(-n // STATE_BLOCK)
                d.exp_avg_scale = take(exp_avg_scales, i, blocks, torch.uint8, "exp_avg_scales")
                d.exp_avg_sq_scale = take(exp_avg_sq_scales, i, blocks, torch.uint8,
                                          "exp_avg_sq_scales")
            d.copy = take(copies, i, n, torch.bfloat16, "copies")
            d.n = n
            d.offset = at if offsets is None else int(offsets[i])
            at += -(-n // STATE_BLOCK) * STATE_BLOCK
            d.weight_decay = 0.0 if weight_decays is None else float(weight_decays[i])
        self.count, self.amax_out, self.rng_state = count, amax_out, rng_state

    def step(self, step: int, *, lr: float, beta1: float = 0.9, beta2: float = 0.95,
             eps: float = 1e-8, grad_scale: Optional[torch.Tensor] = None,
             scalars: Optional[torch.Tensor] = None) -> None:
        """One step (`step` counts from 1) on the current stream.  grad_scale
        (one float32 on the device) multiplies the gradients; scalars (three
        float32 on the device: lr, 1 - beta1^step, 1 - beta2^step) take the
        place of lr and step in a captured step."""
        for name, t, n in (("grad_scale", grad_scale, 1), ("scalars", scalars, 3)):
            _word(t, name, n)
            if t is not None and t.device != self.device:
                raise ValueError(f"{name}: not on {self.device}")
        with torch.cuda.device(self.device):
            ops.adamw_step(self._table, self.count, self.param_dtype, self.grad_dtype,
                           int(self.eight), lr, beta1, beta2, eps, step, grad_scale, scalars,
                           self.amax_out, self.rng_state)


@_on_device_of_first
def adamw_unpack_state(codes: torch.Tensor, scales: torch.Tensor, moment: str,
                       out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an 8-bit moment ("exp_avg" or "exp_avg_sq"), for a
    checkpoint in floating point or for inspection."""
    n = codes.numel()
    _same_device(codes, scales)
    if codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise ValueError("codes: expected contiguous uint8")
    if (scales.dtype != torch.uint8 or not scales.is_contiguous()
            or scales.numel() != -(-n // STATE_BLOCK)):
        raise ValueError(f"scales: expected {-(-n // STATE_BLOCK)} contiguous uint8")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"unexpected out_dtype {out_dtype}")
    out = torch.empty(codes.shape, dtype=out_dtype, device=codes.device)
    ops.adamw_unpack_state(codes, scales, n, moment, out, out_dtype)
    return out
