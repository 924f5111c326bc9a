"""The operators of a training step around the NVFP4 cast, on torch tensors:
products of NVFP4 operands, layer norm forward and backward, AdamW.

Each function checks its tensors, allocates its outputs and any scratch with
torch (so both belong to the stream, and inside a capture to the graph), and
launches on the current stream of the tensors' device.  Bad arguments raise
ValueError here or NVFP4Error from the library.  The pointer-level forms, with
explicit streams and workspaces, are in ops."""
from __future__ import annotations

from itertools import accumulate
from typing import Optional, Sequence

import torch

from . import ops
from ._native import AdamWTensor, check, load

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32 = torch.float32
STATE_BLOCK = 128   # elements that share one scale byte of an 8-bit state

# A small product or norm takes a few microseconds on the device, so these
# wrappers look at each tensor once and call the library without the layers of
# the pointer-level forms; the stream is asked for as an address (a Stream
# object costs more than a launch).
_raw_stream = torch._C._cuda_getCurrentRawStream


def _device(x) -> int:
    """Index of a CUDA tensor's device."""
    d = x.get_device() if isinstance(x, torch.Tensor) else -1
    if d < 0:
        raise ValueError("expected a CUDA tensor")
    return d


def _call(device: int, name: str, *args) -> None:
    """A library call on the device's current stream (the last argument of every
    entry point)."""
    fn = getattr(load(), name)
    if device == torch.cuda.current_device():
        status = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(device))
    if status:
        check(name, status)


def _rows(t: torch.Tensor, m: int, n: int, dtype, device: int, name: str) -> int:
    """Row stride of an m x n tensor with unit inner stride."""
    if t.dtype != dtype or t.dim() != 2 or tuple(t.shape) != (m, n):
        raise ValueError(f"{name}: expected {(m, n)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name}: not on cuda:{device}")
    if t.is_contiguous():
        return n
    if n > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the inner stride must be 1")
    # A single row has no row stride to speak of.
    return t.stride(0) if m > 1 else max(t.stride(0), n)


def _vector(t: torch.Tensor, n: int, device: int, name: str) -> int:
    """Address of n contiguous values."""
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name}: expected {n} contiguous values on cuda:{device}, got "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _words(t: Optional[torch.Tensor], n: int, device: int, name: str) -> Optional[int]:
    """Address of n float32 on the device, or None."""
    if t is None:
        return None
    if t.numel() != n or t.dtype != _F32 or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name}: expected {n} float32 on cuda:{device}")
    return t.data_ptr()


def _operand(codes: torch.Tensor, scales: torch.Tensor, amax: torch.Tensor, device: int,
             name: str):
    if (codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.is_contiguous()
            or codes.get_device() != device):
        raise ValueError(f"{name}: codes are a contiguous 2-D uint8 tensor on cuda:{device}")
    rows, half = codes.shape
    if half % 16:
        raise ValueError(f"{name}: k must be a multiple of 32, got {2 * half}")
    if (scales.element_size() != 1 or tuple(scales.shape) != (rows, half // 8)
            or not scales.is_contiguous() or scales.get_device() != device):
        raise ValueError(f"{name}: scales are contiguous bytes of shape {(rows, half // 8)} "
                         f"on cuda:{device}")
    return rows, 2 * half, _words(amax, 1, device, f"{name}: amax")


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
    device = _device(a)
    m, k, pa = _operand(a, a_scales, a_amax, device, "a")
    n, kb, pb = _operand(b, b_scales, b_amax, device, "b")
    if k != kb:
        raise ValueError(f"a and b differ in k: {k} and {kb}")
    act = ops._activation(activation)
    if out is None:
        code = _DTYPES.get(out_dtype)
        if code is None:
            raise ValueError(f"unexpected out_dtype {out_dtype}")
        out = a.new_empty((m, n), dtype=out_dtype)
        ldd = n
    else:
        out_dtype = out.dtype
        code = _DTYPES.get(out_dtype)
        if code is None:
            raise ValueError(f"out: unexpected type {out_dtype}")
        ldd = _rows(out, m, n, out_dtype, device, "out")
    bias_ptr, bias_code = None, 0
    if bias is not None:
        bias_code = _DTYPES.get(bias.dtype)
        if bias_code is None:
            raise ValueError(f"bias: unexpected type {bias.dtype}")
        bias_ptr = _vector(bias, n, device, "bias")
    res_ptr, ldr = None, n
    if residual is not None:
        ldr = _rows(residual, m, n, out_dtype, device, "residual")
        res_ptr = residual.data_ptr()
    amax_ptr = _words(amax_out, 1, device, "amax_out")
    aux = a.new_empty((m, n), dtype=out_dtype) if with_aux else None
    nbytes = load().nvfp4_gemm_workspace_bytes(m, n, k)
    ws = a.new_empty(nbytes) if nbytes else None
    _call(device, "nvfp4_gemm", m, n, k, a.data_ptr(), a_scales.data_ptr(), pa, b.data_ptr(),
          b_scales.data_ptr(), pb, out.data_ptr(), ldd, code, bias_ptr, bias_code, res_ptr, ldr,
          act, aux.data_ptr() if with_aux else None, n, amax_ptr,
          ws.data_ptr() if nbytes else None, nbytes, 0)
    return out, aux


def matmul_nvfp4_dact(a: torch.Tensor, a_scales: torch.Tensor, a_amax: torch.Tensor,
                      b: torch.Tensor, b_scales: torch.Tensor, b_amax: torch.Tensor,
                      aux: torch.Tensor, *, activation: str, with_dbias: bool = False,
                      amax_out: Optional[torch.Tensor] = None):
    """(A B^T) act'(aux), of aux's type, and its column sums in fp32 (the bias
    gradient) or None."""
    device = _device(a)
    m, k, pa = _operand(a, a_scales, a_amax, device, "a")
    n, kb, pb = _operand(b, b_scales, b_amax, device, "b")
    if k != kb:
        raise ValueError(f"a and b differ in k: {k} and {kb}")
    act = ops._activation(activation)
    dtype = aux.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"aux: unexpected type {dtype}")
    ldaux = _rows(aux, m, n, dtype, device, "aux")
    amax_ptr = _words(amax_out, 1, device, "amax_out")
    d = a.new_empty((m, n), dtype=dtype)
    dbias = a.new_empty(n, dtype=_F32) if with_dbias else None
    lib = load()
    nbytes = (lib.nvfp4_gemm_dact_workspace_bytes if with_dbias
              else lib.nvfp4_gemm_workspace_bytes)(m, n, k)
    ws = a.new_empty(nbytes) if nbytes else None
    _call(device, "nvfp4_gemm_dact", m, n, k, a.data_ptr(), a_scales.data_ptr(), pa, b.data_ptr(),
          b_scales.data_ptr(), pb, aux.data_ptr(), ldaux, act, d.data_ptr(), n, code,
          dbias.data_ptr() if with_dbias else None, amax_ptr, ws.data_ptr() if nbytes else None,
          nbytes, 0)
    return d, dbias


def _norm(x: torch.Tensor, gamma: torch.Tensor, device: int):
    """(rows, cols, codes of both types, row stride, address of gamma)."""
    dtype = x.dtype
    code, weight = _DTYPES.get(dtype), _DTYPES.get(gamma.dtype)
    if x.dim() != 2 or code is None:
        raise ValueError("x: expected a 2-D float32, bfloat16 or float16 tensor")
    if weight is None or weight not in (0, code):
        raise ValueError(f"gamma: expected {dtype} or float32, got {gamma.dtype}")
    rows, cols = x.shape
    return rows, cols, code, weight, _rows(x, rows, cols, dtype, device, "x"), _vector(
        gamma, cols, device, "gamma")


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor] = None,
              eps: float = 1e-5, *, amax_out: Optional[torch.Tensor] = None):
    """Layer norm over the last dimension of a 2-D tensor.  Returns (y, mean,
    rstd); `amax_out` (one float32) receives max |y| for the cast of y."""
    device = _device(x)
    rows, cols, code, weight, ldx, gamma_ptr = _norm(x, gamma, device)
    beta_ptr = None
    if beta is not None:
        if beta.dtype != gamma.dtype:
            raise ValueError(f"beta: expected {gamma.dtype}, got {beta.dtype}")
        beta_ptr = _vector(beta, cols, device, "beta")
    amax_ptr = _words(amax_out, 1, device, "amax_out")
    y = x.new_empty((rows, cols))
    mean, rstd = x.new_empty(rows, dtype=_F32), x.new_empty(rows, dtype=_F32)
    _call(device, "nvfp4_layernorm_fwd", rows, cols, x.data_ptr(), ldx, gamma_ptr, beta_ptr, code,
          weight, eps, y.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr(), amax_ptr)
    return y, mean, rstd


def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       gamma: torch.Tensor, *, residual: Optional[torch.Tensor] = None):
    """Gradients (dx, dgamma, dbeta) of layernorm; `residual` is added to dx
    (the gradient that reaches x past the norm).  dgamma and dbeta have
    gamma's type."""
    device = _device(x)
    rows, cols, code, weight, ldx, gamma_ptr = _norm(x, gamma, device)
    lddy = _rows(dy, rows, cols, x.dtype, device, "dy")
    res_ptr, ldr = None, cols
    if residual is not None:
        ldr = _rows(residual, rows, cols, x.dtype, device, "residual")
        res_ptr = residual.data_ptr()
    mean_ptr, rstd_ptr = _words(mean, rows, device, "mean"), _words(rstd, rows, device, "rstd")
    dx = x.new_empty((rows, cols))
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
    nbytes = load().nvfp4_layernorm_bwd_workspace_bytes(rows, cols)
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _call(device, "nvfp4_layernorm_bwd", rows, cols, dy.data_ptr(), lddy, x.data_ptr(), ldx,
          mean_ptr, rstd_ptr, gamma_ptr, res_ptr, ldr, code, weight, dx.data_ptr(), cols,
          dgamma.data_ptr(), dbeta.data_ptr(), ws.data_ptr(), nbytes)
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
        self._device = _device(params[0])
        amax_ptr = _words(amax_out, count, self._device, "amax_out")
        state = torch.uint8 if self.eight else torch.float32

        # The tensors are held as long as their addresses are.
        self._keep = [t for t in (amax_out, rng_state) if t is not None]
        sizes = [p.numel() for p in params]
        blocks = [-(-n // STATE_BLOCK) for n in sizes]

        def take(seq, sizes, dtype, name):
            """The addresses of contiguous tensors of these sizes."""
            if seq is None:
                return [0] * count
            for i, (t, n) in enumerate(zip(seq, sizes)):
                if (t.get_device() != self._device or t.dtype != dtype or t.numel() != n
                        or not t.is_contiguous()):
                    raise ValueError(f"{name}[{i}]: expected {n} contiguous {dtype} on "
                                     f"{self.device}")
            self._keep.extend(seq)
            return [t.data_ptr() for t in seq]

        if offsets is None:
            offsets = [0, *accumulate(b * STATE_BLOCK for b in blocks)][:count]
        fields = (take(params, sizes, self.param_dtype, "params"),
                  take(grads, sizes, self.grad_dtype, "grads"),
                  take(exp_avgs, sizes, state, "exp_avgs"),
                  take(exp_avg_sqs, sizes, state, "exp_avg_sqs"),
                  take(exp_avg_scales if self.eight else None, blocks, torch.uint8,
                       "exp_avg_scales"),
                  take(exp_avg_sq_scales if self.eight else None, blocks, torch.uint8,
                       "exp_avg_sq_scales"),
                  take(copies, sizes, torch.bfloat16, "copies"), sizes, map(int, offsets),
                  map(float, weight_decays) if weight_decays is not None else [0.0] * count)
        own = [p for p, n in zip(fields[0], sizes) if n]
        if len(set(own)) != len(own):
            raise ValueError("params: the same tensor twice")
        self._table = (AdamWTensor * count)(*zip(*fields))
        self.count = count
        self._fixed = (self._table, count, _DTYPES[self.param_dtype], _DTYPES[self.grad_dtype],
                       int(self.eight))
        self._words = (amax_ptr, None if rng_state is None else rng_state.data_ptr())

    def step(self, step: int, *, lr: float, beta1: float = 0.9, beta2: float = 0.95,
             eps: float = 1e-8, grad_scale: Optional[torch.Tensor] = None,
             scalars: Optional[torch.Tensor] = None) -> None:
        """One step (`step` counts from 1) on the current stream.  grad_scale
        (one float32 on the device) multiplies the gradients; scalars (three
        float32 on the device: lr, 1 - beta1^step, 1 - beta2^step) take the
        place of lr and step in a captured step."""
        d = self._device
        _call(d, "nvfp4_adamw_step", *self._fixed, lr, beta1, beta2, eps, step,
              _words(grad_scale, 1, d, "grad_scale"), _words(scalars, 3, d, "scalars"),
              *self._words)


def adamw_unpack_state(codes: torch.Tensor, scales: torch.Tensor, moment: str,
                       out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an 8-bit moment ("exp_avg" or "exp_avg_sq"), for a
    checkpoint in floating point or for inspection."""
    device = _device(codes)
    n = codes.numel()
    if codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise ValueError("codes: expected contiguous uint8")
    if (scales.dtype != torch.uint8 or not scales.is_contiguous()
            or scales.numel() != -(-n // STATE_BLOCK) or scales.get_device() != device):
        raise ValueError(f"scales: expected {-(-n // STATE_BLOCK)} contiguous uint8 on "
                         f"cuda:{device}")
    if out_dtype not in (_F32, torch.bfloat16):
        raise ValueError(f"unexpected out_dtype {out_dtype}")
    if moment not in ops.MOMENTS:
        raise ValueError(f"unknown moment {moment!r}: one of {', '.join(ops.MOMENTS)}")
    out = codes.new_empty(codes.shape, dtype=out_dtype)
    _call(device, "nvfp4_adamw_unpack_state", codes.data_ptr(), scales.data_ptr(), n,
          ops.MOMENTS[moment], out.data_ptr(), _DTYPES[out_dtype])
    return out
