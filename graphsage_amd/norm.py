"""Layer norm and dropout between the layers of a deeper encoder, and the two joined with a residual sum.

``layer_norm(x, weight, bias)``, ``dropout(x, p)`` and ``dropout_add_layer_norm(x, residual, weight, bias, p)``
(``LayerNorm(residual + dropout(x))`` in one pass) on fp32, bf16 or fp16 tables: arithmetic in fp32, outputs
rounded once.  ``GraphSAGE(norm="layer")`` runs its hidden layers through them; the reference's experimental
``FlexibleGraphSAGE`` (src/model/graphsage.py:160-296) composes the same from nn.LayerNorm, nn.Dropout and a sum.

Dropout masks are those of the projection kernels: element ``i`` (row-major) is kept or not by a counter hash of
``(seed, i)`` alone (host mirror: :func:`graphsage_amd.rng.dropout_keep_mask`), so a mask is never stored and the
backward draws it again.  Of tables below 2^32 elements the seed's two 32-bit halves count by their xor alone: 2^32 masks
in all, seeds 1 and 2^32 the same one.  A dropped element gives exactly 0, forward and backward, whatever it holds.
``seed`` is an int, a one-element int64 tensor on the device (read when the kernel runs: a captured graph that
rewrites it draws other masks on each replay, where an int is frozen into the graph), or None: one draw from
torch's CPU generator.

Derivatives are reverse mode, once: forward mode raises ``NotImplementedError``, a second derivative ``RuntimeError``.
``torch.jit.trace`` records a call as a Python function (an int or drawn seed frozen into it).

A backward is captured into a graph like any other of torch's: with no eager graph of the same leaves alive, whose
gradient nodes torch would run on the stream they were made on.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_M64 = (1 << 64) - 1

Seed = Union[int, torch.Tensor, None]


def _table(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU (graphsage_amd has no CPU path)")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return t.contiguous()


def _like(t: torch.Tensor, x: torch.Tensor, name: str) -> torch.Tensor:
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must have the input's shape, type and device ({tuple(x.shape)}, {x.dtype}, {x.device}), "
                         f"got {tuple(t.shape)}, {t.dtype}, {t.device}")
    return t.contiguous()


def _affine(t: torch.Tensor, x: torch.Tensor, name: str) -> torch.Tensor:
    if t.device != x.device:
        raise ValueError(f"{name} must live on the input's device {x.device}, got {t.device}")
    if t.dim() != 1 or t.numel() != x.size(-1):
        raise ValueError(f"{name} must be [{x.size(-1)}], got {tuple(t.shape)}")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 or of the input's type {x.dtype}, got {t.dtype}")
    return t.contiguous()


def _rate(p: float) -> float:
    p = float(p)
    if not 0.0 <= p < 1.0 - 2.0 ** -25:           # (an fp32 number below 1)
        raise ValueError(f"dropout rate must be in [0, 1), got {p}")
    return p if p > 2.0 ** -150 else 0.0          # (what is 0 as an fp32 number drops nothing)


def _seed(seed: Seed, device: torch.device) -> Union[int, torch.Tensor]:
    if seed is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("dropout inside a graph capture needs a seed: a one-element int64 tensor on the device "
                               "that the graph rewrites (or an int, for the same mask on every replay)")
        # CPU generator: reproducible under torch.manual_seed, no device sync
        return int(torch.empty((), dtype=torch.int64).random_().item())
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a seed tensor must be one int64 element on {device}, got {seed.dtype} "
                             f"{tuple(seed.shape)} on {seed.device}")
        return seed
    return int(seed) & _M64


def _split(seed) -> Tuple[int, Optional[int]]:
    """(seed by value, seed's device pointer) for the C ABI."""
    return (0, seed.data_ptr()) if torch.is_tensor(seed) else (seed, None)


# ----------------------------------------------------------------------------------------------- raw ops
def _call(tag: str, device: torch.device, entry, *args) -> None:
    """``entry(*args, stream)`` on ``device``'s current stream.  Allocations belong to a device whichever is current;
    the launch does not."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(tag, device, entry, *args)
    if ops._timer is None:
        status = entry(*args, _lib.stream_handle())
    else:
        with ops._bracket(tag):
            status = entry(*args, _lib.stream_handle())
    if status:
        _lib.check(status, "gsage_" + tag)


def _dropout(x: torch.Tensor, p: float, seed) -> torch.Tensor:
    value, pointer = _split(seed)
    out = torch.empty_like(x)
    _call("dropout", x.device, _lib.load().gsage_dropout, x.data_ptr(), int(x.numel()), _DTYPES[x.dtype], p, value, pointer,
          out.data_ptr())
    return out


def layer_norm_fwd(x, residual, weight, bias, eps: float, p: float, seed, want_sum: bool, want_stats: bool):
    """gsage_layer_norm_fwd on contiguous operands -> (y, sum or None, [mean, rstd] as fp32 [2, M] or None)."""
    value, pointer = _split(seed)
    F = int(x.size(-1))           # (sizes are tensors while torch.jit.trace records)
    M = int(x.numel()) // F
    y = torch.empty_like(x)
    total = torch.empty_like(x) if want_sum else None
    stats = mean = rstd = None
    if want_stats:
        stats = torch.empty((2, M), dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * M
    code = _DTYPES[x.dtype]
    affine = weight if weight is not None else bias
    _call("layer_norm_fwd", x.device, _lib.load().gsage_layer_norm_fwd, x.data_ptr(), _lib.ptr(residual),
          _lib.ptr(weight), _lib.ptr(bias), M, F, code, code if affine is None else _DTYPES[affine.dtype], eps, p, value,
          pointer, y.data_ptr(), _lib.ptr(total), mean, rstd)
    return y, total, stats


def layer_norm_bwd(grad_y, grad_sum, x, residual, weight, stats, p: float, seed, need, wdtype: torch.dtype):
    """gsage_layer_norm_bwd -> (grad_x, grad_residual, grad_weight, grad_bias), None where ``need`` is false."""
    lib = _lib.load()
    value, pointer = _split(seed)
    dev, code = x.device, _DTYPES[x.dtype]
    F = int(x.size(-1))
    M = int(x.numel()) // F
    gx = torch.empty_like(x) if need[0] else None
    gres = torch.empty_like(x) if need[1] else None
    gw = torch.empty(F, dtype=wdtype, device=dev) if need[2] else None
    gb = torch.empty(F, dtype=wdtype, device=dev) if need[3] else None
    ws, ws_bytes = None, 0
    if need[2] or need[3]:
        joined = residual is not None or grad_sum is not None or p > 0.0
        ws_bytes = (lib.gsage_layer_norm_bwd_joined_workspace_bytes if joined
                    else lib.gsage_layer_norm_bwd_workspace_bytes)(M, F, code)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    mean = stats.data_ptr()
    _call("layer_norm_bwd", dev, lib.gsage_layer_norm_bwd, grad_y.data_ptr(), _lib.ptr(grad_sum), x.data_ptr(),
          _lib.ptr(residual), _lib.ptr(weight), mean, mean + 4 * M, M, F, code, _DTYPES[wdtype], p, value, pointer,
          _lib.ptr(gx), _lib.ptr(gres), _lib.ptr(gw), _lib.ptr(gb), _lib.ptr(ws), ws_bytes)
    return gx, gres, gw, gb


# ----------------------------------------------------------------------------------------- autograd glue
def _keep_seed(ctx, seed, *tensors) -> None:
    # a seed tensor is saved like any operand: rewriting it between forward and backward is an error,
    # not another mask
    if torch.is_tensor(seed):
        ctx.seed = None
        ctx.save_for_backward(*tensors, seed)
    else:
        ctx.seed = seed
        ctx.save_for_backward(*tensors)


def _once(backward):
    """A backward of raw kernels: not differentiable again.  torch's own wrapper for that only where a graph of the
    backward is wanted (it costs as much as a launch)."""
    refusing = once_differentiable(backward)

    def call(ctx, *grads):
        return refusing(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call


def _watched() -> bool:
    """Whether torch has to see the call though no gradient is wanted: a launch on raw pointers would give an output
    without a tangent in forward mode (through the function it raises) and leave the kernel out of a trace."""
    return forward_ad._current_level >= 0 or torch._C._is_tracing()


class DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p: float, seed):
        ctx.p = p
        _keep_seed(ctx, seed)
        return _dropout(x, p, seed)

    @staticmethod
    @_once
    def backward(ctx, grad_out):
        seed = ctx.seed if ctx.seed is not None else ctx.saved_tensors[0]
        return _dropout(grad_out.contiguous(), ctx.p, seed), None, None


class LayerNormFunction(torch.autograd.Function):
    """y (and z with ``return_sum``) = LayerNorm(z), z = residual + dropout(x)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps: float, p: float, seed, return_sum: bool):
        y, total, stats = layer_norm_fwd(x, residual, weight, bias, eps, p, seed, return_sum, True)
        ctx.p = p
        affine = weight if weight is not None else bias
        ctx.wdtype = torch.float32 if affine is None else affine.dtype
        _keep_seed(ctx, seed, x, residual, weight, stats)
        ctx.set_materialize_grads(False)
        return (y, total) if return_sum else y

    @staticmethod
    @_once
    def backward(ctx, grad_y, grad_sum=None):
        if grad_y is None and grad_sum is None:
            return (None,) * 8
        saved = ctx.saved_tensors
        x, residual, weight, stats = saved[:4]
        grad_y = torch.zeros_like(x) if grad_y is None else grad_y.contiguous()
        if grad_sum is not None:
            grad_sum = grad_sum.contiguous()
        grads = layer_norm_bwd(grad_y, grad_sum, x, residual, weight, stats, ctx.p,
                               ctx.seed if ctx.seed is not None else saved[4], ctx.needs_input_grad, ctx.wdtype)
        return (*grads, None, None, None, None)


# ------------------------------------------------------------------------------------------- entry points
def dropout(x: torch.Tensor, p: float = 0.5, training: bool = True, seed: Seed = None) -> torch.Tensor:
    """``x_i / (1 - p)`` where element ``i`` is kept (probability ``1 - p``), else 0; ``x`` itself when not training
    or ``p`` is 0."""
    p = _rate(p)
    x = _table(x, "x")
    if not training or p == 0.0:
        return x
    seed = _seed(seed, x.device)
    if (torch.is_grad_enabled() and x.requires_grad) or _watched():
        return DropoutFunction.apply(x, p, seed)
    return _dropout(x, p, seed)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension; ``weight`` and ``bias`` are [F], float32 or of x's type."""
    return dropout_add_layer_norm(x, None, weight, bias, eps=eps)


def dropout_add_layer_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                           weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                           p: float = 0.0, eps: float = 1e-5, training: bool = True, seed: Seed = None,
                           return_sum: bool = False):
    """``layer_norm(z)`` of ``z = residual + dropout(x)`` in one pass; ``(layer_norm(z), z)`` with ``return_sum``.
    The norm is taken of z before it is rounded."""
    p, eps = _rate(p), float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    x = _table(x, "x")
    if x.dim() == 0 or x.size(-1) == 0:
        raise ValueError(f"layer norm needs at least one column, got x of shape {tuple(x.shape)}")
    if residual is not None:
        residual = _like(residual, x, "residual")
    if weight is not None:
        weight = _affine(weight, x, "weight")
    if bias is not None:
        bias = _affine(bias, x, "bias")
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not training:
        p = 0.0
    seed = _seed(seed, x.device) if p > 0.0 else 0
    if (torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad) or
                                     (weight is not None and weight.requires_grad) or
                                     (bias is not None and bias.requires_grad))) or _watched():
        return LayerNormFunction.apply(x, residual, weight, bias, eps, p, seed, return_sum)
    y, total, _ = layer_norm_fwd(x, residual, weight, bias, eps, p, seed, return_sum, False)
    return (y, total) if return_sum else y


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one dimension (its parameters, names and initialisation) on :func:`layer_norm`."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, **kw):
        super().__init__(normalized_shape, eps, elementwise_affine, **kw)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm covers the last dimension only, got {self.normalized_shape}")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.size(-1) != self.normalized_shape[0]:
            raise ValueError(f"x must have {self.normalized_shape[0]} columns, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
