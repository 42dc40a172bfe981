"""Layer norm of rows and its gradients."""
from typing import Optional, Tuple

import torch

from .._cabi import lib, torch_calls
from ._operands import DTYPES, Matrix, check_rows, launch, like, vector


def layer_norm(x_input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None,
               non_blocking: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)`` with ``y = (x - mean) rstd weight + bias`` and ``rstd = (mean((x - mean)^2) + eps)^-1/2`` of every
    row; ``mean`` and ``rstd`` are float32, one value a row, for the backward pass.  ``weight`` and ``bias`` are float32 or of
    the type of ``x_input``, both alike; ``out`` may be ``x_input``."""
    done = torch_calls().layer_norm(x_input, weight, bias, eps, out, non_blocking)
    if done is not None:
        return done
    x = Matrix(check_rows(x_input, "x_input"), "x_input")
    types = (torch.float32, x_input.dtype)
    w = vector(weight, x_input, x.cols, types, "weight")
    b = vector(bias, x_input, x.cols, types if w is None else (w.dtype,), "bias")
    given = w if w is not None else b
    if out is None:
        out = torch.empty(x_input.shape, dtype=x_input.dtype, device=x_input.device)
    y = like(out, x_input, x_input.shape, "out", written=True)
    mean, rstd = torch.empty((2, *x_input.shape[:-1]), dtype=torch.float32, device=x_input.device)
    launch(x_input.device, non_blocking,
           lambda device, stream: lib().rpu_layer_norm(
               x.ptr, x.ld, None if w is None else w.data_ptr(), None if b is None else b.data_ptr(),
               0 if given is None else DTYPES[given.dtype], y.ptr, y.ld, mean.data_ptr(), rstd.data_ptr(), DTYPES[x_input.dtype],
               x.rows, x.cols, float(eps), device, stream))
    return out, mean, rstd


def layer_norm_backward(d_input: torch.Tensor, x_input: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, base: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None, non_blocking: bool = False
                        ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(dx, dweight, dbias)`` from the gradient ``d_input`` of the output and what the forward pass took and left.

    ``base`` is added to ``dx``: the gradient that reaches ``x`` past the norm.  ``dweight`` and ``dbias`` have the type of
    ``weight`` and are None without it.  ``out`` (dx) may be ``d_input``, ``x_input`` or ``base``.  Sums over rows are added in
    an order that depends on the sizes alone."""
    done = torch_calls().layer_norm_backward(d_input, x_input, mean, rstd, weight, base, out, non_blocking)
    if done is not None:
        return done
    x = Matrix(check_rows(x_input, "x_input"), "x_input")
    d = like(d_input, x_input, x_input.shape, "d_input")
    mean = vector(mean, x_input, x.rows, (torch.float32,), "mean")
    rstd = vector(rstd, x_input, x.rows, (torch.float32,), "rstd")
    if mean is None or rstd is None:
        raise RuntimeError("The statistics of the forward pass are needed.")
    w = vector(weight, x_input, x.cols, (torch.float32, x_input.dtype), "weight")
    add = None if base is None else like(base, x_input, x_input.shape, "base")
    if out is None:
        out = torch.empty(x_input.shape, dtype=x_input.dtype, device=x_input.device)
    dx = like(out, x_input, x_input.shape, "out", written=True)
    dw = db = scratch = None
    scratch_bytes = 0
    if w is not None:
        dw, db = torch.empty_like(weight, memory_format=torch.contiguous_format), torch.empty_like(weight, memory_format=torch.contiguous_format)
        scratch_bytes = lib().rpu_layer_norm_backward_scratch(x.rows, x.cols)
        scratch = torch.empty(scratch_bytes // 4, dtype=torch.float32, device=x_input.device)

    def ptr(tensor):
        return None if tensor is None else tensor.data_ptr()

    launch(x_input.device, non_blocking,
           lambda device, stream: lib().rpu_layer_norm_backward(
               d.ptr, d.ld, x.ptr, x.ld, mean.data_ptr(), rstd.data_ptr(), ptr(w), 0 if w is None else DTYPES[w.dtype],
               add.ptr if add else None, add.ld if add else 0, dx.ptr, dx.ld, ptr(dw), ptr(db), DTYPES[x_input.dtype], x.rows,
               x.cols, ptr(scratch), scratch_bytes, device, stream))
    return out, dw, db
