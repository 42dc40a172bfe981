"""Dropout of activations."""
import ctypes as C
from typing import Optional, Union

import torch

from .._cabi import lib, torch_calls
from ._operands import DTYPES, Matrix, check_rows, drop_params, launch, like


def dropout(x_input: torch.Tensor, p: float, seed: int, call: Union[int, torch.Tensor] = 0, base: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, non_blocking: bool = False) -> torch.Tensor:
    """``base + drop(x_input)``: every element is dropped with probability ``p`` and scaled by ``1 / (1 - p)`` otherwise.

    The mask is a function of ``(seed, call, row, column)`` alone (Philox4x32-10, rpu_amd.h has its definition) and is not
    stored: the backward pass is the same call on the gradient.  ``call`` is a number of its own for every mask that is drawn
    with one seed, or an int64 tensor of one value on the GPU, read when the kernel runs, so that a captured step draws new
    masks in every replay.  Dropped elements count as zero also where they are infinite or NaN.  ``out`` may be ``x_input``
    or ``base``."""
    done = torch_calls().dropout(x_input, p, seed, call, base, out, non_blocking)
    if done is not None:
        return done
    x = Matrix(check_rows(x_input, "x_input"), "x_input")
    add = None if base is None else like(base, x_input, x_input.shape, "base")
    params = drop_params(p, seed, call, x_input.device)
    if out is None:
        out = torch.empty(x_input.shape, dtype=x_input.dtype, device=x_input.device)
    y = like(out, x_input, x_input.shape, "out", written=True)
    launch(x_input.device, non_blocking,
           lambda device, stream: lib().rpu_dropout(x.ptr, x.ld, add.ptr if add else None, add.ld if add else 0, y.ptr, y.ld,
                                                    DTYPES[x_input.dtype], x.rows, x.cols, C.byref(params), device, stream))
    return out
