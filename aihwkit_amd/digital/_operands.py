"""Operands of the digital operators: checks, and how a tensor is handed to the C entry points."""
import ctypes as C

import torch

from .._cabi import DropoutParams

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # enum rpu_dtype


def check_rows(tensor, what: str) -> torch.Tensor:
    """A GPU tensor of one of the three types with at least one dimension and one column."""
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if tensor.dtype not in DTYPES:
        raise RuntimeError(f"{what} must be a float32, float16 or bfloat16 tensor")
    if not tensor.is_cuda:
        raise RuntimeError(f"{what} must be a CUDA tensor")
    if tensor.dim() < 1 or tensor.size(-1) < 1:
        raise RuntimeError(f"{what} must have at least one column")
    return tensor


def _in_rows(tensor: torch.Tensor) -> bool:
    if tensor.is_contiguous():
        return True
    return tensor.dim() == 2 and (tensor.size(1) == 1 or tensor.stride(1) == 1) and \
        (tensor.size(0) < 2 or tensor.stride(0) >= tensor.size(1))


class Matrix:
    """Rows of a tensor: the tensor (a copy where its layout is not one of rows) and the distance of its rows."""

    __slots__ = ("tensor", "rows", "cols", "ld")

    def __init__(self, tensor: torch.Tensor, what: str, written: bool = False):
        if not _in_rows(tensor):
            if written:
                raise RuntimeError(f"{what} must be contiguous or a matrix with unit column stride")
            tensor = tensor.contiguous()
        self.tensor = tensor
        self.cols = tensor.size(-1)
        self.rows = tensor.numel() // self.cols
        self.ld = tensor.stride(0) if tensor.dim() == 2 and tensor.size(0) > 1 else self.cols

    @property
    def ptr(self):
        return self.tensor.data_ptr()


def like(tensor, other: torch.Tensor, shape, what: str, written: bool = False) -> Matrix:
    """An operand beside ``other``: the same type and GPU, and the shape it must have."""
    check_rows(tensor, what)
    if tensor.dtype != other.dtype:
        raise RuntimeError(f"{what} must be of type {other.dtype}")
    if tensor.device != other.device:
        raise RuntimeError(f"{what} must be on {other.device}")
    if tuple(tensor.shape) != tuple(shape):
        raise RuntimeError(f"Invalid {what} dimensions: expected {list(shape)}, got {list(tensor.shape)}")
    return Matrix(tensor, what, written)


def vector(tensor, other: torch.Tensor, count: int, dtypes, what: str):
    """A dense vector of ``count`` values beside ``other`` (None stays None)."""
    if tensor is None:
        return None
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if tensor.dtype not in dtypes:
        raise RuntimeError(f"{what} must be of type {' or '.join(str(d) for d in dtypes)}")
    if tensor.device != other.device:
        raise RuntimeError(f"{what} must be on {other.device}")
    if tensor.numel() != count:
        raise RuntimeError(f"Invalid {what} dimensions: expected {count} values, got {tensor.numel()}")
    return tensor.contiguous()


def drop_params(p: float, seed: int, call, device: torch.device) -> DropoutParams:
    """``call``: a number of its own for every mask drawn with one seed, or a tensor of one int64 on the GPU that is read when
    the kernel runs."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError("The dropout probability must be in [0, 1].")
    if not 0 <= int(seed) < 1 << 64:
        raise RuntimeError("The seed must be in 0 .. 2^64 - 1.")
    params = DropoutParams(p=p, seed=int(seed))
    if isinstance(call, torch.Tensor):
        if call.dtype != torch.int64 or call.numel() != 1 or call.device != device:
            raise RuntimeError(f"The call must be a number or one int64 on {device}")
        params.call_dev = call.data_ptr()
    else:
        if not 0 <= int(call) < 1 << 32:
            raise RuntimeError("The call must be in 0 .. 2^32 - 1.")
        params.call = int(call)
    return params


def launch(device: torch.device, non_blocking: bool, call) -> None:
    """``call(device_id, stream)`` on the current stream of the device."""
    from .._cabi import check

    stream = torch.cuda.current_stream(device)
    check(call(device.index, C.c_void_p(stream.cuda_stream)))
    if not non_blocking:
        stream.synchronize()
