"""Low-rank adapters of many requests beside one projection."""
import ctypes as C
from typing import Optional, Tuple, Union

import torch

from .._cabi import Adapters, check, lib, torch_calls
from ._operands import DTYPES, Matrix, check_rows, drop_params, launch, like

MOST_SIZE = 1 << 21   # inputs or outputs of an adapter, as the C entry points take them
FEW_ROWS = 64   # RPU_ADAPTER_FEW_ROWS: a forward call groups so many rows by itself


def _check_index(index: torch.Tensor) -> torch.Tensor:
    if not isinstance(index, torch.Tensor):
        raise TypeError("index must be a torch.Tensor")
    if index.dtype != torch.int32 or not index.is_cuda:
        raise RuntimeError("index must be an int32 CUDA tensor")
    return index.contiguous()


class AdapterRows:
    """Rows grouped by adapter, for any number of calls on as many rows: a step's layers share one.

    ``index``: int32 CUDA tensor, the adapter of every row; a row whose number is not in ``0 .. n_adapters - 1`` has none.  The
    grouping is made on the current stream when the object is, of the numbers that ``index`` holds then, and nothing waits for it on the
    host.  Calls on other streams wait for it on the GPU, and its memory is kept until they are done.  A capture cannot wait for what is
    not captured: by then the grouping has to be done (``torch.cuda.graph`` waits for the GPU before it begins), and the object lives
    as long as the graph.  Made within a capture, the grouping is done by each replay, and not before the first."""

    def __init__(self, index: torch.Tensor, n_adapters: int):
        index = _check_index(index)
        self.n_adapters, self.rows, self.device = int(n_adapters), index.numel(), index.device
        self._device = self.device.index
        self._stream = torch._C._cuda_getCurrentRawStream(self._device)
        self._plan = torch_calls().adapter_plan(index, self.n_adapters)
        if self._plan is not None:
            self._bytes = self._plan.numel()
            return
        self._bytes = 0
        if 1 <= self.n_adapters <= 65535:
            self._bytes = lib().rpu_adapter_plan_bytes(self.rows, self.n_adapters)
        if not self._bytes:
            raise RuntimeError("The number of adapters must be in 1 .. 65535, that of rows at most 2^28.")
        self._plan = torch.empty(self._bytes, dtype=torch.uint8, device=index.device)
        check(lib().rpu_adapter_plan(index.data_ptr(), self.rows, self.n_adapters, self._plan.data_ptr(), self._bytes,
                                     self._device, C.c_void_p(self._stream)))

    def _plan_here(self) -> torch.Tensor:
        """The plan, for work on the current stream: on another one than its own, after it has been made."""
        if torch._C._cuda_getCurrentRawStream(self._device) != self._stream:
            self._order_after(torch.cuda.current_stream(self.device))
        return self._plan

    def _order_after(self, here: torch.cuda.Stream) -> None:
        made = torch.cuda.ExternalStream(self._stream, device=self.device)

        def captured(stream):      # the default stream never is
            with torch.cuda.stream(stream):
                return stream.cuda_stream != 0 and torch.cuda.is_current_stream_capturing()

        if captured(made):
            if not captured(here):
                raise RuntimeError("The stream that the rows were grouped on is being captured, the current one is not.")
        elif captured(here):
            return                 # done by now, as the class's description asks for
        else:
            self._plan.record_stream(here)
        here.wait_stream(made)


class LowRankAdapters:
    """``n`` adapters of a projection: ``y = base + scale_i b_i (a_i drop(x))`` with ``i`` the adapter of the row.

    ``a`` [n, rank, in_size], ``b`` [n, out_size, rank] (float32, float16 or bfloat16) and ``scale`` [n] (float32; None: ones)
    are the caller's tensors, dense and on one GPU, and are used as they are at every call: an optimizer may write them, or they may be replaced
    by others of their shape.  Beside 16-bit rows the matrices are of the rows' type.  An adapter of a smaller rank than the
    others has zeros in the rest.  Infinities and NaN of a row stay with it, and in gradients with its adapter; beside 16-bit
    rows a product with an infinity may be NaN where the formula has an infinity."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: Optional[torch.Tensor] = None):
        for tensor, what in ((a, "a"), (b, "b")):
            check_rows(tensor, what)
            if tensor.dim() != 3:
                raise RuntimeError(f"{what} must have three dimensions")
        self.n_adapters, self.rank, self.in_size = a.shape
        self.out_size = b.size(1)
        if self.n_adapters < 1 or self.n_adapters > 65535:
            raise RuntimeError("The number of adapters must be in 1 .. 65535.")
        if self.rank < 1 or self.rank > 128:
            raise RuntimeError("The rank of the adapters must be in 1 .. 128.")
        if not 1 <= self.out_size <= MOST_SIZE or self.in_size > MOST_SIZE:
            raise RuntimeError("The sizes of the adapters must be in 1 .. 2^21.")
        self.a, self.b = a, b
        self._a_shape, self._b_shape = a.shape, torch.Size((self.n_adapters, self.out_size, self.rank))
        self.scale = torch.ones(self.n_adapters, dtype=torch.float32, device=a.device) if scale is None else scale
        self._operand(a)

    def _operand(self, x_input: torch.Tensor) -> Adapters:
        """The C structure of the tensors as they are now."""
        a, b, scale = self.a, self.b, self.scale
        if tuple(a.shape) != (self.n_adapters, self.rank, self.in_size) or not a.is_contiguous():
            raise RuntimeError("Invalid a: expected a dense [%d,%d,%d] tensor" % (self.n_adapters, self.rank, self.in_size))
        if tuple(b.shape) != (self.n_adapters, self.out_size, self.rank) or not b.is_contiguous():
            raise RuntimeError("Invalid b: expected a dense [%d,%d,%d] tensor" % (self.n_adapters, self.out_size, self.rank))
        if a.dtype not in DTYPES or a.dtype != b.dtype:
            raise RuntimeError("a and b must be of one type")
        if not isinstance(scale, torch.Tensor) or tuple(scale.shape) != (self.n_adapters,) or scale.dtype != torch.float32 \
                or not scale.is_contiguous():
            raise RuntimeError("Invalid scale: expected a dense float32 tensor of %d values" % self.n_adapters)
        if a.device != x_input.device or b.device != a.device or scale.device != a.device:
            raise RuntimeError(f"a, b, scale and the rows must be on one GPU, {x_input.device}")
        return Adapters(a_dev=a.data_ptr(), b_dev=b.data_ptr(), scale_dev=scale.data_ptr(), n=self.n_adapters,
                        in_size=self.in_size, out_size=self.out_size, rank=self.rank, w_dtype=DTYPES[a.dtype])

    @staticmethod
    def _checked_rows(tensor: torch.Tensor, size: int, what: str) -> torch.Tensor:
        check_rows(tensor, what)
        if tensor.size(-1) != size:
            raise RuntimeError(f"Invalid {what} dimensions: expected {size} columns, got {tensor.size(-1)}")
        return tensor

    def _rows(self, tensor: torch.Tensor, size: int, what: str) -> Matrix:
        return Matrix(self._checked_rows(tensor, size, what), what)

    def _chosen(self, rows: Union[torch.Tensor, AdapterRows], x_input: torch.Tensor):
        """(index, plan) as given, one of them None."""
        if isinstance(rows, AdapterRows):
            if rows.n_adapters != self.n_adapters:
                raise RuntimeError("The rows were grouped for %d adapters, not %d" % (rows.n_adapters, self.n_adapters))
            index, plan = None, rows
            count, device = rows.rows, rows.device
        else:
            index, plan = _check_index(rows), None
            count, device = index.numel(), index.device
        expected = x_input.numel() // x_input.size(-1)
        if count != expected:
            raise RuntimeError("Invalid index dimensions: expected %d rows, got %d" % (expected, count))
        if device != x_input.device:
            raise RuntimeError(f"The index must be on {x_input.device}")
        return index, plan

    def _grouped(self, rows: Union[torch.Tensor, AdapterRows], x: Matrix, few: int):
        """(index, plan) of a call: an index of more than ``few`` rows is grouped first."""
        index, plan = self._chosen(rows, x.tensor)
        if plan is None and index.numel() > few:
            plan = AdapterRows(index, self.n_adapters)
        return index, plan

    def check_forward(self, x_input: torch.Tensor, rows: Union[torch.Tensor, AdapterRows], out_size: int) -> None:
        """Raises what ``forward`` would raise for rows beside a projection of ``out_size`` outputs, without computing anything: for a
        projection that is not to run in vain."""
        self._checked_rows(x_input, self.in_size, "x_input")
        self._operand(x_input)
        if x_input.dtype != torch.float32 and x_input.dtype != self.a.dtype:
            raise RuntimeError("Adapters beside 16-bit rows must be of the rows' type.")
        if out_size != self.out_size:
            raise RuntimeError("The adapters have %d outputs, the projection %d" % (self.out_size, out_size))
        self._chosen(rows, x_input)

    def _native(self, rows, x_input):
        """(index, plan) for the native calls, (None, None) for what the general path has to look at."""
        a, b = self.a, self.b
        if not isinstance(a, torch.Tensor) or not isinstance(b, torch.Tensor) or not isinstance(x_input, torch.Tensor) or \
                a.shape != self._a_shape or b.shape != self._b_shape:
            return None, None
        if not isinstance(rows, AdapterRows):
            return rows, None
        if rows.n_adapters != self.n_adapters or rows.rows * self.in_size != x_input.numel():
            return None, None
        return None, rows._plan_here()

    def forward(self, x_input: torch.Tensor, rows: Union[torch.Tensor, AdapterRows], base: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None, return_hidden: bool = False, p: float = 0.0, seed: int = 0,
                call: Union[int, torch.Tensor] = 0, non_blocking: bool = False
                ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """``y``, or ``(y, hidden)`` with ``hidden = a drop(x)`` (float32, for the backward pass) if ``return_hidden``.

        ``rows``: the adapter of every row, an int32 CUDA tensor, or ``AdapterRows`` that several calls share.  ``base``: the
        projection's output, which ``out`` may be.  Rows without adapter get ``base`` (zeros without it).  ``p``, ``seed`` and
        ``call`` are those of ``dropout``, applied to ``x_input``."""
        index, plan = self._native(rows, x_input)
        if index is not None or plan is not None:
            done = torch_calls().adapter_forward(self.a, self.b, self.scale, x_input, index, plan, base, out, return_hidden, p, seed,
                                                 call, non_blocking)
            if done is not None:
                return done if return_hidden else done[0]
        x = self._rows(x_input, self.in_size, "x_input")
        adapters = self._operand(x_input)
        shape = (*x_input.shape[:-1], self.out_size)
        add = None if base is None else like(base, x_input, shape, "base")
        drop = drop_params(p, seed, call, x_input.device)
        index, plan = self._grouped(rows, x, FEW_ROWS)
        if out is None:
            out = torch.empty(shape, dtype=x_input.dtype, device=x_input.device)
        y = like(out, x_input, shape, "out", written=True)
        hidden = torch.empty((*x_input.shape[:-1], self.rank), dtype=torch.float32, device=x_input.device) \
            if return_hidden or plan else None
        launch(x_input.device, non_blocking,
               lambda device, stream: lib().rpu_adapter_forward(
                   C.byref(adapters), x.ptr, x.ld, None if plan else index.data_ptr(), plan._plan_here().data_ptr() if plan else None,
                   plan._bytes if plan else 0, C.byref(drop), add.ptr if add else None, add.ld if add else 0, y.ptr, y.ld,
                   hidden.data_ptr() if hidden is not None else None, DTYPES[x_input.dtype], x.rows, device, stream))
        return (out, hidden) if return_hidden else out

    def backward(self, d_input: torch.Tensor, x_input: torch.Tensor, rows: Union[torch.Tensor, AdapterRows], hidden: torch.Tensor,
                 base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, p: float = 0.0, seed: int = 0,
                 call: Union[int, torch.Tensor] = 0, non_blocking: bool = False
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``(dx, da, db)`` from the gradient ``d_input`` of ``y`` and what the forward pass took and left (``rows``, ``p``,
        ``seed`` and ``call`` as there).  ``base``: added to ``dx``, the input gradient of the projection; ``out`` (dx) may be
        it.  ``da`` and ``db`` are like ``a`` and ``b``, zeros for adapters without rows."""
        index, plan = self._native(rows, x_input)
        if index is not None or plan is not None:
            done = torch_calls().adapter_backward(self.a, self.b, self.scale, d_input, x_input, index, plan, hidden, base, out, p, seed,
                                                  call, non_blocking)
            if done is not None:
                return done
        x = self._rows(x_input, self.in_size, "x_input")
        adapters = self._operand(x_input)
        d = like(d_input, x_input, (*x_input.shape[:-1], self.out_size), "d_input")
        if not isinstance(hidden, torch.Tensor) or hidden.dtype != torch.float32 or hidden.device != x_input.device \
                or hidden.numel() != x.rows * self.rank or not hidden.is_contiguous():
            raise RuntimeError("hidden must be what forward returned")
        add = None if base is None else like(base, x_input, x_input.shape, "base")
        drop = drop_params(p, seed, call, x_input.device)
        _, plan = self._grouped(rows, x, -1)
        if out is None:
            out = torch.empty(x_input.shape, dtype=x_input.dtype, device=x_input.device)
        dx = like(out, x_input, x_input.shape, "out", written=True)
        da, db = torch.empty_like(self.a), torch.empty_like(self.b)
        scratch_bytes = lib().rpu_adapter_backward_scratch(C.byref(adapters), x.rows)
        scratch = torch.empty(scratch_bytes // 4, dtype=torch.float32, device=x_input.device)
        launch(x_input.device, non_blocking,
               lambda device, stream: lib().rpu_adapter_backward(
                   C.byref(adapters), d.ptr, d.ld, x.ptr, x.ld, hidden.data_ptr(), plan._plan_here().data_ptr(), plan._bytes,
                   C.byref(drop), add.ptr if add else None, add.ld if add else 0, dx.ptr, dx.ld, da.data_ptr(), db.data_ptr(),
                   DTYPES[x_input.dtype], x.rows, scratch.data_ptr(), scratch_bytes, device, stream))
        return out, da, db
