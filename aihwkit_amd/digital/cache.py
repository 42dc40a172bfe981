"""Attention between tiles: a paged cache of keys and values, what fills it and what reads it."""
import ctypes as C
import math
from typing import Optional

import torch

from .._cabi import Cache, CacheRows, lib, torch_calls
from ._operands import DTYPES, check_rows, launch

MOST_POSITIONS = 1 << 30     # of a table
NUMBER = 1 << 31


def rotation_frequencies(head_size: int, base: float = 10000.0) -> torch.Tensor:
    """Angles by which the pairs of a head turn from a position to the next, in radians: ``base ** (-2 i / head_size)`` (float64)."""
    return float(base) ** (-torch.arange(head_size // 2, dtype=torch.float64) * 2 / head_size)


class _Heads:
    """Rows of heads [rows, heads, head_size], the values of a row in a row: the tensor (a copy where it is laid out otherwise) and the
    distance of its rows."""

    __slots__ = ("tensor", "rows", "heads", "ld")

    def __init__(self, tensor, head_size: int, what: str, beside: Optional[torch.Tensor] = None, written: bool = False):
        check_rows(tensor, what)
        if tensor.dim() != 3 or tensor.size(2) != head_size or tensor.size(1) < 1:
            raise RuntimeError(f"Invalid {what} dimensions: expected [rows, heads, {head_size}], got {list(tensor.shape)}")
        if beside is not None:
            if tensor.dtype != beside.dtype:
                raise RuntimeError(f"{what} must be of type {beside.dtype}")
            if tensor.device != beside.device:
                raise RuntimeError(f"{what} must be on {beside.device}")
        self.rows, self.heads = tensor.size(0), tensor.size(1)
        width = self.heads * head_size
        if not (tensor.stride(2) == 1 and (self.heads == 1 or tensor.stride(1) == head_size) and (self.rows < 2 or tensor.stride(0) >= width)):
            if written:
                raise RuntimeError(f"The values of a row of {what} must lie in a row")
            tensor = tensor.contiguous()
        self.tensor = tensor
        self.ld = tensor.stride(0) if self.rows > 1 else width

    @property
    def ptr(self):
        return self.tensor.data_ptr()


def _int32(tensor, device: torch.device, dims: int, what: str) -> torch.Tensor:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if tensor.dtype != torch.int32 or tensor.device != device:
        raise RuntimeError(f"{what} must be an int32 tensor on {device}")
    if tensor.dim() != dims:
        raise RuntimeError(f"{what} must have {dims} dimension{'s' if dims > 1 else ''}")
    return tensor


class PagedCache:
    """Keys and values of the tokens of many sequences, in pages that sequences take as they grow.

    ``keys`` and ``values`` [pages, heads, page_size, head_size] (float32, float16 or bfloat16) are the caller's tensors, dense and on one
    GPU, and are used as they are at every call.  ``page_size`` is a power of two, 8 to 65536, ``head_size`` a multiple of 8 up to 256.
    ``frequencies`` (None: no rotation): the angles, in radians, by which the pairs of a head turn from a position to the next, at most
    ``head_size / 2`` of them (``rotation_frequencies``); they are copied, as float64.  Pair ``i`` is columns ``(i, i + pairs)`` or, with
    ``neighbours``, ``(2 i, 2 i + 1)``; columns from ``2 pairs`` on are not rotated.

    Both calls name the sequences of their rows in the same way, by int32 tensors on the GPU that are read when the kernels run (a captured
    step follows what they hold at each replay):

    ``tables`` [n, width]: the pages of every sequence in the order of its positions.  A page number that the cache does not have, such as -1,
    stands for positions that are not there: they are not written and not seen.
    ``lengths`` [n]: positions of every sequence, the new rows included: the ``i``-th of its ``m`` new rows is at ``length - m + i``.
    ``starts`` [n + 1] (None: as many rows for every sequence): rows ``starts[s] .. starts[s + 1] - 1`` are those of sequence ``s``;
    not decreasing.  Rows of no sequence are left as they are in an ``out`` that is given, and are zeros in a new one.

    Rows are float32 beside any cache, or of the cache's type."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, frequencies: Optional[torch.Tensor] = None, neighbours: bool = False):
        for tensor, what in ((keys, "keys"), (values, "values")):
            check_rows(tensor, what)
            if tensor.dim() != 4 or tensor.numel() == 0:
                raise RuntimeError(f"{what} must be of four dimensions: pages, heads, positions of a page, values of a head")
        self.pages, self.n_heads, self.page_size, self.head_size = keys.shape
        if self.page_size & (self.page_size - 1) or not 8 <= self.page_size <= 65536:
            raise RuntimeError("The size of a page must be a power of two, 8 to 65536.")
        if self.head_size % 8 or self.head_size > 256:
            raise RuntimeError("The size of a head must be a multiple of 8 up to 256.")
        if self.n_heads > 65536 or self.pages >= NUMBER:
            raise RuntimeError("A cache has at most 65536 heads and 2^31 - 1 pages.")
        if keys[0].numel() * keys.element_size() >= NUMBER:
            raise RuntimeError("The keys of a page must take less than 2 GB.")
        self._shape = keys.shape
        self.keys, self.values = keys, values
        self.neighbours = bool(neighbours)
        self._turns, self.pairs = None, 0
        if frequencies is not None:
            if not isinstance(frequencies, torch.Tensor):
                raise TypeError("frequencies must be a torch.Tensor")
            if frequencies.dim() != 1 or 2 * frequencies.numel() > self.head_size or not frequencies.is_floating_point():
                raise RuntimeError("frequencies must be one dimension of at most half a head's size")
            self.pairs = frequencies.numel()
            if self.pairs:
                self._turns = (frequencies.detach().to("cpu", torch.float64) / (2 * math.pi)).to(keys.device)
        self._operand()

    def _operand(self) -> Cache:
        """The C structure of the tensors as they are now."""
        keys, values = self.keys, self.values
        for tensor, what in ((keys, "keys"), (values, "values")):
            if not isinstance(tensor, torch.Tensor) or tensor.shape != self._shape or not tensor.is_contiguous():
                raise RuntimeError("Invalid %s: expected a dense %s tensor" % (what, list(self._shape)))
        if keys.dtype not in DTYPES or keys.dtype != values.dtype:
            raise RuntimeError("keys and values must be of one type")
        if not keys.is_cuda or keys.device != values.device or (self._turns is not None and self._turns.device != keys.device):
            raise RuntimeError("keys and values must be on one GPU")
        return Cache(k_dev=keys.data_ptr(), v_dev=values.data_ptr(), turns_dev=None if self._turns is None else self._turns.data_ptr(),
                     pages=self.pages, page_size=self.page_size, heads=self.n_heads, head_size=self.head_size, dtype=DTYPES[keys.dtype],
                     pairs=self.pairs, neighbours=int(self.neighbours))

    def _check_beside(self, rows: _Heads) -> None:
        if rows.tensor.device != self.keys.device:
            raise RuntimeError(f"Rows and cache must be on one GPU, {self.keys.device}")
        if rows.tensor.dtype not in (torch.float32, self.keys.dtype):
            raise RuntimeError("A cache beside 16-bit rows must be of the rows' type.")

    def _sequences(self, tables, lengths, starts, rows: int):
        """The C structure, and the tensors that it points into."""
        device = self.keys.device
        tables = _int32(tables, device, 2, "tables")
        n, width = tables.shape
        lengths = _int32(lengths, device, 1, "lengths").contiguous()
        if n < 1 or lengths.numel() != n:
            raise RuntimeError("tables and lengths must be of as many sequences, one at least")
        if width < 1 or width * self.page_size > MOST_POSITIONS:
            raise RuntimeError("A table must hold 1 .. 2^30 positions.")
        if (width > 1 and tables.stride(1) != 1) or (n > 1 and tables.stride(0) < width):
            tables = tables.contiguous()
        if starts is not None:
            starts = _int32(starts, device, 1, "starts").contiguous()
            if starts.numel() != n + 1:
                raise RuntimeError("Invalid starts dimensions: expected %d values, got %d" % (n + 1, starts.numel()))
        elif rows % n:
            raise RuntimeError("Without starts, the sequences have as many rows each.")
        given = CacheRows(tables_dev=tables.data_ptr(), lengths_dev=lengths.data_ptr(), starts_dev=None if starts is None else starts.data_ptr(),
                          table_ld=tables.stride(0) if n > 1 else width, n=n, table_width=width, rows=rows)
        return given, (tables, lengths, starts)

    @staticmethod
    def _output(out, like: torch.Tensor, starts, head_size: int) -> _Heads:
        if out is None:
            out = (torch.empty if starts is None else torch.zeros)(like.shape, dtype=like.dtype, device=like.device)
        given = _Heads(out, head_size, "out", like, written=True)
        if given.tensor.shape != like.shape:
            raise RuntimeError(f"Invalid out dimensions: expected {list(like.shape)}, got {list(given.tensor.shape)}")
        return given

    def append(self, keys: torch.Tensor, values: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
               queries: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, non_blocking: bool = False) -> Optional[torch.Tensor]:
        """Writes the new rows' ``keys`` (rotated by their positions) and ``values`` [rows, heads, head_size] into the cache.

        ``queries`` [rows, any number of heads, head_size]: rotated in the same way into ``out``, which may be ``queries``, and returned.
        Angles are taken in 64 bits; results are rounded once.  Two rows for one place of the cache leave either's values."""
        done = torch_calls().cache_append(self.keys, self.values, self._shape, self._turns, self.neighbours, keys, values, tables, lengths, starts,
                                          queries, out, non_blocking)
        if done is not None:
            return done[0]
        cache = self._operand()
        k = _Heads(keys, self.head_size, "keys")
        v = _Heads(values, self.head_size, "values", keys)
        self._check_beside(k)
        if k.heads != self.n_heads or v.tensor.shape != k.tensor.shape:
            raise RuntimeError("keys and values must have the cache's %d heads, and as many rows" % self.n_heads)
        given, held = self._sequences(tables, lengths, starts, k.rows)
        q = y = None
        if queries is not None:
            q = _Heads(queries, self.head_size, "queries", keys)
            if q.rows != k.rows:
                raise RuntimeError("Invalid queries dimensions: expected %d rows, got %d" % (k.rows, q.rows))
            y = self._output(out, queries, starts, self.head_size)
        elif out is not None:
            raise RuntimeError("There are no queries to write to out.")
        launch(self.keys.device, non_blocking,
               lambda device, stream: lib().rpu_cache_append(
                   C.byref(cache), C.byref(given), k.ptr, k.ld, v.ptr, v.ld, q.ptr if q else None, q.ld if q else 0, y.ptr if q else None,
                   y.ld if q else 0, q.heads if q else 0, DTYPES[keys.dtype], device, stream))
        del held
        return y.tensor if q else None

    def attend(self, queries: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, window: int = 0, sinks: int = 0, longest: Optional[int] = None, out: Optional[torch.Tensor] = None,
               non_blocking: bool = False) -> torch.Tensor:
        """Attention of the new rows [rows, heads, head_size] over what the cache holds, their own keys and values included.

        The row at position ``p`` sees positions ``j <= p``; with a ``window`` > 0 those of ``j > p - window`` or ``j < sinks``.  ``heads`` is a
        multiple of the cache's, each of which serves as many neighbouring ones.  ``scale`` (None: ``head_size ** -0.5``; up to 1e30)
        multiplies the products of queries and keys.  ``longest``: a number that no length exceeds (None: what the tables hold); how the work is
        shared goes by it, the results are right without it.  A row that sees nothing becomes zeros, and so does one whose weights are all
        zero.  What a row does not see does not reach it, infinities and NaN included; one among the values that a head of a row sees makes its
        column of that head infinite or NaN, one among the keys that it sees, or in its query, may make all of its columns so.  The products of
        queries and keys, and the sums of the values by weights of up to 1, are to stay below the largest float.  ``out`` may be ``queries``."""
        done = torch_calls().cache_attend(self.keys, self.values, self._shape, queries, tables, lengths, starts, scale, window, sinks, longest, out,
                                          non_blocking)
        if done is not None:
            return done
        cache = self._operand()
        q = _Heads(queries, self.head_size, "queries")
        self._check_beside(q)
        if q.heads % self.n_heads:
            raise RuntimeError("The heads of a row must be a multiple of the cache's.")
        window, sinks, longest = int(window), int(sinks), 0 if longest is None else int(longest)
        if not (0 <= window < NUMBER and 0 <= sinks < NUMBER and 0 <= longest < NUMBER):
            raise RuntimeError("window, sinks and longest must be in 0 .. 2^31 - 1.")
        scale = self.head_size ** -0.5 if scale is None else float(scale)
        given, held = self._sequences(tables, lengths, starts, q.rows)
        y = self._output(out, queries, starts, self.head_size)
        bytes_ = lib().rpu_cache_attend_scratch(C.byref(cache), C.byref(given), q.heads, DTYPES[queries.dtype], window, sinks, longest)
        scratch = torch.empty(bytes_ // 4, dtype=torch.float32, device=queries.device) if bytes_ else None
        launch(self.keys.device, non_blocking,
               lambda device, stream: lib().rpu_cache_attend(
                   C.byref(cache), C.byref(given), q.ptr, q.ld, y.ptr, y.ld, q.heads, DTYPES[queries.dtype], scale, window, sinks, longest,
                   scratch.data_ptr() if bytes_ else None, bytes_, device, stream))
        del held
        return y.tensor
