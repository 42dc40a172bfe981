"""Digital operators beside and between analog tiles, as HIP kernels on the GPU.

Weights that were programmed into tiles are not trained any more; what adapts such a network, is trained beside the tiles or
differs from request to request is digital: low-rank adapters of a tile's projection (``LowRankAdapters``, also through
``InferenceTile.forward``), dropout whose mask is never stored (``dropout``), the layer norms between the tiles
(``layer_norm``, ``layer_norm_backward``) and, where the tiles are a transformer's linear layers, attention over a paged cache of keys and
values (``PagedCache``).  The reference leaves these to torch.

Tensors are on the GPU, float32, float16 or bfloat16; the last dimension holds the columns, the others together are the rows.
Matrices whose rows are apart (column slices) are read and written in place; other layouts of inputs are copied first.
Everything is computed in 32 bits and rounded once.  As with the tiles, calls go to the current stream of the tensors' GPU and
wait for it unless ``non_blocking`` is set (``AdapterRows`` never waits: calls that use it come after it on whatever stream), and nothing
takes part in autograd: forward and backward are calls of their own.
"""
from .adapters import AdapterRows, LowRankAdapters
from .cache import PagedCache, rotation_frequencies
from .elementwise import dropout
from .norm import layer_norm, layer_norm_backward

__all__ = ["AdapterRows", "LowRankAdapters", "PagedCache", "dropout", "layer_norm", "layer_norm_backward", "rotation_frequencies"]
