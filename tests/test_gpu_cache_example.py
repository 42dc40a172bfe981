"""The documented example of attention over a paged cache, as it stands, against the definition in 64 bits."""
import os
import re

import pytest
import torch

from aihwkit_amd.inference import InferenceTile
from aihwkit_amd.rpu_base import devices as dv
from cache_oracle import U, rotated
from test_gpu_digital import rand

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_documented_example():
    """Keys and values are rounded to bf16, half a step of 2^-8, once: the oracle rounds what the tile gives in the same way, and the few values whose
    rounding hangs on the last bits of the tile's sums are off by a whole step.  A step of one value of 16 in a mean of up to 90: 2^-8 of
    the largest weight's value and of a score of order one; 4 steps cover both."""
    with open(os.path.join(ROOT, "INTEGRATION.md")) as text:
        block, = [b for b in re.findall(r"```python\n(.*?)```", text.read(), re.S) if "PagedCache(" in b]
    io = dv.AnalogTileInputOutputParameter()
    io.is_perfect = True
    heads, head_size, width = 4, 16, 64
    project = InferenceTile(3 * width, width, forward_io=io)
    project.set_weights(rand(1, 3 * width, width, std=0.1).cpu())
    project.cuda()
    prompts, tokens = rand(2, 130, width), rand(3, 3, width)
    counts = [89, 1, 40]
    names = dict(torch=torch, project=project, heads=heads, head_size=head_size, pages=6, prompts=prompts, tokens=tokens,
                 tables=torch.tensor([[4, 1], [0, -1], [2, -1]], dtype=torch.int32, device="cuda"),
                 lengths=torch.tensor(counts, dtype=torch.int32, device="cuda"), starts=torch.tensor([0, 89, 90, 130], dtype=torch.int32, device="cuda"))
    exec(block, names)
    torch.cuda.synchronize()
    w, f = project.get_weights().double(), torch.tensor([10000.0 ** (-i / 8) for i in range(8)], dtype=torch.float64)
    for s in range(3):
        first = sum(counts[:s])
        x = torch.cat((prompts[first:first + counts[s]], tokens[s:s + 1])).double().cpu()
        q, k, v = (x @ w.T).view(-1, 3, heads, head_size).unbind(1)
        position = torch.arange(len(x))
        q, k = rotated(q, position, f, False), rotated(k, position, f, False).bfloat16().double()
        scores = torch.einsum("ihd,jhd->hij", q, k) * head_size ** -0.5
        scores = scores.masked_fill(torch.triu(torch.ones(len(x), len(x), dtype=torch.bool), 1), -float("inf"))
        expected = torch.einsum("hij,jhd->ihd", torch.softmax(scores, -1), v.bfloat16().double()).reshape(-1, width)
        got = torch.cat((names["prompted"][first:first + counts[s]], names["generated"][s:s + 1])).double().cpu()
        limit = (4 * 2.0 ** -8 + 1000 * U) * max(1.0, float(v.abs().max()))
        assert float((got - expected).abs().max()) <= limit
    assert names["generated"].dtype == torch.float32 and names["generated"].shape == (3, width)
