"""The documented example of the digital operators, as it stands: that it runs, and its gradients."""
import os
import re

import pytest
import torch

from aihwkit_amd.inference import InferenceTile
from aihwkit_amd.rpu_base import devices as dv
from test_gpu_digital import U, kept, rand

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    with open(os.path.join(ROOT, "INTEGRATION.md")) as text:
        blocks = re.findall(r"```python\n(.*?)```", text.read(), re.S)
    block, = [b for b in blocks if "LowRankAdapters(" in b]
    return block


def test_the_documented_example():
    """Against torch's autograd in 64 bits on the same masks.  The results are sums over up to 96 terms in each of five stages and over 70
    rows in the gradients; 400 U of the largest value covers any order of them, all values being of order one."""
    io = dv.AnalogTileInputOutputParameter()
    io.is_perfect = True
    tile = InferenceTile(64, 96, forward_io=io)
    tile.set_weights(rand(1, 64, 96, std=0.1).cpu())
    tile.cuda()
    given = dict(a=rand(2, 3, 8, 96, std=0.1), b=rand(3, 3, 64, 8, std=0.1), scale=rand(4, 3), x=rand(5, 70, 96), dz=rand(6, 70, 64),
                 residual=rand(7, 70, 64), w=1 + rand(8, 64, std=0.1), bias=rand(9, 64), index=(torch.arange(70, device="cuda") % 4 - 1).to(torch.int32))
    names = dict(given, tile=tile, seed=12, step=4)
    exec(example(), names)
    torch.cuda.synchronize()
    f = {k: v.detach().double().cpu().requires_grad_(v.is_floating_point()) for k, v in given.items() if k != "index"}
    chosen, weights = given["index"].cpu().long(), tile.get_weights().double()
    one = torch.nn.functional.one_hot(chosen + 1, 4)[:, 1:].double()              # rows without an adapter: zeros

    def adapted(x):
        v = torch.stack([x @ f["a"][k].T for k in range(3)], 1)
        u = torch.stack([v[:, k] @ f["b"][k].T for k in range(3)], 1)
        return (u * (one * f["scale"])[:, :, None]).sum(1)

    plain = f["x"] @ weights.T
    served = plain + adapted(f["x"])
    y = plain + adapted(f["x"] * kept(70, 96, 0.1, 12, 4).double() / 0.9)
    r = f["residual"] + y * kept(70, 64, 0.1, 12, 5).double() / 0.9
    c = r - r.mean(1, keepdim=True)
    z = c * (c.square().mean(1, keepdim=True) + 1e-5) ** -0.5 * f["w"] + f["bias"]
    (z * f["dz"].detach()).sum().backward()
    for name, expected in dict(served=served, z=z, dx=f["x"].grad, da=f["a"].grad, db=f["b"].grad, dw=f["w"].grad, dbias=f["bias"].grad,
                               dr=f["residual"].grad).items():
        expected = expected.detach()
        limit = 400 * U * max(1.0, float(expected.abs().max()))
        assert float((names[name].double().cpu() - expected).abs().max()) <= limit, name
