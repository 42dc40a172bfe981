"""The digital operators that stand beside and between analog tiles, as cases that can be timed and compared.

A case is a dict of plain values; ``kind`` names the operator, the rest are its sizes and options:

  ``dropout``         dropout from counter-based draws (the backward pass is the same map of the gradient)
  ``norm``            layer norm, forward
  ``norm_backward``   its gradients, weight and bias included
  ``adapters``        low-rank adapters chosen by the row beside a projection whose output they add to
  ``adapters_train``  the same, forward and backward

With ``own`` false the operators are computed in their plain form, by elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # hidden layer of the 784-256-128-10 MLP at its batch of 64: a launch and little else
        dict(name="dropout_small", kind="dropout", rows=64, cols=256, type="f32", p=0.5, base=False),
        # end of a transformer block in training: dropout of a projection's output and the residual sum
        dict(name="dropout_residual", kind="dropout", rows=16384, cols=768, type="bf16", p=0.1, base=True),
        # rows of odd length (a layer of 785 lines), half precision
        dict(name="dropout_ragged", kind="dropout", rows=4099, cols=785, type="f16", p=0.2, base=False),
        # one token of a generated sequence: latency
        dict(name="norm_token", kind="norm", rows=1, cols=768, type="f32", weight="f32"),
        # a large batch of prompts
        dict(name="norm_rows", kind="norm", rows=16384, cols=1024, type="bf16", weight="f32"),
        # training step of a block of 768 channels; the gradient of the residual path is added
        dict(name="norm_backward", kind="norm_backward", rows=8192, cols=768, type="f32", weight="f32", base=True),
        # odd rows, half precision throughout
        dict(name="norm_backward_ragged", kind="norm_backward", rows=1037, cols=1537, type="f16", weight="f16", base=False),
        # eight requests, each with an adapter of its own, generate a token each beside a tile of 768 x 2304
        dict(name="adapters_decode", kind="adapters", rows=8, x=768, d=2304, rank=16, adapters=32, type="f32", weight="bf16",
             order="mixed"),
        # prompts of sixteen requests in a row
        dict(name="adapters_prefill", kind="adapters", rows=8192, x=768, d=2304, rank=16, adapters=16, type="f32", weight="bf16",
             order="runs"),
        # wide layer, larger rank, 16-bit activations, rows of the adapters mixed
        dict(name="adapters_wide", kind="adapters", rows=4096, x=4096, d=4096, rank=64, adapters=4, type="bf16", weight="bf16",
             order="mixed"),
        # adapting a programmed layer: one adapter, all rows, dropout on its input
        dict(name="adapters_train", kind="adapters_train", rows=8192, x=768, d=2304, rank=16, adapters=1, type="f32",
             weight="f32", order="runs", p=0.1),
        # seven adapters trained at once, odd sizes, some rows without one
        dict(name="adapters_train_ragged", kind="adapters_train", rows=1037, x=785, d=300, rank=5, adapters=7, type="bf16",
             weight="bf16", order="mixed", p=0.0),
    ]


def _log_int(rng, low, high):
    """An integer of [low, high], uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("dropout", "norm", "norm_backward", "adapters", "adapters", "adapters_train"))
    if kind.startswith("adapters"):
        x, d, rank = _log_int(rng, 32, 4096), _log_int(rng, 10, 4096), _log_int(rng, 1, 64)
        most = (1 << 24) // (x + d)
        type_, weight = rng.choice((("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")))
        case = dict(kind=kind, rows=_log_int(rng, 1, min(16384, most)), x=x, d=d, rank=rank, adapters=_log_int(rng, 1, 32),
                    type=type_, weight=weight, order=rng.choice(("runs", "mixed")))
        if kind == "adapters_train":
            case["p"] = rng.choice((0.0, 0.05, 0.1))
        return case
    cols = _log_int(rng, 16, 8192)
    case = dict(kind=kind, rows=_log_int(rng, 1, min(65536, (1 << 24) // cols)), cols=cols, type=rng.choice(("f32", "bf16", "f16")))
    if kind == "dropout":
        return dict(case, p=rng.choice((0.1, 0.25, 0.5)), base=rng.random() < 0.5)
    case["weight"] = rng.choice(("f32", case["type"]))
    if kind == "norm_backward":
        case["base"] = rng.random() < 0.5
    return case


# -- inputs ------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    state = dict(case=case, seed=(seed * 0x9E3779B97F4A7C15 + 1) % (1 << 64), call=seed % 1000)
    rows = case["rows"]
    if case["kind"] == "dropout":
        shape = (rows, case["cols"])
        return dict(state, x=normal(*shape), base=normal(*shape) if case["base"] else None)
    if case["kind"].startswith("norm"):
        cols, w = case["cols"], TYPES[case["weight"]]
        # rows of unlike size with an offset, as a residual stream has them
        scale = torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
        x = (torch.randn((rows, cols), generator=gen, device="cuda") * scale + 0.3).to(t)
        state.update(x=x, w=(1.0 + normal(cols, std=0.1, dtype=torch.float32)).to(w), b=normal(cols, std=0.1, dtype=w))
        if case["kind"] == "norm_backward":
            # what the forward pass left behind
            f = x.double()
            mean = f.mean(1)
            rstd = torch.rsqrt((f - mean[:, None]).square().mean(1) + EPS)
            state.update(mean=mean.float(), rstd=rstd.float(), d=normal(rows, cols, std=0.1),
                         base=normal(rows, cols, std=0.1) if case["base"] else None)
        return state
    n, r, x_size, d_size, w = case["adapters"], case["rank"], case["x"], case["d"], TYPES[case["weight"]]
    if case["order"] == "runs":        # prompts one after the other, of unlike lengths, adapters in any order
        cuts = torch.rand(n, generator=gen, device="cuda").cumsum(0)
        at = (torch.arange(rows, device="cuda") + 0.5) / rows * cuts[-1]
        index = torch.randperm(n, generator=gen, device="cuda")[torch.searchsorted(cuts, at).clamp_(max=n - 1)]
    else:                              # any row any adapter, some none
        index = torch.randint(-1, n, (rows,), generator=gen, device="cuda")
    state.update(index=index.to(torch.int32), x=normal(rows, x_size), base=normal(rows, d_size),
                 a=normal(n, r, x_size, std=x_size ** -0.5, dtype=w), b=normal(n, d_size, r, std=r ** -0.5, dtype=w),
                 scale=torch.rand(n, generator=gen, device="cuda") + 0.5)
    if case["kind"] == "adapters_train":
        state.update(d=normal(rows, d_size, std=0.1), dx_base=normal(rows, x_size, std=0.1))
    return state


# -- plain forms -------------------------------------------------------------------------------------------------------

def _product32(a, m):
    """High and low word of 32-bit numbers (held in 64 bits) times a constant; 64-bit products wrap."""
    p = a * m
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _draws(rows, cols, seed, call, purpose):
    """16 random bits an element: halves of Philox4x32-10 blocks, counter (column / 8, row, call, purpose), key the seed."""
    blocks = -(-cols // 8)
    c0 = torch.arange(blocks, device="cuda").expand(rows, blocks)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, blocks)
    c2, c3 = torch.full_like(c0, call), torch.full_like(c0, purpose)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _product32(c0, 0xD2511F53)
        h1, l1 = _product32(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0, c1, c2, c3), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, blocks * 8)[:, :cols]


def _kept(rows, cols, p, seed, call):
    limit = int(p * 4294967296.0 + 0.5)
    u, v = _draws(rows, cols, seed, call, 18), _draws(rows, cols, seed, call, 19)
    return (u > limit >> 16) | ((u == limit >> 16) & (v >= limit & 0xFFFF))


def _dropped(x, p, seed, call):
    if p == 0.0:
        return x
    return torch.where(_kept(*x.shape, p, seed, call), x * (1.0 / (1.0 - p)), 0.0)


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    y = _dropped(x.float(), case["p"], s["seed"], s["call"])
    return (y if s["base"] is None else y + s["base"].float()).to(x.dtype)


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = torch.rsqrt(c.square().mean(1) + EPS)
    y = c * rstd[:, None] * s["w"].float() + s["b"].float()
    return y.to(s["x"].dtype), mean, rstd


def _plain_norm_backward(s):
    x, d, w, rstd = s["x"].float(), s["d"].float(), s["w"].float(), s["rstd"][:, None]
    h = (x - s["mean"][:, None]) * rstd
    g = d * w
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    if s["base"] is not None:
        dx = dx + s["base"].float()
    return dx.to(s["x"].dtype), (d * h).sum(0).to(s["w"].dtype), d.sum(0).to(s["w"].dtype)


def _own_part(full, index, n):
    """[rows, n, r] with zero wherever the row has another adapter."""
    return torch.where(index[:, None, None] == torch.arange(n, device="cuda")[None, :, None], full, 0.0)


def _plain_adapters(s):
    case, a, b = s["case"], s["a"].float(), s["b"].float()
    n, r, x_size = a.shape
    rows, d_size = case["rows"], case["d"]
    p = case.get("p", 0.0)
    x = _dropped(s["x"].float(), p, s["seed"], s["call"])
    flat_a = a.reshape(n * r, x_size)
    flat_b = b.permute(0, 2, 1).reshape(n * r, d_size)
    scale = s["scale"][:, None]
    hidden = _own_part((x @ flat_a.T).view(rows, n, r), s["index"], n)
    y = s["base"].float() + (hidden * scale).view(rows, n * r) @ flat_b
    y = y.to(s["x"].dtype)
    if case["kind"] == "adapters":
        return y
    d = s["d"].float()
    up = _own_part((d @ flat_b.T).view(rows, n, r) * scale, s["index"], n).view(rows, n * r)
    dx = s["dx_base"].float() + _dropped(up @ flat_a, p, s["seed"], s["call"])
    da = (up.T @ x).view(n, r, x_size)
    db = ((hidden * scale).view(rows, n * r).T @ d).view(n, r, d_size).permute(0, 2, 1).contiguous()
    return y, dx.to(s["x"].dtype), da.to(s["a"].dtype), db.to(s["b"].dtype)


# -- the framework's calls ---------------------------------------------------------------------------------------------

def _own_dropout(s):
    from aihwkit_amd import digital
    return digital.dropout(s["x"], s["case"]["p"], s["seed"], s["call"], base=s["base"], non_blocking=True)


def _own_norm(s):
    from aihwkit_amd import digital
    return digital.layer_norm(s["x"], s["w"], s["b"], EPS, non_blocking=True)


def _own_norm_backward(s):
    from aihwkit_amd import digital
    return digital.layer_norm_backward(s["d"], s["x"], s["mean"], s["rstd"], s["w"], base=s["base"], non_blocking=True)


def _own_adapters(s):
    from aihwkit_amd import digital
    if "handle" not in s:
        s["handle"] = digital.LowRankAdapters(s["a"], s["b"], s["scale"])
    adapters = s["handle"]
    if s["case"]["kind"] == "adapters":
        return adapters.forward(s["x"], s["index"], base=s["base"], non_blocking=True)
    drop = dict(p=s["case"]["p"], seed=s["seed"], call=s["call"])
    rows = digital.AdapterRows(s["index"], adapters.n_adapters)      # one grouping of the rows for both directions
    y, hidden = adapters.forward(s["x"], rows, base=s["base"], return_hidden=True, non_blocking=True, **drop)
    dx, da, db = adapters.backward(s["d"], s["x"], rows, hidden, base=s["dx_base"], non_blocking=True, **drop)
    return y, dx, da, db


def run(state):
    kind = state["case"]["kind"]
    if kind.startswith("adapters"):
        return _own_adapters(state) if own else _plain_adapters(state)
    if kind == "dropout":
        return _own_dropout(state) if own else _plain_dropout(state)
    if kind == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_norm_backward(state) if own else _plain_norm_backward(state)


# -- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    rows, e = case["rows"], SIZES[case["type"]]
    if case["kind"] == "dropout":
        values = rows * case["cols"]
        return dict(bytes=e * values * (3 if case["base"] else 2), flops=values * (2 if case["base"] else 1))
    if case["kind"] == "norm":
        values = rows * case["cols"]
        return dict(bytes=2 * e * values + 8 * rows + 2 * SIZES[case["weight"]] * case["cols"], flops=7 * values)
    if case["kind"] == "norm_backward":
        values = rows * case["cols"]
        return dict(bytes=(4 if case["base"] else 3) * e * values + 8 * rows + 3 * SIZES[case["weight"]] * case["cols"],
                    flops=13 * values)
    x, d, r, n = case["x"], case["d"], case["rank"], case["adapters"]
    used = min(n, rows)
    matrices = SIZES[case["weight"]] * r * (x + d)
    forward = dict(bytes=e * rows * (x + 2 * d) + 4 * rows + used * (matrices + 4), flops=2 * rows * r * (x + d))
    if case["kind"] == "adapters":
        return forward
    # x and the weights count once for both directions; gradients of all adapters are written
    return dict(bytes=forward["bytes"] + e * rows * (d + 2 * x) + n * matrices, flops=3 * forward["flops"])


# -- the definition in 64 bits -----------------------------------------------------------------------------------------

def _exact_kept(rows, cols, p, seed, call):
    """The same draws with numpy's unsigned integers, written from the generator's definition."""
    u32, mask = np.uint64(32), np.uint64(0xFFFFFFFF)
    row, block = np.meshgrid(np.arange(rows, dtype=np.uint64), np.arange((cols + 7) // 8, dtype=np.uint64), indexing="ij")
    bits = []
    for purpose in (18, 19):
        ctr = [block.copy(), row.copy(), np.full_like(row, call), np.full_like(row, purpose)]
        key = [seed % (1 << 32), seed // (1 << 32)]
        for _ in range(10):
            left, right = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            ctr = [(right >> u32) ^ ctr[1] ^ np.uint64(key[0]), right & mask,
                   (left >> u32) ^ ctr[3] ^ np.uint64(key[1]), left & mask]
            key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
        half = np.empty(row.shape + (8,), dtype=np.uint64)
        for k in range(4):
            half[..., 2 * k], half[..., 2 * k + 1] = ctr[k] % np.uint64(65536), ctr[k] // np.uint64(65536)
        bits.append(half.reshape(rows, -1)[:, :cols])
    limit = np.uint64(int(math.floor(p * 2.0 ** 32 + 0.5)))
    return torch.from_numpy(bits[0] * np.uint64(65536) + bits[1] >= limit).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "dropout":
        y = f["x"] / (1.0 - case["p"]) * _exact_kept(case["rows"], case["cols"], case["p"], s["seed"], s["call"])
        return y + f["base"] if case["base"] else y
    if case["kind"] == "norm":
        var, mean = torch.var_mean(f["x"], 1, correction=0)
        rstd = (var + EPS) ** -0.5
        return (f["x"] - mean[:, None]) * rstd[:, None] * f["w"] + f["b"], mean, rstd
    if case["kind"] == "norm_backward":
        # gradient of sum(d * y) at the given statistics, from its pieces: d/dx of (x - mean) rstd
        h = (f["x"] - f["mean"][:, None]) * f["rstd"][:, None]
        g = f["d"] * f["w"]
        n = case["cols"]
        dx = f["rstd"][:, None] * (g - (g.sum(1, keepdim=True) + h * (g * h).sum(1, keepdim=True)) / n)
        return dx + f["base"] if case["base"] else dx, torch.einsum("tc,tc->c", f["d"], h), f["d"].sum(0)
    p = case.get("p", 0.0)
    rows, x_size = case["rows"], case["x"]
    keep = _exact_kept(rows, x_size, p, s["seed"], s["call"]).double() / (1.0 - p) if p else torch.ones_like(f["x"])
    y, dx = f["base"].clone(), f.get("dx_base", torch.zeros(1)).clone()
    da, db = torch.zeros_like(f["a"]), torch.zeros_like(f["b"])
    for k in range(case["adapters"]):
        at = torch.nonzero(s["index"] == k)[:, 0]
        x, a, b, scale = f["x"][at] * keep[at], f["a"][k], f["b"][k], f["scale"][k]
        v = x @ a.T
        y[at] += scale * (v @ b.T)
        if case["kind"] == "adapters_train":
            u = scale * (f["d"][at] @ b)
            dx[at] += (u @ a) * keep[at]
            da[k], db[k] = u.T @ x, scale * (f["d"][at].T @ v)
    return y if case["kind"] == "adapters" else (y, dx, da, db)
