"""The head of a classifier as work that can be timed: dropout whose mask is never stored, and the last linear layer with
its softmax cross entropy without keeping the logits.

A case is one pass as a training step (forward, then every gradient) or a validation step (forward under `no_grad`) runs
it.  With `own` set, `run` calls the framework's operators; otherwise it computes the same values from elementary torch
operations in 32 bits.  `exact` computes them in 64 bits.

    dropout                y[i] = x[i] * [draw(i // run) >= round(p * 2^32)] / (1 - p), run = elements that share a draw.
                           Philox4x32-10(counter = (j // 8, offset), key = seed) gives the upper 16 bits of the draws 8 (j // 8)
                           ... + 7, low halves of its words first; the lower 16 bits come from the counter j // 8 + 2^63
    linear_cross_entropy   z = x W^T + b,  loss_t = logsumexp(z_t) - (1 - s) z_t[y_t] - s mean(z_t), averaged or summed
                           over the rows that are not ignored, or one by one
"""
import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_IGNORE = -100


def _dropout(name, shape, dtype, p, shared_dims=0, grad=True):
    return dict(name=name, op="dropout", shape="x".join(map(str, shape)), dtype=dtype, p=p, shared_dims=shared_dims, grad=grad)


def _head(name, rows, features, classes, dtype, smoothing=0.0, bias=True, ignored=0.0, reduction="mean", grad=True):
    return dict(name=name, op="head", rows=rows, features=features, classes=classes, dtype=dtype, smoothing=smoothing, bias=bias,
                ignored=ignored, reduction=reduction, grad=grad)


def listed():
    return [
        # the dropout in front of a mobile classifier: pooled features of 128 images, nothing but latency
        _dropout("dropout_fp16_pooled", (128, 1280), "fp16", 0.2),
        # every element of the largest layer of the sweep: nothing but bandwidth
        _dropout("dropout_fp16_c96_112", (128, 96, 112, 112), "fp16", 0.1),
        # whole feature planes at once, full precision
        _dropout("dropout_fp32_planes", (64, 144, 56, 56), "fp32", 0.2, shared_dims=2),
        # dense prediction: rows and planes of odd sizes
        _dropout("dropout_bf16_ragged", (8, 72, 75, 101), "bf16", 0.5),
        # one image through the classifier of a service, its loss only: nothing but latency
        _head("head_fp16_one_image", 1, 1280, 1000, "fp16", grad=False),
        # training steps of the mobile classifier: one GPU's share of the images, and all of them with smoothed labels
        _head("head_fp16_b128", 128, 1280, 1000, "fp16"),
        _head("head_fp16_b1024_smooth", 1024, 1280, 1000, "fp16", smoothing=0.1),
        # the same in full precision
        _head("head_fp32_b256", 256, 1280, 1000, "fp32"),
        # dense prediction: every pixel of 8 planes of 56 x 56 a row, few features and classes, unlabelled pixels
        _head("head_fp16_pixels", 8 * 56 * 56, 256, 150, "fp16", ignored=0.1),
        # validation over a large vocabulary, one loss a row, all three sizes odd
        _head("head_bf16_ragged_eval", 1777, 1021, 32003, "bf16", bias=False, ignored=0.05, reduction="none", grad=False),
        # training with the 21841 classes of a large image collection
        _head("head_bf16_21k", 4096, 1280, 21841, "bf16", smoothing=0.1),
        # the largest: long batches over a large vocabulary, no bias
        _head("head_bf16_65k", 8192, 2048, 65536, "bf16", bias=False, ignored=0.05, reduction="sum"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _nameless(case):
    del case["name"]
    return case


def draw(rng):
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    if rng.random() < 0.35:
        shape = [_spread(rng, 1, 128), _spread(rng, 1, 960)]
        shared = 0
        if rng.random() < 0.7:
            side = _spread(rng, 1, 112)
            shape += [side, _spread(rng, max(1, side // 2), min(112, 2 * side))]
            shared = rng.choice([0, 0, 2, 3])
        else:
            shape[1] = _spread(rng, 1, 4096)
        limit = 128 * 96 * 112 * 112 // (2 if dtype == "fp32" else 1)
        while math.prod(shape) > limit:
            shape[0] = max(1, shape[0] // 2)
            if shape[0] == 1:
                shape[1] = max(1, shape[1] // 2)
        return _nameless(_dropout(None, shape, dtype, round(rng.uniform(0.02, 0.9), 3), shared, rng.random() < 0.7))
    rows, features, classes = _spread(rng, 1, 16384), _spread(rng, 16, 2560), _spread(rng, 2, 65536)
    # the products of 32-bit operands cost several times those of 16-bit ones
    limit = 8192 * 2048 * 65536 // (16 if dtype == "fp32" else 1)
    while rows * features * classes > limit or rows * classes > 8192 * 65536:
        rows = max(1, rows // 2)
    reduction = rng.choice(["mean", "mean", "sum", "none"])
    return _nameless(_head(None, rows, features, classes, dtype, rng.choice([0.0, 0.0, 0.1]), rng.random() < 0.7,
                           rng.choice([0.0, 0.0, 0.1]), reduction, rng.random() < 0.7))


def _shape(case):
    return [int(v) for v in case["shape"].split("x")]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)

    st = dict(case)
    if case["op"] == "dropout":
        shape = _shape(case)
        st["x"] = normal(*shape)
        st["dy"] = normal(*shape) if case["grad"] else None
        # what a training program keeps on the device: the seed and the number of the draw
        st["state"] = torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 63), 1000 + seed % 1000], device="cuda", dtype=torch.int64)
        st["x"].requires_grad_(case["grad"])
        return st
    t, d, v = case["rows"], case["features"], case["classes"]
    w = normal(v, d, std=1.5 / math.sqrt(d))
    y = torch.randint(0, v, (t,), device="cuda", generator=gen)
    # features of a network that has learned something: they lean towards the row of their class
    lean = torch.rand(t, 1, device="cuda", generator=gen) * 3
    st["x"] = (torch.randn(t, d, device="cuda", generator=gen) + lean * w[y].float()).to(dtype)
    st["w"] = w
    st["b"] = normal(v, std=0.1) if case["bias"] else None
    if case["ignored"]:
        drop = torch.rand(t, device="cuda", generator=gen) < case["ignored"]
        drop[0] = False                              # a batch has a label
        y = torch.where(drop, torch.full_like(y, _IGNORE), y)
    st["y"] = y
    if case["grad"]:
        # what arrives from behind the loss: the scale that keeps 16-bit gradients out of the subnormal numbers
        up = torch.full((), 1024.0 if case["dtype"] == "fp16" else 1.0, device="cuda")
        if case["reduction"] == "none":
            up = up * torch.rand(t, device="cuda", generator=gen) / t
        elif case["reduction"] == "sum":
            up = up / t
        st["up"] = up
    for k in ("x", "w", "b"):
        if st[k] is not None:
            st[k].requires_grad_(case["grad"])
    return st


def _philox(group, state):
    """Ten rounds on the counters (group, offset) under the key `seed`: eight half words a counter, in int64."""
    low = 0xFFFFFFFF
    zero = torch.zeros_like(group)
    c0, c1 = group & low, (group >> 32) & low
    c2, c3 = zero + (state[1] & low), zero + ((state[1] >> 32) & low)
    k0, k1 = state[0] & low, (state[0] >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57     # modulo 2^64, which holds the whole product
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).view(-1)


def _draws(count, state):
    group = torch.arange((count + 7) // 8, device=state.device, dtype=torch.int64)
    return ((_philox(group, state) << 16) | _philox(group | -(1 << 63), state))[:count]


def _plain_dropout(st):
    x = st["x"]
    shared = st["shared_dims"]
    lead = x.shape[:x.dim() - shared]
    keep = (_draws(math.prod(lead), st["state"]) >= int(math.floor(st["p"] * 2.0 ** 32 + 0.5))).view(*lead, *[1] * shared)
    scale = 1.0 / (1.0 - st["p"])
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero).to(x.dtype)
    if not st["grad"]:
        return {"y": y}
    return {"y": y, "dx": torch.where(keep, st["dy"].float() * scale, zero).to(x.dtype)}


def _plain_head(st):
    x, w, y = st["x"].float(), st["w"].float(), st["y"]
    s, v = st["smoothing"], st["classes"]
    z = x @ w.t()
    if st["b"] is not None:
        z += st["b"].float()
    top = z.amax(1, keepdim=True)
    live = y != _IGNORE
    at = torch.where(live, y, torch.zeros_like(y)).unsqueeze(1)
    loss = (1 - s) * (top.squeeze(1) - z.gather(1, at).squeeze(1))
    if s:
        loss = loss + s * (top.squeeze(1) - z.mean(1))
    z -= top
    z.exp_()
    total = z.sum(1, keepdim=True)
    loss = torch.where(live, loss + total.squeeze(1).log(), torch.zeros((), device=x.device))
    count = live.sum()
    red = st["reduction"]
    out = {"loss": loss if red == "none" else loss.sum() if red == "sum" else loss.sum() / count}
    if st["grad"]:
        g = st["up"] * live.float()
        if red == "mean":
            g = torch.where(live, g / count, torch.zeros((), device=x.device))
        z /= total
        z.scatter_add_(1, at, torch.full_like(at, s - 1.0, dtype=torch.float32))
        if s:
            z -= s / v
        z *= g.unsqueeze(1)
        out["dx"] = (z @ w).to(st["x"].dtype)
        out["dw"] = (z.t() @ x).to(st["w"].dtype)
        if st["b"] is not None:
            out["db"] = z.sum(0).to(st["b"].dtype)
    return out


@functools.lru_cache(maxsize=None)
def _functions():
    sys.path[:0] = [p for p in [os.path.abspath("deformable-kernels_b200")] if p not in sys.path]
    from deformable_kernels.ops.deform_kernel import functions
    return functions


def _own_dropout(st):
    dropout = _functions().dropout
    if not st["grad"]:
        with torch.no_grad():
            return {"y": dropout(st["x"], st["p"], st["state"], shared_dims=st["shared_dims"])}
    y = dropout(st["x"], st["p"], st["state"], shared_dims=st["shared_dims"])
    return {"y": y.detach(), "dx": torch.autograd.grad(y, st["x"], st["dy"])[0]}


def _own_head(st):
    linear_cross_entropy = _functions().linear_cross_entropy
    kw = dict(bias=st["b"], ignore_index=_IGNORE, reduction=st["reduction"], label_smoothing=st["smoothing"])
    if not st["grad"]:
        with torch.no_grad():
            return {"loss": linear_cross_entropy(st["x"], st["w"], st["y"], **kw)}
    loss = linear_cross_entropy(st["x"], st["w"], st["y"], **kw)
    leaves = [st["x"], st["w"]] + ([st["b"]] if st["b"] is not None else [])
    return dict(zip(("loss", "dx", "dw", "db"), (loss.detach(), *torch.autograd.grad(loss, leaves, st["up"]))))


def run(state):
    if own:
        return (_own_dropout if state["op"] == "dropout" else _own_head)(state)
    with torch.no_grad():
        return (_plain_dropout if state["op"] == "dropout" else _plain_head)(state)


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "dropout":
        n = math.prod(_shape(case))
        passes = 2 if case["grad"] else 1
        return {"bytes": 2 * passes * n * size, "flops": passes * n}
    t, d, v = case["rows"], case["features"], case["classes"]
    read = (t * d + v * d + (v if case["bias"] else 0)) * size
    loss = 4 * (t if case["reduction"] == "none" else 1)
    # a training step reads the same operands once, writes as many gradients, and has two more products of the same size
    return {"bytes": read * (2 if case["grad"] else 1) + 8 * t + loss, "flops": 2 * t * d * v * (3 if case["grad"] else 1)}


def _exact_keep(count, seed, offset, p, device):
    """Philox4x32-10 once more, with the products taken from 16-bit halves."""
    def product(c, m):
        lo, hi = c & 0xFFFF, c >> 16
        a, b = lo * m, hi * m                        # below 2^48
        mid = (a >> 16) + (b & 0xFFFFFFFFFFFF)       # b < 2^48: the sum of the upper parts, below 2^49
        return mid >> 16, ((mid & 0xFFFF) << 16) | (a & 0xFFFF)

    n = -(-count // 8)
    index = torch.arange(n, device=device, dtype=torch.int64)
    draws = torch.zeros(n, 8, device=device, dtype=torch.int64)
    for part in range(2):
        words = [index % (1 << 32), index // (1 << 32) + part * (1 << 31),
                 torch.full_like(index, offset % (1 << 32)), torch.full_like(index, offset >> 32)]
        for r in range(10):
            h0, l0 = product(words[0], 0xD2511F53)
            h1, l1 = product(words[2], 0xCD9E8D57)
            key = ((seed % (1 << 32)) + r * 0x9E3779B9) % (1 << 32), ((seed >> 32) + r * 0xBB67AE85) % (1 << 32)
            words = [h1 ^ words[1] ^ key[0], l1, h0 ^ words[3] ^ key[1], l0]
        for i in range(8):
            half = (words[i // 2] // (1 << 16 * (i % 2))) % (1 << 16)
            draws[:, i] += half * (1 << 16 * (1 - part))
    return (draws >= round(p * (1 << 32))).flatten()[:count]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dropout":
        x = st["x"].detach().double()
        lead = x[(...,) + (0,) * case["shared_dims"]].shape
        keep = _exact_keep(lead.numel(), int(st["state"][0]), int(st["state"][1]), case["p"], x.device)
        keep = keep.reshape(lead + (1,) * case["shared_dims"]).expand_as(x)
        out = {"y": (x / (1 - case["p"])).masked_fill_(~keep, 0)}
        if case["grad"]:
            out["dx"] = (st["dy"].double() / (1 - case["p"])).masked_fill_(~keep, 0)
        return out
    leaves = [st[k].detach().double().requires_grad_(case["grad"]) for k in ("x", "w", "b") if st[k] is not None]
    with torch.enable_grad():
        z = leaves[0] @ leaves[1].t()
        if st["b"] is not None:
            z = z + leaves[2]
        live = st["y"] != _IGNORE
        logp = torch.log_softmax(z, 1)
        picked = -logp[torch.arange(len(z), device=z.device), st["y"].clamp(min=0)]
        each = (picked * (1 - case["smoothing"]) - logp.mean(1) * case["smoothing"]).masked_fill(~live, 0)
        loss = {"none": lambda: each, "sum": each.sum, "mean": lambda: each.sum() / live.sum()}[case["reduction"]]()
    out = {"loss": loss.detach()}
    if case["grad"]:
        out.update(zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, st["up"].double())))
    return out
