"""Plain implementations in 64 bits of the classifier head's operators, and how far a kernel may be from them.

A rounding to a type is off by at most u = finfo(type).eps / 2 relative to the value (2^-24, 2^-11, 2^-8), or half of its
smallest subnormal.  The fp32 sums of the kernels are those of the tensor cores, whose additions may cut instead of
round: 2^-23 of the magnitudes for each addition.
"""
import math

import numpy as np
import torch

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "fp64": torch.float64}


# ------------------------------------------------------------------ dropout

def philox(counter, key):
    """Philox4x32-10 on uint64 arrays that hold 32-bit words: counter [4][n], key (k0, k1) -> [4][n]."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = list(key)
    mask = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(index, seed, offset):
    """The 32-bit draws of the given indices (uint64 array)."""
    index = np.asarray(index, dtype=np.uint64)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    group, i = index >> np.uint64(3), (index & np.uint64(7)).astype(np.int64)
    out = np.zeros(index.shape, dtype=np.uint64)
    for part in range(2):
        w = philox([group & np.uint64(0xFFFFFFFF), (group >> np.uint64(32)) | np.uint64(part << 31),
                    np.full_like(index, offset & 0xFFFFFFFF), np.full_like(index, offset >> 32)],
                   (seed & 0xFFFFFFFF, seed >> 32))
        word = np.choose(i // 2, w)
        half = (word >> (np.uint64(16) * (i % 2).astype(np.uint64))) & np.uint64(0xFFFF)
        out |= half << np.uint64(16 * (1 - part))
    return out


def keep_mask(shape, p, seed, offset, shared_dims=0):
    lead = tuple(shape[:len(shape) - shared_dims])
    n = int(np.prod(lead, dtype=np.int64)) if lead else 1
    keep = draws(np.arange(n, dtype=np.uint64), seed, offset) >= np.uint64(math.floor(p * 2.0 ** 32 + 0.5))
    return torch.from_numpy(keep).reshape(lead + (1,) * shared_dims).expand(shape)


def dropout(x, p, seed, offset=0, shared_dims=0):
    """The operator's definition, rounding included (one product with the reciprocal in the arithmetic type)."""
    keep = keep_mask(x.shape, p, seed, offset, shared_dims)
    a = x if x.dtype == torch.float64 else x.float()
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=a.dtype)
    return torch.where(keep, a * scale, torch.zeros((), dtype=a.dtype)).to(x.dtype)


# ------------------------------------------------------------------ linear layer + cross entropy

def head(x, w, y, b=None, up=None, ignore_index=-100, reduction="mean", label_smoothing=0.0, device="cpu"):
    """Loss and gradients in 64 bits, and the bounds of their errors: ({name: value}, {name: bound}), on the CPU; `device`:
    where they are computed."""
    with torch.device(device):
        out, far = _head(x.to(device), w.to(device), y.to(device), b.to(device) if b is not None else None,
                         up.to(device) if up is not None else None, ignore_index, reduction, label_smoothing)
    return {k: v.cpu() for k, v in out.items()}, {k: v.cpu() for k, v in far.items()}


def _head(x, w, y, b, up, ignore_index, reduction, label_smoothing):
    dtype = x.dtype
    x, w = x.double(), w.double()
    b = b.double() if b is not None else None
    t, d = x.shape
    v = w.shape[0]
    s = label_smoothing
    live = y != ignore_index
    xs = torch.where(live[:, None], x, torch.zeros((), dtype=torch.double))    # an ignored row has no say at all
    z = xs @ w.T + (b if b is not None else 0)
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, y, torch.zeros_like(y))
    each = lse - (1 - s) * z.gather(1, at[:, None]).squeeze(1)
    if s:
        each = each - s * z.mean(1)
    each = torch.where(live, each, torch.zeros((), dtype=torch.double))
    count = live.sum().double()
    out = {"loss": each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / count}
    exact64 = dtype == torch.float64
    step = 2.0 ** -52 if exact64 else 2.0 ** -23
    # logits: d products and sums, the bias, the change to base 2 (8 roundings); the largest of a row bounds its lse
    fat = xs.abs() @ w.abs().T + (b.abs() if b is not None else 0)
    fat = torch.where(torch.isfinite(fat), fat, torch.zeros((), dtype=torch.double))
    dz_err = ((d + 8) * step * fat).amax(1) + 8 * step * (1 + lse.abs().nan_to_num(0, 0, 0))
    # the row's sum of exponentials: v additions and two roundings of each exponential
    row_err = 3 * dz_err + (min(v, 512) + 8) * step
    row_err = torch.where(live, row_err, torch.zeros((), dtype=torch.double))
    far = {"loss": row_err + 4 * step * each.abs() if reduction == "none" else
           (row_err + 4 * step * each.abs()).sum() / (count if reduction == "mean" else 1)}
    if up is None:
        return out, far
    up = up.double()
    g = torch.where(live, up / count if reduction == "mean" else up * torch.ones(t, dtype=torch.double), torch.zeros((), dtype=torch.double))
    p = torch.exp(z - lse[:, None])
    dz = p - s / v
    dz[torch.arange(t), at] -= 1 - s
    dz = torch.where(live[:, None], dz * g[:, None], torch.zeros((), dtype=torch.double))
    out["dx"], out["dw"] = dz @ w, dz.T @ xs
    u = 0.0 if exact64 else torch.finfo(dtype).eps / 2
    tiny = 0.0 if dtype != torch.float16 else 2.0 ** -25
    # dz: its own error from the logits, and its rounding to the operand type (fp16 is scaled so that the largest g has 2^14)
    gmax = g.abs().max().item() if t else 0.0
    dz_far = (p * row_err[:, None] + 4 * step) * g.abs()[:, None] + u * dz.abs() + tiny * gmax / 2 ** 13
    dz_far = torch.where(live[:, None], dz_far, torch.zeros((), dtype=torch.double))
    aw, ax = w.abs(), xs.abs()

    def bound(value, k, magnitude, moved):
        return 1.01 * (moved + (k + 16) * step * magnitude + (u + 2.0 ** -40 if not exact64 else step) * value.abs()) + tiny + 1e-300
    far["dx"] = bound(out["dx"], v, dz.abs() @ aw, dz_far @ aw)
    far["dw"] = bound(out["dw"], t, dz.abs().T @ ax, dz_far.T @ ax)
    if b is not None:
        out["db"] = dz.sum(0)
        far["db"] = bound(out["db"], t, dz.abs().sum(0), dz_far.sum(0))
    return out, far
