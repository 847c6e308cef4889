"""fp32 calls of the classifier head whose results need all 24 bits of every operand, and bounds that show it.

Every row has two features that are not zero and all but three classes are taken out by a bias of -inf, so every sum has a few
terms and its bound a few roundings.  The last eight bits of every value are such that two bf16 pieces (16 bits) would lose about
2^-18.5 of it, always downwards, and signs are such that nothing cancels: losses add up.
"""
import torch

import head_oracle as H

U, CUT = 2.0 ** -24, 2.0 ** -23   # a rounding; an addition on the tensor cores, which may cut
SIZES = [(5, 72, 40), (12, 1280, 1000), (64, 520, 4099), (200, 1280, 1000), (300, 96, 5000), (33, 33, 65)]


def pieces(v, n):
    """The sum of the n leading bf16 pieces of fp32 values."""
    out, left = torch.zeros_like(v), v
    for _ in range(n):
        p = left.bfloat16().float()
        out, left = out + p, left - p
    return out


def values(n, gen):
    """n fp32 values in [1, 2) that are 2^-19.2 to 2^-18 above their two leading pieces."""
    found = torch.empty(0)
    while found.numel() < n:
        v = 1 + torch.rand(8 * n + 64, generator=gen)
        lost = (v - pieces(v, 2)) / v
        found = torch.cat([found, v[(lost > 2.0 ** -19.2) & (lost < 2.0 ** -17.9)]])
    return found[:n]


def case(t, d, v, scale):
    gen = torch.Generator().manual_seed(t * d + v)
    own = int(torch.randint(0, v, (1,), generator=gen))
    others = torch.tensor([c % v for c in (own + 1, own + v // 2)])
    w = values(v * d, gen).view(v, d).clone()
    w[own].neg_()
    x = torch.zeros(t, d)
    at = torch.rand(t, d, generator=gen).argsort(1)[:, :2]
    x.scatter_(1, at, values(2 * t, gen).view(t, 2) * scale)
    b = torch.full((v,), float("-inf"))
    b[own] = 0.0
    b[others] = 0.0
    return x, w, torch.full((t,), own), b


def bounds(x, w, y, b):
    """The result of the call (the sum of its losses, and its gradients) in 64 bits, and bounds."""
    live = torch.isfinite(b)
    out, _ = H.head(x.double(), w.double(), y, b.double(), torch.tensor(1.0), reduction="sum")
    z = x.double() @ w[live].double().T
    reach = (z.amax(1) - z.amin(1)).max().item()
    fat = (x.double().abs() @ w[live].double().abs().T).amax(1)
    off_z = 5 * CUT * fat                                    # two products, the sum of the small ones, theirs, the products left out
    off_e = 3 * U * reach + 2 * CUT                          # an exponential relative to itself: its argument, ex2
    each = H.head(x.double(), w.double(), y, b.double(), reduction="none")[0]["loss"]
    far = {"loss": (2 * off_z + off_e + 8 * U * (1 + each)).sum()}
    p = torch.softmax(z, 1)
    hit = live[:, None] & (torch.arange(len(b))[:, None] == y[None])
    dz = p - hit[live].T.double()
    off_dz = p * (4 * off_z + 2 * off_e + 8 * U)[:, None] + U + 2 * U * dz.abs()
    rows = (x != 0).sum(0).max().item()

    def bound(value, terms, magnitude, moved):
        return moved + (terms + 5) * CUT * magnitude + 2 * U * value.abs() + 1e-300
    aw, ax = w[live].double().abs(), x.double().abs()
    far["dx"] = bound(out["dx"], 3, dz.abs() @ aw, off_dz @ aw)
    far["dw"] = torch.zeros_like(out["dw"])
    far["dw"][live] = bound(out["dw"][live], rows, dz.abs().T @ ax, off_dz.T @ ax)
    return out, far
