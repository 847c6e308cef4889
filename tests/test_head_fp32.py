"""The cases of head_fp32 tell three bf16 pieces from two: a mistake planted in the oracle is found by every one of its bounds."""
import pytest
import torch

import head_fp32 as F
import head_oracle as H


def over(got, out, far, name):
    return ((got[name].double() - out[name]).abs() / far[name].clamp(min=1e-300)).nan_to_num(0).max().item()


@pytest.mark.parametrize("t, d, v", F.SIZES)
def test_bounds_hold_for_24_bits_and_not_for_16(t, d, v):
    for scale, names in ((2.0, ("loss",)), (2.0 ** -6, ("dx", "dw"))):
        x, w, y, b = F.case(t, d, v, scale)
        out, far = F.bounds(x, w, y, b)
        for n, holds in ((3, True), (2, False)):
            got, _ = H.head(F.pieces(x, n).double(), F.pieces(w, n).double(), y, b.double(), torch.tensor(1.0), reduction="sum")
            for name in names:
                assert (over(got, out, far, name) <= 1) == holds, (name, n, over(got, out, far, name))
        # one operand with too few bits is enough
        for args in ((F.pieces(x, 2), w), (x, F.pieces(w, 2))):
            got, _ = H.head(args[0].double(), args[1].double(), y, b.double(), torch.tensor(1.0), reduction="sum")
            assert max(over(got, out, far, name) for name in names) > 1


@pytest.mark.parametrize("t, d, v", F.SIZES)
def test_bounds_do_not_hold_for_16_bits_of_the_logits_gradient(t, d, v):
    x, w, y, b = F.case(t, d, v, 2.0 ** -6)
    out, far = F.bounds(x, w, y, b)
    dz = torch.softmax(x.double() @ w.double().T + b.double(), 1)
    dz[torch.arange(t), y] -= 1
    live = torch.isfinite(b)[:, None]
    for n, holds in ((3, True), (2, False)):
        q = F.pieces(dz.float(), n).double()
        assert (over({"dx": q @ torch.where(live, w, 0 * w).double()}, out, far, "dx") <= 1) == holds
        assert (over({"dw": q.T @ x.double()}, out, far, "dw") <= 1) == holds
