"""The classifier head without a GPU: the oracle's own checks, refusals, modules."""
import ctypes

import numpy as np
import pytest
import torch

import head_oracle as H


def test_generator_of_the_oracle_gives_the_published_answers():
    def words(c, k):
        return [int(w[0]) for w in H.philox([[v] for v in c], k)]
    assert words([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_oracle_draws_have_the_right_share_and_no_common_bits():
    d = H.draws(np.arange(1 << 16, dtype=np.uint64), 5, 9)
    # 2^16 draws: the share below p is off by less than five standard deviations
    for p in (0.01, 0.2, 0.5, 0.9):
        share = float((d < np.uint64(p * 2 ** 32)).mean())
        assert abs(share - p) < 5 * (p * (1 - p) / 2 ** 16) ** 0.5
    assert len(np.unique(d)) > 65000
    assert not np.array_equal(d, H.draws(np.arange(1 << 16, dtype=np.uint64), 5, 10))


@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_oracle_head_is_torchs(smoothing, reduction):
    torch.manual_seed(0)
    x, w, b = (torch.randn(*s, dtype=torch.double, requires_grad=True) for s in ((7, 5), (11, 5), (11,)))
    y = torch.randint(0, 11, (7,))
    y[3] = -100
    loss = torch.nn.functional.cross_entropy(x @ w.T + b, y, reduction=reduction, label_smoothing=smoothing)
    up = torch.rand_like(loss)
    out, far = H.head(x.detach(), w.detach(), y, b.detach(), up, reduction=reduction, label_smoothing=smoothing)
    got = (loss,) + torch.autograd.grad(loss, [x, w, b], up)
    for name, v in zip(("loss", "dx", "dw", "db"), got):
        assert torch.allclose(out[name], v.detach(), rtol=1e-12, atol=1e-14), name
        assert far[name].shape == out[name].shape


def _functions():
    from deformable_kernels.ops.deform_kernel import functions
    return functions


def test_cpu_tensors_are_refused():
    f = _functions()
    with pytest.raises(NotImplementedError):
        f.dropout(torch.zeros(4), 0.5, 1)
    with pytest.raises(NotImplementedError):
        f.linear_cross_entropy(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))


def test_arguments_of_the_wrong_kind_are_refused():
    f = _functions()
    with pytest.raises(TypeError):
        f.dropout([1.0], 0.5, 1)
    with pytest.raises(TypeError):
        f.dropout(torch.zeros(4), 0.5, 1.5)
    with pytest.raises(TypeError):
        f.linear_cross_entropy(torch.zeros(2, 4), torch.zeros(3, 4), [0, 1])
    with pytest.raises(ValueError):
        f.linear_cross_entropy(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64), reduction="batchmean")


def test_library_refuses_bad_calls_before_any_launch():
    from deformable_kernels import _cabi as C
    one, null = ctypes.c_void_p(16), ctypes.c_void_p(0)

    def drop(x=one, y=one, count=8, run=1, p=0.5, dtype=0, state=null, used=null):
        return C.lib.dk_dropout(x, y, count, run, p, 0, 0, state, used, dtype, null)
    assert drop(x=null) == 1 and drop(y=null) == 1 and drop(count=0) == 1 and drop(run=0) == 1 and drop(dtype=4) == 1
    assert drop(p=-0.1) == 1 and drop(p=1.1) == 1 and drop(p=float("nan")) == 1
    assert drop(state=ctypes.c_void_p(12)) == 1 and drop(state=one, used=ctypes.c_void_p(20)) == 1 and drop(used=one) == 1

    def forward(x=one, w=one, y=one, loss=one, rows=2, features=8, classes=3, reduction=1, smoothing=0.0, dtype=0, ws=null, size=0):
        return C.lib.dk_linear_cross_entropy_forward(x, w, null, y, loss, null, rows, features, classes, -100, reduction, smoothing, dtype,
                                                     ws, size, null)
    for bad in (dict(x=null), dict(w=null), dict(y=null), dict(loss=null), dict(rows=0), dict(features=0), dict(classes=0), dict(reduction=3),
                dict(reduction=-1), dict(smoothing=-0.1), dict(smoothing=1.5), dict(smoothing=float("nan")), dict(dtype=4)):
        assert forward(**bad) == 1, bad
    assert forward(x=ctypes.c_void_p(24)) == 1 and forward(ws=ctypes.c_void_p(24), size=1 << 30) == 1
    assert forward() == 3 and forward(ws=one, size=16) == 3                                   # no workspace, too little

    def backward(up=one, saved=one, dtype=0, ws=null, size=0, rows=2):
        return C.lib.dk_linear_cross_entropy_backward(up, one, one, null, one, saved, one, one, null, rows, 8, 3, -100, 1, 0.0, dtype,
                                                      ws, size, null)
    assert backward(up=null) == 1 and backward(saved=null) == 1 and backward(dtype=9) == 1 and backward(rows=-1) == 1
    assert backward() == 3 and backward(ws=one, size=16) == 3
    for q in (C.lib.dk_linear_cross_entropy_forward_workspace_bytes, C.lib.dk_linear_cross_entropy_backward_workspace_bytes):
        assert q(0, 8, 3, 0) == 0 and q(2, 8, 3, 7) == 0 and q(2, 8, 3, C.DK_BF16) > 0


def test_workspace_does_not_grow_with_the_vocabulary_like_logits():
    from deformable_kernels import _cabi as C
    rows, features, classes = 16384, 1280, 262144
    logits = rows * classes * 2
    assert C.lib.dk_linear_cross_entropy_backward_workspace_bytes(rows, features, classes, C.DK_BF16) < logits // 8
    assert C.lib.dk_linear_cross_entropy_forward_workspace_bytes(rows, features, classes, C.DK_BF16) < logits // 8


def test_modules_have_the_stock_parameters():
    from deformable_kernels.modules import Dropout, LinearCrossEntropy
    torch.manual_seed(3)
    head = LinearCrossEntropy(12, 5, dropout=0.2, label_smoothing=0.1)
    stock = torch.nn.Linear(12, 5)
    head.load_state_dict(stock.state_dict())
    x = torch.randn(3, 12)
    head.eval()
    assert torch.equal(head(x), stock(x))                        # logits need no kernel of ours
    assert "label_smoothing=0.1" in repr(head)
    d = Dropout(0.3, shared_dims=2)
    assert d.eval()(x) is x and Dropout(0.0)(x) is x
    assert not list(d.state_dict()) and not list(d.buffers())
    with pytest.raises(ValueError):
        Dropout(1.5)
