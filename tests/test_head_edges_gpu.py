"""The classifier head on the GPU where its kernels end: ragged tiles, long sums, values at the ends of a type's range, layouts,
second derivatives, waits that run out."""
import pytest
import torch

import head_fp32 as F
import head_oracle as H
from test_head_gpu import DEV, check, functions, make, no_wait_ran_out  # noqa: F401  (the fixture watches every test)

pytestmark = pytest.mark.gpu


def padded(x, w, y, b, rows, classes):
    """The same call with `rows` more rows, which are ignored, and `classes` more classes, which a bias of -inf takes out."""
    t, d = x.shape
    x2 = torch.cat([x, torch.randn(rows, d, generator=torch.Generator().manual_seed(1)).to(x.dtype)])
    w2 = torch.cat([w, torch.randn(classes, d, generator=torch.Generator().manual_seed(2)).to(w.dtype)])
    return x2, w2, torch.cat([y, torch.full((rows,), -100)]), torch.cat([b, torch.full((classes,), float("-inf"), dtype=b.dtype)])


@pytest.mark.parametrize("features", [33, 72, 200])
@pytest.mark.parametrize("rows, classes", [(r, c) for r in (1, 2, 3, 5, 31, 33, 62, 63) for c in (7, 30, 63)] + [(1501, 130), (130, 9001)])
def test_fp32_gradients_of_ragged_tiles_are_those_of_whole_ones(rows, classes, features):
    """The last tile of rows and of classes ends anywhere: nothing that its lanes skip changes what the others store.  The same
    call with whole tiles adds zeros only (ignored rows, classes without a chance): the same bits, call after call.  Short sums,
    and long ones that are split and joined."""
    x, w, y, b, _ = make(rows, features, classes, "fp32", seed=rows + classes)
    more = -rows % 64, -classes % 64

    def grads(x, w, y, b):
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
        loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2], reduction="sum")
        return torch.autograd.grad(loss, leaves)
    want = [t[:n] for t, n in zip(grads(*padded(x, w, y, b, *more)), (rows, classes, classes))]
    for _ in range(3):
        got = grads(x, w, y, b)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    check(x, w, y, b, torch.tensor(1.0), reduction="sum")


def test_more_classes_than_the_kernels_count_are_refused():
    from deformable_kernels._cabi import DkError
    w = torch.zeros(2 ** 31 - 1, 1, dtype=torch.float16, device=DEV)
    x, y = torch.zeros(1, 1, dtype=torch.float16, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    with pytest.raises(DkError, match="unsupported|supported"):
        functions().linear_cross_entropy(x, w, y)
    with pytest.raises(DkError):
        functions().linear_cross_entropy(x.requires_grad_(True), w, y)
    del w
    torch.cuda.empty_cache()


WAITS = """
import sys
sys.path[:0] = [%r, %r]
import torch
from deformable_kernels import _cabi as C
import test_head_gpu as T
ran_out = 0
for rows, features, classes, dtype, kw in %r:
    x, w, y, b, up = T.make(rows, features, classes, dtype, ignored=0.1, reduction="none")
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y, up = y.cuda(), up.cuda()

    def step():
        loss = T.functions().linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="none", **kw)
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves, up))
    assert C.lib.dk_linear_cross_entropy_wait_limit(0) in (1, 2000000000)
    want = step()
    torch.cuda.synchronize()
    before = C.lib.dk_ring_error_status()
    assert C.lib.dk_linear_cross_entropy_wait_limit(1) == 2000000000
    got = step()
    torch.cuda.synchronize()
    after = C.lib.dk_ring_error_status()
    gave_up = [bool(torch.isnan(a).any()) for a in got]
    for a, c in zip(got, want):
        assert not torch.isnan(c).any()
        assert (torch.isnan(a) | (a == c)).all(), (rows, features, classes, dtype)
    assert after == 1 or (before == 0 and not any(gave_up)), (before, after, gave_up)
    if gave_up[0]:
        # what is ignored has no loss, whatever happened; the loss that is NaN has gradients that are
        assert gave_up[1] and gave_up[2] and gave_up[3] and (got[0][y == -100] == 0).all()
    print(rows, features, classes, dtype, gave_up, flush=True)
    ran_out += gave_up[0]
    C.lib.dk_linear_cross_entropy_wait_limit(0)
    assert all(torch.equal(a, c) for a, c in zip(step(), want))      # the next call is none the worse
    C.lib.dk_linear_cross_entropy_wait_limit(1)
assert ran_out
"""


def test_waits_that_run_out_leave_nan_and_a_status():
    """With a limit of a nanosecond the kernels give up where the tensor cores or the copies keep them waiting: every value is
    then NaN or the right one, the status says so, and the process goes on.  Tiles of one SM and of two; the longer the sum
    the longer the wait.  In a process of its own: the status stays."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cases = [(64, 4096, 48, "bf16", {}), (300, 4096, 10000, "bf16", {}), (2 ** 18, 2048, 128, "bf16", {}), (64, 2 ** 17, 48, "fp32", {}),
             (300, 2 ** 15, 1000, "fp32", dict(label_smoothing=0.1))]
    code = WAITS % (os.path.join(root, "deformable-kernels_b200"), os.path.join(root, "tests"), cases)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert out.returncode == 0, (out.stdout[-1000:], out.stderr[-2000:])
    print(out.stdout)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows, features, classes", [(40, 8, 5), (200, 8, 70), (300, 16, 300)])
def test_bias_gradients_are_sums_of_unrounded_values(rows, features, classes, dtype):
    """dz is rounded to 16 bits for the two products, not for the bias gradient: its errors are those of fp32 sums (the
    bound of the same call in fp32) and one rounding of the result.  Few features keep the first below what a rounding of
    every dz would add where a class's dz cancel."""
    x, w, y, b, up = make(rows, features, classes, dtype, seed=rows)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2])
    db, = torch.autograd.grad(loss, leaves[2:], up.to(DEV))
    out, far = H.head(x.float(), w.float(), y, b.float(), up)
    info = torch.finfo(H.DTYPES[dtype])
    bound = far["db"] + info.eps / 2 * out["db"].abs() + info.smallest_normal * info.eps / 2
    assert ((db.cpu().double() - out["db"]).abs() <= bound).all()


@pytest.mark.parametrize("rows, classes, dtype", [(100, 3000, "bf16"), (100, 30000, "bf16"), (300, 20000, "bf16"), (2100, 70000, "bf16"), (70000, 2100, "fp16"),
                                                  (100, 3000, "fp32"), (300, 20000, "fp32"), (2100, 24000, "fp32"), (24000, 2100, "fp32")])
def test_gradients_of_losses_near_zero_in_every_tile_shape(rows, classes, dtype):
    """1 - p of a class that is nearly certain is the difference of the forward's logits and the backward's, which have to be the
    same to the last bit in every shape of tiles, in calls that are cut into pieces too.  Logits of up to 24: one that
    was off by a single step (2^-20) would be 2^-20 / 1e-5 = 10 % of it.  Else the others' probabilities are off by the two
    logits' errors, (64 + 8) 2^-23 24, and 1 - p by three roundings of one; 16-bit dz and results are rounded once each."""
    gen = torch.Generator().manual_seed(rows)
    lift = 11.5 + torch.tensor(float(classes)).log().item()
    y = torch.arange(rows) % 7 * (classes // 7)
    w = torch.randn(classes, 64, generator=gen) * 0.05
    x = torch.randn(rows, 64, generator=gen) * 0.1 + lift * w[y] / w[y].square().sum(1, keepdim=True)
    x, w = (t.to(H.DTYPES[dtype]).to(DEV) for t in (x, w))
    y, b = y.to(DEV), torch.zeros(classes, dtype=x.dtype, device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    loss = functions().linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="sum")
    got = torch.autograd.grad(loss, leaves)
    with torch.no_grad():
        z = x.double() @ w.double().t()
        lse = torch.logsumexp(z, 1)
        dz = z.sub_(lse[:, None]).exp_()
        dz[torch.arange(rows, device=DEV), y] = 0
        rest = dz.sum(1)
        assert 1e-6 < rest.min() and rest.max() < 1e-2
        dz[torch.arange(rows, device=DEV), y] = -rest
        u = 0.0 if dtype == "fp32" else torch.finfo(x.dtype).eps / 2
        tol = 72 * 2.0 ** -23 * 24 * 2 + 2.0 ** -22 / rest.min().item() + 2.1 * u
        for a, c in zip(got, (dz @ w.double(), dz.t() @ x.double(), dz.sum(0))):
            assert (a.double() - c).norm() < tol * c.norm(), ((a.double() - c).norm() / c.norm()).item()
    del z, dz
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [12, 200])
def test_fp32_values_at_the_end_of_the_range(rows):
    """The largest fp32 values are finite as three bf16 pieces too.  x = +-max with w = +-2^-125 in features of their own: logits of
    8 (1 - 2^-24), exact but for the last bit; one product a logit that is not zero."""
    big, classes = torch.finfo(torch.float32).max, 6
    x, w = torch.zeros(rows, 16), torch.zeros(classes, 16)
    for c in range(classes):
        w[c, c] = 2.0 ** -125
    y = torch.arange(rows) % classes
    x[torch.arange(rows), y] = big * (1 - 2 * (torch.arange(rows) // classes % 2)).float()
    b = torch.zeros(classes)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2], reduction="none")
    grads = torch.autograd.grad(loss.mean() * 2.0 ** -10, leaves)
    ref = [t.double().requires_grad_(True) for t in (x, w, b)]
    want = torch.nn.functional.cross_entropy(ref[0] @ ref[1].t() + ref[2], y, reduction="none")
    want_grads = torch.autograd.grad(want.mean() * 2.0 ** -10, ref)
    # a logit of 8 is off by 2^-21, what follows by a few roundings
    assert ((loss.cpu().double() - want).abs() <= 2.0 ** -20 + 2.0 ** -21 * want).all()
    # dz is off by that of itself and by three roundings of one (p - 1); a class's dz cancel in its bias gradient, their errors do not:
    # the bound is of the sum of magnitudes
    with torch.no_grad():
        z = ref[0] @ ref[1].t()
        dz = (torch.softmax(z, 1) - torch.nn.functional.one_hot(y, classes)).abs()
        off = (2.0 ** -19 * dz + 2.0 ** -22) * (2.0 ** -10 / rows)
        for a, c, bound in zip(grads[1:], want_grads[1:], (off.t() @ ref[0].abs(), off.sum(0))):
            assert ((a.cpu().double() - c).abs() <= bound).all()
    # w is of the size of fp32's smallest normal numbers, which a sum of less than that keeps to 2^-149
    assert (grads[0].cpu().double() - want_grads[0]).abs().max() <= 2.0 ** -125 * 2.0 ** -8


@pytest.mark.parametrize("t, d, v", F.SIZES)
def test_fp32_keeps_24_bits_of_every_operand(t, d, v):
    for scale, names in ((2.0, ("loss",)), (2.0 ** -6, ("dx", "dw"))):
        x, w, y, b = F.case(t, d, v, scale)
        out, far = F.bounds(x, w, y, b)
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w)]
        loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), b.to(DEV), reduction="sum")
        got = dict(zip(("loss", "dx", "dw"), (loss.detach(),) + torch.autograd.grad(loss, leaves)))
        with torch.no_grad():
            got["alone"] = functions().linear_cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), b.to(DEV), reduction="sum")
        out["alone"], far["alone"] = out["loss"], far["loss"]
        for name in names + ("alone",) * (scale == 2.0):
            assert ((got[name].cpu().double() - out[name]).abs() <= far[name]).all(), name


def test_dropout_of_nothing_has_a_gradient():
    """An empty batch goes through a training step like any other."""
    f = functions()
    state = torch.tensor([3, 4], device=DEV)
    for seed in (1, state):
        x = torch.zeros(0, 8, device=DEV, requires_grad=True)
        w = torch.ones(3, 8, device=DEV, requires_grad=True)
        y = f.dropout(x, 0.5, seed)
        assert y.requires_grad and y.shape == (0, 8)
        dx, dw = torch.autograd.grad((y @ w.t()).sum(), [x, w])
        assert dx.shape == (0, 8) and (dw == 0).all()
        dx, = torch.autograd.grad(f.dropout(x, 0.5, seed).sum(), x)
        assert dx.shape == (0, 8)


def test_second_derivatives_through_dropout():
    """The gradient of a gradient goes through the mask as well: d/dx of |d/dx (sum of squares of what is kept)|^2."""
    f = functions()
    state = torch.tensor([3, 4], device=DEV)
    for seed in (7, state):
        x = torch.randn(40, 16, device=DEV, dtype=torch.double, requires_grad=True)
        keep = (f.dropout(torch.ones_like(x), 0.25, seed) != 0).detach()
        outcomes = []
        for drop in (lambda t: f.dropout(t, 0.25, seed), lambda t: torch.where(keep, t / 0.75, torch.zeros_like(t))):
            dx, = torch.autograd.grad(drop(x).pow(3).sum(), x, create_graph=True)
            assert dx.requires_grad
            ddx, = torch.autograd.grad(dx.square().sum(), x, create_graph=True)
            dddx, = torch.autograd.grad(ddx.square().sum(), x)
            outcomes.append((dx.detach(), ddx.detach(), dddx))
        for a, c in zip(*outcomes):
            assert torch.allclose(a, c, rtol=1e-13, atol=0)


def test_second_derivatives_of_the_loss_are_refused():
    """Its gradients are no constants: a term made of them raises instead of having no derivative."""
    x, w, y, b, up = (t.to(DEV) for t in make(20, 16, 30, "fp32", seed=2))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(functions().linear_cross_entropy(x, w, y, b), leaves)
    loss = functions().linear_cross_entropy(x, w, y, b)
    got = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(a, c) and a.requires_grad for a, c in zip(got, want))
    for g in got:
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(g.square().sum(), leaves, retain_graph=True, allow_unused=True)
    loss = functions().linear_cross_entropy(x, w, y, b, reduction="none")
    up = torch.ones(20, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(loss, x, up, create_graph=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(dx.sum(), up)
    # asked for and not used: as without it
    functions().linear_cross_entropy(x, w, y, b).backward(create_graph=True)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1]) and torch.equal(b.grad, want[2])
    for t in leaves:
        t.grad = None


def test_autocast_leaves_fp64_alone():
    from deformable_kernels.modules import LinearCrossEntropy
    torch.manual_seed(1)
    head = LinearCrossEntropy(20, 7).to(DEV, torch.float64)
    x, y = torch.randn(30, 20, device=DEV, dtype=torch.float64), torch.randint(0, 7, (30,), device=DEV)
    want = head(x, y)
    for dtype in (torch.float16, torch.bfloat16):
        with torch.autocast("cuda", dtype=dtype):
            got = head(x, y)
        assert got.dtype == torch.float64 and torch.equal(got, want)


@pytest.mark.parametrize("shared", [0, 1, 2, 3])
def test_dropout_module_keeps_the_memory_format(shared):
    """As nn.Dropout does: channels last, transposed batches, planes of a permuted batch; elements that share a draw still do."""
    from deformable_kernels.modules import Dropout
    m = Dropout(0.4, shared_dims=shared)
    base = torch.randn(12, 10, 9, 7, device=DEV)
    views = [base, base.contiguous(memory_format=torch.channels_last), base.transpose(0, 1), base.permute(3, 1, 0, 2), base.permute(1, 0, 3, 2),
             base[:, :1].contiguous(memory_format=torch.channels_last), base[:, :, 2:], base[:1].expand(12, 10, 9, 7)]
    for x in views:
        x = x.detach().requires_grad_(True)
        torch.manual_seed(3)
        y = m(x)
        stock = torch.nn.functional.dropout(x, 0.4)
        # (the stride of a dimension of size one addresses nothing)
        assert y.shape == x.shape and all(a == c or n == 1 for a, c, n in zip(y.stride(), stock.stride(), x.shape))
        keep = y.detach() != 0
        assert torch.equal(y.detach(), torch.where(keep, x.detach() * (1 / 0.6), torch.zeros_like(x)))
        runs = keep.reshape(*x.shape[:4 - shared], -1)
        assert shared == 0 or torch.equal(runs.all(-1), runs.any(-1))
        share = runs[..., 0].float().mean().item()
        assert abs(share - 0.6) < 5 * (0.24 / runs[..., 0].numel()) ** 0.5
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(dx != 0, keep)


@pytest.mark.parametrize("rows, features, classes, dtype", [(64, 2 ** 18, 90, "bf16"), (64, 2 ** 18, 90, "fp16"), (300, 2 ** 16 + 8, 9500, "bf16"), (4, 2 ** 18, 90, "bf16"),
                                                            (40, 2 ** 17 + 3, 64, "bf16"), (150, 4160, 19000, "fp16"), (64, 2 ** 18, 90, "fp32")])
def test_long_sums_of_one_sign(rows, features, classes, dtype):
    """Logits whose products all have the same sign: the tensor cores' additions cut, always downwards.  In registers every 2048
    features (128 additions of 2^-23 at most, then one of 2^-24 each), the sum keeps its precision however long it is."""
    gen = torch.Generator(device=DEV).manual_seed(features)
    share = torch.linspace(0, 1, classes, device=DEV)[:, None]
    w = (torch.rand(1, features, generator=gen, device=DEV) + 0.5) * share * (8.0 / features)
    x = torch.rand(rows, features, generator=gen, device=DEV) + 0.5
    if dtype == "fp16":
        w, x = w * 256, x / 256      # out of the subnormal numbers
    x, w = (t.to(H.DTYPES[dtype]) for t in (x, w))
    y = torch.arange(rows, device=DEV) % 2       # among the smallest logits: the loss is that of the largest
    z = torch.cat([x.double() @ part.double().t() for part in w.split(1000)], 1)
    lse = torch.logsumexp(z, 1)
    want = lse - z.gather(1, y[:, None]).squeeze(1)
    additions = (128 + features // 2048 / 2) * 2.0 ** -23
    tol = 2 * additions * z.amax(1) + 2.0 ** -20 * (1 + lse)
    with torch.no_grad():
        alone = functions().linear_cross_entropy(x, w, y, reduction="none")
    x.requires_grad_(True)
    loss = functions().linear_cross_entropy(x, w, y, reduction="none")
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert ((loss.detach().double() - want).abs() <= tol).all(), ((loss.detach().double() - want).abs() / tol).max().item()
    assert ((alone.double() - want).abs() <= tol).all()
    # and the backward's logits are the same: the gradients are theirs
    dz = torch.exp(z - lse[:, None])
    dz[torch.arange(rows, device=DEV), y] -= 1
    want_dx = sum(dz[:, i:i + 1000] @ w[i:i + 1000].double() for i in range(0, classes, 1000))
    u = torch.finfo(x.dtype).eps / 2
    mag = sum(dz[:, i:i + 1000].abs() @ w[i:i + 1000].double().abs() for i in range(0, classes, 1000))
    assert ((dx.double() - want_dx).abs() <= (2 * tol.max() + u + (classes + 16) * 2.0 ** -23) * mag + u * want_dx.abs() + torch.finfo(x.dtype).smallest_normal).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_long_gradient_sums_of_one_sign(dtype):
    """dw of 2^20 equal rows: without weights p is 1/8 and dz -7/8 or 1/8, exactly, so a class's gradient is a sum of equal terms.
    At most 4096 additions of a sum cut (2^-23 each), its parts are rounded, the result is rounded once."""
    rows, features, classes = 2 ** 20, 8192, 8
    one = (torch.rand(features, generator=torch.Generator().manual_seed(1)) + 1).to(H.DTYPES[dtype]).to(DEV)
    x = one.expand(rows, features).contiguous()
    w = torch.zeros(classes, features, dtype=x.dtype, device=DEV, requires_grad=True)
    y = torch.zeros(rows, dtype=torch.int64, device=DEV)
    loss = functions().linear_cross_entropy(x, w, y)
    dw, = torch.autograd.grad(loss, w)
    dz = torch.full((classes, 1), 0.125, dtype=torch.double, device=DEV)
    dz[0] -= 1
    tol = 4096 * 2.0 ** -23 + 300 * 2.0 ** -24 + torch.finfo(x.dtype).eps / 2
    want = dz * one.double()
    assert ((dw.double() - want).abs() <= tol * want.abs()).all(), ((dw.double() - want).abs() / want.abs()).max().item()
    del x
    torch.cuda.empty_cache()


def test_features_in_the_millions():
    """2^23 + 3 features (one bf16 row of 17 MB): the loss and its gradients against fp64."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    d = 2 ** 23 + 3
    for rows in (2, 9):
        x = (torch.randn(rows, d, generator=gen, device=DEV)).bfloat16()
        w = (torch.randn(3, d, generator=gen, device=DEV) * 2.0 ** -11).bfloat16()
        y = torch.arange(rows, device=DEV) % 3
        leaves = [x.requires_grad_(True), w.requires_grad_(True)]
        loss = functions().linear_cross_entropy(x, w, y, reduction="none")
        dx, dw = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        xd, wd = x.detach().double(), w.detach().double()
        z = xd @ wd.t()
        want = torch.nn.functional.cross_entropy(z, y, reduction="none")
        # sums of 2^23 random terms of 2^-11: magnitudes of 2^23 2^-11 2 / pi, of which 128 additions cut at a time; two logits a loss
        off = 2 * (128 * 2.0 ** -23 * 2.0 ** 11 / 2048 + 4096 * 2.0 ** -24 * 4) + 2.0 ** -20
        assert ((loss.detach().double() - want).abs() <= off * (1 + want)).all(), (loss.detach().double() - want).abs().max().item()
        dz = torch.softmax(z, 1)
        dz[torch.arange(rows), y] -= 1
        for a, c in ((dx, dz @ wd), (dw, dz.t() @ xd)):
            assert (a.double() - c).norm() <= (2.0 ** -7 + 4 * off) * c.norm()


@pytest.mark.parametrize("rows, classes", [(9, 2), (40, 2), (200, 2), (200, 3000)])
def test_fp32_sums_are_cut_no_more_than_sixteen_times(rows, classes):
    """A one and then small products, one for every addition of the tensor cores, each a little less than the last bit of the sum so
    far: a cut loses it whole.  Of 32 such additions sixteen may meet in one accumulator before sums that round take over;
    the exact logit is 1 + 31 (255 / 256) 2^-23.  The loss of the other class, log(classes - 1 + e^z), moves by less than
    the logit and is rounded in four places."""
    x, w = torch.zeros(rows, 512), torch.zeros(classes, 512)
    x[:, ::16], w[0, ::16] = 2.0 ** -11, 2.0 ** -12 * 255 / 256
    x[:, 0], w[0, 0] = 1.0, 1.0
    y = torch.ones(rows, dtype=torch.int64)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w)]
    loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), reduction="none").detach().cpu().double()
    z = 1 + 31 * (255 / 256) * 2.0 ** -23
    want = torch.log(torch.tensor(classes - 1 + torch.exp(torch.tensor(z, dtype=torch.double)).item(), dtype=torch.double)).item()
    share = torch.exp(torch.tensor(z, dtype=torch.double)).item() / torch.exp(torch.tensor(want, dtype=torch.double)).item()
    assert ((loss - want).abs() <= share * 16 * 2.0 ** -23 + 4 * 2.0 ** -24 * want).all(), ((loss - want).abs().max().item() * 2 ** 23, share)


@pytest.mark.parametrize("rows", [3, 60])
@pytest.mark.parametrize("dtype", list(H.DTYPES))
def test_weights_that_are_not_finite(dtype, rows):
    """A logit of -inf takes its class out of the row; in fp32, whose pieces of an infinity are not finite, the loss may be NaN
    instead.  +inf and NaN make NaN."""
    x, w, y, b, _ = make(rows, 40, 30, dtype, seed=rows)
    y[y == 7] = 8
    out = torch.nn.functional.cross_entropy(*[(x.double() @ w.double().t() + b.double())[:, [i for i in range(30) if i != 7]], y - (y > 7).long()],
                                            reduction="none")
    for bad in (float("inf"), float("-inf"), float("nan")):
        w2 = w.clone()
        w2[7, 11] = bad
        loss = functions().linear_cross_entropy(x.to(DEV), w2.to(DEV), y.to(DEV), b.to(DEV), reduction="none").cpu().double()
        gone = x[:, 11].double() * bad == float("-inf")
        assert torch.isnan(loss[~gone]).all()
        right = (loss - out).abs() < 1e-4 * (1 + out)
        assert (right | (torch.isnan(loss) if dtype == "fp32" else torch.zeros_like(right)))[gone].all()


@pytest.mark.parametrize("dtype", ["fp16", "fp32", "fp64"])
def test_dropout_of_runs_on_both_sides_of_the_rule(dtype):
    for run in (8, 248, 256, 312, 320, 328, 384, 1016, 1024, 1032, 2056):
        x = torch.randn(37, run, generator=torch.Generator().manual_seed(run)).to(H.DTYPES[dtype])
        assert torch.equal(functions().dropout(x.to(DEV), 0.3, 9, 2, shared_dims=1).cpu(), H.dropout(x, 0.3, 9, 2, 1))
