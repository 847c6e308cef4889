"""The classifier head on the GPU: dropout bit by bit, the loss and its gradients within derived bounds."""
import pytest
import torch
import torch.utils.checkpoint

import head_oracle as H

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def functions():
    from deformable_kernels.ops.deform_kernel import functions as f
    return f


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from deformable_kernels import _cabi
    assert _cabi.lib.dk_ring_error_status() == 0


# ------------------------------------------------------------------ dropout

@pytest.mark.parametrize("dtype", list(H.DTYPES))
@pytest.mark.parametrize("shape, shared", [((1,), 0), ((7,), 0), ((8,), 0), ((9, 3), 1), ((300, 1001), 0), ((5, 6, 7, 9), 2), ((5, 6, 7, 9), 3),
                                           ((4, 3, 64, 64), 2), ((3, 7, 8, 32), 2), ((2, 5, 41, 40), 2), ((6, 3, 40, 40), 3), ((3, 5, 2), 1), ((2, 3), 2), ((), 0)])
def test_dropout_is_its_definition(shape, shared, dtype):
    torch.manual_seed(1)
    x = torch.randn(shape).to(H.DTYPES[dtype])
    dy = torch.randn(shape).to(H.DTYPES[dtype])
    for p, seed, offset in ((0.2, 12345, 0), (0.5, 2 ** 63 + 17, 2 ** 40 + 3)):
        xg = x.to(DEV).requires_grad_(True)
        y = functions().dropout(xg, p, seed, offset, shared_dims=shared)
        dx, = torch.autograd.grad(y, xg, dy.to(DEV))
        assert y.dtype == x.dtype and y.shape == x.shape
        assert torch.equal(y.detach().cpu(), H.dropout(x, p, seed, offset, shared))
        assert torch.equal(dx.cpu(), H.dropout(dy, p, seed, offset, shared))


def test_dropout_looks_at_the_lower_half_where_the_upper_is_the_thresholds():
    n = 1 << 19
    x = torch.ones(n, device=DEV)
    for p in (0.3, 1e-6, 2.0 ** -16, 1 - 2.0 ** -16, 2.0 ** -32):
        assert torch.equal(functions().dropout(x, p, 77, 5).cpu(), H.dropout(torch.ones(n), p, 77, 5))
    assert torch.equal(functions().dropout(x, 0.0, 1), x)
    assert not functions().dropout(x, 1.0, 1).any()


def test_dropout_of_values_that_are_not_finite_is_zero_where_dropped():
    x = torch.tensor([float("inf"), float("nan"), float("-inf"), 1.0] * 64)
    keep = H.keep_mask(x.shape, 0.5, 3, 0)
    for t in (x, x.half()):
        y = functions().dropout(t.to(DEV), 0.5, 3).cpu()
        assert (y[~keep] == 0).all()
        assert torch.equal(y[keep].isnan(), t[keep].isnan()) and torch.equal(y[keep].isinf(), t[keep].isinf())


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_dropout_of_views(dtype):
    base = torch.randn(6, 40, 33).to(H.DTYPES[dtype])
    for view in (lambda t: t[:, 1:, 3:], lambda t: t.transpose(0, 2), lambda t: t.flatten()[1:], lambda t: t[:, :1].expand(6, 5, 33)):
        y = functions().dropout(view(base.to(DEV)), 0.3, 4)
        assert torch.equal(y.cpu(), H.dropout(view(base).contiguous(), 0.3, 4))


def test_dropout_state_on_the_device_and_replayed_graphs():
    x = torch.randn(1000, device=DEV)
    state = torch.tensor([99, 10], device=DEV)
    want = [H.dropout(x.cpu(), 0.4, 99, 10 + i) for i in range(6)]
    assert torch.equal(functions().dropout(x, 0.4, state).cpu(), want[0])
    assert torch.equal(functions().dropout(x, 0.4, state, 2).cpu(), want[2])
    # the backward draws what its forward drew, although the state has moved on
    xg = x.clone().requires_grad_(True)
    y = functions().dropout(xg, 0.4, state)
    state[1] += 1
    dx, = torch.autograd.grad(y, xg, x)
    assert torch.equal(y.detach().cpu(), want[0]) and torch.equal(dx.cpu(), want[0])

    # captured: what the tensor holds at each replay
    state.copy_(torch.tensor([99, 10]))
    xs = x.clone().requires_grad_(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = functions().dropout(xs, 0.4, state)
        state[1] += 1
        dx, = torch.autograd.grad(y, xs, x)
    for i in range(3):
        g.replay()
        assert torch.equal(y.detach().cpu(), want[i]) and torch.equal(dx.cpu(), want[i])


def test_dropout_module_draws_from_torchs_generator():
    from deformable_kernels.modules import Dropout
    m = Dropout(0.4, shared_dims=1)
    x = torch.randn(200, 3, device=DEV)

    def run(seed, f=m):
        torch.manual_seed(seed)
        xs = x.clone().requires_grad_(True)
        y = f(xs)
        return y.detach(), torch.autograd.grad(y, xs, x)[0]
    (a, ga), (b, gb), (c, _) = run(5), run(5), run(6)
    assert torch.equal(a, b) and torch.equal(ga, gb) and torch.equal(a, ga) and not torch.equal(a, c)
    # a checkpointed call makes the same mask again for its backward
    d, gd = run(5, lambda t: torch.utils.checkpoint.checkpoint(m, t, use_reentrant=False))
    assert torch.equal(a, d) and torch.equal(a, gd)
    # replays draw anew, and their backwards what they drew
    xs = x.clone().requires_grad_(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(xs)
        dx, = torch.autograd.grad(y, xs, x)
    seen = []
    for _ in range(3):
        g.replay()
        assert torch.equal(y, dx)
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_dropout_beyond_32_bits():
    """2^33 + 24 elements: the index of a draw and the offsets of elements pass 32 bits, the launch is split."""
    n = 2 ** 33 + 24
    x = torch.ones(n, device=DEV, dtype=torch.float16)
    y = functions().dropout(x, 0.3, 11, 2 ** 35 + 1)
    index = torch.cat([torch.arange(64), torch.arange(2 ** 32 - 32, 2 ** 32 + 32), torch.arange(2 ** 33 - 32, n)])
    keep = torch.from_numpy(H.draws(index.numpy(), 11, 2 ** 35 + 1).astype("int64")) >= int(0.3 * 2 ** 32 + 0.5)
    assert torch.equal(y[index.to(DEV)].cpu() != 0, keep)
    del x, y
    torch.cuda.empty_cache()


def test_dropout_refusals():
    f = functions()
    x = torch.zeros(4, 4, device=DEV)
    for kw in (dict(p=1.5), dict(p=-0.5), dict(p=float("nan")), dict(shared_dims=3), dict(shared_dims=-1),
               dict(seed=torch.zeros(3, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            f.dropout(x, **kw)
    with pytest.raises(TypeError):
        f.dropout(x, 0.5, torch.zeros(2, device=DEV))
    with pytest.raises(TypeError):
        f.dropout(x.int(), 0.5, 1)
    with pytest.raises(NotImplementedError):
        f.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    assert f.dropout(x[:0], 0.5, 1).shape == (0, 4)


# ------------------------------------------------------------------ linear layer + cross entropy

def make(t, d, v, dtype, bias=True, ignored=0.0, reduction="mean", seed=0):
    gen = torch.Generator().manual_seed(seed)
    dt = H.DTYPES[dtype]
    w = (torch.randn(v, d, generator=gen) * (1.5 / d ** 0.5)).to(dt)
    y = torch.randint(0, v, (t,), generator=gen)
    x = (torch.randn(t, d, generator=gen) + 3 * torch.rand(t, 1, generator=gen) * w[y].float()).to(dt)
    b = (torch.randn(v, generator=gen) * 0.1).to(dt) if bias else None
    if ignored:
        y = torch.where(torch.rand(t, generator=gen) < ignored, torch.full_like(y, -100), y)
    scale = 1024.0 if dtype == "fp16" else 1.0
    up = torch.rand(t, generator=gen) * scale if reduction == "none" else torch.tensor(scale / (t if reduction == "sum" else 1))
    return x, w, y, b, up.double() if dtype == "fp64" else up


def check(x, w, y, b, up, where="", device="cpu", **kw):
    """One call and its gradients against the 64-bit oracle, every value within its bound."""
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b) if t is not None]
    loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2] if b is not None else None, **kw)
    grads = torch.autograd.grad(loss, leaves, up.to(DEV))
    out, far = H.head(x, w, y, b, up, device=device, **kw)
    got = dict(zip(("loss", "dx", "dw", "db"), (loss.detach(),) + grads))
    assert loss.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    for name, v in got.items():
        v = v.cpu()
        assert v.dtype == (loss.dtype if name == "loss" else x.dtype) and v.shape == out[name].shape, name
        assert torch.isfinite(v).all() == torch.isfinite(out[name]).all(), (where, name)
        over = ((v.double() - out[name]).abs() / far[name]).nan_to_num(0).max().item() if v.numel() else 0
        assert over <= 1, (where, name, over, (v.double() - out[name]).abs().max().item(), out[name].abs().max().item())
    with torch.no_grad():
        again = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2] if b is not None else None, **kw)
    if x.shape[0] > 8:  # a few rows without a backward are summed in another order
        assert torch.equal(again, loss.detach()) or not torch.isfinite(again).all()
    else:
        over = ((again.cpu().double() - out["loss"]).abs() / far["loss"]).nan_to_num(0).max().item()
        assert over <= 1 and again.shape == loss.shape and torch.isfinite(again).all() == torch.isfinite(out["loss"]).all(), (where, over)
    return got


SIZES = [(1, 8, 2), (2, 100, 5000), (3, 256, 1200), (4, 72, 4800), (5, 64, 5001), (8, 33, 700), (1, 1280, 1000), (2, 1, 1), (31, 24, 7), (33, 33, 65), (127, 64, 130), (128, 128, 256), (129, 200, 257), (300, 96, 1000),
         (257, 65, 1031), (64, 520, 4099), (1030, 40, 64)]


@pytest.mark.parametrize("dtype", list(H.DTYPES))
@pytest.mark.parametrize("t, d, v", SIZES)
def test_head_sizes(t, d, v, dtype):
    check(*make(t, d, v, dtype, seed=t + d + v))


# tiles shared by two SMs, in one or all products; several pieces of the classes, of the rows; long sums that are split
LARGE = [(2100, 72, 5000), (1500, 520, 4600), (3000, 136, 24100), (24100, 40, 3001), (9000, 64, 40), (20, 72, 30000), (4700, 1032, 600), (1100, 1280, 1000),
         (700, 256, 2100), (100, 264, 11000)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("t, d, v", LARGE)
def test_head_large_sizes(t, d, v, dtype):
    check(*make(t, d, v, dtype, ignored=0.1, seed=t + d + v), device=DEV, label_smoothing=0.1)


@pytest.mark.parametrize("dtype", list(H.DTYPES))
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
def test_head_options(dtype, reduction, smoothing):
    for bias, ignored in ((True, 0.0), (False, 0.3)):
        check(*make(150, 72, 203, dtype, bias, ignored, reduction, seed=5), reduction=reduction, label_smoothing=smoothing)


@pytest.mark.parametrize("dtype", list(H.DTYPES))
def test_ignored_rows_have_no_say_whatever_they_hold(dtype):
    x, w, y, b, up = make(140, 48, 90, dtype, ignored=0.4, seed=6)
    dead = y == -100
    clean = check(x, w, y, b, up)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(x.dtype).max):
        x2 = x.clone()
        x2[dead] = bad
        dirty = check(x2, w, y, b, up)
        for k in clean:
            assert torch.equal(clean[k], dirty[k]), (k, bad)
    y2 = torch.where(dead, torch.full_like(y, 255), y)
    other = check(x, w, y2, b, up, ignore_index=255)
    assert all(torch.equal(clean[k], other[k]) for k in clean)


@pytest.mark.parametrize("dtype", list(H.DTYPES))
def test_all_rows_ignored(dtype):
    x, w, y, b, up = make(40, 16, 10, dtype)
    y[:] = -100
    for reduction, want in (("mean", float("nan")), ("sum", 0.0), ("none", 0.0)):
        u = up if reduction != "none" else up * torch.ones(40, dtype=up.dtype)
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
        loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2], reduction=reduction)
        grads = torch.autograd.grad(loss, leaves, u.to(DEV))
        assert torch.isnan(loss).all() if want != want else (loss == want).all()
        assert all((g == 0).all() for g in grads)


@pytest.mark.parametrize("dtype", list(H.DTYPES))
def test_classes_taken_out_by_an_infinite_bias(dtype):
    x, w, y, b, up = make(70, 40, 300, dtype, seed=8)
    out = torch.rand(300, generator=torch.Generator().manual_seed(1)) < 0.5
    out[y] = False
    out[64:192] = True
    y[y >= 64] = int((~out).nonzero()[0])
    b[out] = float("-inf")
    b[y] = 0.0
    check(x, w, y, b, up)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_targets_that_are_no_class_make_the_loss_nan(dtype):
    x, w, y, b, up = make(130, 40, 30, dtype, reduction="none")
    for wrong in (30, -1, 2 ** 40, -(2 ** 62)):
        y2 = y.clone()
        y2[7] = wrong
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
        loss = functions().linear_cross_entropy(leaves[0], leaves[1], y2.to(DEV), leaves[2], reduction="none")
        dx, dw, db = torch.autograd.grad(loss, leaves, up.to(DEV))
        bad = torch.isnan(loss)
        assert bad[7] and int(bad.sum()) == 1
        assert torch.isnan(dx[7]).all() and torch.isfinite(dx[8:]).all() and torch.isfinite(dx[:7]).all()
        assert torch.isnan(dw).all() and torch.isnan(db).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_rows_with_features_that_are_not_finite_keep_to_themselves(dtype):
    x, w, y, b, up = make(130, 40, 300, dtype, reduction="none")
    x[5, 3], x[77, 0] = float("nan"), float("inf")
    loss = functions().linear_cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), b.to(DEV), reduction="none").cpu()
    bad = torch.isnan(loss)
    assert bad[5] and bad[77] and int(bad.sum()) == 2


def test_large_and_small_logits():
    """Logits of a few hundred: the sum of exponentials is taken from the largest one."""
    for dtype in H.DTYPES:
        x, w, y, b, up = make(50, 64, 200, dtype, seed=3)
        check(x * 16, w * 4, y, b, up)
        check(x * 0, w, y, b, up)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 40])
def test_losses_near_zero(rows, dtype):
    """The row's own logit far above the others: the loss is log(1 + e), not the difference of two large numbers.  Logits are
    whole numbers (exact), e is off by 2^-22 of itself, 1 + e by 2^-24, its logarithm by 2^-23 of itself and twice that
    in steps; 60 losses of a sum change nothing, the mean is one of equal values."""
    for gap in (3.0, 8.0, 11.0):
        x = torch.zeros(rows, 16)
        x[:, 0] = 1.0
        w = torch.zeros(2, 16)
        w[0, 0], w[1, 0] = 20.0, 20.0 - gap
        y = torch.zeros(rows, dtype=torch.int64)
        dt = H.DTYPES[dtype]
        got = functions().linear_cross_entropy(x.to(dt).to(DEV), w.to(dt).to(DEV), y.to(DEV)).item()
        want = torch.log1p(torch.exp(torch.tensor(-gap, dtype=torch.double))).item()
        assert abs(got - want) < 2.0 ** -23 + 2.0 ** -21 * want


@pytest.mark.parametrize("rows", [1, 3, 8, 40])
def test_gradients_of_losses_near_zero(rows):
    """p - 1 of a class that is nearly certain: it takes the backward's logits to be the forward's.  fp32 features whose
    products are not exact; dz is off by the logits' error relative to itself (1e-5 at these sizes, 64 products of a
    few units) and by three roundings of one, 2^-22, against 1 - p."""
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 64, generator=gen)
    y = torch.arange(rows) % 4
    for lift in (9.0, 11.0):
        w = torch.randn(5, 64, generator=gen) * 0.05
        x2 = x.clone()
        b = torch.zeros(5)
        # the row's own class lifted through its features: x . w_y = lift, about nothing for the others
        for t in range(rows):
            x2[t] = x[t] * 0.1 + lift * w[y[t]] / w[y[t]].square().sum()
        leaves = [t.to(DEV).requires_grad_(True) for t in (x2, w, b)]
        loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2])
        got = torch.autograd.grad(loss, leaves)
        ref = [t.double().requires_grad_(True) for t in (x2, w, b)]
        z = ref[0] @ ref[1].t() + ref[2]
        want = torch.autograd.grad(torch.nn.functional.cross_entropy(z, y), ref)
        rest = 1 - torch.softmax(z.detach(), 1).gather(1, y[:, None]).min().item()
        least = 1 - torch.softmax(z.detach(), 1).gather(1, y[:, None]).max().item()
        assert rest < 0.1
        for a, c in zip(got, want):
            assert (a.cpu().double() - c).norm() < (1e-5 + 2.0 ** -22 / least) * c.norm()


def test_leading_dimensions_views_and_dtypes():
    f = functions()
    x, w, y, b, up = make(60, 32, 50, "fp16", seed=4)
    base = check(x, w, y, b, up)
    # [N, H, W, features] and a transposed feature map
    x4 = x.view(3, 4, 5, 32).to(DEV).requires_grad_(True)
    loss = f.linear_cross_entropy(x4, w.to(DEV), y.view(3, 4, 5).to(DEV), b.to(DEV))
    dx, = torch.autograd.grad(loss, x4, up.to(DEV))
    assert torch.equal(loss.detach(), base["loss"]) and torch.equal(dx.view(60, 32), base["dx"])
    xt = x.t().contiguous().to(DEV).requires_grad_(True)
    loss = f.linear_cross_entropy(xt.t(), w.to(DEV), y.to(DEV), b.to(DEV))
    dxt, = torch.autograd.grad(loss, xt, up.to(DEV))
    assert torch.equal(loss.detach(), base["loss"]) and torch.equal(dxt.t(), base["dx"])
    assert torch.equal(f.linear_cross_entropy(x4.detach(), w.to(DEV), y.view(3, 4, 5).to(DEV), b.to(DEV), reduction="none").view(60),
                       f.linear_cross_entropy(x.to(DEV), w.to(DEV), y.to(DEV), b.to(DEV), reduction="none"))
    # storage that does not begin on 16 bytes, a strided target
    odd = torch.cat([x.flatten()[:1], x.flatten()]).to(DEV)[1:].view(60, 32)
    oddw = torch.cat([w.flatten()[:3], w.flatten()]).to(DEV)[3:].view(50, 32)
    y2 = torch.stack([y, y], 1).to(DEV)[:, 0]
    assert torch.equal(f.linear_cross_entropy(odd, oddw, y2, b.to(DEV)), base["loss"])
    # fp32 parameters follow 16-bit features, and get fp32 gradients
    wp, bp = w.float().to(DEV).requires_grad_(True), b.float().to(DEV).requires_grad_(True)
    loss = f.linear_cross_entropy(x.to(DEV), wp, y.to(DEV), bp)
    dw, db = torch.autograd.grad(loss, [wp, bp], up.to(DEV))
    assert dw.dtype == db.dtype == torch.float32
    assert torch.equal(dw.half(), base["dw"]) and torch.equal(db.half(), base["db"])


def test_single_gradients_and_empty_batches():
    f = functions()
    x, w, y, b, up = (t.to(DEV) for t in make(60, 32, 50, "fp32", seed=4))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(f.linear_cross_entropy(full[0], full[1], y, full[2]), full, up)
    for i in range(3):
        part = [x, w, b]
        part[i] = part[i].clone().requires_grad_(True)
        got, = torch.autograd.grad(f.linear_cross_entropy(part[0], part[1], y, part[2]), part[i], up)
        assert torch.equal(got, want[i])
    for reduction in ("none", "mean", "sum"):
        leaves = [x[:0].clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
        loss = f.linear_cross_entropy(leaves[0], leaves[1], y[:0], leaves[2], reduction=reduction)
        assert {"none": loss.shape == (0,), "mean": loss.isnan().all(), "sum": (loss == 0).all()}[reduction]
        dx, dw, db = torch.autograd.grad(loss.sum(), leaves)
        assert dx.shape == (0, 32) and (dw == 0).all() and (db == 0).all()


def test_refusals():
    f = functions()
    x, w, y, b, _ = (t.to(DEV) for t in make(6, 8, 5, "fp32"))
    for args in ((x, w[:, :7], y), (x, w, y[:5]), (x, w.flatten(), y), (x, w, y.view(6, 1)), (x, w, y, b[:4]), (x, w[:0], y), (x[:, :0], w[:, :0], y)):
        with pytest.raises(ValueError):
            f.linear_cross_entropy(*args)
    for kw in (dict(label_smoothing=1.1), dict(label_smoothing=-0.1), dict(reduction="max")):
        with pytest.raises(ValueError):
            f.linear_cross_entropy(x, w, y, b, **kw)
    for args in ((x, w, y.int()), (x, w, y.float()), (x.int(), w.int(), y)):
        with pytest.raises(TypeError):
            f.linear_cross_entropy(*args)
    with pytest.raises(NotImplementedError):
        f.linear_cross_entropy(x, w, y.cpu())
    loss = f.linear_cross_entropy(x.requires_grad_(True), w, y)
    loss.backward()
    with pytest.raises(RuntimeError):
        loss.backward()
    loss = f.linear_cross_entropy(x, w, y)
    with torch.no_grad():
        x += 1
    with pytest.raises(RuntimeError):
        loss.backward()


def test_gradients_against_differences():
    """fp64, central differences of the operator itself: the step 1e-5 leaves h^2 / 6 of a third derivative that is
    below one, and 2^-52 / h of a loss below ten: under 1e-8 together."""
    x, w, y, b, _ = make(9, 6, 5, "fp64", ignored=0.2, seed=12)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    for kw in (dict(), dict(label_smoothing=0.2, reduction="sum")):
        grads = torch.autograd.grad(functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2], **kw), leaves)
        for i, g in enumerate(grads):
            for j in range(0, g.numel(), 3):
                at = []
                for s in (1e-5, -1e-5):
                    moved = [t.detach().clone() for t in leaves]
                    moved[i].view(-1)[j] += s
                    at.append(functions().linear_cross_entropy(moved[0], moved[1], y.to(DEV), moved[2], **kw).item())
                assert abs((at[0] - at[1]) / 2e-5 - g.view(-1)[j].item()) < 1e-8


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_the_same_call_gives_the_same_bits(dtype):
    args = make(700, 136, 1500, dtype, ignored=0.1, seed=9)
    a, b = check(*args), check(*args)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_head_on_another_stream_and_captured():
    f = functions()
    x, w, y, b, up = (t.to(DEV) for t in make(200, 64, 500, "bf16", seed=2))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        loss = f.linear_cross_entropy(x, w, y, b, label_smoothing=0.1)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, up)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            g.replay()
        for g, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want, out))


def test_one_row_without_a_batch_and_inference_mode():
    f = functions()
    x, w, y, b, _ = (t.to(DEV) for t in make(3, 40, 30, "fp32"))
    each = f.linear_cross_entropy(x, w, y, b, reduction="none")
    for reduction in ("none", "mean", "sum"):
        one = f.linear_cross_entropy(x[1], w, y[1], b, reduction=reduction)
        assert one.shape == () and abs(one - each[1]) < 1e-6
    with torch.inference_mode():
        assert torch.equal(f.linear_cross_entropy(x, w, y, b, reduction="none"), each)
        assert torch.equal(f.dropout(x, 0.5, 3), f.dropout(x, 0.5, 3))


def test_replays_whose_ignored_rows_become_strange():
    """What an ignored row holds is looked at on the device: a captured step meets NaN in one replay and none in the next."""
    f = functions()
    x, w, y, b, up = make(300, 64, 500, "bf16", ignored=0.3, seed=40)
    dead = y == -100
    xs = x.to(DEV).requires_grad_(True)
    ws = w.to(DEV).requires_grad_(True)
    ys, bs = y.to(DEV), b.to(DEV)

    def step():
        loss = f.linear_cross_entropy(xs, ws, ys, bs)
        return (loss.detach(),) + torch.autograd.grad(loss, [xs, ws])
    want = [t.clone() for t in step()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for bad in (0.0, float("nan"), 1.0, float("inf")):
        with torch.no_grad():
            xs[dead.to(DEV)] = bad
        g.replay()
        assert all(torch.equal(a, c) for a, c in zip(want, out)), bad


def test_two_streams_at_once():
    """Calls of different sizes on two streams, none waiting for the other: each has its own scratch, and what is on the
    chip of an SM belongs to one block at a time."""
    f = functions()
    cases = [make(3000, 264, 5000, "bf16", seed=21), make(40, 64, 300, "fp32", seed=22)]
    streams = [torch.cuda.Stream() for _ in cases]

    def step(case):
        x, w, y, b, up = (t.to(DEV) for t in case)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        loss = f.linear_cross_entropy(x, w, y, b)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, up)
    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(want[i], g))


def test_gradients_that_arrive_expanded_or_in_another_dtype():
    x, w, y, b, _ = make(50, 40, 60, "fp16", reduction="none", seed=30)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    loss = functions().linear_cross_entropy(leaves[0], leaves[1], y.to(DEV), leaves[2], reduction="none")
    want = torch.autograd.grad(loss, leaves, torch.ones(50, device=DEV), retain_graph=True)
    for got in (torch.autograd.grad(loss.sum(), leaves, retain_graph=True), torch.autograd.grad(loss.double().sum(), leaves, retain_graph=True),
                torch.autograd.grad(loss, leaves, torch.ones(1, device=DEV).expand(50))):
        assert all(torch.equal(a, c) for a, c in zip(want, got))


def test_gradients_of_broadcast_inputs_and_shared_weights():
    """One feature row for many targets, one weight in two losses: autograd sums what the operator gives for each."""
    f = functions()
    x, w, y, b, _ = (t.to(DEV) for t in make(30, 24, 40, "fp64", seed=31))
    one = x[:1].clone().requires_grad_(True)
    wp = w.clone().requires_grad_(True)
    loss = f.linear_cross_entropy(one.expand(30, 24), wp, y, b) + f.linear_cross_entropy(x, wp, y.flip(0), b, label_smoothing=0.2)
    got = torch.autograd.grad(loss, [one, wp])
    want = torch.nn.functional.cross_entropy(one.expand(30, 24) @ wp.t() + b, y) + \
        torch.nn.functional.cross_entropy(x @ wp.t() + b, y.flip(0), label_smoothing=0.2)
    for a, c in zip(got, torch.autograd.grad(want, [one, wp])):
        assert torch.allclose(a, c, rtol=1e-11, atol=1e-13)


def test_head_and_dropout_together_as_a_training_step():
    """Features -> dropout -> linear -> loss, as the module runs it, against the oracles one after the other."""
    from deformable_kernels.modules import LinearCrossEntropy
    torch.manual_seed(5)
    x, w, y, b, up = make(90, 56, 120, "fp32", seed=15)
    head = LinearCrossEntropy(56, 120, dropout=0.25, label_smoothing=0.1).to(DEV)
    with torch.no_grad():
        head.weight.copy_(w), head.bias.copy_(b)
    for step in range(3):
        torch.manual_seed(step)
        seed, offset = torch.randint(0, 2 ** 63 - 1, (2,), device=DEV).tolist()
        torch.manual_seed(step)
        xg = x.to(DEV).requires_grad_(True)
        loss = head(xg, y.to(DEV))
        dx, dw, db = torch.autograd.grad(loss, [xg, head.weight, head.bias])
        dropped = H.dropout(x, 0.25, seed, offset)
        out, far = H.head(dropped, w, y, b, torch.tensor(1.0), label_smoothing=0.1)
        keep = H.keep_mask(x.shape, 0.25, seed, offset).double() / 0.75
        out["dx"], far["dx"] = out["dx"] * keep, far["dx"] * keep + out["dx"].abs() * 2.0 ** -22 + 1e-300
        for name, v in (("loss", loss), ("dx", dx), ("dw", dw), ("db", db)):
            assert ((v.detach().cpu().double() - out[name]).abs() <= far[name]).all(), (step, name)
    head.eval()
    with torch.no_grad():
        assert torch.equal(head(x.to(DEV), y.to(DEV)), functions().linear_cross_entropy(x.to(DEV), head.weight, y.to(DEV), head.bias,
                                                                                       label_smoothing=0.1))
    with torch.autocast("cuda", dtype=torch.float16):
        loss = head(x.to(DEV), y.to(DEV))
        assert loss.dtype == torch.float32
        loss.backward()
    assert head.weight.grad.dtype == torch.float32


def test_calls_from_threads_that_have_not_used_the_gpu_yet():
    """Forward, and backward on autograd's thread, as the first thing a process and its threads do; two threads at once."""
    import subprocess
    import sys
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys, threading
sys.path[:0] = [%r, %r]
import torch
import torch.utils.checkpoint
import head_oracle as H
import test_head_gpu as T
cases = [T.make(60, 32, 50, "bf16", seed=s) for s in range(4)]
wrong = []
def work(case):
    try:
        for _ in range(20):
            T.check(*case)
    except BaseException as e:
        wrong.append(e)
x, w, y, b, up = (t.cuda() for t in cases[0])
x.requires_grad_(True)
torch.autograd.grad(T.functions().linear_cross_entropy(x, w, y, b), x, up)
threads = [threading.Thread(target=work, args=(c,)) for c in cases]
[t.start() for t in threads]
[t.join() for t in threads]
assert not wrong, wrong
""" % (os.path.join(root, "deformable-kernels_b200"), os.path.join(root, "tests"))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert out.returncode == 0, out.stderr[-2000:]


def test_features_and_weights_beyond_32_bits():
    """More than 2^32 features or weights: what is far behind is what a call on those rows or classes alone gives."""
    f = functions()
    gen = torch.Generator(device=DEV).manual_seed(3)
    t, d, v = 2 ** 21 + 5, 2056, 24
    x = torch.randn(t, d, device=DEV, generator=gen, dtype=torch.bfloat16)
    w = torch.randn(v, d, device=DEV, generator=gen, dtype=torch.bfloat16) / 32
    y = torch.randint(0, v, (t,), device=DEV, generator=gen)
    x.requires_grad_(True)
    loss = f.linear_cross_entropy(x, w, y, reduction="none")
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    loss = loss.detach()
    for lo in (0, 2 ** 20 - 100, t - 300):
        part = x.detach()[lo:lo + 300].clone().requires_grad_(True)
        want = f.linear_cross_entropy(part, w, y[lo:lo + 300], reduction="none")
        dpart, = torch.autograd.grad(want, part, torch.ones_like(want))
        # the same products in another tiling: 2056 cutting additions of 2^-23 each at most, a rounding of dz and of dx that may fall to the
        # other side (2^-7 of the value, 2^-8 of every class's part)
        assert (loss[lo:lo + 300] - want.detach()).abs().max() < 1e-3
        assert (dx[lo:lo + 300].float() - dpart.float()).abs().max() < 2.0 ** -6 * w.float().abs().max()
    del x, dx, loss
    torch.cuda.empty_cache()
    t, v = 40, 2 ** 21 + 5
    x = torch.randn(t, d, device=DEV, generator=gen, dtype=torch.bfloat16)
    w = (torch.randn(v, d, device=DEV, generator=gen, dtype=torch.bfloat16) / 32).requires_grad_(True)
    y = torch.randint(0, v, (t,), device=DEV, generator=gen)
    y[:4] = torch.tensor([0, 2 ** 20, v - 1, v - 2])
    loss = f.linear_cross_entropy(x, w, y, reduction="none")
    dw, = torch.autograd.grad(loss, w, torch.ones_like(loss))
    z = torch.cat([x.float() @ w.detach()[i:i + 2 ** 18].float().t() for i in range(0, v, 2 ** 18)], 1)
    lse = torch.logsumexp(z, 1)
    assert (loss.detach() - (lse - z.gather(1, y[:, None]).squeeze(1))).abs().max() < 1e-2
    for lo in (0, 2 ** 20 - 50, v - 100):
        dz = torch.exp(z[:, lo:lo + 100] - lse[:, None])
        hit = (y >= lo) & (y < lo + 100)
        dz[hit, y[hit] - lo] -= 1
        want = dz.t() @ x.float()
        # dz and dw are rounded to bf16: 2^-8 of the magnitudes each; the logits' error moves p by a few 1e-3 of itself
        assert ((dw[lo:lo + 100].float() - want).abs() <= 2.0 ** -6 * (dz.abs().t() @ x.float().abs()) + 1e-6).all()
    del w, dw, z
    torch.cuda.empty_cache()


def test_training_step_of_the_bench_with_the_fused_head():
    """MobileNetV2-DK with its classifier and loss as LinearCrossEntropy against the same network with the stock modules:
    fp32, running statistics (no dropout then), loss and the gradients at both ends of the network."""
    import bench
    old = (torch.backends.cudnn.allow_tf32, torch.backends.cuda.matmul.allow_tf32)
    torch.backends.cudnn.allow_tf32 = torch.backends.cuda.matmul.allow_tf32 = False
    try:
        torch.manual_seed(0)
        stock, _ = bench.build_mobilenet_dk()
        stock = stock.to(DEV).eval()
        with torch.no_grad():
            stock.classifier[1].weight.normal_(0, 0.05)
        x = torch.randn(4, 3, 96, 96, device=DEV)
        y = torch.randint(0, 1000, (4,), device=DEV)
        loss = torch.nn.functional.cross_entropy(stock(x), y)
        loss.backward()
        want = {n: p.grad.clone() for n, p in stock.named_parameters() if p.grad is not None}
        stock.zero_grad(set_to_none=True)
        fused = bench.ClassifierStep(stock).eval().to(DEV)
        loss2 = fused(x, y)
        loss2.backward()
        assert abs(loss.item() - loss2.item()) < 1e-5 * abs(loss.item())
        for mine, theirs in (("head.weight", "classifier.1.weight"), ("head.bias", "classifier.1.bias"),
                             ("net.features.18.0.weight", "features.18.0.weight"),
                             ("net.features.1.conv.0.0.inner_conv.weight", "features.1.conv.0.0.inner_conv.weight")):
            a, b = fused.get_parameter(mine).grad.double(), want[theirs].double()
            assert (a - b).norm() < 1e-4 * b.norm(), mine
        fused.train()
        with torch.autocast("cuda", dtype=torch.float16):
            losses = [fused(x, y) for _ in range(2)]
        assert all(v.dtype == torch.float32 and torch.isfinite(v) for v in losses)
    finally:
        torch.backends.cudnn.allow_tf32, torch.backends.cuda.matmul.allow_tf32 = old
