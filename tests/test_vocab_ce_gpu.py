"""loss_fns.linear_cross_entropy against the definition in float64 on the same (already rounded) inputs.

Tolerances, with e = 2^-24 (half a step of fp32), u = 2^-8 for bf16 and 2^-24 for fp32 (half a step of the output type), and
A_m = max_v sum_k |x_mk w_vk| + |b_v|:
  a score z is a sum of D fp32 terms and the bias:                   |dz| <= (D + 2) e A
  exponentials and their sum (positive terms, the hardware's exp2 good to a step): relative error of the sum <= 512 e, so
  the row's loss is off by at most                                   t = (2 (D + 2) A + 512) e, and by e |loss| in the end
  a softmax value p is off by 2 t p; a gradient of the scores g = c (p - keep [v = t] - s) is then off by
                                                                     E = |c| (2 t p + 4 e (p + keep + s)) + u |g|  (g is held in T)
  a product over n of them adds n e of the sum of magnitudes, and the output's own rounding u |out|."""
import math

import pytest
import torch
import torch.nn.functional as F

from image_segmentation_amd import _C
from image_segmentation_amd._C import LsamError
from image_segmentation_amd.loss_fns import linear_cross_entropy

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def make(M, D, V, dtype, bias, seed, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) * (2 / D ** 0.5)
    t = torch.randint(0, V, (M,), generator=g)
    x = torch.randn(M, D, generator=g) + w[t] * (0.5 * D ** 0.5) * torch.rand(M, 1, generator=g)
    t[torch.rand(M, generator=g) < ignored] = -100
    b = torch.randn(V, generator=g).cuda() if bias else None
    return x.to("cuda", dtype), w.to("cuda", dtype), t.cuda(), b, torch.rand(M, generator=g).cuda()


def bounds(x, w, t, b, smoothing, c):
    """(tolerance of each row's loss, dx, dw, db) for row coefficients c (fp64, 0 where ignored)."""
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else E
    X, W = x.detach().double(), w.detach().double()
    B = torch.zeros(W.shape[0], dtype=torch.float64, device=X.device) if b is None else b.detach().double()
    (M, D), V = X.shape, W.shape[0]
    A = (X.abs() @ W.abs().t() + B.abs()).amax(1)
    tz = (2 * (D + 2) * A + 512) * E
    p = torch.softmax(X @ W.t() + B, 1)
    hot = F.one_hot(t.clamp_min(0), V).double()
    g = c[:, None] * (p - (1 - smoothing) * hot - smoothing / V)
    err = c.abs()[:, None] * (2 * tz[:, None] * p + 4 * E * (p + (1 - smoothing) * hot + smoothing / V)) + u * g.abs()
    dx = err @ W.abs() + V * E * (g.abs() @ W.abs()) + u * (g @ W).abs()
    dw = err.t() @ X.abs() + M * E * (g.abs().t() @ X.abs()) + u * (g.t() @ X).abs()
    db = (c.abs()[:, None] * (2 * tz[:, None] * p + 4 * E * (p + (1 - smoothing) * hot + smoothing / V))).sum(0) + M * E * g.abs().sum(0)
    return tz, dx + 1e-30, dw + 1e-30, db + 1e-30


def check(x, w, t, b, gout, smoothing, reduction, **kw):
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b) if v is not None]
    lx, lw, lb = leaves[0], leaves[1], leaves[2] if b is not None else None
    loss = linear_cross_entropy(lx, lw, t, bias=lb, label_smoothing=smoothing, reduction=reduction, **kw)
    go = gout if reduction == "none" else torch.ones_like(loss)
    grads = torch.autograd.grad(loss, leaves, go)
    rows = t != -100
    ref_leaves = [v.detach().double().requires_grad_(True) for v in (x, w, b) if v is not None]
    ref = F.cross_entropy(F.linear(ref_leaves[0], ref_leaves[1], ref_leaves[2] if b is not None else None), t, label_smoothing=smoothing,
                          reduction=reduction)
    want = torch.autograd.grad(ref, ref_leaves, go.double())
    n = int(rows.sum())
    c = torch.where(rows, gout.double() if reduction == "none" else torch.ones_like(gout, dtype=torch.float64) / (n if reduction == "mean" else 1),
                    0.0)
    tz, *tol = bounds(x, w, t, b, smoothing, c)
    row = torch.where(rows, tz, 0.0)
    lim = row if reduction == "none" else row.sum() / (n if reduction == "mean" else 1)
    assert loss.dtype == torch.float32 and loss.shape == ref.shape
    assert ((loss.double() - ref).abs() <= lim + 4 * E * ref.abs()).all()
    for got, exp, lim, name in zip(grads, want, tol, ("dx", "dw", "db")):
        assert got.dtype == {"dx": x, "dw": w, "db": b}[name].dtype and got.shape == exp.shape
        bad = (got.double() - exp).abs() > lim
        assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[:4].tolist())
    assert (grads[0][~rows] == 0).all()
    return loss, grads


SHAPES = [(1, 8, 2), (1, 256, 1000), (2, 1, 3), (3, 7, 5), (16, 256, 1000), (37, 100, 301), (64, 12, 70), (257, 64, 513), (300, 252, 1000),
          (255, 33, 257), (700, 896, 2050), (513, 320, 255)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M, D, V", SHAPES)
@pytest.mark.parametrize("bias, smoothing, reduction", [(True, 0.0, "mean"), (False, 0.1, "none"), (True, 1.0, "sum"), (False, 0.0, "sum")])
def test_matches_float64(M, D, V, dtype, bias, smoothing, reduction):
    x, w, t, b, g = make(M, D, V, dtype, bias, 1000 * M + D + V)
    if (t == -100).all():
        t[0] = 0
    check(x, w, t, b, g, smoothing, reduction)


# large tiles (bf16): one and several tiles a workgroup, one to four k-tiles, an odd number of them, rows and classes that end inside a
# tile, a weight gradient whose last tiles go apart
LARGE = [(4096, 16, 4096), (4000, 100, 8200), (5001, 448, 8192), (3900, 200, 8300), (1100, 256, 67300), (300, 896, 66000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M, D, V", LARGE)
def test_large_tiles(M, D, V, dtype):
    x, w, t, b, g = make(M, D, V, dtype, M % 2 == 0, M + D + V)
    check(x, w, t, b, g, 0.1 if D == 100 else 0.0, "none" if D == 200 else "mean")


# few rows against many classes (sums over hundreds of splits), many against few, and rows of dW of every alignment
FEW = [(1, 100, 20000), (6, 587, 9001), (30, 101, 30000), (5, 592, 24000), (9000, 70, 5), (2100, 254, 40), (2100, 257, 700), (130, 129, 4000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M, D, V", FEW)
def test_long_and_narrow(M, D, V, dtype):
    x, w, t, b, g = make(M, D, V, dtype, True, M + D + V, ignored=0.0 if M < 10 else 0.2)
    check(x, w, t, b, g, 0.1 if D % 2 else 0.0, "sum" if M < 100 else "none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_several_pieces_of_the_classes(dtype):
    # gradients of the scores over a piece's 1 GiB in either type: the products accumulate over pieces
    x, w, t, b, g = make(36000, 16, 15990 if dtype == torch.bfloat16 else 8000, dtype, True, 5)
    check(x, w, t, b, g, 0.1, "mean")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["one", "first", "last", "none"])
def test_rows_that_count(dtype, kind):
    x, w, t, b, g = make(600, 64, 300, dtype, True, 7, ignored=0.0)
    keep = torch.zeros(600, dtype=torch.bool, device="cuda")
    keep[{"one": slice(311, 312), "first": slice(0, 1), "last": slice(599, 600), "none": slice(0, 0)}[kind]] = True
    t = torch.where(keep, t, -100)
    # what ignored rows hold reaches nothing
    x[~keep] = float("nan")
    if kind == "none":
        leaves = [v.requires_grad_(True) for v in (x, w, b)]
        for red, want in (("mean", float("nan")), ("sum", 0.0)):
            loss = linear_cross_entropy(x, w, t, bias=b, reduction=red)
            assert loss.isnan() if want != want else float(loss.detach()) == want
            for gr in torch.autograd.grad(loss, leaves):
                assert (gr == 0).all()
        assert (linear_cross_entropy(x, w, t, bias=b, reduction="none") == 0).all()
        return
    loss, grads = linear_cross_entropy(x, w, t, bias=b), None
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(*leaves[:2], t, bias=leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    xs, ts = x.detach()[keep], t[keep]
    ref_loss, ref = check(xs, w.detach(), ts, b.detach(), g[keep], 0.0, "mean")
    assert torch.equal(loss, ref_loss)
    assert torch.equal(grads[0][keep], ref[0]) and torch.equal(grads[2], ref[2])
    assert (grads[0][~keep] == 0).all() and torch.isfinite(grads[1]).all()
    # dW splits its sum over the rows by the rows that could count: same terms, another order
    assert (grads[1].double() - ref[1].double()).abs().max() <= 2.0 ** -7 * ref[1].abs().max()


@pytest.mark.parametrize("M", [8191, 8192, 8193, 30000])
def test_many_rows(M):
    # rows of several selecting workgroups, whole ones of them ignored
    x, w, t, b, g = make(M, 24, 60, torch.float32, True, M, ignored=0.5)
    t[8000:16500] = -100
    check(x, w, t, b, g, 0.0, "none")


def test_second_derivative_is_refused():
    x, w, t, b, g = make(20, 8, 30, torch.float32, False, 3)
    x.requires_grad_(True)
    with pytest.raises(LsamError, match="second derivative"):
        torch.autograd.grad(linear_cross_entropy(x, w, t), x, create_graph=True)


def test_no_rows():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.randn(40, 16, device="cuda", requires_grad=True)
    b = torch.randn(40, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.long, device="cuda")
    for red in ("none", "mean", "sum"):
        loss = linear_cross_entropy(x, w, t, bias=b, reduction=red)
        assert loss.shape == ((0,) if red == "none" else ())
        gx, gw, gb = torch.autograd.grad(loss.sum(), (x, w, b))
        assert gx.shape == (0, 16) and (gw == 0).all() and (gb == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    M, D, V = 130, 72, 333
    x, w, t, b, g = make(M, D, V, dtype, True, 11)
    want_loss, want = check(x, w, t, b, g, 0.1, "none")
    wide = torch.full((M, D + 9), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:3 + D] = x                                       # rows off any vector's alignment
    wide_w = torch.full((V, D + 5), float("nan"), dtype=dtype, device="cuda")
    wide_w[:, 1:1 + D] = w
    forms = [(wide[:, 3:3 + D], wide_w[:, 1:1 + D]), (x.t().contiguous().t(), w.t().contiguous().t()), (x, w.repeat_interleave(2, 0)[::2])]
    for xs, ws in forms:
        loss, grads = check(xs, ws, t, b, g, 0.1, "none")
        assert torch.equal(loss, want_loss)
        assert all(torch.equal(a, e) for a, e in zip(grads, want))
    # int32 targets, [N, H, W, D] features, a bias in bf16
    loss = linear_cross_entropy(x.view(2, 13, 5, D), w, t.view(2, 13, 5).int(), bias=b, label_smoothing=0.1, reduction="none")
    assert torch.equal(loss.view(-1), want_loss)
    bl = b.bfloat16().requires_grad_(True)
    (gb,) = torch.autograd.grad(linear_cross_entropy(x, w, t, bias=bl), bl)
    assert gb.dtype == torch.bfloat16
    # broadcast rows (stride 0)
    xe = x[:1].expand(M, D)
    assert torch.equal(linear_cross_entropy(xe, w, t, bias=b, reduction="none"), linear_cross_entropy(xe.contiguous(), w, t, bias=b, reduction="none"))


def test_masked_classes_and_extreme_scores():
    x, w, t, b, g = make(300, 64, 700, torch.bfloat16, True, 13, ignored=0.0)
    b[256:520] = float("-inf")                                # a whole tile of classes and parts of two others
    t = torch.where((t >= 256) & (t < 520), 3, t)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    live = torch.ones(700, dtype=torch.bool, device="cuda")
    live[256:520] = False
    t2 = torch.where(t >= 520, t - 264, t)
    _, want = check(x, w[live].contiguous(), t2, b[live].contiguous(), g, 0.0, "mean")
    assert (grads[1][~live] == 0).all() and (grads[2][~live] == 0).all()
    assert (grads[0].double() - want[0].double()).abs().max() <= 2.0 ** -7 * want[0].abs().max()
    # the type's lowest value as a mask, and scores of several thousand: finite
    for low, scale in ((torch.finfo(torch.float32).min, 1.0), (-1e4, 300.0)):
        b2 = torch.where(live, b, low)
        loss = linear_cross_entropy(x * scale, w, t, bias=b2, reduction="none")
        ref = F.cross_entropy(F.linear((x * scale).double(), w.double(), b2.double()), t, reduction="none")
        assert torch.isfinite(loss).all()
        A = ((x * scale).double().abs() @ w.double().abs().t() + torch.where(live, b2, 0.0).double().abs()).amax(1)
        assert ((loss - ref).abs() <= (2 * 66 * A + 512) * E + 4 * E * ref.abs()).all()


def test_not_finite():
    x, w, t, b, g = make(70, 32, 300, torch.float32, True, 17, ignored=0.0)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[5, 3] = bad
        loss = linear_cross_entropy(y, w, t, bias=b, reduction="none")
        assert loss[5].isnan() and torch.isfinite(loss[torch.arange(70, device="cuda") != 5]).all()
    for wrong in (300, -1, 2 ** 31, -2 ** 40):                 # outside [0, V): NaN, and nothing read out of range
        t2 = t.clone()
        t2[9] = wrong
        y = x.clone().requires_grad_(True)
        loss = linear_cross_entropy(y, w, t2, bias=b, reduction="none")
        assert loss[9].isnan() and int(loss.isnan().sum()) == 1
        (gx,) = torch.autograd.grad(loss.sum(), y)
        assert gx[9].isnan().all() and int(gx.isnan().any(1).sum()) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_magnitudes(dtype):
    # columns of x scaled by powers of two and those of w by their inverses: every product, and so every score, stays what it was, and
    # the gradients scale with them, all without a rounding
    x, w, t, b, _ = make(150, 96, 500, dtype, True, 43)
    k = torch.linspace(-60, 60, 96, device="cuda").round()
    k = torch.where(torch.arange(96, device="cuda") % 2 == 0, k, -k)
    up = torch.exp2(k).to(dtype)

    def step(x, w):
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], label_smoothing=0.05)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    want, got = step(x, w), step(x * up, w / up)
    got[1], got[2] = got[1] * up, got[2] / up
    assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_gradient_against_differences():
    x, w, t, b, _ = make(20, 24, 50, torch.float32, True, 19)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, bias=b, label_smoothing=0.2)
    grads = torch.autograd.grad(loss, leaves)
    gen = torch.Generator().manual_seed(3)
    h = 2.0 ** -6
    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=gen).cuda()
        val = []
        for sgn in (1, -1):
            moved = [v.detach() + (sgn * h * d if j == i else 0) for j, v in enumerate(leaves)]
            val.append(float(linear_cross_entropy(moved[0], moved[1], t, bias=moved[2], label_smoothing=0.2)))
        # central difference: truncation h^2 |third derivative| / 6 (softmax cumulants along d: at most (max |dz|)^3, dz the scores' change)
        along = d.abs().max() if i == 2 else d.abs().sum(1).max() * w.detach().abs().max() if i == 0 else d.abs().max() * x.detach().abs().sum(1).max()
        got = float((grads[i] * d).sum())
        assert abs((val[0] - val[1]) / (2 * h) - got) <= h * h / 6 * float(along) ** 3 + 2e-5 / h


def test_only_some_gradients_and_same_bits_twice():
    x, w, t, b, _ = make(500, 128, 1200, torch.bfloat16, True, 23)
    full = torch.autograd.grad(linear_cross_entropy(*(l := [v.detach().requires_grad_(True) for v in (x, w, b)])[:2], t, bias=l[2]), l)
    again = torch.autograd.grad(linear_cross_entropy(*(l := [v.detach().requires_grad_(True) for v in (x, w, b)])[:2], t, bias=l[2]), l)
    assert all(torch.equal(a, c) for a, c in zip(full, again))
    for i in range(3):
        l = [v.detach().requires_grad_(i == j) for j, v in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(linear_cross_entropy(l[0], l[1], t, bias=l[2]), [l[i]])
        assert torch.equal(g, full[i])
    assert not linear_cross_entropy(x, w, t, bias=b).requires_grad
    # the rows may change between forward and backward: the forward's own are used
    l = [v.detach().clone().requires_grad_(True) for v in (x, w, b)]
    y = l[0] * 1
    loss = linear_cross_entropy(y, l[1], t, bias=l[2])
    with torch.no_grad():
        y.zero_()
    assert torch.equal(torch.autograd.grad(loss, l)[1], full[1])


def test_stream_and_graph():
    x, w, t, b, _ = make(300, 96, 700, torch.bfloat16, True, 29)

    def step(leaves, t):
        loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    fresh = lambda: [v.detach().clone().requires_grad_(True) for v in (x, w, b)]
    want = step(fresh(), t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = fresh()
        ts = t.clone()
        for a, e in zip(step(leaves, ts), want):
            assert torch.equal(a, e)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(leaves, ts)
    for seed in (31, 37, 41):
        x2, w2, t2, b2, _ = make(300, 96, 700, torch.bfloat16, True, seed, ignored=0.1 * (seed - 30))
        with torch.no_grad():
            for leaf, v in zip(leaves, (x2, w2, b2)):
                leaf.copy_(v)
            ts.copy_(t2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = step([v.detach().requires_grad_(True) for v in (x2, w2, b2)], t2)
        for a, e in zip(out, eager):                           # the last replay has no row left: its mean is NaN on both sides
            assert torch.allclose(a, e, rtol=0, atol=0, equal_nan=True)


def test_refusals():
    x, w, t = torch.zeros(4, 8, device="cuda"), torch.zeros(5, 8, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    for args in ((x, w[:, :7], t), (x, w.bfloat16(), t), (x.half(), w.half(), t), (x, w, t[:3]), (x, w, t.float()), (x, w, t, torch.zeros(4, device="cuda")),
                 (x, w, t, torch.zeros(5, dtype=torch.long, device="cuda")), (x, w.cpu(), t), (x, w, t.cpu()), (x, w, t, torch.zeros(5)), (x, w[:0], t)):
        with pytest.raises(LsamError):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(ValueError):
        linear_cross_entropy(x, w, t, label_smoothing=1.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [0, 20, 24, 25, 26, 31, 40, 80, 117])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_scores_of_any_size(power, smoothing, dtype):
    """One column, whole numbers times 2^power: every score is exact in fp32, and so is what a bias of such numbers makes of it.  What is left:
    an exponential's argument is rounded where it is 64 at most (2^-17), the exponentials are good to a step, their sum has 700 terms:
    2^-13 of the sum in all.  The mean of the scores is a sum of 700 terms in fp32."""
    g = torch.Generator().manual_seed(power)
    M, V = 60, 700
    w = torch.randint(0, 50, (V, 1), generator=g).double()
    w[[3, 200, 301, 640]] = 50.0                               # ties of the highest score, in several tiles
    x = (torch.randint(1, 4, (M, 1), generator=g) * (1 - 2 * torch.randint(0, 2, (M, 1), generator=g))).double() * 2.0 ** power
    t = torch.randint(0, V, (M,), generator=g).cuda()
    t[:4] = torch.tensor([3, 640, 5, -100])
    x, w = x.to("cuda", dtype), w.to("cuda", dtype)
    b = (torch.randint(-3, 4, (V,), generator=g).double() * 2.0 ** power).float().cuda()
    b[[3, 200, 301, 640]] = 0.0
    gout = torch.rand(M, generator=g).cuda()
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2], label_smoothing=smoothing, reduction="none")
    grads = torch.autograd.grad(loss, leaves, gout)
    X, W, B = (v.detach().double().requires_grad_(True) for v in (x, w, b))
    Z = X @ W.t() + B
    ref = F.cross_entropy(Z, t, label_smoothing=smoothing, reduction="none")
    want = torch.autograd.grad(ref, (X, W, B), gout.double())
    z = Z.detach()
    assert torch.isfinite(loss).all()
    assert ((loss - ref.detach()).abs() <= 2.0 ** -13 + 8 * E * ref.detach().abs() + smoothing * V * E * z.abs().amax(1)).all()
    u = 2.0 ** -8 if dtype == torch.bfloat16 else E
    rows = t >= 0
    size = torch.softmax(z, 1) + F.one_hot(t.clamp_min(0), V).double() + smoothing / V
    size = torch.where(rows, gout.double(), 0.0)[:, None] * size
    X, W = X.detach().abs(), W.detach().abs()
    for got, exp, lim in zip(grads, want, (size @ W, size.t() @ X, size.sum(0))):
        assert ((got.double() - exp).abs() <= (2.0 ** -12 + u) * lim + u * exp.abs() + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e9, -3e9, -1e20, -1e38])
def test_masks_of_any_size(mask, dtype):
    # finite masks are the bias that they say: the loss of a masked target, and the mean of the scores that smoothing takes.  A score next to a mask
    # keeps fp32's 24 bits of the larger one
    x, w, t, b, _ = make(50, 24, 600, dtype, True, 47, ignored=0.0)
    b[100:400] = mask
    t[:8] = 150
    z = x.double() @ w.double().t() + b.double()
    for smoothing in (0.0, 0.1):
        loss = linear_cross_entropy(x, w, t, bias=b, label_smoothing=smoothing, reduction="none")
        ref = F.cross_entropy(z, t, label_smoothing=smoothing, reduction="none")
        assert ((loss - ref).abs() <= 1e-4 + (600 * smoothing + 8) * E * ref.abs()).all()
    # nothing but the type's lowest value: fp32 scores are all alike there
    leaves = [v.detach().requires_grad_(True) for v in (x, w, torch.full_like(b, torch.finfo(torch.float32).min))]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    assert abs(float(loss.detach()) - math.log(600)) < 1e-4
    assert all(torch.isfinite(v).all() for v in torch.autograd.grad(loss, leaves))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wanted", range(1, 8))
def test_no_rows_at_the_c_boundary(wanted, dtype):
    # no rows, every pointer set: nothing of dx exists, dw and db are zeros
    L, code, D, V = _C.lib(), _C.dtype_code(dtype), 16, 40
    w = torch.randn(V, D, device="cuda").to(dtype)
    state = torch.empty(L.lsam_linear_ce_state_bytes(code, 0, D), dtype=torch.uint8, device="cuda")
    ws = torch.empty(max(L.lsam_linear_ce_ws_bytes(code, 0, D, V, w.data_ptr(), D, 0.0, f) for f in (0, wanted)), dtype=torch.uint8, device="cuda")
    loss, gout = torch.empty(1, device="cuda"), torch.ones(1, device="cuda")
    dx, dw, db = torch.full((4, D), 7.0, dtype=dtype, device="cuda"), torch.full((V, D), 7.0, dtype=dtype, device="cuda"), torch.full((V,), 7.0, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    assert L.lsam_linear_ce_fwd(code, 0, D, w.data_ptr(), D, 0, 0, 0, D, V, -100, 0.0, 2, loss.data_ptr(), state.data_ptr(), ws.data_ptr(), ws.numel(), s) == 0
    assert L.lsam_linear_ce_bwd(code, w.data_ptr(), D, 0, gout.data_ptr(), 0, D, V, 0.0, 2, state.data_ptr(), dx.data_ptr() if wanted & 1 else 0, D,
                                dw.data_ptr() if wanted & 2 else 0, D, db.data_ptr() if wanted & 4 else 0, ws.data_ptr(), ws.numel(), s) == 0
    assert float(loss) == 0.0 and (dx == 7.0).all()
    assert (dw == (0.0 if wanted & 2 else 7.0)).all() and (db == (0.0 if wanted & 4 else 7.0)).all()


@pytest.mark.parametrize("M, D, V, dtype", [(2_200_000, 16, 300, torch.bfloat16), (750_000, 16, 300, torch.float32), (9_000_000, 8, 20, torch.bfloat16)])
def test_rows_beyond_a_piece(M, D, V, dtype):
    # so many rows that 256 classes' gradients of the scores are more than a GiB, and more than 2^31 of them in the last case
    x, w, t, b, g = make(M, D, V, dtype, True, V)
    check(x, w, t, b, g, 0.0, "none")
