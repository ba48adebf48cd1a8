"""Softmax cross entropy over the catalogue (rs_softmax_ce): refusals on the CPU, values against the definition in
64 bits on the GPU.

Tolerances.  u = eps / 2 is half a step of a type.  A logit is a sum of k products held in fp32: its error is at most
(k + 4) u32 sum |h w| plus, for the base-2 exponent, 3 u32 |l| (one rounding each for the scale, the sum with the
bias and the difference); fp16 pairs leave 3 u32 |h w| of a product more.  With L the largest
sum |h w| + |bias| of a row, e_l = (k + 10) u32 (L + 1) bounds a logit's error, the loss and lse take 2 e_l, and a
probability is off by 2 e_l and 4 u32 of itself (its exponential, the sum, the division and a product).  A coefficient c = weight (p - [target]) is then rounded to
fp16 or a pair of them (U_C), and the sum over the rows or items adds (terms) u32 of the sum of magnitudes.
Outputs add half a step of their type.  (exp2 and log2 are good to 2 units, inside the 10.)
"""
import ctypes as C
import math

import numpy as np
import pytest

import rsgpu

torch = pytest.importorskip("torch")

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24
U_C = {"f32": 2 * U32, "bf16": 2.0 ** -11, "f16": 2.0 ** -22}  # a coefficient's rounding: a pair, one fp16 value, a pair


def half_step(t):
    return torch.finfo(t).eps / 2


def reference(H, W, target, bias=None, weight=None):
    """The definition in 64 bits, on the CPU, with the rules for rows and items that take no part."""
    H, W = H.double().cpu(), W.double().cpu()
    n, v = H.shape[0], W.shape[0]
    b = torch.zeros(v, dtype=torch.float64) if bias is None else bias.double().cpu()
    g = torch.ones(n, dtype=torch.float64) if weight is None else weight.double().cpu()
    gone = b == -math.inf
    t = target.cpu().long()
    known = (t >= 0) & (t < v)
    tt = torch.where(known, t, torch.zeros_like(t))
    Wm = torch.where(gone[:, None], torch.zeros_like(W), W)
    Hm = torch.where(known[:, None], H, torch.zeros_like(H))
    z = Hm @ Wm.T + b
    empty = bool(gone.all())
    lse = torch.full((n,), -math.inf, dtype=torch.float64) if empty else torch.logsumexp(z, 1)
    live = known & ~gone[tt] & (not empty)
    loss = torch.zeros(n, dtype=torch.float64)
    loss[live] = (lse - z[torch.arange(n), tt])[live]
    if not empty:
        loss[known & gone[tt]] = math.inf
    lse = torch.where(known, lse, torch.zeros_like(lse))
    p = torch.where(live[:, None], torch.exp(z - lse[:, None]), torch.zeros_like(z))
    prob = p.clone()
    p[torch.arange(n)[live], tt[live]] -= 1
    gl = torch.where(live, g, torch.zeros_like(g))
    c = p * gl[:, None]
    L = (Hm.abs() @ Wm.abs().T + torch.where(gone, torch.zeros_like(b), b).abs()).amax(1) if v else torch.zeros(n)
    return dict(loss=loss, lse=lse, dH=c @ Wm, dW=c.T @ Hm, db=c.sum(0), L=L, live=live, c=c, Hm=Hm, Wm=Wm, g=gl, p=prob)


def make(n, v, k, ty, seed=0, spread=1.5, bias=False, gone=0.0, unknown=0.0, weight=True, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    H = (torch.randn(n, k, generator=g) * spread / k ** 0.5).to(T[ty])
    W = torch.randn(v, k, generator=g).to(T[ty])
    target = torch.randint(0, v, (n,), generator=g, dtype=torch.int32)
    b = None
    if bias:
        b = torch.randn(v, generator=g)
        if gone:
            b[torch.rand(v, generator=g) < gone] = -math.inf
            b[0] = 0.5
    if unknown:
        target[torch.rand(n, generator=g) < unknown] = -1
    w = torch.rand(n, generator=g) + 0.5 if weight else None
    to = lambda t: None if t is None else t.to(dev)
    return to(H), to(W), to(target), to(b), to(w)


def check(out, ref, ty, k, grad=True):
    t = T[ty]
    loss, lse = (x.double().cpu() for x in out[:2])
    e_l = (k + 10) * U32 * (ref["L"] + 1)
    for name, x in (("loss", loss), ("lse", lse)):
        r = ref[name]
        fin = torch.isfinite(r)
        assert torch.equal(torch.isfinite(x), fin) and torch.equal(x[~fin], r[~fin]), name
        assert (((x - r).abs() - 2 * e_l - 4 * U32 * r.abs())[fin] <= 0).all(), (name, float((x - r)[fin].abs().max()))
    if not grad:
        return
    u_c = U_C[ty]
    n, v = ref["c"].shape
    # error of a coefficient: its probability's, then its rounding; an fp16 coefficient of any type keeps at least 2^-25 of
    # 2^-13 of the largest weight (it is held scaled to below 2^14)
    gmax = ref["g"].abs().max() if n else 0.0
    floor = float(gmax) * 2.0 ** -38
    p = ref["p"]
    ec = ref["g"].abs()[:, None] * (2 * e_l[:, None] + 4 * U32) * p + u_c * ref["c"].abs() + floor * ref["live"][:, None]
    bound_H = ec @ ref["Wm"].abs() + (v + 4) * U32 * (ref["c"].abs() @ ref["Wm"].abs())
    bound_W = ec.T @ ref["Hm"].abs() + (n + 4) * U32 * (ref["c"].abs().T @ ref["Hm"].abs())
    # db sums the coefficients before they are rounded
    bound_b = ec.sum(0) + (n + 4) * U32 * ref["c"].abs().sum(0)
    # dH is the difference of the mean item and the target's: both sides of it round in fp32
    bound_H = bound_H + 6 * U32 * ref["g"].abs()[:, None] * ref["Wm"].abs().max()
    for name, x, b in (("dH", out[2], bound_H), ("dW", out[3], bound_W), ("db", out[4], bound_b)):
        r = ref[name]
        ut = half_step(x.dtype)
        tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        err = (x.double().cpu() - r).abs()
        lim = b * (1 + ut) + ut * r.abs() + tiny
        assert (err <= lim).all(), (name, float((err - lim).max()), float((err / lim.clamp(min=1e-300)).max()))


SHAPES = [(1, 1, 1), (1, 2, 3), (3, 1, 8), (5, 31, 7), (33, 129, 15), (128, 128, 32), (130, 1682, 20), (257, 500, 33),
          (64, 3706, 100), (100, 257, 128), (40, 300, 129), (70, 90, 256), (130, 260, 300), (20, 1000, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,k", SHAPES)
def test_values_and_gradients(ctx, n, v, k, ty):
    H, W, target, b, w = make(n, v, k, ty, seed=n * 1000 + v, bias=True)
    ref = reference(H, W, target, b, w)
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), ref, ty, k)
    check(ctx.softmax_ce(H, W, target, bias=b), ref, ty, k, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,k", [(1, 1100, 20), (2, 9000, 30), (309, 25322, 22), (4, 48241, 43), (1, 20000, 64), (33, 60000, 8),
                                   (40, 9000, 110), (3, 5001, 200), (6000, 150, 25), (20000, 3, 9)])
def test_split_sums(ctx, n, v, k, ty):
    """A few rows against many items, and many rows against a few: the sums come from up to hundreds of pieces."""
    H, W, target, b, w = make(n, v, k, ty, seed=n + v, bias=True, gone=0.1)
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), ty, k)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 17, 8), (2, 130, 100), (3, 129, 128), (4, 1000, 129), (4, 5000, 256), (1, 70001, 257), (2, 9001, 317),
                                   (4, 2000, 512), (5, 2000, 60)])
def test_a_few_rows_without_gradients(ctx, n, v, k, ty):
    H, W, target, b, _ = make(n, v, k, ty, seed=n + v, bias=v > 1, gone=0.1)
    big = torch.full((v, k + 3), math.nan, dtype=T[ty], device="cuda")
    big[:, :k] = W
    for table in (W, big[:, :k]):  # (aligned rows, and others)
        check(ctx.softmax_ce(H, table, target, bias=b), reference(H, W, target, b), ty, k, grad=False)
    if n > 1:
        target[1], H[1] = -1, math.nan
        W[v // 2] = math.nan
        if b is not None and v > 2:
            b[v // 2] = -math.inf
            check(ctx.softmax_ce(H, W, target, bias=b), reference(H, W, target, b), ty, k, grad=False)
    gone = torch.full((v,), -math.inf, device="cuda")
    loss, lse = ctx.softmax_ce(H, W, target, bias=gone)
    known = target >= 0
    assert (lse[known] == -math.inf).all() and (loss == 0).all() and (lse[~known] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
def test_no_bias_no_weight(ctx, ty):
    H, W, target, _, _ = make(77, 333, 40, ty, seed=3)
    check(ctx.softmax_ce(H, W, target, grad=True), reference(H, W, target), ty, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
def test_withdrawn_items_and_unknown_rows_hold_anything(ctx, ty):
    """NaN, infinities and the type's largest values in withdrawn items' and unknown rows' places reach no output."""
    n, v, k = 150, 700, 50
    H, W, target, b, w = make(n, v, k, ty, seed=5, bias=True, gone=0.3, unknown=0.2)
    gone = b == -math.inf
    target = torch.where((target >= 0) & gone[target.clamp(min=0).long()], torch.zeros_like(target), target)
    target[3], target[7] = v, 2 ** 31 - 1  # past the catalogue: unknown too
    ref = reference(H, W, target, b, w)
    bad = [math.nan, math.inf, -math.inf, torch.finfo(T[ty]).max, torch.finfo(T[ty]).min]
    off = ((target < 0) | (target >= v)).nonzero().flatten().tolist()
    for i, x in enumerate(off):
        H[x] = bad[i % 5]
        w[x] = bad[(i + 1) % 5]
    for i, x in enumerate(gone.nonzero().flatten().tolist()):
        W[x] = bad[i % 5]
    out = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    check(out, ref, ty, k)
    assert (out[2][off] == 0).all() and (out[0][off] == 0).all() and (out[1][off] == 0).all()
    assert (out[3][gone] == 0).all() and (out[4][gone] == 0).all()


@pytest.mark.gpu
def test_everything_withdrawn_and_withdrawn_targets(ctx):
    H, W, target, b, w = make(40, 90, 16, "f32", seed=6, bias=True)
    target[0] = -1
    none = torch.full_like(b, -math.inf)
    loss, lse, dH, dW, db = ctx.softmax_ce(H, W, target, bias=none, weight=w, grad=True)
    assert (loss == 0).all() and (lse[1:] == -math.inf).all() and lse[0] == 0
    assert (dH == 0).all() and (dW == 0).all() and (db == 0).all()
    b[target[5].item()] = -math.inf  # row 5 (and rows of the same target) ask for a withdrawn item
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), "f32", 16)
    ids = torch.full_like(target, -1)
    for x in ctx.softmax_ce(H, W, ids, bias=b, weight=w, grad=True):
        assert (x == 0).all()


@pytest.mark.gpu
def test_bias_of_the_lowest_value(ctx):
    """A bias of the type's lowest value is no withdrawal, and no infinity: the item only never wins."""
    H, W, target, b, w = make(30, 64, 24, "f32", seed=8, bias=True)
    b[10:20] = torch.finfo(torch.float32).min
    target[:] = 30
    ref = reference(H, W, target, b, w)
    ref["L"] = ref["L"] * 0 + (H.double().abs() @ W.double().abs().T).max().cpu() + 5  # the lowest values' logits decide nothing
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), ref, "f32", 24)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(5, 33), (200, 3000)])
def test_every_bias_of_the_lowest_value(ctx, n, v):
    """Every logit is the type's lowest value (the products vanish beside it): each item has the probability 1 / v."""
    H, W, target, b, w = make(n, v, 16, "f32", seed=15, bias=True)
    b[:] = torch.finfo(torch.float32).min
    loss, lse, dH, dW, db = (x.double().cpu() for x in ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True))
    assert torch.isfinite(lse).all() and (lse < -1e35).all()
    u = 16 * U32
    assert ((loss - math.log(v)).abs() <= u * math.log(v)).all()
    c = torch.full((n, v), 1.0 / v, dtype=torch.float64)
    c[torch.arange(n), target.cpu().long()] -= 1
    c *= w.double().cpu()[:, None]
    Hd, Wd = H.double().cpu(), W.double().cpu()
    assert ((dH - c @ Wd).abs() <= (u + v * U32) * (c.abs() @ Wd.abs())).all()
    assert ((dW - c.T @ Hd).abs() <= (u + n * U32) * (c.abs().T @ Hd.abs())).all()
    assert ((db - c.sum(0)).abs() <= (u + n * U32) * c.abs().sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("where", ["late", "zeros", "huge", "tiny"])
def test_scales_from_a_sample(ctx, ty, where):
    """Tables too large to be looked through before they are scaled: the sampled rows mislead about the rest."""
    n, v, k = 700, 4000, 64
    H, W, target, b, w = make(n, v, k, ty, seed=16, bias=True)
    if where == "late":  # one row far above the others, which no sample of every 30th row meets
        W[1237] *= 300.0
        H[333] *= 0.01
    elif where == "zeros":
        W[::31] = 0
        H[::5] = 0
    elif where == "huge":
        H *= 1e-18
        W *= 1e18
    else:
        W *= 1e-25
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), ty, k)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_large_logits(ctx, ty):
    """Rows whose logits spread over hundreds: one item takes nearly all, the running maximum moves through the catalogue."""
    H, W, target, b, w = make(65, 900, 64, ty, seed=9, spread=80.0, bias=True)
    W = W[torch.argsort((H[0].float() @ W.float().T))].contiguous()  # row 0's logits ascend
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), ty, 64)


@pytest.mark.gpu
def test_fp32_spread_of_magnitudes(ctx):
    """fp32 pairs are scaled by the largest element of a matrix: rows thousands of times smaller keep their values."""
    H, W, target, b, w = make(96, 400, 60, "f32", seed=10, bias=True)
    W[::7] *= 1e-4
    H[::5] *= 1e-4
    W[3] *= 30
    check(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), "f32", 60)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_strided_and_unaligned_rows(ctx, ty):
    H, W, target, b, w = make(50, 260, 37, ty, seed=11, bias=True)
    big = torch.full((50, 90), math.nan, dtype=T[ty], device="cuda")
    big[:, 3:40] = H
    tab = torch.full((260, 41), math.nan, dtype=T[ty], device="cuda")
    tab[:, 1:38] = W
    ref = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    out = ctx.softmax_ce(big[:, 3:40], tab[:, 1:38], target, bias=b, weight=w, grad=True)
    for x, y in zip(out, ref):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_gradient_against_differences(ctx):
    """dH, dW and dbias against central differences of the operator's own loss (in fp32: steps of 2^-6, error h^2 of
    the third derivative, bounded by 1 for these sizes, and the loss's rounding over the step)."""
    H, W, target, b, w = make(12, 40, 8, "f32", seed=12, bias=True)
    _, _, dH, dW, db = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    h = 2.0 ** -6
    def total(H, W, b):
        return float((ctx.softmax_ce(H, W, target, bias=b)[0].double() * w.double()).sum())
    L = float((H.double().abs() @ W.double().abs().T).max()) + 4
    # sum of 12 losses, each off by 2 (k + 10) u32 (L + 1); third derivative of a loss along a unit coordinate: below |x|^3
    tol = 12 * 1.5 * (2 * 18 * U32 * (L + 1)) / h + 12 * 1.5 * h * h * max(float(H.abs().max()), float(W.abs().max()), 1.0) ** 3
    for M, g, idx in ((H, dH, [(0, 0), (5, 7), (11, 3)]), (W, dW, [(0, 0), (39, 7), (int(target[2]), 4)])):
        for i, j in idx:
            keep = M[i, j].item()
            M[i, j] = keep + h
            up = total(H, W, b)
            M[i, j] = keep - h
            dn = total(H, W, b)
            M[i, j] = keep
            assert abs((up - dn) / (2 * h) - float(g[i, j])) <= tol
    for i in (0, int(target[1]), 39):
        keep = b[i].item()
        b[i] = keep + h
        up = total(H, W, b)
        b[i] = keep - h
        dn = total(H, W, b)
        b[i] = keep
        assert abs((up - dn) / (2 * h) - float(db[i])) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("v,k,top", [(2, 33, 4.0), (9, 64, 8.0), (300, 20, 12.0), (500, 100, 16.0)])
def test_rows_that_are_nearly_learnt(ctx, ty, v, k, top):
    """Targets with a probability near one (their bias is `top` above the others', a target's logit passes the others' by
    up to 2 top): the gradients are the others' small coefficients c and their sum for the target, each off by 2 e_l and
    8 u32 of itself (the target's besides by the roundings of a sum of v) and its own rounding, not by a step of the
    target's row; the loss is their log1p, off by the same relative error."""
    n = 64
    H, W, _, _, w = make(n, v, k, ty, seed=v, spread=1.0)
    target = torch.full((n,), v // 2, dtype=torch.int32, device="cuda")
    b = torch.linspace(-0.5, 0.5, v, device="cuda")
    b[v // 2] = top
    loss, lse, dH, dW, db = (x.double().cpu() for x in ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True))
    ref = reference(H, W, target, b, w)
    e_l = (k + 10) * U32 * (ref["L"] + 1)
    assert ((loss - ref["loss"]).abs() <= (2 * e_l + (v + 8) * U32) * ref["loss"]).all()
    c, g = ref["c"], ref["g"]
    others = c.clone()
    others[:, v // 2] = 0.0
    c[:, v // 2] = -others.sum(1)
    u_c = U_C[ty]
    ec = (2 * e_l[:, None] + 8 * U32 + u_c) * c.abs()
    ec[:, v // 2] += v * U32 * c[:, v // 2].abs()
    floor = float(g.max()) * 2.0 ** -38  # (fp16 coefficients of the items' pass)
    Wm, Hm = W.double().cpu(), H.double().cpu()
    for name, x, r, lim in (("dH", dH, c @ Wm, ec @ Wm.abs() + (v + 4) * U32 * (c.abs() @ Wm.abs())),
                            ("dW", dW, c.T @ Hm, (ec + floor).T @ Hm.abs() + (n + 4) * U32 * (c.abs().T @ Hm.abs())),
                            ("db", db, c.sum(0), (ec + floor).sum(0) + (n + 4) * U32 * c.abs().sum(0))):
        ut = U32 if name == "db" else half_step(T[ty])
        tiny = 2.0 ** -24 if ty == "f16" and name != "db" else 1e-38
        err = (x - r).abs()
        lim = lim * (1 + ut) + ut * r.abs() + tiny
        assert (err <= lim).all(), (name, float((err / lim).max()))


@pytest.mark.gpu
def test_many_rows(ctx):
    """More rows than one axis of a launch holds waves for.  Two items of one factor: l = h w_v, p = sigmoid.  A few fp32
    roundings of lse; a coefficient's 2^-11 and half a step of bf16 for dH; the sums of dW and dbias besides by a rounding
    for each of at most 2^26 / 16 products of a split, which stay below 2^-11 of the sum of magnitudes too."""
    n = 2 ** 26 + 300
    h = (torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) / 4).bfloat16()
    W = torch.tensor([[0.5], [-1.25]], device="cuda").bfloat16()
    target = (torch.arange(n, device="cuda") % 3 - 1).int()
    loss, lse, dH, dW, db = ctx.softmax_ce(h[:, None], W, target, grad=True)
    dW, db = dW.double(), db.double()
    w = W.double()[:, 0]
    gw, gb, mag = torch.zeros(2, dtype=torch.float64, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda"), 0.0
    for a in range(0, n, 1 << 24):
        x, t = h[a:a + (1 << 24)].double(), target[a:a + (1 << 24)].long()
        there = t >= 0
        l = x[:, None] * w
        z = torch.logsumexp(l, 1)
        assert ((lse[a:a + (1 << 24)] - z * there).abs() <= 16 * 2.0 ** -24 * (1 + l.abs().amax(1))).all()
        lt = l.gather(1, t.clamp(min=0)[:, None])[:, 0]
        assert ((loss[a:a + (1 << 24)] - (z - lt) * there).abs() <= 16 * 2.0 ** -24 * (1 + l.abs().amax(1))).all()
        c = (torch.exp(l - z[:, None]) - torch.nn.functional.one_hot(t.clamp(min=0), 2)) * there[:, None]
        d = (c * w).sum(1)
        assert ((dH[a:a + (1 << 24), 0] - d).abs() <= 2.0 ** -8 * d.abs() + 2.0 ** -10 * w.abs().sum()).all()
        gw += (x[:, None] * c).sum(0)
        gb += c.sum(0)
        mag += float((c.abs() * (1 + x.abs()[:, None])).sum())
    assert ((dW[:, 0] - gw).abs() <= 2.0 ** -8 * gw.abs() + 2.0 ** -10 * mag).all()
    assert ((db - gb).abs() <= 2.0 ** -10 * mag).all()


@pytest.mark.gpu
def test_rows_far_apart(ctx):
    """Rows of H and W further apart than 32 bits of elements."""
    step = 2 ** 31 + 8
    big = torch.empty(2 * step + 64, dtype=torch.float16, device="cuda")
    far = big.as_strided((3, 20), (step, 1))
    far.copy_(torch.randn(3, 20, generator=torch.Generator().manual_seed(1)))
    W = torch.randn(70, 20, generator=torch.Generator().manual_seed(2)).half().cuda()
    target = torch.tensor([4, 69, 0], dtype=torch.int32, device="cuda")
    for x, y in zip(ctx.softmax_ce(far, W, target, grad=True), ctx.softmax_ce(far.contiguous(), W, target, grad=True)):
        assert torch.equal(x, y)
    target = torch.arange(70, dtype=torch.int32, device="cuda") % 3
    for x, y in zip(ctx.softmax_ce(W, far, target, grad=True), ctx.softmax_ce(W, far.contiguous(), target, grad=True)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_same_call_same_bits(ctx):
    H, W, target, b, w = make(300, 5000, 48, "f32", seed=13, bias=True)
    one = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    two = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    for x, y in zip(one, two):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_side_stream_and_graph(ctx):
    H, W, target, b, w = make(200, 3000, 64, "f32", seed=14, bias=True)
    ref = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(out, ref):
        assert torch.equal(x, y)
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    with torch.cuda.graph(g2):
        out2 = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    for step in range(3):
        H.mul_(0.5)
        W[step] += 1.0
        for x in out + out2:
            x.fill_(7.0)
        g.replay()
        g2.replay()
        torch.cuda.synchronize()
        ref = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
        for x, z, y in zip(out, out2, ref):
            assert torch.equal(x, y) and torch.equal(z, y)


@pytest.mark.gpu
def test_tensor_refusals(ctx):
    H, W, target, b, w = make(8, 20, 6, "f32", bias=True)
    with pytest.raises(ValueError):
        ctx.softmax_ce(H.cpu(), W, target)
    with pytest.raises(ValueError):
        ctx.softmax_ce(H, W[:, :5], target)
    with pytest.raises(TypeError):
        ctx.softmax_ce(H, W, target.long())
    with pytest.raises(TypeError):
        ctx.softmax_ce(H, W.half(), target)
    with pytest.raises(TypeError):
        ctx.softmax_ce(H.double(), W.double(), target)
    with pytest.raises(ValueError):
        ctx.softmax_ce(H, W, target[:7])
    with pytest.raises(ValueError):
        ctx.softmax_ce(H.t().contiguous().t(), W, target)
    with pytest.raises(ValueError):
        ctx.softmax_ce(H[:0], W, target[:0])
    with pytest.raises(rsgpu.RsError) as e:
        ctx.softmax_ce(torch.zeros(2, 513, device="cuda"), torch.zeros(3, 513, device="cuda"), target[:2])
    assert e.value.code == rsgpu.RS_ERR_UNSUPPORTED


def test_entry_point_refusals():
    """The C entry points refuse before they touch a device (no context, and one whose memory is never read)."""
    L = rsgpu.lib()
    need = C.c_int64(-1)
    assert L.rs_softmax_ce_workspace(None, 0, 10, 20, 8, 1, C.byref(need)) == rsgpu.RS_OK and need.value > 0
    assert L.rs_softmax_ce_workspace(None, 0, 10, 20, 8, 1, None) == rsgpu.RS_ERR_INVALID
    assert L.rs_softmax_ce_workspace(None, 3, 10, 20, 8, 1, C.byref(need)) == rsgpu.RS_ERR_INVALID
    assert L.rs_softmax_ce_workspace(None, 0, -1, 20, 8, 1, C.byref(need)) == rsgpu.RS_ERR_INVALID
    assert L.rs_softmax_ce_workspace(None, 0, 1, 2 ** 31, 8, 1, C.byref(need)) == rsgpu.RS_ERR_INVALID
    assert L.rs_softmax_ce_workspace(None, 0, 1, 2, 0, 1, C.byref(need)) == rsgpu.RS_ERR_INVALID
    assert L.rs_softmax_ce_workspace(None, 0, 1, 2, 513, 1, C.byref(need)) == rsgpu.RS_ERR_UNSUPPORTED
    assert L.rs_softmax_ce_workspace(None, 0, 0, 5, 8, 1, C.byref(need)) == rsgpu.RS_OK and need.value == 0

    buf = C.create_string_buffer(1 << 16)
    base = (C.addressof(buf) + 255) & ~255
    good = dict(type=0, n=4, v=6, k=8, H=base, ldh=8, W=base, ldw=8, bias=None, target=base, weight=None, loss=base,
                lse=base, dH=None, lddh=8, dW=None, lddw=8, db=None, ws=base, ws_bytes=1 << 40, stream=None)

    def call(**kw):
        a = dict(good, **kw)
        return L.rs_softmax_ce(None, a["type"], a["n"], a["v"], a["k"], a["H"], a["ldh"], a["W"], a["ldw"], a["bias"], a["target"],
                               a["weight"], a["loss"], a["lse"], a["dH"], a["lddh"], a["dW"], a["lddw"], a["db"], a["ws"],
                               a["ws_bytes"], a["stream"])
    for kw in (dict(), dict(type=7), dict(n=-1), dict(v=0), dict(n=0), dict(k=0), dict(H=None), dict(H=base + 2), dict(ldh=7),
               dict(W=None), dict(ldw=5), dict(target=None), dict(target=base + 1), dict(loss=None), dict(lse=None), dict(dH=base),
               dict(dH=base, dW=base), dict(dH=base, dW=base, db=base, lddw=3), dict(bias=base + 2), dict(weight=base + 1),
               dict(ws=None), dict(ws=base + 4), dict(ws_bytes=100)):
        assert call(**kw) == rsgpu.RS_ERR_INVALID, kw  # (the first: no context)
        assert L.rs_last_error(None)
    assert call(k=600, ldh=600, ldw=600) == rsgpu.RS_ERR_UNSUPPORTED
    assert call(n=0, v=0) == rsgpu.RS_OK
