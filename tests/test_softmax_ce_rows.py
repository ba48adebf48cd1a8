"""Softmax cross entropy over the catalogue, row by row: every row of the gradients is held to its own terms, however
improbable the item, small the weight or large the table's elements.

Tolerances.  The names are test_softmax_ce.py's: a logit is off by e_l, a probability by 2 e_l and 4 u32 of itself, a
coefficient c besides by its rounding U_C and by FLOOR of the largest coefficient of its own sum: a sum holds its
coefficients times a power of two that keeps the largest so far at 2^8 (dW; 2^7: dH) or more, and fp16 rounds to steps
of 2^-24, half of one at most.  A probability below 2^-126 counts as zero.  An element of an fp32 table is held as a
pair: off by 2^-23 of itself (the step of the second piece, half of it), or by 2^-38 of the largest one.  The sums
take a rounding (u32 of their magnitudes) for each term, outputs half a step of their type, subnormal ones two steps.
"""
import math

import pytest

import rsgpu  # noqa: F401  (the library is built)

torch = pytest.importorskip("torch")

from test_softmax_ce import T, U32, U_C, half_step, make, reference  # noqa: E402

FLOOR = {"dH": 2.0 ** -32, "dW": 2.0 ** -33}


def check_rows(out, ref, ty, k):
    e_l = (k + 10) * U32 * (ref["L"] + 1)
    loss, lse = out[0].double().cpu(), out[1].double().cpu()
    assert ((loss - ref["loss"]).abs() <= 2 * e_l + 4 * U32 * ref["loss"].abs()).all()
    assert ((lse - ref["lse"]).abs() <= 2 * e_l + 4 * U32 * ref["lse"].abs()).all()
    n, v = ref["c"].shape
    c, g, p, Hm, Wm = ref["c"].abs(), ref["g"].abs(), ref["p"], ref["Hm"].abs(), ref["Wm"].abs()
    ec = g[:, None] * (2 * e_l[:, None] + 4 * U32) * p + U_C[ty] * c + g[:, None] * 2.0 ** -126
    lost = 2.0 ** -38 if ty == "f32" else 0.0
    size_H, size_W = c @ Wm, c.T @ Hm
    # the target's share of dH is the sum of the others' in fp32, not a difference (a target that takes all): its error is theirs
    eh = ec + FLOOR["dH"] * c.amax(1, keepdim=True)
    ew = ec + FLOOR["dW"] * c.amax(0, keepdim=True)
    bound = {"dH": eh @ Wm + (v + 12) * U32 * size_H + lost * Wm.max() * c.sum(1)[:, None],
             "dW": ew.T @ Hm + (n + 12) * U32 * size_W + lost * Hm.max() * c.sum(0)[:, None],
             "db": ec.sum(0) + (n + 4) * U32 * c.sum(0)}
    for name, x in (("dH", out[2]), ("dW", out[3]), ("db", out[4])):
        r, b, ut = ref[name], bound[name], half_step(x.dtype)
        tiny = 2 * torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        err = (x.double().cpu() - r).abs()
        lim = b * (1 + ut) + ut * r.abs() + tiny
        assert (err <= lim).all(), (name, float((err / lim).max()), int((err > lim).sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,k", [(128, 20000, 8), (128, 20000, 64), (1500, 900, 20), (20000, 60, 9), (65, 700, 200), (40, 300, 300)])
def test_improbable_items(ctx, n, v, k, ty):
    """Logits that spread over tens: most items of a row have probabilities of 1e-9 and less."""
    H, W, target, _, w = make(n, v, k, ty, seed=n + v, spread=10.0)
    check_rows(ctx.softmax_ce(H, W, target, weight=w, grad=True), reference(H, W, target, None, w), ty, k)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(70, 800), (3000, 300)])
def test_items_that_nobody_takes(ctx, ty, n, v):
    """Biases down to -75: probabilities of 1e-33, and a row of dW that is made of them alone."""
    k = 24
    H, W, target, _, w = make(n, v, k, ty, seed=n, spread=1.0)
    b = torch.linspace(0.0, -75.0, v, device="cuda")
    target %= v // 8
    out = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    check_rows(out, reference(H, W, target, b, w), ty, k)
    assert (out[3].float().abs().amax(1) > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(70, 3000), (3000, 300)])
def test_weights_far_apart(ctx, ty, n, v):
    """Weights over thirty powers of ten, ascending, descending and mixed along the batch."""
    k = 20
    H, W, target, b, _ = make(n, v, k, ty, seed=n, bias=True)
    w = torch.logspace(-25, 5, n, device="cuda")
    target[:] = torch.arange(n, device="cuda") % v  # an item has few rows of its own
    for order in (w, w.flip(0), w[torch.randperm(n, generator=torch.Generator().manual_seed(1))]):
        check_rows(ctx.softmax_ce(H, W, target, bias=b, weight=order, grad=True), reference(H, W, target, b, order), ty, k)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_one_item_takes_nearly_all(ctx, ty):
    """An item far above all others, which is nobody's target: the others' probabilities are 2^-30 and less."""
    n, v, k = 60, 5000, 16
    H, W, target, _, w = make(n, v, k, ty, seed=2, spread=1.0)
    b = torch.zeros(v, device="cuda")
    b[v // 2] = 24.0
    target[target == v // 2] = 0
    check_rows(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), ty, k)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("eh,ew", [(117, -117), (-117, 117), (124, -124), (-124, 122), (90, -90), (-140, 124), (60, -100), (-100, -100)])
def test_elements_of_any_size(ctx, ty, eh, ew):
    """Finite elements up to the type's largest and down to its subnormal ones, the logits between them of ordinary size or
    none."""
    n, v, k = 70, 500, 40
    H, W, target, b, w = make(n, v, k, ty, seed=3, spread=1.0, bias=True)
    H, W = (H.double() * 2.0 ** eh).to(T[ty]), (W.double() * 2.0 ** ew).to(T[ty])
    assert torch.isfinite(H).all() and torch.isfinite(W).all()
    ref = reference(H, W, target, b, w)
    check_rows(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), ref, ty, k)
    e_l = (k + 10) * U32 * (ref["L"] + 1)
    for rows in (70, 3):  # the loss alone, and its path for a few rows
        loss, _ = ctx.softmax_ce(H[:rows], W, target[:rows], bias=b)
        assert ((loss.double().cpu() - ref["loss"][:rows]).abs() <= (2 * e_l + 4 * U32 * ref["loss"])[:rows]).all()


@pytest.mark.gpu
def test_zeros_between_the_largest_elements(ctx):
    """Both tables at the type's largest, in columns where the other one is zero: logits of exactly the biases."""
    n, v, k = 40, 90, 32
    H, W, target, b, w = make(n, v, k, "f32", seed=4, bias=True)
    H[:, ::2], W[:, 1::2] = 0.0, 0.0
    H[:, 1::2] *= 2.0 ** 120
    W[:, ::2] *= 2.0 ** 120
    w = w * 2.0 ** -30
    check_rows(ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True), reference(H, W, target, b, w), "f32", k)


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", [(50, 400), (5000, 130)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_withdrawn_items_beside_rows_that_are_not_finite(ctx, ty, n, v, bad):
    """A known row that holds a NaN or an infinity reaches the items that are there, and the rows of dW and dbias of no
    withdrawn one: those are zero."""
    H, W, target, b, w = make(n, v, 24, ty, seed=5, bias=True, gone=0.3)
    gone = b == -math.inf
    target = torch.where(gone[target.long()], torch.zeros_like(target), target)
    H[7, 3] = bad
    loss, lse, dH, dW, db = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    assert (dW[gone] == 0).all() and (db[gone] == 0).all()
    assert torch.isnan(loss[7]) and torch.isnan(dW[~gone].float()).any(1).all()
    rest = [i for i in range(n) if i != 7]
    assert torch.isfinite(loss[rest]).all() and torch.isfinite(dH[rest].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_the_last_rows_of_many(ctx, grad):
    """More rows than one axis of a launch holds waves for, known ones only here and there: one in 2^20 of the first 2^26 and
    every third of the 300 behind them, so that each is seen in the sums.  Two items of one factor: bounds as in check_rows,
    with sums of the known rows' terms alone."""
    n, ty, k = 2 ** 26 + 300, "bf16", 1
    h = (torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) / 4).to(T[ty])
    W = torch.tensor([[0.5], [-1.25]], device="cuda").to(T[ty])
    target = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    known = torch.cat([torch.arange(5, 2 ** 26, 2 ** 20), torch.arange(2 ** 26, n, 3)]).cuda()
    target[known] = (torch.arange(len(known), device="cuda") % 2).int()
    w = torch.full((n,), math.nan, device="cuda")
    w[known] = torch.rand(len(known), device="cuda", generator=torch.Generator("cuda").manual_seed(2)) + 0.5
    ref = reference(h[known][:, None], W, target[known], None, w[known])
    if not grad:
        loss, lse = ctx.softmax_ce(h[:, None], W, target)
        e_l = (k + 10) * U32 * (ref["L"] + 1)
        assert ((loss[known].double().cpu() - ref["loss"]).abs() <= 2 * e_l + 4 * U32 * ref["loss"]).all()
        assert int((loss != 0).sum()) == len(known) and int((lse != 0).sum()) <= len(known)
        return
    loss, lse, dH, dW, db = ctx.softmax_ce(h[:, None], W, target, weight=w, grad=True)
    assert int((dH != 0).sum()) == len(known) and int((loss != 0).sum()) == len(known)
    check_rows((loss[known], lse[known], dH[known], dW, db), ref, ty, k)
    # a row less than all of them would be seen
    least = float((ref["c"].abs() * ref["Hm"].abs())[-100:].amax(1).median())
    assert least > 4 * float(half_step(T[ty]) * ref["dW"].abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("k", [64, 128, 256, 300, 512])
def test_sums_whose_scale_keeps_moving(ctx, ty, k):
    """Logits that ascend along the items by 100 (the users' sums follow a new maximum in every block) and weights that ascend
    along the rows by ten powers of ten (the items' sums follow a new largest coefficient)."""
    n, v = 600, 1000
    H, W, target, _, _ = make(n, v, k, ty, seed=k, spread=1.0)
    b = torch.linspace(-100.0, 0.0, v, device="cuda")
    w = torch.logspace(-6, 4, n, device="cuda") if ty != "f16" else torch.logspace(-3, 1, n, device="cuda")
    target[:] = torch.arange(n, device="cuda") % v
    out = ctx.softmax_ce(H, W, target, bias=b, weight=w, grad=True)
    check_rows(out, reference(H, W, target, b, w), ty, k)
