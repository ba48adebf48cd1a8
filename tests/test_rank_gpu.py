"""The dense operators on a plan's resident factors: the ranking step (loss, gradient and orthogonalised update together)
against the same step in 64 bits, the catalogue's scores against the plan's own predictions, and both among epochs."""
import math

import numpy as np
import pytest

import rsgpu

COEF = (3.4445, -4.7750, 2.0315)
U32 = 2.0 ** -24


def make_plan(ctx, n_users=60, n_items=90, k=20, nnz=1500, seed=0):
    rng = np.random.default_rng(seed)
    u = rng.integers(0, n_users, nnz).astype(np.int32)
    i = np.minimum(rng.geometric(0.05, nnz) - 1, n_items - 1).astype(np.int32)
    r = rng.integers(1, 6, nnz).astype(np.float64)
    plan = ctx.svd_plan(rsgpu.Ratings(u, i, r, n_users, n_items), k)
    P, Q = rng.normal(0, 0.5, (n_users, k)), rng.normal(0, 0.5, (n_items, k))
    plan.upload(P.astype(np.float32), Q.astype(np.float32), rng.normal(0, 0.2, n_users).astype(np.float32),
                rng.normal(0, 0.2, n_items).astype(np.float32), 3.5)
    return plan


def orthogonalized(G):
    X = G / np.linalg.norm(G)
    a, b, c = COEF
    for _ in range(5):
        A = X.T @ X if X.shape[0] >= X.shape[1] else X @ X.T
        M = b * A + c * A @ A
        X = a * X + (X @ M if X.shape[0] >= X.shape[1] else M @ X)
    return X


def reference_step(P, Q, bi, users, items, lr, q_lr, reg):
    ok = (users >= 0) & (users < len(P)) & (items >= 0) & (items < len(Q))
    u, t = users[ok], items[ok]
    m = len(u)
    H = P[u]
    z = H @ Q.T + bi
    z -= z.max(1, keepdims=True)
    lse = np.log(np.exp(z).sum(1))
    loss = float((lse - z[np.arange(m), t]).mean())
    c = np.exp(z - lse[:, None])
    c[np.arange(m), t] -= 1
    c /= m
    gP = np.zeros_like(P)
    np.add.at(gP, u, c @ Q)
    cnt = np.bincount(u, minlength=len(P))
    gQ, gb = c.T @ H, c.sum(0)
    P1 = P - lr * (gP + reg * (cnt / m)[:, None] * P)
    return loss, P1, Q - q_lr * (orthogonalized(gQ) + reg * Q), bi - lr * gb, gP, gQ


def logit_bound(P, Q, bi):
    """Logits of up to L, products of k terms and a bias in fp32 (operands rounded from pairs: one more step each)."""
    k = P.shape[1]
    return (k + 10) * U32 * (np.abs(P).max() * np.abs(Q).max() * k + np.abs(bi).max() + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [5, 20, 100])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_step_against_64_bits(ctx, n, k):
    plan = make_plan(ctx, k=k)
    rng = np.random.default_rng(n)
    users, items = rng.integers(0, 60, n).astype(np.int32), rng.integers(0, 90, n).astype(np.int32)
    if n > 1:
        users[3], items[5], users[7], items[9] = -1, -1, 60, 90   # unknown
        users[10:14] = users[10]                                  # one user several times
    P, Q, bu, bi, gb = plan.download()
    lr, q_lr, reg = 0.7, 0.05, 0.01
    loss, P1, Q1, b1, gP, gQ = reference_step(P, Q, bi, users, items, lr, q_lr, reg)
    got = plan.rank_step(users, items, lr, q_lr, reg)
    Pg, Qg, bug, big, gbg = plan.download()
    # logits off by e; a gradient's coefficients by 2 e + 8 u32 of themselves, its sums by their length's roundings, a
    # row's coefficients sum to at most 2 weight; a step adds four roundings of the row
    e = logit_bound(P, Q, bi)
    assert abs(got - loss) <= 2 * e + 4 * U32 * loss
    rel = 2 * e + (n + 98) * U32
    assert np.abs(Pg - P1).max() <= lr * rel * 2 * np.abs(Q).max() + 6 * U32 * np.abs(P1).max()
    assert np.abs(big - b1).max() <= lr * rel * 2 + 6 * U32
    # the update of the items: its gradient's relative error is carried by the polynomials to at most a^5 of the weakest
    # direction's share; the errors of the gradient are random, so against its norm they are e-sized
    O, Og = (Q - Q1) / q_lr - reg * Q, (Q - Qg) / q_lr - reg * Q
    assert np.linalg.norm(Og - O) <= (COEF[0] ** 5 * rel + 8 * U32 * np.sqrt(O.size) * np.abs(Q).max() / q_lr / np.linalg.norm(O)) * np.linalg.norm(O)
    assert np.array_equal(bu, bug) and gb == gbg
    untouched = np.setdiff1d(np.arange(60), users)
    assert np.array_equal(P[untouched], Pg[untouched])
    plan.close()


@pytest.mark.gpu
def test_steps_between_epochs(ctx):
    """Epochs, steps and scores on one plan, as a program mixes them: everything stays finite and each call sees the
    factors that the one before left."""
    plan = make_plan(ctx, k=16)
    rng = np.random.default_rng(3)
    users, items = rng.integers(0, 60, 200).astype(np.int32), rng.integers(0, 90, 200).astype(np.int32)
    plan.epochs(2)
    for _ in range(3):
        P, Q, bu, bi, gb = plan.download()
        want = reference_step(P, Q, bi, users, items, 1.0, 0.02, 0.0)[0]
        got = plan.rank_step(users, items)
        assert abs(got - want) <= 2 * logit_bound(P, Q, bi) + 4 * U32 * want
        plan.epochs(1)
    out = plan.score_items(np.arange(60))
    assert np.isfinite(out).all()
    assert all(np.isfinite(x).all() for x in plan.download()[:4])
    plan.close()


@pytest.mark.gpu
def test_item_copies_follow_a_step(ctx):
    """The hybrid schedule keeps copies of hot items' rows: after a step they hold the stepped rows (an epoch that learns
    nothing leaves the factors as they are, up to its fixed point of 2^-24)."""
    plan = make_plan(ctx, k=12, nnz=4000)
    plan.set_mode(rsgpu.WB_ATOMIC)
    plan.set_hot_replicas(16, 4)
    plan.epochs(1)
    users = np.arange(40, dtype=np.int32)
    plan.rank_step(users, (users * 2).astype(np.int32), q_lr=0.5)
    before = plan.download()
    plan.epochs(1, lr=0.0, reg=0.0)
    after = plan.download()
    for a, b in zip(before[:4], after[:4]):
        assert np.abs(a - b).max() <= 2.0 ** -24
    plan.close()


@pytest.mark.gpu
def test_nothing_known(ctx):
    plan = make_plan(ctx)
    before = plan.download()
    assert math.isnan(plan.rank_step([], []))
    assert math.isnan(plan.rank_step([-1, 60, 3], [4, 4, 90]))
    for a, b in zip(before, plan.download()):
        assert np.array_equal(a, b)
    assert plan.score_items([]).shape == (0, 90)
    with pytest.raises(ValueError):
        plan.rank_step([1, 2], [3])
    with pytest.raises(rsgpu.RsError):
        plan.rank_step([1], [2], lr=math.nan)
    with pytest.raises(rsgpu.RsError):
        plan.rank_step([1], [2], q_lr=1e300)  # finite, but no float
    with pytest.raises(rsgpu.RsError):
        plan.rank_step(np.zeros((1 << 20) + 1, np.int32), np.zeros((1 << 20) + 1, np.int32))
    for a, b in zip(before, plan.download()):
        assert np.array_equal(a, b)
    plan.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(1, 20), (30, 7), (200, 100)])
def test_scores_against_predictions(ctx, n, k):
    plan = make_plan(ctx, k=k)
    rng = np.random.default_rng(n)
    users = rng.integers(-1, 62, n).astype(np.int32)  # some unknown
    out = plan.score_items(users).astype(np.float64)
    P, Q, bu, bi, gb = plan.download()
    want = np.stack([plan.predict(np.full(90, u, np.int32), np.arange(90, dtype=np.int32)) for u in users])
    known = (users >= 0) & (users < 60)
    p = np.where(known[:, None], P[np.clip(users, 0, 59)], 0)
    sp, sq = np.abs(p).max(1) / 127, np.abs(Q).max(1) / 127
    bound = (sp[:, None] * np.abs(Q).sum(1) + np.abs(p).sum(1)[:, None] * sq) / 2 + k * sp[:, None] * sq / 4
    bound = bound * (1 + 1e-6) + 8 * U32 * (np.abs(want) + np.abs(p) @ np.abs(Q).T + 5)
    assert (np.abs(out - want) <= bound).all()
    assert np.array_equal(out[~known], np.broadcast_to((np.float32(gb) + bi.astype(np.float32)).astype(np.float64), (int((~known).sum()), 90)))
    plan.close()


def test_entry_point_refusals():
    L = rsgpu.lib()
    assert L.rs_svd_plan_rank_step(None, 0, None, None, 0.1, 0.1, 0.0, None) == rsgpu.RS_ERR_INVALID
    assert L.rs_svd_plan_score_items(None, 0, None, None) == rsgpu.RS_ERR_INVALID


def tables(plan):
    return [x.copy() if isinstance(x, np.ndarray) else x for x in plan.download()]


@pytest.mark.gpu
@pytest.mark.parametrize("why", ["logits", "row", "rate", "item rate", "bias"])
def test_a_step_out_of_range_changes_nothing(ctx, why):
    """A logit, a gradient or a stepped value that is not finite: RS_ERR_NUMERIC, and every factor and bias as it was."""
    plan = make_plan(ctx)
    users, items = np.arange(40, dtype=np.int32), (np.arange(40) * 2).astype(np.int32)
    good = tables(plan)
    P, Q, bu, bi, gb = tables(plan)
    rates = dict(lr=0.5, q_lr=0.05)
    if why == "logits":
        P, Q = P * 1e22, Q * 1e22
    elif why == "row":
        P[7, 3] = np.nan
    elif why == "bias":
        bi[11] = np.inf
    elif why == "rate":
        rates["lr"] = 3e38
        P, Q = P * 2.0, Q * 50.0
    else:
        rates["q_lr"] = 3e38
        Q[5] = 3e38 * np.sign(Q[5] + 1e-3)
        P = P * 1e-39
    plan.upload(*(x.astype(np.float32) for x in (P, Q, bu, bi)), gb)
    before = tables(plan)
    with pytest.raises(rsgpu.RsError) as e:
        plan.rank_step(users, items, reg=0.01, **rates)
    assert e.value.code == rsgpu.RS_ERR_NUMERIC
    for a, b in zip(before, tables(plan)):
        assert np.array_equal(a, b, equal_nan=True)
    plan.upload(*(x.astype(np.float32) for x in good[:4]), gb)  # and the plan goes on
    assert np.isfinite(plan.rank_step(users, items))
    assert all(np.isfinite(x).all() for x in plan.download()[:4])
    plan.close()


@pytest.mark.gpu
def test_a_withdrawn_item_stays_withdrawn(ctx):
    """An item bias of -inf withdraws the item; a step leaves it so, and is none that leaves the range."""
    plan = make_plan(ctx)
    P, Q, bu, bi, gb = tables(plan)
    bi[4] = -np.inf
    plan.upload(*(x.astype(np.float32) for x in (P, Q, bu, bi)), gb)
    users = np.arange(50, dtype=np.int32)
    items = np.where(users % 90 == 4, 5, users).astype(np.int32)
    assert np.isfinite(plan.rank_step(users, items))
    got = plan.download()
    assert got[3][4] == -np.inf and np.isfinite(np.delete(got[3], 4)).all() and all(np.isfinite(x).all() for x in got[:2])
    plan.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n_items,k", [(90, 5), (90, 100), (300, 280), (270, 300), (1200, 64)])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_step_is_its_operators(ctx, n_items, k, n):
    """A step is softmax_ce of the gathered rows with weights 1 / m, orthogonalize of its dW and the documented sums in fp32:
    the same bits as those calls and numpy's fp32 give (each operator has its own tests against 64 bits)."""
    torch = pytest.importorskip("torch")
    plan = make_plan(ctx, n_items=n_items, k=k)
    rng = np.random.default_rng(n + k)
    users, items = rng.integers(0, 60, n).astype(np.int32), rng.integers(0, n_items, n).astype(np.int32)
    if n > 1:
        users[3], items[5], users[7], items[9] = -1, -1, 60, n_items   # unknown
        users[10:14] = users[10]                                       # one user several times
    P, Q, bu, bi, gb = plan.download()
    P, Q, bi = P.astype(np.float32), Q.astype(np.float32), bi.astype(np.float32)
    ok = (users >= 0) & (users < 60) & (items >= 0) & (items < n_items)
    m = int(ok.sum())
    H = np.where(((users >= 0) & (users < 60))[:, None], P[np.clip(users, 0, 59)], np.float32(0))
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    loss, _, dH, dW, db = ctx.softmax_ce(dev(H), dev(Q), dev(np.where(ok, items, -1).astype(np.int32)), bias=dev(bi),
                                         weight=torch.full((n,), 1.0 / m, device="cuda"), grad=True)
    O = ctx.orthogonalize(dW).cpu().numpy()
    dH, db = dH.cpu().numpy(), db.cpu().numpy()
    lr, q_lr, reg = np.float32(0.7), np.float32(0.05), np.float32(0.01)
    P1, Q1 = P.copy(), Q - q_lr * (O + reg * Q)
    for u in np.unique(users[ok]):
        rows = np.nonzero(ok & (users == u))[0]
        g = np.zeros(k, np.float32)
        for r in rows:
            g = g + dH[r]
        P1[u] = P[u] - lr * (g + (reg / np.float32(m) * np.float32(len(rows))) * P[u])
    got = plan.rank_step(users, items, 0.7, 0.05, 0.01)
    Pg, Qg, bug, big, gbg = plan.download()
    assert np.array_equal(Pg.astype(np.float32), P1) and np.array_equal(Qg.astype(np.float32), Q1)
    assert np.array_equal(big.astype(np.float32), bi - lr * db) and np.array_equal(bu, bug) and gb == gbg
    assert got == float(loss.cpu().numpy().astype(np.float64)[ok].sum() / m) or abs(got - float(loss.double().sum()) / m) <= n * 2.0 ** -52 * got
    plan.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n_items,k,n", [(90, 100, 40), (90, 100, 1), (300, 280, 60)])
def test_item_update_against_64_bits(ctx, n_items, k, n):
    """The whole item update in 64 bits, with factors whose logits are near 0.  The gradient G is off by at most E = rel (|c|^T
    |H|), rel the coefficients' and the sums' errors; the steps' polynomial of a matrix moves by at most its steepest slope,
    a^5 = 485 at 0, times what moves G / |G|, 2 |E| / |G| at most; the operator's own error is test_ortho.py's bound, and
    reading O back from the step costs 8 roundings of Q / q_lr.  All in all below a quarter: an update that is missing is off
    by 1, one of the wrong sign by 2."""
    import test_ortho
    torch = pytest.importorskip("torch")
    plan = make_plan(ctx, n_items=n_items, k=k)
    rng = np.random.default_rng(k)
    small = lambda *s: rng.normal(0, 0.03, s).astype(np.float32)
    plan.upload(small(60, k), small(n_items, k), small(60), small(n_items), 3.5)
    users, items = rng.integers(0, 60, n).astype(np.int32), rng.integers(0, n_items, n).astype(np.int32)
    P, Q, bu, bi, gb = plan.download()
    lr, q_lr, reg = 0.7, 0.05, 0.01
    _, _, Q1, _, _, gQ = reference_step(P, Q, bi, users, items, lr, q_lr, reg)
    plan.rank_step(users, items, lr, q_lr, reg)
    Qg = plan.download()[1]
    H = P[users]
    e = (k + 10) * U32 * ((np.abs(H) @ np.abs(Q).T).max() + np.abs(bi).max() + 1)
    z = H @ Q.T + bi
    c = np.exp(z - z.max(1, keepdims=True))
    c /= c.sum(1, keepdims=True)
    c[np.arange(n), items] -= 1
    E = (2 * e + 8 * U32 + (n + 4) * U32) * (np.abs(c).T @ np.abs(H)) / n
    O, Og = (Q - Q1) / q_lr - reg * Q, (Q - Qg) / q_lr - reg * Q
    _, own = test_ortho.reference(torch.from_numpy(gQ), gram=0.0)
    tol = 2 * COEF[0] ** 5 * np.linalg.norm(E) / np.linalg.norm(gQ)
    tol = tol + float(own.norm()) + 8 * U32 * np.linalg.norm(Q) / q_lr
    assert tol < 0.25 * np.linalg.norm(O)
    assert np.linalg.norm(Og - O) <= tol
    plan.close()


@pytest.mark.gpu
def test_scores_in_several_batches(ctx):
    """More scores than are held on the device at a time (2^26): a user's row is the same wherever it stands."""
    plan = make_plan(ctx, k=7)
    users = np.concatenate([np.arange(-1, 61), np.random.default_rng(1).integers(-1, 61, 2 ** 26 // 90 + 700)]).astype(np.int32)
    out = plan.score_items(users)
    one = plan.score_items(np.arange(-1, 61))
    assert out.shape == (len(users), 90)
    for a in range(0, len(users), 1 << 17):
        assert np.array_equal(out[a:a + (1 << 17)], one[users[a:a + (1 << 17)] + 1])
    plan.close()
