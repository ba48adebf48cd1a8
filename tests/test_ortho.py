"""Orthogonalised updates (rs_orthogonalize): refusals on the CPU, values against the steps in 64 bits on the GPU.

X = G T / |G| with T = f(A), A = G^T G / |G|^2 (or G G^T), f the steps' polynomials over s, formed in fp64.  Three errors:
- the Gram matrix: fp16 pairs leave 3 u32 of each product of two elements (2^-24 of each element, the dropped lo lo),
  and the fp32 sums of a piece of the long side take a rounding for each of its at most 2 (512 / 16) products of 16 and
  at most 16 inside each: 83 roundings, each at most u32 of (|G|^T |G|)_ij / |G|^2.  They are independent: an entry of
  dA has a variance of at most v_ij = 83 u32^2 (|G|^T |G|)_ij^2 / |G|^4.  T moves by V (D o V^T dA V) V^T, V the
  eigenvectors of A and D the divided differences of f on its eigenvalues (f' on the diagonal), to first order, so an
  element of X by a sum of variance ((G V)^2 (D^2 o (V^2)^T v V^2) (V^2)^T) / |G|^2, squares taken of each entry; 8 of its
  standard deviations are allowed.  (The worst case of all roundings at once is no use as a bound: it passes X itself.)
- T as pairs (2^-24 of an element), the table's too, the dropped lo lo, and S sums in fp32: (S + 6) u32 |G| |T| / |G|.
- the factor 1 / |G| and half a step of X's own type.
"""
import ctypes as C
import math

import pytest

import rsgpu

torch = pytest.importorskip("torch")

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24
COEF = (3.4445, -4.7750, 2.0315)


def reference(G, steps=5, coef=COEF, gram=1.0):
    """(X, bound): the steps in 64 bits, and what an element may be off before its own type's rounding (gram: how much of
    the Gram matrix's variance counts)."""
    G = G.double().cpu()
    norm = torch.linalg.vector_norm(G)
    if norm == 0:
        return torch.zeros_like(G), torch.zeros_like(G)
    a, b, c = coef
    flip = G.shape[0] < G.shape[1]
    Y = (G.T if flip else G) / norm
    Y0 = Y
    for _ in range(steps):
        A = Y.T @ Y
        Y = a * Y + Y @ (b * A + c * (A @ A))
    w, V = torch.linalg.eigh(Y0.T @ Y0)
    s = w.clamp(min=0).sqrt()
    amp = torch.ones_like(s)
    for _ in range(steps):
        p = a + b * s ** 2 + c * s ** 4
        amp, s = amp * p, s * p
    Tm = V @ torch.diag(amp) @ V.T
    # f'(w) by f = amp: d log amp, accumulated along the steps
    w0 = w.clamp(min=0)
    s, val, der = w0.clone(), torch.ones_like(w0), torch.zeros_like(w0)  # s^2, f and f' at w0
    ds = torch.ones_like(w0)
    for _ in range(steps):
        p, dp = a + b * s + c * s * s, (b + 2 * c * s) * ds
        val, der = val * p, der * p + val * dp
        s, ds = s * p * p, ds * p * p + s * 2 * p * dp
    gap = w0[:, None] - w0[None, :]
    near = gap.abs() < 1e-7 * w0.max().clamp(min=1e-300)
    D = torch.where(near, torch.maximum(der.abs()[:, None], der.abs()[None, :]), ((val[:, None] - val[None, :]) / torch.where(near, torch.ones_like(gap), gap)).abs())
    v = gram * 83 * U32 ** 2 * (Y0.abs().T @ Y0.abs()) ** 2
    V2 = V ** 2
    move = 8 * ((Y0 @ V) ** 2 @ (D ** 2 * (V2.T @ v @ V2)) @ V2.T).sqrt()
    S = Y0.shape[1]
    bound = (S + 6) * U32 * (Y0.abs() @ Tm.abs()) + move
    return (Y.T, bound.T) if flip else (Y, bound)


def check(X, G, steps=5, coef=COEF):
    ref, bound = reference(G, steps, coef)
    ut = torch.finfo(X.dtype).eps / 2
    tiny = torch.finfo(X.dtype).smallest_normal * torch.finfo(X.dtype).eps
    err = (X.double().cpu() - ref).abs()
    lim = bound * (1 + ut) + (ut + 2 * U32) * ref.abs() + tiny
    assert (err <= lim).all(), (float((err - lim).max()), float((err / lim.clamp(min=1e-300)).max()))


def update(rows, cols, ty, seed=0, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    r = min(4, rows, cols)
    G = torch.randn(rows, r, generator=g) @ torch.randn(r, cols, generator=g) + torch.randn(rows, cols, generator=g)
    G *= 0.2 + torch.rand(cols, generator=g)
    return (G * scale).to(T[ty]).cuda()


SHAPES = [(1, 1), (1, 7), (9, 1), (3, 3), (33, 20), (20, 33), (64, 64), (130, 65), (1682, 20), (100, 600), (700, 129), (257, 256),
          (300, 511), (2000, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_values(ctx, rows, cols, ty):
    G = update(rows, cols, ty, seed=rows + cols)
    keep = G.clone()
    check(ctx.orthogonalize(G), G)
    assert torch.equal(G, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 9])
def test_steps_and_coefficients(ctx, steps):
    G = update(200, 40, "f32", seed=steps)
    coef = (1.5, -0.5, 0.0)
    check(ctx.orthogonalize(G, steps=steps, coef=coef), G, steps, coef)
    if steps < 5:
        check(ctx.orthogonalize(G, steps=steps), G, steps)


@pytest.mark.gpu
def test_cubic_steps_end_in_an_orthogonal_matrix(ctx):
    """(1.5, -0.5, 0) converges: X^T X = 1 within the rounding of its fp32 entries (S u32 and the chain's own)."""
    G = update(500, 24, "f32", seed=3)
    X = ctx.orthogonalize(G, steps=16, coef=(1.5, -0.5, 0.0)).double()
    assert float((X.T @ X - torch.eye(24, device="cuda", dtype=torch.float64)).abs().max()) < 1e-4


@pytest.mark.gpu
def test_degenerate(ctx):
    Z = torch.zeros(50, 10, device="cuda")
    assert (ctx.orthogonalize(Z) == 0).all()
    one = torch.zeros(90, 30, device="cuda")
    one[17, 5] = -1e-20
    check(ctx.orthogonalize(one), one)
    same = torch.ones(60, 12, device="cuda") * 1e15  # rank one
    check(ctx.orthogonalize(same), same)
    G = update(80, 16, "f32", seed=5)
    G[3, 4] = math.nan
    assert torch.isnan(ctx.orthogonalize(G)).all()
    G[3, 4] = math.inf
    assert not torch.isfinite(ctx.orthogonalize(G)).any()


@pytest.mark.gpu
def test_spread_of_singular_values(ctx):
    """Directions 1000 times weaker than the strongest are amplified by up to a^5 = 485: inside the bound by T."""
    g = torch.Generator().manual_seed(6)
    U, _ = torch.linalg.qr(torch.randn(400, 50, generator=g, dtype=torch.float64))
    V, _ = torch.linalg.qr(torch.randn(50, 50, generator=g, dtype=torch.float64))
    G = (U @ torch.diag(torch.logspace(0, -3, 50, dtype=torch.float64)) @ V.T).float().cuda()
    check(ctx.orthogonalize(G), G)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(300, 70), (70, 300)])
def test_strided_in_place_and_beside(ctx, rows, cols):
    G = update(rows, cols, "f32", seed=8)
    want = ctx.orthogonalize(G)
    big = torch.full((rows, cols + 11), 3.0, device="cuda")
    big[:, 5:5 + cols] = G
    assert torch.equal(ctx.orthogonalize(big[:, 5:5 + cols]), want)
    ctx.orthogonalize(big[:, 5:5 + cols], out=big[:, 5:5 + cols])
    assert torch.equal(big[:, 5:5 + cols], want)
    big[:, 5:5 + cols] = 3.0
    assert (big == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 2), (10, 12), (33, 31), (40, 40), (64, 64), (100, 97), (129, 160), (260, 256),
                                       (512, 512), (300, 511), (2048, 512), (2048, 5), (20, 2047)])
def test_near_square_updates(ctx, rows, cols):
    """Small singular values: the Gram matrix of an fp32 update of up to 2048 long-side rows is exact but for fp64's
    roundings, so the errors are T's and the table's as pairs, S fp32 sums and the output's rounding, without what fp32 sums
    of the Gram matrix would move T by (fp64's 2^-53 times the largest divided difference, under 486 S: nothing)."""
    G = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows + cols)).cuda() * 1e-3
    ref, bound = reference(G, gram=0.0)
    err = (ctx.orthogonalize(G).double().cpu() - ref).abs()
    lim = bound * (1 + U32) + 3 * U32 * ref.abs()
    assert (err <= lim).all(), float((err / lim).max())


@pytest.mark.gpu
def test_rows_far_apart(ctx):
    """Rows of G and X further apart than 32 bits of elements."""
    step = 2 ** 31 + 8
    big = torch.empty(2 * step + 64, dtype=torch.float16, device="cuda")
    G, X = big.as_strided((3, 20), (step, 1)), big.as_strided((3, 20), (step, 1), 32)
    G.copy_(torch.randn(3, 20, generator=torch.Generator().manual_seed(1)))
    ctx.orthogonalize(G, out=X)
    assert torch.equal(X, ctx.orthogonalize(G.contiguous()))


@pytest.mark.gpu
def test_columns_beside_and_overlapping(ctx):
    big = torch.randn(60, 50, device="cuda")
    G = big[:, :20]
    want = ctx.orthogonalize(G)
    assert torch.equal(ctx.orthogonalize(G, out=big[:, 20:40]), want) and torch.equal(ctx.orthogonalize(G, out=big[:, 30:]), want)
    for bad in (big[:, 1:21], big[:, 19:39], big[1:, :20]):
        with pytest.raises(rsgpu.RsError):
            ctx.orthogonalize(G[:len(bad)], out=bad)
    assert torch.equal(ctx.orthogonalize(big[:30, :20], out=big[30:, :20]), ctx.orthogonalize(big[:30, :20]))


@pytest.mark.gpu
def test_transposed_update(ctx):
    """A tall update and its transpose are the same operator: equal up to the order of the sums."""
    G = update(500, 90, "f32", seed=9)
    check(ctx.orthogonalize(G), G)
    check(ctx.orthogonalize(G.T.contiguous()).T, G)


@pytest.mark.gpu
def test_side_stream_and_graph(ctx):
    G = update(900, 100, "f32", seed=10)
    ref = ctx.orthogonalize(G)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ctx.orthogonalize(G)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ctx.orthogonalize(G)
        both = ctx.orthogonalize(G, steps=2)
    for i in range(3):
        G[i] *= 3.0
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ctx.orthogonalize(G)) and torch.equal(both, ctx.orthogonalize(G, steps=2))


@pytest.mark.gpu
def test_tensor_refusals(ctx):
    G = update(30, 8, "f32")
    with pytest.raises(ValueError):
        ctx.orthogonalize(G.cpu())
    with pytest.raises(TypeError):
        ctx.orthogonalize(G.double())
    with pytest.raises(ValueError):
        ctx.orthogonalize(G[:, ::2])
    with pytest.raises(ValueError):
        ctx.orthogonalize(G, out=G[:20])
    with pytest.raises(ValueError):
        ctx.orthogonalize(G[:0])
    for kw in (dict(steps=0), dict(steps=17), dict(coef=(math.nan, 0, 0))):
        with pytest.raises(rsgpu.RsError):
            ctx.orthogonalize(G, **kw)
    with pytest.raises(rsgpu.RsError) as e:
        ctx.orthogonalize(torch.zeros(513, 513, device="cuda"))
    assert e.value.code == rsgpu.RS_ERR_UNSUPPORTED


def test_entry_point_refusals():
    L = rsgpu.lib()
    need = C.c_int64(-1)
    assert L.rs_orthogonalize_workspace(None, 100, 20, C.byref(need)) == rsgpu.RS_OK and need.value > 0
    assert L.rs_orthogonalize_workspace(None, 100, 20, None) == rsgpu.RS_ERR_INVALID
    assert L.rs_orthogonalize_workspace(None, -1, 20, C.byref(need)) == rsgpu.RS_ERR_INVALID
    assert L.rs_orthogonalize_workspace(None, 513, 513, C.byref(need)) == rsgpu.RS_ERR_UNSUPPORTED
    assert L.rs_orthogonalize_workspace(None, 0, 20, C.byref(need)) == rsgpu.RS_OK and need.value == 0
    buf = C.create_string_buffer(1 << 12)
    p = (C.addressof(buf) + 255) & ~255
    good = dict(ty=0, r=4, c=3, G=p, ldg=3, steps=5, a=1.5, b=-0.5, cc=0.0, X=p, ldx=3, ws=p, n=1 << 40)

    def call(**kw):
        a = dict(good, **kw)
        return L.rs_orthogonalize(None, a["ty"], a["r"], a["c"], a["G"], a["ldg"], a["steps"], a["a"], a["b"], a["cc"], a["X"], a["ldx"], a["ws"], a["n"], None)
    for kw in (dict(), dict(ty=5), dict(r=-1), dict(G=None), dict(G=p + 2), dict(ldg=2), dict(steps=0), dict(steps=17), dict(a=math.inf),
               dict(X=None), dict(ldx=2), dict(ldx=4), dict(ws=None), dict(ws=p + 8), dict(n=64)):
        assert call(**kw) == rsgpu.RS_ERR_INVALID, kw  # (the first: no context)
    assert call(r=600, c=600, ldg=600, ldx=600) == rsgpu.RS_ERR_UNSUPPORTED
    assert call(r=0) == rsgpu.RS_OK


LARGE = [("f32", 2049, 20), ("f32", 6041, 100), ("f32", 100, 6041), ("f32", 2500, 300), ("f32", 300, 2500), ("f32", 4099, 512), ("f32", 511, 4100)] + \
    [(ty, r, c) for ty in ("f32", "bf16", "f16") for r, c in ((40001, 64), (64, 40001), (26745, 128), (20001, 250), (250, 20001), (9001, 500))]


@pytest.mark.gpu
@pytest.mark.parametrize("ty,rows,cols", LARGE)
def test_large_tables(ctx, ty, rows, cols):
    """Past the fp64 Gram matrix (2048 long-side rows): up to 79 pieces of it, summed in groups, several tiles for each
    workgroup of the last pass.  A piece is at most 1024 rows dealt to 8 groups of waves, or 512 or fewer to one or two: the
    roundings of an entry stay within the 83 of the bound."""
    G = update(rows, cols, ty, seed=rows + cols)
    X = ctx.orthogonalize(G)
    check(X, G)
    if min(rows, cols) <= 256:  # in place, between columns that stay as they are
        big = torch.full((rows, cols + 9), 3.0, dtype=G.dtype, device="cuda")
        big[:, 4:4 + cols] = G
        ctx.orthogonalize(big[:, 4:4 + cols], out=big[:, 4:4 + cols])
        assert torch.equal(big[:, 4:4 + cols], X)
        assert (big[:, :4] == 3.0).all() and (big[:, 4 + cols:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(30001, 100), (100, 30001), (20001, 250), (1500, 60)])
@pytest.mark.parametrize("up", [True, False])
def test_rows_of_growing_size(ctx, ty, rows, cols, up):
    """The long side's elements grow (or shrink) by a factor of ten every eighth of it, over eight powers of ten: sums so far
    follow the scale as it moves.  An fp32 element is off by 2^-23 of itself or 2^-49 of |G|, a bf16 one by 2^-38 of |G|:
    small rows of X keep their own precision (bf16: what lies above that)."""
    G = update(rows, cols, "f32", seed=rows, scale=1.0).double().cpu()
    n = max(rows, cols)
    f = 10.0 ** (torch.arange(n, dtype=torch.float64) * 8 // n - 4)
    f = f if up else f.flip(0)
    G = (G * (f[:, None] if rows >= cols else f)).to(T[ty]).cuda()
    X = ctx.orthogonalize(G)
    ref, bound = reference(G)
    Gd = G.double().cpu()
    Tm = transform(Gd)
    floor = (2.0 ** -49 if ty == "f32" else 2.0 ** -38) * (Tm.abs().sum(0) if rows >= cols else Tm.abs().sum(0)[:, None])
    ut = torch.finfo(X.dtype).eps / 2
    err = (X.double().cpu() - ref).abs()
    lim = (bound + floor) * (1 + ut) + (ut + 2 * U32) * ref.abs()
    assert (err <= lim).all(), (float((err / lim).max()), int((err > lim).sum()))


def transform(G, steps=5, coef=COEF):
    """T of X = G T / |G| (T G / |G| where G is wide), in 64 bits."""
    G = G / torch.linalg.vector_norm(G)
    A = G.T @ G if G.shape[0] >= G.shape[1] else G @ G.T
    a, b, c = coef
    T_ = torch.eye(len(A), dtype=torch.float64)
    for _ in range(steps):
        M = a * torch.eye(len(A), dtype=torch.float64) + b * A + c * A @ A
        T_, A = T_ @ M, M @ A @ M
    return T_
