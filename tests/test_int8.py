"""Rows in 8 bits (rs_quantize_rows) and the int8 product with scales (rs_i8_matmul): refusals on the CPU, values
against integers and 64 bits on the GPU.

The sums are exact.  After them an output takes the rounding of the sum to fp32 (past 2^24), of the two scales'
product, of the product with it and one or two sums with biases: at most 3 u32 of the product and 2 u32 of the partial
sums (u32 = 2^-24), then half a step of its own type.
"""
import ctypes as C
import math

import numpy as np
import pytest

import rsgpu

torch = pytest.importorskip("torch")

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def quantize_reference(x):
    """The definition with the exact quotient: fractions of 64-bit integers."""
    x = x.float().cpu().numpy()
    amax = np.abs(x).max(axis=1)
    s = (amax * (np.float32(1) / np.float32(127))).astype(np.float32)
    q = np.zeros(x.shape, np.int64)
    ok = np.isfinite(amax) & (s > 0)
    # |x| against the ties (j + 1/2) s, exact in 64 bits
    ax = np.abs(x.astype(np.float64))
    for r in np.nonzero(ok)[0]:
        ties = (np.arange(128) + 0.5) * np.float64(s[r])
        above = np.searchsorted(ties, ax[r], side="left")  # ties strictly below |x|
        at = np.isin(ax[r], ties)
        above = above + (at & (above % 2 == 1))            # a tie goes to the even neighbour
        q[r] = np.minimum(above, 127) * np.where(x[r] < 0, -1, 1)
    s = np.where(np.isfinite(amax), s, np.float32(np.nan))
    return torch.from_numpy(q), torch.from_numpy(s)


def product_reference(A, sa, B, sb, rb=None, cb=None):
    acc = A.cpu().double() @ B.cpu().double().T
    out = acc * sa.cpu().double()[:, None] * sb.cpu().double()
    mag = out.abs()
    if rb is not None:
        out, mag = out + rb.cpu().double()[:, None], mag + rb.cpu().double().abs()[:, None]
    if cb is not None:
        out, mag = out + cb.cpu().double(), mag + torch.where(torch.isinf(cb), torch.zeros_like(cb), cb).cpu().double().abs()
    return out, mag


def check_product(out, ref, mag):
    ut = torch.finfo(out.dtype).eps / 2
    x = out.double().cpu()
    fin = torch.isfinite(ref)
    assert torch.equal(x[~fin], ref[~fin])
    tiny = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    lim = 5 * U32 * mag * (1 + ut) + ut * ref.abs() + tiny
    err = (x - ref).abs()
    assert (err[fin] <= lim[fin]).all(), float((err - lim)[fin].max())


def codes(m, k, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (m, k + pad), generator=g, dtype=torch.int8).cuda()[:, :k]


def scales(m, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(m, generator=g) * 0.02 + 1e-4).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 64), (70, 100), (37, 128), (35, 129), (19, 256), (33, 257), (9, 1025), (6, 2048), (7, 2049), (4, 4099), (3, 16390)])
def test_quantize(ctx, m, k, ty):
    g = torch.Generator().manual_seed(m * 100 + k)
    x = (torch.randn(m, k, generator=g) * torch.rand(m, 1, generator=g)).to(T[ty]).cuda()
    q, s = ctx.quantize_rows(x)
    rq, rs = quantize_reference(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu().long(), rq)


@pytest.mark.gpu
def test_quantize_ties_and_borders(ctx):
    """Values on ties and one step of fp32 beside them; the smallest and largest scales; zeros; rows that are not finite."""
    base = torch.cat([torch.arange(0, 127) + 0.5, torch.tensor([127.0])])
    rows = []
    for e in (0, -20, 30, -130, 120):
        r = base * 2.0 ** e
        rows += [r, -r, torch.nextafter(r, r * 2), torch.nextafter(r, r * 0)]
    x = torch.stack(rows).float()
    x[:, -1] = torch.where(x[:, -1].abs() > 0, x[:, -1], torch.ones(1))
    extra = torch.zeros(8, x.shape[1])
    extra[1, 5], extra[2, 6], extra[3, 7] = math.inf, math.nan, -math.inf
    extra[4, :3] = torch.tensor([1e-45, 3e-45, -1e-45])     # the scale underflows
    extra[5, :3] = torch.tensor([1e-43, -7e-44, 3e-44])     # a subnormal scale
    extra[6, 0] = torch.finfo(torch.float32).max
    extra[7, 0], extra[7, 1] = torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max
    x = torch.cat([x, extra]).cuda()
    q, s = ctx.quantize_rows(x)
    rq, rs = quantize_reference(x)
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(rs, nan=-1.0))
    assert torch.equal(q.cpu().long(), rq)


@pytest.mark.gpu
def test_quantize_many_rows_and_far_rows(ctx):
    """More rows than one axis of a launch holds waves for, and rows further apart than 32 bits of elements."""
    n = 2 ** 26 + 77
    x = (torch.arange(n, device="cuda") % 255 - 127).to(torch.float16)[:, None]
    q, s = ctx.quantize_rows(x)
    assert torch.equal(q, (x > 0).to(torch.int8) * 127 - (x < 0).to(torch.int8) * 127)
    assert torch.equal(s, x[:, 0].abs().float() * torch.tensor(1 / 127, dtype=torch.float32, device="cuda"))
    del x, q, s
    far = torch.empty(2 * (2 ** 31 + 16) + 40, dtype=torch.float16, device="cuda").as_strided((3, 40), (2 ** 31 + 16, 1))
    far.copy_(torch.randn(3, 40, generator=torch.Generator().manual_seed(1)))
    q, s = ctx.quantize_rows(far)
    rq, rs = quantize_reference(far)
    assert torch.equal(q.cpu().long(), rq) and torch.equal(s.cpu(), rs)


@pytest.mark.gpu
def test_product_of_far_rows(ctx):
    """Rows of A, B and C further apart than 32 bits of elements."""
    step = 2 ** 31 + 32
    big = torch.empty(2 * step + 64, dtype=torch.int8, device="cuda")
    A = big.as_strided((3, 40), (step, 1))
    A.copy_(codes(3, 40, 1))
    sa, sb = scales(3, 2), scales(70, 3)
    B = codes(70, 40, 4)
    near = ctx.i8_matmul(A.contiguous(), sa, B, sb)
    assert torch.equal(ctx.i8_matmul(A, sa, B, sb), near)
    assert torch.equal(ctx.i8_matmul(B, sb, A, sa), near.T)
    out = torch.empty(2 * step + 70, dtype=torch.float16, device="cuda").as_strided((3, 70), (step, 1))
    ctx.check(rsgpu.lib().rs_i8_matmul(ctx.h, 3, 70, 40, A.data_ptr(), step, sa.data_ptr(), B.data_ptr(), 40, sb.data_ptr(), None, None,
                                       rsgpu.dense.TYPE_F16, out.data_ptr(), step, rsgpu.dense.STREAM_DEFAULT))
    assert torch.equal(out, near.half())


@pytest.mark.gpu
def test_quantize_strided_leaves_the_rest(ctx):
    x = torch.randn(6, 40, device="cuda")
    q, s = ctx.quantize_rows(x[:, 1:30])
    q2, s2 = ctx.quantize_rows(x[:, 1:30].contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    L = rsgpu.lib()
    buf = torch.full((6, 40), 77, dtype=torch.int8, device="cuda")
    ctx.check(L.rs_quantize_rows(ctx.h, 0, 6, 29, x.data_ptr() + 4, 40, buf.data_ptr() + 3, 40, s2.data_ptr(), rsgpu.dense.STREAM_DEFAULT))
    assert torch.equal(buf[:, 3:32], q) and (buf[:, :3] == 77).all() and (buf[:, 32:] == 77).all()


SHAPES = [(1, 1, 1), (1, 3706, 100), (2, 17, 16), (16, 64, 64), (16, 1000, 250), (17, 33, 65), (5, 40, 4096), (5, 40, 4100),
          (33, 129, 128), (128, 128, 64), (129, 257, 300), (300, 70, 31), (200, 513, 1040), (64, 256, 128), (257, 640, 96), (20, 90, 1024), (50, 33, 900), (50, 33, 1100), (65, 20, 64),
          (3000, 4100, 72), (4097, 4096, 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ctx, m, n, k, out):
    A, B = codes(m, k, 1, pad=(-k) % 16), codes(n, k, 2, pad=(-k) % 16)
    sa, sb = scales(m, 3), scales(n, 4)
    rb, cb = torch.randn(m, device="cuda"), torch.randn(n, device="cuda")
    check_product(ctx.i8_matmul(A, sa, B, sb, rb, cb, T[out]), *product_reference(A, sa, B, sb, rb, cb))
    check_product(ctx.i8_matmul(A, sa, B, sb, out_dtype=T[out]), *product_reference(A, sa, B, sb))
    # rows at any address and stride: the same bits
    A1, B1 = codes(m, k + 3, 1)[:, 3:], codes(n, k + 5, 2)[:, 5:]
    A1.copy_(A), B1.copy_(B)
    assert torch.equal(ctx.i8_matmul(A1, sa, B1, sb, rb, cb, T[out]), ctx.i8_matmul(A, sa, B, sb, rb, cb, T[out]))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40])
def test_largest_sums(ctx, m):
    """k = 65536 of -128 and 127: the largest sums, exact."""
    k = 65536
    A = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    B = torch.stack([torch.full((k,), x, dtype=torch.int8) for x in (-128, 127, 1)]).cuda()
    one = torch.ones(m, device="cuda")
    out = ctx.i8_matmul(A, one, B, torch.ones(3, device="cuda"))
    ref = torch.tensor([2.0 ** 30, -128.0 * 127 * k, -128.0 * k]).cuda()
    assert torch.equal(out, ref.expand(m, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 70])
def test_masks_and_rows_that_are_not_finite(ctx, m):
    n, k = 100, 48
    X = torch.randn(m, k, device="cuda")
    X[1, 5] = math.nan
    A, sa = ctx.quantize_rows(X)
    B, sb = ctx.quantize_rows(torch.randn(n, k, device="cuda"))
    cb = torch.randn(n, device="cuda")
    cb[::3] = -math.inf
    out = ctx.i8_matmul(A, sa, B, sb, col_bias=cb)
    assert torch.isnan(out[1]).all()
    keep = [r for r in range(m) if r != 1]
    assert (out[keep][:, ::3] == -math.inf).all()
    ref, mag = product_reference(A, sa, B, sb, None, cb)
    check_product(out[keep], ref[keep], mag[keep])


@pytest.mark.gpu
def test_output_rows_beside_are_left(ctx):
    """C inside a larger buffer: nothing outside the m x n block is written."""
    L = rsgpu.lib()
    for m, n, k in ((1, 37, 20), (50, 131, 70)):
        A, B, sa, sb = codes(m, k, 5), codes(n, k, 6), scales(m, 7), scales(n, 8)
        want = ctx.i8_matmul(A, sa, B, sb)
        big = torch.full((m + 2, n + 9), 5.0, device="cuda")
        ctx.check(L.rs_i8_matmul(ctx.h, m, n, k, A.data_ptr(), k, sa.data_ptr(), B.data_ptr(), k, sb.data_ptr(), None, None, 0,
                                 big[1:, 4:].data_ptr(), n + 9, rsgpu.dense.STREAM_DEFAULT))
        assert torch.equal(big[1:m + 1, 4:n + 4], want)
        big[1:m + 1, 4:n + 4] = 5.0
        assert (big == 5.0).all()


@pytest.mark.gpu
def test_empty(ctx):
    A, B, sa, sb = codes(3, 8, 1), codes(4, 8, 2), scales(3, 3), scales(4, 4)
    assert ctx.i8_matmul(A[:0], sa[:0], B, sb).shape == (0, 4)
    assert ctx.i8_matmul(A, sa, B[:0], sb[:0]).shape == (3, 0)
    q, s = ctx.quantize_rows(torch.empty(0, 5, device="cuda"))
    assert q.shape == (0, 5) and s.shape == (0,)


@pytest.mark.gpu
def test_side_stream_and_graph(ctx):
    X, W = torch.randn(20, 72, device="cuda"), torch.randn(400, 72, device="cuda")
    B, sb = ctx.quantize_rows(W)

    def step(x):
        q, s = ctx.quantize_rows(x)
        return ctx.i8_matmul(q, s, B, sb, out_dtype=torch.bfloat16), ctx.i8_matmul(q[:1], s[:1], B, sb)
    ref = step(X)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step(X)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(out, ref))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(X)
    for i in range(3):
        X.mul_(1.5)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step(X)))


@pytest.mark.gpu
def test_tensor_refusals(ctx):
    A, B, sa, sb = codes(3, 8, 1), codes(4, 8, 2), scales(3, 3), scales(4, 4)
    with pytest.raises(TypeError):
        ctx.i8_matmul(A.float(), sa, B, sb)
    with pytest.raises(TypeError):
        ctx.i8_matmul(A, sa, B, sb, out_dtype=torch.int32)
    with pytest.raises(ValueError):
        ctx.i8_matmul(A, sa, B[:, :7], sb)
    with pytest.raises(ValueError):
        ctx.i8_matmul(A, sb, B, sb)
    with pytest.raises(ValueError):
        ctx.i8_matmul(A.cpu(), sa, B, sb)
    with pytest.raises(TypeError):
        ctx.quantize_rows(A)
    with pytest.raises(ValueError):
        ctx.quantize_rows(torch.empty(3, 0, device="cuda"))
    with pytest.raises(rsgpu.RsError) as e:
        ctx.i8_matmul(torch.zeros(1, 65537, dtype=torch.int8, device="cuda"), sa[:1], torch.zeros(1, 65537, dtype=torch.int8, device="cuda"), sb[:1])
    assert e.value.code == rsgpu.RS_ERR_UNSUPPORTED


def test_entry_point_refusals():
    L = rsgpu.lib()
    buf = C.create_string_buffer(1 << 12)
    p = (C.addressof(buf) + 255) & ~255
    good = dict(m=2, n=3, k=8, A=p, lda=8, sa=p, B=p, ldb=8, sb=p, rb=None, cb=None, ty=0, C=p, ldc=3)

    def call(**kw):
        a = dict(good, **kw)
        return L.rs_i8_matmul(None, a["m"], a["n"], a["k"], a["A"], a["lda"], a["sa"], a["B"], a["ldb"], a["sb"], a["rb"], a["cb"], a["ty"],
                              a["C"], a["ldc"], None)
    for kw in (dict(), dict(m=-1), dict(n=-1), dict(k=0), dict(A=None), dict(lda=7), dict(B=None), dict(ldb=7), dict(sa=None), dict(sb=p + 2),
               dict(rb=p + 1), dict(cb=p + 1), dict(ty=9), dict(C=None), dict(C=p + 2), dict(ldc=2), dict(m=2 ** 31)):
        assert call(**kw) == rsgpu.RS_ERR_INVALID, kw  # (the first: no context)
    assert call(k=65537, lda=65537, ldb=65537) == rsgpu.RS_ERR_UNSUPPORTED
    assert call(m=0) == rsgpu.RS_OK and call(n=0) == rsgpu.RS_OK
    quant = lambda ty=0, r=2, c=4, X=p, ldx=4, q=p, ldq=4, s=p: L.rs_quantize_rows(None, ty, r, c, X, ldx, q, ldq, s, None)
    for kw in (dict(), dict(ty=3), dict(r=-1), dict(c=0), dict(X=None), dict(X=p + 1), dict(ldx=3), dict(q=None), dict(ldq=3), dict(s=None)):
        assert quant(**kw) == rsgpu.RS_ERR_INVALID, kw
    assert quant(r=0) == rsgpu.RS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_quantize_subnormal_scales(ctx, ty):
    """max * (1/127) below 2^-126 is rounded to a multiple of 2^-149, by up to half of itself: the quotient of the largest
    value passes 127 (190 * 2^-149 has the scale 2^-149) and is held there."""
    units = torch.cat([torch.arange(1, 700), torch.arange(700, 16200, 37), torch.tensor([16064, 16065, 16128, 16129, 65536, 131072, 8388607, 8388608])])
    x = torch.zeros(2 * len(units), 5)
    x[:, 0] = torch.cat([units, units]).to(torch.int32).view(torch.float32)
    x[:, 1] = -x[:, 0]
    x[:, 2] = (torch.cat([units, units]) * 2 // 3).to(torch.int32).view(torch.float32)
    x[:, 3] = -1.0 * torch.ones(1, dtype=torch.int32).view(torch.float32)
    x[len(units):] *= -1
    x = x.to(T[ty]).cuda()
    q, s = ctx.quantize_rows(x)
    rq, rs = quantize_reference(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu().long(), rq)
    assert (q.cpu().long().abs() <= 127).all()
