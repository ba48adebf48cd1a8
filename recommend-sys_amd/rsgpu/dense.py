"""Dense operators over factor tables, on torch tensors in device memory (rs_softmax_ce, rs_quantize_rows,
rs_i8_matmul, rs_orthogonalize of include/rsgpu_dense.h).  They are methods of Context.

Each call enqueues its kernels on torch's current stream of the tensors' device and returns at once: nothing is
synchronised, and a call may be captured into a graph.  Outputs and workspaces are new torch tensors.  Tensors live
on the context's device, matrices have contiguous rows (any row stride).  The operators return gradients
themselves; they are not recorded by autograd.
"""
from __future__ import annotations

import ctypes as C

TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
DENSE_MAX_FACTORS = 512
STREAM_DEFAULT = 1  # RS_STREAM_DEFAULT: torch's default stream (0 would name the context's own)

_vp, _i32, _i64, _dbl = C.c_void_p, C.c_int32, C.c_int64, C.c_double

SIGNATURES = {
    "rs_softmax_ce_workspace": (C.c_int, [_vp, _i32, _i64, _i64, _i32, _i32, C.POINTER(_i64)]),
    "rs_softmax_ce": (C.c_int, [_vp, _i32, _i64, _i64, _i32, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp,
                                _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp]),
    "rs_quantize_rows": (C.c_int, [_vp, _i32, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _vp]),
    "rs_i8_matmul": (C.c_int, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _i32, _vp, _i64, _vp]),
    "rs_orthogonalize_workspace": (C.c_int, [_vp, _i64, _i64, C.POINTER(_i64)]),
    "rs_orthogonalize": (C.c_int, [_vp, _i32, _i64, _i64, _vp, _i64, _i32, _dbl, _dbl, _dbl, _vp, _i64, _vp, _i64, _vp]),
    "rs_svd_plan_rank_step": (C.c_int, [_vp, _i64, _vp, _vp, _dbl, _dbl, _dbl, C.POINTER(_dbl)]),
    "rs_svd_plan_score_items": (C.c_int, [_vp, _i64, _vp, _vp]),
}

# torch, the library and the element types, set by the first call (this module imports neither)
_torch = _lib = _types = None


def _load():
    global _torch, _lib, _types
    import torch

    from . import lib
    _types = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}
    _lib, _torch = lib(), torch


def _type(dtype, name):
    ty = _types.get(dtype)
    if ty is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, not {dtype}")
    return ty


class DenseOps:
    """The device-tensor operators of a Context."""

    def _mat(self, t, name, dtype=None):
        """Checks a 2-D device tensor; returns its row stride in elements."""
        if t.dim() != 2:
            raise ValueError(f"{name} must have two dimensions")
        self._place(t, name, dtype)
        rows, cols = t.shape
        ld, one = t.stride()
        if one != 1 and cols > 1:
            raise ValueError(f"{name} must have contiguous rows (stride 1 along the columns)")
        return ld if rows > 1 or ld > cols else (cols or 1)  # (one row: its stride says nothing)

    def _vec(self, t, name, n, dtype):
        """Checks a contiguous 1-D device tensor (None passes); returns its pointer."""
        if t is None:
            return None
        if t.dim() != 1 or t.shape[0] != n:
            raise ValueError(f"{name} must have {n} values, not {tuple(t.shape)}")
        self._place(t, name, dtype)
        if n > 1 and t.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr()

    def _place(self, t, name, dtype):
        if not t.is_cuda or t.get_device() != self.device:
            raise ValueError(f"{name} is on {t.device}, the context on cuda:{self.device}")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, not {t.dtype}")

    def _stream(self):
        return _torch._C._cuda_getCurrentRawStream(self.device) or STREAM_DEFAULT

    def softmax_ce(self, H, W, target, bias=None, weight=None, grad=False):
        """Softmax cross entropy of every row of H (n x k) against the catalogue W (items x k), the logits
        H W^T + bias never kept (rs_softmax_ce).  target: int32 item ids, -1 (or any id outside the catalogue):
        the row takes no part.  bias: fp32, -inf withdraws an item.  Returns (loss, lse) of every row, and with
        grad=True also (dH, dW, dbias), the gradient of sum(weight * loss) (weight None: ones)."""
        if _torch is None:
            _load()
        ty = _type(H.dtype, "H")
        ldh, ldw = self._mat(H, "H"), self._mat(W, "W", H.dtype)
        (n, k), items = H.shape, W.shape[0]
        if W.shape[1] != k:
            raise ValueError(f"H has {k} columns, W {W.shape[1]}")
        f32, empty, dev = _torch.float32, _torch.empty, H.device
        pt = self._vec(target, "target", n, _torch.int32)
        pb = self._vec(bias, "bias", items, f32)
        pw = self._vec(weight, "weight", n, f32)
        if n == 0 or items == 0:
            raise ValueError("softmax_ce needs at least one row and one item")
        need = _i64(0)
        self.check(_lib.rs_softmax_ce_workspace(self.h, ty, n, items, k, int(bool(grad)), C.byref(need)))
        ws = empty(need.value, dtype=_torch.uint8, device=dev)
        loss, lse = empty(n, dtype=f32, device=dev), empty(n, dtype=f32, device=dev)
        if not grad:
            self.check(_lib.rs_softmax_ce(self.h, ty, n, items, k, H.data_ptr(), ldh, W.data_ptr(), ldw, pb, pt, pw, loss.data_ptr(),
                                          lse.data_ptr(), None, k, None, k, None, ws.data_ptr(), need.value, self._stream()))
            return loss, lse
        dH, dW = empty((n, k), dtype=H.dtype, device=dev), empty((items, k), dtype=H.dtype, device=dev)
        db = empty(items, dtype=f32, device=dev)
        self.check(_lib.rs_softmax_ce(self.h, ty, n, items, k, H.data_ptr(), ldh, W.data_ptr(), ldw, pb, pt, pw, loss.data_ptr(),
                                      lse.data_ptr(), dH.data_ptr(), k, dW.data_ptr(), k, db.data_ptr(), ws.data_ptr(), need.value,
                                      self._stream()))
        return loss, lse, dH, dW, db

    def quantize_rows(self, X):
        """The rows of X in 8 bits with a scale each (rs_quantize_rows): (q int8, scale fp32), x ~ scale * q with
        scale = max |x| * (1/127) of the row.  q's rows are 16-byte multiples apart, as i8_matmul reads them fastest."""
        if _torch is None:
            _load()
        ty = _type(X.dtype, "X")
        ldx = self._mat(X, "X")
        m, k = X.shape
        if k == 0:
            raise ValueError("X has no columns")
        ldq = (k + 15) & ~15
        q = _torch.empty((m, ldq), dtype=_torch.int8, device=X.device)
        scale = _torch.empty(m, dtype=_torch.float32, device=X.device)
        self.check(_lib.rs_quantize_rows(self.h, ty, m, k, X.data_ptr(), ldx, q.data_ptr(), ldq, scale.data_ptr(), self._stream()))
        return (q if ldq == k else q[:, :k]), scale

    def i8_matmul(self, A, a_scale, B, b_scale, row_bias=None, col_bias=None, out_dtype=None):
        """C = (A B^T) * a_scale[:, None] * b_scale + row_bias[:, None] + col_bias for int8 A (m x k) and B (n x k)
        with a scale per row (rs_i8_matmul); C of out_dtype (float32 by default), m x n."""
        if _torch is None:
            _load()
        f32, i8 = _torch.float32, _torch.int8
        out_dtype = f32 if out_dtype is None else out_dtype
        ty = _type(out_dtype, "out_dtype")
        lda, ldb = self._mat(A, "A", i8), self._mat(B, "B", i8)
        (m, k), n = A.shape, B.shape[0]
        if B.shape[1] != k or k == 0:
            raise ValueError(f"A has {k} columns, B {B.shape[1]}")
        pa, pb = self._vec(a_scale, "a_scale", m, f32), self._vec(b_scale, "b_scale", n, f32)
        pr, pc = self._vec(row_bias, "row_bias", m, f32), self._vec(col_bias, "col_bias", n, f32)
        if pa is None or pb is None:
            raise ValueError("a_scale and b_scale are needed")
        out = _torch.empty((m, n), dtype=out_dtype, device=A.device)
        self.check(_lib.rs_i8_matmul(self.h, m, n, k, A.data_ptr(), lda, pa, B.data_ptr(), ldb, pb, pr, pc, ty, out.data_ptr(), n or 1,
                                     self._stream()))
        return out

    def orthogonalize(self, G, steps=5, coef=(3.4445, -4.7750, 2.0315), out=None):
        """The orthogonalised form of the update G of a factor table by Newton-Schulz products (rs_orthogonalize): G / |G|
        with every singular value s taken `steps` times through a s + b s^3 + c s^5.  out: where to write it (it may be
        G itself where the shorter side is at most 256)."""
        if _torch is None:
            _load()
        ty = _type(G.dtype, "G")
        ldg = self._mat(G, "G")
        rows, cols = G.shape
        if rows == 0 or cols == 0:
            raise ValueError("G is empty")
        if out is None:
            out = _torch.empty((rows, cols), dtype=G.dtype, device=G.device)
            ldx = cols
        else:
            ldx = self._mat(out, "out", G.dtype)
            if out.shape != G.shape:
                raise ValueError(f"out must be {tuple(G.shape)}, not {tuple(out.shape)}")
        a, b, c = coef
        need = _i64(0)
        self.check(_lib.rs_orthogonalize_workspace(self.h, rows, cols, C.byref(need)))
        ws = _torch.empty(need.value, dtype=_torch.uint8, device=G.device)
        self.check(_lib.rs_orthogonalize(self.h, ty, rows, cols, G.data_ptr(), ldg, int(steps), a, b, c, out.data_ptr(), ldx, ws.data_ptr(),
                                         need.value, self._stream()))
        return out
