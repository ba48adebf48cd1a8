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
}


def _types():
    import torch
    return {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}


def _type(t, name):
    ty = _types().get(t.dtype)
    if ty is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return ty


class DenseOps:
    """The device-tensor operators of a Context."""

    def _mat(self, t, name, shape=None, dtype=None):
        """Checks a 2-D device tensor; returns its row stride in elements."""
        if t.dim() != 2:
            raise ValueError(f"{name} must have two dimensions")
        self._on_device(t, name, dtype)
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{name} must have contiguous rows (stride 1 along the columns)")
        return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)

    def _vec(self, t, name, n, dtype):
        """Checks a contiguous 1-D device tensor (None passes); returns its pointer."""
        if t is None:
            return None
        if t.dim() != 1 or t.shape[0] != n:
            raise ValueError(f"{name} must have {n} values, not {tuple(t.shape)}")
        self._on_device(t, name, dtype)
        if n > 1 and t.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr()

    def _on_device(self, t, name, dtype):
        if t.device.type != "cuda" or t.device.index != self.device:
            raise ValueError(f"{name} is on {t.device}, the context on cuda:{self.device}")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, not {t.dtype}")

    def _dense(self, name, *args):
        from . import lib
        self.check(getattr(lib(), name)(self.h, *args))

    def _stream(self, t):
        import torch
        return torch.cuda.current_stream(t.device).cuda_stream or STREAM_DEFAULT

    def softmax_ce(self, H, W, target, bias=None, weight=None, grad=False):
        """Softmax cross entropy of every row of H (n x k) against the catalogue W (items x k), the logits
        H W^T + bias never kept (rs_softmax_ce).  target: int32 item ids, -1 (or any id outside the catalogue):
        the row takes no part.  bias: fp32, -inf withdraws an item.  Returns (loss, lse) of every row, and with
        grad=True also (dH, dW, dbias), the gradient of sum(weight * loss) (weight None: ones)."""
        import torch
        ty = _type(H, "H")
        ldh, ldw = self._mat(H, "H"), self._mat(W, "W", dtype=H.dtype)
        (n, k), items = H.shape, W.shape[0]
        if W.shape[1] != k:
            raise ValueError(f"H has {k} columns, W {W.shape[1]}")
        pt = self._vec(target, "target", n, torch.int32)
        pb = self._vec(bias, "bias", items, torch.float32)
        pw = self._vec(weight, "weight", n, torch.float32)
        if n == 0 or items == 0:
            raise ValueError("softmax_ce needs at least one row and one item")
        need = _i64(0)
        self._dense("rs_softmax_ce_workspace", ty, n, items, k, int(bool(grad)), C.byref(need))
        dev = H.device
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        loss, lse = (torch.empty(n, dtype=torch.float32, device=dev) for _ in range(2))
        dH = dW = db = None
        if grad:
            dH = torch.empty(n, k, dtype=H.dtype, device=dev)
            dW = torch.empty(items, k, dtype=H.dtype, device=dev)
            db = torch.empty(items, dtype=torch.float32, device=dev)
        ptr = lambda t: None if t is None else t.data_ptr()
        self._dense("rs_softmax_ce", ty, n, items, k, H.data_ptr(), ldh, W.data_ptr(), ldw, pb, pt, pw, loss.data_ptr(),
                    lse.data_ptr(), ptr(dH), k, ptr(dW), k, ptr(db), ws.data_ptr(), need.value, self._stream(H))
        return (loss, lse, dH, dW, db) if grad else (loss, lse)

    def quantize_rows(self, X):
        """The rows of X in 8 bits with a scale each (rs_quantize_rows): (q int8, scale fp32), x ~ scale * q with
        scale = max |x| * (1/127) of the row.  q's rows are 16-byte multiples apart, as i8_matmul reads them fastest."""
        import torch
        ty = _type(X, "X")
        ldx = self._mat(X, "X")
        m, k = X.shape
        if k == 0:
            raise ValueError("X has no columns")
        q = torch.empty(m, (k + 15) // 16 * 16, dtype=torch.int8, device=X.device)[:, :k]
        scale = torch.empty(m, dtype=torch.float32, device=X.device)
        self._dense("rs_quantize_rows", ty, m, k, X.data_ptr(), ldx, q.data_ptr(), (k + 15) // 16 * 16, scale.data_ptr(), self._stream(X))
        return q, scale

    def i8_matmul(self, A, a_scale, B, b_scale, row_bias=None, col_bias=None, out_dtype=None):
        """C = (A B^T) * a_scale[:, None] * b_scale + row_bias[:, None] + col_bias for int8 A (m x k) and B (n x k)
        with a scale per row (rs_i8_matmul); C of out_dtype (float32 by default), m x n."""
        import torch
        out_dtype = torch.float32 if out_dtype is None else out_dtype
        ty = _types().get(out_dtype)
        if ty is None:
            raise TypeError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
        lda, ldb = self._mat(A, "A", dtype=torch.int8), self._mat(B, "B", dtype=torch.int8)
        (m, k), n = A.shape, B.shape[0]
        if B.shape[1] != k or k == 0:
            raise ValueError(f"A has {k} columns, B {B.shape[1]}")
        pa, pb = self._vec(a_scale, "a_scale", m, torch.float32), self._vec(b_scale, "b_scale", n, torch.float32)
        pr, pc = self._vec(row_bias, "row_bias", m, torch.float32), self._vec(col_bias, "col_bias", n, torch.float32)
        out = torch.empty(m, n, dtype=out_dtype, device=A.device)
        self._dense("rs_i8_matmul", m, n, k, A.data_ptr(), lda, pa, B.data_ptr(), ldb, pb, pr, pc, ty, out.data_ptr(), max(n, 1),
                    self._stream(A))
        return out

    def orthogonalize(self, G, steps=5, coef=(3.4445, -4.7750, 2.0315), out=None):
        """The orthogonalised form of the update G of a factor table by Newton-Schulz products (rs_orthogonalize): G / |G|
        with every singular value s taken `steps` times through a s + b s^3 + c s^5.  out: where to write it (it may be
        G itself)."""
        import torch
        ty = _type(G, "G")
        ldg = self._mat(G, "G")
        rows, cols = G.shape
        if rows == 0 or cols == 0:
            raise ValueError("G is empty")
        X = torch.empty(rows, cols, dtype=G.dtype, device=G.device) if out is None else out
        ldx = self._mat(X, "out", shape=G.shape, dtype=G.dtype)
        a, b, c = (float(v) for v in coef)
        need = _i64(0)
        self._dense("rs_orthogonalize_workspace", rows, cols, C.byref(need))
        ws = torch.empty(need.value, dtype=torch.uint8, device=G.device)
        self._dense("rs_orthogonalize", ty, rows, cols, G.data_ptr(), ldg, int(steps), a, b, c, X.data_ptr(), ldx, ws.data_ptr(), need.value,
                    self._stream(G))
        return X
