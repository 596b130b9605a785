"""Operator-level entry points over the C ABI, taking torch CUDA tensors.

These mirror the reference's three custom ops (cuda/wrapper.cpp:45-129, called from
modules/matmul.py:42-49, :70-80 and modules/wkv.py:18): a one- or three-matrix uint8
GEMV and the WKV recurrence.  They validate, pass raw device pointers to the library and
launch on torch's current stream.  No CPU path.
"""
from __future__ import annotations

import ctypes as C
import struct
from contextlib import nullcontext
from functools import lru_cache
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .quant import QuantMatrix


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The operators below are called once per projection or step with a few rows, where the host's share of a call counts: a
# raw stream handle instead of a stream object, and no change of device where it is the current one already.
def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


_HERE = nullcontext()


def _on(index: int):
    return _HERE if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def _cmatrix(m: QuantMatrix) -> _lib.Matrix:
    return _lib.Matrix(_lib.ptr(m.qt), _lib.ptr(m.ry), _lib.ptr(m.my), _lib.ptr(m.rx), _lib.ptr(m.mx),
                       float(m.half), m.n_out, m.k_in)


_workspaces = {}


def gemv_workspace(device, k_in: int, nmat: int) -> torch.Tensor:
    """Zeroed scratch for ``gemv_u8``, cached per device, size AND current CUDA stream: calls that share
    a workspace must be ordered on one stream, so every stream gets its own.  Its first int32 is the
    kernels' status word."""
    n = int(_lib.lib().b200rwkv_gemv_workspace_bytes(k_in, nmat))
    key = (str(device), n, _stream(device))
    if key not in _workspaces:
        _workspaces[key] = torch.zeros(n, dtype=torch.uint8, device=device)
    return _workspaces[key]


def gemv_u8(mats: Sequence[QuantMatrix], xs: Sequence[torch.Tensor], ys: Optional[Sequence[torch.Tensor]] = None,
            accumulate: bool = False, workspace: Optional[torch.Tensor] = None,
            trace: Optional[torch.Tensor] = None) -> List[torch.Tensor]:
    """``ys[i] = xs[i] @ W_i`` for 1..3 quantised matrices of equal k_in, one launch.

    ``xs[i]`` fp32 ``[k_in]`` on the matrices' CUDA device; ``ys[i]`` fp32 ``[n_out_i]``
    (allocated when omitted; with ``accumulate`` the result is added onto them, which is
    what the reference ops do with their zero-filled ``y``).  ``trace``: optional int64
    ``[1024, 8]`` CUDA tensor that receives the per-CTA phase timeline (profiling).
    ``workspace``: scratch from ``gemv_workspace`` (a cached one is used when omitted)."""
    n = len(mats)
    if n < 1 or n > 3 or len(xs) != n:
        raise ValueError("gemv_u8 takes 1..3 matrices and as many input vectors")
    dev = mats[0].qt.device
    if dev.type != "cuda":
        raise RuntimeError("gemv_u8 needs CUDA tensors (no CPU path)")
    if ys is None:
        if accumulate:
            raise ValueError("accumulate needs caller-provided outputs")
        ys = [torch.empty(m.n_out, dtype=torch.float32, device=dev) for m in mats]
    for m, x, y in zip(mats, xs, ys):
        if x.dtype != torch.float32 or y.dtype != torch.float32 or not x.is_contiguous() or not y.is_contiguous():
            raise ValueError("gemv_u8 needs contiguous fp32 vectors")
        if x.numel() != m.k_in or y.numel() != m.n_out or x.device != dev or y.device != dev:
            raise ValueError("gemv_u8 vector shape/device does not match its matrix")
    cm = (_lib.Matrix * n)(*[_cmatrix(m) for m in mats])
    cx = (C.c_void_p * n)(*[x.data_ptr() for x in xs])
    cy = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
    if workspace is None:
        workspace = gemv_workspace(dev, mats[0].k_in, n)
    with torch.cuda.device(dev):
        if trace is None:
            _lib.check(_lib.lib().b200rwkv_gemv_u8(n, cm, cx, cy, int(accumulate), workspace.data_ptr(),
                                                   workspace.numel(), _stream(dev)))
        else:
            _lib.check(_lib.lib().b200rwkv_gemv_u8_traced(n, cm, cx, cy, int(accumulate), workspace.data_ptr(),
                                                          workspace.numel(), trace.data_ptr(), _stream(dev)))
    return list(ys)


def gemm_u8(mats: Sequence[QuantMatrix], xs: Sequence[torch.Tensor],
            ys: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
    """``ys[i] = xs[i] @ W_i`` for 1..3 quantised matrices of equal k_in and ``xs[i]`` fp32
    ``[rows, k_in]``: the many-rows (tensor-core) form of ``gemv_u8``, which the reference serves by
    dequantising the matrix (modules/matmul.py:64-68).  Returns fp32 ``[rows, n_out_i]``."""
    n = len(mats)
    if n < 1 or n > 3 or len(xs) != n:
        raise ValueError("gemm_u8 takes 1..3 matrices and as many input matrices")
    dev = mats[0].qt.device
    if dev.type != "cuda":
        raise RuntimeError("gemm_u8 needs CUDA tensors (no CPU path)")
    rows = xs[0].shape[0]
    if ys is None:
        ys = [torch.empty(rows, m.n_out, dtype=torch.float32, device=dev) for m in mats]
    for m, x, y in zip(mats, xs, ys):
        if x.dtype != torch.float32 or y.dtype != torch.float32 or not x.is_contiguous() or not y.is_contiguous():
            raise ValueError("gemm_u8 needs contiguous fp32 matrices")
        if tuple(x.shape) != (rows, m.k_in) or tuple(y.shape) != (rows, m.n_out) or x.device != dev or y.device != dev:
            raise ValueError("gemm_u8 operand shape/device does not match its matrix")
    cm = (_lib.Matrix * n)(*[_cmatrix(m) for m in mats])
    cx = (C.c_void_p * n)(*[x.data_ptr() for x in xs])
    cy = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
    nbytes = int(_lib.lib().b200rwkv_gemm_workspace_bytes(mats[0].k_in, n, rows))
    key = (str(dev), "gemm", nbytes)
    if key not in _workspaces:
        _workspaces[key] = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
    ws = _workspaces[key]
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().b200rwkv_gemm_u8(n, cm, cx, cy, rows, ws.data_ptr(), ws.numel(), _stream(dev)))
    status = int(ws[:4].view(torch.int32).item())
    if status:
        ws[:4].zero_()
        raise _lib.B200RWKVError(_lib.ETIMEOUT, f"gemm_u8: a bounded device-side wait expired (status bits {status})")
    return list(ys)


def wkv_scan(w: torch.Tensor, u: torch.Tensor, k: torch.Tensor, v: torch.Tensor, aa: torch.Tensor,
             bb: torch.Tensor, pp: torch.Tensor, convention: int = 0) -> torch.Tensor:
    """WKV-4 over ``k, v [B,T,C]`` (or ``[T,C]``); ``aa, bb, pp [B,C]`` (or ``[C]``) updated in
    place.  ``convention`` 0 = max-trick state, 1 = the reference FASTQUANT state."""
    if k.dim() == 2:
        k, v = k.unsqueeze(0), v.unsqueeze(0)
    B, T, Cc = k.shape
    for t in (w, u, k, v, aa, bb, pp):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.device.type != "cuda":
            raise ValueError("wkv_scan needs contiguous fp32 CUDA tensors")
    if aa.numel() != B * Cc or bb.numel() != B * Cc or pp.numel() != B * Cc or w.numel() != Cc or u.numel() != Cc:
        raise ValueError("wkv_scan state/parameter shapes do not match k")
    y = torch.empty_like(k)
    with torch.cuda.device(k.device):
        _lib.check(_lib.lib().b200rwkv_wkv_scan(B, T, Cc, w.data_ptr(), u.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                y.data_ptr(), aa.data_ptr(), bb.data_ptr(), pp.data_ptr(),
                                                convention, _stream(k.device)))
    return y


def sample_typical(logits: torch.Tensor, temp: float = 1.0, tau: float = 0.95, u: Optional[torch.Tensor] = None,
                   generator: Optional[torch.Generator] = None, return_probs: bool = False):
    """Typical sampling of one token per row of ``logits [rows,V]`` (or ``[V]``) on the device:
    the arithmetic of the reference's ``typical(logits, temp, tau)`` (samplers/typical.py:1-17)
    with the draw made by inverse CDF from ``u`` (device f32 [rows] uniform in [0,1); drawn from
    ``generator`` when absent).  Returns device int64 [rows], and with ``return_probs`` also the
    masked, tempered, unnormalised probabilities [rows,V] the draw was made from."""
    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    if x.dtype != torch.float32 or x.device.type != "cuda" or x.stride(1) != 1:
        raise ValueError("sample_typical needs fp32 CUDA logits with contiguous rows")
    rows, n = x.shape
    if u is None:
        u = torch.rand(rows, device=x.device, dtype=torch.float32, generator=generator)
    if u.dtype != torch.float32 or u.device != x.device or u.numel() != rows or not u.is_contiguous():
        raise ValueError("u must be a contiguous fp32 tensor of one number per row on the logits' device")
    out = torch.empty(rows, dtype=torch.int64, device=x.device)
    probs = torch.empty(rows, n, dtype=torch.float32, device=x.device) if return_probs else None
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().b200rwkv_sample_typical(x.data_ptr(), rows, n, x.stride(0), float(temp), float(tau),
                                                      u.data_ptr(), out.data_ptr(),
                                                      probs.data_ptr() if return_probs else None, None, None, 0,
                                                      _stream(x.device)))
    return (out, probs) if return_probs else out


def argmax_rows(logits: torch.Tensor) -> torch.Tensor:
    """Index of the largest value of every row of ``logits [rows,V]`` (fp32, CUDA, contiguous rows), on the
    device: int64 [rows]; ties go to the lowest index like ``torch.argmax`` on a CPU tensor."""
    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    if x.dtype != torch.float32 or x.device.type != "cuda" or x.stride(1) != 1:
        raise ValueError("argmax_rows needs fp32 CUDA logits with contiguous rows")
    rows, n = x.shape
    out = torch.empty(rows, dtype=torch.int64, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().b200rwkv_argmax(x.data_ptr(), rows, n, x.stride(0), out.data_ptr(), None, None, 0, _stream(x.device)))
    return out


_DENSE_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def gemv_dense(w: torch.Tensor, x: torch.Tensor, y: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Unquantised matrix-vector product ``y[o] = sum_j x[j] * w[o,j]`` for ``w [out,in]`` of bf16,
    fp16 or fp32 with contiguous rows (a row stride >= in is allowed) and fp32 ``x [in]``:
    x is rounded to the weights' type, products are summed in fp32, the result is rounded to the
    weights' type and returned as fp32 - what the reference's TORCH-mode ``matvec`` computes
    (agnostic/backends/torch.py:162-164)."""
    if w.dim() != 2 or w.dtype not in _DENSE_DTYPES or w.device.type != "cuda" or w.stride(1) != 1:
        raise ValueError("gemv_dense needs a CUDA [out,in] matrix of bf16/fp16/fp32 with contiguous rows")
    n_out, k_in = w.shape
    if x.dtype != torch.float32 or x.device != w.device or x.numel() != k_in or not x.is_contiguous():
        raise ValueError(f"x must be a contiguous fp32 vector of {k_in} values on the weights' device")
    if y is None:
        y = torch.empty(n_out, dtype=torch.float32, device=w.device)
    elif y.dtype != torch.float32 or y.device != w.device or y.numel() != n_out or not y.is_contiguous():
        raise ValueError(f"y must be a contiguous fp32 vector of {n_out} values on the weights' device")
    with torch.cuda.device(w.device):
        _lib.check(_lib.lib().b200rwkv_gemv_dense(w.data_ptr(), _DENSE_DTYPES[w.dtype], k_in, n_out, w.stride(0),
                                                  x.data_ptr(), y.data_ptr(), _stream(w.device)))
    return y


def pack_adapters(adapters: Sequence[Tuple[torch.Tensor, torch.Tensor, float]], dtype: Optional[torch.dtype] = None,
                  device=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A bank for ``adapt_rows`` from one projection's adapters ``(a [r,in], b [out,r], scale)``, whose ranks r may differ:
    ``(a [n,rank,in], b [n,out,rank], scale f32 [n])`` with rank the largest one, rounded up to a multiple of 4; the
    ranks that an adapter lacks are zeros.  Laid out once, when adapters are loaded."""
    if not adapters:
        raise ValueError("pack_adapters needs at least one adapter")
    a0, b0, _ = adapters[0]
    dtype, device = dtype or a0.dtype, device or a0.device
    for a, b, _ in adapters:
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[1] != a0.shape[1] or b.shape[0] != b0.shape[0]:
            raise ValueError("pack_adapters takes a [r,in] and b [out,r] of one projection")
    rank = max(4, -(-max(a.shape[0] for a, _, _ in adapters) // 4) * 4)
    pa = torch.zeros(len(adapters), rank, a0.shape[1], dtype=dtype, device=device)
    pb = torch.zeros(len(adapters), b0.shape[0], rank, dtype=dtype, device=device)
    for i, (a, b, _) in enumerate(adapters):
        pa[i, :a.shape[0]] = a.to(device=device, dtype=dtype)
        pb[i, :, :b.shape[1]] = b.to(device=device, dtype=dtype)
    return pa, pb, torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=device)


def adapt_rows(banks: Sequence[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]], xs: Sequence[torch.Tensor], ids: torch.Tensor,
               ys: Sequence[torch.Tensor], outs: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
    """Low-rank adapters of many requests beside 1..3 shared projections of equal k_in (``gemm_u8``'s or
    others'): ``outs[i][r] = ys[i][r] + scale_i[id] * (xs[i][r] @ A_i[id].T) @ B_i[id].T`` with the adapter
    ``id = ids[r // T]`` of the row's stream, T = rows // len(ids); an id outside ``[0, n)`` (say -1) means none.

    ``banks[i] = (a [n,rank,k_in], b [n,n_out_i,rank], scale f32 [n] or None)`` of bf16, fp16 or fp32 (see
    ``pack_adapters``), ``xs[i] [rows,k_in]`` and ``ys[i] [rows,n_out_i]`` of fp32 or the banks' type, ``ids`` int64
    ``[streams]``; all contiguous on one CUDA device.  Rank a multiple of 4 up to 256, k_in of 8 up to 2^30, up to 65535
    rows.  In place on ``ys`` when ``outs`` is omitted; an output may be its own y and overlaps nothing else.  ``h = x A^T``
    is fp32 whatever the types, products leave out less than 2^-21 of themselves, and the result is rounded once.  A row of
    x that holds an infinity or a NaN comes out as NaN where it has an adapter; rows without one are left as they are.
    Should a bounded device-side wait of the forms for many rows expire, its rows come out as NaN and ``check_status`` raises."""
    n = len(banks)
    outs = ys if outs is None else outs
    if n < 1 or n > 3 or len(xs) != n or len(ys) != n or len(outs) != n:
        raise ValueError("adapt_rows takes 1..3 banks and as many inputs and outputs")
    a0, x0 = banks[0][0], xs[0]
    index, dt, row_dt = a0.get_device(), a0.dtype, x0.dtype
    if index < 0:
        raise RuntimeError("adapt_rows needs CUDA tensors (no CPU path)")
    if dt not in _DENSE_DTYPES or (row_dt != torch.float32 and row_dt != dt):
        raise ValueError("adapt_rows needs banks of bf16, fp16 or fp32 and rows of fp32 or the banks' type")
    bank_shape, x_shape = a0.shape, x0.shape
    if len(bank_shape) != 3 or len(x_shape) != 2 or ids.dim() != 1:
        raise ValueError("adapt_rows needs a [n,rank,k_in], x [rows,k_in] and ids [streams]")
    count, rank, k_in = bank_shape
    rows, streams = x_shape[0], ids.shape[0]
    if ids.dtype != torch.int64 or ids.get_device() != index or not ids.is_contiguous() or (rows % streams if streams else rows):
        raise ValueError("ids must be contiguous int64 on the banks' device, one per stream, and the rows a multiple of them")
    if (count | k_in | rows) >> 31:
        raise ValueError("adapt_rows takes sizes of 32 bits")
    packed, px, py, po, n_out = [], [], [], [], []
    x_want = (rows, k_in)
    for (a, b, s), x, y, o in zip(banks, xs, ys, outs):
        b_shape = b.shape
        if a.shape != bank_shape or len(b_shape) != 3 or b_shape[0] != count or b_shape[2] != rank:
            raise ValueError("adapt_rows banks must share n, rank and k_in: a [n,rank,k_in], b [n,n_out,rank]")
        if (a.dtype != dt or b.dtype != dt or not a.is_contiguous() or not b.is_contiguous() or a.get_device() != index
                or b.get_device() != index):
            raise ValueError("adapt_rows banks must be contiguous, of one type, on one device")
        if s is not None and (s.dtype != torch.float32 or s.get_device() != index or s.shape != (count,) or not s.is_contiguous()):
            raise ValueError("an adapter bank's scale must be contiguous fp32 [n] on its device")
        n_o = b_shape[1]
        if n_o >> 31:
            raise ValueError("adapt_rows takes sizes of 32 bits")
        y_want = (rows, n_o)
        if (x.shape != x_want or y.shape != y_want or x.dtype != row_dt or y.dtype != row_dt or x.get_device() != index
                or y.get_device() != index or not x.is_contiguous() or not y.is_contiguous()):
            raise ValueError("adapt_rows rows must be contiguous, of one type, on the banks' device, and match their bank")
        if o is not y and (o.shape != y_want or o.dtype != row_dt or o.get_device() != index or not o.is_contiguous()):
            raise ValueError("adapt_rows outputs must be contiguous, of the rows' type and shape, on the banks' device")
        packed += (a.data_ptr(), b.data_ptr(), 0 if s is None else s.data_ptr(), n_o)
        px.append(x.data_ptr())
        py.append(y.data_ptr())
        po.append(o.data_ptr())
        n_out.append(n_o)
    if rows == 0:
        return list(outs)
    # the C side's arrays as one buffer: n b200rwkv_adapters (three pointers, an int32 and its padding), three times n pointers
    arrays = C.create_string_buffer(_ADAPT_PACK[n].pack(*packed, *px, *py, *po), 56 * n)
    at = C.addressof(arrays)
    code = _DENSE_DTYPES[dt]
    tokens = rows // streams
    nbytes = _adapt_workspace(tuple(n_out), count, rank, k_in, code, streams, tokens)
    with _on(index):
        ws = ids.new_empty(nbytes // 8)
        _lib.check(_lib.lib().b200rwkv_adapt_rows(n, at, count, rank, k_in, code, at + 32 * n, at + 40 * n, at + 48 * n, _DENSE_DTYPES[row_dt],
                                                  ids.data_ptr(), streams, tokens, ws.data_ptr(), nbytes, _raw_stream(index)))
    return list(outs)


def check_status(device=None) -> None:
    """Raise if a device-side wait of an ``adapt_rows`` call that has ended on ``device`` (the current one when omitted)
    expired since the last check.  Waits for the device's current stream."""
    with torch.cuda.device(device):
        _lib.check(_lib.lib().b200rwkv_adapt_rows_status(_stream(device)))


_ADAPT_PACK = {n: struct.Struct("=" + "QQQi4x" * n + "%dQ" % (3 * n)) for n in (1, 2, 3)}


@lru_cache(maxsize=1024)
def _adapt_workspace(n_out: Tuple[int, ...], count: int, rank: int, k_in: int, dtype: int, streams: int, tokens: int) -> int:
    """Bytes of scratch for a call of this shape; a refused shape gets a few, for the call to say why."""
    banks = (_lib.Adapters * len(n_out))(*[_lib.Adapters(None, None, None, o) for o in n_out])
    return max(256, int(_lib.lib().b200rwkv_adapt_rows_workspace_bytes(len(n_out), banks, count, rank, k_in, dtype, streams, tokens)))


def verify_drafts(target: torch.Tensor, draft: Optional[torch.Tensor], tokens: torch.Tensor, u: torch.Tensor,
                  lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Accept or replace drafted tokens so that what comes out is distributed as the target's own draws.

    ``target`` fp32 ``[B,K+1,V]``: the target's weights behind each of the K drafted tokens and in front of the first
    (``sample_typical``'s ``return_probs``: they need not sum to one; what is not above zero counts as zero).  ``draft``
    fp32 ``[B,K,V]``: the weights that ``tokens`` int64 ``[B,K]`` were drawn from, or None where the draft is sure of
    them.  ``u`` fp32 ``[B,K+1]`` uniform in [0,1): one number per drafted token and one for the draw.  ``lengths`` int64
    ``[B]``: how many of the K tokens a stream has (all, when omitted).  Token t is accepted where
    ``u_t q_t/Q_t < p_t/P_t``; the first refused one is replaced by a draw from ``max(0, p/P - q/Q)``, and where none is,
    one more is drawn from the target's next row.  Returns int64 ``[B,K+1]`` (the accepted tokens, the drawn one, -1
    behind it) and the number accepted, int64 ``[B]``.  Rows must be contiguous; streams and rows may be strided."""
    index = target.get_device()
    if target.dim() != 3 or tokens.dim() != 2 or target.dtype != torch.float32 or index < 0:
        raise ValueError("verify_drafts needs fp32 CUDA weights [B,K+1,V] and tokens [B,K]")
    (B, K), V = tokens.shape, target.shape[2]
    if (B | K | V) >> 31:
        raise ValueError("verify_drafts takes sizes of 32 bits")
    t_stream, t_row, t_step = target.stride()
    if target.shape != (B, K + 1, V) or (V > 1 and t_step != 1):
        raise ValueError(f"target must be [{B},{K + 1},V] with contiguous rows, got {tuple(target.shape)}")
    d_ptr, d_stream, d_row = None, 0, 0
    if draft is not None:
        if draft.shape != (B, K, V) or draft.dtype != torch.float32 or draft.get_device() != index or (V > 1 and draft.stride(2) != 1):
            raise ValueError(f"draft must be fp32 [{B},{K},{V}] with contiguous rows on the target's device")
        d_ptr, (d_stream, d_row, _) = draft.data_ptr(), draft.stride()
    if tokens.dtype != torch.int64 or tokens.get_device() != index or not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous int64 on the target's device")
    if u.dtype != torch.float32 or u.get_device() != index or u.shape != (B, K + 1) or not u.is_contiguous():
        raise ValueError(f"u must be contiguous fp32 [{B},{K + 1}] on the target's device")
    if lengths is not None and (lengths.dtype != torch.int64 or lengths.get_device() != index or lengths.shape != (B,) or not lengths.is_contiguous()):
        raise ValueError(f"lengths must be contiguous int64 [{B}] on the target's device")
    # (sizes one by one, and new_empty, parse faster than a tuple with a type and a device)
    out = torch.empty(B, K + 1, dtype=torch.int64, device=target.device)
    accepted = tokens.new_empty(B)
    if B == 0:
        return out, accepted
    with _on(index):
        nbytes = _verify_workspace(B, K, V)
        ws = tokens.new_empty(nbytes // 8)
        _lib.check(_lib.lib().b200rwkv_verify_drafts(target.data_ptr(), t_stream, t_row, d_ptr, d_stream, d_row, tokens.data_ptr(),
                                                     u.data_ptr(), None if lengths is None else lengths.data_ptr(), B, K, V, out.data_ptr(),
                                                     accepted.data_ptr(), ws.data_ptr(), nbytes, _raw_stream(index)))
    return out, accepted


@lru_cache(maxsize=1024)
def _verify_workspace(B: int, K: int, V: int) -> int:
    return max(8, int(_lib.lib().b200rwkv_verify_drafts_workspace_bytes(B, K, V)))


def advance_state(state: torch.Tensor, counts: torch.Tensor, trace: torch.Tensor, params: torch.Tensor,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The state of B streams after the first ``counts[b]`` of a step's T tokens, for a step whose later tokens were refused
    (a recurrent state cannot drop them).  ``state`` fp32 ``[B,L,5,C]`` in front of the step, ``counts`` int64 ``[B]``
    (clamped to 0..T; 0 leaves the state as it is), ``trace`` fp32 ``[L,4,B,T,C]``: of every block and token the residual
    stream in front of ln1, in front of ln2, the key and the value; ``params`` fp32 ``[L,5,C]``: ln1 weight and bias, ln2
    weight and bias, ``-exp(time_decay)``.  Carries become the layer norms of the last accepted token, the WKV sums take
    ``counts[b]`` steps (agnosticRwkv.py:68-103).  In place when ``out`` is omitted; returns the new state."""
    index, shape = state.get_device(), state.shape
    if len(shape) != 4 or shape[2] != 5 or trace.dim() != 5:
        raise ValueError("advance_state needs state [B,L,5,C] and trace [L,4,B,T,C]")
    B, L, _, Cc = shape
    T = trace.shape[3]
    if (B | L | T | Cc) >> 31:
        raise ValueError("advance_state takes sizes of 32 bits")
    out = state if out is None else out
    for t, want in ((state, shape), (out, shape), (trace, (L, 4, B, T, Cc)), (params, (L, 5, Cc))):
        if t.dtype != torch.float32 or index < 0 or t.get_device() != index or t.shape != want or not t.is_contiguous():
            raise ValueError("advance_state needs contiguous fp32 CUDA tensors: state and out [B,L,5,C], trace [L,4,B,T,C], params [L,5,C]")
    if counts.dtype != torch.int64 or counts.get_device() != index or counts.shape != (B,) or not counts.is_contiguous():
        raise ValueError(f"counts must be contiguous int64 [{B}] on the state's device")
    if B == 0 or T == 0:
        return out if out is state else out.copy_(state)
    with _on(index):
        _lib.check(_lib.lib().b200rwkv_advance_state(state.data_ptr(), out.data_ptr(), counts.data_ptr(), trace.data_ptr(), params.data_ptr(),
                                                     B, L, T, Cc, _raw_stream(index)))
    return out


def matvec(W: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """The reference's TORCH-mode op table entry ``matvec(W, x)`` (agnostic/backends/torch.py:162-164)
    for one vector: ``W`` is the ``[in,out]`` transposed view the reference's ``initTensor`` makes of
    the checkpoint's ``[out,in]`` tensor; the result has ``x``'s dtype.  A matrix that is not such a
    view (its transpose does not have contiguous rows) is refused rather than copied."""
    if W.dim() != 2 or W.stride(0) != 1:
        raise ValueError("matvec expects the transposed view of an [out,in] matrix (stride 1 along the input index)")
    xv = x.reshape(-1)
    if xv.numel() != W.shape[0]:
        raise ValueError("matvec handles one vector per call")
    y = gemv_dense(W.t(), xv.float().contiguous())
    return y.to(x.dtype).reshape(*x.shape[:-1], W.shape[1])
