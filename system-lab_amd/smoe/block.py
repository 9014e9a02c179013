"""Operators of an unquantised expert block: token rows to their experts and
back, the norms before and after the block, and matrix products with bias,
activation and residual in their epilogue, each with its gradient.

They take bf16 and fp16 (the row movers and norms fp32 too).  An input's rows
may lie apart (any row stride; the last dimension is contiguous) and be of any
length; weights, maps and outputs are contiguous.  As every op of this
package they are ordered on the current stream, allocate through torch and
never synchronise.  Empty batches return empty tensors without a launch.
"""
from __future__ import annotations

import ctypes

import torch

from . import _C
from .ops import _check, _ptr, _status_workspace, route_sort

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # SMOE_BF16 / _F16 / _F32
_ALL, _HALF = tuple(DTYPES), (torch.bfloat16, torch.float16)
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5}  # SMOE_ACT_*
NORM_MAX_H = 65536
_F32 = torch.float32


def _here(t, name: str) -> None:
    """A tensor on the current GPU (a call's checks cost a few microseconds, as
    much as a small kernel: cheap questions first)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (got {t.device}); the HIP kernels are the only path")
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name} is on {t.device} but the current device is cuda:{torch.cuda.current_device()}")


def _stream() -> int:
    """The current stream's handle on the current device."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _dense(t, name: str, dtypes, shape) -> None:
    """Check a contiguous tensor of a given shape."""
    _here(t, name)
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {tuple(dtypes)}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _rows(t: torch.Tensor, name: str, dtypes, cols: int | None = None, rows: int | None = None) -> int:
    """Check a 2-D input whose rows may lie apart; -> elements between rows."""
    _here(t, name)
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {tuple(dtypes)}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    r, c = t.shape
    if (rows is not None and r != rows) or (cols is not None and c != cols):
        raise ValueError(f"{name} must be [{'*' if rows is None else rows}, {'*' if cols is None else cols}], "
                         f"got {(r, c)}")
    ld, one = t.stride()
    if one != 1 and c > 1 and r > 0:
        raise ValueError(f"{name}'s rows must be contiguous (strides {t.stride()})")
    return ld


def _like(t: torch.Tensor, dtype, shape) -> torch.Tensor:
    return t.new_empty(shape, dtype=dtype)


def _out(out: torch.Tensor | None, like: torch.Tensor, shape, name: str = "out") -> torch.Tensor:
    if out is None:
        return _like(like, like.dtype, shape)
    _dense(out, name, (like.dtype,), shape)
    return out


# ------------------------------------------------------------------ tokens
def _pairs(inv_map, top_k: int, topk_w, T: int) -> None:
    if not 0 < top_k <= 32:
        raise ValueError(f"top_k must be in [1, 32], got {top_k}")
    _check(inv_map, "inv_map", (torch.int32,))
    if inv_map.numel() != T * top_k:
        raise ValueError(f"inv_map must have T*K = {T * top_k} entries, got {inv_map.numel()}")
    if topk_w is not None:
        _dense(topk_w, "topk_w", (_F32,), (T, top_k))


def _tokens_of(rows: int, top_k: int, name: str) -> int:
    if not 0 < top_k <= 32:
        raise ValueError(f"top_k must be in [1, 32], got {top_k}")
    if rows % top_k:
        raise ValueError(f"{name} must have T*K rows, got {rows} for K = {top_k}")
    return rows // top_k


def permute_tokens_rows(x: torch.Tensor, inv_map: torch.Tensor, top_k: int, topk_w: torch.Tensor | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Row inv_map[t*K+k] of the result is x[t], times topk_w[t,k] where given:
    x [T,H] -> [T*K,H] in x's type.  The unquantised ``permute_quant_rows``.
    Rows no pair maps to (ids outside [0, E) have inv_map -1) are not written."""
    ld = _rows(x, "x", _ALL)
    T, H = x.shape
    _pairs(inv_map, top_k, topk_w, T)
    xp = _out(out, x, (T * top_k, H))
    if T and H:
        _C.call("smoe_permute_tokens", _ptr(x), ld, _ptr(inv_map), _ptr(topk_w), T, top_k, H, DTYPES[x.dtype],
                _ptr(xp), _stream())
    return xp


def permute_tokens(x: torch.Tensor, topk_idx: torch.Tensor, num_experts: int, topk_w: torch.Tensor | None = None):
    """Expert sort and row permute: the unquantised ``permute_quant``, with the
    router's weights applied on the way in where ``topk_w`` [T,K] is given.
    x [T,H], topk_idx [T,K] i32 -> (xp [T*K,H], row_map, inv_map, counts,
    offsets) as ``route_sort`` numbers the rows."""
    ld = _rows(x, "x", _ALL)
    T, H = x.shape
    _here(topk_idx, "topk_idx")
    if topk_idx.dim() != 2 or topk_idx.shape[0] != T:
        raise ValueError(f"topk_idx must be [{T}, K], got {list(topk_idx.shape)}")
    K, E, i32 = topk_idx.shape[1], int(num_experts), torch.int32
    _dense(topk_idx, "topk_idx", (i32,), (T, K))
    if not 0 < K <= min(E, 32):
        raise ValueError(f"top-k must be in [1, min(E, 32)], got {K} of {E}")
    if topk_w is not None:
        _dense(topk_w, "topk_w", (_F32,), (T, K))
    R = T * K
    xp, row_map, inv_map = x.new_empty((R, H)), x.new_empty(R, dtype=i32), x.new_empty(R, dtype=i32)
    counts, offsets = x.new_empty(E, dtype=i32), x.new_empty(E + 1, dtype=i32)
    if T == 0:
        return xp, row_map, inv_map, counts.zero_(), offsets.zero_()
    if H == 0:
        return (xp, *route_sort(topk_idx, E))
    ws = _status_workspace(int(_C.lib().smoe_route_sort_workspace_size(T, K, E)), x.device)
    _C.call("smoe_sort_permute_tokens", _ptr(x), ld, _ptr(topk_idx), _ptr(topk_w), T, K, E, H, DTYPES[x.dtype],
            _ptr(row_map), _ptr(inv_map), _ptr(counts), _ptr(offsets), _ptr(xp), _ptr(ws), ws.numel(), _stream())
    return xp, row_map, inv_map, counts, offsets


def unpermute_tokens(y: torch.Tensor, inv_map: torch.Tensor, top_k: int, topk_w: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum over k of topk_w[t,k] * y[inv_map[t*K+k]] (plain rows
    without ``topk_w``): fp32 sums in k order, rounded once.  y [T*K,H] ->
    [T,H] in y's type.  ``unpermute_combine`` for every type and row length."""
    ld = _rows(y, "y", _ALL)
    T, H = _tokens_of(y.shape[0], top_k, "y"), y.shape[1]
    _pairs(inv_map, top_k, topk_w, T)
    o = _out(out, y, (T, H))
    if T and H:
        _C.call("smoe_unpermute_tokens", _ptr(y), ld, _ptr(inv_map), _ptr(topk_w), T, top_k, H, DTYPES[y.dtype],
                _ptr(o), _stream())
    return o


def permute_tokens_bwd(dxp: torch.Tensor, inv_map: torch.Tensor, top_k: int, x: torch.Tensor | None = None,
                       topk_w: torch.Tensor | None = None):
    """Gradient of ``permute_tokens_rows``: dxp [T*K,H] -> dx [T,H]; with
    ``topk_w`` (then ``x`` is needed too) -> (dx, dtopk_w [T,K] f32)."""
    if topk_w is None:
        return unpermute_tokens(dxp, inv_map, top_k)
    ld = _rows(dxp, "dxp", _ALL)
    T, H = _tokens_of(dxp.shape[0], top_k, "dxp"), dxp.shape[1]
    _pairs(inv_map, top_k, topk_w, T)
    if x is None:
        raise ValueError("the weights' gradient needs x")
    ldx = _rows(x, "x", (dxp.dtype,), H, T)
    dx, dw = _like(dxp, dxp.dtype, (T, H)), _like(dxp, _F32, (T, top_k))
    if T and H:
        _C.call("smoe_permute_tokens_bwd", _ptr(dxp), ld, _ptr(x), ldx, _ptr(inv_map), _ptr(topk_w), T, top_k, H,
                DTYPES[dxp.dtype], _ptr(dx), _ptr(dw), _stream())
    return dx, dw if H else dw.zero_()


def unpermute_tokens_bwd(dout: torch.Tensor, inv_map: torch.Tensor, top_k: int, y: torch.Tensor | None = None,
                         topk_w: torch.Tensor | None = None):
    """Gradient of ``unpermute_tokens``: dout [T,H] -> dy [T*K,H]; with
    ``topk_w`` (then ``y`` is needed too) -> (dy, dtopk_w [T,K] f32).  Rows of
    dy no pair maps to are not written."""
    if topk_w is None:
        return permute_tokens_rows(dout, inv_map, top_k)
    ld = _rows(dout, "dout", _ALL)
    T, H = dout.shape
    _pairs(inv_map, top_k, topk_w, T)
    if y is None:
        raise ValueError("the weights' gradient needs y")
    ldy = _rows(y, "y", (dout.dtype,), H, T * top_k)
    dy, dw = _like(dout, dout.dtype, (T * top_k, H)), _like(dout, _F32, (T, top_k))
    if T and H:
        _C.call("smoe_unpermute_tokens_bwd", _ptr(dout), ld, _ptr(y), ldy, _ptr(inv_map), _ptr(topk_w), T, top_k, H,
                DTYPES[dout.dtype], _ptr(dy), _ptr(dw), _stream())
    return dy, dw if H else dw.zero_()


# ------------------------------------------------------------------- norms
def _norm_weight(weight, v: torch.Tensor) -> int:
    if not 0 < v.shape[1] <= NORM_MAX_H:
        raise ValueError(f"rows must have 1 to {NORM_MAX_H} values, got {v.shape[1]}")
    if weight is None:
        return 0
    _dense(weight, "weight", (v.dtype, _F32), (v.shape[1],))
    return int(weight.dtype == _F32)


def _norm_gate(gate, v: torch.Tensor):
    """(SMOE_GATE_*, row stride, gate is f32) of a gate [H], [T,1] or [T,H]."""
    if gate is None:
        return 0, 0, 0
    T, H = v.shape
    f32 = int(gate.dtype == _F32)
    if gate.dim() == 1:
        _dense(gate, "gate", (v.dtype, _F32), (H,))
        return 1, 0, f32
    ld = _rows(gate, "gate", (v.dtype, _F32), None, T)
    if gate.shape[1] == 1 and H != 1:
        return 2, ld, f32
    if gate.shape[1] != H:
        raise ValueError(f"gate must be [{H}], [{T}, 1] or [{T}, {H}], got {list(gate.shape)}")
    return 3, ld, f32


def _eps(eps: float) -> float:
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"eps must be positive, got {eps}")
    return float(eps)


def _rstd(rstd, T: int) -> None:
    _dense(rstd, "rstd", (_F32,), (T,))


def block_norm_in(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6):
    """The RMS norm before a block: h = x * rstd * weight with rstd =
    1 / sqrt(mean(x^2) + eps) over each row.  x [T,H], weight [H] in x's type
    or fp32 -> (h [T,H], rstd [T] f32); rstd is what the gradient needs."""
    ld = _rows(x, "x", _ALL)
    T, H = x.shape
    wf = _norm_weight(weight, x)
    h, rstd = _like(x, x.dtype, (T, H)), _like(x, _F32, (T,))
    if T:
        _C.call("smoe_block_norm_in", _ptr(x), ld, _ptr(weight), wf, _eps(eps), T, H, DTYPES[x.dtype], _ptr(h),
                _ptr(rstd), _stream())
    return h, rstd


def block_norm_out(y: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None = None,
                   gate: torch.Tensor | None = None, residual_scale: float = 1.0, eps: float = 1e-6):
    """The norm after a block with the block's gate and the scaled residual, in
    one pass: out = residual_scale * x + gate * (y * rstd * weight), rstd of
    y's rows.  ``gate``: None, [H] (a channel), [T,1] (a token) or [T,H].
    -> (out [T,H], rstd [T] f32)."""
    ldy = _rows(y, "y", _ALL)
    T, H = y.shape
    ldx = _rows(x, "x", (y.dtype,), H, T)
    wf = _norm_weight(weight, y)
    mode, ldg, gf = _norm_gate(gate, y)
    out, rstd = _like(y, y.dtype, (T, H)), _like(y, _F32, (T,))
    if T:
        _C.call("smoe_block_norm_out", _ptr(y), ldy, _ptr(x), ldx, _ptr(weight), _ptr(gate), ldg, mode, wf | gf << 1,
                float(residual_scale), _eps(eps), T, H, DTYPES[y.dtype], _ptr(out), _ptr(rstd), _stream())
    return out, rstd


def _norm_bwd_ws(T: int, H: int, like: torch.Tensor, need: bool):
    n = int(_C.lib().smoe_block_norm_bwd_workspace_size(T, H)) if need else 0
    return (torch.empty(n, dtype=torch.uint8, device=like.device) if n else None), n


def block_norm_in_bwd(dh: torch.Tensor, x: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                      dskip: torch.Tensor | None = None, skip_scale: float = 1.0):
    """Gradient of ``block_norm_in``: -> (dx [T,H], dweight [H] in weight's
    type, None without weight).  ``dskip`` [T,H] is the gradient that reaches x
    past the block: dx then also holds skip_scale * dskip (the residual of
    ``block_norm_out``: its dout and residual_scale)."""
    ldx = _rows(x, "x", _ALL)
    T, H = x.shape
    ldh = _rows(dh, "dh", (x.dtype,), H, T)
    lds = 0 if dskip is None else _rows(dskip, "dskip", (x.dtype,), H, T)
    wf = _norm_weight(weight, x)
    _rstd(rstd, T)
    dx = _like(x, x.dtype, (T, H))
    dw = None if weight is None else torch.empty_like(weight)
    if T == 0:
        return dx, dw if dw is None else dw.zero_()
    ws, n = _norm_bwd_ws(T, H, x, dw is not None)
    _C.call("smoe_block_norm_in_bwd", _ptr(dh), ldh, _ptr(x), ldx, _ptr(rstd), _ptr(weight), wf, _ptr(dskip), lds,
            float(skip_scale), T, H, DTYPES[x.dtype], _ptr(dx), _ptr(dw), _ptr(ws), n, _stream())
    return dx, dw


def block_norm_out_bwd(dout: torch.Tensor, y: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                       gate: torch.Tensor | None = None):
    """Gradient of ``block_norm_out`` by y, weight and gate: -> (dy [T,H],
    dweight [H] | None, dgate in gate's shape and type | None).  The
    residual's gradient is residual_scale * dout (``block_norm_in_bwd`` adds
    it: ``dskip``)."""
    ldy = _rows(y, "y", _ALL)
    T, H = y.shape
    ldo = _rows(dout, "dout", (y.dtype,), H, T)
    wf = _norm_weight(weight, y)
    mode, ldg, gf = _norm_gate(gate, y)
    _rstd(rstd, T)
    dy = _like(y, y.dtype, (T, H))
    dw = None if weight is None else torch.empty_like(weight)
    dg = None if gate is None else _like(gate, gate.dtype, gate.shape)
    if T == 0:
        return dy, dw if dw is None else dw.zero_(), dg if dg is None else dg.zero_()
    ws, n = _norm_bwd_ws(T, H, y, dw is not None or mode == 1)
    _C.call("smoe_block_norm_out_bwd", _ptr(dout), ldo, _ptr(y), ldy, _ptr(rstd), _ptr(weight), _ptr(gate), ldg, mode,
            wf | gf << 1, T, H, DTYPES[y.dtype], _ptr(dy), _ptr(dw), _ptr(dg), _ptr(ws), n, _stream())
    return dy, dw, dg


# ------------------------------------------------------------------ linear
def _linear_weight(w, x: torch.Tensor, act: str, bias, offsets):
    """(E, N, K) of a weight [N,K], or [E,N,K] with offsets [E+1]."""
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
    _here(w, "w")
    if w.dim() != (2 if offsets is None else 3):
        raise ValueError(f"w must be [N, K], or [E, N, K] with offsets; got shape {tuple(w.shape)}")
    _dense(w, "w", (x.dtype,), w.shape)
    E = 1 if offsets is None else w.shape[0]
    N, K = w.shape[-2:]
    if x.shape[1] != K:
        raise ValueError(f"x has {x.shape[1]} columns, w's rows {K}")
    if act == "swiglu" and N % 2:
        raise ValueError("w's rows must be gate | up halves for act='swiglu'")
    if offsets is not None:
        _dense(offsets, "offsets", (torch.int32,), (E + 1,))
    if bias is not None:
        _dense(bias, "bias", (x.dtype, _F32), w.shape[:-1])
    if not (E and N and K):
        raise ValueError(f"w must not be empty, got {list(w.shape)}")
    return E, N, K


def linear_act(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, act: str = "none",
               residual: torch.Tensor | None = None, offsets: torch.Tensor | None = None, save_z: bool = False,
               out: torch.Tensor | None = None):
    """act(x W^T + bias) + residual in bf16 or fp16, bias, activation and
    residual applied to the product's fp32 sums and rounded once.

    x [R,K]; w [N,K], or [E,N,K] with ``offsets`` [E+1] i32: rows
    [offsets[e], offsets[e+1]) of x go through w[e] and rows of no expert are
    not written.  ``bias`` [N] / [E,N] in x's type or fp32.  ``act``: "none",
    "relu", "silu", "gelu" (erf), "gelu_tanh" or "swiglu" (w's rows are gate |
    up halves, the result silu(gate) * up has N/2 columns).  ``residual`` and
    the result are [R, N or N/2].  ``save_z`` also returns z = x W^T + bias
    [R,N], what ``linear_act_bwd`` needs for any act but "none"."""
    ldx = _rows(x, "x", _HALF)
    E, N, K = _linear_weight(w, x, act, bias, offsets)
    R, M = x.shape[0], N // 2 if act == "swiglu" else N
    ldr = 0 if residual is None else _rows(residual, "residual", (x.dtype,), M, R)
    o = _out(out, x, (R, M))
    z = _like(x, x.dtype, (R, N)) if save_z else None
    if R:
        n = int(_C.lib().smoe_linear_act_workspace_size(R, N, K, E, ACTS[act]))
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        a = _C.LinearFwd(R, N, K, E, ACTS[act], DTYPES[x.dtype], int(bias is not None and bias.dtype == _F32),
                         _ptr(x), ldx, _ptr(w), _ptr(bias), _ptr(residual), ldr, _ptr(offsets), _ptr(o), _ptr(z),
                         _ptr(ws), n)
        _C.call("smoe_linear_act", ctypes.byref(a), _stream())
    return (o, z) if save_z else o


def linear_act_bwd(dout: torch.Tensor, x: torch.Tensor, w: torch.Tensor, z: torch.Tensor | None = None,
                   act: str = "none", bias: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
                   need_dx: bool = True, need_dw: bool = True, dw_out: torch.Tensor | None = None,
                   accumulate: bool = False):
    """Gradients of ``linear_act``: -> (dx [R,K], dw like w, dbias like bias),
    None for what is not asked for (``need_dx``, ``need_dw``, ``bias`` None).
    ``z`` is the forward's (``save_z``).  ``dw_out`` (w's shape, fp32 or w's
    type) receives dw, added to what it holds with ``accumulate`` (a
    ``main_grad``); without it dw is in w's type.  dz = dout act'(z) is
    rounded to x's type as both products' operand; sums are fp32.  Experts
    without rows get zero gradients (nothing is added to ``dw_out``).  The
    residual's gradient is dout."""
    ldx = _rows(x, "x", _HALF)
    E, N, K = _linear_weight(w, x, act, bias, offsets)
    R, M = x.shape[0], N // 2 if act == "swiglu" else N
    ldo = _rows(dout, "dout", (x.dtype,), M, R)
    if act != "none":
        if z is None:
            raise ValueError(f"the gradient of act={act!r} needs z (linear_act's save_z)")
        _dense(z, "z", (x.dtype,), (R, N))
    if accumulate and dw_out is None:
        raise ValueError("accumulate needs the buffer to add into (dw_out)")
    if dw_out is not None:
        _dense(dw_out, "dw_out", (_F32, w.dtype), w.shape)
    dx = _like(x, x.dtype, (R, K)) if need_dx else None
    dw = (dw_out if dw_out is not None else torch.empty_like(w)) if need_dw else None
    db = None if bias is None else torch.empty_like(bias)
    if R == 0:
        if dw is not None and not accumulate:
            dw.zero_()
        return dx, dw, db if db is None else db.zero_()
    n = int(_C.lib().smoe_linear_act_bwd_workspace_size(R, N, K, E, ACTS[act], int(db is not None)))
    ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
    mode = (0 if dw is None or dw.dtype == _F32 else 2) | int(accumulate)
    a = _C.LinearBwd(R, N, K, E, ACTS[act], DTYPES[x.dtype], int(bias is not None and bias.dtype == _F32), mode,
                     _ptr(dout), ldo, _ptr(x), ldx, _ptr(w), _ptr(z) if act != "none" else None, _ptr(offsets),
                     _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n)
    _C.call("smoe_linear_act_bwd", ctypes.byref(a), _stream())
    return dx, dw, db
