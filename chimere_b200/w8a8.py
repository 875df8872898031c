"""Products of 8-bit integers with a scale per token and a scale per output channel (W8A8), over the C ABI.

The form int8 checkpoints have for the projections around the MoE layer and for experts.  The reference has no counterpart: its
weights are ggml blocks.  Every computation happens in the CUDA library; torch owns memory and streams.  All launches go to torch's
current stream of the tensors' device, nothing synchronises, and every call can be captured in a CUDA graph.

int8 rows start on 16-byte boundaries: a matrix whose width is no multiple of 16 lies in rows that are wider (`padded_i8`).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import abi

_TYPES = {torch.float32: abi.TYPE_F32, torch.float16: abi.TYPE_F16, torch.bfloat16: abi.TYPE_BF16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _call(what: str, device: torch.device, *args) -> None:
    """One C entry on the device's current stream."""
    fn = getattr(abi.load(), what)
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        abi.check(rc, what)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _vector(t: Optional[torch.Tensor], name: str, shape: tuple, dtype: torch.dtype, device: torch.device) -> Optional[int]:
    if t is None:
        return None
    _need(t.dtype == dtype and t.shape == shape and t.device == device and t.is_contiguous(), f"{name}: contiguous {dtype} {shape} on {device}")
    return t.data_ptr()


def _rows_ok(t: torch.Tensor, name: str) -> int:
    """Distance between rows of a matrix whose rows are contiguous."""
    _need(t.stride(-1) == 1 or t.shape[-1] == 1, f"{name}: the values of a row lie side by side")
    return t.stride(-2) if t.shape[-2] > 1 else (t.shape[-1] + 15) // 16 * 16


def _weight(w: torch.Tensor, name: str, device: torch.device) -> Tuple[int, int]:
    _need(w.dtype == torch.int8 and w.device == device, f"{name}: int8 on {device}")
    ld = _rows_ok(w, name)
    _need(ld % 16 == 0 and w.data_ptr() % 16 == 0, f"{name}: rows start on 16-byte boundaries (padded_i8 lays a matrix out so)")
    return w.data_ptr(), ld


def _output(out: Optional[torch.Tensor], rows: int, cols: int, dtype: Optional[torch.dtype], device: torch.device) -> torch.Tensor:
    if out is None:
        _need(dtype in _TYPES, "out_dtype: float32, float16 or bfloat16")
        return torch.empty(rows, cols, dtype=dtype, device=device)
    _need(out.dim() == 2 and out.shape == (rows, cols) and out.device == device and out.dtype in _TYPES and (dtype is None or dtype == out.dtype),
          f"out: [{rows}, {cols}] of float32, float16 or bfloat16 on {device}")
    _need(out.stride(1) == 1 or cols == 1, "out: the values of a row lie side by side")
    _need(rows <= 1 or out.stride(0) >= cols, "out: rows do not overlap")
    return out


def _ld_out(out: torch.Tensor) -> int:
    return out.stride(0) if out.shape[0] > 1 else max(out.stride(0), out.shape[1])


def padded_i8(q: torch.Tensor) -> torch.Tensor:
    """The same int8 matrix (or stack of matrices) with rows that start on 16-byte boundaries: a copy where they do not already."""
    _need(q.dtype == torch.int8 and q.dim() >= 2, "padded_i8: an int8 matrix or a stack of them")
    K = q.shape[-1]
    if K % 16 == 0:
        return q.contiguous()
    out = torch.zeros(*q.shape[:-1], (K + 15) // 16 * 16, dtype=torch.int8, device=q.device)[..., :K]
    out.copy_(q)
    return out


def quantize_i8(x: torch.Tensor, rows: Optional[torch.Tensor] = None, rows_div: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): int8 rows and their f32 scales, q = rint(x / scale), scale = max|row| / 127.  x [n, K] float32, float16 or bfloat16 on
    the device.  With `rows` (int32 [M]) row i is row rows[i] // rows_div of x -- a dispatch permutation and top_k, say; an index outside x gives
    a row of zeros with scale 0.  A row with an infinity or a NaN has scale NaN.  q is a view of rows padded to 16 bytes."""
    _need(x.is_cuda and x.dim() == 2 and x.dtype in _TYPES, "x: [n, K] of float32, float16 or bfloat16 on a CUDA device")
    _need(x.stride(1) == 1 or x.shape[1] == 1, "x: the values of a row lie side by side")
    M, K = x.shape[0] if rows is None else rows.shape[0], x.shape[1]
    rp = None if rows is None else _vector(rows, "rows", (M,), torch.int32, x.device)
    ld = (K + 15) // 16 * 16
    q = torch.empty(M, ld, dtype=torch.int8, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    _need(x.shape[0] <= 1 or x.stride(0) >= K, "x: rows do not overlap")
    _call("chimere_b200_quantize_i8", x.device, x.data_ptr(), _TYPES[x.dtype], max(x.stride(0), K), x.shape[0], rp, rows_div, M, K, q.data_ptr(), ld,
          scale.data_ptr())
    return q[:, :K], scale


def matmul_w8a8(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = abi.ACT_NONE,
                out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act((q . w^T) * q_scale[:, None] * w_scale + bias): q int8 [M, K], w int8 [N, K], or [2 N, K] with the gate's rows in front of the up matrix'
    for ACT_SWIGLU; w_scale and bias f32, one per row of w.  The integer sums are exact.  out_dtype: float32 unless given."""
    _need(q.is_cuda and q.dim() == 2 and w.dim() == 2 and q.shape[1] == w.shape[1], "q [M, K] and w [N, K] on a CUDA device")
    dev, (M, K), R = q.device, q.shape, w.shape[0]
    _need(act != abi.ACT_SWIGLU or R % 2 == 0, "w: gate and up rows in equal number")
    N = R // 2 if act == abi.ACT_SWIGLU else R
    out = _output(out, M, N, out_dtype or (None if out is not None else torch.float32), dev)
    xp, ldx = _weight(q, "q", dev)
    wp, ldw = _weight(w, "w", dev)
    _call("chimere_b200_matmul_w8a8", dev, xp, ldx, _vector(q_scale, "q_scale", (M,), torch.float32, dev), wp, ldw,
          _vector(w_scale, "w_scale", (R,), torch.float32, dev), _vector(bias, "bias", (R,), torch.float32, dev), M, N, K, act, out.data_ptr(), _TYPES[out.dtype],
          _ld_out(out), _vector(status, "status", (1,), torch.int32, dev))
    return out


def _stack(w: torch.Tensor, name: str, device: torch.device) -> Tuple[int, int, int]:
    _need(w.dim() == 3, f"{name}: [E, rows, K]")
    p, ld = _weight(w, name, device)
    plane = w.stride(0) if w.shape[0] > 1 else w.shape[1] * ld
    _need(plane % 16 == 0, f"{name}: matrices start on 16-byte boundaries")
    return p, ld, plane


def matmul_w8a8_grouped(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        act: int = abi.ACT_NONE, out_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                        out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same with a matrix per group of rows: rows offsets[e] .. offsets[e + 1] of q (int32 [E + 1], as the router's dispatch leaves them) by w[e];
    w int8 [E, N or 2 N, K], w_scale and bias f32 [E, N or 2 N].  With out_rows (int32 [M]) row i goes to row out_rows[i] of `out`.  Rows that belong to no
    group, and rows with an index outside `out`, are not written: `out` keeps what it held there (without `out` those rows are not initialised)."""
    _need(q.is_cuda and q.dim() == 2 and w.dim() == 3 and q.shape[1] == w.shape[2], "q [M, K] and w [E, N, K] on a CUDA device")
    dev, (M, K), (E, R) = q.device, q.shape, w.shape[:2]
    _need(act != abi.ACT_SWIGLU or R % 2 == 0, "w: gate and up rows in equal number")
    N = R // 2 if act == abi.ACT_SWIGLU else R
    y_rows = M if out is None or out_rows is None else out.shape[0]
    out = _output(out, y_rows, N, out_dtype or (None if out is not None else torch.float32), dev)
    xp, ldx = _weight(q, "q", dev)
    wp, ldw, plane = _stack(w, "w", dev)
    _call("chimere_b200_matmul_w8a8_grouped", dev, xp, ldx, _vector(q_scale, "q_scale", (M,), torch.float32, dev), wp, ldw, plane,
          _vector(w_scale, "w_scale", (E, R), torch.float32, dev), _vector(bias, "bias", (E, R), torch.float32, dev),
          _vector(offsets, "offsets", (E + 1,), torch.int32, dev), E, M, N, K, act, out.data_ptr(), _TYPES[out.dtype], _ld_out(out), y_rows,
          _vector(out_rows, "out_rows", (M,), torch.int32, dev), _vector(status, "status", (1,), torch.int32, dev))
    return out


def linear_w8a8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = abi.ACT_NONE,
                out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """matmul_w8a8(*quantize_i8(x), w, w_scale, ...) in one call.  out_dtype: that of x unless given."""
    _need(x.is_cuda and x.dim() == 2 and x.dtype in _TYPES, "x: [M, K] of float32, float16 or bfloat16 on a CUDA device")
    _need(w.dim() == 2 and x.shape[1] == w.shape[1], "x [M, K] and w [N, K]")
    dev, (M, K), R = x.device, x.shape, w.shape[0]
    _need(x.stride(1) == 1 or K == 1, "x: the values of a row lie side by side")
    _need(M <= 1 or x.stride(0) >= K, "x: rows do not overlap")
    _need(act != abi.ACT_SWIGLU or R % 2 == 0, "w: gate and up rows in equal number")
    N = R // 2 if act == abi.ACT_SWIGLU else R
    out = _output(out, M, N, out_dtype or (None if out is not None else x.dtype), dev)
    wp, ldw = _weight(w, "w", dev)
    nbytes = abi.load().chimere_b200_linear_w8a8_bytes(M, K)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call("chimere_b200_linear_w8a8", dev, x.data_ptr(), _TYPES[x.dtype], max(x.stride(0), K), wp, ldw, _vector(w_scale, "w_scale", (R,), torch.float32, dev),
          _vector(bias, "bias", (R,), torch.float32, dev), M, N, K, act, out.data_ptr(), _TYPES[out.dtype], _ld_out(out), ws.data_ptr(), nbytes,
          _vector(status, "status", (1,), torch.int32, dev))
    return out


def experts_w8a8(x: torch.Tensor, perm: torch.Tensor, offsets: torch.Tensor, top_k: int, w_up: torch.Tensor, up_scale: torch.Tensor, w_down: torch.Tensor,
                 down_scale: torch.Tensor, act: int = abi.ACT_SWIGLU, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                 status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows [T * top_k, H] of the routed pairs: down_e . act(gate|up_e . x[pair // top_k]), pair by pair (row t * top_k + j is slot j of token t).  perm int32 [T * top_k]
    and offsets int32 [E + 1]: the router's dispatch (MoeScratch.perm / .offsets).  w_up int8 [E, 2 F, H] (gate rows, then up) for ACT_SWIGLU, [E, F, H] for
    ACT_RELU2; w_down int8 [E, H, F]; scales f32 [E, rows].  Pairs of no expert are not written (without `out`: not initialised).  out_dtype: that of x."""
    _need(x.is_cuda and x.dim() == 2 and x.dtype in _TYPES, "x: [T, H] of float32, float16 or bfloat16 on a CUDA device")
    _need(act in (abi.ACT_SWIGLU, abi.ACT_RELU2), "act: ACT_SWIGLU or ACT_RELU2")
    _need(w_up.dim() == 3 and w_down.dim() == 3, "w_up [E, F or 2 F, H], w_down [E, H, F]")
    dev, (T, H), (E, R), F = x.device, x.shape, w_up.shape[:2], w_down.shape[2]
    _need(R == (2 * F if act == abi.ACT_SWIGLU else F) and w_up.shape[2] == H and w_down.shape[:2] == (E, H), "w_up [E, F or 2 F, H], w_down [E, H, F]")
    _need(x.stride(1) == 1 or H == 1, "x: the values of a row lie side by side")
    _need(T <= 1 or x.stride(0) >= H, "x: rows do not overlap")
    _need(top_k >= 1, "top_k: at least 1")
    P = T * top_k
    out = _output(out, P, H, out_dtype or (None if out is not None else x.dtype), dev)
    up, ld_up, plane_up = _stack(w_up, "w_up", dev)
    down, ld_down, plane_down = _stack(w_down, "w_down", dev)
    nbytes = abi.load().chimere_b200_experts_w8a8_bytes(P, H, F)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call("chimere_b200_experts_w8a8", dev, x.data_ptr(), _TYPES[x.dtype], max(x.stride(0), H), T, _vector(perm, "perm", (P,), torch.int32, dev),
          _vector(offsets, "offsets", (E + 1,), torch.int32, dev), top_k, E, up, ld_up, plane_up, _vector(up_scale, "up_scale", (E, R), torch.float32, dev),
          down, ld_down, plane_down, _vector(down_scale, "down_scale", (E, H), torch.float32, dev), H, F, act, out.data_ptr(), _TYPES[out.dtype], _ld_out(out),
          ws.data_ptr(), nbytes, _vector(status, "status", (1,), torch.int32, dev))
    return out
