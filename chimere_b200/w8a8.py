"""Products of 8-bit integers with a scale per token and a scale per output channel (W8A8), over the C ABI.

The form int8 checkpoints have for the projections around the MoE layer and for experts.  The reference has no counterpart: its
weights are ggml blocks.  Every computation happens in the CUDA library; torch owns memory and streams.  All launches go to torch's
current stream of the tensors' device, nothing synchronises, and every call can be captured in a CUDA graph.  Nothing here is differentiable: results carry no gradient and no tangent.

int8 rows start on 16-byte boundaries: a matrix whose width is no multiple of 16 lies in rows that are wider (`padded_i8`).
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import abi

_TYPES = {torch.float32: abi.TYPE_F32, torch.float16: abi.TYPE_F16, torch.bfloat16: abi.TYPE_BF16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda i: torch.cuda.current_stream(i).cuda_stream
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _call(what: str, index: int, *args) -> None:
    """One C entry on the current stream of a device."""
    fn = getattr(abi._lib or abi.load(), what)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        abi.check(rc, what)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(all_bits: int) -> None:
    """Of sizes and options that the C ABI takes as 32-bit integers, or-ed together: ctypes would cut what is wider."""
    if all_bits >> 31:
        raise ValueError("sizes and options: whole numbers from 0 to 2^31 - 1")


def _vector(t: Optional[torch.Tensor], name: str, shape: tuple, dtype: torch.dtype, index: int) -> Optional[int]:
    """Address of a contiguous tensor."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} {shape} on device {index}")
    return t.data_ptr()


def _weight(w: torch.Tensor, name: str, index: int) -> Tuple[int, int]:
    """Address and distance between rows of an int8 matrix (or stack)."""
    rows, K = w.shape[-2:]
    strides = w.stride()
    p, ld = w.data_ptr(), strides[-2] if rows > 1 else (K + 15) // 16 * 16
    if w.dtype is not torch.int8 or w.get_device() != index or (strides[-1] != 1 and K != 1) or ld % 16 or p % 16:
        raise ValueError(f"{name}: int8 on device {index}, the values of a row side by side, rows on 16-byte boundaries (padded_i8 lays a matrix out so)")
    return p, ld


def _floats(x: torch.Tensor, name: str) -> Tuple[int, int, int, int, int]:
    """(rows, width, address, type, distance between rows) of a matrix of float32, float16 or bfloat16."""
    if x.dim() != 2 or x.dtype not in _TYPES or not x.is_cuda:
        raise ValueError(f"{name}: a matrix of float32, float16 or bfloat16 on a CUDA device")
    M, K = x.shape
    ld, step = x.stride()
    if (step != 1 and K != 1) or (M > 1 and ld < K):
        raise ValueError(f"{name}: the values of a row lie side by side, rows do not overlap")
    return M, K, x.data_ptr(), _TYPES[x.dtype], ld if M > 1 else K


def _output(out: Optional[torch.Tensor], rows: int, cols: int, dtype: Optional[torch.dtype], like: torch.Tensor) -> Tuple[torch.Tensor, int, int, int]:
    """(out, address, type, distance between rows)."""
    if out is None:
        if dtype not in _TYPES:
            raise ValueError("out_dtype: float32, float16 or bfloat16")
        out = torch.empty(rows, cols, dtype=dtype, device=like.device)
        return out, out.data_ptr(), _TYPES[dtype], cols
    if dtype is not None and out.dtype is not dtype:
        raise ValueError("out: not of out_dtype")
    m, n, p, kind, ld = _floats(out, "out")
    if m != rows or n != cols or out.get_device() != like.get_device():
        raise ValueError(f"out: [{rows}, {cols}] on device {like.get_device()}")
    return out, p, kind, ld


def padded_i8(q: torch.Tensor) -> torch.Tensor:
    """The same int8 matrix (or stack of matrices) with rows that start on 16-byte boundaries: itself if it is contiguous and they do, else a copy."""
    _need(q.dtype == torch.int8 and q.dim() >= 2, "padded_i8: an int8 matrix or a stack of them")
    K = q.shape[-1]
    if K % 16 == 0:
        q = q.contiguous()
        if q.data_ptr() % 16 == 0:
            return q
    out = torch.zeros(*q.shape[:-1], (K + 15) // 16 * 16, dtype=torch.int8, device=q.device)[..., :K]
    out.copy_(q)
    return out


def quantize_i8(x: torch.Tensor, rows: Optional[torch.Tensor] = None, rows_div: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): int8 rows and their f32 scales, q = rint(x / scale), scale = max|row| / 127.  x [n, K] float32, float16 or bfloat16 on
    the device.  With `rows` (int32 [M]) row i is row rows[i] // rows_div of x -- a dispatch permutation and top_k, say; an index outside x gives
    a row of zeros with scale 0.  A row with an infinity or a NaN has scale NaN.  q is a view of rows padded to 16 bytes."""
    n, K, xp, kind, ldx = _floats(x, "x")
    _ints(K | rows_div)
    index = x.get_device()
    M = n if rows is None else rows.numel()
    rp = _vector(rows, "rows", (M,), torch.int32, index)
    ld = (K + 15) // 16 * 16
    q = torch.empty(M, ld, dtype=torch.int8, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    _call("chimere_b200_quantize_i8", index, xp, kind, ldx, n, rp, rows_div, M, K, q.data_ptr(), ld, scale.data_ptr())
    return q[:, :K], scale


def matmul_w8a8(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = abi.ACT_NONE,
                out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act((q . w^T) * q_scale[:, None] * w_scale + bias): q int8 [M, K], w int8 [N, K], or [2 N, K] with the gate's rows in front of the up matrix'
    for ACT_SWIGLU; w_scale and bias f32, one per row of w.  The integer sums are exact.  out_dtype: float32 unless given."""
    _need(q.is_cuda and q.dim() == 2 and w.dim() == 2 and q.shape[1] == w.shape[1], "q [M, K] and w [N, K] on a CUDA device")
    index, (M, K), R = q.get_device(), q.shape, w.shape[0]
    _ints(K | R | act + 1)
    N = _outputs(R, act)
    out, yp, kind, ldy = _output(out, M, N, out_dtype or (None if out is not None else torch.float32), q)
    xp, ldx = _weight(q, "q", index)
    wp, ldw = _weight(w, "w", index)
    _call("chimere_b200_matmul_w8a8", index, xp, ldx, _vector(q_scale, "q_scale", (M,), torch.float32, index), wp, ldw,
          _vector(w_scale, "w_scale", (R,), torch.float32, index), _vector(bias, "bias", (R,), torch.float32, index), M, N, K, act, yp, kind, ldy,
          _vector(status, "status", (1,), torch.int32, index))
    return out


def _outputs(rows: int, act: int) -> int:
    if act != abi.ACT_SWIGLU:
        return rows
    _need(rows % 2 == 0, "w: gate and up rows in equal number")
    return rows // 2


def _stack(w: torch.Tensor, name: str, index: int) -> Tuple[int, int, int]:
    p, ld = _weight(w, name, index)
    plane = w.stride(0) if w.shape[0] > 1 else w.shape[1] * ld
    if plane % 16:
        raise ValueError(f"{name}: matrices start on 16-byte boundaries")
    return p, ld, plane


def matmul_w8a8_grouped(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        act: int = abi.ACT_NONE, out_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                        out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same with a matrix per group of rows: rows offsets[e] .. offsets[e + 1] of q (int32 [E + 1], ascending, as the router's dispatch leaves them) by w[e];
    w int8 [E, N or 2 N, K], w_scale and bias f32 [E, N or 2 N].  With out_rows (int32 [M]) row i goes to row out_rows[i] of `out` (no index
    twice, or either row's values may end up there).  Rows that belong to no
    group, and rows with an index outside `out`, are not written: `out` keeps what it held there (without `out` those rows are not initialised)."""
    _need(q.is_cuda and q.dim() == 2 and w.dim() == 3 and q.shape[1] == w.shape[2], "q [M, K] and w [E, N, K] on a CUDA device")
    index, (M, K), (E, R) = q.get_device(), q.shape, w.shape[:2]
    _ints(K | R | E | act + 1)
    N = _outputs(R, act)
    y_rows = M if out is None or out_rows is None else out.shape[0]
    out, yp, kind, ldy = _output(out, y_rows, N, out_dtype or (None if out is not None else torch.float32), q)
    xp, ldx = _weight(q, "q", index)
    wp, ldw, plane = _stack(w, "w", index)
    _call("chimere_b200_matmul_w8a8_grouped", index, xp, ldx, _vector(q_scale, "q_scale", (M,), torch.float32, index), wp, ldw, plane,
          _vector(w_scale, "w_scale", (E, R), torch.float32, index), _vector(bias, "bias", (E, R), torch.float32, index),
          _vector(offsets, "offsets", (E + 1,), torch.int32, index), E, M, N, K, act, yp, kind, ldy, y_rows,
          _vector(out_rows, "out_rows", (M,), torch.int32, index), _vector(status, "status", (1,), torch.int32, index))
    return out


def linear_w8a8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = abi.ACT_NONE,
                out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """matmul_w8a8(*quantize_i8(x), w, w_scale, ...) in one call.  out_dtype: that of x unless given.  `out` may share memory with x."""
    M, K, xp, x_kind, ldx = _floats(x, "x")
    _need(w.dim() == 2 and w.shape[1] == K, "x [M, K] and w [N, K]")
    index, R = x.get_device(), w.shape[0]
    _ints(K | R | act + 1)
    N = _outputs(R, act)
    given = out
    out, yp, kind, ldy = _output(out, M, N, out_dtype or (None if out is not None else x.dtype), x)
    wp, ldw = _weight(w, "w", index)
    ws, nbytes = _scratch(x, _linear_bytes(M, N, K))
    if given is not None and nbytes == 0 and _share_memory(x, ldx, out, ldy):     # (what needs no scratch is one launch, which stores while it reads)
        return matmul_w8a8(*quantize_i8(x), w, w_scale, bias, act, out=out, status=status)
    _call("chimere_b200_linear_w8a8", index, xp, x_kind, ldx, wp, ldw, _vector(w_scale, "w_scale", (R,), torch.float32, index),
          _vector(bias, "bias", (R,), torch.float32, index), M, N, K, act, yp, kind, ldy, None if ws is None else ws.data_ptr(), nbytes,
          _vector(status, "status", (1,), torch.int32, index))
    return out


def _share_memory(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int) -> bool:
    """Whether two matrices' ranges meet, but for matrices side by side in one wider one."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (rows, wa), (rows_b, wb) = ((t.shape[0], t.shape[1] * t.element_size()) for t in (a, b))
    pitch, pitch_b, lo, hi = lda * a.element_size(), ldb * b.element_size(), a.data_ptr(), b.data_ptr()
    if lo + pitch * (rows - 1) + wa <= hi or hi + pitch_b * (rows_b - 1) + wb <= lo:
        return False
    if rows == 1 or rows_b == 1 or pitch != pitch_b:
        return True
    if lo > hi:
        lo, hi, wa, wb = hi, lo, wb, wa
    off = (hi - lo) % pitch
    return off < wa or off + wb > pitch


@lru_cache(maxsize=4096)
def _linear_bytes(M: int, N: int, K: int) -> int:
    return abi.load().chimere_b200_linear_w8a8_bytes(M, N, K)


@lru_cache(maxsize=4096)
def _experts_bytes(T: int, top_k: int, H: int, F: int) -> int:
    return abi.load().chimere_b200_experts_w8a8_bytes(T, top_k, H, F)


def _scratch(like: torch.Tensor, nbytes: int) -> Tuple[Optional[torch.Tensor], int]:
    if nbytes < 0:
        abi.check(nbytes, "scratch size")
    return (torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None), nbytes


def experts_w8a8(x: torch.Tensor, perm: torch.Tensor, offsets: torch.Tensor, top_k: int, w_up: torch.Tensor, up_scale: torch.Tensor, w_down: torch.Tensor,
                 down_scale: torch.Tensor, act: int = abi.ACT_SWIGLU, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                 status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows [T * top_k, H] of the routed pairs: down_e . act(gate|up_e . x[pair // top_k]), pair by pair (row t * top_k + j is slot j of token t).  perm int32 [T * top_k]
    and offsets int32 [E + 1]: the router's dispatch (MoeScratch.perm / .offsets).  w_up int8 [E, 2 F, H] (gate rows, then up) for ACT_SWIGLU, [E, F, H] for
    ACT_RELU2; w_down int8 [E, H, F]; scales f32 [E, rows].  Pairs of no expert are not written (without `out`: not initialised).  out_dtype: that of x.  `out` may share memory with x."""
    T, H, xp, x_kind, ldx = _floats(x, "x")
    _need(act in (abi.ACT_SWIGLU, abi.ACT_RELU2), "act: ACT_SWIGLU or ACT_RELU2")
    _need(w_up.dim() == 3 and w_down.dim() == 3, "w_up [E, F or 2 F, H], w_down [E, H, F]")
    index, (E, R, K), F = x.get_device(), w_up.shape, w_down.shape[2]
    _need(K == H and R == (2 * F if act == abi.ACT_SWIGLU else F) and w_down.shape[0] == E and w_down.shape[1] == H, "w_up [E, F or 2 F, H], w_down [E, H, F]")
    _need(top_k >= 1, "top_k: at least 1")
    _ints(E | R | H | F | top_k)
    P = T * top_k
    out, yp, kind, ldy = _output(out, P, H, out_dtype or (None if out is not None else x.dtype), x)
    up, ld_up, plane_up = _stack(w_up, "w_up", index)
    down, ld_down, plane_down = _stack(w_down, "w_down", index)
    ws, nbytes = _scratch(x, _experts_bytes(T, top_k, H, F))
    _call("chimere_b200_experts_w8a8", index, xp, x_kind, ldx, T, _vector(perm, "perm", (P,), torch.int32, index),
          _vector(offsets, "offsets", (E + 1,), torch.int32, index), top_k, E, up, ld_up, plane_up, _vector(up_scale, "up_scale", (E, R), torch.float32, index),
          down, ld_down, plane_down, _vector(down_scale, "down_scale", (E, H), torch.float32, index), H, F, act, yp, kind, ldy,
          None if ws is None else ws.data_ptr(), nbytes, _vector(status, "status", (1,), torch.int32, index))
    return out
