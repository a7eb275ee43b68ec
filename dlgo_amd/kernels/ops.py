"""Python faces of the HIP kernels: each checks on the host what its kernel and
grid assume (device, dtype, contiguity, shapes), then launches on torch's current
stream.  There is no other implementation behind these: on a machine without the
GPU or the compiler they raise.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Dict, List, Optional, Sequence

import torch

from . import build

PAGE = 64   # tokens per cache page; the kernels are compiled with the same number

EPI_STORE, EPI_ACCUM_F32, EPI_SWIGLU, EPI_STORE_F32 = 0, 1, 2, 3
GEMM_AUTO, GEMM_STREAM, GEMM_TILE128, GEMM_TILE64, GEMM_TILE32, GEMM_ROWS16 = 0, 1, 2, 3, 4, 5
GEMM_FEW_ROWS = 64      # up to this many rows of x the weight-streaming kernels can be chosen
GEMM_SPLIT_FLOATS = 1 << 22   # scratch that lets gemm() share the inner size of a product out over blocks
GEMM_VERY_WIDE = 65536   # from this many weight rows on (a vocabulary: 16 blocks of 16 rows for each of 256 compute units) the tiled kernel is faster for any number of rows of x
GEMM_FEW_ROWS_WIDE = 16  # ... and up to this many when the weight has very many rows (there the tiled kernel is faster)

_DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1}


class KernelError(RuntimeError):
    pass


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError:
        raise KernelError(f"kernels run in float32 or bfloat16, not {dtype}") from None


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)    # the handle without a Stream object around it


_raw_device = getattr(torch._C, "_cuda_getDevice", None)              # the current device without torch.cuda's start-up check


def _stream() -> ctypes.c_void_p:
    """torch's current stream on the current device, as the launches take it (asked at every launch: a recording has
    a stream of its own)."""
    if _raw_stream is not None and _raw_device is not None:
        return ctypes.c_void_p(_raw_stream(_raw_device()))
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t: Optional[torch.Tensor]) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _need(t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None, dims: Optional[int] = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise KernelError(f"{name}: expected a tensor on the GPU")
    if dtype is not None and t.dtype != dtype:
        raise KernelError(f"{name}: expected {dtype}, found {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise KernelError(f"{name}: expected {dims} dimensions, found shape {tuple(t.shape)}")


def _rows(t: torch.Tensor, name: str) -> int:
    """Row stride (elements) of a 2-d tensor whose rows are contiguous."""
    strides = t.stride()
    if len(strides) != 2 or (strides[1] != 1 and t.shape[1] > 1):
        raise KernelError(f"{name}: expected rows that are contiguous in memory, found shape {tuple(t.shape)} strides {strides}")
    return strides[0] if t.shape[0] > 1 else max(strides[0], t.shape[1])


def _rows32(t: torch.Tensor, name: str) -> int:
    """_rows() for a kernel that takes the stride as a 32-bit number."""
    stride = _rows(t, name)
    if stride >= 2 ** 31:
        raise KernelError(f"{name}: rows {stride} elements apart, at most {2 ** 31 - 1} are taken")
    return stride


def _check(err: Optional[bytes]) -> None:
    if err:
        raise KernelError(err.decode())


_libs: dict = {}      # (module, defines) -> loaded library with its return types set; looked up at every launch


def _lib(module: str, defines=()):
    key = (module, tuple(defines))
    lib = _libs.get(key)
    if lib is None:
        lib = build.load(module, defines)
        for name in ("dlgo_embed", "dlgo_copy_rows", "dlgo_rmsnorm", "dlgo_rope_kv", "dlgo_gemm", "dlgo_gemm_accum_norm", "dlgo_gemm_parts", "dlgo_gemm_rows", "dlgo_gemm_rmsnorm", "dlgo_gemm_rows_leave_parts", "dlgo_gemm_rows_scaled", "dlgo_gemm_tile_leave", "dlgo_gemm_tile_scaled", "dlgo_attention_rows",
                     "dlgo_attention_prefill", "dlgo_attention_prefill_f32", "dlgo_attention_decode", "dlgo_attention_decode_f32", "dlgo_argmax", "dlgo_sample", "dlgo_bias_add", "dlgo_head_rmsnorm",
                     "dlgo_rope_kv_q8", "dlgo_attention_q8", "dlgo_verify_drafts"):
            if hasattr(lib, name):
                getattr(lib, name).restype = ctypes.c_char_p
        _libs[key] = lib
    return lib


# ---------------------------------------------------------------------------
def embed(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """out[t, :] = table[ids[t], :] as float32."""
    _need(table, "embed table", dims=2)
    _need(ids, "token ids", torch.int32, 1)
    _need(out, "embed output", torch.float32, 2)
    n, d = ids.shape[0], table.shape[1]
    if not table.is_contiguous() or not out.is_contiguous() or tuple(out.shape) != (n, d):
        raise KernelError(f"embed: output {tuple(out.shape)} does not fit {n} tokens of width {d}")
    _check(_lib("embed").dlgo_embed(_ptr(table), dtype_code(table.dtype), _ptr(ids), _ptr(out), n, d, table.shape[0], _stream()))
    return out


def copy_rows(src: torch.Tensor, dst: torch.Tensor, src_rows: Optional[torch.Tensor] = None,
              dst_rows: Optional[torch.Tensor] = None, n: Optional[int] = None) -> torch.Tensor:
    """dst[dst_rows[i]] = src[src_rows[i]] for i < n (a missing list stands for i itself; n defaults to the lists'
    length, or to src's rows).  Rows of any element type whose bytes are a multiple of 4; 1-d tensors are rows of one
    element.  The lists are int32 on the device and hold row numbers inside the two tensors (the caller's duty: they
    are not read here); source and destination rows must not overlap."""
    given = dst
    if src.dim() == 1:
        src = src.unsqueeze(1)
    if dst.dim() == 1:
        dst = dst.unsqueeze(1)
    _need(src, "rows to copy", dims=2)
    _need(dst, "copied rows", src.dtype, 2)
    for name, r in (("source rows", src_rows), ("destination rows", dst_rows)):
        if r is not None:
            _need(r, name, torch.int32, 1)
    if n is None:
        n = src_rows.shape[0] if src_rows is not None else (dst_rows.shape[0] if dst_rows is not None else src.shape[0])
    es = src.element_size()
    if src.shape[1] != dst.shape[1] or (src.shape[1] * es) % 4 or n < 0 \
            or any(r is not None and r.shape[0] < n for r in (src_rows, dst_rows)) \
            or (src_rows is None and src.shape[0] < n) or (dst_rows is None and dst.shape[0] < n):
        raise KernelError(f"copy_rows: {n} rows of {tuple(src.shape)} into {tuple(dst.shape)} (rows of equal width, a multiple of 4 bytes)")
    _check(_lib("embed").dlgo_copy_rows(_ptr(src), _ptr(src_rows), _ptr(dst), _ptr(dst_rows), n, ctypes.c_longlong(src.shape[1] * es),
                                        ctypes.c_longlong(_rows(src, "rows to copy") * es), ctypes.c_longlong(_rows(dst, "copied rows") * es),
                                        _stream()))
    return given


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor,
            rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[r] = rmsnorm(x[rows[r]] if rows is given else x[r]) * weight; x float32, out in its own dtype."""
    _need(x, "rmsnorm input", torch.float32, 2)
    _need(weight, "rmsnorm weight", torch.float32, 1)
    _need(out, "rmsnorm output", dims=2)
    d = x.shape[1]
    n = out.shape[0]
    if rows is not None:
        _need(rows, "rmsnorm rows", torch.int32, 1)
        if rows.shape[0] != n:
            raise KernelError("rmsnorm: one output row per gathered row")
    elif x.shape[0] != n:
        raise KernelError(f"rmsnorm: {x.shape[0]} input rows, {n} output rows")
    if weight.shape[0] != d or out.shape[1] != d or not x.is_contiguous() or not out.is_contiguous():
        raise KernelError(f"rmsnorm: width mismatch or strided operands (x {tuple(x.shape)}, w {tuple(weight.shape)}, out {tuple(out.shape)})")
    _check(_lib("rmsnorm").dlgo_rmsnorm(_ptr(x), _ptr(rows), _ptr(weight), _ptr(out), dtype_code(out.dtype), n, d,
                                        ctypes.c_float(eps), _stream()))
    return out


def bias_add(y: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """y[t, n] += bias[n]; y rows in float32 or bfloat16 (row stride free), bias float32."""
    _need(y, "rows", dims=2)
    _need(bias, "bias", torch.float32, 1)
    if bias.shape[0] != y.shape[1] or not bias.is_contiguous():
        raise KernelError(f"bias_add: bias {tuple(bias.shape)} does not fit rows {tuple(y.shape)}")
    _check(_lib("rowwise").dlgo_bias_add(_ptr(y), dtype_code(y.dtype), y.shape[0], y.shape[1], _rows(y, "rows"), _ptr(bias), _stream()))
    return y


def head_rmsnorm(x: torch.Tensor, first_col: int, n_heads: int, head_dim: int, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """Each of n_heads heads of head_dim consecutive elements, from column first_col on, of every row of x is RMS-normalised
    in place over its own elements and multiplied by weight [head_dim] (float32)."""
    _need(x, "rows", dims=2)
    _need(weight, "head norm weight", torch.float32, 1)
    if weight.shape[0] != head_dim or not weight.is_contiguous() or first_col < 0 or first_col + n_heads * head_dim > x.shape[1]:
        raise KernelError(f"head_rmsnorm: {n_heads} heads of {head_dim} from column {first_col} and weight {tuple(weight.shape)} do not fit rows {tuple(x.shape)}")
    _check(_lib("rowwise").dlgo_head_rmsnorm(_ptr(x), dtype_code(x.dtype), x.shape[0], _rows(x, "rows"), first_col, n_heads, head_dim,
                                             _ptr(weight), ctypes.c_float(eps), _stream()))
    return x


_cus: dict = {}


def compute_units(device=None) -> int:
    """Compute units of the device (256 on an MI355X): what the rules below count blocks against."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    if index not in _cus:
        _cus[index] = torch.cuda.get_device_properties(index).multi_processor_count
    return _cus[index]


def stream_plan(weight: torch.Tensor, t: int):
    """(waves a block, kilobytes of a row a wave takes in turn, groups of 16 weight rows a block works through) of the
    streamed products for this weight and t rows of x, or None if they do not take it."""
    if weight.dim() != 2 or weight.stride(1) != 1 or not (1 <= t <= 16):
        return None
    lib = _lib("gemm_rows", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    lib.dlgo_gemm_rows_stream_plan.restype = ctypes.c_int
    waves, turns, groups = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    ok = lib.dlgo_gemm_rows_stream_plan(dtype_code(weight.dtype), weight.shape[0], t, weight.shape[1], weight.stride(0),
                                        ctypes.byref(waves), ctypes.byref(turns), ctypes.byref(groups))
    return (waves.value, turns.value, groups.value) if ok else None


def _streams_rows(weight: torch.Tensor, t: int, kind: int, has_scratch: bool, splits: int) -> bool:
    """Whether a product of t rows with this weight goes to the kernels that stream W against a few rows of x (else to
    the tiled ones).  The rules count bytes, blocks and rows, not the sizes of a model:

      row_bytes  what a block reads of one weight row; in 128-byte pieces the tiles can load it straight into LDS, and
                 from 32 pieces (4 KB) on they can share k out over blocks, given scratch (`can_split`);
      blocks16   blocks of the streamed kernels (16 weight rows each), tiles64 those of the small tiles (64 rows each),
                 both against the device's compute units.

    Up to 16 rows stream, except: (a) so few blocks that compute units stay idle and rows long enough to share out
    (the split tiles use every unit); (b) rows that a wave takes in several turns, from 8 rows of x on, where k can be
    shared out (the streamed kernel for such rows has one group of weight rows a block, and every block reads all of
    x again: with 10 KB rows and 8 rows of x the split tiles are 10 to 30% faster, with 40 KB rows also for one row);
    (c) a matrix with 16 and more blocks a unit (a vocabulary), which streams only with up to 8 rows and a wave per
    kilobyte of a row, or when the tiles cannot load its rows.  17 to 64 rows go to the kernel that reads W into
    registers only where the tiles are few and cannot split."""
    n, k = weight.shape
    es = weight.element_size()
    row_bytes = k * es
    pieces = row_bytes // 128 if row_bytes % 128 == 0 else 0
    can_split = has_scratch and splits != 1 and pieces >= 32
    if kind != GEMM_AUTO or splits > 1:
        return kind in (GEMM_STREAM, 5, 6, 7, 8, 9, 10, 11, 15, 16, 17, 18, 19)
    cus = compute_units(weight.device)
    blocks16, tiles64 = (n + 15) // 16, (n + 63) // 64
    very_wide = blocks16 >= 16 * cus
    if t <= GEMM_FEW_ROWS_WIDE:
        plan = stream_plan(weight, t)
        waves, turns, groups = plan if plan is not None else (0, 1, 1)
        if very_wide:                                                                       # (c)
            return pieces == 0 or (t <= 8 and plan is not None and turns == 1 and waves not in (5, 7))
        if can_split and blocks16 <= cus and pieces >= 64:                                  # (a)
            return False
        if can_split and plan is not None and turns > 1 and (t >= 8 or pieces >= 256):      # (b)
            return False
        return True
    if t <= GEMM_FEW_ROWS:
        return blocks16 < 4 * cus and not (can_split and tiles64 <= cus // 2 and (pieces >= 48 or t >= 24)) and (t <= 40 or pieces == 0)
    return False


def gemm_streams(weight: torch.Tensor, rows: int, has_scratch: bool = True) -> bool:
    """Which family gemm() gives a product of `rows` rows of x with this weight when the choice is its own: the kernels
    that stream W against a few rows (True) or the tiled ones (False).  The rules are _streams_rows'."""
    return _streams_rows(weight, rows, GEMM_AUTO, has_scratch, 0)


def gemm_accum_then_norm(weight: torch.Tensor, x: torch.Tensor, residual: torch.Tensor, scratch: Optional[torch.Tensor],
                         norm_weight: torch.Tensor, eps: float, normed: torch.Tensor) -> bool:
    """residual += x @ weight.T and, beside it, normed = rmsnorm(residual) * norm_weight of the new rows, if this
    product is one whose inner size gemm() would share out over blocks (then the sum of the runs gives the norm for
    nothing).  Returns False, having done nothing, if it is not: the caller then runs gemm() and the norm."""
    _need(weight, "gemm weight", dims=2)
    _need(x, "gemm input", weight.dtype, 2)
    n, k = weight.shape
    t = x.shape[0]
    if scratch is None or t == 0 or n % 4 or n > 8192 or _streams_rows(weight, t, GEMM_AUTO, True, 0):
        return False
    _need(scratch, "gemm scratch", torch.float32, 1)
    lib = _lib("gemm", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    ldw, ldx = _rows(weight, "gemm weight"), _rows(x, "gemm input")
    splits = lib.dlgo_gemm_auto_splits(dtype_code(weight.dtype), n, t, k, ldw, ldx, ctypes.c_longlong(scratch.numel()))
    if splits <= 1:
        return False
    _need(residual, "residual rows", torch.float32, 2)
    _need(norm_weight, "norm weight", torch.float32, 1)
    _need(normed, "normed rows", weight.dtype, 2)
    if x.shape[1] != k or tuple(residual.shape) != (t, n) or tuple(normed.shape) != (t, n) or norm_weight.shape[0] != n:
        raise KernelError(f"gemm_accum_then_norm: x {tuple(x.shape)}, residual {tuple(residual.shape)}, normed {tuple(normed.shape)} "
                          f"and norm weight {tuple(norm_weight.shape)} do not fit weight {tuple(weight.shape)}")
    _check(lib.dlgo_gemm_accum_norm(_ptr(weight), _ptr(x), _ptr(residual), dtype_code(weight.dtype), n, t, k, ldw, ldx,
                                    _rows(residual, "residual rows"), splits, _ptr(scratch), ctypes.c_longlong(scratch.numel()),
                                    _ptr(norm_weight), ctypes.c_float(eps), _ptr(normed), _rows(normed, "normed rows"), _stream()))
    return True


class UnsummedRows:
    """The rows x @ weight.T as gemm_runs leaves them: `runs` float32 planes [T, N] one after the other in `scratch`, each
    the sum over one run of k; the rows themselves are the planes added in order.  A kernel that reads the rows once
    can do that sum as it reads (rope_kv does) and save the pass that would write them out."""
    __slots__ = ("scratch", "runs", "rows", "cols")

    def __init__(self, scratch, runs, rows, cols):
        self.scratch, self.runs, self.rows, self.cols = scratch, runs, rows, cols


def gemm_runs(weight: torch.Tensor, x: torch.Tensor, scratch: Optional[torch.Tensor]) -> Optional[UnsummedRows]:
    """x @ weight.T left as unsummed runs of k in `scratch`, if this product is one whose inner size gemm() would share
    out over blocks; None, having done nothing, if it is not (the caller then runs gemm())."""
    _need(weight, "gemm weight", dims=2)
    _need(x, "gemm input", weight.dtype, 2)
    n, k = weight.shape
    t = x.shape[0]
    if scratch is None or t == 0 or n % 4 or _streams_rows(weight, t, GEMM_AUTO, True, 0):
        return None
    _need(scratch, "gemm scratch", torch.float32, 1)
    if x.shape[1] != k:
        raise KernelError(f"gemm_runs: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    lib = _lib("gemm", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    ldw, ldx = _rows(weight, "gemm weight"), _rows(x, "gemm input")
    splits = lib.dlgo_gemm_auto_splits(dtype_code(weight.dtype), n, t, k, ldw, ldx, ctypes.c_longlong(scratch.numel()))
    if splits <= 1:
        return None
    runs = ctypes.c_int(0)
    _check(lib.dlgo_gemm_parts(_ptr(weight), _ptr(x), dtype_code(weight.dtype), n, t, k, ldw, ldx, splits, _ptr(scratch),
                               ctypes.c_longlong(scratch.numel()), ctypes.byref(runs), _stream()))
    return UnsummedRows(scratch, runs.value, t, n)


def gemm(weight: torch.Tensor, x: torch.Tensor, out: torch.Tensor, epilogue: int = EPI_STORE,
         kind: int = GEMM_AUTO, scratch: Optional[torch.Tensor] = None, splits: int = 0) -> torch.Tensor:
    """out (epilogue)= x @ weight.T with weight [N, K], x [T, K].

    scratch: float32 of GEMM_SPLIT_FLOATS elements (optional).  With it, a product of few rows with a long inner
    size may share k out over several blocks (splits: 0 = let the kernel choose, 1 = never, n = n runs of k).

    EPI_STORE: out [T, N] in the run dtype.  EPI_ACCUM_F32: out float32 [T, N], added to.
    EPI_SWIGLU: weight rows are (gate_0, up_0, gate_1, up_1, ...), out [T, N/2] = silu(gate) * up.
    EPI_STORE_F32: out float32 [T, N].
    """
    _need(weight, "gemm weight", dims=2)
    _need(x, "gemm input", weight.dtype, 2)
    n, k = weight.shape
    t = x.shape[0]
    if x.shape[1] != k:
        raise KernelError(f"gemm: input width {x.shape[1]} does not match weight {tuple(weight.shape)}")
    want_dtype = torch.float32 if epilogue in (EPI_ACCUM_F32, EPI_STORE_F32) else weight.dtype
    _need(out, "gemm output", want_dtype, 2)
    cols = n // 2 if epilogue == EPI_SWIGLU else n
    if tuple(out.shape) != (t, cols):
        raise KernelError(f"gemm: output {tuple(out.shape)}, expected {(t, cols)}")
    if scratch is not None:
        _need(scratch, "gemm scratch", torch.float32, 1)
    elif splits > 1:
        raise KernelError("gemm: a split product needs scratch")
    rows_kernel = _streams_rows(weight, t, kind, scratch is not None, splits)
    args = (_ptr(weight), _ptr(x), _ptr(out), dtype_code(weight.dtype), n, t, k, _rows(weight, "gemm weight"),
            _rows(x, "gemm input"), _rows(out, "gemm output"), epilogue)
    if rows_kernel:
        fn = _lib("gemm_rows", (("DLGO_ELEM", dtype_code(weight.dtype)),)).dlgo_gemm_rows
        _check(fn(*args, 0 if kind in (GEMM_AUTO, GEMM_ROWS16) else kind, _stream()))
    else:
        fn = _lib("gemm", (("DLGO_ELEM", dtype_code(weight.dtype)),)).dlgo_gemm
        _check(fn(*args, kind, splits, _ptr(scratch), ctypes.c_longlong(scratch.numel() if scratch is not None else 0), _stream()))
    return out


FUSED_NORM_ROWS = 64   # most rows of the residual stream that gemm_rmsnorm takes
FUSED_NORM_PAYS = 16   # up to this many rows the fused norm is faster than a norm kernel and a plain product


def fused_norm_pays(weight: torch.Tensor, rows: int) -> bool:
    """Whether gemm_rmsnorm beats a norm kernel followed by gemm for this weight and this many rows."""
    tiled = weight.shape[0] >= GEMM_VERY_WIDE and weight.shape[1] % (128 // weight.element_size()) == 0
    return rows <= FUSED_NORM_PAYS and not tiled


def gemm_rmsnorm(weight: torch.Tensor, x: torch.Tensor, norm_weight: torch.Tensor, eps: float, out: torch.Tensor,
                 epilogue: int = EPI_STORE, kind: int = GEMM_AUTO) -> torch.Tensor:
    """out (epilogue)= (rmsnorm(x) * norm_weight) @ weight.T for up to 64 rows x of the float32 residual stream,
    without writing the normed rows.  Epilogues as gemm().  kind: 0 = chosen by the shape, 10 = the weights go through
    LDS in whole 1 KB runs wherever that kernel applies (up to 16 rows, weight rows of 2 to 16 whole KB), 11 = never."""
    _need(weight, "gemm weight", dims=2)
    _need(x, "residual rows", torch.float32, 2)
    _need(norm_weight, "norm weight", torch.float32, 1)
    n, k = weight.shape
    t = x.shape[0]
    if x.shape[1] != k or norm_weight.shape[0] != k or t > FUSED_NORM_ROWS:
        raise KernelError(f"gemm_rmsnorm: rows {tuple(x.shape)} and norm weight {tuple(norm_weight.shape)} do not fit weight {tuple(weight.shape)} (at most {FUSED_NORM_ROWS} rows)")
    want_dtype = torch.float32 if epilogue in (EPI_ACCUM_F32, EPI_STORE_F32) else weight.dtype
    _need(out, "gemm output", want_dtype, 2)
    cols = n // 2 if epilogue == EPI_SWIGLU else n
    if tuple(out.shape) != (t, cols):
        raise KernelError(f"gemm_rmsnorm: output {tuple(out.shape)}, expected {(t, cols)}")
    _check(_lib("gemm_rows", (("DLGO_ELEM", dtype_code(weight.dtype)),)).dlgo_gemm_rmsnorm(_ptr(weight), _ptr(x), _ptr(norm_weight), ctypes.c_float(eps), _ptr(out),
                                          dtype_code(weight.dtype), n, t, k, _rows(weight, "gemm weight"),
                                          _rows(x, "residual rows"), _rows(out, "gemm output"), epilogue, kind, _stream()))
    return out


class UnscaledNorm:
    """What gemm_accum_leave_norm leaves of rmsnorm(residual) * norm_weight: the rows it wrote hold residual * norm_weight,
    and `parts` [T, n_parts] (float32) each row's sum of squares in n_parts shares; rmsnorm's factor of row t is
    1 / sqrt(sum(parts[t]) / width + eps).  It is a scalar per row, so a product of the rows can apply it to its sums:
    gemm_scaled does."""
    __slots__ = ("rows", "parts", "n_parts", "width", "eps")

    def __init__(self, rows, parts, n_parts, width, eps):
        self.rows, self.parts, self.n_parts, self.width, self.eps = rows, parts, n_parts, width, eps


ROLE_PLAIN, ROLE_LEAVES_NORM, ROLE_APPLIES_NORM = 0, 1, 2


def streams_few_rows(weight: torch.Tensor, rows: int, role: int = ROLE_PLAIN) -> bool:
    """Whether the streamed products take this weight with this many rows of x: up to 16 rows and weight rows of whole
    KB; as the product that leaves a norm (ROLE_LEAVES_NORM) or applies one left to it (ROLE_APPLIES_NORM) also a
    normed width that its shares of the sums of squares cover."""
    if weight.dim() != 2 or weight.stride(1) != 1 or not (1 <= rows <= 16):
        return False
    lib = _lib("gemm_rows", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    lib.dlgo_gemm_rows_streams.restype = ctypes.c_int
    return bool(lib.dlgo_gemm_rows_streams(dtype_code(weight.dtype), weight.shape[0], rows, weight.shape[1], weight.stride(0), int(role)))


def _tiles_take_norm(weight: torch.Tensor, rows: int, role: int) -> bool:
    """Whether the tiled products leave (role 1) or apply (role 2) a norm for this weight and this many rows: steps of
    many rows whose product gemm() would give to tiles that sum the whole of k."""
    if weight.dim() != 2 or weight.stride(1) != 1 or rows <= 16:
        return False
    lib = _lib("gemm", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    lib.dlgo_gemm_tile_norm_takes.restype = ctypes.c_int
    return bool(lib.dlgo_gemm_tile_norm_takes(dtype_code(weight.dtype), weight.shape[0], rows, weight.shape[1], weight.stride(0),
                                              weight.shape[1], role, ctypes.c_longlong(GEMM_SPLIT_FLOATS)))


def can_leave_unscaled(weight: torch.Tensor, rows: int) -> bool:
    """Whether gemm_accum_leave_norm takes this weight with this many rows of x (contiguous rows of x assumed)."""
    return streams_few_rows(weight, rows, ROLE_LEAVES_NORM) or _tiles_take_norm(weight, rows, 1)


def can_take_unscaled(weight: torch.Tensor, rows: int) -> bool:
    """Whether gemm_scaled takes this weight with this many rows (contiguous rows assumed)."""
    return streams_few_rows(weight, rows, ROLE_APPLIES_NORM) or _tiles_take_norm(weight, rows, 2)


def gemm_accum_leave_norm(weight: torch.Tensor, x: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                          unscaled: torch.Tensor, parts: torch.Tensor) -> UnscaledNorm:
    """residual += x @ weight.T, and of rmsnorm(residual) * norm_weight of the new rows what UnscaledNorm describes
    (unscaled: [T, N] in the run dtype; parts: float32 scratch of at least T * ceil(N / 8) elements).  For weights
    and rows that can_leave_unscaled accepts: few rows go to the streamed product, many to tiles."""
    _need(weight, "gemm weight", dims=2)
    _need(x, "gemm input", weight.dtype, 2)
    _need(residual, "residual rows", torch.float32, 2)
    _need(norm_weight, "norm weight", torch.float32, 1)
    _need(unscaled, "unscaled rows", weight.dtype, 2)
    _need(parts, "norm parts", torch.float32, 1)
    n, k = weight.shape
    t = x.shape[0]
    if x.shape[1] != k or tuple(residual.shape) != (t, n) or tuple(unscaled.shape) != (t, n) or norm_weight.shape[0] != n:
        raise KernelError(f"gemm_accum_leave_norm: x {tuple(x.shape)}, residual {tuple(residual.shape)}, unscaled {tuple(unscaled.shape)} "
                          f"and norm weight {tuple(norm_weight.shape)} do not fit weight {tuple(weight.shape)}")
    n_parts = ctypes.c_int(0)
    tiled = t > 16
    lib = _lib("gemm" if tiled else "gemm_rows", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    fn = lib.dlgo_gemm_tile_leave if tiled else lib.dlgo_gemm_rows_leave_parts
    _check(fn(_ptr(weight), _ptr(x), _ptr(residual), dtype_code(weight.dtype), n, t, k,
              _rows(weight, "gemm weight"), _rows(x, "gemm input"), _rows(residual, "residual rows"),
              _ptr(norm_weight), _ptr(unscaled), _rows(unscaled, "unscaled rows"), _ptr(parts),
              ctypes.c_longlong(parts.numel()), ctypes.byref(n_parts), _stream()))
    return UnscaledNorm(unscaled, parts, n_parts.value, n, eps)


def gemm_scaled(weight: torch.Tensor, left: UnscaledNorm, out: torch.Tensor, epilogue: int = EPI_STORE) -> torch.Tensor:
    """out (epilogue)= rmsnorm's factor of each row * (left.rows @ weight.T): the product of the normed rows that `left`
    describes.  Epilogues as gemm() for few rows, store and SwiGLU for many; for weights and rows that can_take_unscaled
    accepts."""
    _need(weight, "gemm weight", dims=2)
    x = left.rows
    _need(x, "unscaled rows", weight.dtype, 2)
    n, k = weight.shape
    t = x.shape[0]
    if x.shape[1] != k or left.width != k or left.parts.numel() < t * left.n_parts:
        raise KernelError(f"gemm_scaled: rows {tuple(x.shape)} of a norm over {left.width} with {left.n_parts} parts do not fit weight {tuple(weight.shape)}")
    want_dtype = torch.float32 if epilogue in (EPI_ACCUM_F32, EPI_STORE_F32) else weight.dtype
    _need(out, "gemm output", want_dtype, 2)
    cols = n // 2 if epilogue == EPI_SWIGLU else n
    if tuple(out.shape) != (t, cols):
        raise KernelError(f"gemm_scaled: output {tuple(out.shape)}, expected {(t, cols)}")
    tiled = t > 16
    lib = _lib("gemm" if tiled else "gemm_rows", (("DLGO_ELEM", dtype_code(weight.dtype)),))
    fn = lib.dlgo_gemm_tile_scaled if tiled else lib.dlgo_gemm_rows_scaled
    _check(fn(_ptr(weight), _ptr(x), _ptr(out), dtype_code(weight.dtype), n, t, k, _rows(weight, "gemm weight"),
              _rows(x, "unscaled rows"), _rows(out, "gemm output"), epilogue, _ptr(left.parts), left.n_parts,
              left.width, ctypes.c_float(left.eps), _stream()))
    return out


def rope_kv(qkv: torch.Tensor, n_heads: int, n_kv: int, head_dim: int, rot: int, interleaved: bool,
            cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], positions: torch.Tensor,
            tok_seq: Optional[torch.Tensor], slots: Optional[torch.Tensor], page_table: Optional[torch.Tensor],
            cache: Optional[torch.Tensor], page_stride: int, v_off: int, write_kv: bool = True,
            unsummed: Optional[UnsummedRows] = None, single_tokens: bool = False,
            seq_pages: Optional[torch.Tensor] = None) -> None:
    """Rotate the query heads of qkv [T, (H+2KV)*hd] in place; rotate the key heads and copy the value heads
    into the cache page of each token (cache: the first element of this layer's pages).  unsummed: the rows are not
    in qkv yet but in the runs that gemm_runs left (see rope_takes_unsummed); the rotated queries are written to qkv.
    single_tokens: every row is a sequence of its own (a hint for how the transposed values are best stored; the
    result is the same).  seq_pages: for such a step, the sequences' page-table rows in the order of the rows
    ([>= T, the table's width], row i = page_table[slots[tok_seq[i]]]); the kernel then reads a row's page from there
    without going through its sequence and slot."""
    _need(qkv, "qkv rows", dims=2)
    _need(positions, "positions", torch.int32, 1)
    t = qkv.shape[0]
    if positions.shape[0] != t:
        raise KernelError("rope_kv: one position per row")
    table_rows = 0
    if cos is not None:
        _need(cos, "cos table", torch.float32, 2)
        _need(sin, "sin table", torch.float32, 2)
        if cos.shape != sin.shape or cos.shape[1] != rot // 2 or not cos.is_contiguous() or not sin.is_contiguous():
            raise KernelError(f"rope_kv: tables {tuple(cos.shape)} do not fit a rotated width of {rot}")
        table_rows = cos.shape[0]
    max_pages = 0
    if write_kv:
        _need(tok_seq, "token->sequence", torch.int32, 1)
        _need(slots, "slots", torch.int32, 1)
        _need(page_table, "page table", torch.int32, 2)
        _need(cache, "cache", qkv.dtype)
        if tok_seq.shape[0] != t or not page_table.is_contiguous():
            raise KernelError("rope_kv: one sequence index per row and a contiguous page table")
        max_pages = page_table.shape[1]
    by_row = write_kv and seq_pages is not None
    if by_row:
        _need(seq_pages, "pages by sequence", torch.int32, 2)
        if not single_tokens or seq_pages.shape[0] < t or seq_pages.shape[1] != max_pages or not seq_pages.is_contiguous():
            raise KernelError(f"rope_kv: pages by sequence {tuple(seq_pages.shape)} do not fit {t} single-token rows "
                              f"and a table {max_pages} wide")
        page_table = seq_pages
    part = (_ptr(None), 0, ctypes.c_longlong(0), 0)
    if unsummed is not None:
        if unsummed.rows != t or unsummed.cols < (n_heads + (2 * n_kv if write_kv else 0)) * head_dim:
            raise KernelError(f"rope_kv: unsummed rows [{unsummed.rows}, {unsummed.cols}] do not fit {t} rows of qkv")
        part = (_ptr(unsummed.scratch), unsummed.runs, ctypes.c_longlong(unsummed.rows * unsummed.cols), unsummed.cols)
    _check(_lib("rope_kv").dlgo_rope_kv(_ptr(qkv), dtype_code(qkv.dtype), t, _rows(qkv, "qkv rows"), n_heads, n_kv, head_dim,
                                        rot, int(interleaved), _ptr(cos), _ptr(sin), table_rows, _ptr(positions),
                                        _ptr(tok_seq), _ptr(slots), _ptr(page_table), max_pages, _ptr(cache),
                                        ctypes.c_longlong(page_stride), ctypes.c_longlong(v_off), int(write_kv), *part,
                                        int(single_tokens), int(by_row), _stream()))


def rope_takes_unsummed(dtype: torch.dtype, head_dim: int, rot: int) -> bool:
    """Whether rope_kv can read rows that gemm_runs left unsummed: it does so in whole 16-byte pieces."""
    epc = 4 if dtype == torch.float32 else 8
    return head_dim % epc == 0 and rot % (2 * epc) == 0


def attention_rows(q: torch.Tensor, out: torch.Tensor, n_heads: int, n_kv: int, head_dim: int,
                   positions: torch.Tensor, tok_seq: torch.Tensor, slots: torch.Tensor, page_table: torch.Tensor,
                   cache: torch.Tensor, page_stride: int, v_off: int, window: int = 0,
                   scale: Optional[float] = None, n_splits: int = 1, scratch=None) -> torch.Tensor:
    """One wave per (row, head): the general kernel, every dtype, every step shape.  n_splits > 1 deals each row's
    pages to that many waves, whose partial results (in scratch(n): float32, n elements) a second kernel merges."""
    _need(q, "query rows", dims=2)
    _need(out, "attention output", q.dtype, 2)
    for name, v in (("positions", positions), ("token->sequence", tok_seq), ("slots", slots)):
        _need(v, name, torch.int32, 1)
    _need(page_table, "page table", torch.int32, 2)
    _need(cache, "cache", q.dtype)
    t = q.shape[0]
    if out.shape[0] != t or positions.shape[0] != t or tok_seq.shape[0] != t or not page_table.is_contiguous():
        raise KernelError("attention: one position, sequence index and output row per query row")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    lib = _lib("attention", (("HEAD_DIM", head_dim),))
    part = None
    if n_splits > 1:
        need = t * n_heads * n_splits * (head_dim + 4)
        part = scratch(need) if scratch is not None else torch.empty(need, dtype=torch.float32, device=q.device)
        _need(part, "attention scratch", torch.float32, 1)
    _check(lib.dlgo_attention_rows(_ptr(q), _rows(q, "query rows"), _ptr(out), _rows(out, "attention output"),
                                   dtype_code(q.dtype), t, n_heads, n_kv, head_dim, _ptr(positions), _ptr(tok_seq),
                                   _ptr(slots), _ptr(page_table), page_table.shape[1], _ptr(cache),
                                   ctypes.c_longlong(page_stride), ctypes.c_longlong(v_off), int(window),
                                   ctypes.c_float(scale), int(n_splits), _ptr(part),
                                   ctypes.c_longlong(part.numel() if part is not None else 0), _stream()))
    return out


def attention_fuses_rotation(dtype: torch.dtype, head_dim: int, group: int, max_q_len: int, rot_width: int,
                             n_seq: int = 1, n_kv: int = 8) -> bool:
    """True if attention() should rotate the queries and take in the new keys and values itself for such a step:
    one row per sequence, bfloat16, a rotated width that is a multiple of 16 or no rotation at all; at most one
    (sequence, kv head) pair for every compute unit, so that a kernel launch costs more than the rotation repeated in
    every wave (with 8 kv heads on 256 units: up to 32 sequences; measured at 64: 62 against 9 + 52 us), and no more
    than 32 sequences whatever the heads (the largest step the fused variant is tested with); and heads small enough
    that eight waves of a block each keep a page (keys and values of 64 tokens) in 128 KB of LDS (at a head size of 128
    the kernel of its own is faster)."""
    page_bytes = 2 * PAGE * head_dim * 2
    return (dtype == torch.bfloat16 and 8 * page_bytes <= 128 * 1024 and group <= 128 and max_q_len == 1 and rot_width % 16 == 0
            and n_seq * n_kv * ((group + 15) // 16) <= compute_units() and n_seq <= 32)


def attention(q: torch.Tensor, out: torch.Tensor, n_heads: int, n_kv: int, head_dim: int, positions: torch.Tensor,
              tok_seq: torch.Tensor, slots: torch.Tensor, page_table: torch.Tensor, cache: torch.Tensor, page_stride: int,
              v_off: int, q_lens: Sequence[int], start_pos: Sequence[int], window: int = 0,
              scale: Optional[float] = None, cu_q: Optional[torch.Tensor] = None,
              start_pos_dev: Optional[torch.Tensor] = None, scratch=None,
              max_pages_used: Optional[int] = None, kernel: str = "auto", rotation=None, new_kv: bool = False,
              split_variant: int = 0, seq_pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a step's query rows over the cache, with the kernel chosen by the step's shape and dtype.

    q_lens, start_pos: per sequence, on the host (rows of the step, and the length before it).  cu_q and
    start_pos_dev are the same numbers on the device (built here if not given).  scratch(n) returns a
    float32 buffer of at least n elements (partials of long sequences in decode).  max_pages_used bounds the pages any sequence
    of the step holds (default: from q_lens and start_pos; a captured step passes the context's bound).
    kernel: "auto", "rows", "tiled" (prefill) or "split" (decode).  All kernels compute the same thing.
    rotation = (cos, sin, width, interleaved) and new_kv: only where attention_fuses_rotation() says so; then q
    holds the step's unrotated [q | k | v] rows, which the kernel rotates, and with new_kv it also takes each
    token's own key and value from its row and writes them to the cache (what rope_kv() does otherwise).
    split_variant (bfloat16 split kernel): 0 or 2 = a page goes through LDS in whole 1 KB runs, 1 = it is read straight
    into the operands' registers.
    seq_pages (steps of single tokens): the sequences' rows of page_table in the order of the step, [>= n_seq, the table's
    width]: row i holds what row slots[i] of page_table holds.  The bfloat16 split kernel then finds a sequence's pages
    without waiting for its slot, and asks for its first page's number together with the position.
    """
    n_seq = len(q_lens)
    max_q = int(max(q_lens)) if n_seq else 0
    group = n_heads // n_kv
    fast_ok = q.dtype == torch.bfloat16 and head_dim <= 256 and group <= 128
    tiled_f32 = q.dtype == torch.float32 and head_dim <= 128 and group <= 128       # prompts in float32: a kernel of their own
    split_f32 = q.dtype == torch.float32 and head_dim <= 128 and group <= 128      # and so have steps of single tokens
    if kernel == "auto":
        if fast_ok:
            kernel = "split" if max_q == 1 else "tiled"
        else:
            kernel = "split" if split_f32 and max_q == 1 else ("tiled" if tiled_f32 and max_q > 1 else "rows")
    if (rotation is not None or new_kv) and not (kernel == "split" and fast_ok and max_q == 1):
        raise KernelError("attention: only the bfloat16 split kernel rotates and stores by itself")
    if kernel == "rows" or n_seq == 0:
        # a few rows with long histories (a decode step off the fast kernels): each row's pages go to several waves
        n_splits = 1
        if max_q == 1 and n_seq > 0:
            pages = max_pages_used if max_pages_used is not None else (int(max(start_pos)) + PAGE) // PAGE
            n_splits = max(1, min(pages // 2, 2048 // max(1, n_seq * n_heads)))
        return attention_rows(q, out, n_heads, n_kv, head_dim, positions, tok_seq, slots, page_table, cache, page_stride,
                              v_off, window, scale, n_splits, scratch)
    if not fast_ok and not (tiled_f32 and kernel == "tiled") and not (split_f32 and kernel == "split"):
        raise KernelError("attention: the tiled and split kernels take bfloat16, head sizes up to 256 and up to 128 heads per kv head "
                          "(and float32 with head sizes up to 128)")
    _need(q, "query rows", q.dtype, 2)
    _need(out, "attention output", q.dtype, 2)
    _need(slots, "slots", torch.int32, 1)
    _need(page_table, "page table", torch.int32, 2)
    _need(cache, "cache", q.dtype)
    if slots.shape[0] != n_seq or out.shape[0] != q.shape[0] or q.shape[0] != int(sum(q_lens)) or not page_table.is_contiguous():
        raise KernelError("attention: rows, sequences and slots do not match")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    lib = _lib("attention", (("HEAD_DIM", head_dim),))
    if kernel == "split":
        if max_q != 1:
            raise KernelError("attention: the split kernel takes one row per sequence")
        _need(positions, "positions", torch.int32, 1)
        if positions.shape[0] != n_seq:
            raise KernelError("attention: one position per sequence")
        max_pages = page_table.shape[1]
        if max_pages_used is None:
            max_pages_used = (int(max(start_pos)) + 1 + PAGE - 1) // PAGE
        max_pages_used = max(1, min(max_pages_used, max_pages))
        cos = sin = None
        rot_width, interleaved = 0, False
        if rotation is not None:
            cos, sin, rot_width, interleaved = rotation
            _need(cos, "cos table", torch.float32, 2)
            _need(sin, "sin table", torch.float32, 2)
            if cos.shape != sin.shape or cos.shape[1] != rot_width // 2 or not cos.is_contiguous() or not sin.is_contiguous():
                raise KernelError(f"attention: tables {tuple(cos.shape)} do not fit a rotated width of {rot_width}")
        if seq_pages is not None:
            _need(seq_pages, "pages by sequence", torch.int32, 2)
            if seq_pages.shape[0] < n_seq or seq_pages.shape[1] != max_pages or not seq_pages.is_contiguous():
                raise KernelError(f"attention: pages by sequence {tuple(seq_pages.shape)} do not fit {n_seq} sequences and a table {max_pages} wide")
        lib.dlgo_attention_decode_splits.restype = ctypes.c_int
        variant = split_variant if q.dtype == torch.bfloat16 else 1
        n_splits = lib.dlgo_attention_decode_splits(n_seq, n_heads, n_kv, max_pages_used, int(rotation is not None or new_kv), variant)
        part = None
        if n_splits > 1:
            need = n_seq * n_heads * n_splits * (head_dim + 4)
            part = scratch(need) if scratch is not None else torch.empty(need, dtype=torch.float32, device=q.device)
            _need(part, "attention scratch", torch.float32, 1)
        if q.dtype == torch.float32:
            _check(lib.dlgo_attention_decode_f32(_ptr(q), _rows(q, "query rows"), _ptr(out), _rows(out, "attention output"), _ptr(part),
                                                 ctypes.c_longlong(part.numel() if part is not None else 0), n_seq, n_heads, n_kv,
                                                 head_dim, _ptr(positions), _ptr(slots), _ptr(page_table), max_pages, max_pages_used,
                                                 _ptr(cache), ctypes.c_longlong(page_stride), ctypes.c_longlong(v_off), int(window),
                                                 ctypes.c_float(scale), _stream()))
            return out
        _check(lib.dlgo_attention_decode(_ptr(q), _rows(q, "query rows"), _ptr(out), _rows(out, "attention output"), _ptr(part),
                                         ctypes.c_longlong(part.numel() if part is not None else 0), n_seq, n_heads, n_kv,
                                         head_dim, _ptr(positions), _ptr(slots), _ptr(page_table), max_pages, max_pages_used,
                                         _ptr(cache), ctypes.c_longlong(page_stride), ctypes.c_longlong(v_off), int(window),
                                         ctypes.c_float(scale), _ptr(cos), _ptr(sin), cos.shape[0] if cos is not None else 0,
                                         int(rot_width), int(interleaved), int(new_kv), int(variant), _ptr(seq_pages), _stream()))
        return out
    if kernel != "tiled":
        raise KernelError(f"attention: unknown kernel {kernel!r}")
    if cu_q is None:
        import numpy as np
        cu = np.concatenate([[0], np.cumsum(np.asarray(q_lens, dtype=np.int64))]).astype(np.int32)
        cu_q = torch.from_numpy(cu).to(q.device)
        start_pos_dev = torch.as_tensor(list(start_pos), dtype=torch.int32).to(q.device)
    _need(cu_q, "row offsets", torch.int32, 1)
    _need(start_pos_dev, "start positions", torch.int32, 1)
    if cu_q.shape[0] != n_seq + 1 or start_pos_dev.shape[0] != n_seq:
        raise KernelError("attention: row offsets and start positions do not match the sequences")
    entry = lib.dlgo_attention_prefill_f32 if q.dtype == torch.float32 else lib.dlgo_attention_prefill
    _check(entry(_ptr(q), _rows(q, "query rows"), _ptr(out), _rows(out, "attention output"), n_seq, max_q,
                                      n_heads, n_kv, head_dim, _ptr(cu_q), _ptr(start_pos_dev), _ptr(slots), _ptr(page_table),
                                      page_table.shape[1], _ptr(cache), ctypes.c_longlong(page_stride),
                                      ctypes.c_longlong(v_off), int(window), ctypes.c_float(scale), _stream()))
    return out


Q8_MAX_HEAD_DIM = 256      # head sizes of the 8-bit cache: multiples of 16 up to this one


def q8_page_bytes(n_kv: int, head_dim: int) -> int:
    """Bytes of one layer's part of a page of the 8-bit cache: for each kv head 64 tokens' keys and values in a byte an
    element, and a byte for the power of two of each token's key and value (csrc/q8_page.h)."""
    return n_kv * 2 * PAGE * (head_dim + 1)


def _q8_cache(name: str, cache: torch.Tensor, page_stride: int, n_kv: int, head_dim: int) -> int:
    """How many whole pages a cache tensor holds (the kernels touch no page beyond)."""
    if not isinstance(cache, torch.Tensor) or cache.dtype is not torch.uint8 or cache.dim() != 1 or not cache.is_cuda:
        _need(cache, f"{name}: cache", torch.uint8, 1)
    if head_dim % 16 or not 16 <= head_dim <= Q8_MAX_HEAD_DIM:
        raise KernelError(f"{name}: the 8-bit cache takes head sizes in steps of 16, up to {Q8_MAX_HEAD_DIM}, not {head_dim}")
    page, size = q8_page_bytes(n_kv, head_dim), cache.numel()
    if page_stride < page or size < page or not cache.is_contiguous():
        raise KernelError(f"{name}: a cache of {size} bytes with pages {page_stride} bytes apart does not hold pages of {page} bytes")
    return min((size - page) // page_stride + 1, 2 ** 31 - 1)


def _same_device(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """Everything on one device, and that device the current one: the launches go to its current stream."""
    for t in others:
        if t is not None and t.device != first.device:
            raise KernelError(f"{name}: tensors on {first.device} and {t.device}")
    if first.device.index != torch.cuda.current_device():
        raise KernelError(f"{name}: tensors on {first.device}, the current device is cuda:{torch.cuda.current_device()}")


_BF16, _F32, _I32, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def _given_scratch(name: str, t: torch.Tensor, dtype: torch.dtype, beside: torch.Tensor) -> torch.Tensor:
    """A caller's scratch buffer: its elements lie in a row in memory (the kernels count on as many as it has), beside the others."""
    _need(t, f"{name}: scratch", dtype, 1)
    if not t.is_contiguous() or t.device != beside.device:
        raise KernelError(f"{name}: scratch must lie in a row in memory on {beside.device} (strides {t.stride()}, {t.device})")
    return t


def _current_device() -> int:
    return _raw_device() if _raw_device is not None else torch.cuda.current_device()


def _is_vector(t: torch.Tensor, n: int, dev: int, dtype: torch.dtype = _I32) -> bool:
    """n elements of dtype in a row in memory, on device `dev`."""
    return t.dtype is dtype and t.numel() == n and t.get_device() == dev and t.is_contiguous()


def _rope_kv_q8_check(qkv, q_out, n_heads, n_kv, head_dim, rot, cos, sin, positions, tok_seq, slots, page_table, cache, write_kv):
    """What rope_kv_q8() needs of its arguments, one after the other; returns (rows of the rotation tables, rows and
    width of the page table, sequences)."""
    _need(qkv, "rope_kv_q8: qkv rows", torch.bfloat16, 2)
    _need(q_out, "rope_kv_q8: query rows", torch.bfloat16, 2)
    _need(positions, "rope_kv_q8: positions", torch.int32, 1)
    t = qkv.shape[0]
    if head_dim % 16 or not 16 <= head_dim <= Q8_MAX_HEAD_DIM:
        raise KernelError(f"rope_kv_q8: the 8-bit cache takes head sizes in steps of 16, up to {Q8_MAX_HEAD_DIM}, not {head_dim}")
    if n_heads < 1 or n_kv < 0 or (write_kv and n_kv < 1):
        raise KernelError(f"rope_kv_q8: {n_heads} query and {n_kv} kv heads")
    if positions.shape[0] != t or not positions.is_contiguous():
        raise KernelError("rope_kv_q8: one position per row, in a row in memory")
    if qkv.shape[1] < (n_heads + (2 * n_kv if write_kv else 0)) * head_dim or q_out.shape[0] != t or q_out.shape[1] != n_heads * head_dim:
        raise KernelError(f"rope_kv_q8: rows {tuple(qkv.shape)} and query rows {tuple(q_out.shape)} do not fit {n_heads} query and {n_kv} kv heads of {head_dim}")
    table_rows = 0
    if (cos is None) != (sin is None):
        raise KernelError("rope_kv_q8: cos and sin tables come together")
    if cos is not None:
        _need(cos, "rope_kv_q8: cos table", torch.float32, 2)
        _need(sin, "rope_kv_q8: sin table", torch.float32, 2)
        if cos.shape != sin.shape or cos.shape[1] != rot // 2 or not cos.is_contiguous() or not sin.is_contiguous():
            raise KernelError(f"rope_kv_q8: tables {tuple(cos.shape)} do not fit a rotated width of {rot}")
        table_rows = cos.shape[0]
    max_pages = n_slots = n_seq = 0
    if write_kv:
        for what, v, dims in (("token->sequence", tok_seq, 1), ("slots", slots, 1), ("page table", page_table, 2)):
            _need(v, f"rope_kv_q8: {what}", torch.int32, dims)
            if not v.is_contiguous():
                raise KernelError(f"rope_kv_q8: {what} must be contiguous")
        if tok_seq.shape[0] != t:
            raise KernelError("rope_kv_q8: one sequence index per row")
        _need(cache, "rope_kv_q8: cache", torch.uint8, 1)
        n_slots, max_pages = page_table.shape
        n_seq = slots.shape[0]
    _same_device("rope_kv_q8", qkv, q_out, positions, cos, sin, *((tok_seq, slots, page_table, cache) if write_kv else ()))
    return table_rows, n_slots, max_pages, n_seq


def rope_kv_q8(qkv: torch.Tensor, q_out: torch.Tensor, n_heads: int, n_kv: int, head_dim: int, rot: int, interleaved: bool,
               cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], positions: torch.Tensor,
               tok_seq: Optional[torch.Tensor], slots: Optional[torch.Tensor], page_table: Optional[torch.Tensor],
               cache: Optional[torch.Tensor], page_stride: int, write_kv: bool = True,
               unsummed: Optional[UnsummedRows] = None) -> None:
    """rope_kv() for the 8-bit cache: the query heads of qkv [T, (H+2KV)*hd] (bfloat16) rotated into q_out [T, H*hd], which
    may be their own place in qkv; the key heads rotated and, with the values, stored in 8 bits in the page of each token
    (cache: uint8, from the first byte of this layer's part of page 0 on; page_stride in bytes).  positions [T], tok_seq
    [T] (each row's index into slots) and slots are int32.  A token's key (value) of a head is stored as e4m3 numbers times the least power of
    two (from 2^-126 on) that brings its largest magnitude within 448; each element is rounded once, from float32.  A token whose key
    or value is not finite is marked as a whole, and every row that sees it becomes NaN in that kv head's queries' results.
    Rows whose position has no page (a hole in the table, a page the cache does not hold) store nothing.  Positions must
    lie inside the rotation tables, and no two rows may be the same token.  write_kv=False: queries only.  unsummed: as in
    rope_kv() (the sums are not rounded before they are rotated and stored)."""
    # the usual call is told by one look at each tensor; any other goes through the checks that can say what is wrong
    n_pages = max_pages = n_slots = n_seq = 0
    try:
        dev = qkv.get_device()
        t, width = qkv.shape
        table_rows, half = cos.shape
        plain = (dev >= 0 and dev == _current_device() and n_heads > 0 and n_kv > 0 and head_dim > 0 and qkv.dtype is _BF16 and q_out.dtype is _BF16
                 and q_out.shape == (t, n_heads * head_dim) and q_out.get_device() == dev
                 and width >= (n_heads + (2 * n_kv if write_kv else 0)) * head_dim and _is_vector(positions, t, dev)
                 and half * 2 == rot and sin.shape == cos.shape and _is_vector(cos, table_rows * half, dev, _F32) and _is_vector(sin, table_rows * half, dev, _F32))
        if plain and write_kv:
            n_slots, max_pages = page_table.shape
            n_seq = slots.numel()
            plain = (_is_vector(tok_seq, t, dev) and _is_vector(slots, n_seq, dev) and _is_vector(page_table, n_slots * max_pages, dev)
                     and cache.get_device() == dev)
    except (AttributeError, TypeError, ValueError):        # something that is no tensor, or has other dimensions
        plain = False
    if not plain:
        table_rows, n_slots, max_pages, n_seq = _rope_kv_q8_check(qkv, q_out, n_heads, n_kv, head_dim, rot, cos, sin, positions, tok_seq,
                                                                  slots, page_table, cache, write_kv)
        t = qkv.shape[0]
    if write_kv:
        n_pages = _q8_cache("rope_kv_q8", cache, page_stride, n_kv, head_dim)
    if t == 0:
        return
    part = (_ptr(None), 0, ctypes.c_longlong(0), 0)
    if unsummed is not None:
        if unsummed.rows != t or unsummed.cols < (n_heads + (2 * n_kv if write_kv else 0)) * head_dim or unsummed.scratch.get_device() != qkv.get_device():
            raise KernelError(f"rope_kv_q8: unsummed rows [{unsummed.rows}, {unsummed.cols}] do not fit {t} rows of qkv")
        part = (_ptr(unsummed.scratch), unsummed.runs, ctypes.c_longlong(unsummed.rows * unsummed.cols), unsummed.cols)
    _check(_lib("kv_q8").dlgo_rope_kv_q8(_ptr(qkv), _rows32(qkv, "rope_kv_q8: qkv rows"), _ptr(q_out), _rows32(q_out, "rope_kv_q8: query rows"),
                                         t, n_heads, n_kv, head_dim, rot, int(interleaved), _ptr(cos), _ptr(sin), table_rows,
                                         _ptr(positions), _ptr(tok_seq), _ptr(slots), n_seq, _ptr(page_table), n_slots, max_pages,
                                         _ptr(cache), ctypes.c_longlong(page_stride), n_pages, int(write_kv), *part, _stream()))


def _attention_q8_check(q, out, n_heads, n_kv, head_dim, cu_q, start_pos, slots, page_table, cache, page_stride, max_q_len, max_kv_len, window):
    """What attention_q8() needs of its arguments, one after the other."""
    _need(q, "attention_q8: query rows", torch.bfloat16, 2)
    _need(out, "attention_q8: output", torch.bfloat16, 2)
    for what, v, dims in (("row offsets", cu_q, 1), ("start positions", start_pos, 1), ("slots", slots, 1), ("page table", page_table, 2)):
        if v is None and what == "slots":
            continue
        _need(v, f"attention_q8: {what}", torch.int32, dims)
        if not v.is_contiguous():
            raise KernelError(f"attention_q8: {what} must be contiguous")
    _q8_cache("attention_q8", cache, page_stride, n_kv, head_dim)
    t, n_seq = q.shape[0], start_pos.shape[0]
    if n_kv < 1 or n_heads % n_kv or q.shape[1] != n_heads * head_dim or out.shape != q.shape:
        raise KernelError(f"attention_q8: query rows {tuple(q.shape)} and output {tuple(out.shape)} do not fit {n_heads} heads of {head_dim} over {n_kv} kv heads")
    if cu_q.shape[0] != n_seq + 1 or (slots is not None and slots.shape[0] != n_seq) or (slots is None and page_table.shape[0] < n_seq):
        raise KernelError("attention_q8: row offsets, start positions and slots do not fit each other")
    if max_q_len < 0 or max_kv_len < 0 or window < 0:
        raise KernelError("attention_q8: bounds and window must not be negative")
    _same_device("attention_q8", q, out, cu_q, start_pos, slots, page_table, cache)


@functools.lru_cache(maxsize=4096)
def _attention_q8_scratch(head_dim, rows, n_seq, n_heads, n_kv, max_q_len, max_kv_len, window) -> int:
    """Floats of scratch that a launch of these sizes needs."""
    lib = _lib("attention_q8", (("HEAD_DIM", head_dim),))
    lib.dlgo_attention_q8_scratch.restype = ctypes.c_longlong
    return lib.dlgo_attention_q8_scratch(rows, n_seq, n_heads, n_kv, max_q_len, max_kv_len, window)


def attention_q8_fuses_rotation(head_dim: int, group: int, max_q_len: int, rot_width: int, interleaved: bool, n_seq: int, n_kv: int) -> bool:
    """True if attention_q8() should rotate the queries and take in the new keys and values itself for such a step: one row a
    sequence, heads rotated whole, in halves, of sizes in steps of 32 up to 128, up to 16 of them a kv head; and so few
    (sequence, kv head) pairs that a launch costs more than the rotation repeated in every wave: two a compute unit with heads of
    up to 64, one with 128 (8 layers of 32 heads over 8 behind 1,024 tokens, ms a step fused and not: head size 64, 8, 32 and 64
    sequences 0.529 and 0.561, 0.632 and 0.644, 0.719 and 0.734; 128, 16, 32 and 48 sequences 1.210 and 1.234, 1.269 and 1.267,
    1.427 and 1.381)."""
    return (max_q_len == 1 and head_dim % 32 == 0 and head_dim <= 128 and rot_width == head_dim and not interleaved and group <= 16
            and n_seq * n_kv * max(head_dim, 64) <= 128 * compute_units())


def attention_q8(q: torch.Tensor, out: torch.Tensor, n_heads: int, n_kv: int, head_dim: int, cu_q: torch.Tensor,
                 start_pos: torch.Tensor, slots: Optional[torch.Tensor], page_table: torch.Tensor, cache: torch.Tensor,
                 page_stride: int, max_q_len: int, max_kv_len: int, window: int = 0, scale: Optional[float] = None,
                 scratch=None, rotation=None) -> torch.Tensor:
    """Attention of a step's (rotated) query rows q [T, H*hd] over the 8-bit cache that rope_kv_q8() writes, which holds
    the step's own tokens already; out [T, H*hd], both bfloat16 and apart in memory.

    cu_q [n_seq + 1], start_pos [n_seq], slots [n_seq]: int32 on the device.  Sequence i brings rows cu_q[i] to cu_q[i+1]
    (none, one, a few drafted tokens, a prompt), at positions from start_pos[i] on, and its pages are row slots[i] of
    page_table (row i if slots is None).  A row sees the keys up to its own position, with window > 0 the last `window`
    of them.  Rows behind the last sequence's are left as they were.  max_q_len and max_kv_len (host) bound the
    rows a sequence brings and the tokens it holds afterwards: a captured step passes what it allows for; rows and
    tokens beyond the bounds are left out or slow, never out of bounds.  scratch(n) returns a float32 buffer of at least n elements for what
    several blocks find of a row (allocated here if not given).  A row that finds no page at all is zeros.  A query head that
    is not finite gives NaN, or zeros where all its scores are -inf.

    rotation = (cos, sin), where attention_q8_fuses_rotation() says so (one row a sequence): q holds the step's unrotated
    [q | k | v] rows, the kernel rotates the queries and does what rope_kv_q8() does for the keys and values, to the bit."""
    # as in rope_kv_q8(): one look at each tensor, and the checks that can say what is wrong where that is not enough
    try:
        dev = q.get_device()
        t, width = q.shape
        n_seq = start_pos.numel()
        n_slots, max_pages = page_table.shape
        plain = (dev >= 0 and dev == _current_device() and n_kv > 0 and n_heads % n_kv == 0 and q.dtype is _BF16
                 and width == (n_heads if rotation is None else n_heads + 2 * n_kv) * head_dim
                 and out.dtype is _BF16 and out.shape == (t, n_heads * head_dim) and out.get_device() == dev and _is_vector(cu_q, n_seq + 1, dev)
                 and _is_vector(start_pos, n_seq, dev) and (n_slots >= n_seq if slots is None else _is_vector(slots, n_seq, dev))
                 and _is_vector(page_table, n_slots * max_pages, dev) and cache.get_device() == dev
                 and max_q_len >= 0 and max_kv_len >= 0 and window >= 0)
    except (AttributeError, TypeError, ValueError):
        plain = False
    if not plain:
        _attention_q8_check(q if rotation is None else q[:, :n_heads * head_dim], out, n_heads, n_kv, head_dim, cu_q, start_pos, slots, page_table, cache, page_stride, max_q_len, max_kv_len, window)
        t, n_seq = q.shape[0], start_pos.shape[0]
        n_slots, max_pages = page_table.shape
    n_pages = _q8_cache("attention_q8", cache, page_stride, n_kv, head_dim)
    cos = sin = None
    if rotation is not None:
        cos, sin = rotation
        if q.shape[1] < (n_heads + 2 * n_kv) * head_dim or max_q_len != 1:
            raise KernelError(f"attention_q8: rows {tuple(q.shape)} of up to {max_q_len} a sequence are not single tokens' [q | k | v] of {n_heads} and {n_kv} heads of {head_dim}")
        for what, v in (("cos", cos), ("sin", sin)):
            _need(v, f"attention_q8: {what} table", torch.float32, 2)
            if v.shape != cos.shape or v.shape[1] != head_dim // 2 or v.shape[0] < 1 or not v.is_contiguous() or v.get_device() != q.get_device():
                raise KernelError(f"attention_q8: {what} table {tuple(v.shape)} does not rotate heads of {head_dim}")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    if t == 0 or n_seq == 0 or max_q_len == 0:
        return out
    max_q_len = min(int(max_q_len), t)
    max_kv_len = max(1, min(int(max_kv_len), max_pages * PAGE))
    window = min(int(window), 2 ** 31 - 1)          # (no sequence is longer)
    need = _attention_q8_scratch(head_dim, t, n_seq, n_heads, n_kv, max_q_len, max_kv_len, window)
    lib = _lib("attention_q8", (("HEAD_DIM", head_dim),))
    part = None
    if need:
        part = scratch(need) if scratch is not None else torch.empty(need, dtype=torch.float32, device=q.device)
        _given_scratch("attention_q8", part, torch.float32, q)
    _check(lib.dlgo_attention_q8(_ptr(q), _rows32(q, "attention_q8: query rows"), _ptr(out), _rows32(out, "attention_q8: output"), t, n_seq,
                                 n_heads, n_kv, head_dim, _ptr(cu_q), _ptr(start_pos), _ptr(slots), _ptr(page_table),
                                 n_slots, max_pages, _ptr(cache), ctypes.c_longlong(page_stride), n_pages,
                                 max_q_len, max_kv_len, window, ctypes.c_float(scale), _ptr(part),
                                 ctypes.c_longlong(part.numel() if part is not None else 0), _ptr(cos), _ptr(sin),
                                 0 if cos is None else cos.shape[0], _stream()))
    return out


_argmax_scratch: dict = {}


def argmax(logits: torch.Tensor, out: torch.Tensor, scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[r] = index of the first maximum of row r.  scratch: 512 bytes per row (kept here per device if not given)."""
    _need(logits, "logits", torch.float32, 2)
    _need(out, "argmax output", torch.int32, 1)
    n = logits.shape[0]
    if out.shape[0] != n:
        raise KernelError("argmax: one output per row")
    if scratch is None:
        scratch = _argmax_scratch.get(logits.device)
        if scratch is None or scratch.numel() < n * 512:
            scratch = torch.empty(max(n, 256) * 512, dtype=torch.uint8, device=logits.device)
            _argmax_scratch[logits.device] = scratch
    _check(_lib("sampling").dlgo_argmax(_ptr(logits), _rows(logits, "logits"), n, logits.shape[1], _ptr(scratch),
                                        ctypes.c_longlong(scratch.numel() * scratch.element_size()), _ptr(out), _stream()))
    return out


def sample(logits: torch.Tensor, work: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor,
           top_p: torch.Tensor, min_p: torch.Tensor, penalty: torch.Tensor, recent: Optional[torch.Tensor],
           uniform: torch.Tensor, out: torch.Tensor, recent_rows: Optional[torch.Tensor] = None,
           counts: Optional[torch.Tensor] = None, dealt_rows: bool = True) -> torch.Tensor:
    """One token per row of float32 logits, each row with its own options.  work: float32 scratch [rows, vocab].  recent [rows, w]: the row's recent tokens
    (-1 where empty) for the repetition penalty.  With recent_rows [rows] and counts: recent is a table of rings, row
    recent_rows[r] of it belongs to row r and holds its last min(counts, w) tokens; the chosen token is added to it.
    dealt_rows=False: the caller, who has the options on the host, knows that no row is of a kind that several blocks
    share over a wide vocabulary (a top-k of 1 to 1,024, or neither top-k nor top-p); the kernels for those are
    then not launched."""
    _need(logits, "logits", torch.float32, 2)
    n, v = logits.shape
    for name, t, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                        ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32),
                        ("penalty", penalty, torch.float32), ("uniform", uniform, torch.float32),
                        ("sample output", out, torch.int32)):
        _need(t, name, dt, 1)
        if t.shape[0] != n:
            raise KernelError(f"sample: {name} has {t.shape[0]} entries for {n} rows")
    _need(work, "work", torch.float32, 2)
    if work.shape[0] < n or work.shape[1] != v or not work.is_contiguous():
        raise KernelError(f"sample: scratch {tuple(work.shape)} too small for {(n, v)}")
    n_recent = 0
    if (recent_rows is None) != (counts is None):
        raise KernelError("sample: a table of rings needs both recent_rows and counts")
    if recent is not None:
        _need(recent, "recent tokens", torch.int32, 2)
        if not recent.is_contiguous() or (counts is None and recent.shape[0] != n):
            raise KernelError("sample: one row of recent tokens per row of logits")
        n_recent = recent.shape[1]
    if counts is not None:
        _need(recent_rows, "rows of the recent tokens", torch.int32, 1)
        _need(counts, "counts of recent tokens", torch.int32, 1)
        if recent is None or recent_rows.shape[0] != n or counts.shape[0] != recent.shape[0]:
            raise KernelError("sample: recent_rows has one entry per row of logits, counts one per row of the table")
    _check(_lib("sampling").dlgo_sample(_ptr(logits), _rows(logits, "logits"), n, v, _ptr(work), _ptr(temperature),
                                        _ptr(top_k), _ptr(top_p), _ptr(min_p), _ptr(penalty), _ptr(recent), n_recent,
                                        _ptr(recent_rows), _ptr(counts), _ptr(uniform), _ptr(out), int(bool(dealt_rows)),
                                        _stream()))
    return out


def _verify_drafts_check(logits, draft_tokens, cu_drafts, temperature, uniform, accepted, token, max_drafts, draft_logits, probs):
    """What verify_drafts() needs of its arguments, one after the other."""
    _need(temperature, "verify_drafts: temperature", torch.float32, 1)
    _need(draft_tokens, "verify_drafts: draft tokens", torch.int32, 1)
    _need(logits, "verify_drafts: logits", torch.float32, 2)
    n, v = temperature.shape[0], logits.shape[1]
    d = draft_tokens.shape[0]
    for what, x, dt, size in (("draft tokens", draft_tokens, torch.int32, d), ("draft offsets", cu_drafts, torch.int32, n + 1),
                              ("temperature", temperature, torch.float32, n), ("uniform numbers", uniform, torch.float32, d + n),
                              ("accepted", accepted, torch.int32, n), ("token", token, torch.int32, n), ("probs", probs, torch.float32, d)):
        if x is None and what == "probs":
            continue
        _need(x, f"verify_drafts: {what}", dt, 1)
        if x.shape[0] != size or not x.is_contiguous():
            raise KernelError(f"verify_drafts: {what} has shape {tuple(x.shape)}, {size} entries in a row are needed ({n} sequences, {d} drafts)")
    if logits.shape[0] != d + n or v < 1:
        raise KernelError(f"verify_drafts: {n} sequences with {d} drafts need {d + n} rows of logits, found {tuple(logits.shape)}")
    if draft_logits is not None:
        _need(draft_logits, "verify_drafts: draft logits", torch.float32, 2)
        if tuple(draft_logits.shape) != (d, v):
            raise KernelError(f"verify_drafts: draft logits {tuple(draft_logits.shape)}, expected {(d, v)}")
    if max_drafts < 0:
        raise KernelError("verify_drafts: max_drafts must not be negative")
    _same_device("verify_drafts", logits, draft_tokens, cu_drafts, temperature, uniform, accepted, token, draft_logits, probs)


@functools.lru_cache(maxsize=4096)
def _verify_drafts_scratch(n, d, vocab, model_drafts) -> int:
    """Bytes of scratch that a call of these sizes needs."""
    lib = _lib("verify")
    lib.dlgo_verify_drafts_scratch.restype = ctypes.c_longlong
    return lib.dlgo_verify_drafts_scratch(n, d, vocab, int(model_drafts))


def verify_drafts(logits: torch.Tensor, draft_tokens: torch.Tensor, cu_drafts: torch.Tensor, temperature: torch.Tensor,
                  uniform: torch.Tensor, accepted: torch.Tensor, token: torch.Tensor, max_drafts: int,
                  draft_logits: Optional[torch.Tensor] = None, probs: Optional[torch.Tensor] = None, scratch=None) -> None:
    """How many of each sequence's drafted tokens the target model keeps, and the token that follows them.

    Sequence i drafted the tokens cu_drafts[i] to cu_drafts[i+1] of draft_tokens (int32, D in all; none is allowed, more
    than max_drafts are not looked at) and
    brings one row of the target's float32 logits [D + n, V] for the place of each draft and one for the place after them,
    from row cu_drafts[i] + i on; uniform [D + n] has a number in [0, 1) for each of those rows.  temperature [n]; 0 is
    greedy.  draft_logits [D, V]: the logits that the drafts were drawn from (at the same temperature); None: the drafts
    are certain of their tokens (looked up, or a greedy draft model's).

    With p = softmax(logits / T) and q = softmax(draft_logits / T) (or one for the drafted token), draft j is kept while
    uniform_j * q(token_j) < p(token_j); accepted[i] (int32) counts the kept ones, token[i] (int32) is drawn from max(p - q, 0)
    of the first refused draft's row, or from p of the last row, as the first index whose running sum exceeds the
    sequence's last uniform number times the whole.  Greedy: a draft is kept if it is the row's maximum (lowest index), and the token is
    the maximum.  Sums are 64-bit, in an order that only the shapes decide.  A logit of -inf or NaN has no weight.  A token
    outside the vocabulary is refused.  probs [D] (float32, optional): p(token_j) for every draft.  scratch(n) returns a uint8 buffer of at least n
    bytes (allocated here if not given)."""
    # as in rope_kv_q8(): one look at each tensor, and the checks that can say what is wrong where that is not enough
    try:
        dev = logits.get_device()
        n, d = temperature.numel(), draft_tokens.numel()
        rows, v = logits.shape
        plain = (dev >= 0 and dev == _current_device() and logits.dtype is _F32 and rows == d + n and v > 0 and max_drafts >= 0
                 and _is_vector(temperature, n, dev, _F32) and _is_vector(draft_tokens, d, dev) and _is_vector(cu_drafts, n + 1, dev)
                 and _is_vector(uniform, d + n, dev, _F32) and _is_vector(accepted, n, dev) and _is_vector(token, n, dev)
                 and (probs is None or _is_vector(probs, d, dev, _F32))
                 and (draft_logits is None or (draft_logits.dtype is _F32 and draft_logits.shape == (d, v) and draft_logits.get_device() == dev)))
    except (AttributeError, TypeError, ValueError):
        plain = False
    if not plain:
        _verify_drafts_check(logits, draft_tokens, cu_drafts, temperature, uniform, accepted, token, max_drafts, draft_logits, probs)
        n, d, v = temperature.shape[0], draft_tokens.shape[0], logits.shape[1]
    if n == 0:
        return
    model_drafts = draft_logits is not None and d > 0
    lib = _lib("verify")
    need = _verify_drafts_scratch(n, d, v, model_drafts)
    work = scratch(need) if scratch is not None else torch.empty(need, dtype=torch.uint8, device=logits.device)
    _given_scratch("verify_drafts", work, torch.uint8, logits)
    _check(lib.dlgo_verify_drafts(_ptr(logits), ctypes.c_longlong(_rows(logits, "verify_drafts: logits")), _ptr(draft_tokens),
                                  _ptr(draft_logits if model_drafts else None),
                                  ctypes.c_longlong(_rows(draft_logits, "verify_drafts: draft logits") if model_drafts else 0),
                                  _ptr(cu_drafts), _ptr(temperature), _ptr(uniform), n, d, v, min(int(max_drafts), d), _ptr(accepted),
                                  _ptr(token), _ptr(probs), _ptr(work), ctypes.c_longlong(work.numel()), _stream()))


# ---------------------------------------------------------------------------
# Timing the launches one by one (what computerex/dlgo's gpu_timing_main.go:73-119 does for its operations): inside a
# `with Timings() as t:` block every face above that launches something is bracketed by two events on the current
# stream; t.microseconds() then gives, per label, the time between them summed over the block.  A product's label
# carries its weight's shape, which is what tells the products of a layer apart.  The steps inside the block must run
# as they are (a replayed recording calls no face).  Outside such a block a face costs one comparison more.
_recorder: Optional[list] = None


class Timings:
    def __enter__(self) -> "Timings":
        global _recorder
        self.events: List[tuple] = []
        self._outer, _recorder = _recorder, self.events
        return self

    def __exit__(self, *exc) -> None:
        global _recorder
        _recorder = self._outer

    def microseconds(self) -> Dict[str, float]:
        torch.cuda.synchronize()
        out: Dict[str, float] = {}
        for label, start, end in self.events:
            out[label] = out.get(label, 0.0) + start.elapsed_time(end) * 1000.0
        return out

    def launches(self) -> Dict[str, int]:
        out: Dict[str, int] = {}
        for label, _, _ in self.events:
            out[label] = out.get(label, 0) + 1
        return out


def _timed(fn):
    name = fn.__name__
    by_weight = name.startswith("gemm")

    @functools.wraps(fn)
    def face(*args, **kwargs):
        rec = _recorder
        if rec is None:
            return fn(*args, **kwargs)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        result = fn(*args, **kwargs)
        end.record()
        if result is False or (result is None and name == "gemm_runs"):
            return result                # it declined: nothing was launched
        label = name
        if by_weight and args and isinstance(args[0], torch.Tensor):
            label = f"{name}[{args[0].shape[0]}x{args[0].shape[1]}]"
        rec.append((label, start, end))
        return result
    return face


for _name in ("embed", "copy_rows", "rmsnorm", "bias_add", "head_rmsnorm", "gemm_accum_then_norm", "gemm_runs", "gemm", "gemm_rmsnorm",
              "gemm_accum_leave_norm", "gemm_scaled", "rope_kv", "attention", "argmax", "sample", "rope_kv_q8", "attention_q8", "verify_drafts"):
    globals()[_name] = _timed(globals()[_name])
del _name
