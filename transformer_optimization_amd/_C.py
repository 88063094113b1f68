"""ctypes binding of ``libtx_hip.so`` (declared in ``include/tx_api.h``).

The library is loaded lazily, after ``import torch``, so that it binds to the
HIP runtime torch already mapped (both resolve ``libamdhip64.so.7`` by
SONAME).  If the library is missing, every wrapper raises -- there is no
fallback path.  Wrappers take torch tensors, check devices / dtypes /
contiguity, pass raw pointers and ``torch.cuda.current_stream()`` and turn a
non-zero status into :class:`TxError`.  They never synchronise, so they are
capturable into a graph.
"""

from __future__ import annotations

import array
import contextlib
import ctypes
import math
import os
import threading
from pathlib import Path
from typing import Optional, Tuple

import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libtx_hip.so"
ABI_VERSION = 4

TX_OK, TX_EINVAL, TX_EUNSUPPORTED, TX_EHIP, TX_ESCRATCH = 0, 1, 2, 3, 4
TX_F32, TX_F16, TX_BF16 = 0, 1, 2

LN_HAS_DELTA, LN_MASK_DELTA, LN_MASK_X, LN_MASK_OUT, LN_WRITE_X, LN_SPLIT_Y = 1, 2, 4, 8, 16, 32
EPI_BIAS, EPI_GELU_ERF, EPI_RESIDUAL, EPI_MASK_DELTA, EPI_MASK_OUT, EPI_SPLIT_OUT = 1, 2, 4, 8, 16, 32
SOFTMAX_EAGER, SOFTMAX_ONLINE = 0, 1
SELECT_GEMM, SELECT_ATTN_ROWRES = 0, 1
SOFTMAX_MODES = {"eager": SOFTMAX_EAGER, "online": SOFTMAX_ONLINE}
# Longest sequence the eager-exact softmax serves (tx_flash_attn_fwd returns
# TX_EUNSUPPORTED above it: 1024 key tiles of 64); below it, the lengths
# eager_softmax_supported accepts.
EAGER_MAX_SEQ = 65536
# Shared memory per block assumed where no device can be asked (the usual
# value; it only decides lengths from ~16K keys up).
DEFAULT_SHARED_MEM_PER_BLOCK = 65536

# Every symbol include/tx_api.h declares.
EXPORTED_SYMBOLS = (
    "tx_abi_version",
    "tx_status_string",
    "tx_device_cu_count",
    "tx_eager_softmax_supported",
    "tx_layernorm_residual",
    "tx_gemm",
    "tx_qkv_proj",
    "tx_flash_attn_fwd",
    "tx_flash_attn_fwd_strided",
    "tx_flash_attn_fwd_noalloc",
    "tx_rotary_append",
    "tx_flash_attn_packed",
    "tx_flash_attn_paged",
    "tx_flash_attn_paged_workspace",
    "tx_select_kernel",
)

# Rows (batch * heads * seq) the fixed scratch of tx_flash_attn_fwd_noalloc holds.
NOALLOC_MAX_STAT_ROWS = 1 << 20

_DT = {torch.float32: TX_F32, torch.float16: TX_F16, torch.bfloat16: TX_BF16}


class TxError(RuntimeError):
    """A libtx_hip entry point returned a non-zero status."""

    def __init__(self, fn: str, code: int, msg: str):
        super().__init__(f"{fn} failed: {msg} (status {code})")
        self.code = code
        self.fn = fn


_lib: Optional[ctypes.CDLL] = None
_lock = threading.Lock()

_i64, _i32, _u32, _f32, _vp = ctypes.c_int64, ctypes.c_int, ctypes.c_uint32, ctypes.c_float, ctypes.c_void_p


def _declare(lib: ctypes.CDLL) -> None:
    lib.tx_abi_version.restype = _i32
    lib.tx_abi_version.argtypes = []
    lib.tx_status_string.restype = ctypes.c_char_p
    lib.tx_status_string.argtypes = [_i32]
    lib.tx_device_cu_count.restype = _i32
    lib.tx_device_cu_count.argtypes = []
    lib.tx_select_kernel.restype = _i32
    lib.tx_select_kernel.argtypes = [_i32, _i32]
    lib.tx_eager_softmax_supported.restype = _i32
    lib.tx_eager_softmax_supported.argtypes = [_i64, _i64]
    lib.tx_layernorm_residual.restype = _i32
    lib.tx_layernorm_residual.argtypes = [
        _vp, _vp, _vp, _vp, _vp, _vp, _vp,  # x delta x_out y gamma beta row_valid
        _vp, _vp,                           # mean_out rstd_out
        _i64, _i64, _f32,                   # rows d eps
        _i32, _i32, _i32, _i32,             # x_dt delta_dt y_dt param_dt
        _u32, _vp,                          # flags stream
    ]
    lib.tx_gemm.restype = _i32
    lib.tx_gemm.argtypes = [
        _vp, _i64, _vp, _i64,               # a lda w ldw
        _vp, _vp, _i64,                     # bias residual ldr
        _vp, _i64, _i64, _i64, _i64,        # c ldc m n k
        _i32, _i32, _i32, _i32, _u32,       # ab_dt c_dt bias_dt res_dt epilogue
        _vp, _vp,                           # row_valid stream
    ]
    lib.tx_qkv_proj.restype = _i32
    lib.tx_qkv_proj.argtypes = [
        _vp, _vp, _vp, _vp, _vp, _i64,      # a w_qkv b_qkv qk vt ldvt
        _i64, _i64, _i64, _i64, _i32, _vp,  # batch seq d_model heads dt stream
    ]
    lib.tx_flash_attn_fwd.restype = _i32
    lib.tx_flash_attn_fwd.argtypes = [
        _vp, _vp, _i64, _vp, _vp,           # qk vt ldvt o key_valid
        _i64, _i64, _i64, _i64,             # batch seq heads head_dim
        _f32, _i32, _i32, _vp,              # scale causal softmax_mode row_stats
        _i32, _vp,                          # dt stream
    ]
    lib.tx_flash_attn_fwd_strided.restype = _i32
    lib.tx_flash_attn_fwd_strided.argtypes = [
        _vp, _vp, _vp, _vp,                 # q k v o
        _vp, _vp, _vp, _vp,                 # q/k/v/o strides (int64[4] each)
        _vp, _i64,                          # key_valid key_valid_sb
        _i64, _i64, _i64, _i64,             # batch heads seq head_dim
        _f32, _i32, _i32, _vp,              # scale causal softmax_mode row_stats
        _i32, _vp,                          # dt stream
    ]
    lib.tx_flash_attn_fwd_noalloc.restype = _i32
    lib.tx_flash_attn_fwd_noalloc.argtypes = [
        _vp, _vp, _i64, _vp, _vp,           # qk vt ldvt o key_valid
        _i64, _i64, _i64, _i64,             # batch seq heads head_dim
        _f32, _i32, _i32, _i32, _vp,        # scale causal softmax_mode dt stream
    ]
    lib.tx_rotary_append.restype = _i32
    lib.tx_rotary_append.argtypes = [
        _vp, _vp, _vp, _vp,                 # q strides q_out strides
        _vp, _vp, _vp, _vp, _vp, _vp,       # k strides k_out strides v strides
        _vp, _vp, _vp, _vp,                 # k_cache strides v_cache strides
        _vp, _vp, _vp, _vp, _vp, _i64,      # steps positions cu_seqlens kv_lens block_table table_ld
        _i64, _i64, _i64, _i64, _i64, _i64,  # tokens batch q_heads kv_heads head_dim rotary_dim
        _i64, _i64, _i64,                   # num_pages page_size max_pages
        _f32, _i32, _i32, _vp,              # amplitude interleaved dt stream
    ]
    lib.tx_flash_attn_packed.restype = _i32
    lib.tx_flash_attn_packed.argtypes = [
        _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,  # q k v o, each with its strides
        _vp, _i64, _i64, _i64, _i64, _i64,  # cu_seqlens tokens batch q_heads kv_heads head_dim
        _f32, _i32, _i32, _vp,              # scale causal dt stream
    ]
    lib.tx_flash_attn_paged.restype = _i32
    lib.tx_flash_attn_paged.argtypes = [
        _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,  # q k_cache v_cache o, each with its strides
        _vp, _vp, _vp, _i64,                # cu_seqlens kv_lens block_table table_ld
        _i64, _i64, _i64, _i64, _i64,       # tokens batch q_heads kv_heads head_dim
        _i64, _i64, _i64, _i64,             # num_pages page_size max_pages max_q_len
        _f32, _i32, _vp, _i64, _i32, _vp,   # scale causal workspace workspace_floats dt stream
    ]
    lib.tx_flash_attn_paged_workspace.restype = _i32
    lib.tx_flash_attn_paged_workspace.argtypes = [_i64] * 8 + [_vp]


def _hip_runtime_mappings() -> set:
    paths = set()
    try:
        with open("/proc/self/maps") as fh:
            for line in fh:
                if "libamdhip64" in line:
                    paths.add(line.split()[-1])
    except OSError:
        pass
    return paths


def load_library() -> ctypes.CDLL:
    """Load and check libtx_hip.so once per process (raises if absent)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise ImportError(
                f"{LIB_PATH} is not built; run `python -m transformer_optimization_amd.build` "
                "(or __graft_entry__.build()). There is no fallback path."
            )
        lib = ctypes.CDLL(str(LIB_PATH), mode=os.RTLD_NOW | os.RTLD_LOCAL)
        _declare(lib)
        if lib.tx_abi_version() != ABI_VERSION:
            raise ImportError(f"libtx_hip ABI {lib.tx_abi_version()} != expected {ABI_VERSION}")
        maps = _hip_runtime_mappings()
        if len(maps) > 1:
            raise ImportError(
                "two HIP runtimes are mapped into this process "
                f"({sorted(maps)}); load libtx_hip after `import torch`"
            )
        _lib = lib
        return lib


def status_string(code: int) -> str:
    return load_library().tx_status_string(code).decode()


def _check(fn: str, code: int) -> None:
    if code != TX_OK:
        raise TxError(fn, code, status_string(code))


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _require_cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and t.device.type != "cuda":
            raise ValueError("libtx_hip operates on GPU tensors only (got a CPU tensor)")


def _dt(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


def cu_count() -> int:
    return int(load_library().tx_device_cu_count())


def select_kernel(op: int, variant: int) -> None:
    """Tests and timing: the kernel that this thread's later calls of ``op``
    (``SELECT_GEMM``, ``SELECT_ATTN_ROWRES``) take; -1 restores the choice."""
    _check("tx_select_kernel", load_library().tx_select_kernel(int(op), int(variant)))


_eager_ok: dict = {}


def eager_softmax_supported(seq: int, device: Optional[torch.device] = None) -> bool:
    """Whether the eager-exact softmax serves rows of ``seq`` keys on
    ``device`` (``tx_eager_softmax_supported``; the device's shared memory
    per block, as torch reports it, decides the longest lengths).  Without a
    device, the usual 64 KiB is assumed.  Memoised per (seq, device)."""
    key = (int(seq), device)
    got = _eager_ok.get(key)
    if got is None:
        if device is not None and device.type == "cuda":
            smem = int(torch.cuda.get_device_properties(device).shared_memory_per_block)
        else:
            smem = DEFAULT_SHARED_MEM_PER_BLOCK
        got = _eager_ok[key] = load_library().tx_eager_softmax_supported(int(seq), smem) == 1
    return got


# ------------------------------------------------------------ launch record
class Launch:
    """One entry-point call as the wrappers made it: the C function, its
    arguments (all but the trailing stream), the tensors they point into
    (kept alive) and a description of the work.  Calling it enqueues the same
    launch again on the current stream."""

    __slots__ = ("fn", "args", "keep", "info")

    def __init__(self, fn: str, args: tuple, keep: tuple, info: dict):
        self.fn, self.args, self.keep, self.info = fn, args, keep, info

    def __call__(self) -> None:
        _check(self.fn, getattr(load_library(), self.fn)(*self.args, _stream()))

    def __repr__(self) -> str:
        return f"Launch({self.fn}, {self.info})"


_recorder: Optional[list] = None


@contextlib.contextmanager
def record_launches():
    """Collect every launch the wrappers make inside the block, in order, as
    :class:`Launch` objects (used to time exactly the kernels a forward runs)."""
    global _recorder
    prev, _recorder = _recorder, []
    try:
        yield _recorder
    finally:
        _recorder = prev


def _launch(fn: str, args: tuple, keep: tuple, info: dict) -> None:
    """Call ``lib.<fn>(*args, stream)`` on the current stream; raise on a
    non-zero status; record the call when a recording is active."""
    _check(fn, getattr(load_library(), fn)(*args, _stream()))
    if _recorder is not None:
        _recorder.append(Launch(fn, args, keep, info))


# ----------------------------------------------------------------- wrappers
def layernorm_residual(
    x: torch.Tensor,
    gamma: torch.Tensor,
    beta: torch.Tensor,
    *,
    delta: Optional[torch.Tensor] = None,
    x_out: Optional[torch.Tensor] = None,
    y: Optional[torch.Tensor] = None,
    y_dtype: Optional[torch.dtype] = None,
    row_valid: Optional[torch.Tensor] = None,
    flags: int = 0,
    eps: float = 1e-5,
    mean_out: Optional[torch.Tensor] = None,
    rstd_out: Optional[torch.Tensor] = None,
    split: bool = False,
) -> torch.Tensor:
    """``y = LN(x [+ delta])`` over the last dim; see ``tx_layernorm_residual``.
    ``mean_out`` / ``rstd_out`` (fp32, one per row) receive the row statistics.
    ``split=True`` writes y as [rows, 2d]: the rounded value, then the rounded
    remainder (a two-term operand for the fp32-residual policy)."""
    load_library()
    _require_cuda(x, gamma, beta, delta, x_out, y, row_valid, mean_out, rstd_out)
    d = x.shape[-1]
    rows = x.numel() // d
    if y is None:
        shape = (*x.shape[:-1], 2 * d) if split else x.shape
        y = torch.empty(shape, dtype=y_dtype or x.dtype, device=x.device)
    if y.numel() != rows * d * (2 if split else 1):
        raise ValueError("y has the wrong number of elements")
    if split:
        flags |= LN_SPLIT_Y
    for t in (x, y, delta, x_out):
        if t is not None and not t.is_contiguous():
            raise ValueError("layernorm_residual needs contiguous rows")
    if delta is not None:
        flags |= LN_HAS_DELTA
    if x_out is not None:
        flags |= LN_WRITE_X
    for t in (mean_out, rstd_out):
        if t is not None and (t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous()):
            raise ValueError("mean_out / rstd_out must be contiguous fp32 with one entry per row")
    rv = row_valid.contiguous() if row_valid is not None else None
    args = (
        x.data_ptr(), _ptr(delta), _ptr(x_out), y.data_ptr(), gamma.data_ptr(), beta.data_ptr(),
        _ptr(rv), _ptr(mean_out), _ptr(rstd_out), rows, d, float(eps), _dt(x),
        _dt(delta) if delta is not None else _dt(x), _dt(y), _dt(gamma), flags,
    )
    info = {"op": "layernorm", "rows": rows, "d": d, "x_bytes": x.element_size(),
            "y_bytes": y.element_size(), "param_bytes": gamma.element_size(), "flags": flags,
            "delta_bytes": delta.element_size() if delta is not None else 0}
    _launch("tx_layernorm_residual", args, (x, delta, x_out, y, gamma, beta, rv, mean_out, rstd_out), info)
    return y


def gemm(
    a: torch.Tensor,
    w: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    residual: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    gelu: bool = False,
    row_valid: Optional[torch.Tensor] = None,
    mask_delta: bool = False,
    mask_out: bool = False,
    split_out: bool = False,
) -> torch.Tensor:
    """``out = epilogue(a @ w.T)`` for a 2-D ``a`` [M,K] and nn.Linear ``w`` [N,K].
    ``split_out=True`` stores the unrounded fp32 result as a hi/lo pair in
    ``out`` [M, 2N] (``out_dtype`` = the operand dtype)."""
    load_library()
    _require_cuda(a, w, bias, residual, out, row_valid)
    if a.dim() != 2 or w.dim() != 2 or a.shape[1] != w.shape[1]:
        raise ValueError(f"gemm shapes: a {tuple(a.shape)} w {tuple(w.shape)}")
    m, k = a.shape
    n = w.shape[0]
    if a.stride(1) != 1 or w.stride(1) != 1:
        raise ValueError("gemm operands must be K-contiguous")
    ncols = 2 * n if split_out else n
    if out is None:
        out = torch.empty((m, ncols), dtype=out_dtype or a.dtype, device=a.device)
    if out.shape != (m, ncols) or out.stride(1) != 1:
        raise ValueError(f"gemm output must be [M, {ncols}] with unit column stride")
    epi = 0
    if bias is not None:
        epi |= EPI_BIAS
    if gelu:
        epi |= EPI_GELU_ERF
    ldr = 0
    if residual is not None:
        if residual.shape != (m, n) or residual.stride(1) != 1:
            raise ValueError("residual must be [M, N] with unit column stride")
        epi |= EPI_RESIDUAL
        ldr = residual.stride(0)
    if split_out:
        epi |= EPI_SPLIT_OUT
    if mask_delta:
        epi |= EPI_MASK_DELTA
    if mask_out:
        epi |= EPI_MASK_OUT
    rv = row_valid.contiguous() if row_valid is not None else None
    args = (
        a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0),
        _ptr(bias), _ptr(residual), ldr,
        out.data_ptr(), out.stride(0), m, n, k,
        _dt(a), _dt(out), _dt(bias) if bias is not None else _dt(a),
        _dt(residual) if residual is not None else _dt(out), epi,
        _ptr(rv),
    )
    info = {"op": "gemm", "m": m, "n": n, "k": k, "epilogue": epi, "ab_bytes": a.element_size(),
            "c_bytes": out.element_size()}
    _launch("tx_gemm", args, (a, w, bias, residual, out, rv), info)
    return out


def vt_ld(seq: int) -> int:
    """Row stride of the head-transposed V buffer: seq rounded up to 8."""
    return (seq + 7) // 8 * 8


def qkv_proj(
    a: torch.Tensor,
    w_qkv: torch.Tensor,
    b_qkv: torch.Tensor,
    batch: int,
    seq: int,
    heads: int,
    *,
    qk: Optional[torch.Tensor] = None,
    vt: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Packed QKV projection -> (qk [M, 2D], vt [B, H, hd, ldvt])."""
    load_library()
    _require_cuda(a, w_qkv, b_qkv, qk, vt)
    m, d = a.shape
    if m != batch * seq or w_qkv.shape != (3 * d, d) or b_qkv.shape != (3 * d,):
        raise ValueError("qkv_proj shapes")
    for t in (a, w_qkv, b_qkv):
        if not t.is_contiguous():
            raise ValueError("qkv_proj operands must be contiguous")
    hd = d // heads
    ld = vt_ld(seq)
    if qk is None:
        qk = torch.empty((m, 2 * d), dtype=a.dtype, device=a.device)
    if vt is None:
        vt = torch.empty((batch, heads, hd, ld), dtype=a.dtype, device=a.device)
    args = (a.data_ptr(), w_qkv.data_ptr(), b_qkv.data_ptr(), qk.data_ptr(), vt.data_ptr(), ld,
            batch, seq, d, heads, _dt(a))
    info = {"op": "qkv_proj", "m": m, "n": 3 * d, "k": d, "ab_bytes": a.element_size()}
    _launch("tx_qkv_proj", args, (a, w_qkv, b_qkv, qk, vt), info)
    return qk, vt


def flash_attn(
    qk: torch.Tensor,
    vt: torch.Tensor,
    batch: int,
    seq: int,
    heads: int,
    head_dim: int,
    scale: float,
    causal: bool,
    *,
    key_valid: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    softmax: str = "eager",
    row_stats: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention over the ``qkv_proj`` layouts -> o [B*S, H*hd].

    ``softmax="eager"`` reproduces the eager fp32 softmax bit for bit and uses
    ``row_stats`` (fp32, 2*B*H*S; allocated here when omitted);
    ``softmax="online"`` is the one-pass online softmax."""
    load_library()
    _require_cuda(qk, vt, key_valid, out, row_stats)
    if softmax not in SOFTMAX_MODES:
        raise ValueError(f"softmax must be one of {sorted(SOFTMAX_MODES)}")
    mode = SOFTMAX_MODES[softmax]
    d = heads * head_dim
    if qk.shape != (batch * seq, 2 * d) or not qk.is_contiguous():
        raise ValueError("qk must be contiguous [B*S, 2D]")
    if vt.dim() != 4 or tuple(vt.shape[:3]) != (batch, heads, head_dim) or not vt.is_contiguous():
        raise ValueError("vt must be contiguous [B, H, hd, ldvt]")
    if out is None:
        out = torch.empty((batch * seq, d), dtype=qk.dtype, device=qk.device)
    kv = None
    if key_valid is not None:
        if key_valid.dtype not in (torch.bool, torch.uint8) or key_valid.numel() != batch * seq:
            raise ValueError("key_valid must be bool/uint8 with B*S elements")
        kv = key_valid.contiguous()
    if mode == SOFTMAX_EAGER:
        if row_stats is None:
            row_stats = torch.empty(2 * batch * heads * seq, dtype=torch.float32, device=qk.device)
        if row_stats.dtype != torch.float32 or row_stats.numel() < 2 * batch * heads * seq:
            raise ValueError("row_stats must be fp32 with at least 2*B*H*S elements")
    args = (qk.data_ptr(), vt.data_ptr(), vt.shape[3], out.data_ptr(), _ptr(kv),
            batch, seq, heads, head_dim, float(scale), 1 if causal else 0, mode,
            _ptr(row_stats) if mode == SOFTMAX_EAGER else None, _dt(qk))
    info = {"op": "flash_attn", "batch": batch, "seq": seq, "heads": heads, "head_dim": head_dim,
            "causal": bool(causal), "softmax": softmax}
    _launch("tx_flash_attn_fwd", args, (qk, vt, out, kv, row_stats), info)
    return out


def _strides4(t: torch.Tensor):
    return (ctypes.c_int64 * 4)(*t.stride())


def flash_attn_strided(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    causal: bool,
    *,
    key_valid: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    softmax: str = "eager",
    row_stats: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention over strided [B, H, S, hd] views (``tx_flash_attn_fwd_strided``),
    the call shape of the reference's ``_triton_short_attention(q, k, v, scale,
    causal, mask_active, valid_token_mask)`` (TTB:1596-1668): q / k / v may be
    column slices of a packed [B, S, 3D] projection viewed as [B, H, S, hd].
    Returns ``out``, a [B, H, S, hd] view; by default the permuted view of a
    fresh [B, S, H, hd] tensor, i.e. heads merged in memory ([B, S, D])."""
    load_library()
    _require_cuda(q, k, v, key_valid, out, row_stats)
    if softmax not in SOFTMAX_MODES:
        raise ValueError(f"softmax must be one of {sorted(SOFTMAX_MODES)}")
    mode = SOFTMAX_MODES[softmax]
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("q, k, v must be [B, H, S, hd] views of one shape")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k, v must share a dtype")
    b, h, s, hd = q.shape
    if out is None:
        out = torch.empty((b, s, h, hd), dtype=q.dtype, device=q.device).permute(0, 2, 1, 3)
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must be a [B, H, S, hd] view of the operand dtype")
    kv, kv_sb = None, 0
    if key_valid is not None:
        if key_valid.dtype not in (torch.bool, torch.uint8) or tuple(key_valid.shape) != (b, s):
            raise ValueError("key_valid must be a bool/uint8 [B, S] tensor")
        kv = key_valid if key_valid.stride(1) == 1 else key_valid.contiguous()
        kv_sb = kv.stride(0)
    if mode == SOFTMAX_EAGER:
        if row_stats is None:
            row_stats = torch.empty(2 * b * h * s, dtype=torch.float32, device=q.device)
        if row_stats.dtype != torch.float32 or row_stats.numel() < 2 * b * h * s:
            raise ValueError("row_stats must be fp32 with at least 2*B*H*S elements")
    st = tuple(_strides4(t) for t in (q, k, v, out))
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            ctypes.addressof(st[0]), ctypes.addressof(st[1]), ctypes.addressof(st[2]),
            ctypes.addressof(st[3]), _ptr(kv), kv_sb, b, h, s, hd, float(scale), 1 if causal else 0,
            mode, _ptr(row_stats) if mode == SOFTMAX_EAGER else None, _dt(q))
    info = {"op": "flash_attn", "batch": b, "seq": s, "heads": h, "head_dim": hd,
            "causal": bool(causal), "softmax": softmax}
    # st stays with the recorded launch: a re-launch passes the same stride arrays.
    _launch("tx_flash_attn_fwd_strided", args, (q, k, v, out, kv, row_stats, st), info)
    return out


def flash_attn_noalloc(
    qk: torch.Tensor,
    vt: torch.Tensor,
    batch: int,
    seq: int,
    heads: int,
    head_dim: int,
    scale: float,
    causal: bool,
    *,
    key_valid: Optional[torch.Tensor] = None,
    out: torch.Tensor,
    softmax: str = "eager",
) -> torch.Tensor:
    """``flash_attn`` through ``tx_flash_attn_fwd_noalloc``: the eager softmax's
    row statistics live in the library's fixed device scratch, so nothing is
    allocated (``out`` is the caller's).  batch * heads * seq above
    ``NOALLOC_MAX_STAT_ROWS`` raises TxError (TX_ESCRATCH)."""
    load_library()
    _require_cuda(qk, vt, key_valid, out)
    if softmax not in SOFTMAX_MODES:
        raise ValueError(f"softmax must be one of {sorted(SOFTMAX_MODES)}")
    d = heads * head_dim
    if qk.shape != (batch * seq, 2 * d) or not qk.is_contiguous():
        raise ValueError("qk must be contiguous [B*S, 2D]")
    if vt.dim() != 4 or tuple(vt.shape[:3]) != (batch, heads, head_dim) or not vt.is_contiguous():
        raise ValueError("vt must be contiguous [B, H, hd, ldvt]")
    if out.shape != (batch * seq, d) or not out.is_contiguous() or out.dtype != qk.dtype:
        raise ValueError("out must be contiguous [B*S, D] of the operand dtype")
    kv = None
    if key_valid is not None:
        if key_valid.dtype not in (torch.bool, torch.uint8) or key_valid.numel() != batch * seq:
            raise ValueError("key_valid must be bool/uint8 with B*S elements")
        if not key_valid.is_contiguous():
            raise ValueError("key_valid must be contiguous (no copy is made)")
        kv = key_valid
    args = (qk.data_ptr(), vt.data_ptr(), vt.shape[3], out.data_ptr(), _ptr(kv),
            batch, seq, heads, head_dim, float(scale), 1 if causal else 0, SOFTMAX_MODES[softmax], _dt(qk))
    info = {"op": "flash_attn", "batch": batch, "seq": seq, "heads": heads, "head_dim": head_dim,
            "causal": bool(causal), "softmax": softmax, "noalloc": True}
    _launch("tx_flash_attn_fwd_noalloc", args, (qk, vt, out, kv), info)
    return out


# ------------------------------------------- packed sequences, paged cache
ROTARY_SCALINGS = ("none", "linear", "base", "ramp")


def rotary_steps(
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: str = "none",
    factor: float = 1.0,
    original_len: int = 0,
    low_turns: float = 1.0,
    high_turns: float = 32.0,
    device: Optional[torch.device] = None,
) -> Tuple[torch.Tensor, float]:
    """``(steps, amplitude)`` of :func:`rotary_append`, made once per model.

    ``steps`` (int64 ``[rotary_dim / 2]``) holds each pair's turn per position in units of 2^-64 turn:
    ``f_i / (2 pi)`` with ``f_i = base^(-2i / rotary_dim)``, scaled for contexts ``factor`` times as long as the
    model was trained on (``original_len`` positions):

    * ``"linear"``: ``f_i / factor`` (positions interpolated);
    * ``"base"``: ``base * factor^(r / (r - 2))``, which divides the lowest frequency by ``factor`` and keeps the
      highest;
    * ``"ramp"``: by parts: pairs that turn more than ``high_turns`` times within ``original_len`` keep their
      frequency, those below ``low_turns`` turns are divided by ``factor``, a linear ramp between; the turned
      values grow by ``0.1 ln(factor) + 1``, the amplitude.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be positive and even")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}")
    if not (math.isfinite(base) and base > 0.0) or not (math.isfinite(factor) and factor > 0.0):
        raise ValueError("base and factor must be positive and finite")
    if scaling == "ramp" and (original_len <= 0 or not low_turns < high_turns):
        raise ValueError("ramp scaling needs original_len > 0 and low_turns < high_turns")
    if scaling == "base":
        if rotary_dim <= 2:
            raise ValueError("base scaling needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    amplitude = 1.0
    steps = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        if scaling == "linear":
            f /= factor
        elif scaling == "ramp":
            keep = (original_len * f / (2.0 * math.pi) - low_turns) / (high_turns - low_turns)
            keep = min(1.0, max(0.0, keep))
            f = f * keep + f / factor * (1.0 - keep)
        # Whole turns fall away; the fraction as a signed 64-bit integer.
        turn = math.ldexp(math.fmod(f / (2.0 * math.pi), 1.0), 64)
        step = int(round(turn)) % (1 << 64)
        steps.append(step - (1 << 64) if step >= 1 << 63 else step)
    if scaling == "ramp" and factor > 1.0:
        amplitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(steps, dtype=torch.int64, device=device), amplitude


# The checks below run on every call of a decoding loop: one comparison each
# where all is well, the message only when not.
def _heads3(name: str, t: torch.Tensor, rows: int, heads: int, hd: int, dtype: torch.dtype) -> tuple:
    if t.shape != (rows, heads, hd):
        raise ValueError(f"{name} must be [{rows}, {heads}, {hd}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must share the other tensors' dtype {dtype}")
    st = t.stride()
    if st[2] != 1 and hd > 1:
        raise ValueError(f"{name} must be contiguous in head_dim")
    return st


def _dims3(name: str, t: torch.Tensor) -> Tuple[int, int, int]:
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(shape)}")
    return shape


def _int_vector(name: str, t: torch.Tensor, n: int, dtype: torch.dtype = torch.int32) -> None:
    if t.shape != (n,) or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype).replace('torch.', '')} [{n}] tensor")


def _check_cache(k_cache, v_cache, block_table, batch: int, hd: int, dtype: torch.dtype) -> tuple:
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape or shape[3] != hd:
        raise ValueError(f"k_cache and v_cache must be [pages, kv_heads, page_size, {hd}] of one shape")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError(f"the caches must share the other tensors' dtype {dtype}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and hd > 1:
        raise ValueError("the caches must be contiguous in head_dim")
    table = block_table.shape
    if len(table) != 2 or table[0] != batch or block_table.dtype != torch.int32:
        raise ValueError("block_table must be an int32 [batch, max_pages] tensor")
    ld, unit = block_table.stride()
    if unit != 1 and table[1] > 1:
        raise ValueError("block_table rows must be contiguous")
    return ks, vs, (shape[0], shape[1], shape[2], table[1], ld)


def _starts(cu_seqlens: torch.Tensor) -> int:
    shape = cu_seqlens.shape
    if len(shape) != 1 or shape[0] < 1 or cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous int32 [batch + 1] tensor")
    return shape[0] - 1


def _one_device(first: torch.Tensor, *rest: Optional[torch.Tensor]) -> int:
    at = first.get_device()  # -1 on the CPU
    if at < 0:
        _require_cuda(first)
    for t in rest:
        if t is not None and t.get_device() != at:
            _require_cuda(t)
            raise ValueError(f"tensors on two devices ({first.device} and {t.device})")
    return at


def _launch_on(at: int, fn: str, args: tuple, keep: tuple, info) -> None:
    """``_launch`` on the current stream of device ``at``; ``info`` is called when a recording is active."""
    if at != torch.cuda.current_device():
        with torch.cuda.device(at):
            _launch_on(at, fn, args, keep, info)
        return
    code = getattr(_lib, fn)(*args, torch._C._cuda_getCurrentRawStream(at))
    if code != TX_OK:
        _check(fn, code)
    if _recorder is not None:
        _recorder.append(Launch(fn, args, keep, info()))


_NO_STRIDES = (0, 0, 0)


def rotary_append(
    q: Optional[torch.Tensor],
    k: torch.Tensor,
    v: Optional[torch.Tensor],
    steps: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    kv_lens: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    k_cache: Optional[torch.Tensor] = None,
    v_cache: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    amplitude: float = 1.0,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Rotary positions on packed q ``[T, heads, hd]`` and k ``[T, kv_heads, hd]``, and with a cache the
    turned k and v written into its pages (``tx_rotary_append``).  Returns ``(q_out, k_out)``.

    ``steps``, ``amplitude``: from :func:`rotary_steps`; its length is half the rotary dim.  A row's position is
    ``positions[t]`` (int64), by default its key index ``kv_lens[b] - n + i`` (``i`` without ``kv_lens``).  The
    caches are ``[pages, kv_heads, page_size, hd]`` views of any strides (a cache kept token by token passes
    ``.transpose(1, 2)``); ``kv_lens`` counts the new tokens already.  q_out and k_out may be q and k
    themselves; k_out is made when omitted only where there is no cache (else it is None).  Rows outside every
    sequence are left as they were (in a tensor made here: undefined)."""
    t, kvh, hd = _dims3("k", k)
    dtype = k.dtype
    ks = _heads3("k", k, t, kvh, hd, dtype)
    qs = qos = kos = vs = kcs = vcs = _NO_STRIDES
    batch = _starts(cu_seqlens)
    half = steps.shape[0] if steps.dim() == 1 else 0
    if not 0 < 2 * half <= hd or steps.dtype != torch.int64 or not steps.is_contiguous():
        raise ValueError(f"steps must be a contiguous int64 [rotary_dim / 2] tensor with rotary_dim <= {hd}")
    heads = kvh
    if q is not None:
        heads = _dims3("q", q)[1]
        qs = _heads3("q", q, t, heads, hd, dtype)
        if q_out is not None:
            qos = _heads3("q_out", q_out, t, heads, hd, dtype)
    elif q_out is not None:
        raise ValueError("q_out without q")
    if k_out is not None:
        kos = _heads3("k_out", k_out, t, kvh, hd, dtype)
    if kv_lens is not None:
        _int_vector("kv_lens", kv_lens, batch)
    if positions is not None:
        _int_vector("positions", positions, t, torch.int64)
    pages = page_size = max_pages = table_ld = 0
    if k_cache is not None or v_cache is not None:
        if k_cache is None or v_cache is None or block_table is None or kv_lens is None or v is None:
            raise ValueError("a cache needs k_cache, v_cache, block_table, kv_lens and v")
        vs = _heads3("v", v, t, kvh, hd, dtype)
        kcs, vcs, (pages, cache_heads, page_size, max_pages, table_ld) = _check_cache(k_cache, v_cache, block_table, batch,
                                                                                     hd, dtype)
        if cache_heads != kvh:
            raise ValueError("the caches must hold k's heads")
    else:
        block_table = v = None
    at = _one_device(k, q, v, steps, cu_seqlens, kv_lens, positions, block_table, k_cache, v_cache, q_out, k_out)
    load_library()
    if q is not None and q_out is None:
        q_out = torch.empty((t, heads, hd), dtype=dtype, device=k.device)
        qos = (heads * hd, hd, 1)
    if k_cache is None and k_out is None:
        k_out = torch.empty((t, kvh, hd), dtype=dtype, device=k.device)
        kos = (kvh * hd, hd, 1)
    if t == 0 or batch == 0:
        return q_out, k_out
    # The strides in one array, kept with the launch, and their addresses in it.
    st = array.array("q", (*qs, *qos, *ks, *kos, *vs, *kcs, *vcs))
    sa = st.buffer_info()[0]
    cached = k_cache is not None
    args = (q.data_ptr() if q is not None else None, sa, q_out.data_ptr() if q_out is not None else None, sa + 24,
            k.data_ptr(), sa + 48, k_out.data_ptr() if k_out is not None else None, sa + 72,
            v.data_ptr() if cached else None, sa + 96, k_cache.data_ptr() if cached else None, sa + 120,
            v_cache.data_ptr() if cached else None, sa + 120 + 8 * len(kcs), steps.data_ptr(),
            positions.data_ptr() if positions is not None else None, cu_seqlens.data_ptr(),
            kv_lens.data_ptr() if kv_lens is not None else None, block_table.data_ptr() if cached else None, table_ld,
            t, batch, heads, kvh, hd, 2 * half, pages, page_size, max_pages, float(amplitude), 1 if interleaved else 0,
            _DT.get(dtype, -1))
    _launch_on(at, "tx_rotary_append", args,
               (q, k, v, steps, cu_seqlens, kv_lens, positions, block_table, k_cache, v_cache, q_out, k_out, st),
               lambda: {"op": "rotary_append", "tokens": t, "heads": heads, "kv_heads": kvh, "head_dim": hd,
                        "cache": k_cache is not None})
    return q_out, k_out


def flash_attn_packed(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: float,
    causal: bool,
    *,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of packed sequences: q ``[T, heads, hd]``, k and v ``[T, kv_heads, hd]`` (strided views, e.g.
    columns of one projection), sequence b in rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` (int32, on the
    device; not read by the host).  Query head h reads K/V head ``h // (heads // kv_heads)``.  Returns out
    ``[T, heads, hd]``; rows outside every sequence are left as they were (``tx_flash_attn_packed``)."""
    t, heads, hd = _dims3("q", q)
    dtype = q.dtype
    qs = _heads3("q", q, t, heads, hd, dtype)
    kvh = _dims3("k", k)[1]
    ks = _heads3("k", k, t, kvh, hd, dtype)
    vs = _heads3("v", v, t, kvh, hd, dtype)
    if kvh <= 0 or heads % kvh:
        raise ValueError(f"{kvh} K/V heads do not divide {heads} query heads")
    batch = _starts(cu_seqlens)
    if out is not None:
        os_ = _heads3("out", out, t, heads, hd, dtype)
    at = _one_device(q, k, v, cu_seqlens, out)
    load_library()
    if out is None:
        out = torch.empty((t, heads, hd), dtype=dtype, device=q.device)
        os_ = (heads * hd, hd, 1)
    if t == 0 or batch == 0:
        return out
    st = array.array("q", (*qs, *ks, *vs, *os_))
    sa = st.buffer_info()[0]
    args = (q.data_ptr(), sa, k.data_ptr(), sa + 24, v.data_ptr(), sa + 48, out.data_ptr(), sa + 72,
            cu_seqlens.data_ptr(), t, batch, heads, kvh, hd, float(scale), 1 if causal else 0, _DT.get(dtype, -1))
    _launch_on(at, "tx_flash_attn_packed", args, (q, k, v, out, cu_seqlens, st),
               lambda: {"op": "flash_attn_packed", "tokens": t, "batch": batch, "heads": heads, "kv_heads": kvh,
                        "head_dim": hd, "causal": bool(causal)})
    return out


def flash_attn_paged_workspace(tokens: int, batch: int, heads: int, kv_heads: int, head_dim: int, page_size: int,
                               max_pages: int, max_q_len: int = 0) -> int:
    """fp32 values of workspace that :func:`flash_attn_paged` needs for these sizes (0: none): at most ``tokens * heads
    * parts * (head_dim + 2)`` with up to ``256 / kv_heads`` parts of the keys, 512 at head dim 64 (``tx_api.h``)."""
    n = ctypes.c_int64(0)
    _check("tx_flash_attn_paged_workspace",
           load_library().tx_flash_attn_paged_workspace(tokens, batch, heads, kv_heads, head_dim, page_size, max_pages,
                                                        max_q_len, ctypes.addressof(n)))
    return n.value


def flash_attn_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    kv_lens: torch.Tensor,
    scale: float,
    causal: bool = True,
    *,
    max_q_len: int = 0,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of each sequence's new tokens over its paged cache (``tx_flash_attn_paged``): one token per
    sequence when decoding, a chunk of a prompt, or any mixture.  q ``[T, heads, hd]`` packed by ``cu_seqlens``;
    caches ``[pages, kv_heads, page_size, hd]`` (any strides) that already hold the new tokens; ``kv_lens``
    counts them.  Row i of n sees the keys up to its own, ``kv_lens[b] - n + i``, when causal, else all of them.
    A page index outside ``[0, pages)`` makes the rows that need it NaN.

    ``max_q_len``: a bound on the rows of one sequence that the caller knows (0: T), to choose the kernel by.
    ``workspace``: fp32, at least :func:`flash_attn_paged_workspace` values, made here when omitted (and kept by a
    captured graph); calls that overlap in time need one each, others may share one."""
    t, heads, hd = _dims3("q", q)
    dtype = q.dtype
    qs = _heads3("q", q, t, heads, hd, dtype)
    batch = _starts(cu_seqlens)
    _int_vector("kv_lens", kv_lens, batch)
    ks, vs, (pages, kvh, page_size, max_pages, table_ld) = _check_cache(k_cache, v_cache, block_table, batch, hd, dtype)
    if kvh <= 0 or heads % kvh:
        raise ValueError(f"{kvh} K/V heads do not divide {heads} query heads")
    if out is not None:
        os_ = _heads3("out", out, t, heads, hd, dtype)
    at = _one_device(q, k_cache, v_cache, block_table, cu_seqlens, kv_lens, out, workspace)
    load_library()
    if out is None:
        out = torch.empty((t, heads, hd), dtype=dtype, device=q.device)
        os_ = (heads * hd, hd, 1)
    if t == 0 or batch == 0:
        return out
    if workspace is None:
        if at != torch.cuda.current_device():
            with torch.cuda.device(at):
                need = flash_attn_paged_workspace(t, batch, heads, kvh, hd, page_size, max_pages, max_q_len)
        else:
            need = flash_attn_paged_workspace(t, batch, heads, kvh, hd, page_size, max_pages, max_q_len)
        if need > 0:
            workspace = torch.empty(need, dtype=torch.float32, device=q.device)
    elif workspace.dtype != torch.float32 or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous fp32")
    st = array.array("q", (*qs, *ks, *vs, *os_))
    sa = st.buffer_info()[0]
    args = (q.data_ptr(), sa, k_cache.data_ptr(), sa + 24, v_cache.data_ptr(), sa + 56, out.data_ptr(), sa + 88,
            cu_seqlens.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(), table_ld, t, batch, heads, kvh,
            hd, pages, page_size, max_pages, max_q_len, float(scale), 1 if causal else 0,
            workspace.data_ptr() if workspace is not None else None, 0 if workspace is None else workspace.numel(),
            _DT.get(dtype, -1))
    _launch_on(at, "tx_flash_attn_paged", args,
               (q, k_cache, v_cache, out, cu_seqlens, kv_lens, block_table, workspace, st),
               lambda: {"op": "flash_attn_paged", "tokens": t, "batch": batch, "heads": heads, "kv_heads": kvh,
                        "head_dim": hd, "causal": bool(causal), "page_size": page_size})
    return out
