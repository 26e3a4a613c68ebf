"""Torch-facing wrappers of the decode-step entry points (libb200dec.so via ctypes).

Every function takes CUDA tensors the caller owns, checks shapes/dtypes on the host, launches
on torch's current stream and returns the output tensor(s).  Bad arguments raise ValueError
(the library's B2D_ERR_* status), CUDA / NCCL failures raise B2DError.  There is no CPU path:
calling these without the CUDA library or a GPU raises.

Reference mapping (LK = ios_kernels/kernels/unsloth__Llama-3.2-1B-Instruct/
kernel_metal_f16_20261024-1620): gemv* <- matvec_f16 / matvec_gate_up_silu
(LK/kernels.metal:106-173), rmsnorm <- LK/kernels.metal:71-89, paged_decode_attn <-
attention + rope_kv (LK/kernels.metal:182-305), lm_head_argmax <- argmax (:307-345).

A step with several rows per sequence (drafted tokens, prompt chunks) is paged_plan, then per layer
qk_norm_rope_append and paged_tree_attn, then token_logprobs.  These four run on the device and the
current stream of their tensors' device, keep nothing between calls and use no shared workspace.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import call, raise_status

_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16}
EPILOGUES = {
    "store": _lib.EPI_STORE,
    "add": _lib.EPI_ADD,
    "gelu_mul": _lib.EPI_GELU_MUL,
    "swiglu": _lib.EPI_SWIGLU,
}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _need_cuda(*ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("all tensors must be CUDA tensors (no CPU path exists)")
        if t is not None and not t.is_contiguous():
            raise ValueError("tensors must be contiguous")


@dataclass
class QWeight:
    """32-block quantized matrix: fmt 'q8' (q int8 [M, K]) or 'q4' (q uint8 [M, K/2]),
    scales fp16 [M, K/32].  See include/b200dec.h for the exact bit layout."""

    fmt: str
    q: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, int]:
        m = self.q.shape[0]
        k = self.q.shape[1] * (2 if self.fmt == "q4" else 1)
        return m, k

    @property
    def dtype_code(self) -> int:
        return _lib.Q8_32 if self.fmt == "q8" else _lib.Q4_32


class Workspace:
    """Zero-filled device scratch, grown on demand and reused (kernels leave it re-zeroed)."""

    def __init__(self):
        self._buf: dict[int, torch.Tensor] = {}

    def get(self, nbytes: int, device: torch.device) -> torch.Tensor:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        b = self._buf.get(idx)
        if b is None or b.numel() < nbytes:
            b = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            self._buf[idx] = b
        return b


_WS_ATTN = Workspace()
_WS_ARGMAX = Workspace()


def gemv(
    W,
    x: torch.Tensor,
    *,
    gamma: torch.Tensor | None = None,
    eps: float = 1e-6,
    epilogue: str = "store",
    W_up=None,
    aux: torch.Tensor | None = None,
    y: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """y[b] = epilogue(W @ rmsnorm?(x[b])) for x [batch, K] (or [K]); W is a fp32/fp16 tensor
    [M, K] or a QWeight.  For 'add', y is read and updated in place."""
    squeeze = x.dim() == 1
    x2 = x.unsqueeze(0) if squeeze else x
    if isinstance(W, QWeight):
        wq, ws, wcode = W.q, W.scales, W.dtype_code
        M, K = W.shape
    else:
        if W.dtype not in _DT:
            raise ValueError(f"unsupported weight dtype {W.dtype}")
        wq, ws, wcode = W, None, _DT[W.dtype]
        M, K = W.shape
    if x2.dtype not in _DT or x2.shape[-1] != K:
        raise ValueError(f"x must be fp32/fp16 [batch, {K}]")
    up_q = up_s = None
    if W_up is not None:
        if isinstance(W_up, QWeight):
            up_q, up_s = W_up.q, W_up.scales
        else:
            up_q = W_up
    batch = x2.shape[0]
    if y is None:
        if epilogue == "add":
            raise ValueError("epilogue 'add' needs y")
        y = torch.empty(batch, M, dtype=out_dtype, device=x.device)
    y2 = y.unsqueeze(0) if y.dim() == 1 else y
    _need_cuda(wq, ws, up_q, up_s, x2, gamma, aux, y2)
    if y2.dtype not in _DT or tuple(y2.shape) != (batch, M):
        raise ValueError(f"y must be fp32/fp16 [{batch}, {M}]")
    call(
        "b2d_gemv",
        wcode,
        _ptr(wq),
        _ptr(ws),
        _ptr(up_q),
        _ptr(up_s),
        _DT[x2.dtype],
        _ptr(x2),
        K,
        _ptr(gamma),
        float(eps),
        EPILOGUES[epilogue],
        _DT[y2.dtype],
        _ptr(y2),
        M,
        _ptr(aux),
        M,
        K,
        batch,
        _stream(),
    )
    return y2[0] if squeeze and y.dim() == 1 else y


_MMA_FMT = {"f16": _lib.F16, "q8": _lib.Q8_32, "q4": _lib.Q4_32, "int8_b1": 4}


def gemv_mma_formats(formats: set[str] | None = None) -> set[str]:
    """Weight formats ('f16', 'q8', 'q4') that gemv() runs on the tensor-core GEMV, plus
    'int8_b1' (a quantized single token on the integer tensor cores); `formats` replaces the set
    (process-wide).  Returns the previous set."""
    mask = -1 if formats is None else sum(1 << _MMA_FMT[f] for f in formats)
    prev = _lib.lib().b2d_gemv_mma_formats(mask)
    return {f for f, d in _MMA_FMT.items() if (prev >> d) & 1}


def gemv_f32(W: torch.Tensor, x: torch.Tensor, y: torch.Tensor | None = None) -> torch.Tensor:
    """Config 1: fp32 y = W @ x (x [K])."""
    M, K = W.shape
    if W.dtype != torch.float32 or x.dtype != torch.float32 or x.shape != (K,):
        raise ValueError("gemv_f32 needs fp32 W [M, K] and x [K]")
    y = torch.empty(M, dtype=torch.float32, device=x.device) if y is None else y
    _need_cuda(W, x, y)
    call("b2d_gemv_f32", W.data_ptr(), x.data_ptr(), y.data_ptr(), M, K, _stream())
    return y


def dequant(Wq: QWeight) -> torch.Tensor:
    """Exact fp32 dequantized weights [M, K]."""
    M, K = Wq.shape
    w = torch.empty(M, K, dtype=torch.float32, device=Wq.q.device)
    _need_cuda(Wq.q, Wq.scales)
    name = "b2d_dequant_q8_32" if Wq.fmt == "q8" else "b2d_dequant_q4_32"
    call(name, Wq.q.data_ptr(), Wq.scales.data_ptr(), w.data_ptr(), M, K, _stream())
    return w


def lm_head_argmax(
    W: torch.Tensor,
    x: torch.Tensor,
    gamma: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    index_offset: int = 0,
    return_logits: bool = False,
    return_max: bool = False,
):
    """tokens[b] = argmax(W @ rmsnorm?(x[b])) + index_offset (fp16 W [V, K], fp32 x [B, K])."""
    V, K = W.shape
    x2 = x.unsqueeze(0) if x.dim() == 1 else x
    B = x2.shape[0]
    if W.dtype != torch.float16 or x2.dtype != torch.float32 or x2.shape[1] != K:
        raise ValueError("lm_head_argmax needs fp16 W [V, K] and fp32 x [B, K]")
    tokens = torch.empty(B, dtype=torch.int32, device=x.device)
    logits = torch.empty(B, V, dtype=torch.float32, device=x.device) if return_logits else None
    mx = torch.empty(B, dtype=torch.float32, device=x.device) if return_max else None
    _need_cuda(W, x2, gamma)
    nbytes = _lib.lib().b2d_lm_head_argmax_workspace_bytes(V, B)
    ws = _WS_ARGMAX.get(nbytes, x.device)
    call(
        "b2d_lm_head_argmax",
        W.data_ptr(),
        x2.data_ptr(),
        K,
        _ptr(gamma),
        float(eps),
        V,
        K,
        B,
        int(index_offset),
        _ptr(logits),
        tokens.data_ptr(),
        _ptr(mx),
        ws.data_ptr(),
        ws.numel(),
        _stream(),
    )
    out = [tokens]
    if return_logits:
        out.append(logits)
    if return_max:
        out.append(mx)
    return out[0] if len(out) == 1 else tuple(out)


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    x2 = x.unsqueeze(0) if x.dim() == 1 else x
    y = torch.empty_like(x2)
    _need_cuda(x2, w)
    call("b2d_rmsnorm", x2.data_ptr(), w.data_ptr(), y.data_ptr(), x2.shape[0], x2.shape[1], float(eps), _stream())
    return y.view_as(x)


def embed_f16(E: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    V, Dm = E.shape
    x = torch.empty(tokens.numel(), Dm, dtype=torch.float32, device=E.device)
    _need_cuda(E, tokens)
    call("b2d_embed_f16", E.data_ptr(), tokens.data_ptr(), x.data_ptr(), Dm, tokens.numel(), _stream())
    return x


def argmax_f32(logits: torch.Tensor, index_offset: int = 0) -> torch.Tensor:
    l2 = logits.unsqueeze(0) if logits.dim() == 1 else logits
    out = torch.empty(l2.shape[0], dtype=torch.int32, device=logits.device)
    _need_cuda(l2)
    call("b2d_argmax_f32", l2.data_ptr(), l2.shape[1], l2.shape[0], out.data_ptr(), int(index_offset), _stream())
    return out


def argmax_combine(vals: torch.Tensor, idxs: torch.Tensor) -> torch.Tensor:
    """vals/idxs [n_parts, batch] -> tokens [batch] (ties -> lowest index)."""
    out = torch.empty(vals.shape[1], dtype=torch.int32, device=vals.device)
    _need_cuda(vals, idxs)
    call("b2d_argmax_combine", vals.data_ptr(), idxs.data_ptr(), vals.shape[0], vals.shape[1], out.data_ptr(), _stream())
    return out


def inv_freq(head_dim: int, theta: float) -> torch.Tensor:
    """RoPE inverse frequencies (host double -> fp32), as a CPU tensor."""
    out = (ctypes.c_float * (head_dim // 2))()
    call("b2d_inv_freq", head_dim, float(theta), ctypes.addressof(out))
    return torch.tensor(list(out), dtype=torch.float32)


def rope_kv_append(qkv, k_pages, v_pages, block_table, ctx_lens, inv_freq_dev, n_heads, n_kv_heads, head_dim):
    """Rotate q in place in qkv and write rotated k / v at pos = ctx_lens[b] (paged)."""
    _need_cuda(qkv, k_pages, v_pages, block_table, ctx_lens, inv_freq_dev)
    call(
        "b2d_rope_kv_append",
        qkv.data_ptr(),
        _DT[qkv.dtype],
        qkv.shape[1],
        k_pages.data_ptr(),
        v_pages.data_ptr(),
        block_table.data_ptr(),
        block_table.shape[1],
        k_pages.shape[0],
        ctx_lens.data_ptr(),
        inv_freq_dev.data_ptr(),
        n_heads,
        n_kv_heads,
        head_dim,
        qkv.shape[0],
        _stream(),
    )


def to_f16x2(x: torch.Tensor) -> torch.Tensor:
    """fp32 [B, K] -> the B2D_F16X2 form fp16 [2, B, K]: hi = fp16(x), lo = fp16(x - hi)."""
    hi = x.to(torch.float16)
    return torch.stack([hi, (x - hi.float()).to(torch.float16)])


def from_f16x2(t: torch.Tensor) -> torch.Tensor:
    """fp16 [2, B, K] hi + lo planes -> fp32 [B, K]."""
    return t[0].float() + t[1].float()


def _is_x2(t: torch.Tensor | None) -> bool:
    return t is not None and t.dim() == 3 and t.shape[0] == 2 and t.dtype == torch.float16


def attn_workspace_bytes(batch, n_heads, n_kv_heads, head_dim, max_ctx) -> int:
    return int(_lib.lib().b2d_paged_attn_workspace_bytes(batch, n_heads, n_kv_heads, head_dim, max_ctx))


def paged_decode_attn(
    qkv: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    ctx_lens: torch.Tensor,
    inv_freq_dev: torch.Tensor | None,
    n_heads: int,
    n_kv_heads: int,
    head_dim: int,
    max_ctx: int,
    *,
    scale: float = 0.0,
    window: int = 0,
    append: bool = True,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Ragged paged decode attention; see include/b200dec.h b2d_paged_decode_attn.  `out` may be
    fp16 [2, B, Hq*HD]: the output as B2D_F16X2 hi + lo planes."""
    B = qkv.shape[0]
    if out is None:
        out = torch.empty(B, n_heads * head_dim, dtype=out_dtype, device=qkv.device)
    out_dt = _lib.F16X2 if _is_x2(out) else _DT[out.dtype]
    nbytes = attn_workspace_bytes(B, n_heads, n_kv_heads, head_dim, max_ctx)
    ws = workspace if workspace is not None else _WS_ATTN.get(nbytes, qkv.device)
    _need_cuda(qkv, k_pages, v_pages, block_table, ctx_lens, inv_freq_dev, out, ws)
    if block_table.dtype != torch.int32 or ctx_lens.dtype != torch.int32:
        raise ValueError("block_table and ctx_lens must be int32")
    call(
        "b2d_paged_decode_attn",
        qkv.data_ptr(),
        _DT[qkv.dtype],
        qkv.shape[1],
        k_pages.data_ptr(),
        v_pages.data_ptr(),
        block_table.data_ptr(),
        block_table.shape[1],
        k_pages.shape[0],
        ctx_lens.data_ptr(),
        _ptr(inv_freq_dev),
        n_heads,
        n_kv_heads,
        head_dim,
        B,
        max_ctx,
        float(scale),
        int(window),
        1 if append else 0,
        out.data_ptr(),
        out_dt,
        out.shape[-1],
        ws.data_ptr(),
        ws.numel(),
        _stream(),
    )
    return out


_WS_TC = Workspace()
_TC_EPI = {"store": _lib.EPI_STORE, "add": _lib.EPI_ADD, "gelu_mul": _lib.EPI_GELU_MUL, "swiglu": _lib.EPI_SWIGLU, "argmax": _lib.EPI_ARGMAX, "silu_mul": _lib.EPI_SILU_MUL}


@dataclass
class TcPacked:
    """fp16 weights [M, K] in the tensor-core tile layout (b2d_tc_pack_f16): 16 KB tiles of 128
    rows x 64 columns, already in the MMA's swizzled shared-memory image."""

    buf: torch.Tensor  # uint8 [b2d_tc_packed_bytes(M, K)]
    M: int
    K: int

    @property
    def shape(self) -> tuple[int, int]:
        return self.M, self.K


def pack_tc(W: torch.Tensor) -> TcPacked:
    """Repack fp16 W [M, K] (row-major) into the tensor-core tile layout."""
    if W.dtype != torch.float16 or W.dim() != 2 or W.stride(1) != 1:
        raise ValueError("pack_tc needs fp16 W [M, K] with unit column stride")
    M, K = W.shape
    buf = torch.empty(_lib.lib().b2d_tc_packed_bytes(M, K), dtype=torch.uint8, device=W.device)
    _need_cuda(W, buf)
    call("b2d_tc_pack_f16", W.data_ptr(), W.stride(0), M, K, buf.data_ptr(), _stream())
    return TcPacked(buf, M, K)


def tc_workspace_bytes(M: int, K: int, batch: int, epilogue: str = "store") -> int:
    return int(_lib.lib().b2d_gemm_tc_workspace_bytes(M, K, batch, _TC_EPI[epilogue]))


def gemm_tc(
    W: torch.Tensor | TcPacked,
    X: torch.Tensor,
    *,
    epilogue: str = "store",
    W_up: torch.Tensor | TcPacked | None = None,
    aux: torch.Tensor | None = None,
    y: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
    index_offset: int = 0,
    return_logits: bool = False,
    workspace: torch.Tensor | None = None,
):
    """Tensor-core batched GEMV (tcgen05): y[b] = epilogue(W @ X[b]) for fp16 W [M, K] and fp16
    X [batch <= 32, K], or X fp16 [2, batch, K]: fp32-precision activations as B2D_F16X2 hi + lo
    planes (to_f16x2).  y may be fp16 [2, batch, M] (B2D_F16X2 output) as well.  For 'argmax'
    returns tokens (and logits if asked).  W (and W_up) may be row-major or packed by pack_tc."""
    M, K = W.shape
    x2 = _is_x2(X)
    B = X.shape[-2]
    packed = isinstance(W, TcPacked)
    if packed != (W_up is None or isinstance(W_up, TcPacked)) and W_up is not None:
        raise ValueError("W and W_up must both be packed or both row-major")
    if (not packed and W.dtype != torch.float16) or X.dtype != torch.float16 or X.shape[-1] != K:
        raise ValueError("gemm_tc needs fp16 W [M, K] and fp16 X [batch, K] (or [2, batch, K])")
    if packed and x2:
        raise ValueError("hi/lo activations run on row-major weights")
    Wt = W.buf if packed else W
    Wu = (W_up.buf if packed else W_up) if W_up is not None else None
    ws = workspace if workspace is not None else _WS_TC.get(tc_workspace_bytes(M, K, B, epilogue), X.device)
    tokens = logits = None
    if epilogue == "argmax":
        tokens = torch.empty(B, dtype=torch.int32, device=X.device)
        logits = torch.empty(B, M, dtype=torch.float32, device=X.device) if return_logits else None
        ydt = _lib.F32
    else:
        if y is None:
            if epilogue == "add":
                raise ValueError("epilogue 'add' needs y")
            y = torch.empty(B, M, dtype=out_dtype, device=X.device)
        if _is_x2(y) and tuple(y.shape) == (2, B, M):
            ydt = _lib.F16X2
        elif y.dtype in _DT and tuple(y.shape) == (B, M):
            ydt = _DT[y.dtype]
        else:
            raise ValueError(f"y must be fp32/fp16 [{B}, {M}] or fp16 [2, {B}, {M}]")
    _need_cuda(Wt, X, Wu, aux, y, ws, tokens, logits)
    head = () if packed else (_lib.F16X2 if x2 else _lib.F16,)
    call(
        "b2d_gemm_tc_packed" if packed else "b2d_gemm_tc_ex",
        *head,
        Wt.data_ptr(),
        _ptr(Wu),
        X.data_ptr(),
        K,
        _TC_EPI[epilogue],
        ydt,
        _ptr(y),
        M,
        _ptr(aux),
        M,
        K,
        B,
        _ptr(logits),
        _ptr(tokens),
        None,
        int(index_offset),
        ws.data_ptr(),
        ws.numel(),
        _stream(),
    )
    if epilogue == "argmax":
        return (tokens, logits) if return_logits else tokens
    return y


def gemm_tc_q(
    Wq: QWeight,
    X: torch.Tensor,
    *,
    epilogue: str = "store",
    aux: torch.Tensor | None = None,
    y: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Tensor-core batched GEMV over 32-block quantized weights: y[b] = epilogue(W @ X[b]) with
    W = scale * q dequantized in shared memory to fp16 (the MMA operand), fp16 X [batch <= 32, K]
    or hi + lo planes fp16 [2, batch, K].  Epilogues 'store', 'add', 'gelu_mul'."""
    M, K = Wq.shape
    x2 = _is_x2(X)
    B = X.shape[-2]
    if X.dtype != torch.float16 or X.shape[-1] != K:
        raise ValueError("gemm_tc_q needs fp16 X [batch, K] (or [2, batch, K])")
    if epilogue not in ("store", "add", "gelu_mul", "silu_mul"):
        raise ValueError(f"gemm_tc_q: unsupported epilogue {epilogue!r}")
    ws = workspace if workspace is not None else _WS_TC.get(tc_workspace_bytes(M, K, B, epilogue), X.device)
    if y is None:
        if epilogue == "add":
            raise ValueError("epilogue 'add' needs y")
        y = torch.empty(B, M, dtype=out_dtype, device=X.device)
    if y.dtype not in _DT or tuple(y.shape) != (B, M):
        raise ValueError(f"y must be fp32/fp16 [{B}, {M}]")
    _need_cuda(Wq.q, Wq.scales, X, aux, y, ws)
    call(
        "b2d_gemm_tc_q_ex",
        _lib.F16X2 if x2 else _lib.F16,
        Wq.dtype_code,
        Wq.q.data_ptr(),
        Wq.scales.data_ptr(),
        X.data_ptr(),
        K,
        _TC_EPI[epilogue],
        _DT[y.dtype],
        y.data_ptr(),
        M,
        _ptr(aux),
        M,
        K,
        B,
        ws.data_ptr(),
        ws.numel(),
        _stream(),
    )
    return y


def _ptr_array(ts) -> ctypes.Array:
    return (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])


def tp_allreduce_add_rmsnorm(
    parts: list[torch.Tensor],
    sigs: list[torch.Tensor],
    epochs: torch.Tensor,
    rank: int,
    x: torch.Tensor,
    err: torch.Tensor,
    gamma: torch.Tensor | None = None,
    eps: float = 1e-5,
    out16: torch.Tensor | None = None,
    slot0: int = 0,
    timeout_ns: int = 10_000_000_000,
) -> torch.Tensor | None:
    """x += parts[0] + ... + parts[tp-1] (rank order) after a per-row barrier on the ranks'
    signal arrays; returns fp16 rmsnorm(x) * gamma if gamma is given.  parts: the ranks'
    partials [rows, D] fp32 as mapped in this process; sigs: the ranks' uint32 signal arrays;
    epochs: this rank's uint32 epoch counters; err: device int32 error word (a barrier that
    times out writes B2D_ERR_TIMEOUT there and leaves its row unchanged)."""
    rows, D = x.shape
    if gamma is not None and out16 is None:
        out16 = torch.empty(rows, D, dtype=torch.float16, device=x.device)
    _need_cuda(x, err, epochs, gamma, out16, *parts, *sigs)
    call(
        "b2d_tp_allreduce_add_rmsnorm",
        ctypes.cast(_ptr_array(parts), ctypes.c_void_p),
        ctypes.cast(_ptr_array(sigs), ctypes.c_void_p),
        epochs.data_ptr(),
        rank,
        len(parts),
        slot0,
        x.data_ptr(),
        _ptr(gamma),
        float(eps),
        _ptr(out16),
        D,
        rows,
        int(timeout_ns),
        err.data_ptr(),
        _stream(),
    )
    return out16


def tp_argmax_gather(
    vals: list[torch.Tensor],
    idxs: list[torch.Tensor],
    sigs: list[torch.Tensor],
    epochs: torch.Tensor,
    rank: int,
    slot: int,
    err: torch.Tensor,
    timeout_ns: int = 10_000_000_000,
) -> torch.Tensor:
    """Best (value, index) over the ranks' LM-head candidates per token (ties -> lower index)."""
    B = vals[0].numel()
    tokens = torch.empty(B, dtype=torch.int32, device=vals[0].device)
    _need_cuda(tokens, epochs, err, *vals, *idxs, *sigs)
    call(
        "b2d_tp_argmax_gather",
        ctypes.cast(_ptr_array(vals), ctypes.c_void_p),
        ctypes.cast(_ptr_array(idxs), ctypes.c_void_p),
        ctypes.cast(_ptr_array(sigs), ctypes.c_void_p),
        epochs.data_ptr(),
        rank,
        len(vals),
        slot,
        B,
        tokens.data_ptr(),
        int(timeout_ns),
        err.data_ptr(),
        _stream(),
    )
    return tokens


def add_rmsnorm_f16(x: torch.Tensor, gamma: torch.Tensor, eps: float, p: torch.Tensor | None = None, x2: bool = False) -> torch.Tensor:
    """x += p (if given, in place); returns fp16 rmsnorm(x) * gamma, or with x2 the B2D_F16X2
    hi + lo planes fp16 [2, rows, D]."""
    out = torch.empty(((2,) if x2 else ()) + tuple(x.shape), dtype=torch.float16, device=x.device)
    _need_cuda(x, gamma, p)
    call(
        "b2d_add_rmsnorm", x.data_ptr(), _ptr(p), gamma.data_ptr(), float(eps), _lib.F16X2 if x2 else _lib.F16,
        out.data_ptr(), x.shape[0], x.shape[1], _stream(),
    )
    return out


# -- several rows per sequence: drafted tokens and prompt chunks ---------------------------------


def _check(name: str, t: torch.Tensor | None, dtypes, d: int, shape, rows: bool = False) -> None:
    """t (None passes) is on CUDA device d, of one of dtypes and of `shape`, contiguous (with rows: only
    each row is, at any row stride)."""
    if t is None or t.dtype in dtypes and t.get_device() == d and t.shape == shape and t.is_contiguous():
        return
    if not t.is_cuda or t.get_device() != d:
        raise ValueError(f"{name} must be a CUDA tensor on the device of the first one (no CPU path exists)")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has dtype {t.dtype}, expected one of {[str(x) for x in dtypes]}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {list(t.shape)}, expected {list(shape)}")
    if not rows:
        raise ValueError(f"{name} must be contiguous")
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name} needs contiguous rows that do not overlap")


def _on_gpu(t: torch.Tensor) -> int:
    """The CUDA device of a wrapper's first tensor."""
    d = t.get_device()
    if d < 0:
        raise ValueError("all tensors must be CUDA tensors (no CPU path exists)")
    return d


def _ld(t: torch.Tensor) -> int:
    """Row stride of a [rows, n] tensor whose rows do not overlap (a single row's says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _two_dims(name: str, t: torch.Tensor) -> None:
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, not {t.dim()}")


def _fits32(*args: int) -> None:
    """ctypes cuts an int to its low 32 bits without a word."""
    if max(args) > 0x7FFFFFFF or min(args) < -0x80000000:
        raise ValueError(f"an integer argument or row stride does not fit 32 bits: {max(args, key=abs)}")


# the current stream's handle without a Stream object around it (1.2 us less per call), where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda d: torch.cuda.current_stream(d).cuda_stream
)


@functools.cache
def _entry(name: str):
    return getattr(_lib.lib(), name)


def _call_on(d: int, name: str, *args) -> None:
    """The entry point with the current stream of CUDA device d as its last argument, on that device."""
    if d == torch.cuda.current_device():
        st = _entry(name)(*args, _raw_stream(d))
    else:
        with torch.cuda.device(d):
            st = _entry(name)(*args, _raw_stream(d))
    if st != _lib.OK:
        raise_status(name, st)


_I32, _I64, _F32, _F16 = (torch.int32,), (torch.int64,), (torch.float32,), (torch.float16,)
_FLOATS = (torch.float32, torch.float16)


@dataclass(slots=True)
class PagedPlan:
    """paged_plan()'s outputs for a batch of B requests and R rows.  Rows from cu_q[B] on belong to no
    request and are left as they were."""

    cu_q: torch.Tensor  # int32 [B + 1]: first row of each request, then their total
    slots: torch.Tensor  # int64 [R]: page * 16 + place in the page, -1 for none
    positions: torch.Tensor  # int32 [R]
    mask: torch.Tensor | None  # int32 [R, words]: bit j = row j of the request is an ancestor, or the row itself
    status: torch.Tensor  # int32 [B]: _lib.PLAN_OK, PLAN_PAGES, PLAN_TABLE, PLAN_ROWS or PLAN_TREE
    n_pages: torch.Tensor  # int32 [B]: pages each request has now
    n_free: torch.Tensor  # int32 [1]: pages left on the free stack

    @property
    def n_rows(self) -> torch.Tensor:
        """int32 [1], on the device: the number of rows in use (qk_norm_rope_append's n_rows)."""
        return self.cu_q[-1:]


def paged_plan(
    ctx_lens: torch.Tensor,
    q_lens: torch.Tensor,
    block_table: torch.Tensor,
    n_pages: torch.Tensor,
    free_pages: torch.Tensor,
    n_free: torch.Tensor,
    max_tokens: int,
    *,
    parents: torch.Tensor | None = None,
    mask_words: int = 0,
    out: PagedPlan | None = None,
) -> PagedPlan:
    """Pages, slots, positions and tree masks of a step that adds q_lens[b] rows to request b (a
    negative number ends it and gives its pages back); block_table and free_pages are updated in
    place, n_pages and n_free if `out` holds them.  A request with status != PLAN_OK was not served:
    its rows exist without slots, and what a step computes for them is to be dropped.  See
    include/b200dec.h b2d_paged_plan.  ctx_lens,
    q_lens, n_pages int32 [B]; block_table int32 [B, max_blocks]; free_pages int32 [capacity]; n_free
    int32 [1]; parents int32 [max_tokens] with mask_words (<= 8) words of 32 nodes per row.  A batch of
    no requests gives no rows; max_tokens is at least 1."""
    d, B = _on_gpu(ctx_lens), ctx_lens.numel()
    _two_dims("block_table", block_table)
    _fits32(max_tokens, mask_words)
    _check("ctx_lens", ctx_lens, _I32, d, (B,))
    _check("q_lens", q_lens, _I32, d, (B,))
    _check("block_table", block_table, _I32, d, (B, block_table.shape[1]))
    _check("n_pages", n_pages, _I32, d, (B,))
    _check("free_pages", free_pages, _I32, d, (free_pages.numel(),))
    _check("n_free", n_free, _I32, d, (1,))
    _check("parents", parents, _I32, d, (max_tokens,))
    if (parents is None) != (mask_words == 0):
        raise ValueError("parents and mask_words go together")
    if max_tokens < 1:
        raise ValueError("max_tokens must be at least 1 (a step without rows has buffers too)")
    if out is None:
        new = ctx_lens.new_empty
        out = PagedPlan(
            new(B + 1),
            new(max_tokens, dtype=torch.int64),
            new(max_tokens),
            new((max_tokens, mask_words)) if mask_words else None,
            new(B),
            new(B),
            new(1),
        )
    else:
        _check("out.cu_q", out.cu_q, _I32, d, (B + 1,))
        _check("out.slots", out.slots, _I64, d, (max_tokens,))
        _check("out.positions", out.positions, _I32, d, (max_tokens,))
        _check("out.status", out.status, _I32, d, (B,))
        _check("out.n_pages", out.n_pages, _I32, d, (B,))
        _check("out.n_free", out.n_free, _I32, d, (1,))
        if mask_words:
            if out.mask is None:
                raise ValueError("out.mask is missing")
            _check("out.mask", out.mask, _I32, d, (max_tokens, mask_words))
    if B == 0:  # no requests: no rows, and the free stack as it was
        out.cu_q.zero_()
        torch.clamp(n_free, 0, free_pages.numel(), out=out.n_free)
        return out
    _call_on(
        d,
        "b2d_paged_plan",
        ctx_lens.data_ptr(),
        q_lens.data_ptr(),
        _ptr(parents),
        block_table.data_ptr(),
        block_table.shape[1],
        n_pages.data_ptr(),
        free_pages.data_ptr(),
        free_pages.numel(),
        n_free.data_ptr(),
        B,
        max_tokens,
        mask_words,
        out.cu_q.data_ptr(),
        out.slots.data_ptr(),
        out.positions.data_ptr(),
        out.mask.data_ptr() if mask_words else None,
        out.status.data_ptr(),
        out.n_pages.data_ptr(),
        out.n_free.data_ptr(),
    )
    return out


def _check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, n_kv_heads: int, head_dim: int, d: int) -> None:
    _check("k_pages", k_pages, _F16, d, (*k_pages.shape[:1], n_kv_heads, 16, head_dim))
    _check("v_pages", v_pages, _F16, d, k_pages.shape)


def qk_norm_rope_append(
    qkv: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    inv_freq_dev: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    n_heads: int,
    n_kv_heads: int,
    head_dim: int,
    *,
    q_gamma: torch.Tensor | None = None,
    k_gamma: torch.Tensor | None = None,
    eps: float = 1e-6,
    v_norm: bool = False,
    n_rows: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """Per-head norms of q and k (where a gamma is given), rotation by positions and append of k and
    v to their slots, for rows of qkv [R, (Hq + 2 Hkv) * HD]; returns the rotated q [R, Hq * HD].
    See include/b200dec.h b2d_qk_norm_rope_append.  positions int32 [R], slots int64 [R] and n_rows
    (int32 [1], optional: rows in use) as paged_plan returns them."""
    _two_dims("qkv", qkv)
    d, R, nq = _on_gpu(qkv), qkv.shape[0], n_heads * head_dim
    _check("qkv", qkv, _FLOATS, d, (R, (n_heads + 2 * n_kv_heads) * head_dim), rows=True)
    if q_out is None:
        q_out = qkv.new_empty((R, nq), dtype=out_dtype)
    _check("q_out", q_out, _FLOATS, d, (R, nq), rows=True)
    _check("positions", positions, _I32, d, (R,))
    _check("slots", slots, _I64, d, (R,))
    _check("inv_freq_dev", inv_freq_dev, _F32, d, (head_dim // 2,))
    _check("q_gamma", q_gamma, _F32, d, (head_dim,))
    _check("k_gamma", k_gamma, _F32, d, (head_dim,))
    _check("n_rows", n_rows, _I32, d, (1,))
    _check_pages(k_pages, v_pages, n_kv_heads, head_dim, d)
    if R == 0:
        return q_out
    _fits32(_ld(qkv), _ld(q_out), n_heads, n_kv_heads, head_dim, R, k_pages.shape[0])
    _call_on(
        d,
        "b2d_qk_norm_rope_append",
        qkv.data_ptr(),
        _DT[qkv.dtype],
        _ld(qkv),
        _ptr(q_gamma),
        _ptr(k_gamma),
        eps,
        1 if v_norm else 0,
        positions.data_ptr(),
        slots.data_ptr(),
        _ptr(n_rows),
        inv_freq_dev.data_ptr(),
        q_out.data_ptr(),
        _DT[q_out.dtype],
        _ld(q_out),
        k_pages.data_ptr(),
        v_pages.data_ptr(),
        k_pages.shape[0],
        n_heads,
        n_kv_heads,
        head_dim,
        R,
    )
    return q_out


def tree_attn_workspace_bytes(batch, rows, n_heads, n_kv_heads, head_dim, max_q, max_ctx) -> int:
    return _entry("b2d_paged_tree_attn_workspace_bytes")(batch, rows, n_heads, n_kv_heads, head_dim, max_q, max_ctx)


def paged_tree_attn(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    ctx_lens: torch.Tensor,
    cu_q: torch.Tensor,
    n_heads: int,
    n_kv_heads: int,
    head_dim: int,
    max_q: int,
    max_ctx: int,
    *,
    mask: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    scale: float = 0.0,
    window: int = 0,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of the rows cu_q[b] .. cu_q[b + 1] of each sequence over its ctx_lens[b] cached tokens
    and, of the step's own rows, those its mask names (mask None: the rows up to itself).  q [R, Hq *
    HD] is rotated, the rows' k and v are in the cache.  See include/b200dec.h b2d_paged_tree_attn;
    `out` may be fp16 [2, R, Hq * HD]: the output as B2D_F16X2 hi + lo planes.  The workspace (any
    contents) is allocated from torch's caching allocator unless given."""
    _two_dims("q", q)
    _two_dims("block_table", block_table)
    if mask is not None:
        _two_dims("mask", mask)
    d, R, nq, B = _on_gpu(q), q.shape[0], n_heads * head_dim, ctx_lens.numel()
    _check("q", q, _FLOATS, d, (R, nq), rows=True)
    if out is None:
        out = q.new_empty((R, nq), dtype=out_dtype)
    x2 = _is_x2(out)
    if x2:
        _check("out", out, _F16, d, (2, R, nq))
    else:
        _check("out", out, _FLOATS, d, (R, nq), rows=True)
    _check_pages(k_pages, v_pages, n_kv_heads, head_dim, d)
    _check("ctx_lens", ctx_lens, _I32, d, (B,))
    _check("block_table", block_table, _I32, d, (B, block_table.shape[1]))
    _check("cu_q", cu_q, _I32, d, (B + 1,))
    _check("mask", mask, _I32, d, None if mask is None else (R, mask.shape[1]))
    _check("positions", positions, _I32, d, (R,))
    if R == 0 or B == 0:  # no row belongs to a sequence
        return out
    ldout = nq if x2 else _ld(out)
    _fits32(_ld(q), ldout, n_heads, n_kv_heads, head_dim, R, k_pages.shape[0], max_q, max_ctx, window)
    nbytes = tree_attn_workspace_bytes(B, R, n_heads, n_kv_heads, head_dim, max_q, max_ctx)
    if workspace is None:
        if nbytes:
            workspace = q.new_empty(nbytes, dtype=torch.uint8)
    else:
        _check("workspace", workspace, (torch.uint8,), d, (workspace.numel(),))
    _call_on(
        d,
        "b2d_paged_tree_attn",
        q.data_ptr(),
        _DT[q.dtype],
        _ld(q),
        k_pages.data_ptr(),
        v_pages.data_ptr(),
        block_table.data_ptr(),
        block_table.shape[1],
        k_pages.shape[0],
        ctx_lens.data_ptr(),
        cu_q.data_ptr(),
        _ptr(mask),
        0 if mask is None else mask.shape[1],
        _ptr(positions),
        n_heads,
        n_kv_heads,
        head_dim,
        B,
        R,
        max_q,
        max_ctx,
        scale,
        window,
        out.data_ptr(),
        _lib.F16X2 if x2 else _DT[out.dtype],
        ldout,
        _ptr(workspace),
        0 if workspace is None else workspace.numel(),
    )
    return out


def tree_attn_check() -> None:
    """Synchronize and raise if a bounded wait of a paged_tree_attn call on the current device gave up."""
    call("b2d_paged_tree_attn_error")


@dataclass(slots=True)
class TokenLogprobs:
    """token_logprobs()'s outputs for R rows; the fields that were not asked for are None."""

    logprobs: torch.Tensor | None  # fp32, the shape of the targets
    entropy: torch.Tensor  # fp32 [R], nats
    top_ids: torch.Tensor | None  # int32 [R, k], falling logits, equal ones by rising index
    top_logprobs: torch.Tensor | None  # fp32 [R, k]


def token_logprobs(
    logits: torch.Tensor,
    targets: torch.Tensor | None = None,
    top_k: int = 0,
    *,
    n_rows: torch.Tensor | None = None,
    out: TokenLogprobs | None = None,
) -> TokenLogprobs:
    """Log probabilities of targets (int32 [R] or [R, n]; ids outside the vocabulary: -inf) under the
    rows of logits [R, V] (fp32 or fp16, any row stride), each row's entropy, and its top_k <= 32 most
    likely tokens.  See include/b200dec.h b2d_token_logprobs.  Rows from n_rows (int32 [1], on the
    device) on are skipped: pass `out` to keep what it held there."""
    d = _on_gpu(logits)
    if logits.dim() != 2:
        raise ValueError("logits must be [rows, V]")
    R, V = logits.shape
    _check("logits", logits, _FLOATS, d, logits.shape, rows=True)
    if targets is not None and (targets.dim() not in (1, 2) or targets.shape[0] != R):
        raise ValueError(f"targets must be int32 [{R}] or [{R}, n]")
    _check("targets", targets, _I32, d, None if targets is None else targets.shape)
    _check("n_rows", n_rows, _I32, d, (1,))
    if out is None:
        new, f32 = logits.new_empty, torch.float32
        out = TokenLogprobs(
            None if targets is None else new(targets.shape, dtype=f32),
            new(R, dtype=f32),
            new((R, top_k), dtype=torch.int32) if top_k > 0 else None,
            new((R, top_k), dtype=f32) if top_k > 0 else None,
        )
    else:
        if (targets is not None and out.logprobs is None) or (top_k > 0 and (out.top_ids is None or out.top_logprobs is None)):
            raise ValueError("out lacks a field that was asked for")
        if targets is not None:
            _check("out.logprobs", out.logprobs, _F32, d, tuple(targets.shape))
        _check("out.entropy", out.entropy, _F32, d, (R,))
        if top_k > 0:
            _check("out.top_ids", out.top_ids, _I32, d, (R, top_k))
            _check("out.top_logprobs", out.top_logprobs, _F32, d, (R, top_k))
    if R == 0:
        return out
    _fits32(R, V, top_k)
    _call_on(
        d,
        "b2d_token_logprobs",
        logits.data_ptr(),
        _DT[logits.dtype],
        _ld(logits),
        V,
        R,
        _ptr(n_rows),
        _ptr(targets),
        0 if targets is None else targets.numel() // R,
        top_k,
        None if targets is None else out.logprobs.data_ptr(),
        _ptr(out.entropy),
        out.top_ids.data_ptr() if top_k > 0 else None,
        out.top_logprobs.data_ptr() if top_k > 0 else None,
    )
    return out
