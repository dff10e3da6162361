"""torch-facing wrappers of the C ABI, named after the reference's operator calls.

Each wrapper validates dtypes/devices, passes raw device pointers and the
current CUDA stream to ``libslang_b200.so`` and raises ``SlangError`` on a
non-zero status.  Buffers are owned by the caller (as the reference runners own
theirs); wrappers only allocate an output when none is given.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import SB_BF16, SB_F16, SB_F32

_DT = {torch.float16: SB_F16, torch.float32: SB_F32}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, name: str, dtypes=None, cuda=True):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if cuda and not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def group_of(scales: torch.Tensor, n_in: int) -> int:
    """Values per scale along K, read off the scale tensor's shape."""
    groups = 1 if scales.dim() == 1 else scales.shape[-1]
    if n_in % groups:
        raise ValueError(f"{groups} scale groups do not tile n_in={n_in}")
    return n_in // groups


def dequant_f16(packed: torch.Tensor, scales: torch.Tensor, n_in: int, n_out: int,
                out: torch.Tensor | None = None, bits: int | None = None) -> torch.Tensor:
    """``PrefillGPU._dq`` (gemma4_150/prefill_gpu.py:186-200): packed -> f16 [n_out, n_in].

    As in the reference, the bit width is read off the packed buffer's size
    unless given.
    """
    _need(packed, "packed", (torch.uint8, torch.int32, torch.uint32))
    _need(scales, "scales", (torch.float16, torch.float32))
    nbytes = packed.numel() * packed.element_size()
    if bits is None:
        bits = nbytes * 8 // (n_in * n_out)
    if bits not in (2, 4, 8) or nbytes * 8 != bits * n_in * n_out:
        raise ValueError(f"odd width for [{n_out}x{n_in}] from {nbytes} packed bytes")
    if out is None:
        out = torch.empty((n_out, n_in), dtype=torch.float16, device=packed.device)
    _need(out, "out", (torch.float16,))
    _lib.call("sb_dequant_f16", _ptr(packed), bits, _ptr(scales), _DT[scales.dtype],
              group_of(scales, n_in), _ptr(out), n_out, n_in, _stream())
    return out


def gemv_q4(w: torch.Tensor, scales: torch.Tensor, x: torch.Tensor,
            y: torch.Tensor | None = None, bits: int = 4) -> torch.Tensor:
    """Decode GEMV ``y[m, n] = x[m] . W[n]`` (matvec_dq4, gemma4/qat_kernels.py:33-77);
    ``bits=2`` for the checkpoint's 2-bit weights (gateup_95 / down_96)."""
    _need(w, "w", (torch.uint8,))
    _need(scales, "scales", (torch.float16, torch.float32))
    _need(x, "x", (torch.float16, torch.float32))
    if bits not in (2, 4):
        raise ValueError(f"bits={bits}: the GEMV takes 2- or 4-bit codes")
    n, k = w.shape[0], w.shape[1] * 8 // bits
    x2 = x.reshape(-1, k)
    m = x2.shape[0]
    if y is None:
        y = torch.empty((m, n), dtype=torch.float32, device=w.device)
    _need(y, "y", (torch.float32,))
    _lib.call("sb_gemv_q4" if bits == 4 else "sb_gemv_q2", _ptr(w), _ptr(scales), _DT[scales.dtype],
              group_of(scales, k), _ptr(x2), _DT[x.dtype], _ptr(y), y.shape[-1], m, n, k, _stream())
    return y


def gemv_srq(w: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, in_scale: float, out_scale=0.0,
             y: torch.Tensor | None = None, bits: int = 4) -> torch.Tensor:
    """SRQ linear ``y = srq(W @ srq(x, in_scale), out)`` (``ReferenceSRQ._qlin``,
    gemma4_150/reference.py:96-101); ``out_scale`` a float or a per-row f32
    tensor [n] (concatenated linears)."""
    _need(w, "w", (torch.uint8,))
    _need(scales, "scales", (torch.float16, torch.float32))
    _need(x, "x", (torch.float16, torch.float32))
    n, k = w.shape[0], w.shape[1] * 8 // bits
    x2 = x.reshape(-1, k)
    m = x2.shape[0]
    if y is None:
        y = torch.empty((m, n), dtype=torch.float32, device=w.device)
    _need(y, "y", (torch.float32,))
    rows = None
    if isinstance(out_scale, torch.Tensor):
        _need(out_scale, "out_scale", (torch.float32,))
        if out_scale.numel() != n:
            raise ValueError("per-row out_scale must hold one scale per output row")
        rows, out_scale = out_scale, 0.0
    _lib.call("sb_gemv_srq", _ptr(w), bits, _ptr(scales), _DT[scales.dtype], group_of(scales, k), _ptr(x2),
              _DT[x.dtype], float(in_scale), float(out_scale), _ptr(rows), _ptr(y), y.shape[-1], m, n, k, _stream())
    return y


def gemv_norm_add(w: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, hidden: torch.Tensor, w_add: torch.Tensor,
                  eps: float, w_next: torch.Tensor | None = None, h_out: torch.Tensor | None = None,
                  h16_out: torch.Tensor | None = None, y: torch.Tensor | None = None,
                  counter: torch.Tensor | None = None, bits: int = 4) -> torch.Tensor:
    """Decode GEMV ``y = W @ x`` whose last-arriving CTA then runs
    ``hidden += rmsnorm(y) * w_add`` and ``h = rmsnorm(hidden) * w_next`` (the
    reference's oproj_73 / down_75 tails); returns y."""
    _need(w, "w", (torch.uint8,))
    _need(scales, "scales", (torch.float16, torch.float32))
    _need(x, "x", (torch.float16, torch.float32))
    for t, name in ((hidden, "hidden"), (w_add, "w_add")):
        _need(t, name, (torch.float32,))
    n, k = w.shape[0], w.shape[1] * 8 // bits
    x2 = x.reshape(-1, k)
    m = x2.shape[0]
    if hidden.numel() != m * n:
        raise ValueError("hidden must hold m x n values")
    if y is None:
        y = torch.empty((m, n), dtype=torch.float32, device=w.device)
    if counter is None:
        counter = _counter(w.device)
    _lib.call("sb_gemv_norm_add", _ptr(w), bits, _ptr(scales), _DT[scales.dtype], group_of(scales, k), _ptr(x2),
              _DT[x.dtype], _ptr(y), m, n, k, _ptr(hidden), _ptr(w_add), _ptr(w_next), _ptr(h_out), _ptr(h16_out),
              float(eps), _ptr(counter), _stream())
    return y


def srq(x: torch.Tensor, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Elementwise ``clip(round(x / scale), -128, 127) * scale`` (gemma4_150/reference.py:30-31)."""
    _need(x, "x", (torch.float16, torch.float32))
    if out is None:
        out = torch.empty_like(x)
    _need(out, "out", (torch.float16, torch.float32))
    _lib.call("sb_srq", _ptr(x), _DT[x.dtype], x.numel(), float(scale), _ptr(out), _DT[out.dtype], _stream())
    return out


def lmhead_argmax(emb: torch.Tensor, scales: torch.Tensor, h: torch.Tensor, row_offset: int = 0,
                  keys: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
                  logits: torch.Tensor | None = None, want_tokens: bool = True, bits: int = 4):
    """Fused ``logits_33`` + ``argmax1_34``/``argmax2_35``; returns (keys, tokens).
    ``bits=2`` for the checkpoint's 2-bit lm_head."""
    _need(emb, "emb", (torch.uint8,))
    _need(scales, "scales", (torch.float16, torch.float32))
    _need(h, "h", (torch.float16, torch.float32))
    if bits not in (2, 4):
        raise ValueError(f"bits={bits}: the lm_head takes 2- or 4-bit codes")
    v, k = emb.shape[0], emb.shape[1] * 8 // bits
    h2 = h.reshape(-1, k)
    m = h2.shape[0]
    dev = emb.device
    if keys is None:
        keys = torch.empty(m, dtype=torch.int64, device=dev)
    if want_tokens and tokens is None:
        tokens = torch.empty(m, dtype=torch.int32, device=dev)
    _lib.call("sb_lmhead_argmax" if bits == 4 else "sb_lmhead_argmax_q2", _ptr(emb), _ptr(scales), _DT[scales.dtype],
              group_of(scales, k),
              _ptr(h2), _DT[h.dtype], m, v, k, int(row_offset), _ptr(keys),
              _ptr(tokens) if want_tokens else None, _ptr(logits), _stream())
    return keys, tokens


def keys_to_tokens(keys: torch.Tensor, tokens: torch.Tensor | None = None) -> torch.Tensor:
    if tokens is None:
        tokens = torch.empty(keys.numel(), dtype=torch.int32, device=keys.device)
    _lib.call("sb_keys_to_tokens", _ptr(keys), _ptr(tokens), keys.numel(), _stream())
    return tokens


def gemm(A: torch.Tensor, W: torch.Tensor, C: torch.Tensor, M: int, N: int, K: int, alpha: float = 1.0,
         tr: bool = True, acols: int | None = None, ccols: int | None = None, aoff: int = 0,
         boff: int = 0, coff: int = 0, bcols: int | None = None) -> torch.Tensor:
    """``PrefillGPU._gemm`` (gemma4_150/prefill_gpu.py:151-184) on tcgen05.

    ``C[M,N] = alpha * A[M,K] @ (W[N,K]^T if tr else W[K,N])``, all f16; acols,
    ccols are row strides wider than the operation and aoff/boff/coff are BYTE
    offsets into the buffers, exactly as in the reference.
    """
    for t, nm in ((A, "A"), (W, "W"), (C, "C")):
        _need(t, nm, (torch.float16,))
    lda = acols or K
    ldb = bcols or (K if tr else N)
    ldc = ccols or N
    _lib.call("sb_gemm_f16", A.data_ptr() + aoff, W.data_ptr() + boff, C.data_ptr() + coff, M, N, K,
              float(alpha), 1 if tr else 0, lda, ldb, ldc, _stream())
    return C


def attn_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor | None = None,
                 split: bool = True, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal prompt attention (the reference's attn_prefill / _attn_gemm,
    gemma4_150/prefill_gpu.py:259-314): q [S, nh, hd], k, v [S, hd] f16 ->
    out [S, nh, hd] f16 = softmax(q k^T, causal) v, one fused kernel
    (hd in {64, 128, 256})."""
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, nm, (torch.float16,))
        if not t.is_contiguous():
            raise ValueError(f"{nm} must be contiguous")
    S, nh, hd = q.shape
    if k.shape[0] < S or v.shape[0] < S or k.shape[1] != hd or v.shape[1] != hd:
        raise ValueError("k and v must be [>= S, head_dim]")
    if out is None:
        out = torch.empty_like(q)
    _need(out, "out", (torch.float16,))
    if not split:
        _lib.call("sb_attn_prefill", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), S, nh, hd, _stream())
        return out
    if workspace is None:
        workspace = _workspace(q.device, _lib.load().sb_attn_prefill_workspace_size(S, nh, hd))
    nbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _lib.call("sb_attn_prefill_ws", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), S, nh, hd,
              _ptr(workspace) if workspace is not None else None, nbytes, _stream())
    return out


def attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                out: torch.Tensor | None = None, f16: bool = False,
                workspace: torch.Tensor | None = None, window: int = 0) -> torch.Tensor:
    """Decode attention (the reference's ``attn_101``, gemma4_150/kernels_dsl.py) for a
    batch of sequences: q [m, nh, hd] f32, caches [m, max_seq, hd] f32 (one KV head),
    pos [m] int32 = each sequence's last cached position; returns softmax(q k^T) v over
    keys 0..pos (the last ``window`` of them for a sliding-window layer) as
    [m, nh, hd] f32 (f16 with ``f16``)."""
    _need(q, "q", (torch.float32,))
    _need(k_cache, "k_cache", (torch.float32,))
    _need(v_cache, "v_cache", (torch.float32,))
    _need(pos, "pos", (torch.int32,))
    m, nh, hd = q.shape
    max_seq = k_cache.shape[1]
    if k_cache.shape != (m, max_seq, hd) or v_cache.shape != k_cache.shape or pos.numel() != m:
        raise ValueError("caches must be [m, max_seq, head_dim] and pos [m]")
    if out is None:
        out = torch.empty((m, nh, hd), dtype=torch.float16 if f16 else torch.float32, device=q.device)
    _need(out, "out", (torch.float16,) if f16 else (torch.float32,))
    need = int(_lib.load().sb_attn_decode_workspace_size(m, nh, hd, max_seq))
    if workspace is None:
        workspace = _workspace(q.device, need)
    nbytes = workspace.numel() * workspace.element_size()
    _lib.call("sb_attn_decode_f16" if f16 else "sb_attn_decode", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
              max_seq * hd, pos.data_ptr(), m, nh, hd, max_seq, int(window), out.data_ptr(), workspace.data_ptr(),
              nbytes, _stream())
    return out


def attn_prefill_gemm(q16: torch.Tensor, k16: torch.Tensor, v16: torch.Tensor, out16: torch.Tensor, S: int,
                      window: int = 0, scores: torch.Tensor | None = None, p16: torch.Tensor | None = None
                      ) -> torch.Tensor:
    """Causal prefill attention as the reference's ``_attn_gemm`` chain
    (gemma4_150/prefill_gpu.py:259-313): scores = q k^T on the tcgen05 f16
    GEMM (f32 out), the causal -- and, with ``window``, sliding-window --
    softmax to f16, out = P v.  Any head_dim the GEMM takes (the
    checkpoint's 512 included).  q16 [S, nh, hd], k16 / v16 [>= S, hd],
    out16 [S, nh * hd]; rows of ``scores`` / ``p16`` are [S * nh, >= S]."""
    nh, hd = q16.shape[1], q16.shape[2]
    ld = ((S + 7) // 8) * 8
    if scores is None:
        scores = torch.empty((S * nh, ld), dtype=torch.float32, device=q16.device)
    if p16 is None:
        p16 = torch.empty((S * nh, ld), dtype=torch.float16, device=q16.device)
    lds, ldp = scores.stride(0), p16.stride(0)
    s = _stream()
    _lib.call("sb_gemm_f16_f32out", q16.data_ptr(), k16.data_ptr(), scores.data_ptr(), S * nh, S, hd, 1.0, 1, hd, hd,
              lds, s)
    _lib.call("sb_softmax_causal", scores.data_ptr(), lds, S * nh, nh, 0, S, int(window), p16.data_ptr(), ldp, s)
    _lib.call("sb_gemm_f16", p16.data_ptr(), v16.data_ptr(), out16.data_ptr(), S * nh, hd, S, 1.0, 0, ldp, hd, hd, s)
    return out16


def gemm_q4(A: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, C: torch.Tensor | None = None,
            alpha: float = 1.0, workspace: torch.Tensor | None = None, geglu: bool = False,
            bits: int = 4) -> torch.Tensor:
    """Fused ``_dq`` + ``_gemm``: ``C = f16(alpha * A @ dq_f16(W)^T)``.

    With ``geglu``, W's rows are interleaved (gate, up) pairs and C [M, N/2]
    receives ``f16(gelu_tanh(gate) * up)`` of the f16-rounded pair (the
    reference's gate/up GEMMs + geglu_b, gemma4_150/prefill_gpu.py:365-372)."""
    _need(A, "A", (torch.float16,))
    _need(w, "w", (torch.uint8,))
    _need(scales, "scales", (torch.float16, torch.float32))
    M, K = A.shape
    N = w.shape[0]
    if bits not in (2, 4):
        raise ValueError(f"bits={bits}: the fused GEMM takes 2- or 4-bit codes")
    if w.shape[1] * 8 // bits != K:
        raise ValueError("packed weight does not match A's K")
    if C is None:
        C = torch.empty((M, N // 2 if geglu else N), dtype=torch.float16, device=A.device)
    _need(C, "C", (torch.float16,))
    if workspace is None:
        need = gemm_q4_workspace_size(M, N, K)
        workspace = _workspace(A.device, need)
    fn = ("sb_gemm_q4" if bits == 4 else "sb_gemm_q2") + ("_geglu" if geglu else "")
    _lib.call(fn, _ptr(A), _ptr(w), _ptr(scales), _DT[scales.dtype], group_of(scales, K),
              _ptr(C), M, N, K, float(alpha), K, C.shape[1], _ptr(workspace) if workspace is not None else None,
              0 if workspace is None else workspace.numel() * workspace.element_size(), _stream())
    return C


def gemm_q4_argmax(A: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, row_offset: int = 0,
                   keys: torch.Tensor | None = None, tokens: torch.Tensor | None = None, alpha: float = 1.0,
                   want_tokens: bool = True):
    """lm_head + greedy argmax for every row of A on the tcgen05 GEMM (the
    batched form of ``lmhead_argmax``); returns (keys, tokens)."""
    _need(A, "A", (torch.float16,))
    _need(w, "w", (torch.uint8,))
    _need(scales, "scales", (torch.float16, torch.float32))
    M, K = A.shape
    N = w.shape[0]
    if w.shape[1] * 2 != K:
        raise ValueError("packed weight does not match A's K")
    if keys is None:
        keys = torch.empty(M, dtype=torch.int64, device=A.device)
    if want_tokens and tokens is None:
        tokens = torch.empty(M, dtype=torch.int32, device=A.device)
    _lib.call("sb_gemm_q4_argmax", _ptr(A), _ptr(w), _ptr(scales), _DT[scales.dtype], group_of(scales, K), M, N, K,
              float(alpha), A.stride(0), int(row_offset), _ptr(keys), _ptr(tokens) if want_tokens else None,
              _stream())
    return keys, tokens


def gemm_q4_workspace_size(M: int, N: int, K: int) -> int:
    return int(_lib.load().sb_gemm_q4_workspace_size(M, N, K))


def gemm_q4_kernels(M: int, N: int, K: int) -> int:
    """Kernels one gemm_q4 call of this shape launches (1, or 2 with a split-K finalize)."""
    return int(_lib.load().sb_gemm_q4_kernels(M, N, K))


_WS: dict = {}


def _workspace(device, nbytes: int):
    """A per-device split-K scratch buffer, grown on demand and reused."""
    if nbytes == 0:
        return None
    key = str(device)
    buf = _WS.get(key)
    if buf is None or buf.numel() * 4 < nbytes:
        buf = torch.empty((nbytes + 3) // 4, dtype=torch.float32, device=device)
        _WS[key] = buf
    return buf


def device_status() -> None:
    """Raise if a bounded device-side wait has timed out since the last check."""
    _lib.call("sb_device_status", _stream())


# ---------------------------------------------------------------- per-layer embeddings (PLE)

def _rows(t: torch.Tensor, name: str, n: int) -> int:
    """Row stride of an f32 [m, n] operand whose rows may be spaced (a slice of a wider tensor)."""
    if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != n or t.stride(1) != 1 or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA f32 [m, {n}] tensor with unit column stride")
    return t.stride(0)


def gemv_q8(codes: torch.Tensor, row_scale: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None,
            ple: torch.Tensor | None = None) -> torch.Tensor:
    """8-bit linear ``y = x @ ((codes - 128) * row_scale).T`` for decode rows (``sb_gemv_q8``).

    ``codes`` [n, k] u8 are the checkpoint's int8 weights +128-biased
    (gemma4_150/export.py:155-157), ``row_scale`` [n] or [n, 1] f32.  With
    ``ple`` ([m, n] f32, rows may be spaced, e.g. ``ple_in[:, layer]``) the
    result is ``gelu_tanh(y) * ple``: the PLE input gate of
    gemma4/reference.py:159 (``plegate_76``).
    """
    _need(codes, "codes", (torch.uint8,))
    _need(row_scale, "row_scale", (torch.float32,))
    n, k = codes.shape
    if row_scale.numel() != n:
        raise ValueError("row_scale must hold one scale per output row")
    x2 = x.reshape(-1, k) if x.is_contiguous() else x
    ldx = _rows(x2, "x", k)
    m = x2.shape[0]
    if out is None:
        out = torch.empty(m, n, dtype=torch.float32, device=x.device)
    ldy = _rows(out, "out", n)
    ld_ple = _rows(ple, "ple", n) if ple is not None else 0
    if ple is not None and ple.shape[0] != m:
        raise ValueError("ple must have one row per activation row")
    _lib.call("sb_gemv_q8", _ptr(codes), _ptr(row_scale), _ptr(x2), ldx, _ptr(out), ldy, m, n, k, _ptr(ple), ld_ple,
              _stream())
    return out


def gemv_bf16(w: torch.Tensor, x: torch.Tensor, alpha: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y = alpha * x @ w.T`` for a bf16 weight [n, k] (``sb_gemv_bf16``; an f16
    weight, as export.py stores the per-layer projection, takes ``sb_gemv_f16``),
    f32 rows in and out."""
    _need(w, "w", (torch.bfloat16, torch.int16, torch.float16))
    n, k = w.shape
    x2 = x.reshape(-1, k) if x.is_contiguous() else x
    ldx = _rows(x2, "x", k)
    m = x2.shape[0]
    if out is None:
        out = torch.empty(m, n, dtype=torch.float32, device=x.device)
    ldy = _rows(out, "out", n)
    fn = "sb_gemv_f16" if w.dtype == torch.float16 else "sb_gemv_bf16"
    _lib.call(fn, _ptr(w), float(alpha), _ptr(x2), ldx, _ptr(out), ldy, m, n, k, _stream())
    return out


def ple_gather(ids: torch.Tensor, table: torch.Tensor, scales: torch.Tensor, ple_scale: float,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Scaled 4-bit PLE table rows [m, cols] (``sb_ple_gather``; plegather_01,
    gemma4_150/kernels_dsl.py:457-478).  ``table`` [vocab, cols/2] u8,
    ``scales`` [vocab, cols/group] f32, ``ids`` [m] int32."""
    _need(ids, "ids", (torch.int32,))
    _need(table, "table", (torch.uint8,))
    _need(scales, "scales", (torch.float32,))
    vocab, cols = table.shape[0], table.shape[1] * 2
    group = group_of(scales, cols)
    m = ids.numel()
    if out is None:
        out = torch.empty(m, cols, dtype=torch.float32, device=ids.device)
    _need(out, "out", (torch.float32,))
    _lib.call("sb_ple_gather", _ptr(ids), _ptr(table), _ptr(scales), vocab, cols, group, float(ple_scale), _ptr(out),
              m, _stream())
    return out


def ple_input(x: torch.Tensor, ids: torch.Tensor, table: torch.Tensor, scales: torch.Tensor, w_proj: torch.Tensor,
              w_norm: torch.Tensor, n_layers: int, d: int, eps: float, ple_scale: float,
              out: torch.Tensor | None = None, ctx: torch.Tensor | None = None,
              w_proj16: torch.Tensor | None = None) -> torch.Tensor:
    """Per-layer inputs [m, n_layers, d] of ``ReferenceGemma4._ple_input``
    (gemma4/reference.py:92-101): the bf16 model projection of the scaled
    embedding ``x`` times hidden**-0.5, RMS-normed per layer slice, plus the
    gathered table row, times 2**-0.5 (``sb_gemv_bf16`` + ``sb_ple_combine``).
    With more than ``PLE_GEMV_ROWS`` rows and an f16 copy of the projection
    (``w_proj16``) the projection runs as a tcgen05 GEMM on f16 operands."""
    _need(ids, "ids", (torch.int32,))
    _need(table, "table", (torch.uint8,))
    _need(scales, "scales", (torch.float32,))
    _need(w_norm, "w_norm", (torch.float32,))
    hidden = x.shape[-1]
    m = ids.numel()
    cols = n_layers * d
    if table.shape[1] * 2 != cols or w_proj.shape != (cols, hidden) or w_norm.numel() != d:
        raise ValueError("PLE table, projection or norm does not match n_layers * d")
    if m > PLE_GEMV_ROWS and w_proj16 is not None:
        _need(w_proj16, "w_proj16", (torch.float16,))
        x2 = x.reshape(m, hidden)
        _need(x2, "x", (torch.float32,))
        x16 = torch.empty(m, hidden, dtype=torch.float16, device=x.device)
        _lib.call("sb_cast_f16", _ptr(x2), _ptr(x16), m * hidden, _stream())
        if ctx is None:
            ctx = torch.empty(m, cols, dtype=torch.float32, device=x.device)
        _lib.call("sb_gemm_f16_f32out", _ptr(x16), _ptr(w_proj16), _ptr(ctx), m, cols, hidden,
                  float(hidden ** -0.5), 1, hidden, hidden, cols, _stream())
    else:
        ctx = gemv_bf16(w_proj, x.reshape(m, hidden), alpha=float(hidden ** -0.5), out=ctx)
    if out is None:
        out = torch.empty(m, n_layers, d, dtype=torch.float32, device=x.device)
    _need(out, "out", (torch.float32,))
    _lib.call("sb_ple_combine", _ptr(ctx), _ptr(ids), _ptr(table), _ptr(scales), table.shape[0], _ptr(w_norm),
              n_layers, d, group_of(scales, cols), float(ple_scale), float(eps), _ptr(out), m, _stream())
    return out


def ple_norm_add(proj: torch.Tensor, hidden: torch.Tensor, w_post: torch.Tensor, layer_scalar: float, eps: float,
                 w_next: torch.Tensor | None = None, h_out: torch.Tensor | None = None,
                 h16_out: torch.Tensor | None = None) -> torch.Tensor:
    """In place ``hidden = (hidden + rmsnorm(proj) * w_post) * layer_scalar``
    (gemma4/reference.py:160-163), then optionally the next layer's input
    norm into ``h_out`` / ``h16_out`` (``sb_ple_norm_add``)."""
    for t, name in ((proj, "proj"), (hidden, "hidden"), (w_post, "w_post")):
        _need(t, name, (torch.float32,))
    n = hidden.shape[-1]
    m = hidden.numel() // n
    if proj.shape != hidden.shape:
        raise ValueError("proj and hidden must have the same shape")
    _lib.call("sb_ple_norm_add", _ptr(proj), _ptr(hidden), _ptr(w_post), float(layer_scalar), _ptr(w_next),
              _ptr(h_out), _ptr(h16_out), m, n, float(eps), _stream())
    return hidden


def ple_block(hidden: torch.Tensor, ple_in: torch.Tensor, layer: dict, eps: float,
              w_next: torch.Tensor | None = None, h_out: torch.Tensor | None = None,
              h16_out: torch.Tensor | None = None) -> torch.Tensor:
    """One layer's PLE block on ``hidden`` [m, H] in place (gemma4/reference.py:154-163):
    ``g = gelu_tanh(W_gate @ x) * ple_in``, ``x = (x + rmsnorm(W_proj @ g) * w_post) * scalar``.

    ``ple_in`` is that layer's [m, d] slice of :func:`ple_input`; ``layer``
    holds ``gate``/``proj`` (codes, row scales) on the device, ``post_norm``
    and ``scalar``.  Up to ``PLE_GEMV_ROWS`` rows (decode): three launches,
    gate GEMV + GELU * ple, projection GEMV, norm-add tail, all f32.  More rows
    (prefill): the two linears run as tcgen05 GEMMs on f16 operands (the 8-bit
    weights dequantised to f16 once, cached in ``layer`` as ``gate16`` /
    ``proj16``), as the reference's prefill does (gemma4_150/kernels_dsl.py:1775).
    """
    m, H = hidden.shape
    if m <= PLE_FUSED_TAIL_ROWS:
        # gate GEMV (+ gelu * ple), then the projection GEMV whose last CTA runs the norm-add tail
        g = gemv_q8(layer["gate"][0], layer["gate"][1], hidden, ple=ple_in)
        return ple_proj_norm_add(layer["proj"][0], layer["proj"][1], g, hidden, layer["post_norm"],
                                 layer["scalar"], eps, w_next, h_out, h16_out)
    if m <= PLE_GEMV_ROWS:
        g = gemv_q8(layer["gate"][0], layer["gate"][1], hidden, ple=ple_in)
        proj = gemv_q8(layer["proj"][0], layer["proj"][1], g)
    else:
        d = layer["gate"][0].shape[0]
        if "gate16" not in layer:
            layer["gate16"] = dequant_f16(layer["gate"][0], layer["gate"][1].reshape(-1), H, d, bits=8)
            layer["proj16"] = dequant_f16(layer["proj"][0], layer["proj"][1].reshape(-1), d, H, bits=8)
        dev = hidden.device
        x16 = torch.empty(m, H, dtype=torch.float16, device=dev)
        _lib.call("sb_cast_f16", _ptr(hidden), _ptr(x16), m * H, _stream())
        # the gate's output is one or two 128 x 256 tiles wide: split K so the GEMM covers the SMs
        kbs, tiles = -(-H // 64), -(-m // 128) * -(-d // 256)
        splits = max(z for z in range(1, 9) if kbs % z == 0 and (z == 1 or tiles * z <= _num_sms(dev)))
        pre = torch.empty(splits, m, d, dtype=torch.float32, device=dev)
        _lib.call("sb_gemm_f16_f32out_splitk", _ptr(x16), _ptr(layer["gate16"]), _ptr(pre), m, d, H, 1.0, 1, H, H,
                  d, splits, _stream())
        g16 = torch.empty(m, d, dtype=torch.float16, device=dev)
        _lib.call("sb_ple_gate_act", _ptr(pre), d, m * d, splits, _ptr(ple_in), _rows(ple_in, "ple_in", d),
                  _ptr(g16), d, m, d, _stream())
        proj = torch.empty(m, H, dtype=torch.float32, device=dev)
        _lib.call("sb_gemm_f16_f32out", _ptr(g16), _ptr(layer["proj16"]), _ptr(proj), m, H, d, 1.0, 1, d, d, H,
                  _stream())
    return ple_norm_add(proj, hidden, layer["post_norm"], layer["scalar"], eps, w_next, h_out, h16_out)


PLE_GEMV_ROWS = 16
# rows up to which ple_block runs the projection with its norm-add tail in one launch
# (sb_ple_proj_norm_add).  Off: a block alone measured 7.65 against 8.27 us at one row, but
# the 35-layer decode chain 280 against 253 us per token, because the separate tail kernel's
# launch overlaps the GEMV under programmatic dependent launch while the last CTA's tail does
# not; at 8 rows (26.5 against 20.1 us) the last CTA also runs every row's tail in turn.
PLE_FUSED_TAIL_ROWS = 0
_SMS: dict = {}
_COUNTERS: dict = {}


def _counter(dev) -> torch.Tensor:
    """A zeroed device u32 per device for last-arriver tails; each launch re-arms it."""
    key = str(dev)
    if key not in _COUNTERS:
        _COUNTERS[key] = torch.zeros(1, dtype=torch.int32, device=dev)
    return _COUNTERS[key]


def ple_proj_norm_add(codes: torch.Tensor, row_scale: torch.Tensor, g: torch.Tensor, hidden: torch.Tensor,
                      w_post: torch.Tensor, layer_scalar: float, eps: float, w_next: torch.Tensor | None = None,
                      h_out: torch.Tensor | None = None, h16_out: torch.Tensor | None = None,
                      proj: torch.Tensor | None = None, counter: torch.Tensor | None = None) -> torch.Tensor:
    """PLE projection GEMV + norm-add tail in one launch (``sb_ple_proj_norm_add``,
    ``pleproj_77``): hidden [m <= 8, H] updated in place.  Launches on one
    stream may share the counter; concurrent streams need their own."""
    _need(codes, "codes", (torch.uint8,))
    _need(row_scale, "row_scale", (torch.float32,))
    for t, name in ((g, "g"), (hidden, "hidden"), (w_post, "w_post")):
        _need(t, name, (torch.float32,))
    n, k = codes.shape
    m = hidden.shape[0]
    if tuple(hidden.shape) != (m, n) or tuple(g.shape) != (m, k):
        raise ValueError("hidden must be [m, n] and g [m, k] for codes [n, k]")
    if proj is None:
        proj = torch.empty(m, n, dtype=torch.float32, device=hidden.device)
    if counter is None:
        counter = _counter(hidden.device)
    _lib.call("sb_ple_proj_norm_add", _ptr(codes), _ptr(row_scale), _ptr(g), k, _ptr(proj), m, n, k, _ptr(hidden),
              _ptr(w_post), float(layer_scalar), _ptr(w_next), _ptr(h_out), _ptr(h16_out), float(eps),
              _ptr(counter), _stream())
    return hidden


def _num_sms(dev) -> int:
    key = str(dev)
    if key not in _SMS:
        _SMS[key] = torch.cuda.get_device_properties(dev).multi_processor_count
    return _SMS[key]


# ---------------------------------------------------------------- paged-cache serving
#
# A decode step makes these calls once per layer and its kernels run for a few
# microseconds, so their checks are the cheapest that say the same: attribute
# reads without helper objects, the stream's raw handle (0.1 against 3.2 us for a
# torch.cuda.Stream), and messages formed only on the way out.

_I32, _I64, _F32T = torch.int32, torch.int64, torch.float32
_DT_PAGED = {torch.float16: SB_F16, torch.bfloat16: SB_BF16}
_DT_ALL = {torch.float16: SB_F16, torch.bfloat16: SB_BF16, torch.float32: SB_F32}
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_empty = torch.empty


def _gpu(t: torch.Tensor, name: str) -> int:
    """The GPU of an operator's leading tensor, which has to be the current one."""
    gpu = t.get_device() if isinstance(t, torch.Tensor) else -1
    if gpu < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if gpu != _current_device():
        raise ValueError(f"{name} is on cuda:{gpu}, the current device is cuda:{_current_device()}")
    return gpu


def _refuse(t: torch.Tensor, name: str, dtype, shape, gpu: int):
    """What is wrong with an operand that is not a contiguous tensor of this type and shape."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype:
        raise TypeError(f"{name} has dtype {getattr(t, 'dtype', type(t))}, expected {dtype}")
    raise ValueError(f"{name} must be a contiguous {list(shape)} tensor on cuda:{gpu}, got {list(t.shape)} on {t.device}")


def _vec(t: torch.Tensor | None, name: str, dtype, n: int, gpu: int) -> int | None:
    """Address of a contiguous vector of n values (None passes through)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != n or t.dim() != 1 or not t.is_contiguous() or t.get_device() != gpu:
        _refuse(t, name, dtype, (n,), gpu)
    return t.data_ptr()


class PagedKV:
    """One layer's paged key-value cache: ``k`` and ``v`` are f16 or bf16 tensors (or views)
    [n_pages, n_kv_heads, page_size, head_dim] with the same strides and unit stride in
    head_dim.  A cache laid out token by token inside a page, [n_pages, page_size,
    n_kv_heads, head_dim], is passed as its ``transpose(1, 2)``."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        for t, name in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor")
            if t.dtype not in _DT_PAGED:
                raise TypeError(f"{name} has dtype {t.dtype}, expected torch.float16 or torch.bfloat16")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be [n_pages, n_kv_heads, page_size, head_dim] of one type on one GPU")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v must have the same strides, with unit stride in head_dim")
        self.k, self.v = k, v
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device, self.gpu = k.dtype, k.device, k.get_device()
        self.desc = _lib.PagedKVDesc(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                                     _DT_PAGED[k.dtype], self.n_pages, self.page_size, self.n_kv_heads, self.head_dim)
        self.ptr = ctypes.addressof(self.desc)

    @classmethod
    def allocate(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=torch.float16,
                 device="cuda") -> "PagedKV":
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def kv_append_paged(qkv: torch.Tensor, cache: PagedKV, page_table: torch.Tensor, pos: torch.Tensor,
                    cos: torch.Tensor, sin: torch.Tensor, n_heads: int, seq: torch.Tensor | None = None,
                    q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, v_norm: bool = False,
                    eps: float = 1e-6, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                    v_out: torch.Tensor | None = None) -> torch.Tensor:
    """Normalise (optionally), rotate and append new tokens to a paged cache
    (``sb_kv_append_paged``); returns the rotated queries [t, n_heads, head_dim] in the
    cache's type.

    ``qkv`` [t, (n_heads + 2 n_kv_heads) head_dim] f16, bf16 or f32 (rows may be spaced);
    ``page_table`` [n_seqs, max_pages] and ``pos`` [t] int32; ``seq`` [t] int32 is each
    token's row of the page table (None: token i is sequence i, a decode step).
    ``cos`` / ``sin`` [max_pos, rot/2] f32 rotate values j and j + rot/2 of every q and k
    head.  A token whose position is negative or past the tables is padding.  ``k_out`` /
    ``v_out`` [t, n_kv_heads, head_dim] receive the same keys and values packed, for
    :func:`attn_prefill_packed`."""
    gpu, hd, nkv = _gpu(qkv, "qkv"), cache.head_dim, cache.n_kv_heads
    src = _DT_ALL.get(qkv.dtype)
    if src is None:
        raise TypeError(f"qkv has dtype {qkv.dtype}, expected f16, bf16 or f32")
    width = (n_heads + 2 * nkv) * hd
    shape, step, tab, angles = qkv.shape, qkv.stride(), page_table.shape, cos.shape
    if len(shape) != 2 or shape[1] != width or step[1] != 1 or gpu != cache.gpu:
        raise ValueError(f"qkv must be [t, {width}] rows with unit column stride on {cache.device}")
    t = shape[0]
    if page_table.dtype is not _I32 or len(tab) != 2 or not page_table.is_contiguous() or page_table.get_device() != gpu:
        _refuse(page_table, "page_table", _I32, ("n_seqs", "max_pages"), gpu)
    if len(angles) != 2 or angles != sin.shape:
        raise ValueError("cos and sin must be [max_pos, rot / 2]")
    if cos.dtype is not _F32T or not cos.is_contiguous() or cos.get_device() != gpu:
        _refuse(cos, "cos", _F32T, cos.shape, gpu)
    if sin.dtype is not _F32T or not sin.is_contiguous() or sin.get_device() != gpu:
        _refuse(sin, "sin", _F32T, sin.shape, gpu)
    if q_out is None:
        q_out = cache.k.new_empty((t, n_heads, hd))
    elif q_out.dtype is not cache.dtype or q_out.shape != (t, n_heads, hd) or not q_out.is_contiguous() or \
            q_out.get_device() != gpu:
        raise ValueError(f"q_out must be a contiguous [{t}, {n_heads}, {hd}] tensor of the cache's type")
    if k_out is not None or v_out is not None:
        for o, name in ((k_out, "k_out"), (v_out, "v_out")):
            if o is not None and (o.dtype is not cache.dtype or o.shape != (t, nkv, hd) or not o.is_contiguous() or
                                  o.get_device() != gpu):
                raise ValueError(f"{name} must be a contiguous [{t}, {nkv}, {hd}] tensor of the cache's type")
    _lib.call("sb_kv_append_paged", cache.ptr, page_table.data_ptr(), tab[0], tab[1], qkv.data_ptr(), src,
              step[0] if t > 1 else width, t, n_heads, None if seq is None else _vec(seq, "seq", _I32, t, gpu),
              _vec(pos, "pos", _I32, t, gpu), None if q_norm is None else _vec(q_norm, "q_norm", _F32T, hd, gpu),
              None if k_norm is None else _vec(k_norm, "k_norm", _F32T, hd, gpu), v_norm, eps, cos.data_ptr(),
              sin.data_ptr(), 2 * angles[1], angles[0], q_out.data_ptr(), None if k_out is None else k_out.data_ptr(),
              None if v_out is None else v_out.data_ptr(), _raw_stream(gpu))
    return q_out


def attn_decode_paged_workspace(cache: PagedKV, n_heads: int, batch: int) -> torch.Tensor:
    """A zeroed workspace for :func:`attn_decode_paged` calls that run one after another, of up to
    ``batch`` sequences in any order (and for caches of other shapes whose own workspace is
    no larger); calls that may overlap on the GPU need their own."""
    n = int(_lib.load().sb_attn_decode_paged_workspace_size(cache.ptr, n_heads, batch))
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=cache.device)


def attn_decode_paged(q: torch.Tensor, cache: PagedKV, page_table: torch.Tensor, pos: torch.Tensor,
                      scale: float = 1.0, window: int = 0, out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over the paged cache
    (``sb_attn_decode_paged``): q [b, n_heads, head_dim] of the cache's type,
    ``page_table`` [b, max_pages], ``pos`` [b] int32 = each sequence's last cached
    position (negative: no key, a zero row); over keys 0..pos, or the last ``window``
    of them.  ``workspace`` from :func:`attn_decode_paged_workspace`; without one a fresh
    one is made for the call."""
    gpu = _gpu(q, "q")
    if q.dtype is not cache.dtype:
        raise TypeError(f"q has dtype {q.dtype}, expected the cache's {cache.dtype}")
    shape, tab = q.shape, page_table.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or gpu != cache.gpu:
        raise ValueError(f"q must be [b, n_heads, {cache.head_dim}] on {cache.device}")
    b, nh, hd = shape
    dense = q.is_contiguous()
    if not dense and (q.stride(2) != 1 or (nh > 1 and q.stride(1) != hd)):
        raise ValueError("each sequence's heads of q must be contiguous")
    if page_table.dtype is not _I32 or len(tab) != 2 or tab[0] != b or not page_table.is_contiguous() or \
            page_table.get_device() != gpu:
        _refuse(page_table, "page_table", _I32, (b, "max_pages"), gpu)
    if out is None:
        out = torch.empty_like(q) if dense else torch.empty((b, nh, hd), dtype=q.dtype, device=q.device)
    elif out.dtype is not q.dtype or out.shape != shape or not out.is_contiguous() or out.get_device() != gpu:
        raise ValueError("out must be contiguous and match q")
    if workspace is None:
        workspace = attn_decode_paged_workspace(cache, nh, b)
    elif not workspace.is_contiguous() or workspace.get_device() != gpu:
        raise ValueError(f"workspace must be a contiguous tensor on cuda:{gpu}")
    _lib.call("sb_attn_decode_paged", cache.ptr, page_table.data_ptr(), tab[1], _vec(pos, "pos", _I32, b, gpu), b,
              q.data_ptr(), q.stride(0) if b > 1 else nh * hd, nh, window, scale,
              out.data_ptr(), workspace.data_ptr(), workspace.nbytes, _raw_stream(gpu))
    return out


class PackedPlan:
    """The query tiles of a packed batch of prompts for :func:`attn_prefill_packed`, made
    once per batch (host lengths) and shared by its layers.  ``kv_lens`` longer than
    ``q_lens``: the sequences' first keys come from a cached prefix."""

    def __init__(self, q_lens, n_heads: int, n_kv_heads: int, head_dim: int, kv_lens=None, window: int = 0,
                 device="cuda"):
        q = np.ascontiguousarray(q_lens, dtype=np.int32)
        k = q if kv_lens is None else np.ascontiguousarray(kv_lens, dtype=np.int32)
        if q.ndim != 1 or k.shape != q.shape:
            raise ValueError("q_lens and kv_lens must be lists of the same length")
        n = ctypes.c_int(0)
        args = (q.ctypes.data, k.ctypes.data, q.size, n_heads, n_kv_heads, head_dim, window)
        _lib.call("sb_attn_packed_plan", *args, None, 0, ctypes.addressof(n))
        tiles = np.zeros((n.value, 8), dtype=np.int32)
        _lib.call("sb_attn_packed_plan", *args, tiles.ctypes.data, n.value, ctypes.addressof(n))
        self.n_tiles = n.value
        self.tiles = torch.from_numpy(tiles).to(device)
        self.gpu = self.tiles.get_device()
        self.total_q, self.total_k = int(q.sum()), int(k.sum())
        self.n_heads, self.n_kv_heads, self.head_dim, self.window = n_heads, n_kv_heads, head_dim, window


def attn_prefill_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan, scale: float = 1.0,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts (``sb_attn_prefill_packed``): q [total_q, n_heads,
    head_dim], k, v [total_k, n_kv_heads, head_dim] f16 or bf16, each sequence's queries
    aligned with the end of its keys, the plan's window; returns [total_q, n_heads,
    head_dim].  Tokens and heads may be spaced."""
    gpu = _gpu(q, "q")
    dtype = _DT_PAGED.get(q.dtype)
    if dtype is None or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError("q, k and v must all be f16 or all be bf16")
    nh, nkv, hd = plan.n_heads, plan.n_kv_heads, plan.head_dim
    q_shape, q_step, k_shape, k_step = q.shape, q.stride(), k.shape, k.stride()
    if q_shape != (plan.total_q, nh, hd) or q_step[2] != 1:
        raise ValueError(f"q must be [{plan.total_q}, {nh}, {hd}] with unit stride in head_dim")
    if k_shape != (plan.total_k, nkv, hd) or v.shape != k_shape or k_step != v.stride() or k_step[2] != 1:
        raise ValueError(f"k and v must be [{plan.total_k}, {nkv}, {hd}] with the same strides, unit in head_dim")
    if k.get_device() != gpu or v.get_device() != gpu or plan.gpu != gpu:
        raise ValueError(f"k, v and the plan must be on cuda:{gpu}")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((plan.total_q, nh, hd))
    elif out.dtype is not q.dtype or out.shape != q_shape or out.stride(2) != 1 or out.get_device() != gpu:
        raise ValueError("out must match q, with unit stride in head_dim")
    _lib.call("sb_attn_prefill_packed", q.data_ptr(), *_steps(q_shape, q_step), k.data_ptr(), v.data_ptr(),
              *_steps(k_shape, k_step), out.data_ptr(), *_steps(q_shape, out.stride()), dtype, q_shape[0], k_shape[0], nh,
              nkv, hd, plan.window, scale, plan.tiles.data_ptr(), plan.n_tiles, _raw_stream(gpu))
    return out


def _steps(shape, step) -> tuple[int, int]:
    """Strides of tokens and heads; that of a dimension of one says nothing, so the rows' own width stands in."""
    return step[0] if shape[0] > 1 else shape[2], step[1] if shape[1] > 1 else shape[2]


def sample(logits: torch.Tensor, seeds: torch.Tensor, pos: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           softcap: float = 0.0, tokens: torch.Tensor | None = None) -> torch.Tensor:
    """Draw one token per row of ``logits`` [rows, vocab] (``sb_sample``): temperature, then
    top-k, then top-p, then min-p, each a per-row tensor on the device or None for off.
    ``softcap`` > 0 caps the logits first (softcap * tanh(x / softcap)).
    ``seeds`` [rows] int64 and ``pos`` [rows] int32 decide the draw: the same seed,
    position and logits give the same token.  Returns int32 tokens, -1 for a row whose
    logits are all -inf."""
    gpu = _gpu(logits, "logits")
    dtype = _DT_ALL.get(logits.dtype)
    if dtype is None:
        raise TypeError(f"logits has dtype {logits.dtype}, expected f16, bf16 or f32")
    shape, step = logits.shape, logits.stride()
    if len(shape) != 2 or (step[1] != 1 and shape[1] > 1):
        raise ValueError("logits must be [rows, vocab] with unit column stride")
    rows, vocab = shape
    if tokens is None:
        tokens = _empty(rows, dtype=_I32, device=logits.device)
    _lib.call("sb_sample", logits.data_ptr(), dtype, step[0] if rows > 1 else vocab, rows, vocab,
              _vec(seeds, "seeds", _I64, rows, gpu), _vec(pos, "pos", _I32, rows, gpu),
              _vec(temperature, "temperature", _F32T, rows, gpu), _vec(top_k, "top_k", _I32, rows, gpu),
              _vec(top_p, "top_p", _F32T, rows, gpu), _vec(min_p, "min_p", _F32T, rows, gpu), softcap,
              _vec(tokens, "tokens", _I32, rows, gpu), _raw_stream(gpu))
    return tokens
