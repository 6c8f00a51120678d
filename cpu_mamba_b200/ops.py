"""Tensor-level ops over the C ABI (CUDA tensors in, CUDA tensors out).

selective_scan mirrors the reference's native op selective_scan_cpu
(src/cpu_mamba/selective_scan_cpu.cpp:19-41): same arguments, same checks and
RuntimeError messages, newly allocated output.  The other ops expose the fused
stages of the block for tests and for callers composing their own pipeline.
"""
from __future__ import annotations

import contextlib
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, dtype_code, lib, ptr, require_cuda, stream_of


def selective_scan(x, dt, A, B, C, D, h0: Optional[torch.Tensor] = None,
                   return_last_state: bool = False):
    """GPU drop-in for selective_scan_cpu(x, dt, A, B, C, D) -> y.

    x, dt: (batch, T, d_inner); A: (d_inner, d_state); B, C: (batch, T, d_state);
    D: (d_inner).  All contiguous float32 (the reference's contract, cpp:27-32).
    Optional h0 / return_last_state carry the recurrence state across calls.
    """
    tensors = (x, dt, A, B, C, D)
    if not all(t.is_contiguous() for t in tensors):
        raise RuntimeError("all inputs must be contiguous")
    if x.dtype != torch.float32:
        raise RuntimeError("fp32 only in this build")
    if not (x.dim() == 3 and dt.dim() == 3 and A.dim() == 2 and B.dim() == 3
            and C.dim() == 3 and D.dim() == 1):
        raise RuntimeError("shape mismatch")
    require_cuda(*tensors, h0, what="selective_scan")
    bsz, T, di = x.shape
    S = A.shape[1]
    if S > 256:
        raise RuntimeError("d_state > 256 not supported (stack limit)")
    if (dt.shape != x.shape or A.shape[0] != di or B.shape != (bsz, T, S)
            or C.shape != (bsz, T, S) or D.shape[0] != di):
        raise RuntimeError("shape mismatch")
    if any(t.dtype != torch.float32 for t in tensors):
        raise RuntimeError("fp32 only in this build")
    if h0 is not None:
        h0 = h0.contiguous()
        if h0.shape != (bsz, di, S) or h0.dtype != torch.float32:
            raise RuntimeError("h0 must be float32 (batch, d_inner, d_state)")
    y = torch.empty_like(x)
    h_last = torch.empty(bsz, di, S, device=x.device, dtype=torch.float32) if return_last_state else None
    check(lib().mb2_selective_scan(ptr(x), ptr(dt), ptr(A), ptr(B), ptr(C), ptr(D), ptr(y),
                                   bsz, T, di, S, ptr(h0), ptr(h_last), stream_of(x)),
          "selective_scan")
    return (y, h_last) if return_last_state else y


def conv1d_silu(x_in: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                batch: int, seqlen: int, d_inner: int, return_tail: bool = False,
                out: Optional[torch.Tensor] = None):
    """silu(causal depthwise conv1d(x) + bias) over rows of x_in (token-major,
    first d_inner columns; row stride = x_in.stride(0)).  weight: (d_inner, 1, K)
    or (d_inner, K)."""
    require_cuda(x_in, weight, bias, what="conv1d_silu")
    if x_in.stride(-1) != 1:
        raise RuntimeError("conv1d_silu: rows must be contiguous")
    K = weight.shape[-1]
    w = weight.reshape(d_inner, K).contiguous()
    xc = out if out is not None else torch.empty(batch * seqlen, d_inner, device=x_in.device,
                                                 dtype=x_in.dtype)
    tail = (torch.empty(batch, d_inner, K - 1, device=x_in.device, dtype=x_in.dtype)
            if return_tail else None)
    check(lib().mb2_conv1d_silu(dtype_code(x_in.dtype), ptr(x_in), x_in.stride(0), ptr(w),
                                ptr(bias), ptr(xc), xc.stride(0), ptr(tail), batch, seqlen,
                                d_inner, K, stream_of(x_in)), "conv1d_silu")
    return (xc, tail) if return_tail else xc


def scan_fused(xc, dt_low, Bm, Cm, z, w_dt, b_dt, A_log, D, batch, seqlen, h0=None,
               return_last_state=False, out=None):
    """The block's scan stage in one kernel: dt = softplus(dt_low W_dt^T + b_dt),
    A = -exp(A_log), selective scan, D skip, cast and SiLU(z) gate.

    xc, z: (N, d_inner) row views (N = batch*seqlen, any row stride);
    dt_low, Bm, Cm: (N, dt_rank) / (N, d_state) row views (e.g. the column
    slices of x_proj's output); w_dt: (d_inner, dt_rank).  Returns y (N, d_inner)."""
    require_cuda(xc, dt_low, Bm, Cm, z, w_dt, A_log, what="scan_fused")
    di, S = A_log.shape
    R = w_dt.shape[1]
    y = out if out is not None else torch.empty(batch * seqlen, di, device=xc.device, dtype=xc.dtype)
    h_last = (torch.empty(batch, di, S, device=xc.device, dtype=torch.float32)
              if return_last_state else None)
    A_log, w_dt = A_log.contiguous(), w_dt.contiguous()   # keep alive across the call
    h0 = None if h0 is None else h0.contiguous()
    check(lib().mb2_scan_fused(dtype_code(xc.dtype), ptr(xc), xc.stride(0), ptr(dt_low),
                               dt_low.stride(0), ptr(Bm), Bm.stride(0), ptr(Cm), Cm.stride(0),
                               ptr(z), z.stride(0), ptr(w_dt), ptr(b_dt), ptr(A_log), ptr(D),
                               ptr(h0), ptr(h_last), ptr(y), y.stride(0), batch, seqlen, di, S, R,
                               stream_of(xc)), "scan_fused")
    return (y, h_last) if return_last_state else y


def scan_gated(xc, dt, Bm, Cm, z, A_log, D, batch, seqlen, h0=None, return_last_state=False,
               out=None):
    """scan_fused given dt_proj's output dt = linear(dt_low, W_dt, b_dt) (before
    the softplus, which this kernel applies): A = -exp(A_log), selective scan,
    D skip, cast and SiLU(z) gate.
    xc, dt, z: (N, d_inner) row views; Bm, Cm: (N, d_state) row views."""
    require_cuda(xc, dt, Bm, Cm, z, A_log, what="scan_gated")
    di, S = A_log.shape
    y = out if out is not None else torch.empty(batch * seqlen, di, device=xc.device, dtype=xc.dtype)
    h_last = (torch.empty(batch, di, S, device=xc.device, dtype=torch.float32)
              if return_last_state else None)
    A_log = A_log.contiguous()
    h0 = None if h0 is None else h0.contiguous()
    # T-segment scratch for long sequences over few chains (0 bytes otherwise)
    ws_bytes = lib().mb2_scan_workspace_bytes(batch, seqlen, di, S)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=xc.device) if ws_bytes else None
    check(lib().mb2_scan_gated_ws(dtype_code(xc.dtype), ptr(xc), xc.stride(0), ptr(dt),
                                  dt.stride(0), ptr(Bm), Bm.stride(0), ptr(Cm), Cm.stride(0),
                                  ptr(z), z.stride(0), ptr(A_log), ptr(D), ptr(h0), ptr(h_last),
                                  ptr(y), y.stride(0), batch, seqlen, di, S, ptr(ws), ws_bytes,
                                  stream_of(xc)), "scan_gated")
    return (y, h_last) if return_last_state else y


def linear_recurrence(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """h[t] = a[t] * h[t-1] + b[t] (h[-1] = 0) along dim 1 of (B, T, ...)
    tensors: the reference's _associative_prefix_scan (scan_assoc.py:24-55)."""
    require_cuda(a, b, what="linear_recurrence")
    if a.shape != b.shape or a.dim() < 2:
        raise RuntimeError("linear_recurrence: a and b must have the same (B, T, ...) shape")
    if a.dtype != b.dtype:
        raise RuntimeError("linear_recurrence: a and b must share a dtype")
    a, b = a.contiguous(), b.contiguous()
    h = torch.empty_like(a)
    Bt, T = a.shape[0], a.shape[1]
    inner = a.numel() // max(Bt * T, 1) if a.numel() else 0
    check(lib().mb2_linear_recurrence(dtype_code(a.dtype), ptr(a), ptr(b), ptr(h), Bt, T, inner,
                                      stream_of(a)), "linear_recurrence")
    return h


def split_tf32(w: torch.Tensor) -> torch.Tensor:
    """(2, *w.shape) float32: TF32 hi and lo halves of w (a derived cache)."""
    require_cuda(w, what="split_tf32")
    w = w.detach().contiguous()
    if w.dtype != torch.float32:
        raise TypeError("split_tf32 needs float32")
    out = torch.empty((2,) + tuple(w.shape), device=w.device, dtype=torch.float32)
    check(lib().mb2_split_tf32(ptr(w), ptr(out), w.numel(), stream_of(w)), "split_tf32")
    return out


def split_f16(w: torch.Tensor) -> torch.Tensor:
    """The scaled fp16 halves of a float32 (N, K) weight for the F16X3 GEMM
    (mb2_split_f16's layout, a derived cache): a uint8 device buffer."""
    require_cuda(w, what="split_f16")
    w = w.detach().contiguous()
    if w.dtype != torch.float32 or w.dim() != 2:
        raise TypeError("split_f16 needs a float32 matrix")
    n = lib().mb2_split_f16_bytes(w.shape[0], w.shape[1])
    out = torch.empty(n, device=w.device, dtype=torch.uint8)   # 256-byte aligned by torch
    check(lib().mb2_split_f16(ptr(w), w.shape[0], w.shape[1], ptr(out), stream_of(w)),
          "split_f16")
    return out


def fold_norm(weight: torch.Tensor, norm_weight: torch.Tensor) -> torch.Tensor:
    """weight * norm_weight[None, :] rounded to weight's dtype: an RMSNorm
    weight folded into the columns of the projection that follows it."""
    require_cuda(weight, norm_weight, what="fold_norm")
    w = weight.detach().contiguous()
    g = norm_weight.detach().to(w.dtype).contiguous()
    if g.shape != (w.shape[-1],):
        raise RuntimeError(f"fold_norm: norm weight {tuple(g.shape)} vs weight {tuple(w.shape)}")
    out = torch.empty_like(w)
    check(lib().mb2_fold_norm(dtype_code(w.dtype), ptr(w), ptr(g), ptr(out), w.shape[0],
                              w.shape[-1], stream_of(w)), "fold_norm")
    return out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           weight_split: Optional[torch.Tensor] = None, softplus: bool = False,
           out: Optional[torch.Tensor] = None,
           weight_f16: Optional[torch.Tensor] = None, sm_pair: int = -1) -> torch.Tensor:
    """y = x W^T + b over the last dim of x (nn.Linear semantics); softplus=True
    applies F.softplus to the result in the same kernel (dt_proj's epilogue).
    float32 with weight_f16 (split_f16(weight)): the F16X3 tensor-core GEMM
    (sm_pair: 1 pairs of SMs, 0 or -1 single SMs); with
    weight_split (split_tf32(weight)): the 3xTF32 one."""
    require_cuda(x, weight, bias, what="linear")
    N, K = weight.shape
    lead = x.shape[:-1]
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    y = out if out is not None else torch.empty(x2.shape[0], N, device=x.device, dtype=x.dtype)
    if weight_f16 is not None and x.dtype == torch.float32:
        scratch = torch.empty(lib().mb2_linear_f16_scratch_bytes(), device=x.device,
                              dtype=torch.uint8)
        check(lib().mb2_linear_f16(ptr(x2), x2.stride(0), ptr(weight_f16), ptr(bias), ptr(y),
                                   y.stride(0), x2.shape[0], N, K,
                                   _lib.EPI_SOFTPLUS if softplus else _lib.EPI_NONE,
                                   sm_pair, ptr(scratch), stream_of(x)), "linear_f16")
        return y if out is not None else y.reshape(*lead, N)
    weight = weight.contiguous()
    check(lib().mb2_linear(dtype_code(x.dtype), ptr(x2), x2.stride(0), ptr(weight),
                           ptr(weight_split), ptr(bias), ptr(y), y.stride(0), x2.shape[0], N, K,
                           _lib.EPI_SOFTPLUS if softplus else _lib.EPI_NONE, stream_of(x)), "linear")
    return y if out is not None else y.reshape(*lead, N)


def quantize(scheme: str, w: torch.Tensor, group_size: Optional[int] = None
             ) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """(weight_q, scale, in_dim) with quant.py's exact codes, on the GPU.
    group_size: None for quant.py's one scale per row, or the number of input
    columns per scale (blockwise; scale is then (rows, ceil(cols / group)))."""
    require_cuda(w, what="quantize")
    w = w.detach().to(torch.float32).contiguous()
    rows, cols = w.shape
    if scheme == "int8":
        q = torch.empty(rows, cols, device=w.device, dtype=torch.int8)
    else:
        q = torch.empty(rows, (cols + 1) // 2, device=w.device, dtype=torch.uint8)
    if group_size:
        s = torch.empty(rows, -(-cols // group_size), device=w.device, dtype=torch.float32)
        check(lib().mb2_quantize_grouped(_lib.SCHEMES[scheme], ptr(w), rows, cols, group_size,
                                         ptr(q), ptr(s), stream_of(w)), f"quantize_{scheme}")
    else:
        s = torch.empty(rows, device=w.device, dtype=torch.float32)
        check(lib().mb2_quantize(_lib.SCHEMES[scheme], ptr(w), rows, cols, ptr(q), ptr(s),
                                 stream_of(w)), f"quantize_{scheme}")
    return q, s, cols


def dequantize(scheme: str, weight_q: torch.Tensor, scale: torch.Tensor, in_dim: int,
               group_size: Optional[int] = None) -> torch.Tensor:
    require_cuda(weight_q, scale, what="dequantize")
    weight_q = weight_q.contiguous()
    scale = scale.to(torch.float32).contiguous()
    out = torch.empty(weight_q.shape[0], in_dim, device=weight_q.device, dtype=torch.float32)
    check(lib().mb2_dequantize_grouped(_lib.SCHEMES[scheme], ptr(weight_q), ptr(scale),
                                       weight_q.shape[0], in_dim, group_size or 0, ptr(out),
                                       stream_of(weight_q)), f"dequantize_{scheme}")
    return out


def qlinear(x: torch.Tensor, scheme: str, weight_q: torch.Tensor, scale: torch.Tensor,
            bias: Optional[torch.Tensor], in_features: int, softplus: bool = False,
            group_size: Optional[int] = None) -> torch.Tensor:
    """QuantizedLinear.forward: y = x deq(W)^T + b with W dequantised in-kernel."""
    require_cuda(x, weight_q, scale, bias, what="qlinear")
    N = weight_q.shape[0]
    lead = x.shape[:-1]
    x2 = x.reshape(-1, in_features)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    y = torch.empty(x2.shape[0], N, device=x.device, dtype=x.dtype)
    weight_q, scale = weight_q.contiguous(), scale.to(torch.float32).contiguous()
    check(lib().mb2_qlinear_grouped(_lib.SCHEMES[scheme], group_size or 0, dtype_code(x.dtype),
                                    ptr(x2), x2.stride(0), ptr(weight_q), ptr(scale), ptr(bias),
                                    ptr(y), N, x2.shape[0], N, in_features,
                            _lib.EPI_SOFTPLUS if softplus else _lib.EPI_NONE, stream_of(x)),
          f"qlinear_{scheme}")
    return y.reshape(*lead, N)


# The operators below are called once per token or per layer, where the host's time
# per call counts: their descriptors are packed in one go (the C structures of
# mamba_b200.h, no padding but at the end) and device and stream are plain integers.
def _device_of(what: str, first: torch.Tensor, *others) -> int:
    i = first.get_device()
    if i < 0:
        require_cuda(first, what=what)
    for t in others:
        if t is not None and t.get_device() != i:
            require_cuda(t, what=what)
            raise RuntimeError(f"{what}: tensors on cuda:{i} and {t.device}")
    return i


def _on(index: int):
    """Device ``index`` as the current one for a launch."""
    if index == torch._C._cuda_getDevice():
        return contextlib.nullcontext()
    return torch.cuda.device(index)


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its last index contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _addr(t) -> int:
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------ decay attention
_DECAY = struct.Struct("=2i8q5Q15q3Qqf4x")


def _decay_descriptor(what, q, k, v, g, scale, o, tokens: bool, state_in=0, state_out=0, cu=0,
                      seqs=0, new=True) -> bytes:
    """Argument checks shared by the prompt and the one-token form, and the
    descriptor (mb2_decay_attn).  ``tokens``: q, k, v and o carry a token index
    after the batch.  ``new``: o was made for this call."""
    lead = 2 if tokens else 1
    qs, ks, vs, gs = q.shape, k.shape, v.shape, g.shape
    names = "(batch, tokens, heads, width)" if tokens else "(batch, heads, width)"
    if not len(qs) == len(ks) == len(vs) == lead + 2:
        raise RuntimeError(f"{what}: q, k and v must be {names}, got {tuple(qs)}, {tuple(ks)}, "
                           f"{tuple(vs)}")
    dtype = v.dtype
    if q.dtype != dtype or k.dtype != dtype:
        raise RuntimeError(f"{what}: q, k and v must share a dtype")
    code = dtype_code(dtype)
    if g.dtype != torch.float32:
        raise RuntimeError(f"{what}: g must be float32")
    batch, dk, dv, H = vs[0], qs[-1], vs[-1], gs[-1]
    if (qs[0] != batch or ks[0] != batch or dk != ks[-1]
            or (tokens and (qs[1] != vs[1] or ks[1] != vs[1]))):
        raise RuntimeError(f"{what}: shape mismatch: q {tuple(qs)}, k {tuple(ks)}, v {tuple(vs)}")
    if len(gs) != 1 and gs[:-1] != vs[:lead]:
        raise RuntimeError(f"{what}: g must be (heads,) or {names[:-8]}), got {tuple(gs)}")
    hq, hk, hv = qs[-2], ks[-2], vs[-2]
    if not (H and hq and hk and hv and dk and dv) or H % hq or H % hk or H % hv:
        raise RuntimeError(f"{what}: the heads of q, k and v ({hq}, {hk}, {hv}; widths {dk}, {dv}) "
                           f"must divide the {H} decays of g")
    if not new and (o.shape != vs[:lead] + (H, dv) or o.dtype != dtype
                    or (dv > 1 and o.stride(-1) != 1)):
        raise RuntimeError(f"{what}: out must be {tuple(vs[:lead]) + (H, dv)} in {dtype} with its "
                           "last index contiguous")
    qt, kt, vt, ot, gt = q.stride(), k.stride(), v.stride(), o.stride(), g.stride()
    if not new and any(st == 0 and n > 1 for st, n in zip(ot, o.shape)):
        raise RuntimeError(f"{what}: out holds several of its elements in one place")
    if tokens:
        strides = (qt[0], qt[1], qt[2], kt[0], kt[1], kt[2], vt[0], vt[1], vt[2],
                   *((0, 0, gt[0]) if len(gt) == 1 else gt), ot[0], ot[1], ot[2])
    else:
        strides = (qt[0], 0, qt[1], kt[0], 0, kt[1], vt[0], 0, vt[1],
                   *((0, 0, gt[0]) if len(gt) == 1 else (gt[0], 0, gt[1])), ot[0], 0, ot[1])
    return _DECAY.pack(code, tokens and new, batch, vs[1] if tokens else 1, H, hq, hk, hv, dk, dv,
                       q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), o.data_ptr(),
                       *strides, state_in, state_out, cu, seqs, scale)


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                    scale: float = 1.0, initial_state: Optional[torch.Tensor] = None,
                    cu_seqlens: Optional[torch.Tensor] = None, return_final_state: bool = False,
                    out: Optional[torch.Tensor] = None):
    """Linear attention with a decay for each head, over whole prompts:

        S_t = exp(g_t) S_{t-1} + k_t v_t^T,     o_t = scale * S_t^T q_t

    q: (B, T, Hq, Dk), k: (B, T, Hk, Dk), v: (B, T, Hv, Dv), float32 or bfloat16
    (any strides with a contiguous last index); g: float32 log decays (B, T, H)
    or (H,), at most 0 (-inf forgets the state); Hq, Hk and Hv divide H, and head
    h reads q head h // (H // Hq).  Dk <= 256.  initial_state: float32
    (N, H, Dk, Dv), zeros when None.

    cu_seqlens (int, N + 1 offsets on the device) packs N sequences along T with
    B = 1; rows before the first and behind the last one are zero in a new output
    and untouched in ``out``, which must not overlap the inputs.  Sequences that
    overlap leave the rows they share and their final states undefined.  Otherwise
    N = B.

    Returns o (B, T, H, Dv), with the final state (N, H, Dk, Dv) float32 when
    ``return_final_state``.  An empty sequence's final state is its initial one.
    The state is float32 throughout; a bfloat16 output is off by its own rounding
    and 2^-16 of its terms.  A kernel's wait that runs out leaves outputs incomplete
    and is reported by ``_lib.device_status()``.  Forward only."""
    what = "decay_attention"
    dev = _device_of(what, q, k, v, g, initial_state, cu_seqlens, out)
    if v.dim() != 4 or q.dim() != 4 or k.dim() != 4 or g.dim() not in (1, 3):
        raise RuntimeError(f"{what}: q, k and v must be (batch, tokens, heads, width) and g "
                           f"(heads,) or (batch, tokens, heads), got {tuple(q.shape)}, "
                           f"{tuple(k.shape)}, {tuple(v.shape)} and {tuple(g.shape)}")
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, T, _, dv = v.shape
    H, dk = g.shape[-1], q.shape[-1]
    n, cu = B, 0
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or B != 1 or (
                cu_seqlens.dtype not in (torch.int32, torch.int64)):
            raise RuntimeError(f"{what}: cu_seqlens must hold N + 1 integer offsets into a "
                               "batch of 1")
        cu_seqlens = cu_seqlens.to(torch.int32).contiguous()
        n, cu = cu_seqlens.shape[0] - 1, cu_seqlens.data_ptr()
    if initial_state is not None:
        if initial_state.shape != (n, H, dk, dv) or initial_state.dtype != torch.float32:
            raise RuntimeError(f"{what}: initial_state must be float32 {(n, H, dk, dv)}")
        initial_state = initial_state.contiguous()
    with _on(dev):
        o = v.new_empty((B, T, H, dv)) if out is None else out
        h_last = (torch.empty((n, H, dk, dv), device=v.device, dtype=torch.float32)
                  if return_final_state else None)
        d = _decay_descriptor(what, q, k, v, g, scale, o, True, _addr(initial_state),
                              _addr(h_last), cu, n, out is None)
        nbytes = lib().mb2_decay_attention_workspace_bytes(d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=v.device) if nbytes else None
        rc = lib().mb2_decay_attention(d, _addr(ws), nbytes, _raw_stream(dev))
        if rc:
            check(rc, what)
    return (o, h_last) if return_final_state else o


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                         state: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """decay_attention for one token: q (B, Hq, Dk), k (B, Hk, Dk), v (B, Hv, Dv),
    g (B, H) or (H,); ``state`` (B, H, Dk, Dv) float32 contiguous is advanced in
    place.  Returns o (B, H, Dv)."""
    what = "decay_attention_step"
    dev = _device_of(what, q, k, v, g, state)
    if v.dim() != 3 or q.dim() != 3 or k.dim() != 3 or g.dim() not in (1, 2):
        raise RuntimeError(f"{what}: q, k and v must be (batch, heads, width) and g (heads,) or "
                           f"(batch, heads), got {tuple(q.shape)}, {tuple(k.shape)}, "
                           f"{tuple(v.shape)} and {tuple(g.shape)}")
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, _, dv = v.shape
    H = g.shape[-1]
    if (state.shape != (B, H, q.shape[-1], dv) or state.dtype != torch.float32
            or not state.is_contiguous()):
        raise RuntimeError(f"{what}: state must be contiguous float32 {(B, H, q.shape[-1], dv)}")
    with _on(dev):
        o = v.new_empty((B, H, dv))
        d = _decay_descriptor(what, q, k, v, g, scale, o, False)
        rc = lib().mb2_decay_attention_step(d, state.data_ptr(), _raw_stream(dev))
        if rc:
            check(rc, what)
    return o


# ------------------------------------------------------- norms around a block
_NORM = struct.Struct("=2i3q8Q5q2f4i")


def _norm_rows(name: str, t: torch.Tensor, shape, W: int) -> torch.Tensor:
    if t.shape != shape:
        raise RuntimeError(f"gated_norm: {name} {tuple(t.shape)} does not match x {tuple(shape)}")
    t = _rows(t)
    return t if t.dim() == 2 else t.reshape(-1, W)


def _norm_vector(name: str, t: torch.Tensor, W: int, dtype) -> torch.Tensor:
    if t.shape != (W,) or t.dtype not in (dtype, torch.float32):
        raise RuntimeError(f"gated_norm: {name} must be ({W},) in {dtype} or float32")
    return t if t.is_contiguous() else t.contiguous()


def gated_norm(x: torch.Tensor, gate: Optional[torch.Tensor] = None,
               weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
               residual_scale=None, next_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-5, group_size: Optional[int] = None,
               norm_before_gate: bool = True, out: Optional[torch.Tensor] = None):
    """The norm after a block, its gate, the residual add and the norm before
    the next block, in one pass over the rows of x (..., width):

        u = RMSNorm(x) * weight * silu(gate)      (norm_before_gate)
        u = RMSNorm(x * silu(gate)) * weight      (otherwise)
        r = residual + residual_scale * u
        n = RMSNorm(r) * next_weight

    Without ``weight`` there is no first norm, without ``gate`` no gate; the
    first norm runs over groups of ``group_size`` columns (None: all of them).
    x and gate share a dtype (float32 or bfloat16); residual is in it or in
    float32; residual_scale is a number (default 1) or a (width,) tensor, and
    the (width,) tensors are in x's dtype or float32.  width <= 16384.

    Returns u without a residual, r with one, (r, n) with ``next_weight``; r in
    residual's dtype, u and n in x's, n computed from the unrounded r.  ``out``
    receives the first result; it may be ``residual`` itself (and overlap no
    other input).  Forward only."""
    what = "gated_norm"
    scale_t = residual_scale if isinstance(residual_scale, torch.Tensor) else None
    dev = _device_of(what, x, gate, weight, residual, scale_t, next_weight, out)
    shape, dtype = x.shape, x.dtype
    if len(shape) < 1 or shape[-1] < 1:
        raise RuntimeError(f"{what}: x must be (..., width), got {tuple(shape)}")
    W = shape[-1]
    code = dtype_code(dtype)
    if group_size is not None and (group_size < 1 or W % group_size):
        raise RuntimeError(f"{what}: group_size {group_size} does not divide width {W}")
    x2 = _norm_rows("x", x, shape, W)
    z2 = r2 = None
    first, rcode, scale = dtype, code, 1.0
    if gate is not None:
        if gate.dtype != dtype:
            raise RuntimeError(f"{what}: gate must be in {dtype}")
        z2 = _norm_rows("gate", gate, shape, W)
    if weight is not None:
        weight = _norm_vector("weight", weight, W, dtype)
    if residual is not None:
        first = residual.dtype
        if first not in (dtype, torch.float32):
            raise RuntimeError(f"{what}: residual must be in {dtype} or float32")
        rcode = dtype_code(first)
        r2 = _norm_rows("residual", residual, shape, W)
        if scale_t is not None:
            scale_t = _norm_vector("residual_scale", scale_t, W, dtype)
        elif residual_scale is not None:
            scale = residual_scale
        if next_weight is not None:
            next_weight = _norm_vector("next_weight", next_weight, W, dtype)
    elif residual_scale is not None or next_weight is not None:
        raise RuntimeError(f"{what}: residual_scale and next_weight need a residual")
    with _on(dev):
        if out is None:
            out = (x if first == dtype else residual).new_empty(shape)
        elif out.shape != shape or out.dtype != first or not out.is_contiguous():
            raise RuntimeError(f"{what}: out must be contiguous {tuple(shape)} in {first}")
        n = None if next_weight is None else x.new_empty(shape)
        f32 = torch.float32
        d = _NORM.pack(code, rcode, x2.shape[0], W, group_size or 0, x2.data_ptr(), _addr(z2),
                       _addr(weight), _addr(r2), _addr(scale_t), _addr(next_weight),
                       out.data_ptr(), _addr(n), x2.stride(0), 0 if z2 is None else z2.stride(0),
                       0 if r2 is None else r2.stride(0), W, W, scale, eps, norm_before_gate,
                       weight is not None and weight.dtype == f32,
                       scale_t is not None and scale_t.dtype == f32,
                       next_weight is not None and next_weight.dtype == f32)
        rc = lib().mb2_gated_norm(d, _raw_stream(dev))
        if rc:
            check(rc, what)
    return out if n is None else (out, n)


# ---------------------------------------------------------------- beam search
def beam_select(logits: torch.Tensor, scores: torch.Tensor, num: Optional[int] = None,
                finished: Optional[torch.Tensor] = None, pad_token: int = 0
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The best ``num`` continuations of each batch over its beams and the
    vocabulary: the candidates scores[b, k] + log_softmax(logits[b, k])[v] in
    order, ties to the lowest beam and then the lowest token.

    logits: (B, K, V) float32 or bfloat16 (strided batch and beams; an expanded
    beam index is fine); scores: (B, K) float32.  ``num`` defaults to K.  A beam
    flagged in ``finished`` (B, K) bool has the one continuation ``pad_token``
    at its own score.  A beam whose score or normaliser is not finite has none;
    such candidates and masked (-inf or NaN) logits are worth -inf and come
    last, lowest index first.  K <= 32, num <= 64, V <= 2^20.

    Returns (scores (B, num) float32, parents (B, num), tokens (B, num)), the
    last two int64, parents being beams 0 .. K-1."""
    what = "beam_select"
    dev = _device_of(what, logits, scores, finished)
    shape = logits.shape
    if len(shape) != 3 or shape[1] == 0 or shape[2] == 0:
        raise RuntimeError(f"{what}: logits must be (batch, beams, vocab), got {tuple(shape)}")
    B, K, V = shape
    if scores.shape != (B, K) or scores.dtype != torch.float32:
        raise RuntimeError(f"{what}: scores must be float32 {(B, K)}")
    if finished is not None:
        if finished.shape != (B, K) or finished.dtype != torch.bool:
            raise RuntimeError(f"{what}: finished must be bool {(B, K)}")
        finished = finished.contiguous()
    num = K if num is None else int(num)
    code = dtype_code(logits.dtype)
    logits, scores = _rows(logits), scores.contiguous()
    with _on(dev):
        n = max(num, 0)
        best = scores.new_empty((B, n))
        parents = torch.empty((B, n), device=logits.device, dtype=torch.int64)
        tokens = torch.empty_like(parents)
        nbytes = lib().mb2_beam_select_workspace_bytes(code, B, K, V, num)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device)
        rc = lib().mb2_beam_select(code, logits.data_ptr(), logits.stride(0), logits.stride(1),
                                   scores.data_ptr(), _addr(finished), pad_token, B, K, V, num,
                                   best.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                                   ws.data_ptr(), nbytes, _raw_stream(dev))
        if rc:
            check(rc, what)
    return best, parents, tokens


def _leaves(states, out: list) -> list:
    if isinstance(states, torch.Tensor):
        out.append(states)
        return out
    for s in states.values() if isinstance(states, dict) else states:
        if isinstance(s, torch.Tensor):
            out.append(s)
        else:
            _leaves(s, out)
    return out


def reorder_states(states, parents: torch.Tensor):
    """Beams follow their parents, in place: row b * K + j of every tensor in
    ``states`` (a tensor, or nested lists, tuples and dicts of them, such as
    MambaStack's or CPUMamba's decode states) becomes row b * K + parents[b, j].

    Each tensor is contiguous with B * K rows (its first index) of any dtype;
    parents: (B, K) int64 or int32 beams, K <= 32; a parent outside 0 .. K-1
    leaves its row as it is.  Tensors that overlap, the same one twice among them,
    are refused.  Returns ``states``."""
    what = "reorder_states"
    if parents.dim() != 2 or parents.shape[1] == 0 or (
            parents.dtype not in (torch.int64, torch.int32)):
        raise RuntimeError(f"{what}: parents must be (batch, beams) int64 or int32, got "
                           f"{tuple(parents.shape)} {parents.dtype}")
    B, K = parents.shape
    rows = B * K
    tensors = _leaves(states, [])
    dev = _device_of(what, parents, *tensors)
    for t in tensors:
        if t.dim() < 1 or t.shape[0] != rows or not t.is_contiguous():
            raise RuntimeError(f"{what}: states must be contiguous with {rows} rows, got "
                               f"{tuple(t.shape)}")
    ptrs = [t.data_ptr() for t in tensors]
    sizes = [t.nbytes // (rows or 1) for t in tensors]
    parents = parents.to(torch.int64).contiguous()
    n = len(ptrs)
    with _on(dev):
        rc = lib().mb2_reorder_rows(struct.pack(f"{n}Q", *ptrs), struct.pack(f"{n}q", *sizes), n,
                                    parents.data_ptr(), B, K, _raw_stream(dev))
        if rc:
            check(rc, what)
    return states
