"""Torch-tensor front end over the C ABI.

Each function takes CUDA tensors, checks shapes/dtypes, passes raw pointers
and the current torch stream to ``libmagma_cuda.so`` and returns torch
tensors. PyTorch supplies device memory and streams only; every op here runs
as a kernel of this library. Names mirror the fused-node targets the reference
graph would dispatch (``magma.layer_norm_fwd`` etc.) and the reference's op
semantics (cited per function).
"""
from __future__ import annotations

import ctypes as C
import functools
from array import array

import torch

from . import lib

_DT = {torch.float32: lib.F32, torch.bfloat16: lib.BF16}
_WS: dict[int, torch.Tensor] = {}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _dtype(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32 or bfloat16") from None


def _check_cuda(*ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("magma_b200 ops take CUDA tensors")


def workspace(nbytes: int, device: torch.device | None = None) -> torch.Tensor:
    """A per-device scratch buffer of at least ``nbytes`` (grown on demand).

    Ops on one stream may share it: each consumer finishes with it before the
    next kernel on that stream starts.
    """
    dev = torch.device(device or torch.cuda.current_device())
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    buf = _WS.get(idx)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _WS[idx] = buf
    return buf


# Operators of encoder-decoder models run on the current stream of their
# tensors' device, whichever device is current, and take a workspace of their
# own from torch's allocator at each call, so that calls on several streams and
# calls in captured graphs share none. Their smallest calls take a few
# microseconds on the GPU, so the checks on the way there are kept short.
def _raw_stream(i: int) -> int:
    return torch.cuda.current_stream(i).cuda_stream


# the same value without the Stream object around it, where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
_I64x12, _I64x24 = C.c_int64 * 12, C.c_int64 * 24


def _same_device(first: torch.Tensor, *ts: torch.Tensor | None) -> int:
    """The CUDA device index that all tensors share."""
    i = first.get_device()
    if i < 0:
        raise ValueError("magma_b200 ops take CUDA tensors")
    for t in ts:
        if t is not None and t.get_device() != i:
            _check_cuda(t)
            raise ValueError(f"tensors on different devices: cuda:{i} and {t.device}")
    return i


def _call_on(i: int, name: str, *args) -> None:
    """lib.call on device i with its current stream as the last argument."""
    if i == torch.cuda.current_device():
        lib.call(name, *args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            lib.call(name, *args, _raw_stream(i))


@functools.lru_cache(maxsize=256)
def _bytes_on(i: int, name: str, *sizes) -> int:
    """A workspace query: it depends on the sizes and the device's SM count."""
    with torch.cuda.device(i):
        return lib.query(name, *sizes)


def _rows_ld(t: torch.Tensor, what: str) -> int:
    """Row stride of a 2-D tensor whose rows are contiguous."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be a 2-D tensor with contiguous rows")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# --------------------------------------------------------------------------- LN
def layer_norm_fwd(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5,
                   out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None):
    """nn.LayerNorm.forward (Module.swift:2754-2791) -> (y, mean, rstd)."""
    _check_cuda(x, gamma, beta)
    dim = x.shape[-1]
    rows = x.numel() // dim
    assert x.is_contiguous() and gamma.dtype == torch.float32 and beta.dtype == torch.float32
    y = out if out is not None else torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    lib.call("magma_layernorm_fwd", _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), _ptr(mean),
             _ptr(rstd), rows, dim, eps, _dtype(x), _dtype(y), _stream())
    return y, mean, rstd


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor, mean: torch.Tensor,
                   rstd: torch.Tensor, dx: torch.Tensor | None = None, accumulate_dx: bool = False,
                   dgamma: torch.Tensor | None = None, dbeta: torch.Tensor | None = None,
                   accumulate_params: bool = False):
    """LayerNorm VJP (Autodiff.swift:57-94,221-257,351-370) -> (dx, dgamma, dbeta)."""
    _check_cuda(dy, x, gamma, mean, rstd)
    dim = x.shape[-1]
    rows = x.numel() // dim
    if dx is None:
        dx = torch.empty(x.shape, dtype=torch.float32 if accumulate_dx else x.dtype, device=x.device)
    if dgamma is None:
        dgamma = torch.empty(dim, dtype=torch.float32, device=x.device)
    if dbeta is None:
        dbeta = torch.empty(dim, dtype=torch.float32, device=x.device)
    ws_n = lib.query("magma_layernorm_bwd_workspace_size", rows, dim)
    ws = workspace(ws_n, x.device)
    lib.call("magma_layernorm_bwd", _ptr(dy), _ptr(x), _ptr(gamma), _ptr(mean), _ptr(rstd),
             _ptr(dx), _ptr(dgamma), _ptr(dbeta), rows, dim, _dtype(dy), _dtype(x), _dtype(dx),
             int(accumulate_dx), int(accumulate_params), _ptr(ws), ws.numel(), _stream())
    return dx, dgamma, dbeta


def layer_norm_bwd_residual(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor,
                            mean: torch.Tensor, rstd: torch.Tensor, dx: torch.Tensor,
                            accumulate_dx: bool = True, bf16_copy: bool = True,
                            col_sums: bool = True):
    """LayerNorm VJP into an F32 residual gradient dx (added, or written), with
    the BF16 copy of the final dx and its column sums (the bias gradient of the
    Linear feeding the residual, Autodiff.swift:221-257) ->
    (dx, dx_bf16 | None, dgamma, dbeta, dcol | None)."""
    _check_cuda(dy, x, gamma, mean, rstd, dx)
    assert x.dtype == torch.float32 and dx.dtype == torch.float32
    dim = x.shape[-1]
    rows = x.numel() // dim
    copy = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device) if bf16_copy else None
    dgamma = torch.empty(dim, dtype=torch.float32, device=x.device)
    dbeta = torch.empty(dim, dtype=torch.float32, device=x.device)
    dcol = torch.empty(dim, dtype=torch.float32, device=x.device) if col_sums else None
    ws_n = lib.query("magma_layernorm_bwd_residual_workspace_size", rows, dim)
    ws = workspace(ws_n, x.device)
    lib.call("magma_layernorm_bwd_residual", _ptr(dy), _ptr(x), _ptr(gamma), _ptr(mean),
             _ptr(rstd), _ptr(dx), _ptr(copy), _ptr(dgamma), _ptr(dbeta), _ptr(dcol), rows, dim,
             _dtype(dy), int(accumulate_dx), 0, _ptr(ws), ws.numel(), _stream())
    return dx, copy, dgamma, dbeta, dcol


# ------------------------------------------------------------------------- GEMM
def gemm(a: torch.Tensor, b: torch.Tensor, *, trans_a: bool = False, trans_b: bool = False,
         out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
         epilogue: int = lib.EPI_NONE, bias: torch.Tensor | None = None,
         aux_in: torch.Tensor | None = None, aux_out: torch.Tensor | None = None) -> torch.Tensor:
    """c = opA(a) . opB(b) + epilogue (Tensor.matmul, Tensor.swift:1102-1121).

    a is [m, k] (or [k, m] with trans_a); b is [k, n] (or [n, k] with trans_b).
    Row-major 2-D tensors; the leading dimension is the row stride.
    """
    _check_cuda(a, b, out, bias, aux_in, aux_out)
    assert a.dim() == 2 and b.dim() == 2 and a.dtype == b.dtype
    assert a.stride(1) == 1 and b.stride(1) == 1
    m, k = (a.shape[1], a.shape[0]) if trans_a else (a.shape[0], a.shape[1])
    kb, n = (b.shape[1], b.shape[0]) if trans_b else (b.shape[0], b.shape[1])
    if k != kb:
        raise ValueError(f"gemm: inner dimensions differ ({k} vs {kb})")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype or a.dtype, device=a.device)
    assert out.shape == (m, n) and out.stride(1) == 1
    if epilogue == lib.EPI_ROWSTATS:
        # aux_out: float2 softmax partials [ceil(n / 64)][m]
        assert aux_out is not None and aux_out.dtype == torch.float32
        assert aux_out.numel() >= (n + 63) // 64 * m * 2
    else:
        for t in (aux_in, aux_out):
            if t is not None:
                assert t.shape == (m, n) and t.stride(0) == out.stride(0)
    ws_n = lib.query("magma_gemm_workspace_size", m, n, k, _dtype(a))
    ws = workspace(ws_n, a.device) if ws_n else None
    lib.call("magma_gemm", _ptr(a), _ptr(b), _ptr(out), m, n, k, a.stride(0), b.stride(0),
             out.stride(0), int(trans_a), int(trans_b), _dtype(a), _dtype(out), int(epilogue),
             _ptr(bias), _ptr(aux_in), _ptr(aux_out), _ptr(ws), 0 if ws is None else ws.numel(),
             _stream())
    return out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """nn.Linear.forward (Module.swift:266-300): x . W^T + b, W [out, in]."""
    shp = x.shape
    y = gemm(x.reshape(-1, shp[-1]), weight, trans_b=True, out_dtype=out_dtype,
             epilogue=lib.EPI_BIAS if bias is not None else lib.EPI_NONE, bias=bias)
    return y.reshape(*shp[:-1], weight.shape[0])


# -------------------------------------------------------------------- attention
def _strides4(t: torch.Tensor):
    """(batch, head, seq) strides of a [B, H, S, D] view with unit D stride."""
    assert t.dim() == 4 and t.stride(3) == 1
    return (C.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2))


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                  causal: bool = True, out: torch.Tensor | None = None):
    """Causal SDPA (main.swift:467-481) on [B, H, S, D] views -> (o, lse)."""
    _check_cuda(q, k, v)
    B, H, S, D = q.shape
    assert k.stride() == q.stride() and v.stride() == q.stride()
    o = out if out is not None else torch.empty((B, H, S, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, S), dtype=torch.float32, device=q.device)
    lib.call("magma_attention_fwd", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), B, H, S, D,
             _strides4(q), _strides4(o), scale, int(causal), _dtype(q), _stream())
    return o, lse


def attention_bwd(q, k, v, o, d_o, lse, scale: float, causal: bool = True,
                  dq=None, dk=None, dv=None):
    """Attention VJP (Autodiff.swift:309-317,379-386) -> (dq, dk, dv)."""
    _check_cuda(q, k, v, o, d_o, lse)
    B, H, S, D = q.shape
    assert k.stride() == q.stride() and v.stride() == q.stride() and d_o.stride() == o.stride()
    if dq is None:
        dq = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=q.device)
        dk = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=q.device)
        dv = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=q.device)
    assert dq.stride() == q.stride() and dk.stride() == q.stride() and dv.stride() == q.stride()
    ws_n = lib.query("magma_attention_bwd_workspace_size", B, H, S, D, _dtype(q))
    ws = workspace(ws_n, q.device)
    lib.call("magma_attention_bwd", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(d_o), _ptr(lse),
             _ptr(dq), _ptr(dk), _ptr(dv), B, H, S, D, _strides4(q), _strides4(o), scale,
             int(causal), _dtype(q), _ptr(ws), ws.numel(), _stream())
    return dq, dk, dv


def _heads_view(t: torch.Tensor, what: str, shape, dtype) -> tuple:
    """Strides of a [B, H, S, D] view with unit D stride."""
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} has dtype {t.dtype}, expected {dtype}")
    st = t.stride()
    if st[3] != 1 and shape[3] > 1:
        raise ValueError(f"the last dimension of {what} must be contiguous")
    return st[:3]


def _cross_sizes(q, k, v, kv_lens):
    qs, ks, dt = q.shape, k.shape, q.dtype
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError("q, k and v must be [batch, heads, length, head_dim]")
    if ks[0] != qs[0] or ks[3] != qs[3]:
        raise ValueError(f"q {tuple(qs)} and k {tuple(ks)} differ in batch or head_dim")
    if kv_lens is not None and (kv_lens.dtype is not torch.int32 or kv_lens.shape != qs[:1] or
                                not kv_lens.is_contiguous()):
        raise ValueError("kv_lens must be a contiguous int32 tensor of one length per sequence")
    strides = (*_heads_view(q, "q", qs, dt), *_heads_view(k, "k", ks, dt),
               *_heads_view(v, "v", ks, dt))
    return (qs[0], qs[1], ks[1], qs[2], ks[2], qs[3]), strides


def cross_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        scale: float | None = None, kv_lens: torch.Tensor | None = None,
                        out: torch.Tensor | None = None):
    """Attention over another sequence's keys and values (nn.MultiheadAttention,
    Module.swift:2456-2660) -> (o, lse).

    q [B, H, Sq, D]; k, v [B, Hkv, Skv, D], H a multiple of Hkv; views with any
    strides whose last dimension is contiguous. kv_lens (int32 [B]): the keys
    that each sequence has; what k and v hold behind them has no influence, and
    a sequence without keys gives zero rows and lse -inf. scale: D ** -0.5 by
    default. One query per sequence (a decoding step) and few queries over long
    sources split the keys over the GPU. out (by default like q, with q's strides
    where they are dense) may not share memory with an input.
    """
    i = _same_device(q, k, v, kv_lens, out)
    sizes, st = _cross_sizes(q, k, v, kv_lens)
    if out is None:
        out = torch.empty_like(q)
    at = C.addressof(stb := _I64x12(*st, *_heads_view(out, "out", q.shape, q.dtype)))
    lse = q.new_empty(q.shape[:3], dtype=torch.float32)
    dt = _dtype(q)
    n = _bytes_on(i, "magma_cross_attention_fwd_workspace_size", *sizes, dt)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _call_on(i, "magma_cross_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(),
             out.data_ptr(), lse.data_ptr(), _ptr(kv_lens), *sizes, at, at + 24, at + 48, at + 72,
             sizes[5] ** -0.5 if scale is None else scale, dt, _ptr(ws), n)
    del stb
    return out, lse


def cross_attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                        d_o: torch.Tensor, lse: torch.Tensor, scale: float | None = None,
                        kv_lens: torch.Tensor | None = None, dq: torch.Tensor | None = None,
                        dk: torch.Tensor | None = None, dv: torch.Tensor | None = None):
    """VJP of cross_attention_fwd (Autodiff.swift:309-317,379-386) -> (dq, dk, dv).

    o and lse are the forward pass's; dk and dv are summed over the query heads
    that share a key head and are zero behind kv_lens. The outputs are written
    whole; given ones may have any strides without overlap, and may not share
    memory with an input."""
    i = _same_device(q, k, v, o, d_o, lse, kv_lens, dq, dk, dv)
    sizes, st = _cross_sizes(q, k, v, kv_lens)
    if lse.dtype != torch.float32 or lse.shape != q.shape[:3] or not lse.is_contiguous():
        raise ValueError("lse must be the forward pass's contiguous float32 [B, H, Sq]")
    if dq is None:
        dq = torch.empty_like(q)
    if dk is None:
        dk = torch.empty_like(k)
    if dv is None:
        dv = torch.empty_like(v)
    qs, ks, t = q.shape, k.shape, q.dtype
    stb = _I64x24(*st, *_heads_view(o, "o", qs, t), *_heads_view(d_o, "d_o", qs, t),
                  *_heads_view(dq, "dq", qs, t), *_heads_view(dk, "dk", ks, t),
                  *_heads_view(dv, "dv", ks, t))
    at = C.addressof(stb)
    dt = _dtype(q)
    n = _bytes_on(i, "magma_cross_attention_bwd_workspace_size", *sizes, dt)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _call_on(i, "magma_cross_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(),
             o.data_ptr(), d_o.data_ptr(), lse.data_ptr(), _ptr(kv_lens), dq.data_ptr(),
             dk.data_ptr(), dv.data_ptr(), *sizes, *range(at, at + 192, 24),
             sizes[5] ** -0.5 if scale is None else scale, dt, _ptr(ws), n)
    return dq, dk, dv


# ------------------------------------------------------------------------- Adam
def adam_step(params: torch.Tensor, grads: torch.Tensor, m: torch.Tensor, v: torch.Tensor, *,
              step: int, lr: float, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
              weight_decay: float = 0.0, grad_scale: float = 1.0,
              shadow_bf16: torch.Tensor | None = None) -> None:
    """optim.Adam.step (Optimizer.swift:354-412) over a flat F32 arena, in place."""
    _check_cuda(params, grads, m, v, shadow_bf16)
    n = params.numel()
    assert grads.numel() == n and m.numel() == n and v.numel() == n
    assert all(t.dtype == torch.float32 and t.is_contiguous() for t in (params, grads, m, v))
    if shadow_bf16 is not None:
        assert shadow_bf16.numel() == n and shadow_bf16.dtype == torch.bfloat16
    lib.call("magma_adam_step", _ptr(params), _ptr(grads), _ptr(m), _ptr(v), _ptr(shadow_bf16), n,
             lr, beta1, beta2, eps, weight_decay, step, grad_scale, _stream())


def grad_norm_workspace(n: int, device=None) -> torch.Tensor:
    """Scratch for grad_norm over n elements (per-block partial sums)."""
    nbytes = lib.query("magma_grad_norm_workspace_size", n)
    return torch.empty(max(nbytes // 4, 1), dtype=torch.float32, device=device)


def grad_norm(grads: torch.Tensor, *, grad_scale: float = 1.0, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Global L2 norm of grads * grad_scale (optim.clipGradNorm,
    Optimizer.swift:1229-1247) as a one-element device tensor."""
    _check_cuda(grads, out, workspace)
    assert grads.dtype == torch.float32 and grads.is_contiguous()
    n = grads.numel()
    out = out if out is not None else torch.empty(1, dtype=torch.float32, device=grads.device)
    ws = workspace if workspace is not None else grad_norm_workspace(n, grads.device)
    lib.call("magma_grad_norm", _ptr(grads), n, grad_scale, _ptr(out), _ptr(ws),
             ws.numel() * ws.element_size(), _stream())
    return out


def adam_step_clipped(params: torch.Tensor, grads: torch.Tensor, m: torch.Tensor, v: torch.Tensor,
                      *, step: int, lr: float, grad_norm: torch.Tensor, max_norm: float,
                      beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                      weight_decay: float = 0.0, grad_scale: float = 1.0,
                      shadow_bf16: torch.Tensor | None = None) -> None:
    """clipGradNorm's scaling (by the device norm, Optimizer.swift:1249-1267)
    then optim.Adam.step, in one pass over the arena, in place."""
    _check_cuda(params, grads, m, v, grad_norm, shadow_bf16)
    n = params.numel()
    assert grads.numel() == n and m.numel() == n and v.numel() == n
    assert all(t.dtype == torch.float32 and t.is_contiguous() for t in (params, grads, m, v))
    lib.call("magma_adam_step_clipped", _ptr(params), _ptr(grads), _ptr(m), _ptr(v),
             _ptr(shadow_bf16), n, lr, beta1, beta2, eps, weight_decay, step, grad_scale,
             _ptr(grad_norm), max_norm, _stream())


def _tensor_list(ts, what: str, i: int | None = None):
    """Device index, pointers, dtypes and sizes of contiguous tensors."""
    n = len(ts)
    if n == 0:
        raise ValueError(f"at least one of the {what} is needed")
    if i is None:
        i = ts[0].get_device()
    if i < 0 or [t.get_device() for t in ts] != [i] * n:
        _same_device(ts[0], *ts)
        raise ValueError(f"{what} on another device than cuda:{i}")
    if not all([t.is_contiguous() for t in ts]):
        raise ValueError(f"{what} must be contiguous tensors")
    try:
        dtypes = [_DT[t.dtype] for t in ts]
    except KeyError as e:
        raise TypeError(f"unsupported dtype {e.args[0]}; expected float32 or bfloat16") from None
    return (i, array("Q", [t.data_ptr() for t in ts]), array("i", dtypes),
            array("q", [t.numel() for t in ts]))


def _addr(a: array) -> int:
    return a.buffer_info()[0]


def _norm_out(norm: torch.Tensor | None, first: torch.Tensor) -> torch.Tensor:
    if norm is None:
        return first.new_empty(1, dtype=torch.float32)
    if norm.dtype != torch.float32 or norm.numel() != 1:
        raise ValueError("the norm is one float32 value")
    _same_device(first, norm)
    return norm


def grad_norm_multi(grads, *, grad_scale: float = 1.0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Global L2 norm of grads * grad_scale over a list of float32 or bfloat16
    tensors (optim.clipGradNorm, Optimizer.swift:1229-1247) as a one-element
    device tensor. The squares are added in 64 bits."""
    grads = list(grads)
    i, ptrs, dtypes, sizes = _tensor_list(grads, "gradients")
    norm = _norm_out(out, grads[0])
    n = _bytes_on(i, "magma_grad_norm_multi_workspace_size", len(grads))
    ws = norm.new_empty(n, dtype=torch.uint8)
    _call_on(i, "magma_grad_norm_multi", _addr(ptrs), _addr(sizes), _addr(dtypes), len(grads),
             grad_scale, norm.data_ptr(), ws.data_ptr(), n)
    return norm


def clip_grad_norm(grads, max_norm: float, *, grad_scale: float = 1.0, out=None,
                   norm: torch.Tensor | None = None) -> torch.Tensor:
    """optim.clipGradNorm (Optimizer.swift:1229-1267) over a list of tensors:
    out_i = (grads_i * grad_scale) * min(1, max_norm / (norm + 1e-6)), with norm
    the global L2 norm of grads * grad_scale, which is returned as a one-element
    device tensor. out: None to clip in place, else one tensor per gradient
    (float32 or bfloat16, the gradient itself or memory of its own). Nothing is
    copied to the host; a NaN norm leaves the gradients unclipped, as the
    reference's mask does."""
    grads = list(grads)
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"{len(outs)} outputs for {len(grads)} gradients")
    i, ptrs, dtypes, sizes = _tensor_list(grads, "gradients")
    optrs, odtypes = ptrs, dtypes
    if out is not None:
        if [o.shape for o in outs] != [g.shape for g in grads]:
            raise ValueError("an output differs in shape from its gradient")
        _, optrs, odtypes, _ = _tensor_list(outs, "outputs", i)
    norm = _norm_out(norm, grads[0])
    n = _bytes_on(i, "magma_grad_norm_multi_workspace_size", len(grads))
    ws = norm.new_empty(n, dtype=torch.uint8)
    _call_on(i, "magma_clip_grad_norm_multi", _addr(ptrs), _addr(optrs), _addr(sizes),
             _addr(dtypes), _addr(odtypes), len(grads), grad_scale, max_norm, norm.data_ptr(),
             ws.data_ptr(), n)
    return norm


def lr_warmup_cosine(base_lr: float, min_lr: float, warmup_steps: int, total_steps: int,
                     step: int) -> float:
    """optim.WarmupCosineScheduler.currentLR (Optimizer.swift:766-803) at
    scheduler step `step` (0 for the first training step). Host only."""
    out = C.c_float()
    lib.call("magma_lr_warmup_cosine", base_lr, min_lr, warmup_steps, total_steps, step,
             C.byref(out))
    return out.value


def adam_step_multi(params, grads, ms, vs, *, step: int, lr: float, beta1: float = 0.9,
                    beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 0.0,
                    grad_scale: float = 1.0) -> None:
    """The same update over lists of tensors (multi-tensor apply)."""
    cnt = len(params)
    arr = lambda ts: (C.c_void_p * cnt)(*[t.data_ptr() for t in ts])  # noqa: E731
    sizes = (C.c_int64 * cnt)(*[t.numel() for t in params])
    lib.call("magma_adam_step_multi", arr(params), arr(grads), arr(ms), arr(vs), sizes, cnt, lr,
             beta1, beta2, eps, weight_decay, step, grad_scale, _stream())


# ------------------------------------------------------------------------- glue
def embedding_fwd(tokens: torch.Tensor, wte: torch.Tensor, wpe: torch.Tensor | None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """tok + pos embedding gather (Data.swift:856-886, main.swift:454-458)."""
    B, S = tokens.shape
    D = wte.shape[1]
    out = out if out is not None else torch.empty((B * S, D), dtype=torch.float32, device=wte.device)
    lib.call("magma_embedding_fwd", _ptr(tokens), _ptr(wte), _ptr(wpe), _ptr(out), B, S, D,
             wte.shape[0], _stream())
    return out


def embedding_bwd(tokens: torch.Tensor, dout: torch.Tensor, dwte: torch.Tensor,
                  dwpe: torch.Tensor | None) -> None:
    """Scatter-add VJP of the gather (Data.swift:890-907), accumulating."""
    B, S = tokens.shape
    lib.call("magma_embedding_bwd", _ptr(tokens), _ptr(dout), _ptr(dwte), _ptr(dwpe), B, S,
             dwte.shape[1], dwte.shape[0], _stream())


def embedding_bwd_deterministic(tokens: torch.Tensor, dout: torch.Tensor, dwte: torch.Tensor,
                                dwpe: torch.Tensor | None,
                                workspace: torch.Tensor | None = None,
                                accumulate_dwpe: bool = True) -> None:
    """The scatter-add VJP with rows added to each token row in row order
    (identical on every run), accumulating into dwte; dwpe is added to, or
    written with accumulate_dwpe=False."""
    B, S = tokens.shape
    need = lib.query("magma_embedding_bwd_workspace_size", B, S)
    ws = workspace if workspace is not None else torch.empty(
        max(need // 4, 1), dtype=torch.int32, device=dwte.device)
    lib.call("magma_embedding_bwd_deterministic", _ptr(tokens), _ptr(dout), _ptr(dwte),
             _ptr(dwpe), B, S, dwte.shape[1], dwte.shape[0], int(accumulate_dwpe), _ptr(ws),
             ws.numel() * ws.element_size(), _stream())


def _tokens(tokens: torch.Tensor) -> tuple[int, int]:
    if tokens.dim() != 2 or tokens.dtype != torch.int32 or not tokens.is_contiguous():
        raise ValueError("tokens must be a contiguous int32 [batch, seq] tensor")
    return tokens.shape[0], tokens.shape[1]


def embedding_scaled_fwd(tokens: torch.Tensor, table: torch.Tensor,
                         pos: torch.Tensor | None = None, *, scale: float = 1.0,
                         out: torch.Tensor | None = None,
                         out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """nn.Embedding (Module.swift:339-410) with a scale and an optional learned
    position row: out[b*S+s] = scale * table[tokens[b, s]] + pos[s], as a
    [B*S, D] tensor (the table's dtype by default). table [V, D] with contiguous
    rows, pos [>= S, D] of the same dtype; float32 or bfloat16."""
    i = _same_device(tokens, table, pos, out)
    b, n = _tokens(tokens)
    ld = _rows_ld(table, "table")
    v, d = table.shape
    if pos is not None and (pos.dtype != table.dtype or pos.dim() != 2 or pos.shape[0] < n or
                            pos.shape[1] != d or not pos.is_contiguous()):
        raise ValueError(f"pos must be a contiguous {table.dtype} tensor of at least [{n}, {d}]")
    if out is None:
        out = table.new_empty((b * n, d), dtype=out_dtype)
    elif out.shape != (b * n, d) or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{b * n}, {d}] tensor")
    _call_on(i, "magma_embedding_scaled_fwd", tokens.data_ptr(), table.data_ptr(), ld, _ptr(pos),
             out.data_ptr(), b, n, d, v, scale, _dtype(table), _dtype(out))
    return out


def embedding_scaled_bwd(tokens: torch.Tensor, dout: torch.Tensor, vocab: int, *,
                         scale: float = 1.0, padding_idx: int | None = None, pos: bool = False,
                         dtable: torch.Tensor | None = None, dpos: torch.Tensor | None = None,
                         accumulate: bool = False, accumulate_pos: bool = False,
                         dtype: torch.dtype = torch.float32):
    """VJP of embedding_scaled_fwd -> (dtable [V, D], dpos [S, D] or None), by
    sorted tokens: the same bits on every run.

    dout [B*S, D] with contiguous rows, float32 or bfloat16. dtable (of `dtype`,
    or the given tensor) is written whole, zeros where a token does not occur
    and at padding_idx, or added to with accumulate. dpos (float32; wanted with
    pos=True or by giving it, then of at least S rows, those from S on left as
    they are) is written, or added to with accumulate_pos."""
    if (accumulate and dtable is None) or (accumulate_pos and dpos is None):
        raise ValueError("accumulating needs the tensor that is added to")
    i = _same_device(tokens, dout, dtable, dpos)
    b, n = _tokens(tokens)
    ld = _rows_ld(dout, "dout")
    d = dout.shape[1]
    if dout.shape[0] != b * n:
        raise ValueError(f"dout has {dout.shape[0]} rows for {b * n} tokens")
    if dtable is None:
        dtable = dout.new_empty((vocab, d), dtype=dtype)
    elif dtable.shape != (vocab, d):
        raise ValueError(f"dtable must be [{vocab}, {d}]")
    if dpos is None and pos:
        dpos = dout.new_empty((n, d), dtype=torch.float32)
    elif dpos is not None and (dpos.dtype != torch.float32 or dpos.dim() != 2 or
                               dpos.shape[0] < n or dpos.shape[1] != d or
                               not dpos.is_contiguous()):
        raise ValueError(f"dpos must be a contiguous float32 tensor of at least [{n}, {d}]")
    pad = -1 if padding_idx is None else padding_idx
    if padding_idx is not None and not 0 <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} outside [0, {vocab})")
    nws = _bytes_on(i, "magma_embedding_scaled_bwd_workspace_size", b, n, d)
    ws = dout.new_empty(nws, dtype=torch.uint8) if nws else None
    _call_on(i, "magma_embedding_scaled_bwd", tokens.data_ptr(), dout.data_ptr(), ld,
             dtable.data_ptr(), _rows_ld(dtable, "dtable"), _ptr(dpos), b, n, d, vocab, scale, pad,
             int(accumulate), int(accumulate_pos), _dtype(dout), _dtype(dtable), _ptr(ws), nws)
    return dtable, dpos


def cross_entropy_fwd_bwd(logits: torch.Tensor, targets: torch.Tensor, classes: int | None = None,
                          grad_scale: float | None = None, losses: torch.Tensor | None = None):
    """Softmax CE (main.swift:412-433): per-row losses; logits become dlogits in place."""
    rows, ld = logits.shape
    classes = classes or ld
    grad_scale = 1.0 / rows if grad_scale is None else grad_scale
    losses = losses if losses is not None else torch.empty(rows, dtype=torch.float32,
                                                           device=logits.device)
    lib.call("magma_cross_entropy_fwd_bwd", _ptr(logits), _ptr(targets), _ptr(losses), rows,
             classes, logits.stride(0), grad_scale, _dtype(logits), _stream())
    return losses


def lm_head_cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, classes: int,
                          logits: torch.Tensor, grad_scale: float | None = None,
                          losses: torch.Tensor | None = None):
    """Fused lm-head + softmax CE (main.swift:412-433): logits[:, :classes] =
    x . w[:classes]^T as BF16 with the GEMM's per-row softmax partials, then the
    loss and dlogits (in place, padded columns zeroed) from one read of the
    logits. x [rows, D] BF16, w [>= classes, D] BF16, logits [rows, ld] BF16.
    Returns the per-row losses."""
    _check_cuda(x, w, targets, logits)
    rows, d = x.shape
    ld = logits.stride(0)
    grad_scale = 1.0 / rows if grad_scale is None else grad_scale
    losses = losses if losses is not None else torch.empty(rows, dtype=torch.float32,
                                                           device=x.device)
    stats = torch.empty((classes + 63) // 64 * rows * 2, dtype=torch.float32, device=x.device)
    lib.call("magma_gemm", _ptr(x), _ptr(w), _ptr(logits), rows, classes, d, x.stride(0),
             w.stride(0), ld, 0, 1, lib.BF16, lib.BF16, lib.EPI_ROWSTATS, None, None, _ptr(stats),
             None, 0, _stream())
    lib.call("magma_cross_entropy_fwd_bwd_rowstats", _ptr(logits), _ptr(stats), _ptr(targets),
             _ptr(losses), rows, classes, ld, grad_scale, lib.BF16, _stream())
    return losses


def reduce_sum(x: torch.Tensor, scale: float = 1.0, out: torch.Tensor | None = None):
    out = out if out is not None else torch.empty(1, dtype=torch.float32, device=x.device)
    lib.call("magma_reduce_sum", _ptr(x), _ptr(out), x.numel(), scale, _stream())
    return out


def gelu_fwd(x: torch.Tensor) -> torch.Tensor:
    y = torch.empty_like(x)
    lib.call("magma_gelu_fwd", _ptr(x), _ptr(y), x.numel(), _dtype(x), _stream())
    return y


def gelu_bwd(x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    dx = torch.empty_like(x)
    lib.call("magma_gelu_bwd", _ptr(x), _ptr(dy), _ptr(dx), x.numel(), _dtype(x), _stream())
    return dx


def relu_fwd(x: torch.Tensor) -> torch.Tensor:
    y = torch.empty_like(x)
    lib.call("magma_relu_fwd", _ptr(x), _ptr(y), x.numel(), _dtype(x), _stream())
    return y


def relu_bwd(x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    dx = torch.empty_like(x)
    lib.call("magma_relu_bwd", _ptr(x), _ptr(dy), _ptr(dx), x.numel(), _dtype(x), _stream())
    return dx


def bias_grad(dy: torch.Tensor, out: torch.Tensor | None = None,
              accumulate: bool = False) -> torch.Tensor:
    """db[c] = sum_r dy[r, c] (sumAlongBroadcastDims, Autodiff.swift:221-257)."""
    rows, cols = dy.shape
    out = out if out is not None else torch.empty(cols, dtype=torch.float32, device=dy.device)
    ws = workspace(lib.query("magma_bias_grad_workspace_size", rows, cols), dy.device)
    lib.call("magma_bias_grad", _ptr(dy), _ptr(out), rows, cols, dy.stride(0), _dtype(dy),
             int(accumulate), _ptr(ws), ws.numel(), _stream())
    return out


def convert(src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    lib.call("magma_convert", _ptr(src), _ptr(dst), src.numel(), _dtype(src), _dtype(dst),
             _stream())
    return dst


def scale_(y: torch.Tensor, alpha: float) -> torch.Tensor:
    lib.call("magma_scale", _ptr(y), y.numel(), alpha, _stream())
    return y


def device_error_check() -> int:
    code = C.c_int32(0)
    lib.call("magma_device_error_check", _stream(), C.byref(code))
    return code.value


def init(device: int | None = None) -> None:
    """magma_init on the current (or given) CUDA device."""
    lib.call("magma_init", int(torch.cuda.current_device() if device is None else device))
