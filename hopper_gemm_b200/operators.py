"""The operators of a served attention layer, over CUDA tensors.

    qkv    = lora(x, w_qkv, down, up, scale, seg_start, seg_adapter)
    q, k   = qk_norm_rope(q_view, k_view, q_weight, k_weight, positions, inv_freq)
    o      = attn_prompt(q, k, v_view, cu_seqlens)
    y      = lora(o, w_out, ...)

Each function checks its tensors, allocates what is not given (outputs, workspace) and launches
on `stream` (default: the current stream of the tensors' device) through the C ABI of
libhgemm_b200.so, whose header states the formulas and ranges. Launches are asynchronous; what depends
on the batch is read on the device, so a captured call follows its tensors at replay. A refused
call raises HgemmError (or TypeError / ValueError for tensors of the wrong type or shape).
"""
import contextlib
import ctypes

import torch

from ._native import HGEMM_OK, HgemmAttnPrompt, HgemmLora, HgemmQkNormRope, lib

_byref = ctypes.byref


def _half(name, t, ndim, device):
    if t.dtype != torch.float16:
        raise TypeError(f"{name} must be float16, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {t.dim()}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, is on {t.device}")
    return t


def _dense(name, t, dtype, shape, device):
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous on {device}")
    return t


def _heads(name, t, device):
    """tokens x heads x head_dim with the heads of a token adjacent; returns the token stride."""
    _half(name, t, 3, device)
    n, h, d = t.shape
    s = t.stride()
    if n and h and ((d > 1 and s[2] != 1) or (h > 1 and s[1] != d)):
        raise ValueError(f"the heads of a token must be adjacent in {name}")
    return s[0] if n > 1 else max(s[0], h * d)


def _cuda(t):
    if not t.is_cuda:
        raise ValueError("the operators take CUDA tensors")
    return t.device


def _on(device, stream):
    """The stream to launch on, and the context in which a call's own tensors are allocated: memory
    taken from the launching stream's pool is free for work on that stream."""
    if stream is None:
        return torch.cuda.current_stream(device), contextlib.nullcontext()
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device)
    return stream, torch.cuda.stream(stream)


def _call(fn, args, device, stream):
    on = (contextlib.nullcontext() if torch.cuda.current_device() == device.index
          else torch.cuda.device(device))
    with on:
        st = fn(_byref(args), stream.cuda_stream)
    if st != HGEMM_OK:
        from . import HgemmError
        raise HgemmError(st, fn.__name__)


def _scratch(need, workspace, device):
    """The caller's workspace, or one allocated for this call, and its address and bytes."""
    if workspace is None:
        if need == 0:
            return None, None, 0
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous on {device}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def lora(X, W, down, up, scale, seg_start, seg_adapter, Y=None, workspace=None, stream=None):
    """Y = X W + scale[a] (X Down[a]) Up[a] with the adapter a of each token's segment.

    X tokens x K, W K x N, down adapters x K x rank, up adapters x rank x N (float16, contiguous);
    scale float32 [adapters]; seg_start int32 [segments + 1], seg_adapter int32 [segments], an
    index outside [0, adapters) for none. Returns Y (tokens x N)."""
    device = _cuda(X)
    _half("X", X, 2, device)
    T, K = X.shape
    N = W.shape[-1]
    A, _, r = down.shape
    S = seg_adapter.shape[0]
    if not X.is_contiguous():
        raise ValueError("X must be contiguous")
    _dense("W", W, torch.float16, (K, N), device)
    _dense("down", down, torch.float16, (A, K, r), device)
    _dense("up", up, torch.float16, (A, r, N), device)
    _dense("scale", scale, torch.float32, (A,), device)
    _dense("seg_start", seg_start, torch.int32, (S + 1,), device)
    _dense("seg_adapter", seg_adapter, torch.int32, (S,), device)
    stream, ours = _on(device, stream)
    with ours:
        if Y is None:
            Y = torch.empty((T, N), dtype=torch.float16, device=device)
        else:
            _dense("Y", Y, torch.float16, (T, N), device)
        keep, ws, nbytes = _scratch(lib.hgemm_lora_workspace_bytes(T, N, K, r, A, S), workspace,
                                    device)
    _call(lib.hgemm_lora,
          HgemmLora(X.data_ptr(), W.data_ptr(), Y.data_ptr(), down.data_ptr(), up.data_ptr(),
                    scale.data_ptr(), seg_start.data_ptr(), seg_adapter.data_ptr(), ws, nbytes,
                    T, N, K, r, A, S), device, stream)
    return Y


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, axis_of=None,
                 interleaved=False, q_out=None, k_out=None, stream=None):
    """Norm of every query and key head and the rotation of its first 2 * len(inv_freq) elements.

    q tokens x heads_q x head_dim, k tokens x heads_kv x head_dim (float16, views of a fused
    projection's rows are fine); weights float16 [head_dim]; positions int32 [tokens] or
    [axes, tokens]; inv_freq float32; axis_of uint8 [len(inv_freq)], the axis of each pair, with more
    than one axis. q_out and k_out may be q and k. Returns (q_out, k_out)."""
    device = _cuda(q)
    qs, ks = _heads("q", q, device), _heads("k", k, device)
    T, hq, d = q.shape
    hk = k.shape[1]
    if k.shape[0] != T or k.shape[2] != d:
        raise ValueError(f"q and k differ: {tuple(q.shape)} and {tuple(k.shape)}")
    _dense("q_weight", q_weight, torch.float16, (d,), device)
    _dense("k_weight", k_weight, torch.float16, (d,), device)
    axes = positions.shape[0] if positions.dim() == 2 else 1
    _dense("positions", positions, torch.int32,
           (axes, T) if positions.dim() == 2 else (T,), device)
    half = inv_freq.shape[0]
    _dense("inv_freq", inv_freq, torch.float32, (half,), device)
    if axis_of is not None:
        _dense("axis_of", axis_of, torch.uint8, (half,), device)
    stream, ours = _on(device, stream)
    with ours:
        if q_out is None:
            q_out = torch.empty((T, hq, d), dtype=torch.float16, device=device)
        if k_out is None:
            k_out = torch.empty((T, hk, d), dtype=torch.float16, device=device)
    if q_out.shape != q.shape or k_out.shape != k.shape:
        raise ValueError("an output has another shape than its input")
    qos, kos = _heads("q_out", q_out, device), _heads("k_out", k_out, device)
    _call(lib.hgemm_qk_norm_rope,
          HgemmQkNormRope(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                          q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(),
                          axis_of.data_ptr() if axis_of is not None else None,
                          inv_freq.data_ptr(), qs, ks, qos, kos, T, hq, hk, d, 2 * half, axes,
                          1 if interleaved else 0, eps), device, stream)
    return q_out, k_out


def attn_prompt(q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None, lse=None,
                workspace=None, stream=None):
    """Attention over packed sequences with grouped heads.

    q tokens x heads_q x head_dim, k and v tokens x heads_kv x head_dim (float16, views of a fused
    projection's rows are fine); cu_q and cu_k int32 [batch + 1], the rows where the sequences
    start (cu_k None: as cu_q). causal: the last query of a sequence sees all of its keys. scale
    defaults to head_dim ** -0.5. lse, if given, is a float32 [tokens, heads_q] output. Returns
    out (tokens x heads_q x head_dim); rows behind the last sequence are not written."""
    device = _cuda(q)
    qs, ks, vs = _heads("q", q, device), _heads("k", k, device), _heads("v", v, device)
    Tq, hq, d = q.shape
    Tk, hkv, _ = k.shape
    if k.shape != v.shape or k.shape[2] != d:
        raise ValueError(f"q, k, v differ: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B = cu_q.shape[0] - 1
    _dense("cu_q", cu_q, torch.int32, (B + 1,), device)
    if cu_k is not None:
        _dense("cu_k", cu_k, torch.int32, (B + 1,), device)
    stream, ours = _on(device, stream)
    with ours:
        if out is None:
            out = torch.empty((Tq, hq, d), dtype=torch.float16, device=device)
        keep, ws, nbytes = _scratch(
            lib.hgemm_attn_prompt_workspace_bytes(Tq, Tk, B, hq, hkv, d), workspace, device)
    if out.shape != q.shape:
        raise ValueError("out has another shape than q")
    os = _heads("out", out, device)
    if lse is not None:
        _dense("lse", lse, torch.float32, (Tq, hq), device)
    _call(lib.hgemm_attn_prompt,
          HgemmAttnPrompt(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                          lse.data_ptr() if lse is not None else None, cu_q.data_ptr(),
                          cu_k.data_ptr() if cu_k is not None else None, qs, ks, vs, os, ws,
                          nbytes, Tq, Tk, B, hq, hkv, d, 1 if causal else 0,
                          d ** -0.5 if scale is None else scale), device, stream)
    return out
