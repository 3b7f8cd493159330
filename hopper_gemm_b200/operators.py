"""The operators of a served attention layer, over CUDA tensors.

    qkv    = lora(x, w_qkv, down, up, scale, seg_start, seg_adapter)
    q, k   = qk_norm_rope(q_view, k_view, q_weight, k_weight, positions, inv_freq)
    o      = attn_prompt(q, k, v_view, cu_seqlens)
    y      = lora(o, w_out, ...)

Each function checks its tensors, allocates what is not given (outputs, workspace) and launches
on `stream` (default: the current stream of the tensors' device) through the C ABI of
libhgemm_b200.so, whose header states the formulas and ranges. Launches are asynchronous; what depends
on the batch is read on the device, so a captured call follows its tensors at replay. A refused
call raises HgemmError (or TypeError / ValueError for tensors of the wrong type or shape). They serve:
no gradients are formed.
"""
import ctypes
import functools
import struct

import torch

from ._native import HGEMM_OK, HgemmAttnPrompt, HgemmLora, HgemmQkNormRope, lib

_HALF, _I32, _F32, _U8 = torch.float16, torch.int32, torch.float32, torch.uint8


def _packer(cls):
    """Packs one of the argument structures from its fields in order (a fifth of the time that
    filling the ctypes structure takes; small calls are bound by the host)."""
    codes = {ctypes.c_void_p: "P", ctypes.c_int: "i", ctypes.c_longlong: "q",
             ctypes.c_size_t: "N", ctypes.c_float: "f"}
    packer = struct.Struct("@" + "".join(codes[t] for _, t in cls._fields_))
    assert packer.size <= ctypes.sizeof(cls)  # the end may be padded to the structure's alignment
    tail = bytes(ctypes.sizeof(cls) - packer.size)
    return packer.pack if not tail else lambda *v: packer.pack(*v) + tail


_pack_lora, _pack_norm, _pack_attn = (_packer(c) for c in (HgemmLora, HgemmQkNormRope,
                                                           HgemmAttnPrompt))
# The same functions, taking the packed bytes.
_entry = {}
for _name in ("hgemm_lora", "hgemm_qk_norm_rope", "hgemm_attn_prompt"):
    _entry[_name] = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)(
        (_name, lib))


def _refuse(name, t, dtype, shape, dev):
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous on cuda:{dev}")


def _dense(name, t, dtype, shape, dev):
    if (t.dtype is not dtype or t.shape != shape or t.get_device() != dev or
            not t.is_contiguous()):
        _refuse(name, t, dtype, shape, dev)
    return t.data_ptr()


def _heads(name, t, dev):
    """tokens x heads x head_dim with the heads of a token adjacent; returns the token stride."""
    if t.dtype is not _HALF:
        raise TypeError(f"{name} must be float16, got {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name} must have 3 dimensions, got {t.dim()}")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on cuda:{dev}")
    n, h, d = t.shape
    s, sh, sd = t.stride()
    if n and h and ((d > 1 and sd != 1) or (h > 1 and sh != d)):
        raise ValueError(f"the heads of a token must be adjacent in {name}")
    return s if n > 1 else max(s, h * d)


def _cuda(t):
    dev = t.get_device()
    if dev < 0:
        raise ValueError("the operators take CUDA tensors")
    return dev


def _new(shape, like, stream):
    """A float16 tensor of this call on the launching stream: memory from that stream's pool is free for
    work on it."""
    if stream is None:
        return like.new_empty(shape)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=like.device)
    with torch.cuda.stream(stream):
        return like.new_empty(shape)


# What a call needs depends on its sizes alone.
_lora_bytes = functools.lru_cache(1024)(lambda *sizes: lib.hgemm_lora_workspace_bytes(*sizes))
_attn_bytes = functools.lru_cache(1024)(lambda *sizes: lib.hgemm_attn_prompt_workspace_bytes(*sizes))


def _scratch(need, workspace, like, stream):
    """The caller's workspace, or one of this call, and its address and bytes."""
    if workspace is None:
        if need == 0:
            return None, 0, 0
        workspace = _new(((need + 1) // 2,), like, stream)
    elif workspace.get_device() != like.get_device() or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous on {like.device}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _call(name, args, dev, stream):
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(dev)
    elif not isinstance(stream, int):
        stream = stream.cuda_stream
    if torch.cuda.current_device() == dev:
        st = _entry[name](args, stream)
    else:
        with torch.cuda.device(dev):
            st = _entry[name](args, stream)
    if st != HGEMM_OK:
        from . import HgemmError
        raise HgemmError(st, name)


def lora(X, W, down, up, scale, seg_start, seg_adapter, Y=None, workspace=None, stream=None):
    """Y = X W + scale[a] (X Down[a]) Up[a] with the adapter a of each token's segment.

    X tokens x K, W K x N, down adapters x K x rank, up adapters x rank x N (float16, contiguous);
    scale float32 [adapters]; seg_start int32 [segments + 1], seg_adapter int32 [segments], an
    index outside [0, adapters) for none. Returns Y (tokens x N)."""
    dev = _cuda(X)
    T, K = X.shape
    N = W.shape[-1]
    A, r = down.shape[0], down.shape[-1]
    S = seg_adapter.shape[0]
    x = _dense("X", X, _HALF, (T, K), dev)
    w = _dense("W", W, _HALF, (K, N), dev)
    d = _dense("down", down, _HALF, (A, K, r), dev)
    u = _dense("up", up, _HALF, (A, r, N), dev)
    sc = _dense("scale", scale, _F32, (A,), dev)
    ss = _dense("seg_start", seg_start, _I32, (S + 1,), dev)
    sa = _dense("seg_adapter", seg_adapter, _I32, (S,), dev)
    if Y is None:
        Y = _new((T, N), X, stream)
        y = Y.data_ptr()
    else:
        y = _dense("Y", Y, _HALF, (T, N), dev)
    keep, ws, nbytes = _scratch(_lora_bytes(T, N, K, r, A, S), workspace, X, stream)
    _call("hgemm_lora",
          _pack_lora(x, w, y, d, u, sc, ss, sa, ws, nbytes, T, N, K, r, A, S), dev, stream)
    return Y


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, axis_of=None,
                 interleaved=False, q_out=None, k_out=None, stream=None):
    """Norm of every query and key head and the rotation of its first 2 * len(inv_freq) elements.

    q tokens x heads_q x head_dim, k tokens x heads_kv x head_dim (float16, views of a fused
    projection's rows are fine); weights float16 [head_dim]; positions int32 [tokens] or
    [axes, tokens]; inv_freq float32; axis_of uint8 [len(inv_freq)], the axis of each pair, with more
    than one axis. q_out and k_out may be q and k. Returns (q_out, k_out)."""
    dev = _cuda(q)
    qs, ks = _heads("q", q, dev), _heads("k", k, dev)
    T, hq, d = q.shape
    hk = k.shape[1]
    if k.shape[0] != T or k.shape[2] != d:
        raise ValueError(f"q and k differ: {tuple(q.shape)} and {tuple(k.shape)}")
    wq = _dense("q_weight", q_weight, _HALF, (d,), dev)
    wk = _dense("k_weight", k_weight, _HALF, (d,), dev)
    axes, shape = (1, (T,)) if positions.dim() == 1 else (positions.shape[0],
                                                          (positions.shape[0], T))
    pos = _dense("positions", positions, _I32, shape, dev)
    half = inv_freq.shape[0]
    inv = _dense("inv_freq", inv_freq, _F32, (half,), dev)
    axis = _dense("axis_of", axis_of, _U8, (half,), dev) if axis_of is not None else 0
    if q_out is None:
        q_out = _new((T, hq, d), q, stream)
        qos = hq * d
    else:
        qos = _heads("q_out", q_out, dev)
    if k_out is None:
        k_out = _new((T, hk, d), q, stream)
        kos = hk * d
    else:
        kos = _heads("k_out", k_out, dev)
    if q_out.shape != q.shape or k_out.shape != k.shape:
        raise ValueError("an output has another shape than its input")
    _call("hgemm_qk_norm_rope",
          _pack_norm(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), wq, wk, pos,
                     axis, inv, qs, ks, qos, kos, T, hq, hk, d, 2 * half, axes,
                     1 if interleaved else 0, eps), dev, stream)
    return q_out, k_out


def attn_prompt(q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None, lse=None,
                workspace=None, stream=None):
    """Attention over packed sequences with grouped heads.

    q tokens x heads_q x head_dim, k and v tokens x heads_kv x head_dim (float16, views of a fused
    projection's rows are fine); cu_q and cu_k int32 [batch + 1], the rows where the sequences
    start (cu_k None: as cu_q). causal: the last query of a sequence sees all of its keys. scale
    defaults to head_dim ** -0.5. lse, if given, is a float32 [tokens, heads_q] output. Returns
    out (tokens x heads_q x head_dim); rows behind the last sequence are not written."""
    dev = _cuda(q)
    qs, ks, vs = _heads("q", q, dev), _heads("k", k, dev), _heads("v", v, dev)
    Tq, hq, d = q.shape
    Tk, hkv, dk = k.shape
    if k.shape != v.shape or dk != d:
        raise ValueError(f"q, k, v differ: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B = cu_q.shape[0] - 1
    cq = _dense("cu_q", cu_q, _I32, (B + 1,), dev)
    ck = _dense("cu_k", cu_k, _I32, (B + 1,), dev) if cu_k is not None else 0
    if out is None:
        out = _new((Tq, hq, d), q, stream)
        os = hq * d
    elif out.shape != q.shape:
        raise ValueError("out has another shape than q")
    else:
        os = _heads("out", out, dev)
    ls = _dense("lse", lse, _F32, (Tq, hq), dev) if lse is not None else 0
    keep, ws, nbytes = _scratch(_attn_bytes(Tq, Tk, B, hq, hkv, d), workspace, q, stream)
    _call("hgemm_attn_prompt",
          _pack_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ls, cq, ck, qs, ks,
                     vs, os, ws, nbytes, Tq, Tk, B, hq, hkv, d, 1 if causal else 0,
                     d ** -0.5 if scale is None else scale), dev, stream)
    return out
