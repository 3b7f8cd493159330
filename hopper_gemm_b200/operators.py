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

import torch  # (the library's tensors and allocator, which _operators is linked to)

from . import HgemmError
from ._native import lib

try:
    from . import _operators
except ImportError as e:
    raise ImportError(f"hopper_gemm_b200/_operators.so: {e}; build it with "
                      "`python hopper_gemm_b200/build.py`") from e
if _operators.built_for.split()[-1] != torch.__version__:  # the layout of its tensors is that torch's
    raise ImportError(f"hopper_gemm_b200/_operators.so is built for torch {_operators.built_for.split()[-1]}, this is "
                      f"{torch.__version__}; build it with `python hopper_gemm_b200/build.py`")

_operators.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
    "hgemm_lora", "hgemm_lora_workspace_bytes", "hgemm_qk_norm_rope", "hgemm_attn_prompt",
    "hgemm_attn_prompt_workspace_bytes")), HgemmError)


def lora(X, W, down, up, scale, seg_start, seg_adapter, Y=None, workspace=None, stream=None):
    """Y = X W + scale[a] (X Down[a]) Up[a] with the adapter a of each token's segment.

    X tokens x K, W K x N, down adapters x K x rank, up adapters x rank x N (float16, contiguous);
    scale float32 [adapters]; seg_start int32 [segments + 1], seg_adapter int32 [segments], an
    index outside [0, adapters) for none. Returns Y (tokens x N)."""
    return _operators.lora(X, W, down, up, scale, seg_start, seg_adapter, Y, workspace, stream)


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, axis_of=None,
                 interleaved=False, q_out=None, k_out=None, stream=None):
    """Norm of every query and key head and the rotation of its first 2 * len(inv_freq) elements.

    q tokens x heads_q x head_dim, k tokens x heads_kv x head_dim (float16, views of a fused
    projection's rows are fine); weights float16 [head_dim]; positions int32 [tokens] or
    [axes, tokens]; inv_freq float32; axis_of uint8 [len(inv_freq)], the axis of each pair, with more
    than one axis. q_out and k_out may be q and k. Returns (q_out, k_out)."""
    return _operators.qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps, axis_of,
                                   interleaved, q_out, k_out, stream)


def attn_prompt(q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None, lse=None,
                workspace=None, stream=None):
    """Attention over packed sequences with grouped heads.

    q tokens x heads_q x head_dim, k and v tokens x heads_kv x head_dim (float16, views of a fused
    projection's rows are fine); cu_q and cu_k int32 [batch + 1], the rows where the sequences
    start (cu_k None: as cu_q). causal: the last query of a sequence sees all of its keys. scale
    defaults to head_dim ** -0.5. lse, if given, is a float32 [tokens, heads_q] output. Returns
    out (tokens x heads_q x head_dim); rows behind the last sequence are not written."""
    return _operators.attn_prompt(q, k, v, cu_q, cu_k, scale, causal, out, lse, workspace, stream)
