"""CPU: refusals and workspace sizes of the attention layer's operators; no GPU calls here (every refused call
returns before the first CUDA call)."""
import ctypes

import pytest

import hopper_gemm_b200 as hg
from hopper_gemm_b200 import lib
from hopper_gemm_b200._native import HgemmAttnPrompt, HgemmLora, HgemmQkNormRope

BAD = hg.HGEMM_ERR_INVALID_ARG
P = 1 << 20  # a 16-byte aligned address that is never touched


def call(fn, st):
    return fn(ctypes.byref(st), None)


def lora_args(**over):
    st = HgemmLora(P, P, P, P, P, P, P, P, P, 1 << 40, 16, 64, 64, 16, 4, 2)
    for k, v in over.items():
        setattr(st, k, v)
    return st


def norm_args(**over):
    st = HgemmQkNormRope(P, P, P, P, P, P, P, None, P, 1024, 1024, 1024, 1024, 16, 8, 2, 128, 128,
                         1, 0, 1e-6)
    for k, v in over.items():
        setattr(st, k, v)
    return st


def attn_args(**over):
    st = HgemmAttnPrompt(P, P, P, P, None, P, None, 1024, 256, 256, 1024, P, 1 << 40, 16, 16, 2, 8,
                         2, 128, 1, 0.1)
    for k, v in over.items():
        setattr(st, k, v)
    return st


@pytest.mark.parametrize("over", [
    dict(tokens=-1), dict(N=-8), dict(N=12), dict(K=0), dict(K=60), dict(rank=0), dict(rank=12),
    dict(rank=264), dict(adapters=-1), dict(segments=-1), dict(X=None), dict(W=None), dict(Y=None),
    dict(down=None), dict(up=None), dict(scale=None), dict(seg_start=None), dict(seg_adapter=None),
    dict(X=P + 2), dict(W=P + 8), dict(Y=P + 8), dict(down=P + 4), dict(up=P + 4),
    dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=0),
])
def test_lora_refuses(over):
    assert call(lib.hgemm_lora, lora_args(**over)) == BAD
    assert hg.last_status() == BAD


def test_lora_without_work():
    assert lib.hgemm_lora(None, None) == BAD
    assert call(lib.hgemm_lora, lora_args(tokens=0)) == hg.HGEMM_OK
    assert call(lib.hgemm_lora, lora_args(N=0)) == hg.HGEMM_OK


def test_lora_workspace_bytes():
    size = lib.hgemm_lora_workspace_bytes
    assert size(16, 64, 64, 16, 0, 2) == 0 and size(16, 64, 64, 16, 4, 0) == 0
    assert size(16, 64, 60, 16, 4, 2) == 0 and size(-1, 64, 64, 16, 4, 2) == 0
    for T in (1, 48, 1037, 8192):
        need = size(T, 4096, 4096, 64, 12, 40)
        assert 0 < need < 1 << 30
        st = lora_args(tokens=T, N=4096, K=4096, rank=64, adapters=12, segments=40,
                       workspace_bytes=need - 1)
        assert call(lib.hgemm_lora, st) == BAD


@pytest.mark.parametrize("over", [
    dict(tokens=-1), dict(heads_q=-1), dict(heads_kv=-1), dict(head_dim=0), dict(head_dim=12),
    dict(head_dim=264), dict(rot_dim=-16), dict(rot_dim=8), dict(rot_dim=144), dict(axes=0),
    dict(axes=2), dict(eps=-1.0), dict(eps=float("nan")), dict(q=None), dict(k=None),
    dict(q_out=None), dict(k_out=None), dict(q_weight=None), dict(k_weight=None),
    dict(positions=None), dict(inv_freq=None), dict(q=P + 2), dict(k_out=P + 8),
    dict(q_weight=P + 8), dict(q_stride=1020), dict(q_stride=1016), dict(k_stride=248),
    dict(q_out_stride=1016), dict(q_out_stride=2048), dict(k_out_stride=1028),
])
def test_qk_norm_rope_refuses(over):
    assert call(lib.hgemm_qk_norm_rope, norm_args(**over)) == BAD


def test_qk_norm_rope_without_work():
    assert lib.hgemm_qk_norm_rope(None, None) == BAD
    assert call(lib.hgemm_qk_norm_rope, norm_args(tokens=0)) == hg.HGEMM_OK
    assert call(lib.hgemm_qk_norm_rope, norm_args(heads_q=0, heads_kv=0)) == hg.HGEMM_OK


@pytest.mark.parametrize("over", [
    dict(total_q=-1), dict(total_k=-1), dict(batch=-1), dict(heads_kv=0), dict(heads_q=0),
    dict(heads_q=7), dict(heads_q=258), dict(head_dim=0), dict(head_dim=20), dict(head_dim=136),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-0.1), dict(q=None), dict(k=None), dict(v=None),
    dict(out=None), dict(cu_q=None), dict(total_k=32), dict(q=P + 2), dict(k=P + 8),
    dict(v=P + 4), dict(out=P + 8), dict(q_stride=1016), dict(q_stride=1028), dict(k_stride=248),
    dict(v_stride=260), dict(out_stride=512),
])
def test_attn_prompt_refuses(over):
    assert call(lib.hgemm_attn_prompt, attn_args(**over)) == BAD


def test_attn_prompt_without_work():
    assert lib.hgemm_attn_prompt(None, None) == BAD
    assert call(lib.hgemm_attn_prompt, attn_args(total_q=0, total_k=0)) == hg.HGEMM_OK
    assert call(lib.hgemm_attn_prompt, attn_args(batch=0)) == hg.HGEMM_OK


def test_attn_prompt_workspace():
    size = lib.hgemm_attn_prompt_workspace_bytes
    assert size(-1, 1, 1, 1, 1, 64) == 0 and size(1, 1, 1, 3, 2, 64) == 0
    need = size(16, 1 << 17, 16, 32, 8, 128)
    if need:
        st = attn_args(total_q=16, total_k=1 << 17, batch=16, heads_q=32, heads_kv=8, cu_k=P,
                       q_stride=4096, out_stride=4096, k_stride=1024, v_stride=1024)
        for over in (dict(workspace=None), dict(workspace=P + 8),
                     dict(workspace_bytes=need - 1)):
            bad = HgemmAttnPrompt.from_buffer_copy(st)
            for k, v in over.items():
                setattr(bad, k, v)
            assert call(lib.hgemm_attn_prompt, bad) == BAD


def test_public_functions_refuse_host_tensors():
    import torch
    x = torch.zeros((4, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        hg.lora(x, x, x[None], x[None], x[0], x, x)
    with pytest.raises(ValueError):
        hg.attn_prompt(x[None], x[None], x[None], x[0])
    with pytest.raises(ValueError):
        hg.qk_norm_rope(x[None], x[None], x[0], x[0], x[0], x[0])
    with pytest.raises(AttributeError):
        hg.no_such_operator


def test_outputs_over_inputs_are_refused():
    """With everything else in order (each pointer a place of its own)."""
    far = {n: P + (i + 1) * (1 << 24) for i, n in enumerate(("X", "W", "down", "up", "q", "k", "v"))}
    st = {k: far[k] for k in ("X", "W", "down", "up")}
    for over in (dict(Y=far["X"]), dict(Y=far["W"])):
        assert call(lib.hgemm_lora, lora_args(**st, **over)) == BAD
    st = {k: far[k] for k in ("q", "k", "v")}
    for name in ("q", "k", "v"):
        assert call(lib.hgemm_attn_prompt, attn_args(**st, out=far[name])) == BAD
