"""CPU: sizes, workspaces and outputs that the attention layer's operators refuse, with every other argument in
order and a place of its own for each pointer; no GPU calls (a refused call returns before the first)."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import hopper_gemm_b200 as hg
from hopper_gemm_b200 import lib
from hopper_gemm_b200._native import HgemmAttnPrompt, HgemmLora, HgemmQkNormRope

BAD, TOO_LARGE = hg.HGEMM_ERR_INVALID_ARG, 9
LIMIT = 2 ** 31 - 2 ** 16  # the most rows of a call: 0x7fffffff - 0xffff


def filled(cls, **values):
    st = cls()
    for i, (name, kind) in enumerate(cls._fields_):
        if kind is ctypes.c_void_p:
            setattr(st, name, (i + 1) << 44)  # never touched
    for name, v in values.items():
        setattr(st, name, v)
    return st


def lora_args(**over):
    return filled(HgemmLora, **{**dict(workspace_bytes=1 << 43, tokens=16, N=64, K=64, rank=16, adapters=4,
                                       segments=2), **over})


def norm_args(**over):
    return filled(HgemmQkNormRope, **{**dict(q_stride=1024, k_stride=256, q_out_stride=1024, k_out_stride=256,
                                             tokens=16, heads_q=8, heads_kv=2, head_dim=128, rot_dim=128,
                                             axes=1, eps=1e-6), **over})


def attn_args(**over):
    return filled(HgemmAttnPrompt, **{**dict(q_stride=1024, k_stride=256, v_stride=256, out_stride=1024,
                                             workspace_bytes=1 << 43, total_q=16, total_k=16, batch=2, heads_q=8,
                                             heads_kv=2, head_dim=128, causal=1, scale=0.1), **over})


def status(st):
    fn = {HgemmLora: lib.hgemm_lora, HgemmQkNormRope: lib.hgemm_qk_norm_rope,
          HgemmAttnPrompt: lib.hgemm_attn_prompt}[type(st)]
    return fn(ctypes.byref(st), None)


@pytest.mark.parametrize("st", [
    lora_args(tokens=LIMIT + 1), lora_args(tokens=2 ** 31 - 1), lora_args(N=2 ** 31 - 8), lora_args(K=2 ** 31 - 8),
    lora_args(segments=2 ** 30 + 1), norm_args(tokens=LIMIT + 1), norm_args(tokens=2 ** 31 - 1),
    norm_args(heads_q=(1 << 20) + 1, q_stride=1 << 32, q_out_stride=1 << 32),
    attn_args(total_q=LIMIT + 1), attn_args(total_q=2 ** 31 - 1, total_k=2 ** 31 - 1), attn_args(total_k=2 ** 31 - 1),
    attn_args(batch=2 ** 31 - 1)])
def test_sizes_that_32_bits_would_not_hold_are_refused(st):
    assert status(st) == TOO_LARGE
    assert hg.last_status() == TOO_LARGE


def test_workspaces_of_refused_and_of_the_largest_sizes():
    lora, attn = lib.hgemm_lora_workspace_bytes, lib.hgemm_attn_prompt_workspace_bytes
    assert lora(2 ** 31 - 1, 64, 64, 16, 4, 2) == 0 and lora(16, 64, 64, 16, 4, 2 ** 30 + 1) == 0
    assert attn(2 ** 31 - 1, 2 ** 31 - 1, 2, 1, 1, 64) == 0 and attn(1, 2 ** 31 - 1, 1, 1, 1, 64) == 0
    assert lora(LIMIT, 64, 64, 16, 4, 2) > 0
    assert 0 < attn(1, LIMIT, 1, 8, 1, 64) < 1 << 20
    assert 0 <= attn(LIMIT, LIMIT, 2 ** 20, 8, 1, 64) < 1 << 62


def test_a_scale_that_overflows_in_log2_units_is_refused():
    """A masked score of -infinity, and a score of 0, would become NaN."""
    for scale in (2.4e38, 3.4e38):
        assert status(attn_args(scale=scale)) == BAD


@pytest.mark.parametrize("T,N,K,r,A,S,most", [
    (4096, 4096, 4096, 64, 8, 4096, 8 << 20), (8192, 4096, 4096, 128, 32, 8192, 80 << 20),
    (4096, 4096, 4096, 64, 1 << 20, 1, 8 << 20), (1 << 20, 4096, 4096, 16, 1 << 20, 3, 256 << 20)])
def test_lora_workspace_goes_by_the_adapters_too(T, N, K, r, A, S, most):
    """Operand blocks of 128 or 256 rows of 64 columns for each adapter of each row tile: min(adapters, one more than
    the segments) of them at most, not one for every segment."""
    assert lib.hgemm_lora_workspace_bytes(T, N, K, r, A, S) <= most


def few_tokens(T, N, K, r, A, S):
    """Whether these sizes take the path of few tokens, whose workspace is its partial sums of X Down."""
    slices = max(1, min(16, 592 // T, K // 64))
    return lib.hgemm_lora_workspace_bytes(T, N, K, r, A, S) == slices * T * r * 4


@pytest.mark.parametrize("K,N", [(4096, 4096), (4096, 14336), (4096, 28672), (14336, 4096), (28672, 8192),
                                 (8192, 57344), (4096, 128256)])
def test_lora_path_goes_by_the_width_of_the_projection(K, N):
    """One token is W's bytes, which the path that splits K streams at any width (4096 x 28672: 39 us against 58, 8192 x
    57344: 139 against 192); 128 tokens of a wide projection are read twice there (4096 x 28672: 125 us against 51)."""
    assert few_tokens(1, N, K, 16, 1, 1)
    assert few_tokens(1, N, K, 64, 32, 1)
    if N >= 14336:
        assert not few_tokens(128, N, K, 16, 1, 1)
        assert not few_tokens(256, N, K, 64, 32, 256)


def test_lora_path_goes_by_the_adapters():
    """Every adapter of a row tile is more k-blocks there (64 tokens x 4096 x 4096 of 32 adapters, rank 64: 45 us against
    25 here), of one adapter's tokens it takes all at once (512 tokens, rank 16: 45 against 57)."""
    assert few_tokens(64, 4096, 4096, 64, 32, 64)
    assert not few_tokens(512, 4096, 4096, 16, 1, 1)
    assert few_tokens(256, 880, 5760, 64, 32, 256)


WITHOUT = """
import importlib.abc, sys
class Gone(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path=None, target=None):
        if name in {names}:
            raise ModuleNotFoundError("No module named " + repr(name), name=name)
if {blank}:
    sys.modules.update(dict.fromkeys({names}))
else:
    sys.meta_path.insert(0, Gone())
from hopper_gemm_b200 import *
import hopper_gemm_b200 as hg
assert callable(launch) and hg.plan(64, 64, 64)["path"] == 1
assert not hasattr(hg, "lora") and "lora" not in globals() and "torch" not in [m for m in sys.modules if sys.modules[m]]
"""


@pytest.mark.parametrize("names", [["torch"], ["hopper_gemm_b200._operators"]])
@pytest.mark.parametrize("blank", [False, True])
def test_the_package_works_without_torch_or_the_binding(names, blank):
    """Star import and everything but the operators, which are no attributes then."""
    code = WITHOUT.format(names=names, blank=blank)
    if names != ["torch"]:
        code = code.replace(' and "torch" not in [m for m in sys.modules if sys.modules[m]]', "")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]


def test_star_import_brings_the_operators():
    names = {}
    exec("from hopper_gemm_b200 import *", names)
    assert callable(names["lora"]) and callable(names["qk_norm_rope"]) and callable(names["attn_prompt"])


def order(st):
    """Nothing is refused: the call gets as far as the device, of which there is none."""
    return status(st) != BAD


@pytest.mark.skipif(torch.cuda.is_available(), reason="an accepted call would run on made-up addresses")
@pytest.mark.parametrize("st", [lora_args(), norm_args(), attn_args(), attn_args(cu_k=None), norm_args(axes=3),
                                lora_args(adapters=0, down=None, up=None, scale=None), attn_args(lse=None)])
def test_arguments_in_order_are_not_refused(st):
    assert order(st)


@pytest.mark.parametrize("out", ["Y", "workspace"])
@pytest.mark.parametrize("name,last", [("X", 16 * 64 * 2), ("W", 64 * 64 * 2), ("down", 4 * 64 * 16 * 2),
                                       ("up", 4 * 64 * 16 * 2), ("scale", 16), ("seg_start", 12), ("seg_adapter", 8)])
def test_lora_outputs_over_inputs(out, name, last):
    """At an input's first byte, and at the 16 bytes that hold its last one."""
    at = getattr(lora_args(), name)
    for where in (at, at + (last - 1) // 16 * 16):
        assert status(lora_args(**{out: where})) == BAD


def test_lora_output_over_the_workspace():
    need = lib.hgemm_lora_workspace_bytes(16, 64, 64, 16, 4, 2)
    ws = lora_args().workspace
    for where in (ws, ws + (need - 1) // 16 * 16, ws - 16 * 64 * 2 + 16):
        assert status(lora_args(Y=where)) == BAD


@pytest.mark.parametrize("out,ins", [("q_out", "k"), ("k_out", "q"), ("q_out", "k_out"), ("q_out", "q_weight"),
                                     ("k_out", "k_weight"), ("k_out", "positions"), ("q_out", "inv_freq")])
def test_norm_outputs_over_other_operands(out, ins):
    assert status(norm_args(**{out: getattr(norm_args(), ins)})) == BAD


@pytest.mark.parametrize("over", [
    dict(q_out=16), dict(q_out=-16), dict(q_out=1024 * 2 * 15), dict(q_out=2048 - 16)])
def test_norm_output_over_a_part_of_its_input(over):
    """Shifted against the input, by less than a row or by whole rows."""
    base = norm_args().q
    assert status(norm_args(q_out=base + over["q_out"])) == BAD


@pytest.mark.parametrize("name", ["q", "k", "v", "cu_q", "cu_k"])
@pytest.mark.parametrize("out", ["out", "lse"])
def test_attn_outputs_over_inputs(out, name):
    st = attn_args()
    assert status(attn_args(**{out: getattr(st, name)})) == BAD


def test_attn_outputs_over_each_other_and_the_workspace():
    st = attn_args(total_q=2, total_k=20000)
    assert lib.hgemm_attn_prompt_workspace_bytes(2, 20000, 2, 8, 2, 128) > 0
    for a, b in (("out", "lse"), ("out", "workspace"), ("lse", "workspace"), ("workspace", "q"), ("workspace", "v")):
        assert status(attn_args(total_q=2, total_k=20000, **{a: getattr(st, b)})) == BAD


@pytest.mark.skipif(torch.cuda.is_available(), reason="an accepted call would run on made-up addresses")
def test_other_columns_of_the_same_rows_are_no_overlap():
    """Queries, keys, values and outputs as columns of one buffer, rows of 8 + 2 + 2 + 8 heads; the norm in place and
    into the columns behind."""
    wide, at = 20 * 128, 1 << 50
    cols = dict(q=at, k=at + 2 * 8 * 128, v=at + 2 * 10 * 128, out=at + 2 * 12 * 128, q_stride=wide, k_stride=wide,
                v_stride=wide, out_stride=wide)
    assert order(attn_args(**cols))
    for shift in (-16, 16):
        assert not order(attn_args(**{**cols, "out": cols["out"] + shift}))
    norm = dict(q=at, k=at + 2 * 8 * 128, q_out=at, k_out=at + 2 * 8 * 128, q_stride=wide, k_stride=wide,
                q_out_stride=wide, k_out_stride=wide)
    assert order(norm_args(**norm))
    assert order(norm_args(**{**norm, "q_out": at + 2 * 10 * 128}))
    assert not order(norm_args(**{**norm, "q_out": at + 2 * 9 * 128}))
    assert not order(norm_args(**{**norm, "k_out": at + 2 * 7 * 128}))
    # one token: its row ends where the row does
    assert order(norm_args(tokens=1, q=at, q_out=at + 2 * 1024)) and not order(norm_args(tokens=1, q=at, q_out=at + 16))


@pytest.mark.parametrize("st", [norm_args(q_stride=1 << 39), norm_args(k_out_stride=1 << 62), attn_args(v_stride=1 << 40),
                                attn_args(out_stride=1 << 60), attn_args(total_q=LIMIT, total_k=LIMIT, cu_k=None,
                                                                         q_stride=1 << 38, out_stride=1 << 38)])
def test_strides_beyond_any_memory_are_refused(st):
    """The last: rows of 2^31 times 2^39 bytes reach over every other operand."""
    assert status(st) == BAD


def test_the_binding_is_built_for_the_installed_torch(tmp_path, monkeypatch):
    """Another torch, an older binding, or none: it is built again."""
    from hopper_gemm_b200 import _operators, build
    where, version = build._torch()
    assert version == torch.__version__ and os.path.samefile(where, os.path.dirname(torch.__file__))
    assert _operators.built_for == build._built_for(version)
    assert not build._binding_stale(version)
    for other in ("1.0.0", version + "1", version[:-1]):
        assert build._binding_stale(other)
    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_operators.so"))
    assert build._binding_stale(version)


def test_products_of_the_largest_sizes_are_no_overlap_by_wrapping():
    """W of 2^31 x 2^31 halves is more than 64 bits count: it ends somewhere behind every other operand here, and a place
    inside it is refused."""
    most = LIMIT - LIMIT % 8
    st = lora_args(N=most, K=most)
    assert status(lora_args(N=most, K=most, Y=st.W + (1 << 30))) == BAD
    assert status(attn_args(total_q=LIMIT, total_k=LIMIT, cu_k=None, heads_q=1 << 20, heads_kv=1 << 20, head_dim=8,
                            q_stride=1 << 23, k_stride=1 << 23, v_stride=1 << 23, out_stride=1 << 23)) == BAD
