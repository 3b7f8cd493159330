"""GPU: the attention layer's operators at the values, masks and sizes where a rounding, a mask or a
repair shows. References and tolerances are plain 64-bit forms derived beside each test."""
import math
import os
import subprocess
import sys

import pytest
import torch

from tests import operators_ref as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
U16, U32 = ref.U16, ref.U32


def rand(seed, shape, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).half()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------- norm + rotation
@pytest.mark.parametrize("d,rot", [(80, 64), (64, 0), (128, 64), (256, 32), (24, 16), (128, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_of_a_head_with_an_infinity(cuda, d, rot, interleaved):
    """x * rsqrt(inf) is 0 wherever x is finite; NaN in the infinity's own place, and in its partner's where
    the pair turns. Every place of a head once, in a token and head of its own."""
    T, hq = d, 3
    q = rand(d, (T, hq + 1, d))
    for t in range(T):
        q[t, t % (hq + 1), t] = math.inf if t % 2 else -math.inf
    k, q = q[:, hq:], q[:, :hq]
    w = rand(1, (d,))
    pos = torch.arange(T, dtype=torch.int32, device=DEV) * 3 + 1
    inv = torch.rand(rot // 2, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    got = cuda.qk_norm_rope(q, k, w, w, pos, inv, interleaved=interleaved)
    axis = torch.zeros(rot // 2, device=DEV)
    for x, y, name in ((q, got[0], "q"), (k, got[1], "k")):
        want, tol = ref.qk_norm_rope(x, w, pos, inv, axis, 1e-6, interleaved)
        ref.close(y, want, tol, f"{name} d{d} rot{rot}")


# ------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("gap", [8.0, 15.0, 17.5, 19.0])
@pytest.mark.parametrize("rows,keys,hq,hkv", [(1, 131072, 8, 2), (1, 131072, 2, 2), (300, 131072, 2, 2), (17, 30000, 16, 1), (3000, 3000, 8, 2)])
def test_attn_one_key_above_many_small_ones(cuda, gap, rows, keys, hq, hkv):
    """Key 0 has the value 0 and scores `gap` above all others, whose values are 1: out = n e^-gap / (1 + n e^-gap).

    A weight's rounding to binary16 is U16 of it, and 2^-32 of the maximum at least (2^-25 under an exponent raised by 7);
    its exponential is 8 U32 off, the score itself exact; sums of n terms n U32; one rounding of the output."""
    d, n = 128, keys - 1
    q = torch.zeros((rows, hq, d), dtype=torch.float16, device=DEV)
    k = torch.zeros((keys, hkv, d), dtype=torch.float16, device=DEV)
    v = torch.ones((keys, hkv, d), dtype=torch.float16, device=DEV)
    q[..., 3] = 1
    k[0, :, 3] = gap
    v[0] = 0
    lse = torch.empty((rows, hq), device=DEV)
    out = cuda.attn_prompt(q, k, v, i32([0, rows]), i32([0, keys]), scale=1.0, causal=False, lse=lse)
    w = math.exp(-gap)
    want = n * w / (1 + n * w)
    tol = n * (w * (U16 + 8 * U32) + 2.0 ** -32) / (1 + n * w) + (n + 16) * U32 * want + U16 * want + ref.TINY
    err = (out.double() - want).abs().max().item()
    assert err <= tol, (err, tol, want)
    z = math.log1p(n * w)
    assert (lse.double() - (gap + z)).abs().max().item() <= (n + 16) * U32 + 8 * U32 * gap


@pytest.mark.parametrize("q_lens,k_lens,hq,hkv,d", [([70, 5], [70, 5], 4, 2, 64), ([1, 1], [9000, 40], 8, 2, 128), ([1], [700], 4, 4, 64),
                                                    ([40], [5000], 4, 1, 128), ([2], [20000], 8, 2, 64)])
def test_attn_rows_whose_scores_are_all_minus_infinity(cuda, q_lens, k_lens, hq, hkv, d):
    """Seen keys of score -infinity are no missing keys: softmax is 0 / 0, so NaN, and the sum's logarithm -infinity,
    whether the keys are split into ranges or not."""
    tq, tk = sum(q_lens), sum(k_lens)
    q, k, v = rand(1, (tq, hq, d)), rand(2, (tk, hkv, d)), rand(3, (tk, hkv, d))
    q[..., 0] = q[..., 0].abs() + 1
    k[:k_lens[0], 0, 0] = -math.inf
    lse = torch.full((tq, hq), 7.0, device=DEV)
    cq, ck = i32([0] + list(torch.tensor(q_lens).cumsum(0))), i32([0] + list(torch.tensor(k_lens).cumsum(0)))
    out = cuda.attn_prompt(q, k, v, cq, ck, lse=lse)
    g, n = hq // hkv, q_lens[0]
    assert out[:n, :g].isnan().all()
    assert (lse[:n, :g] == -math.inf).all()
    assert out[:n, g:].isfinite().all() and out[n:].isfinite().all()


@pytest.mark.parametrize("q_len,keys", [(1, 9000), (1, 700), (40, 5000), (200, 900)])
def test_attn_some_ranges_of_minus_infinity(cuda, q_len, keys):
    """Weights of exactly 0 in whole key ranges: they count for nothing, but 0 * infinity is NaN in the one column
    where a value among them is infinite."""
    hq, hkv, d = 4, 2, 64
    q, k, v = rand(4, (q_len, hq, d)), rand(5, (keys, hkv, d)), rand(6, (keys, hkv, d))
    q[..., 0] = q[..., 0].abs() + 1
    dead = slice(0, keys * 3 // 4)
    k[dead, :, 0] = -math.inf
    want, tol, wl, tl = ref.attn(q, k[dead.stop:], v[dead.stop:], [q_len], [keys - dead.stop], d ** -0.5, True)
    lse = torch.empty((q_len, hq), device=DEV)
    out = cuda.attn_prompt(q, k, v, i32([0, q_len]), i32([0, keys]), lse=lse)
    ref.close(out, want, tol, "dead keys")
    ref.close(lse, wl, tl, "lse")
    v[keys // 3, 1, 7] = math.inf
    out = cuda.attn_prompt(q, k, v, i32([0, q_len]), i32([0, keys]))
    want[:, 2:, 7] = math.nan
    ref.close(out, want, tol, "an infinite value among them")


@pytest.mark.parametrize("rows,hq", [(1, 1), (1, 32), (16, 8)])
def test_attn_few_rows_keep_22_bits_of_a_weight(cuda, rows, hq):
    """Two keys whose weights differ by 2^-13, values 1 and -1: 1 - (1 - 2^-13) is lost where weights have 11 bits.
    With 22 they are off by 2^-23, their exponentials by 8 U32 and the scores' product by 132 U32 of 2^-13."""
    d, eps = 128, 2.0 ** -13
    q = torch.zeros((rows, hq, d), dtype=torch.float16, device=DEV)
    k = torch.zeros((2, hq, d), dtype=torch.float16, device=DEV)
    v = torch.ones((2, hq, d), dtype=torch.float16, device=DEV)
    q[..., 5] = 1
    k[1, :, 5] = -eps
    v[1] = -1
    out = cuda.attn_prompt(q, k, v, i32([0, rows]), i32([0, 2]), scale=1.0, causal=False)
    w = math.exp(-eps)
    want = (1 - w) / (1 + w)
    tol = (2.0 ** -23 + 8 * U32 + 132 * U32 * eps) + U16 * want + ref.TINY
    assert (out.double() - want).abs().max().item() <= tol


# ------------------------------------------------------------------------------- lora
def pass_us(fn):
    best = math.inf
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        fn()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


def test_lora_a_request_of_nan_does_not_stall_the_others(cuda):
    """Half of 1200 tokens are NaN: their rows are NaN and cost no more than a few calls' time."""
    T, K, N, r, A = 1200, 4096, 4096, 16, 6
    X, W = rand(1, (T, K)), rand(2, (K, N), K ** -0.5)
    down, up = rand(3, (A, K, r), K ** -0.5), rand(4, (A, r, N), r ** -0.5)
    scale = torch.ones(A, device=DEV)
    seg, ids = i32([0, 200, 800, 1000, T]), i32([1, 4, 2, 0])
    args = (W, down, up, scale, seg, ids)
    want = cuda.lora(X, *args)
    bad = X.clone()
    bad[200:800] = math.nan
    got = cuda.lora(bad, *args)
    assert got[200:800].isnan().all()
    assert torch.equal(got[:200], want[:200]) and torch.equal(got[800:], want[800:])
    clean, stalled = pass_us(lambda: cuda.lora(X, *args)), pass_us(lambda: cuda.lora(bad, *args))
    assert stalled < 10 * clean + 500, (clean, stalled)


@pytest.mark.parametrize("what", [math.inf, math.nan])
def test_lora_an_adapter_of_infinities_costs_the_others_little(cuda, what):
    """One adapter's Up is not finite in some columns: its own tokens show it there, the other tokens of its
    row tiles are formed again, in a few calls' time."""
    T, K, N, r, A = 1200, 4096, 4096, 24, 6
    X, W = rand(1, (T, K)), rand(2, (K, N), K ** -0.5)
    down, up = rand(3, (A, K, r), K ** -0.5), rand(4, (A, r, N), r ** -0.5)
    scale = torch.ones(A, device=DEV)
    starts, ids = [0, 200, 210, 800, 1000, T], [1, 4, 2, -1, 0]
    broken = [5, 64, 1000, 1001, N - 1]
    want, tol = ref.lora(X, W, down, up, scale, ref.token_adapters(T, starts, ids, A))
    up[4, :, broken] = what
    call = lambda: cuda.lora(X, W, down, up, scale, i32(starts), i32(ids))  # noqa: E731
    got = call()
    assert not got[200:210][:, broken].isfinite().any()
    want[200:210, broken] = got[200:210, broken].double()
    ref.close(got, want, tol, "other tokens")
    up[4] = what
    got = call()
    assert not got[200:210].isfinite().any()
    want[200:210] = got[200:210].double()
    ref.close(got, want, tol, "all columns")
    us = pass_us(call)
    print("one adapter of infinities:", us, "us")
    assert us < 20000, us


# ------------------------------------------------------------------------------- lora: tables and tiles
@pytest.mark.parametrize("T,A,segs,K,N", [
    (1500, 5, 1500, 256, 512), (1500, 1100, 1500, 256, 512), (1500, 1100, 9, 256, 512),
    (4100, 3, 4100, 512, 4096), (4100, 40, 70, 512, 4096), (1025, 2, 1024, 64, 264), (700, 300, 1023, 128, 136)])
def test_lora_tables_of_many_segments_and_adapters(cuda, T, A, segs, K, N):
    """More segments and adapters than the tables in shared memory hold, entries by tiles and by segments, several
    adapters to a tile, empty segments."""
    r = 24
    X, W = rand(T, (T, K)), rand(A, (K, N), K ** -0.5)
    down, up = rand(segs, (A, K, r), K ** -0.5), rand(K, (A, r, N), r ** -0.5)
    scale = torch.rand(A, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) + 0.5
    cut = [min(T, s * T // segs + (s % 3 == 1 and segs < T)) for s in range(segs)] + [T]
    ids = [(s * 7919) % (A + 1) - 1 for s in range(segs)]
    got = cuda.lora(X, W, down, up, scale, i32(cut), i32(ids))
    want, tol = ref.lora(X, W, down, up, scale, ref.token_adapters(T, cut, ids, A))
    ref.close(got, want, tol, "lora")
    assert cuda.device_status(clear=True) == (0, 0)


TILES = {(1, 64): (700, 520, 1024), (1, 128): (700, 520, 264), (1, 256): (700, 4104, 512),
         (2, 128): (777, 2056, 2048), (2, 256): (700, 6144, 1024), (2, 512): (1037, 6144, 1024)}


@pytest.mark.parametrize("tile", sorted(TILES))
def test_lora_infinities_do_not_leak_in_any_tile(cuda, tile):
    """Columns of one adapter's Up are infinite: in every tile of the GEMM its blocks are listed and the other
    requests' rows formed again."""
    T, N, K = TILES[tile]
    r, A = 72, 4
    plan = cuda.plan(T, N, K)
    assert (plan["pair"], plan["tile_n"]) == tile and plan["ksplit"] == 1
    X, W = rand(T, (T, K)), rand(N, (K, N), K ** -0.5)
    down, up = rand(3, (A, K, r), K ** -0.5), rand(4, (A, r, N), r ** -0.5)
    scale = torch.ones(A, device=DEV)
    cut, ids = [0, T // 3, T // 3 + 5, T - 70, T - 1, T], [0, 2, 1, -1, 3]
    want, tol = ref.lora(X, W, down, up, scale, ref.token_adapters(T, cut, ids, A))
    broken = [0, 9, N // 2, N // 2 + 1, N - 1]
    up[2, :, broken] = math.inf
    up[3, 5, broken] = -math.inf
    got = cuda.lora(X, W, down, up, scale, i32(cut), i32(ids))
    for own in (slice(T // 3, T // 3 + 5), slice(T - 1, T)):
        assert not got[own][:, broken].isfinite().any()
        want[own, broken] = got[own, broken].double()
    ref.close(got, want, tol, f"tile {tile}")
    assert cuda.device_status(clear=True) == (0, 0)


@pytest.mark.parametrize("T,K,N,r", [(1, 264, 28672, 16), (1, 64, 128256, 8), (48, 1024, 14336, 32), (70, 520, 33352, 16),
                                     (16, 14336, 136, 64), (200, 14336, 264, 16), (130, 512, 28672, 64)])
def test_lora_wide_and_long_projections(cuda, T, K, N, r):
    A = 6
    X, W = rand(T, (T, K)), rand(N, (K, N), K ** -0.5)
    down, up = rand(K, (A, K, r), K ** -0.5), rand(r, (A, r, N), r ** -0.5)
    scale = torch.rand(A, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) + 0.5
    cut, ids = list(range(T + 1)), [(5 * t) % (A + 1) - 1 for t in range(T)]
    for cut, ids in ((cut, ids), ([0, T // 2, T], [3, 1])):
        got = cuda.lora(X, W, down, up, scale, i32(cut), i32(ids))
        want, tol = ref.lora(X, W, down, up, scale, ref.token_adapters(T, cut, ids, A))
        ref.close(got, want, tol, f"lora {T}x{K}x{N}")
    assert cuda.device_status(clear=True) == (0, 0)


# ------------------------------------------------------------------------------- after a device reset
RESET = """
import ctypes, glob, os, sys
import hopper_gemm_b200 as hg
from hopper_gemm_b200._native import HgemmAttnPrompt, HgemmLora, HgemmQkNormRope
cudart = ctypes.CDLL("libcudart.so.12")

def once():
    def mem(n):
        p = ctypes.c_void_p()
        assert cudart.cudaMalloc(ctypes.byref(p), ctypes.c_size_t(n)) == 0
        assert cudart.cudaMemset(p, 0, ctypes.c_size_t(n)) == 0
        return p.value
    a = HgemmLora()
    for n in ("X", "W", "Y", "down", "up", "scale", "seg_start", "seg_adapter", "workspace"):
        setattr(a, n, mem(1 << 22))
    a.workspace_bytes, a.N, a.K, a.rank, a.adapters, a.segments = 1 << 22, 512, 512, 16, 2, 2
    out = []
    for a.tokens in (3, 700):
        out.append(hg.lib.hgemm_lora(ctypes.byref(a), None))
    b = HgemmAttnPrompt()
    for n in ("q", "k", "v", "out", "cu_q", "workspace"):
        setattr(b, n, mem(1 << 22))
    b.q_stride = b.k_stride = b.v_stride = b.out_stride = 512
    b.workspace_bytes, b.total_q, b.total_k, b.batch = 1 << 22, 300, 300, 2
    b.heads_q, b.heads_kv, b.head_dim, b.causal, b.scale = 4, 4, 128, 1, 0.1
    out.append(hg.lib.hgemm_attn_prompt(ctypes.byref(b), None))
    out.append(hg.lib.hgemm_launch(a.X, a.W, a.Y, 512, 512, 512, 1.0, 0.0, None))
    return out + [cudart.cudaDeviceSynchronize()] + list(hg.device_status(clear=True))

assert once() == [0] * 7
assert cudart.cudaDeviceReset() == 0
hg.release()
got = once()
assert got == [0] * 7, got
"""


def test_calls_after_a_device_reset(cuda):
    """hgemm_release() forgets what a reset of the device took: the calls of a new context set it up again."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, LD_LIBRARY_PATH="/usr/local/cuda/lib64:" + os.environ.get("LD_LIBRARY_PATH", ""))
    run = subprocess.run([sys.executable, "-c", RESET], cwd=root, env=env, timeout=120, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]


# ------------------------------------------------------------------------------- outputs that autograd has saved
def test_outputs_of_the_caller_are_known_as_written(cuda):
    """A tensor that another operation keeps for its gradient, written by an operator: backward says so instead of going on
    with other values. Inference tensors have no such count."""
    w = rand(1, (64,))
    pos, inv = i32(list(range(6))), torch.ones(32, device=DEV)
    x = rand(2, (6, 4, 64)).requires_grad_()

    def kept():
        y = x * 2
        return y, (y * y).sum()

    y, z = kept()
    cuda.qk_norm_rope(y[:, :3], y[:, 3:], w, w, pos, inv, q_out=y[:, :3])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    y, z = kept()
    cuda.qk_norm_rope(y[:, :3], y[:, 3:], w, w, pos, inv, k_out=y[:, 3:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    y, z = kept()
    q = rand(3, (6, 4, 64))
    cuda.attn_prompt(q, q, q, i32([0, 6]), out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    lse = torch.ones((6, 4), device=DEV, requires_grad=True) * 2
    z = (lse * lse).sum()
    cuda.attn_prompt(q, q, q, i32([0, 6]), lse=lse)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    y, z = kept()
    down, up = rand(4, (1, 64, 8)), rand(5, (1, 8, 64))
    cuda.lora(rand(6, (24, 64)), rand(7, (64, 64)), down, up, torch.ones(1, device=DEV), i32([0, 24]), i32([0]),
              Y=y.view(24, 64))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    y, z = kept()
    cuda.attn_prompt(q, q, q, i32([0, 6]))
    z.backward()
    with torch.inference_mode():
        out = torch.empty_like(q)
        cuda.attn_prompt(q, q, q, i32([0, 6]), out=out)
    assert torch.equal(out, cuda.attn_prompt(q, q, q, i32([0, 6])))
    cuda.attn_prompt(q, q, q, i32([0, 6]), out=out)


# ------------------------------------------------------------------------------- a cache with room to grow
@pytest.mark.parametrize("behind", [0.0, 7.0, math.nan])
def test_attn_cache_of_slots_with_room(cuda, behind):
    """Single tokens over slots that are not full: a sequence without queries stands for the rest of each. A captured step
    follows the starts as the sequences grow."""
    slots, size, hq, hkv, d = 5, 700, 8, 2, 128
    fill = [1, 64, 130, 699, 317]
    k, v, q = rand(1, (slots * size, hkv, d)), rand(2, (slots * size, hkv, d)), rand(3, (slots, hq, d))
    store = [k.clone(), v.clone()]

    def cu_k():
        return [0] + [x for s in range(slots) for x in (s * size + fill[s], (s + 1) * size)]

    def blank():
        for t, full in zip((k, v), store):
            for s in range(slots):
                t[s * size:(s + 1) * size] = full[s * size:(s + 1) * size]
                t[s * size + fill[s]:(s + 1) * size] = behind

    cq, ck = i32([0] + [x for s in range(slots) for x in (s + 1, s + 1)]), i32(cu_k())
    out = torch.empty_like(q)

    def check():
        for s in range(slots):
            rows = slice(s * size, s * size + fill[s])
            want, tol, _, _ = ref.attn(q[s:s + 1], k[rows], v[rows], [1], [fill[s]], d ** -0.5, True)
            ref.close(out[s:s + 1], want, tol, f"slot {s} of {fill[s]}")

    blank()
    cuda.attn_prompt(q, k, v, cq, ck, out=out)
    check()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cuda.attn_prompt(q, k, v, cq, ck, out=out)
    for _ in range(2):
        fill = [min(size, n + 1) for n in fill]
        blank()
        ck.copy_(i32(cu_k()))
        graph.replay()
        check()
    assert cuda.device_status(clear=True) == (0, 0)
