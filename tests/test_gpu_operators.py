"""GPU: the attention layer's operators against plain 64-bit forms, at the sizes, masks, strides and
values where they can go wrong."""
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

from tests import operators_ref as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def rand(g, shape, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).half()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def status_clear(hg):
    assert hg.device_status(clear=True) == (0, 0)


# ------------------------------------------------------------------------------- lora
def lora_case(T, K, N, r, A, seed=0):
    g = gen(seed)
    return (rand(g, (T, K)), rand(g, (K, N), K ** -0.5), rand(g, (A, K, r), K ** -0.5),
            rand(g, (A, r, N), r ** -0.5), torch.rand(A, generator=g, device=DEV) * 2 - 0.5)


def check_lora(hg, T, K, N, r, A, seg_start, seg_adapter, seed=0):
    X, W, down, up, scale = lora_case(T, K, N, r, A, seed)
    Y = hg.lora(X, W, down, up, scale, i32(seg_start), i32(seg_adapter))
    ids = ref.token_adapters(T, seg_start, seg_adapter, A)
    want, tol = ref.lora(X, W, down, up, scale, ids)
    ref.close(Y, want, tol, f"lora {T}x{K}x{N} r{r}")
    status_clear(hg)


@pytest.mark.parametrize("T,K,N,r", [
    (1, 8, 8, 8), (1, 4096, 4096, 16), (1, 520, 1000, 40), (2, 64, 72, 8), (3, 1000, 136, 24),
    (16, 512, 264, 64), (17, 2048, 4096, 16), (33, 136, 2000, 32), (48, 4096, 6144, 32),
    (63, 1032, 520, 128), (64, 256, 256, 256), (65, 256, 520, 72), (127, 776, 1032, 16),
    (128, 512, 512, 64), (129, 64, 64, 8), (257, 1096, 1800, 128), (300, 2048, 4104, 200),
    (777, 1544, 2056, 64), (1025, 1024, 2048, 16)])
def test_lora_sizes(cuda, T, K, N, r):
    """Three segments of three adapters over the tokens, or one for a single token."""
    if T < 3:
        check_lora(cuda, T, K, N, r, 2, [0, T], [1])
    else:
        a, b = T // 3, T - T // 4
        check_lora(cuda, T, K, N, r, 3, [0, a, b, T], [2, 0, 1])


@pytest.mark.parametrize("T,N,K", [
    (65, 72, 512), (65, 512, 512), (65, 8, 64), (65, 512, 64), (513, 4096, 64), (257, 4104, 1024),
    (513, 2048, 1024), (2049, 2056, 264), (1500, 4096, 264), (3000, 2056, 2048), (777, 8192, 1024),
    (4100, 4096, 2048)])
def test_lora_tiles(cuda, T, N, K):
    """Every tile of the GEMM, whole in N and not, with several adapters to a tile and a rank of two
    64-column blocks."""
    cut = [0, T // 9, T // 5, T // 5 + 1, T // 2, T - T // 3, T - 2, T]
    check_lora(cuda, T, K, N, 72, 6, cut, [5, 0, -1, 3, 0, 4, 1], seed=N)


@pytest.mark.parametrize("T,N,K", [(65, 72, 512), (65, 512, 512), (65, 8, 64), (65, 512, 64),
                                   (40, 520, 136), (9, 136, 72)])
def test_lora_tiles_of_few_tokens_at_a_high_rank(cuda, T, N, K):
    """Few tokens whose adapters weigh more than the projection."""
    cut = [0, T // 9, T // 5, T // 5 + 1, T // 2, T - T // 3, T - 2, T]
    check_lora(cuda, T, K, N, 256, 6, cut, [5, 0, -1, 3, 0, 4, 1], seed=T)


@pytest.mark.parametrize("T", [63, 64, 65, 127, 128, 129, 300, 511, 512, 513])
@pytest.mark.parametrize("K,N", [(1032, 264), (64, 1160), (2048, 128)])
def test_lora_tokens_in_chunks_of_64(cuda, T, K, N):
    """Batches that one CTA's 64 tokens do not hold, at a low rank; requests across the chunks."""
    cut = [0, 1, T // 3, T // 3 + 1, T - 20, T - 3]
    check_lora(cuda, T, K, N, 8, 5, cut, [2, 4, -1, 0, 3], seed=T)


@pytest.mark.parametrize("T", [40, 64, 200, 515])
@pytest.mark.parametrize("r", [16, 96])
def test_lora_segments(cuda, T, r):
    """Empty segments, one-token segments, gaps before and behind, no adapter, an index behind the pool,
    one adapter in many segments."""
    seg = [2, 2, 3, 4, 9, 9, 20, 21, 30, T - 3]
    check_lora(cuda, T, 264, 528, r, 5, seg, [0, 1, 2, -1, 3, 4, 7, 2, 1], seed=T + r)


@pytest.mark.parametrize("T", [1, 31, 64, 150, 300])
def test_lora_one_token_segments(cuda, T):
    """A decoding batch: every token its own request, adapters shared and not."""
    ids = [(7 * t) % 50 - 1 for t in range(T)]
    check_lora(cuda, T, 512, 1024, 32, 48, list(range(T + 1)), ids, seed=T)
    check_lora(cuda, T, 512, 1024, 16, T, list(range(T + 1)), list(range(T)), seed=T)


def test_lora_without_adapters(cuda):
    for T in (5, 200):
        X, W, down, up, scale = lora_case(T, 264, 520, 16, 2)
        base, tol = ref.lora(X, W, down, up, scale, [-1] * T)
        none = torch.empty(0, dtype=torch.int32, device=DEV)
        ref.close(cuda.lora(X, W, down, up, scale, i32([0]), none), base, tol, "no segment")
        ref.close(cuda.lora(X, W, down, up, scale, i32([0, T]), i32([-1])), base, tol, "none")
        empty = cuda.lora(X, W, down[:0], up[:0], scale[:0], i32([0, T]), i32([0]))
        ref.close(empty, base, tol, "no adapters")


@pytest.mark.parametrize("T", [6, 64, 130, 400])
def test_lora_other_adapters_and_tokens_do_not_leak(cuda, T):
    """NaN and infinities in adapters that a token does not use, and in other tokens' rows."""
    X, W, down, up, scale = lora_case(T, 328, 520, 24, 4, seed=T)
    seg, ids = [0, 2, T // 2, T - 1, T], [0, 1, 2, 0]
    down[3], up[3], scale[3] = math.nan, math.inf, math.nan
    up[1] = math.nan
    X[T - 1] = math.inf
    owner = ref.token_adapters(T, seg, ids, 4)
    Y = cuda.lora(X, W, down, up, scale, i32(seg), i32(ids))
    clean = [t for t in range(T - 1) if owner[t] != 1]
    up2 = up.clone()
    up2[1] = 0
    want, tol = ref.lora(X[:T - 1], W, down, up2, scale, owner[:T - 1])
    ref.close(Y[clean], want[clean], tol[clean], "other adapters")
    assert not Y[2:T // 2].isfinite().any()
    status_clear(cuda)


@pytest.mark.parametrize("T", [4, 70, 300])
def test_lora_starts_that_are_not_ascending_stay_in_bounds(cuda, T):
    """Any contents of the segment tensors: no fault, and tokens of no adapter exact."""
    X, W, down, up, scale = lora_case(T, 128, 256, 16, 2)
    guard = torch.full((T + 64, 256), 7.0, dtype=torch.float16, device=DEV)
    for seg, ids in (([T, 5, -9, 1 << 30], [0, 1, 1]), ([0, 1 << 30, 3, T], [1, 0, 1]),
                     ([-5, -1, -3, 2], [0, 1, 0])):
        cuda.lora(X, W, down, up, scale, i32(seg), i32(ids), Y=guard[:T])
        assert (guard[T:] == 7).all()
    status_clear(cuda)


def test_lora_offsets_beyond_32_bits(cuda):
    """An adapter pool larger than 2^32 bytes: its last adapter."""
    A, K, N, r = 1100, 8192, 8192, 256
    X, W = rand(gen(1), (70, K)), rand(gen(2), (K, N), K ** -0.5)
    down = torch.zeros((A, K, r), dtype=torch.float16, device=DEV)
    up = torch.zeros((A, r, N), dtype=torch.float16, device=DEV)
    assert down[-1].data_ptr() - down.data_ptr() > 1 << 32
    down[-1] = rand(gen(3), (K, r), K ** -0.5)
    up[-1] = rand(gen(4), (r, N), r ** -0.5)
    scale = torch.ones(A, device=DEV)
    for T in (3, 70):
        Y = cuda.lora(X[:T], W, down, up, scale, i32([0, T]), i32([A - 1]))
        want, tol = ref.lora(X[:T], W, down, up, scale, [A - 1] * T)
        ref.close(Y, want, tol, "last adapter")


# ------------------------------------------------------------------------------- norm + rotation
def check_norm(hg, T, hq, hk, d, rot, axes=1, interleaved=False, far=1000, eps=1e-6, in_place=False,
               seed=0, std=1.0):
    g = gen(seed)
    qkv = rand(g, (T, hq + 2 * hk + 1, d), std)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    wq, wk = rand(g, (d,)), rand(g, (d,))
    pos = torch.randint(-far, far, (axes, T), generator=g, device=DEV, dtype=torch.int32)
    inv = torch.tensor([10000.0 ** (-2 * i / max(rot, 1)) for i in range(rot // 2)],
                       dtype=torch.float32, device=DEV)
    axis = torch.tensor([i % axes for i in range(rot // 2)], dtype=torch.uint8, device=DEV)
    want = [ref.qk_norm_rope(x, w, pos, inv, axis, eps, interleaved) for x, w in ((q, wq), (k, wk))]
    rest = qkv[:, hq + hk:].clone()
    over = dict(q_out=q, k_out=k) if in_place else {}
    got = hg.qk_norm_rope(q, k, wq, wk, pos if axes > 1 else pos[0], inv, eps=eps,
                          axis_of=axis if axes > 1 else None, interleaved=interleaved, **over)
    for o, (w, tol), name in zip(got, want, "qk"):
        ref.close(o, w, tol, f"{name} T{T} d{d} rot{rot}")
    assert torch.equal(qkv[:, hq + hk:], rest)


@pytest.mark.parametrize("d,rot", [(8, 0), (16, 16), (24, 16), (64, 64), (64, 32), (72, 64), (80, 80),
                                   (96, 48), (112, 112), (128, 128), (128, 64), (136, 128),
                                   (192, 192), (256, 256), (256, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_dims(cuda, d, rot, interleaved):
    check_norm(cuda, 37, 6, 2, d, rot, interleaved=interleaved, seed=d + rot)


@pytest.mark.parametrize("T,hq,hk", [(1, 32, 8), (2, 1, 1), (5, 71, 1), (48, 32, 8), (295, 3, 3),
                                     (296, 40, 8), (1183, 12, 4), (4737, 8, 2), (9001, 5, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_tokens(cuda, T, hq, hk, in_place):
    check_norm(cuda, T, hq, hk, 128, 128, in_place=in_place, seed=T)


@pytest.mark.parametrize("axes", [2, 3, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_axes(cuda, axes, interleaved):
    check_norm(cuda, 301, 4, 2, 80, 64, axes=axes, interleaved=interleaved, seed=axes)


def test_norm_far_positions(cuda):
    """The whole range of int32: an angle of 2^31 - 1 turns as exactly as a near one."""
    check_norm(cuda, 64, 4, 2, 128, 128, far=2 ** 31 - 1)
    check_norm(cuda, 64, 4, 2, 64, 64, far=2 ** 31 - 1, interleaved=True)


def test_norm_small_and_zero_rows(cuda):
    check_norm(cuda, 9, 2, 2, 128, 128, std=1e-4)
    check_norm(cuda, 9, 2, 2, 128, 128, std=0.0)
    check_norm(cuda, 9, 2, 2, 64, 64, std=2000.0, eps=0.0)


def test_norm_one_side(cuda):
    """Queries without keys, as where the keys come from a cache."""
    g = gen(3)
    q, w = rand(g, (10, 4, 64)), rand(g, (64,))
    pos = torch.arange(10, dtype=torch.int32, device=DEV)
    inv = torch.rand(32, generator=g, device=DEV)
    out, none = cuda.qk_norm_rope(q, q[:, :0], w, w, pos, inv)
    want, tol = ref.qk_norm_rope(q, w, pos, inv, torch.zeros(32, device=DEV), 1e-6, False)
    ref.close(out, want, tol, "q alone")
    assert none.shape == (10, 0, 64)


def test_norm_axis_behind_the_last_counts_as_the_last(cuda):
    g = gen(4)
    q, k, w = rand(g, (7, 2, 64)), rand(g, (7, 1, 64)), rand(g, (64,))
    pos = torch.randint(0, 99, (2, 7), generator=g, device=DEV, dtype=torch.int32)
    inv = torch.rand(32, generator=g, device=DEV)
    wild = torch.full((32,), 200, dtype=torch.uint8, device=DEV)
    last = torch.ones(32, dtype=torch.uint8, device=DEV)
    a = cuda.qk_norm_rope(q, k, w, w, pos, inv, axis_of=wild)
    b = cuda.qk_norm_rope(q, k, w, w, pos, inv, axis_of=last)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------- attention
def attn_case(q_lens, k_lens, hq, hkv, d, seed=0, extra=0, packed=False, std=1.0):
    g = gen(seed)
    tq, tk = sum(q_lens) + extra, sum(k_lens) + extra
    if packed:
        qkv = rand(g, (tq, hq + 2 * hkv, d), std)
        return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    return rand(g, (tq, hq, d), std), rand(g, (tk, hkv, d), std), rand(g, (tk, hkv, d))


def check_attn(hg, q_lens, k_lens, hq, hkv, d, causal=True, scale=None, seed=0, extra=0,
               packed=False, std=1.0, edit=None):
    q, k, v = attn_case(q_lens, k_lens, hq, hkv, d, seed, extra, packed, std)
    if edit:
        edit(q, k, v)
    scale = d ** -0.5 if scale is None else scale
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    same = q_lens == k_lens
    got = hg.attn_prompt(q, k, v, i32(starts(q_lens)), None if same else i32(starts(k_lens)),
                         scale=scale, causal=causal, out=out, lse=lse)
    assert got is out
    want, tol, wl, tl = ref.attn(q, k, v, q_lens, k_lens, scale, causal)
    n = sum(q_lens)
    ref.close(out[:n], want[:n], tol[:n], f"out {q_lens[:6]} {k_lens[:6]} d{d}")
    if edit is None:
        ref.close(lse[:n], wl[:n], tl[:n], f"lse {q_lens[:6]} {k_lens[:6]} d{d}")
    assert (out[n:] == 7).all() and (lse[n:] == 7).all(), "rows behind the last sequence"
    status_clear(hg)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 1031])
@pytest.mark.parametrize("d", [64, 128])
def test_attn_lengths(cuda, n, d):
    check_attn(cuda, [n], [n], 8, 2, d, seed=n)
    check_attn(cuda, [n], [n], 2, 2, d, causal=False, seed=n)


@pytest.mark.parametrize("d", [8, 16, 24, 40, 56, 72, 80, 96, 104, 112, 120])
def test_attn_head_dims(cuda, d):
    check_attn(cuda, [150, 3, 77], [150, 3, 77], 4, 2, d, seed=d, extra=5)
    check_attn(cuda, [2, 140], [400, 141], 4, 2, d, seed=d)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 1), (6, 2), (7, 1), (16, 1), (33, 1), (64, 1),
                                    (65, 1), (71, 1), (128, 1), (48, 8), (16, 16)])
def test_attn_groups(cuda, hq, hkv):
    check_attn(cuda, [45, 130], [45, 130], hq, hkv, 64, seed=hq)
    check_attn(cuda, [1, 3], [300, 900], hq, hkv, 128, seed=hq)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("packed", [True, False])
def test_attn_packed_sequences(cuda, causal, packed):
    """Uneven lengths, empty sequences, single tokens, rows behind the last one."""
    lens = [0, 5, 129, 0, 1, 64, 300, 1, 1, 17, 256, 0]
    check_attn(cuda, lens, lens, 8, 2, 128, causal=causal, extra=37, packed=packed)
    check_attn(cuda, lens, lens, 6, 2, 64, causal=causal, extra=37, packed=packed)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_attn_appended_prompts(cuda, causal, d):
    """Keys before the first query; fewer keys than queries (rows without a key); no keys at all."""
    q = [3, 70, 128, 1, 200, 5, 0, 9, 260]
    k = [500, 71, 129, 1000, 60, 0, 77, 3, 1]
    check_attn(cuda, q, k, 8, 2, d, causal=causal, seed=3)


@pytest.mark.parametrize("nk", [1, 2, 127, 128, 129, 1000, 5000, 20011])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (14, 2, 80)])
def test_attn_single_tokens(cuda, nk, hq, hkv, d):
    """One new token each over keys of uneven lengths, down to one key and none."""
    check_attn(cuda, [1, 1, 1, 1], [nk, max(1, nk // 3), 0, 1], hq, hkv, d, seed=nk)
    check_attn(cuda, [1], [nk], hq, hkv, d, seed=nk)


@pytest.mark.parametrize("q,k,hq,hkv,d", [
    ([300], [7000], 4, 1, 128), ([700, 1, 650], [7000, 12000, 6200], 16, 8, 128),
    ([129, 65], [6200, 6300], 8, 8, 96), ([1000, 0, 40, 900], [6000, 9000, 20000, 900], 16, 8, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_long_keys(cuda, q, k, hq, hkv, d, causal):
    """Prompts over many keys: two row tiles to a CTA, key ranges joined and not, one tile without rows."""
    check_attn(cuda, q, k, hq, hkv, d, causal=causal, seed=len(q))


def test_attn_many_sequences(cuda):
    lens = [(i * 37) % 90 for i in range(300)]
    check_attn(cuda, lens, lens, 4, 1, 64, extra=3)
    check_attn(cuda, [1] * 300, [(i * 91) % 700 for i in range(300)], 8, 2, 128)


def test_attn_growing_maximum(cuda):
    """Scores that rise and fall over hundreds of units along the keys, so that the running maximum moves often."""
    def edit(q, k, v):
        n = k.shape[0]
        ramp = torch.linspace(-6, 6, n, device=DEV)[:, None, None]
        k.copy_((k.float() * 0.2 + ramp).half())
        q.copy_((q.float().abs() + 1).half())
    for d in (64, 128):
        check_attn(cuda, [700], [700], 4, 2, d, edit=edit)
        check_attn(cuda, [2], [3000], 4, 2, d, edit=edit)

    def fall(q, k, v):
        edit(q, k, v)
        k.copy_(k.flip(0))
    check_attn(cuda, [700], [700], 4, 2, 128, edit=fall)
    check_attn(cuda, [300], [7000], 4, 1, 128, edit=edit)
    check_attn(cuda, [700], [6500], 16, 8, 128, edit=edit)


def test_attn_scale(cuda):
    check_attn(cuda, [200], [200], 4, 2, 64, scale=0.0)
    check_attn(cuda, [200], [200], 4, 2, 64, scale=2.0)


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, 65504.0])
@pytest.mark.parametrize("d", [64, 128])
def test_attn_masked_places_do_not_matter(cuda, what, d):
    """Anything may stand in later tokens, in other sequences and behind the last one: a row sees none of
    it. Rows that do see it are left out."""
    lens, hq, hkv = [70, 200, 131], 4, 2
    q, k, v = attn_case(lens, lens, hq, hkv, d, seed=5, extra=40)
    clean = [t.clone() for t in (q, k, v)]
    first = 70 + 150  # this token and all behind it hold `what`, the third sequence but its first
    for t in (k, v):
        t[first:270] = what
        t[271:] = what
    cu = i32(starts(lens))
    out = cuda.attn_prompt(q, k, v, cu)
    want, tol, _, _ = ref.attn(*clean, lens, lens, d ** -0.5, True)
    rows = list(range(first)) + [270]
    ref.close(out[rows], want[rows], tol[rows], f"{what}")
    status_clear(cuda)


def test_attn_values_that_are_seen_propagate(cuda):
    def edit(q, k, v):
        v[40, 0, 3] = math.nan
        v[300, 1, 5] = math.inf
    q, k, v = attn_case([400], [400], 4, 2, 64, seed=6)
    edit(q, k, v)
    out = cuda.attn_prompt(q, k, v, i32([0, 400]))
    for h in range(4):
        assert torch.equal(out[:, h, 3].isnan(), (torch.arange(400, device=DEV) >= 40) & (h < 2))
        assert torch.equal(~out[:, h, 5].isfinite(), (torch.arange(400, device=DEV) >= 300) & (h >= 2))
    out = cuda.attn_prompt(q[:1], k, v, i32([0, 1]), i32([0, 400]))
    assert out[0, :2, 3].isnan().all() and not out[0, 2:, 5].isfinite().any()
    assert torch.isfinite(out).sum() == out.numel() - 4


@pytest.mark.parametrize("d", [64, 128])
def test_attn_starts_that_are_not_ascending_stay_in_bounds(cuda, d):
    q, k, v = attn_case([200], [200], 4, 2, d)
    guard = torch.full((264, 4, d), 7.0, dtype=torch.float16, device=DEV)
    for cu in ([0, 1 << 30, 50, 200], [-7, 3, -100, 90], [190, 20, 400, 100], [5, 5, 5, 5]):
        cuda.attn_prompt(q, k, v, i32(cu), out=guard[:200])
        cuda.attn_prompt(q, k, v, i32([0, 1, 2, 3]), i32(cu), out=guard[:200])
        cuda.attn_prompt(q[:3], k, v, i32(cu), i32(cu[::-1]), out=guard[:3])
        assert (guard[200:] == 7).all()
    status_clear(cuda)


def test_attn_offsets_beyond_32_bits(cuda):
    """A long cache whose rows are far apart: the last sequence lies behind 2^32 bytes."""
    stride = 1 << 17
    n = 17000
    store = torch.empty((n, stride), dtype=torch.float16, device=DEV)
    assert (n - 1) * stride * 2 > 1 << 32
    g = gen(8)
    k = store[:, :256].view(n, 2, 128)
    v = store[:, 1024:1280].view(n, 2, 128)
    k.copy_(rand(g, (n, 2, 128)))
    v.copy_(rand(g, (n, 2, 128)))
    q_lens, k_lens = [1, 130], [n - 400, 400]
    q = rand(g, (131, 8, 128))
    out = cuda.attn_prompt(q, k, v, i32(starts(q_lens)), i32(starts(k_lens)))
    want, tol, _, _ = ref.attn(q, k, v, q_lens, k_lens, 128 ** -0.5, True)
    ref.close(out, want, tol, "far rows")


# ------------------------------------------------------------------------------- together, streams, graphs
def layer(hg, st):
    hq, hk, d = st["heads"]
    qkv = hg.lora(st["x"], st["w_in"], st["down_in"], st["up_in"], st["scale"], st["seg"], st["ids"])
    qkv = qkv.view(-1, hq + 2 * hk, d)
    q, k = hg.qk_norm_rope(qkv[:, :hq], qkv[:, hq:hq + hk], st["wq"], st["wk"], st["pos"], st["inv"])
    o = hg.attn_prompt(q, k, qkv[:, hq + hk:], st["seg"])
    y = hg.lora(o.view(-1, hq * d), st["w_out"], st["down_out"], st["up_out"], st["scale"],
                st["seg"], st["ids"])
    return qkv, q, k, o, y


def layer_state(lens, seed, heads=(8, 2, 64), K=512, r=16, A=3):
    hq, hk, d = heads
    g, T = gen(seed), sum(lens)
    n = (hq + 2 * hk) * d
    return dict(heads=heads, lens=lens, x=rand(g, (T, K)), w_in=rand(g, (K, n), K ** -0.5),
                down_in=rand(g, (A, K, r), K ** -0.5), up_in=rand(g, (A, r, n), r ** -0.5),
                w_out=rand(g, (hq * d, K), (hq * d) ** -0.5),
                down_out=rand(g, (A, hq * d, r), (hq * d) ** -0.5),
                up_out=rand(g, (A, r, K), r ** -0.5), scale=torch.rand(A, generator=g, device=DEV),
                seg=i32(starts(lens)), ids=i32([i % (A + 1) - 1 for i in range(len(lens))]),
                wq=rand(g, (d,)), wk=rand(g, (d,)),
                pos=torch.cat([torch.arange(n_, dtype=torch.int32, device=DEV) for n_ in lens]),
                inv=torch.tensor([10000.0 ** (-2 * i / d) for i in range(d // 2)],
                                 dtype=torch.float32, device=DEV))


def check_layer(st, got):
    """Each operator against its 64-bit form on what the one before it returned."""
    qkv, q, k, o, y = got
    hq, hk, d = st["heads"]
    T, A = st["x"].shape[0], st["scale"].shape[0]
    ids = ref.token_adapters(T, st["seg"].tolist(), st["ids"].tolist(), A)
    want, tol = ref.lora(st["x"], st["w_in"], st["down_in"], st["up_in"], st["scale"], ids)
    ref.close(qkv.reshape(T, -1), want, tol, "qkv")
    axis = torch.zeros(d // 2, device=DEV)
    for x, w, out in ((qkv[:, :hq], st["wq"], q), (qkv[:, hq:hq + hk], st["wk"], k)):
        want, tol = ref.qk_norm_rope(x, w, st["pos"], st["inv"], axis, 1e-6, False)
        ref.close(out, want, tol, "norm")
    want, tol, _, _ = ref.attn(q, k, qkv[:, hq + hk:], st["lens"], st["lens"], d ** -0.5, True)
    ref.close(o, want, tol, "attention")
    want, tol = ref.lora(o.reshape(T, -1), st["w_out"], st["down_out"], st["up_out"], st["scale"], ids)
    ref.close(y, want, tol, "y")


@pytest.mark.parametrize("lens", [[1], [1] * 20, [33, 1, 129, 70], [300, 211, 90]])
def test_layer(cuda, lens):
    st = layer_state(lens, seed=len(lens))
    check_layer(st, layer(cuda, st))
    status_clear(cuda)


def test_layer_on_another_stream(cuda):
    st = layer_state([120, 41], seed=9)
    want = layer(cuda, st)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = layer(cuda, st)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    y = cuda.lora(st["x"], st["w_in"], st["down_in"], st["up_in"], st["scale"], st["seg"], st["ids"],
                  stream=s)
    z = cuda.lora(st["x"], st["w_in"], st["down_in"], st["up_in"], st["scale"], st["seg"], st["ids"],
                  stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(y, z) and torch.equal(y, want[0].reshape(161, -1))


def test_two_streams_at_once(cuda):
    """Calls that overlap on the GPU each have their own workspace."""
    states = [layer_state([90, 200, 3], seed=s) for s in (1, 2)]
    want = [layer(cuda, st) for st in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(10):
        got = []
        for st, s in zip(states, streams):
            with torch.cuda.stream(s):
                got.append(layer(cuda, st))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("lens,other", [([64, 100, 37], [100, 100, 1]), ([1] * 12, [1] * 12)])
def test_captured_layer_follows_its_tensors(cuda, lens, other):
    """A captured layer replayed with other lengths, adapters and values in the same tensors."""
    st = layer_state(lens, seed=1)
    layer(cuda, st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(cuda, st)
    new = layer_state(other, seed=2)
    for name, t in new.items():
        if isinstance(t, torch.Tensor):
            st[name].copy_(t)
    st["ids"].copy_(i32([(i + 1) % 3 for i in range(len(lens))]))
    st["lens"] = other
    graph.replay()
    torch.cuda.synchronize()
    check_layer(st, got)


def test_two_graphs_do_not_share_a_workspace(cuda):
    states = [layer_state([40, 90], seed=s) for s in (3, 4)]
    want = [[t.clone() for t in layer(cuda, st)] for st in states]
    graphs, got = [], []
    for st in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(layer(cuda, st))
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(10):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


CAPTURED_FIRST = """
import torch, hopper_gemm_b200 as hg
T, d = {T}, 64
g = torch.Generator(device="cuda").manual_seed(0)
n = lambda *s: torch.randn(s, generator=g, device="cuda").half()
x, w, down, up, wn = n(T, 256), n(256, 384) / 16, n(2, 256, 16) / 16, n(2, 16, 384) / 4, n(d)
i32 = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)
scale, seg, ids, pos = torch.ones(2, device="cuda"), i32([0, 3, T]), i32([1, 0]), i32(list(range(T)))
inv = torch.ones(d // 2, device="cuda") / 100
def layer():
    qkv = hg.lora(x, w, down, up, scale, seg, ids).view(T, 6, d)
    q, k = hg.qk_norm_rope(qkv[:, :4], qkv[:, 4:5], wn, wn, pos, inv)
    return hg.attn_prompt(q, k, qkv[:, 5:], seg)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = layer()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(got, layer())
"""


@pytest.mark.parametrize("T", [20, 200])
def test_first_call_of_a_process_is_captured(T):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.format(T=T)], cwd=root, timeout=120,
                         capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]


def test_explicit_workspace_on_another_stream(cuda):
    """The caller's workspace, a view of its own buffer, with prompts in key ranges and single tokens."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for q, k in (([1] * 3, [900, 4000, 70]), ([40], [5000])):
        Q, K, V = (torch.randn((n, h, 64), generator=g, device="cuda").half()
                   for n, h in ((sum(q), 4), (sum(k), 2), (sum(k), 2)))
        cq, ck = i32(starts(q)), i32(starts(k))
        want = cuda.attn_prompt(Q, K, V, cq, ck)
        need = cuda.lib.hgemm_attn_prompt_workspace_bytes(sum(q), sum(k), len(q), 4, 2, 64)
        assert need > 0
        ws = torch.full((need + 512,), 0x7f, device="cuda", dtype=torch.uint8)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = cuda.attn_prompt(Q, K, V, cq, ck, workspace=ws[256:256 + need], stream=s)
        s.synchronize()
        assert torch.equal(got, want)
        assert bool((ws[:256] == 0x7f).all()) and bool((ws[256 + need:] == 0x7f).all())
        with pytest.raises(cuda.HgemmError):
            cuda.attn_prompt(Q, K, V, cq, ck, workspace=ws[256:255 + need])


def test_calls_from_several_threads(cuda):
    """Four threads, a stream each; one adapter for two requests; tensors that ask for gradients."""
    T = 70
    X, W, down, up, scale = lora_case(T, 256, 384, 16, 3)
    seg, ids = i32([0, 30, T]), i32([1, 1])
    want = cuda.lora(X, W, down, up, scale, seg, ids)
    with torch.inference_mode():
        assert torch.equal(cuda.lora(X, W, down, up, scale, seg, ids), want)
    assert torch.equal(cuda.lora(X.clone().requires_grad_(), W, down, up, scale, seg, ids), want)
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(50):
                    got = cuda.lora(X, W, down, up, scale, seg, ids)
                s.synchronize()
                assert torch.equal(got, want)
        except BaseException as e:  # noqa: B036  (handed to the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("over", [dict(scale=float("nan")), dict(scale=1e60), dict(scale="x"),
                                  dict(stream="s"), dict(lse=3), dict(workspace=torch.zeros(4))])
def test_attn_refuses_through_python(cuda, over):
    q = torch.zeros((5, 4, 64), dtype=torch.float16, device=DEV)
    with pytest.raises((cuda.HgemmError, TypeError, ValueError, AttributeError)):
        cuda.attn_prompt(q, q[:, :2], q[:, 2:], i32([0, 5]), **over)
    with pytest.raises(cuda.HgemmError):
        cuda.attn_prompt(q, q[:, :2], q[:, 2:], i32([0, 5]), out=q)
    with pytest.raises(cuda.HgemmError):
        cuda.attn_prompt(q, q[:, :2], q[:, 2:], i32([]))
    status_clear(cuda)


def test_repeated_runs_are_identical(cuda):
    for lens in ([1] * 40, [700, 5]):
        st = layer_state(lens, seed=11)
        first = layer(cuda, st)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(layer(cuda, st), first))


def test_public_functions_refuse_wrong_tensors(cuda):
    st = layer_state([5, 6], seed=1)
    args = [st[n] for n in ("x", "w_in", "down_in", "up_in", "scale", "seg", "ids")]
    for i, bad, err in ((0, args[0].bfloat16(), TypeError), (0, args[0][:, ::2], ValueError),
                        (1, args[1].t(), ValueError), (2, args[2][:, :, :8], ValueError),
                        (4, args[4].half(), TypeError), (5, args[5].long(), TypeError),
                        (5, args[5][1:], ValueError), (6, args[6].cpu(), ValueError),
                        (0, args[0].cpu(), ValueError)):
        with pytest.raises(err):
            cuda.lora(*[bad if j == i else a for j, a in enumerate(args)])
    with pytest.raises(cuda.HgemmError):  # K not a multiple of 8
        cuda.lora(args[0][:, :508].contiguous(), args[1][:508].contiguous(),
                  args[2][:, :508].contiguous(), *args[3:])
    q = torch.zeros((4, 2, 64), dtype=torch.float16, device=DEV)
    w, inv = q[0, 0], torch.zeros(32, device=DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        cuda.qk_norm_rope(q, q[:3], w, w, pos, inv)
    with pytest.raises(TypeError):
        cuda.qk_norm_rope(q, q, w, w, pos.long(), inv)
    with pytest.raises(ValueError):
        cuda.qk_norm_rope(q.transpose(0, 1), q.transpose(0, 1), w, w, pos[:2], inv)
    with pytest.raises(cuda.HgemmError):  # not on a 16-byte boundary
        flat = torch.zeros(4 * 2 * 64 + 1, dtype=torch.float16, device=DEV)
        cuda.qk_norm_rope(flat[1:].view(4, 2, 64), q, w, w, pos, inv)
    cu = i32([0, 4])
    with pytest.raises(ValueError):
        cuda.attn_prompt(q, q, q[:3], cu)
    with pytest.raises(ValueError):
        cuda.attn_prompt(q, q, q, cu, lse=torch.zeros((4, 3), device=DEV))
    with pytest.raises(TypeError):
        cuda.attn_prompt(q, q, q, cu.long())
    with pytest.raises(cuda.HgemmError):  # three query heads over two
        cuda.attn_prompt(torch.zeros((4, 3, 64), dtype=torch.float16, device=DEV), q, q, cu)
