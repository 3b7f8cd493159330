"""GPU: the attention layer's operators at the values, masks and sizes where a rounding, a mask or a
repair shows. References and tolerances are plain 64-bit forms derived beside each test."""
import math

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
