"""Linear attention at the decays where its forms could part: growth, resets, very strong decays, NaN. Each against the
recurrence in 64 bits.

Tolerances (u: the type's unit roundoff, e = 2^-23; OA, A: outputs and state of the recurrence over absolute values):
  outputs  u |o| for their own rounding; what enters the products does so to u^2 (two terms of the type), the exponents
           and sums to (D + 200 + G) e, G the largest sum of |decay| over two chunks (128 tokens)
  state    (D + 200 + G) e A + 3 u^3 A
Both plus what float32 does not hold: 1e-30 (products of exponentials below 2^-126 are zero)."""

import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}
E = 2.0 ** -23
INF, NAN = float("inf"), float("nan")


def recurrence(q, k, v, g, S, scale):
    n, t, hk, dk = q.shape
    hv, dv = v.shape[2:]
    q, k = (x.double().repeat_interleave(hv // hk, 2) for x in (q, k))
    v, g = v.double(), g.double()
    S = torch.zeros((n, hv, dk, dv), dtype=torch.float64, device=q.device) if S is None else S.double()
    A, O, OA = S.abs(), torch.zeros_like(v), torch.zeros_like(v)
    for i in range(t):
        a = torch.exp(g[:, i])[..., None, None]
        kv = k[:, i, :, :, None] * v[:, i, :, None, :]
        S, A = a * S + kv, a * A + kv.abs()
        O[:, i] = (q[:, i, :, :, None] * S).sum(2) * scale
        OA[:, i] = (q[:, i, :, :, None].abs() * A).sum(2) * abs(scale)
    return O, S, OA, A


def check(q, k, v, g, S, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    kept = None if S is None else S.clone()
    out, state = context.linear_attention(q, k, v, g, state=S, scale=scale)
    assert S is None or torch.equal(S.view(torch.int32), kept.view(torch.int32))
    O, F, OA, A = recurrence(q, k, v, g, S, scale)
    u, d = U[q.dtype], q.shape[-1]
    G = 128 * g.nan_to_num(0.0, posinf=0.0, neginf=0.0).clamp(min=-104.0).abs().amax().item()
    e = (d + 200 + G) * E
    for got, want, tol in ((out, O, u * O.abs() + (u * u + e) * OA + 1e-30), (state, F, (e + 3 * u ** 3) * A + 1e-30)):
        assert torch.equal(got.isnan(), want.isnan())
        err = torch.where(want.isnan(), 0.0, (got.double() - want).abs())
        ratio = torch.where(want.isnan(), 0.0, err / tol)
        assert (ratio <= 1).all(), ratio.max().item()
    _lib.check_device_errors()
    return out, state


def make(n, t, hk, hv, dk, dv, dtype, seed=0, stated=True):
    g = torch.Generator(device="cuda").manual_seed(seed + t)
    q, k = (torch.randn((n, t, hk, dk), generator=g, device="cuda").to(dtype) for _ in range(2))
    v = torch.randn((n, t, hv, dv), generator=g, device="cuda").to(dtype)
    r = torch.rand((n, t, hv), generator=g, device="cuda")
    S = torch.randn((n, hv, dk, dv), generator=g, device="cuda") if stated else None
    return q, k, v, r, S


SHAPES = [(1, 40, 1, 2, 64, 64, BF), (1, 200, 1, 2, 128, 128, BF), (2, 1100, 1, 1, 128, 64, BF), (1, 150, 2, 2, 64, 48, HF)]


@pytest.mark.parametrize("rate", [0.01, 0.05])
@pytest.mark.parametrize("kind", ["growth", "mixed"])
@pytest.mark.parametrize("stated", [False, True])
@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", SHAPES)
def test_growth(cuda, n, t, hk, hv, dk, dv, dtype, stated, kind, rate):
    """Decays above 0, alone and among others, over one chunk, several, and several segments. At 0.05 a token a state
    grows e^55-fold over the longest prompt."""
    if dtype == HF and rate == 0.05:
        rate = 0.02  # outputs within float16's range
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype, stated=stated)
    check(q, k, v, rate * torch.ones_like(r) if kind == "growth" else 20 * rate * (r - 0.45), S)


def test_growth_of_tenths_a_token(cuda):
    """A chunk's sum of 6.4 and a prompt's of 30: e^30."""
    q, k, v, r, S = make(1, 300, 1, 1, 128, 128, BF)
    check(q, k, v, torch.full_like(r, 0.1), S)
