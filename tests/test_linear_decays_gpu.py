"""Linear attention at the decays where its forms could part: growth, resets, very strong decays, NaN. Each against the
recurrence in 64 bits.

Tolerances (u: the type's unit roundoff, e = 2^-23; OA, A: outputs and state of the recurrence over absolute values):
  outputs  u |o| for their own rounding; what enters the products does so to u^2 (two terms of the type), the exponents
           and sums to (D + 200 + G) e, G the largest sum of |decay| over two chunks (128 tokens)
  state    (D + 200 + G) e A + 3 u^3 A
Both plus what float32 does not hold: 1e-30 (products of exponentials below 2^-126 are zero), and outputs half of their
type's least value (2^-25 in float16)."""

import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}
LEAST = {BF: 2.0 ** -134, HF: 2.0 ** -25}
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
    past = O.abs() > torch.finfo(q.dtype).max  # outputs past the type's range are its infinities
    assert torch.equal(out.isinf(), past) and torch.equal(out[past] > 0, O[past] > 0)
    out_tol = u * O.abs() + (u * u + e) * OA + 1e-30 + LEAST[q.dtype]
    for got, want, tol, skip in ((out, O, out_tol, past), (state, F, (e + 3 * u ** 3) * A + 1e-30, False)):
        assert torch.equal(got.isnan(), want.isnan())
        ratio = torch.where(want.isnan() | skip, 0.0, (got.double() - want).abs() / tol)
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


SHAPES = [(1, 40, 1, 2, 64, 64, BF), (1, 200, 1, 2, 128, 128, BF), (2, 1100, 1, 1, 128, 64, BF),
          (1, 150, 2, 2, 64, 48, HF)]


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


LONG = [(1, 64, 1, 2, 64, 64, BF), *SHAPES[1:]]
LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("value", [-INF, LOWEST, -105.0])
@pytest.mark.parametrize("where", ["chunk's ends", "often", "every token", "the first", "the last"])
@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", LONG)
def test_resets_forget(cuda, n, t, hk, hv, dk, dv, dtype, where, value):
    """A decay of -inf, or one whose exponential is zero in float32: nothing of an earlier token or of a state twelve
    orders larger is left."""
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype)
    at = torch.arange(t, device="cuda")
    hit = {"chunk's ends": (at % 64 == 63) | (at % 128 == 0), "often": r > 0.95, "every token": r >= 0,
           "the first": at == 0, "the last": at == t - 1}[where]
    hit = hit if hit.dim() == 3 else hit[:, None].expand_as(r)
    check(q, k, v, torch.where(hit, value, -0.02 * r), S * 1e12)


@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", LONG)
@pytest.mark.parametrize("last", [0, 5, 63, 64, 149])
def test_nothing_is_left_where_nothing_is_added(cuda, n, t, hk, hv, dk, dv, dtype, last):
    """Behind the last reset the keys are zero: so are the outputs and the state, exactly."""
    last = min(last, t - 1)
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype)
    k[:, last:] = 0
    g = -0.1 * r
    g[:, last] = -INF
    out, state = check(q, k, v, g, S)
    assert (out[:, last:] == 0).all() and (state == 0).all()


@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", LONG)
def test_strong_decays_are_their_exponentials(cuda, n, t, hk, hv, dk, dv, dtype):
    """e^-31 to e^-80, with nothing added behind them that would cover what they leave."""
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype)
    k[:, 20:] = 0
    g = -0.001 * r
    g[:, 30] = -31.0 - 49.0 * r[:, 30]
    check(q, k, v, g, S)
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype, seed=1)
    check(q, k, v, torch.where(r > 0.9, -100.0 * r, -0.01 * r), S)


@pytest.mark.parametrize("at", [0, 1, 40, 63, 64, 100, 149])
@pytest.mark.parametrize("resets", ["none", "before", "after", "around"])
@pytest.mark.parametrize("stated", [False, True])
@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", LONG)
def test_a_broken_gate_shows(cuda, n, t, hk, hv, dk, dv, dtype, at, resets, stated):
    """A NaN decay of one head: NaN in every output of the head from its token on and in the state, though resets follow
    (0 times NaN); the tokens before it and the other heads are as they were."""
    at = min(at, t - 1)
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype, stated=stated)
    g = -0.05 * r
    if resets in ("before", "around"):
        g[:, max(0, at - 3)] = -INF
    if resets in ("after", "around"):
        g[:, min(t - 1, at + 2)] = -INF
    g[0, at, hv - 1] = NAN
    out, state = check(q, k, v, g, S)
    assert out[0, at:, hv - 1].isnan().all() and state[0, hv - 1].isnan().all()
    assert not out[0, :at].isnan().any() and not out[0, :, : hv - 1].isnan().any()


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("at", [0, 1, 40, 63, 64, 100, 149])
@pytest.mark.parametrize("resets", [False, True])
@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", LONG)
def test_a_value_does_not_reach_earlier_tokens(cuda, n, t, hk, hv, dk, dv, dtype, resets, at, value):
    """A value that is not finite, in a masked place for the tokens before it: their outputs are what they are without it,
    and so are the other value dimensions and heads; from its token on its dimension is not finite."""
    at = min(at, t - 1)
    q, k, v, r, S = make(n, t, hk, hv, dk, dv, dtype)
    g = -0.05 * r
    if resets:
        g[:, max(0, at - 20)] = -INF
    O, F, OA, A = recurrence(q, k, v, g, S, dk ** -0.5)
    u, e = U[dtype], (dk + 200 + 128 * 0.05) * E
    v[0, at, hv - 1, 5] = value
    v[0, min(t - 1, at + 3), hv - 1, dv - 1] = value
    out, state = context.linear_attention(q, k, v, g, state=S)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, at:, hv - 1, 5] = True
    bad[0, min(t - 1, at + 3) :, hv - 1, dv - 1] = True
    assert not out[bad].isfinite().any() and not state[0, hv - 1, :, 5].isfinite().any()
    ratio = torch.where(bad, 0.0, (out.double() - O).abs() / (u * O.abs() + (u * u + e) * OA + 1e-30 + LEAST[dtype]))
    assert (ratio <= 1).all(), ratio.max().item()
    _lib.check_device_errors()


@pytest.mark.parametrize("t", [100, 1100])
def test_in_place_with_a_value_that_is_not_finite(cuda, t):
    """The library's call with one array for the state before and after: the same bits as with two."""
    q, k, v, r, S = make(2, t, 2, 2, 128, 128, BF)
    g = -0.05 * r
    v[0, 70, 1, 9] = INF
    v[1, 20, 0, 100] = NAN
    out, state = context.linear_attention(q, k, v, g, state=S)
    got, place, lib = torch.empty_like(out), S.clone(), _lib.lib()
    strides = [x for y in (q, k, v, g) for x in y.stride()[:3]]
    call = context._LINEAR.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), place.data_ptr(), place.data_ptr(),
                                0, got.data_ptr(), *strides, 2, t, 2, 2, 128, 128, 2, 128 ** -0.5)
    size = lib.sc_linear_attention_workspace(call)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    assert lib.sc_linear_attention(call, ws.data_ptr(), size, _lib.error_word().data_ptr(), _lib.stream()) == 0
    assert torch.equal(got.view(torch.int16), out.view(torch.int16))
    assert torch.equal(place.isnan(), state.isnan()) and torch.equal(place[state.isfinite()], state[state.isfinite()])
    assert got[0, :70, 1, 9].isfinite().all() and got[1, :20, 0, 100].isfinite().all()
    _lib.check_device_errors()


def test_every_value_is_not_finite(cuda):
    """The mending over all dimensions and heads of a long prompt, in several segments and in one."""
    for n, hv in ((1, 2), (8, 16)):
        q, k, v, r, S = make(n, 4096, 2, hv, 128, 128, BF)
        v[:, 4000:] = NAN
        out, state = context.linear_attention(q, k, v, -0.05 * r, state=S)
        assert out[:, :4000].isfinite().all() and out[:, 4000:].isnan().all() and state.isnan().all()
        want = context.linear_attention(*(x[:, :4000] for x in (q, k, v, -0.05 * r)), state=S)[0]
        assert torch.allclose(out[:, :4000].float(), want.float(), rtol=2.0 ** -6, atol=1e-2)
        _lib.check_device_errors()
