"""The context operators over tensors that lie otherwise: heads before tokens, tokens before sequences, rows of a wider
buffer, axes of one entry whose strides are anything. The same bits as over contiguous copies."""

import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def lay(x, how):
    """x (batch, tokens, heads, dim) with the same values, lying in memory as `how` says."""
    if how == "heads first":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "tokens first":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "heads outermost":
        return x.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    if how == "padded":
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 8), float("nan"), dtype=x.dtype, device=x.device)
        wide[..., : x.shape[-1]] = x
        return wide[..., : x.shape[-1]]
    if how == "every other token":
        wide = torch.full((x.shape[0], 2 * x.shape[1], *x.shape[2:]), float("nan"), dtype=x.dtype, device=x.device)
        wide[:, ::2] = x
        return wide[:, ::2]
    return x.transpose(-1, -2).contiguous().transpose(-1, -2)  # dims not adjacent: copied by the call


@pytest.mark.parametrize("how", ["heads first", "tokens first", "heads outermost", "padded", "every other token", "dims"])
@pytest.mark.parametrize("t, dtype", [(5, BF), (150, BF), (1100, BF), (60, HF)])
def test_linear_attention_layouts(cuda, how, t, dtype):
    g = torch.Generator(device="cuda").manual_seed(t)
    q, k = (torch.randn((2, t, 2, 64), generator=g, device="cuda").to(dtype) for _ in range(2))
    v = torch.randn((2, t, 4, 64), generator=g, device="cuda").to(dtype)
    d = -0.1 * torch.rand((2, t, 4), generator=g, device="cuda")
    want = context.linear_attention(q, k, v, d)
    got = context.linear_attention(lay(q, how), lay(k, how), lay(v, how), d.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a, b = want[1].clone(), want[1].clone()
    x = context.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], a)
    y = context.linear_attention_step(lay(q, how)[:, 0], lay(k, how)[:, 0], lay(v, how)[:, 0], d[:, 0], b)
    assert torch.equal(x, y) and torch.equal(a, b)
    _lib.check_device_errors()


def odd(x, *axes):
    """x with an odd stride at axes of one entry."""
    st = list(x.stride())
    for a in axes:
        assert x.shape[a] == 1
        st[a] = 12345
    return x.as_strided(x.shape, st)


@pytest.mark.parametrize("t", [1, 5, 100])
def test_an_axis_of_one_entry_has_any_stride(cuda, t):
    """As views of a row whose width is no multiple of 8 have."""
    q, k, v = (torch.randn((1, t, 1, 64), device="cuda").to(BF) for _ in range(3))
    d = -0.1 * torch.rand((1, t, 1), device="cuda")
    axes = (0, 2) if t > 1 else (0, 1, 2)
    want = context.linear_attention(q, k, v, d)
    got = context.linear_attention(odd(q, *axes), odd(k, *axes), odd(v, *axes), d)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    S, T = want[1].clone(), want[1].clone()
    a = context.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], S)
    b = context.linear_attention_step(*(odd(x[:, 0], 0, 1) for x in (q, k, v)), d[:, 0], T)
    assert torch.equal(a, b) and torch.equal(S, T)
    cache = torch.randn((2, 1, 64), device="cuda").to(BF)[:, None]  # pages of one slot, one head
    table, n = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda")
    one = torch.randn((1, 1, 64), device="cuda").to(BF)
    want = context.decode_attention(one, cache, cache, table, n)
    assert torch.equal(context.decode_attention(odd(one, 0, 1), odd(cache, 1, 2), odd(cache, 1, 2), table, n), want)
    page = torch.randn((1, 16, 1, 64), device="cuda").to(BF)
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    want = context.decode_attention(one, page, page, table, n)
    assert torch.equal(context.decode_attention(odd(one, 0, 1), odd(page, 0, 2), odd(page, 0, 2), table, n), want)
    _lib.check_device_errors()
