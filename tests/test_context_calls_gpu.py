"""What the context operators' calls put on the stream, and how they stand calls from several threads and odd arguments."""

import ctypes

import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def cache(lengths=(300, 77), hkv=2, d=64, page=16, tracked=True):
    n, per = len(lengths), -(-max(lengths) // page)
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((n * per, page, hkv, d), generator=g, device="cuda").to(BF) for _ in range(2))
    table = torch.arange(n * per, dtype=torch.int32, device="cuda").reshape(n, per)
    w = torch.rand((n, per * page), generator=g, device="cuda") if tracked else None
    pos = torch.arange(per * page, dtype=torch.int32, device="cuda").repeat(n, 1)
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return context.KVPages(k, v, table, lengths, weight=w, position=pos)


def nodes(call) -> int:
    """The nodes of the graph that a call is captured as."""
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    n = ctypes.c_size_t()
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(g.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


def test_a_captured_call_is_its_two_kernels(cuda):
    """No fill of a workspace among them."""
    c = cache()
    q, out = torch.randn((2, 8, 64), device="cuda").to(BF), torch.empty((2, 8, 64), dtype=BF, device="cuda")
    assert nodes(lambda: c.attend(q, out=out)) == 2
    seen = c.lengths.clone()
    aside = torch.empty_like(c.weight), torch.empty_like(c.position), torch.empty_like(c.lengths)
    assert nodes(lambda: c.evict(seen, 100, sinks=4, recent=10, out=aside)) == 2


def test_a_workspace_may_hold_anything(cuda):
    """NaN and largest integers in the memory that the workspaces get."""
    q = torch.randn((2, 8, 64), device="cuda").to(BF)
    got = []
    for fill in (0, 255, 127):
        c = cache()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        junk = [torch.full((n << 10,), fill, dtype=torch.uint8, device="cuda") for n in (1, 16, 256, 4096, 65536)]
        del junk
        out = c.attend(q)
        c.evict(c.lengths.clone(), 100, sinks=4, recent=10)
        got.append((out, c.weight[:, :77].clone(), c.position[:, :77].clone(), c.lengths.clone(), c.k[:5].clone()))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    _lib.check_device_errors()


def test_a_batch_past_the_limit_is_named(cuda):
    k = torch.zeros((1, 16, 1, 64), dtype=BF, device="cuda")
    table = torch.zeros((65536, 1), dtype=torch.int32, device="cuda")
    cache = context.KVPages(k, k.clone(), table, torch.ones(65536, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="65535"):
        cache.attend(torch.zeros((65536, 1, 64), dtype=BF, device="cuda"))
