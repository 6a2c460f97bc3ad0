"""Eviction from caches longer than a cluster's shared memory holds keys for (409,600 slots): keys made anew at each pass.
Against the definition; exact."""

import numpy as np
import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu


def kept(w, pos, seen, keep, sinks, recent):
    """The slots that stay, and what each slot below the new length holds."""
    n, m = len(w), min(len(w), keep)
    nan = np.isnan(w)
    key = np.where(nan, np.inf, w.astype(np.float64))
    safe = (pos < sinks) | (pos >= seen - recent)
    stays = np.zeros(n, dtype=bool)
    stays[np.lexsort((np.arange(n), -key, ~nan, ~safe))[:m]] = True
    take = np.arange(m)
    take[~stays[:m]] = m + np.flatnonzero(stays[m:])
    return take


@pytest.mark.parametrize("weights", ["spread", "equal", "odd"])
@pytest.mark.parametrize("places", ["each once", "repeated"])
@pytest.mark.parametrize("lengths, keep, sinks, recent, page", [
    ([420000, 409601], 100003, 4, 5000, 64), ([430000, 0, 17], 3, 1, 2, 16), ([409664, 200000], 409600, 0, 100, 64)])
def test_evict_past_shared_memory(cuda, lengths, keep, sinks, recent, page, places, weights):
    """Positions that repeat make more places kept than slots stay (all slots' position a sink's): only those are ranked."""
    g = np.random.default_rng(keep)
    n, per = len(lengths), -(-max(lengths) // page)
    slots = per * page
    assert slots > 409600
    k, v = (torch.randn((n * per, page, 1, 8), device="cuda").to(torch.bfloat16) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    table = torch.randperm(n * per, device="cuda").to(torch.int32).reshape(n, per)
    w = {"spread": np.round(g.random((n, slots)) * 1e5).astype(np.float32) / 1e5,
         "equal": np.full((n, slots), 0.5, dtype=np.float32),
         "odd": g.choice(np.array([0.0, -0.0, -1.0, 1e-45, 1.0, 3e38, np.inf, -np.inf, np.nan], dtype=np.float32),
                         size=(n, slots))}[weights]
    if places == "each once":
        pos = np.stack([g.permutation(slots) for _ in lengths]).astype(np.int32)
        seen = np.full(n, slots + 9, dtype=np.int32)
    else:  # a third of the slots at position 0: with sinks or recent, more than stay
        pos = np.where(g.random((n, slots)) < 0.34, 0, 5).astype(np.int32)
        seen = np.full(n, 1000000 if sinks else recent, dtype=np.int32)
    cw, cp = torch.from_numpy(w.copy()).cuda(), torch.from_numpy(pos.copy()).cuda()
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cache = context.KVPages(k, v, table, length, weight=cw, position=cp)
    cache.evict(torch.from_numpy(seen).cuda(), keep, sinks=sinks, recent=recent)
    for b, m in enumerate(lengths):
        take = kept(w[b, :m], pos[b, :m], seen[b], keep, sinks, recent)
        left = len(take)
        assert int(length[b]) == left
        assert np.array_equal(cw[b, :left].cpu().numpy().view(np.int32), w[b, take].view(np.int32))
        assert np.array_equal(cp[b, :left].cpu().numpy(), pos[b, take])
        at, src = (table[b].long()[x // page] * page + x % page
                   for x in (torch.arange(left, device="cuda"), torch.from_numpy(take).cuda()))
        for pool, was in ((k, k0), (v, v0)):
            assert torch.equal(pool.view(-1, 8)[at], was.view(-1, 8)[src])
    _lib.check_device_errors()


@pytest.mark.parametrize("slots", [9216, 10240, 11264, 12288, 81920, 98304, 409600])
def test_evict_at_the_limits_of_shared_memory(cuda, slots):
    """Around the slots a block gets shared memory for without asking, and up to the most that it holds keys of."""
    g = np.random.default_rng(slots)
    keep = slots // 3
    k, v = (torch.randn((slots // 16, 16, 1, 8), device="cuda").to(torch.bfloat16) for _ in range(2))
    k0 = k.clone()
    table = torch.arange(slots // 16, dtype=torch.int32, device="cuda")[None]
    w, pos = g.random((1, slots)).astype(np.float32), np.arange(slots, dtype=np.int32)[None]
    cw, cp = torch.from_numpy(w.copy()).cuda(), torch.from_numpy(pos.copy()).cuda()
    length = torch.tensor([slots], dtype=torch.int32, device="cuda")
    context.KVPages(k, v, table, length, weight=cw, position=cp).evict(length.clone(), keep, sinks=4, recent=keep // 2)
    take = kept(w[0], pos[0], slots, keep, 4, keep // 2)
    assert int(length[0]) == keep and np.array_equal(cp[0, :keep].cpu().numpy(), take)
    assert torch.equal(k.view(-1, 8)[:keep], k0.view(-1, 8)[torch.from_numpy(take).cuda()])
    _lib.check_device_errors()
