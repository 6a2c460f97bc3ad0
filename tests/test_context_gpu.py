"""The context operators against their definitions in 64 bits.

Tolerances, from the arithmetic (u: the activation type's unit roundoff, 2^-8 bfloat16, 2^-11 float16; e = 2^-23,
which covers a float32 rounding and a truncating accumulation):
  scores      a sum of D products: |ds| <= (D + 4) e S, S = scale sum |q_i k_i|; so a probability is off by at most
              2 ds (itself and the sum) plus the sums' n e
  attention   u |o| for the output's rounding, and (2 ds + (n + 64) e + u^2) sum p |v|: the value product takes a
              probability as two terms of the type, u^2 apart from it at most
  weights     (2 ds + (n + 64) e) sum p for what was added, e |w| for the addition
  linear      u |o| + (rounded operands of the products) 3 u A + (D + 200 + G) e A, A the same recurrence over absolute
              values and G the largest decay within 128 tokens, whose sums round at e G
  state       (D + 200 + G) e A + 3 u^3 A: three terms of the type
"""

import math

import numpy as np
import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -23
BF, HF = torch.bfloat16, torch.float16


def pool(lengths, hkv, d, page, dtype, seed=0, layout="plain", room=0, spread=1.0):
    """A cache whose unused slots and pages hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = len(lengths)
    per = max(1, -(-(max(lengths) + room) // page))
    pages = n * per + 3
    if layout == "plain":
        k, v = (torch.full((pages, page, hkv, d), float("nan"), device="cuda", dtype=dtype) for _ in range(2))
    elif layout == "joined":  # keys and values of a page side by side
        kv = torch.full((pages, 2, page, hkv, d), float("nan"), device="cuda", dtype=dtype)
        k, v = kv[:, 0], kv[:, 1]
    else:  # heads before tokens, rows padded
        k, v = (torch.full((pages, hkv, page, d + 8), float("nan"), device="cuda", dtype=dtype)[..., :d].transpose(1, 2)
                for _ in range(2))
    table = torch.randperm(pages, generator=g, device="cuda")[: n * per].to(torch.int32).reshape(n, per)
    K, V = [], []
    for b, m in enumerate(lengths):
        slots = torch.arange(m, device="cuda")
        at = table[b].long()[slots // page], slots % page
        K.append((torch.randn((m, hkv, d), generator=g, device="cuda") * spread).to(dtype))
        V.append(torch.randn((m, hkv, d), generator=g, device="cuda").to(dtype))
        k[at], v[at] = K[-1], V[-1]
    return k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), K, V


def check_attention(q, K, V, out, scale, added=None, before=None):
    n, hq, d = q.shape
    u = U[q.dtype]
    for b in range(n):
        m, hk = K[b].shape[:2]
        if m == 0:
            assert (out[b] == 0).all()
            if added is not None:
                assert torch.equal(added[b], before[b])
            continue
        qd = q[b].double().reshape(hk, hq // hk, d)
        k, v = K[b].double(), V[b].double()
        p = torch.softmax(torch.einsum("hgd,thd->hgt", qd, k) * scale, -1)
        s = torch.einsum("hgd,thd->hgt", qd.abs(), k.abs()).amax(-1, keepdim=True) * abs(scale)
        ds = (d + 4) * E * s
        o = torch.einsum("hgt,thd->hgd", p, v)
        tol = u * o.abs() + (2 * ds + (m + 64) * E + u * u) * torch.einsum("hgt,thd->hgd", p, v.abs()) + 1e-7
        err = (out[b].double().reshape(hk, hq // hk, d) - o).abs()
        assert (err <= tol).all(), (b, m, (err / tol).max().item())
        if added is not None:
            w = p.sum((0, 1))
            tol = ((2 * ds + (m + 64) * E) * p).sum((0, 1)) + E * (before[b, :m].double() + w)
            err = (added[b, :m].double() - before[b, :m].double() - w).abs()
            assert (err <= tol).all(), (b, m, (err / tol).max().item())
            assert torch.equal(added[b, m:], before[b, m:])


ATTEND = [  # lengths, q_heads, kv_heads, head_dim, page, type
    ([8], 16, 2, 256, 16, BF), ([0, 1, 2, 15, 16, 17], 8, 1, 128, 16, BF), ([300, 0, 77, 1023], 12, 4, 64, 16, HF),
    ([1000], 3, 3, 80, 8, BF), ([129, 513], 20, 4, 96, 32, HF), ([64, 65, 63], 16, 1, 256, 64, HF),
    ([5003, 1, 2500], 32, 8, 128, 16, HF), ([20001], 16, 2, 256, 16, BF), ([31, 4097], 40, 1, 160, 1, BF),
    ([7, 250] * 40, 5, 1, 8, 4, BF), ([33000, 2], 14, 7, 64, 256, BF), ([127, 128, 129, 255, 257], 1, 1, 248, 16, HF)]


@pytest.mark.parametrize("tracked", [False, True])
@pytest.mark.parametrize("lengths, hq, hkv, d, page, dtype", ATTEND)
def test_decode_attention(cuda, lengths, hq, hkv, d, page, dtype, tracked):
    k, v, table, n, K, V = pool(lengths, hkv, d, page, dtype, seed=len(lengths) + d)
    q = torch.randn((len(lengths), hq, d), device="cuda").to(dtype)
    before = torch.rand((len(lengths), table.shape[1] * page), device="cuda") if tracked else None
    w = before.clone() if tracked else None
    cache = context.KVPages(k, v, table, n, weight=w)
    out = cache.attend(q)
    check_attention(q, K, V, out, d ** -0.5, w, before)
    if tracked:
        w.copy_(before)
    again = cache.attend(q)  # the same bits on every run
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    _lib.check_device_errors()


@pytest.mark.parametrize("layout", ["joined", "heads"])
def test_decode_attention_takes_strided_caches_and_queries(cuda, layout):
    lengths, hq, hkv, d = [100, 39], 6, 3, 64
    k, v, table, n, K, V = pool(lengths, hkv, d, 16, BF, layout=layout)
    qkv = torch.randn((2, hq + 2 * hkv, d), device="cuda").to(BF)
    q = qkv[:, :hq]
    check_attention(q, K, V, context.decode_attention(q, k, v, table, n), d ** -0.5)
    wide = torch.full((2, 7), 1 << 20, dtype=torch.int32, device="cuda")  # rows of a wider table
    wide[:, : table.shape[1]] = table
    out = torch.empty((2, hq, d), dtype=BF, device="cuda")
    got = context.decode_attention(q, k, v, wide[:, : table.shape[1]], n, scale=0.5, out=out)
    assert got is out
    check_attention(q, K, V, out, 0.5)


def test_decode_attention_of_sharp_and_flat_scores(cuda):
    """Scores thousands apart give one slot; equal scores an average; a slot at minus infinity nothing."""
    d = 64
    k, v, table, n, K, V = pool([600, 600], 1, d, 16, BF, spread=400.0)
    q = torch.randn((2, 4, d), device="cuda").to(BF) * 30
    check_attention(q, K, V, context.decode_attention(q, k, v, table, n), d ** -0.5)
    q.zero_()
    check_attention(q, K, V, context.decode_attention(q, k, v, table, n), d ** -0.5)
    q[:] = 0
    q[..., 0] = 1.0
    flat = k.view(-1, 1, d)
    rows = (table[0].long()[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)
    flat[rows[::2][:300], :, 0] = float("-inf")
    flat[rows[1::2][:300], :, 0] = 0.0
    out = context.decode_attention(q, k, v, table, n)
    want = V[0][1::2].double().mean(0)
    assert ((out[0].double() - want).abs() <= U[BF] * want.abs() + (700 * E + U[BF] ** 2) * V[0][1::2].double().abs().mean(0)).all()


def test_decode_attention_of_rows_that_share_pages(cuda):
    """A prompt's tokens as sequences over one row of the table: causal attention."""
    t, hq, hkv, d = 40, 4, 2, 64
    k, v, table, n, K, V = pool([t], hkv, d, 16, BF)
    q = torch.randn((t, hq, d), device="cuda").to(BF)
    lengths = torch.arange(1, t + 1, dtype=torch.int32, device="cuda")
    out = context.decode_attention(q, k, v, table.expand(t, -1), lengths)
    check_attention(q, [K[0][: i + 1] for i in range(t)], [V[0][: i + 1] for i in range(t)], out, d ** -0.5)


def test_decode_attention_past_32_bits_of_offset(cuda):
    """Pages on both sides of 2^31 values of a pool."""
    page, hkv, d = 16, 2, 128
    far = (1 << 31) // (page * hkv * d) + 5
    pools = [torch.empty((far + 2, page, hkv, d), dtype=BF, device="cuda") for _ in range(2)]
    table = torch.tensor([[far, 0, far + 1, far - 20]], dtype=torch.int32, device="cuda")
    rows = [torch.randn((4, page, hkv, d), device="cuda").to(BF) for _ in range(2)]
    for p, r in zip(pools, rows):
        p[table[0].long()] = r
    lengths = torch.tensor([60], dtype=torch.int32, device="cuda")
    q = torch.randn((1, 4, d), device="cuda").to(BF)
    w, pos = torch.rand((1, 64), device="cuda"), torch.arange(64, dtype=torch.int32, device="cuda")[None].clone()
    before = w.clone()
    cache = context.KVPages(*pools, table, lengths, weight=w, position=pos)
    K, V = ([r.reshape(-1, hkv, d)[:60]] for r in rows)
    check_attention(q, K, V, cache.attend(q), d ** -0.5, w, before)
    w.copy_(torch.arange(64, device="cuda", dtype=torch.float32))  # the last ones stay
    cache.evict(lengths.clone(), 20, sinks=0)
    for p, r in zip(pools, rows):
        got = p[table[0].long()].reshape(-1, hkv, d)[:20]
        assert torch.equal(got, r.reshape(-1, hkv, d)[40:60])


def test_decode_attention_from_a_graph_and_on_another_stream(cuda):
    d = 128
    k, v, table, n, K, V = pool([500, 90], 2, d, 16, BF, room=40)
    q = torch.randn((2, 8, d), device="cuda").to(BF)
    cache = context.KVPages(k, v, table, n)
    out = torch.empty_like(q)
    cache.attend(q, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(q, out=out)
    for m in ([400, 1], [37, 0], [500, 90]):  # lengths are read at each replay
        n.copy_(torch.tensor(m, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check_attention(q, [a[:b] for a, b in zip(K, m)], [a[:b] for a, b in zip(V, m)], out, d ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = cache.attend(q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, again)


def test_bad_pages_and_lengths_are_recorded(cuda):
    k, v, table, n, K, V = pool([40, 40], 1, 64, 16, BF)
    q = torch.randn((2, 2, 64), device="cuda").to(BF)
    bad = table.clone()
    bad[0, 1] = k.shape[0]
    bad[1, 2] = -1
    w, pos = torch.rand((2, 48), device="cuda"), torch.zeros((2, 48), dtype=torch.int32, device="cuda")
    out = context.decode_attention(q, k, v, bad, n, weight=w)
    keep = [torch.cat([torch.arange(16), torch.arange(32, 40)]), torch.arange(32)]
    check_attention(q, [a[i.cuda()] for a, i in zip(K, keep)], [a[i.cuda()] for a, i in zip(V, keep)], out, 0.125)
    with pytest.raises(_lib.StrataError, match="SC_ERR_PAGE"):
        _lib.check_device_errors()
    n[0], n[1] = -3, 49
    table[1, 2] = table[1, 1]
    out = context.decode_attention(q, k, v, table, n)
    assert (out[0] == 0).all()
    with pytest.raises(_lib.StrataError, match="SC_ERR_PAGE"):
        _lib.check_device_errors()
    context.KVPages(k, v, bad, torch.tensor([40, 40], dtype=torch.int32, device="cuda"), w, pos).evict(n.clone(), 20)
    with pytest.raises(_lib.StrataError, match="SC_ERR_PAGE"):
        _lib.check_device_errors()
    _lib.check_device_errors()


# ---- eviction


def kept_slots(w, pos, seen, keep, sinks, recent):
    """The slots that stay, by their definition, and slot i < keep's source."""
    n = len(w)
    m = min(n, keep)
    w = np.where(np.isnan(w), np.inf, w.astype(np.float64)), np.isnan(w)
    safe = (pos < sinks) | (pos >= seen - recent)
    stays = np.zeros(n, dtype=bool)
    stays[np.lexsort((np.arange(n), -w[0], ~w[1], ~safe))[:m]] = True
    take = np.arange(m)
    take[~stays[:m]] = m + np.flatnonzero(stays[m:])
    return take


EVICT = [  # lengths, keep, sinks, recent, kv_heads, head_dim, page, type
    ([100], 60, 4, 10, 2, 256, 16, BF), ([0, 1, 2, 3, 50], 2, 0, 0, 1, 64, 16, HF), ([500, 20, 300], 100, 4, 30, 3, 80, 8, BF),
    ([1000, 1024, 1025], 1000, 4, 996, 2, 64, 32, HF), ([5000, 1], 1234, 1, 0, 8, 8, 16, BF),
    ([40, 39], 0, 0, 0, 1, 64, 16, BF), ([33, 70], 200, 4, 10, 1, 64, 16, BF), ([140000, 9, 70001], 20011, 4, 128, 1, 8, 64, BF),
    ([2304], 2048, 4, 256, 2, 256, 16, BF), ([4096] * 3, 1, 1, 0, 1, 16, 1, HF),
    ([8191, 30, 4097], 3001, 4, 500, 2, 64, 16, BF), ([10001, 16000], 9999, 0, 1, 1, 32, 16, HF)]


@pytest.mark.parametrize("weights", ["spread", "equal", "odd"])
@pytest.mark.parametrize("lengths, keep, sinks, recent, hkv, d, page, dtype", EVICT)
def test_evict(cuda, lengths, keep, sinks, recent, hkv, d, page, dtype, weights):
    k, v, table, n, K, V = pool(lengths, hkv, d, page, dtype, seed=keep, layout="joined" if keep % 2 else "plain")
    g = np.random.default_rng(keep + d)
    slots = table.shape[1] * page
    w = np.round(g.random((len(lengths), slots)) * 1e4).astype(np.float32) / 1e4 if weights == "spread" else np.full(
        (len(lengths), slots), 0.25, dtype=np.float32)
    if weights == "odd":
        w = g.choice(np.array([0.0, -0.0, -1.0, 1e-45, 1e-38, 1.0, 3e38, np.inf, -np.inf, np.nan, -np.nan],
                              dtype=np.float32), size=w.shape)
    pos = np.stack([g.permutation(slots) for _ in lengths]).astype(np.int32)
    seen = np.array([max(pos[b, :m], default=0) + 1 for b, m in enumerate(lengths)], dtype=np.int32)
    cw, cp, cs = (torch.from_numpy(a.copy()).cuda() for a in (w, pos, seen))
    cache = context.KVPages(k, v, table, n, weight=cw, position=cp)
    m = max(1, min(keep, slots))
    aside = (torch.full((len(lengths), m), -7.0, device="cuda"), torch.full((len(lengths), m), -7, dtype=torch.int32,
                                                                            device="cuda"), torch.zeros_like(n))
    for out in (aside, None):  # next to the cache's arrays, then in place: the same rows move
        cache.evict(cs, keep, sinks=sinks, recent=recent, out=out)
        torch.cuda.synchronize()
        got = [a.cpu().numpy() for a in (aside if out else (cw, cp, n))]
        for b, length in enumerate(lengths):
            take = kept_slots(w[b, :length], pos[b, :length], seen[b], keep, sinks, recent)
            left = len(take)
            assert got[2][b] == left
            assert np.array_equal(got[0][b, :left].view(np.int32), w[b, take].view(np.int32))
            assert np.array_equal(got[1][b, :left], pos[b, take])
            if out:
                assert (got[1][b, left:] == -7).all()
            at = torch.arange(left, device="cuda")
            at = table[b].long()[at // page], at % page
            src = torch.from_numpy(take).cuda()
            assert torch.equal(k[at], K[b][src]) and torch.equal(v[at], V[b][src])
        if out:
            assert torch.equal(cw.cpu().view(torch.int32), torch.from_numpy(w).view(torch.int32))
    _lib.check_device_errors()


def test_attention_over_a_cache_held_to_its_budget(cuda):
    """Steps of append, attend and evict: what is attended to are the tokens that were kept."""
    hq, hkv, d, page, keep = 8, 2, 64, 16, 48
    k, v, table, n, K, V = pool([60, 50], hkv, d, page, BF, room=80)
    slots = table.shape[1] * page
    w = torch.zeros((2, slots), device="cuda")
    pos = torch.arange(slots, dtype=torch.int32, device="cuda").repeat(2, 1)
    seen = n.clone()
    cache = context.KVPages(k, v, table, n, weight=w, position=pos)
    for step in range(6):
        if step % 2:
            before = n.cpu().tolist(), w.cpu().numpy(), pos.cpu().numpy(), seen.cpu().numpy()
            cache.evict(seen, keep, sinks=4, recent=8)
            for b, m in enumerate(before[0]):
                take = torch.from_numpy(kept_slots(before[1][b, :m], before[2][b, :m], before[3][b], keep, 4, 8)).cuda()
                K[b], V[b] = K[b][take], V[b][take]
        for b in range(2):  # append a token
            s = int(n[b])
            K[b], V[b] = (torch.cat([a, torch.randn((1, hkv, d), device="cuda").to(BF)]) for a in (K[b], V[b]))
            k[table[b, s // page].long(), s % page], v[table[b, s // page].long(), s % page] = K[b][-1], V[b][-1]
            w[b, s], pos[b, s] = 0, seen[b]
        n += 1
        seen += 1
        q = torch.randn((2, hq, d), device="cuda").to(BF)
        old = w.clone()
        check_attention(q, K, V, cache.attend(q), d ** -0.5, w, old)
    assert n.tolist() == [keep + 2, keep + 2] or n.tolist() == [keep + 1, keep + 1]


def test_python_refusals(cuda):
    k, v, table, n, K, V = pool([20], 2, 64, 16, BF)
    w, pos = torch.zeros((1, 32), device="cuda"), torch.zeros((1, 32), dtype=torch.int32, device="cuda")
    q = torch.zeros((1, 4, 64), dtype=BF, device="cuda")
    KV = context.KVPages
    for bad in (dict(v=v.half()), dict(k=k.float(), v=v.float()), dict(v=v[:, :8]), dict(table=table.long()),
                dict(table=table[0]), dict(lengths=n.long()), dict(lengths=n.expand(2)), dict(weight=w[:, :31]),
                dict(weight=w.half()), dict(position=pos.long()), dict(k=k.cpu())):
        with pytest.raises(ValueError):
            KV(**{**dict(k=k, v=v, table=table, lengths=n), **bad})
    cache = KV(k, v, table, n)
    for bad in (q.half(), q[..., :32], q[0], q.cpu(), torch.zeros((1, 3, 64), dtype=BF, device="cuda")):
        with pytest.raises(ValueError):
            cache.attend(bad)
    with pytest.raises(ValueError):
        cache.attend(q, out=torch.zeros((1, 4, 64), device="cuda"))
    with pytest.raises(ValueError):
        cache.evict(n, 4)  # no weight, no position
    cache = KV(k, v, table, n, w, pos)
    for bad in (dict(keep=-1), dict(keep=4, sinks=4, recent=1), dict(keep=4, seen=n.long()),
                dict(keep=8, out=(w[:, :7], pos, n)), dict(keep=8, out=(w, pos, n.float()))):
        with pytest.raises(ValueError):
            cache.evict(**{**dict(seen=n), **bad})
    odd = torch.zeros((4, 16, 2, 68), dtype=BF, device="cuda")[..., :64]
    with pytest.raises(ValueError):
        KV(odd, odd, table, n).attend(q)  # rows 136 bytes apart
    x, g, S = torch.zeros((1, 3, 2, 64), dtype=BF, device="cuda"), torch.zeros((1, 3, 2), device="cuda"), torch.zeros(
        (1, 2, 64, 64), device="cuda")
    for bad in (dict(q=x.float()), dict(k=x.half()), dict(v=x[:, :2]), dict(decay=g.half()), dict(decay=g[:, :2]),
                dict(state=S.half()), dict(state=S[:, :1]), dict(lengths=torch.zeros(1, device="cuda")),
                dict(v=torch.zeros((1, 3, 3, 64), dtype=BF, device="cuda")), dict(state=S.cpu())):
        with pytest.raises(ValueError):
            context.linear_attention(**{**dict(q=x, k=x, v=x, decay=g), **bad})
    big = torch.zeros((1, 3, 2, 136), dtype=BF, device="cuda")
    with pytest.raises(ValueError):
        context.linear_attention(big, big, x, g)
    with pytest.raises(ValueError):
        context.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], g[:, 0], S, out=torch.zeros((1, 2, 64), device="cuda"))


# ---- linear attention


def recurrence(q, k, v, g, S, lengths, scale):
    """Token by token in 64 bits: outputs, the state, and both over absolute values (for the tolerances)."""
    n, t, hk, dk = q.shape
    hv, dv = v.shape[2:]
    rep = hv // hk
    q, k = (x.double().repeat_interleave(rep, 2) for x in (q, k))
    v, g = v.double(), g.double()
    S = torch.zeros((n, hv, dk, dv), dtype=torch.float64, device=q.device) if S is None else S.double()
    A, O, OA = S.abs(), torch.zeros_like(v), torch.zeros_like(v)
    for i in range(t):
        live = torch.ones(n, dtype=torch.bool, device=q.device) if lengths is None else i < lengths
        m = live[:, None, None]
        a = torch.exp(g[:, i])[..., None, None]
        kv = k[:, i, :, :, None] * v[:, i, :, None, :]
        S = torch.where(m[..., None], a * S + kv, S)
        A = torch.where(m[..., None], a * A + kv.abs(), A)
        O[:, i] = torch.where(m, (q[:, i, :, :, None] * S).sum(2) * scale, 0.0)
        OA[:, i] = torch.where(m, (q[:, i, :, :, None].abs() * A).sum(2) * scale, 0.0)
    return O, S, OA, A


def check_linear(args, out, state):
    q, k, v, g, S, lengths, scale = args
    O, F, OA, A = recurrence(*args)
    u, dk = U[q.dtype], q.shape[-1]
    G = 128 * g.clamp(min=-30.0, max=0.0).abs().amax().item() if g.numel() else 0.0
    e = (dk + 200 + G) * E
    tol = u * O.abs() + (3 * u + e) * OA + 1e-7
    err = (out.double() - O).abs()
    assert (err <= tol).all(), (err / tol).max().item()
    tol = (e + 3 * u ** 3) * A + 1e-30
    err = (state.double() - F).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def make(n, t, hk, hv, dk, dv, dtype, decay="spread", stated=True, lengths=None, seed=0, fused=False):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * t + dk)
    if fused:  # q, k and v as views of one projection
        x = torch.randn((n, t, 2 * hk * dk + hv * dv), generator=g, device="cuda").to(dtype)
        q = x[..., : hk * dk].unflatten(-1, (hk, dk))
        k = x[..., hk * dk : 2 * hk * dk].unflatten(-1, (hk, dk))
        v = x[..., 2 * hk * dk :].unflatten(-1, (hv, dv))
    else:
        q, k = (torch.randn((n, t, hk, dk), generator=g, device="cuda").to(dtype) for _ in range(2))
        v = torch.randn((n, t, hv, dv), generator=g, device="cuda").to(dtype)
    r = torch.rand((n, t, hv), generator=g, device="cuda")
    if decay == "spread":
        d = -torch.logspace(-3, 0, hv, device="cuda") * r
    elif decay == "none":
        d = torch.zeros(hv, device="cuda").expand(n, t, hv)  # a fixed decay a head
    elif decay == "fixed":
        d = -torch.logspace(-3, 0, hv, device="cuda").expand(n, t, hv)
    elif decay == "resets":  # documents behind one another: everything before is forgotten
        d = torch.where(r < 0.05, float("-inf"), -0.01 * r)
    else:  # strong: far past what float32 holds over a chunk
        d = -50.0 * r
    if lengths is not None:  # nothing past a length is read
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        dead = torch.arange(t, device="cuda") >= lengths[:, None]
        q, k, v, d = (x.clone() for x in (q, k, v, d))
        for x in (q, k, v, d):
            x[dead] = float("nan")
    S = torch.randn((n, hv, dk, dv), generator=g, device="cuda") if stated else None
    return q, k, v, d, S, lengths, dk ** -0.5


def clean(args):
    q, k, v, d, S, lengths, scale = args
    return (*(x.nan_to_num(0.0, neginf=float("-inf")) if lengths is not None else x for x in (q, k, v, d)), S, lengths, scale)


LINEAR = [  # batch, tokens, k_heads, v_heads, k_dim, v_dim, type
    (1, 1, 1, 1, 64, 64, BF), (2, 2, 2, 2, 128, 128, BF), (2, 63, 2, 4, 64, 64, BF), (1, 64, 1, 1, 128, 128, BF),
    (1, 65, 1, 3, 128, 64, BF), (3, 127, 1, 2, 64, 128, BF), (1, 128, 2, 2, 72, 80, BF), (2, 129, 1, 1, 8, 8, BF),
    (1, 200, 2, 2, 96, 32, HF), (1, 1000, 2, 2, 128, 128, BF), (1, 1000, 1, 2, 64, 48, HF), (2, 3001, 1, 1, 128, 128, BF)]


@pytest.mark.parametrize("decay", ["spread", "none", "resets", "strong"])
@pytest.mark.parametrize("n, t, hk, hv, dk, dv, dtype", LINEAR)
def test_linear_attention(cuda, n, t, hk, hv, dk, dv, dtype, decay):
    args = make(n, t, hk, hv, dk, dv, dtype, decay, stated=t % 2 == 1)
    q, k, v, d, S, _, _ = args
    kept = None if S is None else S.clone()
    out, state = context.linear_attention(q, k, v, d, state=S)
    check_linear(args, out, state)
    assert S is None or torch.equal(S, kept)
    again = context.linear_attention(q, k, v, d, state=S)  # the same bits on every run
    assert torch.equal(out, again[0]) and torch.equal(state, again[1])
    _lib.check_device_errors()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lengths", [[0, 1, 5], [64, 63, 65], [128, 129, 300], [0, 0, 0], [300, 2, 191]])
def test_linear_attention_of_ragged_prompts(cuda, lengths, dtype):
    args = make(3, 300, 1, 2, 128, 64, dtype, lengths=lengths)
    out, state = context.linear_attention(*args[:4], state=args[4], lengths=args[5])
    check_linear(clean(args), out, state)
    for b, m in enumerate(lengths):
        assert (out[b, m:] == 0).all()
        if m == 0:
            assert torch.equal(state[b], args[4][b])


def test_linear_attention_of_long_ragged_prompts(cuda):
    lengths = [1100, 0, 513, 64]  # in several segments, most of them short or empty
    args = make(4, 1100, 2, 2, 128, 128, BF, lengths=lengths)
    out, state = context.linear_attention(*args[:4], state=args[4], lengths=args[5])
    check_linear(clean(args), out, state)
    assert all((out[b, m:] == 0).all() for b, m in enumerate(lengths)) and torch.equal(state[1], args[4][1])


def test_linear_attention_of_views_and_nothing(cuda):
    args = make(2, 150, 2, 4, 64, 64, BF, "fixed", fused=True)
    out, state = context.linear_attention(*args[:4], state=args[4], scale=0.3)
    check_linear((*args[:6], 0.3), out, state)
    out, state = context.linear_attention(*(x[:, :0] for x in args[:4]), state=args[4])
    assert out.shape == (2, 0, 4, 64) and torch.equal(state, args[4])
    out, state = context.linear_attention(*(x[:0] for x in args[:4]))
    assert out.shape == (0, 150, 4, 64) and state.shape == (0, 4, 64, 64)
    k, v, table, n, _, _ = pool([20], 2, 64, 16, BF)
    none = context.decode_attention(torch.empty((0, 4, 64), dtype=BF, device="cuda"), k, v, table[:0], n[:0])
    assert none.shape == (0, 4, 64)


def test_a_prompt_in_parts_and_then_token_by_token(cuda):
    n, t, h, d = 2, 301, 2, 128
    q, k, v, g, S, _, scale = args = make(n, t, h, h, d, d, BF)
    cut = [0, 130, 131, 290]
    outs, state = [], S
    for a, b in zip(cut, cut[1:]):
        o, state = context.linear_attention(*(x[:, a:b] for x in (q, k, v, g)), state=state)
        outs.append(o)
    for i in range(290, t):
        outs.append(context.linear_attention_step(*(x[:, i] for x in (q, k, v, g)), state)[:, None])
    check_linear(args, torch.cat(outs, 1), state)


STEP = [(1, 1, 1, 64, 64, BF), (3, 2, 6, 128, 128, HF), (70, 2, 2, 72, 80, BF), (1, 16, 16, 128, 128, BF),
        (2, 4, 4, 8, 128, HF), (5, 1, 3, 128, 8, BF), (33, 8, 32, 96, 96, HF)]


@pytest.mark.parametrize("decay", ["spread", "none", "resets"])
@pytest.mark.parametrize("n, hk, hv, dk, dv, dtype", STEP)
def test_linear_attention_step(cuda, n, hk, hv, dk, dv, dtype, decay):
    q, k, v, g, S, _, scale = args = make(n, 1, hk, hv, dk, dv, dtype, decay)
    state = S.clone()
    out = context.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state)
    check_linear(args, out[:, None], state)
    buf = torch.empty_like(out)
    state.copy_(S)
    assert context.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, out=buf) is buf
    assert torch.equal(buf, out)
