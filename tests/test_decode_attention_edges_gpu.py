"""Decode attention where its sums could lose something: long float16 tails under a peak, and batches of more sequences
than a block has threads. Against the definition in 64 bits.

Tolerances (u: the type's unit roundoff, e = 2^-23, m: slots, D: head_dim): a score is off by ds = (D + 4) e S at most, S
the largest scale sum |q_i k_i|. Outputs: u |o| for their rounding, half of their type's least value (2^-25 in float16),
and (2 ds + (m + 64) e + u^2) sum p |v| as a probability enters the value product as two terms of the type; a float16
term has no bits below 2^-24, which is 2^-39 of the largest probability a warp has met, so a slot's is off by 2^-40 of the
peak's at most: 2^-40 sum |v| more. Weights: (2 ds + (m + 64) e) p and e of the sum."""

import pytest
import torch

from strata_mlx_b200 import _lib, context

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}
LEAST = {BF: 2.0 ** -134, HF: 2.0 ** -25}
E = 2.0 ** -23


def pool(lengths, hkv, d, page, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, per = len(lengths), max(1, -(-max(lengths) // page))
    k, v = (torch.randn((n * per, page, hkv, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(n * per, generator=g, device="cuda").to(torch.int32).reshape(n, per)
    return k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check(q, k, v, table, lengths, weight=None):
    """attend against softmax in 64 bits, sequence by sequence."""
    n, hq, d = q.shape
    page, hk = k.shape[1:3]
    scale, u = d ** -0.5, U[q.dtype]
    before = None if weight is None else weight.clone()
    out = context.decode_attention(q, k, v, table, lengths, weight=weight)
    for b, m in enumerate(lengths.tolist()):
        if m == 0:
            assert (out[b] == 0).all() and (weight is None or torch.equal(weight[b], before[b]))
            continue
        rows = table[b, : -(-m // page)].long()
        K, V = (x[rows].reshape(-1, hk, d)[:m].double() for x in (k, v))
        Q = q[b].double().reshape(hk, hq // hk, d)
        p = torch.softmax(torch.einsum("hgd,thd->hgt", Q, K) * scale, -1)
        ds = (d + 4) * E * scale * torch.einsum("hgd,thd->hgt", Q.abs(), K.abs()).amax(-1, keepdim=True)
        o, av = torch.einsum("hgt,thd->hgd", p, V), V.abs()
        tol = (u * o.abs() + LEAST[q.dtype] + (2 * ds + (m + 64) * E + u * u) * torch.einsum("hgt,thd->hgd", p, av)
               + 2.0 ** -40 * p.amax(-1, keepdim=True) * av.sum(0)[:, None])
        ratio = (out[b].double().reshape(hk, hq // hk, d) - o).abs() / tol
        assert (ratio <= 1).all(), (b, m, ratio.max().item())
        if weight is not None:
            w = p.sum((0, 1))
            tol = ((2 * ds + (m + 64) * E) * p).sum((0, 1)) + E * (before[b, :m].double() + w) + 2.0 ** -126
            ratio = (weight[b, :m].double() - before[b, :m].double() - w).abs() / tol
            assert (ratio <= 1).all(), (b, m, ratio.max().item())
            assert torch.equal(weight[b, m:], before[b, m:])
    _lib.check_device_errors()
    return out


def sinks(n, m, d, dtype, tail, value, at):
    """n sequences of m slots, of which the slots `at` hold most of the attention, with a value of zero or an ordinary
    one, and the others lie `tail` nats below, flat for one query head and spread for the other."""
    k, v, table, lengths = pool([m] * n, 1, d, 64, dtype)
    v.abs_()  # so that the tail's sum is not near zero
    k[..., 0] = 0
    q = torch.zeros((n, 2, d), dtype=dtype, device="cuda")
    q[..., 0] = float(d) ** 0.5
    q[:, 1, 1] = 0.01 * float(d) ** 0.5
    for s in at:
        page = table[:, s // 64].long()
        k[page, s % 64, 0, 0] = tail
        v[page, s % 64, 0] = value
    return q, k, v, table, lengths


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("tail", [12.0, 17.7, 18.5, 20.0])
@pytest.mark.parametrize("value", [0.0, 1.0])
def test_a_long_tail_under_one_peak(cuda, dtype, d, tail, value):
    check(*sinks(1, 131072, d, dtype, tail, value, [44807]))


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("n, d", [(448, 64), (448, 128), (150, 256)])
@pytest.mark.parametrize("tail", [8.0, 16.0, 17.7, 18.5, 20.0])
@pytest.mark.parametrize("value", [0.0, 1.0])
def test_long_tails_under_sinks(cuda, dtype, n, d, tail, value):
    """So many sequences that a block has whole ones, their first slots sinks: each warp meets one, and the tail behind it."""
    q, k, v, table, lengths = sinks(n, 8192, d, dtype, tail, value, range(0, 256, 8))
    out = context.decode_attention(q, k, v, table, lengths)
    some = torch.tensor([0, 1, n // 2, n - 1], device="cuda")
    got = check(q[some], k, v, table[some].contiguous(), lengths[some])
    rows = table[some].long()
    for b, r in zip(some.tolist(), rows):  # as check, for the whole batch's outputs
        K, V = (x[r].reshape(-1, d).double() for x in (k, v))
        p = torch.softmax(q[b].double() @ K.T * d ** -0.5, -1)
        o, u = p @ V, U[dtype]
        ds = (d + 4) * E * d ** -0.5 * (q[b].double().abs() @ K.abs().T).amax(-1, keepdim=True)
        tol = (u * o.abs() + LEAST[dtype] + (2 * ds + (8192 + 64) * E + u * u) * (p @ V.abs())
               + 2.0 ** -40 * p.amax(-1, keepdim=True) * V.abs().sum(0))
        ratio = (out[b].double() - o).abs() / tol
        assert (ratio <= 1).all(), (b, ratio.max().item())
    assert got.shape == (4, 2, d)


def ragged(n, most, seed):
    """Lengths of n sequences, empty ones among them and around the ends of runs of 128 and 256."""
    g = torch.Generator().manual_seed(seed)
    got = torch.randint(1, most + 1, (n,), generator=g)
    got[torch.randperm(n, generator=g)[: n // 4]] = 0
    for at in (0, 126, 127, 128, 129, 254, 255, 256, 257, 511, 512, 513, n - 1):
        if at < n:
            got[at] = 0 if at % 3 else most
    return got.tolist()


@pytest.mark.parametrize("tracked", [False, True])
@pytest.mark.parametrize("d, hq, hkv, dtype", [(64, 6, 2, HF), (128, 4, 4, BF), (256, 8, 1, BF)])
@pytest.mark.parametrize("n", [2, 127, 128, 129, 256, 257, 300, 511, 512, 513, 1100])
def test_more_sequences_than_a_block_has_threads(cuda, n, d, hq, hkv, dtype, tracked):
    lengths = ragged(n, 200, n + d)
    k, v, table, t = pool(lengths, hkv, d, 16, dtype)
    q = torch.randn((n, hq, d), device="cuda").to(dtype)
    weight = torch.rand((n, table.shape[1] * 16), device="cuda") if tracked else None
    check(q, k, v, table, t, weight)


@pytest.mark.parametrize("tracked", [False, True])
@pytest.mark.parametrize("lengths", [[0] * 300, [0] * 299 + [1], [1] + [0] * 299, [0] * 150 + [700] + [0] * 149])
def test_hardly_a_sequence_with_tokens(cuda, lengths, tracked):
    k, v, table, t = pool(lengths, 2, 64, 16, BF)
    q = torch.randn((300, 4, 64), device="cuda").to(BF)
    check(q, k, v, table, t, torch.rand((300, table.shape[1] * 16), device="cuda") if tracked else None)


def test_thousands_of_sequences(cuda):
    """Some of them against the definition; the whole twice, with the same bits."""
    n, d = 20000, 64
    lengths = torch.randint(0, 90, (n,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    k, v = (torch.randn((500, 16, 2, d), device="cuda").to(BF) for _ in range(2))
    table = torch.randint(0, 500, (n, 6), device="cuda", dtype=torch.int32)
    q = torch.randn((n, 4, d), device="cuda").to(BF)
    weight = torch.zeros((n, 96), device="cuda")
    out = context.decode_attention(q, k, v, table, lengths, weight=weight)
    some = torch.cat([torch.arange(0, n, 499), torch.tensor([n - 1])]).cuda()
    alone = torch.zeros((len(some), 96), device="cuda")
    want = check(q[some], k, v, table[some].contiguous(), lengths[some], alone)
    assert torch.equal(out[some], want)  # such short sequences lie in one unit each: the same sums
    assert torch.equal(weight[some], alone)
    assert torch.equal(out, context.decode_attention(q, k, v, table, lengths))


def test_time_grows_with_the_batch_not_its_square(cuda):
    """65,535 sequences of up to 64 tokens: under 2 ms of work. Where every block counted all lengths: 134 ms."""
    n, d = 65535, 64
    lengths = torch.randint(0, 65, (n,), dtype=torch.int32, device="cuda")
    k, v = (torch.randn((512, 16, 2, d), device="cuda").to(BF) for _ in range(2))
    table = torch.randint(0, 512, (n, 4), device="cuda", dtype=torch.int32)
    q = torch.randn((n, 16, d), device="cuda").to(BF)
    cache, out, best = context.KVPages(k, v, table, lengths), torch.empty_like(q), float("inf")
    for _ in range(4):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        cache.attend(q, out=out)
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    assert best < 20.0, best
