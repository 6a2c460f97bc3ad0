"""The hybrid decoder's prompts: rows past what one attention call takes, and its layers one at a time against 64 bits."""

import pytest
import torch

from strata_mlx_b200 import _lib
from strata_mlx_b200 import hybrid as H

pytestmark = pytest.mark.gpu


def make(**kw):
    return H.HybridDecoder(**{**dict(layers=2, batch=3, capacity=96, keep=64, sinks=2, recent=16, hidden=256, linear_heads=2,
                                     linear_dim=64, q_heads=4, kv_heads=2, experts=0, vocab=256, max_pos=512), **kw})


def test_more_prompt_rows_than_a_call_takes(cuda):
    """35 prompts of up to 2000 tokens: 70,000 rows of attention."""
    dec = make(batch=35, capacity=2000, keep=1000, max_pos=2048, layers=1, every=1, hidden=64, q_heads=1, kv_heads=1)
    lengths = torch.randint(1, 2001, (35,), dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, 256, (35, 2000), device="cuda")
    logits = dec.prompt(tokens, lengths)
    assert torch.isfinite(logits).all()
    mixer = dec.layers[0][0]
    at = torch.arange(2000, device="cuda")
    # every token that is seen gives its one head's weight, 1 in all: as much as there are tokens
    assert torch.allclose(mixer.weight.sum(1), lengths.float(), rtol=1e-3)  # 2000 slots' sums round at 2^-23 each
    assert (mixer.weight[at >= lengths[:, None]] == 0).all()
    _lib.check_device_errors()


def test_rows_in_pieces_are_rows_at_once(cuda, monkeypatch):
    lengths = torch.tensor([90, 1, 63], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, 256, (3, 90), device="cuda")
    a, b = make(), make()
    whole = a.prompt(tokens, lengths)
    monkeypatch.setattr(H, "ROWS", 21)  # seven tokens of each
    pieces = b.prompt(tokens, lengths)
    assert torch.equal(whole, pieces)  # short rows lie in one unit each: the same sums
    wa, wb = a.layers[1][0].weight, b.layers[1][0].weight
    assert torch.allclose(wa, wb, rtol=1e-5, atol=1e-6)
    _lib.check_device_errors()


def close(a, b):
    """Head by head, to bfloat16 roundings of inputs, products and outputs: 8 x 2^-8 of a head's 2-norm."""
    a, b = a.float(), b.float()
    ratio = (a - b).norm(dim=-1) / (2.0 ** -5 * b.norm(dim=-1) + 1e-6)
    assert (ratio <= 1).all(), ratio.max().item()


def test_a_cache_layer_s_prompt_is_its_steps(cuda):
    """One full attention layer on the same inputs: every head of every token, the caches and what slots gathered."""
    t, lengths = 70, torch.tensor([70, 1, 33], dtype=torch.int32, device="cuda")
    a, b = make(layers=1, every=1), make(layers=1, every=1)
    h = torch.randn((3, t, 256), device="cuda").to(torch.bfloat16)
    x, y = a.layers[0][0], b.layers[0][0]
    x.wo = y.wo = lambda out: out  # the heads as they are
    whole = x.prompt(h, lengths).unflatten(-1, (4, -1))
    for i in range(t):
        b.lengths += 1
        close(y.step(h[:, i].contiguous()).unflatten(-1, (4, -1))[lengths > i], whole[:, i][lengths > i])
        b.seen += 1
    for n, m in enumerate(lengths.tolist()):
        rows = [d.rows(torch.arange(m, device="cuda").expand(3, m))[n] for d in (a, b)]
        for p, q in ((x.k, y.k), (x.v, y.v)):
            close(p.view(-1, 2, 256)[rows[0]], q.view(-1, 2, 256)[rows[1]])
        assert torch.equal(x.position[n, :m], y.position[n, :m])
    assert torch.allclose(x.weight[0, :70], y.weight[0, :70], rtol=2.0 ** -5)


def test_a_linear_layer_s_prompt_is_its_steps(cuda):
    t = 70
    lengths = torch.tensor([70, 1, 33], dtype=torch.int32, device="cuda")
    a, b = make(layers=1, linear_heads=4), make(layers=1, linear_heads=4)
    h = torch.randn((3, t, 256), device="cuda").to(torch.bfloat16)
    x, y = a.layers[0][0], b.layers[0][0]
    x.wo = y.wo = lambda out: out
    whole = x.prompt(h, lengths).unflatten(-1, (4, -1))
    y.state = torch.zeros_like(x.state)
    for i in range(t):
        close(y.step(h[:, i].contiguous()).unflatten(-1, (4, -1))[lengths > i], whole[:, i][lengths > i])
        for n in (lengths == i + 1).nonzero()[:, 0].tolist():
            close(y.state[n].flatten(1), x.state[n].flatten(1))
