"""The hybrid decoder (hybrid.HybridDecoder): linear and full attention layers over a batch, prompts and steps, caches
held to a budget."""

import pytest
import torch

from strata_mlx_b200 import _lib
from strata_mlx_b200 import hybrid as H

pytestmark = pytest.mark.gpu


def make(**kw):
    return H.HybridDecoder(**{**dict(layers=4, batch=3, capacity=96, keep=64, sinks=2, recent=16, hidden=512, linear_heads=4,
                                     linear_dim=64, q_heads=4, kv_heads=2, experts=0, vocab=256, max_pos=512), **kw})


def test_a_prompt_is_its_tokens_one_by_one(cuda):
    """Without MoE blocks (whose routes could differ at near-ties) the two ways agree to bfloat16's rounding through
    four layers: 4 x 2 roundings of 2^-8 in the residual stream, an eighth of it at most in the logits' 2-norm."""
    g = torch.Generator(device="cuda").manual_seed(0)
    lengths = torch.tensor([40, 1, 23], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, 256, (3, 40), generator=g, device="cuda")
    a, b = make(), make()
    logits = a.prompt(tokens, lengths)
    one = b.prompt(tokens[:, :1], torch.ones(3, dtype=torch.int32, device="cuda"))
    last = torch.where(lengths[:, None] == 1, one, 0.0)
    for i in range(1, 40):
        out = b.step(tokens[:, i])
        last = torch.where(lengths[:, None] == i + 1, out, last)
    assert ((logits - last).norm(dim=-1) <= 0.125 * last.norm(dim=-1)).all()
    for (m, _), (n, _) in zip(a.layers, b.layers):
        if isinstance(m, H.LinearMixer):  # the state of the longest prompt, which both have read whole
            assert (m.state[0] - n.state[0]).norm() <= 0.125 * n.state[0].norm()
    _lib.check_device_errors()


@pytest.mark.parametrize("experts", [0, 16])
def test_caches_stay_within_their_budget(cuda, experts):
    kw = dict(hidden=2048, inter=512, experts=16, top_k=4) if experts else {}
    dec = make(batch=2, **kw)
    lengths = torch.tensor([50, 7], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, 256, (2, 50), device="cuda")
    nxt = dec.prompt(tokens, lengths).argmax(-1)
    for i in range(150):
        logits = dec.step(nxt)
        nxt = logits.argmax(-1)
    assert torch.isfinite(logits).all()
    assert dec.seen.tolist() == [200, 157]
    assert dec.most <= 96 and (dec.lengths <= dec.most).all() and (dec.lengths >= 64).all()
    for mixer, _ in dec.layers:
        if isinstance(mixer, H.CacheMixer):
            for b, n in enumerate(dec.lengths.tolist()):
                at = mixer.position[b, :n].tolist()
                seen = dec.seen[b].item()
                assert len(set(at)) == n and max(at) < seen  # each slot another token
                assert {0, 1} <= set(at)  # the sinks
                # the tokens since the last eviction, and the 16 recent ones that it kept
                assert set(range(seen - (n - 64) - 16, seen)) <= set(at)
    _lib.check_device_errors()


def test_refusals(cuda):
    with pytest.raises(ValueError):
        make(capacity=90)
    with pytest.raises(ValueError):
        make(keep=96)
    with pytest.raises(ValueError):
        make(recent=64)
    dec = make()
    with pytest.raises(ValueError):
        dec.prompt(torch.zeros((3, 97), dtype=torch.int64, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        dec.prompt(torch.zeros((2, 9), dtype=torch.int64, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"))
