"""The hybrid decoder without a GPU: what it refuses, or holds to its bounds, before anything is launched."""

import pytest
import torch

from strata_mlx_b200 import hybrid as H


def make(**kw):
    return H.HybridDecoder(**{**dict(layers=1, batch=2, capacity=48, keep=32, sinks=2, recent=8, hidden=64, linear_heads=2,
                                     linear_dim=8, experts=0, vocab=16, max_pos=40, device="cpu"), **kw})


def test_positions_past_the_rotary_table_are_refused():
    """On the GPU an index past the table's end is a failed assertion of the device."""
    dec = make()
    lengths = torch.tensor([3, 41], dtype=torch.int32)
    with pytest.raises(ValueError, match="max_pos"):
        dec.prompt(torch.zeros((2, 41), dtype=torch.int64), lengths)
    dec.layers = []  # the embedding and the head alone
    dec.prompt(torch.zeros((2, 38), dtype=torch.int64), torch.tensor([38, 5], dtype=torch.int32))
    for _ in range(2):
        dec.step(torch.zeros(2, dtype=torch.int64))
    assert dec.seen.tolist() == [40, 7]
    with pytest.raises(ValueError, match="max_pos"):
        dec.step(torch.zeros(2, dtype=torch.int64))
    assert dec.seen.tolist() == [40, 7] and dec.lengths.tolist() == [40, 7]
    dec.prompt(torch.zeros((2, 5), dtype=torch.int64), torch.tensor([5, 5], dtype=torch.int32))  # a new prompt starts over
    dec.step(torch.zeros(2, dtype=torch.int64))


def test_lengths_past_the_prompts_are_held_to_them():
    """A length outside the prompt's width would index past the tokens here, and past the cache at the next step."""
    dec = make()
    dec.layers = []
    tokens = torch.arange(16).reshape(2, 8)
    logits = dec.prompt(tokens, torch.tensor([99, 8], dtype=torch.int32))
    assert torch.equal(logits, dec.prompt(tokens, torch.tensor([8, 8], dtype=torch.int32)))
    dec.prompt(tokens, torch.tensor([99, -4], dtype=torch.int32))
    assert dec.lengths.tolist() == [8, 0] and dec.seen.tolist() == [8, 0]
