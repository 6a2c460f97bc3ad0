"""KVPages without a GPU, against a library that only records: what its calls do on the host."""

import threading
import time

import pytest
import torch

from strata_mlx_b200 import context


class Recorder:
    """Stands for the library: notes the arguments, and whether a call came while another was under way."""

    def __init__(self):
        self.busy, self.overlaps, self.calls = 0, 0, []

    def _call(self, name, args):
        self.busy += 1
        self.overlaps += self.busy > 1
        time.sleep(0.002)
        self.calls.append((name, args))
        self.busy -= 1
        return 0

    def sc_decode_attention(self, *args):
        return self._call("attend", args)

    def sc_evict(self, *args):
        return self._call("evict", args)

    def sc_error_string(self, code):
        return b"refused"

    def sc_decode_attention_workspace(self, *args):
        return 64

    def sc_evict_workspace(self, *args):
        return 64


@pytest.fixture
def cache(monkeypatch):
    """A cache on the CPU whose calls reach the recorder."""
    monkeypatch.setattr(context, "_here", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(context, "_stream", lambda index: 0)
    monkeypatch.setattr(context, "_capturing", lambda: False)
    monkeypatch.setattr(context._lib, "error_word", lambda device=None: torch.zeros(4, dtype=torch.int32))
    lib = Recorder()
    monkeypatch.setattr(context._lib, "lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    k = torch.zeros((4, 16, 1, 64), dtype=torch.bfloat16)
    table = torch.arange(4, dtype=torch.int32).reshape(2, 2)
    lengths = torch.tensor([20, 9], dtype=torch.int32)
    c = context.KVPages(k, k.clone(), table, lengths, torch.zeros((2, 32)), torch.zeros((2, 32), dtype=torch.int32))
    c._index = -1  # the index of a tensor on the CPU
    return c, lib


def test_two_threads_calls_follow_each_other(cache):
    """A call is two launches over one workspace: another's launch must not come between them."""
    c, lib = cache
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    seen = c.lengths.clone()

    def work():
        for _ in range(5):
            c.attend(q)
            c.evict(seen, 12, sinks=0)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(lib.calls) == 40 and lib.overlaps == 0


def test_a_call_that_fails_does_not_hold_the_others_up(cache):
    c, lib = cache
    lib.sc_decode_attention = lambda *args: -2
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for _ in range(2):
        with pytest.raises(ValueError):
            c.attend(q)
    c.evict(c.lengths.clone(), 12, sinks=0)
    assert [name for name, _ in lib.calls] == ["evict"]


@pytest.mark.parametrize("keep", [1 << 31, 1 << 32, (1 << 32) + 5, 1 << 40])
def test_a_budget_past_32_bits_is_refused(cache, keep):
    """It would reach the library as its low 32 bits: 2^32 as a budget of nothing."""
    c, lib = cache
    with pytest.raises(ValueError, match="keep"):
        c.evict(c.lengths.clone(), keep, sinks=0)
    assert not lib.calls
    c.evict(c.lengths.clone(), (1 << 31) - 1, sinks=0)
    assert lib.calls[0][1][2] == (1 << 31) - 1


def test_rows_that_are_written_may_not_overlap(cache):
    """Sequences are worked on side by side: one row of weights for several would be a race."""
    c, lib = cache
    kv = c.k, c.v, c.table, c.lengths
    one, pos = torch.zeros((1, 32)), torch.zeros((2, 32), dtype=torch.int32)
    for bad in (dict(weight=one.expand(2, -1)), dict(weight=torch.zeros(48).as_strided((2, 32), (16, 1))),
                dict(weight=c.weight, position=pos[:1].expand(2, -1))):
        with pytest.raises(ValueError, match="overlap"):
            context.KVPages(*kv, **bad)
    for out in ((one.expand(2, -1), pos, c.lengths), (torch.zeros((2, 32)), pos[:1].expand(2, -1), c.lengths)):
        with pytest.raises(ValueError, match="overlap"):
            c.evict(c.lengths.clone(), 12, sinks=0, out=out)
    alone = context.KVPages(c.k, c.v, c.table[:1], c.lengths[:1], weight=one.as_strided((1, 32), (0, 1)))
    alone._index = -1
    alone.attend(torch.zeros((1, 4, 64), dtype=torch.bfloat16))
    assert [name for name, _ in lib.calls] == ["attend"]
