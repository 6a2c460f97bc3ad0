"""The context operators without a GPU: argument checks of the C entry points answer before any launch, workspaces
have their sizes, and the Python calls refuse tensors off the GPU."""

import ctypes

import pytest
import torch

from strata_mlx_b200 import _lib, context

FAKE = 0x1000  # never dereferenced


def pages(**kw) -> "_lib.SCPages":
    P = _lib.SCPages()
    P.k = P.v = P.table = P.lengths = P.weight = P.position = FAKE
    P.batch, P.kv_heads, P.head_dim, P.page, P.pool_pages, P.max_pages, P.dtype = 2, 2, 64, 16, 8, 4, 2
    P.k_head = P.v_head = 64
    P.k_token = P.v_token = 128
    P.k_page = P.v_page = 2048
    P.table_row, P.weight_row, P.position_row = 4, 64, 64
    for name, v in kw.items():
        setattr(P, name, v)
    return P


def attend(P, q=FAKE, q_row=256, q_head=64, heads=4, out=FAKE, ws=FAKE, ws_bytes=None):
    lib = _lib.load()
    n = lib.sc_decode_attention_workspace(ctypes.addressof(P), heads) if ws_bytes is None else ws_bytes
    return lib.sc_decode_attention(ctypes.addressof(P), q, q_row, q_head, heads, ctypes.c_float(1.0), out, ws, n, None,
                                   None)


BAD_PAGES = [({"k": None}, -5), ({"table": None}, -5), ({"lengths": None}, -5), ({"batch": -1}, -5),
             ({"dtype": 0}, -3), ({"dtype": 7}, -3), ({"head_dim": 60}, -2), ({"head_dim": 264}, -2),
             ({"page": 12}, -2), ({"page": 0}, -2), ({"kv_heads": 0}, -2), ({"pool_pages": 0}, -2),
             ({"max_pages": 0}, -2), ({"max_pages": 1 << 27}, -2), ({"k": FAKE + 8}, -4), ({"v_head": 68}, -4),
             ({"k_token": 4}, -4)]


@pytest.mark.parametrize("change, code", BAD_PAGES)
def test_a_cache_the_kernels_do_not_take_is_refused(change, code):
    lib = _lib.load()
    P = pages(**change)
    assert attend(P, ws_bytes=1 << 20) == code
    assert lib.sc_decode_attention_workspace(ctypes.addressof(P), 4) == 0
    assert lib.sc_evict_workspace(ctypes.addressof(P), 16) == 0
    assert lib.sc_evict(ctypes.addressof(P), FAKE, 16, 4, 4, FAKE, 64, FAKE, 64, FAKE, FAKE, 1 << 20, None, None) == code


def test_decode_attention_refusals():
    P = pages()
    assert attend(P, q=None) == -5 and attend(P, out=None) == -5 and attend(P, ws=None) == -5
    assert attend(P, heads=3) == -2 and attend(P, heads=0) == -2  # not a multiple of the cache's heads
    assert attend(P, q=FAKE + 2) == -4 and attend(P, q_row=252) == -4 and attend(P, q_head=4) == -4
    assert attend(P, out=FAKE + 8) == -4
    n = _lib.load().sc_decode_attention_workspace(ctypes.addressof(P), 4)
    assert n > 0 and attend(P, ws_bytes=n - 1) == -7
    assert attend(pages(batch=0)) == 0  # nothing to do, nothing launched
    assert _lib.load().sc_decode_attention(None, FAKE, 0, 0, 1, ctypes.c_float(1.0), FAKE, FAKE, 64, None, None) == -5


def test_evict_refusals():
    lib = _lib.load()
    P = pages()
    n = lib.sc_evict_workspace(ctypes.addressof(P), 16)

    def evict(P=P, seen=FAKE, keep=16, sinks=4, recent=4, ws=FAKE, ws_bytes=n, w=FAKE, lengths=FAKE):
        return lib.sc_evict(ctypes.addressof(P), seen, keep, sinks, recent, w, 64, FAKE, 64, lengths, ws, ws_bytes,
                            None, None)

    assert n > 0 and evict(ws_bytes=n - 1) == -7
    assert evict(seen=None) == -5 and evict(w=None) == -5 and evict(lengths=None) == -5 and evict(ws=None) == -5
    assert evict(pages(weight=None)) == -5 and evict(pages(position=None)) == -5
    assert evict(keep=-1) == -5 and evict(sinks=-1) == -5 and evict(recent=-1) == -5
    assert evict(sinks=10, recent=7) == -2  # more than is kept
    assert evict(recent=(1 << 31) - 1, sinks=4) == -2  # a sum past 32 bits
    assert evict(ws=FAKE + 4) == -4
    assert evict(pages(batch=0)) == 0
    # the lists hold what can move: nothing when every slot is kept
    assert lib.sc_evict_workspace(ctypes.addressof(P), 16) > lib.sc_evict_workspace(ctypes.addressof(P), 64)


def linear(**kw) -> "_lib.SCLinear":
    A = _lib.SCLinear()
    A.q = A.k = A.v = A.decay = A.state_in = A.state_out = A.out = FAKE
    A.batch, A.tokens, A.k_heads, A.v_heads, A.k_dim, A.v_dim, A.dtype = 2, 1, 2, 4, 64, 64, 2
    A.q_head = A.k_head = A.v_head = 64
    for name, v in kw.items():
        setattr(A, name, v)
    return A


@pytest.mark.parametrize("change, code", [
    ({"q": None}, -5), ({"decay": None}, -5), ({"state_out": None}, -5), ({"out": None}, -5), ({"batch": -1}, -5),
    ({"tokens": -1}, -5), ({"dtype": 0}, -3), ({"v_heads": 3}, -2), ({"k_heads": 0}, -2), ({"k_dim": 136}, -2),
    ({"k_dim": 60}, -2), ({"v_dim": 136}, -2), ({"v_dim": 4}, -2), ({"v": FAKE + 2}, -4), ({"q_head": 60}, -4),
    ({"state_in": FAKE + 4}, -4), ({"out": FAKE + 8}, -4)])
def test_linear_attention_refusals(change, code):
    lib = _lib.load()
    A = linear(**change)
    assert lib.sc_linear_attention_workspace(ctypes.addressof(A)) == 0
    assert lib.sc_linear_attention(ctypes.addressof(A), FAKE, 1 << 40, None, None) == code
    assert lib.sc_linear_attention_step(ctypes.addressof(A), None) == code


def test_linear_attention_workspace_and_the_step_form():
    lib = _lib.load()
    A = linear(tokens=4096, q_token=128, k_token=128, v_token=256, q_row=1 << 20, k_row=1 << 20, v_row=1 << 20)
    n = lib.sc_linear_attention_workspace(ctypes.addressof(A))
    assert n > 0 and lib.sc_linear_attention(ctypes.addressof(A), FAKE, n - 1, None, None) == -7
    assert lib.sc_linear_attention(ctypes.addressof(A), None, n, None, None) == -5
    assert lib.sc_linear_attention(ctypes.addressof(A), FAKE + 8, n, None, None) == -4
    assert lib.sc_linear_attention_workspace(ctypes.addressof(linear(tokens=8))) == 0  # the recurrence needs none
    assert lib.sc_linear_attention_step(ctypes.addressof(A), None) == -2  # one token a sequence
    assert lib.sc_linear_attention_step(ctypes.addressof(linear(lengths=FAKE)), None) == -2
    assert lib.sc_linear_attention_step(ctypes.addressof(linear(batch=0)), None) == 0
    assert lib.sc_linear_attention(ctypes.addressof(linear(batch=0)), FAKE, n, None, None) == 0


def test_the_packed_call_is_the_structure():
    """linear_attention packs sc_linear field by field: the same bytes as the structure."""
    A = linear(tokens=7, batch=3, scale=0.25)
    for i, (name, kind) in enumerate(A._fields_):
        setattr(A, name, i + 1)
    assert context._LINEAR.pack(*(getattr(A, name) for name, _ in A._fields_)) == bytes(A)


def test_calls_refuse_tensors_off_the_gpu():
    k = torch.zeros((2, 16, 1, 64), dtype=torch.bfloat16)
    table, lengths = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        context.KVPages(k, k, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        context.decode_attention(torch.zeros((1, 4, 64), dtype=torch.bfloat16), k, k, table, lengths)
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    g, state = torch.zeros((1, 2)), torch.zeros((1, 2, 64, 64))
    with pytest.raises(ValueError, match="CUDA"):
        context.linear_attention_step(x, x, x, g, state)
    with pytest.raises(ValueError, match="CUDA"):
        context.linear_attention(x[:, None], x[:, None], x[:, None], g[:, None])
    with pytest.raises(ValueError):
        context.linear_attention(x, x, x, g)  # a prompt has a token axis
    with pytest.raises(ValueError):
        context.linear_attention_step(x, x, x, g, None)
