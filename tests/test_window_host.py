"""Sliding windows on the CPU: the attention's torch route against the definition, the token counts of the split plan
and the refusals of the C entry points."""
import pytest
import torch

from threadcut_amd import _lib, attention
from threadcut_amd.paged import PageTable


def definition(q, k, v, window, sinks):
    t, n = q.shape[2], k.shape[2]
    p = torch.arange(n - t, n)[:, None]
    j = torch.arange(n)
    hidden = (j > p) | ((j <= p - window) & (j >= sinks))
    g = q.shape[1] // k.shape[1]
    s = q @ k.repeat_interleave(g, 1).transpose(2, 3) * q.shape[-1] ** -0.5
    return (torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ v.repeat_interleave(g, 1)).transpose(1, 2)


@pytest.mark.parametrize("t,n,window,sinks", [(1, 50, 8, 2), (1, 50, 60, 0), (7, 50, 8, 2), (50, 50, 8, 0), (50, 50, 90, 0),
                                              (7, 50, 90, 0), (1, 50, 1, 0), (20, 30, 4, 100)])
def test_attention_on_the_host(t, n, window, sinks):
    g = torch.Generator().manual_seed(t * n)
    q, k, v = (torch.randn(2, h, m, 16, generator=g, dtype=torch.float64) for h, m in ((6, t), (2, n), (2, n)))
    out = attention.attention(None, q, k, v, None, sliding_window=window, sink_tokens=sinks)[0]
    assert torch.allclose(out, definition(q, k, v, window, sinks), rtol=0, atol=1e-12)
    masked = attention.attention(None, q, k, v, torch.ones(1, 1, t, n, dtype=torch.bool), sliding_window=window)[0]
    assert torch.allclose(masked, attention.attention(None, q, k, v, torch.ones(1, 1, t, n, dtype=torch.bool))[0])


def test_window_tokens():
    f = _lib.load().tc_decode_window_tokens
    assert f(1000, 100, 0) == 100 and f(1000, 100, 4) == 116 and f(1000, 100, 16) == 116 and f(1000, 100, 17) == 132
    assert f(100, 100, 0) == f(100, 60, 40) == f(100, 1 << 40, 1 << 40) == 100
    assert f(0, 5, 5) == 0
    assert f(10, 0, 0) == f(10, 1, -1) == f(-1, 1, 0) == -_lib.TC_ERR_INVALID_ARGUMENT


def test_entry_refusals():
    lib = _lib.load()
    st = _lib.i64x3(1 << 24, 1 << 20, 128)

    def decode(n=100, window=10, sinks=0, split=64, q=4096, **kw):
        return lib.tc_decode_window_attention(q, st, 8192, st, 12288, st, None, n, window, sinks, 1, 8, 4, kw.get("d", 128),
                                              0, 0.088, split, 4096, kw.get("ws", 1 << 20), 16384, st, None)

    assert decode(window=0) == decode(sinks=-1) == decode(n=-1) == _lib.TC_ERR_INVALID_ARGUMENT
    assert decode(d=64) == _lib.TC_ERR_UNSUPPORTED
    assert decode(ws=100) == _lib.TC_ERR_WORKSPACE
    assert decode(q=4100) == _lib.TC_ERR_ALIGNMENT
    assert decode(q=0) == _lib.TC_ERR_INVALID_ARGUMENT

    def prefill(window=10, sinks=0, q_len=16, n=64, **kw):
        return lib.tc_prefill_window_attention(4096, st, 8192, st, 12288, st, window, sinks, q_len, n, 1,
                                               kw.get("hq", 32), 8, 128, 0, 0.088, 1, None, 0, kw.get("out", 16384), st, None)

    assert prefill(window=0) == prefill(sinks=-1) == prefill(q_len=65) == prefill(out=0) == _lib.TC_ERR_INVALID_ARGUMENT
    assert prefill(hq=24) == _lib.TC_ERR_UNSUPPORTED
    assert prefill(q_len=0) == _lib.TC_OK
    assert lib.tc_prefill_window_num_splits(1, 10, 5, 1, 0, 32, 8) == -_lib.TC_ERR_INVALID_ARGUMENT
    assert lib.tc_prefill_window_num_splits(1, 5, 10, 0, 0, 32, 8) == -_lib.TC_ERR_INVALID_ARGUMENT
    rc = lib.tc_prefill_paged_window_attention(4096, st, 8192, 12288, st, 1 << 12, 4096, 64, 10, 0, 16, 64, 1, 32, 8, 128, 0,
                                               0.088, 1, None, 0, 16384, st, None)
    assert rc == _lib.TC_ERR_UNSUPPORTED and b"2 GiB" in lib.tc_last_error()
    rc = lib.tc_decode_append_window_attention(4096, st, 8192, st, 12288, st, 4096, _lib.i64x2(0, 128), 0, _lib.i64x2(0, 128),
                                               None, 100, 10, 0, 1, 8, 4, 128, 0, 0.088, 64, 4096, 1 << 20, 16384, st, None)
    assert rc == _lib.TC_ERR_INVALID_ARGUMENT


def test_visible_fragments():
    """The tile table of a window holds the sinks' and the window's slots, whatever holes the sequence has."""
    t = PageTable(60, 16, batch=3)
    for _ in range(5):
        for b in (0, 1):
            t.reserve(b, 50)
    t.prune(0, 30, 77, 250 - 77)
    t.reserve(0, 13)
    for window, sinks in ((1, 0), (10, 3), (100, 20), (40, 31), (200, 5), (500, 0), (180, 16)):
        tab, cnt = t.tile_table(window, sinks)
        for b in range(3):
            slots = t.token_slots(b).tolist()
            n = len(slots)
            want = [s for j, s in enumerate(slots) if j >= n - window or j < sinks]
            got = [[p, s + i] for p, s, rows, _ in tab[b, :cnt[b]].tolist() for i in range(rows)]
            assert got == want
