"""Pages shared by several sequences (PageTable.fork) against a brute-force model, and the argument checks of rotated
appends, on the CPU."""
import ctypes
import random

import numpy as np
import pytest

from threadcut_amd import _lib
from threadcut_amd.paged import PageTable, _placed


def check(t, model):
    """Every sequence reads its own tokens, whatever the others wrote since: model[b] is its list of token names, and
    `written` what each slot holds."""
    for b, tokens in enumerate(model["tokens"]):
        got = [model["written"][tuple(x)] for x in t.token_slots(b).tolist()]
        assert got == tokens
    users = {}
    for b in range(t.batch):
        for p in set(t.frags[b][:, 0].tolist()):
            users[p] = users.get(p, 0) + 1
    assert sorted(t.free) == sorted(set(range(t.num_pages)) - set(users))
    assert len(set(t.free)) == len(t.free)
    assert t.users == {p: n for p, n in users.items() if n > 1}


@pytest.mark.parametrize("page_tokens", [16, 40, 64])
@pytest.mark.parametrize("seed", range(8))
def test_forks_match_brute_force(seed, page_tokens):
    rnd = random.Random(seed)
    t = PageTable(300, page_tokens, batch=5)
    model = {"tokens": [[] for _ in range(5)], "written": {}}
    name = 0
    for _ in range(150):
        b = rnd.randrange(5)
        tokens = model["tokens"][b]
        what = rnd.random()
        if what < 0.45:
            n = rnd.choice([1, 1, 5, 16, 30, rnd.randint(1, 150)])
            if t.pages_needed(b, n) > len(t.free):
                with pytest.raises(RuntimeError, match="pages needed"):
                    t.reserve(b, n)
                continue
            free = len(t.free)
            need = t.pages_needed(b, n)
            for slot in t.reserve(b, n).tolist():
                model["written"][tuple(slot)] = name  # a slot that another sequence reads would change its token
                tokens.append(name)
                name += 1
            assert free - len(t.free) == need
        elif what < 0.7:
            src = rnd.randrange(5)
            n = rnd.randint(0, len(model["tokens"][src]))
            if src == b or tokens:
                with pytest.raises(ValueError, match="empty"):
                    t.fork(src, b, n)
                continue
            t.fork(src, b, n)
            model["tokens"][b] = model["tokens"][src][:n]
        elif what < 0.88:
            a = rnd.randint(0, len(tokens))
            c0 = rnd.randint(a, len(tokens))
            c = rnd.randint(0, len(tokens) - c0)
            t.prune(b, a, c0, c)
            model["tokens"][b] = tokens[:a] + tokens[c0:c0 + c]
        else:
            t.release(b)
            model["tokens"][b] = []
        check(t, model)
    for b in range(5):
        t.release(b)
    assert len(t.free) == 300 and not t.users


def test_fork_refusals():
    t = PageTable(8, 16, batch=3)
    t.reserve(0, 20)
    for src, dst, n, match in ((0, 0, 5, "empty"), (0, 1, 21, "21 tokens"), (0, 1, -1, "tokens")):
        with pytest.raises(ValueError, match=match):
            t.fork(src, dst, n)
    t.fork(0, 1, 0)  # nothing shared
    assert t.length(1) == 0 and not t.users
    t.fork(0, 1, 20)
    with pytest.raises(ValueError, match="empty"):
        t.fork(0, 1, 20)
    assert t.reserve(0, 1).tolist() == [[2, 0]]  # neither writes behind the other's last token
    assert t.reserve(1, 1).tolist() == [[3, 0]]


def test_rotated_append_validation():
    lib = _lib.load()
    st = _lib.i64x3(0, 1 << 20, 128)
    p, f = _lib.ptr_array([4096]), (ctypes.c_float * 64)()
    pool = _lib.i64x3(8 * 16 * 128, 16 * 128, 128)

    def rope(k=p, ks=st, slots=4096, pages=4, P=16, q=None, qs=None, qo=None, hq=0, host=f, dev=None, layers=1, b=1, h=8,
             rows=3, d=128, dt=0, ps=pool):
        return lib.tc_paged_append_rope(k, ks, p, st, p, p, ps, pages, P, slots, q, qs, qo, qs, hq, host, dev, layers,
                                        b, h, rows, d, dt, None)

    assert rope(slots=None) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(slots=4104) == _lib.TC_ERR_ALIGNMENT
    assert rope(pages=0) == rope(P=0) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(host=None) == _lib.TC_ERR_INVALID_ARGUMENT and b"frequencies" in lib.tc_last_error()
    assert rope(dev=4096) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(host=None, dev=4098) == _lib.TC_ERR_ALIGNMENT
    assert rope(k=_lib.ptr_array([0])) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(k=_lib.ptr_array([4100])) == _lib.TC_ERR_ALIGNMENT
    assert rope(ks=_lib.i64x3(0, 1 << 20, 130)) == _lib.TC_ERR_ALIGNMENT
    assert rope(ps=_lib.i64x3(0, 0, 64)) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(hq=8) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(hq=8, q=p, qs=st, qo=_lib.ptr_array([0])) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(d=64) == rope(dt=5) == _lib.TC_ERR_UNSUPPORTED
    assert rope(b=0) == rope(layers=-1) == rope(rows=-1) == _lib.TC_ERR_INVALID_ARGUMENT
    assert rope(rows=1 << 30, b=4) == _lib.TC_ERR_UNSUPPORTED
    assert rope(h=40000) == _lib.TC_ERR_UNSUPPORTED
    assert rope(rows=0, slots=None, host=None) == rope(layers=0, slots=None) == _lib.TC_OK
    assert _placed([[4, 1], [5, 0]], 7).tolist() == [[4, 1, 7, 0], [5, 0, 8, 0]]


def test_shared_fragments():
    t = PageTable(40, 16, batch=3)
    t.reserve(0, 70)
    t.fork(0, 1, 70)
    t.fork(0, 2, 40)
    t.reserve(2, 5)
    assert t.shared_frags() == 2  # the third page has 16 tokens in two sequences, 8 in the third
    t.release(2)
    assert t.shared_frags() == 0
    t.fork(1, 2, 70)
    assert t.shared_frags() == 5
    whole, counts = t.tile_table()
    own, none = t.tile_table(skip=5)
    assert own.shape == (3, 0, 4) and none.tolist() == [0, 0, 0]
    for b, n in enumerate((1, 20, 33)):
        t.reserve(b, n)
    assert t.shared_frags() == 5
    head, _ = t.tile_table()
    own, mine = t.tile_table(skip=5)
    assert mine.tolist() == [1, 2, 3]
    for b in range(3):
        assert head[b, :5].tolist() == whole[b, :5].tolist()
        assert own[b, :mine[b]].tolist() == head[b, 5:5 + mine[b]].tolist()
    assert PageTable(4, 16).shared_frags() == 0


def test_table_refusals():
    f = _lib.load().tc_page_table
    frags = np.array([[3, 0, 10], [5, 4, 30]], dtype=np.int64)
    args = np.array([frags.__array_interface__["data"][0], 2], dtype=np.int64)
    base = args.__array_interface__["data"][0]
    tab, cnt = np.zeros((1, 4, 4), dtype=np.int32), np.zeros(1, dtype=np.int32)
    ptr = lambda a: a.__array_interface__["data"][0]
    call = lambda P=64, first=0, w=0, s=0, t=None, pitch=0, c=None, b=1: f(base, base + 8, b, P, first, w, s, t, pitch, c)
    # Token 5 of 40 (slot 5 of page 3) and token 20 (slot 14 of page 5) begin a tile of their own behind the sinks'.
    assert call() == 4 and call(w=1) == 1 and call(w=35, s=2) == 5 and call(w=20, s=1) == 4
    assert call(P=32) == call(first=-1) == call(w=-1) == call(s=-1) == call(b=0) == -_lib.TC_ERR_INVALID_ARGUMENT
    assert call(t=ptr(tab), pitch=3) == -_lib.TC_ERR_INVALID_ARGUMENT  # no counts
    assert call(t=ptr(tab), pitch=3, c=ptr(cnt)) == -_lib.TC_ERR_INVALID_ARGUMENT  # four tiles
    assert call(w=20, s=1, t=ptr(tab), pitch=4, c=ptr(cnt)) == 4
    assert cnt.tolist() == [4] and tab[0].tolist() == [[3, 0, 1, 0], [5, 14, 2, 20], [5, 16, 16, 22], [5, 32, 2, 38]]


def test_shared_entry_refusals():
    lib = _lib.load()
    st = _lib.i64x3(1 << 24, 1 << 20, 128)
    s2 = _lib.i64x2(1 << 20, 128)

    def shared(prefix=100, n=0, d=128, g=4, q=4096, kp=8192, ps=s2):
        return lib.tc_decode_shared_attention(q, st, kp, ps, 12288, s2, prefix, 4096, st, 4096, st, None, n, 2, 8, g, d, 0,
                                              0.088, 4096, 1 << 20, 16384, st, None)

    assert shared(prefix=-1) == shared(n=-1) == _lib.TC_ERR_INVALID_ARGUMENT
    assert shared(d=64) == shared(g=9) == _lib.TC_ERR_UNSUPPORTED
    assert lib.tc_decode_shared_num_splits(0, 8, 4, 100, 0, 0) == -_lib.TC_ERR_INVALID_ARGUMENT
    assert lib.tc_decode_shared_num_splits(2, 8, 4, 1 << 40, 0, 0) == -_lib.TC_ERR_INVALID_ARGUMENT

    def pages(pages=4, P=16, table=4096, tiles=3, own=4096, max_tiles=2, kn=None, vn=None):
        return lib.tc_decode_paged_shared_attention(4096, st, 8192, 12288, st, pages, P, table, tiles, own, own, max_tiles,
                                                    kn, s2, vn, s2, 2, 8, 4, 128, 0, 0.088, 4096, 1 << 20, 16384, st, None)

    assert pages(pages=0) == pages(P=0) == pages(table=None) == pages(own=None) == _lib.TC_ERR_INVALID_ARGUMENT
    assert pages(tiles=-1) == pages(max_tiles=-1) == pages(max_tiles=1 << 28) == _lib.TC_ERR_INVALID_ARGUMENT
    assert pages(table=4104) == pages(own=4104) == _lib.TC_ERR_ALIGNMENT
    assert pages(kn=4096) == pages(kn=4096, vn=4096, max_tiles=0) == _lib.TC_ERR_INVALID_ARGUMENT
    assert pages(kn=4100, vn=4096) == _lib.TC_ERR_ALIGNMENT


@pytest.mark.parametrize("n", [1, 3, 16, 40])
def test_a_step_reserves_what_each_sequence_would(n):
    """reserve_all against reserve on an equal table, from empty sequences, shared and full last pages on."""
    tables = [PageTable(300, 16, 4) for _ in range(2)]
    for t in tables:
        t.reserve(0, 33)
        t.fork(0, 1, 33)
        t.reserve(2, 32)
    for step in range(12):
        a, b = tables
        if step == 5:
            for t in tables:
                t.release(1)
        starts = [a.length(i) for i in range(4)]
        rows = a.reserve_all(n)
        assert rows.dtype == np.int32 and rows.shape == (4, n, 4)
        for i in range(4):
            assert np.array_equal(rows[i, :, :2], b.reserve(i, n))
            assert rows[i, :, 2].tolist() == list(range(starts[i], starts[i] + n)) and not rows[i, :, 3].any()
            assert a.length(i) == b.length(i) == starts[i] + n == int(a.frags[i][:, 2].sum())
            assert np.array_equal(a.frags[i], b.frags[i])
        assert a.free == b.free and a.users == b.users
        if step % 3 == 2:  # the last token goes again
            for t in tables:
                for i in range(4):
                    t.prune(i, t.length(i) - 1, t.length(i), 0)
    short = PageTable(4, 16, 2)
    short.reserve(0, 16)
    with pytest.raises(RuntimeError, match="pages needed"):
        short.reserve_all(33)
    assert short.length(0) == 16 and short.length(1) == 0 and len(short.free) == 3
