"""Decode over a prefix that all sequences share, against the definition in float64: the contiguous entry point, forked
sequences of a paged cache, and a run of the paged operators together."""
import types

import pytest
import torch

from threadcut_amd import _lib, flash_decode, paged, workloads
from threadcut_amd.match import Split

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5


def rand(seed, shape, dtype, dev):
    return torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def definition(q, k, v):
    """(out, A) in float64 of q [hkv, g, d] on k/v [hkv, n, d]; A is the sum of the weights times |v|."""
    if k.shape[1] == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    w = torch.softmax(torch.bmm(q.double(), k.double().transpose(1, 2).contiguous()) * SCALE, -1)
    return torch.bmm(w, v.double()), torch.bmm(w, v.double().abs())


def close(got, want, spread, columns):
    """Rounded once (eps / 2), the rest in fp32: weights to 2^-16, sums and merges far below 2^-14 of the spread. More
    than 32 query rows a KV head: the prefix's weights are rounded to the type (eps / 2 of each), in the sum over v and
    in the one that divides it."""
    f = torch.finfo(got.dtype)
    bound = f.eps / 2 * want.abs() + 2.0 ** -14 * spread + f.smallest_normal
    if columns > 32:
        bound = bound * (1 + f.eps) + f.eps / 2 * (spread + want.abs())
    off = (got.double() - want).abs()
    assert torch.all(off <= bound), f"worst {(off / bound).max().item():.3g} of the bound"


def check(out, q, kp, vp, k, v, lens):
    for i, n in enumerate(lens):
        close(out[i], *definition(q[i], torch.cat((kp, k[i, :, :n]), 1), torch.cat((vp, v[i, :, :n]), 1)),
              q.shape[0] * q.shape[2])


CASES = [  # batch, kv heads, group, prefix, own tokens (one number: all of them)
    (4, 8, 4, 2000, [200, 1, 57, 16]), (2, 8, 1, 1, [3, 0]), (16, 8, 4, 500, [33] * 16), (3, 8, 8, 4097, [0, 0, 0]),
    (64, 2, 8, 700, list(range(64))), (5, 3, 3, 31, [17, 400, 0, 5, 64]), (1, 8, 4, 1000, [100]), (33, 1, 1, 17, [2] * 33),
    (2, 8, 4, 20000, [1000, 30]), (65, 4, 2, 15, [16] * 65), (8, 8, 2, 16, [300] * 8), (9, 8, 7, 333, [12] * 9),
    (4, 64, 2, 600, [40] * 4), (13, 8, 4, 900, [9] * 13), (17, 4, 8, 2500, [3] * 17), (40, 2, 8, 1200, [0] * 40), (300, 2, 4, 100, [7] * 300), (2, 1, 4, 40000, [100, 100])]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,hkv,g,prefix,lens", CASES)
def test_shared(gpu, dtype, b, hkv, g, prefix, lens):
    print(f"case: {b} x {hkv} heads x {g}, prefix {prefix}, own {lens[:6]}", flush=True)
    n = max(lens)
    kp, vp = (torch.full((1, hkv, prefix + 9, D), float("nan"), dtype=dtype, device=gpu) for _ in range(2))
    k, v = (torch.full((b, hkv, n + 9, D), float("nan"), dtype=dtype, device=gpu) for _ in range(2))
    for i, t in enumerate((kp, vp)):
        t[:, :, :prefix] = rand(i, (1, hkv, prefix, D), dtype, gpu)
    for i, t in enumerate((k, v)):
        for j, m in enumerate(lens):
            t[j, :, :m] = rand(10 + 1000 * i + j, (hkv, m, D), dtype, gpu)
    kp, vp, k, v = kp[:, :, :prefix], vp[:, :, :prefix], k[:, :, :n], v[:, :, :n]
    q = rand(3, (b, hkv, g, D), dtype, gpu)
    t = torch.tensor(lens, dtype=torch.int32, device=gpu)
    out = flash_decode.decode_attention_shared(q, kp, vp, k, v, SCALE, lens=t)
    check(out, q, kp[0], vp[0], k, v, lens)
    if min(lens) == n:  # one length: none to tell, and the prefix as [Hkv, P, D], the output given
        given = torch.empty_like(out)
        assert flash_decode.decode_attention_shared(q, kp[0], vp[0], k, v, SCALE, out=given) is given
        check(given, q, kp[0], vp[0], k, v, lens)


def test_other_strides(gpu):
    """Tokens first, heads of a wider buffer, a transposed query and a strided output."""
    b, hkv, g, prefix, n = 6, 4, 4, 300, 50
    kp, vp = (rand(i, (prefix, hkv + 2, D), torch.float16, gpu)[:, 1:1 + hkv].transpose(0, 1) for i in range(2))
    k, v = (rand(5 + i, (n, b, hkv, D), torch.float16, gpu).permute(1, 2, 0, 3) for i in range(2))
    q = rand(9, (hkv, g, b, D), torch.float16, gpu).permute(2, 0, 1, 3)
    out = torch.zeros(b, hkv, g, 2 * D, dtype=torch.float16, device=gpu)
    flash_decode.decode_attention_shared(q, kp, vp, k, v, SCALE, out=out[..., :D])
    check(out[..., :D], q, kp, vp, k, v, [n] * b)
    assert not out[..., D:].any()


def test_no_prefix_is_the_plain_call(gpu):
    q, k, v = (rand(i, s, torch.float16, gpu) for i, s in enumerate(((3, 8, 4, D), (3, 8, 90, D), (3, 8, 90, D))))
    lens = torch.tensor([90, 0, 5], dtype=torch.int32, device=gpu)
    out = flash_decode.decode_attention_shared(q, k[0, :, :0], v[0, :, :0], k, v, SCALE, lens=lens)
    assert torch.equal(out, flash_decode.decode_attention_batched(q, k, v, SCALE, lens=lens))
    assert not out[1].any()
    empty = flash_decode.decode_attention_shared(q, k[0, :, :0], v[0, :, :0], k[:, :, :0], v[:, :, :0], SCALE)
    assert not empty.any()


def test_extreme_scores(gpu):
    """The prefix's scores far above or below a sequence's own: nothing overflows in the merge."""
    q = rand(1, (4, 2, 4, D), torch.float16, gpu)
    kp, vp = rand(2, (2, 500, D), torch.float16, gpu), rand(3, (2, 500, D), torch.float16, gpu)
    k, v = rand(4, (4, 2, 30, D), torch.float16, gpu), rand(5, (4, 2, 30, D), torch.float16, gpu)
    for scale in (SCALE, 30.0, -30.0, 0.0):
        out = flash_decode.decode_attention_shared(q, kp, vp, k, v, scale)
        for i in range(4):
            s = torch.bmm(q[i].double(), torch.cat((kp, k[i]), 1).double().transpose(1, 2).contiguous()) * scale
            w = torch.softmax(s, -1)
            vv = torch.cat((vp, v[i]), 1).double()
            want, spread = torch.bmm(w, vv), torch.bmm(w, vv.abs())
            # Scores of up to 2000 carry 2^-12 (scale 30), and so do the weights, relative to what they are.
            slack = (2.0 ** -14 if abs(scale) < 1 else 2.0 ** -9) * spread
            assert torch.all((out[i].double() - want).abs() <= 2.0 ** -11 * want.abs() + slack + 1e-7)


def test_captured_and_replayed(gpu):
    b, hkv, g, prefix, n = 12, 8, 4, 1500, 80
    kp, vp = (rand(i, (hkv, prefix, D), torch.float16, gpu) for i in range(2))
    k, v = (rand(5 + i, (b, hkv, n, D), torch.float16, gpu) for i in range(2))
    lens = torch.zeros(b, dtype=torch.int32, device=gpu)
    q = torch.zeros(b, hkv, g, D, dtype=torch.float16, device=gpu)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flash_decode.decode_attention_shared(q, kp, vp, k, v, SCALE, lens=lens, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flash_decode.decode_attention_shared(q, kp, vp, k, v, SCALE, lens=lens, out=out)
    for i in range(4):
        q.copy_(rand(30 + i, q.shape, torch.float16, gpu))
        now = [(7 * i + j) % (n + 1) for j in range(b)]
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(out, q, kp, vp, k, v, now)
        eager = flash_decode.decode_attention_shared(q, kp, vp, k, v, SCALE, lens=lens)
        assert torch.equal(eager, out)


def test_refusals(gpu):
    q, k = rand(1, (2, 2, 4, D), torch.float16, gpu), rand(2, (2, 2, 30, D), torch.float16, gpu)
    p = k[0]
    f = flash_decode.decode_attention_shared
    with pytest.raises(ValueError, match="prefix"):
        f(q, k, k, k, k, SCALE)  # a prefix for each sequence
    with pytest.raises(ValueError, match="prefix"):
        f(q, p[:1], p[:1], k, k, SCALE)
    with pytest.raises(ValueError, match="prefix"):
        f(q, p, p[:, :5], k, k, SCALE)
    with pytest.raises(ValueError, match="prefix"):
        f(q, p.bfloat16(), p.bfloat16(), k, k, SCALE)
    with pytest.raises(ValueError, match="contiguous"):
        f(q, p.transpose(1, 2).contiguous().transpose(1, 2), p, k, k, SCALE)
    with pytest.raises(ValueError, match="lens"):
        f(q, p, p, k, k, SCALE, lens=torch.zeros(2, dtype=torch.int64, device=gpu))
    with pytest.raises(ValueError, match="out"):
        f(q, p, p, k, k, SCALE, out=torch.empty(2, 2, 4, D, device=gpu))
    with pytest.raises(RuntimeError, match="GPU"):
        f(q, p.cpu(), p.cpu(), k, k, SCALE)
    with pytest.raises(RuntimeError, match="not finite"):
        f(q, p, p, k, k, float("nan"))
    with pytest.raises(RuntimeError, match="unsupported"):
        f(rand(1, (2, 2, 9, D), torch.float16, gpu), p, p, k, k, SCALE)


class Forked:
    """A paged cache of two layers whose sequences begin with the same tokens, and every sequence's rows in order."""

    def __init__(self, dev, prefix, lens, page_tokens, dtype=torch.float16, heads=8, cut=None):
        b = len(lens)
        P = page_tokens
        self.cache = paged.PagedKV(2, heads, -(-prefix // P) + b * (-(-(max(lens) + 40) // P) + 1) + 2, P, batch=b,
                                   dtype=dtype, device=dev)
        for t in self.cache.k_pools + self.cache.v_pools:
            t.fill_(float("nan"))
        head = rand(1, (2, 2, heads, prefix, D), dtype, dev)
        self.cache.append(0, list(head[0]), list(head[1]))
        for i in range(1, b):
            self.cache.fork(0, i, cut[i] if cut else None)
        self.rows = []
        for i, n in enumerate(lens):
            own = rand(50 + i, (2, 2, heads, n, D), dtype, dev)
            self.cache.append(i, list(own[0]), list(own[1]))
            self.rows.append(torch.cat((head[:, :, :, :cut[i]] if cut and i else head, own), 3))

    def check(self, out, q, layer):
        for i, r in enumerate(self.rows):
            close(out[i], *definition(q[i], r[0, layer], r[1, layer]), q.shape[0] * q.shape[2])


def few(monkeypatch):
    """Short prefixes are read once too (by default they take the plain call, which is faster there)."""
    monkeypatch.setattr(paged, "SHARED_MIN_ROWS", 2048)
    monkeypatch.setattr(paged, "SHARED_MIN_ROWS_FEW", 2048)


@pytest.fixture(params=["native", "Python"])
def calls(request, monkeypatch):
    """Which decode calls read the prefix once, through either path of the wrappers."""
    _lib.load()
    taken = []
    fast = types.SimpleNamespace(**{n: getattr(_lib.FAST, n) for n in dir(_lib.FAST) if n[0] != "_"})
    shared, attend = fast.paged_shared, paged.PagedKV._attend_shared

    def native(*a):
        done = shared(*a)
        if done is not None:
            taken.append(1)
        return done

    fast.paged_shared = native
    monkeypatch.setattr(_lib, "FAST", fast if request.param == "native" else None)
    few(monkeypatch)
    monkeypatch.setattr(paged.PagedKV, "_attend_shared", lambda self, *a: taken.append(2) or attend(self, *a))
    yield taken
    assert set(taken) == {1 if request.param == "native" else 2}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("prefix,lens,page_tokens,heads,g", [
    (1000, [30, 1, 200], 64, 8, 4), (320, [0, 0], 16, 8, 2), (999, [5] * 20, 32, 2, 8), (2049, [100, 0, 7], 40, 8, 1),
    (5000, [64] * 70, 64, 2, 4)])
def test_forked_sequences(gpu, calls, dtype, prefix, lens, page_tokens, heads, g):
    print(f"case: prefix {prefix}, own {lens[:5]}, pages of {page_tokens}", flush=True)
    f = Forked(gpu, prefix, lens, page_tokens, dtype, heads)
    b = len(lens)
    for layer in range(2):
        q = rand(7 + layer, (b, heads, g, D), dtype, gpu)
        f.check(f.cache.decode(layer, q, SCALE), q, layer)
    for step in range(2):  # steps with the append fused in
        f.cache.reserve_step()
        new = []
        for layer in range(2):
            q, kn, vn = (rand(100 * step + 10 * layer + i, s, dtype, gpu) for i, s in
                         enumerate(((b, heads, g, D), (b, heads, D), (b, heads, 1, D))))
            out = f.cache.decode_append(layer, q, kn, vn, SCALE)
            new.append((kn, vn[:, :, 0], q, out))
        for i in range(b):
            add = torch.stack([torch.stack([new[l][kv][i] for l in range(2)]) for kv in range(2)])
            f.rows[i] = torch.cat((f.rows[i], add[:, :, :, None]), 3)
        for layer in range(2):
            f.check(new[layer][3], new[layer][2], layer)
            for i in range(b):
                gk, gv = f.cache.gather(layer, i)
                assert torch.equal(gk, f.rows[i][0, layer]) and torch.equal(gv, f.rows[i][1, layer])
    assert len(calls) == 6


def test_what_is_shared_changes(gpu, calls):
    """Forks at different lengths, a sequence that leaves, prunes: decode follows the table."""
    f = Forked(gpu, 1000, [30, 10, 20], 64, cut=[1000, 700, 1000])
    q = rand(1, (3, 8, 4, D), torch.float16, gpu)
    f.check(f.cache.decode(0, q, SCALE), q, 0)
    assert len(calls) == 1
    with pytest.raises(RuntimeError, match="share"):
        f.cache.prune(1, Split(10, 300, 200), workloads.inv_freq())
    f.check(f.cache.decode(0, q, SCALE), q, 0)
    # A sequence's own tokens move, and shared ones can be dropped.
    inv = workloads.inv_freq()
    before = f.cache.gather(1, 0)[0]
    f.cache.prune(2, Split(1003, 1010, 5), inv)
    f.cache.prune(1, Split(100, 100, 0), inv)
    k, v = f.cache.gather(0, 2)
    f.rows[2] = torch.stack((torch.stack((k, k)), torch.stack((v, v))))
    f.rows[1] = f.rows[1][:, :, :, :100]
    f.check(f.cache.decode(0, q, SCALE), q, 0)
    assert len(calls) == 2  # the sequences share fewer tokens than pay now
    assert torch.equal(f.cache.gather(1, 0)[0], before)
    f.cache.table.release(1)
    f.cache.table.release(2)
    f.rows[1], f.rows[2] = (r[:, :, :, :0] for r in f.rows[1:])
    f.check(f.cache.decode(0, q, SCALE), q, 0)
    assert not f.cache.table.users
    f.cache.fork(0, 1)
    f.rows[1] = f.rows[0]
    f.check(f.cache.decode(0, q, SCALE), q, 0)
    f.cache.reserve_step()
    with pytest.raises(RuntimeError, match="incomplete"):
        f.cache.fork(0, 2)


@pytest.mark.parametrize("short", [True, False])
def test_the_paged_operators_together(gpu, monkeypatch, short):
    """A prompt, forks of it, a chunk of new tokens and decode steps, keys and queries rotated on the way, with and
    without a window: against float64 from the rows as they were handed over."""
    if short:
        few(monkeypatch)
    b, heads, g, prefix, chunk = 3, 8, 4, 700, 40
    inv = workloads.inv_freq().to(gpu)
    cache = paged.PagedKV(2, heads, 60, 64, batch=b, device=gpu)
    head = rand(1, (2, 2, 1, heads, prefix, D), torch.float16, gpu)
    cache.append(0, list(head[0]), list(head[1]), inv_freq=inv)
    for i in range(1, b):
        cache.fork(0, i)
    keys = [[head[0, l, 0]] * b for l in range(2)]
    values = [[head[1, l, 0]] * b for l in range(2)]

    def turned(x, start):  # rotated in float64, rounded as the cache and the kernel's query are
        z = torch.complex(x[..., :64].double(), x[..., 64:].double())
        pos = start + torch.arange(x.shape[-2], dtype=torch.float64, device=gpu)
        z = z * torch.polar(torch.ones((), dtype=torch.float64, device=gpu), torch.outer(pos, inv.double()))
        return torch.cat((z.real, z.imag), -1).half()

    n = prefix
    for t in (chunk, 1, 1):
        cache.reserve_step(t)
        for l in range(2):
            k, v, q = (rand(100 * n + 10 * l + i, (b, t, h, D), torch.float16, gpu).transpose(1, 2)
                       for i, h in enumerate((heads, heads, heads * g)))
            q2 = cache.write_step(l, k, v, inv_freq=inv, query=q)
            for i in range(b):
                keys[l] = keys[l][:i] + [torch.cat((keys[l][i], k[i]), 1)] + keys[l][i + 1:]
                values[l] = values[l][:i] + [torch.cat((values[l][i], v[i]), 1)] + values[l][i + 1:]
            for window, sinks in ((None, 0), (100, 4)):
                if t > 1:
                    out = cache.prefill(l, q2, SCALE, causal=True, window=window, sink_tokens=sinks).transpose(1, 2)
                else:
                    out = cache.decode(l, q2.reshape(b, heads, g, D), SCALE, window=window, sink_tokens=sinks)
                    out = out.reshape(b, heads * g, 1, D)
                for i in range(b):
                    kk = turned(keys[l][i], 0).repeat_interleave(g, 0)
                    vv = values[l][i].repeat_interleave(g, 0).double()
                    p = n + torch.arange(t, device=gpu)[:, None]
                    j = torch.arange(n + t, device=gpu)
                    hidden = (j > p) | ((j <= p - window) & (j >= sinks)) if window else j > p
                    s = torch.bmm(turned(q[i], n).double(), kk.double().transpose(1, 2).contiguous()) * SCALE
                    w = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
                    want, spread = torch.bmm(w, vv), torch.bmm(w, vv.abs())
                    # Keys and queries rounded to the neighbour where float64 and fp32 straddle a border: a step of
                    # 2^-11 in a few of 128 dims, 2^-11 * |q| |k| / sqrt(d) at most in a score; prefill's weights.
                    off = (out[i].double() - want).abs()
                    assert torch.all(off <= 2.0 ** -11 * want.abs() + (2.0 ** -10 if t > 1 else 2.0 ** -11) * spread + 1e-7)
        n += t


def test_fork_on_another_stream(gpu, monkeypatch):
    few(monkeypatch)
    f = Forked(gpu, 600, [10, 20], 64)
    q = rand(1, (2, 8, 4, D), torch.float16, gpu)
    first = f.cache.decode(0, q, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = f.cache.decode(0, q, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    f.check(first, q, 0)


def test_bad_tiles_count_as_empty(gpu):
    """Entries outside the pool or the page, and of more than 16 rows, read nothing."""
    heads, g, P = 2, 4, 32
    pool = rand(1, (4, heads, P, D), torch.float16, gpu)
    vpool = rand(2, (4, heads, P, D), torch.float16, gpu)
    table = torch.tensor([[0, 0, 16, 0], [4, 0, 16, 0], [-1, 0, 16, 0], [1, 20, 13, 0], [1, -1, 5, 0], [2, 3, 17, 0],
                          [3, 16, 16, 0], [2, 5, -2, 0], [1 << 30, 0, 1, 0], [2, 31, 1, 0]], dtype=torch.int32, device=gpu)
    q = rand(3, (3, heads, g, D), torch.float16, gpu)
    out = torch.empty_like(q)
    lib = _lib.load()
    s = lib.tc_decode_shared_num_splits(3, heads, g, 160, 0, 1)
    ws = torch.empty(lib.tc_decode_workspace_bytes(3, heads, g, D, s), dtype=torch.uint8, device=gpu)
    _lib.check(lib.tc_decode_paged_shared_attention(
        q.data_ptr(), _lib.i64x3(*q.stride()[:3]), pool.data_ptr(), vpool.data_ptr(), _lib.i64x3(*pool.stride()[:3]), 4, P,
        table.data_ptr(), 10, None, None, 0, None, None, None, None, 3, heads, g, D, 0, SCALE, ws.data_ptr(), ws.numel(),
        out.data_ptr(), _lib.i64x3(*out.stride()[:3]), _lib.stream_of(gpu)), "shared")
    k = torch.cat((pool[0, :, :16], pool[3, :, 16:], pool[2, :, 31:]), 1)
    v = torch.cat((vpool[0, :, :16], vpool[3, :, 16:], vpool[2, :, 31:]), 1)
    for i in range(3):
        close(out[i], *definition(q[i], k, v), 12)


def test_what_pays(gpu):
    """By default short prefixes, and few sequences, take the plain call."""
    x = torch.zeros(8, 2100, D, dtype=torch.float16, device=gpu)
    for b, prefix, group, pays in ((2, 2100, 4, False), (4, 2100, 4, True), (4, 1000, 4, False), (4, 2100, 8, False),
                                   (8, 2100, 4, False), (9, 2100, 4, True), (8, 900, 2, True), (17, 1100, 4, True),
                                   (3, 2100, 16, False)):
        c = paged.PagedKV(1, 8, 34, 64, batch=b, device=gpu)
        c.append(0, [x[:, :prefix]], [x[:, :prefix]])
        assert c.shared_tables(group) is None
        for i in range(1, b):
            c.fork(0, i)
        assert (c.shared_tables(group) is not None) == pays, (b, prefix, group)


@pytest.mark.parametrize("window", [None, 300])
def test_paged_calls_captured_and_replayed(gpu, monkeypatch, window):
    """Forked and windowed decode of pages in a graph, after an eager call (which uploads the tables): every replay
    against the eager call on the same queries, with eager calls between them."""
    few(monkeypatch)
    b, heads, g = 4, 8, 4
    c = paged.PagedKV(1, heads, 60, 64, batch=b, device=gpu)
    x = rand(1, (heads, 900, D), torch.float16, gpu)
    c.append(0, [x], [x])
    for i in range(1, b):
        c.fork(0, i)
        c.append(i, [x[:, :30 * i]], [x[:, 5:5 + 30 * i]])
    q = rand(2, (b, heads, g, D), torch.float16, gpu)
    c.decode(0, q, SCALE, window=window)
    assert (c.shared_tables(g) is not None)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = c.decode(0, q, SCALE, window=window)
    for seed in range(3, 7):
        q.copy_(rand(seed, q.shape, q.dtype, gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.decode(0, q, SCALE, window=window))


def test_no_query_heads(gpu, monkeypatch):
    few(monkeypatch)
    c = paged.PagedKV(1, 8, 40, 64, batch=3, device=gpu)
    x = torch.zeros(8, 600, D, dtype=torch.float16, device=gpu)
    c.append(0, [x], [x])
    for i in (1, 2):
        c.fork(0, i)
    with pytest.raises((ValueError, RuntimeError)):
        c.decode(0, x.new_empty(3, 8, 0, D), SCALE)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,hkv,g,prefix,most", [(300, 1, 5, 700, 33), (43, 3, 8, 1234, 400), (130, 8, 1, 5, 16), (128, 8, 1, 3000, 0)])
def test_many_rows(gpu, dtype, b, hkv, g, prefix, most):
    """1024 rows and more, which another kernel joins: rows that do not fill a work-group, sequences without own tokens,
    outputs whose heads are not next to each other, their neighbours left as they were."""
    lens = [(7 * i) % (most + 1) for i in range(b)]
    kp, vp = (rand(i, (hkv, prefix, D), dtype, gpu) for i in range(2))
    k, v = (rand(5 + i, (b, hkv, most, D), dtype, gpu) for i in range(2))
    q = rand(3, (b, hkv, g, D), dtype, gpu)
    t = torch.tensor(lens, dtype=torch.int32, device=gpu)
    buf = torch.full((b, g, hkv + 1, D + 8), 7.0, dtype=dtype, device=gpu)
    out = buf[:, :, :hkv, :D].transpose(1, 2)
    assert flash_decode.decode_attention_shared(q, kp, vp, k, v, SCALE, lens=t, out=out) is out
    check(out, q, kp, vp, k, v, lens)
    buf[:, :, :hkv, :D] = 7.0
    assert torch.all(buf == 7.0)
