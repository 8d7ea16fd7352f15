"""Rotated appends into a paged cache (tc_paged_append_rope): the keys and queries of new tokens are rotated to their
positions on the way, against the rotation in float64; values are copied bit for bit, and nothing else of the pools
changes."""
import types

import pytest
import torch

from threadcut_amd import _lib, paged, workloads
from threadcut_amd.match import Split

pytestmark = pytest.mark.gpu

D = 128


def rand(seed, shape, dtype, dev):
    return torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def turned(x, start, inv_freq):
    """x [heads, n, 128] at positions start .. in float64, from the complex form of the rotation."""
    x = x.double()
    pos = start + torch.arange(x.shape[1], dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       torch.outer(pos, inv_freq.to(x.device).double()))
    z = torch.complex(x[..., :64], x[..., 64:]) * turn
    return torch.cat((z.real, z.imag), -1)


def close(got, x, start, inv_freq):
    """A rotated row is rounded once to its type (half a step of eps, half a subnormal step for fp16), after cos, sin,
    two products and a sum in fp32: sin and cos within 4 steps of 2^-24 of the angle's (whose part of a turn carries
    2^-25 turns, another 4), each product and the sum within one of 2^-24, so 16 steps of |lo| + |hi|."""
    want = turned(x, start, inv_freq)
    f = torch.finfo(got.dtype)
    both = (x[..., :64].double().abs() + x[..., 64:].double().abs()).repeat(1, 1, 2)
    slack = 16 * 2.0 ** -24 * both
    bound = (want.abs() + slack) * f.eps / 2 + slack + f.smallest_normal * f.eps / 2
    off = (got.double() - want).abs()
    assert torch.all(off <= bound), f"worst {(off / bound).max().item():.3g} of the bound"


def forms(form, seed, b, h, n, dtype, dev):
    if form == "heads first":
        return rand(seed, (b, h, n, D), dtype, dev)
    if form == "tokens first":
        return rand(seed, (b, n, h, D), dtype, dev).transpose(1, 2)
    if form == "fused qkv":
        return rand(seed, (b, n, h + 3, D), dtype, dev)[:, :, 2:2 + h].transpose(1, 2)
    if form == "misaligned":
        return rand(seed, (b, h, n, D + 4), dtype, dev)[..., 3:131]
    raise ValueError(form)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["heads first", "tokens first", "fused qkv", "misaligned"])
@pytest.mark.parametrize("heads,before,n,page_tokens,layers", [
    (8, 0, 1, 16, 1), (8, 37, 100, 64, 2), (3, 5, 33, 40, 1), (1, 100, 32, 32, 3), (17, 63, 65, 64, 1), (8, 9, 700, 64, 49)])
def test_append(gpu, dtype, form, heads, before, n, page_tokens, layers):
    print(f"case: {heads} heads, {before} + {n} tokens, pages of {page_tokens}, {layers} layers, {form}", flush=True)
    inv = workloads.inv_freq()
    cache = paged.PagedKV(layers, heads, -(-(before + n) // page_tokens) + 2, page_tokens, dtype=dtype, device=gpu)
    for t in cache.k_pools + cache.v_pools:
        t.fill_(7.0)
    old = rand(1, (heads, before, D), dtype, gpu)
    cache.append(0, [old] * layers, [-old] * layers)
    wk, wv = [t.clone() for t in cache.k_pools], [t.clone() for t in cache.v_pools]
    ks = [forms(form, 10 + i, 1, heads, n, dtype, gpu) for i in range(layers)]
    vs = [forms(form, 100 + i, 1, heads, n, dtype, gpu) for i in range(layers)]
    # A cache's rows of [Hkv, n, D] are taken too; the frequencies from the host or the GPU.
    cache.append(0, [t[0] for t in ks] if layers == 2 else ks, vs, inv_freq=inv.to(gpu) if before % 2 else inv)
    slots = torch.from_numpy(cache.table.token_slots(0)[before:]).to(gpu)
    for i in range(layers):
        close(cache.k_pools[i][slots[:, 0], :, slots[:, 1]].transpose(0, 1), ks[i][0], before, inv)
        wk[i][slots[:, 0], :, slots[:, 1]] = cache.k_pools[i][slots[:, 0], :, slots[:, 1]]
        wv[i][slots[:, 0], :, slots[:, 1]] = vs[i][0].transpose(0, 1)
        assert torch.equal(cache.k_pools[i], wk[i]) and torch.equal(cache.v_pools[i], wv[i])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_heads,heads,n", [(32, 8, 1), (9, 3, 1), (8, 8, 21), (64, 8, 3)])
def test_step(gpu, dtype, q_heads, heads, n):
    """Sequences of different lengths, one of them empty: each token at its own position, queries too."""
    print(f"case: {q_heads} over {heads} heads, {n} tokens", flush=True)
    inv = workloads.inv_freq().to(gpu)
    lens = [0, 16, 333]
    cache = paged.PagedKV(2, heads, 40, 16, batch=3, dtype=dtype, device=gpu)
    for b, m in enumerate(lens):
        old = rand(b, (heads, m, D), dtype, gpu)
        cache.append(b, [old] * 2, [old] * 2)
    cache.reserve_step(n)
    assert [cache.length(b) for b in range(3)] == [m + n for m in lens]
    for layer in range(2):
        k, v = (forms("tokens first", 10 * layer + i, 3, heads, n, dtype, gpu) for i in range(2))
        q = forms("fused qkv", 50 + layer, 3, q_heads, n, dtype, gpu)
        before = q.clone()
        out = cache.write_step(layer, k, v, inv_freq=inv, query=q)
        assert out.shape == q.shape and torch.equal(q, before)
        for b, m in enumerate(lens):
            close(out[b], q[b], m, inv)
            gk, gv = cache.gather(layer, b)
            close(gk[:, m:], k[b], m, inv)
            assert torch.equal(gv[:, m:], v[b])
            assert torch.equal(gk[:, :m], rand(b, (heads, m, D), dtype, gpu))
    cache.reserve_step()  # the step is complete
    cache.cancel_step()
    assert cache.length(2) == 333 + n


def test_steps_of_several_tokens_are_cancelled_whole(gpu):
    cache = paged.PagedKV(2, 2, 9, 16, batch=2, device=gpu)
    x = rand(1, (2, 2, 20, D), torch.float16, gpu)
    cache.append(0, [x[:1]] * 2, [x[:1]] * 2)
    cache.reserve_step(20)
    cache.write_step(0, x, -x)
    with pytest.raises(RuntimeError, match="20 tokens a sequence"):
        cache.decode_append(1, x[:, :, :1], x[:, :, 0], x[:, :, 0], 1.0)
    with pytest.raises(RuntimeError, match="incomplete"):
        cache.decode(1, x[:, :, :1], 1.0)
    gk, gv = cache.gather(0, 1)  # rows that are not rotated arrive bit for bit
    assert torch.equal(gk, x[1]) and torch.equal(gv, -x[1])
    cache.cancel_step()
    assert [cache.length(b) for b in range(2)] == [20, 0]
    with pytest.raises(RuntimeError, match="pages needed"):
        cache.reserve_step(100)
    assert [cache.length(b) for b in range(2)] == [20, 0] and len(cache.table.free) == 7


def test_far_positions(gpu):
    """A product in 32 bits would be off by up to 0.06 rad here."""
    inv = workloads.inv_freq()
    n, start = 64, 1_999_990
    x = rand(3, (1, 1, n, D), torch.float16, gpu)
    out = torch.empty_like(x)
    pool = torch.zeros(1, 1, n, D, dtype=torch.float16, device=gpu)
    vpool = torch.zeros_like(pool)
    slots = torch.zeros(1, n, 4, dtype=torch.int32, device=gpu)
    slots[0, :, 1] = torch.arange(n)
    slots[0, :, 2] = start + torch.arange(n)
    slots[0, 5, 0], slots[0, 6, 1], slots[0, 7, 0] = 1, n, -1  # outside the pool: skipped, the query all the same
    st = _lib.i64x3(n * D, n * D, D)
    p = lambda t: _lib.ptr_array([t.data_ptr()])
    _lib.check(_lib.load().tc_paged_append_rope(
        p(x), st, p(x), st, p(pool), p(vpool), st, 1, n, slots.data_ptr(), p(x), st, p(out), st, 1,
        _lib.float_array(inv), None, 1, 1, 1, n, D, 0, _lib.stream_of(gpu)), "tc_paged_append_rope")
    close(out[0], x[0], start, inv)
    want, copied = out[0, 0].clone(), x[0, 0].clone()
    want[5:8], copied[5:8] = 0, 0
    assert torch.equal(pool[0, 0], want) and torch.equal(vpool[0, 0], copied)


def test_torch_rotates_what_autograd_tracks(gpu):
    """A query that requires a gradient is rotated by torch operations: the gradient is the rotation back."""
    inv = workloads.inv_freq().to(gpu)
    cache = paged.PagedKV(1, 2, 4, 16, device=gpu)
    x = rand(1, (1, 2, 5, D), torch.float16, gpu)
    cache.append(0, [x], [x])
    cache.reserve_step(5)
    q = rand(2, (1, 4, 5, D), torch.float16, gpu).requires_grad_()
    out = cache.write_step(0, x, x, inv_freq=inv, query=q)
    close(out.detach()[0], q.detach()[0], 5, inv)
    w = rand(3, out.shape, torch.float16, gpu)
    out.backward(w)
    back = torch.complex(w.double()[..., :64], w.double()[..., 64:])
    angle = torch.outer(5 + torch.arange(5, device=gpu).double(), inv.double())
    back = back * torch.polar(torch.ones_like(angle), -angle)
    want = torch.cat((back.real, back.imag), -1)[0]
    assert (q.grad[0].double() - want).abs().max() <= 2.0 ** -11 * 8 + 1e-5  # |w| < 8, half a step


def test_kernel_takes_the_usual_rows(gpu, monkeypatch):
    """Which calls the kernel serves: torch's fallback gives the same rows, so only the count tells."""
    _lib.load()
    native = _lib.FAST.rope_rows
    monkeypatch.setattr(_lib, "FAST", None)
    taken, write = [], paged.PagedKV._write_rotated
    monkeypatch.setattr(paged.PagedKV, "_write_rotated", lambda *a: taken.append(write(*a)) or taken[-1])
    inv = workloads.inv_freq()
    cache = paged.PagedKV(2, 2, 9, 16, device=gpu)
    for form in ("heads first", "tokens first", "fused qkv", "misaligned"):
        x = forms(form, 1, 1, 2, 7, torch.float16, gpu)
        cache.append(0, [x] * 2, [x] * 2, inv_freq=inv)
    cache.append(0, [x.float()] * 2, [x] * 2, inv_freq=inv)
    assert taken == [True, True, True, False, False]
    del taken[:]
    monkeypatch.setattr(paged.PagedKV, "_write_rotated", write)
    monkeypatch.setattr(_lib, "FAST", types.SimpleNamespace(rope_rows=lambda *a: taken.append(native(*a)) or taken[-1]))
    inv = inv.to(gpu)
    x = forms("tokens first", 1, 1, 2, 7, torch.float16, gpu)
    bad = forms("misaligned", 1, 1, 2, 7, torch.float16, gpu)
    for k, f in ((x, inv), (x[0], inv), (bad, inv), (x.float(), inv), (x, inv.cpu()), (x, inv.double())):
        cache.append(0, [k] * 2, [x] * 2, inv_freq=f)
        cache.table.prune(0, 20, cache.length(), 0)
    assert taken == [True, True, None, None, None, None]
    cache.append(0, [x, x.transpose(1, 2).contiguous().transpose(1, 2)], [x] * 2, inv_freq=inv)  # strides that differ
    assert taken[-1] is None or x.transpose(1, 2).is_contiguous()


def test_rotation_and_prune_agree(gpu):
    """Rows rotated on the way in and moved by a prune are where they would have been put (one more rounding)."""
    inv = workloads.inv_freq()
    x = rand(1, (1, 4, 200, D), torch.float16, gpu)
    a, b = (paged.PagedKV(1, 4, 8, 32, device=gpu) for _ in range(2))
    a.append(0, [x], [x], inv_freq=inv)
    a.prune(0, Split(20, 70, 130), inv)
    kept = torch.cat((x[:, :, :20], x[:, :, 70:]), 2)
    b.append(0, [kept], [kept], inv_freq=inv)
    (ka, va), (kb, vb) = a.gather(0), b.gather(0)
    assert torch.equal(va, vb)
    size = 2 * x.float().abs().max().item()
    # Two roundings and one, of values up to |lo| + |hi|; the prune's angle in 32 bits: 70 rad * 2^-23.
    assert (ka.float() - kb.float()).abs().max().item() <= size * (3 * 2.0 ** -11 + 70 * 2.0 ** -22)


def test_other_stream_and_device_tables(gpu):
    """A step written on another stream than the one it was reserved on."""
    inv = workloads.inv_freq().to(gpu)
    cache = paged.PagedKV(2, 2, 9, 16, batch=2, device=gpu)
    x = rand(1, (2, 2, 3, D), torch.float16, gpu)
    cache.reserve_step(3)
    cache.write_step(0, x, x, inv_freq=inv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = cache.write_step(1, x, x, inv_freq=inv, query=x)
    torch.cuda.current_stream().wait_stream(side)
    for layer in range(2):
        for b in range(2):
            close(cache.gather(layer, b)[0], x[b], 0, inv)
            close(out[b], x[b], 0, inv)


def test_refusals(gpu):
    inv = workloads.inv_freq()
    cache = paged.PagedKV(1, 2, 9, 16, batch=2, device=gpu)
    x = rand(1, (2, 2, 1, D), torch.float16, gpu)
    with pytest.raises(ValueError, match="inv_freq"):
        cache.append(0, [x[:1]], [x[:1]], inv_freq=inv[:10])
    assert cache.length(0) == 0
    with pytest.raises(ValueError, match="0 tokens"):
        cache.reserve_step(0)
    cache.reserve_step()
    for kw, match in ((dict(inv_freq=inv.long()), "inv_freq"), (dict(query=x), "missing"),
                      (dict(inv_freq=inv, query=x[:1]), "query"), (dict(inv_freq=inv, query=x.float()), "query"),
                      (dict(inv_freq=inv, query=x.cpu()), "query")):
        with pytest.raises(ValueError, match=match):
            cache.write_step(0, x, x, **kw)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="not captured"):
            cache.write_step(0, x, x, inv_freq=inv)
    assert cache.write_step(0, x, x, inv_freq=inv) is None
    assert y is not None


def test_step_without_native_paths(gpu, monkeypatch):
    """The same rows without _fast.so."""
    _lib.load()
    inv = workloads.inv_freq().to(gpu)
    got = []
    for fast in (_lib.FAST, None):
        monkeypatch.setattr(_lib, "FAST", fast)
        cache = paged.PagedKV(1, 8, 20, 16, batch=2, device=gpu)
        x, q = rand(1, (2, 8, 1, D), torch.float16, gpu), rand(2, (2, 32, 1, D), torch.float16, gpu)
        cache.append(1, [x[:1]], [x[:1]])
        cache.reserve_step()
        got.append((cache.write_step(0, x, x, inv_freq=inv, query=q), cache.k_pools[0], cache.v_pools[0]))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_rows_that_do_not_fit_change_nothing(gpu):
    inv = workloads.inv_freq().to(gpu)
    cache = paged.PagedKV(2, 2, 9, 16, device=gpu)
    x, y = rand(1, (1, 2, 20, D), torch.float16, gpu), rand(1, (1, 2, 19, D), torch.float16, gpu)
    cache.append(0, [x] * 2, [x] * 2, inv_freq=inv)
    table, pools = cache.table.frags[0].copy(), [t.clone() for t in cache.k_pools + cache.v_pools]
    free = list(cache.table.free)
    for ks, vs in (([x, y], [x, x]), ([x, x], [x, y]), ([x, x.expand(2, 2, 20, D)], [x, x])):
        with pytest.raises(ValueError, match="append"):
            cache.append(0, ks, vs, inv_freq=inv)
    assert (cache.table.frags[0] == table).all() and cache.table.free == free
    assert all(torch.equal(a, b) for a, b in zip(cache.k_pools + cache.v_pools, pools))


def test_a_refused_append_takes_no_slots(gpu):
    """Rows on the host, or a call inside a capture: the sequence and the free pages stay as they were."""
    inv = workloads.inv_freq().to(gpu)
    cache = paged.PagedKV(1, 2, 9, 16, device=gpu)
    x = rand(1, (1, 2, 20, D), torch.float16, gpu)
    cache.append(0, [x], [x], inv_freq=inv)
    table, free = cache.table.frags[0].copy(), list(cache.table.free)
    with pytest.raises(RuntimeError):
        cache.append(0, [x.cpu()], [x.cpu()], inv_freq=inv)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="not captured"):
            cache.append(0, [x], [x], inv_freq=inv)
    assert (cache.table.frags[0] == table).all() and cache.table.free == free and y is not None
    cache.append(0, [x], [x], inv_freq=inv)
    close(cache.gather(0)[0][:, 20:], x[0], 20, inv)
