"""Sliding-window attention with sink tokens against the definition in float64: decode (one length, per-sequence
lengths, with the append fused in), prefill, and both over page pools.

A query at position p sees keys j <= p with j > p - window or j < sinks."""
import pytest
import torch

from threadcut_amd import attention, flash_decode, kv, paged, prefill
from threadcut_amd.match import Split

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5


def rand(seed, shape, dtype, dev):
    return torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def definition(q, k, v, first, window, sinks):
    """(out, A) in float64 of queries q [hq, t, d] at positions first .. on keys k/v [hkv, n, d] (rows past the last
    query's position do not count): out [hq, t, d] and A, the sum of the weights times |v|. A row that sees nothing is 0."""
    hq, t, _ = q.shape
    g = hq // k.shape[0]
    p = first + torch.arange(t, device=q.device)[:, None]
    j = torch.arange(k.shape[1], device=q.device)[None]
    hidden = ~((j <= p) & ((j > p - window) | (j < sinks)))
    k, v = k.double().repeat_interleave(g, 0), v.double().repeat_interleave(g, 0)
    s = torch.bmm(q.double(), k.transpose(1, 2).contiguous()) * SCALE
    w = torch.softmax(s.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)
    return torch.bmm(w, v), torch.bmm(w, v.abs())


def close(got, want, spread, rounded_weights):
    """The output is rounded once (eps / 2 of its value); scores, exponentials, sums and weights are held in fp32 (a
    score of up to 40 with 2^-22, so a weight with 2^-16; decode's weights, as two numbers of the type, with 2^-16).
    Prefill rounds a weight to the type (eps / 2 of each), in the sum over v and in the one that divides it."""
    f = torch.finfo(got.dtype)
    bound = f.eps / 2 * want.abs() + 2.0 ** -14 * spread + f.smallest_normal
    if rounded_weights:
        bound = bound * (1 + f.eps) + f.eps / 2 * (spread + want.abs())
    off = (got.double() - want).abs()
    assert torch.all(off <= bound), f"worst {(off / bound).max().item():.3g} of the bound"


def cache(seed, b, hkv, n, dtype, dev, spare=40):
    """Views of buffers with room for more, whose unused rows are NaN: reading one would show."""
    out = []
    for i in range(2):
        buf = torch.full((b, hkv, n + spare, D), float("nan"), dtype=dtype, device=dev)
        buf[:, :, :n] = rand(seed + i, (b, hkv, n, D), dtype, dev)
        out.append(buf[:, :, :n])
    return out


def check_decode(out, q, k, v, lens, window, sinks):
    """out, q [b, hkv, g, d]; query b at the last of its lens[b] tokens."""
    for i, n in enumerate(lens):
        want, spread = definition(q[i].reshape(-1, 1, D), k[i, :, :n], v[i, :, :n], n - 1, window, sinks)
        close(out[i].reshape(-1, 1, D), want, spread, False)


DECODE = [  # batch, kv heads, group, tokens, window, sinks
    (1, 8, 4, 1000, 100, 4), (1, 8, 4, 1000, 1, 0), (2, 8, 1, 500, 16, 1), (3, 2, 8, 2000, 640, 16),
    (1, 1, 3, 5000, 1111, 17), (1, 8, 4, 200, 150, 50), (1, 8, 4, 201, 150, 50), (1, 8, 4, 202, 150, 50),
    (1, 8, 4, 40, 7, 33), (1, 8, 4, 40, 6, 33), (16, 8, 4, 3000, 2048, 4), (1, 8, 4, 33000, 8192, 100),
    (64, 2, 2, 300, 64, 5), (1, 8, 2, 70, 1000, 4), (1, 8, 4, 1, 1, 0), (4, 8, 4, 20000, 17, 2), (2, 8, 4, 4097, 1, 1000)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,hkv,g,n,window,sinks", DECODE)
def test_decode(gpu, dtype, b, hkv, g, n, window, sinks):
    print(f"case: {b} x {hkv} heads x {g}, {n} tokens, window {window}, {sinks} sinks", flush=True)
    k, v = cache(1, b, hkv, n, dtype, gpu)
    hidden = max(n - window, 0)
    if hidden > sinks:  # what no query sees is not read
        k[:, :, sinks:hidden] = float("nan")
        v[:, :, sinks:hidden] = float("nan")
    q = rand(3, (b, hkv, g, D), dtype, gpu)
    out = flash_decode.decode_attention_batched(q, k, v, SCALE, window=window, sink_tokens=sinks)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    check_decode(out, q, k, v, [n] * b, window, sinks)
    # Through the registered attention, as a model hands the query over.
    qm = q.reshape(b, 1, hkv * g, D).transpose(1, 2)
    again = attention.attention(None, qm, k, v, None, scaling=SCALE, sliding_window=window, sink_tokens=sinks)[0]
    check_decode(again.view(b, hkv, g, D), q, k, v, [n] * b, window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,window,sinks", [
    ([0, 1, 15, 16, 17, 700], 16, 1), ([700, 0, 0], 64, 40), ([5, 1200, 130, 129, 128], 128, 0),
    ([3000, 2999, 1, 2000], 1999, 500), ([100] * 70, 30, 3), ([4000, 64], 1, 0), ([900, 20, 64, 65, 66], 48, 16)])
def test_decode_lengths(gpu, dtype, lens, window, sinks):
    print(f"case: lengths {lens[:8]}, window {window}, {sinks} sinks", flush=True)
    b, n = len(lens), max(lens)
    k, v = cache(1, b, 4, n, dtype, gpu)
    for i, m in enumerate(lens):
        k[i, :, m:], v[i, :, m:] = float("nan"), float("nan")
    q = rand(3, (b, 4, 4, D), dtype, gpu)
    t = torch.tensor(lens, dtype=torch.int32, device=gpu)
    out = flash_decode.decode_attention_batched(q, k, v, SCALE, lens=t, window=window, sink_tokens=sinks)
    check_decode(out, q, k, v, lens, window, sinks)
    for split in (64, 256):  # the caller's split length
        again = flash_decode.decode_attention_batched(q, k, v, SCALE, lens=t, split=split, window=window,
                                                      sink_tokens=sinks)
        check_decode(again, q, k, v, lens, window, sinks)


def test_windows_that_hide_nothing_are_the_plain_call(gpu):
    k, v = cache(1, 2, 8, 300, torch.float16, gpu)
    q = rand(3, (2, 8, 4, D), torch.float16, gpu)
    plain = flash_decode.decode_attention_batched(q, k, v, SCALE)
    for window, sinks in ((300, 0), (1 << 40, 0), (200, 100), (1, 299), (5, 1 << 40)):
        assert torch.equal(plain, flash_decode.decode_attention_batched(q, k, v, SCALE, window=window, sink_tokens=sinks))
    qp = rand(4, (2, 32, 50, D), torch.float16, gpu)
    plain = prefill.prefill_attention(qp, k, v, None, SCALE, True)
    assert torch.equal(plain, prefill.prefill_attention(qp, k, v, None, SCALE, True, window=300))
    assert torch.equal(plain, prefill.prefill_attention(qp, k, v, None, SCALE, True, window=100, sink_tokens=200))
    qm = q.reshape(2, 1, 32, D).transpose(1, 2)
    assert torch.equal(attention.attention(None, qm, k, v, None)[0],
                       attention.attention(None, qm, k, v, None, sliding_window=300)[0])


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("n,window,sinks", [(500, 100, 4), (100, 1, 0), (64, 60, 3), (64, 61, 3), (64, 62, 3), (3, 2, 0)])
def test_growing_cache_steps(gpu, fused, n, window, sinks):
    """A decode loop over a GrowingLayer, its rows written by the attention kernel or before it."""
    layer = kv.GrowingLayer()
    layer.fused_append = fused
    k, v = rand(1, (2, 8, n, D), torch.float16, gpu), rand(2, (2, 8, n, D), torch.float16, gpu)
    layer.update(k, v)
    for step in range(3):
        kn, vn = rand(10 + step, (2, 8, 1, D), torch.float16, gpu), rand(20 + step, (2, 8, 1, D), torch.float16, gpu)
        q = rand(30 + step, (2, 32, 1, D), torch.float16, gpu)
        k, v = torch.cat((k, kn), 2), torch.cat((v, vn), 2)
        keys, values = layer.update(kn, vn)
        assert (layer.pending is not None) == fused
        out = attention.attention(None, q, keys, values, None, scaling=SCALE, sliding_window=window,
                                  sink_tokens=sinks)[0]
        assert layer.pending is None and torch.equal(layer.keys, k) and torch.equal(layer.values, v)
        check_decode(out.view(2, 8, 4, D), q.view(2, 8, 4, D), k, v, [n + step + 1] * 2, window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_at_device_positions_replayed(gpu, dtype):
    """One captured step serves every position: short of the window, at its edge, past it."""
    b, hkv, g, cap, window, sinks = 3, 8, 4, 700, 90, 5
    lens = [0, 93, 400]
    k, v = cache(1, b, hkv, cap, dtype, gpu, spare=0)
    for i, m in enumerate(lens):
        k[i, :, m:], v[i, :, m:] = float("nan"), float("nan")
    wk, wv = k.clone(), v.clone()
    pos = torch.tensor(lens, dtype=torch.int32, device=gpu)
    q, kn, vn = (torch.empty(s, dtype=dtype, device=gpu) for s in ((b, hkv, g, D), (b, hkv, D), (b, hkv, D)))
    out = torch.empty_like(q)

    def step():
        flash_decode.decode_append_at(q, k, v, kn, vn, pos, SCALE, out, window=window, sink_tokens=sinks)
        pos.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    pos.sub_(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(8):
        q.copy_(rand(50 + i, q.shape, dtype, gpu))
        kn.copy_(rand(60 + i, kn.shape, dtype, gpu))
        vn.copy_(rand(70 + i, vn.shape, dtype, gpu))
        graph.replay()
        for j, m in enumerate(lens):
            wk[j, :, m + i], wv[j, :, m + i] = kn[j], vn[j]
        torch.cuda.synchronize()
        assert torch.equal(k.nan_to_num(9.0), wk.nan_to_num(9.0)) and torch.equal(v.nan_to_num(9.0), wv.nan_to_num(9.0))
        check_decode(out, q, k, v, [m + i + 1 for m in lens], window, sinks)


PREFILL = [  # batch, q heads, kv heads, queries, past, window, sinks
    (1, 32, 8, 300, 0, 64, 4), (1, 32, 8, 300, 700, 100, 0), (2, 16, 8, 77, 500, 33, 70), (1, 8, 8, 1000, 0, 1, 0),
    (1, 64, 8, 130, 2000, 256, 16), (1, 16, 4, 2, 3000, 700, 1), (1, 32, 8, 2, 5, 3, 0), (1, 32, 8, 1500, 0, 1000, 0),
    (1, 32, 8, 93, 9000, 4096, 4), (1, 8, 2, 2000, 3000, 129, 200), (4, 32, 8, 40, 1000, 64, 64),
    (1, 32, 8, 64, 64, 127, 1), (1, 32, 8, 3, 20000, 1500, 130), (1, 8, 1, 4100, 0, 513, 65), (2, 32, 32, 700, 100, 300, 4),
    (1, 16, 8, 1, 500, 100, 3), (1, 32, 8, 513, 9000, 2000, 1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,hq,hkv,t,past,window,sinks", PREFILL)
def test_prefill(gpu, dtype, b, hq, hkv, t, past, window, sinks):
    print(f"case: {b} x {hq} over {hkv} heads, {t} on {past}, window {window}, {sinks} sinks", flush=True)
    n = t + past
    k, v = cache(1, b, hkv, n, dtype, gpu)
    q = rand(3, (b, t, hq, D), dtype, gpu).transpose(1, 2)
    out = prefill.prefill_attention(q, k, v, None, SCALE, True, window=window, sink_tokens=sinks)
    seen = [definition(q[i], k[i], v[i], past, window, sinks) for i in range(b)]
    for i in range(b):
        close(out[i].transpose(0, 1), *seen[i], True)
    for splits in (1, 3, 32):
        again = prefill.prefill_attention(q, k, v, None, SCALE, True, splits=splits, window=window, sink_tokens=sinks)
        for i in range(b):
            close(again[i].transpose(0, 1), *seen[i], True)
    if t > 1:
        model = attention.attention(None, q, k, v, None, scaling=SCALE, sliding_window=window, sink_tokens=sinks)[0]
        assert torch.equal(model, out)
    # A mask that says the same.
    mask = prefill.band_mask(t, n, window, sinks, gpu)
    masked = attention.attention(None, q, k, v, mask, scaling=SCALE, sliding_window=7)[0]
    for i in range(b):
        close(masked[i].transpose(0, 1), *seen[i], True)


def test_prefill_keys_out_of_one_range(gpu):
    """Rows so far apart that a head's slab spans more than 31 bits."""
    n, t, window, sinks = 700, 40, 100, 4
    big = [torch.empty(n * (1 << 21), dtype=torch.float16, device=gpu).as_strided((1, 2, n, D), (0, D, 1 << 21, 1))
           for _ in range(2)]
    k, v = (x.copy_(rand(i, (1, 2, n, D), torch.float16, gpu)) for i, x in enumerate(big))
    q = rand(3, (1, 8, t, D), torch.float16, gpu)
    out = prefill.prefill_attention(q, k, v, None, SCALE, True, window=window, sink_tokens=sinks)
    close(out[0].transpose(0, 1), *definition(q[0], k[0], v[0], n - t, window, sinks), True)
    q1 = rand(4, (1, 2, 4, D), torch.float16, gpu)
    out = flash_decode.decode_attention_batched(q1, k, v, SCALE, window=window, sink_tokens=sinks)
    check_decode(out, q1, k, v, [n], window, sinks)


def filled(dev, lens, page_tokens, dtype, seed, prune=True):
    """A paged cache of two layers whose sequences mix their pages, with a hole in each, and its rows in order."""
    b = len(lens)
    c = paged.PagedKV(2, 8, 2 * b * (-(-(max(lens) + 90) // page_tokens) + 3), page_tokens, batch=b, dtype=dtype, device=dev)
    for t in c.k_pools + c.v_pools:
        t.fill_(float("nan"))
    gap = 37 if prune else 0
    rows = [[rand(seed + i, (2, 2, 8, n + gap, D), dtype, dev) for i, n in enumerate(lens)]][0]
    for at in range(0, max(lens) + gap, 100):
        for i, n in enumerate(lens):
            part = rows[i][:, :, :, at:min(at + 100, n + gap)]
            if part.shape[3]:
                c.append(i, list(part[0]), list(part[1]))
    for i, n in enumerate(lens):
        if prune and n:  # a span after the first token is dropped; the rows behind it stay as they are (no rotation)
            first = min(20, n)
            c.table.prune(i, first, first + gap, n - first)
            rows[i] = torch.cat((rows[i][:, :, :, :first], rows[i][:, :, :, first + gap:]), 3)
        elif prune:
            c.table.prune(i, 0, gap, 0)
            rows[i] = rows[i][:, :, :, :0]
    return c, rows


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,page_tokens,window,sinks", [
    ([500, 20, 333, 0], 16, 100, 4), ([1000], 64, 257, 33), ([64, 65, 66, 300], 40, 64, 1), ([700, 90], 128, 1, 0),
    ([5000, 300], 64, 2048, 100), ([40, 30], 16, 60, 4)])
def test_paged_decode(gpu, dtype, lens, page_tokens, window, sinks):
    print(f"case: lengths {lens}, pages of {page_tokens}, window {window}, {sinks} sinks", flush=True)
    c, rows = filled(gpu, lens, page_tokens, dtype, 1)
    b = len(lens)
    for layer in range(2):
        q = rand(40 + layer, (b, 8, 4, D), dtype, gpu)
        out = c.decode(layer, q, SCALE, window=window, sink_tokens=sinks)
        full = c.decode(layer, q, SCALE)  # both tables at once
        for i, n in enumerate(lens):
            check_decode(out[i:i + 1], q[i:i + 1], rows[i][0, layer][None], rows[i][1, layer][None], [n], window, sinks)
            check_decode(full[i:i + 1], q[i:i + 1], rows[i][0, layer][None], rows[i][1, layer][None], [n], n + 1, 0)
    for step in range(2):  # the fused step: the new token is the window's last
        c.reserve_step()
        for layer in range(2):
            q, kn, vn = (rand(60 + 10 * step + i, s, dtype, gpu) for i, s in
                         enumerate(((b, 8, 4, D), (b, 8, D), (b, 8, D))))
            out = c.decode_append(layer, q, kn, vn, SCALE, window=window, sink_tokens=sinks)
            for i in range(b):
                gk, gv = c.gather(layer, i)
                assert torch.equal(gk[:, -1], kn[i]) and torch.equal(gv[:, -1], vn[i])
                check_decode(out[i:i + 1], q[i:i + 1], gk[None], gv[None], [lens[i] + step + 1], window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,t,page_tokens,window,sinks", [
    (600, 50, 16, 100, 4), (900, 900, 64, 130, 0), (3000, 300, 64, 700, 70), (333, 2, 40, 64, 1), (2500, 1, 128, 1000, 3)])
def test_paged_prefill(gpu, dtype, n, t, page_tokens, window, sinks):
    print(f"case: {t} of {n}, pages of {page_tokens}, window {window}, {sinks} sinks", flush=True)
    c, rows = filled(gpu, [n, n], page_tokens, dtype, 1)
    q = rand(3, (2, 32, t, D), dtype, gpu)
    out = c.prefill(1, q, SCALE, causal=True, window=window, sink_tokens=sinks)
    for i in range(2):
        close(out[i].transpose(0, 1), *definition(q[i], rows[i][0, 1], rows[i][1, 1], n - t, window, sinks), True)


class Config:
    num_hidden_layers = 1

    def get_text_config(self, decoder=True):
        return self


@pytest.mark.parametrize("group", [4, 3])
def test_paged_cache_behind_the_attention(gpu, group):
    """Prompt, chunk and decode steps of a paged cache through the registered attention; three query heads a KV head
    go through torch's attention in prefill."""
    window, sinks = 50, 3
    cache = paged.new_paged_cache(Config(), 40, 16)
    k, v = (torch.zeros(1, 8, 0, D, dtype=torch.float16, device=gpu) for _ in range(2))
    for step, t in enumerate((120, 33, 1, 1)):
        kn, vn, q = (rand(10 * step + i, (1, h, t, D), torch.float16, gpu) for i, h in enumerate((8, 8, 8 * group)))
        k, v = torch.cat((k, kn), 2), torch.cat((v, vn), 2)
        kp, vp = cache.update(kn, vn, 0)
        out = attention.attention(None, q, kp, vp, None, scaling=SCALE, sliding_window=window, sink_tokens=sinks)[0]
        close(out[0].transpose(0, 1), *definition(q[0], k[0], v[0], k.shape[2] - t, window, sinks), t > 1)


@pytest.mark.parametrize("form", ["float32", "host", "group 16"])
def test_calls_the_kernels_do_not_take(gpu, form):
    """They keep torch's attention, with the band as its mask. With u half a step of the type and S the largest sum of
    |q k| scale: both factors and the score may be rounded to the type, and 128 terms added in fp32, so a score is off by
    (3 u + 128 2^-24) S, a weight by twice that (itself and the sum of weights) and 2 u, and the result by u again."""
    dev, dtype, hq = (gpu, torch.float16, 16 * 2) if form == "group 16" else (torch.device("cpu") if form == "host" else gpu,
                                                                             torch.float32, 8)
    for t in (1, 30):
        k, v = rand(1, (1, 2, 200, D), dtype, dev), rand(2, (1, 2, 200, D), dtype, dev)
        q = rand(3, (1, hq, t, D), dtype, dev)
        out = attention.attention(None, q, k, v, None, scaling=SCALE, sliding_window=40, sink_tokens=3)[0]
        want, spread = definition(q[0], k[0], v[0], 200 - t, 40, 3)
        u = torch.finfo(dtype).eps / 2
        most = SCALE * max((q[0].double().abs() @ h.double().abs().t().contiguous()).max().item() for h in k[0])
        bound = spread * (2 * (3 * u + 128 * 2.0 ** -24) * most + 2 * u) + u * want.abs()
        assert torch.all((out[0].transpose(0, 1).double() - want).abs() <= bound)


def test_extreme_scores(gpu):
    """Scores of +-60000 / sqrt(d): the running maximum and the hidden keys' -inf."""
    n, window, sinks = 300, 40, 5
    k, v = cache(1, 1, 2, n, torch.float16, gpu)
    k[:, :, ::7] *= 400
    k[:, :, sinks:n - window] = float("inf")
    v[:, :, sinks:n - window] = float("nan")
    q = rand(3, (1, 2, 4, D), torch.float16, gpu)
    out = flash_decode.decode_attention_batched(q, k, v, SCALE, window=window, sink_tokens=sinks)
    assert torch.isfinite(out).all()
    k[:, :, sinks:n - window], v[:, :, sinks:n - window] = 0, 0
    # Scores of up to 2000 carry 2^-12 in fp32, so weights 2^-11 relative to what they are.
    want, spread = definition(q[0].reshape(8, 1, D), k[0], v[0], n - 1, window, sinks)
    assert torch.all((out.double().view(8, 1, D) - want).abs() <= 2.0 ** -9 * spread + 2.0 ** -11 * want.abs())


def test_another_stream(gpu):
    c, rows = filled(gpu, [500, 90], 16, torch.float16, 1)
    q = rand(3, (2, 8, 4, D), torch.float16, gpu)
    first = c.decode(0, q, SCALE, window=100, sink_tokens=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = c.decode(0, q, SCALE, window=100, sink_tokens=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    c.prune(0, Split(400, 500, 0), None)  # the tables of before do not serve any more
    out = c.decode(0, q, SCALE, window=100, sink_tokens=4)
    check_decode(out[:1], q[:1], rows[0][0, 0, :, :400][None], rows[0][1, 0, :, :400][None], [400], 100, 4)


def test_refusals(gpu):
    k, v = cache(1, 1, 2, 50, torch.float16, gpu)
    q = rand(3, (1, 2, 4, D), torch.float16, gpu)
    for kw in (dict(window=0), dict(window=-1), dict(window=5, sink_tokens=-1), dict(sink_tokens=4)):
        with pytest.raises(ValueError):
            flash_decode.decode_attention_batched(q, k, v, SCALE, **kw)
        with pytest.raises(ValueError):
            prefill.prefill_attention(q, k, v, None, SCALE, True, **kw)
        c, _ = filled(gpu, [30], 16, torch.float16, 1)
        with pytest.raises(ValueError):
            c.decode(0, q.expand(1, 2, 4, D).repeat(1, 4, 1, 1), SCALE, **kw)
        with pytest.raises(ValueError):
            c.prefill(0, rand(1, (1, 8, 4, D), torch.float16, gpu), SCALE, causal=True, **kw)
    with pytest.raises(ValueError, match="is_causal"):
        prefill.prefill_attention(q, k, v, None, SCALE, window=5)
    with pytest.raises(ValueError, match="causal"):
        c.prefill(0, rand(1, (1, 8, 4, D), torch.float16, gpu), SCALE, window=5)
    with pytest.raises(ValueError, match="is_causal"):
        prefill.prefill_attention(q, k, v, prefill.band_mask(4, 50, 5, 0, gpu), SCALE, window=5)
