"""GQA-aware attention registered into transformers as ``"threadcut"``.

Drop-in for threadcut/attention.py:22-51. Decode (one query token, no mask):
the g query heads sharing a KV head are handed to the split-KV HIP kernels of
``flash_decode`` together with the unexpanded cache views, for any batch
size (the reference used its GPU kernel for b == 1 and SDPA otherwise; both
compute the same softmax), whenever the kernels take the tensors
(``flash_decode.supports``: GPU, float16/bfloat16, head_dim 128, g <= 8).
Other decode calls, host tensors included, keep the reference's own decode
path for them (threadcut/attention.py:40-42): SDPA with each group's query
heads folded into a length-g query against the unexpanded cache. Prefill
(threadcut/attention.py:43-46) runs the GQA-native HIP kernel of ``prefill``
on the unexpanded K/V for GPU tensors in float16/bfloat16 with head_dim 128,
g in (1, 2, 4, 8) and no mask or a boolean [b|1, 1, q, n] mask (what the
registered ``sdpa_mask`` produces). Other prefill calls keep the reference's
own path: expand KV once and run SDPA. A paged cache (``paged.new_paged_cache``)
hands over its page pools; its layers run the paged decode and prefill kernels.
"""
import torch
import torch.nn.functional as F
from transformers import AttentionInterface
from transformers.masking_utils import AttentionMaskInterface, sdpa_mask

from . import _lib, kv, paged, prefill
from .flash_decode import decode_append_at, decode_append_into, decode_into, supports as decode_supports

NAME = "threadcut"


def repeat_kv(x, n):
    """[b, h, s, d] -> [b, h*n, s, d], each KV head repeated n times in place order."""
    if n == 1:
        return x
    b, h, s, d = x.shape
    return x.unsqueeze(2).expand(b, h, n, s, d).reshape(b, h * n, s, d)


def attention(module, query, key, value, attention_mask, dropout=0.0, scaling=None, **kwargs):
    """transformers attention interface (threadcut/attention.py:30-47).

    query [b, hq, q, d] (usually a transposed view), key/value [b, hkv, n, d]
    (views into the cache). Returns ([b, q, hq, d] contiguous, None).

    ``sliding_window`` (which transformers passes for its sliding layers) holds
    where there is no mask: each query then sees the last `sliding_window` keys
    up to its own and the first `sink_tokens` (default 0). A mask holds its own.
    """
    window, sinks = kwargs.get("sliding_window"), kwargs.get("sink_tokens") or 0
    if not window or attention_mask is not None:
        window, sinks = None, 0
    b, hq, q, d = query.shape
    scaling = scaling if scaling is not None else query.shape[-1] ** -0.5
    layer = paged.layer_of(key)
    if layer is not None:  # a paged cache layer handed over its pools
        return paged.attention(layer, query, attention_mask, scaling, window, sinks), None
    hkv = key.shape[1]
    g = hq // hkv
    pending = kv.take_pending(key)
    if window is not None and (_lib.check_window(window, sinks, key.shape[2], NAME) or 1 < q < key.shape[2]):
        return _windowed(query, key, value, pending, scaling, int(window), int(sinks)), None
    fast = _lib.FAST
    if q == 1 and attention_mask is None and fast is not None and query.is_cuda:
        # The whole call in native code; None for what it does not take (then as below).
        stream = _lib.raw_stream(query.get_device())
        if pending is None:
            out = fast.decode(query, key, value, scaling, stream)
        else:
            out = fast.decode_append(query, pending.kbuf, pending.vbuf, *pending.pending,
                                     pending.n if pending.device_pos is None else pending.device_pos, scaling, stream)
        if out is not None:
            if pending is not None:
                pending.pending = None
            return out, None
    if q == 1 and attention_mask is None and not decode_supports(query, key, value):
        # The reference's decode path for calls its GPU kernel does not serve
        # (attention.py:40-42): the g query heads of a KV head as a length-g query.
        if pending is not None:
            pending.flush()
        out = F.scaled_dot_product_attention(query.reshape(b, hkv, g, d), key, value, scale=scaling)
        return out.reshape(b, hq, 1, d).transpose(1, 2).contiguous(), None
    if q == 1 and attention_mask is None:
        # [b, 1, hq, d] contiguous is [b, hkv, g, d] with head index h*g + i.
        out = torch.empty((b, 1, hq, d), dtype=query.dtype, device=query.device)
        if pending is not None:
            # GrowingLayer deferred this token's append: write it and attend in one launch.
            k_new, v_new = pending.pending
            pending.pending = None
            if pending.device_pos is not None:  # graph-captured step: the position lives on the device
                decode_append_at(query.reshape(b, hkv, g, d), pending.kbuf, pending.vbuf, k_new, v_new,
                                 pending.device_pos, scaling, out.view(b, hkv, g, d))
            else:
                decode_append_into(query.reshape(b, hkv, g, d), pending.kbuf, pending.vbuf, k_new, v_new, pending.n,
                                   scaling, out.view(b, hkv, g, d))
        else:
            decode_into(query.reshape(b, hkv, g, d), key, value, scaling, out.view(b, hkv, g, d))
        return out, None
    if pending is not None:  # a deferred append must land before SDPA reads the cache
        pending.flush()
    is_causal = attention_mask is None and q > 1 and q == key.shape[2]
    if prefill.supports(query, key, attention_mask):
        return prefill.prefill_attention(query, key, value, attention_mask, scaling, is_causal), None
    out = F.scaled_dot_product_attention(query, repeat_kv(key, g), repeat_kv(value, g),
                                         attn_mask=attention_mask, scale=scaling, is_causal=is_causal)
    return out.transpose(1, 2).contiguous(), None


def _windowed(query, key, value, pending, scaling, window, sinks):
    """The call under a sliding window: the decode and prefill kernels where they take the tensors, else SDPA."""
    b, hq, q, d = query.shape
    hkv, n = key.shape[1], key.shape[2]
    g = hq // hkv
    fast = _lib.FAST
    if q == 1 and fast is not None and query.is_cuda:
        stream = _lib.raw_stream(query.get_device())
        if pending is None:
            out = fast.decode(query, key, value, scaling, stream, window, sinks)
        else:
            out = fast.decode_append(query, pending.kbuf, pending.vbuf, *pending.pending,
                                     pending.n if pending.device_pos is None else pending.device_pos, scaling, stream,
                                     window, sinks)
        if out is not None:
            if pending is not None:
                pending.pending = None
            return out
    if q == 1 and decode_supports(query, key, value):
        out = torch.empty((b, 1, hq, d), dtype=query.dtype, device=query.device)
        qg, og = query.reshape(b, hkv, g, d), out.view(b, hkv, g, d)
        if pending is None:
            decode_into(qg, key, value, scaling, og, window=window, sink_tokens=sinks)
            return out
        k_new, v_new = pending.pending
        pending.pending = None
        if pending.device_pos is not None:
            decode_append_at(qg, pending.kbuf, pending.vbuf, k_new, v_new, pending.device_pos, scaling, og,
                             window=window, sink_tokens=sinks)
        else:
            decode_append_into(qg, pending.kbuf, pending.vbuf, k_new, v_new, pending.n, scaling, og, window=window,
                               sink_tokens=sinks)
        return out
    if pending is not None:
        pending.flush()
    if prefill.supports(query, key, None):
        return prefill.prefill_attention(query, key, value, None, scaling, True, window=window, sink_tokens=sinks)
    out = F.scaled_dot_product_attention(query, repeat_kv(key, g), repeat_kv(value, g), scale=scaling,
                                         attn_mask=prefill.band_mask(q, n, window, sinks, query.device))
    return out.transpose(1, 2).contiguous()


AttentionInterface.register(NAME, attention)
AttentionMaskInterface.register(NAME, sdpa_mask)
