"""Paged KV cache: page pools, per-sequence fragment lists, decode over a tile
table, and a prune that frees the dropped span's pages and re-rotates the kept
suffix's keys in place.

threadcut keeps each layer's cache in one growing buffer, so a prune moves the
whole kept suffix C (threadcut/kv.py:28-41, 83-92). Its README
(README.md:141-144) names the next step: with a paged cache, dropping the span
frees pages and C needs only a key re-rotation. This module is that cache:

- Every layer has a K pool and a V pool ``[pages, Hkv, P, D]``. A page holds P
  consecutive token slots of one sequence, and every layer uses the same page
  ids, so one page table serves all of them.
- A sequence is an ordered list of fragments ``(page, first slot, count)``.
  Appends extend the last fragment while its page has room, then take a new
  page. A prune cuts the list at the dropped span. A page no fragment uses any
  more goes back to the free list, and the kept fragments stay where they are.
- Decode reads a tile table: each fragment is cut into tiles of at most 16
  slots, entries ``{page, first slot, rows, first logical position}``
  (``tc_decode_paged_attention``). Attention over a set of keys does not
  depend on their order, so holes left by prunes cost nothing.
- The prune's only device work is ``tc_paged_rotate_keys``: C's keys rotated
  in place by -(c0 - a) positions with the reference's rotation
  (threadcut/kv.py:20-25), for every layer in one launch. V is not touched.

``PageTable`` is the bookkeeping alone (no device; its fragment arithmetic is the
host code of ``tc_page_tiles``, ``tc_page_prune`` and ``tc_page_token_offsets``),
``PagedKV`` adds the pools.
"""
import ctypes
import weakref

import numpy as np
import torch
import torch.nn.functional as F
from torch.autograd.graph import increment_version
from transformers import DynamicCache
from transformers.cache_utils import DynamicLayer

from . import _lib
from .flash_decode import HEAD_DIM, _on_device, _plan, _shared_workspace
from .kv import _plain, rope_table, rotate_half, rows_ok, watched
from .prefill import GROUPS, band_mask

TILE = 16  # rows per tile-table entry (the decode kernel's tile)
# Rows of K (tokens times KV heads) whose repeated reading has to be saved for decode to read what all sequences share
# once for all: the one launch for both, with large work-groups, takes longer than the plain one where there is little
# to save. At most 16 query rows a KV head take a lighter work-group. Shared against plain (us on the GPU, sequences of
# 60 to 200 own tokens, 8 KV heads, sequences x rows of a head): 2 x 4 4096 shared tokens 8.9, 8.5, 8192 10.8, 11.8;
# 4 x 4 1024 8.1, 7.4, 2048 8.1, 8.7; 8 x 2 1024 8.2, 8.8; 8 x 4 1024 10.5, 9.0, 2048 10.7, 11.5; 16 x 4 512 12.5,
# 9.8, 1024 12.7, 13.0; 16 x 8 1024 14.4, 14.6; 32 x 4 512 14.2, 14.4, 1024 16.1, 21.9; of 2 KV heads: 8 x 4 8192
# 12.1, 11.9; 16 x 4 4096 13.1, 12.3, 8192 14.7, 18.3.
SHARED_MIN_ROWS = 131072
SHARED_MIN_ROWS_FEW = 49152
_I64P = ctypes.POINTER(ctypes.c_int64)


_EMPTY = np.zeros((0, 3), dtype=np.int64)


def _cut(frags, lo, hi):
    """The fragments (rows of an int64 [F, 3] array) covering logical tokens [lo, hi)."""
    if hi <= lo or len(frags) == 0:
        return _EMPTY
    ends = np.cumsum(frags[:, 2])
    begins = ends - frags[:, 2]
    i0 = int(np.searchsorted(ends, lo, side="right"))
    i1 = int(np.searchsorted(begins, hi, side="left"))
    sub = frags[i0:i1].copy()
    if len(sub):
        skip = lo - begins[i0]
        if skip > 0:
            sub[0, 1] += skip
            sub[0, 2] -= skip
        over = ends[i1 - 1] - hi
        if over > 0:
            sub[-1, 2] -= over
        sub = sub[sub[:, 2] > 0]
    return sub


def _to_device(arr, device):
    """A host numpy array as a device tensor: staged in pinned memory and copied on the
    current stream without a host wait (torch keeps the staging block until the copy ran)."""
    return torch.from_numpy(np.ascontiguousarray(arr)).pin_memory().to(device, non_blocking=True)


def _upload(arrays, device):
    """int32 arrays as device tensors, in one copy (each a multiple of 16 bytes but the last)."""
    flat = _to_device(np.concatenate([a.ravel() for a in arrays]), device)
    return tuple(t.view(a.shape) for t, a in zip(flat.split([a.size for a in arrays]), arrays))


def _as_batch(t):
    """[Hkv, n, D] as [1, Hkv, n, D]."""
    return t if t.dim() == 4 else t.unsqueeze(0)


def _addr(a):
    return a.__array_interface__["data"][0]


def _rotated(x, positions, inv_freq):
    """x [B, heads, n, 128] rotated to int positions [B, n] by torch operations: the angles in 64 bits, the rotation in
    fp32, the result in x's type (what tc_paged_append_rope computes)."""
    angle = positions[..., None].double() * inv_freq.to(x.device).float().double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    f = x.float()
    return (f * torch.cat((cos, cos), -1) + rotate_half(f) * torch.cat((sin, sin), -1)).to(x.dtype)


def _rows_strides(t):
    """(batch, head, token) strides of [B, heads, n, D] rows."""
    return _lib.i64x3(*t.stride()[:3])


def _frag_arg(frags):
    f = frags
    if not (isinstance(f, np.ndarray) and f.dtype == np.int64 and f.ndim == 2 and f.flags.c_contiguous):
        f = np.ascontiguousarray(np.asarray(frags, dtype=np.int64).reshape(-1, 3))
    return f, _addr(f), len(f)


def _tiles(frags, page_tokens, first_pos=0):
    """Tile entries {page, first slot, rows, logical start} of a fragment array of pages of
    page_tokens slots, int32 [T, 4] (tc_page_tiles): each fragment cut at multiples of 16
    slots."""
    lib = _lib.load()
    f, fp, nf = _frag_arg(frags)
    n = lib.tc_page_tiles(fp, nf, int(page_tokens), int(first_pos), None, 0)
    if n < 0:
        _lib.check(-n, "tc_page_tiles")
    out = np.empty((n, 4), dtype=np.int32)
    if n:
        _lib.check(0 if lib.tc_page_tiles(fp, nf, int(page_tokens), int(first_pos), _addr(out), n) == n
                   else _lib.TC_ERR_INVALID_ARGUMENT, "tc_page_tiles")
    return out


def tiles_of(frags, page_tokens):
    """Tile entries (page, first slot, rows) of a fragment array of pages of page_tokens
    slots, int32 [T, 3]: each fragment is cut at multiples of 16 slots, so full tiles are
    16-slot aligned."""
    return np.ascontiguousarray(_tiles(frags, page_tokens)[:, :3])


def _placed(slots, start):
    """int64 [n, 2] slots of consecutive tokens as int32 [n, 4] rows (page, slot, position, 0), the first at `start`."""
    out = np.zeros((len(slots), 4), dtype=np.int32)
    out[:, :2] = slots
    out[:, 2] = np.arange(start, start + len(slots))
    return out


def _check_inv_freq(f, what):
    if not isinstance(f, torch.Tensor) or f.shape != (HEAD_DIM // 2,) or not f.is_floating_point():
        raise ValueError(f"PagedKV.{what}: inv_freq must be a float tensor of {HEAD_DIM // 2} inverse frequencies")


def _query_ok(t, pool, rows):
    """rows_ok for the query heads of new tokens (any number of heads)."""
    sh, st = t.shape, t.stride()
    return (t.is_cuda and len(sh) == 4 and sh[3] == HEAD_DIM and sh[2] == rows and t.dtype == pool.dtype
            and t.get_device() == pool.get_device() and st[3] == 1 and not (st[0] | st[1] | st[2]) & 7
            and not t.data_ptr() & 15 and _plain(t))


class PageTable:
    """Pages of `page_tokens` slots shared by `batch` sequences (host bookkeeping).

    frags[b] is sequence b's int64 [F, 3] array of (page, first slot, count).
    """

    def __init__(self, num_pages, page_tokens, batch=1):
        if num_pages < 1 or page_tokens < 1 or batch < 1:
            raise ValueError("PageTable needs num_pages, page_tokens and batch >= 1")
        self.num_pages = int(num_pages)
        self.page_tokens = int(page_tokens)
        self.free = list(range(self.num_pages - 1, -1, -1))  # pop() hands out the lowest id first
        self.frags = [_EMPTY.copy() for _ in range(batch)]
        self._lengths = {}  # (the fragments it was counted from, tokens) of each sequence
        self.users = {}  # pages that more than one sequence uses (fork): how many do
        self.version = 0  # bumped on every change, so device copies know when to refresh

    @property
    def batch(self):
        return len(self.frags)

    def length(self, b):
        known, fr = self._lengths.get(b), self.frags[b]
        if known is None or known[0] is not fr:  # (fragments are replaced, never changed in place)
            known = self._lengths[b] = (fr, int(fr[:, 2].sum()))
        return known[1]

    def _extend(self, b, n):
        """n tokens more (or fewer) on the last page of sequence b."""
        length, fr = self.length(b) + n, self.frags[b].copy()
        fr[-1, 2] += n
        self.frags[b] = fr
        self._lengths[b] = (fr, length)
        self.version += 1

    def _room(self, b):
        """Slots that sequence b's next tokens find on its last page (none on a shared one: the others' tokens are,
        or will be, behind its own)."""
        fr = self.frags[b]
        if len(fr) == 0:
            return 0
        page, first, count = fr[-1].tolist()
        return 0 if page in self.users else self.page_tokens - first - count

    def _drop(self, pages):
        """Takes one user from each of `pages`; returns those that nobody uses any more."""
        freed = []
        for p in pages:
            n = self.users.pop(p, 1) - 1
            if n > 1:
                self.users[p] = n
            elif n == 0:
                freed.append(p)
        return freed

    def fork(self, src, dst, n):
        """Sequence dst (empty) starts with the first n tokens of sequence src, in the same pages. They stay where
        they are until the last of the sequences that use them lets them go."""
        if src == dst or len(self.frags[dst]):
            raise ValueError(f"fork: sequence {dst} is not an empty one beside sequence {src}")
        if not 0 <= n <= self.length(src):
            raise ValueError(f"fork: {n} tokens of a sequence of {self.length(src)}")
        fr = _cut(self.frags[src], 0, n)
        for p in set(fr[:, 0].tolist()):
            self.users[p] = self.users.get(p, 1) + 1
        self.frags[dst] = fr.copy()
        self.version += 1

    def pages_needed(self, b, n):
        """Pages that the next n tokens of sequence b take from the free list."""
        return -(-max(0, n - self._room(b)) // self.page_tokens)

    def reserve(self, b, n):
        """Slots of the next n tokens of sequence b, in order: int64 [n, 2] of (page, slot)."""
        if n < 0:
            raise ValueError("reserve: n must be >= 0")
        n, P = int(n), self.page_tokens
        fr = self.frags[b]
        room = self._room(b)
        if 0 < n <= room:  # the usual step: behind the last token
            page, first, count = fr[-1].tolist()
            self._extend(b, n)
            out = np.empty((n, 2), dtype=np.int64)
            out[:, 0] = page
            out[:, 1] = np.arange(first + count, first + count + n)
            return out
        take = min(n, room)
        rest = n - take
        k = -(-rest // P)
        if k > len(self.free):
            raise RuntimeError(f"PageTable: {k} pages needed, {len(self.free)} free")
        out = np.empty((n, 2), dtype=np.int64)
        if take:
            page, end = int(fr[-1, 0]), int(fr[-1, 1] + fr[-1, 2])
            out[:take, 0] = page
            out[:take, 1] = np.arange(end, end + take)
            fr = fr.copy()
            fr[-1, 2] += take
        if k:
            more = np.zeros((k, 3), dtype=np.int64)
            more[:, 0] = [self.free.pop() for _ in range(k)]
            more[:, 2] = P
            more[-1, 2] = rest - (k - 1) * P
            fr = np.concatenate([fr, more])
            out[take:, 0] = np.repeat(more[:, 0], more[:, 2])
            out[take:, 1] = np.arange(rest) % P
        self.frags[b] = fr
        self.version += 1
        return out

    def reserve_all(self, n):
        """Slots of the next n tokens of every sequence, rows (page, slot, position, 0), int32 [B, n, 4]. Without room
        for all of them nothing is reserved."""
        n, P = int(n), self.page_tokens
        at = [(*fr[-1].tolist(), self.length(b)) if len(fr) else (-1, 0, P, 0) for b, fr in enumerate(self.frags)]
        if all(first + count + n <= P and page not in self.users for page, first, count, _ in at):  # the usual step
            out = np.zeros((self.batch, n, 4), dtype=np.int32)
            out[:, :, :3] = np.array([(page, first + count, start) for page, first, count, start in at])[:, None]
            if n > 1:
                out[:, :, 1:3] += np.arange(n)[:, None]
            for b in range(self.batch):
                self._extend(b, n)
            return out
        need = sum(self.pages_needed(b, n) for b in range(self.batch))
        if need > len(self.free):
            raise RuntimeError(f"PageTable: {need} pages needed, {len(self.free)} free")
        return np.stack([_placed(self.reserve(b, n), start) for b, (*_, start) in enumerate(at)])

    def prune(self, b, a, c0, c):
        """Keep tokens [0, a) and [c0, c0 + c) of sequence b; returns (the kept
        suffix's fragments, the pages freed) (tc_page_prune)."""
        old = self.frags[b]
        n = self.length(b)
        if not (0 <= a <= c0 and c >= 0 and c0 + c <= n):
            raise ValueError(f"prune: split (a={a}, c0={c0}, c={c}) outside a sequence of {n} tokens")
        if c == 0 and len(old) and n - int(old[-1, 2]) < a:  # last tokens of the last fragment go: it keeps its page
            self._extend(b, a - n)
            return _EMPTY.copy(), []
        f, fp, nf = _frag_arg(old)
        # One buffer: kept (nf + 1 rows), suffix (nf rows), freed (nf), counts (3).
        buf = np.empty(7 * nf + 6, dtype=np.int64)
        base = _addr(buf)
        rc = _lib.load().tc_page_prune(fp, nf, self.page_tokens, int(a), int(c0), int(c), base,
                                       base + 8 * (3 * nf + 3), base + 8 * (6 * nf + 3),
                                       ctypes.cast(base + 8 * (7 * nf + 3), _I64P))
        _lib.check(rc, "tc_page_prune")
        nk, ns, nfr = (int(x) for x in buf[7 * nf + 3:])
        self.frags[b] = buf[:3 * nk].reshape(nk, 3).copy()
        freed = self._drop(buf[6 * nf + 3:6 * nf + 3 + nfr].tolist())
        self.free += freed[::-1]
        self.version += 1
        return buf[3 * nf + 3:3 * nf + 3 + 3 * ns].reshape(ns, 3).copy(), freed

    def release(self, b):
        """Drop sequence b entirely (the pages that no other sequence shares return to the free list)."""
        self.free += sorted(self._drop(set(self.frags[b][:, 0].tolist())), reverse=True)
        self.frags[b] = _EMPTY.copy()
        self.version += 1

    def token_slots(self, b):
        """(page, slot) of every token of sequence b in logical order, int64 [n, 2]."""
        fr = self.frags[b]
        if len(fr) == 0:
            return np.zeros((0, 2), dtype=np.int64)
        rep = np.repeat(np.arange(len(fr)), fr[:, 2])
        i = np.arange(len(rep)) - np.repeat(np.cumsum(fr[:, 2]) - fr[:, 2], fr[:, 2])
        return np.stack([fr[rep, 0], fr[rep, 1] + i], axis=1)

    def tile_table(self, window=None, sink_tokens=0, skip=0):
        """int32 [B, max_tiles, 4] and tiles int32 [B] (numpy): entries {page, first slot,
        rows, first logical position} in logical order. With a window, of each sequence's last
        `window` tokens and its first `sink_tokens`; with `skip`, without its first `skip`
        fragments (the same in every sequence)."""
        lib, B = _lib.load(), self.batch
        # One array of what the call reads, the lists' addresses and then their lengths, over one array of the lists.
        frags, args = np.concatenate(self.frags, dtype=np.int64), np.empty((2, B), dtype=np.int64)
        args[1] = [len(f) for f in self.frags]
        args[0] = _addr(frags) + 24 * (args[1].cumsum() - args[1] + skip)
        args[1] -= skip
        base = _addr(args)
        start = int(self.frags[0][:skip, 2].sum()) if skip else 0
        fixed = (base, base + 8 * B, B, self.page_tokens, start, min(int(window or 0), 1 << 40),
                 min(int(sink_tokens), 1 << 40))
        most = lib.tc_page_table(*fixed, None, 0, None)
        tab = np.empty((B, max(1, most) if not skip else max(0, most), 4), dtype=np.int32)
        cnt = np.empty(B, dtype=np.int32)
        if most < 0 or lib.tc_page_table(*fixed, _addr(tab), tab.shape[1], _addr(cnt)) != most:
            _lib.check(_lib.TC_ERR_INVALID_ARGUMENT, "tc_page_table")
        return tab, cnt

    def shared_frags(self):
        """Leading fragments that are the same in every sequence."""
        if not self.users or self.batch < 2:
            return 0
        most = min(len(f) for f in self.frags)
        first = self.frags[0][:most]
        for f in self.frags[1:]:
            apart = (f[:most] != first[:most]).any(axis=1)
            most = int(apart.argmax()) if apart.any() else most
        return most

    def token_offsets(self, page_bytes, slot_bytes, pitch=None):
        """int32 [B, pitch]: byte offset of every logical token's row within a head slab of
        the pools (page * page_bytes + slot * slot_bytes); past a sequence's end, INT32_MIN,
        which no buffer range covers."""
        n = max([self.length(b) for b in range(self.batch)] + [1])
        pitch = max(n, int(pitch or 0))
        off = np.empty((self.batch, pitch), dtype=np.int32)
        lib = _lib.load()
        for b in range(self.batch):
            f, fp, nf = _frag_arg(self.frags[b])
            if lib.tc_page_token_offsets(fp, nf, self.page_tokens, int(page_bytes), int(slot_bytes), _addr(off[b]),
                                         pitch) < 0:
                raise RuntimeError("PageTable.token_offsets: pools of 2 GiB or more need 64-bit offsets")
        return off


class PagedKV:
    """A paged KV cache of `layers` layers on one GPU.

    K/V pools are ``[num_pages, kv_heads, page_tokens, 128]`` per layer (zeroed
    at creation); `page_tokens` should be a multiple of 16 so that full tiles
    are aligned. Sequences grow with `append` and shrink with `prune`.
    """

    def __init__(self, layers, kv_heads, num_pages, page_tokens=64, batch=1, dtype=torch.float16, device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("PagedKV: the pools must live on a GPU (the kernels are HIP only)")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"PagedKV: dtype {dtype} unsupported (float16, bfloat16)")
        self.table = PageTable(num_pages, page_tokens, batch)
        shape = (num_pages, kv_heads, page_tokens, HEAD_DIM)
        self.k_pools = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.v_pools = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.kv_heads = kv_heads
        self.dtype = dtype
        # The pools' own device, with its index ("cuda" alone names the current device).
        self.device = self.k_pools[0].device if self.k_pools else torch.device(
            "cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        # (version, what device_table or device_offsets returns, for each stream)
        self._dev_table = self._dev_off = self._dev_window = self._dev_shared = (None, None)
        self._last_tables = (None, None, None)  # what the last decode() read, and for which table, window and stream

    @property
    def layers(self):
        return len(self.k_pools)

    def length(self, b=0):
        return self.table.length(b)

    def _strides(self):
        return _lib.i64x3(*self.k_pools[0].stride()[:3])

    def append(self, b, ks, vs, inv_freq=None):
        """Append tokens to sequence b: ks/vs are per-layer [Hkv, n, D] (or
        [1, Hkv, n, D]) tensors on the pools' device. With ``inv_freq`` (float [D / 2])
        the keys are not rotated yet: they are rotated to their positions, length(b)
        onwards, on the way into their slots."""
        if len(ks) != self.layers or len(vs) != self.layers:
            raise ValueError(f"append: {self.layers} layers of K and V expected")
        n = ks[0].shape[-2]
        native = inv_freq is not None and _lib.FAST is not None  # (which checks the rows itself)
        if not native:
            self._check_rows(ks, vs, n)
        if inv_freq is not None:
            _check_inv_freq(inv_freq, "append")
            if torch.cuda.is_current_stream_capturing():  # (a replay would write the same slots again)
                raise RuntimeError("PagedKV.append: rotated rows are not captured")
        start = self.table.length(b)
        slots = self.table.reserve(b, n)
        if n == 0:
            return
        if inv_freq is not None and self.layers:
            try:
                at = _to_device(_placed(slots, start)[None], self.device)
                if native:
                    if _lib.FAST.rope_rows(ks, vs, self.k_pools, self.v_pools, at, inv_freq, None,
                                           _lib.raw_stream(self.device.index)):
                        return
                    self._check_rows(ks, vs, n)
                ks, vs = [_as_batch(t) for t in ks], [_as_batch(t) for t in vs]
                if self._write_rotated(range(self.layers), ks, vs, at, inv_freq):
                    return
                ks = [_rotated(t.reshape(1, self.kv_heads, n, HEAD_DIM), at[..., 2], inv_freq) for t in ks]
            except Exception:
                self.table.prune(b, start, start + n, 0)  # the sequence is as it was
                raise
        idx = _to_device(slots, self.device)
        if self.layers and self._write_rows(range(self.layers), [_as_batch(t) for t in ks], [_as_batch(t) for t in vs],
                                            idx):
            return
        pages, sl = idx[:, 0], idx[:, 1]
        for kp, vp, k, v in zip(self.k_pools, self.v_pools, ks, vs):
            k = k.reshape(self.kv_heads, n, HEAD_DIM)
            v = v.reshape(self.kv_heads, n, HEAD_DIM)
            kp[pages, :, sl] = k.transpose(0, 1).to(self.dtype)
            vp[pages, :, sl] = v.transpose(0, 1).to(self.dtype)

    def _check_rows(self, ks, vs, n):
        for t in list(ks) + list(vs):
            if t.shape[-2] != n or t.numel() != self.kv_heads * n * HEAD_DIM:
                raise ValueError(f"append: every layer's K and V must be [{self.kv_heads}, {n}, {HEAD_DIM}]")

    def _write_rows(self, layers, ks, vs, slots):
        """New tokens' rows, per layer [B, Hkv, n, D], into the pools' slots (int64 [B, n, 2] of (page, slot) on the
        device, or [n, 2] for one sequence) with one launch (tc_paged_append_rows). False if the kernel does not
        take the tensors (another type, strides that differ between layers): nothing is written then."""
        if watched():
            return False
        b, n = (1, slots.shape[0]) if slots.dim() == 2 else slots.shape[:2]
        k0, v0 = ks[0], vs[0]
        for i, k, v in zip(layers, ks, vs):
            if not (k.shape[0] == v.shape[0] == b and k.stride() == k0.stride() and v.stride() == v0.stride()
                    and rows_ok(k, self.k_pools[i], n) and rows_ok(v, self.v_pools[i], n)):
                return False
        pool = self.k_pools[0]
        with _on_device(self.device):
            rc = _lib.load().tc_paged_append_rows(
                _lib.ptr_array([t.data_ptr() for t in ks]), _lib.i64x3(*k0.stride()[:3]),
                _lib.ptr_array([t.data_ptr() for t in vs]), _lib.i64x3(*v0.stride()[:3]),
                _lib.ptr_array([self.k_pools[i].data_ptr() for i in layers]),
                _lib.ptr_array([self.v_pools[i].data_ptr() for i in layers]), self._strides(), pool.shape[0],
                pool.shape[2], slots.data_ptr(), len(ks), b, self.kv_heads, n, HEAD_DIM, _lib.dtype_code(self.dtype),
                _lib.stream_of(self.device))
        _lib.check(rc, "tc_paged_append_rows")
        increment_version([pools[i] for i in layers for pools in (self.k_pools, self.v_pools)])
        return True

    def _write_rotated(self, layers, ks, vs, slots, inv_freq, qs=(), q_outs=()):
        """New tokens' rows, per layer [B, Hkv, n, D], into the pools' slots (int32 [B, n, 4] of (page, slot, position,
        0) on the device), the keys rotated to their positions, and the queries qs of the same tokens, rotated, into
        q_outs (per layer [B, Hq, n, D]), with one launch (tc_paged_append_rope). False if the kernel does not take the
        tensors: nothing is written then."""
        if watched():
            return False
        b, n = slots.shape[:2]
        for group, pools, ok in ((ks, self.k_pools, rows_ok), (vs, self.v_pools, rows_ok), (qs, self.k_pools, _query_ok)):
            for i, t in zip(layers, group):
                if t.shape[0] != b or t.stride() != group[0].stride() or not ok(t, pools[i], n):
                    return False
        pool, dev = self.k_pools[0], inv_freq.is_cuda
        f = inv_freq.to(self.device if dev else "cpu", torch.float32).contiguous()
        heads = qs[0].shape[1] if len(qs) else 0
        with _on_device(self.device):
            rc = _lib.load().tc_paged_append_rope(
                _lib.ptr_array([t.data_ptr() for t in ks]), _rows_strides(ks[0]),
                _lib.ptr_array([t.data_ptr() for t in vs]), _rows_strides(vs[0]),
                _lib.ptr_array([self.k_pools[i].data_ptr() for i in layers]),
                _lib.ptr_array([self.v_pools[i].data_ptr() for i in layers]), self._strides(), pool.shape[0],
                pool.shape[2], slots.data_ptr(),
                _lib.ptr_array([t.data_ptr() for t in qs]) if heads else None, _rows_strides(qs[0]) if heads else None,
                _lib.ptr_array([t.data_ptr() for t in q_outs]) if heads else None,
                _rows_strides(q_outs[0]) if heads else None, heads, None if dev else _lib.float_array(f),
                f.data_ptr() if dev else None, len(ks), b, self.kv_heads, n, HEAD_DIM, _lib.dtype_code(self.dtype),
                _lib.stream_of(self.device))
        _lib.check(rc, "tc_paged_append_rope")
        increment_version([pools[i] for i in layers for pools in (self.k_pools, self.v_pools)])
        return True

    def gather(self, layer, b=0):
        """Sequence b's K and V of one layer in logical order, [Hkv, n, D] copies."""
        slots = self.table.token_slots(b)
        if len(slots) == 0:
            z = torch.empty(self.kv_heads, 0, HEAD_DIM, dtype=self.dtype, device=self.device)
            return z, z.clone()
        idx = _to_device(slots, self.device)
        k = self.k_pools[layer][idx[:, 0], :, idx[:, 1]].transpose(0, 1).contiguous()
        v = self.v_pools[layer][idx[:, 0], :, idx[:, 1]].transpose(0, 1).contiguous()
        return k, v

    def fork(self, src, dst, n=None):
        """Sequence dst (empty) starts with the first n tokens (default: all) of sequence src, in the same
        pages: nothing is copied, and decode() reads what all sequences share once for all of them. Both grow
        on pages of their own. Shared tokens can be dropped by each sequence; prune() does not move them."""
        self._refuse_during_step("fork")
        self.table.fork(src, dst, self.table.length(src) if n is None else n)

    def device_table(self):
        """(tile table int32 [B, max_tiles, 4], tiles int32 [B], max_tiles) on the device."""
        version, copies = self._dev_table
        if version != self.table.version:
            copies = {}
            self._dev_table = (self.table.version, copies)
        return (copies.get(_lib.raw_stream(self.device.index))
                or _lib.per_stream(copies, self.device.index, self._upload_table))

    def shared_tables(self, group):
        """(the tiles that every sequence begins with, int32 [T, 4], each sequence's own in device_table's form, on
        the device) of a cache with forked sequences, or None where they share less than pays (for `group` query
        heads a KV head)."""
        if not self.table.users:
            return None
        version, copies = self._dev_shared
        if version != self.table.version:
            t, head = self.table.shared_frags(), self.table.frags[0]
            copies = False
            if t:
                saved = (self.table.batch - 1) * int(head[:t, 2].sum()) * self.kv_heads
                copies = (saved, _tiles(head[:t], self.table.page_tokens), *self.table.tile_table(skip=t), {})
            self._dev_shared = (self.table.version, copies)
        if copies is False:
            return None
        saved, head, own, cnt, streams = copies
        if saved < (SHARED_MIN_ROWS_FEW if self.table.batch * group <= 16 else SHARED_MIN_ROWS):
            return None
        return (streams.get(_lib.raw_stream(self.device.index))
                or _lib.per_stream(streams, self.device.index, lambda: _upload((head, own, cnt), self.device)))

    def _attend_shared(self, tables, layer, q, k_new, v_new, scale, out):
        """decode (k_new None) or decode_append of checked tensors over shared_tables."""
        head, own, cnt = tables
        b, hkv, g, d = q.shape
        kp, vp = self.k_pools[layer], self.v_pools[layer]
        nbytes = _shared_workspace(self.device.index, b, hkv, g, d, TILE * head.shape[0], TILE * own.shape[1], b > 1)
        st = lambda t: None if t is None else _lib.i64x2(t.stride(0), t.stride(1))
        ptr = lambda t: None if t is None else t.data_ptr()
        with _on_device(self.device):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            rc = _lib.load().tc_decode_paged_shared_attention(
                q.data_ptr(), _lib.i64x3(*q.stride()[:3]), kp.data_ptr(), vp.data_ptr(), self._strides(), kp.shape[0],
                kp.shape[2], head.data_ptr(), head.shape[0], own.data_ptr(), cnt.data_ptr(), own.shape[1],
                ptr(k_new), st(k_new), ptr(v_new), st(v_new), b, hkv, g, d, _lib.dtype_code(self.dtype), float(scale),
                ws.data_ptr(), ws.numel(), out.data_ptr(), _lib.i64x3(*out.stride()[:3]), _lib.stream_of(self.device))
            _lib.check(rc, "tc_decode_paged_shared_attention")
        return out

    def window_table(self, window, sink_tokens, what):
        """device_table of the tokens that a sliding window shows each sequence's newest token: its last `window` and
        its first `sink_tokens`. Attention over a set of keys does not depend on their order, so the decode kernels
        take it like the whole table. One table serves every layer of a step."""
        if window is None and not sink_tokens:
            return self.device_table()
        version, tables = self._dev_window
        if version != self.table.version:
            tables = {}
            self._dev_window = (self.table.version, tables)
        copies = tables.get((window, sink_tokens))
        if copies is None:  # False: the window hides nothing
            most = max(map(self.table.length, range(self.table.batch)))
            copies = tables[window, sink_tokens] = {} if _lib.check_window(window, sink_tokens, most, what) else False
        if copies is False:
            return self.device_table()
        return (copies.get(_lib.raw_stream(self.device.index))
                or _lib.per_stream(copies, self.device.index, lambda: self._upload_table(window, sink_tokens)))

    def _upload_table(self, window=None, sink_tokens=0):
        tab, cnt = self.table.tile_table(window, sink_tokens)
        return *_upload((tab, cnt), self.device), tab.shape[1]

    def device_offsets(self):
        """(token offsets int32 [B, pitch], pitch) on the device: the byte offset of each logical
        token's row in a head slab of the pools (PageTable.token_offsets), for the paged prefill
        and the device-length decode step."""
        version, copies = self._dev_off
        if version != self.table.version:
            copies = {}
            self._dev_off = (self.table.version, copies)
        return (copies.get(_lib.raw_stream(self.device.index))
                or _lib.per_stream(copies, self.device.index, self._upload_offsets))

    def _upload_offsets(self):
        st = self.k_pools[0].stride()
        off = self.table.token_offsets(st[0] * 2, st[2] * 2)
        return _to_device(off, self.device), off.shape[1]

    def prefill(self, layer, query, scale, mask=None, causal=False, out=None, window=None, sink_tokens=0):
        """The prefill branch of threadcut/attention.py:43-46 over the pools: query
        [B, Hq, q, D] (any strides, last dim contiguous) attends the first n keys of every
        sequence (n = the sequences' common length; the last q of them are the queries'
        own tokens), in logical order, with no mask, is_causal (and then, with a ``window``,
        only the last `window` keys up to its own and the first `sink_tokens`), or a boolean mask
        [B|1, 1, q, n]. Returns [B, q, Hq, D] (the reference's transposed output)."""
        from . import prefill as pf

        self._refuse_during_step("prefill", layer)
        _lib.require_gpu(query, what="PagedKV.prefill")
        b, hq, ql, d = query.shape
        lens = {self.table.length(i) for i in range(self.table.batch)}
        if b != self.table.batch or d != HEAD_DIM or query.dtype != self.dtype or query.device != self.device:
            raise ValueError(f"PagedKV.prefill: query {tuple(query.shape)} {query.dtype} does not fit the cache")
        if len(lens) != 1:
            raise ValueError(f"PagedKV.prefill: sequences of different lengths {sorted(lens)}")
        n = lens.pop()
        if not 0 <= ql <= n or hq % self.kv_heads:
            raise ValueError(f"PagedKV.prefill: {ql} queries over {n} keys, {hq} query heads")
        if out is None:
            out = torch.empty((b, ql, hq, d), dtype=query.dtype, device=query.device)
        if ql == 0:
            return out
        if mask is not None and causal:
            raise ValueError("PagedKV.prefill: pass either a mask or causal")
        if window is not None and not causal:
            raise ValueError("PagedKV.prefill: a window needs causal (a mask holds its own)")
        w = _lib.check_window(window, sink_tokens, n, "PagedKV.prefill")
        off, pitch = self.device_offsets()
        tiles, tiles_bytes, mptr, mst = None, 0, None, _lib.i64x3(0, 0, 1)
        if mask is not None:
            m = mask
            if m.dtype != torch.bool or m.dim() != 4 or m.shape[1] != 1 or m.shape[0] not in (1, b) \
                    or tuple(m.shape[2:]) != (ql, n) or m.device != self.device:
                raise ValueError(f"PagedKV.prefill: the mask must be bool [B|1, 1, {ql}, {n}] on the pools' device")
            if m.stride(3) != 1 and n > 1:  # the kernel reads mask rows as contiguous bytes
                m = m.contiguous()
            tiles = pf.mask_tiles(m, hq, self.kv_heads)
            tiles_bytes = tiles.numel()
            m = m[:, 0]
            mptr, mst = m.data_ptr(), pf._mask_strides(m)
        lib = _lib.load()
        kp, vp = self.k_pools[layer], self.v_pools[layer]
        splits, nbytes = pf._plan(self.device.index, b, ql, n, w, hq, self.kv_heads)
        with _on_device(self.device):
            ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=self.device)
            if w is not None:
                rc = lib.tc_prefill_paged_window_attention(
                    query.data_ptr(), pf._strides(query, (0, 1, 2)), kp.data_ptr(), vp.data_ptr(), self._strides(),
                    kp.shape[0], off.data_ptr(), pitch, *w, ql, n, b, hq, self.kv_heads, d,
                    _lib.dtype_code(self.dtype), float(scale), splits, ws.data_ptr(), ws.numel(), out.data_ptr(),
                    pf._strides(out, (0, 1, 2)), _lib.stream_of(self.device))
                _lib.check(rc, "tc_prefill_paged_window_attention")
                return out
            rc = lib.tc_prefill_paged_attention(
                query.data_ptr(), pf._strides(query, (0, 1, 2)), kp.data_ptr(), vp.data_ptr(), self._strides(),
                kp.shape[0], off.data_ptr(), pitch, mptr, mst,
                None if tiles is None else tiles.data_ptr(), tiles_bytes, int(bool(causal)), ql, n, b, hq,
                self.kv_heads, d, _lib.dtype_code(self.dtype), float(scale), splits, ws.data_ptr(), ws.numel(),
                out.data_ptr(), pf._strides(out, (0, 1, 2)), _lib.stream_of(self.device))
            _lib.check(rc, "tc_prefill_paged_attention")
        return out

    def _step_pending(self, layer=None):
        """True between reserve_step() and the last layer's decode_append of that step:
        the tile table then includes slots not every layer has written yet. With `layer`,
        True only while that layer's own row of the step is unwritten."""
        step = getattr(self, "_step", None)
        if step is None or step[0] != self.table.version:
            return False
        return bool(step[1]) if layer is None else layer in step[1]

    def _refuse_during_step(self, what, layer=None):
        """Refuse a read of the tile table while the reserved step's slots are unwritten: in
        every layer (layer None: prune, a new reservation), or in the layer to be read."""
        if self._step_pending(layer):
            raise RuntimeError(f"PagedKV.{what}: a reserved decode step is incomplete; run decode_append for "
                               "every layer (or cancel_step()) first")

    def cancel_step(self):
        """Drop the slots of an incomplete reserved step (each sequence's last tokens)."""
        if not self._step_pending():
            return
        for b in range(self.table.batch):
            n = self.table.length(b)
            self.table.prune(b, n - self._step[2], n, 0)
        self._step = None

    def decode(self, layer, q, scale, out=None, split=None, window=None, sink_tokens=0):
        """softmax(q·Kᵀ·scale)·V over each sequence's keys of one layer, with a ``window``
        over its last `window` ones and its first `sink_tokens`.

        q [B, Hkv, G, D] (G query heads per KV head, last dim contiguous) in the
        pools' dtype; returns out [B, Hkv, G, D]. Enqueued on the current stream.
        """
        self._refuse_during_step("decode", layer)
        fast = _lib.FAST
        if fast is not None and split is None and q.is_cuda and q.dim() == 4 and 0 <= layer < self.layers:
            # The whole call in native code; None for what it does not take (then as below).
            stream = _lib.raw_stream(self.device.index)
            key = (self.table.version, window, sink_tokens, stream, q.shape[2])
            last = self._last_tables  # (read once: another thread may replace it)
            if last[0] != key:  # the layers of a step ask for the same ones
                shared = self.shared_tables(q.shape[2]) if window is None else None
                last = self._last_tables = (key, shared, None if shared else self.window_table(window, sink_tokens, "decode"))
            _, shared, table = last
            if shared:
                done = fast.paged_shared(q, self.k_pools[layer], self.v_pools[layer], *shared, None, None, out, scale,
                                         stream)
            else:
                done = fast.paged_decode(q, self.k_pools[layer], self.v_pools[layer], table[0], table[1], out, scale,
                                         stream)
            if done is not None:
                return done
        _lib.require_gpu(q, what="PagedKV.decode")
        b, hkv, g, d = q.shape
        if b != self.table.batch or hkv != self.kv_heads or d != HEAD_DIM or q.dtype != self.dtype:
            raise ValueError(f"PagedKV.decode: q {tuple(q.shape)} {q.dtype} does not fit the cache")
        if q.stride(3) != 1:
            raise ValueError("PagedKV.decode: q must have a contiguous last dimension")
        if q.device != self.device:
            raise ValueError(f"PagedKV.decode: q is on {q.device}, the pools on {self.device}")
        if not 0 <= layer < self.layers:
            raise IndexError(f"PagedKV.decode: layer {layer} outside [0, {self.layers})")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(3) != 1:
            raise ValueError("PagedKV.decode: out must match q in shape, dtype and device")
        tables = self.shared_tables(g) if window is None and split is None else None
        if tables is not None:
            return self._attend_shared(tables, layer, q, None, None, scale, out)
        tab, cnt, mt = self.window_table(window, sink_tokens, "decode")
        lib = _lib.load()
        kp, vp = self.k_pools[layer], self.v_pools[layer]
        _, nbytes = _plan(q.device.index, b, hkv, g, d, TILE * mt, split, b > 1)
        with _on_device(q.device):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            rc = lib.tc_decode_paged_attention(
                q.data_ptr(), _lib.i64x3(*q.stride()[:3]), kp.data_ptr(), vp.data_ptr(), self._strides(),
                kp.shape[0], kp.shape[2], tab.data_ptr(), cnt.data_ptr(), mt, b, hkv, g, d,
                _lib.dtype_code(self.dtype), float(scale), int(split or 0), ws.data_ptr(), ws.numel(),
                out.data_ptr(), _lib.i64x3(*out.stride()[:3]), _lib.stream_of(q.device))
            _lib.check(rc, "tc_decode_paged_attention")
        return out

    def reserve_step(self, n=1):
        """Reserve the slots of the next n tokens of every sequence (once per step,
        before layer 0); every layer's `decode_append` (one token) or `write_step` of that
        step then writes its new K/V rows there. Without room for all of them nothing is
        reserved."""
        if n < 1:
            raise ValueError(f"PagedKV.reserve_step: {n} tokens")
        self._refuse_during_step("reserve_step")
        slots = self.table.reserve_all(n)
        # (table version, layers not written yet, tokens, the slots and their copy for each stream)
        self._step = (self.table.version, set(range(self.layers)), int(n), slots, {})

    def _step_slots(self, step):
        """The reserved step's slots on the device (int32 [B, n, 4])."""
        if torch.cuda.is_current_stream_capturing():  # (a replay would write this step's slots again)
            raise RuntimeError("PagedKV.write_step: rotated rows are not captured; decode_append_at is")
        return _lib.per_stream(step[4], self.device.index, lambda: _to_device(step[3], self.device))

    def write_step(self, layer, k_new, v_new, inv_freq=None, query=None):
        """The unfused order of a step: write one layer's new K/V rows ([B, Hkv, n, D], or
        [B, Hkv, D] of one token) into the slots reserve_step(n) took. Once a layer's rows
        are written (here or by decode_append), decode() and prefill() of that layer read the
        new tokens; prune() and the next reserve_step() wait for every layer.

        With ``inv_freq`` (float [D / 2]) the keys are not rotated yet: they are rotated to
        their positions on the way, and so are the tokens' queries, if given ([B, Hq, n, D];
        returned as a new tensor of that shape)."""
        step = getattr(self, "_step", None)
        if step is None or step[0] != self.table.version or layer not in step[1]:
            raise RuntimeError(f"PagedKV.write_step: layer {layer} has no reserved slot in this step")
        if inv_freq is not None and _lib.FAST is not None and k_new.is_cuda:
            # The whole call in native code; None for what it does not take (then as below).
            done = _lib.FAST.rope_rows((k_new,), (v_new,), (self.k_pools[layer],), (self.v_pools[layer],),
                                       self._step_slots(step), inv_freq, query, _lib.raw_stream(self.device.index))
            if done is not None:
                step[1].discard(layer)
                return None if done is True else done
        b, n = self.table.batch, step[2]
        kn = k_new.reshape(b, self.kv_heads, n, HEAD_DIM)
        vn = v_new.reshape(b, self.kv_heads, n, HEAD_DIM)
        out = None
        if inv_freq is not None:
            _check_inv_freq(inv_freq, "write_step")
        if query is not None:
            if inv_freq is None:
                raise ValueError("PagedKV.write_step: a query is rotated by inv_freq, which is missing")
            if query.dim() != 4 or query.shape[0] != b or query.shape[2:] != (n, HEAD_DIM) or \
                    query.dtype != self.dtype or query.device != self.device:
                raise ValueError(f"PagedKV.write_step: query {tuple(query.shape)} {query.dtype} on {query.device}, "
                                 f"expected [{b}, Hq, {n}, {HEAD_DIM}] {self.dtype} on {self.device}")
        done = False
        if inv_freq is not None:
            at = self._step_slots(step)
            if query is not None:
                out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
            done = self._write_rotated([layer], [kn], [vn], at, inv_freq, *(([query], [out]) if query is not None else ()))
            if not done:
                kn = _rotated(kn, at[..., 2], inv_freq)
                out = _rotated(query, at[..., 2], inv_freq) if query is not None else None
        if not done:
            for i, slots in enumerate(step[3]):  # a run of slots of one page at a time
                ends = np.flatnonzero(np.diff(slots[:, 0])) + 1
                for lo, hi in zip([0, *ends.tolist()], [*ends.tolist(), n]):
                    page, first = int(slots[lo, 0]), int(slots[lo, 1])
                    self.k_pools[layer][page, :, first:first + hi - lo] = kn[i, :, lo:hi]
                    self.v_pools[layer][page, :, first:first + hi - lo] = vn[i, :, lo:hi]
        step[1].discard(layer)
        return out

    def decode_append(self, layer, q, k_new, v_new, scale, out=None, split=None, window=None, sink_tokens=0):
        """One decode step of one layer with the append fused in: k_new/v_new
        [B, Hkv, D] (or [B, Hkv, 1, D]) go to the slots `reserve_step` took, and q
        attends every key of its sequence including the new one, or with a ``window`` the
        last `window` of them, the new one among them, and the first `sink_tokens`. Returns
        out [B, Hkv, G, D]."""
        step, fast = getattr(self, "_step", None), _lib.FAST
        if step is not None and step[2] != 1 and step[0] == self.table.version:
            raise RuntimeError(f"PagedKV.decode_append: the step has {step[2]} tokens a sequence (write_step takes them)")
        if (fast is not None and split is None and q.is_cuda and q.dim() == 4 and step is not None
                and step[0] == self.table.version and layer in step[1]):
            # The whole call in native code; None for what it does not take (then as below).
            tables = self.shared_tables(q.shape[2]) if window is None else None
            stream = _lib.raw_stream(q.get_device())
            if tables is not None:
                done = fast.paged_shared(q, self.k_pools[layer], self.v_pools[layer], *tables, k_new, v_new, out, scale,
                                         stream)
            else:
                tab, cnt, _ = self.window_table(window, sink_tokens, "decode_append")
                done = fast.paged_append(q, self.k_pools[layer], self.v_pools[layer], tab, cnt, k_new, v_new, out,
                                         scale, stream)
            if done is not None:
                step[1].discard(layer)
                return done
        _lib.require_gpu(q, k_new, v_new, what="PagedKV.decode_append")
        b, hkv, g, d = q.shape
        if b != self.table.batch or hkv != self.kv_heads or d != HEAD_DIM or q.dtype != self.dtype:
            raise ValueError(f"PagedKV.decode_append: q {tuple(q.shape)} {q.dtype} does not fit the cache")
        if not 0 <= layer < self.layers:
            raise IndexError(f"PagedKV.decode_append: layer {layer} outside [0, {self.layers})")
        kn = k_new.reshape(b, hkv, HEAD_DIM) if k_new.dim() == 4 else k_new
        vn = v_new.reshape(b, hkv, HEAD_DIM) if v_new.dim() == 4 else v_new
        for name, t in (("q", q), ("k_new", kn), ("v_new", vn)):
            if t.stride(-1) != 1 or t.dtype != self.dtype or t.device != self.device:
                raise ValueError(f"PagedKV.decode_append: {name} must be {self.dtype} on {self.device}, "
                                 "last dim contiguous")
        if kn.shape != (b, hkv, HEAD_DIM) or vn.shape != (b, hkv, HEAD_DIM):
            raise ValueError("PagedKV.decode_append: k_new/v_new must be [B, Hkv, D]")
        if step is None or step[0] != self.table.version or layer not in step[1]:
            raise RuntimeError(f"PagedKV.decode_append: layer {layer} has no reserved slot in this step "
                               "(call reserve_step() once per step, then each layer once)")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(3) != 1:
            raise ValueError("PagedKV.decode_append: out must match q in shape, dtype and device")
        tables = self.shared_tables(g) if window is None and split is None else None
        if tables is not None:
            self._attend_shared(tables, layer, q, kn, vn, scale, out)
            step[1].discard(layer)
            return out
        tab, cnt, mt = self.window_table(window, sink_tokens, "decode_append")
        lib = _lib.load()
        kp, vp = self.k_pools[layer], self.v_pools[layer]
        _, nbytes = _plan(q.device.index, b, hkv, g, d, TILE * mt, split, b > 1)
        with _on_device(q.device):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            rc = lib.tc_decode_paged_append_attention(
                q.data_ptr(), _lib.i64x3(*q.stride()[:3]), kp.data_ptr(), vp.data_ptr(), self._strides(),
                kp.shape[0], kp.shape[2], tab.data_ptr(), cnt.data_ptr(), mt,
                kn.data_ptr(), _lib.i64x2(kn.stride(0), kn.stride(1)), vn.data_ptr(),
                _lib.i64x2(vn.stride(0), vn.stride(1)), b, hkv, g, d, _lib.dtype_code(self.dtype), float(scale),
                int(split or 0), ws.data_ptr(), ws.numel(), out.data_ptr(), _lib.i64x3(*out.stride()[:3]),
                _lib.stream_of(q.device))
            _lib.check(rc, "tc_decode_paged_append_attention")
        step[1].discard(layer)
        return out

    def decode_append_at(self, layer, q, k_new, v_new, lens, scale, out=None):
        """decode_append with the sequence lengths on the device (int32 [B], tokens before the
        step), for a captured step: the new rows go to logical positions lens[b], whose slots
        must already be in the table (reserved ahead), and q attends positions [0, lens[b]].
        Nothing here reads lens on the host, so a graph of this call stays valid while lens
        advances; the table must not change meanwhile."""
        b, hkv, g, d = q.shape
        kn = k_new.reshape(b, hkv, HEAD_DIM)
        vn = v_new.reshape(b, hkv, HEAD_DIM)
        for name, t in (("q", q), ("k_new", kn), ("v_new", vn)):
            if t.stride(-1) != 1 or t.dtype != self.dtype or t.device != self.device:
                raise ValueError(f"PagedKV.decode_append_at: {name} must be {self.dtype} on {self.device}, "
                                 "last dim contiguous")
        if lens.dtype != torch.int32 or lens.shape != (b,) or lens.device != self.device:
            raise ValueError("PagedKV.decode_append_at: lens must be int32 [B] on the pools' device")
        if out is None:
            out = torch.empty_like(q)
        tab, cnt, mt = self.device_table()
        off, pitch = self.device_offsets()
        lib = _lib.load()
        kp, vp = self.k_pools[layer], self.v_pools[layer]
        _, nbytes = _plan(self.device.index, b, hkv, g, d, TILE * mt, None, b > 1)
        with _on_device(self.device):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            rc = lib.tc_decode_paged_append_attention_at(
                q.data_ptr(), _lib.i64x3(*q.stride()[:3]), kp.data_ptr(), vp.data_ptr(), self._strides(),
                kp.shape[0], kp.shape[2], tab.data_ptr(), cnt.data_ptr(), mt, off.data_ptr(), pitch, lens.data_ptr(),
                kn.data_ptr(), _lib.i64x2(kn.stride(0), kn.stride(1)), vn.data_ptr(),
                _lib.i64x2(vn.stride(0), vn.stride(1)), b, hkv, g, d, _lib.dtype_code(self.dtype), float(scale), 0,
                ws.data_ptr(), ws.numel(), out.data_ptr(), _lib.i64x3(*out.stride()[:3]), _lib.stream_of(self.device))
            _lib.check(rc, "tc_decode_paged_append_attention_at")
        return out

    def prune(self, b, s, inv_freq):
        """Keep tokens [0, s.a) and [s.c0, s.c0 + s.c) of sequence b (a threadcut
        Split): the dropped span's pages are freed and the kept suffix's keys are
        re-rotated in place by -(c0 - a) positions in every layer. Returns the
        freed page ids."""
        self._refuse_during_step("prune")
        gap = s.c0 - s.a
        if gap and s.c and self.table.users:
            kept = _cut(self.table.frags[b], s.c0, s.c0 + s.c)[:, 0].tolist()
            if any(p in self.table.users for p in kept):
                raise RuntimeError(f"PagedKV.prune: tokens [{s.c0}, {s.c0 + s.c}) of sequence {b} would move, and other "
                                   "sequences share their pages")
        suffix, freed = self.table.prune(b, s.a, s.c0, s.c)
        if gap and len(suffix):
            tiles = tiles_of(suffix, self.table.page_tokens)
            t = np.zeros((len(tiles), 4), dtype=np.int32)
            t[:, :3] = tiles
            td = _to_device(t, self.device)
            table = _lib.float_array(rope_table(-gap, inv_freq))
            lib = _lib.load()
            kp = _lib.ptr_array([p.data_ptr() for p in self.k_pools])
            with torch.cuda.device(self.device):
                rc = lib.tc_paged_rotate_keys(kp, self.layers, self._strides(), self.k_pools[0].shape[0],
                                              self.k_pools[0].shape[2], td.data_ptr(), len(tiles), self.kv_heads,
                                              HEAD_DIM, _lib.dtype_code(self.dtype), table,
                                              _lib.stream_of(self.device))
                _lib.check(rc, "tc_paged_rotate_keys")
        return freed


# ---------------------------------------------------------------------------
# The paged cache behind transformers' cache interface.
# ---------------------------------------------------------------------------

# PagedLayers by the address of their K pool: update() returns the pools, and
# the "threadcut" attention finds the layer behind them here. The entries are
# weak: a cache that nothing else holds is freed with its pools, and its
# entries leave the registry with it.
_LAYERS = weakref.WeakValueDictionary()


def layer_of(key):
    """The PagedLayer whose K pool `key` is, or None."""
    if not isinstance(key, torch.Tensor) or not key.is_cuda:
        return None
    layer = _LAYERS.get(key.data_ptr())
    if layer is None or layer.owner.kv is None or layer.owner.kv.k_pools[layer.index] is not key:
        return None
    return layer


class PagedCacheState:
    """What the layers of one paged cache share: the PagedKV (made at the first update,
    when the head count, dtype and device are known), the fused-append switch and, while
    a DecodeGraph holds the cache, the device lengths of its captured step."""

    def __init__(self, num_layers, num_pages, page_tokens, batch, fused_append):
        self.num_layers, self.num_pages, self.page_tokens, self.batch = num_layers, num_pages, page_tokens, batch
        self.fused_append = fused_append
        self.kv = None
        self.layers = []
        self.device_lens = None
        self.in_graph_step = False
        self._slots = {}

    def ensure_pools(self, like):
        if self.kv is None:
            if like.dim() != 4 or like.shape[0] != self.batch or like.shape[-1] != HEAD_DIM:
                raise ValueError(f"paged cache: K/V {tuple(like.shape)} for a batch of {self.batch} at head_dim "
                                 f"{HEAD_DIM}")
            self.kv = PagedKV(self.num_layers, like.shape[1], self.num_pages, self.page_tokens, batch=self.batch,
                              dtype=like.dtype, device=like.device)

    def check_not_captured(self, what):
        if self.device_lens is not None and not self.in_graph_step:
            raise RuntimeError(f"paged cache {what}: a DecodeGraph holds this cache; close() it first")

    def write(self, layer, keys, values):
        """Rows of positions [layer.n, layer.n + add) of every sequence into the layer's pools,
        reserving the slots when this is the first layer to reach them."""
        kv = self.kv
        add = keys.shape[-2]
        need = layer.n + add - kv.table.length(0)
        if need > 0:
            for b in range(self.batch):
                kv.table.reserve(b, need)
        slots = self.slots_on_device(layer.n, layer.n + add)
        if add and kv._write_rows([layer.index], [keys], [values], slots):
            return
        kp, vp = kv.k_pools[layer.index], kv.v_pools[layer.index]
        for b in range(self.batch):
            sl = slots[b]
            kp[sl[:, 0], :, sl[:, 1]] = keys[b].transpose(0, 1).to(kv.dtype)
            vp[sl[:, 0], :, sl[:, 1]] = values[b].transpose(0, 1).to(kv.dtype)

    def slots_on_device(self, lo, hi):
        """(page, slot) of every sequence's positions [lo, hi), int64 [B, hi - lo, 2] on the device; every
        layer of a step writes the same positions, so the upload is kept (for each stream) for the table version."""
        key = (self.kv.table.version, lo, hi)
        if self._slots and next(iter(self._slots))[0] != key[0]:
            self._slots.clear()
        return _lib.per_stream(self._slots.setdefault(key, {}), self.kv.device.index, lambda: _to_device(
            np.stack([self.kv.table.token_slots(b)[lo:hi] for b in range(self.batch)]), self.kv.device))

    def reserve_step_for(self, layer):
        """A decode step's slot per sequence: reserved by the first layer of the step."""
        if layer.n == self.kv.table.length(0):
            self.kv.reserve_step()


class PagedLayer(DynamicLayer):
    """A transformers cache layer whose K/V rows live in the pools of a PagedKV shared by
    every layer of the cache (one page table for all).

    update() writes the new tokens' rows into their slots and returns the layer's K and V
    pools, which the "threadcut" attention recognises (layer_of) and serves with the paged
    kernels: decode over the tile table, prefill through the token offsets. With
    fused_append a one-token update reserves the step's slot and leaves the row pending;
    the decode kernel writes it while it attends.
    """

    def __init__(self, owner, index):
        super().__init__()
        self.owner, self.index = owner, index
        self.n = 0
        self.pending = None

    @property
    def kv(self):
        return self.owner.kv

    def lazy_initialization(self, key_states, value_states):
        super().lazy_initialization(key_states, value_states)
        self.owner.ensure_pools(key_states)
        self.n = 0

    def flush(self):
        """Write a pending row that no attention call consumed. In a captured step (device
        lengths) only the decode kernel can place the row, at lens[b]; a row left pending
        there would be lost, so that raises."""
        if self.pending is not None:
            k, v = self.pending
            self.pending = None
            if self.owner.device_lens is not None:
                raise RuntimeError(
                    "paged cache: a one-token update of a captured decode step reached no decode attention "
                    "call (an attention mask, or a second update before attention); its K/V row would be lost")
            self.kv.write_step(self.index, k, v)

    def update(self, key_states, value_states, *args, **kwargs):
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        self.owner.check_not_captured("update")
        self.flush()
        add = key_states.shape[-2]
        if add == 1 and self.owner.device_lens is not None:
            self.pending = (key_states, value_states)  # written at lens[b] by the captured kernel
        elif add == 1 and self.owner.fused_append and key_states.is_cuda:
            self.owner.reserve_step_for(self)
            self.pending = (key_states, value_states)
        else:
            self.owner.write(self, key_states, value_states)
        self.n += add
        kp = self.kv.k_pools[self.index]
        _LAYERS[kp.data_ptr()] = self
        return kp, self.kv.v_pools[self.index]

    def get_seq_length(self):
        return self.n if self.is_initialized else 0

    def crop(self, max_length):
        raise NotImplementedError("PagedLayer.crop: shorten a paged cache with kv.splice (a prune) instead")


def new_paged_cache(config, num_pages, page_tokens=64, batch=1, fused_append=True):
    """A DynamicCache whose layers keep their K/V in page pools (PagedKV): the engine's
    cache (threadcut/kv.py:95-98) in the layout the reference's README.md:141-144 proposes.
    Use it with the "threadcut" attention; kv.splice prunes it (pages of the dropped span
    freed, the kept suffix's keys re-rotated in place)."""
    cache = DynamicCache(config=config)
    state = PagedCacheState(len(cache.layers), num_pages, page_tokens, batch, fused_append)
    cache.layers = [PagedLayer(state, i) for i in range(len(cache.layers))]
    state.layers = cache.layers
    return cache


def state_of(cache):
    """The PagedCacheState of a new_paged_cache() cache, or None."""
    layers = getattr(cache, "layers", None)
    if layers and all(isinstance(l, PagedLayer) for l in layers):
        return layers[0].owner
    return None


def attention(layer, query, attention_mask, scaling, window=None, sink_tokens=0):
    """The "threadcut" attention for a paged layer: query [B, Hq, q, D] -> [B, q, Hq, D]. A window is that of a call
    without a mask."""
    b, hq, q, d = query.shape
    kv = layer.kv
    hkv = kv.kv_heads
    g = hq // hkv
    if q == 1 and attention_mask is None:
        out = torch.empty((b, 1, hq, d), dtype=query.dtype, device=query.device)
        qg, og = query.reshape(b, hkv, g, d), out.view(b, hkv, g, d)
        if layer.pending is not None:
            k_new, v_new = layer.pending
            layer.pending = None
            if layer.owner.device_lens is not None:
                if _lib.check_window(window, sink_tokens, layer.n, "paged cache") is not None:
                    raise RuntimeError("paged cache: the captured decode step has no sliding window")
                kv.decode_append_at(layer.index, qg, k_new, v_new, layer.owner.device_lens, scaling, out=og)
            else:
                kv.decode_append(layer.index, qg, k_new, v_new, scaling, out=og, window=window, sink_tokens=sink_tokens)
        else:
            kv.decode(layer.index, qg, scaling, out=og, window=window, sink_tokens=sink_tokens)
        return out
    layer.flush()
    is_causal = attention_mask is None and q > 1 and (q == layer.n or window is not None)
    m = attention_mask
    if g in GROUPS and (m is None or (m.dtype == torch.bool and m.dim() == 4 and m.shape[1] == 1)):
        return kv.prefill(layer.index, query, scaling, m, is_causal, window=window if is_causal else None,
                          sink_tokens=sink_tokens if is_causal else 0)
    # Other masks and group sizes: the reference's route (repeat_kv + SDPA) on the gathered keys.
    ks, vs = zip(*[kv.gather(layer.index, i) for i in range(b)])
    k, v = torch.stack(ks), torch.stack(vs)
    if window is not None:
        m, is_causal = band_mask(q, k.shape[2], window, sink_tokens, k.device), False
    out = F.scaled_dot_product_attention(query, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1),
                                         attn_mask=m, scale=scaling, is_causal=is_causal)
    return out.transpose(1, 2).contiguous()
