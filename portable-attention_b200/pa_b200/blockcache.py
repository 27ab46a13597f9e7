"""A key/value cache with block scales: quantising append, decode, eviction by weight.

The reference's SdpaBackend takes dense key/value tensors
(``src/portable_attention/dispatch.py:53-76``); a serving stack keeps them in a
cache that it fills token by token, stores in 8 bits and holds to a budget.
These entry points are the three calls such a loop makes
(``pa_cache_append`` / ``pa_cache_decode`` / ``pa_cache_evict`` of
include/pa_b200.h, where the arithmetic is written down):

* append: new keys and values go behind each sequence's length, in 8 bits with
  one power-of-two scale per block of ``scale_block`` tokens, page and head;
* decode: ``reference.py:139-162`` for one query row per sequence over its own
  keys, optionally adding every row's softmax weight to ``weights``;
* evict: every (sequence, kv head) keeps its ``budget`` rows of the largest
  weight, the ``recent`` newest and the first ``sinks`` positions always.

Caches are ``(pages, kv_heads, page_size, head_dim)`` (``layout="hnd"``) or
``(pages, page_size, kv_heads, head_dim)`` (``"nhd"``), paged through a block
table or one page per sequence. ``kv_format`` is ``None`` (the query's 16-bit
type), ``"e4m3"`` (``uint8`` bit patterns) or ``"int8"``; 8-bit caches come with
float32 scales ``(pages, kv_heads, ceil(page_size / scale_block))``. ``weights``
and ``positions`` are ``(batch, kv_heads, rows)``.

The ``*_device`` functions launch on device pointers (no copies, no sync) on
``stream``; the others take NumPy arrays, copy them to the device and return new
arrays, and never change their inputs.
"""

from __future__ import annotations

import ctypes
from collections import namedtuple

import numpy as np

from ._lib import PA_I8, BlockCacheDesc, check, lib
from .device import Stream, sync_device_status
from .kvcache import kv_cache_desc

__all__ = [
    "AppendResult", "EvictResult", "block_cache_desc", "cache_append", "cache_append_device",
    "cache_decode", "cache_decode_device", "cache_decode_workspace_size", "cache_evict",
    "cache_evict_device", "cache_evict_workspace_size",
]

_FORMATS = (None, "e4m3", "int8")

AppendResult = namedtuple("AppendResult", "key_cache value_cache k_scales v_scales seq_lens weights positions")
EvictResult = namedtuple("EvictResult",
                         "key_cache value_cache k_scales v_scales seq_lens weights positions kept")


def block_cache_desc(batch, q_heads, head_dim, cache_shape, *, layout="hnd", q_dtype="f16",
                     kv_format=None, paged=False, max_pages_per_seq=0, max_seq_len=None,
                     scale=None, scale_block=None, rows=None) -> BlockCacheDesc:
    """Fill a ``pa_block_cache_desc`` for dense cache, scale and per-row arrays.

    ``scale_block`` defaults to ``page_size`` (one scale per page and head);
    ``rows`` is the last dimension of the per-row arrays (default ``max_seq_len``).
    """
    if kv_format not in _FORMATS:
        raise ValueError(f"kv_format must be one of {_FORMATS}, got {kv_format!r}")
    desc = BlockCacheDesc()
    desc.cache = kv_cache_desc(batch, q_heads, head_dim, cache_shape, layout=layout, q_dtype=q_dtype,
                               kv_format="e4m3" if kv_format == "e4m3" else None, paged=paged,
                               max_pages_per_seq=max_pages_per_seq, max_seq_len=max_seq_len, scale=scale)
    c = desc.cache
    if kv_format == "int8":
        c.kv_dtype = PA_I8
    if c.page_size < 1:
        raise ValueError(f"the cache has pages of {c.page_size} keys")
    block = int(c.page_size if scale_block is None else scale_block)
    if block < 1:
        raise ValueError(f"scale_block must be positive, got {block}")
    blocks = -(-c.page_size // block)
    desc.scale_block, desc.scale_head_stride = block, blocks
    desc.scale_page_stride = c.kv_heads * blocks
    rows = int(c.max_seq_len if rows is None else rows)
    desc.row_head_stride, desc.row_seq_stride = rows, c.kv_heads * rows
    return desc


def _handle(stream):
    return stream.handle if stream is not None else None


def cache_append_device(desc: BlockCacheDesc, k_ptr, v_ptr, new_len, k_cache_ptr, v_cache_ptr,
                        seq_lens_ptr, *, strides=None, new_lens_ptr=None, k_scales_ptr=None,
                        v_scales_ptr=None, block_table_ptr=None, weights_ptr=None,
                        positions_ptr=None, start_positions_ptr=None, seq_lens_out_ptr=None,
                        stream: Stream | None = None) -> None:
    """Launch ``pa_cache_append`` on device pointers (asynchronous on ``stream``).

    ``strides`` gives the element strides (sequence, token, head) of the new
    keys and values; the default is dense ``(batch, new_len, kv_heads, head_dim)``.
    """
    c = desc.cache
    if strides is None:
        strides = (new_len * c.kv_heads * c.head_dim, c.kv_heads * c.head_dim, c.head_dim)
    check(lib().pa_cache_append(ctypes.byref(desc), k_ptr, v_ptr, new_len, *strides, new_lens_ptr,
                                k_cache_ptr, v_cache_ptr, k_scales_ptr, v_scales_ptr,
                                block_table_ptr, seq_lens_ptr, weights_ptr, positions_ptr,
                                start_positions_ptr, seq_lens_out_ptr, _handle(stream)))


def cache_decode_workspace_size(desc: BlockCacheDesc, paged: bool, weights: bool = False) -> int:
    n = ctypes.c_size_t(0)
    check(lib().pa_cache_decode_workspace_size(ctypes.byref(desc), int(bool(paged)),
                                               int(bool(weights)), ctypes.byref(n)))
    return int(n.value)


def cache_decode_device(desc: BlockCacheDesc, q_ptr, k_cache_ptr, v_cache_ptr, out_ptr, *,
                        k_scales_ptr=None, v_scales_ptr=None, block_table_ptr=None,
                        seq_lens_ptr=None, lse_ptr=None, weights_ptr=None,
                        stream: Stream | None = None, workspace=(None, 0)) -> None:
    """Launch ``pa_cache_decode`` on device pointers (asynchronous on ``stream``)."""
    check(lib().pa_cache_decode(ctypes.byref(desc), q_ptr, k_cache_ptr, v_cache_ptr, k_scales_ptr,
                                v_scales_ptr, block_table_ptr, seq_lens_ptr, out_ptr, lse_ptr,
                                weights_ptr, workspace[0], workspace[1], _handle(stream)))


def cache_evict_workspace_size(desc: BlockCacheDesc, paged: bool, budget: int) -> int:
    n = ctypes.c_size_t(0)
    check(lib().pa_cache_evict_workspace_size(ctypes.byref(desc), int(bool(paged)), budget,
                                              ctypes.byref(n)))
    return int(n.value)


def cache_evict_device(desc: BlockCacheDesc, k_cache_ptr, v_cache_ptr, seq_lens_ptr, weights_ptr,
                       budget, seq_lens_out_ptr, kept_ptr, *, recent=0, sinks=0,
                       positions_ptr=None, next_positions_ptr=None, k_scales_ptr=None,
                       v_scales_ptr=None, block_table_ptr=None, weights_out_ptr=None,
                       positions_out_ptr=None, stream: Stream | None = None,
                       workspace=(None, 0)) -> None:
    """Launch ``pa_cache_evict`` on device pointers (asynchronous on ``stream``)."""
    check(lib().pa_cache_evict(ctypes.byref(desc), k_cache_ptr, v_cache_ptr, k_scales_ptr,
                               v_scales_ptr, block_table_ptr, seq_lens_ptr, weights_ptr,
                               positions_ptr, next_positions_ptr, budget, recent, sinks,
                               weights_out_ptr, positions_out_ptr, seq_lens_out_ptr, kept_ptr,
                               workspace[0], workspace[1], _handle(stream)))


# ------------------------------------------------------------- NumPy entry points

_CACHE_DTYPE = {None: np.float16, "e4m3": np.uint8, "int8": np.int8}


def _int32(x, name):
    """``x`` as contiguous int32; values that int32 does not hold are refused, not wrapped or cut off."""
    x = np.asarray(x)
    if x.dtype == np.int32:
        return np.ascontiguousarray(x)
    with np.errstate(invalid="ignore"):
        y = np.ascontiguousarray(x.astype(np.int32))
    if not np.array_equal(x, y):
        raise ValueError(f"{name} must hold whole numbers of 32 bits")
    return y


def _table(block_table):
    """A block table as int32. Entries behind the rows in use may hold anything: one that int32 does not
    hold becomes -1, which is no page."""
    t = np.asarray(block_table)
    if t.dtype == np.int32:
        return np.ascontiguousarray(t)
    ok = (t >= -(2 ** 31)) & (t < 2 ** 31)
    out = np.full(t.shape, -1, np.int32)
    out[ok] = _int32(t[ok], "block_table")
    return out


def _check_arrays(key_cache, value_cache, k_scales, v_scales, block_table, batch, *, layout,
                  kv_format, scale_block):
    """Contiguous cache, scale and table arrays, and the scale block they imply."""
    if kv_format not in _FORMATS:
        raise ValueError(f"kv_format must be one of {_FORMATS}, got {kv_format!r}")
    want = np.dtype(_CACHE_DTYPE[kv_format])
    k, v = np.ascontiguousarray(key_cache), np.ascontiguousarray(value_cache)
    if k.dtype != want or v.dtype != want:
        raise ValueError(f"caches must be {want.name} for kv_format={kv_format!r}")
    if k.shape != v.shape:
        raise ValueError(f"key and value caches differ in shape: {k.shape} vs {v.shape}")
    if k.ndim != 4:
        raise ValueError(f"cache must be 4-D (pages, ..., head_dim), got shape {k.shape}")
    if layout not in ("hnd", "nhd"):
        raise ValueError(f"layout must be one of ('hnd', 'nhd'), got {layout!r}")
    heads, page_size = (k.shape[1], k.shape[2]) if layout == "hnd" else (k.shape[2], k.shape[1])
    ks = vs = None
    if kv_format is None:
        if k_scales is not None or v_scales is not None:
            raise ValueError("16-bit caches have no scales")
    else:
        if k_scales is None or v_scales is None:
            raise ValueError("8-bit caches need k_scales and v_scales")
        ks = np.ascontiguousarray(k_scales, dtype=np.float32)
        vs = np.ascontiguousarray(v_scales, dtype=np.float32)
        scale_block = page_size if scale_block is None else int(scale_block)
        if scale_block < 1:
            raise ValueError(f"scale_block must be positive, got {scale_block}")
        shape = (k.shape[0], heads, -(-page_size // scale_block))
        if ks.shape != shape or vs.shape != shape:
            raise ValueError(f"scales must have shape {shape}, got {ks.shape} and {vs.shape}")
    bt = None
    if block_table is not None:
        bt = _table(block_table)
        if bt.ndim != 2 or bt.shape[0] != batch:
            raise ValueError(f"block_table must be (batch, max_pages_per_seq), got {bt.shape}")
    elif k.shape[0] < batch:
        raise ValueError(f"without a block_table the cache needs one page per sequence: {k.shape[0]} < {batch}")
    capacity = bt.shape[1] * page_size if bt is not None else page_size
    return k, v, ks, vs, bt, heads, capacity, scale_block


def _per_sequence(x, name, batch):
    x = _int32(x, name)
    if x.shape != (batch,):
        raise ValueError(f"{name} must have shape ({batch},), got {x.shape}")
    return x


def _per_row(x, name, dtype, batch, heads, rows):
    if x is None:
        return None
    x = _int32(x, name) if dtype == np.int32 else np.ascontiguousarray(x, dtype=dtype)
    if x.ndim != 3 or x.shape[:2] != (batch, heads) or x.shape[2] < rows:
        raise ValueError(f"{name} must be (batch, kv_heads, at least {rows} rows), got {x.shape}")
    return x


def _on_device(arrays, extra, launch, results):
    """Copy ``arrays`` in, run ``launch(ptrs, stream)`` and copy ``results(ptrs)`` back.

    ``extra`` gives the bytes of further device buffers; the pointers come in the
    order of ``arrays`` then ``extra`` (None for an absent array).
    """
    from .backend import _arena, _stream

    L, st, arena = lib(), _stream(), _arena()
    with arena.lock:
        ptrs = arena.carve([0 if x is None else x.nbytes for x in arrays] + list(extra))
        ptrs = [None if i < len(arrays) and arrays[i] is None else p for i, p in enumerate(ptrs)]
        for x, p in zip(arrays, ptrs):
            if x is not None and x.nbytes:
                check(L.pa_memcpy_h2d(p, x.ctypes.data, x.nbytes, st.handle))
        launch(ptrs, st)
        for out, p in results(ptrs):
            if out is not None and out.nbytes:
                check(L.pa_memcpy_d2h(out.ctypes.data, p, out.nbytes, st.handle))
        st.synchronize()
    sync_device_status()


def _like(x):
    return None if x is None else np.empty_like(x)


def cache_append(k_new, v_new, key_cache, value_cache, seq_lens, block_table=None, *, new_lens=None,
                 k_scales=None, v_scales=None, scale_block=None, layout="hnd", kv_format=None,
                 weights=None, positions=None, start_positions=None) -> AppendResult:
    """Write float16 tokens ``(batch, T, kv_heads, head_dim)`` behind each sequence.

    ``new_lens`` gives each sequence's number of new tokens (default T). Returns
    the updated arrays; ``weights`` is 0 and ``positions`` is
    ``start_positions + t`` (default: the row) in the new rows.
    """
    kn, vn = np.ascontiguousarray(k_new), np.ascontiguousarray(v_new)
    if kn.dtype != np.float16 or vn.dtype != np.float16 or kn.ndim != 4 or kn.shape != vn.shape:
        raise ValueError("k_new and v_new must be float16 (batch, T, kv_heads, head_dim) of one shape, "
                         f"got {kn.dtype} {kn.shape} and {vn.dtype} {vn.shape}")
    B, T, H, D = kn.shape
    k, v, ks, vs, bt, heads, capacity, block = _check_arrays(
        key_cache, value_cache, k_scales, v_scales, block_table, B, layout=layout,
        kv_format=kv_format, scale_block=scale_block)
    if H != heads or D != k.shape[3]:
        raise ValueError(f"new tokens have {H} heads of {D}, the cache {heads} of {k.shape[3]}")
    lens = _per_sequence(seq_lens, "seq_lens", B)
    nl = None if new_lens is None else _per_sequence(new_lens, "new_lens", B)
    add = np.full(B, T, np.int32) if nl is None else nl
    if B and (lens.min() < 0 or add.min() < 0 or add.max() > T):
        raise ValueError("seq_lens and new_lens must be in range (0 <= new_lens <= T)")
    top = int((lens.astype(np.int64) + add).max()) if B else 0
    if top > capacity:
        raise ValueError(f"the cache holds {capacity} rows per sequence, {top} are needed")
    w = _per_row(weights, "weights", np.float32, B, H, top)
    p = _per_row(positions, "positions", np.int32, B, H, top)
    if w is not None and p is not None and w.shape != p.shape:
        raise ValueError(f"weights and positions differ in shape: {w.shape} vs {p.shape}")
    sp = None if start_positions is None else _per_sequence(start_positions, "start_positions", B)
    if sp is not None and p is None:
        raise ValueError("start_positions needs positions")
    rows = w.shape[2] if w is not None else p.shape[2] if p is not None else capacity
    out = AppendResult(_like(k), _like(v), _like(ks), _like(vs), (lens + add).astype(np.int32), _like(w), _like(p))
    if B == 0 or T == 0:
        return AppendResult(*(None if x is None else x.copy() for x in (k, v, ks, vs, lens, w, p)))
    desc = block_cache_desc(B, H, D, k.shape, layout=layout, kv_format=kv_format, paged=bt is not None,
                            max_pages_per_seq=bt.shape[1] if bt is not None else 0,
                            max_seq_len=min(capacity, rows), scale_block=block, rows=rows)

    def launch(q, st):
        cache_append_device(desc, q[0], q[1], T, q[2], q[3], q[7], new_lens_ptr=q[8], k_scales_ptr=q[4],
                            v_scales_ptr=q[5], block_table_ptr=q[6], weights_ptr=q[9], positions_ptr=q[10],
                            start_positions_ptr=q[11], seq_lens_out_ptr=q[12], stream=st)

    _on_device([kn, vn, k, v, ks, vs, bt, lens, nl, w, p, sp], [4 * B], launch,
               lambda q: [(out.key_cache, q[2]), (out.value_cache, q[3]), (out.k_scales, q[4]),
                          (out.v_scales, q[5]), (out.seq_lens, q[12]), (out.weights, q[9]),
                          (out.positions, q[10])])
    return out


def cache_decode(query, key_cache, value_cache, seq_lens=None, block_table=None, *, k_scales=None,
                 v_scales=None, scale=None, scale_block=None, layout="hnd", kv_format=None,
                 max_seq_len=None, weights=None, return_lse=False):
    """Decode ``query`` (batch, q_heads, head_dim) float16 over a block-scaled cache.

    Returns the float16 output; with ``return_lse`` also the float32 natural-log
    lse (batch, q_heads), and with ``weights`` the updated weights, as a tuple.
    """
    q = np.ascontiguousarray(query)
    if q.dtype != np.float16 or q.ndim != 3:
        raise ValueError(f"query must be float16 (batch, q_heads, head_dim), got {q.dtype} {q.shape}")
    B, Hq, D = q.shape
    k, v, ks, vs, bt, heads, capacity, block = _check_arrays(
        key_cache, value_cache, k_scales, v_scales, block_table, B, layout=layout,
        kv_format=kv_format, scale_block=scale_block)
    sl = None
    if seq_lens is not None:
        sl = _per_sequence(seq_lens, "seq_lens", B)
        if max_seq_len is None:
            max_seq_len = int(sl.max()) if B else 0
    if max_seq_len is None:
        max_seq_len = capacity
    w = _per_row(weights, "weights", np.float32, B, heads, max_seq_len)
    out, lse, w_out = np.empty((B, Hq, D), np.float16), np.empty((B, Hq), np.float32), _like(w)
    desc = block_cache_desc(B, Hq, D, k.shape, layout=layout, kv_format=kv_format, paged=bt is not None,
                            max_pages_per_seq=bt.shape[1] if bt is not None else 0, max_seq_len=max_seq_len,
                            scale=scale, scale_block=block, rows=w.shape[2] if w is not None else None)
    if B:
        ws = cache_decode_workspace_size(desc, bt is not None, w is not None)

        def launch(p, st):
            cache_decode_device(desc, p[0], p[1], p[2], p[8], k_scales_ptr=p[3], v_scales_ptr=p[4],
                                block_table_ptr=p[5], seq_lens_ptr=p[6], lse_ptr=p[9], weights_ptr=p[7],
                                stream=st, workspace=(p[10], ws))

        _on_device([q, k, v, ks, vs, bt, sl, w], [out.nbytes, lse.nbytes, ws], launch,
                   lambda p: [(out, p[8]), (lse, p[9]), (w_out, p[7])])
    got = [out] + ([lse] if return_lse else []) + ([w_out] if w is not None else [])
    return got[0] if len(got) == 1 else tuple(got)


def cache_evict(key_cache, value_cache, seq_lens, weights, budget, block_table=None, *, recent=0,
                sinks=0, positions=None, next_positions=None, k_scales=None, v_scales=None,
                scale_block=None, layout="hnd", kv_format=None) -> EvictResult:
    """Keep each (sequence, kv head)'s ``budget`` rows of the largest weight.

    Rows with position ``>= next_positions - recent`` or ``< sinks`` are kept
    first (``positions`` defaults to the row, ``next_positions`` to the length).
    Returns the updated arrays and ``kept`` (batch, kv_heads, budget): the row
    that each row held before, -1 behind a shorter sequence.
    """
    B = int(np.shape(seq_lens)[0]) if np.ndim(seq_lens) == 1 else -1
    if B < 0:
        raise ValueError(f"seq_lens must be one-dimensional, got shape {np.shape(seq_lens)}")
    k, v, ks, vs, bt, heads, capacity, block = _check_arrays(
        key_cache, value_cache, k_scales, v_scales, block_table, B, layout=layout,
        kv_format=kv_format, scale_block=scale_block)
    lens = _per_sequence(seq_lens, "seq_lens", B)
    top = int(lens.max()) if B else 0
    if B and (lens.min() < 0 or top > capacity):
        raise ValueError(f"seq_lens must be in [0, {capacity}]")
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError("budget must be positive and hold recent and sinks (non-negative) together")
    w = _per_row(weights, "weights", np.float32, B, heads, top)
    if w is None:
        raise ValueError("weights must be given")
    p = _per_row(positions, "positions", np.int32, B, heads, top)
    if p is not None and p.shape != w.shape:
        raise ValueError(f"weights and positions differ in shape: {w.shape} vs {p.shape}")
    nx = None if next_positions is None else _per_sequence(next_positions, "next_positions", B)
    if p is not None and nx is None:
        raise ValueError("positions need next_positions")
    kept = np.full((B, heads, budget), -1, np.int32)
    if B == 0 or top == 0:
        return EvictResult(*(None if x is None else x.copy() for x in (k, v, ks, vs, lens, w, p)), kept)
    out = EvictResult(*(_like(x) for x in (k, v, ks, vs, lens, w, p)), kept)
    D = k.shape[3]
    desc = block_cache_desc(B, heads, D, k.shape, layout=layout, kv_format=kv_format, paged=bt is not None,
                            max_pages_per_seq=bt.shape[1] if bt is not None else 0, max_seq_len=top,
                            scale_block=block, rows=w.shape[2])
    ws = cache_evict_workspace_size(desc, bt is not None, budget)

    def launch(q, st):
        cache_evict_device(desc, q[0], q[1], q[5], q[6], budget, q[9], q[10], recent=recent, sinks=sinks,
                           positions_ptr=q[7], next_positions_ptr=q[8], k_scales_ptr=q[2], v_scales_ptr=q[3],
                           block_table_ptr=q[4], weights_out_ptr=q[6], positions_out_ptr=q[7], stream=st,
                           workspace=(q[11], ws))

    _on_device([k, v, ks, vs, bt, lens, w, p, nx], [lens.nbytes, kept.nbytes, ws], launch,
               lambda q: [(out.key_cache, q[0]), (out.value_cache, q[1]), (out.k_scales, q[2]),
                          (out.v_scales, q[3]), (out.seq_lens, q[9]), (out.weights, q[6]),
                          (out.positions, q[7]), (kept, q[10])])
    return out
