"""Block-scaled cache, host side: the oracle's rules, the C struct's layout, and
every refusal (no kernel launches)."""

from __future__ import annotations

import ctypes
import shutil
import subprocess

import numpy as np
import pytest

from oracle.blockcache import append_reference, decode_reference, evict_reference, need_scale, round8
from oracle.kvcache import decode_kv_reference

from conftest import ROOT


@pytest.mark.parametrize("fmt,qmax", [("e4m3", 448.0), ("int8", 127.0)])
def test_need_scale_is_the_least_power_of_two_that_fits(fmt, qmax):
    rng = np.random.default_rng(0)
    for top in list(np.exp(rng.uniform(-20, 20, 200))) + [qmax, np.nextafter(qmax, 1e9), qmax * 2.0 ** -7, 1.0]:
        s = need_scale([0.0, -top, np.nan, np.inf], fmt)
        assert np.log2(s) == round(np.log2(s)) and top <= qmax * s and top > qmax * s / 2
    assert need_scale([0.0], fmt) == need_scale([], fmt) == 2.0 ** -100


def test_round8_int8_and_e4m3_edges():
    assert list(round8([0.5, 1.5, -2.5, 200, -200, np.inf, np.nan], "int8")) == [0, 2, -2, 127, -127, 127, 0]
    got = round8([449, -1e9, np.inf, 17, 2.0 ** -10], "e4m3")
    assert list(got) == [448, -448, 448, 16, 0]
    assert np.isnan(round8([np.nan], "e4m3")[0])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_token_by_token_keeps_every_row_within_a_step(fmt):
    """Rows appended one at a time stand for their inputs to within one step of the block's last scale."""
    rng = np.random.default_rng(1)
    B, H, D, P, bs, n = 1, 2, 8, 16, 8, 30
    x = rng.standard_normal((B, n, H, D)) * np.exp(rng.standard_normal((B, n, H, 1)))
    k = np.zeros((2, H, P, D))
    v = k.copy()
    ks, vs = np.full((2, H, P // bs), np.nan), np.full((2, H, P // bs), np.nan)
    table = np.array([[1, 0]])
    for t in range(n):
        append_reference(x[:, t:t + 1], -x[:, t:t + 1], k, v, [t], [1], ks=ks, vs=vs, table=table, block=bs, fmt=fmt)
    for r in range(n):
        page, at = table[0, r // P], r % P
        s = ks[page, :, at // bs][:, None]
        # int8: half a step for each rounding; a row is rounded once, and again whenever the scale doubles
        # (steps 1/2 + 1/4 + ... < 1). e4m3: a half step is 2^-4 relative, or half the smallest subnormal; a
        # doubling is exact but for subnormals.
        tol = s if fmt == "int8" else np.abs(x[0, r]) * 2.0 ** -4 + s * 2.0 ** -9
        assert (np.abs(k[page, :, at] * s - x[0, r]) <= tol).all()
        assert np.array_equal(v[page, :, at], -k[page, :, at])


def test_decode_oracle_equals_the_per_tensor_oracle():
    rng = np.random.default_rng(2)
    B, Hq, H, D, P = 3, 4, 2, 8, 16
    table = np.array([[3, 1], [0, 5], [2, 4]])
    k, v = rng.standard_normal((6, H, P, D)), rng.standard_normal((6, H, P, D))
    q, lens = rng.standard_normal((B, Hq, D)), np.array([32, 0, 17])
    one = np.ones((6, H, 2))
    got = decode_reference(q, k, v, lens, ks=one * 0.5, vs=one * 0.25, table=table, block=8, weights=np.zeros((B, H, 32)))
    want, lse = decode_kv_reference(q, k, v, lens, block_table=table, k_scale=0.5, v_scale=0.25)
    np.testing.assert_allclose(got["out"], want, rtol=1e-12, atol=1e-14)
    np.testing.assert_allclose(got["lse"], lse, rtol=1e-12)
    np.testing.assert_allclose(got["weights"].sum(-1), np.array([[2, 2], [0, 0], [2, 2]]), atol=1e-12)
    assert (got["weights"][2, :, 17:] == 0).all()


def test_evict_oracle_keeps_the_best_rows_and_attention_over_them():
    rng = np.random.default_rng(3)
    B, H, D, P, n, budget = 1, 2, 8, 64, 50, 20
    k, v = rng.standard_normal((1, H, P, D)), rng.standard_normal((1, H, P, D))
    w = rng.exponential(size=(B, H, P)).astype(np.float32)
    k0, v0, w0 = k.copy(), v.copy(), w.copy()
    pos = np.tile(np.arange(P, dtype=np.int32), (B, H, 1))
    lens, kept = evict_reference(k, v, [n], w, budget, recent=5, sinks=2, positions=pos, next_positions=[n])
    assert lens == [budget]
    for h in range(H):
        best = sorted(range(2, n - 5), key=lambda r: -w0[0, h, r])[:budget - 7]
        assert sorted(kept[0, h]) == sorted([0, 1, *range(n - 5, n), *best])
        assert np.array_equal(pos[0, h, :budget], kept[0, h])
        assert np.array_equal(k[0, h, :budget], k0[0, h, kept[0, h]])
        assert np.array_equal(k[0, h, budget:], k0[0, h, budget:])       # rows behind stay
        stay = kept[0, h] < budget
        assert np.array_equal(kept[0, h][stay], np.flatnonzero(stay))    # only holes receive rows
    q = rng.standard_normal((1, H, D))
    short = decode_reference(q, k, v, lens)["out"]
    for h in range(H):
        alone = decode_reference(q[:, h:h + 1], k0[:, h:h + 1, kept[0, h]], v0[:, h:h + 1, kept[0, h]], [budget])["out"]
        np.testing.assert_allclose(short[:, h], alone[:, 0], rtol=1e-12)


_LAYOUT_C = r"""
#include <stddef.h>
#include <stdio.h>
#include "pa_b200.h"
#define F(m) printf(#m " %zu\n", offsetof(pa_block_cache_desc, m))
int main(void) {
  printf("size %zu\n", sizeof(pa_block_cache_desc));
  F(cache); F(scale_block); F(scale_head_stride); F(scale_page_stride); F(row_head_stride); F(row_seq_stride);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_block_cache_desc_layout_matches_the_c_compiler(tmp_path):
    from pa_b200._lib import BlockCacheDesc

    src = tmp_path / "layout.c"
    src.write_text(_LAYOUT_C)
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    c = {k: int(v) for k, v in (ln.split() for ln in lines if ln)}
    assert c.pop("size") == ctypes.sizeof(BlockCacheDesc)
    for name, off in c.items():
        assert getattr(BlockCacheDesc, name).offset == off, name


def good_desc(**kw):
    import pa_b200

    kw = {"layout": "hnd", "kv_format": "e4m3", "paged": True, "max_pages_per_seq": 8, "scale_block": 8, **kw}
    return pa_b200.block_cache_desc(2, 16, 128, (64, 4, 16, 128), **kw)


def test_block_cache_desc_strides():
    import pa_b200

    d = good_desc(rows=200)
    assert (d.cache.kv_dtype, d.cache.page_size, d.cache.max_seq_len) == (6, 16, 128)
    assert (d.scale_block, d.scale_head_stride, d.scale_page_stride) == (8, 2, 8)
    assert (d.row_head_stride, d.row_seq_stride) == (200, 800)
    d = pa_b200.block_cache_desc(2, 16, 64, (5, 33, 4, 64), layout="nhd", kv_format="int8", scale_block=10)
    assert (d.cache.kv_dtype, d.cache.page_size, d.scale_head_stride, d.scale_page_stride) == (7, 33, 4, 16)
    assert good_desc(kv_format=None).cache.kv_dtype == good_desc().cache.q_dtype == 1
    with pytest.raises(ValueError, match="kv_format"):
        good_desc(kv_format="e5m2")
    with pytest.raises(ValueError, match="scale_block"):
        good_desc(scale_block=0)


def change(d, name, value):
    part = d.cache if hasattr(d.cache, name) else d
    setattr(part, name, value)
    return d


@pytest.mark.parametrize("name,value,status,msg", [
    ("q_dtype", 3, 2, "fp16 or bf16"), ("kv_dtype", 2, 2, "query's dtype, fp8 e4m3 or int8"),
    ("head_dim", 96, 2, "64 or 128"), ("q_heads", 18, 1, "multiple of kv heads"), ("q_heads", 68, 2, "at most 16"),
    ("batch", -1, 1, "batch"), ("kv_heads", 0, 1, "kv_heads"), ("scale", float("inf"), 1, "finite"),
    ("k_scale", 0.5, 1, "must be 1"), ("v_scale", float("nan"), 1, "must be 1"),
    ("max_seq_len", -1, 2, "too many keys"), ("max_seq_len", 129, 1, "cover max_seq_len"),
    ("page_size", 0, 1, "page_size"), ("num_pages", 0, 1, "num_pages"), ("max_pages_per_seq", 7, 1, "cover max_seq_len"),
    ("key_stride", 127, 1, "at least head_dim"), ("key_stride", 136, 1, "16 bytes"), ("head_stride", 1 << 50, 1, "range"),
    ("page_stride", 2050 * 4, 1, "16 bytes"), ("scale_block", 0, 1, "scale_block"), ("scale_block", 3, 1, "divide page_size"),
    ("scale_head_stride", 1, 1, "scale strides"), ("scale_page_stride", 0, 1, "scale strides"),
    ("row_head_stride", 127, 1, "row strides"), ("row_seq_stride", -4, 1, "row strides"),
])
def test_library_refuses_bad_descriptors(name, value, status, msg):
    from pa_b200._lib import PaError, check, lib

    n = ctypes.c_size_t(0)
    d = change(good_desc(), name, value)
    with pytest.raises(PaError, match=msg) as err:
        check(lib().pa_cache_decode_workspace_size(ctypes.byref(d), 1, 1, ctypes.byref(n)))
    assert err.value.status == status
    if name not in ("q_heads", "scale"):
        with pytest.raises(PaError, match=msg) as err:
            check(lib().pa_cache_evict_workspace_size(ctypes.byref(d), 1, 10, ctypes.byref(n)))
        assert err.value.status == status
    if not name.startswith("row_"):
        with pytest.raises(PaError):
            check(lib().pa_cache_decode(ctypes.byref(d), *[16] * 11, 1 << 30, None))
    assert n.value == 0


def test_library_refuses_bad_dense_caches():
    from pa_b200._lib import PaError, check, lib

    n = ctypes.c_size_t(0)
    for name, value, msg in (("page_size", 10, "at least max_seq_len"), ("num_pages", 1, "one page per sequence")):
        d = change(good_desc(paged=False, max_seq_len=16), name, value)
        with pytest.raises(PaError, match=msg):
            check(lib().pa_cache_decode_workspace_size(ctypes.byref(d), 0, 0, ctypes.byref(n)))


def test_library_refuses_bad_calls_before_any_launch():
    """Null, misaligned or contradictory arguments; the pointers are never followed."""
    from pa_b200._lib import PaError, check, lib

    L = lib()
    d = good_desc()
    half = good_desc(kv_format=None)

    def decode(desc=d, q=16, k=16, v=16, ks=16, vs=16, bt=16, lens=16, out=16, lse=None, w=None, ws=16, size=1 << 30):
        check(L.pa_cache_decode(ctypes.byref(desc) if desc else None, q, k, v, ks, vs, bt, lens, out, lse, w, ws, size, None))

    for kw, msg in ((dict(desc=None), "null descriptor"), (dict(q=None), "null q or out"), (dict(out=None), "null q or out"),
                    (dict(q=8), "16-byte aligned"), (dict(k=None), "null cache"), (dict(v=24), "16-byte aligned"),
                    (dict(ks=None), "need k_scales"), (dict(desc=half), "have no scales"), (dict(size=8), "workspace smaller"),
                    (dict(ws=8), "workspace must be"), (dict(bt=None), "page_size must be at least")):
        with pytest.raises(PaError, match=msg):
            decode(**kw)

    def append(desc=d, kn=16, vn=16, T=4, strides=(2048, 512, 128), nl=None, k=16, v=16, ks=16, vs=16, bt=16, lens=16,
               w=None, p=None, start=None, lo=None):
        check(L.pa_cache_append(ctypes.byref(desc), kn, vn, T, *strides, nl, k, v, ks, vs, bt, lens, w, p, start, lo, None))

    for kw, msg in ((dict(T=-1), "new_len"), (dict(T=129), "new_len"), (dict(lens=None), "null seq_lens"),
                    (dict(lo=16), "must not be seq_lens"), (dict(kn=None), "null k_new"), (dict(vn=20), "16-byte aligned"),
                    (dict(strides=(2048, 4, 128)), "multiples of 8"), (dict(strides=(-8, 512, 128)), "multiples of 8"),
                    (dict(start=16), "without positions"), (dict(vs=None), "need k_scales"), (dict(k=None), "null cache")):
        with pytest.raises(PaError, match=msg):
            append(**kw)

    def evict(desc=d, k=16, v=16, ks=16, vs=16, bt=16, lens=16, w=16, p=None, nx=None, budget=10, recent=2, sinks=1,
              wo=None, po=None, lo=32, kept=16, ws=16, size=1 << 30):
        check(L.pa_cache_evict(ctypes.byref(desc), k, v, ks, vs, bt, lens, w, p, nx, budget, recent, sinks, wo, po, lo,
                               kept, ws, size, None))

    for kw, msg in ((dict(budget=0), "budget"), (dict(recent=10), "fit the budget"), (dict(sinks=-1), "fit the budget"),
                    (dict(p=16), "need next_positions"), (dict(lens=None), "null seq_lens"), (dict(w=None), "null seq_lens, weights"),
                    (dict(lo=None), "null seq_lens"), (dict(kept=None), "null seq_lens"), (dict(lo=16), "must not be seq_lens"),
                    (dict(ks=None), "need k_scales"), (dict(k=8), "16-byte aligned"), (dict(size=4), "workspace smaller"),
                    (dict(ws=4), "workspace must be")):
        with pytest.raises(PaError, match=msg):
            evict(**kw)


def arrays():
    k = np.zeros((4, 2, 16, 64), np.uint8)
    s = np.ones((4, 2, 2), np.float32)
    return dict(key_cache=k, value_cache=k.copy(), k_scales=s, v_scales=s.copy(), scale_block=8, kv_format="e4m3")


TABLE = np.array([[0, 1], [2, 3]], np.int32)


@pytest.mark.parametrize("kw,msg", [
    (dict(kv_format="fp4"), "kv_format"), (dict(kv_format="int8"), "must be int8"), (dict(kv_format=None), "must be float16"),
    (dict(value_cache=np.zeros((4, 2, 8, 64), np.uint8)), "differ in shape"), (dict(k_scales=None), "need k_scales"),
    (dict(v_scales=np.ones((4, 2, 1))), "scales must have shape"), (dict(scale_block=0), "scale_block"),
    (dict(layout="bhsd"), "layout"), (dict(block_table=TABLE[:1]), "block_table must be"),
    (dict(seq_lens=[1]), "seq_lens must have shape"),
])
def test_numpy_entry_points_refuse_bad_caches(kw, msg):
    import pa_b200

    a = {**arrays(), "seq_lens": np.array([3, 4]), "block_table": TABLE, **kw}
    x = np.zeros((2, 1, 2, 64), np.float16)
    with pytest.raises(ValueError, match=msg):
        pa_b200.cache_append(x, x, **a)
    with pytest.raises(ValueError, match=msg):
        pa_b200.cache_decode(x[:, 0], **a)
    if "seq_lens" not in kw:
        with pytest.raises(ValueError, match=msg):
            pa_b200.cache_evict(**a, weights=np.zeros((2, 2, 32)), budget=2)


def test_numpy_entry_points_refuse_bad_arguments():
    import pa_b200

    a = {**arrays(), "seq_lens": np.array([3, 4]), "block_table": TABLE}
    x = np.zeros((2, 1, 2, 64), np.float16)
    w, p = np.zeros((2, 2, 32), np.float32), np.zeros((2, 2, 32), np.int32)
    for args, kw, msg in (((x.astype(np.float32), x), {}, "float16"), ((x, x[:, :, :1]), {}, "one shape"),
                          ((x[..., :32], x[..., :32]), {}, "heads of"), ((x, x), dict(new_lens=[2, 0]), "in range"),
                          ((x, x), dict(seq_lens=[32, 0]), "32 rows per sequence"), ((x, x), dict(weights=w[:, :, :3]), "weights must be"),
                          ((x, x), dict(positions=p[:1]), "positions must be"), ((x, x), dict(start_positions=[0, 0]), "needs positions"),
                          ((x, x), dict(weights=w, positions=p[:, :, :31]), "differ in shape")):
        with pytest.raises(ValueError, match=msg):
            pa_b200.cache_append(*args, **{**a, **kw})
    for q, kw, msg in ((x, {}, "query must be float16"), (x[:, 0, :, :32], {}, "does not match"), (x[:, 0, :1], {}, "multiple of kv_heads"),
                       (x[:, 0], dict(weights=w[:, :, :2]), "weights must be")):
        with pytest.raises(ValueError, match=msg):
            pa_b200.cache_decode(q, **{**a, **kw})
    for kw, msg in ((dict(budget=0), "budget must be"), (dict(budget=3, recent=2, sinks=2), "budget must be"),
                    (dict(weights=None), "weights must be given"), (dict(weights=w[:, :, :3]), "weights must be"),
                    (dict(positions=p), "need next_positions"), (dict(positions=p[:, :, :30], next_positions=[4, 4]), "differ in shape"),
                    (dict(seq_lens=[33, 0]), "seq_lens must be in"), (dict(seq_lens=3), "one-dimensional")):
        with pytest.raises(ValueError, match=msg):
            pa_b200.cache_evict(**{**a, "weights": w, "budget": 2, **kw})


def test_a_padded_batch_may_be_wider_than_the_cache():
    """new_len above max_seq_len is refused only where every sequence would take all of it (before any
    launch: without new_lens the check comes first, with it the next argument's)."""
    from pa_b200._lib import PaError, check, lib

    d = good_desc()
    for new_lens, new_len, msg in ((None, 129, "new_len"), (16, 129, "null k_new"), (16, (1 << 31) - 1, "null k_new"),
                                   (16, 1 << 31, "new_len"), (16, -1, "new_len")):
        with pytest.raises(PaError, match=msg):
            check(lib().pa_cache_append(ctypes.byref(d), None, 16, new_len, 2048, 512, 128, new_lens, 16, 16, 16, 16, 16, 16,
                                        None, None, None, None, None))


def test_grids_too_large_are_refused_before_any_launch():
    """Products of accepted sizes that pass 64 bits, or a grid's limit in the second launch only."""
    from pa_b200._lib import PaError, check, lib

    L, n = lib(), ctypes.c_size_t(0)
    d = good_desc(paged=True, max_pages_per_seq=1 << 20, scale_block=1)
    for name, value in (("batch", 65535 * 1024), ("kv_heads", 65535), ("page_size", 2047), ("max_seq_len", (1 << 31) - 65537)):
        change(d, name, value)
    change(change(d, "scale_head_stride", 1 << 20), "scale_page_stride", 1 << 20)
    change(change(d, "row_head_stride", 1 << 31), "row_seq_stride", 1 << 31)
    change(d, "max_pages_per_seq", 1 << 21)
    for new_lens, new_len in ((None, 1 << 20), (16, (1 << 31) - 1)):
        with pytest.raises(PaError, match="grid too large") as err:
            check(L.pa_cache_append(ctypes.byref(d), 16, 16, new_len, 2048, 512, 128, new_lens, 16, 16, 16, 16, 16, 16,
                                    None, None, None, None, None))
        assert err.value.status == 2
    change(change(d, "batch", 64), "kv_heads", 128)
    with pytest.raises(PaError, match="grid too large"):
        check(L.pa_cache_evict_workspace_size(ctypes.byref(d), 1, 1 << 30, ctypes.byref(n)))
    assert n.value == 0


def test_numpy_entry_points_refuse_numbers_that_int32_does_not_hold():
    """2^32 + 3 is no length of 3, and 3.5 none either."""
    import pa_b200

    a = {**arrays(), "block_table": TABLE}
    x, w = np.zeros((2, 1, 2, 64), np.float16), np.zeros((2, 2, 32), np.float32)
    lens = np.array([3, 4])
    for bad in ([2 ** 32 + 3, 4], [3.5, 4.0], np.array([2 ** 63 + 3, 4], np.uint64), [float("nan"), 1.0]):
        for call in (lambda: pa_b200.cache_append(x, x, seq_lens=bad, **a), lambda: pa_b200.cache_append(x, x, seq_lens=lens, new_lens=bad, **a),
                     lambda: pa_b200.cache_decode(x[:, 0], seq_lens=bad, **a),
                     lambda: pa_b200.cache_evict(seq_lens=bad, weights=w, budget=2, **a),
                     lambda: pa_b200.cache_evict(seq_lens=lens, weights=w, budget=2, next_positions=bad, **a),
                     lambda: pa_b200.cache_append(x, x, seq_lens=lens, positions=np.full((2, 2, 32), bad[0]), **a)):
            with pytest.raises(ValueError, match="32 bits"):
                call()


def test_table_entries_that_int32_does_not_hold_are_no_pages():
    from pa_b200.blockcache import _table

    t = _table(np.array([[0, 2 ** 32 + 1], [2 ** 63 - 1, -(2 ** 40)]]))
    assert t.dtype == np.int32 and t.tolist() == [[0, -1], [-1, -1]]
    assert _table(np.array([[7, 2 ** 64 - 1]], np.uint64)).tolist() == [[7, -1]]
    with pytest.raises(ValueError, match="32 bits"):
        _table([[0.5, 1.0]])


def test_lengths_are_not_written_over_what_the_call_reads():
    """seq_lens_out in the memory of new_lens, start_positions or next_positions: other blocks read those."""
    from pa_b200._lib import PaError, check, lib

    L, d = lib(), good_desc()

    def append(new_lens, start, lens_out):
        check(L.pa_cache_append(ctypes.byref(d), 16, 16, 4, 2048, 512, 128, new_lens, 16, 16, 16, 16, 16, 32, None, 16, start,
                                lens_out, None))

    for args in ((48, None, 48), (48, 64, 64)):
        with pytest.raises(PaError, match="seq_lens_out must not be") as err:
            append(*args)
        assert err.value.status == 1
    with pytest.raises(PaError, match="seq_lens_out must not be"):
        check(L.pa_cache_evict(ctypes.byref(d), 16, 16, 16, 16, 16, 16, 16, 16, 48, 10, 2, 1, None, None, 48, 16, 16, 1 << 30, None))
