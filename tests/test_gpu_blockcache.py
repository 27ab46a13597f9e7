"""Block-scaled cache on the GPU against the float64 oracle of oracle/blockcache.py.

Append and evict are exact: their scales are powers of two, so every value is
rounded once and codes, scales, rows and positions must equal the oracle's bit
for bit, and everything they do not own must be left as it was.

Decode bounds (u = half a step of the output type: fp16 2^-11, bf16 2^-8):
  |out - want|  <= u |want| + (2^-11 + 2^-16) sum_j p_j |v_j| + 2^-25
                   final rounding; probabilities rounded to fp16 for the
                   products, relative to the largest of their tile; fp32 sums;
                   half the smallest fp16 subnormal;
  |lse - want|  <= 2^-18 mag + 2^-20 (1 + |lse|),  mag = max_j scale sum_d |q_d k_jd|
                   at most 128 fp32 additions of partial sums below mag, each
                   within 2^-24 of it (2^-17 at the very worst; their signs
                   differ), then exponentials and a logarithm to about 2^-22;
  |w - want|    <= added * (2 dlse + 2^-18) + 2^-23 (|w| + 1):  a weight is exp(s - lse).
Rows and blocks behind a sequence hold NaN, in int8 a NaN scale.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle.blockcache import append_reference, decode_reference, evict_reference, need_scale, round8
from oracle.kvcache import e4m3_to_float, float_to_e4m3

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def to_hnd(x, layout):
    return x if layout == "hnd" else np.ascontiguousarray(np.swapaxes(x, 1, 2))


def codes_of(x, fmt):
    """The stored array of element values: bytes in 8 bits, fp16 otherwise."""
    if fmt == "e4m3":
        return float_to_e4m3(x)
    return x.astype(np.int8 if fmt == "int8" else np.float16)


def values_of(a, fmt):
    return e4m3_to_float(a) if fmt == "e4m3" else a.astype(np.float64)


class Cache:
    """A random paged (or dense) cache in oracle form; everything not in use is NaN."""

    def __init__(self, rng, B, H, D, page, block, fmt, lens, rows, paged=True, odd_scales=False):
        self.fmt, self.block, self.lens = fmt, block, np.asarray(lens, np.int32)
        per = -(-rows // page)
        if paged:
            pages = B * per + 2
            self.table = rng.permutation(pages)[:B * per].reshape(B, per).astype(np.int32)
        else:
            pages, self.table = B, None
            assert per == 1
        nan = np.nan if fmt != "int8" else 77.0
        self.k, self.v = np.full((pages, H, page, D), nan), np.full((pages, H, page, D), nan)
        self.ks = self.vs = None
        if fmt is not None:
            nblk = -(-page // block)
            self.ks, self.vs = np.full((pages, H, nblk), np.nan), np.full((pages, H, nblk), np.nan)
        for b in range(B):
            for r0 in range(0, int(lens[b]), block or page):
                r1 = min(int(lens[b]), r0 + (block or page))
                p, at = (b, r0) if self.table is None else (int(self.table[b, r0 // page]), r0 % page)
                for h in range(H):
                    for c, s in ((self.k, self.ks), (self.v, self.vs)):
                        x = rng.standard_normal((r1 - r0, D)) * np.exp(0.7 * rng.standard_normal())
                        if fmt is None:
                            c[p, h, at:at + r1 - r0] = x.astype(np.float16)
                            continue
                        sc = need_scale(x, fmt) * (np.float32(1 + rng.random()) if odd_scales else 1.0)
                        c[p, h, at:at + r1 - r0] = round8(x / sc, fmt)
                        s[p, h, at // block] = np.float32(sc)

    def arrays(self, layout):
        kw = dict(key_cache=codes_of(to_hnd(self.k, layout), self.fmt), value_cache=codes_of(to_hnd(self.v, layout), self.fmt),
                  block_table=self.table, layout=layout, kv_format=self.fmt)
        if self.fmt is not None:
            kw.update(k_scales=self.ks.astype(np.float32), v_scales=self.vs.astype(np.float32), scale_block=self.block)
        return kw

    def parts(self):
        return dict(ks=self.ks, vs=self.vs, table=self.table, block=self.block)

    def check_equal(self, got, layout):
        for name, want in (("key_cache", self.k), ("value_cache", self.v)):
            np.testing.assert_array_equal(values_of(to_hnd(getattr(got, name), layout), self.fmt), want)
        if self.fmt is not None:
            np.testing.assert_array_equal(got.k_scales, self.ks.astype(np.float32))
            np.testing.assert_array_equal(got.v_scales, self.vs.astype(np.float32))


def check_decode(ref, out, lse, weights=None, before=None, u=U["f16"]):
    out = out.astype(np.float64)
    assert np.isfinite(out).all()
    tol = u * np.abs(ref["out"]) + (2.0 ** -11 + 2.0 ** -16) * ref["pv"] + 2.0 ** -25
    assert (np.abs(out - ref["out"]) <= tol).all(), float((np.abs(out - ref["out"]) / tol).max())
    live = np.isfinite(ref["lse"])
    assert np.array_equal(np.isneginf(lse), ~live)
    dl = 2.0 ** -18 * ref["mag"] + 2.0 ** -20 * (1 + np.abs(np.where(live, ref["lse"], 0)))
    off = np.abs(lse[live] - ref["lse"][live])
    assert (off <= dl[live]).all(), float((off / dl[live]).max())
    if weights is not None:
        G = lse.shape[1] // weights.shape[1]
        d = dl.reshape(lse.shape[0], -1, G).max(-1)[..., None]
        tol = (ref["weights"] - before) * (2 * d + 2.0 ** -18) + 2.0 ** -23 * (np.abs(ref["weights"]) + 1)
        assert (np.abs(weights - ref["weights"]) <= tol).all()


FORMATS = ["e4m3", "int8", None]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,page,block,D,H,T", [
    ("hnd", 16, 16, 128, 2, 1), ("nhd", 32, 8, 64, 3, 50), ("hnd", 64, 32, 128, 1, 200), ("nhd", 5, 5, 64, 2, 23),
    ("hnd", 12, 4, 128, 2, 33), ("hnd", 8, 1, 64, 2, 9), ("nhd", 128, 128, 128, 2, 140),
])
def test_append_equals_the_oracle(fmt, layout, page, block, D, H, T):
    import pa_b200

    rng = np.random.default_rng(page * 100 + T)
    lens = np.array([0, 1, page, page + block // 2 + 1, 2 * page - 1], np.int32)
    B, rows = len(lens), 2 * page + T
    c = Cache(rng, B, H, D, page, block, fmt, lens, rows)
    x = (rng.standard_normal((2, B, T, H, D)) * np.exp(rng.standard_normal((2, B, T, H, 1)))).astype(np.float16)
    new = np.array([T, T // 2, 0, T, max(T - 1, 1)], np.int32)
    w = rng.random((B, H, rows)).astype(np.float32)
    p = rng.integers(0, 1000, (B, H, rows)).astype(np.int32)
    start = rng.integers(0, 10000, B).astype(np.int32)
    a = c.arrays(layout)
    keep = {n: np.copy(v) for n, v in a.items() if isinstance(v, np.ndarray)}
    got = pa_b200.cache_append(x[0], x[1], seq_lens=lens, new_lens=new, weights=w, positions=p, start_positions=start, **a)
    for n, v in keep.items():
        np.testing.assert_array_equal(a[n], v)          # inputs are never changed
    want_w, want_p = w.astype(np.float64), p.copy()
    want_len = append_reference(x[0], x[1], c.k, c.v, lens, new, fmt=fmt, weights=want_w, positions=want_p, start=start, **c.parts())
    c.check_equal(got, layout)
    np.testing.assert_array_equal(got.seq_lens, want_len)
    np.testing.assert_array_equal(got.weights, want_w.astype(np.float32))
    np.testing.assert_array_equal(got.positions, want_p)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_of_zeros_infinities_nan_and_extremes(fmt):
    import pa_b200

    rng = np.random.default_rng(5)
    B, H, D, page = 1, 1, 64, 16
    c = Cache(rng, B, H, D, page, 8, fmt, [3], 64)
    x = rng.standard_normal((2, 1, 40, H, D)).astype(np.float16)
    x[0, 0, 2, 0, :4] = [np.inf, -np.inf, np.nan, 65504]
    x[0, 0, 5:13] = 0.0                                  # a whole block of zeros
    x[0, 0, 13:21] = np.float16(2.0 ** -24)              # the smallest subnormal
    x[0, 0, 21:29] = np.nan                              # a block without a finite value
    x[1, 0, 30, 0, 7] = np.inf
    got = pa_b200.cache_append(x[0], x[1], seq_lens=[3], **c.arrays("hnd"))
    append_reference(x[0], x[1], c.k, c.v, [3], [40], fmt=fmt, **c.parts())
    c.check_equal(got, "hnd")


def test_append_one_token_at_a_time_equals_the_oracle():
    import pa_b200

    rng = np.random.default_rng(6)
    c = Cache(rng, 2, 2, 64, 16, 16, "e4m3", [0, 7], 48)
    lens = c.lens
    for _ in range(20):
        x = (rng.standard_normal((2, 2, 1, 2, 64)) * np.exp(2 * rng.standard_normal())).astype(np.float16)
        got = pa_b200.cache_append(x[0], x[1], seq_lens=lens, **c.arrays("hnd"))
        append_reference(x[0], x[1], c.k, c.v, lens, [1, 1], fmt="e4m3", **c.parts())
        c.check_equal(got, "hnd")
        lens = got.seq_lens
    assert list(lens) == [20, 27]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,page,block,D,Hq,H,odd", [
    ("hnd", 16, 16, 128, 8, 2, False), ("nhd", 32, 8, 64, 16, 2, False), ("hnd", 64, 64, 128, 4, 4, True),
    ("nhd", 16, 4, 128, 16, 1, True), ("hnd", 5, 5, 64, 3, 1, False), ("hnd", 1, 1, 64, 6, 2, True),
    ("nhd", 100, 20, 128, 9, 1, False), ("hnd", 128, 128, 64, 12, 1, False),
])
def test_decode_equals_the_oracle(fmt, layout, page, block, D, Hq, H, odd):
    import pa_b200

    rng = np.random.default_rng(page * 10 + Hq)
    lens = np.array([0, 1, 31, 33, page, 700, 1500], np.int32)
    B, rows = len(lens), 1500
    c = Cache(rng, B, H, D, page, block, fmt, lens, rows, odd_scales=odd)
    q = rng.standard_normal((B, Hq, D)).astype(np.float16)
    w = rng.random((B, H, rows)).astype(np.float32)
    out, lse, got_w = pa_b200.cache_decode(q, seq_lens=lens, weights=w, return_lse=True, **c.arrays(layout))
    ref = decode_reference(q, c.k, c.v, lens, weights=w, **c.parts())
    check_decode(ref, out, lse, got_w, w)
    assert (out[0] == 0).all()
    for b, n in enumerate(lens):
        np.testing.assert_array_equal(got_w[b, :, n:], w[b, :, n:])
    again = pa_b200.cache_decode(q, seq_lens=lens, **c.arrays(layout))
    np.testing.assert_array_equal(again, out)            # the weights do not change the output


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("B,S,Hq,H,D", [(1, 1, 1, 1, 64), (1, 20011, 8, 8, 128), (1, 70001, 4, 1, 64), (40, 77, 32, 8, 128)])
def test_decode_dense_cache_of_one_length(fmt, B, S, Hq, H, D):
    """No block table, no lengths; scale blocks that do not divide the sequence."""
    import pa_b200

    rng = np.random.default_rng(S)
    c = Cache(rng, B, H, D, S, min(S, 48) if fmt else None, fmt, [S] * B, S, paged=False)
    q = rng.standard_normal((B, Hq, D)).astype(np.float16)
    w = np.zeros((B, H, S + 3), np.float32)
    out, lse, got_w = pa_b200.cache_decode(q, weights=w, return_lse=True, scale=0.2, **c.arrays("hnd"))
    ref = decode_reference(q, c.k, c.v, [S] * B, scale=0.2, weights=w, **c.parts())
    check_decode(ref, out, lse, got_w, w)
    assert (got_w[..., S:] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_with_a_sink_token(fmt):
    """One key takes almost all the weight and its values are zero: the others' shares still count."""
    import pa_b200

    rng = np.random.default_rng(8)
    B, H, D, S = 1, 1, 64, 4000
    c = Cache(rng, B, H, D, 16, 1, fmt, [S], S)
    q = rng.standard_normal((B, 2, D)).astype(np.float16)
    p, at = c.table[0, 0], 0
    sink = q[0, 0] / np.linalg.norm(q[0, 0].astype(np.float64)) * 8.0
    if fmt is None:
        c.k[p, 0, at] = sink.astype(np.float16)
    else:
        c.ks[p, 0, at] = need_scale(sink, fmt)
        c.k[p, 0, at] = round8(sink / c.ks[p, 0, at], fmt)
        c.vs[p, 0, at] = 2.0 ** -100
    c.v[p, 0, at] = 0.0
    out, lse = pa_b200.cache_decode(q, seq_lens=[S], return_lse=True, **c.arrays("hnd"))
    ref = decode_reference(q, c.k, c.v, [S], **c.parts())
    check_decode(ref, out, lse)


def test_decode_reads_no_row_behind_the_length_inside_a_block():
    """Rows behind the length share the block's scale; whatever they hold is not used."""
    import pa_b200

    rng = np.random.default_rng(9)
    for fmt, bad in (("e4m3", np.nan), ("int8", -127.0), (None, np.inf)):
        c = Cache(rng, 2, 2, 128, 64, 64, fmt, [37, 65], 128)
        q = rng.standard_normal((2, 8, 128)).astype(np.float16)
        a = pa_b200.cache_decode(q, seq_lens=[37, 65], **c.arrays("hnd"))
        for b, n in ((0, 37), (1, 1)):
            page = c.table[b, 0 if b == 0 else 1]
            c.k[page, :, n:] = bad
            c.v[page, :, n:] = bad
        np.testing.assert_array_equal(pa_b200.cache_decode(q, seq_lens=[37, 65], **c.arrays("hnd")), a)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,page,block,D,H,budget,recent,sinks", [
    ("hnd", 16, 16, 128, 2, 64, 8, 2), ("nhd", 32, 8, 64, 3, 100, 20, 4), ("hnd", 12, 4, 128, 1, 1, 0, 0),
    ("nhd", 5, 5, 64, 2, 33, 33, 0), ("hnd", 64, 64, 64, 2, 130, 0, 1), ("hnd", 8, 1, 128, 2, 77, 10, 3),
    ("hnd", 16, 8, 64, 2, 5000, 100, 4),
])
def test_evict_equals_the_oracle(fmt, layout, page, block, D, H, budget, recent, sinks):
    import pa_b200

    rng = np.random.default_rng(page * 10 + budget)
    big = budget >= 5000
    lens = np.array([9001] if big else [0, 1, budget, budget + 1, 3 * budget + 7, 300 + budget], np.int32)
    B, rows = len(lens), int(lens.max())
    c = Cache(rng, B, H, D, page, block, fmt, lens, rows)
    w = np.round(rng.exponential(size=(B, H, rows)) * 4).astype(np.float32) / 4     # many ties
    w[:, :, 3::11] = np.nan
    w[:, :, 5::13] = -0.0
    w[:, :, 6::17] = -1.5
    pos = np.tile(np.sort(rng.choice(2 * rows + 5, rows, replace=False)).astype(np.int32), (B, H, 1))
    pos[:, :, :sinks] = np.arange(sinks)
    nxt = np.array([pos[b, 0, n - 1] + 1 if n else 0 for b, n in enumerate(lens)], np.int32)
    got = pa_b200.cache_evict(seq_lens=lens, weights=w, budget=budget, recent=recent, sinks=sinks, positions=pos,
                              next_positions=nxt, **c.arrays(layout))
    want_w, want_p = w.copy(), pos.copy()
    want_len, kept = evict_reference(c.k, c.v, lens, want_w, budget, recent=recent, sinks=sinks, positions=want_p,
                                     next_positions=nxt, fmt=fmt, **c.parts())
    np.testing.assert_array_equal(got.kept, kept)
    np.testing.assert_array_equal(got.seq_lens, want_len)
    np.testing.assert_array_equal(got.weights, want_w)
    np.testing.assert_array_equal(got.positions, want_p)
    c.check_equal(got, layout)


def test_evict_without_positions_and_with_equal_weights():
    """All weights equal: the lowest rows stay, apart from the newest; a row's position is its index."""
    import pa_b200

    rng = np.random.default_rng(11)
    c = Cache(rng, 2, 2, 64, 16, 16, "int8", [90, 50], 96)
    w = np.ones((2, 2, 96), np.float32)
    got = pa_b200.cache_evict(seq_lens=c.lens, weights=w, budget=40, recent=10, **c.arrays("hnd"))
    for b, n in enumerate(c.lens):
        assert (got.kept[b] == np.r_[0:30, n - 10:n]).all()
    assert list(got.seq_lens) == [40, 40]


@pytest.mark.parametrize("over", [1, 2, 7, 8, 9])
@pytest.mark.parametrize("fmt", FORMATS)
def test_evict_of_a_few_rows(fmt, over):
    """A budget kept up step by step: few rows over it, ties, protected rows among the smallest."""
    import pa_b200

    rng = np.random.default_rng(over)
    B, H, budget = 4, 3, 261
    lens = np.array([budget + over, budget + 1, budget, budget + over], np.int32)
    c = Cache(rng, B, H, 64, 16, 8, fmt, lens, budget + over)
    w = np.round(rng.exponential(size=(B, H, budget + over)) * 30).astype(np.float32) / 30
    w[0, 0] = 1.0                                       # all equal: the last unprotected rows go
    w[1, 1, 5] = np.nan
    w[3, :, budget:] = 50.0                             # every row behind the budget stays
    w[3, 2, 250:258] = w[3, 2, 3]
    for recent, sinks in ((0, 0), (20, 4), (255, 6)):
        d = Cache.__new__(Cache)
        d.__dict__.update({k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.__dict__.items()})
        got = pa_b200.cache_evict(seq_lens=lens, weights=w, budget=budget, recent=recent, sinks=sinks, **d.arrays("nhd"))
        want_w = w.copy()
        want_len, kept = evict_reference(d.k, d.v, lens, want_w, budget, recent=recent, sinks=sinks, fmt=fmt, **d.parts())
        np.testing.assert_array_equal(got.kept, kept)
        np.testing.assert_array_equal(got.weights, want_w)
        np.testing.assert_array_equal(got.seq_lens, want_len)
        d.check_equal(got, "nhd")


@pytest.mark.parametrize("fmt,B,H,n,budget,page,block", [
    ("int8", 1, 1, 140001, 20003, 64, 64),     # a cluster whose threads hold their rows in two rounds
    (None, 40, 2, 17001, 16990, 1024, 1024),   # one CTA a head, three rounds
    (None, 2, 1, 70000, 69990, 1024, 1024), ("e4m3", 3, 2, 30000, 1000, 16, 16),
])
def test_evict_of_long_sequences(fmt, B, H, n, budget, page, block):
    import pa_b200

    rng = np.random.default_rng(n)
    lens = np.array([n - 7 * (b % 3) for b in range(B)], np.int32)
    c = Cache(rng, B, H, 64, page, block, fmt, lens, n)
    w = np.exp(2 * rng.standard_normal((B, H, n))).astype(np.float32)
    w[:, :, ::5] = np.float32(0.25)            # ties across threads, warps and rounds
    got = pa_b200.cache_evict(seq_lens=lens, weights=w, budget=budget, recent=100, sinks=3, **c.arrays("hnd"))
    want_w = w.copy()
    want_len, kept = evict_reference(c.k, c.v, lens, want_w, budget, recent=100, sinks=3, fmt=fmt, **c.parts())
    np.testing.assert_array_equal(got.kept, kept)
    np.testing.assert_array_equal(got.weights, want_w)
    np.testing.assert_array_equal(got.seq_lens, want_len)
    c.check_equal(got, "hnd")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_dense_cache_append_decode_evict(fmt, layout):
    """No block table: page b is sequence b, and scale blocks need not divide it."""
    import pa_b200

    rng = np.random.default_rng(41)
    B, Hq, H, D, page, block, T, budget = 3, 6, 2, 64, 157, 12, 30, 70
    lens = np.array([100, 0, 127], np.int32)
    c = Cache(rng, B, H, D, page, block, fmt, lens, page, paged=False)
    x = rng.standard_normal((2, B, T, H, D)).astype(np.float16)
    got = pa_b200.cache_append(x[0], x[1], seq_lens=lens, **c.arrays(layout))
    append_reference(x[0], x[1], c.k, c.v, lens, [T] * B, fmt=fmt, **c.parts())
    c.check_equal(got, layout)
    lens = got.seq_lens
    q = rng.standard_normal((B, Hq, D)).astype(np.float16)
    before = rng.random((B, H, page)).astype(np.float32)
    out, lse, w = pa_b200.cache_decode(q, seq_lens=lens, weights=before, return_lse=True, **c.arrays(layout))
    check_decode(decode_reference(q, c.k, c.v, lens, weights=before, **c.parts()), out, lse, w, before)
    want_w = w.copy()
    got = pa_b200.cache_evict(seq_lens=lens, weights=w, budget=budget, recent=9, sinks=2, **c.arrays(layout))
    want_len, kept = evict_reference(c.k, c.v, lens, want_w, budget, recent=9, sinks=2, fmt=fmt, **c.parts())
    np.testing.assert_array_equal(got.kept, kept)
    np.testing.assert_array_equal(got.weights, want_w)
    c.check_equal(got, layout)


def test_a_budgeted_serving_loop():
    """Prompt, then tokens: append, decode with weights, evict when over budget, against the oracle
    (which takes the device's own weights, so a close call in the choice cannot split the two)."""
    import pa_b200

    rng = np.random.default_rng(12)
    for fmt in FORMATS:
        B, Hq, H, D, page, block, budget = 3, 8, 2, 64, 16, 8, 60
        rows = 112
        c = Cache(rng, B, H, D, page, block, fmt, [0, 0, 0], rows)
        w, pos = np.zeros((B, H, rows), np.float32), np.zeros((B, H, rows), np.int32)
        lens, nxt = np.zeros(B, np.int32), np.zeros(B, np.int32)
        for step in range(30):
            T = 90 if step == 0 else 3
            new = np.array([T, T - 1, (T + 1) // 2], np.int32)
            x = rng.standard_normal((2, B, T, H, D)).astype(np.float16)
            got = pa_b200.cache_append(x[0], x[1], seq_lens=lens, new_lens=new, weights=w, positions=pos,
                                       start_positions=nxt, **c.arrays("hnd"))
            append_reference(x[0], x[1], c.k, c.v, lens, new, fmt=fmt, **c.parts())
            c.check_equal(got, "hnd")
            lens, w, pos, nxt = got.seq_lens, got.weights, got.positions, nxt + new
            q = rng.standard_normal((B, Hq, D)).astype(np.float16)
            before = w
            out, lse, w = pa_b200.cache_decode(q, seq_lens=lens, weights=w, return_lse=True, **c.arrays("hnd"))
            check_decode(decode_reference(q, c.k, c.v, lens, weights=before, **c.parts()), out, lse, w, before)
            want_w, want_p = w.copy(), pos.copy()
            got = pa_b200.cache_evict(seq_lens=lens, weights=w, budget=budget, recent=16, sinks=2, positions=pos,
                                      next_positions=nxt, **c.arrays("hnd"))
            want_len, kept = evict_reference(c.k, c.v, lens, want_w, budget, recent=16, sinks=2, positions=want_p,
                                             next_positions=nxt, fmt=fmt, **c.parts())
            np.testing.assert_array_equal(got.kept, kept)
            np.testing.assert_array_equal(got.positions, want_p)
            c.check_equal(got, "hnd")
            lens, w, pos = got.seq_lens, got.weights, got.positions
        assert lens.max() == budget


def test_bad_pages_and_lengths_are_reported_and_harmless():
    import pa_b200
    from pa_b200._lib import PaError

    rng = np.random.default_rng(13)
    c = Cache(rng, 2, 2, 64, 16, 16, "e4m3", [40, 40], 64)
    a = c.arrays("hnd")
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    x = rng.standard_normal((2, 3, 2, 64)).astype(np.float16)
    w = rng.random((2, 2, 64)).astype(np.float32)
    for bad in (10 ** 6, -1):
        t = a["block_table"].copy()
        t[1, 2] = bad
        b = {**a, "block_table": t}
        for call in (lambda: pa_b200.cache_decode(q, seq_lens=[40, 40], **b),
                     lambda: pa_b200.cache_append(x, x, seq_lens=[40, 40], **b),
                     lambda: pa_b200.cache_evict(seq_lens=[40, 40], weights=w, budget=20, recent=8, **b)):
            with pytest.raises(PaError, match="block-table entry") as err:
                call()
            assert err.value.status == 1
    with pytest.raises(PaError, match="sequence length"):
        pa_b200.cache_decode(q, seq_lens=[40, 41], max_seq_len=40, **a)
    with pytest.raises(PaError, match="sequence length"):
        pa_b200.cache_decode(q, seq_lens=[-1, 40], max_seq_len=40, **a)
    out = pa_b200.cache_decode(q, seq_lens=[40, 40], **a)      # and the device goes on
    ref = decode_reference(q, c.k, c.v, [40, 40], **c.parts())
    assert np.abs(out - ref["out"]).max() < 1e-2


def test_table_entries_behind_the_rows_in_use_may_hold_anything():
    import pa_b200

    rng = np.random.default_rng(14)
    c = Cache(rng, 2, 2, 64, 16, 8, "e4m3", [40, 17], 200)
    a = c.arrays("hnd")
    t = a["block_table"].copy()
    t[0, 3:], t[1, 2:] = -7, 10 ** 8
    b = {**a, "block_table": t}
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    w = rng.random((2, 2, 200)).astype(np.float32)
    for x, y in zip(pa_b200.cache_decode(q, seq_lens=[40, 17], weights=w, max_seq_len=200, **a),
                    pa_b200.cache_decode(q, seq_lens=[40, 17], weights=w, max_seq_len=200, **b)):
        np.testing.assert_array_equal(x, y)
    x = rng.standard_normal((2, 8, 2, 64)).astype(np.float16)
    got, want = (pa_b200.cache_append(x, x, seq_lens=[40, 17], **d) for d in (b, a))
    np.testing.assert_array_equal(got.key_cache, want.key_cache)
    np.testing.assert_array_equal(got.k_scales, want.k_scales)
    got = pa_b200.cache_evict(seq_lens=[40, 17], weights=w, budget=11, recent=4, **b)
    want = pa_b200.cache_evict(seq_lens=[40, 17], weights=w, budget=11, recent=4, **a)
    np.testing.assert_array_equal(got.key_cache, want.key_cache)
    np.testing.assert_array_equal(got.kept, want.kept)


# ------------------------------------------------------- device pointers (PyTorch tensors)

class OnDevice:
    """A cache on the GPU in PyTorch tensors, for the *_device entry points."""

    def __init__(self, c, layout, q_dtype="f16"):
        import torch

        self.c, self.layout = c, layout
        t16 = torch.float16 if q_dtype == "f16" else torch.bfloat16

        def up(x):
            x = to_hnd(x, layout)
            if c.fmt is None:
                return torch.from_numpy(x).to("cuda", t16)
            return torch.from_numpy(codes_of(x, c.fmt).view(np.uint8)).cuda()

        self.k, self.v = up(c.k), up(c.v)
        self.ks = self.vs = None
        if c.fmt is not None:
            self.ks, self.vs = (torch.from_numpy(s.astype(np.float32)).cuda() for s in (c.ks, c.vs))
        self.table = None if c.table is None else torch.from_numpy(c.table).cuda()
        self.lens = torch.from_numpy(c.lens).cuda()

    def kw(self):
        ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        return dict(k_scales_ptr=ptr(self.ks), v_scales_ptr=ptr(self.vs), block_table_ptr=ptr(self.table))

    def desc(self, Hq, rows, q_dtype="f16"):
        import pa_b200

        c = self.c
        return pa_b200.block_cache_desc(
            len(c.lens), Hq, c.k.shape[3], tuple(self.k.shape), layout=self.layout, q_dtype=q_dtype, kv_format=c.fmt,
            paged=c.table is not None, max_pages_per_seq=0 if c.table is None else c.table.shape[1], max_seq_len=rows,
            scale_block=c.block if c.fmt else None, rows=rows)

    def values(self, x):
        x = x.cpu()
        if self.c.fmt is None:
            x = x.double().numpy()
        else:
            x = values_of(x.numpy().view(np.int8 if self.c.fmt == "int8" else np.uint8), self.c.fmt)
        return to_hnd(x, self.layout)

    def check_equal(self):
        np.testing.assert_array_equal(self.values(self.k), self.c.k)
        np.testing.assert_array_equal(self.values(self.v), self.c.v)
        if self.ks is not None:
            np.testing.assert_array_equal(self.ks.cpu().numpy(), self.c.ks.astype(np.float32))
            np.testing.assert_array_equal(self.vs.cpu().numpy(), self.c.vs.astype(np.float32))


class On:
    """A stream by its handle, as the entry points take it."""

    def __init__(self, stream):
        self.handle = stream.cuda_stream


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,Hq,H,layout", [(128, 8, 2, "nhd"), (64, 16, 1, "hnd")])
def test_bf16_append_decode_evict_on_device_pointers(fmt, D, Hq, H, layout):
    """bf16 tokens and queries, strided new tokens, a scratch pool instead of a workspace, in-place eviction."""
    import pa_b200
    import torch

    rng = np.random.default_rng(D + Hq)
    lens, page, block, T, rows, budget = [37, 0, 500], 16, 8, 21, 560, 300
    c = Cache(rng, 3, H, D, page, block, fmt, lens, rows)
    if fmt is None:  # values that bf16 holds
        for x in (c.k, c.v):
            x[:] = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    d = OnDevice(c, layout, "bf16")
    desc = d.desc(Hq, rows, "bf16")
    x = torch.from_numpy(rng.standard_normal((3, H, T, 2, D + 8))).to("cuda", torch.bfloat16)
    kn, vn = x[..., 0, :D], x[..., 1, :D]                      # (batch, head, token, D) inside a wider array
    w = torch.from_numpy(rng.random((3, H, rows)).astype(np.float32)).cuda()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda").expand(3, H, rows).contiguous()
    lens2 = torch.empty_like(d.lens)
    pa_b200.cache_append_device(desc, kn.data_ptr(), vn.data_ptr(), T, d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(),
                                strides=(kn.stride(0), kn.stride(2), kn.stride(1)), weights_ptr=w.data_ptr(),
                                positions_ptr=pos.data_ptr(), seq_lens_out_ptr=lens2.data_ptr(), **d.kw())
    ref_w = w.cpu().numpy()
    new = lambda y: y.transpose(1, 2).double().cpu().numpy()  # noqa: E731
    append_reference(new(kn), new(vn), c.k, c.v, lens, [T] * 3, fmt=fmt, **c.parts())
    d.check_equal()
    assert lens2.tolist() == [58, 21, 521]
    q = torch.from_numpy(rng.standard_normal((3, Hq, D))).to("cuda", torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((3, Hq), device="cuda")
    pa_b200.cache_decode_device(desc, q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(),
                                seq_lens_ptr=lens2.data_ptr(), lse_ptr=lse.data_ptr(), weights_ptr=w.data_ptr(), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, lens2.tolist(), weights=ref_w, **c.parts())
    check_decode(ref, out.float().cpu().numpy(), lse.cpu().numpy(), w.cpu().numpy(), ref_w, u=U["bf16"])
    lens3, kept = torch.empty_like(lens2), torch.empty((3, H, budget), dtype=torch.int32, device="cuda")
    want_w, want_p = w.cpu().numpy(), pos.cpu().numpy()
    pa_b200.cache_evict_device(desc, d.k.data_ptr(), d.v.data_ptr(), lens2.data_ptr(), w.data_ptr(), budget, lens3.data_ptr(),
                               kept.data_ptr(), recent=64, sinks=4, positions_ptr=pos.data_ptr(), next_positions_ptr=lens2.data_ptr(),
                               weights_out_ptr=w.data_ptr(), positions_out_ptr=pos.data_ptr(), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    want_len, want_kept = evict_reference(c.k, c.v, lens2.tolist(), want_w, budget, recent=64, sinks=4, positions=want_p,
                                          next_positions=lens2.tolist(), fmt=fmt, **c.parts())
    np.testing.assert_array_equal(kept.cpu().numpy(), want_kept)
    np.testing.assert_array_equal(w.cpu().numpy(), want_w)
    np.testing.assert_array_equal(pos.cpu().numpy(), want_p)
    assert lens3.tolist() == list(want_len)
    d.check_equal()


def test_bf16_cache_with_values_near_the_end_of_the_range():
    import pa_b200
    import torch

    rng = np.random.default_rng(17)
    c = Cache(rng, 2, 1, 64, 16, 16, None, [40, 3], 48)
    for x in (c.k, c.v):
        x[:] = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    c.v *= 2.0 ** 120                                   # up to about 5e36: finite in bf16 and fp32
    d = OnDevice(c, "hnd", "bf16")
    q = torch.from_numpy(rng.standard_normal((2, 4, 64))).to("cuda", torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((2, 4), device="cuda")
    pa_b200.cache_decode_device(d.desc(4, 48, "bf16"), q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(),
                                seq_lens_ptr=d.lens.data_ptr(), lse_ptr=lse.data_ptr(), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, [40, 3], **c.parts())
    check_decode(ref, out.double().cpu().numpy(), lse.cpu().numpy(), u=U["bf16"])


def test_calls_with_an_empty_batch_no_tokens_and_no_rows():
    import pa_b200

    rng = np.random.default_rng(18)
    c = Cache(rng, 2, 2, 64, 16, 16, "e4m3", [20, 0], 32)
    a = c.arrays("hnd")
    none = np.zeros((2, 0, 2, 64), np.float16)
    got = pa_b200.cache_append(none, none, seq_lens=[20, 0], **a)
    c.check_equal(got, "hnd")
    assert list(got.seq_lens) == [20, 0]
    got = pa_b200.cache_evict(seq_lens=[0, 0], weights=np.zeros((2, 2, 32), np.float32), budget=3, **a)
    assert (got.kept == -1).all() and list(got.seq_lens) == [0, 0]
    out, lse = pa_b200.cache_decode(np.ones((2, 4, 64), np.float16), seq_lens=[0, 0], return_lse=True, **a)
    assert (out == 0).all() and np.isneginf(lse).all()
    b = {**a, "block_table": a["block_table"][:0]}
    assert pa_b200.cache_decode(np.ones((0, 4, 64), np.float16), seq_lens=np.zeros(0, np.int32), **b).shape == (0, 4, 64)
    assert pa_b200.cache_append(none[:0], none[:0], seq_lens=np.zeros(0, np.int32), **b).seq_lens.shape == (0,)


def test_a_step_captured_in_a_graph_and_two_graphs_at_once():
    """Append, decode and evict captured on a side stream; two graphs with workspaces of their own replayed
    on two streams give what the calls give one by one."""
    import pa_b200
    import torch

    rng = np.random.default_rng(21)
    B, Hq, H, D, rows, budget = 4, 8, 2, 128, 512, 400
    sides = []
    for i in range(2):
        c = Cache(rng, B, H, D, 16, 16, ["e4m3", "int8"][i], [400, 380, 17, 400], rows)
        d = OnDevice(c, "hnd")
        desc = d.desc(Hq, rows)
        t = dict(x=torch.randn((2, B, 1, H, D), device="cuda").half(), q=torch.randn((B, Hq, D), device="cuda").half(),
                 w=torch.rand((B, H, rows), device="cuda"), pos=torch.arange(rows, dtype=torch.int32, device="cuda").expand(B, H, rows).contiguous())
        t.update(out=torch.zeros_like(t["q"]), lens2=torch.zeros_like(d.lens), lens3=torch.zeros_like(d.lens),
                 kept=torch.zeros((B, H, budget), dtype=torch.int32, device="cuda"),
                 ws=torch.empty((max(pa_b200.cache_decode_workspace_size(desc, True, True),
                                     pa_b200.cache_evict_workspace_size(desc, True, budget)),), dtype=torch.uint8, device="cuda"))

        def step(d=d, desc=desc, t=t, s=None):
            ws = (t["ws"].data_ptr(), t["ws"].numel())
            pa_b200.cache_append_device(desc, t["x"][0].data_ptr(), t["x"][1].data_ptr(), 1, d.k.data_ptr(), d.v.data_ptr(),
                                        d.lens.data_ptr(), weights_ptr=t["w"].data_ptr(), positions_ptr=t["pos"].data_ptr(),
                                        seq_lens_out_ptr=t["lens2"].data_ptr(), stream=s, **d.kw())
            pa_b200.cache_decode_device(desc, t["q"].data_ptr(), d.k.data_ptr(), d.v.data_ptr(), t["out"].data_ptr(),
                                        seq_lens_ptr=t["lens2"].data_ptr(), weights_ptr=t["w"].data_ptr(), stream=s, workspace=ws, **d.kw())
            pa_b200.cache_evict_device(desc, d.k.data_ptr(), d.v.data_ptr(), t["lens2"].data_ptr(), t["w"].data_ptr(), budget,
                                       t["lens3"].data_ptr(), t["kept"].data_ptr(), recent=32, sinks=2, positions_ptr=t["pos"].data_ptr(),
                                       next_positions_ptr=t["lens2"].data_ptr(), weights_out_ptr=t["w"].data_ptr(),
                                       positions_out_ptr=t["pos"].data_ptr(), stream=s, workspace=ws, **d.kw())

        tensors = [d.k, d.v, d.ks, d.vs] + list(t.values())
        first = [x.clone() for x in tensors]
        torch.cuda.synchronize()
        for _ in range(3):
            step()
        torch.cuda.synchronize()
        want = [x.clone() for x in tensors]
        for x, y in zip(tensors, first):
            x.copy_(y)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(s=On(torch.cuda.current_stream()))
        sides.append((graph, stream, tensors, want, t["ws"], d))  # the graph reads d's lengths and table too
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream, *_ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    for graph, stream, tensors, want, ws, d in sides:
        for x, y in zip(tensors, want):
            if x is not ws:
                same = torch.equal(x.view(torch.uint8), y.view(torch.uint8))
                assert same


def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of the cache base (keys and values share the array, which only append distinguishes)."""
    import pa_b200
    import torch

    H, page, D, block = 8, 16, 128, 16
    pages = (5 << 30) // (H * page * D)
    k = torch.zeros((pages, H, page, D), dtype=torch.uint8, device="cuda")
    ks = torch.zeros((pages, H, 1), device="cuda")
    T = 200
    per = 16
    table = torch.arange(pages - 2 * per, pages, dtype=torch.int32, device="cuda").flip(0).reshape(2, per).contiguous()
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    lens2 = torch.zeros_like(lens)
    desc = pa_b200.block_cache_desc(2, 16, D, tuple(k.shape), kv_format="e4m3", paged=True, max_pages_per_seq=per, scale_block=block)
    x = torch.randn((2, T, H, D), device="cuda").half()
    kw = dict(k_scales_ptr=ks.data_ptr(), v_scales_ptr=ks.data_ptr(), block_table_ptr=table.data_ptr())
    pa_b200.cache_append_device(desc, x.data_ptr(), x.data_ptr(), T, k.data_ptr(), k.data_ptr(), lens.data_ptr(),
                                seq_lens_out_ptr=lens2.data_ptr(), **kw)
    q = torch.randn((2, 16, D), device="cuda").half()
    out, lse = torch.empty_like(q), torch.empty((2, 16), device="cuda")
    w = torch.rand((2, H, per * page), device="cuda")
    w0 = w.cpu().numpy()
    pa_b200.cache_decode_device(desc, q.data_ptr(), k.data_ptr(), k.data_ptr(), out.data_ptr(), seq_lens_ptr=lens2.data_ptr(),
                                lse_ptr=lse.data_ptr(), weights_ptr=w.data_ptr(), **kw)
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    small = k[-2 * per:].cpu().numpy()
    sc = ks[-2 * per:].cpu().numpy()
    assert int(k[:-2 * per].count_nonzero()) == 0
    c = np.full((2 * per, H, page, D), np.nan)
    s = np.full((2 * per, H, 1), np.nan)
    tab = table.cpu().numpy() - (pages - 2 * per)
    xs = x.double().cpu().numpy()
    append_reference(xs, xs, c, c.copy(), [0, 0], [T, T], ks=s, vs=s.copy(), table=tab, block=block, fmt="e4m3")
    live = ~np.isnan(c)
    np.testing.assert_array_equal(e4m3_to_float(small)[live], c[live])
    np.testing.assert_array_equal(sc[~np.isnan(s)], s[~np.isnan(s)].astype(np.float32))
    ref = decode_reference(q.cpu().numpy(), c, c, [T, T], ks=s, vs=s, table=tab, block=block, weights=w0)
    check_decode(ref, out.cpu().numpy(), lse.cpu().numpy(), w.cpu().numpy(), w0)


@pytest.mark.parametrize("H,n,budget", [(2, 9004, 4000), (80, 301, 120)])
def test_evict_writes_positions_without_being_given_any(H, n, budget):
    """positions_out holds the rows themselves; weights at an odd address, results apart from the inputs,
    what is behind the new length left as it was (one head in a cluster, many in one CTA each)."""
    import pa_b200
    import torch

    rng = np.random.default_rng(n)
    c = Cache(rng, 1, H, 64, 64, 64, None, [n], n)
    d = OnDevice(c, "hnd")
    w = torch.rand(H * n + 1, device="cuda")[1:]
    w_out, p_out = torch.full((H, n), -2.0, device="cuda"), torch.full((H, n), -3, dtype=torch.int32, device="cuda")
    lens2, kept = torch.empty_like(d.lens), torch.empty((H, budget), dtype=torch.int32, device="cuda")
    want_w = w.cpu().numpy().reshape(1, H, n).copy()
    pa_b200.cache_evict_device(d.desc(H, n), d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(), w.data_ptr(), budget,
                               lens2.data_ptr(), kept.data_ptr(), recent=5, weights_out_ptr=w_out.data_ptr(),
                               positions_out_ptr=p_out.data_ptr(), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    _, want = evict_reference(c.k, c.v, [n], want_w, budget, recent=5, table=c.table)
    np.testing.assert_array_equal(kept.cpu().numpy(), want[0])
    np.testing.assert_array_equal(p_out[:, :budget].cpu().numpy(), want[0])
    np.testing.assert_array_equal(w_out[:, :budget].cpu().numpy(), want_w[0, :, :budget])
    assert (w_out[:, budget:] == -2).all() and (p_out[:, budget:] == -3).all()
    d.check_equal()


def test_two_streams_at_once_without_workspaces_or_lengths():
    """Scratch from the pool; NULL lengths mean full sequences. Each stream's calls repeat bit for bit."""
    import pa_b200
    import torch

    rng = np.random.default_rng(51)
    rows, sides = 1024, []
    for fmt in ("e4m3", None):
        c = Cache(rng, 3, 2, 128, 32, 32, fmt, [rows] * 3, rows)
        d = OnDevice(c, "nhd")
        q = torch.randn((3, 8, 128), device="cuda").half()
        out, w = torch.empty_like(q), torch.zeros((3, 2, rows), device="cuda")
        sides.append((c, d, d.desc(8, rows), q, out, w, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, d, desc, q, out, w, s in sides:
            pa_b200.cache_decode_device(desc, q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(), weights_ptr=w.data_ptr(),
                                        stream=On(s), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    for c, d, desc, q, out, w, s in sides:
        ref = decode_reference(q.cpu().numpy(), c.k, c.v, [rows] * 3, weights=np.zeros((3, 2, rows)), **c.parts())
        tol = U["f16"] * np.abs(ref["out"]) + (2.0 ** -11 + 2.0 ** -16) * ref["pv"] + 2.0 ** -25
        assert (np.abs(out.double().cpu().numpy() - ref["out"]) <= tol).all()
        # Twenty equal additions: each within the single call's bound, and half a step of the sum each time.
        dl = (2.0 ** -18 * ref["mag"] + 2.0 ** -20 * (1 + np.abs(ref["lse"]))).reshape(3, 2, 4).max(-1)[..., None]
        want = 20 * ref["weights"]
        assert (np.abs(w.cpu().numpy() - want) <= want * (2 * dl + 2.0 ** -18 + 20 * 2.0 ** -24)).all()


def test_calls_with_workspaces_allocate_nothing():
    import pa_b200
    import torch

    rng = np.random.default_rng(61)
    c = Cache(rng, 2, 2, 64, 16, 16, "int8", [4000, 9], 4200)
    d = OnDevice(c, "hnd")
    desc = d.desc(4, 4200)
    q, x = torch.randn((2, 4, 64), device="cuda").half(), torch.randn((2, 2, 8, 2, 64), device="cuda").half()
    out, w = torch.empty_like(q), torch.zeros((2, 2, 4200), device="cuda")
    lens2, lens3 = torch.empty_like(d.lens), torch.empty_like(d.lens)
    kept = torch.empty((2, 2, 3000), dtype=torch.int32, device="cuda")
    n1, n2 = pa_b200.cache_decode_workspace_size(desc, True, True), pa_b200.cache_evict_workspace_size(desc, True, 3000)
    ws = torch.empty((max(n1, n2),), dtype=torch.uint8, device="cuda")

    def step():
        pa_b200.cache_append_device(desc, x[0].data_ptr(), x[1].data_ptr(), 8, d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(),
                                    weights_ptr=w.data_ptr(), seq_lens_out_ptr=lens2.data_ptr(), **d.kw())
        pa_b200.cache_decode_device(desc, q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(), seq_lens_ptr=lens2.data_ptr(),
                                    weights_ptr=w.data_ptr(), workspace=(ws.data_ptr(), n1), **d.kw())
        pa_b200.cache_evict_device(desc, d.k.data_ptr(), d.v.data_ptr(), lens2.data_ptr(), w.data_ptr(), 3000, lens3.data_ptr(),
                                   kept.data_ptr(), weights_out_ptr=w.data_ptr(), workspace=(ws.data_ptr(), n2), **d.kw())

    step()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(10):
        step()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == free
    assert lens3.tolist() == [3000, 17]


def test_calls_on_another_device():
    import pa_b200

    if pa_b200.device_count() < 2:
        pytest.skip("needs two GPUs")
    rng = np.random.default_rng(30)
    c = Cache(rng, 2, 2, 64, 16, 16, "e4m3", [30, 64], 64)
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    first = pa_b200.cache_decode(q, seq_lens=c.lens, **c.arrays("hnd"))
    pa_b200.set_device(1)
    try:
        np.testing.assert_array_equal(pa_b200.cache_decode(q, seq_lens=c.lens, **c.arrays("hnd")), first)
    finally:
        pa_b200.set_device(0)
