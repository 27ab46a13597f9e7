"""Block-scaled cache on the GPU at the ends of its ranges: magnitudes, infinities and NaN, wrong
pages and lengths, descriptors far wider than the work.

Bounds and helpers are those of test_gpu_blockcache.py.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle.blockcache import append_reference, decode_reference, evict_reference, need_scale, round8
from test_gpu_blockcache import FORMATS, U, Cache, OnDevice, check_decode

pytestmark = pytest.mark.gpu


def decode(d, q, rows, q_dtype="bf16", weights=None):
    """One call on device pointers; returns float64 output, lse and (if given) the weights afterwards."""
    import pa_b200
    import torch

    B, Hq, _ = q.shape
    out, lse = torch.empty_like(q), torch.empty((B, Hq), device="cuda")
    w = None if weights is None else torch.from_numpy(weights).cuda()
    pa_b200.cache_decode_device(d.desc(Hq, rows, q_dtype), q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(),
                                seq_lens_ptr=d.lens.data_ptr(), lse_ptr=lse.data_ptr(),
                                weights_ptr=None if w is None else w.data_ptr(), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    return out.double().cpu().numpy(), lse.cpu().numpy(), None if w is None else w.cpu().numpy()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,Hq", [(64, 3), (128, 8), (64, 13), (128, 16)])
def test_bf16_query_heads_of_one_group_far_apart_in_magnitude(fmt, D, Hq):
    """Each head's scores are as exact as if it were alone: heads 2^40 apart share a kv head."""
    import torch

    rng = np.random.default_rng(D + Hq)
    rows, lens = 300, [300, 37]
    c = Cache(rng, 2, 1, D, 16, 16, fmt, lens, rows)
    d = OnDevice(c, "hnd")
    x = rng.standard_normal((2, Hq, D))
    x[:, 1::2] *= 2.0 ** -20
    x[:, 2::4] *= 2.0 ** 20
    c.ks *= 2.0 ** 20                     # so that the small heads' scores count
    d.ks.mul_(2.0 ** 20)
    q = torch.from_numpy(x).to("cuda", torch.bfloat16)
    w = rng.random((2, 1, rows)).astype(np.float32)
    out, lse, got_w = decode(d, q, rows, weights=w)
    ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, lens, weights=w, **c.parts())
    check_decode({k: v[:, 1::2] if k != "weights" else v for k, v in ref.items()}, out[:, 1::2], lse[:, 1::2], u=U["bf16"])
    assert np.isfinite(got_w).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("exp", [127, 100, -112, -118, -125])
def test_value_scales_at_the_ends_of_fp32(fmt, exp):
    """Scales of 1 to 1.9 times 2^exp: bf16 holds the results, which are below a code times its scale.

    From 2^-117 down a result may be a bf16 subnormal: half a step of those is 2^-134, and fp32
    sums lose at most 2^-149 a tile (of four), taken relative to 256 rows."""
    import torch

    rng = np.random.default_rng(exp + 200)
    rows, lens = 200, [200, 5]
    c = Cache(rng, 2, 2, 64, 16, 8, fmt, lens, rows)
    live = ~np.isnan(c.vs)
    c.vs[live] = (np.float32(1 + 0.9 * rng.random(live.sum())) * np.float32(2.0) ** np.float32(exp)).astype(np.float64)
    if exp > 0:                                # codes whose product with the scale is finite in bf16
        c.v = np.clip(c.v, -1, 1)
        if exp == 127:
            c.v[:] = np.where(np.isnan(c.v), c.v, 0.0)
            for b in range(2):                 # one row of codes 1, the others 0
                c.v[c.table[b, 0], :, 3] = 1.0
    d = OnDevice(c, "hnd")
    q = torch.from_numpy(rng.standard_normal((2, 4, 64))).to("cuda", torch.bfloat16)
    out, lse, _ = decode(d, q, rows)
    ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, lens, **c.parts())
    assert (np.abs(ref["out"]).max((1, 2)) > 2.0 ** (exp - 12)).all()
    tol = U["bf16"] * np.abs(ref["out"]) + (2.0 ** -11 + 2.0 ** -16) * ref["pv"] + 2.0 ** -134 + 2.0 ** -139
    assert np.isfinite(out).all()
    assert (np.abs(out - ref["out"]) <= tol).all(), float((np.abs(out - ref["out"]) / tol).max())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,S,weights", [(64, 33, False), (128, 300, False), (64, 300, True), (128, 70001, False), (64, 20011, True)])
def test_sums_of_many_values_near_the_end_of_the_range(fmt, D, S, weights):
    """All keys weigh the same and all values are 1.5 * 2^126: their mean is finite, their sum is not."""
    import torch

    rng = np.random.default_rng(S)
    c = Cache(rng, 1, 1, D, 64, 64, fmt, [S], S)
    for x, s in ((c.k, c.ks), (c.v, c.vs)):
        x[~np.isnan(x)] = 0.0 if x is c.k else 1.5 * 2.0 ** 126 if fmt is None else 3.0
        if fmt is not None:
            s[~np.isnan(s)] = 2.0 ** 125
    d = OnDevice(c, "hnd", "bf16")
    q = torch.from_numpy(rng.standard_normal((1, 3, D))).to("cuda", torch.bfloat16)
    w = np.zeros((1, 1, S), np.float32) if weights else None
    out, lse, _ = decode(d, q, S, weights=w)
    assert (np.abs(out / (1.5 * 2.0 ** 126) - 1) <= U["bf16"] + 2.0 ** -11 + 2.0 ** -16).all()
    np.testing.assert_allclose(lse, np.log(S), rtol=2.0 ** -19)


def test_small_bf16_values_keep_their_bits():
    """Values of about 2^-110 over 70001 rows: far below, 17 bits of the sums' range go to the other end."""
    import torch

    rng = np.random.default_rng(70)
    c = Cache(rng, 1, 1, 64, 64, 64, None, [70001], 70001)
    c.v *= 2.0 ** -110
    for x in (c.k, c.v):
        x[:] = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    d = OnDevice(c, "hnd", "bf16")
    q = torch.from_numpy(rng.standard_normal((1, 3, 64))).to("cuda", torch.bfloat16)
    out, _, _ = decode(d, q, 70001)
    ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, [70001], **c.parts())
    # Each of 2188 tiles costs at most 2^-149, taken relative to 2^17 rows: 2^-121.
    tol = U["bf16"] * np.abs(ref["out"]) + 2.0 ** -11 * ref["pv"] + 2.0 ** -120
    assert (np.abs(out - ref["out"]) <= tol).all()


@pytest.mark.parametrize("q_dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["e4m3", None])
@pytest.mark.parametrize("S,weights", [(50, False), (50, True), (5000, True)])
def test_infinities_and_nan_reach_what_they_belong_to(fmt, q_dtype, S, weights):
    """One launch and two: a NaN key or query makes its heads NaN, a NaN value its element, an infinite
    value its element infinite; other heads and sequences are as they would be without."""
    import torch

    rng = np.random.default_rng(S)
    t16 = torch.float16 if q_dtype == "f16" else torch.bfloat16
    B, H, G, D = 5, 2, 3, 64
    c = Cache(rng, B, H, D, 16, 16, fmt, [S] * B, S)
    if fmt is None:
        for x in (c.k, c.v):
            x[:] = torch.from_numpy(x).to(t16).double().numpy()
    at = lambda b, r: (c.table[b, r // 16], r % 16)  # noqa: E731
    p, r = at(0, 41)
    c.k[p, 0, r, 7] = np.nan                     # sequence 0, kv head 0
    p, r = at(1, 17)
    c.v[p, 1, r, 9] = np.nan                     # sequence 1, kv head 1, element 9
    if fmt is None:
        for n, (b, row, x) in enumerate([(2, 3, np.inf), (2, 40, -np.inf)]):
            p, r = at(b, row)
            c.v[p, n, r, 5 + n] = x              # sequence 2: element 5 of kv head 0, 6 of kv head 1
        p, r = at(4, 20)
        c.k[p, 1, r, 0] = np.inf                 # sequence 4, kv head 1: a score of plus or minus infinity
    d = OnDevice(c, "hnd", q_dtype)
    q = torch.from_numpy(rng.standard_normal((B, H * G, D))).to("cuda", t16)
    q[3, 1, 3] = float("nan")                    # sequence 3, head 1
    q[4, H * G - 1, 0] = 2.0                     # an infinite score: that head is NaN
    q[4, H * G - 2, 0] = -2.0                    # minus infinity: a key without weight
    w = rng.random((B, H, S)).astype(np.float32) if weights else None
    out, lse, got_w = decode(d, q, S, q_dtype, weights=w)
    with np.errstate(all="ignore"):
        ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, [S] * B, weights=w, **c.parts())
    assert (ref["lse"][0] != ref["lse"][0]).tolist() == [True] * G + [False] * G
    for got, want in ((out, ref["out"]), (lse, ref["lse"])) + (((got_w, ref["weights"]),) if weights else ()):
        for same in (np.isnan, np.isposinf, np.isneginf):
            np.testing.assert_array_equal(same(got), same(want))
    ok = np.isfinite(ref["out"])
    tol = U[q_dtype] * np.abs(ref["out"]) + (2.0 ** -11 + 2.0 ** -16) * ref["pv"] + 2.0 ** -25
    assert (np.abs(out[ok] - ref["out"][ok]) <= tol[ok]).all()


@pytest.mark.parametrize("fmt,q_dtype", [("e4m3", "f16"), ("int8", "bf16"), (None, "f16"), (None, "bf16")])
@pytest.mark.parametrize("G,H,D", [(1, 2, 64), (4, 2, 128), (3, 1, 64), (5, 1, 128), (8, 2, 64), (9, 1, 128), (16, 1, 64)])
def test_probabilities_keep_more_bits_than_the_output(fmt, q_dtype, G, H, D):
    """Probabilities go into the products as two 16-bit terms: what is lost is 2^-10 of 2^-10 (fp16), 2^-7
    of 2^-7 (bf16 caches), far below half a step of the output even where values cancel; fp32 sums 2^-16."""
    import torch

    rng = np.random.default_rng(G * D)
    lens = [3, 40, 1000, 9, 21]
    c = Cache(rng, 5, H, D, 16, 8, fmt, lens, 1000)
    if fmt is None and q_dtype == "bf16":
        for x in (c.k, c.v):
            x[:] = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    d = OnDevice(c, "hnd", q_dtype)
    q = torch.from_numpy(rng.standard_normal((5, G * H, D))).to("cuda", torch.float16 if q_dtype == "f16" else torch.bfloat16)
    for weights in (None, rng.random((5, H, 1000)).astype(np.float32)):
        out, _, _ = decode(d, q, 1000, q_dtype, weights=weights)
        ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, lens, **c.parts())
        p = 2.0 ** -14 if fmt is None and q_dtype == "bf16" else 2.0 ** -20
        tol = U[q_dtype] * np.abs(ref["out"]) + (p + 2.0 ** -16) * ref["pv"] + (2.0 ** -25 if q_dtype == "f16" else 0)
        assert (np.abs(out - ref["out"]) <= tol).all(), float((np.abs(out - ref["out"]) / tol).max())


def reported(call, text):
    """Runs the call; the device has to report `text`."""
    import pa_b200
    import torch
    from pa_b200._lib import PaError

    call()
    torch.cuda.synchronize()
    with pytest.raises(PaError, match=text):
        pa_b200.sync_device_status()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [10 ** 6, -1])
def test_append_with_a_wrong_page_leaves_its_rows_and_the_length(fmt, bad):
    """The second page of sequence 1's new rows is wrong; sequence 0 is as ever, sequence 2 is too long."""
    import pa_b200
    import torch

    rng = np.random.default_rng(81)
    B, H, D, T, rows = 3, 2, 64, 30, 64
    lens = [11, 12, 50]
    c = Cache(rng, B, H, D, 16, 8, fmt, lens, rows)
    d = OnDevice(c, "hnd")
    good = c.table.copy()
    d.table[1, 1] = bad                                     # rows 16 to 31 of sequence 1
    x = torch.from_numpy(rng.standard_normal((2, B, T, H, D))).to("cuda", torch.float16)
    w, pos = torch.full((B, H, rows), 7.0, device="cuda"), torch.full((B, H, rows), -5, dtype=torch.int32, device="cuda")
    out = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    reported(lambda: pa_b200.cache_append_device(
        d.desc(H, rows), x[0].data_ptr(), x[1].data_ptr(), T, d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(),
        weights_ptr=w.data_ptr(), positions_ptr=pos.data_ptr(), seq_lens_out_ptr=out.data_ptr(), **d.kw()), "code 0x20")
    assert out.tolist() == [41, 12, 50]
    # What the call means: every block that has a page, none of sequence 2.
    before = {n: getattr(c, n) if getattr(c, n) is None else getattr(c, n).copy() for n in ("k", "v", "ks", "vs")}
    xs = x.double().cpu().numpy()
    append_reference(xs[0], xs[1], c.k, c.v, lens, [T, T, 0], fmt=fmt, **c.parts())
    for n in ("k", "v", "ks", "vs"):
        if before[n] is not None:
            getattr(c, n)[good[1, 1]] = before[n][good[1, 1]]
    d.check_equal()
    written = np.zeros((B, 1, rows), bool)
    written[0, :, 11:41] = written[1, :, 12:16] = written[1, :, 32:42] = True
    np.testing.assert_array_equal(w.cpu().numpy(), np.broadcast_to(np.where(written, 0.0, 7.0), (B, H, rows)))
    np.testing.assert_array_equal(pos.cpu().numpy(), np.broadcast_to(np.where(written, np.arange(rows), -5), (B, H, rows)))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,n,budget,page_at", [
    (2, 300, 290, 11), (2, 300, 290, 18),      # few rows go; a page of holes, the last page
    (3, 303, 299, 3), (3, 700, 120, 0),        # few rows go and the CTA moves them; many go
    (1, 9000, 4000, 500),                      # a cluster
])
def test_evict_with_a_wrong_page_leaves_the_sequence(fmt, H, n, budget, page_at):
    """Sequence 1 has a wrong page, sequence 3 a wrong length; 0 shrinks as ever and 2 has nothing to lose."""
    import pa_b200
    import torch

    rng = np.random.default_rng(n + page_at)
    lens = [n, n, min(budget, 37), n]
    c = Cache(rng, 4, H, 64, 16, 8, fmt, lens, n)
    d = OnDevice(c, "hnd")
    d.table[1, page_at] = c.k.shape[0]
    d.table[2, 4] = -3                          # behind its rows: not a page of the sequence
    lens[3] = n + 1
    d.lens[3] = n + 1
    w0, p0 = rng.random((4, H, n)).astype(np.float32), np.tile(np.arange(n, dtype=np.int32) + 5, (4, H, 1))
    for in_place in (False, True):
        w, pos = torch.from_numpy(w0).cuda(), torch.from_numpy(p0).cuda()
        w_out = w if in_place else torch.full_like(w, -2.0)
        p_out = pos if in_place else torch.full_like(pos, -4)
        nxt = torch.full((4,), n + 5, dtype=torch.int32, device="cuda")
        lens2 = torch.full((4,), -1, dtype=torch.int32, device="cuda")
        kept = torch.full((4, H, budget), -7, dtype=torch.int32, device="cuda")
        reported(lambda: pa_b200.cache_evict_device(
            d.desc(H, n), d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(), w.data_ptr(), budget, lens2.data_ptr(),
            kept.data_ptr(), recent=9, sinks=6, positions_ptr=pos.data_ptr(), next_positions_ptr=nxt.data_ptr(),
            weights_out_ptr=w_out.data_ptr(), positions_out_ptr=p_out.data_ptr(), **d.kw()), "code 0x20")
        if not in_place:                        # the second call finds sequence 0's cache shrunk once
            want_w, want_p = w0.copy(), p0.copy()
            _, want = evict_reference(c.k, c.v, [n, 0, 0, 0], want_w, budget, recent=9, sinks=6, positions=want_p,
                                      next_positions=[n + 5] * 4, fmt=fmt, **c.parts())
            d.check_equal()
        assert lens2.tolist() == [budget, n, min(budget, 37), n + 1]
        got = kept.cpu().numpy()
        np.testing.assert_array_equal(got[0], want[0])
        assert (got[1] == -1).all() and (got[3] == -1).all()
        np.testing.assert_array_equal(got[2], np.tile(np.r_[0:37, [-1] * (budget - 37)], (H, 1)))
        np.testing.assert_array_equal(w_out[0, :, :budget].cpu().numpy(), want_w[0, :, :budget])
        np.testing.assert_array_equal(p_out[0, :, :budget].cpu().numpy(), want_p[0, :, :budget])
        for b in (1, 3):
            for got, was, fill in ((w_out[b], w0[b], -2.0), (p_out[b], p0[b], -4)):
                got = got.cpu().numpy()
                assert ((got == was) | (not in_place and got == fill)).all()
                if not in_place:
                    assert (got[:, budget:] == fill).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [100, 5000])
def test_decode_with_wrong_lengths_and_pages(fmt, rows):
    """A length too long counts as the longest, one below 0 as 0, both without weights; a wrong page as zeros."""
    import pa_b200
    import torch

    rng = np.random.default_rng(rows)
    B, H, D = 4, 2, 64
    c = Cache(rng, B, H, D, 16, 8, fmt, [rows] * B, rows)
    d = OnDevice(c, "hnd")
    d.lens.copy_(torch.tensor([rows + 1, -1, rows, 60], dtype=torch.int32))
    d.table[2, 1] = -1
    q = torch.from_numpy(rng.standard_normal((B, 6, D))).to("cuda", torch.float16)
    out, lse = torch.empty_like(q), torch.empty((B, 6), device="cuda")
    w0 = rng.random((B, H, rows)).astype(np.float32)
    w = torch.from_numpy(w0).cuda()
    reported(lambda: pa_b200.cache_decode_device(
        d.desc(6, rows), q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(), seq_lens_ptr=d.lens.data_ptr(),
        lse_ptr=lse.data_ptr(), weights_ptr=w.data_ptr(), **d.kw()), "code 0x20")
    for x in (c.k, c.v) + ((c.ks, c.vs) if fmt else ()):
        x[c.table[2, 1]] = 0.0
    ref = decode_reference(q.double().cpu().numpy(), c.k, c.v, [rows, 0, rows, 60], weights=w0, **c.parts())
    ref["weights"][:2] = w0[:2]
    check_decode(ref, out.cpu().numpy(), lse.cpu().numpy(), w.cpu().numpy(), w0)
    np.testing.assert_array_equal(w[:2].cpu().numpy(), w0[:2])


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_of_a_padded_batch_wider_than_the_cache(fmt):
    import pa_b200

    rng = np.random.default_rng(91)
    c = Cache(rng, 2, 2, 64, 16, 8, fmt, [10, 0], 32)
    x = rng.standard_normal((2, 2, 100, 2, 64)).astype(np.float16)
    w = rng.random((2, 2, 24)).astype(np.float32)                  # arrays of 24 rows
    new = np.array([5, 24], np.int32)
    got = pa_b200.cache_append(x[0], x[1], seq_lens=[10, 0], new_lens=new, weights=w, **c.arrays("hnd"))
    append_reference(x[0], x[1], c.k, c.v, [10, 0], new, fmt=fmt, weights=w, **c.parts())
    c.check_equal(got, "hnd")
    assert list(got.seq_lens) == [15, 24]
    np.testing.assert_array_equal(got.weights, w)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scale_blocks_far_above_the_page_of_a_dense_cache(fmt):
    """One scale a sequence and head, whatever scale_block says above the page's rows."""
    import pa_b200

    rng = np.random.default_rng(95)
    for block in (150, 2 ** 31 - 1):
        c = Cache(rng, 2, 2, 64, 150, 150, fmt, [100, 3], 150, paged=False)
        a = {**c.arrays("hnd"), "scale_block": block}
        x = rng.standard_normal((2, 2, 40, 2, 64)).astype(np.float16)
        got = pa_b200.cache_append(x[0], x[1], seq_lens=[100, 3], **a)
        append_reference(x[0], x[1], c.k, c.v, [100, 3], [40, 40], fmt=fmt, **c.parts())
        c.check_equal(got, "hnd")
        a = {**c.arrays("hnd"), "scale_block": block}
        q = rng.standard_normal((2, 4, 64)).astype(np.float16)
        w0 = np.zeros((2, 2, 150), np.float32)
        out, lse, w = pa_b200.cache_decode(q, seq_lens=[140, 43], weights=w0, return_lse=True, **a)
        check_decode(decode_reference(q, c.k, c.v, [140, 43], weights=w0, **c.parts()), out, lse, w, w0)
        for budget in (137, 64):
            want_w = w.copy()
            got = pa_b200.cache_evict(seq_lens=[140, 43], weights=w, budget=budget, recent=5, **a)
            d = Cache.__new__(Cache)
            d.__dict__.update({k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.__dict__.items()})
            _, kept = evict_reference(d.k, d.v, [140, 43], want_w, budget, recent=5, fmt=fmt, **d.parts())
            np.testing.assert_array_equal(got.kept, kept)
            d.check_equal(got, "hnd")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,page,block,layout", [(128, 16, 16, "hnd"), (128, 128, 64, "nhd"), (64, 128, 128, "hnd"), (128, 8, 2, "nhd")])
@pytest.mark.parametrize("spare", [0, 3, 9, 700, 20000])
def test_evict_of_a_few_rows_from_descriptors_of_any_width(fmt, D, page, block, layout, spare):
    """1 to 8 rows over the budget, in arrays of `spare` rows more than the longest sequence: the CTA that
    selects moves the rows where no sequence can have more than eight to lose, else a second launch does."""
    import pa_b200
    import torch

    rng = np.random.default_rng(D + page + spare)
    B, H, budget = 3, 2, 333
    lens = [budget + 5, budget + 1, budget + 8 - min(spare, 8)]
    rows = max(lens) + spare
    c = Cache(rng, B, H, D, page, block, fmt, lens, rows)
    d = OnDevice(c, layout)
    w0 = np.round(rng.exponential(size=(B, H, rows)) * 30).astype(np.float32) / 30
    w = torch.from_numpy(w0).cuda()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda").expand(B, H, rows).contiguous()
    lens2, kept = torch.empty_like(d.lens), torch.empty((B, H, budget), dtype=torch.int32, device="cuda")
    pa_b200.cache_evict_device(d.desc(H, rows), d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(), w.data_ptr(), budget,
                               lens2.data_ptr(), kept.data_ptr(), recent=20, sinks=3, positions_ptr=pos.data_ptr(),
                               next_positions_ptr=d.lens.data_ptr(), weights_out_ptr=w.data_ptr(), positions_out_ptr=pos.data_ptr(),
                               **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    want_w, want_p = w0.copy(), np.broadcast_to(np.arange(rows, dtype=np.int32), (B, H, rows)).copy()
    want_len, want = evict_reference(c.k, c.v, lens, want_w, budget, recent=20, sinks=3, positions=want_p,
                                     next_positions=lens, fmt=fmt, **c.parts())
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    np.testing.assert_array_equal(w.cpu().numpy(), want_w)
    np.testing.assert_array_equal(pos.cpu().numpy(), want_p)
    assert lens2.tolist() == list(want_len)
    d.check_equal()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_of_bf16_near_the_ends_of_its_range(fmt):
    """Scales up to 2^121 and down to 2^-100; earlier rows 2^200 below are coded to 0."""
    import pa_b200
    import torch

    rng = np.random.default_rng(97)
    c = Cache(rng, 1, 2, 64, 16, 8, fmt, [4], 64)
    d = OnDevice(c, "nhd", "bf16")
    x = rng.standard_normal((2, 1, 40, 2, 64))
    x[0, 0, :12] *= 2.0 ** 125
    x[0, 0, 12:20] *= 2.0 ** -98
    x[1, 0, 20:] *= 2.0 ** -126
    t = torch.from_numpy(x).to("cuda", torch.bfloat16)
    assert bool(torch.isfinite(t).all())
    pa_b200.cache_append_device(d.desc(2, 64, "bf16"), t[0].data_ptr(), t[1].data_ptr(), 40, d.k.data_ptr(), d.v.data_ptr(),
                                d.lens.data_ptr(), **d.kw())
    torch.cuda.synchronize()
    pa_b200.sync_device_status()
    xs = t.double().cpu().numpy()
    append_reference(xs[0], xs[1], c.k, c.v, [4], [40], fmt=fmt, **c.parts())
    d.check_equal()


def pool_high(reset=False):
    """Most bytes in use of the device's default pool since the last reset."""
    import ctypes

    cuda = ctypes.CDLL("libcuda.so.1")
    dev, pool, value = ctypes.c_int(0), ctypes.c_void_p(), ctypes.c_uint64(0)
    import torch

    assert cuda.cuDeviceGet(ctypes.byref(dev), torch.cuda.current_device()) == 0
    assert cuda.cuDeviceGetDefaultMemPool(ctypes.byref(pool), dev) == 0
    used_high = 8                                     # CU_MEMPOOL_ATTR_USED_MEM_HIGH
    if reset:
        assert cuda.cuMemPoolSetAttribute(pool, used_high, ctypes.byref(value)) == 0
    assert cuda.cuMemPoolGetAttribute(pool, used_high, ctypes.byref(value)) == 0
    return value.value


def test_the_pool_is_used_without_workspaces_and_not_with_them():
    """The default pool keeps what it once had, so free memory says nothing: its most bytes in use do."""
    import pa_b200
    import torch

    rng = np.random.default_rng(99)
    c = Cache(rng, 2, 2, 64, 16, 16, "int8", [4000, 9], 4200)
    d = OnDevice(c, "hnd")
    desc = d.desc(4, 4200)
    q, x = torch.randn((2, 4, 64), device="cuda").half(), torch.randn((2, 2, 8, 2, 64), device="cuda").half()
    out, w = torch.empty_like(q), torch.zeros((2, 2, 4200), device="cuda")
    lens2, lens3 = torch.empty_like(d.lens), torch.empty_like(d.lens)
    kept = torch.empty((2, 2, 3000), dtype=torch.int32, device="cuda")
    n1, n2 = pa_b200.cache_decode_workspace_size(desc, True, True), pa_b200.cache_evict_workspace_size(desc, True, 3000)
    ws = torch.empty((max(n1, n2),), dtype=torch.uint8, device="cuda")

    def used(ws1, ws2):
        torch.cuda.synchronize()
        base = pool_high(reset=True)
        for _ in range(3):
            pa_b200.cache_append_device(desc, x[0].data_ptr(), x[1].data_ptr(), 8, d.k.data_ptr(), d.v.data_ptr(), d.lens.data_ptr(),
                                        weights_ptr=w.data_ptr(), seq_lens_out_ptr=lens2.data_ptr(), **d.kw())
            pa_b200.cache_decode_device(desc, q.data_ptr(), d.k.data_ptr(), d.v.data_ptr(), out.data_ptr(),
                                        seq_lens_ptr=lens2.data_ptr(), weights_ptr=w.data_ptr(), workspace=ws1, **d.kw())
            pa_b200.cache_evict_device(desc, d.k.data_ptr(), d.v.data_ptr(), lens2.data_ptr(), w.data_ptr(), 3000, lens3.data_ptr(),
                                       kept.data_ptr(), weights_out_ptr=w.data_ptr(), workspace=ws2, **d.kw())
        torch.cuda.synchronize()
        return pool_high() - base

    used((None, 0), (None, 0))
    assert used((ws.data_ptr(), n1), (ws.data_ptr(), n2)) == 0
    assert used((None, 0), (ws.data_ptr(), n2)) >= n1          # the count sees what the calls take themselves
    assert used((ws.data_ptr(), n1), (None, 0)) >= n2
    pa_b200.sync_device_status()
