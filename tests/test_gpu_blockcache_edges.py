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
