"""The attention over a paged cache at the ends of its scales' and values' ranges, against the formula in 64 bits (the
tolerances of test_paged_gpu.py): scales of an 8-bit cache that are negative, zero or tiny, queries of any size, NaN in
places that a row does not see."""
import math

import pytest

import kore_b200 as K
from tests.test_paged_gpu import BOTH, HINTS, KINDS, Cache, attend, check_attention, dev, gen, ints, rand, starts, u

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@BOTH
@pytest.mark.parametrize("tq", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(scale=-0.2), dict(window=50), dict(causal=False, window=70)])
def test_scales_of_any_sign(kernel, tq, d, kw):
    """A head's value is its 8 bits times its scale, whatever the scale's sign; with a scale of 0 every key scores 0 and
    the outputs are the means of the values."""
    g = gen(31)
    ns, kvs = [1, 37, 150, 6], [400, 37, 900, 129]
    C = Cache(g, "e4m3", 4, d, 64, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    C.ks[0] = 0
    C.ks[1:] *= ints([-1, 1, -4])
    C.vs *= ints([1, -1, 0, 1])
    attend(g, C, 28, ns, tq, kernel, **kw)


@BOTH
@pytest.mark.parametrize("tq", ["f16", "bf16"])
def test_a_factor_too_small_for_32_bits_is_as_good_as_zero(kernel, tq):
    g = gen(32)
    ns, kvs = [1, 90], [300, 131]
    C = Cache(g, "e4m3", 2, 64, 32, kvs)
    C.fill(g, 0), C.fill(g, 1)
    C.ks.fill_(2.0 ** -100)
    attend(g, C, 14, ns, tq, kernel, scale=2.0 ** -60)
    # tiny rows of queries, and no scales of the keys' own
    C.ks, C.vs = torch.ones_like(C.ks), torch.ones_like(C.vs)
    C.cache = K.PagedCache(C.kp, C.vp)
    q = (rand(g, sum(ns), 14, 64) * (2.0 ** -100 if tq == "bf16" else 2.0 ** -14)).to(getattr(torch, {"f16": "float16", "bf16": "bfloat16"}[tq]))
    out = torch.zeros_like(q)
    C.cache.attend(K.PagedBatch(starts(ns), ints(kvs), C.table, **HINTS[kernel]), q, out, scale=2.0 ** -60)
    C.cache.check()
    check_attention(C, q, out, ns, scale=2.0 ** -60)
