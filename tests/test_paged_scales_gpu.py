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


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 48])   # by vectors, and (with rows off their alignment below) one at a time
def test_append_into_a_head_whose_scale_is_zero(t, d):
    """All that such a head can hold is 0: what is stored must not be 0 / 0."""
    g = gen(33)
    C = Cache(g, "e4m3", 3, d, 16, [20], junk=7.0)
    C.ks[0] = C.vs[1] = 0
    x = rand(g, 20, 3, d).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t])
    x[:, 0, ::2] = 0
    x[:, 1, 1::2] = 0
    rows = torch.zeros(20, 3, d + 3, dtype=x.dtype, device=dev())[:, :, 1:d + 1] if d == 48 else torch.empty_like(x)
    rows.copy_(x)
    C.cache.append(K.PagedBatch(ints([0, 20]), ints([20]), C.table, 20), rows, rows)
    C.cache.check()
    k, v = C.rows(0)
    assert (k[:, 0] == 0).all() and (v[:, 1] == 0).all()
    for got, scale, heads in ((k, C.ks, (1, 2)), (v, C.vs, (0, 2))):
        for h in heads:
            sc = scale[h].item()
            want = x[:, h].double()
            tol = u("e4m3") * want.abs() * (1 + 2 ** -20) + 2.0 ** -10 * sc * (1 + 2 ** -20)
            assert ((got[:, h] - want).abs() <= tol).all()


@BOTH
@pytest.mark.parametrize("top", [60, 112, 120])
def test_rows_of_large_bf16_queries_over_8_bits(kernel, top):
    """Scores of ordinary size from queries of 2^top and keys of 2^-top."""
    g = gen(34)
    ns, kvs = [1, 60], [200, 300]
    C = Cache(g, "e4m3", 2, 128, 32, kvs)
    C.fill(g, 0), C.fill(g, 1)
    C.ks *= 2.0 ** -top
    n = sum(ns)
    q = rand(g, n, 14, 128)
    q[::3] *= 0.25
    q[1::7, :, 5] = 100.0   # one large value: 2^6.6 times the others
    q = (q * 2.0 ** top).to(torch.bfloat16)
    assert torch.isfinite(q).all()
    out = torch.zeros_like(q)
    C.cache.attend(K.PagedBatch(starts(ns), ints(kvs), C.table, **HINTS[kernel]), q, out)
    C.cache.check()
    check_attention(C, q, out, ns)


@BOTH
@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
def test_huge_queries_take_one_keys_value(kernel, tc):
    """Scores of 2^60 and more, whose softmax is a 1 at the largest: the output is that key's value, rounded once. (Rows
    whose two largest scores are closer than four times what a score may be off are left out: 2 d u32 sum|q k| each.)"""
    g = gen(35)
    n, kv, d = 40, 300, 128
    C = Cache(g, tc, 1, d, 32, [kv])
    C.fill(g, 0)
    q = (rand(g, n, 7, d) * 2.0 ** 60).to(torch.bfloat16)
    out = torch.zeros_like(q)
    C.cache.attend(K.PagedBatch(starts([n]), ints([kv]), C.table, **HINTS[kernel]), q, out)
    k, v = C.rows(0)
    s = torch.einsum("nhd,td->nht", q.double(), k[:, 0]) * d ** -0.5
    off = torch.einsum("nhd,td->nht", q.double().abs(), k[:, 0].abs()).amax(-1) * d ** -0.5 * 2 * d * 2.0 ** -24
    pos = kv - n + torch.arange(n, device=dev())
    s.masked_fill_(torch.arange(kv, device=dev()) > pos[:, None, None], -math.inf)
    two, at = s.topk(2, -1)
    clear = two[..., 0] - two[..., 1] > 4 * off
    assert clear.double().mean() > 0.9
    want = v[at[..., 0], 0]
    # the value's scale, the sum's reciprocal and the product: three roundings of 32 bits, then the output's
    tol = want.abs() * (u("bf16") + 4 * 2.0 ** -24) * (1 + 2.0 ** -7) + 2.0 ** -134
    assert ((out.double() - want).abs() <= tol)[clear].all()


@BOTH
@pytest.mark.parametrize("tq,tc", KINDS)
@pytest.mark.parametrize("window", [0, 1000])
def test_nan_in_a_value_stays_with_the_rows_of_its_block(kernel, tq, tc, window):
    """NaN in V reaches every row that sees it and no row whose block (256 packed rows at most) sees none: those have the
    bits that they have without it. A window's lost positions and a chunk's later ones are such."""
    g = gen(36)
    n, kv, rep, d = 500, 3000, 8, 128
    C = Cache(g, tc, 2, d, 64, [kv])
    C.fill(g, 0)
    q = rand(g, n, 2 * rep, d).to(getattr(torch, {"f16": "float16", "bf16": "bfloat16"}[tq]))
    batch = K.PagedBatch(starts([n]), ints([kv]), C.table, **HINTS[kernel])
    clean = C.cache.attend(batch, q, window=window)
    check_attention(C, q, clean, [n], window=window)
    spots = [(1600, 0, 3), (2504, 1, 100), (2999, 0, 64), (10, 1, 7)]   # (position, head, d)
    for t, h, e in spots:
        pg, sl = C.places(0, torch.tensor([t], device=dev()))
        C.vp[pg, h, sl, e] = float("nan")
    got = C.cache.attend(batch, q, window=window)
    C.cache.check()
    pos = kv - n + torch.arange(n, device=dev())
    sees = torch.zeros(n, 2, rep, d, dtype=torch.bool, device=dev())
    block = sees.clone()
    tokens = 256 // rep
    for t, h, e in spots:
        s = (t <= pos) & ((t > pos - window) if window else torch.ones_like(pos, dtype=torch.bool))
        sees[s, h, :, e] = True
        near = torch.nn.functional.pad(s, (0, -n % tokens)).view(-1, tokens).any(1).repeat_interleave(tokens)[:n]
        block[near, h, :, e] = True
    sees, block = sees.flatten(1, 2), block.flatten(1, 2)
    assert got[sees].isnan().all()
    assert torch.equal(got[~block], clean[~block])
    assert sees.any() and (~block).any()
