"""The operators on a caller-owned paged cache against plain forms in 64 bits.

Tolerances, derived from the arithmetic (u = eps/2 of a type, the most that one rounding is off):
rotation: each of the two products carries the table's rounding and its own, their sum one more, all fp32:
    3 u32 (|x0 c| + |x1 s|), below 4 u32 amp (|x0| + |x1|); then u of the output's type (and, below its normal range,
    half its smallest step).
attention: the probabilities are rounded to the product's type (u_p); a score is off by at most
    e = 2 d u32 scale sum|q k| (fp32 sums of exact products, twice the bound for sums that are cut, not rounded) plus
    4 u32 |score| (the factor, the subtraction), which moves a probability by 2e relative (its own and the sum's);
    exp2 and the sums add less than 2^-18. So |out - exact| <= (u_p + 2 e + 2^-18) sum p |v| + u_out |out|.
    For 8-bit caches the scales are one rounding each (in 2^-18).
"""
import itertools
import math

import numpy as np
import pytest

import kore_b200 as K

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
U32 = 2.0 ** -24
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134, "e4m3": 2.0 ** -10}   # half the smallest step
GUARD = 7.0   # written around outputs and into pages that nothing may touch


def u(t):
    return torch.finfo(DT[t]).eps / 2


def dev():
    return torch.device("cuda", 0)


def rand(g, *shape):
    return torch.randn(*shape, device=dev(), generator=g)


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=dev())


def strided(x, how):
    """The rows x [n][h][d] laid out otherwise: part of wider rows, heads apart, or off any vector's alignment."""
    n, h, d = x.shape
    if how == "dense":
        return x.contiguous()
    if how == "fused":
        wide = torch.full((n, (h + 3) * d), GUARD, dtype=x.dtype, device=x.device)
        y = wide[:, d:d + h * d].unflatten(1, (h, d))
    elif how == "heads_first":
        y = torch.full((h, n, d), GUARD, dtype=x.dtype, device=x.device).transpose(0, 1)
    else:   # odd
        y = torch.full((n, h, d + 3), GUARD, dtype=x.dtype, device=x.device)[:, :, 1:d + 1]
    y.copy_(x)
    return y


# ---------------------------------------------------------------- rotary positions

def turned(x, pos, freq, amp, interleaved):
    """x [n][h][d] rotated at pos [n], in 64 bits; and the bound's sum |x0| + |x1| at each value."""
    x, r = x.double(), 2 * len(freq)
    a = pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = a.cos()[:, None] * amp, a.sin()[:, None] * amp
    y, m = x.clone(), torch.zeros_like(x)
    e0, e1 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    x0, x1 = x[..., e0], x[..., e1]
    y[..., e0], y[..., e1] = x0 * c - x1 * s, x0 * s + x1 * c
    m[..., e0] = m[..., e1] = (x0.abs() + x1.abs()) * amp
    return y, m


def near_rounded(got, want, m, t):
    tol = 4 * U32 * m + u(t) * (want.abs() + 4 * U32 * m) + TINY[t]
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (got.double() - want).abs()[bad][:4]


SCALED = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=4.0, original_ctx=8192)]


@pytest.mark.parametrize("kw", SCALED)
@pytest.mark.parametrize("rot", [2, 24, 128])
def test_table_is_rounded_from_64_bits(kw, rot):
    n = 40000
    t = K.RopeTable(n, rot, **kw)
    freq, amp = K.rope_frequencies(rot, **kw)
    a = np.outer(np.arange(n, dtype=np.float64), np.array(freq, np.float64))
    want = np.stack([np.cos(a), np.sin(a)], -1) * amp
    err = np.abs(t.table.cpu().numpy().astype(np.float64) - want)
    # a value below amp <= 2 is rounded by at most 2^-24 * 2; the 64-bit sides differ by far less
    assert err.max() <= (2.0 ** -24 if amp == 1 else 2.0 ** -23) * (1 + 1e-6)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (128, 32), (64, 20), (80, 80), (96, 6), (2, 2), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,h,how", [(1, 28, "dense"), (33, 3, "fused"), (7, 14, "odd"), (130, 5, "heads_first")])
def test_rope(t, d, rot, interleaved, n, h, how):
    g = gen(n * d + rot)
    x = strided(rand(g, n, h, d).to(DT[t]), how)
    pos = torch.randint(0, 5000, (n,), device=dev(), generator=g).to(torch.int32)
    table = K.RopeTable(5000, rot, interleaved=interleaved)
    out = strided(torch.full((n, h, d), GUARD, dtype=DT[t], device=dev()), how)
    if n > 1:
        pos[n // 2] = -1   # a row of padding
    table.rotate(x, pos, out=out)
    table.check()
    keep = pos >= 0
    want, m = turned(x, pos, *K.rope_frequencies(rot), interleaved)
    near_rounded(out[keep], want[keep], m[keep], t)
    assert (out[~keep] == GUARD).all()
    assert torch.equal(out[keep][..., rot:], x[keep][..., rot:])   # values behind rot are copied
    before = x.clone()
    table.rotate(x, pos, out=x)   # in place
    assert torch.equal(x[keep], out[keep]) and torch.equal(x[~keep], before[~keep])


def test_rope_positions_outside_the_table_are_reported():
    table = K.RopeTable(16, 8)
    x = torch.ones(3, 1, 16, device=dev())
    out = torch.full_like(x, GUARD)
    table.rotate(x, ints([0, 16, 15]), out=out)
    with pytest.raises(K.KoreCudaError, match="outside the rotation table"):
        table.check()
    assert (out[1] == GUARD).all() and (out[0] == 1).all() and not (out[2] == GUARD).any()
    table.check()   # reported once


def test_rope_refuses_tensors_that_do_not_fit():
    table = K.RopeTable(16, 8)
    x = torch.ones(3, 2, 16, device=dev())
    pos = ints([0, 1, 2])
    for bad in (dict(x=x[0]), dict(x=x.transpose(1, 2)), dict(x=x.cpu()), dict(pos=pos[:2]), dict(pos=pos.long()),
                dict(out=x[:2].clone()), dict(x=x.double(), out=x)):
        a = dict(x=x, pos=pos, out=x)
        a.update(bad)
        with pytest.raises((ValueError, K.KoreCudaError)):
            table.rotate(a["x"], a["pos"], out=a["out"])


# ---------------------------------------------------------------- a paged cache

class Cache:
    """Pages with a page table whose physical pages are shuffled; pages and slots that no position has hold `junk`."""

    def __init__(self, g, t, G, d, P, kvs, spare=2, alternate=False, junk=float("nan")):
        self.t, self.G, self.d, self.P, self.kvs = t, G, d, P, kvs
        used = [-(-k // P) for k in kvs]
        total = sum(used) + spare
        perm = torch.randperm(total, device=dev(), generator=g).tolist()
        width = max(used + [1]) + 1
        table, at = [], 0
        for n in used:
            table.append(perm[at:at + n] + [-1] * (width - n))
            at += n
        self.table = ints(table).reshape(len(kvs), width)
        if alternate:   # K and V by turns in one pool
            pool = torch.full((total, 2, G, P, d), junk, device=dev()).to(DT[t])
            self.kp, self.vp = pool[:, 0], pool[:, 1]
        else:
            self.kp, self.vp = (torch.full((total, G, P, d), junk, device=dev()).to(DT[t]) for _ in range(2))
        self.ks = self.vs = None
        if t == "e4m3":
            self.ks, self.vs = (0.01 * (1 + torch.rand(G, device=dev(), generator=g)) for _ in range(2))
        self.cache = K.PagedCache(self.kp, self.vp, k_scale=self.ks, v_scale=self.vs)

    def places(self, s, p):
        p = p.long()
        return self.table[s].long()[p // self.P], p % self.P

    def fill(self, g, s, amp=1.0):
        """N(0, 1) keys and values at every position of sequence s."""
        n = self.kvs[s]
        pg, sl = self.places(s, torch.arange(n, device=dev()))
        for pages, scale in ((self.kp, self.ks), (self.vp, self.vs)):
            x = rand(g, n, self.G, self.d) * amp
            if scale is not None:
                x = (x / scale[:, None]).clamp(-448, 448)
            pages[pg, :, sl] = x.to(DT[self.t])

    def rows(self, s):
        """The sequence's keys and values [kv][G][d] in 64 bits."""
        pg, sl = self.places(s, torch.arange(self.kvs[s], device=dev()))
        k, v = self.kp[pg, :, sl].double(), self.vp[pg, :, sl].double()
        if self.ks is not None:
            k, v = k * self.ks.double()[:, None], v * self.vs.double()[:, None]
        return k, v


def starts(ns):
    return ints([0] + list(itertools.accumulate(ns)))


@pytest.mark.parametrize("t,c", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f32", "e4m3"), ("f16", "f16"),
                                 ("f16", "e4m3"), ("bf16", "bf16"), ("bf16", "e4m3")])
@pytest.mark.parametrize("G,d,rot,P,how,interleaved", [(4, 128, 128, 64, "fused", False), (2, 64, 32, 16, "dense", True),
                                                       (3, 96, 96, 48, "odd", False), (1, 256, 20, 32, "heads_first", True),
                                                       (2, 16, 0, 16, "dense", False)])
def test_append(t, c, G, d, rot, P, how, interleaved):
    g = gen(d + P)
    ns, past = [1, 0, 3 * P + 5, 2, P, 1], [0, 5, 7, P - 1, P, 40]
    kvs = [a + b for a, b in zip(ns, past)]
    C = Cache(g, c, G, d, P, kvs, alternate=(G == 4), junk=GUARD)
    n, H = sum(ns) + 3, 2 * G + 1
    k, v, q = (strided((rand(g, n, h, d) * 3).to(DT[t]), how) for h in (G, G, H))
    q_out = strided(torch.full((n, H, d), GUARD, dtype=DT[t], device=dev()), how)
    table = K.RopeTable(max(kvs), rot, interleaved=interleaved, scaling="yarn", factor=2.0, original_ctx=64) if rot else None
    kp0, vp0 = C.kp.clone(), C.vp.clone()
    batch = K.PagedBatch(starts(ns), ints(kvs), C.table, max(ns))
    C.cache.append(batch, k, v, rope=table, q=q, q_out=q_out)
    C.cache.check()
    freq, amp = K.rope_frequencies(rot, scaling="yarn", factor=2.0, original_ctx=64) if rot else ([], 1.0)
    touched = torch.zeros(C.kp.shape[:1] + C.kp.shape[2:3], dtype=torch.bool, device=dev())
    at = 0
    for s, m in enumerate(ns):
        pos = torch.arange(past[s], kvs[s], device=dev())
        rows = slice(at, at + m)
        at += m
        pg, sl = C.places(s, pos)
        touched[pg, sl] = True
        for x, pages, scale, turn in ((k, C.kp, C.ks, True), (v, C.vp, C.vs, False)):
            want, mag = turned(x[rows], pos, freq if turn else [], amp, interleaved)
            got = pages[pg, :, sl].double()
            if c == "e4m3":
                sc = scale.double()[:, None]
                # x / scale is rounded once more in fp32, then to 8 bits, at most 448
                lim = (want / sc).clamp(-448, 448)
                tol = u("e4m3") * lim.abs() * (1 + 2 ** -20) + TINY["e4m3"] + 8 * U32 * mag / sc + 2 * U32 * lim.abs()
                assert ((got - lim).abs() <= tol).all()
            else:
                near_rounded(got, want, mag, c)
        want, mag = turned(q[rows], pos, freq, amp, interleaved)
        near_rounded(q_out[rows], want, mag, t)
    # nothing else is written: other slots and pages, rows behind the last sequence
    for pages, before in ((C.kp, kp0), (C.vp, vp0)):
        same = (pages.float() == before.float()).all(-1).all(1)   # [pages][slots]
        assert same[~touched].all()
    assert (q_out[sum(ns):] == GUARD).all()
    # without q, and into the same places: the same bits
    kp1 = C.kp.clone()
    C.cache.append(batch, k, v, rope=table)
    assert torch.equal(C.kp.view(torch.uint8) if c == "e4m3" else C.kp, kp1.view(torch.uint8) if c == "e4m3" else kp1)


def test_append_fp32_keys_are_the_contexts_bits():
    """The fp32 cache of this operator and a context's hold the same key rows, bit for bit."""
    G, d, n = 4, 128, 300
    g = gen(3)
    C = Cache(g, "f32", G, d, 64, [n])
    k, v = rand(g, n, G, d), rand(g, n, G, d)
    C.cache.append(K.PagedBatch(ints([0, n]), ints([n]), C.table, n), k, v, rope=K.RopeTable(n, d))
    ctx = K.KoreCuda(1, 28, G, d, n)
    ctx.append(0, 0, 0, k.cpu().numpy(), v.cpu().numpy())
    kr, vr = ctx.kv_read(0, 0, 0, n)
    ctx.close()
    got_k, got_v = C.rows(0)
    same = np.mean(got_k.float().cpu().numpy().reshape(n, -1) == kr)
    assert same > 0.999   # the tables' cosines may differ where 64-bit values lie at a border of 32
    np.testing.assert_allclose(got_k.cpu().numpy().reshape(n, -1), kr, rtol=0, atol=1e-6)
    assert np.array_equal(got_v.float().cpu().numpy().reshape(n, -1), vr)


def test_append_special_values_into_eight_bits():
    C = Cache(gen(1), "e4m3", 1, 16, 16, [1])
    C.ks.fill_(1.0), C.vs.fill_(2.0)
    x = torch.tensor([0.0, -0.0, 448, 449, 1e30, -1e30, math.inf, -math.inf, math.nan, 2.0 ** -9, 2.0 ** -10,
                      -2.0 ** -11, 17, 18, 1.0625, 1.1875], device=dev()).reshape(1, 1, 16)
    C.cache.append(K.PagedBatch(ints([0, 1]), ints([1]), C.table, 1), x, x * 2)
    # ties to even: 2^-10 -> 0, 17 -> 16, 18 stays, 1.0625 -> 1, 1.1875 -> 1.25
    want = torch.tensor([0.0, 0, 448, 448, 448, -448, 448, -448, math.nan, 2.0 ** -9, 0, 0, 16, 18, 1, 1.25], device=dev())
    pg, sl = C.places(0, torch.zeros(1, device=dev()))
    for pages in (C.kp, C.vp):
        got = pages[pg, 0, sl].float().flatten()
        assert torch.equal(got.nan_to_num(99), want.nan_to_num(99))


@pytest.mark.parametrize("bad,word", [("page", "page id"), ("negative", "page id"), ("short", "bounds"), ("rows", "bounds"),
                                      ("long", "bounds"), ("position", "rotation table")])
def test_append_reports_bad_device_data(bad, word):
    g = gen(2)
    C = Cache(g, "bf16", 2, 64, 16, [20, 20], junk=GUARD)
    table, q_start, kv = C.table.clone(), [0, 4, 8], [20, 20]
    if bad == "page":
        table[1, 1] = C.kp.shape[0]
    elif bad == "negative":
        table[1, 1] = -5
    elif bad == "short":
        kv[1] = 3
    elif bad == "rows":
        q_start[2] = 99
    elif bad == "long":
        kv[1] = table.shape[1] * 16 + 1
    k = torch.ones(8, 2, 64, device=dev(), dtype=torch.bfloat16)
    rope = K.RopeTable(19 if bad == "position" else 64, 64)
    before = C.kp.clone()
    C.cache.append(K.PagedBatch(ints(q_start), ints(kv), table, 4), k, k, rope=rope)
    with pytest.raises(K.KoreCudaError, match=word):
        C.cache.check()
    # the good sequence (its good tokens) is stored; nothing of the bad one
    pg, sl = C.places(0, torch.arange(16, 19, device=dev()))
    assert not (C.kp[pg, :, sl] == GUARD).all(-1).any()
    pg, sl = C.places(1, torch.arange(16, 19, device=dev()))
    if bad != "position":
        assert torch.equal(C.kp[pg, :, sl], before[pg, :, sl])


# ---------------------------------------------------------------- attention

def check_attention(C, q, out, ns, scale=None, causal=True, window=0, lse=None):
    """Every row of out (and lse) against the formula in 64 bits."""
    H, d = q.shape[1:]
    rep = H // C.G
    scale = d ** -0.5 if scale is None else scale
    up = u("f16") if C.t == "e4m3" else u(C.t)
    uo = torch.finfo(out.dtype).eps / 2
    at = 0
    for s, n in enumerate(ns):
        kv = C.kvs[s]
        if n:
            k, v = C.rows(s)
            x = q[at:at + n].double().unflatten(1, (C.G, rep))   # [n][G][rep][d]
            sc = torch.einsum("ngrd,tgd->ngrt", x, k) * scale
            mag = torch.einsum("ngrd,tgd->ngrt", x.abs(), k.abs()) * abs(scale)
            pos = kv - n + torch.arange(n, device=dev())[:, None]
            t = torch.arange(kv, device=dev())
            seen = torch.ones(n, kv, dtype=torch.bool, device=dev())
            if causal:
                seen &= t <= pos
            if window:
                seen &= t > pos - window
            sc = sc.masked_fill(~seen[:, None, None], -math.inf)
            some = seen.any(-1)
            p = torch.softmax(sc, -1).nan_to_num(0.0)
            want = torch.einsum("ngrt,tgd->ngrd", p, v)
            pv = torch.einsum("ngrt,tgd->ngrd", p, v.abs())
            e = (2 * d * U32 * mag + 4 * U32 * sc.abs().nan_to_num(0, 0, 0)).masked_fill(~seen[:, None, None], 0)
            e = e.amax(-1, keepdim=True) if kv else torch.zeros(n, C.G, rep, 1, device=dev())
            tol = (up + 2 * e + 2.0 ** -18) * pv
            tol = tol + uo * (want.abs() + tol) + TINY["f16"]
            got = out[at:at + n].double().unflatten(1, (C.G, rep))
            diff = (got - want).abs()
            assert torch.isfinite(got).all() and (diff <= tol).all(), (s, n, kv, (diff / tol).max().item())
            assert (got[~some] == 0).all()
            if lse is not None:
                wl = torch.logsumexp(sc, -1)
                gl = lse[at:at + n].double().unflatten(1, (C.G, rep))
                assert (gl[~some] == -math.inf).all()
                assert ((gl - wl).abs()[some] <= (e[..., 0] + 2.0 ** -18 + 4 * U32 * wl.abs())[some]).all()
        at += n


# what the host says of the batch chooses the kernel: 16 rows a unit, or 256 on tcgen05
HINTS = {"rows": dict(max_q=1), "tiles": dict(max_q=1 << 20, max_kv=1 << 30)}
BOTH = pytest.mark.parametrize("kernel", list(HINTS))


def attend(g, C, H, ns, tq, kernel, how="dense", pad=2, **kw):
    n = sum(ns) + pad
    q = strided(rand(g, n, H, C.d).to(DT[tq]), how)
    out = strided(torch.full((n, H, C.d), GUARD, dtype=DT[tq], device=dev()), how)
    lse = torch.full((n, H), GUARD, device=dev())
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    C.cache.attend(batch, q, out, lse=lse, **kw)
    C.cache.check()
    check_attention(C, q, out, ns, lse=lse, **kw)
    assert (out[sum(ns):] == GUARD).all() and (lse[sum(ns):] == GUARD).all()   # rows behind the last sequence
    return q, out, batch


KINDS = [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")]

# (new tokens, cached positions) of each sequence
BATCHES = {
    "one": [(1, 1)],
    "tile_edges": [(1, 15), (1, 16), (1, 17), (1, 127), (1, 128), (1, 129), (1, 255), (1, 257)],
    "ragged_steps": [(1, 700), (1, 3), (1, 2049), (1, 64), (1, 1000)],
    "none_and_empty": [(0, 50), (2, 2), (0, 0), (1, 0), (3, 2), (5, 300), (0, 7)],   # 0 keys; a row before position 0
    "chunk": [(40, 40)],
    "chunks": [(130, 390), (1, 511), (257, 257), (19, 1000)],
    "long_chunk": [(300, 1500)],
}


@pytest.mark.parametrize("tq,tc", KINDS)
@pytest.mark.parametrize("H,G,d,P", [(28, 4, 128, 64), (14, 2, 64, 16), (8, 8, 128, 48), (40, 2, 64, 256), (3, 1, 128, 16)])
@pytest.mark.parametrize("which", list(BATCHES))
@BOTH
def test_attention(kernel, tq, tc, H, G, d, P, which):
    g = gen(H + P)
    ns, kvs = map(list, zip(*BATCHES[which]))
    C = Cache(g, tc, G, d, P, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    attend(g, C, H, ns, tq, kernel)


@BOTH
@pytest.mark.parametrize("tq,tc", [("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=100), dict(causal=False), dict(causal=False, window=33),
                                dict(scale=0.5), dict(scale=-0.2), dict(window=100000),
                                dict(window=2 ** 31 - 1)])
def test_attention_masks_and_scales(kernel, tq, tc, kw):
    g = gen(5)
    ns, kvs = [1, 37, 200, 1, 6], [400, 37, 900, 1, 129]
    C = Cache(g, tc, 2, 128, 64, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    attend(g, C, 16, ns, tq, kernel, **kw)


@BOTH
@pytest.mark.parametrize("how", ["fused", "heads_first", "odd"])
@pytest.mark.parametrize("ns,kvs", [([1, 1], [300, 77]), ([150, 3], [300, 77])])
def test_attention_of_strided_rows(kernel, how, ns, kvs):
    g = gen(6)
    for t, d in (("bf16", 128), ("f16", 64)):
        C = Cache(g, t, 2, d, 32, kvs, alternate=True)
        for s in range(2):
            C.fill(g, s)
        attend(g, C, 14, ns, t, kernel, how=how)


@pytest.mark.parametrize("max_q", [0, 1, 17, 100000])
@pytest.mark.parametrize("max_kv", [0, 1, 1 << 30])
def test_attention_whatever_the_hints(max_q, max_kv):
    """max_q and max_kv choose the kernel and bound nothing."""
    g = gen(7)
    ns, kvs = [1, 90, 0, 30], [500, 200, 3, 31]
    C = Cache(g, "bf16", 2, 64, 64, kvs)
    for s in range(4):
        C.fill(g, s)
    q = rand(g, sum(ns), 14, 64).to(torch.bfloat16)
    out = C.cache.attend(K.PagedBatch(starts(ns), ints(kvs), C.table, max_q, max_kv), q)
    C.cache.check()
    check_attention(C, q, out, ns)


@BOTH
@pytest.mark.parametrize("tq,tc", KINDS)
def test_attention_of_large_scores(kernel, tq, tc):
    """Sharp softmaxes and reference maxima that move: keys that grow along the sequence."""
    g = gen(8)
    ns, kvs = [1, 140], [3000, 600]
    C = Cache(g, tc, 2, 128, 64, kvs)
    for s, kv in enumerate(kvs):
        C.fill(g, s)
        pg, sl = C.places(s, torch.arange(kv, device=dev()))
        k = C.kp[pg, :, sl].float() * torch.linspace(0.01, 1.0 if tc == "e4m3" else 8.0, kv, device=dev())[:, None, None]
        C.kp[pg, :, sl] = k.to(DT[tc])
    attend(g, C, 14, ns, tq, kernel)


@BOTH
@pytest.mark.parametrize("tq,tc", KINDS)
def test_attention_of_one_loud_key_among_many_faint_ones(kernel, tq, tc):
    """20000 keys that each have 2^-20 of one key's weight, and together 2 % of it: probabilities far below the smallest
    normal f16."""
    g = gen(20)
    kv, n = 20000, 3
    C = Cache(g, tc, 1, 64, 64, [kv])
    C.fill(g, 0)
    pg, sl = C.places(0, torch.arange(kv, device=dev()))
    scale = C.ks if tc == "e4m3" else torch.ones(1, device=dev())
    one = torch.ones(1, 64, device=dev()) / scale[:, None]   # k: 1 at every value (the loud key: 2)
    C.kp[pg, :, sl] = one.to(DT[tc]).expand(kv, 1, 64)
    C.kp[pg[777], :, sl[777]] = (2 * one).to(DT[tc])
    v = C.vp[pg, :, sl].float().abs()   # of one sign, so that what the faint keys add does not cancel
    C.vp[pg, :, sl] = v.to(DT[tc])
    C.vp[pg[777], :, sl[777]] = 0
    q = torch.full((n, 2, 64), 20 * math.log(2) * 8 / 64, device=dev()).to(DT[tq])
    out = torch.zeros_like(q)
    C.cache.attend(K.PagedBatch(starts([n]), ints([kv]), C.table, **HINTS[kernel]), q, out)
    C.cache.check()
    check_attention(C, q, out, [n])


@BOTH
@pytest.mark.parametrize("tq,tc,top", [("bf16", "e4m3", 60), ("bf16", "bf16", 60), ("f16", "e4m3", 10)])
def test_attention_of_queries_of_any_size(kernel, tq, tc, top):
    """Rows of q that are all zeros, tiny or huge, and a row with one large value (bf16 queries over an 8-bit cache are
    brought to f16 a row at a time)."""
    g = gen(24)
    n = 40
    C = Cache(g, tc, 1, 128, 32, [300])
    C.fill(g, 0)
    q = rand(g, n, 7, 128)
    q[::5] = 0
    q[1::5] *= 2.0 ** -top if tq == "bf16" else 2.0 ** -6
    q[2::5] *= 2.0 ** top
    q[3::5, :, 17] = 1000.0
    q = q.to(DT[tq])
    out = torch.zeros_like(q)
    C.cache.attend(K.PagedBatch(starts([n]), ints([300]), C.table, **HINTS[kernel]), q, out)
    check_attention(C, q, out, [n])


@BOTH
@pytest.mark.parametrize("H,G,d", [(128, 1, 64), (16, 16, 128)])
def test_attention_of_wide_and_of_single_groups(kernel, H, G, d):
    g = gen(21)
    ns, kvs = [3, 1, 20], [200, 333, 20]
    C = Cache(g, "bf16", G, d, 32, kvs)
    for s in range(3):
        C.fill(g, s)
    attend(g, C, H, ns, "bf16", kernel)


@BOTH
def test_attention_of_a_whole_batch_of_sequences(kernel):
    """4096 sequences, some of them empty."""
    g = gen(22)
    kvs = torch.randint(0, 20, (4096,), generator=torch.Generator().manual_seed(2)).tolist()
    ns = [min(1, k) for k in kvs]
    C = Cache(g, "f16", 1, 64, 16, kvs)
    k = rand(g, *C.kp.shape).to(torch.float16)
    C.kp.copy_(k), C.vp.copy_(k.flip(0))
    n = sum(ns)
    q = rand(g, n, 2, 64).to(torch.float16)
    out = torch.zeros_like(q)
    C.cache.attend(K.PagedBatch(starts(ns), ints(kvs), C.table, **HINTS[kernel]), q, out)
    C.cache.check()
    at = [i for i, m in enumerate(ns) if m]
    for j in list(range(0, n, 97)) + [n - 1]:
        D = Cache.__new__(Cache)
        D.__dict__.update(C.__dict__, kvs=[kvs[at[j]]], table=C.table[at[j]:at[j] + 1])
        check_attention(D, q[j:j + 1], out[j:j + 1], [1])


@BOTH
def test_attention_with_a_page_table_of_a_large_capacity(kernel):
    """So wide a table that sums of work are formed in 64 bits."""
    g = gen(23)
    ns, kvs = [700, 600], [700, 1100]
    C = Cache(g, "bf16", 1, 64, 256, kvs)
    C.fill(g, 0), C.fill(g, 1)
    wide = torch.full((2, 1500000), -1, dtype=torch.int32, device=dev())
    wide[:, :C.table.shape[1]] = C.table
    C.table = wide
    attend(g, C, 7, ns, "bf16", kernel)


@BOTH
def test_attention_of_many_short_sequences(kernel):
    g = gen(9)
    kvs = torch.randint(1, 90, (300,), generator=torch.Generator().manual_seed(1)).tolist()
    C = Cache(g, "bf16", 2, 64, 16, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    attend(g, C, 4, [1] * 300, "bf16", kernel)


@pytest.mark.parametrize("tq,tc", [("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("n", [1, 40])
@BOTH
def test_attention_of_a_long_context_is_split_and_the_same_each_time(kernel, tq, tc, n):
    g = gen(10)
    C = Cache(g, tc, 1, 128, 256, [70001])
    C.fill(g, 0)
    q, out, batch = attend(g, C, 8, [n], tq, kernel)
    again = torch.zeros_like(out)
    for _ in range(3):
        C.cache.attend(batch, q, again)
        assert torch.equal(again[:n], out[:n])


@BOTH
def test_attention_offsets_beyond_32_bits(kernel):
    """A pool of more than 2^32 elements: pages at both ends of it."""
    G, d, P, n = 4, 128, 1024, 60
    pages = 2 ** 32 // (G * P * d) + 3
    kp = torch.empty(pages, G, P, d, dtype=torch.bfloat16, device=dev())
    vp = torch.empty_like(kp)
    g = gen(11)
    C = Cache(g, "bf16", G, d, P, [2500], spare=0)
    C.kp, C.vp = kp, vp
    C.cache = K.PagedCache(kp, vp)
    C.table = ints([[pages - 1, 0, pages - 2, -1]])
    C.fill(g, 0)
    attend(g, C, 28, [n], "bf16", kernel)
    k = rand(g, n, G, d).to(torch.bfloat16)
    C.table = ints([[0, 1, pages - 1, -1]])
    C.cache.append(K.PagedBatch(ints([0, n]), ints([2500]), C.table, n), k, k)
    pg, sl = C.places(0, torch.arange(2500 - n, 2500, device=dev()))
    assert torch.equal(kp[pg, :, sl], k) and torch.equal(vp[pg, :, sl], k)


@pytest.mark.parametrize("tq,tc", [("bf16", "bf16"), ("bf16", "e4m3")])
@pytest.mark.parametrize("n", [1, 30])
@BOTH
def test_attention_reads_nothing_before_the_window(kernel, tq, tc, n):
    """Pages wholly before every row's window may be gone from the table."""
    g = gen(12)
    C = Cache(g, tc, 2, 64, 32, [1000])
    C.fill(g, 0)
    kp = C.table.clone()
    first = (1000 - n) - 200 + 1
    q, out, batch = attend(g, C, 14, [n], tq, kernel, window=200)
    C.table[0, :first // 32] = -1
    pg = kp[0, first // 32].long()
    C.kp[pg, :, :first % 32] = float("nan")   # before the window, in its first page
    C.vp[pg, :, :first % 32] = float("nan")
    again = torch.zeros_like(out)
    C.cache.attend(batch, q, again, window=200)
    C.cache.check()
    assert torch.equal(again[:n], out[:n])


@BOTH
def test_attention_passes_nan_and_infinity_on_to_their_rows(kernel):
    g = gen(13)
    for tq, tc in KINDS:
        C = Cache(g, tc, 1, 64, 32, [80, 80])
        C.fill(g, 0), C.fill(g, 1)
        q = rand(g, 2, 2, 64).to(DT[tq])
        q[0, 1, 3] = math.nan
        pg, sl = C.places(1, torch.tensor([11], device=dev()))
        C.vp[pg, 0, sl, 5] = float("nan")
        out = C.cache.attend(K.PagedBatch(ints([0, 1, 2]), ints([80, 80]), C.table, **HINTS[kernel]), q)
        assert torch.isfinite(out[0, 0]).all() and out[0, 1].isnan().all()
        assert out[1, :, 5].isnan().all() and torch.isfinite(out[1, :, :5]).all() and torch.isfinite(out[1, :, 6:]).all()


@pytest.mark.parametrize("n", [1, 50])
@BOTH
@pytest.mark.parametrize("bad,word", [("page", "page id"), ("rows", "bounds"), ("long", "bounds"), ("negative", "bounds")])
def test_attention_reports_bad_device_data(kernel, n, bad, word):
    g = gen(14)
    ns, kvs = [n, n], [150, 150]
    C = Cache(g, "bf16", 2, 64, 16, kvs)
    C.fill(g, 0), C.fill(g, 1)
    q = rand(g, 2 * n, 14, 64).to(torch.bfloat16)
    out = torch.full_like(q, GUARD)
    table, q_start, kv = C.table.clone(), [0, n, 2 * n], list(kvs)
    if bad == "page":
        table[1, 3] = 10 ** 6
    elif bad == "rows":
        q_start[2] = 2 * n + 1
    elif bad == "long":
        kv[1] = 16 * table.shape[1] + 1
    else:
        kv[1] = -1
    C.cache.attend(K.PagedBatch(ints(q_start), ints(kv), table, **HINTS[kernel]), q, out)
    with pytest.raises(K.KoreCudaError, match=word):
        C.cache.check()
    C.kvs = [150]
    check_attention(C, q[:n], out[:n], [n])   # the good sequence
    if bad != "page":
        assert (out[n:] == GUARD).all()
    out2 = torch.full_like(q, GUARD)   # the workspace is as it was: the next call is right
    C.cache.attend(K.PagedBatch(ints([0, n]), ints([150]), C.table[:1].contiguous(), **HINTS[kernel]), q, out2)
    C.cache.check()
    assert torch.equal(out2[:n], out[:n]) or bad == "page"


def test_attention_refuses_tensors_that_do_not_fit():
    g = gen(15)
    C = Cache(g, "bf16", 2, 64, 16, [20])
    C.fill(g, 0)
    batch = K.PagedBatch(ints([0, 1]), ints([20]), C.table, 1)
    q = rand(g, 1, 4, 64).to(torch.bfloat16)
    for bad in (q.half(), q.float(), q[:, :3], q[:, :, :32], q.cpu(), q[0], rand(g, 1, 64, 4).to(torch.bfloat16).transpose(1, 2)):
        with pytest.raises((ValueError, K.KoreCudaError)):
            C.cache.attend(batch, bad)
    for kw in (dict(out=q), dict(out=q[:, :2]), dict(lse=torch.zeros(1, 3, device=dev())), dict(window=-1),
               dict(workspace=torch.zeros(64, dtype=torch.uint8, device=dev()))):
        with pytest.raises((ValueError, K.KoreCudaError)):
            C.cache.attend(batch, q, **kw)
    f = Cache(g, "f32", 2, 64, 16, [20])
    with pytest.raises(K.KoreCudaError, match="type"):
        f.cache.attend(batch, q)
    with pytest.raises(ValueError):
        K.PagedCache(C.kp, C.vp[:-1])
    with pytest.raises(ValueError):
        K.PagedCache(C.kp, C.vp, k_scale=torch.ones(3, device=dev()))
    with pytest.raises(ValueError):
        K.PagedBatch(ints([0, 1, 2]), ints([20]), C.table, 1)


# ---------------------------------------------------------------- streams, graphs, the operators together

@BOTH
def test_calls_on_two_streams_at_once(kernel):
    """Default workspaces are a stream's own."""
    g = gen(16)
    C = Cache(g, "bf16", 1, 128, 256, [30000])
    C.fill(g, 0)
    batch = K.PagedBatch(ints([0, 1]), ints([30000]), C.table, **HINTS[kernel])
    qs = [rand(g, 1, 8, 128).to(torch.bfloat16) for _ in range(2)]
    want = [C.cache.attend(batch, q).clone() for q in qs]
    caches = [C.cache, K.PagedCache(C.kp, C.vp)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(qs[0]) for _ in range(20)] for _ in range(2)]
    for i in range(20):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                caches[j].attend(batch, qs[j], outs[j][i])
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, want[j]) for o in outs[j])


@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 24])
@BOTH
def test_captured_step_follows_the_lengths_on_the_device(kernel, tc, n):
    """A step (rotate and append, attend) captured once and replayed as the sequences grow; and two graphs, captured
    one after the other on one stream, replayed on two streams at once."""
    g = gen(17)
    H, G, d, P, steps = 14, 2, 64, 16, 4
    full = [400 + n * steps, 9000 + n * steps]
    C = Cache(g, tc, G, d, P, full)
    C.fill(g, 0), C.fill(g, 1)
    rope = K.RopeTable(max(full), d)
    kv = ints([400 + n, 9000 + n])
    batch = K.PagedBatch(ints([0, n, 2 * n]), kv, C.table, **HINTS[kernel])
    q, k, v = (rand(g, 2 * n, h, d).to(torch.bfloat16) for h in (H, G, G))
    qr, out = torch.zeros_like(q), torch.zeros_like(q)

    def step(o=out):
        C.cache.append(batch, k, v, rope=rope, q=q, q_out=qr)
        C.cache.attend(batch, qr, o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graphs, outs = [], [torch.zeros_like(q) for _ in range(2)]
        for o in outs:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                step(o)
            graphs.append(gr)
    torch.cuda.synchronize()
    for i in range(steps):
        for x, h in ((q, H), (k, G), (v, G)):
            x.copy_(rand(g, 2 * n, h, d))
        kv.copy_(ints([400 + n * (i + 1), 9000 + n * (i + 1)]))
        graphs[0].replay()
        torch.cuda.synchronize()
        C.kvs = kv.tolist()
        check_attention(C, qr, outs[0], [n, n])
    C.cache.check()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        check_attention(C, qr, outs[1], [n, n])


@pytest.mark.parametrize("tq,tc,H,G,d,P", [("bf16", "bf16", 28, 4, 128, 64), ("f16", "e4m3", 14, 2, 64, 16)])
@BOTH
def test_prompts_and_steps_together(kernel, tq, tc, H, G, d, P):
    """Prompts in two chunks, then tokens, of three conversations of different lengths, as a server would run them:
    every step's attention against the formula over what the cache holds, and the cache against the keys and values
    that went in."""
    g = gen(18)
    lens, steps = [300, 41, 150], 3
    total = [x + steps for x in lens]
    C = Cache(g, tc, G, d, P, total)
    rope = K.RopeTable(max(total), d, scaling="linear", factor=2.0)
    freq, amp = K.rope_frequencies(d, scaling="linear", factor=2.0)
    keys = [rand(g, t, G, d).to(DT[tq]) for t in total]
    vals = [rand(g, t, G, d).to(DT[tq]) for t in total]
    at = [0, 0, 0]
    plan = [[200, 41, 1], [100, 0, 149]] + [[1, 1, 1]] * steps
    for ns in plan:
        C.kvs = [a + n for a, n in zip(at, ns)]
        k = torch.cat([x[a:a + n] for x, a, n in zip(keys, at, ns)])
        v = torch.cat([x[a:a + n] for x, a, n in zip(vals, at, ns)])
        q = rand(g, sum(ns), H, d).to(DT[tq])
        batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
        C.cache.append(batch, k, v, rope=rope, q=q, q_out=q)
        out = C.cache.attend(batch, q)
        C.cache.check()
        check_attention(C, q, out, ns)
        at = C.kvs
    for s, t in enumerate(total):
        pos = torch.arange(t, device=dev())
        want, mag = turned(keys[s], pos, freq, amp, False)
        got_k, got_v = C.rows(s)
        if tc == "e4m3":
            sc = C.ks.double()[:, None]
            assert ((got_k - want).abs() <= u(tc) * want.abs() * (1 + 2 ** -18) + (TINY[tc] + 448 * 0) * sc + 8 * U32 * mag).all()
        else:
            near_rounded(got_k, want, mag, tc)
            assert torch.equal(got_v.float(), vals[s].float())


def test_no_tokens_and_no_sequences():
    g = gen(25)
    C = Cache(g, "bf16", 2, 64, 16, [20])
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev())
    batch = K.PagedBatch(ints([0, 0]), ints([20]), C.table, 1)
    C.cache.append(batch, none, none)
    assert C.cache.attend(batch, none).shape == none.shape
    assert K.RopeTable(4, 64).rotate(none, ints([])).shape == none.shape
    x = torch.full((3, 2, 64), GUARD, dtype=torch.bfloat16, device=dev())
    out = x.clone()
    nobody = K.PagedBatch(ints([0]), ints([]), ints([]).reshape(0, 1), 1)
    C.cache.append(nobody, x, x)
    C.cache.attend(nobody, x + 1, out)
    assert torch.equal(out, x)
    C.cache.check()
    with pytest.raises(ValueError, match="together"):
        C.cache.append(batch, x, x, q_out=x)


def test_sequences_may_share_pages():
    """A common beginning in one set of pages, attended by two sequences."""
    g = gen(26)
    for kernel in HINTS:
        C = Cache(g, "bf16", 2, 64, 16, [64, 100])
        C.fill(g, 0), C.fill(g, 1)
        C.table[0, :4] = C.table[1, :4]
        attend(g, C, 14, [3, 40], "bf16", kernel)


def test_tensors_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    with torch.cuda.device(1):
        g = gen(19)
        C = Cache(g, "bf16", 2, 64, 16, [100])
        C.fill(g, 0)
        q = rand(g, 1, 14, 64).to(torch.bfloat16)
        batch = K.PagedBatch(ints([0, 1]), ints([100]), C.table, 1)
    out = C.cache.attend(batch, q)
    check_attention(C, q, out, [1])
