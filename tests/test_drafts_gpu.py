"""A step with drafted tokens over the paged cache: plans and trims against a model of the pool on the host, stores and
tree attention against 64 bits, acceptance and moves against copies, and a run of them together.

Tolerances, derived from the arithmetic (u = eps/2 of a type; U32 of fp32):
norm and rotation: the d squares and their sum are d roundings of terms of one sign, so the mean is off by at most
    (d + 1) U32 relative and its root by half of that; the division, eps, the reciprocal root (2 units in the last place: 4 U32)
    and two products add less than 8 U32: a normed value is off by (d / 2 + 8) U32 of itself. The rotation adds
    4 U32 (|y0| + |y1|) (tests/test_paged_gpu.py), and one rounding to the type follows.
tree attention: as the attention of chunks there.
"""
import math
import random

import pytest

import kore_b200 as K
from tests.test_paged_gpu import attend as attend_chunks
from tests.test_paged_gpu import DT, GUARD, HINTS, KINDS, TINY, U32, Cache, dev, gen, ints, rand, starts, strided, turned, u

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---------------------------------------------------------------- plan and trim

class Model:
    """A pool on the host."""

    def __init__(self, pool):
        self.P, self.width = pool.view.page_tokens, pool.view.table_stride
        self.free = pool.free.tolist()[: int(pool.n_free)]
        self.table = pool.table.tolist()
        self.length = pool.length.tolist()

    def pages(self, n):
        return -(-n // self.P)

    def plan(self, request, n_new, n_tok):
        """(q_start, kv_len, pages of each, slots, pos) and the failures."""
        q, kv, rows, slots, pos, bad, short = [0], [], [], [-1] * n_tok, [-1] * n_tok, set(), False
        left = len(self.free)
        for r, n in zip(request, n_new):
            if r < 0:
                q.append(q[-1]), kv.append(0), rows.append([])
                continue
            first = q[-1]
            q.append(first + max(n, 0))
            ok = (n >= 0 and r < len(self.length) and request.count(r) == 1 and q[-1] <= n_tok
                  and 0 <= self.length[r] <= self.width * self.P and self.length[r] + n <= self.width * self.P)
            if not ok:
                bad.add(7), kv.append(0), rows.append([])
                continue
            base, total = self.length[r], self.length[r] + n
            need = self.pages(total) - self.pages(base)
            if need and (short or need > left):
                short = True
                bad.add(8), kv.append(0), rows.append([])
                continue
            left -= need
            for j in range(self.pages(base), self.pages(total)):
                self.table[r][j] = self.free.pop()
            self.length[r] = total
            kv.append(total), rows.append(self.table[r][: self.pages(total)])
            for i in range(n):
                p = base + i
                slots[first + i], pos[first + i] = self.table[r][p // self.P] * self.P + p % self.P, p
        return q, kv, rows, slots, pos, bad

    def trim(self, request, keep):
        gone, bad = [], False
        for r, k in zip(request, keep):
            if r < 0:
                continue
            if r >= len(self.length) or request.count(r) > 1 or k < 0:
                bad = True
            elif k < self.length[r]:
                for j in range(self.pages(k), self.pages(self.length[r])):
                    gone.append(self.table[r][j])
                    self.table[r][j] = -1
                self.length[r] = k
        self.free += gone[::-1]
        return bad

    def agrees(self, pool):
        n = len(self.free)
        assert int(pool.n_free) == n and pool.free.tolist()[:n] == self.free
        assert pool.length.tolist() == self.length
        assert pool.table.tolist() == self.table


def planned(pool, model, step, request, n_new):
    before = step.page_table.tolist()
    pool.plan(step, ints(request), ints(n_new))
    q, kv, rows, slots, pos, bad = model.plan(request, n_new, step.slots.shape[0])
    assert step.q_start.tolist() == q and step.kv_len.tolist() == kv
    assert step.slots.tolist() == slots and step.pos.tolist() == pos
    got = step.page_table.tolist()
    assert all(g == r + b[len(r):] for g, r, b in zip(got, rows, before))   # (and nothing behind a sequence's pages)
    model.agrees(pool)
    return bad


@pytest.mark.parametrize("n_seq,n_req,P,most,n_tok", [(1, 1, 16, 3, 8), (5, 7, 48, 60, 200), (33, 60, 16, 40, 700),
                                                      (129, 200, 256, 700, 30011), (700, 1000, 64, 9, 4000),
                                                      (4096, 65536, 16, 4, 9000)])
def test_plans_and_trims(n_seq, n_req, P, most, n_tok):
    r = random.Random(n_seq)
    width = 4 * most // P + 9
    pool = K.PagePool(max(4, 3 * n_seq * (most // P + 1)), P, n_req, width)
    model, step = Model(pool), pool.new_step(n_seq, n_tok, most)
    for turn in range(6):
        who = r.sample(range(n_req), n_seq)
        pad = r.randrange(0, n_seq // 3 + 1)
        request = who[: n_seq - pad] + [-1 - r.randrange(5) for _ in range(pad)]
        if turn % 2:
            r.shuffle(request)
        n_new, room = [], n_tok
        for x in request:
            n = min(r.choice([0, 1, most, r.randrange(most + 1)]), room)
            if x >= 0 and model.length[x] + n > width * P:
                n = 0
            n_new.append(n)
            room -= n if x >= 0 else 0
        bad = planned(pool, model, step, request, n_new)
        assert bad <= {8}
        if bad:
            with pytest.raises(K.KoreCudaError, match="free pages"):
                pool.check()
        pool.check()
        some = [x if r.random() < 0.8 else -1 for x in request]
        keep = [r.choice([0, model.length[x], model.length[x] + 5, max(0, model.length[x] - 1 - r.randrange(most)),
                          model.length[x] // 2]) if x >= 0 else -7 for x in some]
        pool.trim(ints(some), ints(keep))
        assert not model.trim(some, keep)
        model.agrees(pool)
        pool.check()


def test_trimmed_pages_come_again_in_the_same_order():
    pool = K.PagePool(40, 16, 4, 12)
    step = pool.new_step(4, 400, 100)
    request, n = ints([2, 0, 3, 1]), ints([100, 3, 0, 70])
    pool.plan(step, request, n)
    first = [x.clone() for x in (step.slots, step.page_table, pool.table, pool.free, pool.n_free)]
    pool.trim(request, torch.zeros_like(n))
    assert int(pool.n_free) == 40 and (pool.table == -1).all() and (pool.length == 0).all()
    pool.plan(step, request, n)
    assert all(torch.equal(a, b) for a, b in zip(first, (step.slots, step.page_table, pool.table, pool.free, pool.n_free)))
    pool.check()


@pytest.mark.parametrize("n_seq", [8, 1500])
@pytest.mark.parametrize("each", [2, 3])
def test_plan_leaves_out_what_does_not_fit(n_seq, each):
    P, width, r = 16, 5, random.Random(n_seq)
    pool = K.PagePool(each * n_seq, P, 2 * n_seq, width)   # about 3.4 a sequence are asked for
    model, step = Model(pool), pool.new_step(n_seq, 40 * n_seq, 80)
    request = list(range(n_seq))
    n_new = [r.randrange(20, 70) for _ in request]
    bad = planned(pool, model, step, request, n_new)
    assert 8 in bad or each == 3   # from some sequence on the pages are gone (of 1500, the step's rows as well)
    if bad:
        with pytest.raises(K.KoreCudaError, match="free pages" if bad == {8} else None):
            pool.check()
    # those that want none still go on; a request named twice, outside the pool, a negative number, one too long
    n_new = [1] * n_seq
    request[1] = request[0]
    request[2] = 2 * n_seq
    request[3] = 2 ** 31 - 1
    n_new[4], n_new[5] = -1, width * P + 1
    assert 7 in planned(pool, model, step, request, n_new)
    with pytest.raises(K.KoreCudaError, match="bounds|free pages"):   # whichever comes first
        pool.check()
    keep = [0] * n_seq
    keep[6] = -1
    request[4] = -3
    pool.trim(ints(request), ints(keep))
    assert model.trim(request, keep)
    model.agrees(pool)
    with pytest.raises(K.KoreCudaError, match="bounds"):
        pool.check()


def test_rows_beyond_the_steps_and_beyond_32_bits():
    pool = K.PagePool(64, 16, 8, 9)
    step = pool.new_step(4, 50, 40)
    pool.plan(step, ints([0, 1, 2, 3]), ints([30, 2 ** 31 - 1, 5, 2 ** 31 - 1]))
    assert step.q_start.tolist() == [0, 30] + [2 ** 31 - 1] * 3
    assert step.kv_len.tolist() == [30, 0, 0, 0] and pool.length.tolist() == [30] + [0] * 7
    assert (step.slots[30:] == -1).all() and (step.slots[:30] >= 0).all()
    with pytest.raises(K.KoreCudaError, match="bounds"):
        pool.check()


@pytest.mark.parametrize("n_free", [-1, 65, -2 ** 31])
def test_a_list_of_impossible_length_is_reported(n_free):
    pool = K.PagePool(64, 16, 8, 9)
    step = pool.new_step(1, 50, 40)
    pool.n_free.fill_(n_free)
    pool.plan(step, ints([0]), ints([30]))
    assert int(step.kv_len) == 0 and int(pool.n_free) == n_free and int(pool.length[0]) == 0
    with pytest.raises(K.KoreCudaError, match="bounds"):
        pool.check()
    pool.length[0] = 40
    pool.trim(ints([0]), ints([0]))
    assert int(pool.n_free) == n_free and int(pool.length[0]) == 40


def test_more_pages_given_back_than_there_are():
    pool = K.PagePool(4, 16, 2, 9)
    pool.length.fill_(64)   # nobody planned them
    pool.trim(ints([0, 1]), ints([0, 0]))
    assert pool.length.tolist() == [64, 64] and int(pool.n_free) == 4
    with pytest.raises(K.KoreCudaError, match="bounds"):
        pool.check()


def test_steps_of_nothing():
    pool = K.PagePool(4, 16, 2, 9)
    step = pool.new_step(0, 5, 1)
    step.slots.fill_(9), step.pos.fill_(9)
    empty = torch.zeros(0, dtype=torch.int32, device=dev())
    pool.plan(step, empty, empty)
    assert step.q_start.tolist() == [0] and (step.slots == -1).all() and (step.pos == -1).all()
    pool.trim(empty, empty)
    step = pool.new_step(2, 0, 1)
    pool.plan(step, ints([0, -1]), ints([0, 7]))
    assert step.q_start.tolist() == [0, 0, 0] and step.kv_len.tolist() == [0, 0]
    pool.check()


# ---------------------------------------------------------------- store

def normed(x, w, eps):
    x = x.double()
    return x if w is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


def near(got, y, mag, t, d, scale=None):
    """Rows against y in 64 bits; mag: |y0| + |y1| of each rotated pair, 0 where there is none."""
    tol = (d / 2 + 8) * U32 * torch.maximum(y.abs(), mag) + 4 * U32 * mag
    if scale is not None:
        y, tol = (y / scale).clamp(-448, 448), tol / scale.abs() + U32 * (y / scale).abs()
    tol = tol + u(t) * (y.abs() + tol) + TINY[t]
    bad = (got.double() - y).abs() > tol
    assert not bad.any(), ((got.double() - y).abs() / tol).max()


@pytest.mark.parametrize("t,c", [("f32", "f32"), ("f32", "bf16"), ("f32", "e4m3"), ("f16", "f16"), ("f16", "e4m3"),
                                 ("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f16")])
@pytest.mark.parametrize("G,H,d,rot,P,how,inter,wt,each", [
    (4, 28, 128, 128, 64, "fused", False, None, False), (2, 5, 64, 32, 16, "dense", True, "f32", True),
    (3, 7, 96, 96, 48, "odd", False, "bf16", True), (1, 9, 256, 64, 32, "heads_first", True, None, False),
    (2, 0, 16, 0, 16, "dense", False, "f16", False), (5, 3, 32, 32, 16, "dense", False, None, True),
    (2, 14, 64, 20, 16, "odd", True, None, False), (1, 70, 240, 10, 16, "dense", False, None, True)])
def test_store(t, c, G, H, d, rot, P, how, inter, wt, each):
    g = gen(d + P + H)
    n, n_pages = 41, 7
    C = Cache(g, c, G, d, P, [P * n_pages], alternate=(G == 4), junk=GUARD)
    k, v = (strided((rand(g, n, G, d) * 3).to(DT[t]), how) for _ in range(2))
    q = strided((rand(g, n, H, d) * 3).to(DT[t]), how) if H else None
    q_out = strided(torch.full((n, H, d), GUARD, dtype=DT[t], device=dev()), how) if H else None
    slots = torch.randperm(C.kp.shape[0] * P, device=dev(), generator=g)[:n]
    pos = torch.randint(0, 900, (n,), device=dev(), generator=g).to(torch.int32)
    slots[3], slots[n - 1], pos[5] = -1, -2 ** 40, -1   # padding
    rope = K.RopeTable(900, rot, interleaved=inter) if rot else None
    wd = DT[wt or t]
    qw, kw = ((1 + 0.5 * rand(g, *((h, d) if each else (d,)))).to(wd) for h in (max(H, 1), G))
    eps = 1e-5
    norm = K.HeadNorm(qw if H else None, kw, eps=eps)
    kp0, vp0 = C.kp.clone(), C.vp.clone()
    C.cache.store(slots, pos, k, v, rope=rope, norm=norm, q=q, q_out=q_out)
    C.cache.check()
    keep = (slots >= 0) & (pos >= 0)
    freq, amp = K.rope_frequencies(rot) if rot else ([], 1.0)
    pg, sl = slots[keep] // P, slots[keep] % P
    for x, w, pages, scale in ((k, kw, C.kp, C.ks), (v, None, C.vp, C.vs)):
        y = normed(x[keep], w, eps)
        y, mag = turned(y, pos[keep], freq, amp, inter) if w is not None else (y, torch.zeros_like(y))
        near(pages[pg, :, sl], y, mag, c, d, None if scale is None else scale.double()[:, None])
    if H:
        y, mag = turned(normed(q[keep], qw, eps), pos[keep], freq, amp, inter)
        near(q_out[keep], y, mag, t, d)
        assert (q_out[~keep] == GUARD).all()
    touched = torch.zeros(C.kp.shape[:1] + C.kp.shape[2:3], dtype=torch.bool, device=dev())
    touched[pg, sl] = True
    for pages, before in ((C.kp, kp0), (C.vp, vp0)):
        assert (pages.float() == before.float()).all(-1).all(1)[~touched].all()
    if H:   # in place, and without the norm: what append makes of the same
        q2 = strided(q.clone(), how)
        C.cache.store(slots, pos, k, v, rope=rope, norm=norm, q=q2, q_out=q2)
        assert torch.equal(q2[keep], q_out[keep]) and torch.equal(q2[~keep], q[~keep])


@pytest.mark.parametrize("t,c", [("bf16", "bf16"), ("f32", "e4m3")])
@pytest.mark.parametrize("d,rot", [(128, 128), (96, 96)])
def test_store_without_norms_has_appends_bits(t, c, d, rot):
    g = gen(4)
    ns, kvs = [3, 40, 1], [3, 77, 300]
    A, B = (Cache(gen(5), c, 2, d, 16, kvs, junk=GUARD) for _ in range(2))
    n = sum(ns)
    k, v, q = (rand(g, n, h, d).to(DT[t]) for h in (2, 2, 6))
    rope = K.RopeTable(300, rot)
    qa, qb = torch.zeros_like(q), torch.zeros_like(q)
    A.cache.append(K.PagedBatch(starts(ns), ints(kvs), A.table, 40), k, v, rope=rope, q=q, q_out=qa)
    pos = torch.cat([torch.arange(b - a, b, device=dev()) for a, b in zip(ns, kvs)])
    seq = torch.repeat_interleave(torch.arange(3, device=dev()), torch.tensor(ns, device=dev()))
    slots = B.table[seq, pos // 16].long() * 16 + pos % 16
    B.cache.store(slots, pos.int(), k, v, rope=rope, q=q, q_out=qb)
    assert torch.equal(qa, qb)
    assert torch.equal(A.kp.view(torch.uint8), B.kp.view(torch.uint8))
    assert torch.equal(A.vp.view(torch.uint8), B.vp.view(torch.uint8))


@pytest.mark.parametrize("d", [64, 80])
def test_norms_of_heads_of_any_size(d):
    """Squares that pass 32 bits, vanish in them, zeros, and values that are none."""
    g = gen(6)
    x = rand(g, 1, 8, d)
    x[0, 1] *= 2.0 ** 100
    x[0, 2] *= 2.0 ** -100
    x[0, 3] = 0
    x[0, 4, 5] = math.inf
    x[0, 5, 5] = math.nan
    x[0, 6, 5] = 2.0 ** 90
    x[0, 7] = 2.0 ** 127 * x[0, 7].sign()
    C = Cache(g, "f32", 1, d, 16, [16])
    w = 1 + rand(g, d) * 0.1
    out = torch.zeros_like(x)
    one = rand(g, 1, 1, d)
    C.cache.store(torch.zeros(1, dtype=torch.int64, device=dev()), None, one, one, norm=K.HeadNorm(w, eps=1e-6), q=x, q_out=out)
    y = normed(x, w, 1e-6)
    for h in (0, 1, 2, 3, 6, 7):
        near(out[:, h], y[:, h], torch.zeros_like(y[:, h]), "f32", d)
    assert out[0, 5].isnan().all()
    rest = torch.arange(d, device=dev()) != 5
    assert out[0, 4, 5].isnan() and (out[0, 4, rest] == 0).all()
    assert torch.equal(C.kp[0, 0, 0], one[0, 0])   # no norm for the keys


def test_store_into_a_head_of_scale_zero():
    C = Cache(gen(1), "e4m3", 2, 64, 16, [16])
    C.ks.copy_(torch.tensor([0.0, 1.0])), C.vs.copy_(torch.tensor([-0.5, 0.0]))
    x = rand(gen(2), 1, 2, 64)
    C.cache.store(torch.tensor([5], device=dev()), None, x, x)
    assert (C.kp[0, 0, 5].float() == 0).all() and (C.vp[0, 1, 5].float() == 0).all()
    near(C.kp[0, 1, 5], x[0, 1].double(), torch.zeros(64, device=dev()), "e4m3", 64)
    near(C.vp[0, 0, 5], x[0, 0].double(), torch.zeros(64, device=dev()), "e4m3", 64, torch.tensor(-0.5, device=dev()))


def test_store_reports_bad_device_data():
    for bad, word in (("slot", "page id"), ("pos", "rotation table")):
        C = Cache(gen(1), "bf16", 2, 64, 16, [20], junk=GUARD)
        n_slots = C.kp.shape[0] * 16
        slots = torch.tensor([0, n_slots if bad == "slot" else 1, n_slots - 1], device=dev())
        k = torch.ones(3, 2, 64, device=dev(), dtype=torch.bfloat16)
        C.cache.store(slots, ints([0, 16 if bad == "pos" else 1, 15]), k, k, rope=K.RopeTable(16, 64))
        with pytest.raises(K.KoreCudaError, match=word):
            C.cache.check()
        written = (C.vp[:, 0, :, 0] == 1).flatten()
        assert written.nonzero().flatten().tolist() == [0, n_slots - 1]
        C.cache.check()


# ---------------------------------------------------------------- trees

def tree(r, n, kind):
    """Parents of a chunk of n tokens."""
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1 if r.random() < 0.5 or not i else r.randrange(i) for i in range(n)]
    return [-1] + [r.randrange(i) for i in range(1, n)]


def sees(parents):
    """[n][n]: token i sees token j."""
    n = len(parents)
    m = torch.zeros(n, n, dtype=torch.bool)
    for i, x in enumerate(parents):
        if x >= 0:
            m[i] = m[x]
        m[i, i] = True
    return m


def words_of(m, words):
    """Rows of truth values as 32-bit words."""
    bits = torch.nn.functional.pad(m.long(), (0, 32 * words - m.shape[1])).unflatten(1, (words, 32))
    w = (bits << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


@pytest.mark.parametrize("kind", ["chain", "star", "random", "roots"])
@pytest.mark.parametrize("ns,most", [([1], 1), ([8, 0, 3], 8), ([33, 64, 1, 65, 96], 100), ([1024, 5], 1024), ([32], 32)])
def test_masks(kind, ns, most):
    r = random.Random(sum(ns))
    par = [tree(r, n, kind) if n else [] for n in ns]
    kvs = [n + r.randrange(500) for n in ns]
    n_tok = sum(ns) + 3
    t = K.TokenTree(n_tok, most)
    t.mask.fill_(77), t.pos.fill_(77)
    batch = K.PagedBatch(starts(ns), ints(kvs), ints([[0]] * len(ns)), most)
    t.build(batch, ints([x for p in par for x in p] + [5, -9, 0]))
    t.check()
    words, at = t.mask.shape[1], 0
    for n, kv, p in zip(ns, kvs, par):
        m = sees(p) if n else torch.zeros(0, 0, dtype=torch.bool)
        assert torch.equal(t.mask[at:at + n].cpu(), words_of(m, words))
        assert t.pos[at:at + n].tolist() == [kv - n + int(x) - 1 for x in m.sum(1)]
        at += n
    assert (t.mask[at:] == 77).all() and (t.pos[at:] == 77).all()


def test_masks_leave_out_what_is_no_tree():
    t = K.TokenTree(9, 6)
    t.mask.fill_(77), t.pos.fill_(77)
    # a parent behind the token, its child; a token that is its own parent; a chunk longer than its length; one too long
    batch = K.PagedBatch(ints([0, 6, 9]), ints([10, 2]), ints([[0], [0]]), 6)
    t.build(batch, ints([-1, 0, 3, 2, 4, -2, -1, 0, 1]))
    assert t.pos.tolist() == [4, 5, -1, -1, -1, -1, 77, 77, 77]
    assert t.mask[:, 0].tolist() == [1, 3, 0, 0, 0, 0, 77, 77, 77]
    with pytest.raises(K.KoreCudaError, match="bounds"):
        t.check()
    long = K.TokenTree(40, 32)
    long.build(K.PagedBatch(ints([0, 40]), ints([40]), ints([[0]]), 40), ints([-1] * 40))
    assert (long.mask == 0).all()
    with pytest.raises(K.KoreCudaError, match="bounds"):
        long.check()


def check_tree(C, q, out, ns, seen, scale=None, lse=None):
    """Every row of out (and lse) against the formula in 64 bits; seen: [n][n] of each sequence."""
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
            m = torch.cat([torch.ones(n, kv - n, dtype=torch.bool), seen[s]], 1).to(dev())
            k, v = (torch.where(m.any(0)[:, None, None], x, 0.0) for x in (k, v))   # what no token sees may be anything
            x = q[at:at + n].double().unflatten(1, (C.G, rep))
            sc = torch.einsum("ngrd,tgd->ngrt", x, k) * scale
            mag = torch.einsum("ngrd,tgd->ngrt", x.abs(), k.abs()) * abs(scale)
            sc = sc.masked_fill(~m[:, None, None], -math.inf)
            some = m.any(-1)
            p = torch.softmax(sc, -1).nan_to_num(0.0)
            want = torch.einsum("ngrt,tgd->ngrd", p, v)
            pv = torch.einsum("ngrt,tgd->ngrd", p, v.abs())
            e = (2 * d * U32 * mag + 4 * U32 * sc.abs().nan_to_num(0, 0, 0)).masked_fill(~m[:, None, None], 0)
            e = e.amax(-1, keepdim=True)
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


def attend(g, C, H, ns, seen, tq, kernel, how="dense", pad=2, most=None, garbage=0, **kw):
    n = sum(ns) + pad
    q = strided(rand(g, n, H, C.d).to(DT[tq]), how)
    out = strided(torch.full((n, H, C.d), GUARD, dtype=DT[tq], device=dev()), how)
    lse = torch.full((n, H), GUARD, device=dev())
    t = K.TokenTree(n, most or max(ns + [1]))
    words = t.mask.shape[1]
    rows = [words_of(m, words) for m, x in zip(seen, ns) if x]
    t.mask[: sum(ns)] = torch.cat(rows).to(dev())
    if garbage:   # bits behind the chunks
        for x, a in zip(ns, starts(ns).tolist()):
            full = words_of(torch.arange(32 * words)[None] >= x, words).to(dev())
            t.mask[a:a + x] |= full
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    C.cache.attend(batch, q, out, lse=lse, tree=t, **kw)
    C.cache.check()
    check_tree(C, q, out, ns, seen, lse=lse, **kw)
    assert (out[sum(ns):] == GUARD).all() and (lse[sum(ns):] == GUARD).all()
    return q, out, batch, t


TREES = {   # (tokens, cached positions with them)
    "one": [(1, 1)],
    "alone": [(1, 1), (7, 7), (40, 40)],
    "edges": [(3, 15), (3, 16), (3, 17), (5, 130), (64, 128), (65, 193), (33, 257)],
    "ragged": [(8, 700), (0, 30), (16, 16), (1, 2049), (25, 64), (13, 1000)],
    "wide": [(96, 500), (128, 128), (200, 1300)],
    "long": [(12, 9000)],
}
KERNELS = pytest.mark.parametrize("kernel", list(HINTS))


@pytest.mark.parametrize("tq,tc", KINDS)
@pytest.mark.parametrize("H,G,d,P", [(28, 4, 128, 64), (14, 2, 64, 16), (8, 8, 128, 48), (40, 2, 64, 256), (3, 1, 128, 16)])
@pytest.mark.parametrize("which", list(TREES))
@KERNELS
def test_tree_attention(kernel, tq, tc, H, G, d, P, which):
    g, r = gen(H + P), random.Random(H + P)
    ns, kvs = map(list, zip(*TREES[which]))
    C = Cache(g, tc, G, d, P, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    attend(g, C, H, ns, [sees(tree(r, n, "random")) if n else None for n in ns], tq, kernel)


@pytest.mark.parametrize("tq,tc", KINDS)
@KERNELS
def test_tree_attention_of_any_mask(kernel, tq, tc):
    """Rows that see nothing (no context, no token), tokens that see later ones, bits behind the chunk, another scale."""
    g = gen(3)
    ns, kvs = [5, 40, 70, 3], [5, 40, 300, 1000]
    C = Cache(g, tc, 2, 64, 16, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    seen = [torch.rand(n, n, generator=torch.Generator().manual_seed(n)) < 0.3 for n in ns]
    seen[0][2] = False
    seen[1][7] = False
    seen[1][39] = False
    seen[2][0] = False
    for kw in (dict(), dict(scale=-0.3), dict(garbage=1), dict(most=1000, garbage=1)):
        attend(g, C, 14, ns, seen, tq, kernel, **kw)


@pytest.mark.parametrize("tq,tc", KINDS)
@KERNELS
def test_what_no_token_sees_may_be_anything(kernel, tq, tc):
    g, r = gen(4), random.Random(4)
    for n, kv in ((6, 6), (40, 41), (90, 700)):
        C = Cache(g, tc, 2, 128, 32, [kv, kv])
        C.fill(g, 0), C.fill(g, 1)
        seen = sees(tree(r, n, "roots"))
        blind = [j for j in range(1, n) if r.random() < 0.3] + [n - 1]
        seen[:, blind] = False
        for s in range(2):
            pg, sl = C.places(s, torch.tensor([kv - n + j for j in blind], device=dev()))
            C.kp[pg, :, sl] = float("nan")
            C.vp[pg, :, sl] = float("nan") if tc == "e4m3" else float("inf")
        attend(g, C, 14, [n, n], [seen, seen], tq, kernel)


@pytest.mark.parametrize("how", ["fused", "heads_first", "odd"])
@KERNELS
def test_tree_attention_of_strided_rows(kernel, how):
    g, r = gen(5), random.Random(5)
    ns, kvs = [9, 30], [200, 77]
    C = Cache(g, "bf16", 2, 128, 48, kvs, alternate=True)
    for s in range(2):
        C.fill(g, s)
    attend(g, C, 14, ns, [sees(tree(r, n, "random")) for n in ns], "bf16", kernel, how=how)


@pytest.mark.parametrize("H,G,d", [(128, 1, 64), (16, 16, 128), (12, 12, 64)])
@KERNELS
def test_tree_attention_of_wide_and_of_single_groups(kernel, H, G, d):
    g, r = gen(6), random.Random(6)
    ns, kvs = [20, 2, 35], [300, 2, 35]
    C = Cache(g, "f16", G, d, 16, kvs)
    for s in range(3):
        C.fill(g, s)
    attend(g, C, H, ns, [sees(tree(r, n, "random")) for n in ns], "f16", kernel)


@KERNELS
def test_a_chains_attention_is_the_chunks(kernel):
    """A chain is a causal chunk."""
    g = gen(7)
    C = Cache(g, "bf16", 4, 128, 64, [1000, 333])
    C.fill(g, 0), C.fill(g, 1)
    ns = [17, 9]
    q, out, batch, t = attend(g, C, 28, ns, [sees(tree(None, n, "chain")) for n in ns], "bf16", kernel, pad=0)
    same = C.cache.attend(batch, q)
    assert (same.float() - out.float()).abs().max() <= 2.0 ** -6   # each within one rounding (2^-8 of values below 2) of the same


@KERNELS
def test_tree_attention_of_many_sequences(kernel):
    g, r = gen(8), random.Random(8)
    ns = [r.choice([0, 1, 5, 13]) for _ in range(300)]
    kvs = [n + r.choice([0, 1, 30, 200]) for n in ns]
    C = Cache(g, "bf16", 2, 64, 16, kvs)
    for s in range(300):
        C.fill(g, s)
    attend(g, C, 4, ns, [sees(tree(r, n, "random")) if n else None for n in ns], "bf16", kernel)


@pytest.mark.parametrize("n", [6, 50])
@pytest.mark.parametrize("bad,word", [("page", "page id"), ("rows", "bounds"), ("long", "bounds"), ("short", "bounds"),
                                      ("words", "bounds")])
@KERNELS
def test_tree_attention_reports_bad_device_data(kernel, n, bad, word):
    g, r = gen(9), random.Random(9)
    C = Cache(g, "bf16", 2, 64, 16, [100, 100])
    C.fill(g, 0), C.fill(g, 1)
    seen = sees(tree(r, n, "random"))
    q = rand(g, 2 * n, 4, 64).to(torch.bfloat16)
    out = torch.full_like(q, GUARD)
    t = K.TokenTree(2 * n, n if bad != "words" else 1)
    if bad == "words":
        if n <= 32:
            return
    else:
        t.mask.copy_(words_of(torch.cat([seen, seen]), t.mask.shape[1]))
    table, q_start, kv = C.table.clone(), [0, n, 2 * n], [100, 100]
    if bad == "page":
        table[1, 1] = C.kp.shape[0] + 3
    elif bad == "rows":
        q_start[2] = 2 * n + 7
    elif bad == "long":
        kv[1] = table.shape[1] * 16 + 1
    elif bad == "short":
        kv[1] = n - 1
    C.cache.attend(K.PagedBatch(ints(q_start), ints(kv), table, **HINTS[kernel]), q, out, tree=t)
    with pytest.raises(K.KoreCudaError, match=word):
        C.cache.check()
    if bad != "words":
        check_tree(C, q[:n], out[:n], [n], [seen])
    if word == "bounds":
        assert (out[n:] == GUARD).all()
    C.cache.check()


# ---------------------------------------------------------------- acceptance and moves

def accepted(par, token, choice, most):
    path = [0]
    while len(path) < most:
        hit = [i for i in range(len(par)) if par[i] == path[-1] and token[i] == choice[path[-1]]]
        if not hit:
            break
        path.append(hit[0])
    return path


@pytest.mark.parametrize("ns,most", [([1], 1), ([8, 0, 3, 1], 4), ([33, 64, 1, 65, 96, 2], 9), ([1024, 40], 1024)])
def test_accept(ns, most):
    r = random.Random(sum(ns))
    for turn in range(4):
        par = [tree(r, n, r.choice(["chain", "random", "star", "roots"])) if n else [] for n in ns]
        token = [[r.randrange(3) for _ in p] for p in par]   # few tokens: siblings alike, long branches
        choice = [[r.randrange(3) for _ in p] for p in par]
        kvs = [n + r.randrange(300) for n in ns]
        flat = lambda x: ints([z for y in x for z in y] + [0, 0])   # noqa: E731
        p = K.AcceptedPath(len(ns), most)
        for x in (p.path, p.count, p.next_token, p.kept):
            x.fill_(77)
        p.accept(K.PagedBatch(starts(ns), ints(kvs), ints([[0]] * len(ns)), max(ns)), flat(par), flat(token), flat(choice))
        p.check()
        for s, n in enumerate(ns):
            want = accepted(par[s], token[s], choice[s], most) if n else []
            assert p.path[s].tolist() == want + [-1] * (most - len(want))
            assert int(p.count[s]) == len(want) and int(p.kept[s]) == kvs[s] - n + len(want)
            assert int(p.next_token[s]) == (choice[s][want[-1]] if n else -1)


def test_accept_leaves_out_what_does_not_fit():
    p = K.AcceptedPath(3, 4)
    p.accept(K.PagedBatch(ints([0, 2, 4, 99]), ints([10, 1, 200]), ints([[0]] * 3), 4), ints([-1, 0, -1, 0]),
             ints([1, 2, 3, 4]), ints([2, 9, 4, 9]))
    assert p.count.tolist() == [2, 0, 0] and p.kept.tolist() == [10, -1, -1] and p.next_token.tolist() == [9, -1, -1]
    assert p.path.tolist() == [[0, 1, -1, -1]] + [[-1] * 4] * 2
    with pytest.raises(K.KoreCudaError, match="bounds"):
        p.check()


@pytest.mark.parametrize("t,G,d,P,L", [("bf16", 4, 128, 64, 28), ("f16", 2, 64, 16, 3), ("e4m3", 3, 16, 48, 1),
                                       ("f32", 2, 256, 16, 5), ("bf16", 1, 80, 32, 130)])
def test_commit(t, G, d, P, L):
    r, g = random.Random(L), gen(L)
    ns = [1, 12, 0, 40, 3, 64, 8]
    kvs = [n + r.randrange(100) for n in ns]
    C = Cache(g, "bf16", 1, 16, P, kvs)   # its page table
    n_pages = C.kp.shape[0]
    pool = torch.randint(0, 120, (L, 2, n_pages, G, P, d * DT[t].itemsize), device=dev(), generator=g, dtype=torch.uint8)
    pages = pool.view(DT[t])
    layers = K.PagedLayers([K.PagedCache(x[0], x[1]) for x in pages])
    p = K.AcceptedPath(len(ns), 20)
    paths = [[0], [0, 1, 2, 5, 6, 7, 11], [], [0] + sorted(r.sample(range(1, 40), 19)), [0, 2], [0] + sorted(r.sample(range(1, 64), 12)),
             [0, 1, 2, 3]]
    for s, x in enumerate(paths):
        p.path[s, : len(x)] = ints(x)
    p.count.copy_(ints([len(x) for x in paths]))
    want = pool.clone()
    for s, x in enumerate(paths):
        for j, i in enumerate(x):
            (pa, sa), (pb, sb) = (C.places(s, torch.tensor(kvs[s] - ns[s] + y, device=dev())) for y in (i, j))
            want[:, :, pb, :, sb] = pool[:, :, pa, :, sa]
    layers.commit(K.PagedBatch(starts(ns), ints(kvs), C.table, 64), p)
    layers.check()
    assert torch.equal(pool, want)


@pytest.mark.parametrize("bad,word", [("down", "bounds"), ("twice", "bounds"), ("outside", "bounds"), ("low", "bounds"),
                                      ("negative", "bounds"), ("count", "bounds"), ("length", "bounds"), ("page", "page id")])
def test_commit_leaves_out_what_does_not_fit(bad, word):
    g = gen(2)
    C = Cache(g, "bf16", 2, 64, 16, [40, 40])
    C.fill(g, 0), C.fill(g, 1)
    path, count, kv, table = [0, 2, 5, 7], 4, 40, C.table.clone()
    if bad == "down":
        path = [0, 5, 2, 7]
    elif bad == "twice":
        path = [0, 2, 2, 7]
    elif bad == "outside":
        path = [0, 2, 5, 8]
    elif bad == "low":
        path = [1, 2, 3, 2]
    elif bad == "negative":
        path = [-1, 2, 5, 7]
    elif bad == "count":
        count = 5
    elif bad == "length":
        kv = 7
    elif bad == "page":
        table[1, 2] = -1
    p = K.AcceptedPath(2, 4)
    p.path.copy_(ints([[0, 2, 5, 7], path])), p.count.copy_(ints([4, count]))
    k0, v0 = C.kp.clone(), C.vp.clone()
    K1 = K.PagedLayers([C.cache])
    K1.commit(K.PagedBatch(ints([0, 8, 16]), ints([40, kv]), table, 8), p)
    with pytest.raises(K.KoreCudaError, match=word):
        K1.check()
    same = torch.ones(40, dtype=torch.bool, device=dev())
    pg, sl = C.places(1, torch.arange(40, device=dev()))
    assert torch.equal(C.kp[pg, :, sl].nan_to_num(9), k0[pg, :, sl].nan_to_num(9))
    pg, sl = C.places(0, torch.arange(40, device=dev()))
    src = torch.arange(40, device=dev())
    src[32:36] = 32 + torch.tensor([0, 2, 5, 7], device=dev())
    same = (C.vp[pg, :, sl] == v0[pg, :, sl][src]).all()
    assert same


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("tq,tc,H,G,d,P", [("bf16", "bf16", 28, 4, 128, 64), ("f16", "e4m3", 14, 2, 64, 16)])
@KERNELS
def test_steps_with_drafts_leave_what_single_tokens_would(kernel, tq, tc, H, G, d, P):
    """Prompts, then steps of drafted trees whose accepted branches are of any length: the caches hold the accepted
    tokens' rows and nothing between them, the attention sees just them, and the pool's pages are the ones in use."""
    g, r = gen(11), random.Random(11)
    n_req, layers, width = 5, 2, 40
    pool = K.PagePool(60, P, n_req, width)
    pages = [[torch.full((60, G, P, d), float("nan"), device=dev()).to(DT[tc]) for _ in range(2)] for _ in range(layers)]
    scale = [0.01 * (1 + torch.rand(G, device=dev(), generator=g)) for _ in range(2)] if tc == "e4m3" else [None, None]
    caches = [K.PagedCache(*x, k_scale=scale[0], v_scale=scale[1]) for x in pages]
    all_layers = K.PagedLayers(caches)
    rope = K.RopeTable(2000, d)
    qw, kw = (1 + 0.2 * rand(g, d) for _ in range(2))
    norm = K.HeadNorm(qw, kw)
    held = [[[] for _ in range(n_req)] for _ in range(layers)]   # accepted (k row, v row, position): as stored

    def rows(cache, slots):
        return [(x[s // P, :, s % P].clone(), y[s // P, :, s % P].clone()) for x, y, s in
                ((cache.k, cache.v, int(s)) for s in slots)]

    # prompts
    who, n_new = [3, 0, 4, 1], [37, 150, 1, 64]
    step = pool.new_step(4, sum(n_new) + 2, max(n_new))
    pool.plan(step, ints(who), ints(n_new))
    for l, cache in enumerate(caches):
        k, v = (rand(g, step.slots.shape[0], G, d).to(DT[tq]) for _ in range(2))
        cache.store(step.slots, step.pos, k, v, rope=rope, norm=norm)
        at = 0
        for w, n in zip(who, n_new):
            held[l][w] += rows(cache, step.slots[at:at + n].tolist())
            at += n
    for turn in range(5):
        ns = [r.randrange(1, 20) for _ in who]
        par = [tree(r, n, "random") for n in ns]
        n_tok = sum(ns) + 3
        step, t, path = pool.new_step(len(who), n_tok, 20), K.TokenTree(n_tok, 20), K.AcceptedPath(len(who), 6)
        batch_kw = HINTS[kernel]
        step.view.max_q, step.view.max_kv = batch_kw["max_q"], batch_kw.get("max_kv", 0)
        parent = ints([x for p in par for x in p] + [0] * 3)
        pool.plan(step, ints(who), ints(ns))
        t.build(step, parent)
        first = step.slots.tolist()
        for l, cache in enumerate(caches):
            k, v = (rand(g, n_tok, G, d).to(DT[tq]) for _ in range(2))
            q = rand(g, n_tok, H, d).to(DT[tq])
            qr, out = torch.zeros_like(q), torch.full_like(q, GUARD)
            cache.store(step.slots, t.pos, k, v, rope=rope, norm=norm, q=q, q_out=qr)
            cache.attend(step, qr, out, tree=t)
            # the cache that the attention should have seen: the accepted rows, then the drafts
            kvs = [len(held[l][w]) + n for w, n in zip(who, ns)]
            assert step.kv_len.tolist() == kvs
            C = Cache(g, tc, G, d, P, kvs)
            C.ks, C.vs = scale
            at = 0
            for s, (w, n) in enumerate(zip(who, ns)):
                pg, sl = C.places(s, torch.arange(kvs[s], device=dev()))
                mine = held[l][w] + rows(cache, first[at:at + n])
                C.kp[pg, :, sl] = torch.stack([a for a, _ in mine])
                C.vp[pg, :, sl] = torch.stack([b for _, b in mine])
                at += n
            check_tree(C, qr, out, ns, [sees(p) for p in par])
            assert (out[sum(ns):] == GUARD).all()
        token = [[r.randrange(2) for _ in p] for p in par]
        choice = [[r.randrange(2) for _ in p] for p in par]
        flat = lambda x: ints([z for y in x for z in y] + [0] * 3)   # noqa: E731
        path.accept(step, parent, flat(token), flat(choice))
        drafts = [rows(c, first[: sum(ns)]) for c in caches]
        all_layers.commit(step, path)
        pool.trim(ints(who), path.kept)
        at = 0
        for s, (w, n) in enumerate(zip(who, ns)):
            took = accepted(par[s], token[s], choice[s], 6)
            for l in range(layers):
                held[l][w] += [drafts[l][at + i] for i in took]
            at += n
        assert path.kept.tolist() == [len(held[0][w]) for w in who]
        used = sum(-(-len(x) // P) for x in held[0])
        assert pool.length.tolist() == [len(x) for x in held[0]] and int(pool.n_free) == 60 - used
        table = pool.table.tolist()
        for l, cache in enumerate(caches):
            for w in who:
                for p, (a, b) in enumerate(held[l][w]):
                    if p < len(held[l][w]) - 30:
                        continue
                    page = table[w][p // P]
                    assert torch.equal(cache.k[page, :, p % P].float(), a.float())
                    assert torch.equal(cache.v[page, :, p % P].float(), b.float())
        for x in (pool, t, path, all_layers, *caches):
            x.check()
        if turn == 2:   # one request ends and another begins
            pool.trim(ints([0]), ints([0]))
            for l in range(layers):
                held[l][0] = []
            who = [3, 2, 4, 1]


def test_captured_step_with_drafts():
    """A whole step captured once and replayed: it follows requests, counts, trees and choices as they are at its replay."""
    g, r = gen(12), random.Random(12)
    G, H, d, P, n_seq, n_tok = 2, 14, 64, 16, 3, 40
    pool = K.PagePool(200, P, 6, 30)
    kp, vp = (torch.zeros(200, G, P, d, device=dev(), dtype=torch.bfloat16) for _ in range(2))
    cache = K.PagedCache(kp, vp)
    layers, rope, norm = K.PagedLayers([cache]), K.RopeTable(500, d), K.HeadNorm(1 + 0.1 * rand(g, d), 1 + 0.1 * rand(g, d))
    step, t, path = pool.new_step(n_seq, n_tok, 16), K.TokenTree(n_tok, 16), K.AcceptedPath(n_seq, 5)
    request, n_new = ints([0, 1, 2]), ints([1, 1, 1])
    parent, token, choice = (torch.zeros(n_tok, dtype=torch.int32, device=dev()) for _ in range(3))
    q, k, v = (rand(g, n_tok, h, d).to(torch.bfloat16) for h in (H, G, G))
    qr, out = torch.zeros_like(q), torch.zeros_like(q)

    def run():
        pool.plan(step, request, n_new)
        t.build(step, parent)
        cache.store(step.slots, t.pos, k, v, rope=rope, norm=norm, q=q, q_out=qr)
        cache.attend(step, qr, out, tree=t)
        path.accept(step, parent, token, choice)
        layers.commit(step, path)
        pool.trim(request, path.kept)

    parent.copy_(ints([-1] * n_tok))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            run()
    torch.cuda.synchronize()
    lengths = pool.length.tolist()
    assert lengths == [1, 1, 1, 0, 0, 0]
    for turn in range(6):
        who = r.sample(range(6), n_seq - (turn == 3)) + [-1] * (turn == 3)
        ns = [r.randrange(1, 14) if w >= 0 else 0 for w in who]
        par = [tree(r, n, "random") if n else [] for n in ns]
        tk = [[r.randrange(2) for _ in p] for p in par]
        ch = [[r.randrange(2) for _ in p] for p in par]
        fill = lambda x: ints([z for y in x for z in y] + [0] * (n_tok - sum(ns)))   # noqa: E731
        for dst, src in ((request, ints(who)), (n_new, ints(ns)), (parent, fill(par)), (token, fill(tk)), (choice, fill(ch))):
            dst.copy_(src)
        for x, h in ((q, H), (k, G), (v, G)):
            x.copy_(rand(g, n_tok, h, d))
        before = pool.table.clone()
        gr.replay()
        torch.cuda.synchronize()
        C = Cache(g, "bf16", G, d, P, [1] * n_seq)
        for w, n, p, a, b in zip(who, ns, par, tk, ch):
            if w >= 0:
                lengths[w] += len(accepted(p, a, b, 5))
        assert pool.length.tolist() == lengths
        assert int(pool.n_free) == 200 - sum(-(-x // P) for x in lengths)
        # the drafts' rows, before the move, are those of the last store: the attention of a sequence's root alone
        C.kvs, C.kp, C.vp, C.table = [x - n + 1 for x, n in zip(step.kv_len.tolist(), ns)], kp, vp, step.page_table
        roots = [a for a, n in zip(step.q_start.tolist(), ns) if n]
        live = [s for s, n in enumerate(ns) if n]
        C.kvs, C.table = [C.kvs[s] for s in live], C.table[live]
        check_tree(C, qr[roots], out[roots], [1] * len(live), [torch.ones(1, 1, dtype=torch.bool)] * len(live))
        del before
    for x in (pool, t, path, layers, cache):
        x.check()


@KERNELS
def test_tree_attention_on_two_streams(kernel):
    g, r = gen(13), random.Random(13)
    C = Cache(g, "bf16", 2, 64, 16, [3000, 2000])
    C.fill(g, 0), C.fill(g, 1)
    ns = [16, 12]
    q, out, batch, t = attend(g, C, 14, ns, [sees(tree(r, n, "random")) for n in ns], "bf16", kernel, pad=0)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(out) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                C.cache.attend(batch, q, o, tree=t)
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)   # the same call, the same bits


@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("n_seq", [32, 33, 63, 64, 65, 97])
@KERNELS
def test_batches_around_the_sequences_of_a_warp(kernel, n_seq, trees):
    """Up to 32 sequences a lane of each warp has one, up to 64 two, behind that the sums are shared: ragged batches,
    some of whose sequences have no tokens (the 32nd and 33rd too), over shares that begin in either half."""
    g, r = gen(n_seq), random.Random(n_seq)
    for empty in (False, True):
        ns = [0 if r.random() < 0.2 or (empty and 28 <= s < 40) else r.randrange(1, 9) for s in range(n_seq)]
        kvs = [n + r.choice([0, 1, 40, 300, 900]) for n in ns]
        C = Cache(g, "bf16", 2, 64, 16, kvs)
        for s in range(n_seq):
            C.fill(g, s)
        if trees:
            attend(g, C, 14, ns, [sees(tree(r, n, "random")) if n else None for n in ns], "bf16", kernel)
        else:
            attend_chunks(g, C, 14, ns, "bf16", kernel)


@pytest.mark.parametrize("tq,tc", KINDS)
@pytest.mark.parametrize("n,past", [(8, 1000), (24, 300), (24, 6000)])
def test_trees_of_many_sequences_with_their_own_bounds(tq, tc, n, past):
    """The batch's real bounds, by which the tile kernel takes it: few tiles a CTA, or many."""
    g, r = gen(n), random.Random(n)
    ns, kvs = [n] * 16, [n + past - 7 * s for s in range(16)]
    C = Cache(g, tc, 4, 128, 64, kvs)
    for s in range(16):
        C.fill(g, s)
    HINTS["own"] = dict(max_q=n, max_kv=n + past)
    try:
        attend(g, C, 28, ns, [sees(tree(r, n, "random")) for n in ns], tq, "own")
    finally:
        del HINTS["own"]
