"""A step with drafted tokens where it can go wrong: waits of the tree attention that run out (as in
tests/test_paged_failures_gpu.py, without a GPU fault), offsets and slots beyond 32 bits, sequences that a plan left out,
another device than the current one, graphs captured on one stream and replayed on two."""
import random

import pytest

import kore_b200 as K
from kore_b200.paged import set_wait_limit
from tests.test_drafts_gpu import attend, check_tree, sees, tree, words_of
from tests.test_paged_gpu import DT, GUARD, HINTS, Cache, dev, gen, ints, rand, starts

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
KERNELS = pytest.mark.parametrize("kernel", list(HINTS))
BATCHES = {"short": [(3, 90)], "long": [(20, 9000), (40, 700), (1, 3000), (33, 5000)]}


def ready(tc, which, H=14, d=128):
    g, r = gen(1), random.Random(1)
    ns, kvs = map(list, zip(*BATCHES[which]))
    C = Cache(g, tc, 2, d, 64, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    seen = [sees(tree(r, n, "random")) for n in ns]
    t = K.TokenTree(sum(ns), max(ns))
    t.mask.copy_(torch.cat([words_of(m, t.mask.shape[1]) for m in seen]))
    return C, ns, rand(g, sum(ns), H, d).to(torch.bfloat16), seen, t


@KERNELS
@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", list(BATCHES))
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(kernel, tc, d, which):
    C, ns, q, seen, t = ready(tc, which, d=d)
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    ws = C.cache.new_workspace()
    set_wait_limit(1e-9)
    try:
        for _ in range(20):   # (a copy may have landed before the kernel looks)
            C.cache.attend(batch, q, torch.zeros_like(q), tree=t, workspace=ws)
            try:
                C.cache.check()
            except K.KoreCudaError as e:
                assert e.code == -6 and "in time" in str(e)
                break
        else:
            pytest.fail("no wait ran out with a limit of 1 ns")
    finally:
        set_wait_limit(0)
    ws[:K.paged.WORKSPACE_ZEROED].zero_()
    for _ in range(3):
        out = C.cache.attend(batch, q, tree=t, workspace=ws)
        C.cache.check()
        check_tree(C, q, out, ns, seen)
        assert (ws[:K.paged.WORKSPACE_ZEROED] == 0).all()   # as every call leaves it


@KERNELS
@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
def test_one_workspace_for_chunks_and_trees_in_turn(kernel, tc):
    """Both divide their work and join its parts in the same memory."""
    C, ns, q, seen, t = ready(tc, "long")
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    ws = C.cache.new_workspace()
    first = C.cache.attend(batch, q, workspace=ws)
    for _ in range(4):
        out = C.cache.attend(batch, q, tree=t, workspace=ws)
        check_tree(C, q, out, ns, seen)
        assert torch.equal(C.cache.attend(batch, q, workspace=ws), first)
    C.cache.check()
    assert (ws[:K.paged.WORKSPACE_ZEROED] == 0).all()


def test_offsets_beyond_32_bits():
    """Pages behind the first 2^31 values of a pool: stored to, moved in and attended over."""
    g, r = gen(2), random.Random(2)
    G, d, P = 2, 128, 64
    per = G * P * d
    n_pages = 2 ** 31 // per + 40
    kp, vp = (torch.empty(n_pages, G, P, d, device=dev(), dtype=torch.bfloat16) for _ in range(2))
    used = torch.arange(n_pages - 20, n_pages, device=dev()).int()
    n, kv = 24, 1200
    small = Cache(g, "bf16", G, d, P, [kv])
    small.fill(g, 0)
    table = used[: small.table.shape[1]].reshape(1, -1).contiguous()
    pg = small.table[0][: -(-kv // P)].long()
    kp[table[0, : len(pg)].long()], vp[table[0, : len(pg)].long()] = small.kp[pg], small.vp[pg]
    cache = K.PagedCache(kp, vp)
    k, v = (rand(g, n, G, d).to(torch.bfloat16) for _ in range(2))
    pos = torch.arange(kv - n, kv, device=dev())
    cache.store(table[0, pos // P].long() * P + pos % P, None, k, v)
    small.cache.store(small.table[0, pos // P].long() * P + pos % P, None, k, v)
    seen = sees(tree(r, n, "random"))
    t = K.TokenTree(n, n)
    t.mask.copy_(words_of(seen, 1))
    q = rand(g, n, 14, d).to(torch.bfloat16)
    for hints in HINTS.values():
        out = cache.attend(K.PagedBatch(ints([0, n]), ints([kv]), table, **hints), q, tree=t)
        check_tree(small, q, out, [n], [seen])
    p = K.AcceptedPath(1, 8)
    p.path.copy_(ints([[0, 3, 4, 9, 15, 20, -1, -1]])), p.count.fill_(6)
    for c, tab in ((cache, table), (small.cache, small.table)):
        K.PagedLayers([c]).commit(K.PagedBatch(ints([0, n]), ints([kv]), tab, n), p)
    cache.check(), small.cache.check()
    for a, b in ((kp, small.kp), (vp, small.vp)):
        assert torch.equal(a[table[0, pos // P].long(), :, pos % P], b[small.table[0, pos // P].long(), :, pos % P])


def test_slots_beyond_32_bits():
    """A pool of more than 2^31 tokens (8 bits, heads of 16; keys and values, which are alike, in one place)."""
    n_pages = 2 ** 27 + 3
    pool = torch.empty(n_pages, 1, 16, 16, device=dev(), dtype=torch.uint8).view(torch.float8_e4m3fn)
    cache = K.PagedCache(pool, pool)
    slots = torch.tensor([2 ** 31 - 1, 2 ** 31, 2 ** 31 + 16 + 5, n_pages * 16 - 1, n_pages * 16, 3], device=dev())
    x = rand(gen(3), 6, 1, 16)
    cache.store(slots, None, x, x)
    with pytest.raises(K.KoreCudaError, match="page id"):   # the slot behind the last
        cache.check()
    keep = slots < n_pages * 16
    got = pool[slots[keep] // 16, 0, slots[keep] % 16].float()
    assert torch.equal(got, x[keep, 0].to(torch.float8_e4m3fn).float())
    del pool, cache
    torch.cuda.empty_cache()


def test_a_step_in_which_a_sequence_got_no_pages():
    """It is left out of everything behind the plan, reported, and keeps what it held; the others go on."""
    g, r = gen(4), random.Random(4)
    P, G, d, H = 16, 2, 64, 8
    pool = K.PagePool(8, P, 3, 8)
    kp, vp = (torch.full((8, G, P, d), GUARD, device=dev(), dtype=torch.bfloat16) for _ in range(2))
    cache = K.PagedCache(kp, vp)
    step = pool.new_step(2, 40, 30)
    pool.plan(step, ints([0, 1]), ints([30, 10]))
    k, v = (rand(g, 40, G, d).to(torch.bfloat16) for _ in range(2))
    cache.store(step.slots, None, k, v)
    pool.check()
    ns = [20, 96]
    step, t, path = pool.new_step(2, 116, 96), K.TokenTree(116, 96), K.AcceptedPath(2, 4)
    par = [tree(r, n, "random") for n in ns]
    parent = ints(par[0] + par[1])
    pool.plan(step, ints([0, 1]), ints(ns))   # 50 and 106 positions: 4 + 7 pages of 8
    assert step.kv_len.tolist() == [50, 0] and pool.length.tolist() == [50, 10, 0]
    t.build(step, parent)
    k, v, q = (rand(g, 116, h, d).to(torch.bfloat16) for h in (G, G, H))
    cache.store(step.slots, t.pos, k, v, rope=K.RopeTable(60, d), q=q, q_out=q)
    out = torch.full_like(q, GUARD)
    cache.attend(step, q, out, tree=t)
    path.accept(step, parent, torch.zeros_like(parent), torch.ones_like(parent))
    K.PagedLayers([cache]).commit(step, path)
    pool.trim(ints([0, 1]), path.kept)
    assert path.kept.tolist() == [31, -1] and path.count.tolist() == [1, 0]
    assert pool.length.tolist() == [31, 10, 0] and int(pool.n_free) == 8 - 2 - 1
    C = Cache(g, "bf16", G, d, P, [50])
    C.kp, C.vp, C.table = kp, vp, step.page_table[:1]
    check_tree(C, q[:20], out[:20], [20], [sees(par[0])])
    assert (out[20:] == GUARD).all()
    for x, word in ((pool, "free pages"), (t, "bounds"), (cache, "bounds"), (path, "bounds")):
        with pytest.raises(K.KoreCudaError, match=word):
            x.check()


@KERNELS
def test_two_graphs_of_one_stream_on_two_streams(kernel):
    C, ns, q, seen, t = ready("bf16", "long")
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    with torch.cuda.stream(side):
        C.cache.attend(batch, q, tree=t)
        for o in outs:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                C.cache.attend(batch, q, o, tree=t)
            graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    C.cache.check()
    assert torch.equal(*outs)
    check_tree(C, q, outs[0], ns, seen)


def test_norms_of_queries_or_keys_alone():
    g = gen(5)
    C = Cache(g, "bf16", 2, 64, 16, [16])
    k, q = rand(g, 3, 2, 64).to(torch.bfloat16), rand(g, 3, 6, 64).to(torch.bfloat16)
    w = (1 + 0.3 * rand(g, 64)).to(torch.bfloat16)
    slots = torch.arange(3, device=dev())
    both = []
    for norm in (K.HeadNorm(w, w), K.HeadNorm(w, None), K.HeadNorm(None, w), None):
        o = torch.zeros_like(q)
        C.cache.store(slots, None, k, k, norm=norm, q=q, q_out=o)
        both.append((o, C.kp[0, :, :3].clone()))
    C.cache.check()
    assert torch.equal(both[1][0], both[0][0]) and torch.equal(both[2][1], both[0][1])
    assert torch.equal(both[3][0], q) and torch.equal(both[2][0], q)
    assert torch.equal(both[1][1], k.transpose(0, 1)) and torch.equal(both[3][1], k.transpose(0, 1))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two devices")
def test_a_step_on_another_device_than_the_current_one():
    other = torch.device("cuda", 1)
    pool = K.PagePool(8, 16, 3, 8, device=other)
    step, t, path = pool.new_step(1, 5, 5), K.TokenTree(5, 5, device=other), K.AcceptedPath(1, 3, device=other)
    n, who = torch.tensor([5], dtype=torch.int32, device=other), torch.tensor([1], dtype=torch.int32, device=other)
    par = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32, device=other)
    kp, vp = (torch.zeros(8, 2, 16, 64, device=other, dtype=torch.bfloat16) for _ in range(2))
    cache = K.PagedCache(kp, vp)
    q = torch.randn(5, 4, 64, device=other).bfloat16()
    pool.plan(step, who, n)
    t.build(step, par)
    cache.store(step.slots, t.pos, q[:, :2], q[:, 2:], rope=K.RopeTable(8, 64, device=other), q=q, q_out=q)
    out = cache.attend(step, q, tree=t)
    path.accept(step, par, par, par)
    K.PagedLayers([cache]).commit(step, path)
    pool.trim(who, path.kept)
    for x in (pool, t, cache, path):
        x.check()
    assert torch.isfinite(out).all() and torch.cuda.current_device() == 0
