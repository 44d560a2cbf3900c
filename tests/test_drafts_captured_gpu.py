"""A step with drafted tokens captured as two graphs, before and behind the model's choices: every token's attention of
every replay, whose requests, counts and trees are those of its replay."""
import random

import pytest

import kore_b200 as K
from kore_b200.paged import set_tree_kernel
from tests.test_drafts_gpu import accepted, check_tree, sees, tree
from tests.test_paged_gpu import DT, GUARD, Cache, dev, gen, ints, rand

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("tc,H,G,d", [("bf16", 14, 2, 64), ("e4m3", 28, 4, 128)])
def test_every_token_of_a_replayed_step(kernel, tc, H, G, d):
    g, r = gen(d), random.Random(d)
    P, n_seq, n_tok, most = 16, 4, 70, 40
    pool = K.PagePool(200, P, 6, 30)
    kp, vp = (torch.zeros(200, G, P, d, device=dev()).to(DT[tc]) for _ in range(2))
    scales = [0.01 * (1 + torch.rand(G, device=dev(), generator=g)) for _ in range(2)] if tc == "e4m3" else [None, None]
    cache = K.PagedCache(kp, vp, k_scale=scales[0], v_scale=scales[1])
    layers, rope, norm = K.PagedLayers([cache]), K.RopeTable(500, d), K.HeadNorm(1 + 0.1 * rand(g, d), 1 + 0.1 * rand(g, d))
    step, t, path = pool.new_step(n_seq, n_tok, most), K.TokenTree(n_tok, most), K.AcceptedPath(n_seq, 5)
    request, n_new = ints([0, 1, 2, -1]), ints([1, 1, 1, 0])
    parent, token, choice = (torch.zeros(n_tok, dtype=torch.int32, device=dev()) for _ in range(3))
    parent.fill_(-1)
    q, k, v = (rand(g, n_tok, h, d).to(torch.bfloat16) for h in (H, G, G))
    qr, out = torch.zeros_like(q), torch.full_like(q, GUARD)

    def drafted():
        pool.plan(step, request, n_new)
        t.build(step, parent)
        cache.store(step.slots, t.pos, k, v, rope=rope, norm=norm, q=q, q_out=qr)
        cache.attend(step, qr, out, tree=t)

    def chosen():
        path.accept(step, parent, token, choice, tree=t)
        layers.commit(step, path)
        pool.trim(request, path.kept)

    graphs, side = [], torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    set_tree_kernel(kernel)
    try:
        with torch.cuda.stream(side):
            for f in (drafted, chosen):
                f()
                gr = torch.cuda.CUDAGraph()
                with torch.cuda.graph(gr, stream=side):
                    f()
                graphs.append(gr)
    finally:
        set_tree_kernel("auto")
    torch.cuda.synchronize()
    pool.trim(ints([0, 1, 2]), ints([0, 0, 0]))
    lengths = [0] * 6
    for turn in range(8):
        who = r.sample(range(6), n_seq - turn % 2) + [-1] * (turn % 2)
        ns, room = [], n_tok
        for w in who:   # chunks of more than 32 tokens, and none, among them
            ns.append(min(r.choice([0, 1, 7, 33, 40]), room) if w >= 0 else 0)
            room -= ns[-1]
        par = [tree(r, n, r.choice(["random", "roots", "chain"])) if n else [] for n in ns]
        tk = [[r.randrange(2) for _ in p] for p in par]
        ch = [[r.randrange(2) for _ in p] for p in par]
        fill = lambda x: ints([z for y in x for z in y] + [0] * (n_tok - sum(ns)))   # noqa: E731
        for dst, src in ((request, ints(who)), (n_new, ints(ns)), (parent, fill(par)), (token, fill(tk)), (choice, fill(ch))):
            dst.copy_(src)
        for x, h in ((q, H), (k, G), (v, G)):
            x.copy_(rand(g, n_tok, h, d))
        out.fill_(GUARD)
        graphs[0].replay()
        torch.cuda.synchronize()
        live = [s for s, n in enumerate(ns) if n]
        assert step.kv_len.tolist() == [lengths[w] + n if w >= 0 else 0 for w, n in zip(who, ns)]
        if live:
            C = Cache(g, tc, G, d, P, [1])
            C.kvs, C.table = [step.kv_len.tolist()[s] for s in live], step.page_table[live]
            C.kp, C.vp, C.ks, C.vs = kp, vp, *scales
            check_tree(C, qr, out, [ns[s] for s in live], [sees(par[s]) for s in live])
        assert (out[sum(ns):] == GUARD).all()
        graphs[1].replay()
        torch.cuda.synchronize()
        for w, n, p, a, b in zip(who, ns, par, tk, ch):
            if n:
                lengths[w] += len(accepted(p, a, b, 5))
        assert pool.length.tolist() == lengths
        assert int(pool.n_free) == 200 - sum(-(-x // P) for x in lengths)
    for x in (pool, t, path, layers, cache):
        x.check()
