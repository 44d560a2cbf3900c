"""The operators of a step with trees of drafted tokens over the caller-owned paged cache, as cases to measure: the step's
page tables, slots and positions made on the GPU from the requests' lengths (`pages`), the store of a step's keys and
values with norms of queries and keys for each head and the rotation on the way (`store`), the attention of the drafted
tokens over the context and their own branches (`tree`), and what follows it: the branch that the model accepts and its
keys and values moved together, in all layers (`verify`).

Head layouts are those of the attention configurations that the benchmark runs (14/2 heads of 64, 28/4 and 16/2 heads
of 128), with their models' 24, 28 and 36 layers; the lengths run from one token to the 32768 cached positions of its
long-context configuration.

Where `own` is false, run() computes the plain form with elementary torch operations; where it is true it makes the
calls of kore_b200. exact() computes the same in 64 bits (or in Python's whole numbers), sequence by sequence, from the
definition.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
HEADS = {"28/4x128": (28, 4, 128), "16/2x128": (16, 2, 128), "14/2x64": (14, 2, 64)}
LAYERS = {"28/4x128": 28, "16/2x128": 36, "14/2x64": 24}
EPS = 1e-6    # of the norms
BASE = 1e6    # of the rotation
VOCAB = 32000


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a generation step of 32 conversations, a token each: some of them begin a page
        dict(name="pages_step", op="pages", seqs=32, new=1, ragged=False, past=4000, page=64, tree=False, lens=1),
        # the same for 500 conversations with a drafted tree each, whose ancestors and positions are wanted too
        dict(name="pages_trees", op="pages", seqs=500, new=24, ragged=True, past=4000, page=16, tree=True, lens=2),
        # a server's largest step: prompts of many conversations, tens of thousands of tokens
        dict(name="pages_prompts", op="pages", seqs=96, new=2048, ragged=True, past=6000, page=16, tree=False, lens=3),
        # a generation step of 48 conversations: one new key and value each, the step's queries with them
        dict(name="store_step", op="store", heads="28/4x128", type="bf16", cache="bf16", seqs=48, new=1, ragged=False,
             past=4000, page=64, rot=128, interleaved=False, each=False, fused=True, tree=False, lens=4),
        # drafted trees of 64 conversations into an 8-bit cache; a weight of its own for each head
        dict(name="store_trees_e4m3", op="store", heads="16/2x128", type="bf16", cache="e4m3", seqs=64, new=25, ragged=True,
             past=3000, page=128, rot=128, interleaved=False, each=True, fused=True, tree=True, lens=5),
        # prompts of several conversations at once into an empty cache
        dict(name="store_prompts", op="store", heads="28/4x128", type="f16", cache="f16", seqs=6, new=2048, ragged=True,
             past=0, page=256, rot=128, interleaved=False, each=False, fused=True, tree=False, lens=6),
        # one short conversation with a small tree: latency
        dict(name="tree_one_short", op="tree", heads="28/4x128", type="bf16", cache="bf16", seqs=1, new=8, ragged=False,
             past=512, page=64, fused=False, lens=7),
        # a server's step: 32 conversations of any length, 16 drafted tokens each
        dict(name="tree_batch", op="tree", heads="28/4x128", type="bf16", cache="bf16", seqs=32, new=16, ragged=False,
             past=8192, page=256, fused=True, lens=8),
        # large trees at the end of long contexts, in an 8-bit cache: the largest
        dict(name="tree_long_e4m3", op="tree", heads="28/4x128", type="bf16", cache="e4m3", seqs=6, new=60, ragged=True,
             past=32768, page=256, fused=False, lens=9),
        # many conversations, small heads and pages, odd sizes, rows of padding behind them
        dict(name="tree_many", op="tree", heads="14/2x64", type="f16", cache="f16", seqs=48, new=33, ragged=True,
             past=3001, page=16, fused=True, lens=10),
        # the end of one conversation's step
        dict(name="verify_one", op="verify", heads="14/2x64", cache="f16", seqs=1, new=8, ragged=False, past=300, page=16,
             lens=11),
        # the end of a server's step
        dict(name="verify_batch", op="verify", heads="28/4x128", cache="bf16", seqs=64, new=24, ragged=True, past=150,
             page=64, lens=12),
    ]


def _log(rng, lo, hi):
    hi = max(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pages", "store", "tree", "tree", "verify"])
    page, lens = rng.choice([16, 48, 64, 128, 256]), rng.randrange(1 << 30)
    heads = rng.choice(sorted(HEADS))
    d = HEADS[heads][2]
    if op == "pages":
        seqs = _log(rng, 1, 2048)
        kind = rng.choice(["step", "tree", "prompts"])
        new = 1 if kind == "step" else _log(rng, 2, 64 if kind == "tree" else min(2048, 65536 // seqs))
        return dict(op=op, seqs=seqs, new=new, ragged=new > 1 and rng.random() < 0.7, past=_log(rng, 1, 1000000 // seqs) - 1
                    if seqs > 30 else _log(rng, 1, 32768) - 1, page=page, tree=kind == "tree" and seqs <= 512, lens=lens)
    if op == "store":
        kind = rng.choice(["f32", "f16", "bf16"])
        cache = rng.choice([kind, kind, "e4m3"] + (["f16", "bf16"] if kind == "f32" else []))
        tree = rng.random() < 0.4
        seqs = _log(rng, 1, 64)
        new = _log(rng, 2, 64) if tree else 1 if rng.random() < 0.3 else _log(rng, 1, max(1, 8192 // seqs))
        return dict(op=op, heads=heads, type=kind, cache=cache, seqs=seqs, new=new, ragged=new > 1 and rng.random() < 0.7,
                    past=_log(rng, 1, 12000 // max(1, seqs // 8)) - 1, page=page, rot=rng.choice([d, d, d // 2, d // 4]),
                    interleaved=rng.random() < 0.4, each=rng.random() < 0.3, fused=rng.random() < 0.5, tree=tree, lens=lens)
    if op == "tree":
        kind = rng.choice(["f16", "bf16"])
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 96 if seqs <= 4 else 64)
        past = _log(rng, 1, min(32768, 100000 // seqs, 3000000 // (seqs * new))) - 1
        return dict(op=op, heads=heads, type=kind, cache=rng.choice([kind, kind, "e4m3"]), seqs=seqs, new=new,
                    ragged=new > 1 and rng.random() < 0.6, past=past, page=page, fused=rng.random() < 0.5, lens=lens)
    seqs = _log(rng, 1, 64)
    return dict(op=op, heads=heads, cache=rng.choice(["f16", "bf16", "e4m3", "f32"]), seqs=seqs, new=_log(rng, 2, 64),
                ragged=rng.random() < 0.6, past=_log(rng, 1, 150) - 1, page=page, lens=lens)


def _lengths(case):
    """(new tokens, cached positions with them) of each sequence: the case's own, whatever the seed."""
    rng = random.Random(case["lens"])
    n, kv = [], []
    for s in range(case["seqs"]):
        ni = case["new"]
        if case["ragged"] and s:  # the first sequence has the longest chunk
            ni = rng.randrange(1, case["new"] + 1)
        past = case["past"] if s == 0 else rng.randrange(case["past"] // 8, case["past"] + 1)
        n.append(ni)
        kv.append(past + ni)
    return n, kv


def _parents(case):
    """The trees: for each sequence, its tokens' parents (indexes in the sequence's chunk; the root, token 0, has none).
    A drafter goes deep first, then wide: a token's parent is a late one more often than an early one."""
    rng = random.Random(case["lens"] + 1)
    return [[-1] + [max(rng.randrange(i), rng.randrange(i)) for i in range(1, n)] for n in _lengths(case)[0]]


def _accepted(case):
    """How many drafted tokens (the root not counted) each sequence's model accepts."""
    rng = random.Random(case["lens"] + 2)
    return [rng.randrange(0, min(7, (n - 1) // 2) + 1) for n in _lengths(case)[0]]


def work(case):
    n, kv = _lengths(case)
    t, P = sum(n), case["page"]
    if case["op"] == "pages":
        used = sum(-(-k // P) for k in kv)
        fresh = used - sum(-(-(k - i) // P) for i, k in zip(n, kv))
        words = -(-max(n) // 32) if case["tree"] else 0
        # requests, counts, lengths and tables in; bounds, tables, slots and positions out; pages taken and given back;
        # of trees, parents in, ancestors and positions out
        return {"bytes": len(n) * 32 + 8 * used + 12 * t + 24 * fresh + (t * (8 + 4 * words) if case["tree"] else 0),
                "flops": 0}
    H, G, d = HEADS[case["heads"]]
    c = SIZE[case["cache"]]
    if case["op"] == "store":  # q, k, v, slots, positions and their angles in; q, k and v out
        e = SIZE[case["type"]]
        return {"bytes": t * ((H + 2 * G) * d * e + 12 + H * d * e + 2 * G * d * c) + min(t, max(kv)) * case["rot"] * 4,
                "flops": t * (H + G) * (4 * d + 3 * case["rot"])}
    if case["op"] == "tree":
        e = SIZE[case["type"]]
        pairs = 0
        for ni, ki, par in zip(n, kv, _parents(case)):
            depth = []
            for x in par:
                depth.append(1 if x < 0 else depth[x] + 1)
            pairs += ni * (ki - ni) + sum(depth)
        return {"bytes": 2 * sum(kv) * G * d * c + 2 * t * H * d * e + 4 * t * -(-max(n) // 32), "flops": 4 * pairs * H * d}
    # parents, tokens and choices in, path, length and next token out; the moved rows in and out
    return {"bytes": 12 * t + 24 * len(n) + 4 * sum(_accepted(case)) * LAYERS[case["heads"]] * G * d * c, "flops": t}


# ---------------------------------------------------------------- inputs

def _frequencies(rot):
    """The rotation's frequencies, each rounded to 32 bits."""
    return torch.tensor([BASE ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64).to(torch.float32).cuda()


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def _table(ns, kvs, P, g):
    """A batch's page table: pages in any order, -1 behind a sequence's last."""
    used = [-(-k // P) for k in kvs]
    order = torch.randperm(sum(used), device="cuda", generator=g).to(torch.int32).cpu()
    table, at = torch.full((len(ns), max(used)), -1, dtype=torch.int32), 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    return table.cuda(), sum(used)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ns, kvs = _lengths(case)
    P, tokens, pad = case["page"], sum(ns), (3 if case["ragged"] else 0)
    rows = tokens + pad  # rows behind the last sequence, as a padded batch has them
    starts = [0]
    for x in ns:
        starts.append(starts[-1] + x)
    S = dict(case=case, ns=ns, kvs=kvs, tokens=tokens, rows=rows, max_q=max(ns), starts=starts)
    if case["op"] == "pages":
        return _prepare_pages(S, g, pad)
    H, G, d = HEADS[case["heads"]]
    S.update(H=H, G=G, d=d, q_start=_ints(starts), kv_len=_ints(kvs), max_kv=max(kvs))
    S["table_"], total = _table(ns, kvs, P, g)
    cd = DTYPES[case["cache"]]
    if case["op"] == "verify":
        return _prepare_verify(S, g, seed, total, cd)
    dt = DTYPES[case["type"]]
    S["ks"] = S["vs"] = None
    if case["cache"] == "e4m3":  # a value is its 8 bits times its head's scale
        S["ks"] = 0.02 * (1 + torch.rand(G, device="cuda", generator=g))
        S["vs"] = 0.01 * (1 + torch.rand(G, device="cuda", generator=g))

    def filled(scale):
        x = torch.randn((total, G, P, d), device="cuda", generator=g)
        return (x if scale is None else (x / scale[:, None, None]).clamp(-448.0, 448.0)).to(cd)

    S["kp"], S["vp"] = filled(S["ks"]), filled(S["vs"])
    wide = torch.randn(rows, (H + 2 * G) * d, device="cuda", generator=g).to(dt)  # what a fused projection leaves
    q, k, v = (x.unflatten(1, (-1, d)) for x in wide.split([H * d, G * d, G * d], 1))
    S["q"] = q if case["fused"] else q.contiguous()
    S["out"] = torch.zeros(rows, H, d, device="cuda", dtype=dt)
    if case["op"] == "tree":
        words = -(-max(ns) // 32)
        mask = torch.zeros(rows, words, dtype=torch.int64)
        parent = torch.full((rows,), -1, dtype=torch.int32)
        for s, par in enumerate(_parents(case)):
            parent[starts[s]:starts[s + 1]] = _ints(par).cpu()
            bits = []
            for i, x in enumerate(par):
                bits.append((1 << i) | (bits[x] if x >= 0 else 0))
                for w in range(words):
                    mask[starts[s] + i, w] = bits[i] >> (32 * w) & 0xffffffff
        S["mask"] = mask.cuda()  # bit j of a token's words: it sees token j of its chunk
        if own:
            import kore_b200 as K
            S["cache"] = K.PagedCache(S["kp"], S["vp"], k_scale=S["ks"], v_scale=S["vs"])
            S["batch"] = K.PagedBatch(S["q_start"], S["kv_len"], S["table_"], max_q=S["max_q"])
            S["tree"] = K.TokenTree(rows, S["max_q"])
            S["tree"].build(S["batch"], parent.cuda())
        return S
    S["k"], S["v"] = (k, v) if case["fused"] else (k.contiguous(), v.contiguous())
    slots, pos = [], []
    table, trees = S["table_"].cpu().tolist(), _parents(case)
    for s, (n, kv) in enumerate(zip(ns, kvs)):
        slots += [table[s][p // P] * P + p % P for p in range(kv - n, kv)]
        depth = []
        for i, x in enumerate(trees[s]):
            depth.append(i if not case["tree"] else 0 if x < 0 else depth[x] + 1)
        pos += [kv - n + x for x in depth]
    S["slots"], S["pos"] = _ints(slots + [-1] * pad, torch.int64), _ints(pos + [-1] * pad)
    shape = ((H, d), (G, d)) if case["each"] else ((d,), (d,))
    S["qw"], S["kw"] = ((1 + 0.2 * torch.randn(x, device="cuda", generator=g)).to(dt) for x in shape)
    S["freq"] = _frequencies(case["rot"])
    if own:
        import kore_b200 as K
        S["cache"] = K.PagedCache(S["kp"], S["vp"], k_scale=S["ks"], v_scale=S["vs"])
        S["rope"] = K.RopeTable(max(kvs), case["rot"], base=BASE, interleaved=case["interleaved"])
        S["norm"] = K.HeadNorm(S["qw"], S["kw"], eps=EPS)
    return S


def _prepare_pages(S, g, pad):
    """A pool in use: some requests hold pages, the step is of some of them in any order, padded at its end."""
    case, ns, kvs, P = S["case"], S["ns"], S["kvs"], S["case"]["page"]
    n_seq = len(ns) + pad
    n_req = len(ns) + len(ns) // 4 + 1
    width = max(3, -(-(max(kvs) + 1) // P) + 1)
    past = [k - n for n, k in zip(ns, kvs)]
    fresh = sum(-(-k // P) - -(-p // P) for k, p in zip(kvs, past))
    who = torch.randperm(n_req, device="cuda", generator=g).cpu()
    length = torch.zeros(n_req, dtype=torch.int32)
    length[who[: len(ns)]] = torch.tensor(past, dtype=torch.int32)
    length[who[len(ns):]] = 2 * P + 1  # requests that this step does not run
    held = -(-length // P)
    n_pages = int(held.sum()) + fresh + fresh // 8 + 5
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    mine = torch.arange(width)[None] < held[:, None]
    table = torch.full((n_req, width), -1, dtype=torch.int32)
    table[mine] = order[: int(held.sum())].cpu()
    n_free = n_pages - int(held.sum())
    free = torch.full((n_pages,), -1, dtype=torch.int32).cuda()
    free[:n_free] = order[n_pages - n_free:]
    S.update(n_seq=n_seq, width=width, request=_ints(who[: len(ns)].tolist() + [-1] * pad),
             n_new=_ints(ns + [0] * pad), keep=_ints(past + [0] * pad))
    start = dict(free=free, n_free=_ints([n_free]), table=table.cuda(), length=length.cuda())
    if case["tree"]:
        par = [x for p in _parents(case) for x in p]
        S["parent"] = _ints(par + [-1] * pad)
    if own:
        import kore_b200 as K
        S["pool"] = K.PagePool(n_pages, P, n_req, width)
        for name, x in start.items():
            getattr(S["pool"], name).copy_(x)
        S["step"] = S["pool"].new_step(n_seq, S["rows"], max_q=S["max_q"])
        if case["tree"]:
            S["tree"] = K.TokenTree(S["rows"], S["max_q"])
            S["tree"].mask.zero_()
            S["tree"].pos.fill_(-1)
        return S
    S.update(start)
    rows = S["rows"]
    S.update(q_start=torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda"),
             kv_len=torch.zeros(n_seq, dtype=torch.int32, device="cuda"),
             page_table=torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda"),
             slots=torch.full((rows,), -1, dtype=torch.int64, device="cuda"),
             pos=torch.full((rows,), -1, dtype=torch.int32, device="cuda"))
    if case["tree"]:
        words = -(-S["max_q"] // 32)
        S.update(mask=torch.zeros(rows, words, dtype=torch.int32, device="cuda"),
                 tree_pos=torch.full((rows,), -1, dtype=torch.int32, device="cuda"))
    return S


def _prepare_verify(S, g, seed, total, cd):
    """Trees with their drafted tokens, the model's choice behind each token, and every layer's cache. The accepted branch
    of each is not among the tokens whose places it takes, so that a pass leaves what another pass would take."""
    case, ns, G, d, P = S["case"], S["ns"], S["G"], S["d"], S["case"]["page"]
    L = LAYERS[case["heads"]]
    pool = torch.randn((L, 2, total, G, P, d), device="cuda", generator=g, dtype=torch.bfloat16 if cd.itemsize < 4 else cd)
    S["layers"] = pool.to(cd)
    del pool
    rng = random.Random(seed)
    parent, tokens, choice = [], [], []
    for n, par, a in zip(ns, _parents(case), _accepted(case)):
        par = list(par)
        path = [0] + sorted(rng.sample(range(a + 1, n), a))
        for i, x in zip(path, path[1:]):
            par[x] = i
        tok = [rng.randrange(VOCAB) for _ in range(n)]
        ch = [rng.randrange(VOCAB) for _ in range(n)]
        for i, x in zip(path, path[1:]):
            ch[i] = tok[x]
        while any(par[x] == path[-1] and tok[x] == ch[path[-1]] for x in range(n)):
            ch[path[-1]] = rng.randrange(VOCAB)
        for i, x in zip(path, path[1:]):  # of siblings with the same token the first is taken
            for y in range(n):
                if y != x and par[y] == i and tok[y] == tok[x]:
                    tok[y] = (tok[y] + 1) % VOCAB
        parent += par
        tokens += tok
        choice += ch
    pad = S["rows"] - S["tokens"]
    S.update(parent=_ints(parent + [-1] * pad), tok=_ints(tokens + [0] * pad), choice=_ints(choice + [0] * pad), deep=8)
    if own:
        import kore_b200 as K
        S["caches"] = K.PagedLayers([K.PagedCache(x[0], x[1]) for x in S["layers"]])
        S["batch"] = K.PagedBatch(S["q_start"], S["kv_len"], S["table_"], max_q=S["max_q"])
        S["path"] = K.AcceptedPath(len(ns), S["deep"])
    return S


# ---------------------------------------------------------------- the plain form

def _up(a, b):
    return torch.div(a + b - 1, b, rounding_mode="floor")


def _plain_pages(S):
    case, P, width, rows = S["case"], S["case"]["page"], S["width"], S["rows"]
    r = S["request"].long()
    here = r >= 0
    r = r.clamp(min=0)
    base = torch.where(here, S["length"][r].long(), 0)
    n = torch.where(here, S["n_new"].long(), 0)
    ends = n.cumsum(0)
    kv = base + n
    have, want = _up(base, P), _up(kv, P)
    need = want - have
    upto = need.cumsum(0)
    # pages for each sequence in turn, from the end of the list
    s = torch.repeat_interleave(torch.arange(len(n), device="cuda"), need)
    j = torch.arange(s.numel(), device="cuda")
    S["table"][r[s], have[s] + j - (upto - need)[s]] = S["free"][S["n_free"].long() - 1 - j]
    S["n_free"] -= upto[-1].int()
    S["q_start"][1:] = ends.int()
    S["kv_len"].copy_(kv)
    held = (torch.arange(width, device="cuda") < want[:, None])
    S["page_table"].copy_(torch.where(held, S["table"][r], S["page_table"]))
    S["length"].scatter_(0, r[here], kv[here].int())
    t = torch.arange(rows, device="cuda")
    s = torch.searchsorted(ends, t, right=True).clamp(max=len(n) - 1)
    pos = base[s] + t - (ends - n)[s]
    live = t < ends[-1]
    page = S["page_table"][s, torch.where(live, pos // P, 0)].long()
    S["slots"].copy_(torch.where(live, page * P + pos % P, -1))
    S["pos"].copy_(torch.where(live, pos, -1))
    if case["tree"]:
        # ancestors by doubling: those within 2^k steps up, and the one 2^k steps up
        first = (ends - n)[s]
        up = torch.where(live & (S["parent"] >= 0), S["parent"].long() + first, t)
        seen = torch.zeros(rows, S["max_q"], dtype=torch.bool, device="cuda")
        seen[t[live], (t - first)[live]] = True
        for _ in range(max(1, S["max_q"].bit_length())):
            seen |= seen[up]
            up = up[up]
        bits = torch.nn.functional.pad(seen, (0, -S["max_q"] % 32)).unflatten(1, (-1, 32)).long()
        words = (bits << torch.arange(32, device="cuda")).sum(-1)
        S["mask"].copy_(torch.where(words >= 1 << 31, words - (1 << 32), words))
        S["tree_pos"].copy_(torch.where(live, base[s] + seen.sum(1) - 1, -1))
    # and back: the pages behind the kept positions, so that taking them again would give the same
    keep = torch.where(here, S["keep"].long(), 0)
    now = torch.where(here, S["length"][r].long(), 0)
    left, gone = _up(keep, P), _up(now, P) - _up(keep, P)
    upto = gone.cumsum(0)
    s = torch.repeat_interleave(torch.arange(len(n), device="cuda"), gone)
    j = torch.arange(s.numel(), device="cuda")
    at = (r[s], left[s] + j - (upto - gone)[s])
    S["n_free"] += upto[-1].int()
    S["free"][S["n_free"].long() - 1 - j] = S["table"][at]
    S["table"][at] = -1
    S["length"].scatter_(0, r[here], keep[here].int())
    got = [S[x] for x in ("q_start", "kv_len", "page_table", "slots", "pos", "table", "length", "n_free")]
    return got + [S["free"]] + ([S["mask"], S["tree_pos"]] if case["tree"] else [])


def _normed(x, w):
    """x [n][heads][d] in 32 bits over its root mean square, times w [d] or [heads][d]."""
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotate(x, pos, freq, interleaved):
    """x [n][heads][d] in 32 bits, the angles in 64."""
    a = pos.double()[:, None] * freq.double()
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    r, y = 2 * freq.numel(), x.clone()
    if interleaved:
        x0, x1 = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = x0 * c - x1 * s, x0 * s + x1 * c
    else:
        x0, x1 = x[..., : r // 2], x[..., r // 2: r]
        y[..., : r // 2], y[..., r // 2: r] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def _plain_store(S):
    P, n = S["case"]["page"], S["tokens"]
    slots, pos = S["slots"][:n], S["pos"][:n]
    page, slot = slots // P, slots % P
    heads = torch.arange(S["G"], device="cuda")[None]
    rot = (pos, S["freq"], S["case"]["interleaved"])
    for pages, x, scale in ((S["kp"], _rotate(_normed(S["k"][:n], S["kw"]), *rot), S["ks"]),
                            (S["vp"], S["v"][:n].float(), S["vs"])):
        if scale is not None:
            x = (x / scale[None, :, None]).clamp(-448.0, 448.0)
        pages[page[:, None], heads, slot[:, None]] = x.to(pages.dtype)
    S["out"][:n] = _rotate(_normed(S["q"][:n], S["qw"]), *rot).to(S["out"].dtype)
    return S["kp"], S["vp"], S["out"]


def _plain_tree(S):
    H, G, d = S["H"], S["G"], S["d"]
    N, L = S["max_q"], S["max_kv"]

    def gather(pages, scale, table):  # [B][G][L][d]
        x = pages[table.long().clamp(min=0)].float().transpose(1, 2).flatten(2, 3)[:, :, :L]
        return x * scale[None, :, None, None] if scale is not None else x

    i, t = torch.arange(N, device="cuda"), torch.arange(L, device="cuda")
    most = max(1, (1 << 29) // (L * max(G * d, H * N)))  # sequences at a time, so that it fits
    for a in range(0, len(S["ns"]), most):
        b = min(len(S["ns"]), a + most)
        n = (S["q_start"][a + 1: b + 1] - S["q_start"][a:b]).long()
        here = i < n[:, None]  # [B][N]
        tok = torch.where(here, S["q_start"][a:b].long()[:, None] + i, 0)
        kv = S["kv_len"][a:b].long()
        k, v = (gather(S[x], S[y], S["table_"][a:b]) for x, y in (("kp", "ks"), ("vp", "vs")))
        v = torch.where((t < kv[:, None])[:, None, :, None], v, 0.0)
        q = S["q"][tok].float().unflatten(2, (G, H // G)).permute(0, 2, 3, 1, 4).flatten(2, 3)
        s = (q @ k.transpose(2, 3)).unflatten(2, (H // G, N)) / math.sqrt(d)  # [B][G][H/G][N][L]
        own_ = t - (kv - n)[:, None]  # [B][L]: index in the chunk, below 0 in the context
        word = (own_.clamp(min=0) // 32).clamp(max=S["mask"].shape[1] - 1)
        bits = torch.gather(S["mask"][tok], 2, word[:, None].expand(-1, N, -1)) >> (own_.clamp(min=0) % 32)[:, None]
        seen = (own_ < 0)[:, None] | ((bits & 1 > 0) & (own_ < n[:, None])[:, None])
        s.masked_fill_(~seen[:, None, None], -math.inf)
        s -= s.amax(-1, keepdim=True)
        s.exp_()
        out = (s.flatten(2, 3) @ v) / s.sum(-1).flatten(2, 3)[..., None]
        out = out.unflatten(2, (H // G, N)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B][N][H][d]
        S["out"][tok[here]] = out[here].to(S["out"].dtype)
    return S["out"]


def _plain_verify(S):
    n_seq, deep, P = len(S["ns"]), S["deep"], S["case"]["page"]
    first, n = S["q_start"][:-1].long(), (S["q_start"][1:] - S["q_start"][:-1]).long()
    i = torch.arange(S["max_q"], device="cuda")
    here = i < n[:, None]
    at = torch.where(here, first[:, None] + i, 0)
    parent, tok, choice = (S[x][at].long() for x in ("parent", "tok", "choice"))  # [B][N]
    path = torch.full((n_seq, deep), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    now, going, count = torch.zeros_like(n), n > 0, torch.ones_like(n)
    for j in range(1, deep):
        want = choice.gather(1, now[:, None])
        hit = here & (parent == now[:, None]) & (tok == want)
        child = torch.where(hit, i, S["max_q"]).amin(1)
        going &= child < S["max_q"]
        path[:, j] = torch.where(going, child, -1)
        count += going
        now = torch.where(going, child, now)
    after = choice.gather(1, now[:, None])[:, 0]
    base = S["kv_len"].long() - n
    s = torch.arange(n_seq, device="cuda")[:, None].expand(-1, deep)
    j = torch.arange(deep, device="cuda").expand(n_seq, -1)
    move = (path >= 0) & (path != j)
    s, to, src = s[move], (base[:, None] + j)[move], (base[:, None] + path)[move]
    rows = S["layers"][:, :, S["table_"][s, src // P].long(), :, src % P]
    S["layers"][:, :, S["table_"][s, to // P].long(), :, to % P] = rows
    return [x.int() for x in (path, count, after, base + count)] + [S["layers"]]


def run(state):
    S = state
    op = S["case"]["op"]
    if not own:
        return {"pages": _plain_pages, "store": _plain_store, "tree": _plain_tree, "verify": _plain_verify}[op](S)
    if op == "pages":
        pool, step = S["pool"], S["step"]
        pool.plan(step, S["request"], S["n_new"])
        if S["case"]["tree"]:
            S["tree"].build(step, S["parent"])
        pool.trim(S["request"], S["keep"])
        got = [step.q_start, step.kv_len, step.page_table, step.slots, step.pos, pool.table, pool.length, pool.n_free, pool.free]
        return got + ([S["tree"].mask, S["tree"].pos] if S["case"]["tree"] else [])
    if op == "store":
        S["cache"].store(S["slots"], S["pos"], S["k"], S["v"], rope=S["rope"], norm=S["norm"], q=S["q"], q_out=S["out"])
        return S["kp"], S["vp"], S["out"]
    if op == "tree":
        S["cache"].attend(S["batch"], S["q"], S["out"], tree=S["tree"])
        return S["out"]
    path = S["path"]
    path.accept(S["batch"], S["parent"], S["tok"], S["choice"])
    S["caches"].commit(S["batch"], path)
    return path.path, path.count, path.next_token, path.kept, S["layers"]


# ---------------------------------------------------------------- the definition, in 64 bits

def _exact_pages(case, seed):
    """Page by page and token by token, on the host; of a pool that is given back what it held at the start."""
    S = prepare(case, seed)
    P, width, n_seq, rows = case["page"], S["width"], S["n_seq"], S["rows"]
    pool = S["pool"] if own else None
    state = {x: (getattr(pool, x) if own else S[x]).cpu().tolist() for x in ("free", "n_free", "table", "length")}
    start = {x: torch.tensor(state[x], dtype=torch.int32) for x in state}
    free = state["free"][: state["n_free"][0]]
    q_start, kv_len, page_table, slots, pos = [0], [], [], [], []
    for r, n in zip(S["request"].tolist(), S["n_new"].tolist()):
        row = []
        if r >= 0:
            total = state["length"][r] + n
            row = [x for x in state["table"][r] if x >= 0]
            while len(row) * P < total:
                row.append(free.pop())
            for p in range(total - n, total):
                slots.append(row[p // P] * P + p % P)
                pos.append(p)
        q_start.append(q_start[-1] + (n if r >= 0 else 0))
        kv_len.append(total if r >= 0 else 0)
        page_table.append(row + [-1] * (width - len(row)))
    slots += [-1] * (rows - len(slots))
    pos += [-1] * (rows - len(pos))
    got = [torch.tensor(x, dtype=t) for x, t in ((q_start, torch.int32), (kv_len, torch.int32), (page_table, torch.int32),
                                                 (slots, torch.int64), (pos, torch.int32))]
    got += [start[x] for x in ("table", "length", "n_free", "free")]
    if case["tree"]:
        words = -(-S["max_q"] // 32)
        mask, where = torch.zeros(rows, words, dtype=torch.int64), torch.full((rows,), -1, dtype=torch.int32)
        at = 0
        for par, kv in zip(_parents(case), S["kvs"]):
            for i in range(len(par)):
                x, steps = i, -1
                while x >= 0:
                    mask[at + i, x // 32] |= 1 << (x % 32)
                    x, steps = par[x], steps + 1
                where[at + i] = kv - len(par) + steps
            at += len(par)
        got += [torch.where(mask >= 1 << 31, mask - (1 << 32), mask).int(), where]
    return got


def _turned(x, pos, freq, interleaved):
    """Rows as complex numbers times e^(i angle)."""
    r = 2 * freq.numel()
    angle = torch.outer(pos.double(), freq.double())
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if interleaved:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:2], r // 2, 2).contiguous()) * turn
        y = torch.view_as_real(z).reshape(*x.shape[:2], r)
    else:
        z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., r:]], -1)


def _eight_bits(x):
    """The nearest e4m3 values (ties to the even mantissa), saturating."""
    m = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(m.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign((torch.round(m / step) * step).clamp(max=448.0), x)


def _exact_store(case, seed):
    S = prepare(case, seed)
    P, at = case["page"], 0
    table = S["table_"].long()
    kp, vp, out = S["kp"].double(), S["vp"].double(), S["out"].double()

    def unit(x, w):
        x = x.double()
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()

    for s, (n, kv) in enumerate(zip(S["ns"], S["kvs"])):
        here = slice(at, at + n)
        slot, pos = torch.arange(kv - n, kv, device="cuda"), S["pos"][here]
        k, v = _turned(unit(S["k"][here], S["kw"]), pos, S["freq"], case["interleaved"]), S["v"][here].double()
        if S["ks"] is not None:
            k, v = (_eight_bits(x / c.double()[:, None]) for x, c in ((k, S["ks"]), (v, S["vs"])))
        kp[table[s, slot // P], :, slot % P] = k
        vp[table[s, slot // P], :, slot % P] = v
        out[here] = _turned(unit(S["q"][here], S["qw"]), pos, S["freq"], case["interleaved"])
        at += n
    return kp, vp, out


def _exact_tree(case, seed):
    S = prepare(case, seed)
    H, G, d, P = S["H"], S["G"], S["d"], case["page"]
    table, at, out = S["table_"].long(), 0, S["out"].double()
    for s, (n, kv, par) in enumerate(zip(S["ns"], S["kvs"], _parents(case))):
        t = torch.arange(kv, device="cuda")
        k, v = (x[table[s, t // P], :, t % P].double() for x in (S["kp"], S["vp"]))  # [kv][G][d]
        if S["ks"] is not None:
            k, v = k * S["ks"].double()[:, None], v * S["vs"].double()[:, None]
        sees = torch.zeros(n, n, dtype=torch.bool)
        for i, x in enumerate(par):
            if x >= 0:
                sees[i] = sees[x]
            sees[i, i] = True
        seen = torch.cat([torch.ones(n, kv - n, dtype=torch.bool), sees], 1).cuda()
        for h in range(H):
            score = S["q"][at: at + n, h].double() @ k[:, h // (H // G)].T * d ** -0.5
            out[at: at + n, h] = score.masked_fill(~seen, -math.inf).softmax(-1) @ v[:, h // (H // G)]
        at += n
    return out


def _exact_verify(case, seed):
    """Token by token, on the host; the moved rows are copies, so that the caches keep their type."""
    S = prepare(case, seed)
    P, deep = case["page"], S["deep"]
    parent, tok, choice, table = (S[x].tolist() for x in ("parent", "tok", "choice", "table_"))
    layers = S["layers"].clone()
    paths, count, after, kept, at = [], [], [], [], 0
    for s, (n, kv) in enumerate(zip(S["ns"], S["kvs"])):
        path = [0]
        while len(path) < deep:
            hits = [i for i in range(n) if parent[at + i] == path[-1] and tok[at + i] == choice[at + path[-1]]]
            if not hits:
                break
            path.append(hits[0])
        for j, i in enumerate(path):
            a, b = kv - n + i, kv - n + j
            layers[:, :, table[s][b // P], :, b % P] = S["layers"][:, :, table[s][a // P], :, a % P]
        paths.append(path + [-1] * (deep - len(path)))
        count.append(len(path))
        after.append(choice[at + path[-1]])
        kept.append(kv - n + len(path))
        at += n
    return [torch.tensor(x, dtype=torch.int32) for x in (paths, count, after, kept)] + [layers]


def exact(case, seed):
    return {"pages": _exact_pages, "store": _exact_store, "tree": _exact_tree, "verify": _exact_verify}[case["op"]](case, seed)
