"""The operators of the caller-owned paged cache, as cases to measure: rotary positions (`rope`), the append of a ragged
batch's keys and values with the rotation on the way (`append`), and the attention of the batch's new tokens over the
cache (`attend`).

Head layouts are those of the attention configurations that the benchmark runs (14/2 heads of 64, 28/4 and 16/2 heads
of 128); the lengths run from one token to the 32768 cached positions of its long-context configuration.

Where `own` is false, run() computes the plain form with elementary torch operations; where it is true it makes the
calls of kore_b200. exact() computes the same in 64 bits, sequence by sequence, from the definition.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
HEADS = {"28/4x128": (28, 4, 128), "16/2x128": (16, 2, 128), "14/2x64": (14, 2, 64)}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one query row of one generated token, far into a context: the smallest call
        dict(name="rope_one_token", op="rope", heads="28/4x128", type="bf16", tokens=1, rot=128, interleaved=False,
             scaling="none", fused=False, pos0=20011),
        # the queries of a prompt chunk, in a context extended past the trained one
        dict(name="rope_chunk_yarn", op="rope", heads="28/4x128", type="bf16", tokens=4096, rot=128, interleaved=False,
             scaling="yarn", fused=False, pos0=28000),
        # half of each head rotated, neighbouring pairs, read out of a fused q|k|v row
        dict(name="rope_partial_fused", op="rope", heads="14/2x64", type="f32", tokens=777, rot=32, interleaved=True,
             scaling="linear", fused=True, pos0=100),
        # a generation step of 48 conversations: one new key and value each, the step's queries rotated with them
        dict(name="append_step", op="append", heads="28/4x128", type="bf16", cache="bf16", seqs=48, new=1, ragged=False,
             past=4000, page=64, rot=128, interleaved=False, scaling="none", fused=True, lens=1),
        # prompts of several conversations at once into an empty cache
        dict(name="append_prompts", op="append", heads="28/4x128", type="f16", cache="f16", seqs=6, new=2048, ragged=True,
             past=0, page=256, rot=128, interleaved=False, scaling="none", fused=True, lens=2),
        # a chunk of each of three conversations into an 8-bit cache
        dict(name="append_chunk_e4m3", op="append", heads="16/2x128", type="bf16", cache="e4m3", seqs=3, new=1021, ragged=True,
             past=3000, page=128, rot=64, interleaved=True, scaling="yarn", fused=False, lens=3),
        # a short conversation's generation step: latency
        dict(name="attend_step_short", op="attend", heads="28/4x128", type="bf16", cache="bf16", seqs=1, new=1, ragged=False,
             past=512, page=64, window=0, fused=False, lens=4),
        # a generation step of 64 conversations of any length
        dict(name="attend_step_batch", op="attend", heads="16/2x128", type="bf16", cache="bf16", seqs=64, new=1, ragged=False,
             past=8192, page=256, window=0, fused=False, lens=5),
        # a generation step of long conversations in an 8-bit cache
        dict(name="attend_step_e4m3", op="attend", heads="28/4x128", type="f16", cache="e4m3", seqs=12, new=1, ragged=False,
             past=32768, page=256, window=0, fused=False, lens=6),
        # a prompt chunk at the end of a long context: the largest
        dict(name="attend_chunk_long", op="attend", heads="28/4x128", type="bf16", cache="bf16", seqs=1, new=2048, ragged=False,
             past=30720, page=256, window=0, fused=True, lens=7),
        # one step of a server: chunks of some conversations beside single tokens of others, rows of padding behind them
        dict(name="attend_mixed", op="attend", heads="14/2x64", type="f16", cache="f16", seqs=24, new=500, ragged=True,
             past=3001, page=16, window=0, fused=False, lens=8),
        # chunks over an 8-bit cache, each token looking back over a window
        dict(name="attend_chunk_window_e4m3", op="attend", heads="16/2x128", type="bf16", cache="e4m3", seqs=4, new=700,
             ragged=True, past=9000, page=64, window=4096, fused=False, lens=9),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    heads = rng.choice(sorted(HEADS))
    H, G, d = HEADS[heads]
    rot = dict(rot=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.4,
               scaling=rng.choice(["none", "linear", "yarn"]), fused=rng.random() < 0.5)
    if op == "rope":
        return dict(op=op, heads=heads, type=rng.choice(["f32", "f16", "bf16"]), tokens=_log(rng, 1, 4096),
                    pos0=rng.randrange(0, 28000), **rot)
    page, lens = rng.choice([16, 48, 64, 128, 256]), rng.randrange(1 << 30)
    if op == "append":
        kind = rng.choice(["f32", "f16", "bf16"])
        cache = rng.choice([kind, kind, "e4m3"] + (["f16", "bf16"] if kind == "f32" else []))
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, 8192 // seqs))
        return dict(op=op, heads=heads, type=kind, cache=cache, seqs=seqs, new=new, ragged=new > 1 and rng.random() < 0.7,
                    past=_log(rng, 1, 12000 // max(1, seqs // 8)) - 1, page=page, lens=lens, **rot)
    kind = rng.choice(["f16", "bf16"])
    cache = rng.choice([kind, kind, "e4m3"])
    window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
    if rng.random() < 0.5:  # generation steps
        seqs = _log(rng, 1, 96)
        new, past = 1, _log(rng, 1, min(32768, 524288 // seqs)) - 1
    else:  # chunks
        seqs = _log(rng, 1, 16)
        new = _log(rng, 2, 2048 // seqs)
        past = _log(rng, 1, min(30000, 100000 // seqs)) - 1
    return dict(op=op, heads=heads, type=kind, cache=cache, seqs=seqs, new=new, ragged=new > 1 and rng.random() < 0.7,
                past=past, page=page, window=window, fused=rng.random() < 0.5, lens=lens)


def _lengths(case):
    """(new tokens, cached positions after the append) of each sequence: the case's own, whatever the seed."""
    rng = random.Random(case["lens"])
    n, kv = [], []
    for s in range(case["seqs"]):
        ni = case["new"]
        if case["ragged"] and s:  # the first sequence has the longest chunk; half of the others a single token
            ni = 1 if rng.random() < 0.5 else rng.randrange(1, case["new"] + 1)
        past = case["past"] if s == 0 else rng.randrange(case["past"] // 8, case["past"] + 1)
        n.append(ni)
        kv.append(past + ni)
    return n, kv


def work(case):
    H, G, d = HEADS[case["heads"]]
    e = SIZE[case["type"]]
    if case["op"] == "rope":  # the positions and (cos, sin) of each token, the rows in and out
        t = case["tokens"]
        return {"bytes": t * (4 + case["rot"] * 4) + 2 * t * H * d * e, "flops": 3 * t * H * case["rot"]}
    n, kv = _lengths(case)
    c = SIZE[case["cache"]]
    if case["op"] == "append":  # q, k, v and the angles in; q, k and v out
        t = sum(n)
        return {"bytes": t * ((H + 2 * G) * d * e + case["rot"] * 4 + H * d * e + 2 * G * d * c),
                "flops": 3 * t * (H + G) * case["rot"]}
    w = case["window"]
    pairs = keys = 0
    for ni, ki in zip(n, kv):
        first = ki - ni
        if w and w < ki:
            pairs += sum(min(first + i + 1, w) for i in range(ni))
            keys += ki - max(0, first - w + 1)
        else:
            pairs += ni * first + ni * (ni + 1) // 2
            keys += ki
    return {"bytes": 2 * keys * G * d * c + 2 * sum(n) * H * d * e, "flops": 4 * pairs * H * d}


# ---------------------------------------------------------------- inputs

BASE = 1e6  # the rotation's base


def _frequencies(case):
    """The rotation's frequencies (each rounded to 32 bits) and the factor on its cosines and sines. Contexts are
    extended by 4 from a quarter of the positions: evenly (linear), or by wavelength (yarn: Peng et al., 2023)."""
    r, f = case["rot"], []
    factor, trained, fast, slow = 4.0, 8192, 32.0, 1.0

    def dim(turns):
        return r * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(BASE))

    low, high = max(math.floor(dim(fast)), 0), min(math.ceil(dim(slow)), r - 1)
    for i in range(r // 2):
        x = BASE ** (-2.0 * i / r)
        if case["scaling"] == "linear":
            x /= factor
        elif case["scaling"] == "yarn":
            ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            x = x / factor * ramp + x * (1 - ramp)
        f.append(x)
    amp = 0.1 * math.log(factor) + 1.0 if case["scaling"] == "yarn" else 1.0
    return torch.tensor(f, dtype=torch.float64).to(torch.float32), amp


def _table(case, n_pos):
    import kore_b200 as K
    more = {"none": {}, "linear": dict(factor=4.0), "yarn": dict(factor=4.0, original_ctx=8192)}[case["scaling"]]
    return K.RopeTable(n_pos, case["rot"], base=BASE, interleaved=case["interleaved"], scaling=case["scaling"], **more)


def _rows(g, n, heads, d, dtype, fused, extra=0):
    """[n][heads][d] of N(0, 1); fused: a part of wider rows, as a fused projection leaves it."""
    wide = torch.randn(n, (heads + extra) * d, device="cuda", generator=g).to(dtype)
    return wide[:, : heads * d].unflatten(1, (heads, d)) if fused else wide[:, : heads * d].contiguous().view(n, heads, d)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, G, d = HEADS[case["heads"]]
    dt = DTYPES[case["type"]]
    S = dict(case=case, H=H, G=G, d=d)
    if case["op"] == "rope":
        n = case["tokens"]
        S["x"] = _rows(g, n, H, d, dt, case["fused"], 2 * G)
        S["pos"] = (case["pos0"] + torch.arange(n, device="cuda")).to(torch.int32)
        S["out"] = torch.zeros(n, H, d, device="cuda", dtype=dt)
        S["freq"], S["amp"] = _frequencies(case)
        S["freq"] = S["freq"].cuda()
        if own:
            S["table"] = _table(case, case["pos0"] + n)
        return S
    ns, kvs = _lengths(case)
    tokens, pad, P = sum(ns), (3 if case["ragged"] else 0), case["page"]
    rows = tokens + pad  # rows behind the last sequence, as a padded batch has them
    used = [-(-k // P) for k in kvs]
    total, widest = sum(used), max(used)
    where = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table, at = torch.full((len(ns), widest), -1, dtype=torch.int32), 0
    order = where.cpu()
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    starts = [0]
    for x in ns:
        starts.append(starts[-1] + x)
    S.update(table_=table.cuda(), q_start=torch.tensor(starts, dtype=torch.int32).cuda(), max_q=max(ns), max_kv=max(kvs),
             kv_len=torch.tensor(kvs, dtype=torch.int32).cuda(), tokens=tokens, ns=ns, kvs=kvs)
    cd = DTYPES[case["cache"]]
    shape = (total, G, P, d)
    S["ks"] = S["vs"] = None
    if case["cache"] == "e4m3":  # a value is its 8 bits times its head's scale
        S["ks"] = 0.02 * (1 + torch.rand(G, device="cuda", generator=g))
        S["vs"] = 0.01 * (1 + torch.rand(G, device="cuda", generator=g))

    def filled(scale):
        x = torch.randn(shape, device="cuda", generator=g)
        return (x / scale[:, None, None] if scale is not None else x).to(cd)

    S["kp"], S["vp"] = filled(S["ks"]), filled(S["vs"])
    if case["op"] == "append":
        if case["fused"]:
            qkv = torch.randn(rows, (H + 2 * G) * d, device="cuda", generator=g).to(dt)
            S["q"], S["k"], S["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([H * d, G * d, G * d], 1))
        else:
            S["q"], S["k"], S["v"] = (_rows(g, rows, h, d, dt, False) for h in (H, G, G))
        S["q_out"] = torch.zeros(rows, H, d, device="cuda", dtype=dt)
        S["freq"], S["amp"] = _frequencies(case)
        S["freq"] = S["freq"].cuda()
        if own:
            S["table"] = _table(case, max(kvs))
    else:
        S["q"] = _rows(g, rows, H, d, dt, case["fused"], 2 * G)
        S["out"] = torch.zeros(rows, H, d, device="cuda", dtype=dt)
    if own:
        import kore_b200 as K
        S["cache"] = K.PagedCache(S["kp"], S["vp"], k_scale=S["ks"], v_scale=S["vs"])
        S["batch"] = K.PagedBatch(S["q_start"], S["kv_len"], S["table_"], max_q=S["max_q"])
    return S


# ---------------------------------------------------------------- the plain form

def _rotate(x, pos, freq, amp, interleaved):
    """x [n][heads][d] in 32 bits, the angles in 64."""
    a = pos.double()[:, None] * freq.double()
    c, s = (a.cos() * amp).float()[:, None], (a.sin() * amp).float()[:, None]
    x, r = x.float(), 2 * freq.numel()
    y = x.clone()
    if interleaved:
        x0, x1 = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = x0 * c - x1 * s, x0 * s + x1 * c
    else:
        x0, x1 = x[..., : r // 2], x[..., r // 2: r]
        y[..., : r // 2], y[..., r // 2: r] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def _owners(S):
    """Each token's sequence and position."""
    t = torch.arange(S["tokens"], device="cuda")
    s = torch.searchsorted(S["q_start"][1:].long(), t, right=True)
    return s, S["kv_len"].long()[s] - S["q_start"].long()[s + 1] + t


def _store(pages, page, g, slot, x, scale):
    if scale is not None:
        x = (x / scale[None, :, None]).clamp(-448.0, 448.0)
    pages[page[:, None], g, slot[:, None]] = x.to(pages.dtype)


def _plain_append(S):
    n, P = S["tokens"], S["case"]["page"]
    seq, pos = _owners(S)
    page, slot = S["table_"][seq, pos // P].long(), pos % P
    heads = torch.arange(S["G"], device="cuda")[None]
    rot = (S["freq"], S["amp"], S["case"]["interleaved"])
    _store(S["kp"], page, heads, slot, _rotate(S["k"][:n], pos, *rot), S["ks"])
    _store(S["vp"], page, heads, slot, S["v"][:n].float(), S["vs"])
    S["q_out"][:n] = _rotate(S["q"][:n], pos, *rot).to(S["q_out"].dtype)
    return S["kp"], S["vp"], S["q_out"]


def _plain_attend(S):
    case, H, G, d, P = S["case"], S["H"], S["G"], S["d"], S["case"]["page"]
    L, N, B = S["max_kv"], S["max_q"], len(S["ns"])

    def gather(pages, scale):  # [B][G][L][d], zero past each sequence's end
        x = pages[S["table_"].long().clamp(min=0)].float()  # [B][pages][G][P][d]
        x = x.transpose(1, 2).flatten(2, 3)[:, :, :L]
        x = x * scale[None, :, None, None] if scale is not None else x
        return torch.where((torch.arange(L, device="cuda") < S["kv_len"][:, None])[:, None, :, None], x, 0.0)

    k, v = gather(S["kp"], S["ks"]), gather(S["vp"], S["vs"])
    i = torch.arange(N, device="cuda")
    n = (S["q_start"][1:] - S["q_start"][:-1]).long()
    here = i < n[:, None]  # [B][N]
    tok = torch.where(here, S["q_start"][:-1].long()[:, None] + i, 0)
    q = S["q"][tok].float().unflatten(2, (G, H // G))  # [B][N][G][H/G][d]
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B][G][H/G * N][d]
    s = (q @ k.transpose(2, 3)).unflatten(2, (H // G, N)) / math.sqrt(d)  # [B][G][H/G][N][L]
    pos = (S["kv_len"].long() - n)[:, None] + i
    t = torch.arange(L, device="cuda")
    seen = t <= pos[..., None]
    if case["window"]:
        seen &= t > pos[..., None] - case["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    out = (s.flatten(2, 3) @ v) / s.sum(-1).flatten(2, 3)[..., None]
    out = out.unflatten(2, (H // G, N)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B][N][H][d]
    S["out"][tok[here]] = out[here].to(S["out"].dtype)
    return S["out"]


def run(state):
    S = state
    op = S["case"]["op"]
    if own:
        if op == "rope":
            S["table"].rotate(S["x"], S["pos"], out=S["out"])
            return S["out"]
        if op == "append":
            S["cache"].append(S["batch"], S["k"], S["v"], rope=S["table"], q=S["q"], q_out=S["q_out"])
            return S["kp"], S["vp"], S["q_out"]
        S["cache"].attend(S["batch"], S["q"], S["out"], window=S["case"]["window"])
        return S["out"]
    if op == "rope":
        S["out"].copy_(_rotate(S["x"], S["pos"], S["freq"], S["amp"], S["case"]["interleaved"]))
        return S["out"]
    return _plain_append(S) if op == "append" else _plain_attend(S)


# ---------------------------------------------------------------- the definition, in 64 bits

def _turned(x, first, S):
    """Rows first, first + 1, ... of one sequence as complex numbers times e^(i angle)."""
    r, x = S["case"]["rot"], x.double()
    p = torch.arange(first, first + x.shape[0], device="cuda", dtype=torch.float64)
    angle = torch.outer(p, S["freq"].double())
    turn = torch.polar(torch.full_like(angle, S["amp"]), angle)[:, None]
    if S["case"]["interleaved"]:
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


def exact(case, seed):
    S = prepare(case, seed)
    H, G, d = S["H"], S["G"], S["d"]
    if case["op"] == "rope":
        return _turned(S["x"], case["pos0"], S)
    P, at = case["page"], 0
    table = S["table_"].long()
    if case["op"] == "append":
        kp, vp, qo = S["kp"].double(), S["vp"].double(), S["q_out"].double()
        for s, (n, kv) in enumerate(zip(S["ns"], S["kvs"])):
            here = slice(at, at + n)
            p = torch.arange(kv - n, kv, device="cuda")
            k, v = _turned(S["k"][here], kv - n, S), S["v"][here].double()
            if S["ks"] is not None:
                k, v = (_eight_bits(x / c.double()[:, None]) for x, c in ((k, S["ks"]), (v, S["vs"])))
            kp[table[s, p // P], :, p % P] = k
            vp[table[s, p // P], :, p % P] = v
            qo[here] = _turned(S["q"][here], kv - n, S)
            at += n
        return kp, vp, qo
    out = S["out"].double()
    for s, (n, kv) in enumerate(zip(S["ns"], S["kvs"])):
        t = torch.arange(kv, device="cuda")
        k, v = (x[table[s, t // P], :, t % P].double() for x in (S["kp"], S["vp"]))  # [kv][G][d]
        if S["ks"] is not None:
            k, v = k * S["ks"].double()[:, None], v * S["vs"].double()[:, None]
        first = kv - n
        for a in range(0, n, 256):  # some queries at a time
            b = min(n, a + 256)
            p = torch.arange(first + a, first + b, device="cuda")[:, None]
            seen = t <= p
            if case["window"]:
                seen &= t > p - case["window"]
            for h in range(H):
                score = S["q"][at + a: at + b, h].double() @ k[:, h // (H // G)].T * d ** -0.5
                out[at + a: at + b, h] = score.masked_fill(~seen, -math.inf).softmax(-1) @ v[:, h // (H // G)]
        at += n
    return out
