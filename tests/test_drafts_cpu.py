"""The operators of a step with drafted tokens, as far as no GPU is needed: calls that are refused before anything reaches
one (every check stands before the first CUDA call, so placeholder addresses do). CPU only."""
import ctypes
import math
from pathlib import Path
from types import SimpleNamespace

import pytest

import kore_b200 as K
from kore_b200 import drafts
from kore_b200 import paged as P
from tests.test_paged_cpu import BAD_PAGES, A, B, _batch, _pages, _ref, _rows
from tests.test_paged_refusals_cpu import cuda, fake  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer")


def err(rc):
    return rc, P._library().kore_cuda_last_error(None).decode()


def _pool(**kw):
    a = dict(free_pages=A, n_free=A, table=A, length=A, n_pages=8, page_tokens=16, n_requests=4, table_stride=4)
    a.update(kw)
    return P._Pool(*a.values())


def _step(**kw):
    a = dict(q_start=A, kv_len=A, page_table=A, table_stride=4, n_tok=9, slots=A, pos=A)
    a.update(kw)
    return P._Step(*a.values())


def _plan(pool=None, n=1, request=A, n_new=A, step=...):
    step = _step() if step is ... else step
    return err(P._library().kore_cuda_paged_plan_dev(_ref(pool or _pool()), n, request, n_new, _ref(step), None, None))


def _trim(pool=None, n=1, request=A, keep=A):
    return err(P._library().kore_cuda_paged_trim_dev(_ref(pool or _pool()), n, request, keep, None, None))


@pytest.mark.parametrize("kw,word,code", [
    (dict(free_pages=None), "null", -1), (dict(n_free=None), "null", -1), (dict(table=None), "null", -1),
    (dict(length=None), "null", -1), (dict(n_pages=0), "n_pages", -1), (dict(page_tokens=24), "page_tokens", -1),
    (dict(page_tokens=0), "page_tokens", -1), (dict(n_requests=0), "n_requests", -2),
    (dict(n_requests=65537), "n_requests", -2), (dict(table_stride=0), "table_stride", -1)])
def test_bad_pools_refused(kw, word, code):
    for rc, msg in (_plan(pool=_pool(**kw)), _trim(pool=_pool(**kw))):
        assert rc == code and word in msg, msg


def test_bad_plans_and_trims_refused():
    for call in (_plan, _trim):
        assert call(n=-1)[0] == -2 and call(n=4097)[0] == -2 and call(request=None)[0] == -1
    assert _plan(n_new=None)[0] == -1 and _trim(keep=None)[0] == -1 and _plan(step=None)[0] == -1
    for kw in (dict(q_start=None), dict(kv_len=None), dict(page_table=None), dict(table_stride=3), dict(n_tok=-1),
               dict(slots=None), dict(pos=None), dict(slots=A + 4), dict(pos=A + 2)):
        assert _plan(step=_step(**kw))[0] == -1
    assert _trim(n=0)[0] == 0


def _norm(**kw):
    a = dict(q_weight=A, k_weight=A, type=P.BF16, q_head_stride=0, k_head_stride=0, eps=1e-6)
    a.update(kw)
    return P._Norm(*a.values())


def _store(cache=None, n=1, slots=A, pos=A, k=..., v=..., q=None, q_out=None, rope=None, norm=None):
    k, v = _rows() if k is ... else k, _rows() if v is ... else v
    return err(P._library().kore_cuda_paged_store_dev(_ref(cache or _pages()), n, slots, pos, _ref(k), _ref(v), _ref(q),
                                                      _ref(q_out), _ref(rope), _ref(norm), None, None))


@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_bad_pages_refused(kw, word):
    layers = (P._Pages * 2)(_pages(), _pages(**kw))
    for rc, msg in (_store(cache=_pages(**kw)), _commit(layers, 2)):
        assert rc == -1 and word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(n=-1), "n_tok"), (dict(slots=None), "slots"), (dict(slots=A + 4), "aligned"), (dict(pos=A + 2), "aligned"), (dict(k=None), "k is null"), (dict(v=_rows(data=None)), "v is null"),
    (dict(k=_rows(3)), "heads"), (dict(v=_rows(type=P.F16)), "different types"), (dict(q=_rows(4)), "together"),
    (dict(q=_rows(4), q_out=_rows(5)), "heads"), (dict(q=_rows(4), q_out=_rows(4, ts=0), n=2), "overlap"),
    (dict(k=_rows(type=P.F16), v=_rows(type=P.F16)), "do not go"),
    (dict(rope=P._RopeView(A, 8, 66, 0)), "n_rot"), (dict(rope=P._RopeView(A, 8, 8, 0), pos=None), "positions"),
    (dict(norm=_norm(type=P.E4M3)), "type"), (dict(norm=_norm(q_weight=None, k_weight=None)), "no weights"),
    (dict(norm=_norm(k_weight=A + 1)), "aligned"), (dict(norm=_norm(eps=0.0)), "eps"), (dict(norm=_norm(eps=-1.0)), "eps"),
    (dict(norm=_norm(eps=math.inf)), "eps"), (dict(norm=_norm(eps=math.nan)), "eps")])
def test_store_refused(kw, word):
    rc, msg = _store(**kw)
    assert rc == -1 and word in msg, msg


def _masks(batch=None, n=1, parent=A, mask=A, words=1, pos=A):
    return err(P._library().kore_cuda_tree_masks_dev(_ref(batch or _batch()), n, parent, mask, words, pos, None, None))


def _accept(batch=None, n=1, parent=A, token=A, choice=A, out=...):
    out = P._Accepted(A, 4, A, A, A) if out is ... else out
    return err(P._library().kore_cuda_tree_accept_dev(_ref(batch or _batch()), n, parent, token, choice, _ref(out), None, None))


def _commit(layers=None, n=1, batch=None, path=A, stride=4, count=A):
    layers = (P._Pages * 1)(_pages()) if layers is None else layers
    return err(P._library().kore_cuda_paged_commit_dev(layers, n, _ref(batch or _batch()), path, stride, count, None, None))


@pytest.mark.parametrize("kw,code", [(dict(n_seq=-1), -2), (dict(n_seq=4097), -2), (dict(q_start=None), -1),
                                     (dict(kv_len=None), -1)])
def test_bad_batches_refused(kw, code):
    for call in (_masks, _accept, _commit):
        assert call(batch=_batch(**kw))[0] == code


def test_bad_trees_refused():
    for kw in (dict(n=-1), dict(parent=None), dict(mask=None), dict(mask=A + 2), dict(words=0), dict(words=33), dict(pos=None)):
        assert _masks(**kw)[0] == -1
    for kw in (dict(n=-1), dict(parent=None), dict(token=None), dict(choice=None), dict(out=None),
               dict(out=P._Accepted(None, 4, A, A, A)), dict(out=P._Accepted(A, 0, A, A, A)),
               dict(out=P._Accepted(A, 1025, A, A, A)), dict(out=P._Accepted(A, 4, None, A, A)),
               dict(out=P._Accepted(A, 4, A, None, A)), dict(out=P._Accepted(A, 4, A, A, None))):
        assert _accept(**kw)[0] == -1
    for kw in (dict(n=-1), dict(path=None), dict(count=None), dict(stride=0), dict(stride=1025),
               dict(batch=_batch(page_table=None)), dict(batch=_batch(table_stride=0))):
        assert _commit(**kw)[0] == -1
    assert _commit(None, 1, batch=_batch(page_table=None))[0] == -1
    for other in (dict(type=P.F16), dict(n_pages=5), dict(page_tokens=32), dict(n_head_kv=1), dict(head_dim=32),
                  dict(page_stride=4096)):
        rc, msg = _commit((P._Pages * 2)(_pages(), _pages(**other)), 2)
        assert rc == -1 and "layer 1" in msg
    assert _masks(n=0)[0] == 0 and _accept(batch=_batch(n_seq=0))[0] == 0 and _commit(n=0)[0] == 0
    assert all(c[0] == -2 for c in (_store(n=(1 << 30) + 1), _plan(step=_step(n_tok=(1 << 30) + 1))))


def test_a_layer_named_twice_is_refused():
    """Its rows would be moved by two threads at once, the second time from where the first has written."""
    far = [dict(k=B + 4096 * i, v=B + 4096 * i + 2048) for i in range(300)]
    for same in (far[7], dict(k=far[7]["v"], v=B - 4096), dict(k=B - 4096, v=far[299]["k"])):
        layers = (P._Pages * 301)(*[_pages(**x) for x in far + [same]])
        rc, msg = _commit(layers, 301)
        assert rc == -1 and "and 300 have the same pages" in msg
        assert _commit(layers, 300, batch=_batch(n_seq=0))[0] == 0


class _Pool:
    """What PagedLayers looks at of a cache; pages of 2 heads of 16 tokens of 64 values of 2 bytes: 4096 bytes."""

    def __init__(self, k, v, n_pages=8, page_stride=0):
        self.view = P._Pages(k, v, P.BF16, n_pages, 16, 2, 64, page_stride, None, None)
        self.k = SimpleNamespace(element_size=lambda: 2)


@pytest.mark.parametrize("other,page_stride,shared", [
    ((A, B), 0, True), ((A + (1 << 20), A), 0, True), ((A + 4096 * 7, B + (1 << 20)), 0, True),
    ((A + 4096 * 8, B + 4096 * 8), 0, False), ((A + 4096 * 8 - 16, B + 4096 * 8), 0, True), ((A - 4096 * 8, B - 4096 * 8), 0, False),
    ((A - 4096 * 8 + 16, B - 4096 * 8), 0, True), ((A + 4096, B + 4096), 8192, False), ((A + 2048, B + 4096), 8192, True),
    ((A + 8192 + 4096, B + 4096), 8192, False), ((A + 8192 + 4112, B + 4096), 8192, True),
    ((A + 8192 * 7 + 4112, B + (1 << 20)), 8192, True),    # (the first page of the values follows the last of the keys)
    ((A + 8192 * 7 + 4096, B + (1 << 20)), 8192, False)])
def test_caches_that_share_pages_are_refused(other, page_stride, shared):
    """Against the pages one by one."""
    pools = [_Pool(A, B, page_stride=page_stride // 2), _Pool(*other, page_stride=page_stride // 2)]
    page, stride = 4096, page_stride or 4096
    spans = [[range(a + i * stride, a + i * stride + page) for a in (c.view.k, c.view.v) for i in range(8)] for c in pools]
    assert shared == any(max(x.start, y.start) < min(x.stop, y.stop) for x in spans[0] for y in spans[1])
    if shared:
        with pytest.raises(ValueError, match="share"):
            drafts._check_apart(pools)
    else:
        drafts._check_apart(pools)
    assert _commit(batch=_batch(n_seq=0))[0] == 0


def _attend(tree=..., opts=..., n=1):
    L = P._library()
    tree = P._Tree(A, 1) if tree is ... else tree
    opts = P._Opts(0.0, 1, 0) if opts is ... else opts
    q, out = _rows(4), _rows(4, data=B)
    return err(L.kore_cuda_paged_tree_attn_dev(_ref(_pages()), _ref(_batch()), n, _ref(q), _ref(out), None, _ref(opts),
                                               _ref(tree), A, 1 << 40, None, None))


@pytest.mark.parametrize("kw,word", [
    (dict(tree=None), "null"), (dict(tree=P._Tree(None, 1)), "null"), (dict(tree=P._Tree(A + 1, 1)), "aligned"),
    (dict(tree=P._Tree(A, 0)), "words"), (dict(tree=P._Tree(A, 33)), "words"), (dict(opts=None), "opts"),
    (dict(opts=P._Opts(0.0, 0, 0)), "masks"), (dict(opts=P._Opts(0.0, 1, 5)), "masks")])
def test_tree_attention_refused(kw, word):
    rc, msg = _attend(**kw)
    assert rc == -1 and word in msg, msg
    assert _attend(n=0)[0] == 0


def test_structures_are_the_headers():
    """Sizes and offsets as the C compiler lays them out (64-bit pointers first, no holes but before a long long)."""
    assert [ctypes.sizeof(x) for x in (P._Pool, P._Step, P._Norm, P._Tree, P._Accepted)] == [48, 48, 48, 16, 40]


def test_python_objects_refuse_what_does_not_fit(fake):  # noqa: F811
    for kw in (dict(n_pages=0), dict(page_tokens=24), dict(n_requests=65537), dict(table_width=0), dict(n_pages=2 ** 31)):
        with pytest.raises(ValueError):
            K.PagePool(**{**dict(n_pages=8, page_tokens=16, n_requests=4, table_width=4), **kw}, device="cuda:0")
    with pytest.raises(ValueError, match="CUDA"):
        K.TokenTree(4, 4, device="cpu")
    pool = K.PagePool(8, 16, 4, 4, device="cuda:0")
    for a in ((4097, 1, 1), (1, -1, 1), (-1, 1, 1), (1, 2 ** 31, 1)):
        with pytest.raises(ValueError):
            pool.new_step(*a)
    step = pool.new_step(2, 9, 5)
    i32 = lambda n, device="cuda:0": cuda(n, dtype=torch.int32, device=device)   # noqa: E731
    for a in ((i32(3), i32(3)), (i32(2), i32(1)), (cuda(2, dtype=torch.int64), i32(2)), (i32(2, "cuda:1"), i32(2)),
              (i32(4)[::2], i32(2))):
        with pytest.raises(ValueError):
            pool.plan(step, *a)
    narrow = K.PagePool(8, 16, 4, 9, device="cuda:0")
    with pytest.raises(ValueError, match="narrower"):
        narrow.plan(step, i32(2), i32(2))
    with pytest.raises(ValueError):
        pool.trim(i32(2), i32(3))
    for n, most in ((4, 1025), (4, 0), (-1, 4)):
        with pytest.raises(ValueError):
            K.TokenTree(n, most, device="cuda:0")
    tree = K.TokenTree(9, 5, device="cuda:0")
    for parent in (i32(8), cuda(9, dtype=torch.int64), i32(9, "cuda:1")):
        with pytest.raises(ValueError):
            tree.build(step, parent)
    for n, most in ((4097, 4), (4, 1025), (4, 0)):
        with pytest.raises(ValueError):
            K.AcceptedPath(n, most, device="cuda:0")
    path = K.AcceptedPath(3, 4, device="cuda:0")
    with pytest.raises(ValueError, match="sequences"):
        path.accept(step, i32(9), i32(9), i32(9))
    with pytest.raises(ValueError):
        path.accept(step, i32(9), i32(8), i32(9))
    cache = K.PagedCache(cuda(8, 2, 16, 64), cuda(8, 2, 16, 64))
    other = K.PagedCache(*(cuda(8, 2, 16, 64, device="cuda:1") for _ in range(2)))
    with pytest.raises(ValueError):
        K.PagedLayers([])
    with pytest.raises(ValueError, match="devices"):
        K.PagedLayers([cache, other])
    with pytest.raises(ValueError, match="sequences"):
        K.PagedLayers([cache]).commit(step, path)
    k, q = cuda(9, 2, 64), cuda(9, 4, 64)
    slots = cuda(9, dtype=torch.int64)
    norm = K.HeadNorm(cuda(4, 64), cuda(64))
    for a, kw in (((i32(9), None, k, k), {}), ((slots[:8], None, k, k), {}), ((slots, None, k, k[:8]), {}),
                  ((slots, None, k, k), dict(q=q)), ((slots, None, k, k), dict(norm=norm, q=k, q_out=k)),
                  ((slots, None, k, k), dict(rope=SimpleNamespace(device=torch.device("cuda:1")))),
                  ((slots, None, k, k), dict(norm=K.HeadNorm(cuda(32)), q=q, q_out=q))):
        with pytest.raises(ValueError):
            cache.store(*a, **kw)
    for a, kw in (((), {}), ((torch.empty(64),), {}), ((cuda(64, 2)[:, 0],), {}), ((cuda(64, dtype=torch.int32),), {}),
                  ((cuda(64), cuda(64, dtype=torch.float16)), {}), ((cuda(64), cuda(64, device="cuda:1")), {}),
                  ((cuda(64),), dict(eps=0.0)), ((cuda(64),), dict(eps=1e-60)), ((cuda(64),), dict(eps=math.inf))):
        with pytest.raises(ValueError):
            K.HeadNorm(*a, **kw)
    for kw in (dict(tree=tree), dict(tree=K.TokenTree(8, 5, device="cuda:1"))):
        with pytest.raises(ValueError, match="tree"):
            cache.attend(step, q[:8], cuda(8, 4, 64), **kw)


def test_products_and_their_commits_are_one_threads():
    """As tests/test_paged_sources_cpu.py says of the chunks' kernel: a commit follows the operations that its own thread
    issued, so every product and every commit of the trees' stands under elect()."""
    import os
    import re
    from kore_b200.build import CSRC
    with open(os.path.join(CSRC, "paged_tree_tiles.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    calls = [m.start() for m in re.finditer(r"\b(?:commit|mma_ss<[^>]*>|mma_ts<[^>]*>)\(", text)]
    assert len(calls) >= 9
    covered = []
    for g in re.finditer(r"if \(elect\(\)\)\s*", text):
        if text[g.end()] != "{":
            covered.append((g.end(), text.index(";", g.end())))
            continue
        depth, end = 0, g.end()
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            if depth == 0:
                break
            end += 1
        covered.append((g.end(), end))
    assert all(any(a <= c < b for a, b in covered) for c in calls)


def test_tensor_memory_is_taken_between_the_wait_and_the_trigger():
    """A CTA that holds tensor memory and waits for the preceding kernel could stand in the way of its allocation; one
    that lets the following kernel in before it allocates, in its own."""
    src = (Path(__file__).parents[1] / "kore_b200" / "csrc" / "paged_tree_tiles.cu").read_text()
    at = [src.index(x) for x in ("grid_dep_wait();", "tcgen05.alloc", "relinquish_alloc_permit", "find_share<", "grid_dep_launch();")]
    assert at == sorted(at) and all(src.count(x) == 1 for x in ("grid_dep_wait();", "tcgen05.alloc", "grid_dep_launch();"))
