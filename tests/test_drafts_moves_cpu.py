"""Stores into and moves in a cache whose keys and values share memory, and the acceptance of a step with masks, as far as
no GPU is needed. CPU only."""
import random
from types import SimpleNamespace

import pytest

from kore_b200 import drafts
from kore_b200 import paged as P
from tests.test_drafts_cpu import _commit, _norm, _Pool, _store, err
from tests.test_paged_cpu import A, B, _batch, _pages, _ref, _rows

PAGE = 4096   # 2 heads of 16 tokens of 64 values of 2 bytes


@pytest.mark.parametrize("apart,stride,overlap", [(16, 0, True), (PAGE, 0, True), (3 * PAGE, 0, True), (4 * PAGE, 0, False),
                                                  (4 * PAGE - 16, 0, True), (-4 * PAGE + 16, 0, True), (-4 * PAGE, 0, False),
                                                  (PAGE, 2 * PAGE, False), (PAGE + 16, 2 * PAGE, True), (-PAGE, 2 * PAGE, False),
                                                  (6 * PAGE, 2 * PAGE, True), (7 * PAGE + 16, 2 * PAGE, False)])
def test_keys_that_overlap_the_values_are_refused(apart, stride, overlap):
    """Two threads would move the shared rows, the second from where the first has written."""
    k, v = 16 * A, 16 * A + apart
    spans = [[range(x + i * (stride or PAGE), x + i * (stride or PAGE) + PAGE) for i in range(4)] for x in (k, v)]
    assert overlap == any(max(a.start, b.start) < min(a.stop, b.stop) for a in spans[0] for b in spans[1])
    layers = (P._Pages * 2)(_pages(k=A), _pages(k=k, v=v, page_stride=stride // 2))
    layers[0].page_stride, layers[0].v = stride // 2, A + 64 * PAGE   # (of the same geometry, apart)
    rc, msg = _commit(layers, 2)
    assert (rc == -1 and "layer 1: the keys' pages overlap" in msg) == overlap, msg
    pool = _Pool(k, v, n_pages=4, page_stride=stride // 2)
    if overlap:
        with pytest.raises(ValueError, match="cache 0: the keys' pages overlap"):
            drafts._check_own([pool])
    else:
        drafts._check_own([pool])


def test_keys_and_values_in_one_memory_are_no_overlap():
    """Their rows are moved once."""
    for check in (drafts._check_apart, drafts._check_own):
        check([_Pool(A, A), _Pool(16 * A, 16 * A)])
    with pytest.raises(ValueError, match="caches 0 and 1 share pages"):
        drafts._check_apart([_Pool(A, A), _Pool(A, A)])
    rc, msg = _commit()
    assert "overlap" not in msg


@pytest.mark.parametrize("cache,k,v,rope,norm,refused", [
    (dict(), {}, {}, False, None, False), (dict(), {}, dict(data=B), False, None, True),
    (dict(), {}, dict(ts=256), False, None, True), (dict(), {}, {}, True, None, True),
    (dict(), {}, {}, False, dict(k_weight=None), False), (dict(), {}, {}, False, dict(), True),
    (dict(v=A + PAGE), {}, {}, False, None, True), (dict(v=A + 4 * PAGE), {}, dict(data=B), True, dict(), False),
    (dict(v=A + PAGE, page_stride=PAGE), {}, dict(data=B), True, None, False)])
def test_different_rows_into_one_memory_are_refused(cache, k, v, rope, norm, refused):
    """Which of them stayed would be chance."""
    pages, k, v = _pages(**cache), _rows(**k), _rows(**v)
    rope = P._RopeView(A, 8, 64, 0) if rope else None
    calls = [_store(cache=pages, k=k, v=v, rope=rope, norm=None if norm is None else _norm(**norm))]
    if norm is None:
        calls.append(err(P._library().kore_cuda_paged_append_dev(
            _ref(pages), _ref(_batch()), 1, _ref(k), _ref(v), None, None, _ref(rope), None, None)))
    for rc, msg in calls:
        assert (rc == -1 and "share memory" in msg) == refused, msg


@pytest.mark.parametrize("words", [-1, 0, 33])
def test_an_acceptance_with_masks_of_no_size_is_refused(words):
    out = P._Accepted(A, 4, A, A, A)
    call = P._library().kore_cuda_tree_accept_masked_dev
    rc, msg = err(call(_ref(_batch()), 1, words, A, A, A, _ref(out), None, None))
    assert rc == -1 and "words" in msg
    assert err(call(_ref(_batch()), 1, 1, None, A, A, _ref(out), None, None))[0] == -1
    assert call(_ref(_batch(n_seq=0)), 1, 32, A, A, A, _ref(out), None, None) == 0


def test_only_kernels_that_there_are_can_be_set():
    L = P._library()
    for x in (-1, 3, 1 << 30):
        assert L.kore_cuda_paged_set_tree_kernel(x) == -1
    with pytest.raises(ValueError, match="kernel"):
        P.set_tree_kernel("other")
    P.set_tree_kernel("auto")


def test_pools_are_compared_with_those_in_reach():
    """Against every page of every pair, for pools one behind the other, between one another's pages, and anywhere."""
    r = random.Random(0)
    for turn in range(400):
        n_pages, stride = r.choice([1, 2, 3, 8]), r.choice([PAGE, PAGE, 2 * PAGE, 6 * PAGE, 5 * PAGE + 16])
        where = r.choice([lambda: r.randrange(40) * stride * n_pages, lambda: r.randrange(60) * PAGE, lambda: r.randrange(9000) * 16,
                          lambda: r.randrange(4) * 50 * stride + r.randrange(6) * PAGE])
        pools = [_Pool(A + where(), A + where(), n_pages, stride // 2) for _ in range(r.choice([2, 2, 3, 5]))]
        if n_pages == 1 and turn % 2:
            for p in pools:
                p.view.page_stride = 0   # (as a cache of one page has it)
        pages = [[x + i * stride for x in {c.view.k, c.view.v} for i in range(n_pages)] for c in pools]
        shared = any(abs(x - y) < PAGE for i, a in enumerate(pages) for b in pages[i + 1:] for x in a for y in b)
        own = any(c.view.k != c.view.v and abs(c.view.k - c.view.v + (i - j) * stride) < PAGE
                  for c in pools for i in range(n_pages) for j in range(n_pages))
        for check, want, word in ((drafts._check_apart, shared, "share pages"), (drafts._check_own, own, "overlap")):
            if want:
                with pytest.raises(ValueError, match=word):
                    check(pools)
            else:
                check(pools)


def test_many_layers_are_compared_in_linear_time():
    """Layers that follow one another are compared with their neighbours only (128 took 10 ms of all pairs)."""
    seen = 0

    class Counted(int):
        def __sub__(self, other):
            nonlocal seen
            seen += 1
            return int(self) - int(other)

    pools = [SimpleNamespace(view=SimpleNamespace(k=Counted(2 * i << 20), v=Counted(2 * i + 1 << 20), n_pages=8, page_stride=0,
                                                  n_head_kv=2, page_tokens=16, head_dim=64),
                             k=SimpleNamespace(element_size=lambda: 2)) for i in range(500)]
    drafts._check_apart(pools)
    assert 0 < seen <= 1000
