"""Arrays of 32- and 64-bit values off their alignment are refused by every entry point of the paged operators: a kernel's
load of one would fault. CPU only; every other call is as one that a GPU would run."""
import pytest

from kore_b200 import paged as P
from tests.test_drafts_cpu import _norm, _pool, _step
from tests.test_paged_cpu import A, B, _batch, _pages, _ref, _rows

torch = pytest.importorskip("torch")
OFF = [1, 2, 3]


def call(name, *a):
    L = P._library()
    rc = getattr(L, name)(*a)
    return rc, L.kore_cuda_last_error(None).decode()


def plan(pool=None, request=A, n_new=A, step=None, status=A):
    return call("kore_cuda_paged_plan_dev", _ref(pool or _pool()), 1, request, n_new, _ref(step or _step()), status, None)


def trim(pool=None, request=A, keep=A, status=A):
    return call("kore_cuda_paged_trim_dev", _ref(pool or _pool()), 1, request, keep, status, None)


def store(cache=None, slots=A, pos=A, rope=None, status=A):
    return call("kore_cuda_paged_store_dev", _ref(cache or _pages(v=B)), 1, slots, pos, _ref(_rows()), _ref(_rows()), None, None,
                _ref(rope), _ref(_norm()), status, None)


def append(batch=None, cache=None, status=A):
    return call("kore_cuda_paged_append_dev", _ref(cache or _pages(v=B)), _ref(batch or _batch()), 1, _ref(_rows()), _ref(_rows()),
                None, None, None, status, None)


def masks(batch=None, parent=A, mask=A, pos=A, status=A):
    return call("kore_cuda_tree_masks_dev", _ref(batch or _batch()), 1, parent, mask, 1, pos, status, None)


def accept(batch=None, parent=A, token=A, choice=A, out=(A, A, A, A), status=A):
    out = P._Accepted(out[0], 4, *out[1:])
    return call("kore_cuda_tree_accept_dev", _ref(batch or _batch()), 1, parent, token, choice, _ref(out), status, None)


def accept_masked(batch=None, parent=A, token=A, choice=A, out=(A, A, A, A), status=A):
    out = P._Accepted(out[0], 4, *out[1:])
    return call("kore_cuda_tree_accept_masked_dev", _ref(batch or _batch()), 1, 1, parent, token, choice, _ref(out), status, None)


def commit(batch=None, cache=None, path=A, count=A, status=A):
    layers = (P._Pages * 1)(cache or _pages(v=B))
    return call("kore_cuda_paged_commit_dev", layers, 1, _ref(batch or _batch()), path, 4, count, status, None)


def attend(batch=None, cache=None, lse=A, mask=A, status=A):
    return call("kore_cuda_paged_tree_attn_dev", _ref(cache or _pages(v=B)), _ref(batch or _batch()), 1, _ref(_rows(4)),
                _ref(_rows(4, data=B)), lse, _ref(P._Opts(0.0, 1, 0)), _ref(P._Tree(mask, 1)), A, 1 << 40, status, None)


def attend_chunks(batch=None, cache=None, lse=A, status=A):
    return call("kore_cuda_paged_attn_dev", _ref(cache or _pages(v=B)), _ref(batch or _batch()), 1, _ref(_rows(4)),
                _ref(_rows(4, data=B)), lse, _ref(P._Opts(0.0, 1, 0)), A, 1 << 40, status, None)


def rotate(pos=A, status=A):
    return call("kore_cuda_rope_dev", _ref(_rows()), _ref(_rows()), 1, pos, _ref(P._RopeView(A, 8, 64, 0)), status, None)


POOL = [lambda x, f=f: dict(pool=_pool(**{f: x})) for f in ("free_pages", "n_free", "table", "length")]
BATCH = [lambda x, f=f: dict(batch=_batch(**{f: x})) for f in ("q_start", "kv_len", "page_table")]
SCALES = [lambda x, f=f: dict(cache=_pages(type=P.E4M3, v=B, **{f: x})) for f in ("k_scale", "v_scale")]
OUT = [lambda x, i=i: dict(out=tuple(x if j == i else A for j in range(4))) for i in range(4)]


def args(*names):
    return [lambda x, n=n: {n: x} for n in names]


EVERY = [(plan, POOL + args("request", "n_new", "status") + [lambda x, f=f: dict(step=_step(**{f: x}))
                                                              for f in ("q_start", "kv_len", "page_table", "slots", "pos")]),
         (trim, POOL + args("request", "keep", "status")), (store, args("slots", "pos", "status") + SCALES),
         (append, BATCH + args("status") + SCALES), (masks, BATCH[:2] + args("parent", "mask", "pos", "status")),
         (accept, BATCH[:2] + OUT + args("parent", "token", "choice", "status")),
         (accept_masked, BATCH[:2] + OUT + args("parent", "token", "choice", "status")),
         (commit, BATCH + args("path", "count", "status")), (attend, BATCH + args("lse", "mask", "status")),
         (attend_chunks, BATCH + args("lse", "status")), (rotate, args("pos", "status"))]


@pytest.mark.parametrize("f,which", [(f, w) for f, ws in EVERY for w in ws])
def test_arrays_off_their_alignment_are_refused(f, which):
    for off in OFF:
        rc, msg = f(**which(A + off))
        assert rc == -1 and "not aligned" in msg, msg
    _, msg = f(**which(A))
    assert "not aligned" not in msg   # (it goes on to the device)


def test_slots_are_of_64_bits():
    for rc, msg in (store(slots=A + 4), plan(step=_step(slots=A + 4))):
        assert rc == -1 and "not aligned" in msg


@pytest.mark.skipif(torch.cuda.is_available(), reason="with a device it is the addresses that are refused")
def test_the_calls_are_otherwise_complete():
    """Nothing but the device is missing."""
    for f, _ in EVERY:
        rc, msg = f()
        assert rc not in (0, -1, -2) and "CUDA device" in msg, (f.__name__, rc, msg)
