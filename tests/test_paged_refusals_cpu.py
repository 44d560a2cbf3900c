"""Calls of the operators on a caller-owned paged cache that are refused before anything reaches a GPU, on tensors
that have a device, shape and strides and no memory (torch's fake tensors). CPU only."""
import ctypes
import random
import sys
import threading

import pytest

import kore_b200 as K
from kore_b200 import paged as P

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

A, B = 0x10000, 0x20000   # placeholders for aligned device addresses
pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer")


@pytest.fixture
def fake():
    with FakeTensorMode() as mode:
        yield mode


def cuda(*shape, dtype=torch.bfloat16, device="cuda:0"):
    return torch.empty(*shape, dtype=dtype, device=device)


def test_pages_that_overlap_are_refused(fake):
    """A page expanded over the pool has a stride of 0, which the C entry points take as dense pages."""
    one = cuda(1, 2, 16, 64)
    with pytest.raises(ValueError, match="overlap"):
        K.PagedCache(one.expand(4, 2, 16, 64), one.expand(4, 2, 16, 64))
    rows = cuda(5 * 2 * 16 * 64)
    near = rows.as_strided((4, 2, 16, 64), (2 * 16 * 64 - 16, 16 * 64, 64, 1))
    with pytest.raises(ValueError, match="overlap"):
        K.PagedCache(near, near)
    for ok in (one, cuda(4, 2, 16, 64), cuda(4, 2, 2, 16, 64)[:, 0], one.expand(1, 2, 16, 64)):
        K.PagedCache(ok, ok)


def step(n=1, device="cuda:0"):
    """A cache, a batch of one sequence and its queries."""
    pages = cuda(4, 2, 16, 64, device=device)
    ints = [cuda(*s, dtype=torch.int32, device=device) for s in ((2,), (1,), (1, 4))]
    return K.PagedCache(pages, pages), K.PagedBatch(*ints, max_q=1), cuda(n, 4, 64, device=device)


@pytest.mark.parametrize("workspace", [dict(device="cpu"), dict(device="cuda:1"), dict(dtype=torch.float32), dict(step=2)])
def test_workspaces_that_the_kernels_cannot_use_are_refused(fake, workspace):
    cache, batch, q = step()
    skip = workspace.pop("step", 1)
    ws = cuda(1 << 27, **{"dtype": torch.uint8, **workspace})[::skip]
    with pytest.raises(ValueError, match="workspace"):
        cache.attend(batch, q, cuda(1, 4, 64), workspace=ws)


@pytest.mark.parametrize("kw", [dict(window=2 ** 32), dict(window=2 ** 32 + 5), dict(window=2 ** 31), dict(scale=1e-50),
                                dict(scale=-1e-46)])
def test_options_outside_32_bits_are_refused(fake, kw):
    """Cut to 32 bits they would be other options: a window of 5, or none, or the default scale."""
    cache, batch, q = step()
    with pytest.raises(ValueError, match="32 bits"):
        cache.attend(batch, q, cuda(1, 4, 64), **kw)


@pytest.mark.parametrize("kw", [dict(max_q=2 ** 32 + 1), dict(max_q=1, max_kv=2 ** 31), dict(max_q=-2 ** 32)])
def test_hints_outside_32_bits_are_refused(fake, kw):
    with pytest.raises(ValueError, match="32 bits"):
        K.PagedBatch(cuda(2, dtype=torch.int32), cuda(1, dtype=torch.int32), cuda(1, 4, dtype=torch.int32), **kw)


def test_tables_outside_32_bits_are_refused(fake):
    for n_pos, n_rot in ((2 ** 32 + 4, 8), (2 ** 31, 8), (16, 2 ** 32 + 8)):
        with pytest.raises(ValueError, match="32 bits"):
            K.RopeTable(n_pos, n_rot, device="cuda:0")
    with pytest.raises(ValueError, match="32 bits"):
        K.rope_frequencies(2 ** 32 + 8)


def test_more_tokens_than_a_call_can_count_are_refused(fake):
    cache, batch, _ = step()
    rows = cuda(1, 2, 64).expand(2 ** 32 + 1, 2, 64)
    with pytest.raises(ValueError, match="too many"):
        cache.append(batch, rows, rows)


def test_written_rows_that_overlap_are_refused(fake):
    """An expanded tensor may be read, not written: which of its rows stays would be chance."""
    cache, batch, q = step(3)
    k = cuda(3, 2, 64)
    for out in (cuda(1, 4, 64).expand(3, 4, 64), cuda(3, 1, 64).expand(3, 4, 64)):
        for call in (lambda: P._library().kore_cuda_paged_attn_dev(*attention(cache, batch, q, out)),
                     lambda: P._library().kore_cuda_rope_dev(*rotation(q, out)),
                     lambda: P._library().kore_cuda_paged_append_dev(*appended(cache, batch, k, q, out))):
            assert call() == -1
            assert "overlap" in P._library().kore_cuda_last_error(None).decode()


def rows(t, address):
    h, d = t.shape[1:]
    return ctypes.byref(P._Rows(address, P.BF16, h, d, *t.stride()[:2]))


def view(struct, **places):
    """A copy of a structure with addresses in place of the fake tensors'."""
    new = type(struct)(*[places.get(name, getattr(struct, name)) for name, _ in struct._fields_])
    return ctypes.byref(new)


def attention(cache, batch, q, out):
    return (view(cache.view, k=A, v=A), view(batch.view, q_start=A, kv_len=A, page_table=A), q.shape[0], rows(q, A),
            rows(out, B), None, ctypes.byref(P._Opts(0.0, 1, 0)), A, 1 << 40, None, None)


def rotation(q, out):
    return rows(q, A), rows(out, B), q.shape[0], A, ctypes.byref(P._RopeView(A, 8, 8, 0)), None, None


def appended(cache, batch, k, q, out):
    return (view(cache.view, k=A, v=A), view(batch.view, q_start=A, kv_len=A, page_table=A), q.shape[0], rows(k, A),
            rows(k, A), rows(q, A), rows(out, B), None, None, None)


def test_default_workspaces_of_several_threads(monkeypatch):
    """Threads with objects and streams of their own share the table of default workspaces."""
    from types import SimpleNamespace as N
    monkeypatch.setattr(P, "_workspaces", {})
    monkeypatch.setattr(P, "_new_workspace", lambda L, device, d: object())
    monkeypatch.setattr(P, "_torch", N(_C=N(_cuda_getDevice=lambda: 0, _cuda_isCurrentStreamCapturing=lambda: True)))
    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    failed = []

    def work(seed):
        r = random.Random(seed)
        L = N(kore_cuda_capture_id=lambda stream: r.randrange(50))
        try:
            for _ in range(4000):
                assert P._workspace(L, N(index=0), r.randrange(20), 64) is not None
        except Exception as e:   # noqa: BLE001
            failed.append(repr(e))
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        sys.setswitchinterval(before)
    assert not failed
    assert len(P._workspaces) <= P._WORKSPACES_KEPT + 8
