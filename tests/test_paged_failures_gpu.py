"""Waits inside the attention over a paged cache that run out, without a GPU fault: under a limit far below a copy's
latency (kore_cuda_paged_set_wait_limit) real copies land "too late". The kernel reports it, waits for its own copies and
products still in flight, frees its tensor memory and returns; the next call is right."""
import pytest

import kore_b200 as K
from kore_b200.paged import set_wait_limit
from tests.test_paged_gpu import BOTH, Cache, HINTS, check_attention, dev, gen, ints, rand, starts

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# one short unit, whose copies are all issued before the first is missed; and many, of several CTAs each
BATCHES = {"short": [(3, 90)], "long": [(2, 9000), (40, 700), (1, 3000)]}


@pytest.fixture
def impatient():
    set_wait_limit(1e-9)
    yield
    set_wait_limit(0)


def ready(tc, which, seed=1):
    g = gen(seed)
    ns, kvs = map(list, zip(*BATCHES[which]))
    C = Cache(g, tc, 2, 128, 64, kvs)
    for s in range(len(kvs)):
        C.fill(g, s)
    return C, ns, rand(g, sum(ns), 14, 128).to(torch.bfloat16)


def run_out(C, batch, q, **kw):
    """Calls until a wait has run out (a copy may have landed before the kernel looks)."""
    for _ in range(20):
        C.cache.attend(batch, q, torch.zeros_like(q), **kw)
        try:
            C.cache.check()
        except K.KoreCudaError as e:
            return e
    pytest.fail("no wait ran out with a limit of 1 ns")


@BOTH
@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
@pytest.mark.parametrize("which", list(BATCHES))
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(impatient, kernel, tc, which):
    C, ns, q = ready(tc, which)
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    e = run_out(C, batch, q)
    assert e.code == -6 and "in time" in str(e)
    set_wait_limit(0)
    for _ in range(3):
        out = C.cache.attend(batch, q)
        C.cache.check()
        check_attention(C, q, out, ns)


@BOTH
def test_a_workspace_of_the_callers_is_zeroed_again_after_a_failure(impatient, kernel):
    C, ns, q = ready("bf16", "long")
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    ws = C.cache.new_workspace()
    run_out(C, batch, q, workspace=ws)
    set_wait_limit(0)
    ws[:K.paged.WORKSPACE_ZEROED].zero_()
    out = C.cache.attend(batch, q, workspace=ws)
    C.cache.check()
    check_attention(C, q, out, ns)


@BOTH
def test_a_captured_call_keeps_the_limit_of_its_capture(kernel):
    C, ns, q = ready("bf16", "long")
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    out = torch.zeros_like(q)
    C.cache.attend(batch, q, out)
    torch.cuda.synchronize(dev())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C.cache.attend(batch, q, out)
    set_wait_limit(1e-9)
    try:
        graph.replay()
        C.cache.check()
    finally:
        set_wait_limit(0)
    check_attention(C, q, out, ns)


def test_a_limit_that_is_no_time_is_refused():
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            set_wait_limit(bad)


@BOTH
def test_a_run_out_wait_is_reported_before_bad_device_data(impatient, kernel):
    """It is what makes the workspaces unusable: a bad page that was met before must not hide it."""
    C, ns, q = ready("bf16", "long")
    table = C.table.clone()
    table[:, 0] = 10 ** 6
    e = run_out(C, K.PagedBatch(starts(ns), ints(C.kvs), table, **HINTS[kernel]), q)
    assert "in time" in str(e)
    set_wait_limit(0)
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    for _ in range(2):
        out = C.cache.attend(batch, q)
        C.cache.check()
        check_attention(C, q, out, ns)


@BOTH
def test_check_waits_for_every_stream_of_the_device(kernel):
    """A failure of a call on another stream than check()'s own, still on its way when check() is called."""
    C, ns, q = ready("bf16", "short")
    table = C.table.clone()
    table[0, 0] = 10 ** 6
    bad = K.PagedBatch(starts(ns), ints(C.kvs), table, **HINTS[kernel])
    out = torch.zeros_like(q)
    side = torch.cuda.Stream(dev())
    with torch.cuda.stream(side):
        C.cache.attend(K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel]), q, out)   # makes the workspace
    torch.cuda.synchronize(dev())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)   # some 50 ms
        C.cache.attend(bad, q, out)
    other = torch.cuda.Stream(dev())
    with torch.cuda.stream(other), pytest.raises(K.KoreCudaError, match="page id"):
        C.cache.check()
    C.cache.check()
    table = K.RopeTable(8, 64)
    pos, x = ints([9] * q.shape[0]), q[..., :64].contiguous()
    torch.cuda.synchronize(dev())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        table.rotate(x, pos, out=x)
    with torch.cuda.stream(other), pytest.raises(K.KoreCudaError, match="rotation table"):
        table.check()


@BOTH
@pytest.mark.parametrize("n", [3, 300])
def test_starts_that_go_back_are_reported_and_the_sequences_that_fit_are_right(kernel, n):
    """31 sequences over the same rows: the 16 whose bounds fit are worked on (here all with one cache, so that it does
    not matter which of them writes last), the others are left out."""
    g = gen(41)
    C = Cache(g, "bf16", 2, 64, 32, [400])
    C.fill(g, 0)
    q = rand(g, n, 14, 64).to(torch.bfloat16)
    table = C.table.expand(31, -1).contiguous()
    batch = K.PagedBatch(ints([0, n] * 16), ints([400] * 31), table, **HINTS[kernel])
    out = C.cache.attend(batch, q)
    with pytest.raises(K.KoreCudaError, match="bounds"):
        C.cache.check()
    check_attention(C, q, out, [n])


@BOTH
def test_workspaces_of_captures_that_are_over_are_given_back(kernel):
    """They are the graphs' memory: no more than the last one is held here, and the graphs go on replaying."""
    C, ns, q = ready("bf16", "long")
    batch = K.PagedBatch(starts(ns), ints(C.kvs), C.table, **HINTS[kernel])
    stream = torch.cuda.Stream(dev())
    outs, graphs = [torch.zeros_like(q) for _ in range(4)], []
    torch.cuda.synchronize(dev())
    with torch.cuda.stream(stream):
        C.cache.attend(batch, q, outs[0])
        for out in outs:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                C.cache.attend(batch, q, out)
                C.cache.attend(batch, q, out)
    here = [k for k in K.paged._workspaces if k[1] == stream.cuda_stream]
    assert sum(k[2] != 0 for k in here) == 1 and sum(k[2] == 0 for k in here) == 1
    side = [torch.cuda.Stream(dev()) for _ in graphs]
    torch.cuda.synchronize(dev())
    for _ in range(3):
        for graph, s in zip(graphs, side):
            with torch.cuda.stream(s):
                graph.replay()
    C.cache.check()
    for out in outs:
        check_attention(C, q, out, ns)
