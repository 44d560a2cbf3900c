"""The tree attention's two kernels at every size of its tests: what a batch says of itself (tests/test_drafts_gpu.py) leaves
the choice to a rule on sizes, which takes the row kernel for many of them; here each is set."""
import random

import pytest

import kore_b200 as K
from kore_b200.paged import set_tree_kernel
from tests import test_drafts_failures_gpu as F
from tests import test_drafts_gpu as T
from tests.test_paged_gpu import KINDS, Cache, dev, gen, ints, rand, starts

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(params=["rows", "tiles"])
def kernel(request):
    set_tree_kernel(request.param)
    yield "rows"   # (its hints: with them the rule would take the row kernel)
    set_tree_kernel("auto")


def test_the_kernel_that_is_set_is_the_one_that_runs(kernel, request):
    g, r = gen(1), random.Random(1)
    C = Cache(g, "bf16", 2, 64, 16, [50])
    C.fill(g, 0)
    q, t = rand(g, 1, 4, 64).to(torch.bfloat16), K.TokenTree(1, 1)
    t.mask.fill_(1)
    batch = K.PagedBatch(ints([0, 1]), ints([50]), C.table, 1)
    C.cache.attend(batch, q, tree=t)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        C.cache.attend(batch, q, tree=t)
        torch.cuda.synchronize()
    names = " ".join(e.name for e in prof.events())
    if "paged_" not in names:
        pytest.skip("this machine's profiler names no kernels")
    tiles = request.node.callspec.params["kernel"] == "tiles"
    assert ("paged_tree_kernel" in names) == tiles and ("paged_rows_kernel" in names) == (not tiles)


@pytest.mark.parametrize("tq,tc", KINDS)
@pytest.mark.parametrize("H,G,d,P", [(28, 4, 128, 64), (14, 2, 64, 16), (8, 8, 128, 48), (40, 2, 64, 256), (3, 1, 128, 16)])
@pytest.mark.parametrize("which", list(T.TREES))
def test_tree_attention(kernel, tq, tc, H, G, d, P, which):
    T.test_tree_attention(kernel, tq, tc, H, G, d, P, which)


@pytest.mark.parametrize("tq,tc", KINDS)
def test_any_mask_and_what_no_token_sees(kernel, tq, tc):
    T.test_tree_attention_of_any_mask(kernel, tq, tc)
    T.test_what_no_token_sees_may_be_anything(kernel, tq, tc)


@pytest.mark.parametrize("how", ["fused", "heads_first", "odd"])
def test_strided_rows(kernel, how):
    T.test_tree_attention_of_strided_rows(kernel, how)


@pytest.mark.parametrize("H,G,d", [(128, 1, 64), (16, 16, 128), (12, 12, 64)])
def test_wide_and_single_groups(kernel, H, G, d):
    T.test_tree_attention_of_wide_and_of_single_groups(kernel, H, G, d)


def test_a_chain_is_a_chunk(kernel):
    T.test_a_chains_attention_is_the_chunks(kernel)


def test_many_sequences(kernel):
    T.test_tree_attention_of_many_sequences(kernel)


@pytest.mark.parametrize("n_seq", [32, 33, 63, 64, 65, 97])
def test_batches_around_the_sequences_of_a_warp(kernel, n_seq):
    T.test_batches_around_the_sequences_of_a_warp(kernel, n_seq, True)


@pytest.mark.parametrize("n_seq,n_tok", [(4096, 4096), (700, 2000)])
def test_most_sequences(kernel, n_seq, n_tok):
    """The sums' place in shared memory holds those of 4096 sequences."""
    g, r = gen(n_seq), random.Random(n_seq)
    ns = [1] * n_seq
    for _ in range(n_tok - n_seq):
        ns[r.randrange(n_seq)] += 1
    some = set(r.sample(range(n_seq), n_seq // 7))
    ns = [0 if s in some else n for s, n in enumerate(ns)]
    kvs = [n + r.choice([0, 1, 20]) for n in ns]
    C = Cache(g, "bf16", 1, 64, 16, kvs)
    C.kp.copy_(torch.randn(C.kp.shape, device=dev(), generator=g)), C.vp.copy_(torch.randn(C.vp.shape, device=dev(), generator=g))
    T.attend(g, C, 2, ns, [T.sees(T.tree(r, n, "random")) if n else None for n in ns], "bf16", kernel)


@pytest.mark.parametrize("n", [6, 50])
@pytest.mark.parametrize("bad,word", [("page", "page id"), ("rows", "bounds"), ("long", "bounds"), ("short", "bounds")])
def test_bad_device_data(kernel, n, bad, word):
    T.test_tree_attention_reports_bad_device_data(kernel, n, bad, word)


@pytest.mark.parametrize("n", [33, 40, 1000])
def test_chunks_longer_than_their_masks(kernel, n):
    """Left out and reported; the one beside it is not."""
    g, r = gen(n), random.Random(n)
    C = Cache(g, "bf16", 2, 64, 16, [n + 50, 90])
    C.fill(g, 0), C.fill(g, 1)
    seen = T.sees(T.tree(r, 32, "random"))
    q, t = rand(g, n + 32, 4, 64).to(torch.bfloat16), K.TokenTree(n + 32, 32)
    t.mask[:n], t.mask[n:] = -1, T.words_of(seen, 1).to(dev())
    out = torch.full_like(q, T.GUARD)
    C.cache.attend(K.PagedBatch(starts([n, 32]), ints(C.kvs), C.table, 1), q, out, tree=t)
    with pytest.raises(K.KoreCudaError, match="bounds"):
        C.cache.check()
    assert (out[:n] == T.GUARD).all()
    one = Cache(g, "bf16", 2, 64, 16, [90])
    one.kp, one.vp, one.table = C.kp, C.vp, C.table[1:]
    T.check_tree(one, q[n:], out[n:], [32], [seen])


@pytest.mark.parametrize("tq,tc", KINDS)
@pytest.mark.parametrize("n,past", [(8, 1000), (24, 300), (24, 6000), (2, 3000)])
def test_many_trees(kernel, tq, tc, n, past):
    T.test_trees_of_many_sequences_with_their_own_bounds(tq, tc, n, past)


@pytest.mark.parametrize("tq,tc,H,G,d,P", [("bf16", "bf16", 28, 4, 128, 64), ("f16", "e4m3", 14, 2, 64, 16)])
def test_steps_with_drafts(kernel, tq, tc, H, G, d, P):
    T.test_steps_with_drafts_leave_what_single_tokens_would(kernel, tq, tc, H, G, d, P)


def test_a_captured_step_and_streams(kernel):
    T.test_captured_step_with_drafts()
    T.test_tree_attention_on_two_streams(kernel)
    F.test_two_graphs_of_one_stream_on_two_streams(kernel)


def test_offsets_beyond_32_bits(kernel):
    F.test_offsets_beyond_32_bits()


@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
def test_one_workspace_in_turn(kernel, tc):
    F.test_one_workspace_for_chunks_and_trees_in_turn(kernel, tc)


@pytest.mark.parametrize("tc", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", list(F.BATCHES))
def test_a_wait_that_runs_out(kernel, tc, d, which):
    F.test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(kernel, tc, d, which)
