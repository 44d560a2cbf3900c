"""What a step with drafted tokens leaves out stays as it is through the whole step: requests that a plan did not serve,
through acceptance and trim; chunks longer than their masks, through store and acceptance."""
import pytest

import kore_b200 as K
from tests.test_paged_gpu import GUARD, dev, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
MOST = 2 ** 31 - 1


def state(pool):
    return pool.free.tolist()[: int(pool.n_free)], pool.table.tolist(), pool.length.tolist()


def held(lengths, width=9):
    """A pool whose first requests hold so many positions."""
    pool = K.PagePool(64, 16, 8, width)
    step = pool.new_step(len(lengths), sum(lengths), max(lengths))
    pool.plan(step, ints(range(len(lengths))), ints(lengths))
    pool.check()
    return pool


def finished(pool, request, n_new, n_tok=50):
    """Plan, masks, acceptance of token 0 alone and trim; what the plan and the acceptance wrote."""
    step, tree, path = pool.new_step(len(request), n_tok, 40), K.TokenTree(n_tok, 64), K.AcceptedPath(len(request), 4)
    none = ints([-1] * n_tok)
    pool.plan(step, ints(request), ints(n_new))
    tree.build(step, none)
    path.accept(step, none, torch.zeros_like(none), none)
    pool.trim(ints(request), path.kept)
    torch.cuda.synchronize()
    return step, path


@pytest.mark.parametrize("request_,n_new,served", [
    ([3, 0, 1], [60, 0, 0], []),             # two that want nothing, behind one whose rows pass the step's
    ([2, 3, 0], [8, 60, 0], [0]),
    ([0, 1], [-1, 5], [1]),                  # a negative number
    ([3, 0, 1], [MOST, 7, 0], []),           # behind a q_start that stands at the most that 32 bits hold
    ([3, 4, 0, 1], [MOST, MOST, 7, -2], []),
    ([0, 0, 1], [0, 0, 3], [2])])            # named twice
def test_requests_that_a_plan_left_out_keep_what_they_hold(request_, n_new, served):
    lengths = [30, 20, 10]
    pool = held(lengths)
    free, table, _ = state(pool)
    step, path = finished(pool, request_, n_new)
    want = (lengths + [0] * 8)[:8]
    for s in served:
        want[request_[s]] += 1   # token 0
    assert state(pool)[2] == want
    more = [-(-b // 16) - -(-a // 16) for a, b in zip(lengths, want)]
    assert int(pool.n_free) == len(free) - sum(more)
    for r, (row, now) in enumerate(zip(table, pool.table.tolist())):
        assert now[: -(-(lengths + [0] * 5)[r] // 16)] == row[: -(-(lengths + [0] * 5)[r] // 16)]
    left = [s for s, n in enumerate(n_new) if s not in served and n != 0]
    assert all(int(path.kept[s]) == -1 and int(path.count[s]) == 0 for s in left)
    with pytest.raises(K.KoreCudaError, match="bounds"):
        pool.check()


def test_requests_that_want_nothing_are_served_whatever_the_rows():
    """They have no rows that could pass the step's."""
    pool = held([30, 20, 10])
    step, path = finished(pool, [3, 0, 4, 1, -1], [60, 0, 70, 0, 3])
    assert step.kv_len.tolist() == [0, 30, 0, 20, 0] and step.q_start.tolist() == [0, 60, 60, 130, 130, 130]
    assert path.kept.tolist() == [-1, 30, -1, 20, -1] and path.count.tolist() == [0] * 5
    assert pool.length.tolist() == [30, 20, 10] + [0] * 5


def test_a_request_that_holds_nothing_and_wants_nothing_is_no_failure():
    pool = held([30, 20, 10])
    before = state(pool)
    finished(pool, [5, 0, -1, 7], [0, 0, 0, 0])
    assert state(pool) == before
    pool.check()
    pool.trim(ints([5, 0]), ints([-1, -1]))   # the second holds something: a negative number is reported
    assert state(pool) == before
    with pytest.raises(K.KoreCudaError, match="bounds"):
        pool.check()


@pytest.mark.parametrize("most,n", [(32, 33), (32, 40), (64, 300), (1024, 1025)])
def test_masks_of_a_chunk_that_is_too_long_are_not_another_steps(most, n):
    """Its tokens have no position, so that a store leaves out their rows; those of the others are as ever."""
    n_tok = n + 7
    tree = K.TokenTree(n_tok, most)
    chain = ints(range(-1, n_tok - 1))
    tree.build(K.PagedBatch(ints([0, most]), ints([most + 5]), ints([[0]]), most), chain)
    tree.check()
    parent = ints(list(range(-1, n - 1)) + [-1, 0, 0, 1, -1] + [-1, -1])
    tree.mask[n + 5:], tree.pos[n + 5:] = 77, 77
    tree.build(K.PagedBatch(ints([0, n, n + 5]), ints([n + 9, 25]), ints([[0], [0]]), n), parent)
    assert (tree.pos[:n] == -1).all() and (tree.mask[:n] == 0).all()
    assert tree.pos[n:].tolist() == [20, 21, 21, 22, 20, 77, 77]
    assert tree.mask[n:, 0].tolist() == [1, 3, 5, 11, 16, 77, 77]
    with pytest.raises(K.KoreCudaError, match="bounds"):
        tree.check()
    kp, vp = (torch.full((n // 8 + 8, 1, 16, 64), GUARD, device=dev(), dtype=torch.bfloat16) for _ in range(2))
    cache, rows = K.PagedCache(kp, vp), torch.ones(n_tok, 1, 64, device=dev(), dtype=torch.bfloat16)
    q, q_out = rows, torch.full_like(rows, GUARD)
    slots = torch.arange(n_tok, device=dev())
    slots[n + 5:] = -1
    cache.store(slots, tree.pos, rows, rows, rope=K.RopeTable(n + 20, 64), q=q, q_out=q_out)
    cache.check()
    written = (vp[:, 0, :, 0] == 1).flatten().nonzero().flatten().tolist()
    assert written == list(range(n, n + 5))
    assert (q_out[:n] == GUARD).all() and (q_out[n + 5:] == GUARD).all() and not (q_out[n:n + 5] == GUARD).any(-1).any()


@pytest.mark.parametrize("most,n", [(32, 33), (64, 70), (64, 1000)])
def test_a_chunk_that_is_too_long_for_its_masks_is_not_accepted(most, n):
    """What the model chose behind its tokens means nothing: the attention has left them out."""
    pool = K.PagePool(n // 16 + 20, 16, 8, n // 16 + 9)
    step, tree, path = pool.new_step(2, n + 6, n), K.TokenTree(n + 6, most), K.AcceptedPath(2, 4)
    pool.plan(step, ints([0, 1]), ints([n, 6]))
    parent = ints(list(range(-1, n - 1)) + list(range(-1, 5)))
    ones = torch.ones_like(parent)
    tree.build(step, parent)
    path.accept(step, parent, ones, ones, tree=tree)
    assert path.count.tolist() == [0, 4] and path.kept.tolist() == [-1, 4] and path.next_token.tolist() == [-1, 1]
    assert path.path.tolist() == [[-1] * 4, [0, 1, 2, 3]]
    with pytest.raises(K.KoreCudaError, match="bounds"):
        path.check()
    path.accept(step, parent[:n], ones[:n], ones[:n])   # (without the masks, and rows for the first chunk alone)
    assert path.count.tolist() == [4, 0]
    with pytest.raises(K.KoreCudaError, match="bounds"):
        path.check()
    with pytest.raises(ValueError, match="tree"):
        path.accept(step, parent[:n], ones[:n], ones[:n], tree=tree)


@pytest.mark.parametrize("n", [1, 6, 300])   # (walked in shared memory, and not)
@pytest.mark.parametrize("root", [0, 3, -2, -2 ** 31])
def test_a_chunk_whose_first_token_is_no_root_is_not_accepted(n, root):
    """Masks and store leave that token out, and with it all of its branches."""
    batch = K.PagedBatch(ints([0, 4, 4 + n, 8 + n]), ints([9, 50 + n, 4]), ints([[0]] * 3), 300)
    chain = list(range(-1, 3))
    parent = ints(chain + [root] + list(range(n - 1)) + chain)
    tree, path, ones = K.TokenTree(8 + n, 320), K.AcceptedPath(3, 3), torch.ones_like(parent)
    tree.build(batch, parent)
    assert (tree.pos[4:4 + n] == -1).all() and tree.pos[:4].tolist() == [5, 6, 7, 8]
    path.accept(batch, parent, ones, ones, tree=tree)
    assert path.count.tolist() == [3, 0, 3] and path.kept.tolist() == [8, -1, 3] and path.next_token.tolist() == [1, -1, 1]
    assert path.path.tolist() == [[0, 1, 2], [-1] * 3, [0, 1, 2]]
    for x in (tree, path):
        with pytest.raises(K.KoreCudaError, match="bounds"):
            x.check()
