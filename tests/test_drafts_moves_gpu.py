"""Moves of accepted rows in caches whose keys and values are one memory."""
import random

import pytest

import kore_b200 as K
from tests.test_paged_gpu import DT, dev, gen, ints, starts

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("t,G,d,layers", [("bf16", 4, 128, 28), ("e4m3", 2, 64, 3), ("f16", 1, 64, 200)])
@pytest.mark.parametrize("every", [1, 2])
def test_keys_and_values_in_one_memory_move_once(t, G, d, layers, every):
    """Every layer, or every second one; more layers than a launch takes."""
    g, r, P = gen(layers), random.Random(layers), 16
    ns = [6, 64, 1, 40, 9]
    kvs = [n + r.randrange(60) for n in ns]
    used = [-(-x // P) for x in kvs]
    order = torch.randperm(sum(used), device=dev(), generator=g).int()
    table = torch.full((len(ns), max(used)), -1, dtype=torch.int32, device=dev())
    for s, x in enumerate(used):
        table[s, :x] = order[sum(used[:s]): sum(used[:s]) + x]
    bytes_ = torch.randint(0, 120, (layers, 2, sum(used), G, P, d * DT[t].itemsize), device=dev(), generator=g,
                           dtype=torch.uint8)
    pages = bytes_.view(DT[t])
    caches = [K.PagedCache(x[0], x[0] if i % every == 0 else x[1]) for i, x in enumerate(pages)]
    paths = [[0, 2, 3, 5], [0] + sorted(r.sample(range(1, 64), 19)), [0], [0, 1, 2, 9, 10, 11, 12, 20, 21, 22, 23, 39], [0, 8]]
    p = K.AcceptedPath(len(ns), 20)
    for s, x in enumerate(paths):
        p.path[s, : len(x)] = ints(x)
    p.count.copy_(ints([len(x) for x in paths]))
    want = bytes_.clone()
    for s, x in enumerate(paths):
        for j, i in enumerate(x):
            a, b = kvs[s] - ns[s] + i, kvs[s] - ns[s] + j
            want[:, :, table[s, b // P], :, b % P] = bytes_[:, :, table[s, a // P], :, a % P]
    for i in range(0, layers, every):
        want[i, 1] = bytes_[i, 1]   # (nobody's)
    moves = K.PagedLayers(caches)
    moves.commit(K.PagedBatch(starts(ns), ints(kvs), table, 64), p)
    moves.check()
    assert torch.equal(bytes_, want)
