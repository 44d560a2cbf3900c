"""Calls of the operators on a caller-owned paged cache that are refused before anything reaches a GPU, on tensors
that have a device, shape and strides and no memory (torch's fake tensors). CPU only."""
import pytest

import kore_b200 as K

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

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
