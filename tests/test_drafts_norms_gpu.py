"""Norms of heads whose squares pass 32 bits, beside an eps that is of their size."""
import pytest

import kore_b200 as K
from tests.test_drafts_gpu import near, normed
from tests.test_paged_gpu import DT, Cache, dev, gen, rand

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [1e-6, 1e20, 2.0 ** 100, 1e36, 1e38, 3.4e38])
def test_eps_counts_whatever_its_size(t, d, eps):
    """Heads of 2^40 to 2^70 (squares below and above what 32 bits hold), ones and zeros, whole and one value alone."""
    g = gen(d)
    x = rand(g, 3, 9, d)
    for h, p in enumerate((0, 40, 58, 62, 63, 64, 66, 70)):
        x[:, h] *= 2.0 ** p
    x[1, 7, 1:], x[2, 4, 1:] = 0, 0
    x[:, 8] = 0
    x, w = x.to(DT[t]), (1 + 0.2 * rand(g, d)).to(DT[t])
    C = Cache(g, t, 9, d, 16, [16])
    out = torch.zeros_like(x)
    slots = torch.arange(3, device=dev())
    eps32 = float(torch.tensor(eps, dtype=torch.float32))
    C.cache.store(slots, None, x, x, norm=K.HeadNorm(w, w, eps=eps), q=x, q_out=out)
    C.cache.check()
    y = normed(x, w, eps32)
    near(out, y, torch.zeros_like(y), t, d)
    near(C.kp[0].transpose(0, 1)[:3], y, torch.zeros_like(y), t, d)
