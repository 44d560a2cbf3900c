"""The built module that describes torch tensors for the library (kore_b200._tensors) and its Python form: the same
structure, the same addresses, the same refusals. On tensors that have a device, shape and strides and no memory
(torch's fake tensors). CPU only."""
import ctypes

import pytest

from kore_b200 import build
from kore_b200 import paged as P

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer")
P._import_torch()


@pytest.fixture(scope="module")
def native():
    build.build_tensors()
    from kore_b200 import _tensors
    assert _tensors.torch_version == torch.__version__.split("+")[0]
    return _tensors


@pytest.fixture
def fake():
    with FakeTensorMode() as mode:
        yield mode


def cuda(*shape, dtype=torch.bfloat16, device="cuda:0"):
    return torch.empty(*shape, dtype=dtype, device=device)


def outcome(f, *a):
    try:
        return f(*a)
    except ValueError as e:
        return str(e)


def described(f, t, device=0):
    r = P._Rows()
    ctypes.memset(ctypes.addressof(r), 0x5a, ctypes.sizeof(r))
    return outcome(f, ctypes.addressof(r), t, "k", device), bytes(r)


ROWS = {
    "bf16": lambda: cuda(5, 2, 64), "f16": lambda: cuda(5, 2, 64, dtype=torch.float16),
    "f32": lambda: cuda(5, 2, 64, dtype=torch.float32), "e4m3": lambda: cuda(5, 2, 64).to(torch.float8_e4m3fn),
    "another type": lambda: cuda(5, 2, 64, dtype=torch.float64), "strided": lambda: cuda(5, 9, 64)[:, 3:5],
    "heads first": lambda: cuda(2, 5, 64).transpose(0, 1), "one value a head": lambda: cuda(5, 2, 8)[..., ::8],
    "no tokens": lambda: cuda(0, 2, 64), "one": lambda: cuda(1, 1, 1), "broadcast": lambda: cuda(1, 2, 64).expand(7, 2, 64),
    "beyond 32 bits": lambda: cuda(3, 1 << 24, 1 << 10).transpose(0, 1),
    "two dimensions": lambda: cuda(5, 64), "four": lambda: cuda(5, 2, 2, 64), "values apart": lambda: cuda(5, 2, 128)[..., ::2],
    "too many": lambda: cuda(1, 1, 1).expand(1 << 31, 1, 1), "too many heads": lambda: cuda(1, 1, 1).expand(1, 1 << 31, 1),
    "another device": lambda: cuda(5, 2, 64, device="cuda:1"), "cpu": lambda: cuda(5, 2, 64, device="cpu")}


@pytest.mark.parametrize("what", ROWS)
def test_rows_as_in_python(native, fake, what):
    t = ROWS[what]()
    a, b = described(native.rows, t), described(P._rows_of, t)
    assert a == b
    refused = what in ("two dimensions", "four", "values apart", "too many", "too many heads", "another device", "cpu")
    assert isinstance(a[0], str) == refused


INTS = {
    "int32": (lambda: cuda(5, dtype=torch.int32), (1, 4, 5), True), "any length": (lambda: cuda(5, dtype=torch.int32), (1, 4, -1), True),
    "none": (lambda: cuda(0, dtype=torch.int32), (1, 4, 0), True), "table": (lambda: cuda(5, 3, dtype=torch.int32), (2, 4, -1), True),
    "int64": (lambda: cuda(5, dtype=torch.int64), (1, 8, 5), True), "of one": (lambda: cuda(8, dtype=torch.int32)[::8], (1, 4, 1), True),
    "longer": (lambda: cuda(6, dtype=torch.int32), (1, 4, 5), False), "shorter": (lambda: cuda(4, dtype=torch.int32), (1, 4, 5), False),
    "wide": (lambda: cuda(5, dtype=torch.int64), (1, 4, 5), False), "narrow": (lambda: cuda(5, dtype=torch.int32), (1, 8, 5), False),
    "float": (lambda: cuda(5, dtype=torch.float32), (1, 4, 5), False), "strided": (lambda: cuda(10, dtype=torch.int32)[::2], (1, 4, 5), False),
    "matrix": (lambda: cuda(5, 1, dtype=torch.int32), (1, 4, 5), False), "scalar": (lambda: cuda((), dtype=torch.int32), (1, 4, -1), False),
    "another device": (lambda: cuda(5, dtype=torch.int32, device="cuda:1"), (1, 4, 5), False),
    "cpu": (lambda: cuda(5, dtype=torch.int32, device="cpu"), (1, 4, 5), False)}


@pytest.mark.parametrize("what", INTS)
def test_integers_as_in_python(native, fake, what):
    t, (dims, size, length), good = INTS[what][0](), INTS[what][1], INTS[what][2]
    a, b = (outcome(f, t, "pos", 0, dims, size, length) for f in (native.ints, P._ints_of))
    assert a == b
    assert isinstance(a, int) == good


@pytest.mark.parametrize("a", [(), (1, 2, 3), (None, None, None, None), ("x", 0, 0, 0), (0, 1, "k", 0), (0, "k", "k", "k")])
def test_other_arguments_raise(native, a):
    with pytest.raises((TypeError, ValueError)):
        native.rows(*a)


@pytest.mark.parametrize("a", [(), (1, 2), (None,) * 6, (3, "pos", 0, 1, 4, -1), (3, "pos", "x", 1, 4, -1),
                               ([1], "pos", 0, 1, 4, 1 << 80)])
def test_other_arguments_for_integers_raise(native, a):
    with pytest.raises((TypeError, ValueError, OverflowError)):
        native.ints(*a)


@pytest.mark.gpu
def test_on_the_gpu_they_agree(native):
    dev = torch.cuda.current_device()
    x = torch.zeros(6, 4, 64, dtype=torch.float16, device="cuda")
    for t in (x, x[1:, 2:], x.transpose(0, 1), x[:0]):
        a, b = described(native.rows, t, dev), described(P._rows_of, t, dev)
        assert a == b and a[0] == t.shape[0]
    i = torch.zeros(9, 2, dtype=torch.int64, device="cuda")
    for t, dims in ((i, 2), (i[3:], 2), (i[3], 1), (i[:0], 2)):
        assert native.ints(t, "x", dev, dims, 8, -1) == P._ints_of(t, "x", dev, dims, 8, -1) == t.data_ptr()
    assert P._rows_in is native.rows and P._ints_in is native.ints   # the calls go through the module
