"""The operators on a caller-owned paged cache, as far as no GPU is needed: the rotation's frequencies against their
formulas, and the calls that are refused (every check stands before the first CUDA call, so placeholder addresses do).
CPU only."""
import ctypes
import math

import pytest

import kore_b200 as K
from kore_b200 import paged as P

A, B = 0x10000, 0x20000   # placeholders for aligned device addresses


def _f32(x: float) -> float:
    return ctypes.c_float(x).value


@pytest.mark.parametrize("rot", [2, 32, 64, 128, 250])
def test_frequencies_are_kores(rot):
    f, amp = K.rope_frequencies(rot)
    assert amp == 1.0
    assert f == [_f32(1e6 ** (-2.0 * i / rot)) for i in range(rot // 2)]


def test_linear_scaling_divides_the_frequencies():
    f, amp = K.rope_frequencies(64, base=10000.0, scaling="linear", factor=8.0)
    assert amp == 1.0 and f == [_f32(10000.0 ** (-2.0 * i / 64) / 8.0) for i in range(32)]


def test_scaling_by_wavelength():
    rot, base, factor, ctx = 128, 1e6, 4.0, 8192
    f, amp = K.rope_frequencies(rot, base=base, scaling="yarn", factor=factor, original_ctx=ctx)
    assert abs(amp - (0.1 * math.log(factor) + 1)) < 1e-15
    for i, x in enumerate(f):
        plain = base ** (-2.0 * i / rot)
        turns = ctx * plain / (2 * math.pi)
        assert plain / factor * (1 - 1e-6) <= x <= plain * (1 + 1e-6)
        if turns > 32 * 1.3:    # more than a pair's step above beta_fast: kept
            assert x == _f32(plain)
        if turns < 1 / 1.3:     # below beta_slow: divided
            assert x == _f32(plain / factor)
    # a factor that shrinks the context, and a given amplitude
    assert K.rope_frequencies(rot, scaling="yarn", factor=0.5, original_ctx=ctx)[1] == 1.0
    assert K.rope_frequencies(rot, scaling="yarn", factor=4.0, original_ctx=ctx, amplitude=1.25)[1] == 1.25


@pytest.mark.parametrize("kw", [dict(n_rot=0), dict(n_rot=7), dict(n_rot=258), dict(n_rot=8, base=0.0),
                                dict(n_rot=8, base=math.nan), dict(n_rot=8, scaling="linear", factor=0.0),
                                dict(n_rot=8, scaling="yarn", factor=2.0),
                                dict(n_rot=8, scaling="yarn", factor=2.0, original_ctx=100, beta_fast=1, beta_slow=2),
                                dict(n_rot=8, amplitude=-1.0), dict(n_rot=8, amplitude=math.inf)])
def test_frequencies_refused(kw):
    with pytest.raises(K.KoreCudaError) as e:
        K.rope_frequencies(kw.pop("n_rot"), **kw)
    assert e.value.code == -1


def test_unknown_scaling_refused():
    with pytest.raises(ValueError, match="scaling"):
        K.rope_frequencies(8, scaling="other")


def _rows(heads=2, d=64, type=P.BF16, data=A, ts=None, hs=None):
    return P._Rows(data, type, heads, d, heads * d if ts is None else ts, d if hs is None else hs)


def _pages(**kw):
    a = dict(k=A, v=A, type=P.BF16, n_pages=4, page_tokens=16, n_head_kv=2, head_dim=64, page_stride=0, k_scale=None,
             v_scale=None)
    a.update(kw)
    return P._Pages(*a.values())


def _batch(**kw):
    a = dict(n_seq=1, q_start=A, kv_len=A, page_table=A, table_stride=4, max_q=1, max_kv=0)
    a.update(kw)
    return P._Batch(*a.values())


def _ref(x):
    return None if x is None else ctypes.byref(x)


def _append(cache=None, batch=None, n=1, k=..., v=..., q=None, q_out=None, rope=None):
    L = P._library()
    k, v = _rows() if k is ... else k, _rows() if v is ... else v
    return L.kore_cuda_paged_append_dev(_ref(cache or _pages()), _ref(batch or _batch()), n, _ref(k), _ref(v), _ref(q),
                                        _ref(q_out), _ref(rope), None, None), L.kore_cuda_last_error(None).decode()


def _attend(cache=None, batch=None, n=1, q=..., out=..., opts=..., ws=A, ws_bytes=1 << 40):
    L = P._library()
    q, out = _rows(4) if q is ... else q, _rows(4, data=B) if out is ... else out
    opts = P._Opts(0.0, 1, 0) if opts is ... else opts
    return L.kore_cuda_paged_attn_dev(_ref(cache or _pages()), _ref(batch or _batch()), n, _ref(q), _ref(out), None,
                                      _ref(opts), ws, ws_bytes, None, None), L.kore_cuda_last_error(None).decode()


BAD_PAGES = [(dict(k=None), "null"), (dict(type=99), "type"), (dict(n_pages=0), "n_pages"),
             (dict(page_tokens=0), "page_tokens"), (dict(page_tokens=24), "page_tokens"), (dict(n_head_kv=0), "n_head_kv"),
             (dict(head_dim=40), "head_dim"), (dict(head_dim=272), "head_dim"), (dict(v=A + 8), "aligned"),
             (dict(page_stride=2 * 16 * 64 - 8), "page_stride"), (dict(page_stride=2 * 16 * 64 + 4), "page_stride"),
             (dict(k_scale=A), "scales")]
BAD_BATCH = [(dict(n_seq=-1), -2), (dict(n_seq=4097), -2), (dict(q_start=None), -1), (dict(kv_len=None), -1),
             (dict(page_table=None), -1), (dict(table_stride=0), -1), (dict(max_q=-1), -1),
             (dict(max_kv=-1), -1)]


@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_bad_pages_refused(kw, word):
    for rc, msg in (_append(cache=_pages(**kw)), _attend(cache=_pages(**kw))):
        assert rc == -1 and word in msg, msg


@pytest.mark.parametrize("kw,code", BAD_BATCH)
def test_bad_batches_refused(kw, code):
    for rc, msg in (_append(batch=_batch(**kw)), _attend(batch=_batch(**kw)), ):
        assert rc == code and msg
    assert _append(n=-1)[0] == -1 and _attend(n=-1)[0] == -1


@pytest.mark.parametrize("kw,word", [
    (dict(k=None), "k is null"), (dict(v=_rows(data=None)), "v is null"), (dict(k=_rows(3)), "heads"),
    (dict(k=_rows(d=128)), "head_dim"), (dict(v=_rows(type=P.F16)), "different types"), (dict(k=_rows(type=5)), "type"),
    (dict(k=_rows(data=A + 1)), "aligned"), (dict(q=_rows(4)), "together"), (dict(q_out=_rows(4)), "together"),
    (dict(q=_rows(4), q_out=_rows(5)), "heads"), (dict(q=_rows(4, type=P.F16), q_out=_rows(4)), "type"),
    (dict(k=_rows(type=P.F16), v=_rows(type=P.F16)), "do not go"), (dict(cache=_pages(type=P.F32)), "do not go"),
    (dict(rope=P._RopeView(None, 8, 8, 0)), "null"), (dict(rope=P._RopeView(A + 4, 8, 8, 0)), "aligned"),
    (dict(rope=P._RopeView(A, 0, 8, 0)), "positions"), (dict(rope=P._RopeView(A, 8, 7, 0)), "n_rot"),
    (dict(rope=P._RopeView(A, 8, 66, 0)), "n_rot")])
def test_append_refused(kw, word):
    rc, msg = _append(**kw)
    assert rc == -1 and word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "q is null"), (dict(q=_rows(4, type=P.F32), out=_rows(4, type=P.F32)), "F16 or BF16"),
    (dict(out=_rows(4)), "own rows"), (dict(out=_rows(4, type=P.F16)), "one type"), (dict(out=_rows(2)), "number of heads"),
    (dict(q=_rows(4, type=P.F16), out=_rows(4, type=P.F16, data=B)), "does not go"), (dict(cache=_pages(type=P.F32)), "type"),
    (dict(q=_rows(5), out=_rows(5, data=B)), "geometry"), (dict(q=_rows(258), out=_rows(258, data=B)), "geometry"),
    (dict(cache=_pages(head_dim=96), q=_rows(4, 96), out=_rows(4, 96)), "head_dim"), (dict(opts=None), "opts"),
    (dict(opts=P._Opts(0.0, 1, -1)), "window"), (dict(opts=P._Opts(math.nan, 1, 0)), "scale"),
    (dict(ws=None), "workspace"), (dict(ws=A + 16), "workspace"), (dict(ws_bytes=1 << 20), "workspace")])
def test_attention_refused(kw, word):
    rc, msg = _attend(**kw)
    assert rc == -1 and word in msg, msg


def test_rope_refused():
    L = P._library()
    view, x = P._RopeView(A, 8, 8, 0), _rows()

    def call(x=x, out=None, pos=A, view=view, n=1):
        return L.kore_cuda_rope_dev(_ref(x), _ref(out or _rows()), n, pos, _ref(view), None, None)
    assert call(pos=None) == -1 and call(view=None) == -1 and call(n=-1) == -1
    assert call(out=_rows(3)) == -1 and call(out=_rows(type=P.F16)) == -1 and call(x=_rows(d=63)) == -1
    assert call(x=_rows(type=P.E4M3), out=_rows(type=P.E4M3)) == -1
    assert L.kore_cuda_rope_table_dev(ctypes.byref(P._RopeSpec(8, 0, 1e4, 1, 0, 0, 0, 0)), 4, A + 8, None) == -1
    assert L.kore_cuda_rope_table_dev(ctypes.byref(P._RopeSpec(8, 0, 1e4, 1, 0, 0, 0, 0)), 0, A, None) == -1


def test_nothing_to_do_is_no_error():
    assert _append(n=0)[0] == 0 and _attend(n=0)[0] == 0
    assert _append(batch=_batch(n_seq=0))[0] == 0 and _attend(batch=_batch(n_seq=0))[0] == 0


def test_workspace_size():
    L = P._library()
    assert L.kore_cuda_paged_attn_workspace(64) > P.WORKSPACE_ZEROED
    assert L.kore_cuda_paged_attn_workspace(128) > L.kore_cuda_paged_attn_workspace(64)
    assert L.kore_cuda_paged_attn_workspace(96) == -1


def test_host_tensors_refused():
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        K.PagedCache(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        K.PagedBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                     torch.zeros(1, 1, dtype=torch.int32), 1)
