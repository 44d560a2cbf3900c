"""Operators on a caller-owned paged cache of 32, 16 or 8 bits (kore_cuda_rope_dev,
kore_cuda_paged_append_dev, kore_cuda_paged_attn_dev): torch tensors in place of the
C structures.

A step of a batch, on the current stream of the tensors' device::

    rope = RopeTable(n_pos, n_rot)                        # once
    cache = PagedCache(k_pages, v_pages)                  # once a layer
    batch = PagedBatch(q_start, kv_len, page_table, max_q)   # once a step
    cache.append(batch, k, v, rope=rope, q=q, q_out=q)    # a layer: store k and v, rotate k and q
    cache.attend(batch, q, out)

An object is for one host thread at a time, as a context is; nothing here is recorded for gradients. Nothing is copied or synchronised: a failure that a kernel meets in the device
data (a page outside the pool, a sequence that does not fit its page table)
is left in ``status`` and raised by ``check()``.
"""
from __future__ import annotations

import ctypes
import struct

from . import KoreCudaError, load_library

__all__ = ["RopeTable", "PagedCache", "PagedBatch", "rope_frequencies", "set_wait_limit"]

F32, F16, BF16, E4M3 = 0, 1, 30, 1000
WORKSPACE_ZEROED = 1024
SCALINGS = {"none": 0, "linear": 1, "yarn": 2}
DEVICE_FAILURES = {1: "a tile copy or product did not come in time", 3: "page id outside the pool", 6: "position outside the rotation table",
                   7: "a sequence's bounds do not fit the rows, its length or its page table"}

_vp, _i, _ll, _d = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double


class _Rows(ctypes.Structure):
    """kore_cuda_rows."""
    _fields_ = [("data", _vp), ("type", _i), ("n_head", _i), ("head_dim", _i), ("token_stride", _ll),
                ("head_stride", _ll)]


class _RopeSpec(ctypes.Structure):
    """kore_cuda_rope_spec."""
    _fields_ = [("n_rot", _i), ("scaling", _i), ("base", _d), ("factor", _d), ("original_ctx", _d), ("beta_fast", _d),
                ("beta_slow", _d), ("amplitude", _d)]


class _RopeView(ctypes.Structure):
    """kore_cuda_rope_view."""
    _fields_ = [("table", _vp), ("n_pos", _i), ("n_rot", _i), ("interleaved", _i)]


class _Pages(ctypes.Structure):
    """kore_cuda_pages."""
    _fields_ = [("k", _vp), ("v", _vp), ("type", _i), ("n_pages", _i), ("page_tokens", _i), ("n_head_kv", _i),
                ("head_dim", _i), ("page_stride", _ll), ("k_scale", _vp), ("v_scale", _vp)]


class _Batch(ctypes.Structure):
    """kore_cuda_batch."""
    _fields_ = [("n_seq", _i), ("q_start", _vp), ("kv_len", _vp), ("page_table", _vp), ("table_stride", _i),
                ("max_q", _i), ("max_kv", _i)]


class _Opts(ctypes.Structure):
    """kore_cuda_attn_opts."""
    _fields_ = [("scale", ctypes.c_float), ("causal", _i), ("window", _i)]


_fns = None


def _library():
    global _fns
    if _fns is None:
        L = load_library()
        # structures go by their address: a c_void_p costs less a call than a POINTER
        L.kore_cuda_rope_freqs.argtypes = [_vp, _vp, _vp]
        L.kore_cuda_rope_table_dev.argtypes = [_vp, _i, _vp, _vp]
        L.kore_cuda_rope_dev.argtypes = [_vp, _vp, _i, _vp, _vp, _vp, _vp]
        L.kore_cuda_paged_append_dev.argtypes = [_vp, _vp, _i] + [_vp] * 7
        L.kore_cuda_paged_attn_workspace.argtypes = [_i]
        L.kore_cuda_paged_attn_workspace.restype = _ll
        L.kore_cuda_paged_attn_dev.argtypes = [_vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _ll, _vp, _vp]
        L.kore_cuda_paged_set_wait_limit.argtypes = [ctypes.c_ulonglong]
        L.kore_cuda_capture_id.argtypes = [_vp]
        L.kore_cuda_capture_id.restype = ctypes.c_ulonglong
        _fns = L
    return _fns


def _ck(L, rc: int) -> None:
    if rc:
        raise KoreCudaError(rc, L.kore_cuda_last_error(None).decode())


_torch = None
_types: dict = {}


def _import_torch():
    global _torch
    if _torch is None:
        import torch
        _torch = torch
        _types.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3})
    return _torch


_INT_MAX = 2 ** 31 - 1


def _int(x, what: str) -> int:
    """x as a C int (ctypes would cut it to 32 bits)."""
    if not -_INT_MAX <= x <= _INT_MAX:
        raise ValueError(f"{what} = {x} does not fit 32 bits")
    return x


_pack_rows = struct.Struct("@Piiiqq").pack_into   # _Rows, in one step


def _fill(r: _Rows, t, what: str, device) -> int:
    """Describes a [tokens][heads][head_dim] tensor in r; returns its tokens."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{what}: expected [tokens][heads][head_dim], got {tuple(shape)}")
    n, h, d = shape
    if n > _INT_MAX:
        raise ValueError(f"{what}: {n} tokens are too many for one call")
    ts, hs, es = t.stride()
    if es != 1 and d > 1:
        raise ValueError(f"{what}: the values of a head must be contiguous")
    if t.get_device() != device.index:
        raise ValueError(f"{what} is on {t.device}, expected {device}")
    _pack_rows(r, 0, t.data_ptr(), _types.get(t.dtype, -1), h, d, ts, hs)
    return n


def _ints(t, what: str, device, shape_len: int):
    if t.dtype != _torch.int32 or t.dim() != shape_len or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what}: expected a contiguous {shape_len}-d int32 tensor on {device}")
    return t.data_ptr()


def _stream(device) -> int:
    return _torch._C._cuda_getCurrentRawStream(device.index)


def _check_status(status) -> None:
    _torch.cuda.synchronize(status.device)   # the calls may be on any stream
    code = int(status.item())
    if code:
        status.zero_()
        _torch.cuda.synchronize(status.device)   # what is launched from now on, on any stream, is kept
        if code == 1:   # workspaces are not as a call leaves them
            _workspaces.clear()
        raise KoreCudaError(-6, DEVICE_FAILURES.get(code, f"device failure {code}"))


def _spec(n_rot, base, scaling, factor, original_ctx, beta_fast, beta_slow, amplitude) -> _RopeSpec:
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} is none of {sorted(SCALINGS)}")
    return _RopeSpec(_int(n_rot, "n_rot"), SCALINGS[scaling], base, factor, original_ctx, beta_fast, beta_slow, amplitude)


def rope_frequencies(n_rot: int, *, base: float = 1e6, scaling: str = "none", factor: float = 1.0,
                     original_ctx: float = 0, beta_fast: float = 32.0, beta_slow: float = 1.0, amplitude: float = 0.0):
    """The frequencies (a list, each rounded to fp32) and amplitude of a rotation (kore_cuda_rope_freqs; no GPU)."""
    L = _library()
    f, a = (ctypes.c_float * 128)(), _d()
    spec = _spec(n_rot, base, scaling, factor, original_ctx, beta_fast, beta_slow, amplitude)
    _ck(L, L.kore_cuda_rope_freqs(ctypes.byref(spec), f, ctypes.byref(a)))
    return list(f[:n_rot // 2]), a.value


def set_wait_limit(seconds: float) -> None:
    """How long a wait inside an attention launched from now on may take before it is reported (0: 2 s), in the whole
    process (kore_cuda_paged_set_wait_limit)."""
    if not 0 <= seconds <= 1e9:
        raise ValueError(f"seconds = {seconds}")
    L = _library()
    _ck(L, L.kore_cuda_paged_set_wait_limit(int(seconds * 1e9)))


class RopeTable:
    """The (cos, sin) table of a rotation of the first n_rot values of a head, for positions [0, n_pos).

    interleaved: value 2i is paired with 2i + 1, else i with i + n_rot/2 (kore's rope_neox). scaling: "none",
    "linear" (frequencies / factor) or "yarn" (by wavelength: original_ctx, beta_fast, beta_slow; amplitude 0 takes
    0.1 ln(factor) + 1)."""

    def __init__(self, n_pos: int, n_rot: int, *, base: float = 1e6, interleaved: bool = False, scaling: str = "none",
                 factor: float = 1.0, original_ctx: float = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 amplitude: float = 0.0, device=None):
        torch = _import_torch()
        self._L = _library()
        spec = _spec(n_rot, base, scaling, factor, original_ctx, beta_fast, beta_slow, amplitude)
        if _int(n_pos, "n_pos") <= 0:
            raise ValueError(f"n_pos = {n_pos} must be positive")
        rope_frequencies(n_rot, base=base, scaling=scaling, factor=factor, original_ctx=original_ctx,
                         beta_fast=beta_fast, beta_slow=beta_slow, amplitude=amplitude)   # refuses before it allocates
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.table = torch.empty((n_pos, n_rot // 2, 2), dtype=torch.float32, device=device)
        self.device = self.table.device
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._status = self.status.data_ptr()
        _ck(self._L, self._L.kore_cuda_rope_table_dev(ctypes.byref(spec), n_pos, self.table.data_ptr(),
                                                      _stream(self.device)))
        self.view = _RopeView(self.table.data_ptr(), n_pos, n_rot, int(bool(interleaved)))
        self._view = ctypes.addressof(self.view)
        self._x, self._out = _Rows(), _Rows()
        self._px, self._pout = ctypes.addressof(self._x), ctypes.addressof(self._out)

    def rotate(self, x, pos, out=None):
        """Rotates x [tokens][heads][head_dim] (fp32, fp16 or bf16) at the int32 positions pos [tokens] into out
        (a new tensor if None; x itself to rotate in place). A row with a negative position is left as it is in out (in
        a new tensor: whatever the memory holds)."""
        if out is None:
            out = _torch.empty_like(x)
        n = _fill(self._x, x, "x", self.device)
        if _fill(self._out, out, "out", self.device) != n:
            raise ValueError("x and out have different numbers of tokens")
        pp = _ints(pos, "pos", self.device, 1)
        if pos.shape[0] != n:
            raise ValueError(f"{pos.shape[0]} positions for {n} tokens")
        if n == 0:
            return out
        rc = self._L.kore_cuda_rope_dev(self._px, self._pout, n, pp, self._view, self._status, _stream(self.device))
        if rc:
            _ck(self._L, rc)
        return out

    def check(self) -> None:
        """Waits for the device; raises if a rotation met a position outside the table."""
        _check_status(self.status)


class PagedBatch:
    """The sequences of a step: rows q_start[s] .. q_start[s+1]-1 of q, k and v are the new tokens of sequence s,
    which holds kv_len[s] positions with them, in the pages page_table[s]. All int32 on the device, read by the
    kernels when they run, so a captured step follows what they hold at its replay. max_q: the longest chunk; max_kv:
    the longest sequence (0: as much as page_table has room for). They choose a kernel and bound nothing."""

    def __init__(self, q_start, kv_len, page_table, max_q: int, max_kv: int = 0):
        _import_torch()
        if not kv_len.is_cuda:
            raise ValueError("expected CUDA tensors")
        self.device = dev = kv_len.device
        n = kv_len.shape[0]
        view = _Batch(n, _ints(q_start, "q_start", dev, 1), _ints(kv_len, "kv_len", dev, 1),
                      _ints(page_table, "page_table", dev, 2), _int(page_table.shape[1], "page_table's width"),
                      _int(max_q, "max_q"), _int(max_kv, "max_kv"))
        if q_start.shape[0] != n + 1 or page_table.shape[0] != n:
            raise ValueError(f"q_start must have {n + 1} and page_table {n} rows")
        self.q_start, self.kv_len, self.page_table, self.view = q_start, kv_len, page_table, view
        self._view = ctypes.addressof(view)


class PagedCache:
    """One layer's pages, k and v [n_pages][n_head_kv][page_tokens][head_dim] in fp32 (append only), fp16, bf16 or
    float8_e4m3fn (with a scale a head: value = 8 bits * scale). The pages' stride is free (a pool may hold k and v
    by turns)."""

    def __init__(self, k_pages, v_pages, *, k_scale=None, v_scale=None):
        torch = _import_torch()
        self._L = _library()
        for t, what in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if t.dim() != 4 or not t.is_cuda or (t.numel() and not t[0].is_contiguous()):
                raise ValueError(f"{what}: expected a CUDA tensor [pages][heads][tokens][head_dim], contiguous in a page")
        if (k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device
                or k_pages.stride(0) != v_pages.stride(0)):
            raise ValueError("k_pages and v_pages differ in shape, type, device or page stride")
        n, g, p, d = k_pages.shape
        if n > 1 and k_pages.stride(0) < g * p * d:   # (an expanded page; the C side takes a stride of 0 as dense)
            raise ValueError(f"k_pages and v_pages: the pages overlap (page stride {k_pages.stride(0)})")
        self.k, self.v, self.k_scale, self.v_scale = k_pages, v_pages, k_scale, v_scale
        self.device = k_pages.device
        scales = []
        for s, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if s is not None and (s.dtype != torch.float32 or tuple(s.shape) != (g,) or not s.is_contiguous()
                                  or s.device != self.device):
                raise ValueError(f"{what}: expected {g} float32 values on {self.device}")
            scales.append(s.data_ptr() if s is not None else None)
        self.view = _Pages(k_pages.data_ptr(), v_pages.data_ptr(), _types.get(k_pages.dtype, -1), n, p, g, d,
                           k_pages.stride(0) if n > 1 else 0, *scales)
        self._view = ctypes.addressof(self.view)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._status = self.status.data_ptr()
        self._r = [_Rows() for _ in range(4)]
        self._p = [ctypes.addressof(r) for r in self._r]
        self._opts = _Opts()
        self._popts = ctypes.addressof(self._opts)

    def append(self, batch: PagedBatch, k, v, *, rope: RopeTable | None = None, q=None, q_out=None) -> None:
        """Stores k (rotated by rope at each token's position) and v [tokens][n_head_kv][head_dim] in the pages; with
        q, rotates it into q_out (which may be q) in the same launch."""
        dev, r = self.device, self._r
        n = _fill(r[0], k, "k", dev)
        if _fill(r[1], v, "v", dev) != n:
            raise ValueError("k and v have different numbers of tokens")
        pq = pqo = None
        if (q is None) != (q_out is None):
            raise ValueError("q and q_out come together")
        if q is not None:
            if _fill(r[2], q, "q", dev) != n or _fill(r[3], q_out, "q_out", dev) != n:
                raise ValueError("q, q_out and k have different numbers of tokens")
            pq, pqo = self._p[2], self._p[3]
        if batch.device != dev or (rope is not None and rope.device != dev):
            raise ValueError(f"the batch or the table is not on {dev}")
        if n == 0:
            return
        rc = self._L.kore_cuda_paged_append_dev(self._view, batch._view, n, self._p[0], self._p[1], pq, pqo,
                                                rope._view if rope is not None else None, self._status, _stream(dev))
        if rc:
            _ck(self._L, rc)

    def attend(self, batch: PagedBatch, q, out=None, *, scale: float = 0.0, causal: bool = True, window: int = 0,
               lse=None, workspace=None):
        """Attention of q [tokens][n_head][head_dim] (fp16 or bf16) over the batch's cached positions, into out (a new
        tensor if None; never q's own memory). Rows outside every sequence keep what out holds (a new tensor: whatever
        the memory holds).

        scale 0: 1/sqrt(head_dim). window: how many positions back a token sees, itself among them (0: all). lse: an
        optional float32 [tokens][n_head] for the log of the softmax's sums. workspace: a tensor of new_workspace();
        by default one that this device and stream (or the capture that the stream is in) keep."""
        dev, r = self.device, self._r
        if out is None:
            out = _torch.empty(q.shape, dtype=q.dtype, device=q.device)
        n = _fill(r[0], q, "q", dev)
        if _fill(r[1], out, "out", dev) != n:
            raise ValueError("q and out have different numbers of tokens")
        plse = None
        if lse is not None:
            if (lse.dtype != _torch.float32 or tuple(lse.shape) != (n, r[0].n_head) or not lse.is_contiguous()
                    or lse.device != dev):
                raise ValueError("lse: expected a contiguous float32 tensor [tokens][n_head]")
            plse = lse.data_ptr()
        if batch.device != dev:
            raise ValueError(f"the batch is not on {dev}")
        o = self._opts
        o.scale, o.causal, o.window = scale, causal, window
        if o.window != window or (scale and not o.scale):   # (cut to 32 bits, or to 0: the default)
            raise ValueError(f"window = {window} or scale = {scale} is outside the range of 32 bits")
        if workspace is not None and (workspace.dtype != _torch.uint8 or workspace.device != dev
                                      or not workspace.is_contiguous()):
            raise ValueError(f"workspace: expected a contiguous uint8 tensor on {dev}, as new_workspace() makes it")
        if n == 0:
            return out
        s = _stream(dev)
        ws = workspace if workspace is not None else _workspace(self._L, dev, s, self.view.head_dim)
        rc = self._L.kore_cuda_paged_attn_dev(self._view, batch._view, n, self._p[0], self._p[1], plse, self._popts,
                                              ws.data_ptr(), ws.numel(), self._status, s)
        if rc:
            _ck(self._L, rc)
        return out

    def new_workspace(self):
        """A workspace for attend(): calls (or replays) that may overlap on the GPU need one each."""
        return _new_workspace(self._L, self.device, self.view.head_dim)

    def check(self) -> None:
        """Waits for the device, all of its streams; raises if a kernel met a failure in the device data since the
        last check."""
        _check_status(self.status)


def _new_workspace(L, device, head_dim: int):
    n = L.kore_cuda_paged_attn_workspace(head_dim)
    if n < 0:
        _ck(L, n)
    ws = _torch.empty(n, dtype=_torch.uint8, device=device)
    ws[:WORKSPACE_ZEROED].zero_()
    return ws


# The default workspaces: one a (device, stream), and one a capture, so that graphs captured on one stream and
# replayed on several share none. Calls on one stream follow one another, whatever their cache.
_workspaces: dict = {}
_WORKSPACES_KEPT = 16


def _workspace(L, device, stream: int, head_dim: int):
    # (torch's answer is the current device's, and quicker)
    may = _torch._C._cuda_getDevice() != device.index or _torch._C._cuda_isCurrentStreamCapturing()
    key = (device.index, stream, L.kore_cuda_capture_id(stream) if may else 0)
    ws = _workspaces.get(key)
    if ws is None:
        # the larger of the two head sizes serves both. In a capture it is the
        # graph's own memory and its zeroing a node of the graph: the graph keeps it, so
        # that those of earlier captures on the stream, which are over, need no place here
        # (other threads may change the table meanwhile: list() of it is one step)
        for old in list(_workspaces):
            if old[:2] == key[:2] and old[2] not in (0, key[2]):
                _workspaces.pop(old, None)
        ws = _new_workspace(L, device, 128)
        for old in list(_workspaces)[:1 - _WORKSPACES_KEPT]:   # the oldest beyond so many
            _workspaces.pop(old, None)
        _workspaces[key] = ws
    return ws
