"""A step with drafted tokens over the paged cache (kore_cuda_paged_plan_dev and what follows it in kore_cuda.h): torch
tensors in place of the C structures.

A step, on the current stream of the tensors' device::

    pool = PagePool(n_pages, page_tokens, n_requests, table_width)      # once
    step, tree = pool.new_step(n_seq, n_tok, max_q), TokenTree(n_tok, max_q)   # once for each size of step
    path = AcceptedPath(n_seq, max_path)

    pool.plan(step, request, n_new)                        # pages, slots, positions; lengths grow
    tree.build(step, parent)                               # who sees whom, positions by depth
    for cache in layers:                                   # q, k, v of the layer's product
        cache.store(step.slots, tree.pos, k, v, rope=rope, norm=norm, q=q, q_out=q)
        cache.attend(step, q, out, tree=tree)
    path.accept(step, parent, token, choice, tree=tree)    # the branch that the model's choices follow
    PagedLayers(layers).commit(step, path)                 # (made once) its rows moved together
    pool.trim(request, path.kept)                          # the refused drafts' pages

The step of a prompt or of single tokens is the same without tree, path and trim. As in kore_b200/paged.py an object is
for one host thread at a time, nothing is copied or synchronised, and a failure that a kernel meets in the device data is
kept in ``status`` and raised by ``check()``.
"""
from __future__ import annotations

import ctypes

from . import paged as P
from .paged import PagedBatch, PagedCache, _ck, _int, _ints, _stream   # noqa: F401

__all__ = ["PagePool", "PagedStep", "TokenTree", "AcceptedPath", "PagedLayers", "HeadNorm"]

MAX_TREE = 1024


def _device(device):
    torch = P._import_torch()
    d = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"expected a CUDA device, got {d}")
    return torch, torch.device("cuda", torch.cuda.current_device()) if d.index is None else d


def _size(x, what: str, least: int = 1) -> int:
    if _int(x, what) < least:
        raise ValueError(f"{what} = {x} must be at least {least}")
    return x


class PagedStep(PagedBatch):
    """A batch whose arrays a plan fills (PagePool.new_step), with the slot (int64) and the position (int32) of each of
    its n_tok rows; -1 for a row of no sequence."""

    def __init__(self, n_seq: int, n_tok: int, table_width: int, max_q: int, max_kv: int, device):
        torch, dev = _device(device)
        new = lambda *shape, dtype=torch.int32: torch.full(shape, -1, dtype=dtype, device=dev)   # noqa: E731
        q_start, kv_len = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (n_seq + 1, n_seq))
        super().__init__(q_start, kv_len, new(n_seq, table_width), max_q, max_kv)
        self.slots, self.pos = new(n_tok, dtype=torch.int64), new(n_tok)
        self._step = P._Step(q_start.data_ptr(), kv_len.data_ptr(), self.page_table.data_ptr(), table_width, n_tok,
                             self.slots.data_ptr(), self.pos.data_ptr())
        self._pstep = ctypes.addressof(self._step)


class PagePool:
    """The pages of a cache (every layer's, which have the same tables) and the requests that hold them. All of it is
    on the device: free [n_pages] (the first n_free of it are the free pages), table [n_requests][table_width], length
    [n_requests]: the positions that a request holds, in its first ceil(length / page_tokens) pages."""

    def __init__(self, n_pages: int, page_tokens: int, n_requests: int, table_width: int, *, device=None):
        torch, self.device = _device(device)
        self._L = P._library()
        for x, what in ((n_pages, "n_pages"), (page_tokens, "page_tokens"), (n_requests, "n_requests"),
                        (table_width, "table_width")):
            _size(x, what)
        if page_tokens % 16 or n_requests > 65536:
            raise ValueError(f"page_tokens {page_tokens} must be a multiple of 16, n_requests {n_requests} at most 65536")
        new = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=self.device)   # noqa: E731
        self.free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=self.device)
        self.table, self.length = new(n_requests, table_width).fill_(-1), new(n_requests)
        self.view = P._Pool(self.free.data_ptr(), self.n_free.data_ptr(), self.table.data_ptr(), self.length.data_ptr(),
                            n_pages, page_tokens, n_requests, table_width)
        self._view = ctypes.addressof(self.view)
        self.status = new(1)
        self._status = self.status.data_ptr()

    def new_step(self, n_seq: int, n_tok: int, max_q: int, max_kv: int = 0) -> PagedStep:
        """Buffers for the steps of up to n_seq sequences and n_tok rows; max_q and max_kv as for PagedBatch."""
        if _size(n_seq, "n_seq", 0) > 4096:
            raise ValueError(f"n_seq = {n_seq} is more than 4096")
        return PagedStep(n_seq, _size(n_tok, "n_tok", 0), self.view.table_stride, max_q, max_kv, self.device)

    def _two(self, request, amount, what: str):
        pr, n = _ints(request, "request", self.device, 1), request.shape[0]
        return n, pr, _ints(amount, what, self.device, 1, n)

    def plan(self, step: PagedStep, request, n_new) -> None:
        """Plans n_new[s] more positions for request[s] (int32 on the device, each request once; negative: padding) into
        the step, whose sequences they are, and makes them part of the requests' lengths."""
        n, pr, pn = self._two(request, n_new, "n_new")
        if step.device != self.device or n != step.view.n_seq or step._step.table_stride < self.view.table_stride:
            raise ValueError(f"the step has {step.view.n_seq} sequences on {step.device}, the plan {n} on {self.device}"
                             if n != step.view.n_seq or step.device != self.device else
                             "the step's page table is narrower than the pool's")
        rc = self._L.kore_cuda_paged_plan_dev(self._view, n, pr, pn, step._pstep, self._status, _stream(self.device))
        if rc:
            _ck(self._L, rc)

    def trim(self, request, keep) -> None:
        """Keeps the first keep[s] positions of request[s] and gives the pages behind them back (0: the request ends)."""
        n, pr, pk = self._two(request, keep, "keep")
        rc = self._L.kore_cuda_paged_trim_dev(self._view, n, pr, pk, self._status, _stream(self.device))
        if rc:
            _ck(self._L, rc)

    def check(self) -> None:
        """Waits for the device; raises if a plan or trim met a failure in the device data since the last check."""
        P._check_status(self.status)


class HeadNorm:
    """Norms of queries and keys: each head x becomes x / sqrt(mean(x^2) + eps) * weight. Weights are [head_dim], one for
    all heads, or [heads][head_dim], in fp32, fp16 or bf16; None: those heads have no norm."""

    def __init__(self, q_weight=None, k_weight=None, *, eps: float = 1e-6):
        torch = P._import_torch()
        some = [w for w in (q_weight, k_weight) if w is not None]
        if not some:
            raise ValueError("expected weights for the queries or the keys")
        for w in some:
            if (not w.is_cuda or w.dim() not in (1, 2) or (w.numel() and w.stride(-1) != 1) or w.dtype != some[0].dtype
                    or w.device != some[0].device or w.dtype not in (torch.float32, torch.float16, torch.bfloat16)):
                raise ValueError("weights: expected CUDA tensors [head_dim] or [heads][head_dim] of one type (fp32, fp16 "
                                 "or bf16) and device, contiguous in a head")
        if not 2.0 ** -126 <= eps < 2.0 ** 128:
            raise ValueError(f"eps = {eps} must be a positive normal number in 32 bits")
        self.q_weight, self.k_weight, self.eps, self.device = q_weight, k_weight, eps, some[0].device
        self._shapes = [None if w is None else (tuple(w.shape)) for w in (q_weight, k_weight)]
        at = [None if w is None else w.data_ptr() for w in (q_weight, k_weight)]
        strides = [0 if w is None or w.dim() == 1 else w.stride(0) for w in (q_weight, k_weight)]
        self.view = P._Norm(*at, P._types[some[0].dtype], *strides, eps)
        self._view = ctypes.addressof(self.view)
        self._fits = None

    def _for(self, device, d: int, q_heads, k_heads):
        """Its structure, for rows of so many heads."""
        if self._fits != (device, d, q_heads, k_heads):
            if device != self.device:
                raise ValueError(f"the norm's weights are not on {device}")
            for shape, h, what in ((self._shapes[0], q_heads, "q"), (self._shapes[1], k_heads, "k")):
                if shape is not None and h is not None and shape not in ((d,), (h, d)):
                    raise ValueError(f"{what}_weight: expected [{d}] or [{h}][{d}], got {shape}")
            self._fits = (device, d, q_heads, k_heads)
        return self._view


class TokenTree:
    """What the tokens of a step's chunks see of each other: bit j of row t of mask (int32 [n_tok][words], 32 * words the
    longest chunk) is set where token t sees token j of its chunk; all see the context before it. build() fills it
    from parents; a mask of another kind may be written into it."""

    def __init__(self, n_tok: int, max_chunk: int, *, device=None):
        torch, self.device = _device(device)
        self._L = P._library()
        if _size(max_chunk, "max_chunk") > MAX_TREE:
            raise ValueError(f"max_chunk = {max_chunk} is more than {MAX_TREE}")
        words = -(-max_chunk // 32)
        self.mask = torch.zeros((_size(n_tok, "n_tok", 0), words), dtype=torch.int32, device=self.device)
        self.pos = torch.full((n_tok,), -1, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._mask, self._pos, self._status = self.mask.data_ptr(), self.pos.data_ptr(), self.status.data_ptr()
        self.view = P._Tree(self._mask, words)
        self._view = ctypes.addressof(self.view)

    def build(self, batch: PagedBatch, parent) -> None:
        """Masks and positions of the batch's tokens from their parents (int32 [n_tok]: the parent's index in the chunk,
        before the token's own; -1: none): a token sees its ancestors and itself, and stands at the context's
        length and its depth."""
        n = self.mask.shape[0]
        pp = _ints(parent, "parent", self.device, 1, n)
        if batch.device != self.device:
            raise ValueError(f"expected a batch on {self.device}")
        if n == 0:
            return
        rc = self._L.kore_cuda_tree_masks_dev(batch._view, n, pp, self._mask, self.view.words, self._pos, self._status,
                                              _stream(self.device))
        if rc:
            _ck(self._L, rc)

    def check(self) -> None:
        """Waits for the device; raises if a build met a failure in the device data since the last check."""
        P._check_status(self.status)


class AcceptedPath:
    """The accepted branch of each sequence: path [n_seq][max_path] (indexes in the chunk, -1 behind the last), count
    [n_seq], next_token [n_seq] (the model's choice behind the last) and kept [n_seq] (positions held with them; -1 for a
    sequence that is left out, here or by the plan, of whose pages a trim then takes none)."""

    def __init__(self, n_seq: int, max_path: int, *, device=None):
        torch, self.device = _device(device)
        self._L = P._library()
        if _size(n_seq, "n_seq", 0) > 4096 or _size(max_path, "max_path") > MAX_TREE:
            raise ValueError(f"n_seq = {n_seq} is more than 4096 or max_path = {max_path} more than {MAX_TREE}")
        self.path = torch.full((n_seq, max_path), -1, dtype=torch.int32, device=self.device)
        self.count, self.next_token, self.kept, self.status = (
            torch.zeros(n, dtype=torch.int32, device=self.device) for n in (n_seq, n_seq, n_seq, 1))
        self._status = self.status.data_ptr()
        self.view = P._Accepted(self.path.data_ptr(), max_path, self.count.data_ptr(), self.next_token.data_ptr(),
                                self.kept.data_ptr())
        self._view = ctypes.addressof(self.view)

    def accept(self, batch: PagedBatch, parent, token, choice, *, tree: TokenTree | None = None) -> None:
        """From token 0 of each chunk on, the first child whose token is the model's choice behind its parent, and so on
        (parent as for TokenTree.build, token and choice [n_tok]; all int32). tree: the step's, whose masks a chunk may be
        too long for: it is left out then, as it was by build, store and attention (without tree: of chunks beyond 1024
        tokens only)."""
        pp, n = _ints(parent, "parent", self.device, 1), parent.shape[0]
        pt, pc = _ints(token, "token", self.device, 1, n), _ints(choice, "choice", self.device, 1, n)
        if batch.device != self.device or batch.view.n_seq != self.path.shape[0]:
            raise ValueError(f"expected a batch of {self.path.shape[0]} sequences on {self.device}")
        if tree is not None and (tree.device != self.device or tree.mask.shape[0] != n):
            raise ValueError(f"tree: expected masks of {n} tokens on {self.device}")
        if batch.view.n_seq == 0:
            return
        words = tree.view.words if tree is not None else MAX_TREE // 32
        rc = self._L.kore_cuda_tree_accept_masked_dev(batch._view, n, words, pp, pt, pc, self._view, self._status,
                                                      _stream(self.device))
        if rc:
            _ck(self._L, rc)

    def check(self) -> None:
        """Waits for the device; raises if an acceptance met a failure in the device data since the last check."""
        P._check_status(self.status)


def _spans(cache):
    """Bytes of a page, from one page to the next, and from a pool's first byte to its last, of cache's geometry."""
    v, size = cache.view, cache.k.element_size()
    page = v.n_head_kv * v.page_tokens * v.head_dim * size
    stride = v.page_stride * size or page
    return page, stride, (v.n_pages - 1) * stride + page


def _overlap(apart: int, page: int, stride: int, span: int) -> bool:
    """Whether pools that begin so many bytes apart, whose pages may lie between one another's, share memory."""
    rest = apart % stride
    return apart < span and (rest < page or stride - rest < page and apart - rest + stride < span)


def _check_apart(caches) -> None:
    """Raises if two caches' pages share memory."""
    page, stride, span = _spans(caches[0])
    pools = sorted((a or 0, i) for i, c in enumerate(caches) for a in (c.view.k, c.view.v))
    for x, (a, i) in enumerate(pools):
        for y in range(x + 1, len(pools)):
            b, j = pools[y]
            if b - a >= span:   # (so are all behind it)
                break
            if i != j and _overlap(b - a, page, stride, span):
                raise ValueError(f"caches {min(i, j)} and {max(i, j)} share pages")


def _check_own(caches) -> None:
    """Raises if a cache's keys and values share memory and are not one (whose rows are moved once)."""
    for i, c in enumerate(caches):
        apart = abs((c.view.k or 0) - (c.view.v or 0))
        if apart and _overlap(apart, *_spans(c)):
            raise ValueError(f"cache {i}: the keys' pages overlap the values'")


class PagedLayers:
    """The caches of a model's layers, of one type and geometry, whose page tables are the same, each in memory of its own
    (in which its keys and values may be the same)."""

    def __init__(self, caches):
        self.caches = caches = list(caches)
        if not caches:
            raise ValueError("expected at least one cache")
        if any(c.device != caches[0].device for c in caches):
            raise ValueError("the caches are on different devices")
        _check_apart(caches)
        _check_own(caches)
        self._L, self.device = P._library(), caches[0].device
        self.views = (P._Pages * len(caches))(*[c.view for c in caches])
        self._views = ctypes.addressof(self.views)
        self.status = P._torch.zeros(1, dtype=P._torch.int32, device=self.device)
        self._status = self.status.data_ptr()

    def commit(self, batch: PagedBatch, path: AcceptedPath) -> None:
        """Moves the accepted tokens' keys and values together in every layer: from their own places in the chunk to its
        first ones. batch: as the step ran with it."""
        if batch.device != self.device or path.device != self.device or batch.view.n_seq != path.path.shape[0]:
            raise ValueError(f"expected a batch and a path of the same sequences on {self.device}")
        v = path.view
        rc = self._L.kore_cuda_paged_commit_dev(self._views, len(self.caches), batch._view, v.path, v.path_stride, v.count,
                                                self._status, _stream(self.device))
        if rc:
            _ck(self._L, rc)

    def check(self) -> None:
        """Waits for the device; raises if a move met a failure in the device data since the last check."""
        P._check_status(self.status)
