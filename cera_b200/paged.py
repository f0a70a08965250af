"""A paged key/value cache of several sequences, and the operators that read and write it: storing new rows, attention of one token per
sequence and of portions of prompts, with a sliding window and first tokens that stay visible, and eviction by accumulated attention
weight.  The reference keeps one sequence in contiguous rows (cera/src/kv_cache.rs:201-221) and has no counterpart.

Like the other operator calls these take torch CUDA tensors as device memory, launch on torch's current stream and never wait."""
import ctypes as C

import torch

from . import ops
from ._lib import PagedKvDesc, check, lib
from .types import BF16, F16, F32

_TYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _refuse(t, what, dtype, shape, index):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != index:
        raise TypeError(f"{what}: expected a tensor on cuda:{index}, where the cache is")
    if t.dtype != dtype or not t.is_contiguous():
        raise TypeError(f"{what}: expected a contiguous {dtype} tensor, got {t.dtype}")
    raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _take(t, what, dtype, shape, index):
    """The address of t, which is a contiguous tensor of that type and shape on the cache's device.  (A small call takes about as long here as on the GPU: one
    line of cheap questions, and the refusal's words apart.)"""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous()):
        _refuse(t, what, dtype, shape, index)
    return t.data_ptr()


class PagedKv:
    """The tensors of a cache, which stay the caller's: k_pages and v_pages [n_pages, page_size, n_kv_heads, head_dim] of float32, float16 or
    bfloat16 in any strides of whole 16 bytes (head_dim contiguous; keys and values may be interleaved views of one tensor),
    page_table int32 [n_seqs, max_pages] and seq_lens int32 [n_seqs].  Slot j of sequence s is row j % page_size of page
    page_table[s, j // page_size]; an entry outside [0, n_pages) is a page that is not there, whose slots are not seen.  The calls read the
    table and the lengths when they run, so both may be changed in place between calls and under a captured graph.  Sequences may share pages
    (a common beginning) that are only read; what paged_append and paged_evict write must be in pages of one sequence."""

    def __init__(self, k_pages, v_pages, page_table, seq_lens):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("page_table", page_table), ("seq_lens", seq_lens)):
            if not (isinstance(t, torch.Tensor) and t.is_cuda):
                raise TypeError(f"{name}: expected a CUDA tensor: this path has no CPU fallback")
            if t.device != k_pages.device:
                raise ValueError(f"{name} is on {t.device}, k_pages on {k_pages.device}")
        if k_pages.dtype not in _TYPE or v_pages.dtype != k_pages.dtype:
            raise TypeError(f"pages must both be float32, float16 or bfloat16, got {k_pages.dtype} and {v_pages.dtype}")
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise ValueError(f"pages are [n_pages, page_size, n_kv_heads, head_dim], got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if t.stride(3) != 1 or any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
                raise ValueError(f"{name}: head_dim must be contiguous and no row may stand for several, got strides {t.stride()}")
        if page_table.dim() != 2 or seq_lens.dim() != 1 or page_table.shape[0] != seq_lens.shape[0]:
            raise ValueError(f"page_table [n_seqs, max_pages] and seq_lens [n_seqs] do not go together: {tuple(page_table.shape)}, {tuple(seq_lens.shape)}")
        for name, t in (("page_table", page_table), ("seq_lens", seq_lens)):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise TypeError(f"{name}: expected a contiguous int32 tensor, got {t.dtype}")
        self.k_pages, self.v_pages, self.page_table, self.seq_lens = k_pages, v_pages, page_table, seq_lens
        n_pages, page_size, n_kv_heads, head_dim = k_pages.shape
        self.n_seqs, self.n_kv_heads, self.head_dim, self.page_size = seq_lens.shape[0], n_kv_heads, head_dim, page_size
        self.capacity = page_table.shape[1] * page_size  # slots of a sequence
        self.dtype, self.device, self.index = k_pages.dtype, k_pages.device, k_pages.get_device()
        # the stride of an extent of one is no stride
        ks, vs = ([st if n > 1 else 0 for n, st in zip(t.shape, t.stride())] for t in (k_pages, v_pages))
        self._desc = PagedKvDesc(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                                 _TYPE[k_pages.dtype], n_pages, page_size, n_kv_heads, head_dim, self.n_seqs, page_table.shape[1])
        self._ref = C.byref(self._desc)
        self._workspace = {}

    def _stream(self):
        """The current stream, which is one of the cache's device."""
        if ops._raw_stream and ops._device:
            if ops._device() == self.index:
                return ops._raw_stream(self.index)
        elif torch.cuda.current_device() == self.index:
            return torch.cuda.current_stream().cuda_stream
        raise ValueError(f"the cache is on {self.device}, the current device is another: make the cache's current")

    def _rows(self, t, what, n, heads):
        """Rows [n][heads][head_dim] of the cache's type or float32 (None: as many as there are)."""
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise TypeError(f"{what}: expected a tensor of three dimensions")
        shape = (t.shape[0] if n is None else n, t.shape[1] if heads is None else heads, self.head_dim)
        return _take(t, what, torch.float32 if t.dtype is torch.float32 else self.dtype, shape, self.index)

    def _track(self, t, what, dtype, least):
        """Weights or positions [n_seqs][n_kv_heads][at least `least`] -> address and slots."""
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise TypeError(f"{what}: expected a tensor of three dimensions")
        slots = t.shape[2]
        p = _take(t, what, dtype, (self.n_seqs, self.n_kv_heads, slots), self.index)
        if slots < least:
            raise ValueError(f"{what}: {slots} slots, {least} needed")
        return p, slots

    def _starts(self, starts):
        return _take(starts, "starts", torch.int32, (self.n_seqs + 1,), self.index)

    def _scratch(self, workspace, key, ask):
        need = self._workspace.get(key)
        if need is None:
            need = ask()
            if need == 0:
                raise ValueError(ops._lib.last_error())
            if len(self._workspace) > 64:  # a program whose calls differ in size
                self._workspace.clear()
            self._workspace[key] = need
        if workspace is None:
            return torch.empty(need, dtype=torch.uint8, device=self.device)
        _take(workspace, "workspace", torch.uint8, (workspace.numel(),) if isinstance(workspace, torch.Tensor) else (), self.index)
        if workspace.shape[0] < need:
            raise ValueError(f"workspace: {workspace.shape[0]} bytes, {need} needed")
        return workspace


def _visible(window, n_sink):
    if not (0 <= window < 2**32 and 0 <= n_sink < 2**32):
        raise ValueError(f"window {window} and n_sink {n_sink}: counts of slots")


def paged_append(cache, k, v, starts=None, weights=None, positions=None, token_positions=None):
    """Stores new tokens' keys and values, [n_tokens, n_kv_heads, head_dim] of the cache's type or float32 (rounded), in slots that
    seq_lens already counts: sequence s's tokens [starts[s], starts[s + 1]) - int32 [n_seqs + 1]; None: one token each - go to its last slots.
    Per slot and head, [n_seqs, n_kv_heads, at least capacity]: weights (float32) becomes 0, positions (int32) the token's position out of
    token_positions, int32 [n_tokens] (None: its slot)."""
    stream = cache._stream()
    kp = cache._rows(k, "k", None, cache.n_kv_heads)
    n = k.shape[0]
    vp = _take(v, "v", k.dtype, (n, cache.n_kv_heads, cache.head_dim), cache.index)
    wp = pp = tp = None
    stride = 0
    if weights is not None:
        wp, stride = cache._track(weights, "weights", torch.float32, cache.capacity)
    if positions is not None:
        pp, slots = cache._track(positions, "positions", torch.int32, cache.capacity)
        if weights is not None and slots != stride:
            raise ValueError("weights and positions differ in their slots")
        stride = slots
    if token_positions is not None:
        tp = _take(token_positions, "token_positions", torch.int32, (n,), cache.index)
    check(lib.cera_cuda_paged_append(cache._ref, kp, vp, _TYPE[k.dtype], None if starts is None else cache._starts(starts), n, wp, pp, stride, tp, stream))


def paged_decode_attention(cache, q, scale, window=0, n_sink=0, weights=None, out=None, workspace=None):
    """Attention of every sequence's newest token, which is in its last slot: q [n_seqs, n_heads, head_dim] of the cache's type or float32;
    the result is of q's type.  window: only that many last slots are seen, and the first n_sink (0: all).  weights, float32
    [n_seqs, n_kv_heads, at least capacity], has the probabilities of a KV head's query heads added to their slots.  A sequence
    without slots gives zeros.  `out` may be q.  Calls that may overlap need a workspace each; by default every call has its own."""
    stream, ref = cache._stream(), cache._ref
    qp = cache._rows(q, "q", cache.n_seqs, None)
    _visible(window, n_sink)
    heads, stride, wp = q.shape[1], 0, None
    if weights is not None:
        wp, stride = cache._track(weights, "weights", torch.float32, cache.capacity)
    if out is None:
        out = torch.empty_like(q)
    else:
        _take(out, "out", q.dtype, q.shape, cache.index)
    ws = cache._scratch(workspace, (heads, wp is not None), lambda: lib.cera_cuda_paged_decode_attention_workspace_bytes(ref, heads, int(wp is not None)))
    check(lib.cera_cuda_paged_decode_attention(ref, qp, _TYPE[q.dtype], heads, scale, window, n_sink, wp, stride, out.data_ptr(), ws.data_ptr(), ws.shape[0], stream))
    return out


def paged_prefill_attention(cache, q, starts, scale, window=0, n_sink=0, out=None, workspace=None):
    """Causal attention of portions of prompts: q [n_tokens, n_heads, head_dim], of which sequence s has [starts[s], starts[s + 1])
    (int32 [n_seqs + 1], ascending from 0) in its last slots.  Types, window and n_sink as in paged_decode_attention, the window counted
    back from each query; `out` may be q.  Rows past starts[n_seqs] are left as they are in `out`, and undefined without one."""
    stream, ref = cache._stream(), cache._ref
    qp, sp = cache._rows(q, "q", None, None), cache._starts(starts)
    _visible(window, n_sink)
    n, heads = q.shape[0], q.shape[1]
    if out is None:
        out = torch.empty_like(q)
    else:
        _take(out, "out", q.dtype, q.shape, cache.index)
    ws = cache._scratch(workspace, (n, heads, None), lambda: lib.cera_cuda_paged_prefill_attention_workspace_bytes(ref, heads, n))
    check(lib.cera_cuda_paged_prefill_attention(ref, qp, _TYPE[q.dtype], heads, sp, n, scale, window, n_sink, out.data_ptr(), ws.data_ptr(), ws.shape[0], stream))
    return out


def paged_evict(cache, weights, positions, budget, n_sink=0, n_recent=0, weights_out=None, positions_out=None, seq_lens_out=None):
    """Cuts every sequence and KV head down to `budget` slots -> (kept, seq_lens).  Kept are the slots with a position below n_sink or
    among the n_recent latest (newest position - n_recent < position), then those of the largest weight (a NaN is the smallest), ties
    to the lower slot.  What is kept past the budget moves, pages included, into the gaps below it, so slots lose their order: attend without
    a window afterwards.  Slots are picked whether their pages are there or not, and only rows that are there move: a cache that is evicted from should have
    all its pages.  weights (float32) and positions (int32), [n_seqs, n_kv_heads, at least capacity], follow in place or into
    weights_out and positions_out (at least min(budget, capacity) slots).  kept, int32 [n_seqs, n_kv_heads, budget]: the slot that each slot's
    content came from, -1 past the length; seq_lens: min(length, budget) in a new tensor or in seq_lens_out, which may be
    cache.seq_lens.  Pages past the budget are the caller's again."""
    stream = cache._stream()
    _visible(n_recent, n_sink)
    if not n_sink + n_recent <= budget < 2**31 - 256 or budget < 1:
        raise ValueError(f"a budget of {budget} slots for {n_sink} first and {n_recent} recent ones")
    wp, slots = cache._track(weights, "weights", torch.float32, cache.capacity)
    pp, also = cache._track(positions, "positions", torch.int32, cache.capacity)
    least = min(budget, cache.capacity)
    wo, slots_out = (wp, slots) if weights_out is None else cache._track(weights_out, "weights_out", torch.float32, least)
    po, also_out = (pp, also) if positions_out is None else cache._track(positions_out, "positions_out", torch.int32, least)
    if slots != also or slots_out != also_out:
        raise ValueError("weights and positions differ in their slots")
    kept = torch.empty((cache.n_seqs, cache.n_kv_heads, budget), dtype=torch.int32, device=cache.device)
    if seq_lens_out is None:
        seq_lens_out = torch.empty_like(cache.seq_lens)
    else:
        _take(seq_lens_out, "seq_lens_out", torch.int32, (cache.n_seqs,), cache.index)
    check(lib.cera_cuda_paged_evict(cache._ref, wp, pp, slots, budget, n_sink, n_recent, wo, po, slots_out, kept.data_ptr(), seq_lens_out.data_ptr(), stream))
    return kept, seq_lens_out
