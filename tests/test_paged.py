"""What the paged cache's calls refuse, which they do before anything reaches a device (no GPU needed)."""
import ctypes as C

import pytest
import torch

import cera_b200 as cb
from cera_b200._lib import PagedKvDesc, last_error, lib

BAD_ARG, UNSUPPORTED = 1, 2
A = 1 << 20  # an address on a 16-byte boundary that nothing reads


def _desc(**kw):
    d = dict(k_pages=A, v_pages=A, page_table=A, seq_lens=A, k_page_stride=16 * 2 * 64, k_slot_stride=128, k_head_stride=64, v_page_stride=16 * 2 * 64,
             v_slot_stride=128, v_head_stride=64, type=1, n_pages=9, page_size=16, n_kv_heads=2, head_dim=64, n_seqs=3, max_pages=4)
    d.update(kw)
    return C.byref(PagedKvDesc(**d))


def _decode(d=..., q=A, q_type=1, heads=8, weights=None, stride=0, out=A, ws=A, ws_bytes=1 << 30):
    return lib.cera_cuda_paged_decode_attention(_desc() if d is ... else d, q, q_type, heads, 1.0, 0, 0, weights, stride, out, ws, ws_bytes, None)


def _prefill(d=..., q=A, q_type=1, heads=8, starts=A, n=5, out=A, ws=A, ws_bytes=1 << 30):
    return lib.cera_cuda_paged_prefill_attention(_desc() if d is ... else d, q, q_type, heads, starts, n, 1.0, 0, 0, out, ws, ws_bytes, None)


def _append(d=..., k=A, v=A, t=1, starts=A, n=5, weights=None, positions=None, stride=0):
    return lib.cera_cuda_paged_append(_desc() if d is ... else d, k, v, t, starts, n, weights, positions, stride, None, None)


def _evict(d=..., w=A, p=A, stride=64, budget=8, sink=1, recent=2, wo=A, po=A, out_stride=64, kept=A, lens=A):
    return lib.cera_cuda_paged_evict(_desc() if d is ... else d, w, p, stride, budget, sink, recent, wo, po, out_stride, kept, lens, None)


@pytest.mark.parametrize("call", [_decode, _prefill, _append, _evict])
@pytest.mark.parametrize("kw,code", [
    (dict(type=2), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=48), UNSUPPORTED), (dict(head_dim=288), UNSUPPORTED),
    (dict(n_seqs=4097), UNSUPPORTED), (dict(n_kv_heads=0), BAD_ARG), (dict(page_size=0), BAD_ARG), (dict(max_pages=1 << 27), BAD_ARG),
    (dict(k_pages=None), BAD_ARG), (dict(v_pages=None), BAD_ARG), (dict(page_table=None), BAD_ARG), (dict(seq_lens=None), BAD_ARG),
    (dict(k_pages=A + 8), BAD_ARG), (dict(v_pages=A + 2), BAD_ARG), (dict(k_page_stride=100), BAD_ARG), (dict(k_slot_stride=4), BAD_ARG),
    (dict(v_head_stride=63), BAD_ARG), (dict(page_table=A + 2), BAD_ARG), (dict(seq_lens=A + 1), BAD_ARG)], ids=str)
def test_caches(call, kw, code):
    assert call(_desc(**kw)) == code
    assert call.__name__[1:] in last_error()


@pytest.mark.parametrize("call", [_decode, _prefill, _append, _evict])
def test_no_cache(call):
    assert call(C.cast(None, C.POINTER(PagedKvDesc))) == BAD_ARG


@pytest.mark.parametrize("call", [_decode, _prefill])
@pytest.mark.parametrize("kw,code", [
    (dict(heads=0), BAD_ARG), (dict(heads=7), BAD_ARG), (dict(q_type=30), UNSUPPORTED), (dict(q_type=2), UNSUPPORTED), (dict(q=None), BAD_ARG),
    (dict(out=None), BAD_ARG), (dict(q=A + 4), BAD_ARG), (dict(out=A + 8), BAD_ARG), (dict(ws=None), BAD_ARG), (dict(ws=A + 8), BAD_ARG), (dict(ws_bytes=0), BAD_ARG)], ids=str)
def test_attention(call, kw, code):
    assert call(**kw) == code
    assert last_error()


def test_the_rest():
    assert _decode(weights=A, stride=63) == BAD_ARG
    assert _prefill(starts=None) == BAD_ARG
    assert _prefill(n=1 << 30) == BAD_ARG
    assert _append(t=30) == UNSUPPORTED and _append(k=None) == BAD_ARG and _append(v=A + 8) == BAD_ARG
    assert _append(starts=None, n=4) == BAD_ARG
    assert _append(weights=A, stride=63) == BAD_ARG and _append(positions=A, stride=63) == BAD_ARG
    for kw in (dict(budget=0), dict(budget=2), dict(sink=7), dict(recent=2 ** 32 - 1), dict(stride=63), dict(out_stride=7, budget=8), dict(w=None), dict(p=None), dict(wo=None),
               dict(po=None), dict(kept=None), dict(lens=None)):
        assert _evict(**kw) == BAD_ARG, kw
    assert _evict(w=A, wo=A, p=A + 4096, po=A + 8192, stride=64, out_stride=80) == BAD_ARG  # in place, rows apart


def test_nothing_to_do_is_no_error():
    empty = _desc(n_seqs=0)
    assert _decode(empty) == 0 and _prefill(empty) == 0 and _append(empty) == 0 and _evict(empty) == 0
    assert _prefill(n=0) == 0 and _append(n=0) == 0


def test_workspaces():
    d = _desc()
    assert lib.cera_cuda_paged_decode_attention_workspace_bytes(d, 7, 0) == 0 and "7 heads" in last_error()
    assert lib.cera_cuda_paged_prefill_attention_workspace_bytes(d, 0, 5) == 0
    for weights in (0, 1):
        need = lib.cera_cuda_paged_decode_attention_workspace_bytes(d, 8, weights)
        assert need > 0 and _decode(ws_bytes=need - 1, weights=A if weights else None, stride=64) == BAD_ARG


def test_tensors_on_the_cpu_are_refused():
    k = torch.zeros(2, 16, 2, 64)
    with pytest.raises(TypeError, match="CUDA"):
        cb.PagedKv(k, k, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
