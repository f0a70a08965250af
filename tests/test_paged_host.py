"""What the paged cache's calls decide on the host, at the ends of their ranges (no GPU needed)."""
import pytest

from cera_b200._lib import last_error, lib
from test_paged import A, _decode, _desc, _prefill

F32, F16, BF16 = 0, 1, 30


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("head_dim", [32, 128, 256])
def test_room_for_a_prompt_of_any_length(type, head_dim):
    """No token and no sequence ask for something too; more rows than can be counted are refused."""
    wide = dict(type=type, head_dim=head_dim, k_head_stride=head_dim, v_head_stride=head_dim, k_slot_stride=2 * head_dim, v_slot_stride=2 * head_dim)
    ask = lib.cera_cuda_paged_prefill_attention_workspace_bytes
    for d in (_desc(**wide), _desc(n_seqs=0, **wide), _desc(max_pages=0, **wide), _desc(n_pages=0, **wide), _desc(max_pages=1 << 20, **wide)):
        for n in (0, 1, 2, 127, 4097, 500000):
            assert ask(d, 8, n) >= 16, n
        for n in (1 << 29, 1 << 31, 1 << 54, 1 << 63, (1 << 64) - 1):
            assert ask(d, 8, n) == 0 and "tokens" in last_error()


def test_tokens_that_cannot_be_counted_are_refused():
    for n in (1 << 29, 1 << 31, 1 << 62, (1 << 64) - 1):
        assert _prefill(n=n) == 1


def test_a_result_over_a_part_of_its_queries_is_refused():
    """It may be the queries themselves, or lie beside them."""
    for call, rows in ((_decode, 3), (_prefill, 5)):
        for q_type, size in ((1, 2), (0, 4)):
            whole = rows * 8 * 64 * size
            for off in (16, whole // 2, whole - 16, -16, 16 - whole):
                assert call(q=A, out=A + off, q_type=q_type) == 1 and "part of the queries" in last_error(), off
            for off in (0, whole, -whole):
                assert call(q=A, out=A + off, q_type=q_type, ws_bytes=0) == 1 and "workspace" in last_error(), off
