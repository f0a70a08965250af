"""What the paged cache's calls decide on the host, at the ends of their ranges (no GPU needed)."""
import pytest

from cera_b200._lib import last_error, lib
from test_paged import _desc, _prefill

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
