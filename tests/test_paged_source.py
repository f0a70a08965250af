"""Rules of the paged cache's kernels that no run shows: read from the sources (no GPU needed)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cera_b200", "csrc")


def _text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_a_row_that_is_computed_again_is_stored_behind_what_was_stored_first():
    """Other lanes of the warp stored to the same addresses: a vote orders no memory."""
    seen = 0
    for name in sorted(os.listdir(CSRC)):
        text = _text(name)
        for call in re.finditer(r"paged_attend_row<[^;{]*?>\(", text):
            if not name.startswith("paged"):
                continue
            seen += 1
            ahead = text[:call.start()].rstrip()
            assert "__syncwarp();" in ahead[-400:] and ahead.rindex("__syncwarp();") > max(ahead.rfind("__any_sync("), ahead.rfind("__ballot_sync(")), name
    assert seen == 3
