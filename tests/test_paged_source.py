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


def test_every_kernel_reports_in_bits_of_its_own():
    """The compiler checks that the bits lie apart; here: every reader takes its own, and no role of a kernel is outside of them."""
    table = {n: (int(a), int(c)) for n, a, c in re.findall(r"(STATUS_\w+) = \{(\d+), (\d+)\}", _text("common.cuh"))}
    bits = [b for a, c in table.values() for b in range(a, a + c)]
    assert len(set(bits)) == len(bits) and max(bits) < 32
    assert all(re.search(r"all\[\] = \{[^}]*\b%s\b" % n, _text("common.cuh")) for n in table)
    used = {}
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cu") or name == "runtime.cu" or "register_kernel_status(" not in _text(name):
            continue
        text = _text(name)
        owner, = re.findall(r"return (STATUS_\w+)\.of\(v\);", text)
        roles = [int(r) for call in re.findall(r"\b(?:mbar_wait\w*|arrived)\(([^;{]*)", text) for r in re.findall(r", (\d+)u\)", call)]
        assert roles and max(roles) < 1 << table[owner][1], (name, roles)
        assert all(r & (r - 1) == 0 for r in roles), (name, roles)
        used[owner] = name
    assert set(used) == set(table)


def test_no_number_of_sms_by_hand():
    for name in sorted(os.listdir(CSRC)):
        if name.startswith("paged"):
            assert not re.search(r"\b148\b", _text(name)), name


def test_loaders_wait_for_their_copies_before_they_leave():
    """Shared memory may not go to another CTA with a copy on its way into it: where a loader gives a wait up, and at its end too, since those who read what it loaded may give up later."""
    decode = _text("paged_decode.cu")
    decode = decode[decode.index("if (warp >= PD_WARPS) {"):decode.index("float *qs = values")]
    prompt = _text("paged_prefill_tc.cu")
    prompt = prompt[prompt.index("void pp_load("):prompt.index("void pp_multiply(")]
    for text, waits in ((decode, 1), (prompt, 2)):
        body = text[:text.rindex("drain(")]
        assert re.search(r"auto drain = .*?SPIN_LIMIT.*?mbar_test\(&full\[", text, re.S)
        given_up = re.findall(r"if \(!tma::mbar_wait_warp\([^;]*?status, \d+u\)\) return drain\(", body)
        assert len(given_up) == waits == len(re.findall(r"mbar_wait_warp\(", text))
        assert re.fullmatch(r"drain\([^;]*\);\s*(return;\s*)?\}\s*(template <[^{]*)?", text[text.rindex("drain("):]), text[text.rindex("drain("):]


def test_warpgroups_that_ask_for_registers_are_launched_with_enough():
    """setmaxnreg.inc waits until the block has that many to spare, for good if it never had: the host asks before the launch, with the numbers that the kernel has."""
    text = _text("paged_prefill_tc.cu")
    assert re.findall(r'setmaxnreg\.(inc|dec)[^"]*%0;" ::"n"\((\w+)\)', text) == [("inc", "PP_MATH_REGS"), ("dec", "PP_LOAD_REGS")] and text.count("setmaxnreg") == 2
    guard = text[text.index("int32_t pp_registers("):text.index("int32_t pp_launch(")]
    assert "numRegs + 7) / 8 * 8 * threads < (threads - 128) * PP_MATH_REGS + 128 * PP_LOAD_REGS" in guard
    launch = text[text.index("int32_t pp_launch("):]
    assert launch.index("pp_registers<") < launch.index("launch_k(")
