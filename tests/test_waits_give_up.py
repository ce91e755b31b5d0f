"""Waits of the adapter kernel end: a barrier of the four epilogue warps has no limit, so
whether a warp's own (limited) wait came through must not decide whether it reaches one."""
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCE = os.path.join(os.path.dirname(HERE), "qwen3-image21_b200", "csrc", "lora.cu")


def barriers(text):
    """(headers of the blocks around it) of every epilogue barrier in the epilogue's branch."""
    start = text.index("} else if (warp >= 4) {")
    open_blocks, found, header = [], [], start + 1
    at = start + 1
    while at < len(text):
        c = text[at]
        if c in "{};":
            if c == "{":
                open_blocks.append(text[header:at])
            elif c == "}":
                open_blocks.pop()
                if not open_blocks:
                    return found
            header = at + 1
        elif re.match(r"\bepi_(sync|all)\(", text[at:]) and not text[at - 1].isalnum():
            found.append([h.strip() for h in open_blocks])
        at += 1
    raise AssertionError("the epilogue's end was not found")


def test_no_epilogue_barrier_depends_on_a_warp_s_own_wait():
    text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    found = barriers(text)
    assert len(found) >= 3
    for blocks in found:
        for header in blocks:
            assert not re.search(r"\bok\b", header), header
